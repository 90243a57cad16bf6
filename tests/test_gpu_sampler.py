"""GPU tests of GpuSampler: sampling and the best log-probabilities against the
plain restatements of _serving.py (equal tokens and indices; log-probabilities
within the bound derived there), at the sizes, alignments, masks and ties
where a row kernel can go wrong."""
import math

import numpy as np
import pytest

import _serving as ref

pytestmark = pytest.mark.gpu

DT = ["f32", "f16", "bf16"]


@pytest.fixture(scope="module", params=[1, 2], ids=["cluster", "solo"])
def gs(request):
    """Every form for every case: a cluster a row, and a CTA of 512 or 1024 threads a row."""
    import forge_sort
    with pytest.MonkeyPatch.context() as mp:
        mp.setenv("FORGESORT_ROW_FORM", str(request.param))
        s = forge_sort.GpuSampler.new()
    yield s
    s.close()


def _dtype(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _peaked(rows, cols, dtype, seed):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device="cuda") * 2
    lift = torch.empty(rows, cols, device="cuda").exponential_(0.4, generator=g)
    x = torch.where(torch.rand(rows, cols, generator=g, device="cuda") < 0.01, x + lift, x)
    return x.to(_dtype(dtype))


def _uniform(rows, seed):
    import torch
    return torch.rand(rows, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def _check(gs, x, u, temperature=None, top_k=None, top_p=None, min_p=None):
    import torch
    R = x.shape[0]
    dev = lambda v, dt: None if v is None else torch.as_tensor(v, dtype=dt, device="cuda").expand(R).contiguous()  # noqa: E731
    tok, lp = gs.sample(x, u, temperature=dev(temperature, torch.float32), top_k=dev(top_k, torch.int32),
                        top_p=dev(top_p, torch.float32), min_p=dev(min_p, torch.float32), sync=True)
    per = lambda v, off: np.broadcast_to(np.asarray(off if v is None else v), (R,))  # noqa: E731
    T, k, p, m = per(temperature, 1.0), per(top_k, 0), per(top_p, 1.0), per(min_p, 0.0)
    want = [ref.sample(x[r], float(u[r]), float(T[r]), int(k[r]), float(p[r]), float(m[r])) for r in range(R)]
    assert tok.tolist() == [w[0] for w in want]
    a, r = ref.logprob_bound(x.shape[1])
    for got, (_, w) in zip(lp.tolist(), want):
        assert got == w if math.isinf(w) else abs(got - w) <= a + r * abs(w)
    return tok, lp


PARAMS = {
    "plain": {},
    "hot": dict(temperature=1.7),
    "cold": dict(temperature=0.05),
    "greedy": dict(temperature=0.0),
    "top_k": dict(top_k=50, temperature=0.9),
    "top_1": dict(top_k=1),
    "top_p": dict(top_p=0.9, temperature=0.8),
    "all": dict(temperature=1.1, top_k=64, top_p=0.95, min_p=0.02),
}


@pytest.mark.parametrize("cols", [1, 2, 3, 7, 8, 9, 31, 33, 100, 255, 1000, 4097, 20011])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("params", sorted(PARAMS))
def test_sizes(gs, cols, dtype, params):
    x = _peaked(5, cols, dtype, cols)
    _check(gs, x, _uniform(5, cols + 1), **PARAMS[params])


@pytest.mark.parametrize("rows,cols", [(1, 131072), (3, 50021), (2, 262144), (1, 1 << 19), (40, 65537)])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("params", ["plain", "top_p", "all", "greedy"])
def test_large(gs, rows, cols, dtype, params):
    _check(gs, _peaked(rows, cols, dtype, 7), _uniform(rows, 8), **PARAMS[params])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("top_k", [1, 2, 31, 500, 1500, 2047, 2048, 2049, 5000, 30000, 40000])
def test_top_k_range(gs, dtype, top_k):
    x = _peaked(3, 30011, dtype, top_k)
    _check(gs, x, _uniform(3, 3), top_k=top_k)
    _check(gs, x, _uniform(3, 4), top_k=top_k, top_p=0.7, temperature=1.3)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("top_p", [-1.0, 0.0, 1e-6, 0.3, 0.5, 0.9, 0.99, 0.9999, 0.99999994, 1.0, 2.0])
@pytest.mark.parametrize("temperature", [0.7, 3.0])
def test_top_p_range(gs, dtype, top_p, temperature):
    """At temperature 3 the nucleus holds most of the row."""
    _check(gs, _peaked(3, 40009, dtype, 11), _uniform(3, 5), top_p=top_p, temperature=temperature)


@pytest.mark.parametrize("min_p", [-1.0, 0.0, 1e-9, 0.01, 0.5, 1.0, 3.0])
def test_min_p_range(gs, min_p):
    for t in (0.6, 2.5):
        _check(gs, _peaked(4, 9001, "f32", 5), _uniform(4, 6), min_p=min_p, temperature=t)
        _check(gs, _peaked(4, 9001, "f32", 5), _uniform(4, 6), min_p=min_p, temperature=t, top_k=300, top_p=0.9)


@pytest.mark.parametrize("temperature", [float("nan"), -1.0, 1e-30, 1e-45, 1e30, float("inf")])
def test_odd_temperatures(gs, temperature):
    _check(gs, _peaked(3, 5003, "f32", 2), _uniform(3, 2), temperature=temperature, top_p=0.9)
    _check(gs, _peaked(3, 5003, "f32", 2), _uniform(3, 2), temperature=temperature)


def _masks(dtype):
    """name -> a row of 6007 logits."""
    import torch
    dt, n = _dtype(dtype), 6007
    low, inf = torch.finfo(dt).min, math.inf
    base = _peaked(1, n, dtype, 31)[0]
    full = lambda v: torch.full((n,), v, dtype=dt, device="cuda")  # noqa: E731

    def put(x, at, v):
        x = x.clone()
        x[at] = v
        return x

    every_other = torch.arange(n, device="cuda") % 2 == 0
    return {
        "nothing": full(-inf), "nan only": full(math.nan), "one left": put(full(-inf), n - 1, 0.5),
        "first left": put(full(-inf), 0, -3.0), "lowest everywhere": full(low), "lowest but one": put(full(low), 17, low / 2),
        "equal": full(1.25), "zeros of both signs": torch.where(every_other, full(0.0), full(-0.0)),
        "two values": torch.where(every_other, full(1.0), full(0.0)), "half masked": torch.where(every_other, base, full(-inf)),
        "half lowest": torch.where(every_other, base, full(low)), "a nan": put(base, 5, math.nan),
        "a plus infinity": put(base, 4000, inf), "plus infinities": put(put(base, 3, inf), 5000, inf),
        "infinity and lowest": put(put(full(low), 9, inf), 10, -inf), "largest everywhere": full(torch.finfo(dt).max),
        "tiny": (base.float() * 1e-6).to(dt), "negative": -base.abs() - 1,
    }


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("params", ["plain", "greedy", "top_k", "top_1", "top_p", "all"])
def test_masks_and_ties(gs, dtype, params):
    import torch
    rows = list(_masks(dtype).values())
    x = torch.stack(rows)
    for seed in (1, 2):
        _check(gs, x, _uniform(len(rows), seed), **PARAMS[params])
    _check(gs, x, _uniform(len(rows), 3), top_k=2500, top_p=0.5)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("step", [0.25, 0.0625, 3.0])
@pytest.mark.parametrize("params", [dict(top_p=0.5), dict(top_p=0.97, min_p=0.01), dict(top_k=9000), dict(top_k=30000, top_p=0.8)],
                         ids=["top_p", "top_p min_p", "top_k", "top_k top_p"])
def test_wide_cuts_end_among_equal_values(gs, dtype, step, params):
    """Logits of few values: a cut that lies far down ends inside hundreds to
    thousands of equal ones, of either sign, and is told by the index alone."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(11)
    x = torch.round(torch.randn(3, 70001, generator=g, device="cuda") * 1.5 / step) * step
    x[1] -= 7.0
    x[2] += 7.0
    x = x.to(getattr(torch, {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}[dtype]) if isinstance(dtype, str) else dtype)
    for seed in (1, 2):
        _check(gs, x, _uniform(3, seed), temperature=1.3, **params)


def test_draw_ends(gs):
    """u at 0, just below 1, and outside [0, 1)."""
    import torch
    x = _peaked(1, 3001, "f32", 3).expand(6, -1)
    u = torch.tensor([0.0, 1 - 2.0**-24, 1.0, 5.0, -1.0, 2.0**-149], device="cuda")
    _check(gs, x, u)
    _check(gs, x, u, top_k=7)
    _check(gs, x, u, top_p=0.8, temperature=2.0)


@pytest.mark.parametrize("params", ["plain", "top_k", "all"])
def test_draw_sweep(gs, params):
    """One row drawn at 1000 numbers: the whole inverse of its distribution."""
    import torch
    x = _peaked(1, 509, "f32", 13).expand(1000, -1)
    _check(gs, x, (torch.arange(1000, device="cuda") + 0.5) / 1000, **PARAMS[params])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("offset", [0, 1, 3, 5])
@pytest.mark.parametrize("gap", [0, 1, 6])
def test_strides_and_alignment(gs, dtype, offset, gap):
    """Rows that begin anywhere, with NaN and infinities between them."""
    import torch
    rows, cols = 4, 2003
    flat = torch.full((rows * (cols + gap) + 16,), math.nan, dtype=_dtype(dtype), device="cuda")
    flat[::3] = math.inf
    x = flat[offset:offset + rows * (cols + gap)].view(rows, cols + gap)[:, :cols] if gap else \
        flat[offset:offset + rows * cols].view(rows, cols)
    x.copy_(_peaked(rows, cols, dtype, offset))
    for params in ("plain", "all", "greedy"):
        _check(gs, x, _uniform(rows, offset), **PARAMS[params])


def test_rows_apart_by_more_than_32_bits(gs):
    import torch
    step = (1 << 32) + 8
    flat = torch.empty(step + 5000, dtype=torch.bfloat16, device="cuda")
    x = flat.as_strided((2, 4999), (step, 1))
    x.copy_(_peaked(2, 4999, "bf16", 1))
    _check(gs, x, _uniform(2, 1), **PARAMS["all"])
    idx, lp, lse = gs.top_logprobs(x, 9, sync=True)
    assert idx[1].tolist() == ref.best(x[1], 9)[0].tolist()


def test_reversed_and_broadcast_rows(gs):
    import torch
    x = _peaked(1, 700, "f32", 4)
    tok, _ = gs.sample(x.expand(50, -1), _uniform(50, 1), top_k=20, sync=True)
    assert tok.tolist() == [ref.sample(x[0], float(v), top_k=20)[0] for v in _uniform(50, 1)]
    with pytest.raises(ValueError):  # a row with a step
        gs.sample(torch.zeros(8, 16, device="cuda").t(), torch.zeros(16, device="cuda"))


@pytest.mark.parametrize("dtype", DT)
def test_equal_inputs_give_equal_tokens_in_any_batch(gs, dtype):
    """A row alone, in a small batch and in a large one: other cluster sizes,
    the same bits."""
    import torch
    x, u = _peaked(64, 33001, dtype, 6), _uniform(64, 6)
    for kw in (dict(temperature=0.9), dict(top_p=0.95, temperature=2.0), dict(top_k=40, top_p=0.9)):
        tok, lp = gs.sample(x, u, sync=True, **kw)
        big_tok, big_lp = gs.sample(x.repeat(8, 1), u.repeat(8), sync=True, **kw)
        assert torch.equal(big_tok, tok.repeat(8)) and torch.equal(big_lp, lp.repeat(8))
        for r in (0, 31, 63):
            t1, l1 = gs.sample(x[r:r + 1], u[r:r + 1], sync=True, **kw)
            assert t1[0] == tok[r] and l1[0] == lp[r]


def test_mixed_batch(gs):
    R = 48
    rng = np.random.default_rng(5)
    _check(gs, _peaked(R, 17003, "bf16", 9), _uniform(R, 9), temperature=rng.choice([0.0, 0.5, 1.0, 1.5], R),
           top_k=rng.choice([0, 1, 20, 400, 3000], R), top_p=rng.choice([0.2, 0.9, 0.999, 1.0], R),
           min_p=rng.choice([0.0, 0.05, 0.3], R))


# -- the best log-probabilities --------------------------------------------------------
def _check_best(gs, x, n):
    idx, lp, lse = gs.top_logprobs(x, n, sync=True)
    a, r = ref.logprob_bound(x.shape[1])
    for k in range(x.shape[0]):
        wi, wl, ws = ref.best(x[k], n)
        assert idx[k].tolist() == wi.tolist()
        got = lp[k].double().cpu().numpy()
        fin = np.isfinite(wl)
        assert np.array_equal(fin, np.isfinite(got)) and (got[~fin] == -np.inf).all()
        assert (np.abs(got[fin] - wl[fin]) <= a + r * np.abs(wl[fin])).all()
        s = float(lse[k])
        assert s == ws if math.isinf(ws) else abs(s - ws) <= a + r * abs(ws)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("cols", [1, 2, 5, 8, 9, 33, 1000, 8191, 50021])
@pytest.mark.parametrize("n", [1, 2, 5, 20, 33, 128])
def test_best_sizes(gs, dtype, cols, n):
    _check_best(gs, _peaked(4, cols, dtype, cols), n)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n", [500, 777, 1023, 1024])
def test_best_many(gs, dtype, n):
    _check_best(gs, _peaked(3, 30011, dtype, n), n)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n", [1, 6, 100, 1024])
def test_best_masks_and_ties(gs, dtype, n):
    import torch
    _check_best(gs, torch.stack(list(_masks(dtype).values())), n)


def test_best_large(gs):
    _check_best(gs, _peaked(2, 1 << 19, "f32", 1), 50)
    _check_best(gs, _peaked(300, 2001, "bf16", 1), 3)
    _check_best(gs, _peaked(33, 131072, "bf16", 1), 20)


# -- streams, graphs, refusals ------------------------------------------------------------
def test_streams(gs):
    """Calls follow torch's current stream, where their inputs were made."""
    import forge_sort
    import torch
    x, u = _peaked(64, 50021, "f32", 3), _uniform(64, 3)
    want, _ = gs.sample(x, u, top_p=0.9, sync=True)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        z = torch.empty_like(x)
        torch.cuda._sleep(20_000_000)
        z.copy_(x)
        got, _ = gs.sample(z, u, top_p=0.9)
    gs.synchronize()
    assert torch.equal(got, want)
    own = forge_sort.GpuSampler.with_context(0, st)
    with torch.cuda.stream(st):
        torch.cuda._sleep(20_000_000)
        z.copy_(x)
    got, _ = own.sample(z, u, top_p=0.9, sync=True)
    assert torch.equal(got, want)
    own.close()


def test_numbers_on_a_stream_of_its_own(gs):
    """Numbers for all rows are spread on the sampler's stream, not on torch's
    current one, which is busy here."""
    import forge_sort
    import torch
    x, u = _peaked(64, 50021, "f32", 3), _uniform(64, 3)
    want, _ = gs.sample(x, u, temperature=0.7, top_k=40, top_p=0.9, min_p=0.01, sync=True)
    torch.cuda.synchronize()
    for st in (torch.cuda.Stream(), torch.cuda.default_stream()):
        own = forge_sort.GpuSampler.with_context(0, st)
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda._sleep(20_000_000)
            got, _ = own.sample(x, u, temperature=0.7, top_k=40, top_p=0.9, min_p=0.01, sync=True)
            assert torch.equal(got.cpu(), want.cpu())
        own.close()


def test_graph(gs):
    import torch
    x, u = _peaked(8, 30011, "bf16", 3), _uniform(8, 3)
    tok, lp = torch.empty(8, dtype=torch.int32, device="cuda"), torch.empty(8, device="cuda")
    k = torch.full((8,), 30, dtype=torch.int32, device="cuda")
    gs.sample(x, u, top_k=k, tokens=tok, logprobs=lp, sync=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gs.sample(x, u, top_k=k, tokens=tok, logprobs=lp)
    x.copy_(_peaked(8, 30011, "bf16", 44))
    tok.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert tok.tolist() == [ref.sample(x[r], float(u[r]), top_k=30)[0] for r in range(8)]


def test_numbers_for_all_rows(gs):
    import torch
    x, u = _peaked(9, 1001, "f32", 3), _uniform(9, 3)
    a = gs.sample(x, u, temperature=0.7, top_k=11, top_p=0.9, min_p=0.01, sync=True)
    full = lambda v, dt: torch.full((9,), v, dtype=dt, device="cuda")  # noqa: E731
    b = gs.sample(x, u, temperature=full(0.7, torch.float32), top_k=full(11, torch.int32),
                  top_p=full(0.9, torch.float32), min_p=full(0.01, torch.float32), sync=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_empty_batch(gs):
    import torch
    tok, lp = gs.sample(torch.empty(0, 100, device="cuda"), torch.empty(0, device="cuda"), sync=True)
    assert tok.shape == (0,) and lp.shape == (0,)
    idx, _, _ = gs.top_logprobs(torch.empty(0, 100, device="cuda"), 4, sync=True)
    assert idx.shape == (0, 4)


def test_refusals(gs):
    import torch
    x, u = torch.zeros(2, 64, device="cuda"), torch.zeros(2, device="cuda")
    for bad in (x.double(), x.int(), [[0.0]], x.cpu().numpy()):
        with pytest.raises(TypeError):
            gs.sample(bad, u)
    for bad in (x[0], x.cpu(), torch.zeros(2, 0, device="cuda"), torch.zeros(1, (1 << 19) + 1, device="cuda").expand(2, -1)):
        with pytest.raises(ValueError):
            gs.sample(bad, u)
    with pytest.raises(ValueError):
        gs.sample(x, u[:1])
    with pytest.raises(TypeError):
        gs.sample(x, u.double())
    with pytest.raises(ValueError):
        gs.sample(x, u, top_k=torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(TypeError):
        gs.sample(x, u, top_k=torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(TypeError):
        gs.sample(x, u, temperature="hot")
    with pytest.raises(ValueError):
        gs.sample(x, torch.zeros(4, device="cuda")[::2])
    with pytest.raises(TypeError):
        gs.sample(x, u, tokens=torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        gs.sample(x, u, tokens=torch.zeros(3, dtype=torch.int32, device="cuda"))
    for n in (0, -1, 1025):
        with pytest.raises((ValueError, RuntimeError)):
            gs.top_logprobs(x, n)


def test_c_refusals(gs):
    """The C entries' own checks, with the text of each."""
    import torch
    from forge_sort import _lib
    L, h = _lib.load(), gs._s._h
    x, u = torch.zeros(4, 64, device="cuda"), torch.zeros(4, device="cuda")
    tok = torch.zeros(4, dtype=torch.int32, device="cuda")
    host = torch.zeros(4, 64)

    def call(dtype=0, p=x.data_ptr(), rows=4, cols=64, stride=64, uni=u.data_ptr(), out=tok.data_ptr(), hh=h):
        return L.fs_sample_rows(hh, dtype, p, rows, cols, stride, None, None, None, None, uni, out, None, 1, None)

    assert call() == _lib.OK
    assert call(rows=0, p=None) == _lib.OK
    for kw, text in [(dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(p=None), "NULL"), (dict(cols=0), "cols"),
                     (dict(cols=(1 << 19) + 1), "cols"), (dict(stride=-64), "stride"), (dict(rows=1 << 27), "rows"),
                     (dict(p=x.data_ptr() + 2), "aligned"), (dict(uni=None), "NULL"), (dict(out=None), "NULL"),
                     (dict(p=host.data_ptr()), "logits")]:
        assert call(**kw) == _lib.E_INVALID
        assert text in L.fs_last_error(h).decode()
    assert call(hh=None) == _lib.E_INVALID
