"""GPU tests of GpuSampler where a cut or a batch is at its edge, against the
plain restatements of _serving.py: equal tokens, into outputs that hold
something else before.  Every test runs in the default form, which goes by the
batch's size, and in each form by itself."""
import functools

import numpy as np
import pytest

import _serving as ref
from test_gpu_sampler import _check, _check_best, _peaked, _uniform

pytestmark = pytest.mark.gpu

DT = ["f32", "f16", "bf16"]


@pytest.fixture(scope="module", params=[0, 1, 2], ids=["by size", "cluster", "solo"])
def gs(request):
    import forge_sort
    with pytest.MonkeyPatch.context() as mp:
        mp.setenv("FORGESORT_ROW_FORM", str(request.param))
        s = forge_sort.GpuSampler.new()
    yield s
    s.close()


def _dtype(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _sample(gs, x, u, **params):
    """Tokens of gs.sample as a list; params: numbers, or a list of one for each row."""
    import torch
    R = x.shape[0]
    dev = lambda v, dt: torch.as_tensor(v, dtype=dt, device="cuda").expand(R).contiguous()  # noqa: E731
    kw = {k: dev(v, torch.int32 if k == "top_k" else torch.float32) for k, v in params.items()}
    tok = torch.full((R,), -7, dtype=torch.int32, device="cuda")
    lp = torch.full((R,), 7.0, device="cuda")
    gs.sample(x, dev(u, torch.float32), tokens=tok, logprobs=lp, sync=True, **kw)
    assert int((tok == -7).sum()) == 0 and float(lp.max()) < 1e-6  # the logarithm of a sum's rounding may pass 0
    return tok.tolist()


def _draws(kept, spots):
    """Numbers u that put the draw at the given shares of the kept mass of all
    entries but the last, and the tokens that they give."""
    run = np.cumsum(kept)
    total, tail = int(run[-1]), int(run[-2])
    us = [np.float32(min(s * tail / total, 1 - 2.0**-24)) for s in spots] + [np.float32(0.5)]
    at = [min(int(np.floor(float(u) * float(total))), total - 1) for u in us]
    return us, [int(np.searchsorted(run, t, side="right")) for t in at]


def _tail(kind, n, rng):
    if kind == "flat":
        return np.zeros(n)
    if kind == "two values":
        return rng.integers(0, 2, n) * -3.0
    return rng.standard_normal(n) * {"narrow": 0.5, "wide": 3.0}[kind]


@functools.lru_cache(maxsize=None)
def _close_cuts(dtype, heavy, share, top_k, V=20011):
    """Four rows, and for each draw its row, top_p, number and token."""
    import torch
    rng = np.random.default_rng(int(share * 1e6) + heavy)
    rows, of, ps, us, want = [], [], [], [], []
    for kind in ("flat", "two values", "narrow", "wide"):
        z = _tail(kind, V - heavy, rng)
        z += np.log((1 - share) / share) - np.log(np.exp(z).sum())
        # the heavy ones last, so that small numbers u draw from the tail
        row = torch.from_numpy(np.concatenate([z, np.full(heavy, -np.log(heavy))]).astype(np.float32)).to(_dtype(dtype)).cuda()
        x = ref.clean(row)
        _, w = ref.weights(x, 1.0, row.device)
        q = ref.kept(x, w, top_k=top_k)
        least = q[-heavy:].sum() / q.sum()
        for by in (-1e-5, 0.0, 1e-7, 1e-6, 1e-5, 3e-5, 1e-4, 1e-3, 1e-2):
            p = float(np.float32(least * (1 + by)))
            if not 0 < p < 1:
                continue
            k = ref.kept(x, w, top_k=top_k, top_p=p)
            k = np.concatenate([k[:-heavy], [k[-heavy:].sum()]])
            for u, t in zip(*_draws(k, (0.3, 0.9999))):
                of.append(len(rows)), ps.append(p), us.append(u), want.append(t)
        rows.append(row)
    return torch.stack(rows), of, ps, np.array(us), want


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("heavy", [1, 3])
@pytest.mark.parametrize("share", [0.5, 0.99, 0.999, 0.99999])
@pytest.mark.parametrize("top_k", [0, 12000])
def test_a_nucleus_that_ends_close_behind_its_heaviest_entries(gs, dtype, heavy, share, top_k):
    """`heavy` equal entries hold `share` of the mass, and p asks for that much
    and a little more, or less: where the nucleus ends among thousands of light
    entries, no estimate of the heavy ones tells where."""
    rows, of, ps, us, want = _close_cuts(dtype, heavy, share, top_k)
    got = _sample(gs, rows[of], us, top_p=ps, top_k=top_k)
    assert [min(t, rows.shape[1] - heavy) for t in got] == want


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("cols,share,p,spread", [(32000, 0.99997, 0.99999, 0.5), (131072, 0.99997, 0.99999, 2.0),
                                                 (131072, 0.99999, 0.999999, 1.0), (131072, 0.999001, 0.999011, 0.5),
                                                 (4096, 0.9900991, 0.990109, 0.0), (131072, 0.9900991, 0.990109, 0.0)])
def test_confident_rows_with_top_p_close_to_one(gs, dtype, cols, share, p, spread):
    import torch
    rng = np.random.default_rng(cols)
    z = rng.standard_normal(cols - 1) * spread
    z += np.log((1 - share) / share) - np.log(np.exp(z).sum())
    row = torch.from_numpy(np.concatenate([z, [0.0]]).astype(np.float32)).to(_dtype(dtype)).cuda()
    x = ref.clean(row)
    _, w = ref.weights(x, 1.0, row.device)
    us, want = _draws(ref.kept(x, w, top_p=p), (0.001, 0.5, 0.99999))
    assert _sample(gs, row.expand(len(us), -1), np.array(us), top_p=p) == want


@pytest.mark.parametrize("params", [dict(top_p=float("nan")), dict(min_p=float("nan")), dict(top_k=40, top_p=float("nan"), min_p=float("nan")),
                                    dict(top_p=0.8, min_p=float("nan"), temperature=1.5)], ids=["top_p", "min_p", "top_k", "top_p min_p"])
def test_a_parameter_of_nan_is_off(gs, params):
    import math
    import torch
    x = torch.randn(64, 5003, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") * 2
    u = torch.rand(64, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").tolist()
    off = {k: v for k, v in params.items() if not math.isnan(v)}
    assert _sample(gs, x, u, **params) == [ref.sample(x[r], u[r], **off)[0] for r in range(64)]


def test_a_number_of_nan_draws_the_first_kept(gs):
    import torch
    x = torch.randn(4, 5003, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    for kw in ({}, dict(top_k=9), dict(top_p=0.9)):
        assert _sample(gs, x, [float("nan")] * 4, **kw) == [ref.sample(x[r], 0.0, **kw)[0] for r in range(4)]


@pytest.fixture()
def managed():
    """f(numpy array) -> address of a copy in managed memory."""
    import ctypes
    import torch
    rt = ctypes.CDLL("libcudart.so.12")  # torch has loaded it
    held = []

    def put(a):
        p = ctypes.c_void_p()
        assert rt.cudaMallocManaged(ctypes.byref(p), ctypes.c_size_t(a.nbytes), ctypes.c_uint(1)) == 0
        held.append(p)
        ctypes.memmove(p, a.ctypes.data, a.nbytes)
        return p.value

    torch.zeros(1, device="cuda")
    yield put
    torch.cuda.synchronize()
    for p in held:
        rt.cudaFree(p)


@pytest.mark.parametrize("sorters", ["own", "legacy"])
def test_managed_logits(managed, sorters):
    """Logits in managed memory, on a stream other than the sorter's: at once and under a capture."""
    import torch
    import forge_sort
    from forge_sort import _lib
    L = _lib.load()
    s = forge_sort.GpuSorter(0, None if sorters == "own" else torch.cuda.default_stream())
    x = (np.random.default_rng(3).standard_normal((4, 70001)) * 2).astype(np.float32)
    u = np.array([0.1, 0.5, 0.9, 0.99], np.float32)
    want = [ref.sample(torch.from_numpy(x[r]).cuda(), float(u[r]))[0] for r in range(4)]
    at, au = managed(x), managed(u)
    tok = torch.full((4,), -7, dtype=torch.int32, device="cuda")
    call = lambda: L.fs_sample_rows(s._h, 0, at, 4, 70001, 70001, None, None, None, None, au, tok.data_ptr(), None, 0,  # noqa: E731
                                    torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        assert call() == _lib.OK
    torch.cuda.synchronize()
    assert tok.tolist() == want
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rc = call()
    assert rc == _lib.OK
    tok.fill_(-7)
    g.replay()
    torch.cuda.synchronize()
    assert tok.tolist() == want
    s.close()


@pytest.mark.parametrize("dtype,cols,rows", [("bf16", 131072, 40), ("f16", 131072, 40), ("f32", 1 << 19, 5)])
def test_a_nucleus_of_the_lightest_weights(gs, dtype, cols, rows):
    """Thousands of entries of hardly more than 2^-41 of the largest weight,
    which the whole-number masses hold as 2^-40: as many as a CTA of a cluster
    has in one bin, of the greatest sum that a bin can have."""
    import torch
    part = 32768  # entries of a CTA
    x = torch.full((cols,), -32.0, dtype=_dtype(dtype), device="cuda")
    x[cols - part:] = -float("inf")
    x[cols - 1] = 0
    T = float(np.float32(ref.LOG2E * 32 / 40.995))
    h = ref.clean(x)
    _, w = ref.weights(h, T, x.device)
    p = 1 - 2.0**-24
    kept = ref.kept(h, w, top_p=p)
    tail = int((kept[:-1] > 0).sum())
    assert 2.0**-41 < w[0] < 2.0**-40.99 and kept[0] == 1 and part // 2 <= tail < cols - part - 1
    at = [0, 1, part // 2, tail - 1, tail]
    u = [(t + 0.5) / int(kept.sum()) for t in at]
    want = [ref.sample(x, v, temperature=T, top_p=p)[0] for v in u]
    assert want[:-1] == at[:-1] and want[-1] == cols - 1
    of = torch.arange(rows) % len(u)
    got = _sample(gs, x.expand(rows, -1), np.array(u, np.float32)[of], top_p=p, temperature=T)
    assert got == [want[k] for k in of]


def _across(dtype, n):
    """Rows that several CTAs of a cluster share, whose entries above -inf, or whose entries that are to be cleaned, lie
    in some of their parts only."""
    import torch
    dt, inf = _dtype(dtype), float("inf")
    base = _peaked(1, n, dtype, 5)[0]
    full = lambda v: torch.full((n,), v, dtype=dt, device="cuda")  # noqa: E731

    def only(a, b, x=base, rest=-inf):
        y = full(rest)
        y[a:b] = x[a:b]
        return y

    def put(at, v, x=base):
        y = x.clone()
        y[at] = v
        return y

    low = torch.finfo(dt).min
    return [full(-inf), full(float("nan")), only(0, 1), only(n - 1, n), only(n // 2, n // 2 + 1), only(0, 30), only(n - 30, n),
            only(n // 2 - 300, n // 2 + 300), only(n // 3, n // 3 + 5, rest=low), only(n - 9000, n), only(0, 9000, full(0.5)),
            put(n // 2, inf), put(n - 1, inf, put(0, inf)), put(n - 2, float("nan")), put(slice(n // 4, n // 2), float("nan")),
            put(slice(0, n, 2), -inf), put(slice(0, n, 2), low), put(n - 3, inf, full(-inf)), full(low), full(2.0)]


@pytest.mark.parametrize("dtype,cols", [("f32", 70001), ("f16", 70001), ("bf16", 70001), ("f32", 200003), ("bf16", 262139)])
@pytest.mark.parametrize("params", [{}, dict(temperature=0.0), dict(top_k=50), dict(top_k=5000), dict(top_p=0.9), dict(min_p=0.05),
                                    dict(temperature=1.1, top_k=3000, top_p=0.9, min_p=0.01)],
                         ids=["plain", "greedy", "top_k 50", "top_k 5000", "top_p", "min_p", "all"])
def test_masks_across_the_ctas_of_a_row(gs, dtype, cols, params):
    import torch
    x = torch.stack(_across(dtype, cols))
    _check(gs, x, _uniform(x.shape[0], 1), **params)


@pytest.mark.parametrize("dtype,cols", [("f32", 70001), ("f16", 70001), ("bf16", 70001), ("f32", 200003), ("bf16", 262139)])
@pytest.mark.parametrize("n", [1, 20, 700])
def test_best_across_the_ctas_of_a_row(gs, dtype, cols, n):
    import torch
    _check_best(gs, torch.stack(_across(dtype, cols)), n)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("params", [{}, dict(temperature=0.0), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05, temperature=1.5)],
                         ids=["plain", "greedy", "top_k", "top_p", "min_p"])
def test_batches_on_both_sides_of_the_size_rule(gs, dtype, params):
    """Clusters take 20 rows, streaming CTAs 600 of them where nothing is cut by mass: the same bits."""
    import torch
    x, u = _peaked(20, 70001, dtype, 2), _uniform(20, 3)
    tok, lp = _check(gs, x, u, **params)
    big_tok, big_lp = gs.sample(x.repeat(30, 1), u.repeat(30), sync=True, **params)
    assert torch.equal(big_tok, tok.repeat(30)) and torch.equal(big_lp, lp.repeat(30))
    if not params:
        small, big = gs.top_logprobs(x, 9, sync=True), gs.top_logprobs(x.repeat(30, 1), 9, sync=True)
        _check_best(gs, x, 9)
        for a, b in zip(small, big):
            assert torch.equal(a.repeat(30, *[1] * (a.dim() - 1)), b)
