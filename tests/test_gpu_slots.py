"""GPU tests of GpuSampler.plan_slots against the plain loop of _serving.py:
every number equal."""
import numpy as np
import pytest

import _serving as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gs():
    import forge_sort
    s = forge_sort.GpuSampler.new()
    yield s
    s.close()


def _case(ctx, new, page, seed, short=0, spare=3, cursor=2, narrow=0):
    """A table whose rows hold the requests' pages, and a list of free pages
    that `short` pages too few are on; narrow: columns the table lacks."""
    rng = np.random.default_rng(seed)
    c, n = np.maximum(ctx, 0), np.maximum(new, 0)
    have, need = -(-c // page), -(-(c + n) // page)
    width = max(1, int(need.max(initial=1)) - narrow)
    ids = rng.permutation(int(need.sum()) + spare + 5).astype(np.int32)
    table = np.full((len(ctx), width), -1, np.int32)
    at = 0
    for r in range(len(ctx)):
        h = min(int(have[r]), width)
        table[r, :h] = ids[at:at + h]
        at += h
    wanted = int((np.minimum(need, width) - np.minimum(have, width)).sum())
    free = np.concatenate([np.full(cursor, -1, np.int32), ids[at:at + max(0, wanted + spare - short - (spare if short else 0))]])
    return table, free


def _check(gs, ctx, new, page, ints="i32", capacity=None, seed=0, cursor=2, stride=0, **kw):
    import torch
    from forge_sort import GpuExecution
    I = {"i32": torch.int32, "i64": torch.int64}[ints]
    ctx, new = np.asarray(ctx, np.int64), np.asarray(new, np.int64)
    table, free = _case(ctx, new, page, seed, cursor=cursor, **kw)
    total = int(np.maximum(new, 0).sum())
    capacity = total if capacity is None else capacity
    dev = lambda a, dt: torch.from_numpy(np.ascontiguousarray(a)).to(dt).cuda()  # noqa: E731
    big = torch.full((table.shape[0], table.shape[1] + stride), -7, dtype=torch.int32, device="cuda")
    t = big[:, :table.shape[1]]
    t.copy_(dev(table, torch.int32))
    args = (dev(ctx, I), dev(new, I), t, dev(free, torch.int32), dev(np.array([cursor]), torch.int32))
    want = ref.plan(ctx, new, page, table, free, cursor, capacity)
    failed = False
    for again in range(2):  # a call may be repeated
        try:
            plan = gs.plan_slots(*args, page_size=page, capacity=capacity, sync=True)
        except GpuExecution as e:
            assert "slot" in str(e)
            failed = True
            plan = gs.plan_slots(*args, page_size=page, capacity=capacity)
            torch.cuda.synchronize()
            with pytest.raises(GpuExecution):
                gs.synchronize()
        gs.synchronize()
        assert failed == want["missed"]
        for name in ("query_start", "seq_lens", "positions", "requests", "slots"):
            assert getattr(plan, name).tolist() == want[name], name
        assert int(plan.cursor_out) == want["cursor_out"]
        assert np.array_equal(t.cpu().numpy(), table)
    assert (big[:, table.shape[1]:] == -7).all()
    assert plan.seq_lens.dtype == I and plan.positions.dtype == I and plan.slots.dtype == torch.int64


@pytest.mark.parametrize("ints", ["i32", "i64"])
@pytest.mark.parametrize("page", [1, 7, 16, 128])
@pytest.mark.parametrize("requests", [1, 2, 31, 33, 511, 513, 2047, 2048, 2049, 5000])
def test_decode(gs, ints, page, requests):
    rng = np.random.default_rng(requests)
    _check(gs, rng.integers(0, 100, requests), np.ones(requests, int), page, ints)


@pytest.mark.parametrize("ints", ["i32", "i64"])
@pytest.mark.parametrize("page", [1, 16, 48, 64])
def test_mixed_lengths(gs, ints, page):
    rng = np.random.default_rng(page)
    for requests in (1, 5, 40, 300):
        ctx = rng.choice([0, 1, page - 1, page, page + 1, 2 * page, 333], requests)
        new = rng.choice([0, 0, 1, 1, 2, page - 1, page, page + 1, 517], requests)
        _check(gs, ctx, new, page, ints, capacity=int(new.sum()) + 100)
        _check(gs, ctx, new, page, ints, stride=5)


def test_chunk_edges(gs):
    """Requests without tokens on both sides of the scan's chunks, long ones across them."""
    new = np.zeros(6200, int)
    new[[0, 2046, 2047, 2048, 2049, 4095, 4096, 6199]] = [3, 700, 1, 513, 2, 1, 900, 5]
    _check(gs, np.arange(6200) % 50, new, 16)
    _check(gs, np.zeros(4096, int), np.zeros(4096, int), 16, capacity=10)
    one = np.zeros(2500, int)
    one[2400] = 3000
    _check(gs, np.full(2500, 5), one, 16)


def test_nothing_new(gs):
    _check(gs, [5, 0, 17], [0, 0, 0], 16)
    _check(gs, [5, 0, 17], [0, 0, 0], 16, capacity=7)


def test_negative_lengths_read_as_zero(gs):
    _check(gs, [-4, 9, -1], [3, -2, 5], 4, capacity=12)


@pytest.mark.parametrize("short", [1, 2, 9])
def test_free_pages_run_out(gs, short):
    _check(gs, [3, 0, 30, 16], [50, 1, 40, 64], 16, short=short)


@pytest.mark.parametrize("narrow", [1, 3])
def test_table_too_narrow(gs, narrow):
    _check(gs, [3, 0, 30, 16], [50, 1, 40, 64], 16, narrow=narrow)


def test_capacity_too_small(gs):
    _check(gs, [3, 0, 30], [50, 1, 40], 16, capacity=60)


def test_a_held_page_is_missing(gs):
    import torch
    from forge_sort import GpuExecution
    t = torch.full((1, 4), -1, dtype=torch.int32, device="cuda")
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    with pytest.raises(GpuExecution):
        gs.plan_slots(i(3), i(2), t, i(9, 8), i(0), page_size=16, capacity=2, sync=True)
    p = gs.plan_slots(i(3), i(30), t, i(9, 8), i(0), page_size=16, capacity=30)
    torch.cuda.synchronize()
    with pytest.raises(GpuExecution):
        gs.synchronize()
    assert p.slots.tolist() == [-1] * 13 + [9 * 16 + k for k in range(16)] + [8 * 16]
    assert t.tolist() == [[-1, 9, 8, -1]]


def test_long_context_and_page_numbers_beyond_32_bits_of_slots(gs):
    import torch
    t = torch.full((2, 70000), -1, dtype=torch.int32, device="cuda")
    held = 2**31 // 65536 + 1
    t[0, :held] = 2**31 - 2 - torch.arange(held, dtype=torch.int32, device="cuda")
    c = torch.tensor([2**31 + 5, 0], device="cuda")
    n = torch.tensor([3, 2], device="cuda")
    free = torch.tensor([2**31 - 1], dtype=torch.int32, device="cuda")
    cur = torch.zeros(1, dtype=torch.int32, device="cuda")
    p = gs.plan_slots(c, n, t, free, cur, page_size=65536, capacity=5, sync=True)
    page = int(t[0, 2**31 // 65536])
    assert p.slots.tolist() == [page * 65536 + 5 + k for k in range(3)] + [(2**31 - 1) * 65536, (2**31 - 1) * 65536 + 1]
    assert p.seq_lens.tolist() == [2**31 + 8, 2]
    assert p.positions.tolist() == [2**31 + 5, 2**31 + 6, 2**31 + 7, 0, 1]


def test_a_million_tokens(gs):
    """Against torch's own scans."""
    import torch
    R, page = 700, 64
    new = torch.randint(0, 3000, (R,), device="cuda")
    ctx = torch.randint(0, 5000, (R,), device="cuda")
    have, need = (ctx + page - 1) // page, (ctx + new + page - 1) // page
    t = torch.full((R, int(need.max())), -1, dtype=torch.int32, device="cuda")
    col = torch.arange(t.shape[1], device="cuda")[None]
    t[col < have[:, None]] = torch.arange(int(have.sum()), dtype=torch.int32, device="cuda")
    free = torch.arange(int(have.sum()), int(need.sum()), dtype=torch.int32, device="cuda")
    T = int(new.sum())
    p = gs.plan_slots(ctx, new, t, free, torch.zeros(1, dtype=torch.int32, device="cuda"), page_size=page, capacity=T, sync=True)
    r = torch.repeat_interleave(torch.arange(R, device="cuda"), new)
    pos = ctx[r] + torch.arange(T, device="cuda") - (torch.cumsum(new, 0) - new)[r]
    assert torch.equal(p.requests.long(), r) and torch.equal(p.positions, pos)
    assert torch.equal(t[(col >= have[:, None]) & (col < need[:, None])], free)
    assert torch.equal(p.slots, t[r, pos // page].long() * page + pos % page)


@pytest.mark.parametrize("page", [1, 3, 100, 65536])
@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("ints", ["int32", "int64"])
def test_many_tokens_into_given_memory(gs, page, offset, ints):
    """Enough tokens for the wide stores, into tensors that begin at 16-byte
    boundaries and between them, with places behind the last token."""
    import torch
    I = getattr(torch, ints)
    g = torch.Generator(device="cuda").manual_seed(page + offset)
    R, T = 997, 90000
    new = torch.randint(0, 181, (R,), generator=g, device="cuda")
    new = (new * T // int(new.sum())).to(I)
    ctx = torch.randint(0, 300, (R,), generator=g, device="cuda").to(I)
    have, need = (ctx + page - 1) // page, (ctx + new + page - 1) // page
    t = torch.full((R, int(need.max())), -1, dtype=torch.int32, device="cuda")
    col = torch.arange(t.shape[1], device="cuda")[None]
    t[col < have[:, None]] = torch.arange(int(have.sum()), dtype=torch.int32, device="cuda")
    free = torch.arange(int(have.sum()), int(need.sum()), dtype=torch.int32, device="cuda")
    out = lambda dt: torch.full((T + 8,), -5, dtype=dt, device="cuda")[offset:offset + T]  # noqa: E731
    p = gs.plan_slots(ctx, new, t, free, torch.zeros(1, dtype=torch.int32, device="cuda"), page_size=page,
                      positions=out(I), requests=out(torch.int32), slots=out(torch.int64), sync=True)
    n = int(new.sum())
    r = torch.repeat_interleave(torch.arange(R, device="cuda"), new.long())
    pos = ctx.long()[r] + torch.arange(n, device="cuda") - (torch.cumsum(new.long(), 0) - new.long())[r]
    assert torch.equal(p.requests[:n].long(), r) and torch.equal(p.positions[:n].long(), pos)
    assert torch.equal(p.slots[:n], t[r, pos // page].long() * page + pos % page)
    assert n < T and (p.requests[n:] == -1).all() and (p.positions[n:] == 0).all() and (p.slots[n:] == -1).all()
    assert torch.equal(t[(col >= have[:, None]) & (col < need[:, None])], free)


def test_refusals(gs):
    import torch
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    t = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    ok = dict(page_size=16, capacity=2)
    gs.plan_slots(i(1, 2), i(1, 1), t, i(5), i(0), sync=True, **ok)
    with pytest.raises(TypeError):
        gs.plan_slots(i(1, 2).float(), i(1, 1), t, i(5), i(0), **ok)
    with pytest.raises(TypeError):
        gs.plan_slots(i(1, 2), i(1, 1).long(), t, i(5), i(0), **ok)
    with pytest.raises(TypeError):
        gs.plan_slots(i(1, 2), i(1, 1), t.long(), i(5), i(0), **ok)
    with pytest.raises(TypeError):
        gs.plan_slots(i(1, 2), i(1, 1), t, None, i(0), **ok)
    for args in [(i(1, 2), i(1), t, i(5), i(0)), (i(1), i(1), t, i(5), i(0)), (i(1, 2), i(1, 1), t[0], i(5), i(0)),
                 (i(1, 2), i(1, 1), t.t().contiguous().t(), i(5), i(0)), (i(1, 2), i(1, 1), t, i(5), i(0, 1)),
                 (i(1, 2), i(1, 1), t.cpu(), i(5), i(0)), (i(1, 2), i(1, 1), t.expand(2, 4)[:1].expand(2, 4), i(5), i(0))]:
        with pytest.raises(ValueError):
            gs.plan_slots(*args, **ok)
    for page in (0, -1, 2**20 + 1):
        with pytest.raises(ValueError):
            gs.plan_slots(i(1, 2), i(1, 1), t, i(5), i(0), page_size=page, capacity=2)
    with pytest.raises(ValueError):  # no number of tokens
        gs.plan_slots(i(1, 2), i(1, 1), t, i(5), i(0), page_size=16)
    c = i(0)
    with pytest.raises(ValueError):  # the cursor would change while it is read
        gs.plan_slots(i(1, 2), i(1, 1), t, i(5), c, cursor_out=c, **ok)
    with pytest.raises(ValueError):
        gs.plan_slots(i(1, 2), i(1, 1), t, i(5), i(0), slots=torch.zeros(3, dtype=torch.int64, device="cuda"),
                      positions=i(0), page_size=16)
    c, n = i(1, 2), i(1, 1)
    for same in (c, n):  # lengths that would change while they are read
        with pytest.raises(ValueError):
            gs.plan_slots(c, n, t, i(5), i(0), seq_lens=same, **ok)
