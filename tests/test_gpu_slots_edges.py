"""GPU tests of fs_plan_slots at its edges: batches without requests, lengths
that pass their type, memory that inputs and outputs share, streams other than
the sorter's."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gs():
    import forge_sort
    s = forge_sort.GpuSampler.new()
    yield s
    s.close()


def _i32(*v):
    import torch
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("ints", ["int32", "int64"])
@pytest.mark.parametrize("capacity", [0, 1, 7, 100000])
@pytest.mark.parametrize("width", [0, 4])
@pytest.mark.parametrize("cursor,free", [(5, 9), (0, 0), (12, 9), (-3, 2)])
def test_no_requests(gs, ints, capacity, width, cursor, free):
    """A step without requests has places to fill and a cursor to hand on."""
    import torch
    I = getattr(torch, ints)
    none = torch.empty(0, dtype=I, device="cuda")
    out = lambda n, dt: torch.full((n,), -5, dtype=dt, device="cuda")  # noqa: E731
    p = gs.plan_slots(none, none, torch.empty(0, width, dtype=torch.int32, device="cuda"), torch.arange(free, dtype=torch.int32, device="cuda"),
                      _i32(cursor), page_size=16, query_start=out(1, torch.int32), positions=out(capacity, I),
                      requests=out(capacity, torch.int32), slots=out(capacity, torch.int64), cursor_out=out(1, torch.int32),
                      sync=True)
    assert p.query_start.tolist() == [0] and p.seq_lens.shape == (0,)
    assert p.cursor_out.tolist() == [min(max(cursor, 0), free)]
    assert (p.positions == 0).all() and (p.requests == -1).all() and (p.slots == -1).all()


MOST = {"int32": 2**31 - 1, "int64": 2**63 - 1}


def _plan(context, new, page, held, top):
    """What a plan holds, in whole numbers without end; no length passes `top`."""
    start, seq, pos, req, slots = [0], [], [], [], []
    for r, c in enumerate(context):
        n = min(new[r], top - c)
        for p in range(c, c + n):
            page_of = p // page
            pos.append(p), req.append(r), slots.append(held[r][page_of] * page + p % page if page_of < len(held[r]) else -1)
        start.append(start[-1] + n), seq.append(c + n)
    return start, seq, pos, req, slots


@pytest.mark.parametrize("ints", ["int32", "int64"])
@pytest.mark.parametrize("short,extra", [(1, 5), (5, 2), (5, 5), (5, 6), (0, 3), (3, 0)])
def test_lengths_that_pass_their_type(gs, ints, short, extra):
    """A request whose context and new tokens exceed the largest number of its
    type, beside others that do not: reported, and planned up to that number."""
    import torch
    from forge_sort import GpuExecution
    I, top, page = getattr(torch, ints), MOST[ints], 1 << 20
    context, new, capacity = [7, top - short, 3], [4, extra, 9], 32
    width = 2048  # all pages that 32-bit positions have; of 64-bit ones, none of the long request's
    table = torch.arange(3 * width, dtype=torch.int32, device="cuda").view(3, width)
    held = table.tolist()
    args = (torch.tensor(context, device="cuda").to(I), torch.tensor(new, device="cuda").to(I), table,
            torch.empty(0, dtype=torch.int32, device="cuda"), _i32(0))
    p = gs.plan_slots(*args, page_size=page, capacity=capacity)
    torch.cuda.synchronize()
    start, seq, pos, req, slots = _plan(context, new, page, held, top)
    if -1 in slots or extra > short:
        with pytest.raises(GpuExecution, match="slot"):
            gs.synchronize()
    else:
        gs.synchronize()
    n = len(pos)
    assert p.query_start.tolist() == start and p.seq_lens.tolist() == seq
    assert p.positions.tolist() == pos + [0] * (capacity - n) and p.requests.tolist() == req + [-1] * (capacity - n)
    assert p.slots.tolist() == slots + [-1] * (capacity - n)
    assert table.tolist() == held


@pytest.mark.parametrize("page", [1, 3, 16, 1 << 20])
@pytest.mark.parametrize("capacity", [70000, 90000])  # both widths of the stores, enough CTAs for 2^31 tokens
def test_lengths_near_two_to_the_63(gs, page, capacity):
    """Sums of lengths that 64 bits do not hold: every step stays inside its
    memory and ends, and what fits is planned."""
    import torch
    from forge_sort import GpuExecution
    top = 2**63 - 1
    context = [4, top, top - 1, top - 5, 0, top // 2, 0]
    new = [2, top, top, 3, top, top, top]
    table = torch.full((7, 4), -1, dtype=torch.int32, device="cuda")
    table[0] = torch.arange(4, dtype=torch.int32, device="cuda")
    p = gs.plan_slots(torch.tensor(context, device="cuda"), torch.tensor(new, device="cuda"), table,
                      torch.empty(0, dtype=torch.int32, device="cuda"), _i32(0), page_size=page, capacity=capacity)
    torch.cuda.synchronize()
    with pytest.raises(GpuExecution, match="slot"):
        gs.synchronize()
    assert p.query_start.tolist() == [0, 2, 2, 3, 6] + [2**31 - 1] * 3
    assert p.seq_lens.tolist() == [6, top, top, top - 2, top, top, top]
    have = [k * page + at if k < 4 else -1 for k, at in (divmod(x, page) for x in (4, 5))]
    assert p.slots.tolist() == have + [-1] * (capacity - 2)
    assert p.positions.tolist() == [4, 5, top - 1, top - 5, top - 4, top - 3] + list(range(capacity - 6))
    assert p.requests.tolist() == [0, 0, 2, 3, 3, 3] + [4] * (capacity - 6)
    assert table.tolist() == [[0, 1, 2, 3]] + [[-1] * 4] * 6


def test_many_long_requests(gs):
    """A sum of new tokens that 64 bits do not hold, of lengths that they do."""
    import torch
    from forge_sort import GpuExecution
    R, T = 5000, 70000
    new = torch.full((R,), 2**62, device="cuda")
    p = gs.plan_slots(torch.zeros_like(new), new, torch.full((R, 1), -1, dtype=torch.int32, device="cuda"), _i32(9, 8, 7), _i32(1),
                      page_size=2, capacity=T)
    torch.cuda.synchronize()
    with pytest.raises(GpuExecution, match="slot"):
        gs.synchronize()
    assert p.query_start.tolist() == [0] + [2**31 - 1] * R
    assert p.slots.tolist() == [16, 17] + [-1] * (T - 2) and p.positions.tolist() == list(range(T))
    assert p.cursor_out.tolist() == [3] and (p.seq_lens == 2**62).all()


def _overlaps():
    """name -> arguments of a plan in which an output shares some of its memory with something else."""
    import torch
    b = torch.zeros(64, dtype=torch.int32, device="cuda")
    w = torch.zeros(64, dtype=torch.int64, device="cuda")
    return {
        "lengths, one on": dict(context_lens=b[0:3], seq_lens=b[1:4]), "lengths, one back": dict(new_lens=b[5:8], seq_lens=b[3:6]),
        "positions of lengths": dict(context_lens=b[0:3], positions=b[2:14]), "starts of lengths": dict(new_lens=b[0:3], query_start=b[0:4]),
        "requests of free pages": dict(free_pages=b[0:6], requests=b[5:17]), "cursor": dict(cursor=b[0:1], cursor_out=b[0:1]),
        "cursor in starts": dict(cursor=b[3:4], query_start=b[0:4]), "cursors in requests": dict(cursor_out=b[4:5], requests=b[0:12]),
        "positions and requests": dict(positions=b[0:12], requests=b[11:23]),
        "slots and positions": dict(slots=w[0:12], positions=w[11:23].view(torch.int32)[:12]),
    }


@pytest.mark.parametrize("name", ["lengths, one on", "lengths, one back", "positions of lengths", "starts of lengths",
                                  "requests of free pages", "cursor", "cursor in starts", "cursors in requests",
                                  "positions and requests", "slots and positions"])
def test_outputs_that_share_memory_are_refused(gs, name):
    import torch
    args = dict(context_lens=_i32(1, 2, 3), new_lens=_i32(4, 4, 4), block_table=torch.zeros(3, 4, dtype=torch.int32, device="cuda"),
                free_pages=_i32(1, 2, 3, 4, 5, 6), cursor=_i32(0), page_size=16, capacity=12)
    with pytest.raises(ValueError, match="overlap"):
        gs.plan_slots(**{**args, **_overlaps()[name]})


def test_outputs_side_by_side_are_taken(gs):
    """Everything in one allocation, nothing shared."""
    import torch
    b = torch.zeros(64, dtype=torch.int32, device="cuda")
    w = torch.zeros(16, dtype=torch.int64, device="cuda")
    b[0:3], b[3:6], b[6:8], b[8] = _i32(1, 2, 3), _i32(1, 1, 2), _i32(5, 6), 0
    table = torch.zeros(3, 4, dtype=torch.int32, device="cuda")
    p = gs.plan_slots(b[0:3], b[3:6], table, b[6:8], b[8:9], page_size=16, query_start=b[9:13], seq_lens=b[13:16],
                      positions=b[16:20], requests=b[20:24], cursor_out=b[24:25], slots=w[0:4], sync=True)
    assert p.positions.tolist() == [1, 2, 3, 4] and p.requests.tolist() == [0, 1, 2, 2] and p.seq_lens.tolist() == [2, 3, 5]


def test_addresses_between_elements_are_refused(gs):
    """The C entries refuse them before a launch, with the argument's name."""
    import torch
    from forge_sort import _lib
    L, h = _lib.load(), gs._s._h
    b = torch.zeros(4096, dtype=torch.int64, device="cuda")
    at = lambda k: b[64 * k:].data_ptr()  # noqa: E731
    plan = dict(context_lens=at(0), new_lens=at(1), requests=2, page_size=16, block_table=at(2), width=4, stride=4, free_pages=at(3),
                n_free=3, cursor=at(4), query_start=at(5), seq_lens=at(6), positions=at(7), request_of=at(8), slots=at(9),
                capacity=4, cursor_out=at(10))
    rows = dict(logits=at(11), rows=2, cols=8, stride=8, temperature=at(12), top_k=at(13), top_p=at(14), min_p=at(15),
                uniform=at(16), tokens=at(17), logprobs=at(18))
    best = dict(logits=at(11), rows=2, cols=8, stride=8, n=2, indices=at(19), logprobs=at(20), lse=at(21))
    calls = [(lambda a: L.fs_plan_slots(h, 4, *a.values(), 1, None), plan, 4, {"slots": 8}),
             (lambda a: L.fs_plan_slots(h, 8, *a.values(), 1, None), plan, 4,
              dict.fromkeys(("context_lens", "new_lens", "seq_lens", "positions", "slots"), 8)),
             (lambda a: L.fs_sample_rows(h, 0, *a.values(), 1, None), rows, 4, {}),
             (lambda a: L.fs_sample_rows(h, 2, *a.values(), 1, None), rows, 4, {"logits": 2}),
             (lambda a: L.fs_top_logprobs(h, 0, *a.values(), 1, None), best, 4, {})]
    for call, args, size, own in calls:
        assert call(args) == _lib.OK
        for name, v in args.items():
            if v < 4096:  # a number
                continue
            off = own.get(name, size) // 2
            assert call({**args, name: v + off}) == _lib.E_INVALID, name
            text = L.fs_last_error(h).decode()
            assert name in text and "aligned" in text


def _short_plan():
    """Arguments of a plan that finds no page for its only token."""
    import torch
    return dict(context_lens=_i32(0), new_lens=_i32(1), block_table=torch.full((1, 1), -1, dtype=torch.int32, device="cuda"),
                free_pages=_i32(), cursor=_i32(0), page_size=16, capacity=1)


def test_synchronize_waits_for_every_stream(gs):
    """A failure on one stream is reported although the last call was on another."""
    import torch
    from forge_sort import GpuExecution
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    x, u, plan = torch.zeros(2, 64, device="cuda"), torch.zeros(2, device="cuda"), _short_plan()
    torch.cuda.synchronize()
    try:
        for asleep in (1000, 200_000_000):  # the first time for the allocations, which wait for the device
            with torch.cuda.stream(a):
                torch.cuda._sleep(asleep)
                gs.plan_slots(**plan)
            with torch.cuda.stream(b):
                gs.sample(x, u)
            if asleep == 1000:
                torch.cuda.synchronize()
            else:
                assert not a.query()
            with pytest.raises(GpuExecution, match="slot"):
                gs.synchronize()
            assert a.query() and b.query()
            gs.synchronize()  # reported once
    finally:
        torch.cuda.synchronize()


def test_fs_synchronize_waits_for_the_callers_streams():
    import torch
    import forge_sort
    from forge_sort import _lib
    L = _lib.load()
    s = forge_sort.GpuSorter.new()
    st = torch.cuda.Stream()
    v = _i32(0, 1, 0, 0, 0, 0, 0, 0, 0)
    table, slots = _i32(-1), torch.zeros(1, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    p = [v[k:].data_ptr() for k in range(9)]
    try:
        with torch.cuda.stream(st):
            torch.cuda._sleep(200_000_000)
        assert L.fs_plan_slots(s._h, 4, p[0], p[1], 1, 16, table.data_ptr(), 1, 1, None, 0, p[2], p[3], p[5], p[6], p[7],
                               slots.data_ptr(), 1, p[8], 0, st.cuda_stream) == _lib.OK
        assert L.fs_synchronize(s._h) == _lib.E_GPU_EXECUTION
        assert st.query() and slots.tolist() == [-1]
        assert L.fs_synchronize(s._h) == _lib.OK
    finally:
        torch.cuda.synchronize()
        s.close()


def test_close_waits_for_the_callers_streams():
    """A failing plan writes the sorter's error word, which close() frees."""
    import torch
    import forge_sort
    plan, st = _short_plan(), torch.cuda.Stream()
    for asleep in (1000, 200_000_000):
        gs = forge_sort.GpuSampler.new()
        with torch.cuda.stream(st):
            torch.cuda._sleep(asleep)
            gs.plan_slots(**plan)
        gs.close()
        assert st.query()


def test_many_streams(gs):
    """More streams than are busy at a time, a captured call among them."""
    import torch
    from forge_sort import GpuExecution
    plan, good = _short_plan(), {**_short_plan(), "free_pages": _i32(4)}
    good["block_table"] = torch.full((1, 1), -1, dtype=torch.int32, device="cuda")
    out = gs.plan_slots(**plan)
    into = {k: getattr(out, k) for k in ("query_start", "seq_lens", "positions", "requests", "slots", "cursor_out")}
    streams = [torch.cuda.Stream() for _ in range(12)]
    torch.cuda.synchronize()
    with pytest.raises(GpuExecution):
        gs.synchronize()
    for bad in (0, 7, 11, None):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                torch.cuda._sleep(2_000_000)
                gs.plan_slots(**(plan if k == bad else good), **into)
        if bad is not None:
            with pytest.raises(GpuExecution, match="slot"):
                gs.synchronize()
        gs.synchronize()
        assert all(st.query() for st in streams)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gs.plan_slots(**plan, **into)
    gs.synchronize()
    g.replay()
    torch.cuda.synchronize()
    with pytest.raises(GpuExecution, match="slot"):
        gs.synchronize()
    gs.synchronize()
