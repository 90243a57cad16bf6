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
