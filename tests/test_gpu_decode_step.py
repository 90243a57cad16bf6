"""The serving loop of examples/decode_step.py: the paged, batched run against
the same model without a cache, one request at a time, in 64 bits."""
import importlib.util
import os

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "decode_step.py")


@pytest.fixture(scope="module")
def ex():
    spec = importlib.util.spec_from_file_location("decode_step", PATH)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def unpaged_logits(model, ids):
    """Logits of the last of `ids`: the whole sequence, no cache, float64."""
    d = lambda t: t.double()
    x = d(model.embed)[ids] + d(model.place)[torch.arange(len(ids), device="cuda")]
    q, k, v = (x @ d(model.qkv).T).chunk(3, -1)
    split = lambda t: t.unflatten(-1, (model.heads, -1))
    score = torch.einsum("hd,shd->hs", split(q)[-1], split(k)) * (q.shape[-1] // model.heads) ** -0.5
    y = x[-1] + torch.einsum("hs,shd->hd", score.softmax(-1), split(v)).flatten()
    return y @ d(model.out).T


PROMPTS = [[1, 2, 3], list(range(100, 140)), [7], [42] * 16, [5] * 17]


def test_greedy_equals_unpaged(ex):
    """Every token of the loop is the largest logit of the unpaged model run
    over what was generated before it, its log-probability that model's, and
    the alternatives begin with it.  32-bit products of 128 terms of size ~8
    differ by far less than 1e-2 from 64 bits; so do the two largest logits
    where the tokens differ."""
    model = ex.PagedModel(seed=3)
    tokens, logprobs, others = ex.generate(model, PROMPTS, 20, temperature=0.0, seed=1)
    for r, p in enumerate(PROMPTS):
        seq = list(p)
        for s in range(20):
            logits = unpaged_logits(model, torch.tensor(seq, device="cuda"))
            t = int(tokens[r, s])
            assert float(logits.max() - logits[t]) < 1e-2
            assert abs(float(logprobs[r, s]) - float(logits.log_softmax(0)[t])) < 1e-2
            assert int(others[r, s, 0]) == t
            seq.append(t)


def test_same_seed_same_tokens(ex):
    runs = [ex.generate(ex.PagedModel(seed=3), PROMPTS, 12, temperature=0.9, top_k=50, top_p=0.9, seed=5) for _ in range(2)]
    for a, b in zip(*runs):
        assert torch.equal(a, b)
    assert int(runs[0][0].min()) >= 0


def test_out_of_pages_is_reported(ex):
    model = ex.PagedModel(pages=256)
    with pytest.raises(Exception, match="free pages"):
        ex.generate(model, [[1] * 40, [2] * 40], 2, temperature=0.0, pages=3)


def test_tokens_without_a_slot_touch_no_page(ex):
    """A token without a page and a place beyond the last token (slots of -1)
    leave every page as it was; the keys of the others are written."""
    from forge_sort import SlotPlan
    model = ex.PagedModel(pages=8, page_size=4)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    mark = torch.full((2, 8 * 4, model.embed.shape[1]), 3.0, device="cuda")
    model.cache[:, :8 * 4] = mark
    plan = SlotPlan(query_start=i32(0, 1, 2), seq_lens=i32(1, 1), positions=i32(0, 0, 0), requests=i32(0, 1, -1),
                    slots=torch.tensor([-1, 9, -1], device="cuda"), cursor_out=i32(1))
    logits = model.forward(torch.tensor([5, 6, 0], device="cuda"), plan, i32(-1, 2).view(2, 1))
    changed = (model.cache[:, :8 * 4] != mark).any(-1)
    assert changed.nonzero().tolist() == [[0, 9], [1, 9]]
    assert logits.shape[0] == 2 and logits[1].isfinite().all()
