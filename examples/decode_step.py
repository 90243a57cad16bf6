"""A serving loop over forge_sort.GpuSampler: requests of different lengths go
through a small attention model with a paged key/value cache.  Each step is

    plan_slots     where the step's tokens go: their request, position and slot,
                   new pages taken from the list of free ones
    the model      writes keys and values into the slots, reads the block table
    sample         one token of every request from its logits
    top_logprobs   the alternatives a client asked for

and nothing leaves the GPU until the loop ends.  The model (random weights, one
layer) is plain torch; it stands for a real one.

    python examples/decode_step.py [--steps N] [--temperature T] [--top-p P]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "gpu-forge_b200"))
from forge_sort import GpuSampler  # noqa: E402


class PagedModel:
    """One attention layer over a paged cache; forward() gives the logits of
    each request's last token."""

    def __init__(self, vocab=4096, dim=128, heads=4, pages=256, page_size=16, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        w = lambda *shape: torch.randn(*shape, generator=g, device="cuda") / shape[-1] ** 0.5
        self.embed, self.place = w(vocab, dim) * 8, w(page_size * pages, dim) * 8
        self.qkv, self.out = w(3 * dim, dim), w(vocab, dim) * 4
        self.heads, self.page_size = heads, page_size
        # one row more than the pages have: slots of -1 (a token without a page, a place beyond the last token) index
        # the last row, which belongs to nobody
        self.cache = torch.zeros(2, pages * page_size + 1, dim, device="cuda")

    def forward(self, ids, plan, block_table):
        x = self.embed[ids] + self.place[plan.positions]
        q, k, v = (x @ self.qkv.T).chunk(3, -1)
        self.cache[0][plan.slots], self.cache[1][plan.slots] = k, v
        # the slots of all positions of each request, from its row of the block table
        at = (block_table.clamp(min=0).long()[:, :, None] * self.page_size
              + torch.arange(self.page_size, device="cuda")).flatten(1)
        keys, values = self.cache[:, at[plan.requests.long()]]  # [tokens, positions, dim]
        split = lambda t: t.unflatten(-1, (self.heads, -1))
        score = torch.einsum("thd,tshd->ths", split(q), split(keys)) * (q.shape[-1] // self.heads) ** -0.5
        ahead = torch.arange(at.shape[1], device="cuda") > plan.positions[:, None]
        score = score.masked_fill(ahead[:, None], float("-inf")).softmax(-1)
        y = x + torch.einsum("ths,tshd->thd", score, split(values)).flatten(1)
        return y[plan.query_start[1:].long() - 1] @ self.out.T


def generate(model, prompts, steps, *, temperature=None, top_k=None, top_p=None, alternatives=3, seed=0,
             pages=256, width=32):
    """(tokens, logprobs, alternatives) of `steps` tokens per prompt (lists of
    token ids): tensors [requests, steps], [requests, steps] and [requests, steps, n]."""
    gs = GpuSampler.new()
    R = len(prompts)
    i32 = dict(dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(seed)
    free = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((R, width), -1, **i32)
    lens, cursor = torch.zeros(R, **i32), torch.zeros(1, **i32)
    ids = torch.tensor([t for p in prompts for t in p], device="cuda")
    new = torch.tensor([len(p) for p in prompts], **i32)
    tokens, logprobs, others = [], [], []
    for _ in range(steps):
        plan = gs.plan_slots(lens, new, table, free, cursor, page_size=model.page_size, capacity=ids.numel())
        logits = model.forward(ids, plan, table)
        u = torch.rand(R, generator=g, device="cuda")
        token, logprob = gs.sample(logits, u, temperature=temperature, top_k=top_k, top_p=top_p)
        best, _, _ = gs.top_logprobs(logits, alternatives)
        tokens.append(token), logprobs.append(logprob), others.append(best)
        lens, cursor, ids = plan.seq_lens, plan.cursor_out, token.long()
        new = torch.ones(R, **i32)
    gs.synchronize()  # reports a step that ran out of pages
    gs.close()
    return torch.stack(tokens, 1), torch.stack(logprobs, 1), torch.stack(others, 1)


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--temperature", type=float, default=0.8)
    ap.add_argument("--top-p", type=float, default=0.95)
    a = ap.parse_args()
    prompts = [[1, 2, 3], list(range(100, 140)), [7], [42] * 17]
    tokens, logprobs, _ = generate(PagedModel(), prompts, a.steps, temperature=a.temperature, top_p=a.top_p)
    for p, t, lp in zip(prompts, tokens.tolist(), logprobs.tolist()):
        print(f"{len(p):3d} tokens in -> {t}  (mean logprob {sum(lp) / len(lp):.2f})")


if __name__ == "__main__":
    main()
