"""Plain restatements of the serving operators for their tests: whole-number
arithmetic and 64-bit floats on the host, one row (or request) at a time.

The weights of a row are 32-bit numbers by definition (2^-y with y rounded
step by step); numpy's float32 gives the same y as the kernels' rounded
operations, and the exponential is torch.exp2 on the logits' device."""
from __future__ import annotations

import math

import numpy as np
import torch

LOG2E = np.float32(1.4426950408889634)
F32_MAX = np.float32(3.4028234663852886e38)


def clean(row):
    """float32 numpy values of one row of logits as the operators read them."""
    x = torch.nan_to_num(row, nan=-math.inf, neginf=-math.inf).float()
    return x.cpu().numpy()


def weights(x, temperature, device):
    """(y, w) of a row with something above -inf; temperature <= 0 or NaN: 1."""
    t = np.float32(temperature)
    with np.errstate(over="ignore", divide="ignore"):
        c = np.minimum(LOG2E / t, F32_MAX) if t > 0 else LOG2E
        y = (x.max() - x) * c
    w = torch.exp2(-torch.from_numpy(y).to(device)).cpu().numpy()
    return y, w


def kept(x, w, top_k=0, top_p=1.0, min_p=0.0):
    """Whole-number masses of the kept entries (0: cut), in index order."""
    q = np.rint(np.ldexp(w.astype(np.float64), 40)).astype(np.int64)
    order = np.argsort(-x.astype(np.float64), kind="stable")
    order = order[x[order] > -np.inf]
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1.0:
        run = np.cumsum(q[order])
        least = max(1, math.ceil(max(float(np.float32(top_p)), 0.0) * float(run[-1])))
        order = order[: int(np.searchsorted(run, least, side="left")) + 1]
    out = np.zeros_like(q)
    out[order] = q[order]
    out[w < min(np.float32(min_p), np.float32(1))] = 0
    return out


def sample(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log-probability in 64 bits) of one row."""
    x = clean(row)
    if not (x > -np.inf).any():
        return -1, -math.inf
    _, w = weights(x, temperature, row.device)
    if not temperature > 0:
        token = int(np.argmax(x))
    else:
        run = np.cumsum(kept(x, w, top_k, top_p, min_p))
        u = min(max(float(np.float32(u)), 0.0), 1.0)
        token = int(np.searchsorted(run, min(math.floor(u * float(run[-1])), int(run[-1]) - 1), side="right"))
    z = x.astype(np.float64) - float(x.max())
    if temperature > 0:
        z = z / float(np.float32(temperature))
    return token, float(z[token] - np.log(np.exp(z).sum()))


def best(row, n):
    """(indices, log-probabilities, log-sum-exp) of the n best of one row."""
    x = clean(row).astype(np.float64)
    idx, lp = np.full(n, -1), np.full(n, -np.inf)
    if not (x > -np.inf).any():
        return idx, lp, -math.inf
    ln = float(np.log(np.exp(x - x.max()).sum()))
    lse = float(x.max()) + ln
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf][:n]
    idx[: order.size] = order
    lp[: order.size] = (x[order] - x.max()) - ln  # x - lse would lose ln beside the lowest value
    lp[lp < -float(F32_MAX)] = -np.inf  # the lowest value beside the largest: no 32-bit number
    return idx, lp, lse


def logprob_bound(cols):
    """(absolute, relative) bound on a 32-bit log-probability: the total mass
    is off by at most 2^-41 for each entry and 2^-22 of itself (2 ulp of the
    exponential, and y's three roundings, which weigh at most y 2^-y of it),
    its logarithm and the final sum round to 2^-24 each of terms of at most
    the result's size plus ln(cols) <= 14: 2^-20 of slack covers them; y itself
    carries three roundings of 2^-24."""
    return 2.0**-20 + cols * 2.0**-41, 2.0**-21


def plan(context, new, page, table, free, cursor, capacity):
    """dict of what plan_slots writes; `table` (numpy, changed in place)."""
    ctx, new = np.maximum(context, 0).tolist(), np.maximum(new, 0).tolist()
    R, width = table.shape
    before = table.copy()
    start, pos, req, slots, missed = [0], [], [], [], False
    nxt = max(int(cursor), 0)
    for r in range(R):
        have = min(-(-ctx[r] // page), width)
        need = min(-(-(ctx[r] + new[r]) // page), width)
        for k in range(have, need):
            table[r, k] = free[nxt] if nxt < len(free) else -1
            nxt += 1
        for p in range(ctx[r], ctx[r] + new[r]):
            k = p // page
            held = int(table[r, k]) if k < width else -1
            pos.append(p)
            req.append(r)
            slots.append(held * page + p % page if held >= 0 else -1)
            missed |= held < 0
        start.append(start[-1] + new[r])
    missed |= len(pos) > capacity
    pad = max(0, capacity - len(pos))
    assert (before[table == before] == table[table == before]).all()
    return {"query_start": start, "seq_lens": [a + b for a, b in zip(ctx, new)],
            "positions": (pos + [0] * pad)[:capacity], "requests": (req + [-1] * pad)[:capacity],
            "slots": (slots + [-1] * pad)[:capacity], "cursor_out": min(nxt, len(free)), "missed": missed}
