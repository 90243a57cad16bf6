"""The serving operators' measured cases: sampling a token from every row of a
batch of logits, the best log-probabilities of every row, and the block tables
and slot maps of a batch's step over a paged cache.

Each has a plain form in elementary torch operations and, where `own` is true,
the call that a user makes of forge_sort.GpuSampler.

Sampling, for a row x of V logits (NaN reads as -inf, +inf as the type's
largest finite value) with temperature T, top_k, top_p, min_p and one uniform
number u of [0, 1):
  c   = log2(e) / T             (T <= 0: the first maximum is taken, c = log2(e))
  w_j = 2^(-(max x - x_j) c)    in 32 bits
  q_j = w_j rounded to a multiple of 2^-40, as a whole number: every sum of
        weights is a sum of whole numbers and does not depend on its order
  the entries in descending order of x (ties: lowest index first) are cut to
  the first top_k, then to the shortest prefix with at least top_p of the
  mass of those, then to those with w_j >= min_p;
  the token is the first index at which the running sum of the kept q, in
  index order, exceeds floor(u * sum of the kept q).
Its log-probability is that of softmax(x / T) over the whole row.  A row with
nothing but -inf has token -1 and log-probability -inf.
"""
import math

import torch

own = False

LOG2E = 1.4426950408889634
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
INTS = {"i32": torch.int32, "i64": torch.int64}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i32": 4, "i64": 8}
LARGEST = 512 * 131072  # logits of the largest listed case
MOST_TOKENS = 1 << 20  # tokens of the largest listed step


# -- cases ----------------------------------------------------------------------
def listed():
    def sample(name, rows, vocab, dtype, logits, params):
        return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "logits": logits,
                "params": params}

    def best(name, rows, vocab, dtype, n):
        return {"name": name, "op": "top_logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "logits": "peaked",
                "n": n}

    def slots(name, requests, tokens, page, context, ints):
        return {"name": name, "op": "slots", "requests": requests, "tokens": tokens, "page": page, "context": context,
                "ints": ints}

    return [
        # one user's next token: latency counts
        sample("sample 1 row", 1, 32768, "f32", "peaked", "topk_topp"),
        # a small batch whose requests all ask for something else, some greedy
        sample("sample 16 mixed", 16, 131072, "bf16", "peaked", "mixed"),
        # a full serving batch with a nucleus
        sample("sample 256 top-p", 256, 131072, "bf16", "peaked", "topp"),
        # rollouts at temperature 1 from an odd vocabulary: no row but the first is aligned
        sample("sample 200 unfiltered", 200, 100003, "f16", "peaked", "plain"),
        # hot sampling from flat rows: the nucleus holds tens of thousands of tokens
        sample("sample 64 wide nucleus", 64, 131072, "f32", "flat", "topp"),
        # a large decode batch in 32 bits with masked tokens, every request its own filters
        sample("sample 512 mixed", 512, 131072, "f32", "masked", "mixed"),
        # the alternatives to one token
        best("best 5 of 1 row", 1, 32768, "f32", 5),
        # a serving batch that returns the 20 best of each token
        best("best 20 of 128", 128, 131072, "bf16", 20),
        # scoring a prompt's tokens
        best("best 8 of 1024", 1024, 50021, "f32", 8),
        # a step of a small batch that decodes
        slots("slots 32 decode", 32, 32, 16, 2048, "i32"),
        # a step of a large batch that decodes
        slots("slots 4096 decode", 4096, 4096, 16, 4096, "i32"),
        # a step that takes in long prompts beside decoding requests
        slots("slots 512 prompts", 512, MOST_TOKENS, 64, 8192, "i64"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sample", "sample", "top_logprobs", "slots"])
    if op == "slots":
        requests = _log_uniform(rng, 1, 8192)
        tokens = max(requests, _log_uniform(rng, requests, MOST_TOKENS)) if rng.random() < 0.6 else requests
        return {"op": op, "requests": requests, "tokens": min(tokens, MOST_TOKENS), "page": rng.choice([8, 16, 48, 64, 128]),
                "context": _log_uniform(rng, 16, 8192), "ints": rng.choice(["i32", "i64"])}
    vocab = _log_uniform(rng, 1000, 262144)
    rows = _log_uniform(rng, 1, min(2048, LARGEST // vocab))
    c = {"op": op, "rows": rows, "vocab": vocab, "dtype": rng.choice(["f32", "f16", "bf16"]),
         "logits": rng.choice(["peaked", "peaked", "masked", "flat"])}
    if op == "sample":
        return {**c, "params": rng.choice(["topk_topp", "mixed", "topp", "topk", "minp", "plain"])}
    return {**c, "n": _log_uniform(rng, 1, 128)}


# -- inputs -----------------------------------------------------------------------
def _logits(case, g):
    R, V = case["rows"], case["vocab"]
    x = torch.randn(R, V, generator=g, device="cuda")
    if case["logits"] == "flat":
        x = x * 1.25
    else:
        # a bulk of unlikely tokens and one in a few hundred that is likely, by a margin that differs from row to row
        x = x * 2.0
        likely = torch.rand(R, V, generator=g, device="cuda") < 1.0 / 300
        lift = torch.empty(R, V, device="cuda").exponential_(0.35, generator=g)
        sharp = 0.5 + torch.rand(R, 1, generator=g, device="cuda")
        x = torch.where(likely, x + lift * sharp, x)
        del likely, lift
        if case["logits"] == "masked":
            # tokens that a grammar or a ban list rules out; now and then all of a row's
            x = torch.where(torch.rand(R, V, generator=g, device="cuda") < 0.25, torch.full_like(x, -math.inf), x)
            x[R // 2] = torch.where(torch.arange(V, device="cuda") == V // 3, 1.0, -math.inf)
            if R > 4:
                x[R // 3] = -math.inf
    return x.to(DTYPES[case["dtype"]])


def _pick(values, R, g, dtype):
    t = torch.tensor(values, dtype=dtype, device="cuda")
    return t[torch.randint(0, len(values), (R,), generator=g, device="cuda")]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "slots":
        return _prepare_slots(case, g)
    R = case["rows"]
    s = {"case": case, "logits": _logits(case, g)}
    if case["op"] == "top_logprobs":
        s["out"] = {"indices": torch.empty(R, case["n"], dtype=torch.int32, device="cuda"),
                    "logprobs": torch.empty(R, case["n"], device="cuda"), "lse": torch.empty(R, device="cuda")}
        return s
    s["uniform"] = torch.rand(R, generator=g, device="cuda")
    p = case["params"]
    f32, i32 = torch.float32, torch.int32
    s["temperature"] = s["top_k"] = s["top_p"] = s["min_p"] = None
    if p == "mixed":  # 0 switches top_k off, 1 switches top_p off, 0 switches min_p off, temperature 0 is greedy
        s["temperature"] = _pick([0.0, 0.6, 0.7, 0.8, 1.0, 1.0, 1.2], R, g, f32)
        s["top_k"] = _pick([0, 0, 20, 40, 50, 100, 200], R, g, i32)
        s["top_p"] = _pick([1.0, 1.0, 0.8, 0.9, 0.95], R, g, f32)
        s["min_p"] = _pick([0.0, 0.0, 0.0, 0.05], R, g, f32)
    else:
        s["temperature"] = _pick([0.7, 0.8, 1.0], R, g, f32) if p != "plain" else torch.ones(R, device="cuda")
        s["top_k"] = _pick([40, 50, 64], R, g, i32) if p in ("topk_topp", "topk") else None
        s["top_p"] = _pick([0.9, 0.95], R, g, f32) if p in ("topk_topp", "topp") else None
        s["min_p"] = _pick([0.02, 0.05, 0.1], R, g, f32) if p == "minp" else None
    s["out"] = {"tokens": torch.empty(R, dtype=torch.int32, device="cuda"), "logprobs": torch.empty(R, device="cuda")}
    return s


def _prepare_slots(case, g):
    R, T, page, I = case["requests"], case["tokens"], case["page"], INTS[case["ints"]]
    # every request has at least one new token; what is left goes to them in lumps of very different sizes
    new = torch.ones(R, dtype=torch.int64, device="cuda")
    if T > R:
        w = torch.log1p(-(torch.arange(R, device="cuda").double() + 0.5) / R).square()
        share = torch.floor(w / w.sum() * (T - R)).to(torch.int64)
        share[-1] += T - R - share.sum()
        new += share[torch.randperm(R, generator=g, device="cuda")]
    ctx = torch.randint(0, case["context"] + 1, (R,), generator=g, device="cuda")
    have = (ctx + page - 1) // page
    need = (ctx + new + page - 1) // page
    width = (case["context"] + int(new.max()) + page - 1) // page
    held, wanted = int(have.sum()), int((need - have).sum())
    pages = torch.randperm(held + wanted + 7, generator=g, device="cuda").to(torch.int32)
    table = torch.full((R, width), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(width, device="cuda")[None, :] < have[:, None]] = pages[:held]
    # the first entries of the list of free pages were taken by earlier steps
    free = torch.cat([torch.full((5,), -1, dtype=torch.int32, device="cuda"), pages[held:]])
    e = lambda n, t: torch.empty(n, dtype=t, device="cuda")  # noqa: E731
    out = {"query_start": e(R + 1, torch.int32), "seq_lens": e(R, I), "positions": e(T, I), "requests": e(T, torch.int32),
           "slots": e(T, torch.int64), "cursor_out": e(1, torch.int32)}
    return {"case": case, "context_lens": ctx.to(I), "new_lens": new.to(I), "block_table": table, "free_pages": free,
            "cursor": torch.full((1,), 5, dtype=torch.int32, device="cuda"), "out": out}


# -- the plain forms ------------------------------------------------------------------
def _finite(logits):
    return torch.nan_to_num(logits, nan=-math.inf, neginf=-math.inf).float()


def _plain_sample(s):
    x = _finite(s["logits"])
    R, V = x.shape
    m = x.amax(1, keepdim=True)
    empty = m == -math.inf
    T = s["temperature"][:, None] if s["temperature"] is not None else torch.ones_like(m)
    greedy = ~(T > 0)
    c = torch.full_like(T, LOG2E) / torch.where(greedy, 1.0, T)
    y = (torch.where(empty, 0.0, m) - x) * c
    w = torch.exp2(-y)
    q = torch.round(w * 2.0**40).to(torch.int64)
    total = q.sum(1, keepdim=True)
    first = torch.where(x == m, torch.arange(V, device=x.device), V).amin(1, keepdim=True)
    kept = q
    if s["top_k"] is not None or s["top_p"] is not None:
        order = torch.sort(x, dim=1, descending=True, stable=True).indices
        sq = torch.gather(q, 1, order)
        if s["top_k"] is not None:
            k = s["top_k"][:, None]
            k = torch.where(k > 0, k, V)
            sq = torch.where(torch.arange(V, device=x.device) < k, sq, 0)
        if s["top_p"] is not None:
            p = s["top_p"][:, None].clamp(0.0, 1.0).double()
            run = torch.cumsum(sq, 1)
            least = torch.ceil(p * run[:, -1:].double()).to(torch.int64).clamp(min=1)
            sq = torch.where((run - sq < least) | (p >= 1.0), sq, 0)
        kept = torch.zeros_like(q).scatter_(1, order, sq)
    if s["min_p"] is not None:
        kept = torch.where(w >= s["min_p"][:, None].clamp(max=1.0), kept, 0)
    run = torch.cumsum(kept, 1)
    mass = run[:, -1:]
    t = torch.minimum(torch.floor(s["uniform"][:, None].double() * mass.double()).to(torch.int64), mass - 1)
    token = torch.where(greedy, first, (run <= t).sum(1, keepdim=True))
    at = torch.gather(y, 1, token.clamp(0, V - 1))
    logprob = -(at * math.log(2.0)) - torch.log(total.float() * 2.0**-40)
    return {"tokens": torch.where(empty, -1, token)[:, 0].to(torch.int32),
            "logprobs": torch.where(empty, -math.inf, logprob)[:, 0]}


def _plain_top_logprobs(s):
    x = _finite(s["logits"])
    V, n = x.shape[1], s["case"]["n"]
    m = x.amax(1, keepdim=True)
    empty = m == -math.inf
    lse = torch.where(empty, 0.0, m) + torch.log(torch.exp(x - torch.where(empty, 0.0, m)).sum(1, keepdim=True))
    # largest value first, lowest index first among equals: both in one whole number
    bits = torch.where(x == 0, 0.0, x).view(torch.int32).to(torch.int64)
    key = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF)) * 2**32 + (2**32 - 1 - torch.arange(V, device=x.device))
    i = 2**32 - 1 - (torch.topk(key, n, dim=1).values & (2**32 - 1))
    v = torch.gather(x, 1, i)
    out = v == -math.inf
    return {"indices": torch.where(out, -1, i).to(torch.int32), "logprobs": torch.where(out, v, v - lse), "lse": lse[:, 0]}


def _plain_slots(s):
    page, out = s["case"]["page"], s["out"]
    ctx, new, table, free = s["context_lens"].long(), s["new_lens"].long(), s["block_table"], s["free_pages"]
    R, width = table.shape
    T, dev = out["slots"].numel(), table.device
    have = torch.clamp((ctx + page - 1) // page, max=width)
    need = torch.clamp((ctx + new + page - 1) // page, max=width)
    took = torch.cumsum(need - have, 0) - (need - have)  # pages that earlier requests take
    col = torch.arange(width, device=dev)[None, :]
    nth = s["cursor"].long() + took[:, None] + col - have[:, None]
    page_of = torch.where(nth < free.numel(), free[nth.clamp(0, free.numel() - 1)], -1)
    fresh = (col >= have[:, None]) & (col < need[:, None])
    table.copy_(torch.where(fresh, page_of, table))
    start = torch.zeros(R + 1, dtype=torch.int64, device=dev)
    start[1:] = torch.cumsum(new, 0)
    i = torch.arange(T, device=dev)
    r = torch.clamp(torch.searchsorted(start, i, right=True) - 1, 0, R - 1)
    inside = i < start[-1]
    pos = ctx[r] + i - start[r]
    held = table[r, torch.clamp(pos // page, 0, width - 1)].long()
    slot = torch.where(inside & (pos // page < width) & (held >= 0), held * page + pos % page, -1)
    I = s["context_lens"].dtype
    return {"query_start": start.to(torch.int32), "seq_lens": (ctx + new).to(I), "positions": torch.where(inside, pos, 0).to(I),
            "requests": torch.where(inside, r, -1).to(torch.int32), "slots": slot, "block_table": table,
            "cursor_out": torch.clamp(s["cursor"] + (need - have).sum().to(torch.int32), max=free.numel())}


# -- one pass ----------------------------------------------------------------------
_sampler = None


def _own():
    global _sampler
    if _sampler is None:
        import os
        import sys
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gpu-forge_b200"))
        import forge_sort
        _sampler = forge_sort.GpuSampler.new()
    return _sampler


def run(s):
    op, o = s["case"]["op"], s["out"]
    if op == "sample":
        if not own:
            return _plain_sample(s)
        _own().sample(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                      min_p=s["min_p"], tokens=o["tokens"], logprobs=o["logprobs"])
        return o
    if op == "top_logprobs":
        if not own:
            return _plain_top_logprobs(s)
        _own().top_logprobs(s["logits"], s["case"]["n"], indices=o["indices"], logprobs=o["logprobs"], lse=o["lse"])
        return o
    if not own:
        return _plain_slots(s)
    _own().plan_slots(s["context_lens"], s["new_lens"], s["block_table"], s["free_pages"], s["cursor"],
                      page_size=s["case"]["page"], query_start=o["query_start"], seq_lens=o["seq_lens"],
                      positions=o["positions"], requests=o["requests"], slots=o["slots"], cursor_out=o["cursor_out"])
    return {**o, "block_table": s["block_table"]}


# -- what a pass cannot do without ---------------------------------------------------
def work(case):
    if case["op"] == "slots":
        R, T, b = case["requests"], case["tokens"], SIZE[case["ints"]]
        # lengths in, lengths and starts out; a position, a request and a slot for each token; the pages taken, read and written
        return {"bytes": R * (3 * b + 4) + T * (b + 4 + 8) + 8 * (T // case["page"]), "flops": 4 * T}
    R, V = case["rows"], case["vocab"]
    read = R * V * SIZE[case["dtype"]]
    if case["op"] == "top_logprobs":
        return {"bytes": read + R * (8 * case["n"] + 4), "flops": 4 * R * V}
    return {"bytes": read + R * 28, "flops": 6 * R * V}


# -- in 64 bits ------------------------------------------------------------------------
def _exact_token(x, w, u, T, k, p, least_w):
    """The token of one row by the definition: x in 64 bits, w the weights in 32 bits (numpy arrays)."""
    import numpy as np
    V = x.size
    if not np.any(x > -np.inf):
        return -1
    if not T > 0:
        return int(np.argmax(x))
    q = np.rint(np.ldexp(w.astype(np.float64), 40)).astype(np.int64)
    keep = np.ones(V, bool)
    if 0 < k < V or p < 1.0:
        down = np.argsort(-x, kind="stable")
        down = down[:k] if 0 < k < V else down
        if p < 1.0:
            run = np.cumsum(q[down])
            least = max(1, math.ceil(max(p, 0.0) * float(run[-1])))
            down = down[: int(np.searchsorted(run, least, side="left")) + 1]
        keep[:] = False
        keep[down] = True
    keep &= w >= min(least_w, 1.0)
    run = np.cumsum(np.where(keep, q, 0))
    t = min(int(math.floor(u * float(run[-1]))), int(run[-1]) - 1)
    return int(np.searchsorted(run, t, side="right"))


def exact(case, seed):
    if case["op"] == "slots":
        return None  # whole numbers only
    import numpy as np
    s = prepare(case, seed)
    dev = s["logits"].device
    R, V = s["logits"].shape
    top = float(torch.finfo(s["logits"].dtype).max)
    if case["op"] == "top_logprobs":
        lse, best = [], []
        for r0 in range(0, R, 64):
            x = s["logits"][r0:r0 + 64].double()
            x = torch.where(torch.isnan(x), -math.inf, x).clamp(max=top)
            l = torch.logsumexp(x, 1, keepdim=True)
            v = torch.sort(x, dim=1, descending=True).values[:, : case["n"]]
            lse.append(l[:, 0])
            best.append(torch.where(v == -math.inf, v, v - l))
        return {"indices": None, "logprobs": torch.cat(best), "lse": torch.cat(lse)}
    if R * V > 70e6:
        return None  # the tokens of so many entries take the host too long
    host = lambda t, off: t.double().cpu().numpy() if t is not None else np.full(R, off)  # noqa: E731
    u, T, k = host(s["uniform"], 0.0), host(s["temperature"], 1.0), host(s["top_k"], 0)
    p, least_w = host(s["top_p"], 1.0), host(s["min_p"], 0.0)
    out = np.full(R, -math.inf)
    for r in range(R):
        x = s["logits"][r].double()
        x = torch.where(torch.isnan(x), -math.inf, x).clamp(max=top)
        m = x.max()
        if float(m) == -math.inf:
            continue
        hot = T[r] > 0
        # the weights are 32-bit numbers by definition: each step rounded as the definition says
        c = np.float32(LOG2E) / np.float32(T[r] if hot else 1.0)
        w = torch.exp2(-((m.float() - x.float()) * float(c)))
        z = (x - m) / (T[r] if hot else 1.0)
        j = _exact_token(x.cpu().numpy(), w.cpu().numpy(), u[r], T[r], int(k[r]), p[r], least_w[r])
        out[r] = float(z[j] - torch.log(torch.exp(z).sum()))
    return {"tokens": None, "logprobs": torch.from_numpy(out).to(dev)}
