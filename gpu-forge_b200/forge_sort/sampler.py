"""GpuSampler -- the calls of a model's decode step over the CUDA C ABI:
sampling a token of every row of logits (fs_sample_rows), the best
log-probabilities of every row (fs_top_logprobs), and the block tables and
slot maps of a batch's step over a paged cache (fs_plan_slots).

No counterpart in the reference.  Arguments are torch tensors on the
sampler's device; what a call returns are tensors too, new ones or those the
caller passes to be written.  Calls enqueue on torch's current stream (or the
stream the sampler was made with) and return without waiting unless
sync=True.  A device-side failure (a token without a slot) is raised, once, by
whatever waits next on the sampler: synchronize(), or any call with sync=True,
one that succeeded itself among them.  They keep no state between them.
"""
from __future__ import annotations

from typing import NamedTuple

from . import _lib
from .errors import GpuExecution
from .sorter import GpuSorter, _stream_handle

BEST_MAX = 1024  # n of top_logprobs


class SlotPlan(NamedTuple):
    """What plan_slots writes (fs_plan_slots in include/forgesort.h)."""
    query_start: object  # int32 [requests + 1]: where each request's tokens start
    seq_lens: object     # [requests]: context + new
    positions: object    # [capacity]: of each token in its request, 0 beyond the last
    requests: object     # int32 [capacity]: the token's request, -1 beyond the last
    slots: object        # int64 [capacity]: page * page_size + offset, -1 where there is none
    cursor_out: object   # int32 [1]: the cursor for the next step


class GpuSampler:
    """Row sampling, best log-probabilities and slot plans on one CUDA device.

    new() / GpuSampler() follow torch's current stream of device 0;
    with_context(device, stream) enqueues on the caller's stream, which the
    arguments must be ready on and which the results belong to."""

    def __init__(self, device: int = 0, stream=None):
        import torch
        self._torch = torch
        self._s = GpuSorter(device, stream)
        self._L = _lib.load()
        self.device = int(device)
        self._dev = torch.device("cuda", self.device)
        self._fixed = _stream_handle(stream)
        self._last = self._fixed
        # With a stream of its own, what a call makes (outputs, numbers spread over the rows) is made on that stream:
        # on torch's current one it might still be filled, or its memory still be used, when the kernel runs.
        if self._fixed is None:
            self._own = None
        elif self._fixed == 1:  # cudaStreamLegacy
            self._own = torch.cuda.default_stream(self._dev)
        else:
            self._own = torch.cuda.ExternalStream(self._fixed, device=self._dev)
        self._logits = {torch.float32: _lib.LOGITS_F32, torch.float16: _lib.LOGITS_F16,
                        torch.bfloat16: _lib.LOGITS_BF16}
        # torch.cuda.current_stream() makes an object; this gives its handle alone
        self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        self._index = {torch.int32: 4, torch.int64: 8}

    @classmethod
    def new(cls) -> "GpuSampler":
        return cls(0, None)

    @classmethod
    def with_context(cls, device: int, stream) -> "GpuSampler":
        return cls(device, stream)

    def close(self) -> None:
        self._s.close()

    def synchronize(self) -> None:
        """Wait for the last call's stream and for the slot plans on all others,
        and report device-side failures.  Replays of a captured graph on another
        stream are the caller's to wait for before."""
        if self._last is not None and self._L.fs_stream_synchronize(self._last):
            raise GpuExecution(self._L.fs_last_error(None).decode())
        self._s.synchronize()

    def last_launch_count(self) -> int:
        return self._s.last_launch_count()

    # -- plumbing -----------------------------------------------------------------
    def _stream(self):
        if self._fixed is None:
            raw = self._raw_stream
            h = raw(self.device) if raw else self._torch.cuda.current_stream(self._dev).cuda_stream
            self._last = h or 1  # 1: cudaStreamLegacy
        return self._last

    def _made(self, make, *args, **kw):
        if self._own is None:
            return make(*args, **kw)
        with self._torch.cuda.stream(self._own):
            return make(*args, **kw)

    def _vec(self, t, name: str, n: int, dtype):
        """Device address of a contiguous tensor of n elements (None: any number) of dtype."""
        try:  # the checks below in their cheapest form
            if t.dtype is dtype and (n is None or t.numel() == n) and t.is_contiguous() and t.get_device() == self.device:
                return t.data_ptr()
        except AttributeError:
            pass
        if not isinstance(t, self._torch.Tensor):
            raise TypeError(f"{name} must be a tensor")
        if t.dtype is not dtype:
            raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
        if n is not None and t.numel() != n:
            raise ValueError(f"{name} has {t.numel()} elements, expected {n}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        if t.device != self._dev:
            raise ValueError(f"{name} is on {t.device}, the sampler on {self._dev}")
        return t.data_ptr()

    def _param(self, v, name: str, n: int, dtype, keep: list):
        """A per-row parameter: None (off), a number for all rows, or a tensor."""
        if v is None:
            return None
        if isinstance(v, (int, float)):
            v = self._made(self._torch.full, (n,), v, dtype=dtype, device=self._dev)
            keep.append(v)  # until the call has been enqueued; later reuse is ordered by the stream
        return self._vec(v, name, n, dtype)

    def _out(self, t, name: str, shape, dtype):
        if t is None:
            t = self._made(self._torch.empty, shape, dtype=dtype, device=self._dev)
            return t, t.data_ptr()
        try:
            if t.shape == shape and t.dtype is dtype and t.is_contiguous() and t.get_device() == self.device:
                return t, t.data_ptr()
        except AttributeError:
            raise TypeError(f"{name} must be a tensor") from None
        if t.shape != shape:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")
        n = shape[0] if len(shape) == 1 else shape[0] * shape[1]
        return t, self._vec(t, name, n, dtype)

    def _rows(self, x):
        if not isinstance(x, self._torch.Tensor):
            raise TypeError("logits must be a tensor")
        code = self._logits.get(x.dtype)
        if code is None:
            raise TypeError(f"logits has dtype {x.dtype}, expected float32, float16 or bfloat16")
        if x.dim() != 2:
            raise ValueError(f"logits must be 2-D (rows x vocabulary), got {x.dim()}-D")
        rows, cols = x.shape
        stride, step = x.stride()
        if step != 1 and cols > 1:
            raise ValueError(f"logits must have stride 1 along the vocabulary, got {step}")
        if x.get_device() != self.device:
            raise ValueError(f"logits is on {x.device}, the sampler on {self._dev}")
        return code, rows, cols, stride

    # -- the operators ---------------------------------------------------------------
    def sample(self, logits, uniform, *, temperature=None, top_k=None, top_p=None, min_p=None, tokens=None,
               logprobs=None, sync: bool = False):
        """(tokens int32 [rows], logprobs f32 [rows]): one token of every row.

        logits: [rows, vocabulary] f32, f16 or bf16, rows any distance apart;
        uniform: f32 [rows], one number of [0, 1) per row.  temperature, top_p,
        min_p (f32 [rows] or a number) and top_k (int32 [rows] or a number)
        filter as fs_sample_rows describes; None switches each off.  A number
        costs a launch that spreads it over the rows; a loop keeps tensors.
        What comes back is detached: no gradient reaches the logits.  Equal
        inputs give equal tokens, whatever the batch around them; a row with
        nothing above -inf gives token -1."""
        t = self._torch
        code, rows, cols, stride = self._rows(logits)
        f32, keep = t.float32, []
        u = self._vec(uniform, "uniform", rows, f32)
        T = self._param(temperature, "temperature", rows, f32, keep)
        k = self._param(top_k, "top_k", rows, t.int32, keep)
        p = self._param(top_p, "top_p", rows, f32, keep)
        mp = self._param(min_p, "min_p", rows, f32, keep)
        tokens, tp = self._out(tokens, "tokens", (rows,), t.int32)
        logprobs, lp = self._out(logprobs, "logprobs", (rows,), f32)
        rc = self._L.fs_sample_rows(self._s._h, code, logits.data_ptr(), rows, cols, stride, T, k, p, mp, u, tp, lp,
                                    sync, self._stream())
        if rc:
            self._s._call(rc)
        return tokens, logprobs

    def top_logprobs(self, logits, n: int, *, indices=None, logprobs=None, lse=None, sync: bool = False):
        """(indices int32 [rows, n], logprobs f32 [rows, n], lse f32 [rows]):
        the n largest logits of every row in descending order (ties: lowest
        index first), their log-softmax, and the rows' log-sum-exp, detached
        from the logits' graph.  Places beyond a row's entries above -inf hold
        index -1, log-probability -inf."""
        t = self._torch
        code, rows, cols, stride = self._rows(logits)
        indices, ip = self._out(indices, "indices", (rows, n), t.int32)
        logprobs, lp = self._out(logprobs, "logprobs", (rows, n), t.float32)
        lse, sp = self._out(lse, "lse", (rows,), t.float32)
        rc = self._L.fs_top_logprobs(self._s._h, code, logits.data_ptr(), rows, cols, stride, n, ip, lp, sp, sync,
                                     self._stream())
        if rc:
            self._s._call(rc)
        return indices, logprobs, lse

    def plan_slots(self, context_lens, new_lens, block_table, free_pages, cursor, *, page_size: int, capacity=None,
                   query_start=None, seq_lens=None, positions=None, requests=None, slots=None, cursor_out=None,
                   sync: bool = False) -> SlotPlan:
        """Plans the step in which request r, with context_lens[r] tokens in
        a paged cache, gets new_lens[r] more: takes the pages it needs beyond
        those it holds from free_pages[cursor:], in request order, enters them
        in its row of block_table (int32 [requests, width], changed in place)
        and gives every token of the step its request, position and slot.

        Lengths are int32 or int64 (seq_lens and positions take their type).
        capacity is the number of token places to fill: the size of
        positions / requests / slots where one of them is passed."""
        t = self._torch
        I = getattr(context_lens, "dtype", None)
        ib = self._index.get(I)
        if ib is None:
            raise TypeError("context_lens must be a tensor of int32 or int64")
        R = context_lens.numel()
        c = self._vec(context_lens, "context_lens", R, I)
        w = self._vec(new_lens, "new_lens", R, I)
        if not isinstance(block_table, t.Tensor) or block_table.dtype is not t.int32:
            raise TypeError("block_table must be a tensor of int32")
        shape = block_table.shape
        if len(shape) != 2 or shape[0] != R:
            raise ValueError(f"block_table must be [{R}, width], got {tuple(shape)}")
        width = shape[1]
        tstride, tstep = block_table.stride()
        if tstep != 1 and width > 1:
            raise ValueError("block_table must have stride 1 along a row")
        if block_table.get_device() != self.device:
            raise ValueError(f"block_table is on {block_table.device}, the sampler on {self._dev}")
        f = self._vec(free_pages, "free_pages", None, t.int32)
        nf = free_pages.numel()
        cur = self._vec(cursor, "cursor", 1, t.int32)
        if capacity is None:
            for o in (slots, positions, requests):
                if o is not None:
                    capacity = o.numel()
                    break
            else:
                raise ValueError("capacity is required when none of slots, positions and requests is passed")
        query_start, qp = self._out(query_start, "query_start", (R + 1,), t.int32)
        seq_lens, lp = self._out(seq_lens, "seq_lens", (R,), I)
        positions, pp = self._out(positions, "positions", (capacity,), I)
        requests, rp = self._out(requests, "requests", (capacity,), t.int32)
        slots, sp = self._out(slots, "slots", (capacity,), t.int64)
        cursor_out, op = self._out(cursor_out, "cursor_out", (1,), t.int32)
        rc = self._L.fs_plan_slots(self._s._h, ib, c, w, R, page_size, block_table.data_ptr(), width, tstride, f, nf,
                                   cur, qp, lp, pp, rp, sp, capacity, op, sync, self._stream())
        if rc:
            self._s._call(rc)
        return SlotPlan(query_start, seq_lens, positions, requests, slots, cursor_out)
