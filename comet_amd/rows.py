"""Rows held in 8-bit floating point, scores of queries against them, and score rows as distributions (include/comet_gpu.h: comet_fp8_*,
comet_logprobs_*; the formulas and the treatment of masks, NaN and padding slots stand there).

    store = Fp8Rows(ctx, capacity, dim)
    store.write(vectors, slots)                          # quantised as they are written
    result = store.search(queries, k, scale=20.0)        # the k best slots of each query with log softmax(scale * score)
    rows = store.read(result.slots[0])                   # what the slots hold

The ``*_dev`` methods take device addresses (any HIP allocation on the context's device, for instance ``tensor.data_ptr()``) and queue their work on
``stream``: a raw ``hipStream_t`` such as ``torch.cuda.current_stream().cuda_stream`` (0 is the device's null stream), or ``None`` for the context's lane 0.
They return without waiting and may be captured into a HIP graph.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import numpy as np

from ._lib import BF16, F16, F32, check
from .index import Context

_DTYPE = {"f32": F32, "f16": F16, "bf16": BF16}


def _dtype(name: str) -> int:
    if name not in _DTYPE:
        raise ValueError(f"unknown element type {name!r}: one of {', '.join(_DTYPE)}")
    return _DTYPE[name]


def _i32(x: int, what: str) -> int:
    x = int(x)
    if not -(1 << 31) <= x < 1 << 31:
        raise ValueError(f"{what} {x} does not fit 32 bits")
    return x


def _i64(x: int, what: str) -> int:
    x = int(x)
    if not -(1 << 63) <= x < 1 << 63:
        raise ValueError(f"{what} {x} does not fit 64 bits")
    return x


def _host(a: np.ndarray):
    return a.ctypes.data_as(C.c_void_p)


@dataclass
class Fp8SearchResult:
    """Of each query: the best slots (-1 where none is left), their log-probabilities, log sum exp(scale * score) and the distribution's entropy."""
    slots: np.ndarray
    logprobs: np.ndarray
    logsum: np.ndarray
    entropy: np.ndarray


class Fp8Rows:
    """A store of ``capacity`` slots of ``dim`` numbers in e4m3 with a power-of-two scale per block of 128 (comet_fp8_rows)."""

    def __init__(self, ctx: Context, capacity: int, dim: int):
        self.ctx, self.lib = ctx, ctx.lib
        h = C.c_void_p()
        check(self.lib.comet_fp8_create(ctx.h, _i64(capacity, "capacity"), _i32(dim, "dimension"), C.byref(h)))
        self.h = h
        self.capacity, self.dim = int(capacity), int(dim)

    def close(self):
        if getattr(self, "h", None):
            h, self.h = self.h, None
            check(self.lib.comet_fp8_destroy(h))

    def __del__(self):
        try:
            if getattr(self.ctx, "h", None):
                self.close()
        except Exception:
            pass

    def _stream(self, stream: int | None) -> C.c_void_p:
        return C.c_void_p(self.ctx.stream if stream is None else int(stream))

    # device arrays
    def write_dev(self, vecs: int, n: int, dtype: str = "f32", ld: int | None = None, slots: int = 0, first: int = 0, stream: int | None = None) -> None:
        """row i of ``vecs`` (n rows, ``ld`` elements apart) to slot slots[i] (device int64; outside the store: skipped), or first + i"""
        check(self.lib.comet_fp8_write_dev(self.h, C.c_void_p(slots or None), _i64(first, "first slot"), C.c_void_p(vecs or None), _dtype(dtype),
                                           _i64(self.dim if ld is None else ld, "row stride"), _i64(n, "row count"), self._stream(stream)))

    def read_dev(self, out: int, n: int, dtype: str = "f32", ld: int | None = None, slots: int = 0, first: int = 0, stream: int | None = None) -> None:
        """out[i] = the row in slot slots[i] (outside the store: zeros), or first + i"""
        check(self.lib.comet_fp8_read_dev(self.h, C.c_void_p(slots or None), _i64(first, "first slot"), C.c_void_p(out or None), _dtype(dtype),
                                          _i64(self.dim if ld is None else ld, "row stride"), _i64(n, "row count"), self._stream(stream)))

    def scores_dev(self, queries: "Fp8Rows", m: int, out: int, dtype: str = "f32", ld: int | None = None, q_first: int = 0, first: int = 0, n: int | None = None,
                   stream: int | None = None) -> None:
        """out[i][j] = <queries' slot q_first + i, this store's slot first + j>, m x n (default: all slots from ``first``)"""
        n = self.capacity - first if n is None else n
        check(self.lib.comet_fp8_scores_dev(queries.h, _i64(q_first, "first query"), _i64(m, "query count"), self.h, _i64(first, "first slot"), _i64(n, "row count"), C.c_void_p(out or None),
                                            _dtype(dtype), _i64(n if ld is None else ld, "row stride"), self._stream(stream)))

    # host arrays
    def _slots(self, slots, n: int) -> np.ndarray:
        s = np.ascontiguousarray(slots, dtype=np.int64).reshape(-1)
        if len(s) != n:
            raise ValueError(f"{n} rows and {len(s)} slots")
        return s

    def write(self, vecs, slots) -> None:
        v = np.ascontiguousarray(vecs, dtype=np.float32)
        if v.ndim == 1:
            v = v[None, :]
        if v.ndim != 2 or v.shape[1] != self.dim:
            raise ValueError(f"vector dimension mismatch: expected {self.dim}, got {v.shape[-1]}")
        s = self._slots(slots, v.shape[0])
        check(self.lib.comet_fp8_write(self.h, _host(s), _host(v), v.shape[0]))

    def read(self, slots) -> np.ndarray:
        s = np.ascontiguousarray(slots, dtype=np.int64).reshape(-1)
        out = np.empty((len(s), self.dim), np.float32)
        check(self.lib.comet_fp8_read(self.h, _host(s), len(s), _host(out)))
        return out

    def search(self, queries, k: int, scale: float = 1.0, first: int = 0, n: int | None = None) -> Fp8SearchResult:
        """the k slots of [first, first + n) of largest scale * score for each query, as a distribution over all n"""
        q = np.ascontiguousarray(queries, dtype=np.float32)
        if q.ndim == 1:
            q = q[None, :]
        if q.ndim != 2 or q.shape[1] != self.dim:
            raise ValueError(f"query dimension mismatch: expected {self.dim}, got {q.shape[-1]}")
        n = self.capacity - first if n is None else n
        B, k = _i32(q.shape[0], "query count"), _i32(k, "k")
        kk = k if 0 <= k <= 128 else 0           # any other is refused below
        r = Fp8SearchResult(np.empty((B, kk), np.int64), np.empty((B, kk), np.float32), np.empty(B, np.float32), np.empty(B, np.float32))
        check(self.lib.comet_fp8_search(self.h, _i64(first, "first slot"), _i64(n, "row count"), _host(q), B, C.c_float(scale), k, _host(r.slots), _host(r.logprobs), _host(r.logsum), _host(r.entropy)))
        return r


class LogProbs:
    """Score rows as distributions: log-probabilities of given columns, entropy, the k best columns (comet_logprobs_dev). Holds the workspace for calls of up
    to ``m`` rows, ``n`` columns and ``k`` best; calls that may run at once each need a LogProbs of their own."""

    def __init__(self, ctx: Context, m: int, n: int, k: int):
        self.ctx, self.lib = ctx, ctx.lib
        size = C.c_size_t()
        check(self.lib.comet_logprobs_work_bytes(_i64(m, "row count"), _i64(n, "column count"), _i32(k, "k"), C.byref(size)))
        self.work_bytes = size.value
        self.work = ctx.alloc(self.work_bytes) if self.work_bytes else 0

    def close(self):
        if getattr(self, "work", 0):
            w, self.work = self.work, 0
            self.ctx.free(w)

    def __del__(self):
        try:
            if getattr(self.ctx, "h", None):
                self.close()
        except Exception:
            pass

    def run_dev(self, scores: int, dtype: str, m: int, n: int, *, out_logsum: int, out_entropy: int, ld: int | None = None, scale: float = 1.0, counts: int = 0,
                targets: int = 0, n_targets: int = 0, out_logprobs: int = 0, k: int = 0, out_ids: int = 0, out_top_logprobs: int = 0, stream: int | None = None) -> None:
        """scores: m x n, ``ld`` elements apart; counts (m), targets (m x n_targets) and out_ids (m x k) are int32, the other outputs float32"""
        p = lambda a: C.c_void_p(a or None)  # noqa: E731
        check(self.lib.comet_logprobs_dev(self.ctx.h, p(scores), _dtype(dtype), _i64(n if ld is None else ld, "row stride"), _i64(m, "row count"), _i64(n, "column count"), p(counts), C.c_float(scale), p(targets),
                                          _i32(n_targets, "target count"), _i32(k, "k"), p(out_logprobs), p(out_logsum), p(out_entropy), p(out_ids), p(out_top_logprobs), p(self.work),
                                          self.work_bytes, C.c_void_p(self.ctx.stream if stream is None else int(stream))))
