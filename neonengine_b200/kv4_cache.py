"""Python host mirror of the 4-bit paged key/value cache (include/neon_kv4.h).

One :class:`Kv4Cache` serves all layers of a model; the caches themselves are the caller's uint8
tensors ``[n_pages, n_kv_heads, record_bytes]`` (one per layer).  A :class:`Kv4Batch` describes the
sequences of a step and serves every layer of that step.  Calls are enqueued on the current stream (or
``stream``); errors become ``RuntimeError``, unusable arguments ``ValueError``.  torch only owns device
memory and streams; every kernel runs inside ``libneon_moe.so``.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _ints(t, name: str, dims: int):
    _need(t.is_cuda and t.dtype == torch.int32 and t.dim() == dims and (t.shape[-1] <= 1 or t.stride(-1) == 1),
          f"{name}: a contiguous int32 CUDA tensor of {dims} dimension(s)")
    return t.data_ptr()


class Kv4Batch:
    """Sequences of a step: cache lengths (new tokens included), their pages, and which rows are whose.  The tensors
    are read when the kernels run; they may be rewritten in place between the replays of a captured graph."""

    def __init__(self, seq_lens, page_table, cu_q=None):
        n = seq_lens.shape[0]
        _need(page_table.dim() == 2 and page_table.shape[0] == n, "page_table: [batch, pages]")
        _need(cu_q is None or cu_q.shape[0] == n + 1, "cu_q: [batch + 1]")
        _need(all(t is None or t.device == seq_lens.device for t in (page_table, cu_q)), "the batch's tensors are on several devices")
        self._keep = (seq_lens, page_table, cu_q)
        self.device = seq_lens.device
        self.batch = n
        self.one_each = cu_q is None
        self._c = _lib.NeonKv4Batch(_ints(seq_lens, "seq_lens", 1), None if cu_q is None else _ints(cu_q, "cu_q", 1),
                                    _ints(page_table, "page_table", 2), page_table.stride(0) if n > 1 else page_table.shape[1],
                                    page_table.shape[1], n, 0)
        self._ref = ctypes.byref(self._c)
        self._scratch = {}


class Kv4Cache:
    def __init__(self, n_q_heads: int, n_kv_heads: int, head_dim: int, page_size: int = 64, device: int = 0):
        self._lib = _lib.load()
        self.n_q_heads, self.n_kv_heads, self.head_dim, self.page_size = int(n_q_heads), int(n_kv_heads), int(head_dim), int(page_size)
        self.device = torch.device("cuda", int(device))
        cfg = _lib.NeonKv4Config(self.n_q_heads, self.n_kv_heads, self.head_dim, self.page_size, int(device))
        handle = ctypes.c_void_p()
        rc = self._lib.neon_kv4_create(ctypes.byref(cfg), ctypes.byref(handle))
        if rc != 0:
            raise RuntimeError(f"neon_kv4_create failed ({rc}): {self._lib.neon_kv4_last_error(None).decode()}")
        self._h = handle
        self.record_bytes = int(self._lib.neon_kv4_record_bytes(handle))

    def _check(self, rc: int, what: str) -> None:
        if rc != 0:
            raise RuntimeError(f"{what} failed ({rc}): {self._lib.neon_kv4_last_error(self._h).decode()}")

    def _stream(self, stream) -> int:
        return (torch.cuda.current_stream(self.device) if stream is None else stream).cuda_stream

    def _place(self, batch: Kv4Batch, cache) -> int:
        _need(cache.dtype == torch.uint8 and cache.dim() == 3 and cache.shape[1] == self.n_kv_heads and cache.shape[2] == self.record_bytes
              and cache.is_contiguous(), f"cache: contiguous uint8 [n_pages, {self.n_kv_heads}, {self.record_bytes}]")
        _need(cache.device == self.device and batch.device == self.device, f"cache and batch have to be on {self.device}")
        batch._c.n_pages = cache.shape[0]
        return cache.data_ptr()

    def _rows(self, t, heads: int, name: str, rows=None) -> int:
        """Checks [rows, heads, head_dim] with whole rows apart by any stride; returns the stride in elements."""
        _need(t.dim() == 3 and t.shape[1] == heads and t.shape[2] == self.head_dim and (rows is None or t.shape[0] == rows),
              f"{name}: [rows, {heads}, {self.head_dim}]")
        _need(t.stride(2) == 1 and (heads == 1 or t.stride(1) == self.head_dim), f"{name}: the heads of a row have to be contiguous")
        _need(t.device == self.device, f"{name} has to be on {self.device}")
        return t.stride(0) if t.shape[0] > 1 else heads * self.head_dim

    # -- caches and batches ----------------------------------------------------------------
    def new_cache(self, n_pages: int):
        """Pages for one layer; zeros read as zeros."""
        return torch.zeros((n_pages, self.n_kv_heads, self.record_bytes), dtype=torch.uint8, device=self.device)

    def batch(self, seq_lens, page_table, cu_q=None) -> Kv4Batch:
        return Kv4Batch(seq_lens, page_table, cu_q)

    # -- execution -----------------------------------------------------------------------------
    def append(self, batch: Kv4Batch, cache, q, k, v, inv_freq, mscale: float = 1.0, out=None, stream=None):
        """Rotates ``q`` and ``k`` [rows, heads, head_dim] (fp32, bf16 or fp16; columns of one projection's output will do) by
        their rows' positions and writes ``k`` and ``v`` to the pages.  Returns the rotated queries (bf16, or fp16 for fp16
        input, or ``out``'s type); ``q`` may be None."""
        rows = k.shape[0]
        ks, vs = self._rows(k, self.n_kv_heads, "k"), self._rows(v, self.n_kv_heads, "v", rows)
        _need(k.dtype in _DTYPES and v.dtype == k.dtype and (q is None or q.dtype == k.dtype), "q, k and v: one of float32, bfloat16, float16")
        _need(inv_freq.dtype == torch.float32 and inv_freq.shape == (self.head_dim // 2,) and inv_freq.is_contiguous()
              and inv_freq.device == self.device, f"inv_freq: float32 [{self.head_dim // 2}]")
        qs = 0
        if q is not None:
            qs = self._rows(q, self.n_q_heads, "q", rows)
            if out is None:
                out = torch.empty((rows, self.n_q_heads, self.head_dim), dtype=torch.float16 if q.dtype == torch.float16 else torch.bfloat16,
                                  device=self.device)
            self._rows(out, self.n_q_heads, "out", rows)
            _need(out.dtype in (torch.bfloat16, torch.float16) and out.is_contiguous(), "out: contiguous, bfloat16 or float16")
        cache_ptr = self._place(batch, cache)
        self._check(self._lib.neon_kv4_append(
            self._h, batch._ref, cache_ptr, rows, _DTYPES[k.dtype], None if q is None else q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs,
            inv_freq.data_ptr(), mscale, None if q is None else out.data_ptr(), 0 if q is None else _DTYPES[out.dtype], self._stream(stream)),
            "neon_kv4_append")
        return out if q is not None else None

    def read(self, batch: Kv4Batch, cache, rows: int | None = None, dtype=torch.bfloat16, out=None, stream=None):
        """(keys, values) [rows, n_kv_heads, head_dim] that the cache holds at the positions of the batch's rows, bf16 or
        fp32; ``out``: a pair of tensors to write to."""
        if out is None:
            rows = batch.batch if rows is None else rows
            out = [torch.zeros((rows, self.n_kv_heads, self.head_dim), dtype=dtype, device=self.device) for _ in range(2)]
        rows = out[0].shape[0]
        for t in out:
            self._rows(t, self.n_kv_heads, "out", rows)
            _need(t.dtype in (torch.bfloat16, torch.float32) and t.dtype == out[0].dtype and t.is_contiguous(), "out: contiguous, bfloat16 or float32")
        cache_ptr = self._place(batch, cache)
        self._check(self._lib.neon_kv4_read(self._h, batch._ref, cache_ptr, rows, out[0].data_ptr(), out[1].data_ptr(), _DTYPES[out[0].dtype],
                                            self._stream(stream)), "neon_kv4_read")
        return out[0], out[1]

    def attend(self, batch: Kv4Batch, cache, q, sinks=None, window: int = 0, scale: float | None = None, max_rows: int | None = None,
               out=None, stream=None):
        """Attention of ``q`` [rows, n_q_heads, head_dim] (bf16 or fp16, rotated) over the cache; ``sinks``: bf16 [n_q_heads] logits of the
        softmax denominator; ``window`` > 0: only the last so many positions; ``scale``: default head_dim ** -0.5; ``max_rows``: the
        most rows of a sequence, if the host knows it (speed only)."""
        rows = q.shape[0]
        qs = self._rows(q, self.n_q_heads, "q")
        _need(q.dtype in (torch.bfloat16, torch.float16), "q: bfloat16 or float16")
        _need(sinks is None or (sinks.dtype == torch.bfloat16 and sinks.shape == (self.n_q_heads,) and sinks.is_contiguous()
                                and sinks.device == self.device), f"sinks: bfloat16 [{self.n_q_heads}]")
        if out is None:
            out = torch.empty((rows, self.n_q_heads, self.head_dim), dtype=q.dtype, device=self.device)
        self._rows(out, self.n_q_heads, "out", rows)
        _need(out.dtype == q.dtype and out.is_contiguous(), "out: contiguous, q's type")
        if max_rows is None:
            max_rows = 1 if batch.one_each else rows
        cache_ptr = self._place(batch, cache)
        size = batch._scratch.get((rows, max_rows, self._h.value))
        if size is None:
            size = batch._scratch[(rows, max_rows, self._h.value)] = int(self._lib.neon_kv4_attend_workspace(self._h, batch._ref, rows, max_rows))
        st = torch.cuda.current_stream(self.device) if stream is None else stream
        scratch = torch.empty(size, dtype=torch.uint8, device=self.device)
        if stream is not None:
            scratch.record_stream(stream)
        self._check(self._lib.neon_kv4_attend(
            self._h, batch._ref, cache_ptr, rows, _DTYPES[q.dtype], q.data_ptr(), qs, None if sinks is None else sinks.data_ptr(), window,
            self.head_dim ** -0.5 if scale is None else scale, max_rows, out.data_ptr(), scratch.data_ptr(), size, st.cuda_stream),
            "neon_kv4_attend")
        return out

    # -- inspection ----------------------------------------------------------------------------
    def status(self) -> int:
        """Reads and clears the status bits (blocking): 1 a page id outside the cache, 2 a sequence longer than its table
        or cu_q not ascending, 4 a wait inside a kernel ran out."""
        word = ctypes.c_int(0)
        self._check(self._lib.neon_kv4_status(self._h, ctypes.byref(word)), "neon_kv4_status")
        return word.value

    @property
    def launch_count(self) -> int:
        return int(self._lib.neon_kv4_launch_count(self._h))

    def close(self) -> None:
        if getattr(self, "_h", None):
            self._lib.neon_kv4_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
