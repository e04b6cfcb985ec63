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


_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


class Kv4Batch:
    """Sequences of a step: cache lengths (new tokens included), their pages, and which rows are whose.  The tensors
    are read when the kernels run; they may be rewritten in place between the replays of a captured graph."""

    def __init__(self, seq_lens, page_table, cu_q=None):
        shape, stride = page_table.shape, page_table.stride()
        if seq_lens.dtype is not torch.int32 or seq_lens.dim() != 1 or not seq_lens.is_contiguous() or not seq_lens.is_cuda:
            raise ValueError("seq_lens: contiguous int32 [batch] in device memory")
        n, index = seq_lens.shape[0], seq_lens.get_device()
        if page_table.dtype is not torch.int32 or len(shape) != 2 or shape[0] != n or (stride[1] != 1 and shape[1] > 1) \
                or page_table.get_device() != index:
            raise ValueError("page_table: int32 [batch, pages], rows contiguous, where seq_lens is")
        if cu_q is not None and (cu_q.dtype is not torch.int32 or cu_q.shape != (n + 1,) or not cu_q.is_contiguous() or cu_q.get_device() != index):
            raise ValueError("cu_q: contiguous int32 [batch + 1] where seq_lens is")
        self._keep = (seq_lens, page_table, cu_q)
        self.device_index, self.batch, self.one_each = index, n, cu_q is None
        self._c = _lib.NeonKv4Batch(seq_lens.data_ptr(), None if cu_q is None else cu_q.data_ptr(), page_table.data_ptr(),
                                    stride[0] if n > 1 else shape[1], shape[1], n, 0)
        self._ref = ctypes.byref(self._c)


class Kv4Cache:
    def __init__(self, n_q_heads: int, n_kv_heads: int, head_dim: int, page_size: int = 64, device: int = 0):
        self._lib = _lib.load()
        self.n_q_heads, self.n_kv_heads, self.head_dim, self.page_size = int(n_q_heads), int(n_kv_heads), int(head_dim), int(page_size)
        self.device, self._index = torch.device("cuda", int(device)), int(device)
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

    def _place(self, batch: Kv4Batch, cache) -> int:
        shape = cache.shape
        if cache.dtype is not torch.uint8 or len(shape) != 3 or shape[1] != self.n_kv_heads or shape[2] != self.record_bytes \
                or not cache.is_contiguous() or cache.get_device() != self._index or batch.device_index != self._index:
            raise ValueError(f"cache: contiguous uint8 [n_pages, {self.n_kv_heads}, {self.record_bytes}] on {self.device}, where the batch is")
        batch._c.n_pages = shape[0]
        return cache.data_ptr()

    def _rows(self, t, heads: int, rows: int, name: str) -> int:
        """Checks [rows, heads, head_dim] with whole rows any stride apart; returns the stride in elements."""
        stride = t.stride()
        if t.shape != (rows, heads, self.head_dim) or stride[2] != 1 or (stride[1] != self.head_dim and heads > 1) \
                or t.get_device() != self._index:
            raise ValueError(f"{name}: [{rows}, {heads}, {self.head_dim}] on {self.device}, the heads of a row contiguous")
        return stride[0] if rows > 1 else heads * self.head_dim

    # -- caches and batches ----------------------------------------------------------------
    def new_cache(self, n_pages: int):
        """Pages for one layer; zeros read as zeros."""
        return torch.zeros((n_pages, self.n_kv_heads, self.record_bytes), dtype=torch.uint8, device=self.device)

    def batch(self, seq_lens, page_table, cu_q=None) -> Kv4Batch:
        return Kv4Batch(seq_lens, page_table, cu_q)

    # -- execution -----------------------------------------------------------------------------
    def _on(self, stream, call, *args):
        """The call with ``stream`` as the current one, so that what it allocates belongs to that stream too."""
        _need(stream.device_index == self._index, "stream: one of the cache's device")
        with torch.cuda.stream(stream):
            return call(*args)

    def append(self, batch: Kv4Batch, cache, q, k, v, inv_freq, mscale: float = 1.0, out=None, stream=None):
        """Rotates ``q`` and ``k`` [rows, heads, head_dim] (fp32, bf16 or fp16; columns of one projection's output will do) by
        their rows' positions and writes ``k`` and ``v`` to the pages.  Returns the rotated queries (bf16, or fp16 for fp16
        input, or ``out``'s type); ``q`` may be None."""
        if stream is not None:
            return self._on(stream, self.append, batch, cache, q, k, v, inv_freq, mscale, out)
        rows = k.shape[0]
        ks, vs = self._rows(k, self.n_kv_heads, rows, "k"), self._rows(v, self.n_kv_heads, rows, "v")
        dtype = k.dtype
        _need(dtype in _DTYPES and v.dtype is dtype and (q is None or q.dtype is dtype), "q, k and v: one of float32, bfloat16, float16")
        _need(inv_freq.dtype is torch.float32 and inv_freq.shape == (self.head_dim // 2,) and inv_freq.is_contiguous()
              and inv_freq.get_device() == self._index, f"inv_freq: float32 [{self.head_dim // 2}]")
        qs = out_dtype = 0
        q_ptr = out_ptr = None
        if q is not None:
            qs = self._rows(q, self.n_q_heads, rows, "q")
            if out is None:
                out = torch.empty((rows, self.n_q_heads, self.head_dim), dtype=torch.float16 if dtype is torch.float16 else torch.bfloat16,
                                  device=self.device)
            elif out.dtype not in (torch.bfloat16, torch.float16) or out.shape != q.shape or not out.is_contiguous() or out.get_device() != self._index:
                raise ValueError("out: contiguous, bfloat16 or float16, q's shape")
            q_ptr, out_ptr, out_dtype = q.data_ptr(), out.data_ptr(), _DTYPES[out.dtype]
        rc = self._lib.neon_kv4_append(self._h, batch._ref, self._place(batch, cache), rows, _DTYPES[dtype], q_ptr, qs, k.data_ptr(), ks, v.data_ptr(),
                                       vs, inv_freq.data_ptr(), mscale, out_ptr, out_dtype,
                                       _stream_of(self._index))
        if rc:
            self._check(rc, "neon_kv4_append")
        return out if q is not None else None

    def read(self, batch: Kv4Batch, cache, rows: int | None = None, dtype=torch.bfloat16, out=None, stream=None):
        """(keys, values) [rows, n_kv_heads, head_dim] that the cache holds at the positions of the batch's rows, bf16 or
        fp32; ``out``: a pair of tensors to write to.  A batch with row offsets needs ``rows`` or ``out``, as the host does not know
        how many rows it has."""
        if stream is not None:
            return self._on(stream, self.read, batch, cache, rows, dtype, out)
        if out is None:
            _need(rows is not None or batch.one_each, "rows: the number of rows of a batch with row offsets")
            rows = batch.batch if rows is None else rows
            out = [torch.zeros((rows, self.n_kv_heads, self.head_dim), dtype=dtype, device=self.device) for _ in range(2)]
        k, v = out
        rows, dtype = k.shape[0], k.dtype
        self._rows(k, self.n_kv_heads, rows, "out")
        _need(dtype in (torch.bfloat16, torch.float32) and v.dtype is dtype and v.shape == k.shape and k.is_contiguous() and v.is_contiguous()
              and v.get_device() == self._index, "out: two contiguous tensors of bfloat16 or float32")
        rc = self._lib.neon_kv4_read(self._h, batch._ref, self._place(batch, cache), rows, k.data_ptr(), v.data_ptr(), _DTYPES[dtype],
                                     _stream_of(self._index))
        if rc:
            self._check(rc, "neon_kv4_read")
        return k, v

    def attend(self, batch: Kv4Batch, cache, q, sinks=None, window: int = 0, scale: float | None = None, max_rows: int | None = None,
               out=None, stream=None):
        """Attention of ``q`` [rows, n_q_heads, head_dim] (bf16 or fp16, rotated) over the cache; ``sinks``: bf16 [n_q_heads] logits of the
        softmax denominator; ``window`` > 0: only the last so many positions; ``scale``: default head_dim ** -0.5; ``max_rows``: the
        most rows of a sequence, as far as the host knows it; it chooses the kernel.  Without it a batch with row offsets counts as one
        sequence of all rows: a batch of 64 single tokens then takes twice as long as with ``max_rows=1``."""
        if stream is not None:
            return self._on(stream, self.attend, batch, cache, q, sinks, window, scale, max_rows, out)
        rows, dtype = q.shape[0], q.dtype
        qs = self._rows(q, self.n_q_heads, rows, "q")
        _need(dtype is torch.bfloat16 or dtype is torch.float16, "q: bfloat16 or float16")
        _need(sinks is None or (sinks.dtype is torch.bfloat16 and sinks.shape == (self.n_q_heads,) and sinks.is_contiguous()
                                and sinks.get_device() == self._index), f"sinks: bfloat16 [{self.n_q_heads}]")
        if out is None:
            out = torch.empty((rows, self.n_q_heads, self.head_dim), dtype=dtype, device=self.device)
        elif out.dtype is not dtype or out.shape != q.shape or not out.is_contiguous() or out.get_device() != self._index:
            raise ValueError("out: contiguous, q's type and shape")
        if max_rows is None:
            max_rows = 1 if batch.one_each else rows
        cache_ptr = self._place(batch, cache)
        lib, handle, ref = self._lib, self._h, batch._ref
        size = lib.neon_kv4_attend_workspace(handle, ref, rows, max_rows)
        # allocated on the current stream, so that two calls never share it; torch reuses it in stream order
        scratch = torch.empty(size, dtype=torch.uint8, device=self.device)
        rc = lib.neon_kv4_attend(handle, ref, cache_ptr, rows, _DTYPES[dtype], q.data_ptr(), qs, None if sinks is None else sinks.data_ptr(), window,
                                 self.head_dim ** -0.5 if scale is None else scale, max_rows, out.data_ptr(), scratch.data_ptr(), size,
                                 _stream_of(self._index))
        if rc:
            self._check(rc, "neon_kv4_attend")
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
