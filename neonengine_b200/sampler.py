"""Python host mirror of the sampler (include/neon_sampler.h): temperature, top-k, top-p and min-p per row, from
random numbers that the caller gives.

Calls are enqueued on the current stream (or ``stream``); errors become ``RuntimeError``, unusable arguments
``ValueError``.  torch only owns device memory and streams; every kernel runs inside ``libneon_moe.so``.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


class Sampler:
    def __init__(self, vocab: int, device: int = 0):
        self._lib = _lib.load()
        self.vocab, self.device, self._index = int(vocab), torch.device("cuda", int(device)), int(device)
        cfg = _lib.NeonSamplerConfig(self.vocab, int(device))
        handle = ctypes.c_void_p()
        rc = self._lib.neon_sampler_create(ctypes.byref(cfg), ctypes.byref(handle))
        if rc != 0:
            raise RuntimeError(f"neon_sampler_create failed ({rc}): {self._lib.neon_sampler_last_error(None).decode()}")
        self._h = handle
        self._scratch = {}

    def _vector(self, t, rows: int, dtype, name: str):
        if t is None:
            return None
        if t.dtype is not dtype or t.shape != (rows,) or t.get_device() != self._index or not t.is_contiguous():
            raise ValueError(f"{name}: contiguous {dtype} [{rows}] on {self.device}")
        return t.data_ptr()

    def run(self, logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None, out=None, details: bool = False, stream=None):
        """Tokens int32 [rows] of ``logits`` [rows, vocab] (fp32, bf16 or fp16; rows may be any stride apart).  ``uniform``: fp32
        [rows] in [0, 1); ``temperature``, ``top_p``, ``min_p`` fp32 [rows] and ``top_k`` int32 [rows], or None.  With ``details``
        returns (tokens, probability of each among what was kept, how many were kept)."""
        if stream is not None:  # what the run allocates belongs to that stream too
            if stream.device_index != self._index:
                raise ValueError("stream: one of the sampler's device")
            with torch.cuda.stream(stream):
                return self.run(logits, uniform, temperature, top_k, top_p, min_p, out, details)
        shape, stride, dtype, f32 = logits.shape, logits.stride(), logits.dtype, torch.float32
        if len(shape) != 2 or shape[1] != self.vocab or dtype not in _DTYPES or logits.get_device() != self._index or (stride[1] != 1 and shape[1] > 1):
            raise ValueError(f"logits: [rows, {self.vocab}] of float32, bfloat16 or float16 on {self.device}, rows contiguous")
        if uniform is None:
            raise ValueError("uniform: one random number per row")
        rows, vector = shape[0], self._vector
        u, t, k = vector(uniform, rows, f32, "uniform"), vector(temperature, rows, f32, "temperature"), vector(top_k, rows, torch.int32, "top_k")
        p, m = vector(top_p, rows, f32, "top_p"), vector(min_p, rows, f32, "min_p")
        size = self._scratch.get(rows)
        if size is None:
            size = self._scratch[rows] = int(self._lib.neon_sampler_workspace(self._h, rows))
        device = self.device
        tokens = torch.empty(rows, dtype=torch.int32, device=device) if out is None else out
        tokens_ptr = tokens.data_ptr() if out is None else vector(out, rows, torch.int32, "out")
        probs = kept = probs_ptr = kept_ptr = None
        if details:
            probs, kept = torch.empty(rows, dtype=f32, device=device), torch.empty(rows, dtype=torch.int32, device=device)
            probs_ptr, kept_ptr = probs.data_ptr(), kept.data_ptr()
        # allocated on the current stream, so that two runs never share it; torch reuses it in stream order
        scratch = torch.empty(size, dtype=torch.uint8, device=device)
        rc = self._lib.neon_sampler_run(self._h, logits.data_ptr(), _DTYPES[dtype], stride[0] if rows > 1 else self.vocab, rows, u, t, k, p, m,
                                        tokens_ptr, probs_ptr, kept_ptr, scratch.data_ptr(), size, _stream_of(self._index))
        if rc:
            raise RuntimeError(f"neon_sampler_run failed ({rc}): {self._lib.neon_sampler_last_error(self._h).decode()}")
        return (tokens, probs, kept) if details else tokens

    @property
    def launch_count(self) -> int:
        return int(self._lib.neon_sampler_launch_count(self._h))

    def close(self) -> None:
        if getattr(self, "_h", None):
            self._lib.neon_sampler_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
