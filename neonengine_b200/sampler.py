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


class Sampler:
    def __init__(self, vocab: int, device: int = 0):
        self._lib = _lib.load()
        self.vocab, self.device = int(vocab), torch.device("cuda", int(device))
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
        if t.dtype != dtype or t.shape != (rows,) or t.device != self.device or not t.is_contiguous():
            raise ValueError(f"{name}: contiguous {dtype} [{rows}] on {self.device}")
        return t.data_ptr()

    def run(self, logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None, out=None, details: bool = False, stream=None):
        """Tokens int32 [rows] of ``logits`` [rows, vocab] (fp32, bf16 or fp16; rows may be any stride apart).  ``uniform``: fp32
        [rows] in [0, 1); ``temperature``, ``top_p``, ``min_p`` fp32 [rows] and ``top_k`` int32 [rows], or None.  With ``details``
        returns (tokens, probability of each among what was kept, how many were kept)."""
        if logits.dim() != 2 or logits.shape[1] != self.vocab or logits.dtype not in _DTYPES or logits.device != self.device or \
                (self.vocab > 1 and logits.stride(1) != 1):
            raise ValueError(f"logits: [rows, {self.vocab}] of float32, bfloat16 or float16 on {self.device}, rows contiguous")
        rows = logits.shape[0]
        args = (self._vector(uniform, rows, torch.float32, "uniform"), self._vector(temperature, rows, torch.float32, "temperature"),
                self._vector(top_k, rows, torch.int32, "top_k"), self._vector(top_p, rows, torch.float32, "top_p"),
                self._vector(min_p, rows, torch.float32, "min_p"))
        if uniform is None:
            raise ValueError("uniform: one random number per row")
        size = self._scratch.get(rows)
        if size is None:
            size = self._scratch[rows] = int(self._lib.neon_sampler_workspace(self._h, rows))
        tokens = torch.empty((rows,), dtype=torch.int32, device=self.device) if out is None else out
        self._vector(tokens, rows, torch.int32, "out")
        probs = kept = None
        if details:
            probs = torch.empty((rows,), dtype=torch.float32, device=self.device)
            kept = torch.empty((rows,), dtype=torch.int32, device=self.device)
        scratch = torch.empty(max(size, 16), dtype=torch.uint8, device=self.device)
        if stream is not None:
            scratch.record_stream(stream)
        st = torch.cuda.current_stream(self.device) if stream is None else stream
        rc = self._lib.neon_sampler_run(self._h, logits.data_ptr(), _DTYPES[logits.dtype], logits.stride(0) if rows > 1 else self.vocab, rows,
                                        *args, tokens.data_ptr(), probs.data_ptr() if details else None, kept.data_ptr() if details else None,
                                        scratch.data_ptr(), size, st.cuda_stream)
        if rc != 0:
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
