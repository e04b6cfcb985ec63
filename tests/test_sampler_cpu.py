"""The sampler's C ABI where no GPU is needed: symbols, refusals, and the restatement that the GPU tests use."""
import ctypes
import os
import re

import numpy as np
import pytest
import torch

import sampler_reference as ref
from neonengine_b200 import _lib, build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def test_exports_every_declared_symbol(lib):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "neon_sampler.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(neon_sampler_[a-z_0-9]+)\s*\(", text)))
    assert len(names) >= 6 and all(hasattr(lib, n) for n in names)
    assert set(names) == set(_lib.SAMPLER_SIGNATURES), "python binding table out of sync with the header"


@pytest.mark.parametrize("vocab", [0, -5, 393217])
def test_create_rejects_bad_config(lib, vocab):
    h = ctypes.c_void_p()
    cfg = _lib.NeonSamplerConfig(vocab, 0)
    assert lib.neon_sampler_create(ctypes.byref(cfg), ctypes.byref(h)) == 1 and not h.value
    assert b"vocab" in lib.neon_sampler_last_error(None)


def test_no_cpu_fallback(lib):
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    h = ctypes.c_void_p()
    cfg = _lib.NeonSamplerConfig(1000, 0)
    assert lib.neon_sampler_create(ctypes.byref(cfg), ctypes.byref(h)) == 2 and not h.value


def test_calls_without_a_handle(lib):
    assert lib.neon_sampler_create(None, None) == 1
    assert lib.neon_sampler_run(None, None, 0, 1, 1, *[None] * 9, 0, None) == 1
    assert lib.neon_sampler_workspace(None, 1) == 0 and lib.neon_sampler_launch_count(None) == 0
    assert lib.neon_sampler_destroy(None) == 0


def test_restatement():
    """What the definition says, on rows small enough to see it."""
    x = [1.0, 3.0, 2.0, 3.0, -np.inf]
    assert ref.draw(x, 0.99, t=0) == (1, 1.0, 1)                       # the lower of two largest
    assert ref.draw(x, 0.0, k=1)[0] == 1 and ref.draw(x, 0.999, k=1)[0] == 1
    assert ref.draw(x, 0.51, k=2)[::2] == (3, 2)
    assert ref.draw(x, 0.0)[::2] == (0, 4) and ref.draw(x, 0.999999)[0] == 3
    assert ref.draw(x, 0.5, p=0.0)[::2] == (1, 1)
    assert ref.draw(x, 0.5, m=1.0)[2] == 2
    assert ref.draw([np.nan, -np.inf], 0.5) == (-1, 0.0, 0)
    assert ref.draw([np.inf, 1.0, np.inf], 0.6) == (2, 0.5, 3)
    p = np.exp(x) / np.exp(x).sum()
    assert abs(ref.draw(x, 0.0)[1] - p[0]) < 1e-15
