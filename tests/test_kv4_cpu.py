"""The 4-bit paged cache's C ABI where no GPU is needed: symbols, refusals, and the restatement that the GPU tests use."""
import ctypes
import os
import re

import pytest
import torch

import kv4_reference as ref
from neonengine_b200 import _lib, build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def test_exports_every_declared_symbol(lib):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "neon_kv4.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(neon_kv4_[a-z_0-9]+)\s*\(", text)))
    assert len(names) >= 10 and all(hasattr(lib, n) for n in names)
    assert set(names) == set(_lib.KV4_SIGNATURES), "python binding table out of sync with the header"


@pytest.mark.parametrize("config,word", [((64, 8, 96, 64, 0), b"head_dim"), ((64, 8, 64, 48, 0), b"page_size"), ((64, 0, 64, 64, 0), b"n_kv_heads"),
                                         ((60, 8, 64, 64, 0), b"n_q_heads"), ((66, 2, 64, 64, 0), b"n_q_heads"), ((64, 8, 64, 64, -1), b"device")])
def test_create_rejects_bad_config(lib, config, word):
    h = ctypes.c_void_p()
    cfg = _lib.NeonKv4Config(*config)
    assert lib.neon_kv4_create(ctypes.byref(cfg), ctypes.byref(h)) in (1, 2) and not h.value
    assert word in lib.neon_kv4_last_error(None)


def test_no_cpu_fallback(lib):
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    h = ctypes.c_void_p()
    cfg = _lib.NeonKv4Config(64, 8, 64, 64, 0)
    assert lib.neon_kv4_create(ctypes.byref(cfg), ctypes.byref(h)) == 2 and not h.value


def test_calls_without_a_handle(lib):
    assert lib.neon_kv4_create(None, None) == 1
    assert lib.neon_kv4_append(None, None, None, 1, 1, None, 0, None, 0, None, 0, None, 1.0, None, 1, None) == 1
    assert lib.neon_kv4_read(None, None, None, 1, None, None, 1, None) == 1
    assert lib.neon_kv4_attend(None, None, None, 1, 1, None, 0, None, 0, 1.0, 1, None, None, 0, None) == 1
    assert lib.neon_kv4_status(None, None) == 1
    assert lib.neon_kv4_attend_workspace(None, None, 1, 1) == 0 and lib.neon_kv4_record_bytes(None) == 0
    assert lib.neon_kv4_destroy(None) == 0


@pytest.mark.parametrize("P,D", [(16, 64), (32, 128)])
def test_restatement_stores_what_it_loads(P, D):
    g = torch.Generator().manual_seed(P)
    cache = torch.zeros((3, 2, P * (D + D // 16)), dtype=torch.uint8)
    n = P + 5
    page, slot = torch.tensor([2, 0])[torch.arange(n) // P], torch.arange(n) % P
    x = torch.randn((2, n, 2, D), generator=g, dtype=torch.float64) * 2.0 ** torch.randint(-9, 9, (2, n, 2, 1), generator=g)
    for which in range(2):
        codes, byte, value = ref.quantise(x[which])
        ref.store(cache, P, D, page, slot, which, codes, byte)
        assert torch.equal(ref.load(cache, P, D, torch.tensor([2, 0]), n, which), value)
        # a rounding is off by at most half a step (the steps are 1/2, 1, 2 of the scale), or clips 8 to 6
        scale = ref.scale_of(byte).repeat_interleave(32, -1)
        assert ((value - x[which]).abs() <= torch.where(x[which].abs() > 6 * scale, 2.0, 1.0) * scale).all()


def test_decoder_calls_without_a_handle(lib):
    assert lib.neon_decoder_set_sampling(None, None, None, None, None, None) == 1
    assert lib.neon_decoder_set_option(None, b"kv_bits", 4) == 1
