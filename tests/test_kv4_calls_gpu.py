"""Calls of the 4-bit cache that leave something out or ask for too much."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_read_of_ragged_rows_wants_their_number():
    """With row offsets the number of rows is not that of the sequences: it has to be given."""
    from neonengine_b200.kv4_cache import Kv4Cache
    kv = Kv4Cache(8, 2, 64, 32)
    cache = torch.randint(0, 120, (4, 2, kv.record_bytes), device=DEV, dtype=torch.uint8)
    table = torch.arange(4, dtype=torch.int32, device=DEV).view(2, 2)
    lens, cu = torch.tensor([40, 50], dtype=torch.int32, device=DEV), torch.tensor([0, 3, 7], dtype=torch.int32, device=DEV)
    ragged, each = kv.batch(lens, table, cu), kv.batch(lens, table)
    with pytest.raises(ValueError, match="rows"):
        kv.read(ragged, cache)
    k, v = kv.read(ragged, cache, rows=7)
    assert k.shape == v.shape == (7, 2, 64)
    assert torch.equal(kv.read(ragged, cache, out=[torch.zeros_like(k), torch.zeros_like(v)])[0], k)
    one, _ = kv.read(each, cache)
    assert one.shape == (2, 2, 64) and torch.equal(one, k[[2, 6]])
    kv.close()


def test_attention_refuses_more_rows_than_it_can_number():
    """Rows times query heads a key/value head: 2^26 at most.  (The buffers are never looked at.)"""
    from neonengine_b200.kv4_cache import Kv4Cache
    kv = Kv4Cache(32, 1, 64, 32)
    small = torch.zeros(4096, device=DEV, dtype=torch.uint8)
    cu = torch.tensor([0, 2 ** 21 + 1], dtype=torch.int32, device=DEV)
    batch = kv.batch(torch.tensor([40], dtype=torch.int32, device=DEV), torch.zeros((1, 2), dtype=torch.int32, device=DEV), cu)
    batch._c.n_pages = 1
    one = ctypes.c_void_p(small.data_ptr())
    rc = kv._lib.neon_kv4_attend(kv._h, batch._ref, one, 2 ** 21 + 1, 1, one, 2048, None, 0, 1.0, 2 ** 21 + 1, one, one, 1 << 40, None)
    assert rc == 1 and b"query heads" in kv._lib.neon_kv4_last_error(kv._h)
    assert kv.launch_count == 0 and kv.status() == 0
    kv.close()


def test_attention_refuses_more_steps_than_it_can_number():
    """Steps of 64 positions times blocks of rows, as the table's width bounds them.  (The buffers are never looked at.)"""
    from neonengine_b200.kv4_cache import Kv4Cache
    kv = Kv4Cache(128, 128, 64, 64)
    small = torch.zeros(4096, device=DEV, dtype=torch.uint8)
    rows = 2 ** 20
    batch = kv.batch(torch.tensor([40], dtype=torch.int32, device=DEV), torch.zeros((1, 1), dtype=torch.int32, device=DEV),
                     torch.tensor([0, rows], dtype=torch.int32, device=DEV))
    batch._c.n_pages, batch._c.table_width, batch._c.table_stride = 1, 2 ** 24, 2 ** 24
    one = ctypes.c_void_p(small.data_ptr())
    rc = kv._lib.neon_kv4_attend(kv._h, batch._ref, one, rows, 1, one, 8192, None, 0, 1.0, 1, one, one, 1 << 62, None)
    assert rc == 1 and b"page tables" in kv._lib.neon_kv4_last_error(kv._h)
    assert kv.launch_count == 0 and kv.status() == 0
    kv.close()
