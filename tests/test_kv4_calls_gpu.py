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
