"""Windows at the ends of what they and lengths can be."""
import pytest
import torch

import kv4_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def world(nq, nkv, D, P, lens, rows, width, seed):
    from neonengine_b200.kv4_cache import Kv4Cache
    kv, g = Kv4Cache(nq, nkv, D, P), torch.Generator(device=DEV)
    g.manual_seed(seed)
    pages = len(lens) * width
    table = torch.randperm(pages, generator=g, device=DEV).int().view(len(lens), width)
    cache = torch.randint(0, 256, (pages, nkv, kv.record_bytes), generator=g, device=DEV, dtype=torch.uint8)
    for s in ref.parts(cache, P, D)[2:]:
        s.copy_(torch.randint(125, 128, s.shape, generator=g, device=DEV, dtype=torch.uint8))
    q = torch.randn((sum(rows), nq, D), generator=g, device=DEV).to(torch.bfloat16)
    cu = torch.tensor([0, *torch.tensor(rows).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    return kv, table, cache, q, cu, kv.batch(torch.tensor(lens, dtype=torch.int32, device=DEV), table, cu)


def expect(kv, cache, table, q, n, length, window):
    """The formula over the positions that the table names."""
    held = min(length, table.shape[0] * kv.page_size)
    k, v = (ref.load(cache, kv.page_size, kv.head_dim, table[:-(-held // kv.page_size)].long(), held, i) for i in range(2))
    want, mass = ref.attend(q, k, v, torch.arange(length - n, length, device=DEV), None, window, kv.head_dim ** -0.5)
    # a rounding to bf16, one of the probabilities, scores in f32
    return want, 2 ** -8 * want.abs() + (2 ** -11 + 2 ** -13) * mass * 1.01


@pytest.mark.parametrize("form", [(16, 2, 64, 64, 1), (16, 2, 64, 16, 4), (16, 2, 128, 32, 4), (8, 8, 64, 32, 1), (16, 2, 64, 64, 70)])
@pytest.mark.parametrize("window", [1, 63, 100, 128, 200, 10000])
def test_sequences_longer_than_their_table(form, window):
    """Positions that the table does not reach are not there; of the others each row sees those in its window, and no more."""
    nq, nkv, D, P, n = form
    lens, rows = [700, 640, 703, 641, 1100], [n] * 5
    kv, table, cache, q, cu, batch = world(nq, nkv, D, P, lens, rows, 640 // P, n)
    out = torch.full_like(q, 7.0)
    kv.attend(batch, cache, q, window=window, max_rows=n, out=out)
    assert kv.status() == 2
    for b, length in enumerate(lens):
        mine = slice(b * n, (b + 1) * n)
        want, tol = expect(kv, cache, table[b], q[mine], n, length, window)
        assert ((out[mine].double() - want).abs() <= tol).all(), (b, length)
    kv.close()


@pytest.mark.parametrize("form", [(16, 2, 64, 64), (16, 2, 128, 32)])
@pytest.mark.parametrize("rows", [20, 90])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 8, 2 ** 30])
def test_largest_windows(form, rows, window):
    """More rows than positions (the first see none) under a window as large as a number can be: as without one."""
    lens = [11, 300]
    kv, table, cache, q, cu, batch = world(*form, lens, [rows, rows], 300 // form[3] + 1, 3)
    for max_rows in (1, rows, 100):
        out, plain = (kv.attend(batch, cache, q, window=w, max_rows=max_rows) for w in (window, 0))
        assert torch.equal(out, plain)
        for b, length in enumerate(lens):
            want, tol = expect(kv, cache, table[b], q[b * rows:(b + 1) * rows], rows, length, 0)
            assert ((out[b * rows:(b + 1) * rows].double() - want).abs() <= tol).all()
    assert kv.status() == 0
    kv.close()
