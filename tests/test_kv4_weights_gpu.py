"""Attention over the 4-bit cache where weights and values lie far apart: results keep the accuracy of their own terms, whichever
kernel is chosen and however long the sequence is."""
import pytest
import torch

import kv4_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

# (query heads, key/value heads, head size, page size, rows of the sequence, window): an item's columns in one, two and four groups of
# eight, and the kernel for chunks of prompts, which a window that hides nothing chooses
FORMS = [(16, 2, 64, 64, 1, 0), (16, 2, 64, 16, 2, 0), (16, 2, 64, 32, 5, 0), (8, 1, 128, 32, 1, 0), (16, 2, 128, 64, 3, 0), (16, 2, 64, 64, 9, 1)]


def system(form):
    from neonengine_b200.kv4_cache import Kv4Cache
    return Kv4Cache(*form[:4])


def paged(kv, length, g):
    n = -(-length // kv.page_size)
    return torch.randperm(n, generator=g, device=DEV).int()[None], kv.new_cache(n)


def put(kv, cache, table, which, x):
    """x float64 [length, heads, D] at the positions from 0 on."""
    pos = torch.arange(x.shape[0], device=DEV)
    codes, byte, _ = ref.quantise(x)
    ref.store(cache, kv.page_size, kv.head_dim, table[0, pos // kv.page_size].long(), pos % kv.page_size, which, codes, byte)


def check(kv, cache, table, length, q, out, n_sequences=1, window=0, lost=2 ** -11):
    """Results of the last rows of sequences that all have these pages, to the rounding of the result, of the probabilities and their sum
    (2^-12 each) and of the scores (2^-13), and what small probabilities lose at most: 2^-9 of the weights times their values' scales
    (`lost` of the mass, as values are four times their scales or more where nothing else is said)."""
    k, v = (ref.load(cache, kv.page_size, kv.head_dim, table[0].long(), length, i) for i in range(2))
    n = q.shape[0] // n_sequences
    pos = torch.arange(length - n, length, device=DEV)
    half = torch.finfo(q.dtype).eps / 2
    for b in sorted({0, n_sequences // 2, n_sequences - 1}):
        want, mass = ref.attend(q[b * n:(b + 1) * n], k, v, pos, None, window, 1.0)
        tol = half * want.abs() + (2 ** -11 + 2 ** -13 + lost) * mass * (1 + half)
        if q.dtype is torch.float16:
            tol = tol + 2 ** -25  # half of fp16's smallest step
        got = out[b * n:(b + 1) * n].double()
        assert got.isfinite().all()
        off = ((got - want).abs() / tol).max()
        assert off <= 1, (b, float(off))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("gap,small", [(17.25, 12), (19.0, 14), (23.0, 20), (44.0, 55), (64.0, 60), (23.0, 0)])
@pytest.mark.parametrize("n", [1, 600])
def test_much_weight_on_small_values(form, gap, small, n):
    """Nearly all weight lies on the first position, whose values are 2^-small of the others': the result is theirs all the same.  One
    sequence, cut over many warps, and so many (on shared pages) that a warp walks hundreds of steps of one."""
    nq, nkv, D, P, rows, window = form
    kv, g = system(form), torch.Generator(device=DEV)
    g.manual_seed(rows)
    length = 30000 if not window else 400
    gap = gap if not window else gap - 4.25  # (a shorter tail)
    table, cache = paged(kv, length, g)
    x = torch.zeros((length, nkv, D), dtype=torch.float64, device=DEV)
    x[0, :, 0] = 4.0
    put(kv, cache, table, 0, x)
    v = 1 + torch.rand((length, nkv, D), generator=g, device=DEV).double()
    v[0] *= 2.0 ** -small
    put(kv, cache, table, 1, v)
    q = torch.zeros((n * rows, nq, D), device=DEV)
    q[..., 0] = gap / 4
    batch = kv.batch(torch.full((n,), length, dtype=torch.int32, device=DEV), table.expand(n, -1).contiguous(),
                     torch.arange(0, n * rows + 1, rows, dtype=torch.int32, device=DEV))
    for dtype in (torch.bfloat16, torch.float16):
        launched = kv.launch_count
        out = kv.attend(batch, cache, q.to(dtype), scale=1.0, window=window and 440, max_rows=rows)
        assert kv.launch_count == launched + (1 if window else 2)
        check(kv, cache, table, length, q.to(dtype), out, n_sequences=n, window=window and 440)
    assert kv.status() == 0
    kv.close()


@pytest.mark.parametrize("form", FORMS[:5])
@pytest.mark.parametrize("fall,first,growth", [(20.0, 60, 2), (9.0, 100, 1), (30.0, 60, 3), (70.0, 10, 5)])
def test_values_that_grow_along_the_sequence(form, fall, first, growth):
    """Values grow by 2^growth every 64 positions while the weights lie e^-fall below those of the first 64: the last ones are the
    result.  So many sequences (on shared pages) that a warp walks all of it by itself."""
    nq, nkv, D, P, rows, _ = form
    kv, g = system(form), torch.Generator(device=DEV)
    g.manual_seed(7)
    length, n = 40 * 64, 1024
    table, cache = paged(kv, length, g)
    x = torch.zeros((length, nkv, D), dtype=torch.float64, device=DEV)
    x[:64, :, 0] = 4.0
    put(kv, cache, table, 0, x)
    v = 1 + torch.rand((length, nkv, D), generator=g, device=DEV).double()
    put(kv, cache, table, 1, v * 2.0 ** (first - 127 + growth * (torch.arange(length, device=DEV) // 64).double())[:, None, None])
    q = torch.zeros((n * rows, nq, D), device=DEV, dtype=torch.bfloat16)
    q[..., 0] = fall / 4
    batch = kv.batch(torch.full((n,), length, dtype=torch.int32, device=DEV), table.expand(n, -1).contiguous(),
                     torch.arange(0, n * rows + 1, rows, dtype=torch.int32, device=DEV))
    out = kv.attend(batch, cache, q, scale=1.0, max_rows=rows)
    check(kv, cache, table, length, q, out, n_sequences=n)
    assert kv.status() == 0
    kv.close()


@pytest.mark.parametrize("form", FORMS)
def test_scores_that_swing(form):
    """Scores that go up and down by 30 from step to step, values of all sizes against them."""
    nq, nkv, D, P, rows, window = form
    kv, g = system(form), torch.Generator(device=DEV)
    g.manual_seed(5)
    length = 6000 if not window else 440
    table, cache = paged(kv, length, g)
    x = torch.zeros((length, nkv, D), dtype=torch.float64, device=DEV)
    step = torch.arange(length, device=DEV) // 64
    x[:, :, 0] = torch.randint(-4, 5, (int(step.max()) + 1, nkv), generator=g, device=DEV)[step].double().clamp(-4, 4)
    x[:, :, 1] = 0.25 * torch.randn((length, nkv), generator=g, device=DEV).double()
    put(kv, cache, table, 0, x)
    v = torch.randn((length, nkv, D), generator=g, device=DEV).double()
    put(kv, cache, table, 1, v * torch.exp(-x[:, :, :1] * 3.5))
    q = torch.randn((rows, nq, D), generator=g, device=DEV)
    q[..., 0] = 3.75 + 0.25 * torch.randint(0, 2, (rows, nq), generator=g, device=DEV)
    q = q.to(torch.bfloat16)
    batch = kv.batch(torch.tensor([length], dtype=torch.int32, device=DEV), table, torch.tensor([0, rows], dtype=torch.int32, device=DEV))
    out = kv.attend(batch, cache, q, scale=1.0, window=window and 470, max_rows=rows)
    check(kv, cache, table, length, q, out, window=window and 470, lost=2 ** -9)  # (normal values)
    kv.close()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("size", [-2.0 ** 21, 2.0 ** 21])
def test_scores_of_millions(form, size):
    """Equal scores, large ones: the mean of the values."""
    nq, nkv, D, P, rows, window = form
    kv, g = system(form), torch.Generator(device=DEV)
    g.manual_seed(2)
    length = 300
    table, cache = paged(kv, length, g)
    x = torch.zeros((length, nkv, D), dtype=torch.float64, device=DEV)
    x[:, :, 3] = 3.0
    put(kv, cache, table, 0, x)
    put(kv, cache, table, 1, torch.randn((length, nkv, D), generator=g, device=DEV).double())
    q = torch.zeros((rows, nq, D), device=DEV, dtype=torch.bfloat16)
    q[..., 3] = size
    batch = kv.batch(torch.tensor([length], dtype=torch.int32, device=DEV), table, torch.tensor([0, rows], dtype=torch.int32, device=DEV))
    out = kv.attend(batch, cache, q, scale=1.0, window=window and 320, max_rows=rows)
    check(kv, cache, table, length, q, out, window=window and 320, lost=2 ** -9)
    kv.close()
