"""The 4-bit paged cache on the GPU against its restatement in 64 bits."""
import ctypes

import numpy as np
import pytest
import torch

import kv4_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def systems():
    from neonengine_b200.kv4_cache import Kv4Cache
    made = {}

    def get(nq, nkv, D, P):
        if (nq, nkv, D, P) not in made:
            made[nq, nkv, D, P] = Kv4Cache(nq, nkv, D, P)
        return made[nq, nkv, D, P]

    yield get
    for s in made.values():
        assert s.status() == 0
        s.close()


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def same(a, b):
    """Equal, a NaN to a NaN."""
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(nan=0.0, posinf=None, neginf=None), b.nan_to_num(nan=0.0, posinf=None, neginf=None))


def make_batch(kv, rows, lens, g, spare=2, each=False, width=None):
    P = kv.page_size
    need = [-(-max(n, 0) // P) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=g, device=DEV).int()
    table = torch.full((len(lens), width or max(1, max(need))), -7, dtype=torch.int32, device=DEV)  # unused entries name no page
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    cu = torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device=DEV)
    batch = kv.batch(torch.tensor(lens, dtype=torch.int32, device=DEV), table, None if each else cu)
    return batch, table, cu, sum(need) + spare


def random_cache(kv, n_pages, g, spread=1):
    """Pages of normal values whose blocks' magnitudes vary by 2^spread."""
    cache = torch.randint(0, 256, (n_pages, kv.n_kv_heads, kv.record_bytes), generator=g, device=DEV, dtype=torch.uint8)
    D, P = kv.head_dim, kv.page_size
    k, v, ks, vs = ref.parts(cache, P, D)
    for s in (ks, vs):
        s.copy_(torch.randint(125, 126 + spread, s.shape, generator=g, device=DEV, dtype=torch.uint8))
    return cache


def check_attention(kv, batch, table, cu, rows, lens, cache, q, sinks, window, scale, out, flat=True):
    half = torch.finfo(q.dtype).eps / 2
    for b, (n, length) in enumerate(zip(rows, lens)):
        lo = int(cu[b])
        if n == 0:
            continue
        length = max(length, 0)
        pages = table[b, :-(-length // kv.page_size)].long()
        k = ref.load(cache, kv.page_size, kv.head_dim, pages, length, 0)
        v = ref.load(cache, kv.page_size, kv.head_dim, pages, length, 1)
        pos = torch.arange(lens[b] - n, lens[b], device=DEV)
        want, mass = ref.attend(q[lo:lo + n], k, v, pos, sinks, window, scale)
        got = out[lo:lo + n].double()
        # one rounding of the result; one of every probability to f16 (2^-11 of it); scores in f32 from exact products,
        # exponentials to 2^-22: under 2^-13 of the mass for the scores at hand; and f16 probabilities below 2^-14 of the
        # largest are off by 2^-25 each, which counts only where values are of one size (`flat`)
        tol = half * want.abs() + (2 ** -11 + 2 ** -13) * mass * (1 + half)
        if flat and length:
            tol = tol + length * 2 ** -25 * v.abs().nan_to_num().amax()
        else:
            tol = tol + length * 2 ** -16 * mass
        assert torch.equal(got.isnan(), want.isnan())
        bad = ((got - want).abs() > tol) & ~want.isnan()
        assert not bad.any(), (b, n, length, int(bad.sum()), float(((got - want).abs() - tol).nan_to_num().max()))


HEADS = [(64, 8, 64, 64), (8, 8, 64, 16), (6, 2, 64, 32), (20, 1, 64, 64), (32, 8, 128, 16), (2, 2, 128, 64), (16, 1, 128, 32)]


@pytest.mark.parametrize("nq,nkv,D,P", HEADS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window", [0, 37])
def test_attend_one_token(systems, nq, nkv, D, P, dtype, window):
    kv, g = systems(nq, nkv, D, P), gen(nq + 7 * D + P)
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 0, 128, 777, 1500]
    batch, table, cu, pages = make_batch(kv, [1] * len(lens), lens, g, each=True)
    cache = random_cache(kv, pages, g)
    q = torch.randn((len(lens), nq, D), generator=g, device=DEV).to(dtype)
    sinks = torch.randn((nq,), generator=g, device=DEV).to(torch.bfloat16) if window else None
    out = torch.full_like(q, 7.0)
    kv.attend(batch, cache, q, sinks=sinks, window=window, out=out)
    check_attention(kv, batch, table, cu, [1] * len(lens), lens, cache, q, sinks, window, D ** -0.5, out)


@pytest.mark.parametrize("nq,nkv,D,P", HEADS)
@pytest.mark.parametrize("rows,lens,window,sink", [
    ([5, 1, 3, 0, 2], [300, 1, 3, 50, 1000], 0, True),      # drafted tokens; a sequence that is all new; one with no rows
    ([4, 7], [2, 7], 0, False),                               # more rows than positions: the first see none
    ([4, 7], [2, 700], 5, True),
    ([130, 33], [130, 641], 0, False),                        # a prompt and a chunk
    ([65, 40, 1], [400, 129, 90], 48, True),
])
def test_attend_several_rows(systems, nq, nkv, D, P, rows, lens, window, sink):
    kv, g = systems(nq, nkv, D, P), gen(sum(rows) + nq)
    batch, table, cu, pages = make_batch(kv, rows, lens, g)
    cache = random_cache(kv, pages, g)
    pad = 3
    q = torch.randn((sum(rows) + pad, nq, D), generator=g, device=DEV).to(torch.bfloat16)
    sinks = torch.randn((nq,), generator=g, device=DEV).to(torch.bfloat16) if sink else None
    for max_rows in (max(rows), 1):
        out = torch.full_like(q, 7.0)
        kv.attend(batch, cache, q, sinks=sinks, window=window, scale=0.2, max_rows=max_rows, out=out)
        check_attention(kv, batch, table, cu, rows, lens, cache, q, sinks, window, 0.2, out)
        assert (out[sum(rows):] == 7.0).all()  # rows behind the last sequence stay as they were


@pytest.mark.parametrize("D,P", [(64, 64), (64, 16), (128, 32)])
def test_attend_long_and_ragged(systems, D, P):
    """Items cut over many warps, and lengths that differ a hundredfold."""
    kv, g = systems(16, 2, D, P), gen(5)
    lens = [20000, 3, 9000, 777, 64, 12345]
    batch, table, cu, pages = make_batch(kv, [1] * 6, lens, g)
    cache = random_cache(kv, pages, g)
    q = (2 * torch.randn((6, 16, D), generator=g, device=DEV)).to(torch.bfloat16)
    out = kv.attend(batch, cache, q, max_rows=1)
    check_attention(kv, batch, table, cu, [1] * 6, lens, cache, q, None, 0, D ** -0.5, out)


@pytest.mark.parametrize("spread", [3, 9, 40, 100])
@pytest.mark.parametrize("rows", [1, 6, 70])
def test_attend_scales_far_apart(systems, spread, rows):
    """Blocks whose magnitudes differ by up to 2^spread: each head's result keeps the accuracy of its own terms."""
    kv, g = systems(8, 2, 64, 32), gen(spread)
    lens = [500, 230]
    batch, table, cu, pages = make_batch(kv, [rows] * 2, lens, g)
    cache = random_cache(kv, pages, g)
    k, v, ks, vs = ref.parts(cache, 32, 64)
    vs.copy_(torch.randint(120 - spread // 2, 121 + spread // 2, vs.shape, generator=g, device=DEV, dtype=torch.uint8))
    q = torch.randn((2 * rows, 8, 64), generator=g, device=DEV).to(torch.bfloat16)
    out = kv.attend(batch, cache, q, max_rows=rows)
    check_attention(kv, batch, table, cu, [rows] * 2, lens, cache, q, None, 0, 64 ** -0.5, out, flat=False)


@pytest.mark.parametrize("rows", [1, 5, 80])
def test_attend_scales_of_infinities(systems, rows):
    """Value scales of 2^126 and 2^127 count as 2^125, in every kernel."""
    kv, g = systems(16, 2, 64, 32), gen(rows)
    lens = [300]
    batch, table, cu, pages = make_batch(kv, [rows], lens, g)
    cache = random_cache(kv, pages, g)
    scales = ref.parts(cache, 32, 64)[3]
    page, slot = int(table[0, 1]), 7  # every row sees it
    cache_top = cache.clone()
    scales[page, 0, slot, 0] = 254
    scales[page, 1, slot, 1] = 253
    top = ref.parts(cache_top, 32, 64)[3]
    top[page, 0, slot, 0] = 252
    top[page, 1, slot, 1] = 252
    q = torch.randn((rows, 16, 64), generator=g, device=DEV).to(torch.bfloat16)
    out, want = (kv.attend(batch, c, q, max_rows=rows) for c in (cache, cache_top))
    assert same(out, want)
    clear = torch.ones_like(out, dtype=torch.bool)  # columns of other blocks are untouched by them
    clear[:, :8, :32] = clear[:, 8:, 32:] = False
    assert out[clear].isfinite().all() and (out[clear].abs() < 100).all()


@pytest.mark.parametrize("nq,nkv,P,dtype", [(16, 2, 16, torch.bfloat16), (64, 8, 32, torch.float16), (12, 4, 64, torch.float16), (20, 10, 16, torch.bfloat16)])
def test_attend_long_chunks(systems, nq, nkv, P, dtype):
    """Chunks of prompts over many steps, more items than multiprocessors, with and without a window."""
    kv, g = systems(nq, nkv, 64, P), gen(nq + P)
    rows, lens = [333, 1, 700, 64, 250], [5000, 4097, 731, 64, 9001]
    batch, table, cu, pages = make_batch(kv, rows, lens, g)
    cache = random_cache(kv, pages, g)
    q = torch.randn((sum(rows), nq, 64), generator=g, device=DEV).to(dtype)
    sinks = torch.randn((nq,), generator=g, device=DEV).to(torch.bfloat16)
    for window in (0, 1000):
        out = kv.attend(batch, cache, q, sinks=sinks, window=window, max_rows=700)
        check_attention(kv, batch, table, cu, rows, lens, cache, q, sinks, window, 0.125, out)
        again = kv.attend(batch, cache, q, sinks=sinks, window=window, max_rows=700)
        assert torch.equal(out, again)
    assert kv.status() == 0


def test_attend_small_values_at_the_top(systems):
    """All weight on positions whose values are 2^-30 of those that the softmax suppresses: the result is theirs."""
    kv, g = systems(8, 8, 64, 64), gen(3)
    length = 192
    batch, table, cu, pages = make_batch(kv, [1], [length], g)
    cache = random_cache(kv, pages, g)
    x = torch.zeros((length, 8, 64), dtype=torch.float64, device=DEV)
    x[:, :, 0] = -96.0
    x[77, :, 0] = 96.0
    v = torch.randn((length, 8, 64), generator=g, device=DEV).double()
    v[77] *= 2.0 ** -30
    page, slot = table[0, torch.arange(length, device=DEV) // 64].long(), torch.arange(length, device=DEV) % 64
    for which, y in ((0, x), (1, v)):
        codes, byte, _ = ref.quantise(y)
        ref.store(cache, 64, 64, page, slot, which, codes, byte)
    q = torch.zeros((1, 8, 64), device=DEV, dtype=torch.bfloat16)
    q[..., 0] = 8.0
    out = kv.attend(batch, cache, q).double()  # scores 96 and -96: the others' weight is e^-192
    want = ref.load(cache, 64, 64, table[0].long(), length, 1)[77]
    assert ((out[0] - want).abs() <= 2 ** -8 * want.abs() + 2 ** -11 * want.abs()).all()


def test_attend_ignores_what_it_does_not_see(systems):
    """NaN scales and any bytes at positions behind the length, outside the window or after the row: no trace of them."""
    kv, g = systems(8, 2, 64, 32), gen(9)
    rows, lens, window = [3, 2], [70, 41], 20
    batch, table, cu, pages = make_batch(kv, rows, lens, g)
    cache = random_cache(kv, pages, g)
    q = torch.randn((5, 8, 64), generator=g, device=DEV).to(torch.bfloat16)
    clean = kv.attend(batch, cache, q, window=window, max_rows=3)
    _, _, ks, vs = ref.parts(cache, 32, 64)
    dirty = cache.clone()
    _, _, kd, vd = ref.parts(dirty, 32, 64)
    for b, (n, length) in enumerate(zip(rows, lens)):
        for p in list(range(0, length - n - window + 1)) + list(range(length, table.shape[1] * 32)):
            page = int(table[b, p // 32])
            if page < 0:
                continue
            kd[page, :, p % 32] = 255
            vd[page, :, p % 32] = 255
    out = kv.attend(batch, dirty, q, window=window, max_rows=3)
    assert torch.equal(out, clean)
    # the newest position of sequence 0 is seen by its last row alone
    page = int(table[0, 69 // 32])
    vd[page, :, 69 % 32, 0] = 255
    out = kv.attend(batch, dirty, q, window=window, max_rows=3)
    assert torch.equal(out[:2], clean[:2]) and torch.equal(out[3:], clean[3:])
    assert out[2, :, :32].isnan().all() and torch.equal(out[2, :, 32:], clean[2, :, 32:])
    kd[page, :, 69 % 32, 0] = 255  # a NaN key: the whole row
    out = kv.attend(batch, dirty, q, window=window, max_rows=3)
    assert torch.equal(out[:2], clean[:2]) and out[2].isnan().all()


def test_attend_extreme_queries(systems):
    """Queries of any magnitude: rows are scaled by powers of two, so tiny and huge ones lose nothing."""
    kv, g = systems(8, 2, 64, 32), gen(11)
    lens = [200, 200, 200]
    batch, table, cu, pages = make_batch(kv, [1] * 3, lens, g)
    cache = random_cache(kv, pages, g)
    q = torch.randn((3, 8, 64), generator=g, device=DEV)
    q[0] *= 2.0 ** -60
    q[1] *= 2.0 ** 4
    q[2] = 0
    q = q.to(torch.bfloat16)
    out = kv.attend(batch, cache, q)
    check_attention(kv, batch, table, cu, [1] * 3, lens, cache, q, None, 0, 64 ** -0.5, out)
    q[0] = float("nan")
    out2 = kv.attend(batch, cache, q)
    assert out2[0].isnan().all() and torch.equal(out2[1:], out[1:])


def test_attend_strided_queries_and_far_pages(systems):
    """Queries as columns of a wider buffer; pages behind 2 GB of cache."""
    kv, g = systems(64, 8, 64, 64), gen(2)
    record = 8 * kv.record_bytes
    n_pages = (1 << 32) // record + 50
    cache = torch.empty((n_pages, 8, kv.record_bytes), dtype=torch.uint8, device=DEV)
    lens = [300, 129]
    table = torch.tensor([[n_pages - 1, n_pages - 3, 2, n_pages - 9, n_pages - 20], [n_pages - 5, 0, n_pages - 4, 0, 0]], dtype=torch.int32, device=DEV)
    used = table.unique().long()
    cache[used] = random_cache(kv, len(used), g)
    batch = kv.batch(torch.tensor(lens, dtype=torch.int32, device=DEV), table)
    cu = torch.tensor([0, 1, 2], device=DEV)
    wide = torch.randn((2, 80, 64), generator=g, device=DEV).to(torch.bfloat16)
    q = wide[:, 8:72]
    out = kv.attend(batch, cache, q)
    check_attention(kv, batch, table, cu, [1, 1], lens, cache, q, None, 0, 0.125, out)


# ---- append ---------------------------------------------------------------------------------------------------
def inv_freq(D):
    return (150000.0 ** (-torch.arange(D // 2, dtype=torch.float64) * 2 / D)).float().to(DEV)


@pytest.mark.parametrize("nq,nkv,D,P", HEADS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,lens", [([1, 1, 1], [1, 64, 100001]), ([70, 0, 3, 200], [70, 9, 131, 1000])])
def test_append(systems, nq, nkv, D, P, dtype, rows, lens):
    kv, g = systems(nq, nkv, D, P), gen(D + P + sum(lens))
    batch, table, cu, pages = make_batch(kv, rows, lens, g)
    cache = torch.randint(0, 256, (pages, nkv, kv.record_bytes), generator=g, device=DEV, dtype=torch.uint8)
    before = cache.clone()
    n, pad = sum(rows), 2
    wide = torch.randn((n + pad, nq + 2 * nkv, D), generator=g, device=DEV) * torch.exp(3 * torch.randn((n + pad, 1, 1), generator=g, device=DEV))
    wide[n:] = float("nan")
    wide = wide.to(dtype)
    q, k, v = wide[:, :nq], wide[:, nq:nq + nkv], wide[:, nq + nkv:]
    f = inv_freq(D)
    out = torch.full((n + pad, nq, D), 7.0, dtype=torch.float16 if dtype == torch.float16 else torch.bfloat16, device=DEV)
    kv.append(batch, cache, q, k, v, f, mscale=1.25, out=out)
    pos = torch.cat([torch.arange(length - m, length, device=DEV) for m, length in zip(rows, lens)])
    seq = torch.repeat_interleave(torch.arange(len(rows), device=DEV), torch.tensor(rows, device=DEV))
    want = ref.rotate(q[:n], pos, f, 1.25)
    # queries: sine, cosine and their products in f32, then one rounding
    size = torch.cat([sum(x.double().abs() for x in q[:n].chunk(2, -1))] * 2, -1) * 1.25
    tol = torch.finfo(out.dtype).eps / 2 * want.abs() + 4 * 2 ** -24 * size
    if out.dtype == torch.float16:
        tol = tol + 2 ** -25
    # fp16 ends at 65504: what lies from 65520 on (a half step further) rounds to infinity, in inputs and outputs
    ends = want.abs() >= 65520 if out.dtype == torch.float16 else torch.zeros_like(want, dtype=torch.bool)
    assert torch.equal(out[:n][ends].double(), torch.copysign(torch.full_like(want, float("inf")), want)[ends])
    assert torch.equal(out[:n].isnan(), want.isnan())
    fits = ~ends & want.isfinite()
    assert ((out[:n].double() - want).abs() <= tol)[fits].all()
    assert (out[n:] == 7.0).all()
    # keys and values: the bytes that the formula gives, and nothing else touched
    page, slot = table[seq, pos // P].long(), pos % P
    for which, x in ((0, ref.rotate(k[:n], pos, f, 1.25)), (1, v[:n].double())):
        codes, byte, value = ref.quantise(x)
        got_codes, got_byte = ref.parts(cache, P, D)[which][page, :, slot], ref.parts(cache, P, D)[2 + which][page, :, slot]
        assert torch.equal(got_byte.long(), byte.long())
        both = torch.stack([got_codes & 15, got_codes >> 4], -1).flatten(-2).long()
        assert torch.equal(both % 8, codes % 8)
        assert torch.equal(torch.where(codes % 8 == 0, 0, both), torch.where(codes % 8 == 0, 0, codes))
        ref.store(before, P, D, page, slot, which, both, got_byte)
    assert torch.equal(cache, before)
    got = kv.read(batch, cache, rows=n + pad)
    for which, x in ((0, ref.rotate(k[:n], pos, f, 1.25)), (1, v[:n].double())):
        assert same(got[which][:n].double(), ref.quantise(x)[2].to(torch.bfloat16).double())
        assert (got[which][n:] == 0).all()
    wide32 = kv.read(batch, cache, rows=n + pad, dtype=torch.float32)
    assert same(wide32[0].to(torch.bfloat16), got[0]) and same(wide32[1].to(torch.bfloat16), got[1])


def test_append_special_values(systems):
    """Zeros, infinities, NaN, denormals, the largest magnitudes, every tie."""
    kv, g = systems(8, 2, 64, 32), gen(1)
    n = 8
    batch, table, cu, pages = make_batch(kv, [n], [n], g)
    cache = kv.new_cache(pages)
    x = torch.zeros((n, 2, 64), device=DEV)
    x[0, 0, :16] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 7.5], device=DEV)
    x[0, 1, 5] = float("inf")
    x[0, 1, 6] = 3.0
    x[1, 0, 3] = float("nan")
    x[1, 1, 40] = float("nan")
    x[2, 0, :4] = torch.tensor([1e-40, -3e-42, 1e-45, 0.0], device=DEV)
    x[2, 1, :3] = torch.tensor([3.4e38, -3e38, 1e30], device=DEV)
    x[3] = torch.randn((2, 64), generator=g, device=DEV) * 2.0 ** -120
    x[4, 0, ::2] = float("-inf")
    x[5] = torch.randn((2, 64), generator=g, device=DEV)
    x[6, 0, 0], x[6, 0, 1] = 4.0, torch.nextafter(torch.tensor(2.5), torch.tensor(3.0))
    x[6, 0, 2] = torch.nextafter(torch.tensor(0.25), torch.tensor(1.0))
    x[6, 0, 3] = torch.nextafter(torch.tensor(0.75), torch.tensor(0.0))
    k = x.clone()
    f = torch.zeros(32, device=DEV)  # no turn: the keys are kept as they are
    k[0, 1] = 0
    k[4] = 0  # infinity times a sine of zero is not a number
    kv.append(batch, cache, None, k, x, f)
    page, slot = table[0, torch.arange(n, device=DEV) // 32].long(), torch.arange(n, device=DEV) % 32
    # (a turn by nothing is still the formula: a NaN times a sine of zero reaches its partner's block)
    for which, y in ((0, ref.rotate(k, torch.arange(n, device=DEV), f, 1.0)), (1, x)):
        codes, byte, value = ref.quantise(y.double())
        got = ref.parts(cache, 32, 64)[2 + which][page, :, slot].long()
        assert torch.equal(got, byte.long()), which
        both = torch.stack([(c := ref.parts(cache, 32, 64)[which][page, :, slot]) & 15, c >> 4], -1).flatten(-2).long()
        nan = (byte == 255).repeat_interleave(32, -1)
        assert torch.equal((both % 8)[~nan], (codes % 8)[~nan]), which
    ks, vs = kv.read(batch, cache, rows=n, dtype=torch.float32)
    assert vs[1, 0, :32].isnan().all() and not vs[1, 0, 32:].isnan().any()
    assert (vs[0, 1, 5] == float("inf")) and (vs[4, 0, ::2] == float("-inf")).all()


def test_bad_pages_and_lengths_are_reported():
    from neonengine_b200.kv4_cache import Kv4Cache
    kv, g = Kv4Cache(8, 2, 64, 32), gen(4)
    lens = [100, 60]
    batch, table, cu, pages = make_batch(kv, [1, 1], lens, g)
    cache = random_cache(kv, pages, g)
    q = torch.randn((2, 8, 64), generator=g, device=DEV).to(torch.bfloat16)
    good = kv.attend(batch, cache, q)
    assert kv.status() == 0
    table[0, 1] = pages  # one past the last
    out = kv.attend(batch, cache, q)
    assert kv.status() == 1 and torch.equal(out[1], good[1])
    # what is left of sequence 0: its other pages
    keep = torch.tensor([0, 2, 3], device=DEV)
    k, v = (torch.cat([ref.load(cache, 32, 64, table[0, keep[:2]].long(), 64, w), ref.load(cache, 32, 64, table[0, keep[2:]].long(), 4, w)]) for w in (0, 1))
    want, mass = ref.attend(q[:1], k, v, torch.full((1,), 1000, device=DEV), None, 0, 0.125)
    assert ((out[0].double() - want[0]).abs() <= 2 ** -8 * want[0].abs() + 2 ** -10 * mass[0]).all()
    f = inv_freq(64)
    table[0, 3] = -1
    before = cache.clone()
    x = torch.randn((2, 12, 64), generator=g, device=DEV).to(torch.bfloat16)
    kv.append(batch, cache, x[:, :8], x[:, 8:10], x[:, 10:], f)
    assert kv.status() == 1
    changed = (cache != before).flatten(1).any(1).nonzero().flatten().tolist()
    assert changed == [int(table[1, 1])]
    # a length that the table does not reach
    long = kv.batch(torch.tensor([129, 60], dtype=torch.int32, device=DEV), table[:, :2].contiguous())
    before = cache.clone()
    kv.append(long, cache, x[:, :8], x[:, 8:10], x[:, 10:], f)
    assert kv.status() == 2
    kv.attend(long, cache, q)
    assert kv.status() & 2
    kv.read(long, cache, rows=2)
    assert kv.status() == 2
    # row offsets that fall: no row outside the inputs is touched
    falls = kv.batch(torch.tensor([60, 60], dtype=torch.int32, device=DEV), table, torch.tensor([0, 9, 1], dtype=torch.int32, device=DEV))
    table.fill_(0)
    kv.attend(falls, cache, q)
    kv.append(falls, cache, x[:, :8], x[:, 8:10], x[:, 10:], f)
    assert kv.status() & 2
    kv.close()


# ---- together -------------------------------------------------------------------------------------------------
def test_append_then_attend_step_by_step(systems):
    """A conversation: a prompt in one pass, then tokens one at a time, against attention over all rounded keys and values."""
    nq, nkv, D, P = 16, 2, 64, 16
    kv, g = systems(nq, nkv, D, P), gen(21)
    lens, f = [37, 5], inv_freq(D)
    steps = 4
    total = [n + steps for n in lens]
    table = torch.randperm(8, generator=g, device=DEV).int().view(2, 4)
    cache = kv.new_cache(8)
    xs = [torch.randn((t, nq + 2 * nkv, D), generator=g, device=DEV).to(torch.bfloat16) for t in total]
    keys = [ref.quantise(ref.rotate(x[:, nq:nq + nkv], torch.arange(t, device=DEV), f, 1.0))[2] for x, t in zip(xs, total)]
    vals = [ref.quantise(x[:, nq + nkv:].double())[2] for x in xs]
    done = [0, 0]
    for step in range(steps + 1):
        rows = lens if step == 0 else [1, 1]
        now = [d + r for d, r in zip(done, rows)]
        cu = torch.tensor([0, rows[0], sum(rows)], dtype=torch.int32, device=DEV)
        batch = kv.batch(torch.tensor(now, dtype=torch.int32, device=DEV), table, cu)
        x = torch.cat([xs[b][done[b]:now[b]] for b in range(2)])
        q = kv.append(batch, cache, x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:], f)
        out = kv.attend(batch, cache, q, max_rows=max(rows))
        for b in range(2):
            lo, hi = int(cu[b]), int(cu[b + 1])
            want, mass = ref.attend(q[lo:hi], keys[b][:now[b]], vals[b][:now[b]], torch.arange(done[b], now[b], device=DEV), None, 0, D ** -0.5)
            tol = 2 ** -8 * want.abs() + (2 ** -11 + 2 ** -13) * mass * 1.01 + 2 ** -19 * vals[b].abs().max()
            assert ((out[lo:hi].double() - want).abs() <= tol).all()
        done = now


def test_captured_graph_and_streams(systems):
    """Both calls captured into a graph whose batch changes between replays; another graph and another stream beside it."""
    kv, g = systems(16, 2, 64, 32), gen(31)
    f = inv_freq(64)

    def world(lens):
        batch, table, cu, pages = make_batch(kv, [1] * len(lens), lens, g, each=True, width=40)
        return batch, table, random_cache(kv, pages + 40, g), torch.randn((len(lens), 20, 64), generator=g, device=DEV).to(torch.bfloat16)

    worlds = [world([500, 70]), world([900, 133])]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs, lens = [], [], [w[0]._keep[0] for w in worlds]
    step = lambda w: kv.attend(w[0], w[2], kv.append(w[0], w[2], w[3][:, :16], w[3][:, 16:18], w[3][:, 18:], f))  # noqa: E731
    for w in worlds:
        step(w)
    torch.cuda.synchronize()
    for w, st in zip(worlds, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            outs.append(step(w))
        graphs.append(graph)
    for new in ([500, 70], [480, 65], [300, 1]):
        for n in lens:
            n.copy_(torch.tensor(new, dtype=torch.int32, device=DEV))
        torch.cuda.synchronize()
        for _ in range(5):
            for graph, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    graph.replay()
        torch.cuda.synchronize()
        for w, out in zip(worlds, outs):
            assert torch.equal(out, step(w))


def test_results_belong_to_the_given_stream(systems):
    """A call on another stream while the current one still has to write to memory that it freed: the result is not in it."""
    kv, g = systems(16, 2, 64, 32), gen(32)
    batch, table, cu, pages = make_batch(kv, [1] * 8, [200] * 8, g, each=True)
    cache = random_cache(kv, pages, g)
    q = torch.randn((8, 16, 64), generator=g, device=DEV).to(torch.bfloat16)
    want, (want_k, want_v) = kv.attend(batch, cache, q), kv.read(batch, cache)
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    freed = [torch.empty_like(t) for t in (want, want_k, want_v)]
    torch.cuda._sleep(20000000)
    for t in freed:
        t.fill_(7)
    del freed, t
    out = kv.attend(batch, cache, q, stream=other)
    k, v = kv.read(batch, cache, stream=other)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(k, want_k) and torch.equal(v, want_v)


@pytest.mark.parametrize("nq,nkv,D,P,n", [(8, 2, 64, 16, 1024), (128, 128, 64, 64, 3), (32, 1, 128, 32, 1024)])
def test_largest_batches_and_head_counts(systems, nq, nkv, D, P, n):
    """As many sequences and key/value heads as there can be: appended, read back, attended to, by chunks too."""
    kv, g = systems(nq, nkv, D, P), gen(n + nq)
    lens = [1 + i * 7 % 90 for i in range(n)]
    batch, table, cu, pages = make_batch(kv, [1] * n, lens, g, each=True)
    cache = random_cache(kv, pages, g)
    x = torch.randn((n, nq + 2 * nkv, D), generator=g, device=DEV).to(torch.bfloat16)
    f = inv_freq(D)
    q = kv.append(batch, cache, x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:], f)
    vals, _, value = ref.quantise(x[:, nq + nkv:].double())
    assert torch.equal(kv.read(batch, cache, dtype=torch.float32)[1].double(), value)
    some = torch.tensor([0, 1, 2, n // 2, n - 1], device=DEV).unique()
    outs = [kv.attend(batch, cache, q)]
    if D == 64:  # behind a window that hides nothing the chunk kernel is chosen
        wide, held, launched = torch.zeros((n + 64, nq, D), dtype=q.dtype, device=DEV), torch.full((n + 64, nq, D), 7.0, dtype=q.dtype, device=DEV), kv.launch_count
        wide[:n] = q
        outs.append(kv.attend(batch, cache, wide, window=100, max_rows=64, out=held)[:n])
        assert kv.launch_count == launched + 1 and (held[n:] == 7.0).all()
    for out in outs:
        for b in some.tolist():
            page = table[b, :-(-lens[b] // P)].long()
            k, v = (ref.load(cache, P, D, page, lens[b], i) for i in range(2))
            want, mass = ref.attend(q[b:b + 1], k, v, torch.tensor([lens[b] - 1], device=DEV), None, 0, D ** -0.5)
            tol = 2 ** -8 * want.abs() + (2 ** -11 + 2 ** -13) * mass * 1.01 + lens[b] * 2 ** -25 * v.abs().amax()
            assert ((out[b:b + 1].double() - want).abs() <= tol).all()


def test_sequences_share_pages(systems):
    """A common prefix: two tables name the same pages, and each sequence has a last page of its own."""
    kv, g = systems(8, 2, 64, 32), gen(34)
    cache = random_cache(kv, 5, g)
    lens, table = [70, 75], torch.tensor([[3, 1, 0], [3, 1, 4]], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    batch = kv.batch(torch.tensor(lens, dtype=torch.int32, device=DEV), table)
    x = torch.randn((2, 12, 64), generator=g, device=DEV).to(torch.bfloat16)
    before = cache.clone()
    q = kv.append(batch, cache, x[:, :8], x[:, 8:10], x[:, 10:], inv_freq(64))
    assert torch.equal(cache[[1, 2, 3]], before[[1, 2, 3]])
    out = kv.attend(batch, cache, q)
    check_attention(kv, batch, table, cu, [1, 1], lens, cache, q, None, 0, 0.125, out)


def test_captured_behind_copies_and_other_streams(systems):
    """A graph in which append, attention and sampling follow a copy, a fill and work of another stream: each waits for them."""
    from neonengine_b200.sampler import Sampler
    kv, g, sampler = systems(16, 2, 64, 32), gen(33), Sampler(16 * 64)
    batch, table, cu, pages = make_batch(kv, [1] * 8, [700] * 8, g, each=True)
    first = random_cache(kv, pages, g)
    given = torch.randn((8, 20, 64), generator=g, device=DEV).to(torch.bfloat16)
    cache, x, uniform, f = torch.empty_like(first), torch.empty_like(given), torch.empty(8, device=DEV), inv_freq(64)
    side = torch.cuda.Stream()

    def run():
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            torch.cuda._sleep(200000)
            cache.copy_(first)
        x.copy_(given)
        main.wait_stream(side)
        q = kv.append(batch, cache, x[:, :16], x[:, 16:18], x[:, 18:], f)
        uniform.zero_()
        out = kv.attend(batch, cache, q)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            torch.cuda._sleep(200000)
            uniform.fill_(0.5)
        main.wait_stream(side)
        return out, sampler.run(out.flatten(1), uniform)

    out, tokens = (t.clone() for t in run())
    torch.cuda.synchronize()
    plain = kv.attend(batch, cache, kv.append(batch, cache, given[:, :16], given[:, 16:18], given[:, 18:], f))
    assert torch.equal(out, plain) and torch.equal(tokens, sampler.run(out.flatten(1), torch.full((8,), 0.5, device=DEV)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for _ in range(3):
        cache.zero_()
        x.zero_()
        for t in held:
            t.zero_()
        graph.replay()
        assert torch.equal(held[0], out) and torch.equal(held[1], tokens)
    sampler.close()


class Padded:
    """The system, with the queries of every attention call followed by rows that belong to no sequence: so many that the
    kernel for chunks of prompts is chosen (where heads are of 64)."""

    def __init__(self, kv):
        self.kv = kv

    def __getattr__(self, name):
        return getattr(self.kv, name)

    def attend(self, batch, cache, q, sinks=None, window=0, scale=None, max_rows=None, out=None):
        n, total = q.shape[0], q.shape[0] + 40960 // self.kv.n_q_heads
        wide = torch.full((total, *q.shape[1:]), float("nan"), dtype=q.dtype, device=DEV)
        wide[:n] = q
        held = torch.full_like(wide, 7.0)
        if out is not None:
            held[:n] = out
        launched = self.kv.launch_count
        self.kv.attend(batch, cache, wide, sinks, window, scale, total, held)
        assert self.kv.launch_count == launched + 1  # the other kernel takes two
        assert (held[n:] == 7.0).all()
        return held[:n] if out is None else out.copy_(held[:n])


SEVERAL = [([5, 1, 3, 0, 2], [300, 1, 3, 50, 1000], 0, True), ([4, 7], [2, 7], 0, False), ([4, 7], [2, 700], 5, True),
           ([130, 33], [130, 641], 0, False), ([65, 40, 1], [400, 129, 90], 48, True)]


@pytest.mark.parametrize("nq,nkv,D,P", [h for h in HEADS if h[2] == 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_chunk_kernel_shapes(systems, nq, nkv, D, P, dtype):
    def padded(*shape):
        return Padded(systems(*shape))
    for window in (0, 37):
        test_attend_one_token(padded, nq, nkv, D, P, dtype, window)
    for rows, lens, window, sink in SEVERAL:
        test_attend_several_rows(padded, nq, nkv, D, P, rows, lens, window, sink)


@pytest.mark.parametrize("which", ["scales", "infinities", "unseen", "queries"])
def test_chunk_kernel_values(systems, which):
    def padded(*shape):
        return Padded(systems(*shape))
    if which == "scales":
        for spread in (3, 9, 40, 100):
            for rows in (1, 6, 70):
                test_attend_scales_far_apart(padded, spread, rows)
    elif which == "infinities":
        test_attend_scales_of_infinities(padded, 5)
    elif which == "unseen":
        test_attend_ignores_what_it_does_not_see(padded)
        test_attend_small_values_at_the_top(padded)
    else:
        test_attend_extreme_queries(padded)


# ---- refusals ----------------------------------------------------------------------------------------------------
def test_refusals(systems):
    kv, g = systems(8, 2, 64, 32), gen(4)
    batch, table, cu, pages = make_batch(kv, [1, 1], [40, 30], g)
    cache = random_cache(kv, pages, g)
    x = torch.randn((2, 12, 64), device=DEV).to(torch.bfloat16)
    q, k, v, f = x[:, :8], x[:, 8:10], x[:, 10:], inv_freq(64)
    for call in (lambda: kv.append(batch, cache, q, k, v[:1], f), lambda: kv.append(batch, cache, q.float(), k, v, f),
                 lambda: kv.append(batch, cache, q, k, v, f[:5]), lambda: kv.append(batch, cache[:, :, :64], q, k, v, f),
                 lambda: kv.append(batch, cache.cpu(), q, k, v, f), lambda: kv.attend(batch, cache, q.float()),
                 lambda: kv.attend(batch, cache, q[:, :4]), lambda: kv.attend(batch, cache, q, sinks=torch.zeros(8, device=DEV)),
                 lambda: kv.attend(batch, cache, q, out=torch.empty((2, 8, 64), device=DEV)), lambda: kv.batch(torch.zeros(2, device=DEV), table),
                 lambda: kv.batch(table[0, :1], table), lambda: kv.attend(batch, cache, q.transpose(0, 1)),
                 lambda: kv.attend(batch, cache, q[..., ::2])):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: kv.attend(batch, cache, q, window=-1), lambda: kv.attend(batch, cache, q, scale=float("nan"))):
        with pytest.raises(RuntimeError):
            call()
    lib, one = kv._lib, ctypes.c_void_p(cache.data_ptr())
    assert lib.neon_kv4_attend(kv._h, batch._ref, one, 2, 0, one, 512, None, 0, 1.0, 1, one, one, 1 << 30, None) == 1  # fp32 queries
    assert lib.neon_kv4_attend(kv._h, batch._ref, one, 2, 1, one, 512, None, 0, 1.0, 1, one, one, 16, None) == 1       # too little scratch
    assert b"workspace" in lib.neon_kv4_last_error(kv._h)
    assert lib.neon_kv4_attend(kv._h, batch._ref, one, 2, 1, ctypes.c_void_p(cache.data_ptr() + 2), 512, None, 0, 1.0, 1, one, one, 1 << 30, None) == 1
    assert lib.neon_kv4_append(kv._h, batch._ref, one, 2, 1, one, 512, one, 100, one, 128, one, 1.0, one, 1, None) == 1  # short rows
    assert lib.neon_kv4_append(kv._h, batch._ref, one, 2, 1, one, 512, one, 128, one, 128, one, 1.0, None, 1, None) == 1  # q without q_out
    assert lib.neon_kv4_append(kv._h, batch._ref, one, 2, 9, one, 512, one, 128, one, 128, one, 1.0, one, 1, None) == 1
    assert lib.neon_kv4_read(kv._h, batch._ref, one, 2, one, one, 2, None) == 1
    assert lib.neon_kv4_read(kv._h, None, one, 2, one, one, 1, None) == 1
    none = kv.batch(torch.zeros(2, dtype=torch.int32, device=DEV), table, torch.zeros(3, dtype=torch.int32, device=DEV))
    empty = kv.append(none, cache, q[:0], k[:0], v[:0], f)
    assert kv.attend(none, cache, empty).shape == (0, 8, 64) and kv.read(none, cache, rows=0)[0].shape == (0, 2, 64)
    assert kv.status() == 0
