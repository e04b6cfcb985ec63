"""The 4-bit paged cache restated in 64 bits: record layout, rounding, rotation, attention."""
import math

import torch

MAGNITUDES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantise(x):
    """(codes, scale bytes, values) of float64 [..., D]: blocks of 32, scale 2^(floor(log2 amax) - 2), nearest magnitude,
    ties to the even code."""
    b = x.unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1)
    byte = (torch.frexp(amax)[1] - 1 - 2 + 127).clamp(1, 254)
    byte = torch.where(amax == 0, 127, byte)
    byte = torch.where(amax.isinf(), 254, byte)
    nan = b.isnan().any(-1)
    y = torch.ldexp(b.abs(), (127 - byte)[..., None])
    mag = MAGNITUDES.to(x.device)
    away = (y.clamp(max=6.0)[..., None] - mag).abs()
    code = away.argmin(-1)  # the lower of two equally near codes
    up = (code + 1).clamp(max=7)
    tie = (code < 7) & (away.gather(-1, up[..., None])[..., 0] == away.gather(-1, code[..., None])[..., 0])
    code = torch.where(tie & (code % 2 == 1), up, code)
    code = torch.where(nan[..., None], 0, code)
    byte = torch.where(nan, 255, byte)
    value = torch.where(b < 0, -1.0, 1.0) * mag[code] * scale_of(byte)[..., None]
    return (code + 8 * (b < 0)).flatten(-2), byte, value.flatten(-2)


def scale_of(byte):
    return torch.where(byte == 255, float("nan"), torch.ldexp(torch.ones_like(byte, dtype=torch.float64), byte.long() - 127))


def parts(cache, P, D):
    c, s = P * D // 2, P * D // 32
    cut = lambda lo, n: cache[:, :, lo:lo + n].unflatten(-1, (P, n // P))  # noqa: E731
    return cut(0, c), cut(c, c), cut(2 * c, s), cut(2 * c + s, s)


def store(cache, P, D, page, slot, which, codes, byte):
    """Writes codes [n, heads, D] and scale bytes of keys (which = 0) or values (1) to (page, slot) pairs."""
    p = parts(cache, P, D)
    p[which][page, :, slot] = (codes[..., 0::2] | codes[..., 1::2] << 4).to(torch.uint8)
    p[2 + which][page, :, slot] = byte.to(torch.uint8)


def load(cache, P, D, pages, length, which):
    """float64 [length, heads, D] of the first positions of the pages."""
    p = parts(cache, P, D)
    codes, byte = p[which][pages], p[2 + which][pages]  # [pages, heads, P, ..]
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    x = MAGNITUDES.to(cache.device)[both % 8] * torch.where(both >= 8, -1.0, 1.0)
    x = (x.unflatten(-1, (-1, 32)) * scale_of(byte)[..., None]).flatten(-2)
    return x.transpose(1, 2).flatten(0, 1)[:length]


def rotate(x, pos, inv_freq, mscale):
    """x [n, heads, D] by the positions [n]; element j pairs with j + D/2."""
    angle = pos.double()[:, None, None] * inv_freq.double()
    c, s = torch.cos(angle) * mscale, torch.sin(angle) * mscale
    a, b = x.double().chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def attend(q, k, v, pos, sinks, window, scale):
    """q [n, nq, D] at positions pos [n] over k, v [length, nkv, D]; returns (out, sum of weight * |v| over the
    denominator), both [n, nq, D]; rows without a position are zero."""
    n, nq, D = q.shape
    nkv = k.shape[1]
    qg = q.double().unflatten(1, (nkv, nq // nkv))
    p = torch.arange(k.shape[0], device=q.device)
    seen = p[None] <= pos[:, None]
    if window:
        seen &= p[None] > pos[:, None] - window
    # positions that no row sees take no part, whatever they hold
    any_seen = seen.any(0)
    k, v, seen = k[any_seen], v[any_seen], seen[:, any_seen]
    score = torch.einsum("nhgd,shd->nhgs", qg, k) * scale
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True) if score.shape[-1] else torch.full((*score.shape[:-1], 1), -math.inf, dtype=torch.float64, device=q.device)
    if sinks is not None:
        top = torch.maximum(top, sinks.double().view(nkv, -1, 1))
    top = torch.where(top == -math.inf, 0.0, top)
    w = torch.exp(score - top)
    total = w.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + torch.exp(sinks.double().view(nkv, -1, 1) - top)
    w = w / torch.where(total == 0, 1.0, total)
    # a row is not touched by values that it does not see
    vm = torch.where(seen[:, :, None, None], v[None], 0.0) if v.isnan().any() else v.expand(n, *v.shape)
    out = torch.einsum("nhgs,nshd->nhgd", w, vm)
    mass = torch.einsum("nhgs,nshd->nhgd", w, vm.abs())
    return out.flatten(1, 2), mass.flatten(1, 2)
