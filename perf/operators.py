"""What a decoding server does around the dense layers, as measurable cases: appending keys and values to a paged
4-bit cache with the position rotation on the way, attention over that cache (one token a sequence, a few drafted
tokens, a chunk of a prompt), and sampling the next token.

`listed()` holds fixed cases, `draw(rng)` makes more of the same ranges; `prepare(case, seed)` builds what a program
holds before the call, `run(state)` is one pass, `work(case)` what it cannot do without, and `exact(case, seed)` the
same outputs in 64 bits.  `own` chooses between the plain form (elementary torch operations) and the framework's own
entry points.

The cache: uint8 [pages, kv heads, record].  A record holds P positions: P * D/2 bytes of key codes (a position after the
other, even column in the low nibble), as many of value codes, P * D/32 key scales and P * D/32 value scales.  Codes are
e2m1 (sign, two exponent bits, one mantissa bit), scales E8M0, one for 32 columns."""
from __future__ import annotations

import functools
import math
import random

import numpy as np
import torch

DEV = "cuda:0"
own = False
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _append(name, batch, most, position, nq=64, nkv=8, dim=64, page=64, dtype="bf16", pad=0):
    return {"name": name, "kind": "append", "batch": batch, "most": most, "position": position, "nq": nq, "nkv": nkv, "dim": dim,
            "page": page, "dtype": dtype, "pad": pad}


def _attend(name, batch, most, context, ragged=True, nq=64, nkv=8, dim=64, page=64, dtype="bf16", window=0, sinks=True):
    return {"name": name, "kind": "attend", "batch": batch, "most": most, "context": context, "ragged": ragged, "nq": nq, "nkv": nkv,
            "dim": dim, "page": page, "dtype": dtype, "window": window, "sinks": sinks}


def _sample(name, batch, vocab, mode, dtype="fp32", pad=0):
    return {"name": name, "kind": "sample", "batch": batch, "vocab": vocab, "mode": mode, "dtype": dtype, "pad": pad}


def listed():
    return [
        # a decoding batch's new tokens, one a sequence, somewhere in their contexts
        _append("append 8 tokens", 8, 1, 4095),
        # a busy server's decoding step, in a buffer padded to the next captured size
        _append("append 200 tokens padded", 200, 1, 20000, pad=56),
        # a pass of prompt chunks
        _append("append prompt chunks", 6, 2500, 6000),
        # one conversation in the middle of its context: latency is everything
        _attend("attend 1 at 1500", 1, 1, 1500, ragged=False),
        # a full batch at the end of its context
        _attend("attend 8 at 4096", 8, 1, 4096, ragged=False),
        # the sliding-window layers of the same step
        _attend("attend 8 window 128", 8, 1, 4096, ragged=False, window=128),
        # a busy server: many sequences, short and long ones
        _attend("attend 64 ragged to 32768", 64, 1, 32768),
        # drafted tokens under verification, wide heads in small pages
        _attend("attend 5 drafted tokens", 24, 5, 6000, nq=32, nkv=8, dim=128, page=16),
        # chunks of two prompts over what is cached of them
        _attend("attend prompt chunks", 2, 2048, 8192),
        # the next token of one conversation, all filters on
        _sample("sample 1", 1, 201088, "all"),
        # a server's batch: every user has settings of their own
        _sample("sample 64 mixed", 64, 201088, "mixed"),
        # rollouts for training: the whole distribution, no filter
        _sample("sample 256 unfiltered", 256, 201088, "none"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    nkv = rng.choice([1, 2, 4, 8, 8, 8])
    dim = rng.choice([64, 64, 64, 128])
    return {"nq": nkv * rng.choice([1, 2, 4, 8, 8] if dim == 64 else [1, 2, 4, 4]), "nkv": nkv, "dim": dim, "page": rng.choice([16, 32, 64, 64])}


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "sample", "sample"])
    if kind == "append":
        most = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 20, 2500)])
        c = _append("", _log_int(rng, 1, 256) if most <= 8 else rng.randint(1, 6), most, _log_int(rng, 1, 60000),
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), pad=rng.choice([0, rng.randint(1, 40)]), **_heads(rng))
    elif kind == "attend":
        form = rng.choice(["one", "one", "one", "few", "chunk"])
        if form == "one":
            batch = _log_int(rng, 1, 64)
            most, context = 1, _log_int(rng, 1, 32768)
        elif form == "few":
            batch, most, context = _log_int(rng, 1, 32), rng.randint(2, 12), _log_int(rng, 12, 12000)
        else:
            batch, most, context = rng.randint(1, 2), _log_int(rng, 40, 2048), _log_int(rng, 2048, 8192)
        c = _attend("", batch, most, context, rng.random() < 0.7, dtype=rng.choice(["bf16", "bf16", "fp16"]),
                    window=rng.choice([0, 0, 128, rng.randint(1, 1500)]), sinks=rng.random() < 0.6, **_heads(rng))
    else:
        c = _sample("", _log_int(rng, 1, 256), _log_int(rng, 1000, 201088), rng.choice(["none", "top-k", "top-p", "min-p", "all", "mixed", "mixed"]),
                    rng.choice(["fp32", "fp32", "bf16"]), rng.choice([0, 0, rng.randint(1, 60)]))
    c.pop("name", None)
    return c


# ---- 4-bit values -----------------------------------------------------------------------------------------------
def _to_4bit(x):
    """(codes [..., D] in 0..15, scale bytes [..., D/32]) of values in 64 bits."""
    b = x.unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1)
    exponent = torch.frexp(amax)[1] - 1  # floor(log2 amax)
    byte = torch.where(amax > 0, (exponent - 2 + 127).clamp(1, 254), 127)
    y = torch.ldexp(b.abs(), (127 - byte)[..., None])
    code = ((y > 0.25).int() + (y >= 0.75).int() + (y > 1.25).int() + (y >= 1.75).int() + (y > 2.5).int() + (y >= 3.5).int() + (y > 5.0).int())
    return (code + 8 * (b < 0).int()).flatten(-2), byte


def _parts(cache, page, dim):
    """Views of the records' four parts: key codes, value codes [pages, heads, P, D/2], key scales, value scales [.., P, D/32]."""
    c, s = page * dim // 2, page * dim // 32
    cut = lambda lo, n: cache[:, :, lo:lo + n].unflatten(-1, (page, n // page))  # noqa: E731
    return cut(0, c), cut(c, c), cut(2 * c, s), cut(2 * c + s, s)


def _values(codes, scales):
    """fp32 values of packed codes [..., D/2] and scale bytes [..., D/32]."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    return (table[both.int()].unflatten(-1, (-1, 32)) * torch.exp2(scales.float() - 127)[..., None]).flatten(-2)


def _pack(codes):
    return (codes[..., 0::2] | codes[..., 1::2] << 4).to(torch.uint8)


# ---- states -----------------------------------------------------------------------------------------------------
def _lengths(case):
    """(new tokens, cached positions with them) of every sequence; part of the case, the same for each seed."""
    B, most = case["batch"], case["most"]
    rng = random.Random(1000 * B + most)
    top = case["position"] + most if case["kind"] == "append" else case["context"]
    rows, lens = [], []
    for b in range(B):
        full = b == 0 or (case["kind"] == "attend" and not case["ragged"])
        n = most if full or most <= 1 else rng.randint(max(1, most // 3), most)
        lo = max(n, top // 20)
        rows.append(min(n, top))
        lens.append(top if full else max(rows[-1], _log_int(rng, lo, top) if lo < top else top))
    return rows, lens


def _inv_freq(dim):
    """Rotary frequencies of base 150000, stretched by 32 from 4096 positions (by parts), and the factor of cos and sin."""
    theta, factor, first, fast, slow = 150000.0, 32.0, 4096.0, 32.0, 1.0
    at = lambda turns: dim * math.log(first / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    low, high = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), dim - 1)
    i = np.arange(dim // 2)
    freq = theta ** (-2.0 * i / dim)
    ramp = np.clip((i - low) / (high - low), 0, 1)
    return torch.from_numpy((freq / factor * ramp + freq * (1 - ramp)).astype(np.float32)).to(DEV), 0.1 * math.log(factor) + 1.0


def _batch(case, g):
    rows, lens = _lengths(case)
    P = case["page"]
    need = [-(-n // P) for n in lens]
    order = torch.randperm(sum(need) + 3, generator=g, device=DEV)  # pages lie anywhere
    table = torch.zeros((len(lens), max(need)), dtype=torch.int32, device=DEV)
    first = np.concatenate([[0], np.cumsum(need)])
    for b, n in enumerate(need):
        table[b, :n] = order[first[b]:first[b] + n]
    return {"rows": sum(rows), "most": max(rows), "cu_q": torch.tensor([0, *np.cumsum(rows)], dtype=torch.int32, device=DEV),
            "seq_lens": torch.tensor(lens, dtype=torch.int32, device=DEV), "table": table, "pages": sum(need) + 3}


def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _prepare_append(case, seed):
    g = _generator(seed)
    s = {"kind": "append", "case": case, **_batch(case, g)}
    nq, nkv, dim, P = case["nq"], case["nkv"], case["dim"], case["page"]
    s["cache"] = torch.zeros((s["pages"], nkv, P * (dim + dim // 16)), dtype=torch.uint8, device=DEV)
    T = s["rows"] + case["pad"]
    # the projection's output, of which q, k and v are columns; some columns of a head are larger than others
    qkv = torch.randn((T, nq + 2 * nkv, dim), generator=g, device=DEV) * torch.exp(0.5 * torch.randn((nq + 2 * nkv, dim), generator=g, device=DEV))
    qkv = qkv.to(DTYPES[case["dtype"]])
    s["q"], s["k"], s["v"] = qkv[:, :nq], qkv[:, nq:nq + nkv], qkv[:, nq + nkv:]
    s["inv_freq"], s["mscale"] = _inv_freq(dim)
    s["out"] = torch.zeros((T, nq, dim), dtype=torch.float16 if case["dtype"] == "fp16" else torch.bfloat16, device=DEV)
    s["held"] = [torch.zeros((T, nkv, dim), dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    return s


def _prepare_attend(case, seed):
    g = _generator(seed)
    s = {"kind": "attend", "case": case, **_batch(case, g)}
    nq, nkv, dim, P = case["nq"], case["nkv"], case["dim"], case["page"]
    dtype = DTYPES[case["dtype"]]
    s["cache"] = torch.empty((s["pages"], nkv, P * (dim + dim // 16)), dtype=torch.uint8, device=DEV)
    kc, vc, ks, vs = _parts(s["cache"], P, dim)
    wide = torch.exp(0.4 * torch.randn((nkv, 1, dim), generator=g, device=DEV))
    step = max(1, (1 << 25) // (nkv * P * dim))
    for p in range(0, s["pages"], step):
        n = min(step, s["pages"] - p)
        for codes, scales in ((kc, ks), (vc, vs)):
            c, b = _to_4bit(torch.randn((n, nkv, P, dim), generator=g, device=DEV) * wide)
            codes[p:p + n], scales[p:p + n] = _pack(c), b.to(torch.uint8)
    s["q"] = (1.5 * torch.randn((s["rows"], nq, dim), generator=g, device=DEV)).to(dtype)
    s["sinks"] = torch.randn((nq,), generator=g, device=DEV).to(torch.bfloat16) if case["sinks"] else None
    s["out"] = torch.zeros((s["rows"], nq, dim), dtype=dtype, device=DEV)
    return s


def _prepare_sample(case, seed):
    g = _generator(seed)
    B, V, mode = case["batch"], case["vocab"], case["mode"]
    rand = lambda *n: torch.rand(n, generator=g, device=DEV)  # noqa: E731
    logits = torch.randn((B, V + case["pad"]), generator=g, device=DEV) * (1 + 2 * rand(B, 1))
    likely = torch.randint(0, V, (B, 40), generator=g, device=DEV)  # the tokens that the context suggests
    logits.scatter_add_(1, likely, 12 * rand(B, 40) ** 2 + 3)
    logits[:, V:] = float("nan")  # the rows' padding is not read
    s = {"kind": "sample", "logits": logits.to(DTYPES[case["dtype"]])[:, :V], "uniform": rand(B), "temperature": 0.6 + 0.6 * rand(B)}
    on = lambda share: rand(B) < (share if mode == "mixed" else 1.0)  # noqa: E731
    top_k = torch.where(on(0.5), torch.randint(20, 200, (B,), generator=g, device=DEV), 0).int()
    top_p = torch.where(on(0.5), 0.8 + 0.19 * rand(B), 1.0)
    min_p = torch.where(on(0.3), 0.1 * rand(B), 0.0)
    if mode == "mixed":
        s["temperature"] = torch.where(rand(B) < 0.15, 0.0, s["temperature"])  # some users want the likeliest token
    s["top_k"] = top_k if mode in ("top-k", "all", "mixed") else None
    s["top_p"] = top_p if mode in ("top-p", "all", "mixed") else None
    s["min_p"] = min_p if mode in ("min-p", "all", "mixed") else None
    return s


def prepare(case, seed):
    return {"append": _prepare_append, "attend": _prepare_attend, "sample": _prepare_sample}[case["kind"]](case, seed)


# ---- the framework's calls --------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _kv_system(nq, nkv, dim, page):
    """A program holds one of these for its model."""
    from neonengine_b200.kv4_cache import Kv4Cache
    return Kv4Cache(n_q_heads=nq, n_kv_heads=nkv, head_dim=dim, page_size=page)


@functools.lru_cache(maxsize=None)
def _sampler(vocab):
    from neonengine_b200.sampler import Sampler
    return Sampler(vocab)


def _own(s):
    if s["kind"] == "sample":
        sampler = _sampler(s["logits"].shape[1])
        token, prob, kept = sampler.run(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                        min_p=s["min_p"], details=True)
        return {"token": token, "prob": prob, "kept": kept}
    c = s["case"]
    kv = _kv_system(c["nq"], c["nkv"], c["dim"], c["page"])
    batch = kv.batch(s["seq_lens"], s["table"], cu_q=s["cu_q"])
    if s["kind"] == "append":
        q = kv.append(batch, s["cache"], s["q"], s["k"], s["v"], s["inv_freq"], mscale=s["mscale"], out=s["out"])
        k, v = kv.read(batch, s["cache"], out=s["held"])
        return {"q": q, "k": k, "v": v}
    return {"out": kv.attend(batch, s["cache"], s["q"], sinks=s["sinks"], window=c["window"], max_rows=s["most"], out=s["out"])}


# ---- the plain forms --------------------------------------------------------------------------------------------
def _plain_append(s):
    c, n = s["case"], s["rows"]
    P, dim = c["page"], c["dim"]
    row = torch.arange(n, device=DEV)
    seq = torch.searchsorted(s["cu_q"], row, right=True) - 1
    pos = s["seq_lens"][seq].long() - s["cu_q"][seq + 1] + row
    angle = pos.double()[:, None, None] * s["inv_freq"].double()  # in 64 bits: far positions, values next to a border
    cos, sin = torch.cos(angle) * s["mscale"], torch.sin(angle) * s["mscale"]

    def turn(x):
        a, b = x.double().chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    page, at = s["table"][seq, pos // P].long(), pos % P
    kc, vc, ks, vs = _parts(s["cache"], P, dim)
    (k_codes, k_bytes), (v_codes, v_bytes) = _to_4bit(turn(s["k"][:n])), _to_4bit(s["v"][:n].double())
    kc[page, :, at], ks[page, :, at] = _pack(k_codes), k_bytes.to(torch.uint8)
    vc[page, :, at], vs[page, :, at] = _pack(v_codes), v_bytes.to(torch.uint8)
    s["out"][:n] = turn(s["q"][:n]).to(s["out"].dtype)
    s["held"][0][:n] = _values(kc[page, :, at], ks[page, :, at]).to(torch.bfloat16)
    s["held"][1][:n] = _values(vc[page, :, at], vs[page, :, at]).to(torch.bfloat16)
    return {"q": s["out"], "k": s["held"][0], "v": s["held"][1]}


def _plain_attend(s):
    c = s["case"]
    P, dim, nkv, G = c["page"], c["dim"], c["nkv"], c["nq"] // c["nkv"]
    kc, vc, ks, vs = _parts(s["cache"], P, dim)
    pages = s["table"].long()
    k, v = (_values(codes[pages], scales[pages]).transpose(2, 3).flatten(1, 2) for codes, scales in ((kc, ks), (vc, vs)))  # [B, S, heads, D]
    lens, first = s["seq_lens"].long(), s["cu_q"][:-1].long()
    new = s["cu_q"][1:].long() - first
    i = torch.arange(s["most"], device=DEV)
    real = i < new[:, None]  # [B, n]
    row = torch.where(real, first[:, None] + i, 0)
    at = (lens - new)[:, None] + i  # position of each row
    q = s["q"][row].float().unflatten(2, (nkv, G))  # [B, n, heads, G, D]
    score = torch.einsum("bnhgd,bshd->bhgns", q, k) * dim**-0.5
    p = torch.arange(k.shape[1], device=DEV)
    seen = p <= at[..., None]  # [B, n, S]
    if c["window"]:
        seen &= p > at[..., None] - c["window"]
    score = score.masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    sink = None if s["sinks"] is None else s["sinks"].float().view(nkv, G, 1, 1)
    top = top if sink is None else torch.maximum(top, sink)
    weight = score.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    total = total if sink is None else total + torch.exp(sink - top)
    out = torch.einsum("bhgns,bshd->bhgnd", weight, v) / total
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3)  # [B, n, nq, D]
    return {"out": out[real].to(s["out"].dtype)}


def _plain_sample(s):
    x = s["logits"].double()
    B, V = x.shape
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    cold = s["temperature"].double()[:, None] <= 0
    w = torch.exp((x - x[:, :1]) / torch.where(cold, 1.0, s["temperature"].double()[:, None]))
    mass = torch.cumsum(w, 1)
    rank = torch.arange(V, device=DEV)
    keep = (x > float("-inf")) & (~cold | (rank == 0))
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        keep &= (k <= 0) | (rank < k)
    if s["top_p"] is not None:
        whole = mass.gather(1, keep.sum(1, keepdim=True) - 1)
        top_p = s["top_p"].double()[:, None]
        keep &= (top_p >= 1) | (mass - w < top_p * whole)
    if s["min_p"] is not None:
        keep &= w >= s["min_p"].double()[:, None]
    kept = keep.sum(1)
    w = torch.zeros_like(w).scatter_(1, order, w * keep)  # back in the tokens' order
    mass = torch.cumsum(w, 1)
    token = torch.searchsorted(mass, s["uniform"].double()[:, None] * mass[:, -1:], right=True)
    return {"token": token[:, 0].int(), "prob": (w.gather(1, token) / mass[:, -1:])[:, 0].float(), "kept": kept.int()}


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[state["kind"]](state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "sample":
        n = case["batch"] * case["vocab"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + case["batch"] * 32, "flops": 4 * n}
    rows, lens = _lengths(case)
    nq, nkv, dim = case["nq"], case["nkv"], case["dim"]
    held = 2 * nkv * (dim // 2 + dim // 32)  # bytes of one position
    if case["kind"] == "append":
        n, size = sum(rows), 4 if case["dtype"] == "fp32" else 2
        return {"bytes": n * ((nq + 2 * nkv) * dim * size + nq * dim * 2 + 2 * held + 2 * nkv * dim * 2), "flops": n * (nq + nkv) * dim * 3}
    size = 2 * 2 * nq * dim * sum(rows)
    flops = 0
    for n, length in zip(rows, lens):
        window = case["window"] or length
        size += held * min(length, window + n - 1)
        seen = sum(min(length - n + i + 1, window) for i in range(n))
        flops += 4 * dim * nq * seen
    return {"bytes": size, "flops": flops}


# ---- the same in 64 bits, sequence by sequence ---------------------------------------------------------------------
_MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def _exact_4bit(x):
    """The nearest values that four bits and a scale hold, of an array [..., D] in 64 bits."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    amax = np.abs(b).max(-1, keepdims=True)
    scale = np.where(amax > 0, 2.0 ** (np.floor(np.log2(np.where(amax > 0, amax, 1.0))) - 2), 1.0)
    y = np.abs(b) / scale
    best = np.abs(y[..., None] - _MAGNITUDES)
    lower = best.argmin(-1)  # the lower of two equally near ones, which is right where its code is even
    tie = (lower < 7) & (np.abs(y - _MAGNITUDES[lower]) == np.abs(y - _MAGNITUDES[np.minimum(lower + 1, 7)]))
    code = np.where(tie & (lower % 2 == 1), lower + 1, lower)
    return (np.sign(b) * _MAGNITUDES[code] * scale).reshape(x.shape)


def _exact_append(case, seed):
    s = _prepare_append(case, seed)
    rows, lens = _lengths(case)
    pos = np.concatenate([np.arange(length - n, length) for n, length in zip(rows, lens)]).astype(np.float64)
    turns = torch.polar(torch.full((), s["mscale"], dtype=torch.float64), torch.from_numpy(np.outer(pos, s["inv_freq"].cpu().numpy().astype(np.float64))))

    def rotated(x):
        half = x.shape[-1] // 2
        z = torch.complex(x[..., :half].cpu().double(), x[..., half:].cpu().double()) * turns[:, None]
        return torch.cat([z.real, z.imag], -1)

    n, T = sum(rows), s["q"].shape[0]

    def padded(x):
        full = torch.zeros((T, *x.shape[1:]), dtype=torch.float64)
        full[:n] = torch.as_tensor(x)
        return full

    def in_4bit(x):
        return padded(np.concatenate([_exact_4bit(x[i:i + 256]) for i in range(0, n, 256)]))

    return {"q": padded(rotated(s["q"][:n])), "k": in_4bit(rotated(s["k"][:n]).numpy()), "v": in_4bit(s["v"][:n].cpu().double().numpy())}


def _exact_attend(case, seed):
    s = _prepare_attend(case, seed)
    rows, lens = _lengths(case)
    P, dim, nkv, G = case["page"], case["dim"], case["nkv"], case["nq"] // case["nkv"]
    signed = torch.from_numpy(np.concatenate([_MAGNITUDES, -_MAGNITUDES])).to(DEV)
    out = torch.empty((sum(rows), nkv, G, dim), dtype=torch.float64, device=DEV)
    q, half, at = s["q"].double().view(-1, nkv, G, dim), P * dim // 2, 0
    for b, (n, length) in enumerate(zip(rows, lens)):
        record = s["cache"][s["table"][b, :-(-length // P)].long()]
        p = torch.arange(length, device=DEV)
        for h in range(nkv):
            kv = []
            for part in range(2):
                byte = record[:, h, part * half:(part + 1) * half].reshape(-1, dim // 2)[:length].long()
                scale = record[:, h, 2 * half + part * P * dim // 32:][:, :P * dim // 32].reshape(-1, dim // 32)[:length].double()
                x = torch.empty((length, dim), dtype=torch.float64, device=DEV)
                x[:, 0::2], x[:, 1::2] = signed[byte % 16], signed[byte // 16]
                kv.append(x * (2.0 ** (scale - 127)).repeat_interleave(32, 1))
            score = torch.matmul(q[at:at + n, h], kv[0].T) / math.sqrt(dim)  # [n, G, length]
            here = (length - n + torch.arange(n, device=DEV))[:, None]
            hidden = p > here
            if case["window"]:
                hidden |= p <= here - case["window"]
            score.masked_fill_(hidden[:, None], -float("inf"))
            if s["sinks"] is not None:
                score = torch.cat([score, s["sinks"].double().view(nkv, 1, G, 1)[h].expand(n, G, 1)], 2)
            weight = torch.softmax(score, 2)
            out[at:at + n, h] = torch.matmul(weight[..., :length], kv[1])
        at += n
    return {"out": out.flatten(1, 2)}


def _exact_sample(case, seed):
    s = _prepare_sample(case, seed)
    probs = []
    host = {k: None if s[k] is None else s[k].double().cpu().numpy() for k in ("uniform", "temperature", "top_k", "top_p", "min_p")}
    for b, x in enumerate(s["logits"]):
        x = x.double().cpu().numpy()
        if host["temperature"][b] <= 0:
            probs.append(1.0)
            continue
        order = np.argsort(-x, kind="stable")
        p = np.exp((x - x.max()) / host["temperature"][b])
        if host["top_k"] is not None and host["top_k"][b] > 0:
            order = order[:int(host["top_k"][b])]
        if host["top_p"] is not None and host["top_p"][b] < 1:
            mass = np.cumsum(p[order])
            order = order[:np.searchsorted(mass, host["top_p"][b] * mass[-1]) + 1]
        if host["min_p"] is not None:
            order = order[p[order] >= host["min_p"][b]]
        mass = np.cumsum(p[np.sort(order)])
        probs.append(p[np.sort(order)[np.searchsorted(mass, host["uniform"][b] * mass[-1], side="right")]] / mass[-1])
    return {"token": None, "prob": np.array(probs), "kept": None}


def exact(case, seed):
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["kind"]](case, seed)
