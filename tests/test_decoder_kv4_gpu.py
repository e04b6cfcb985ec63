"""The decoder stack over its 4-bit cache and with sampled tokens: append, attention and sampling as one step uses them.

A step's attention is compared with the same kernels' result for the step's own projections in a cache that the test keeps
(bit for bit), and with the formula in 64 bits over what that cache holds.
"""
import dataclasses

import numpy as np
import pytest

import kv4_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
DEV = "cuda:0"


def small_shape(**kw):
    from neonengine_b200.decoder_synth import DecoderShape
    from neonengine_b200.synth import MoeShape
    hidden = kw.pop("hidden", 256)
    return DecoderShape(**{**dict(n_layers=2, hidden=hidden, n_q_heads=8, n_kv_heads=2, vocab=512, window=8,
                                  moe=MoeShape(hidden=hidden, inter=128, n_experts=8, top_k=4)), **kw})


def make(shape, B, ctx, seed, kv_bits=4):
    from neonengine_b200.decoder_synth import make_decoder_weights
    from neonengine_b200.decoder_system import DecoderSystem
    s = DecoderSystem(shape, B, ctx)
    s.set_weights(make_decoder_weights(shape, seed))
    s.set_option("kv_bits", kv_bits)
    return s


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Cache:
    """A cache of the test's own with the decoder's geometry."""

    def __init__(self, shape, B, ctx):
        from neonengine_b200.kv4_cache import Kv4Cache
        self.kv = Kv4Cache(shape.n_q_heads, shape.n_kv_heads, 64, 64)
        self.width = -(-ctx // 64)
        self.table = torch.arange(B * self.width, dtype=torch.int32, device=DEV).view(B, self.width)
        self.cache = self.kv.new_cache(B * self.width)
        self.shape, self.B = shape, B

    def load(self, k, v):
        """bf16 tensors [B, n, heads, 64] at positions 0 .. n - 1, as they are."""
        B, n = k.shape[:2]
        batch = self.kv.batch(torch.full((B,), n, dtype=torch.int32, device=DEV), self.table[:B], ints(*range(0, B * n + 1, n)))
        self.kv.append(batch, self.cache, None, k.flatten(0, 1), v.flatten(0, 1), torch.zeros(32, device=DEV))

    def attend(self, qkv, positions, window, inv_freq, mscale, sinks):
        """qkv fp32 [B, heads, 64] as projected; returns (attention, rotated queries)."""
        nq, nkv = self.shape.n_q_heads, self.shape.n_kv_heads
        batch = self.kv.batch((positions + 1).int(), self.table[:len(positions)])
        out = torch.empty((len(positions), nq, 64), dtype=torch.bfloat16, device=DEV)
        q = self.kv.append(batch, self.cache, qkv[:, :nq], qkv[:, nq:nq + nkv], qkv[:, nq + nkv:], inv_freq, mscale, out=out)
        return self.kv.attend(batch, self.cache, q, sinks=sinks, window=window, max_rows=1), q


def bf16(bits):
    return torch.from_numpy(np.ascontiguousarray(bits).view(np.int16)).view(torch.bfloat16).to(DEV)


@pytest.mark.parametrize("hidden", [256, 2112])  # 2112: the projection's depth is cut into two parts
@pytest.mark.parametrize("B,positions", [(3, [5, 70, 0]), (1, [99]), (8, [31, 63, 64, 65, 8, 9, 0, 127])])
def test_attention_over_the_decoders_cache(hidden, B, positions):
    from neonengine_b200.decoder_synth import make_decoder_weights, make_kv
    shape, ctx = small_shape(hidden=hidden), 128
    s, pos = make(shape, B, ctx, seed=3), torch.tensor(positions, device=DEV)
    w = make_decoder_weights(shape, 3)
    inv_freq = torch.from_numpy(s.read("inv_freq")).to(DEV)
    mscale = float(np.float32(0.1 * np.log(shape.rope_factor) + 1)) if shape.rope_factor > 1 else 1.0
    parts = 2 if hidden > 1536 else 1
    tokens, p32 = ints(*range(5, 5 + B)), pos.int()
    for layer in range(shape.n_layers):
        k, v = (bf16(x) for x in make_kv(shape, layer, B, ctx, 3))
        s.load_kv(layer, k, v)
        mine = Cache(shape, B, ctx)
        mine.load(k, v)
        s.set_option("stop_after_layer", layer + 1)
        s.step(tokens, p32)
        raw = np.empty((parts, B, shape.qkv_rows), np.float32)
        s._check(s._lib.neon_decoder_read(s._h, b"qkv", raw.ctypes.data, raw.nbytes), "read")
        qkv = raw[0] if parts == 1 else raw[0] + raw[1]
        window = shape.window if layer % 2 == 0 else 0
        sinks = bf16(w.attention[layer].sinks)
        want, q = mine.attend(torch.from_numpy(qkv).to(DEV).view(B, -1, 64), pos, window, inv_freq, mscale, sinks)
        got = bf16(s.read("attn", B)).view(B, -1, 64)
        assert torch.equal(got, want)
        for b in range(B):
            n = positions[b] + 1
            kk, vv = (ref.load(mine.cache, 64, 64, mine.table[b].long(), n, i) for i in range(2))
            exact, mass = ref.attend(q[b:b + 1], kk, vv, pos[b:b + 1], sinks, window, 0.125)
            # a rounding to bf16, f16 probabilities, scores in f32 (as in the cache's own tests)
            tol = 2 ** -8 * exact.abs() + (2 ** -11 + 2 ** -13) * mass * 1.01 + n * 2 ** -25 * vv.abs().amax()
            assert ((got[b:b + 1].double() - exact).abs() <= tol).all()
    status = np.empty(1, np.int32)
    s._check(s._lib.neon_decoder_read(s._h, b"kv4_status", status.ctypes.data, 4), "read")
    assert status[0] == 0
    s.close()


def test_load_kv_from_the_host():
    from neonengine_b200.decoder_synth import make_kv
    shape = small_shape()
    k, v = make_kv(shape, 0, 2, 40, 7)
    got = []
    for on_device in (False, True):
        s = make(shape, 2, 64, seed=4)
        s.load_kv(0, *((bf16(k), bf16(v)) if on_device else (k, v)))
        s.set_option("stop_after_layer", 1)
        s.step(ints(3, 4), ints(39, 40))
        got.append(s.read("attn"))
        s.close()
    np.testing.assert_array_equal(*got)
    assert np.abs(got[0].view(np.int16)).max() > 0


def test_steps_replayed_and_back_to_16_bits():
    """A few tokens of two sequences, with graphs and without: the same logits.  Switched to 4 bits and back, the bf16 path
    gives what it gave."""
    shape = dataclasses.replace(small_shape(), window=4)
    s = make(shape, 2, 192, seed=5, kv_bits=16)

    def run(steps=70):
        tokens, pos, nxt = ints(3, 4), ints(0, 100), torch.zeros(2, dtype=torch.int32, device=DEV)
        logits = torch.empty((2, shape.vocab), device=DEV)
        seen = []
        for _ in range(steps):
            s.step(tokens, pos, logits=logits, next_tokens=nxt)
            tokens.copy_(nxt)
            pos += 1
            seen.append(logits.clone())
        torch.cuda.synchronize()
        return torch.stack(seen)

    before = run()
    s.set_option("kv_bits", 4)
    replayed = run()
    s.set_option("kv_bits", 16)
    assert torch.equal(run(), before)
    s.set_option("kv_bits", 4)  # an empty cache again
    s.set_option("use_graphs", 0)
    assert torch.equal(run(), replayed)
    assert replayed.isfinite().all() and not torch.equal(replayed, before)
    bytes4 = s.step_bytes(np.array([99, 9], np.int32))[1]
    s.set_option("kv_bits", 16)
    assert s.step_bytes(np.array([99, 9], np.int32))[1] == bytes4 * 256 / 68
    s.close()


@pytest.mark.parametrize("kv_bits", [4, 16])
def test_sampled_tokens(kv_bits):
    """Every step's tokens are the sampler's for that step's logits; settings change between replays; then the largest again."""
    from neonengine_b200.sampler import Sampler
    shape, B = small_shape(vocab=20000), 3
    s, sampler = make(shape, B, 64, seed=6, kv_bits=kv_bits), Sampler(20000)
    uniform, temperature = torch.rand(4, device=DEV), torch.tensor([0.7, 1.0, 0.0, 2.0], device=DEV)
    top_k, top_p, min_p = ints(0, 50, 7, 1), torch.tensor([0.9, 1.0, 0.5, 1.0], device=DEV), torch.tensor([0.0, 0.01, 0.0, 0.2], device=DEV)
    s.set_sampling(uniform, temperature, top_k, top_p, min_p)
    tokens, pos, nxt = ints(3, 4, 5), ints(0, 1, 2), torch.zeros(B, dtype=torch.int32, device=DEV)
    logits = torch.empty((B, shape.vocab), device=DEV)
    drawn = []
    for i in range(6):
        uniform.copy_(torch.rand(4, device=DEV))
        if i == 3:
            temperature.fill_(1.5)
        s.step(tokens, pos, logits=logits, next_tokens=nxt)
        want = sampler.run(logits, uniform[:B], temperature[:B], top_k[:B], top_p[:B], min_p[:B])
        assert torch.equal(nxt, want)
        drawn.append(nxt.tolist())
        tokens.copy_(nxt)
        pos += 1
    host = s.step_host(nxt.cpu().numpy(), pos.cpu().numpy())
    assert host.shape == (B,) and (host >= 0).all() and (host < shape.vocab).all()
    s.set_sampling()
    s.step(tokens, pos, logits=logits, next_tokens=nxt)
    assert torch.equal(nxt, logits.argmax(-1).int())
    assert len(set(map(tuple, drawn))) > 1
    s.close()
    sampler.close()


def test_refusals():
    shape = small_shape()
    s = make(shape, 2, 64, seed=8)
    with pytest.raises(RuntimeError, match="kv_bits"):
        s.set_option("kv_bits", 8)
    with pytest.raises(RuntimeError, match="uniform"):
        s.set_sampling(temperature=torch.ones(2, device=DEV))
    with pytest.raises(ValueError):
        s.set_sampling(torch.ones(1, device=DEV))  # fewer than max_batch
    with pytest.raises(ValueError):
        s.set_sampling(torch.ones(2, device=DEV), top_k=torch.ones(2, device=DEV))
    with pytest.raises(ValueError):
        s.set_sampling(torch.ones(2))
    s.set_option("kv_bits", 16)
    with pytest.raises(RuntimeError, match="kv4_status"):
        word = np.empty(1, np.int32)
        s._check(s._lib.neon_decoder_read(s._h, b"kv4_status", word.ctypes.data, 4), "read")
    s.close()
    from neonengine_b200.decoder_system import DecoderSystem
    big = DecoderSystem(small_shape(vocab=400000), 1, 64)
    with pytest.raises(RuntimeError, match="vocabular"):
        big.set_sampling(torch.ones(1, device=DEV))
    big.close()
