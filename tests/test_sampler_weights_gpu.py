"""Sampling where weights are next to nothing: logits whose weights round to none, temperatures whose scale leaves f32."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def f32(values):
    return torch.tensor(values, dtype=torch.float32, device=DEV)


def run(sampler, x, u, **kw):
    """(tokens, probabilities, counts), the tokens written over a value that no row can have."""
    out = torch.full((x.shape[0],), -99, dtype=torch.int32, device=DEV)
    token, prob, kept = sampler.run(x, f32(u), out=out, details=True, **kw)
    return token.tolist(), prob.tolist(), kept.tolist()


def units(x, t):
    """Weights of a row as the definition rounds them: whole numbers of 2^-43 of the largest."""
    x = x.double().cpu().numpy()
    return np.rint(np.exp((x - x.max()) / t) * 2.0 ** 43)


@pytest.mark.parametrize("vocab,peak", [(201088, 150000), (201088, 201087), (201088, 200), (7169, 7000), (7169, 200), (20011, 1024)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_too_light_to_be_drawn(vocab, peak, dtype):
    """One logit far above the rest: theirs weigh 2^-43 or less each, and together more.  The token is the first whose running sum
    of ROUNDED weights exceeds the number's share of theirs."""
    from neonengine_b200.sampler import Sampler
    gaps = [29.0, 30.25, 30.75, 31.0, 32.0, 33.0, 34.5, 36.0, 40.0, 100.0]
    numbers = [0.0, float("nan"), -1.0, 2.0 ** -40, 2.0 ** -24, 0.5, 1 - 2.0 ** -24]
    s = Sampler(vocab)
    for t in (1.0, 0.5):
        x = torch.zeros((len(gaps) * len(numbers), vocab), dtype=dtype, device=DEV)
        for i, gap in enumerate(gaps):
            x[i * len(numbers):(i + 1) * len(numbers), peak] = gap * t
        token, prob, kept = run(s, x, numbers * len(gaps), temperature=f32([t] * x.shape[0]))
        for i in range(len(gaps)):
            w = units(x[i * len(numbers)], t)
            mass = np.cumsum(w)
            for j, u in enumerate(numbers):
                u = 0.0 if not u > 0 else u
                # (2^-24 of the sum is more than all light logits weigh, 2^-40 less than the first eight of a chunk)
                want = int(np.searchsorted(mass, u * mass[-1], side="right"))
                row = i * len(numbers) + j
                assert token[row] == want, (gaps[i], numbers[j], token[row], want)
                # the whole row's weight holds what the rounding dropped, up to half a unit a token
                share = w[want] / mass[-1]
                assert abs(prob[row] - share) <= 2 ** -24 * share * 1.01 + 1e-9 + vocab * 2.0 ** -44
                assert kept[row] == vocab
    s.close()


@pytest.mark.parametrize("vocab", [7169, 201088])
def test_light_logits_before_behind_and_between(vocab):
    """Stretches of unequal light logits, all masked ones among them, and a mass of two: every number gives a token."""
    from neonengine_b200.sampler import Sampler
    g = torch.Generator(device=DEV)
    g.manual_seed(vocab)
    n = 64
    x = -31.5 - 3 * torch.rand((n, vocab), generator=g, device=DEV)
    x[:, 1024:2048] = -float("inf")
    x[:, 5000], x[:, 6500] = 0.0, -1.0
    u = [0.0] * 8 + [2.0 ** -e for e in range(149, 93, -1)]
    s = Sampler(vocab)
    token, prob, kept = run(s, x, u)
    assert token == [5000] * n and kept == [vocab - 1024] * n
    token, _, _ = run(s, x, [1 - 2.0 ** -24] * n)
    assert token == [6500] * n
    # with a cut by top_p alone, light logits of the row are not what reaches it either
    token, _, kept = run(s, x, u, top_p=f32([0.999999] * n))
    assert token == [5000] * n and kept == [2] * n
    s.close()


@pytest.mark.parametrize("vocab", [7169, 20011, 201088])
@pytest.mark.parametrize("t", [1e-36, 1e-37, 2e-38, 1e-38, 1e-44])
def test_temperatures_whose_scale_leaves_f32(vocab, t):
    """The largest logit is exactly zero and the temperature next to nothing: the zeros share everything."""
    from neonengine_b200.sampler import Sampler
    g = torch.Generator(device=DEV)
    g.manual_seed(vocab)
    zeros = sorted({1, 1500, vocab // 2, vocab - 3})
    x = -1 - torch.rand((6, vocab), generator=g, device=DEV)
    x[:, zeros] = 0.0
    u = [0.0, 0.2, 0.3, 0.6, 0.8, 0.999]
    want = [zeros[int(v * len(zeros))] for v in u]
    s = Sampler(vocab)
    temperature = f32([t] * 6)
    token, prob, kept = run(s, x, u, temperature=temperature)
    assert token == want and all(abs(p - 1 / len(zeros)) < 1e-7 for p in prob) and kept == [vocab] * 6
    token, prob, kept = run(s, x, u, temperature=temperature, top_p=f32([0.9] * 6))
    assert token == want and kept == [len(zeros)] * 6
    token, prob, kept = run(s, x, u, temperature=temperature, top_p=f32([0.4] * 6))  # reached by the second of them
    assert token == [zeros[int(v * 2)] for v in u] and kept == [2] * 6
    s.close()


@pytest.mark.parametrize("t", [1.0, 0.3, 1e-30, 7.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_largest_logits_that_no_list_holds(t, dtype):
    """Thousands of equal largest logits fill stretches of their own; the only listed tokens weigh little or nothing."""
    from neonengine_b200.sampler import Sampler
    import sampler_reference as ref
    vocab = 20011
    x = torch.full((7, vocab), -60.0, device=DEV)
    x[:, 100:150] = -55.0            # fifty that a stretch lists
    x[:, 10240:14336] = 0.0          # 4096 that none can
    x[:, 11000] = -0.0
    x[3:, 3000:3020] = -1.0          # some more, of weight
    x = x.to(dtype)
    u = [0.0, 0.3, 0.77, 0.9, 1 - 2.0 ** -24, 0.55, 0.1234]
    s, rows = Sampler(vocab), x.double().cpu().numpy()
    for k, p, m in ((0, 0.3, 0.0), (0, 0.9, 0.0), (0, 0.001, 0.0), (0, 1.0, 1.0), (0, 1.0, 0.99), (0, 0.9, 1.0), (0, 0.3, 1e-6), (100, 1.0, 0.0), (5000, 0.3, 0.5)):
        n = x.shape[0]
        token, prob, kept = run(s, x, u, temperature=f32([t] * n), top_k=torch.full((n,), k, dtype=torch.int32, device=DEV),
                                top_p=f32([p] * n), min_p=f32([m] * n))
        for b in range(n):
            want = ref.draw(rows[b], float(np.float32(u[b])), float(np.float32(t)), k, float(np.float32(p)), float(np.float32(m)))
            assert (token[b], kept[b]) == (want[0], want[2]), (k, p, m, b, token[b], kept[b], want)
            assert abs(prob[b] - want[1]) <= 2 ** -24 * want[1] * 1.01 + 1e-9
    s.close()
