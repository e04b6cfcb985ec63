"""The sampler on the GPU against its restatement in 64 bits."""
import numpy as np
import pytest
import torch

import sampler_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def samplers():
    from neonengine_b200.sampler import Sampler
    made = {}

    def get(vocab):
        if vocab not in made:
            made[vocab] = Sampler(vocab)
        return made[vocab]

    yield get
    for s in made.values():
        s.close()


def f32(values):
    return torch.tensor(values, dtype=torch.float32, device=DEV)


def check(sampler, logits, u, t=None, k=None, p=None, m=None):
    """Runs the rows and compares each with the restatement: the same token and count, the probability to its f32 rounding and
    that of the weights (1e-11)."""
    rows = logits.shape[0]
    tensors = [None if v is None else f32(v) for v in (t, p, m)]
    ks = None if k is None else torch.tensor(k, dtype=torch.int32, device=DEV)
    token, prob, kept = sampler.run(logits, f32(u), tensors[0], ks, tensors[1], tensors[2], details=True)
    x = logits.double().cpu().numpy()
    for b in range(rows):
        value = lambda v, none: none if v is None else float(np.float32(v[b]))  # noqa: E731
        want = ref.draw(x[b], value(u, 0), value(t, 1.0), 0 if k is None else k[b], value(p, 1.0), value(m, 0.0))
        got = (int(token[b]), float(prob[b]), int(kept[b]))
        assert (got[0], got[2]) == (want[0], want[2]), (b, got, want)
        assert abs(got[1] - want[1]) <= 2 ** -24 * want[1] * 1.01 + 1e-11, (b, got, want)
    return token, prob, kept


def rows_of(rows, vocab, seed, sigma=(1.0, 3.0), dtype=torch.float32):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    x = torch.randn((rows, vocab), generator=g, device=DEV)
    x *= torch.linspace(sigma[0], sigma[1], rows, device=DEV)[:, None]
    return x.to(dtype), torch.rand((rows,), generator=g, device=DEV).tolist()


# around the list that one CTA takes (6144), a warp's 1024, and the largest
VOCABS = [1, 2, 31, 1000, 6143, 6144, 6145, 7169, 20011, 201088, 393216]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_every_filter(samplers, vocab, dtype):
    n = 16
    x, u = rows_of(n, vocab, vocab, dtype=dtype)
    x[n // 2:] = torch.where(torch.rand((n // 2, vocab), device=DEV) < 0.001, x[n // 2:] * 3 + 4, x[n // 2:])  # some likely tokens
    t = [0.7 + 0.05 * i for i in range(n)]
    k = [0, 1, 5, 50, 0, 0, 0, 200, vocab, vocab + 7, -3, 1000, 3, 40, 0, 2]
    p = [1.0, 1.0, 0.9, 0.5, 0.9, 0.99, 0.0, 0.95, 1.0, 0.3, 0.8, 1.5, 0.99, 1.0, 0.999, 0.4]
    m = [0.0, 0.0, 0.0, 0.01, 0.0, 0.05, 0.0, 0.001, 0.1, 0.0, 0.02, 0.3, 1.0, 2.0, 0.0, -1.0]
    s = samplers(vocab)
    check(s, x, u)
    check(s, x, u, t=t)
    check(s, x, u, t=t, k=k)
    check(s, x, u, t=t, p=p)
    check(s, x, u, t=t, m=m)
    check(s, x, u, t=t, k=k, p=p, m=m)


@pytest.mark.parametrize("vocab", [500, 20011, 201088])
def test_many_rows_and_numbers(samplers, vocab):
    """Random numbers over the whole range, the ends among them."""
    n = 100
    x, u = rows_of(n, vocab, 3)
    u[0], u[1], u[2], u[3], u[4], u[5] = 0.0, 1 - 2.0 ** -24, 1.0, -1.0, float("nan"), 2.0 ** -24
    check(samplers(vocab), x, u)
    check(samplers(vocab), x, u, p=[0.9] * n)
    check(samplers(vocab), x, u, k=[7 * i for i in range(n)], m=[0.001 * i for i in range(n)])


@pytest.mark.parametrize("vocab", [300, 9000, 201088])
def test_equal_logits(samplers, vocab):
    """Ties go to the lowest index: few values, one value, cuts in the middle of equal ones."""
    n = 12
    x, u = rows_of(n, vocab, 5)
    x = (x * 2).round() / 2
    x[0] = 1.5
    x[1] = -0.0
    x[1, ::2] = 0.0
    x[2] = torch.where(torch.arange(vocab, device=DEV) < vocab // 2, 3.0, -2.0)
    k = [7, 100, vocab // 2 + 5, vocab // 3, 50, 1, 2, 3, 0, 0, vocab - 1, 20]
    p = [1.0, 0.5, 0.9, 0.25, 0.9, 1.0, 0.6, 0.99, 0.001, 0.5, 0.7, 1.0]
    s = samplers(vocab)
    check(s, x, u, k=k)
    check(s, x, u, k=k, p=p)
    check(s, x, u, p=p)
    check(s, x, u, t=[0.0] * n)
    check(s, x, u, t=[-1.0] * n, k=k, p=p)


@pytest.mark.parametrize("vocab", [300, 9000])
def test_special_values(samplers, vocab):
    inf, nan = float("inf"), float("nan")
    x = torch.zeros((14, vocab), device=DEV)
    x[0] = -inf                      # nothing can be drawn
    x[1] = nan
    x[2] = -inf
    x[2, vocab - 1] = -1e38          # one token left
    x[3] = nan
    x[3, 7] = 2.0
    x[4, 5], x[4, 250] = inf, inf    # infinities share everything
    x[5] = inf
    x[6] = -3.4e38
    x[6, 3] = 3.4e38
    x[7] = -inf
    x[7, 1::2] = torch.randn((vocab // 2,), device=DEV)  # a mask of every other token
    x[8] = torch.randn((vocab,), device=DEV) * 1e-40
    x[9] = torch.randn((vocab,), device=DEV) * 1e30
    x[10:] = torch.randn((4, vocab), device=DEV)
    x[10, 3:] = -inf                 # fewer left than top_k asks for
    u = [0.5, 0.1, 0.9, 0.3, 0.75, 0.6, 0.2, 0.4, 0.35, 0.8, 0.7, 0.99, 0.01, 0.5]
    s = samplers(vocab)
    for t in (None, [0.0] * 14, [nan] * 14, [1e-30] * 14, [1e30] * 14, [inf] * 14):
        check(s, x, u, t=t)
    check(s, x, u, k=[50] * 14)
    check(s, x, u, p=[0.9] * 14)
    check(s, x, u, m=[0.2] * 14)
    check(s, x, u, k=[50] * 14, p=[0.5] * 14, m=[0.1] * 14)
    check(s, x, u, p=[nan] * 14, m=[nan] * 14)
    check(s, x, u, p=[-1.0] * 14)


@pytest.mark.parametrize("vocab", [20011, 201088])
def test_few_values_and_extreme_temperatures(samplers, vocab):
    """Thousands of equal logits about the cut, and temperatures from next to nothing to infinity."""
    n = 9
    g = torch.Generator(device=DEV)
    g.manual_seed(vocab)
    x = -0.5 * torch.randint(0, 4, (n, vocab), generator=g, device=DEV).float()
    x[5:] = torch.randn((n - 5, vocab), generator=g, device=DEV)
    u = torch.rand((n,), generator=g, device=DEV).tolist()
    t = [1.0, 0.3, 5.0, float("inf"), 1e-30, 1e-38, 1e30, float("inf"), 1e-3]
    p = [0.9, 0.4, 0.97, 0.5, 0.5, 0.3, 0.9, 0.25, 0.9]
    check(samplers(vocab), x, u, t=t, p=p)
    check(samplers(vocab), x, u, t=t, p=p, k=[0, 30000, 0, 9000, 0, 7, 0, 12345, 0])
    check(samplers(vocab), x, u, t=t)


@pytest.mark.parametrize("order", ["descending", "ascending", "one chunk"])
def test_likely_tokens_side_by_side(samplers, order):
    """The largest logits lie together, where a warp's list cannot hold them."""
    vocab = 30000
    x, u = rows_of(8, vocab, 11)
    if order == "one chunk":
        x[:, 5000:5600] += 8
    else:
        x = x.sort(dim=1, descending=order == "descending").values
    s = samplers(vocab)
    check(s, x, u, k=[1, 10, 64, 65, 100, 500, 1000, 10000])
    check(s, x, u, p=[0.1, 0.3, 0.5, 0.7, 0.9, 0.99, 0.999, 0.9999])
    check(s, x, u, m=[0.5, 0.1, 0.01, 0.001, 0.9, 1.0, 0.0, 0.02])
    check(s, x, u, t=[0.3] * 8, k=[1, 10, 64, 65, 100, 500, 1000, 10000], p=[0.95] * 8)


def test_strides_and_alignment(samplers):
    vocab = 20011
    for dtype in (torch.float32, torch.bfloat16):
        for pad, skip in ((0, 0), (1, 0), (5, 3), (13, 8)):
            wide = torch.full((6, vocab + pad + skip), 1e30, device=DEV, dtype=dtype)
            x, u = rows_of(6, vocab, pad)
            wide[:, skip:skip + vocab] = x.to(dtype)
            check(samplers(vocab), wide[:, skip:skip + vocab], u, k=[0, 30, 0, 5, 0, 0], p=[1.0, 1.0, 0.9, 0.9, 1.0, 0.5])


def test_a_row_does_not_depend_on_its_batch(samplers):
    vocab = 50000
    x, u = rows_of(40, vocab, 23)
    k, p = [(i * 13) % 90 for i in range(40)], [0.5 + 0.0125 * i for i in range(40)]
    whole = check(samplers(vocab), x, u, k=k, p=p)
    for b in (0, 17, 39):
        one = check(samplers(vocab), x[b:b + 1], u[b:b + 1], k=k[b:b + 1], p=p[b:b + 1])
        assert all(torch.equal(a[b:b + 1], c) for a, c in zip(whole, one))


def test_frequencies(samplers):
    """Evenly spread numbers draw every kept token as often as its weight says, to one draw."""
    n = 4096
    x = torch.tensor([0.0, 1.0, -1.0, 2.0, 0.5, -8.0], device=DEV).expand(n, 6).contiguous()
    u = ((torch.arange(n, device=DEV) + 0.5) / n).float()
    token = samplers(6).run(x, u, top_k=torch.full((n,), 4, dtype=torch.int32, device=DEV))
    w = np.exp(np.array([0.0, 1.0, 0.0, 2.0, 0.5, 0.0]))
    w[[2, 5]] = 0
    count = np.bincount(token.cpu().numpy(), minlength=6)
    assert (np.abs(count - n * w / w.sum()) <= 1).all()


def test_captured_and_on_two_streams(samplers):
    vocab = 60000
    s = samplers(vocab)
    worlds = []
    for seed in range(2):
        x, u = rows_of(5, vocab, 40 + seed)
        worlds.append((x, f32(u), f32([0.9] * 5), torch.tensor([0, 20, 0, 0, 3], dtype=torch.int32, device=DEV), f32([0.9, 1.0, 0.5, 1.0, 0.8])))
    streams, graphs, outs = [torch.cuda.Stream() for _ in worlds], [], []
    for w, st in zip(worlds, streams):
        s.run(*w)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            outs.append(s.run(*w, details=True))
        graphs.append(graph)
    for step in range(4):
        for w in worlds:
            w[1].copy_(torch.rand((5,), device=DEV))
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    graph.replay()
        torch.cuda.synchronize()
        for w, out in zip(worlds, outs):
            assert all(torch.equal(a, b) for a, b in zip(out, s.run(*w, details=True)))


def test_results_belong_to_the_given_stream(samplers):
    """A run on another stream while the current one still has to write to memory that it freed: the result is not in it."""
    x, u = rows_of(8, 20011, 77)
    u = f32(u)
    s, other = samplers(20011), torch.cuda.Stream()
    want = s.run(x, u, top_p=f32([0.9] * 8), details=True)
    p = f32([0.9] * 8)
    torch.cuda.synchronize()
    freed = [torch.empty_like(t) for t in want]
    torch.cuda._sleep(20000000)
    for t in freed:
        t.fill_(3)
    del freed, t
    got = s.run(x, u, top_p=p, details=True, stream=other)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(samplers):
    s = samplers(1000)
    x, u = torch.zeros((3, 1000), device=DEV), torch.zeros((3,), device=DEV)
    for call in (lambda: s.run(x[:, :999], u), lambda: s.run(x, u[:2]), lambda: s.run(x, None), lambda: s.run(x.double(), u),
                 lambda: s.run(x.cpu(), u), lambda: s.run(x, u, top_k=torch.ones((3,), dtype=torch.int64, device=DEV)),
                 lambda: s.run(x, u, temperature=u.double()), lambda: s.run(torch.zeros((1000, 3), device=DEV).T, u),
                 lambda: s.run(x, u, out=torch.zeros((3,), dtype=torch.int64, device=DEV))):
        with pytest.raises(ValueError):
            call()
    one = x.data_ptr()
    run = lambda **kw: s._lib.neon_sampler_run(s._h, *{**dict(logits=one, dtype=0, stride=1000, batch=3, uniform=one, t=None, k=None, p=None, m=None,  # noqa: E731
                                                               tokens=one, probs=None, kept=None, ws=one, size=1 << 20, stream=None), **kw}.values())
    assert run(dtype=5) == 1 and run(stride=999) == 1 and run(batch=-1) == 1 and run(ws=None) == 1 and run(size=1) == 1
    assert b"workspace" in s._lib.neon_sampler_last_error(s._h)
    assert run(logits=one + 2) == 1 and run(batch=0) == 0 and run(tokens=None) == 1
    assert s.run(torch.zeros((0, 1000), device=DEV), torch.zeros((0,), device=DEV)).shape == (0,)
