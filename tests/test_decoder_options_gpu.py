"""Options of the decoder with a 4-bit cache and sampling."""
import pytest

from test_decoder_kv4_gpu import ints, make, small_shape

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
DEV = "cuda:0"


def programmatic_edges(s):
    """How many of a captured step's edges let a kernel start before its predecessor is over."""
    from cuda.bindings import runtime
    tokens, pos, nxt = ints(3, 4), ints(9, 70), torch.zeros(2, dtype=torch.int32, device=DEV)
    s.step(tokens, pos, next_tokens=nxt)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        s.step(tokens, pos, next_tokens=nxt)
    raw = runtime.cudaGraph_t(graph.raw_cuda_graph())
    err, _, _, _, n = runtime.cudaGraphGetEdges_v2(raw)
    assert err == 0
    err, _, _, data, n = runtime.cudaGraphGetEdges_v2(raw, n)
    assert err == 0 and n > 0
    return sum(int(d.type) == int(runtime.cudaGraphDependencyType.cudaGraphDependencyTypeProgrammatic) for d in data[:n])


@pytest.mark.parametrize("kv_bits", [4, 16])
def test_pdl_option_covers_every_kernel(kv_bits):
    """"pdl" has a bit per kind of kernel, the 4-bit cache's and the sampler's among them: 0 leaves what the MoE layers do by themselves."""
    shape = small_shape(vocab=20000)
    s = make(shape, 2, 128, seed=3, kv_bits=16)
    s.set_option("pdl", 0)
    moe = programmatic_edges(s)
    s.set_option("kv_bits", kv_bits)
    s.set_sampling(torch.rand(2, device=DEV), top_p=torch.full((2,), 0.9, device=DEV))
    # rotation and cache 4, attention 8, merging 16: a kernel a layer; sampler 64: three kernels where rows are cut
    for bits, kernels in ((0, 0), (4, shape.n_layers), (8, shape.n_layers), (16, shape.n_layers), (64, 3)):
        s.set_option("pdl", bits)
        assert programmatic_edges(s) == moe + kernels, bits
    s.close()


@pytest.mark.parametrize("then", ["other", "none"])
def test_sampling_settings_outlive_steps_under_way(then):
    """A step on another stream has not run when new settings are given: what it still reads is not handed out again before."""
    shape, vocab = small_shape(vocab=20000), 20000
    s = make(shape, 2, 64, seed=6)
    side, logits, nxt = torch.cuda.Stream(), torch.empty((2, vocab), device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    tokens, pos = ints(3, 4), ints(0, 1)
    new = [torch.full((2,), 0.5, device=DEV), torch.full((2,), 0.1, device=DEV)]
    given = [torch.full((2,), 0.25, device=DEV), torch.full((2,), 50.0, device=DEV)]
    places = [t.data_ptr() for t in given]
    s.set_sampling(*given)
    s.step(tokens, pos, logits=logits, next_tokens=nxt)
    want = nxt.clone()
    torch.cuda.synchronize()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(40000000)
    s.step(tokens, pos, logits=logits, next_tokens=nxt, stream=side)
    del given
    s.set_sampling(*(new if then == "other" else ()))
    again = [torch.full((2,), x, device=DEV) for x in (0.9, 0.01, 0.9, 0.01)]  # the memory that is free now
    assert set(places) & {t.data_ptr() for t in again}
    torch.cuda.synchronize()
    assert torch.equal(nxt, want)
    s.close()


@pytest.mark.parametrize("kv_bits", [4, 16])
def test_load_kv_refuses_unaligned_tensors(kv_bits):
    """Device tensors are read 16 bytes at a time (16-bit caches' values are not)."""
    shape = small_shape()
    s = make(shape, 2, 64, seed=6, kv_bits=kv_bits)
    flat = torch.randn(2 * 40 * 2 * 64 + 8, device=DEV).to(torch.bfloat16)
    whole, shifted = flat[:-8].view(2, 40, 2, 64), flat[1:-7].view(2, 40, 2, 64)
    with pytest.raises(RuntimeError, match="16-byte"):
        s.load_kv(0, shifted, whole)
    if kv_bits == 4:
        with pytest.raises(RuntimeError, match="16-byte"):
            s.load_kv(0, whole, shifted)
    else:
        s.load_kv(0, whole, shifted)
    s.load_kv(0, whole, whole)
    s.step(ints(3, 4), ints(39, 40))
    assert torch.from_numpy(s.read("logits")).isfinite().all()
    s.close()
