// Host side of the sampler declared in include/neon_sampler.h: checks arguments and enqueues the kernels.
// No CPU fallback exists: a call launches CUDA kernels or fails with an error code.
#include "../../include/neon_sampler.h"

#include <algorithm>
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <new>
#include <string>

#include "sampler_kernels.cuh"
#include "sampler_launch.h"

using namespace neon;

struct neon_sampler_handle {
    neon_sampler_config cfg{};
    std::string err;
    std::atomic<int64_t> launches{0};
};

namespace {
thread_local std::string g_create_error;

int fail(neon_sampler_handle* h, int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    if (h) h->err = buf; else g_create_error = buf;
    return code;
}

// Makes the handle's device current for a scope and the caller's again after it.
struct OnDevice {
    int before = -1;
    bool ok;
    explicit OnDevice(int device) {
        ok = cudaGetDevice(&before) == cudaSuccess && (before == device || cudaSetDevice(device) == cudaSuccess);
        if (before == device) before = -1;
    }
    ~OnDevice() { if (before >= 0) cudaSetDevice(before); }
};
}  // namespace

namespace neon {
namespace sampler {
namespace {
constexpr int kSms = 148, kSharedPerSm = 227 * 1024;
int chunks_of(int vocab) { return vocab <= kList ? 0 : (vocab + kChunk - 1) / kChunk; }
size_t whole_smem(int vocab) { return sizeof(WholeSmem) + (size_t)whole_share(vocab) * sizeof(float); }
size_t round16(size_t n) { return (n + 15) / 16 * 16; }
}  // namespace

cudaError_t configure() {
    static std::atomic<bool> done[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || done[dev & 63]) return e;
    e = cudaFuncSetAttribute(pick_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(PickSmem));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(whole_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedPerSm);
    if (e == cudaSuccess) done[dev & 63] = true;
    return e;
}

uint64_t workspace(int vocab, int batch) {
    const size_t chunks = chunks_of(vocab);
    return std::max<size_t>(16, batch * chunks * (sizeof(ChunkHead) + kSlots * sizeof(uint2)) + round16(batch * sizeof(int)));
}

int launch(const void* logits, int dtype, long long row_stride, int vocab, int batch, const float* uniform, const float* temperature,
           const int32_t* top_k, const float* top_p, const float* min_p, int32_t* tokens, float* probs, int32_t* kept, void* workspace,
           cudaStream_t st, bool pdl) {
    Params p{};
    p.logits = logits; p.dtype = dtype; p.vocab = vocab; p.batch = batch; p.stride = row_stride;
    p.uniform = uniform; p.temperature = temperature; p.top_k = top_k; p.top_p = top_p; p.min_p = min_p;
    p.tokens = tokens; p.probs = probs; p.kept = kept;
    p.chunks = chunks_of(vocab);
    if (p.chunks == 0) {
        pick_kernel<<<batch, kPickThreads, sizeof(PickSmem), st>>>(p, 1);
        return 1;
    }
    const size_t n = (size_t)batch * p.chunks;
    p.entries = static_cast<uint2*>(workspace);
    p.heads = reinterpret_cast<ChunkHead*>(p.entries + n * kSlots);
    p.left = reinterpret_cast<int*>(p.heads + n);
    // A warp lists some 1.4 times as many elements as lanes' maxima pass its bound.  Longer lists let pick settle more rows, but all
    // warps' together have to fit its list.  64 rows with all filters, us by lanes' maxima (16, 8): 98 chunks 35, 71; 147 39, 37; 197 43, 40;
    // 256 47, 44; 293 438, 51.  From 147 to 220 both settle such rows, and 16 reaches deeper.
    p.rank = p.chunks <= 220 ? 16 : 8;
    const unsigned grid = (unsigned)std::min<size_t>((n + kScanWarps - 1) / kScanWarps, 2 * kSms);
    void (*scan)(Params) = dtype == NEON_SAMPLER_F32 ? scan_kernel<0> : dtype == NEON_SAMPLER_BF16 ? scan_kernel<1> : scan_kernel<2>;
    // Each may be set up while its predecessor drains and waits for it before it reads or writes memory.  The first only where
    // setting up is not a small part of it: behind the decoder's projection, 8 rows, that saves 10 us of 14; but 256 rows, run after run,
    // take 76 us instead of 71, since its CTAs take the place of the last ones of what is before.
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = pdl && n <= 8 * kScanWarps * grid;
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kScanWarps * 32);
    cudaLaunchKernelEx(&cfg, scan, static_cast<const Params>(p));
    cfg.numAttrs = pdl;
    cfg.blockDim = dim3(kPickThreads);
    cfg.gridDim = dim3(batch);
    cfg.dynamicSmemBytes = sizeof(PickSmem);
    cudaLaunchKernelEx(&cfg, pick_kernel, static_cast<const Params>(p), 0);
    if (!top_k && !top_p && !min_p) return 2;  // pick leaves nothing
    const size_t smem = whole_smem(vocab);
    const int clusters = std::min(batch, (int)(kSms / kClusterCtas * (kSharedPerSm / (smem + 1024))));
    cfg.gridDim = dim3(std::max(clusters, 1) * kClusterCtas);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchKernelEx(&cfg, whole_kernel, static_cast<const Params>(p));
    return 3;
}

}  // namespace sampler
}  // namespace neon

extern "C" {

const char* neon_sampler_last_error(const neon_sampler_handle* h) { return h ? h->err.c_str() : g_create_error.c_str(); }
int64_t neon_sampler_launch_count(const neon_sampler_handle* h) { return h ? h->launches.load() : 0; }

int neon_sampler_create(const neon_sampler_config* cfg, neon_sampler_handle** out) {
    if (!cfg || !out) return fail(nullptr, NEON_MOE_EINVAL, "null argument");
    *out = nullptr;
    if (cfg->vocab < 1 || cfg->vocab > NEON_SAMPLER_MAX_VOCAB)
        return fail(nullptr, NEON_MOE_EINVAL, "vocab %d outside 1..%d", cfg->vocab, NEON_SAMPLER_MAX_VOCAB);
    int count = 0;
    if (cudaGetDeviceCount(&count) != cudaSuccess || cfg->device < 0 || cfg->device >= count) {
        cudaGetLastError();
        return fail(nullptr, NEON_MOE_ECUDA, "no CUDA device %d", cfg->device);
    }
    auto* h = new (std::nothrow) neon_sampler_handle;
    if (!h) return fail(nullptr, NEON_MOE_ECUDA, "out of host memory");
    h->cfg = *cfg;
    OnDevice dev(cfg->device);
    if (!dev.ok || sampler::configure() != cudaSuccess) {
        const cudaError_t e = cudaGetLastError();
        delete h;
        return fail(nullptr, NEON_MOE_ECUDA, "setting up device %d: %s", cfg->device, cudaGetErrorString(e));
    }
    *out = h;
    return NEON_MOE_OK;
}

int neon_sampler_destroy(neon_sampler_handle* h) {
    delete h;
    return NEON_MOE_OK;
}

uint64_t neon_sampler_workspace(const neon_sampler_handle* h, int batch) { return h && batch > 0 ? sampler::workspace(h->cfg.vocab, batch) : 0; }

int neon_sampler_run(neon_sampler_handle* h, const void* logits, int dtype, int64_t row_stride, int batch, const float* uniform,
                     const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p, int32_t* tokens, float* probs,
                     int32_t* kept, void* workspace, uint64_t workspace_bytes, void* cuda_stream) {
    if (!h) return NEON_MOE_EINVAL;
    if (batch == 0) return NEON_MOE_OK;
    if (!logits || !uniform || !tokens || !workspace) return fail(h, NEON_MOE_EINVAL, "null logits, uniform, tokens or workspace");
    if (dtype != NEON_SAMPLER_F32 && dtype != NEON_SAMPLER_BF16 && dtype != NEON_SAMPLER_F16) return fail(h, NEON_MOE_EINVAL, "dtype %d", dtype);
    if (batch < 0 || batch > 65535) return fail(h, NEON_MOE_EINVAL, "batch %d outside 0..65535", batch);
    if (row_stride < h->cfg.vocab) return fail(h, NEON_MOE_EINVAL, "rows %lld apart are shorter than the vocabulary", (long long)row_stride);
    if (reinterpret_cast<uintptr_t>(logits) % (dtype == NEON_SAMPLER_F32 ? 4 : 2) || reinterpret_cast<uintptr_t>(workspace) % 16)
        return fail(h, NEON_MOE_EINVAL, "logits or workspace are not aligned");
    if (workspace_bytes < sampler::workspace(h->cfg.vocab, batch))
        return fail(h, NEON_MOE_EINVAL, "workspace of %llu bytes, %llu wanted", (unsigned long long)workspace_bytes,
                    (unsigned long long)sampler::workspace(h->cfg.vocab, batch));
    OnDevice dev(h->cfg.device);
    if (!dev.ok) return fail(h, NEON_MOE_ECUDA, "cudaSetDevice(%d) failed", h->cfg.device);
    h->launches += sampler::launch(logits, dtype, row_stride, h->cfg.vocab, batch, uniform, temperature, top_k, top_p, min_p, tokens, probs, kept,
                                   workspace, static_cast<cudaStream_t>(cuda_stream));
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? NEON_MOE_OK : fail(h, NEON_MOE_ECUDA, "launch failed: %s", cudaGetErrorString(e));
}

}  // extern "C"
