// Host side of the 4-bit paged cache declared in include/neon_kv4.h: checks arguments, picks the kernel variant and
// enqueues it.  No CPU fallback exists: a call launches CUDA kernels or fails with an error code.
#include "../../include/neon_kv4.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <new>
#include <string>

#include "kv4_append.cuh"
#include "kv4_attend.cuh"
#include "kv4_launch.h"

using namespace neon;
using namespace neon::kv4;

struct neon_kv4_handle {
    neon_kv4_config cfg{};
    Shape shape{};
    std::string err;
    int* status = nullptr;
    std::atomic<int64_t> launches{0};
};

namespace {
thread_local std::string g_create_error;

int fail(neon_kv4_handle* h, int code, const char* fmt, ...) {
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

#define ON_DEVICE(h)                    \
    OnDevice on_device_((h)->cfg.device); \
    if (!on_device_.ok) return fail((h), NEON_MOE_ECUDA, "cudaSetDevice(%d) failed", (h)->cfg.device)

int launched(neon_kv4_handle* h, int n) {
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail(h, NEON_MOE_ECUDA, "launch failed: %s", cudaGetErrorString(e));
    h->launches += n;
    return NEON_MOE_OK;
}

bool aligned(const void* p, int64_t stride, int dtype) {
    const int size = dtype == NEON_KV4_F32 ? 4 : 2;
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0;
}

int check_batch(neon_kv4_handle* h, const neon_kv4_batch* b, const void* cache, int rows) {
    if (!b || !b->seq_lens || !b->page_table || !cache) return fail(h, NEON_MOE_EINVAL, "null batch, seq_lens, page_table or cache");
    if (b->batch < 1 || b->batch > NEON_KV4_MAX_BATCH)
        return fail(h, NEON_MOE_EINVAL, "batch %d outside 1..%d", b->batch, NEON_KV4_MAX_BATCH);
    if (b->table_width < 1 || b->table_stride < b->table_width || (int64_t)b->table_width * h->cfg.page_size > (1 << 30))
        return fail(h, NEON_MOE_EINVAL, "page table of %d columns, rows %lld apart", b->table_width, (long long)b->table_stride);
    if (b->n_pages < 1) return fail(h, NEON_MOE_EINVAL, "a cache of %lld pages", (long long)b->n_pages);
    if (rows < 0 || (!b->cu_q && rows < b->batch))
        return fail(h, NEON_MOE_EINVAL, "%d rows for %d sequences of one row each", rows, b->batch);
    if (reinterpret_cast<uintptr_t>(cache) % 16) return fail(h, NEON_MOE_EINVAL, "the cache is not 16-byte aligned");
    return NEON_MOE_OK;
}
}  // namespace

namespace neon {
namespace kv4 {

namespace {
constexpr int kSms = 148, kSharedPerSm = 227 * 1024;

// Columns of an item's products, in groups of eight.  More of them read, convert and scale the cache less often; fewer need fewer
// registers, so that two CTAs fit a multiprocessor.  64 sequences of 4000 positions, 8 key/value heads, us by groups of columns:
//   heads of 64    8 rows an item: 48 (1), 104 (4)    16 rows: 82 (1), 108 (4)    32 rows: 146 (1), 113 (4)
//   heads of 128   8 rows: 79 (1), 104 (2)            16 rows: 143 (1), 109 (2)
int column_groups(const Shape& s, int max_rows) {
    const long long rows = (long long)std::max(max_rows, 1) * (s.nq / s.nkv);
    if (s.D == 128) return rows <= 8 ? 1 : 2;
    return rows <= 16 ? 1 : 4;
}
// one instead of two, with eight rows of 64: 56 us instead of 48, with sixteen 102 instead of 82
int ctas_per_sm(const Shape& s, int nt) { return s.D == 64 && nt == 1 ? 2 : 1; }
// steps that there can be in all, as the table's width bounds the lengths
long long most_units(const Shape& s, const Batch& b, int nt) {
    const long long steps = ((long long)b.width * s.P + kStep - 1) / kStep;
    return steps * ((long long)b.rows * (s.nq / s.nkv) / (8 * nt) + b.n) * s.nkv;
}
int attend_grid(const Shape& s, const Batch& b, int nt) {
    const long long most = (most_units(s, b, nt) + kAttendWarps - 1) / kAttendWarps;  // CTAs that there can be steps for
    return (int)std::min<long long>(kSms * ctas_per_sm(s, nt), std::max<long long>(most, 1));
}

// The kernel may be set up while what runs before it on the stream drains (append 6.4 -> 6.3 us, attention of one token 10.0 -> 9.8, 8
// layers of the decoder's step 1097 -> 1090); it waits for that before it reads or writes memory.
template <class F>
void with_pdl(bool pdl, void (*kernel)(F), unsigned grid, int threads, size_t smem, cudaStream_t st, const F& p) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl;
    cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int DIM, int PAGE, int NT>
cudaError_t attend_variant(const AttendParams* run, cudaStream_t st, bool pdl, bool pdl_merge) {
    using W = WarpSmem<DIM>;
    if (!run) return cudaFuncSetAttribute(attend_kernel<DIM, PAGE, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024);
    AttendParams p = *run;
    const int plan = plan_bytes(p.b.n), budget = kSharedPerSm / ctas_per_sm(p.s, NT) - 2048 - plan;
    p.stages = std::min(W::kMaxStages, (budget / kAttendWarps - W::bytes(0)) / W::kRing);
    with_pdl(pdl, attend_kernel<DIM, PAGE, NT>, (unsigned)p.grid, kAttendWarps * 32, plan + kAttendWarps * W::bytes(p.stages), st, p);
    const long long tasks = (long long)p.b.rows * p.s.nq;
    with_pdl(pdl_merge, merge_kernel<DIM>, (unsigned)((tasks + 7) / 8), 256, plan, st, p);
    return cudaSuccess;
}
// Chunks of prompts: 256 rows of a key/value head at a time on tcgen05.  Heads of 64 only: the kernel's three operand stages and
// second query term would not fit a CTA at 128 columns (one with two stages, for bf16 queries, would), and those go to the other
// kernel, 1910 us for two chunks of 2048 rows over up to 8192 positions, 32 and 8 heads.  An item walks its positions alone, 1.2 to 1.5 us a step of 64, whether or not there is work for
// the other multiprocessors; the other kernel splits steps evenly over all of them, 2.9 ns a step of 32 rows.  So the first is faster
// from about 480 blocks of 32 rows for every wave of items on.  At 8 query and key/value heads and 4096 positions (other kernel, this one):
//   8 sequences of 128 rows (256 blocks, 1 wave)     65,  94 us       of 256 rows (512 blocks)            111,  82 us
//   32 sequences of 64 rows (512 blocks, 2 waves)   112, 216 us       of 128 rows (1024 blocks, 2 waves)  206, 187 us
//   one sequence of 512 rows (128 blocks, 1 wave)    38,  79 us
// Where a window leaves a few steps only, the other kernel's split and its second launch cost more than they bring.  Windows of 64, 128,
// 256, 448, 512, 1024, us:
//   32 sequences of 64 rows       23, 24   36, 26   43, 32   50, 40   46, 43   63, 69
//   8 sequences of 128 rows       21, 15   18, 17   30, 20   28, 23   33, 25   36, 36
//   one sequence of 512 rows      18, 19   22, 21   22, 23   24, 27   24, 28   29, 37
// Below 64 rows the products' tiles are nearly empty: 64 sequences of 16 rows, window 128, 22, 46 us.
constexpr int kPrefillRows = 64, kPrefillSpan = 512, kPrefillBlocks = 480;
bool prefills(const Shape& s, const Batch& b, int max_rows, int window) {
    const int G = s.nq / s.nkv;
    const long long most = (long long)std::min(std::max(max_rows, 1), b.rows) * G;  // rows of an item's sequence, as far as known
    if (s.D != 64 || most < kPrefillRows) return false;
    if (window > 0 && (long long)window + max_rows <= kPrefillSpan) return true;
    auto count = [&](int per) { return std::min((long long)b.rows * G / per + b.n, (most + per - 1) / per * b.n) * s.nkv; };
    return count(32) >= kPrefillBlocks * ((count(kPrefillItem) + kSms - 1) / kSms);
}

// Calls f with every variant that there is; the one of a shape and a number of column groups.
template <class F>
cudaError_t each_variant(const F& f) {
    cudaError_t e = cudaSuccess;
#define TRY(DIM, PAGE, NT) if (e == cudaSuccess) e = f(DIM, PAGE, NT, &attend_variant<DIM, PAGE, NT>);
#define PAGES(DIM, NT) TRY(DIM, 16, NT) TRY(DIM, 32, NT) TRY(DIM, 64, NT)
    PAGES(64, 1) PAGES(64, 4) PAGES(128, 1) PAGES(128, 2)
#undef PAGES
#undef TRY
    return e;
}
}  // namespace

cudaError_t configure_attend() {
    static std::atomic<bool> done[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || done[dev & 63]) return e;
    e = each_variant([](int, int, int, auto variant) { return variant(nullptr, nullptr, false, false); });
    if (e == cudaSuccess) e = configure_prefill();
    if (e == cudaSuccess) done[dev & 63] = true;
    return e;
}

bool attend_counts(const Shape& s, const Batch& b, int max_rows, int window) {
    const int nt = column_groups(s, max_rows);
    return prefills(s, b, max_rows, window) || most_units(s, b, nt) / attend_grid(s, b, nt) < kMaxCtaUnits;
}

uint64_t attend_workspace(const Shape& s, const Batch& b, int max_rows) {
    if (prefills(s, b, max_rows, 0)) return 16;  // (whatever the window)
    const int nt = column_groups(s, max_rows);
    return (uint64_t)attend_grid(s, b, nt) * (2 + kAttendWarps) * 8 * nt * (s.D + 2) * sizeof(float);
}

int launch_attend(const Shape& s, const Batch& b, const uint8_t* cache, int dtype, const void* q, long long q_stride, const uint16_t* sinks,
                  int window, float scale, int max_rows, void* out, float* workspace, cudaStream_t st, bool pdl, bool pdl_merge) {
    AttendParams p{};
    p.b = b; p.s = s; p.cache = cache; p.q = q; p.q_stride = q_stride; p.sinks = sinks;
    p.window = window; p.G = s.nq / s.nkv; p.half = dtype == NEON_KV4_F16; p.scale = scale; p.out = out; p.part = workspace;
    const int nt = column_groups(s, max_rows);
    p.grid = attend_grid(s, b, nt);
    p.R = 8 * nt;
    p.G_inverse = (uint32_t)((0x100000000ull + p.G - 1) / p.G);
    if (prefills(s, b, max_rows, window)) {
        launch_prefill(p, st);
        return 1;
    }
    each_variant([&](int dim, int page, int groups, auto variant) {
        return dim == s.D && page == s.P && groups == nt ? variant(&p, st, pdl, pdl_merge) : cudaSuccess;
    });
    return 2;
}

int launch_append(const AppendParams& given, int dtype, int out_dtype, cudaStream_t st, bool pdl) {
    AppendParams p = given;
    // a warp per row, unless there are so few rows that its ten or so rounds would be what takes the time: 8 rows of 80 heads 3.3 us in
    // parts, 6.0 by whole rows; 1024 rows 6.4 with this rule, 7.3 by whole rows, 12.0 in ten parts
    const int heads = (p.q ? p.s.nq : 0) + 2 * p.s.nkv, rounds = (heads * p.s.D / 16 + 31) / 32;
    p.split = std::min(rounds, std::max(1, kSms * 16 / p.b.rows));
    const unsigned grid = (unsigned)(((long long)p.b.rows * p.split + kAppendWarps - 1) / kAppendWarps);
#define RUN(DT, DIM)                                                                                                     \
    if (dtype == DT && p.s.D == DIM) {                                                                                   \
        if (out_dtype == NEON_KV4_F16) with_pdl(pdl, append_kernel<DT, __half, DIM>, grid, kAppendWarps * 32, 0, st, p); \
        else with_pdl(pdl, append_kernel<DT, __nv_bfloat16, DIM>, grid, kAppendWarps * 32, 0, st, p);                    \
    }
    RUN(NEON_KV4_F32, 64) RUN(NEON_KV4_BF16, 64) RUN(NEON_KV4_F16, 64) RUN(NEON_KV4_F32, 128) RUN(NEON_KV4_BF16, 128) RUN(NEON_KV4_F16, 128)
#undef RUN
    return 1;
}

}  // namespace kv4
}  // namespace neon

extern "C" {

const char* neon_kv4_last_error(const neon_kv4_handle* h) { return h ? h->err.c_str() : g_create_error.c_str(); }
int64_t neon_kv4_launch_count(const neon_kv4_handle* h) { return h ? h->launches.load() : 0; }
int64_t neon_kv4_record_bytes(const neon_kv4_handle* h) { return h ? h->shape.record() : 0; }

int neon_kv4_create(const neon_kv4_config* cfg, neon_kv4_handle** out) {
    if (!cfg || !out) return fail(nullptr, NEON_MOE_EINVAL, "null argument");
    *out = nullptr;
    const auto& c = *cfg;
    if (c.head_dim != 64 && c.head_dim != 128) return fail(nullptr, NEON_MOE_EINVAL, "head_dim must be 64 or 128");
    if (c.page_size != 16 && c.page_size != 32 && c.page_size != 64) return fail(nullptr, NEON_MOE_EINVAL, "page_size must be 16, 32 or 64");
    if (c.n_kv_heads < 1 || c.n_kv_heads > 128) return fail(nullptr, NEON_MOE_EINVAL, "n_kv_heads must be 1..128");
    if (c.n_q_heads < c.n_kv_heads || c.n_q_heads % c.n_kv_heads || c.n_q_heads / c.n_kv_heads > 32)
        return fail(nullptr, NEON_MOE_EINVAL, "n_q_heads must be 1 to 32 times n_kv_heads");
    int count = 0;
    if (cudaGetDeviceCount(&count) != cudaSuccess || c.device < 0 || c.device >= count) {
        cudaGetLastError();
        return fail(nullptr, NEON_MOE_ECUDA, "no CUDA device %d", c.device);
    }
    auto* h = new (std::nothrow) neon_kv4_handle;
    if (!h) return fail(nullptr, NEON_MOE_ECUDA, "out of host memory");
    h->cfg = c;
    h->shape = {c.n_q_heads, c.n_kv_heads, c.head_dim, c.page_size};
    OnDevice dev(c.device);
    if (!dev.ok || cudaMalloc(&h->status, sizeof(int)) != cudaSuccess || cudaMemset(h->status, 0, sizeof(int)) != cudaSuccess ||
        configure_attend() != cudaSuccess) {
        const cudaError_t e = cudaGetLastError();
        if (h->status) cudaFree(h->status);
        delete h;
        return fail(nullptr, NEON_MOE_ECUDA, "setting up device %d: %s", c.device, cudaGetErrorString(e));
    }
    *out = h;
    return NEON_MOE_OK;
}

int neon_kv4_destroy(neon_kv4_handle* h) {
    if (!h) return NEON_MOE_OK;
    {
        OnDevice dev(h->cfg.device);
        if (dev.ok && h->status) cudaFree(h->status);  // waits for the device
        cudaGetLastError();
    }
    delete h;
    return NEON_MOE_OK;
}

static Batch device_batch(const neon_kv4_handle* h, const neon_kv4_batch* b, int rows) {
    return {b->seq_lens, b->cu_q, b->page_table, b->table_stride, b->n_pages, b->table_width, b->batch, rows, h->status};
}

int neon_kv4_append(neon_kv4_handle* h, const neon_kv4_batch* batch, void* cache, int rows, int dtype, const void* q, int64_t q_stride,
                    const void* k, int64_t k_stride, const void* v, int64_t v_stride, const float* inv_freq, float mscale, void* q_out,
                    int out_dtype, void* cuda_stream) {
    if (!h) return NEON_MOE_EINVAL;
    if (int rc = check_batch(h, batch, cache, rows)) return rc;
    if (rows == 0) return NEON_MOE_OK;
    if (!k || !v || !inv_freq || !q != !q_out) return fail(h, NEON_MOE_EINVAL, "null k, v or inv_freq, or one of q and q_out without the other");
    if (dtype != NEON_KV4_F32 && dtype != NEON_KV4_BF16 && dtype != NEON_KV4_F16) return fail(h, NEON_MOE_EINVAL, "dtype %d", dtype);
    if (q_out && out_dtype != NEON_KV4_BF16 && out_dtype != NEON_KV4_F16) return fail(h, NEON_MOE_EINVAL, "out_dtype %d", out_dtype);
    const Shape& s = h->shape;
    if (k_stride < s.nkv * s.D || v_stride < s.nkv * s.D || (q && q_stride < s.nq * s.D))
        return fail(h, NEON_MOE_EINVAL, "a row stride is smaller than the row");
    if (!aligned(k, k_stride, dtype) || !aligned(v, v_stride, dtype) || (q && !aligned(q, q_stride, dtype)) || reinterpret_cast<uintptr_t>(q_out) % 16)
        return fail(h, NEON_MOE_EINVAL, "q, k, v and q_out rows have to start on 16-byte boundaries");
    ON_DEVICE(h);
    AppendParams p{};
    p.b = device_batch(h, batch, rows);
    p.s = s;
    p.q = q; p.k = k; p.v = v;
    p.q_stride = q_stride; p.k_stride = k_stride; p.v_stride = v_stride;
    p.n_parts = 1;
    p.inv_freq = inv_freq; p.mscale = mscale; p.q_out = q_out;
    p.cache = static_cast<uint8_t*>(cache);
    return launched(h, launch_append(p, dtype, out_dtype, static_cast<cudaStream_t>(cuda_stream)));
}

int neon_kv4_read(neon_kv4_handle* h, const neon_kv4_batch* batch, const void* cache, int rows, void* k_out, void* v_out, int dtype,
                  void* cuda_stream) {
    if (!h) return NEON_MOE_EINVAL;
    if (int rc = check_batch(h, batch, cache, rows)) return rc;
    if (rows == 0) return NEON_MOE_OK;
    if (dtype != NEON_KV4_F32 && dtype != NEON_KV4_BF16) return fail(h, NEON_MOE_EINVAL, "dtype %d", dtype);
    if (reinterpret_cast<uintptr_t>(k_out) % 16 || reinterpret_cast<uintptr_t>(v_out) % 16)
        return fail(h, NEON_MOE_EINVAL, "k_out and v_out have to be 16-byte aligned");
    if (!k_out && !v_out) return NEON_MOE_OK;
    ON_DEVICE(h);
    // few rows: four warps each, so that a row's rounds do not follow one another (8 rows 2.1 us instead of 3.0; 4096 rows 7.4, not 6.5)
    const ReadParams p{device_batch(h, batch, rows), h->shape, static_cast<const uint8_t*>(cache), k_out, v_out, rows <= 1024 ? 4 : 1};
    cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    const unsigned grid = ((unsigned)rows * p.split + 3) / 4;
    if (dtype == NEON_KV4_F32) with_pdl(true, read_kernel<float>, grid, 128, 0, st, p);
    else with_pdl(true, read_kernel<__nv_bfloat16>, grid, 128, 0, st, p);
    return launched(h, 1);
}

uint64_t neon_kv4_attend_workspace(neon_kv4_handle* h, const neon_kv4_batch* batch, int rows, int max_rows) {
    if (!h || !batch || batch->batch < 1 || rows < 0) return 0;
    return attend_workspace(h->shape, device_batch(h, batch, rows), max_rows);
}

int neon_kv4_attend(neon_kv4_handle* h, const neon_kv4_batch* batch, const void* cache, int rows, int dtype, const void* q, int64_t q_stride,
                    const void* sinks, int window, float scale, int max_rows, void* out, void* workspace, uint64_t workspace_bytes,
                    void* cuda_stream) {
    if (!h) return NEON_MOE_EINVAL;
    if (int rc = check_batch(h, batch, cache, rows)) return rc;
    if (rows == 0) return NEON_MOE_OK;
    if (!q || !out || !workspace) return fail(h, NEON_MOE_EINVAL, "null q, out or workspace");
    if (dtype != NEON_KV4_BF16 && dtype != NEON_KV4_F16) return fail(h, NEON_MOE_EINVAL, "dtype %d", dtype);
    if (window < 0) return fail(h, NEON_MOE_EINVAL, "window %d", window);
    if (!std::isfinite(scale)) return fail(h, NEON_MOE_EINVAL, "scale is not finite");
    const Shape& s = h->shape;
    if (q_stride < s.nq * s.D) return fail(h, NEON_MOE_EINVAL, "a row stride is smaller than the row");
    if ((int64_t)rows * (s.nq / s.nkv) > kMaxHeadRows)
        return fail(h, NEON_MOE_EINVAL, "%d rows of %d query heads a key/value head are more than %d", rows, s.nq / s.nkv, kMaxHeadRows);
    if (!attend_counts(s, device_batch(h, batch, rows), max_rows, window))
        return fail(h, NEON_MOE_EINVAL, "%d rows over page tables of %d columns", rows, batch->table_width);
    if (!aligned(q, q_stride, dtype) || reinterpret_cast<uintptr_t>(out) % 16 || reinterpret_cast<uintptr_t>(workspace) % 16)
        return fail(h, NEON_MOE_EINVAL, "q rows, out and workspace have to start on 16-byte boundaries");
    const Batch b = device_batch(h, batch, rows);
    if (workspace_bytes < attend_workspace(s, b, max_rows))
        return fail(h, NEON_MOE_EINVAL, "workspace of %llu bytes, %llu wanted", (unsigned long long)workspace_bytes,
                    (unsigned long long)attend_workspace(s, b, max_rows));
    ON_DEVICE(h);
    return launched(h, launch_attend(s, b, static_cast<const uint8_t*>(cache), dtype, q, q_stride, static_cast<const uint16_t*>(sinks), window,
                                     scale, max_rows, out, static_cast<float*>(workspace), static_cast<cudaStream_t>(cuda_stream)));
}

int neon_kv4_status(neon_kv4_handle* h, int* status) {
    if (!h || !status) return NEON_MOE_EINVAL;
    ON_DEVICE(h);
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaMemcpy(status, h->status, sizeof(int), cudaMemcpyDeviceToHost);
    if (e == cudaSuccess) e = cudaMemset(h->status, 0, sizeof(int));
    return e == cudaSuccess ? NEON_MOE_OK : fail(h, NEON_MOE_ECUDA, "reading the status: %s", cudaGetErrorString(e));
}

}  // extern "C"
