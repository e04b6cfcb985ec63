// The variants of the kernel for chunks of prompts (kv4_prefill.cuh), which a source file of its own keeps compiled as one unit: how
// well its softmax is scheduled decides its time.
#include "kv4_prefill.cuh"
#include "kv4_launch.h"

namespace neon {
namespace kv4 {

static_assert(kPreRows == kPrefillItem, "rows of an item");

namespace {
constexpr int kSmem = sizeof(PrefillSmem) + 1024;

template <int PAGE>
cudaError_t configure() { return cudaFuncSetAttribute(prefill_kernel<PAGE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem); }
}  // namespace

cudaError_t configure_prefill() {
    cudaError_t e = configure<16>();
    if (e == cudaSuccess) e = configure<32>();
    if (e == cudaSuccess) e = configure<64>();
    return e;
}

void launch_prefill(const AttendParams& p, cudaStream_t st) {
    const long long items = (long long)p.b.rows * p.G / kPreRows + p.b.n;  // as many as there can be
    const unsigned grid = (unsigned)(items * p.s.nkv);
    if (p.s.P == 16) prefill_kernel<16><<<grid, kPreWarps * 32, kSmem, st>>>(p);
    else if (p.s.P == 32) prefill_kernel<32><<<grid, kPreWarps * 32, kSmem, st>>>(p);
    else prefill_kernel<64><<<grid, kPreWarps * 32, kSmem, st>>>(p);
}

}  // namespace kv4
}  // namespace neon
