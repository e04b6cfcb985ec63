// What other parts of the library call of the sampler (neon_sampler.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace neon {
namespace sampler {
// Opts the kernels into their shared memory on the current device.
cudaError_t configure();
uint64_t workspace(int vocab, int batch);
// Enqueues on `st` and returns the number of kernels launched.  Arguments as in neon_sampler.h, checked by the caller.  pdl: may a
// kernel be set up while what runs before it drains.
int launch(const void* logits, int dtype, long long row_stride, int vocab, int batch, const float* uniform, const float* temperature,
           const int32_t* top_k, const float* top_p, const float* min_p, int32_t* tokens, float* probs, int32_t* kept, void* workspace,
           cudaStream_t st, bool pdl = true);
}  // namespace sampler
}  // namespace neon
