// What the 4-bit paged cache's parts (neon_kv4.cu, neon_kv4_prefill.cu) call of one another, and the decoder of it.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace neon {
namespace kv4 {
struct Shape;
struct Batch;
struct AppendParams;
struct AttendParams;

constexpr int kPrefillItem = 256;  // query rows of an item of the kernel for chunks of prompts
cudaError_t configure_prefill();
void launch_prefill(const AttendParams& p, cudaStream_t st);

// Opts the attention kernels into their shared memory on the current device.
cudaError_t configure_attend();
// Each enqueues on `st` and returns the number of kernels launched.  Arguments as in neon_kv4.h, checked by the caller.  pdl: may a
// kernel be set up while what runs before it drains.
int launch_append(const AppendParams& p, int dtype, int out_dtype, cudaStream_t st, bool pdl = true);
uint64_t attend_workspace(const Shape& s, const Batch& b, int max_rows);
// whether the steps of a call can be numbered, whatever its lengths are within the table
bool attend_counts(const Shape& s, const Batch& b, int max_rows, int window);
int launch_attend(const Shape& s, const Batch& b, const uint8_t* cache, int dtype, const void* q, long long q_stride, const uint16_t* sinks,
                  int window, float scale, int max_rows, void* out, float* workspace, cudaStream_t st, bool pdl = true, bool pdl_merge = true);
}  // namespace kv4
}  // namespace neon
