/*
 * neon_sampler.h - C ABI of sampling from logits (same shared library as neon_moe.h): temperature,
 * top-k, top-p and min-p, each a number per row, from random numbers that the caller gives.
 *
 * Relation to the reference engine: none of this exists there.  The calling conventions are those
 * of neon_moe.h (construction checks and owns, NeonEngine/src/water_physics.cpp:23-123;
 * stream-ordered execution, NeonEngine/src/water_physics.hpp:66; errors as values,
 * NeonEngine/src/lve_buffer.hpp:22-28).
 *
 * What a row's token is:
 *   - The order of tokens: logit descending, equal logits by index ascending (-0 equals 0).  A logit of NaN counts as
 *     -infinity, and tokens of -infinity are never drawn.
 *   - temperature <= 0 (or NaN): the first in order.
 *   - Weights w_i = exp((x_i - max) / temperature).  If the maximum is +infinity, tokens that have it weigh 1 and all
 *     others 0.
 *   - Kept are: the first top_k (top_k <= 0 or >= vocab: all); of those the shortest run from the front whose weight reaches
 *     top_p of theirs, at least one token (top_p >= 1 or NaN: all); of those the ones of w_i >= min_p, where more than
 *     1 counts as 1 (min_p <= 0 or NaN: all).
 *   - The token is the first, by INDEX, whose running sum of kept weights exceeds uniform * (their sum); numbers
 *     outside [0, 1) are moved to its nearer end.
 *   - A row of which nothing can be drawn (all -infinity) gives token -1, probability 0, kept 0.
 * Weights are computed to 4e-11 of their value (sums over all of a row: to 1e-9), rounded to 2^-43 of the largest and summed in
 * 64-bit integers, so the result depends neither on the order of sums nor on the batch around a row.
 *
 * All functions return 0 or a NEON_MOE_E* code (neon_moe.h); none throws or aborts.
 */
#ifndef NEON_SAMPLER_H
#define NEON_SAMPLER_H

#include <stdint.h>

#include "neon_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct neon_sampler_handle neon_sampler_handle;

typedef struct neon_sampler_config {
    int vocab;  /* 1 .. NEON_SAMPLER_MAX_VOCAB */
    int device; /* CUDA device ordinal         */
} neon_sampler_config;

#define NEON_SAMPLER_MAX_VOCAB 393216

/* element types of logits */
#define NEON_SAMPLER_F32 0
#define NEON_SAMPLER_BF16 1
#define NEON_SAMPLER_F16 2

int neon_sampler_create(const neon_sampler_config* cfg, neon_sampler_handle** out);
int neon_sampler_destroy(neon_sampler_handle* h);
const char* neon_sampler_last_error(const neon_sampler_handle* h);

/* Bytes of scratch that a run of `batch` rows wants (device memory, 16-byte aligned, its contents mean nothing before and
 * after the call).  Runs that can overlap need scratch of their own. */
uint64_t neon_sampler_workspace(const neon_sampler_handle* h, int batch);

/* One token per row, enqueued on cuda_stream.  Device pointers: logits [batch, vocab] of `dtype`, rows row_stride elements
 * apart (>= vocab; any alignment of whole elements); uniform fp32 [batch]; temperature fp32 [batch] or NULL (1);
 * top_k int32 [batch], top_p fp32 [batch], min_p fp32 [batch], each NULL for none; tokens int32 [batch]; probs fp32 [batch]
 * or NULL: the drawn token's share of the kept weights; kept int32 [batch] or NULL: how many tokens were kept. */
int neon_sampler_run(neon_sampler_handle* h, const void* logits, int dtype, int64_t row_stride, int batch, const float* uniform,
                     const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p, int32_t* tokens,
                     float* probs, int32_t* kept, void* workspace, uint64_t workspace_bytes, void* cuda_stream);

/* Kernels this library launched for the handle so far. */
int64_t neon_sampler_launch_count(const neon_sampler_handle* h);

#ifdef __cplusplus
}
#endif
#endif /* NEON_SAMPLER_H */
