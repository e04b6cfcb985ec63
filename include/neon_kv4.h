/*
 * neon_kv4.h - C ABI of a paged key/value cache held in 4 bits (same shared library as neon_moe.h):
 * appending the new tokens of a ragged batch with the rotary embedding applied on the way, reading
 * positions back, and attention over the cache - one token per sequence, a few drafted tokens, or
 * a chunk of a prompt.
 *
 * Relation to the reference engine: none of this exists there.  The calling conventions are those
 * of neon_moe.h (construction checks and owns, NeonEngine/src/water_physics.cpp:23-123;
 * stream-ordered execution, NeonEngine/src/water_physics.hpp:66; errors as values,
 * NeonEngine/src/lve_buffer.hpp:22-28).
 *
 * The cache is the caller's: uint8 [n_pages, n_kv_heads, record], contiguous, 16-byte aligned.  A
 * record holds the P positions of one page and head:
 *     P * D/2 bytes   key codes: position after position, low nibble = even column, code s|e|e|m (e2m1)
 *     P * D/2 bytes   value codes
 *     P * D/32 bytes  key scales (E8M0, one for 32 columns)
 *     P * D/32 bytes  value scales
 * neon_kv4_record_bytes() = P * (D + D/16).  Per block of 32 columns the scale is 2^(floor(log2
 * amax) - 2), clamped to 2^-126 .. 2^127 (1 for a block of zeros; NaN, with codes of 0, for a block that
 * holds a NaN), and every value is rounded to the nearest e2m1 magnitude, ties to the even code, clipped
 * to 6.
 *
 * A batch (neon_kv4_batch): sequence b owns rows cu_q[b] .. cu_q[b+1]-1 of the row-major inputs,
 * its newest tokens; seq_lens[b] counts its cache positions INCLUDING those rows, so row i of n
 * stands at position seq_lens[b] - n + i.  Position p lies in page page_table[b][p / P], at p % P.
 * These three arrays are device memory and may change between replays of a captured graph.  Rows
 * before position 0 or behind the last sequence are not looked at; of the former attention writes
 * zeros, the latter are left as they were.  A page id outside [0, n_pages) or a length beyond the
 * table (table_width * P positions) never reaches memory: such positions are neither written nor
 * attended to, and neon_kv4_status() reports it.  Sequences may share pages (a common prefix), but no two rows of an
 * append may stand at one place of the cache.  Outputs overlap no inputs.
 *
 * Calls only enqueue work and keep nothing between calls: any number of them may run at once on
 * several streams, and be captured into graphs, as long as no append writes pages that another
 * call reads.  A handle's calls come from one host thread at a time (its error text is one).  All functions return 0 or a NEON_MOE_E* code (neon_moe.h); none throws or aborts.
 */
#ifndef NEON_KV4_H
#define NEON_KV4_H

#include <stdint.h>

#include "neon_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct neon_kv4_handle neon_kv4_handle;

typedef struct neon_kv4_config {
    int n_q_heads;   /* a multiple of n_kv_heads, at most 32 times as many     */
    int n_kv_heads;  /* 1 .. 128                                               */
    int head_dim;    /* 64 or 128                                              */
    int page_size;   /* P: 16, 32 or 64 positions                              */
    int device;      /* CUDA device ordinal                                    */
} neon_kv4_config;

typedef struct neon_kv4_batch {
    const int32_t* seq_lens;    /* device [batch]                                          */
    const int32_t* cu_q;        /* device [batch + 1], from 0, ascending; NULL: one row each */
    const int32_t* page_table;  /* device, row b at page_table + b * table_stride           */
    int64_t table_stride;       /* elements; >= table_width                                 */
    int table_width;            /* pages per sequence that the table can name               */
    int batch;                  /* sequences, 1 .. NEON_KV4_MAX_BATCH                       */
    int64_t n_pages;            /* pages of the cache                                       */
} neon_kv4_batch;

#define NEON_KV4_MAX_BATCH 1024

/* element types of q, k, v and outputs */
#define NEON_KV4_F32 0
#define NEON_KV4_BF16 1
#define NEON_KV4_F16 2

/* bits of neon_kv4_status */
#define NEON_KV4_BAD_PAGE 1    /* a page id outside the cache was met                     */
#define NEON_KV4_BAD_LENGTH 2  /* a sequence longer than its table, or (seen by attention) cu_q not ascending */
#define NEON_KV4_TIMEOUT 4     /* a wait inside a kernel ran out                          */

int neon_kv4_create(const neon_kv4_config* cfg, neon_kv4_handle** out);
int neon_kv4_destroy(neon_kv4_handle* h);
const char* neon_kv4_last_error(const neon_kv4_handle* h);
int64_t neon_kv4_record_bytes(const neon_kv4_handle* h);

/* Rotates q and k of `rows` rows by their positions (element j pairs with j + D/2; angle = position *
 * inv_freq[j], inv_freq fp32 [D/2] in device memory; cos and sin times mscale), writes the rotated
 * queries to q_out ([rows, n_q_heads, D], contiguous, out_dtype BF16 or F16) and keys and values to
 * their pages.  q, k, v: dtype, heads contiguous within a row, rows `*_stride` elements apart (multiples
 * of 8, 16-byte aligned bases: columns of one projection's output will do).  q and q_out may both be NULL.
 * Angles and rotated keys are computed in double precision, so that a key's code does not depend on how
 * far it stands. */
int neon_kv4_append(neon_kv4_handle* h, const neon_kv4_batch* batch, void* cache, int rows, int dtype,
                    const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                    int64_t v_stride, const float* inv_freq, float mscale, void* q_out, int out_dtype,
                    void* cuda_stream);

/* The values that the cache holds at the positions of the batch's rows: k_out, v_out [rows, n_kv_heads, D]
 * contiguous, dtype F32 or BF16 (both exact, but that BF16 and F32 overflow to infinity where the scale is
 * 2^126 or more); either may be NULL. */
int neon_kv4_read(neon_kv4_handle* h, const neon_kv4_batch* batch, const void* cache, int rows, void* k_out,
                  void* v_out, int dtype, void* cuda_stream);

/* Bytes of scratch that neon_kv4_attend wants (device memory, 16-byte aligned, its contents mean nothing
 * before and after the call).  Calls that can run at once need scratch of their own. */
uint64_t neon_kv4_attend_workspace(neon_kv4_handle* h, const neon_kv4_batch* batch, int rows, int max_rows);

/* out[row, head] = sum_p w_p v_p / (sum_p w_p + exp(sinks[head])), w_p = exp(scale * q.k_p), over the positions
 * p <= the row's own (and > own - window where window > 0); query head j reads key/value head
 * j / (n_q_heads / n_kv_heads).  q (rows q_stride elements apart) and out ([rows, n_q_heads, D] contiguous):
 * dtype BF16 or F16.  sinks: bf16 [n_q_heads] or NULL.  Rows that see no position get zeros.  rows * n_q_heads / n_kv_heads
 * is 2^26 at most; a call is refused, too, whose table could hold more than 2^35 steps: 64 positions for 8 to 32 of those
 * products and a key/value head.
 * Value scales above 2^125, which only infinities give, count as 2^125.  From values of about 2^110 on a row's sums
 * may leave the range of fp32; it is infinite or NaN then.  Scores are fp32 sums of exact products, good to 2^-23 of
 * their size; from 2^22 on a row may be zero, infinite or NaN.  Each probability is rounded to 11 bits (12 where a
 * sequence has few rows), and the bits that small ones lose are 2^-8 of the sum of weights times values' scales at most.
 * max_rows: the most rows that a sequence has, as far as the host knows it; it chooses the kernel, so results
 * depend on it by these roundings, and speed does: 64 sequences of one row and 4000 positions 48 us told 1, 104 told 64. */
int neon_kv4_attend(neon_kv4_handle* h, const neon_kv4_batch* batch, const void* cache, int rows, int dtype,
                    const void* q, int64_t q_stride, const void* sinks, int window, float scale, int max_rows,
                    void* out, void* workspace, uint64_t workspace_bytes, void* cuda_stream);

/* Reads and clears the handle's status word (blocking; NEON_KV4_* bits, 0 = nothing happened). */
int neon_kv4_status(neon_kv4_handle* h, int* status);

/* Kernels this library launched for the handle so far. */
int64_t neon_kv4_launch_count(const neon_kv4_handle* h);

#ifdef __cplusplus
}
#endif
#endif /* NEON_KV4_H */
