// What the kernels of the 4-bit paged cache share: the record's layout, the batch as a kernel sees it, element types.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/neon_kv4.h"
#include "moe_common.cuh"

namespace neon {
namespace kv4 {

constexpr int kTopScale = 252;  // attention takes larger scales (of infinities alone: 2^125 holds the largest finite number) for 2^125

struct Shape {
    int nq, nkv, D, P;
    __host__ __device__ int codes() const { return P * D / 2; }        // bytes of a record's key (or value) codes
    __host__ __device__ int scales() const { return P * D / 32; }      // bytes of its key (or value) scales
    __host__ __device__ int record() const { return P * (D + D / 16); }
};

struct Batch {
    const int32_t *seq_lens, *cu_q, *table;
    long long table_stride, n_pages;
    int width, n, rows;  // pages a table row can name, sequences, rows of the inputs
    int* status;
    // first row and number of rows of sequence b, kept inside the inputs whatever cu_q says
    __device__ __forceinline__ int2 span(int b) const {
        if (!cu_q) return b < rows ? make_int2(b, 1) : make_int2(rows, 0);
        const int lo = min(max(cu_q[b], 0), rows), hi = min(max(cu_q[b + 1], lo), rows);
        return make_int2(lo, hi - lo);
    }
};

__device__ __forceinline__ void report(int* status, int bits) { atomicOr(status, bits); }

template <int DT>
struct Elem;
template <>
struct Elem<NEON_KV4_F32> { using T = float; };
template <>
struct Elem<NEON_KV4_BF16> { using T = __nv_bfloat16; };
template <>
struct Elem<NEON_KV4_F16> { using T = __half; };

// eight elements at a 16-byte aligned address as floats
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&x)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void load8(const __half* p, float (&x)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x; x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
    const __half2 r = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2(x[0], x[1], T()), pack2(x[2], x[3], T()), pack2(x[4], x[5], T()), pack2(x[6], x[7], T()));
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// 8 e2m1 codes -> 8 f16, in column order
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t (&r)[4]) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\tcvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
        : "r"(w));
}
// two E8M0 bytes -> their f32 values (255 is NaN)
__device__ __forceinline__ float2 scales_to_f32(uint32_t two) {
    uint32_t r;
    asm("cvt.rn.bf16x2.ue8m0x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
    return make_float2(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
}

}  // namespace kv4
}  // namespace neon
