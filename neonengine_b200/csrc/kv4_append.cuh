// Appending to the 4-bit paged cache and reading positions back.
#pragma once
#include "kv4_common.cuh"

namespace neon {
namespace kv4 {

struct AppendParams {
    Batch b;
    Shape s;
    const void *q, *k, *v;
    long long q_stride, k_stride, v_stride;  // elements between rows
    int n_parts;                             // the inputs are sums of this many parts (1 but for the decoder's K-split projection) ..
    long long part_stride;                   // .. this many elements apart
    const float* inv_freq;
    float mscale;
    void* q_out;
    uint8_t* cache;
};

// The sequence that a row belongs to and the row's position; .x < 0: none.  The whole CTA takes part.
__device__ __forceinline__ int2 locate(const Batch& b, int row) {
    int s = row;
    if (b.cu_q) {
        s = 0;
        for (int i = threadIdx.x; i - threadIdx.x < b.n; i += blockDim.x)  // sequences that end at or before this row
            s += __syncthreads_count(i < b.n && b.cu_q[i + 1] <= row);
    }
    if (s >= b.n) return make_int2(-1, 0);
    const int2 sp = b.span(s);
    if (row < sp.x || row >= sp.x + sp.y) return make_int2(-1, 0);
    return make_int2(s, b.seq_lens[s] - sp.y + row - sp.x);
}

// Where position `pos` of sequence s is held: the page, or -1 (reported) where there is none.
__device__ __forceinline__ long long page_of(const Batch& b, int s, int pos, int P) {
    if (pos / P >= b.width) {
        if (threadIdx.x == 0) report(b.status, NEON_KV4_BAD_LENGTH);
        return -1;
    }
    const int id = b.table[s * b.table_stride + pos / P];
    if (id < 0 || id >= b.n_pages) {
        if (threadIdx.x == 0) report(b.status, NEON_KV4_BAD_PAGE);
        return -1;
    }
    return id;
}

// Rounds to 24 bits so that a later rounding to fewer bits is the one of the exact value: towards zero, the last bit
// set where something was cut off.
__device__ __forceinline__ float round_to_odd(double y) {
    const float f = __double2float_rz(y);
    return (double)f == y ? f : __uint_as_float(__float_as_uint(f) | 1u);
}

// Eight values of a block (the block's others are in the lanes that differ in bits 0 and 1) -> four bytes of codes; the
// block's scale byte in `byte`.  floor(log2 amax) is the largest exponent field.
__device__ __forceinline__ uint32_t quantise8(const double (&x)[8], int& byte) {
    int e = 0;  // biased exponent of the largest magnitude; 0x7ff: infinity, 0x800: NaN
#pragma unroll
    for (int i = 0; i < 8; ++i) e = max(e, x[i] != x[i] ? 0x800 : (__double2hiint(x[i]) >> 20) & 0x7ff);
    e = max(e, __shfl_xor_sync(0xffffffffu, e, 1));
    e = max(e, __shfl_xor_sync(0xffffffffu, e, 2));
    byte = e == 0x800 ? 255 : e == 0 ? 127 : min(max(e - 1023 - 2 + 127, 1), 254);
    const double inv = __hiloint2double((1023 + 127 - byte) << 20, 0);  // 2^(127 - byte)
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float lo = round_to_odd(x[2 * i] * inv), hi = round_to_odd(x[2 * i + 1] * inv);
        uint32_t two;
        asm("{\n\t.reg .b8 c;\n\tcvt.rn.satfinite.e2m1x2.f32 c, %1, %2;\n\tmov.b32 %0, {c, 0, 0, 0};\n\t}" : "=r"(two) : "f"(hi), "f"(lo));
        w |= two << (8 * i);
    }
    return byte == 255 ? 0u : w;
}

// One CTA per row.  A thread turns eight pairs of a head: elements 8c .. 8c+7 and their partners D/2 further; for keys
// and values the four threads of a 32-column block agree on its scale by shuffles.
// The angle position * inv_freq is exact in 53 bits; it is reduced to a fraction of a turn before sine and cosine are
// taken, so its error is 1e-16 of a turn per turn.  Keys are rotated in double precision: a code next to a rounding
// border is then that of the formula, whatever the position (queries are rounded to 16 bits right away and take f32).
// Memory bound from some hundred rows on: 15 KB a row at 64 + 8 + 8 heads of 64.  All loads of a thread are in flight
// before its CTA waits for the angles.
template <int DT, class OutT>
__global__ void __launch_bounds__(512) append_kernel(const AppendParams p) {
    using T = typename Elem<DT>::T;
    __shared__ double cs[64], sn[64];
    const int row = blockIdx.x, D = p.s.D, half = D / 2, per_head = D / 16;
    const int q_units = p.q ? p.s.nq * per_head : 0, kv_units = p.s.nkv * per_head, units = q_units + 2 * kv_units;
    pdl_wait();
    const int2 at = locate(p.b, row);
    if (at.x < 0 || at.y < 0) return;  // uniform over the CTA
    auto fetch = [&](int u, float (&a)[8], float (&b)[8]) {
        const T* base;
        if (u < q_units) base = static_cast<const T*>(p.q) + row * p.q_stride;
        else if ((u -= q_units) < kv_units) base = static_cast<const T*>(p.k) + row * p.k_stride;
        else base = static_cast<const T*>(p.v) + row * p.v_stride, u -= kv_units;
        base += u / per_head * D + u % per_head * 8;
        load8(base, a);
        load8(base + half, b);
        for (int i = 1; i < p.n_parts; ++i) {
            float c[8], d[8];
            load8(base + i * p.part_stride, c);
            load8(base + i * p.part_stride + half, d);
#pragma unroll
            for (int j = 0; j < 8; ++j) { a[j] += c[j]; b[j] += d[j]; }
        }
    };
    float a[8], b[8];
    if (threadIdx.x < units) fetch(threadIdx.x, a, b);
    if (threadIdx.x < half) {
        const double turns = (double)at.y * (double)p.inv_freq[threadIdx.x] * 0.15915494309189533577;  // 1 / (2 pi)
        double s, c;
        sincospi(2.0 * (turns - rint(turns)), &s, &c);
        cs[threadIdx.x] = c * (double)p.mscale;
        sn[threadIdx.x] = s * (double)p.mscale;
    }
    const long long page = page_of(p.b, at.x, at.y, p.s.P);
    __syncthreads();
    const int slot = at.y % p.s.P;
    // whole warps stay together for the shuffles: units is rounded up to the warp
    for (int u0 = threadIdx.x; u0 - (threadIdx.x & 31) < units; u0 += blockDim.x) {
        const int u = min(u0, units - 1);
        if (u0 != threadIdx.x || u != u0) fetch(u, a, b);
        const int c = u % per_head;
        const bool is_q = u < q_units, is_v = u >= q_units + kv_units;
        double x[8], y[8];
        if (is_q) {
            float r0[8], r1[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float co = (float)cs[c * 8 + j], si = (float)sn[c * 8 + j];
                r0[j] = a[j] * co - b[j] * si;
                r1[j] = b[j] * co + a[j] * si;
            }
            if (u0 < units) {
                OutT* o = static_cast<OutT*>(p.q_out) + ((long long)row * p.s.nq + u / per_head) * D + c * 8;
                store8(o, r0);
                store8(o + half, r1);
            }
        }
        if (__all_sync(0xffffffffu, is_q)) continue;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double co = is_v ? 1.0 : cs[c * 8 + j], si = is_v ? 0.0 : sn[c * 8 + j];
            x[j] = is_v ? (double)a[j] : (double)a[j] * co - (double)b[j] * si;
            y[j] = is_v ? (double)b[j] : (double)b[j] * co + (double)a[j] * si;
        }
        int bx, by;
        const uint32_t wx = quantise8(x, bx), wy = quantise8(y, by);
        if (is_q || u0 >= units || page < 0) continue;
        const int head = (u - q_units - (is_v ? kv_units : 0)) / per_head;
        uint8_t* rec = p.cache + (page * p.s.nkv + head) * p.s.record();
        uint8_t* codes = rec + (is_v ? p.s.codes() : 0) + slot * (D / 2) + c * 4;
        *reinterpret_cast<uint32_t*>(codes) = wx;
        *reinterpret_cast<uint32_t*>(codes + half / 2) = wy;
        if (c % 4 == 0) {
            uint8_t* sc = rec + 2 * p.s.codes() + (is_v ? p.s.scales() : 0) + slot * (D / 32) + c / 4;
            sc[0] = (uint8_t)bx;
            sc[half / 32] = (uint8_t)by;
        }
    }
}

struct ReadParams {
    Batch b;
    Shape s;
    const uint8_t* cache;
    void *k_out, *v_out;
};

// One CTA per row; a thread turns eight codes into values.
template <class OutT>
__global__ void __launch_bounds__(256) read_kernel(const ReadParams p) {
    const int row = blockIdx.x, D = p.s.D, per_head = D / 8, units = p.s.nkv * per_head;
    pdl_wait();
    const int2 at = locate(p.b, row);
    if (at.x < 0 || at.y < 0) return;
    const long long page = page_of(p.b, at.x, at.y, p.s.P);
    if (page < 0) return;
    const int slot = at.y % p.s.P;
    for (int i = threadIdx.x; i < 2 * units; i += blockDim.x) {
        const int is_v = i >= units, u = i - is_v * units, head = u / per_head, c = u % per_head;
        OutT* o = static_cast<OutT*>(is_v ? p.v_out : p.k_out);
        if (!o) continue;
        const uint8_t* rec = p.cache + (page * p.s.nkv + head) * p.s.record();
        uint32_t f[4];
        codes_to_f16(*reinterpret_cast<const uint32_t*>(rec + is_v * p.s.codes() + slot * (D / 2) + c * 4), f);
        const float scale = scales_to_f32(rec[2 * p.s.codes() + is_v * p.s.scales() + slot * (D / 32) + c / 4]).x;
        float x[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&f[j]));
            x[2 * j] = v.x * scale;
            x[2 * j + 1] = v.y * scale;
        }
        store8(o + ((long long)row * p.s.nkv + head) * D + c * 8, x);
    }
}

}  // namespace kv4
}  // namespace neon
