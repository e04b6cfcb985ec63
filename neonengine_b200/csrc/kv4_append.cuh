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
    int split;  // warps per row
};

// The sequence that a row belongs to and the row's position; .x < 0: none.  The whole warp takes part.
__device__ __forceinline__ int2 locate(const Batch& b, int row) {
    const int lane = threadIdx.x & 31;
    int s = row;
    if (b.cu_q) {
        s = 0;
#pragma unroll 4
        for (int i0 = 0; i0 < b.n; i0 += 32)  // sequences that end at or before this row
            s += __popc(__ballot_sync(0xffffffffu, i0 + lane < b.n && b.cu_q[min(i0 + lane, b.n - 1) + 1] <= row));
    }
    if (s >= b.n) return make_int2(-1, 0);
    const int2 sp = b.span(s);
    if (row < sp.x || row >= sp.x + sp.y) return make_int2(-1, 0);
    return make_int2(s, b.seq_lens[s] - sp.y + row - sp.x);
}

// The table's entry for position `pos` of sequence s (-2: the table does not reach it), and what page that is: -1, reported,
// where there is none.  Two steps, so that the load is under way early.
__device__ __forceinline__ int entry_of(const Batch& b, int s, int pos, int P) { return pos / P >= b.width ? -2 : max(b.table[s * b.table_stride + pos / P], -1); }
__device__ __forceinline__ long long page_of(const Batch& b, int entry) {
    if (entry >= 0 && entry < b.n_pages) return entry;
    if ((threadIdx.x & 31) == 0) report(b.status, entry == -2 ? NEON_KV4_BAD_LENGTH : NEON_KV4_BAD_PAGE);
    return -1;
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

// The same of f32 values: scaling them by a power of two is exact, but where it makes them less than any code.
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], int& byte) {
    uint32_t top = 0;  // magnitudes' bits are in order; a NaN's are above all
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    byte = top > 0x7f800000u ? 255 : top == 0 ? 127 : min(max((int)(top >> 23) - 2, 1), 254);
    if (top == 0x7f800000u) byte = 254;
    const int e = 127 - byte, half_e = e / 2;  // in two factors, as 2^-127 is none
    const float f = __uint_as_float((127 + half_e) << 23), g = __uint_as_float((127 + e - half_e) << 23);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t two;
        asm("{\n\t.reg .b8 c;\n\tcvt.rn.satfinite.e2m1x2.f32 c, %1, %2;\n\tmov.b32 %0, {c, 0, 0, 0};\n\t}"
            : "=r"(two) : "f"(x[2 * i + 1] * f * g), "f"(x[2 * i] * f * g));
        w |= two << (8 * i);
    }
    return byte == 255 ? 0u : w;
}

// A warp turns the heads of one row, or (`split` > 1: few rows) one of `split` parts of them; 32 eight-pair pieces at a time.  Piece c of
// a head is elements 8c .. 8c+7 and their partners D/2 further; a lane's c never changes, so it gets its sines and cosines once.
// For keys and values the four lanes of a 32-column block agree on its scale by shuffles.
// The angle position * inv_freq is exact in 53 bits; it is reduced to a fraction of a turn before sine and cosine are
// taken, so its error is 1e-16 of a turn per turn.  Keys are rotated in double precision: a code next to a rounding
// border is then that of the formula, whatever the position (queries are rounded to 16 bits right away and take f32).
// Memory bound from some hundred rows on (19 KB a row at 64 + 8 + 8 heads of 64; 13320 rows take 53 us, 4.8 TB/s; 8 rows 3.3 us, a chain
// of loads).  A row's chain of loads (offsets, length, page)
// and the sines hide behind the loads of the first pieces, and behind other warps: no barrier, no shared memory.
constexpr int kAppendWarps = 4;
template <int DT, class OutT, int D>
__global__ void __launch_bounds__(kAppendWarps * 32, 4) append_kernel(const AppendParams p) {
    using T = typename Elem<DT>::T;
    constexpr int half = D / 2, kPieces = D / 16, kHeads = 32 / kPieces, kAhead = sizeof(T) == 2 ? 4 : 2, kAngles = D / 64;
    const int lane = threadIdx.x & 31, c = lane % kPieces;
    const int task = blockIdx.x * kAppendWarps + threadIdx.x / 32, row = task / p.split;
    pdl_wait();
    pdl_launch_dependents();
    if (row >= p.b.rows) return;
    const int first_head = p.q ? 0 : p.s.nq, heads = p.s.nq + 2 * p.s.nkv, v_head = p.s.nq + p.s.nkv;
    // this warp's rounds of kHeads heads
    const int rounds = (heads - first_head + kHeads - 1) / kHeads, part = task - row * p.split;
    const int begin = (int)((long long)rounds * part / p.split), end = (int)((long long)rounds * (part + 1) / p.split);
    struct Raw { uint4 v[sizeof(T) == 2 ? 2 : 4]; };
    auto source = [&](int head) {
        const T* base;
        if (head < p.s.nq) base = static_cast<const T*>(p.q) + row * p.q_stride + head * D;
        else if (head < v_head) base = static_cast<const T*>(p.k) + row * p.k_stride + (head - p.s.nq) * D;
        else base = static_cast<const T*>(p.v) + row * p.v_stride + (head - v_head) * D;
        return base + c * 8;
    };
    auto head_of = [&](int round) { return first_head + round * kHeads + lane / kPieces; };
    auto load = [&](int round) {
        Raw r;
        const T* src = source(min(head_of(round), heads - 1));
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < (int)sizeof(Raw) / 32; ++i) r.v[h * (sizeof(Raw) / 32) + i] = reinterpret_cast<const uint4*>(src + h * half)[i];
        return r;
    };
    Raw raw[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        if (begin + i < end) raw[i] = load(begin + i);
    const int2 at = locate(p.b, row);
    if (at.x < 0 || at.y < 0) return;  // the same for the whole warp
    const int entry = entry_of(p.b, at.x, at.y, p.s.P);
    double cs[kAngles], sn[kAngles];
#pragma unroll
    for (int i = 0; i < kAngles; ++i) {
        const double turns = (double)at.y * (double)p.inv_freq[i * 32 + lane] * 0.15915494309189533577;  // 1 / (2 pi)
        sincospi(2.0 * (turns - rint(turns)), &sn[i], &cs[i]);
        cs[i] *= (double)p.mscale;
        sn[i] *= (double)p.mscale;
    }
    auto angle = [&](const double (&v)[kAngles], int j) {  // of pair 8c + j
        const int k = 8 * c + j;
        if constexpr (kAngles == 1) return __shfl_sync(0xffffffffu, v[0], k);
        const double lo = __shfl_sync(0xffffffffu, v[0], k & 31), hi = __shfl_sync(0xffffffffu, v[kAngles - 1], k & 31);
        return k < 32 ? lo : hi;
    };
    float fc[8], fs[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { fc[j] = (float)angle(cs, j); fs[j] = (float)angle(sn, j); }
    const long long page = page_of(p.b, entry);
    const int slot = at.y % p.s.P;
    for (int r0 = begin; r0 < end; r0 += kAhead) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (r0 + i >= end) break;
            const int head = head_of(r0 + i);
            float a[8], b[8];
            load8(reinterpret_cast<const T*>(&raw[i].v[0]), a);
            load8(reinterpret_cast<const T*>(&raw[i].v[sizeof(Raw) / 32]), b);
            for (int k = 1; k < p.n_parts; ++k) {
                float e[8], f[8];
                const T* src = source(min(head, heads - 1)) + k * p.part_stride;
                load8(src, e);
                load8(src + half, f);
#pragma unroll
                for (int j = 0; j < 8; ++j) { a[j] += e[j]; b[j] += f[j]; }
            }
            if (r0 + kAhead + i < end) raw[i] = load(r0 + kAhead + i);
            if (head < p.s.nq) {
                float x[8], y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    x[j] = a[j] * fc[j] - b[j] * fs[j];
                    y[j] = b[j] * fc[j] + a[j] * fs[j];
                }
                OutT* o = static_cast<OutT*>(p.q_out) + ((long long)row * p.s.nq + head) * D + c * 8;
                store8(o, x);
                store8(o + half, y);
            }
            if (!__any_sync(0xffffffffu, head >= p.s.nq && head < heads)) continue;
            const bool is_v = head >= v_head;
            int bx, by;
            uint32_t wx, wy;
            if (!__any_sync(0xffffffffu, head >= p.s.nq && !is_v)) {  // values alone: as they came
                wx = quantise8(a, bx);
                wy = quantise8(b, by);
            } else {
                double x[8], y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const double co = angle(cs, j), si = angle(sn, j);
                    x[j] = is_v ? (double)a[j] : (double)a[j] * co - (double)b[j] * si;
                    y[j] = is_v ? (double)b[j] : (double)b[j] * co + (double)a[j] * si;
                }
                wx = quantise8(x, bx);
                wy = quantise8(y, by);
            }
            if (head < p.s.nq || head >= heads || page < 0) continue;
            uint8_t* rec = p.cache + (page * p.s.nkv + head - (is_v ? v_head : p.s.nq)) * p.s.record();
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
}

struct ReadParams {
    Batch b;
    Shape s;
    const uint8_t* cache;
    void *k_out, *v_out;
    int split;  // warps per row
};

// A warp (or `split` of them) per row; a lane turns eight codes into values, 32 pieces of the row's heads at a time.  13320 rows of 8 + 8
// heads of 64 to bf16 take 11 us behind the append (2.6 KB a row), 17 from HBM: not the memory bounds it but some 1.8 instructions a
// clock and SM, divisions by the head's and page's size and four bytes of codes a lane among them.  A few rows take 2 us.
template <class OutT>
__global__ void __launch_bounds__(128) read_kernel(const ReadParams p) {
    const int task = blockIdx.x * 4 + threadIdx.x / 32, row = task / p.split, lane = threadIdx.x & 31, D = p.s.D, per_head = D / 8, units = p.s.nkv * per_head;
    pdl_wait();
    pdl_launch_dependents();
    if (row >= p.b.rows) return;
    const int2 at = locate(p.b, row);
    if (at.x < 0 || at.y < 0) return;
    const long long page = page_of(p.b, entry_of(p.b, at.x, at.y, p.s.P));
    if (page < 0) return;
    const int slot = at.y % p.s.P;
#pragma unroll 4
    for (int i = (task - row * p.split) * 32 + lane; i < 2 * units; i += 32 * p.split) {
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
