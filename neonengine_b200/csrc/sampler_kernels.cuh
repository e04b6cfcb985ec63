// Sampling kernels: a token per row of logits after temperature, top-k, top-p and min-p (definitions: neon_sampler.h).
//
//   scan     streams the logits once, a warp per 1024 of a row: their maximum, their weight relative to it, and the
//            elements that could be among the row's largest - all from a bound of the warp's own on;
//   pick     one CTA per row.  No filter: the 1024 that hold the token, from the warps' weights, then the token in them.
//            Filters: cuts and token are found among the listed elements, which suffices whenever the last kept one is not
//            below the highest of the warps' bounds; other rows are left to
//   whole    a cluster per row that keeps the row in its shared memory and finds cuts and token among all of it.
// Vocabularies that fit pick's list go to pick alone.
//
// One histogram over the list cuts it down to what the first filter can keep.  With up to 512 elements every thread then has
// one, and finds its rank and the weight ahead of it by looking at the others; more are cut by histograms over ten bits of the
// key at a time, the key being the logit in descending order (or the index).
// Weights are integers of 2^-43 of the largest, so that sums depend on no order; a histogram keeps them as three words
// of 15 bits each per element, which shared memory can add atomically.
//
// What bounds them, with 201088 fp32 logits a row.  scan: issue slots and the f64 units, for weights (256 rows 74 us with pick, 2.8 TB/s, 2.3
// instructions a clock and SM; without sums it would be 38; 16-bit logits take as long, 79).  pick: a chain of barriers and of
// searches in shared memory, one CTA a row (1 row 17 us; 256 rows without filters 8).  whole: the same and a histogram with two or three
// shared memory atomics an element; a few rows take 55 us, however few.
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/neon_sampler.h"
#include "moe_common.cuh"

namespace neon {
namespace sampler {

namespace cg = cooperative_groups;

constexpr int kChunk = 1024;          // logits of a warp of the scan
constexpr int kSlots = 64;            // list entries a warp can leave
constexpr int kList = 6144;           // list entries of pick
constexpr int kPickThreads = 512, kScanWarps = 8;
constexpr int kBins = 1024, kBinBits = 10;
constexpr int kWeightBits = 43;       // weights are multiples of 2^-43; a row's sum stays below 2^63
constexpr double kUnit = 8796093022208.0;  // 2^43
constexpr int kClusterCtas = 8;
constexpr float kLowest = -3.402823466e38f;  // the lowest that can be drawn
typedef unsigned long long u64;

struct ChunkHead {   // what a warp of the scan leaves about its logits
    float max, bound;   // largest; every logit >= bound is listed
    int listed, valid;  // entries; logits above -infinity
    double weight;      // of all, relative to 2^exponent, or (exponent = kRelative) to max
    int exponent, pad;
};

struct Params {
    const void* logits;
    int dtype, vocab, batch, chunks;
    long long stride;
    const float *uniform, *temperature, *top_p, *min_p;
    const int32_t* top_k;
    int32_t *tokens, *kept;
    float* probs;
    ChunkHead* heads;   // [batch][chunks]
    uint2* entries;     // [batch][chunks][kSlots]: logit bits, index
    int* left;          // [batch]: rows for `whole`
    int rank;           // how many lanes' maxima a warp's bound lets through
};

struct Rule {  // a row's parameters, with what they exclude made plain
    bool greedy, by_k, by_p, by_m;
    double c;  // log2(e) / temperature; at least 2^-500, so that 1/c is finite
    int k;
    double p, m;
    float u;
    __device__ bool filters() const { return by_k || by_p || by_m; }
};
__device__ __forceinline__ Rule rule_of(const Params& p, int row) {
    Rule r;
    const float t = p.temperature ? p.temperature[row] : 1.f;
    r.greedy = !(t > 0.f);
    r.c = r.greedy ? 1.0 : fmax(1.4426950408889634074 / (double)t, 0x1p-500);
    r.k = p.top_k ? p.top_k[row] : 0;
    r.by_k = r.k > 0 && r.k < p.vocab;
    const float tp = p.top_p ? p.top_p[row] : 1.f, mp = p.min_p ? p.min_p[row] : 0.f;
    r.by_p = tp < 1.f;
    r.p = fmax((double)tp, 0.0);
    r.by_m = mp > 0.f;
    r.m = fmin((double)mp, 1.0);
    const float u = p.uniform[row];
    r.u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;
    return r;
}

__device__ __forceinline__ float clean(float x) { return fmaxf(x, -INFINITY); }  // NaN is -infinity
__device__ __forceinline__ float load1(const Params& p, long long i) {
    float x;
    if (p.dtype == 0) x = static_cast<const float*>(p.logits)[i];
    else if (p.dtype == 1) x = __bfloat162float(static_cast<const __nv_bfloat16*>(p.logits)[i]);
    else x = __half2float(static_cast<const __half*>(p.logits)[i]);
    return clean(x);
}
// ascending keys for descending logits
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);  // -0 is 0
    return b & 0x80000000u ? b : ~b & 0x7fffffffu;
}
__device__ __forceinline__ float key_logit(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k : ~k & 0x7fffffffu); }

// 2^(j/64), j < 64, a copy for every lane: reads never share a bank
constexpr int kTable = 64 * 32;
__device__ __forceinline__ void fill_table(double* tab) {
    for (int j = threadIdx.x; j < 64; j += blockDim.x) {
        const double v = exp2(j / 64.0);
        for (int l = 0; l < 32; ++l) tab[j * 32 + ((l + j) & 31)] = v;
    }
}
// exp((x - top) / temperature) to 4e-11: with t = 64 (x - top) log2(e) / temperature = k + r, |r| <= 1/2, a table of 2^(k/64)
// times a cubic in r, whose next term is (ln 2 / 128)^4 / 24 = 3.6e-11.  What is below 2^-60 counts as nothing.
struct Weigher {
    double c, off;  // t = c x + off
    float top, low;
    const double* tab;  // this lane's column
    __device__ __forceinline__ Weigher(float top_, double log2_scale, const double* table) : top(top_), tab(table + (threadIdx.x & 31)) {
        c = 64.0 * log2_scale;
        off = -c * (double)top;
        low = fmaxf((float)((double)top - 60.0 / log2_scale), kLowest);
        if (top == INFINITY) low = INFINITY;  // infinities alone, at weight 1
    }
    // of an x >= low, where top is finite (of another: any number)
    __device__ __forceinline__ double bare(float x) const {
        const double kMagic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low word is the rounded integer
        const double kA = 0.010830424696249145, kB = 5.8649049505537566e-05, kC = 2.1173136998904953e-07;  // A = ln 2 / 64, A^2 / 2, A^3 / 6
        const double t = fma((double)x, c, off), kd = t + kMagic;
        const int k = __double2loint(kd);
        const double r = t - (kd - kMagic), v = tab[(k & 63) * 32];
        const double w = fma(v, r * fma(r, fma(r, kC, kB), kA), v);
        return __hiloint2double(__double2hiint(w) + (k & ~63) * (1 << 14), __double2loint(w));
    }
    __device__ __forceinline__ double operator()(float x) const { return x == top ? 1.0 : x >= low ? bare(x) : 0.0; }  // exactly 1 for the largest
};
// Sums of many weights, at half the instructions: 2^(x log2(e) / temperature), not relative to a largest.  The product's integer
// part is found in f32; what is left of it is exact to 2^-25, as a fused multiply-add rounds once, and so small that the cubic can be
// f32, too: 5e-10 of a weight, and no more than 1e-9 of a row's sum of any number of them.
struct Adder {
    float hi, lo, low;  // 64 log2(e) / temperature as two f32
    const double* tab;
    bool fits;          // the powers are within f64's range and the scale within f32's, and `low` is below the largest by what it should be
    __device__ __forceinline__ Adder(const Weigher& w) : hi((float)w.c), lo((float)(w.c - (double)(float)w.c)), low(w.low), tab(w.tab) {
        fits = hi < INFINITY && fabs(w.off) < 64.0 * 900 && w.top < INFINITY && (double)w.top * w.c - (double)w.low * w.c > 64.0 * 55;
    }
    __device__ __forceinline__ float steps(float x) const { return fmaf(x, hi, 12582912.f); }  // 1.5 * 2^23 + the product's integer part
    __device__ __forceinline__ void add(double& sum, float x) const {
        x = fmaxf(x, low);  // 2^-60 of the largest for nothing
        const float k = steps(x), r = fmaf(x, lo, fmaf(x, hi, 12582912.f - k));
        const uint32_t bits = __float_as_uint(k);  // its low bits are the integer's
        const double v = tab[(bits & 63) * 32];
        const float q = r * fmaf(r, fmaf(r, 2.1173136998904953e-07f, 5.8649049505537566e-05f), 0.010830424696249145f);
        const double w = __hiloint2double(__double2hiint(v) + (int)((bits & ~63u) << 14), __double2loint(v));
        sum += fma(w, (double)q, w);
    }
    // 2^e of about the weight of x, and its inverse's power
    __device__ __forceinline__ int exponent(float x) const { return (int)(__float_as_uint(steps(x)) - 0x4b400000u) >> 6; }
};
constexpr int kRelative = -0x7fffffff - 1;

__device__ __forceinline__ u64 to_units(double w) {  // w <= 2^9, in 2^-43, rounded
    return (u64)(__double_as_longlong(fma(w, kUnit, 4503599627370496.0)) & 0xfffffffffffffll);
}

// A chunk's weight, relative to the row's largest.  Nothing where its largest logit rounds to nothing, since no token of it can be drawn
// then: the sum is one of weights that are not rounded.
__device__ __forceinline__ u64 chunk_units(const ChunkHead& h, const Weigher& w) {
    if (h.max == -INFINITY || to_units(w(h.max)) == 0) return 0;
    const double factor = h.exponent == kRelative ? w(h.max) : exp2((64.0 * h.exponent + w.off) * (1.0 / 64.0));
    return (u64)(h.weight * factor * kUnit);
}

// ---- scan -------------------------------------------------------------------------------------------------------------
// Largest first across the warp's lanes.
__device__ __forceinline__ float warp_sorted(float v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1) {
            const float o = __shfl_xor_sync(0xffffffffu, v, j);
            v = ((lane & k) == 0) == ((lane & j) == 0) ? fmaxf(v, o) : fminf(v, o);
        }
    return v;
}

// Warps go through the chunks of all rows; a chunk's row, its rule and its logits are one after the other in memory, so the
// next chunk's loads need nothing of this one's.
template <int DT>
__global__ void __launch_bounds__(kScanWarps * 32, 2) scan_kernel(const Params p) {
    __shared__ double tab[kTable];
    const int lane = threadIdx.x & 31;
    fill_table(tab);
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    const int tasks = p.batch * p.chunks, step = gridDim.x * kScanWarps;
    constexpr int kSize = DT == 0 ? 4 : 2;
    // element 4 * (32 v + lane) + c of a chunk is x[4 v + c]
    auto fetch = [&](float (&x)[32], int task) {
        if (task >= tasks) return;
        const int row = task / p.chunks, i0 = (task - row * p.chunks) * kChunk, n = min(kChunk, p.vocab - i0);
        const long long base = row * p.stride + i0;
        if (n == kChunk && ((reinterpret_cast<uintptr_t>(p.logits) + base * kSize) & (4 * kSize - 1)) == 0) {
#pragma unroll
            for (int v = 0; v < 8; ++v) {
                const long long at = base + 4 * (32 * v + lane);
                if (DT == 0) {
                    const float4 f = __ldcs(reinterpret_cast<const float4*>(static_cast<const float*>(p.logits) + at));
                    x[4 * v] = f.x; x[4 * v + 1] = f.y; x[4 * v + 2] = f.z; x[4 * v + 3] = f.w;
                } else {
                    const uint2 f = __ldcs(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.logits) + at));
                    const uint32_t w[2] = {f.x, f.y};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (DT == 1) {
                            x[4 * v + 2 * h] = __uint_as_float(w[h] << 16);
                            x[4 * v + 2 * h + 1] = __uint_as_float(w[h] & 0xffff0000u);
                        } else {
                            const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&w[h]));
                            x[4 * v + 2 * h] = g.x;
                            x[4 * v + 2 * h + 1] = g.y;
                        }
                    }
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const int e = 4 * (32 * (i / 4) + lane) + i % 4;
                x[i] = e < n ? load1(p, base + e) : -INFINITY;
            }
        }
    };
    int task = blockIdx.x * kScanWarps + threadIdx.x / 32;
    float x[32], ahead[32];
    fetch(ahead, task);
    for (; task < tasks; task += step) {
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = clean(ahead[i]);
        fetch(ahead, task + step);  // on their way while this chunk is looked at
        const int row = task / p.chunks, i0 = (task - row * p.chunks) * kChunk;
        const Rule r = rule_of(p, row);
        float top = x[0], least = x[0];
#pragma unroll
        for (int i = 1; i < 32; ++i) {
            top = fmaxf(top, x[i]);
            least = fminf(least, x[i]);
        }
        ChunkHead head;
        float bound = INFINITY;
        const bool list_wanted = !r.greedy && r.filters();
        if (list_wanted) bound = __shfl_sync(0xffffffffu, warp_sorted(top), p.rank - 1);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        head.max = top;
        head.valid = kChunk;
        if (__any_sync(0xffffffffu, least == -INFINITY)) {
            int valid = 0;
#pragma unroll
            for (int i = 0; i < 32; ++i) valid += x[i] > -INFINITY;
            head.valid = __reduce_add_sync(0xffffffffu, valid);
        }
        // the whole row's weight counts where nothing but top_p cuts it
        double sum = 0.0;
        head.exponent = kRelative;
        head.pad = 0;
        if (!r.greedy && !r.by_k && (r.by_p || !r.by_m) && top > -INFINITY) {
            const Weigher weight(top, r.c, tab);
            const Adder adder(weight);
            if (adder.fits && head.valid == kChunk) {
                double part[4] = {};
#pragma unroll
                for (int i = 0; i < 32; ++i) adder.add(part[i & 3], x[i]);
                head.exponent = adder.exponent(top);
                sum = ((part[0] + part[1]) + (part[2] + part[3])) * __hiloint2double((1023 - head.exponent) << 20, 0);
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) sum += weight(x[i]);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        head.weight = sum;
        // the list
        int listed = 0;
        if (list_wanted) {
            bound = fmaxf(bound, kLowest);  // -infinity is not listed
            auto count = [&] {
                int c = 0;
#pragma unroll
                for (int i = 0; i < 32; ++i) c += x[i] >= bound;
                return __reduce_add_sync(0xffffffffu, c);
            };
            if (count() > kSlots) {  // many equal ones: those above
                bound = bound < INFINITY ? nextafterf(bound, INFINITY) : bound;
                if (count() > kSlots) bound = __int_as_float(0x7fc00000);  // none: nothing is >= NaN
            }
            uint2* list = p.entries + (long long)task * kSlots;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const bool in = x[i] >= bound;
                const uint32_t b = __ballot_sync(0xffffffffu, in);
                if (in) list[listed + __popc(b & ((1u << lane) - 1))] = make_uint2(__float_as_uint(x[i]), i0 + 4 * (32 * (i / 4) + lane) + i % 4);
                listed += __popc(b);
            }
        }
        // fewer finite logits than the bound lets through: all are listed
        head.bound = listed == head.valid ? -INFINITY : bound;
        head.listed = bound == bound ? listed : kList + 1;  // no list: more than pick takes
        if (lane == 0) p.heads[task] = head;
    }
}

// ---- cuts and token among elements in shared memory ---------------------------------------------------------------------
struct Found {
    uint32_t key;
    u64 before, at;  // sum of the keys before it, sum of the key itself
};

// The CTAs that hold a row's elements, and the histogram they share.
template <int C>
struct Group {
    uint32_t (*hist)[kBins];  // three words of a bin's sum
    u64* scratch;             // [64]
    Weigher weight;
    __device__ void sync() const {
        if constexpr (C == 1) __syncthreads();
        else cg::this_cluster().sync();
    }
    // Sum over the group's CTAs of a value that every thread of this CTA holds a part of; the same in all threads.  slot: a
    // place of scratch that no other sum between two syncs uses.
    __device__ u64 total(u64 v, int slot) const {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
        __syncthreads();
        u64 s = 0;
        for (int w = 0; w < (int)blockDim.x / 32; ++w) s += scratch[w];
        if constexpr (C > 1) {
            if (threadIdx.x == 0) scratch[32 + slot] = s;
            sync();
            s = 0;
            for (int r = 0; r < C; ++r) s += *cg::this_cluster().map_shared_rank(scratch + 32 + slot, r);
        }
        return s;
    }
    __device__ __forceinline__ void add(uint32_t b, u64 units) const {
        atomicAdd(&hist[0][b], (uint32_t)units & 0x7fffu);
        if (units >> 15) {
            atomicAdd(&hist[1][b], (uint32_t)(units >> 15) & 0x7fffu);
            if (units >> 30) atomicAdd(&hist[2][b], (uint32_t)(units >> 30));
        }
    }
    __device__ void clear() const {
        for (int i = threadIdx.x; i < 3 * kBins; i += blockDim.x) (&hist[0][0])[i] = 0;
        __syncthreads();
    }
    // The bin in which the running sum, from f.before on, reaches target (or exceeds it), or the last that is not empty; f.before
    // and f.at become the sums before it and of it.  Begins and ends with a barrier of the group.
    __device__ uint32_t reach(Found& f, u64 target, bool beyond) const {
        constexpr int kSlice = kBins / C, kPer = (kSlice + kPickThreads - 1) / kPickThreads;  // a CTA adds up a slice of the bins
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = C == 1 ? 0 : (int)cg::this_cluster().block_rank();
        sync();
        u64 bin[kPer], mine = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int b = threadIdx.x * kPer + j;
            bin[j] = 0;
            if (b < kSlice)
#pragma unroll
                for (int r = 0; r < C; ++r) {
                    const uint32_t* h = &hist[0][rank * kSlice + b];
                    if constexpr (C > 1) h = cg::this_cluster().map_shared_rank(h, r);
                    bin[j] += (u64)h[0] + ((u64)h[kBins] << 15) + ((u64)h[2 * kBins] << 30);
                }
            mine += bin[j];
        }
        u64 run = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 v = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += v;
        }
        if (lane == 31) scratch[warp] = run;
        __syncthreads();
        u64 part = lane < kPickThreads / 32 ? scratch[lane] : 0, upto = part;
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            const u64 v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        u64 start = run - mine + __shfl_sync(0xffffffffu, upto - part, warp), all = __shfl_sync(0xffffffffu, upto, kPickThreads / 32 - 1);
        if constexpr (C > 1) {  // the slices before this one
            if (threadIdx.x == 0) scratch[60] = all;
            sync();
            u64 theirs = lane < C ? *cg::this_cluster().map_shared_rank(scratch + 60, lane) : 0, sum = theirs;
#pragma unroll
            for (int o = 1; o < C; o <<= 1) {
                const u64 v = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += v;
            }
            start += __shfl_sync(0xffffffffu, sum - theirs, rank);
            all = __shfl_sync(0xffffffffu, sum, C - 1);
        }
        start += f.before;
        const u64 end_of_all = f.before + all, goal = beyond ? min(target, end_of_all - 1) : min(target, end_of_all);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const u64 end = start + bin[j];
            if (bin[j] && (beyond ? start <= goal && end > goal : start < goal && end >= goal)) {  // one bin of all
#pragma unroll
                for (int r = 0; r < C; ++r) {  // told to everybody
                    u64* to = scratch + 56;
                    if constexpr (C > 1) to = cg::this_cluster().map_shared_rank(to, r);
                    to[0] = rank * kSlice + threadIdx.x * kPer + j;
                    to[1] = start;
                    to[2] = bin[j];
                }
            }
            start = end;
        }
        sync();  // also: everybody has read everybody's histogram
        f.before = scratch[57];
        f.at = scratch[58];
        const uint32_t b = (uint32_t)scratch[56];
        __syncthreads();
        return b;
    }
};

// The first key, ascending from klo to khi, at which the running sum (of what comes before klo, `before`, on) reaches
// `target` (or exceeds it, with `beyond`); the last key if none does.  Elements: visit(f) calls f(key, units) for each of this
// thread's that takes part, units being a function.
template <int C, class Visit>
__device__ Found first_key(const Group<C>& g, uint32_t klo, uint32_t khi, u64 target, bool beyond, Visit visit, u64 before = 0) {
    Found f{klo, before, 0};
    int shift = max(0, 32 - __clz(khi - klo) - kBinBits);
    if (khi == klo) shift = 0;
    while (true) {
        for (int i = threadIdx.x; i < 3 * kBins; i += blockDim.x) (&g.hist[0][0])[i] = 0;
        __syncthreads();
        visit([&](uint32_t key, auto units) {
            if (key >= klo && key <= khi) g.add((key - klo) >> shift, units());
        });
        const uint32_t b = g.reach(f, target, beyond);
        klo += b << shift;
        khi = min(khi, klo + ((1u << shift) - 1));
        f.key = klo;
        if (shift == 0) return f;
        shift = max(0, shift - kBinBits);
    }
}

// Smallest of a value that every thread of the group has; slot as for Group::total.
template <int C>
__device__ uint32_t group_min(const Group<C>& g, uint32_t v, int slot) {
    v = __reduce_min_sync(0xffffffffu, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) g.scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    for (int w = 0; w < (int)blockDim.x / 32; ++w) v = min(v, (uint32_t)g.scratch[w]);
    if constexpr (C > 1) {
        if (threadIdx.x == 0) g.scratch[32 + slot] = v;
        g.sync();
        for (int r = 0; r < C; ++r) v = min(v, (uint32_t)*cg::this_cluster().map_shared_rank(g.scratch + 32 + slot, r));
    }
    return v;
}

// A CTA's elements of one bin, by their place in its shared memory: looking at them again costs little.
constexpr int kFew = 1024;
struct Few {
    uint16_t* at;
    uint32_t* count;  // may pass kFew: then all of the CTA's elements have to be looked at
    const float* xs;
    uint32_t i0;      // index of the first
    __device__ __forceinline__ void add(uint32_t index) const {
        const uint32_t j = atomicAdd(count, 1u);
        if (j < kFew) at[j] = (uint16_t)(index - i0);
    }
    template <class Each, class F>
    __device__ __forceinline__ void each(Each all, F f) const {
        const uint32_t n = *count;
        if (n > kFew) return all(f);
        for (uint32_t j = threadIdx.x; j < n; j += blockDim.x) f(xs[at[j]], i0 + at[j]);
    }
};

struct Cut {  // the last kept token: its key, and its index among equals
    uint32_t key, index;
    __device__ __forceinline__ bool keeps(uint32_t k, uint32_t i) const { return k < key || (k == key && i <= index); }
};

// top_k's and top_p's cut of a row whose elements the group holds: each(f) calls f(logit, index) for this thread's, `have` are
// listed in all.  whole: the weight of all tokens.  Elements below `bound` may be missing; false: they are needed.
template <int C, class Each>
__device__ bool find_cut(const Group<C>& g, const Params& p, const Rule& r, u64 have, u64 whole, float bound, float lowest, Each each, Cut& cut,
                         const Few& few = Few{}) {
    cut = {0xffffffffu, 0xffffffffu};
    auto one = [] { return 1ull; };
    // the last of `n` among the equal ones at a key
    auto cut_ties = [&](uint32_t key, u64 n) {
        return first_key<C>(g, 0, p.vocab - 1, n, false, [&](auto f) {
            each([&](float x, uint32_t i) { if (order_key(x) == key && cut.keeps(key, i)) f(i, one); });
        }).key;
    };
    const uint32_t first = order_key(g.weight.top), last = order_key(lowest);
    if (r.by_k) {
        if (have > (u64)r.k) {
            const Found f = first_key<C>(g, first, last, r.k, false, [&](auto f) { each([&](float x, uint32_t) { f(order_key(x), one); }); });
            if (!(key_logit(f.key) >= bound)) return false;
            const u64 n = r.k - f.before;
            const uint32_t index = n < f.at ? cut_ties(f.key, n) : 0xffffffffu;
            cut = {f.key, index};
        } else if (bound > -INFINITY) {
            return false;
        }
    }
    if (r.by_p) {
        u64 mass = whole;
        if (r.by_k) mass = g.total([&] { u64 s = 0; each([&](float x, uint32_t i) { if (cut.keeps(order_key(x), i)) s += to_units(g.weight(x)); }); return s; }(), 1);
        const u64 target = min(max((u64)ceil(r.p * (double)mass), 1ull), mass);
        Found f{first, 0, 0};
        const float top = g.weight.top, range = top - fmaxf(g.weight.low, lowest), per = (float)kBins / range;
        if (C > 1 && range > 0.f && range < INFINITY && per < INFINITY) {
            // first by distance from the largest: a row's bulk spreads over these bins, where keys' leading bits would not part it
            auto bin = [&](float x) { return min((uint32_t)((top - x) * per), (uint32_t)kBins - 1); };
            g.clear();
            each([&](float x, uint32_t i) { if (x >= g.weight.low && cut.keeps(order_key(x), i)) g.add(bin(x), to_units(g.weight(x))); });
            const uint32_t b = g.reach(f, target, false);
            if (threadIdx.x == 0) *few.count = 0;
            __syncthreads();
            uint32_t lo = 0xffffffffu, hi = 0;
            each([&](float x, uint32_t i) {
                if (!(x >= g.weight.low) || bin(x) != b) return;
                const uint32_t k = order_key(x);
                if (cut.keeps(k, i)) { lo = min(lo, k); hi = max(hi, k); few.add(i); }
            });
            lo = group_min(g, lo, 2);  // (with barriers: the list is complete)
            hi = ~group_min(g, ~hi, 3);
            f = first_key<C>(g, lo, hi, target, false, [&](auto f) {
                few.each(each, [&](float x, uint32_t i) { if (cut.keeps(order_key(x), i)) f(order_key(x), [&] { return to_units(g.weight(x)); }); });
            }, f.before);
        } else {
            f = first_key<C>(g, first, last, target, false, [&](auto f) {
                each([&](float x, uint32_t i) { if (cut.keeps(order_key(x), i)) f(order_key(x), [&] { return to_units(g.weight(x)); }); });
            });
        }
        if (f.before + f.at < target) {          // not reached:
            if (!r.by_k && bound > -INFINITY) return false;  // among those listed,
            if (!r.by_k) return true;                        // or by the few units that the parts' sums were rounded by
        }
        if (!(key_logit(f.key) >= bound)) return false;
        const u64 each_one = to_units(g.weight(key_logit(f.key))), n = (target - f.before + each_one - 1) / each_one;
        const uint32_t index = n < f.at / each_one ? cut_ties(f.key, n) : f.key == cut.key ? cut.index : 0xffffffffu;
        cut = {f.key, index};
    }
    return !(r.by_m && !r.by_k && !r.by_p && bound > -INFINITY && g.weight(bound) >= r.m);
}

__device__ __forceinline__ void answer(const Params& p, int row, int token, float prob, int kept) {
    p.tokens[row] = token;
    if (p.probs) p.probs[row] = prob;
    if (p.kept) p.kept[row] = kept;
}

// Sum over the CTA's threads before this one, and all of it in `all`.
__device__ __forceinline__ u64 prefix(u64 v, u64* scratch, u64& all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 run = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 t = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += t;
    }
    __syncthreads();
    if (lane == 31) scratch[warp] = run;
    __syncthreads();
    const u64 part = lane < kPickThreads / 32 ? scratch[lane] : 0;
    u64 upto = part;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
        const u64 t = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += t;
    }
    all = __shfl_sync(0xffffffffu, upto, kPickThreads / 32 - 1);
    const u64 before = __shfl_sync(0xffffffffu, upto - part, warp);
    return before + run - v;
}

// ---- pick ---------------------------------------------------------------------------------------------------------------
struct PickSmem {
    uint32_t hist[3][kBins];
    u64 scratch[64];
    double tab[kTable];
    float x[kList];
    uint32_t index[kList];
};
enum Outcome { kDone, kTooMany, kNeedsMore };

// A row of which one histogram's bins leave at most 512 elements to look at.
__device__ Outcome pick_few(const Group<1>& g, PickSmem& s, const Params& p, int row, const Rule& r, int have, u64 whole, float bound, float lowest) {
    const int tid = threadIdx.x, lane = tid & 31;
    const uint32_t first = order_key(g.weight.top), last = order_key(lowest);
    uint32_t keep_to = last;  // key of the last element that may matter
    bool by_p_late = false;   // top_p's cut lies behind min_p's
    if (r.by_k ? have > r.k : r.by_p) {
        const int shift = max(0, 32 - __clz(last - first) - kBinBits);
        const u64 target = r.by_k ? (u64)r.k : min(max((u64)ceil(r.p * (double)whole), 1ull), whole);
        g.clear();
        for (int i = tid; i < have; i += kPickThreads)
            if (s.x[i] > -INFINITY) {
                const uint32_t b = (order_key(s.x[i]) - first) >> shift;
                if (r.by_k) atomicAdd(&g.hist[0][b], 1u);
                else g.add(b, to_units(g.weight(s.x[i])));
            }
        Found f{first, 0, 0};
        const uint32_t b = g.reach(f, target, false);
        if (f.before + f.at < target) {  // top_p reaches beyond the list; min_p may still cut within it
            if (bound > -INFINITY && !(by_p_late = r.by_m && !(g.weight(bound) >= r.m))) return kNeedsMore;
        } else {
            keep_to = min(last, first + (b << shift) + ((1u << shift) - 1));
        }
    } else if (r.by_k && bound > -INFINITY) {
        return kNeedsMore;
    }
    const bool by_m_alone = r.by_m && !r.by_k && (!r.by_p || by_p_late);
    if (by_m_alone && bound > -INFINITY && g.weight(bound) >= r.m) return kNeedsMore;
    // what is left, side by side in the histogram's place
    u64* list = reinterpret_cast<u64*>(&g.hist[0][0]);
    int* count = reinterpret_cast<int*>(g.scratch + 48);
    __syncthreads();
    if (tid == 0) *count = 0;
    __syncthreads();
    uint32_t takes = 0;  // bit per round: this thread's element is among them
    int upto = 0, warp_total = 0;
    static_assert(kList <= 32 * kPickThreads, "a bit a round");
    for (int i0 = 0, round = 0; i0 < have; i0 += kPickThreads, ++round) {
        const int i = i0 + tid;
        const float x = i < have ? s.x[i] : -INFINITY;
        const bool take = x > -INFINITY && order_key(x) <= keep_to && (!by_m_alone || g.weight(x) >= r.m);
        if (take) takes |= 1u << round;
        warp_total += __popc(__ballot_sync(0xffffffffu, take));
    }
    if (lane == 0 && warp_total) upto = atomicAdd(count, warp_total);
    upto = __shfl_sync(0xffffffffu, upto, 0);
    for (int i0 = 0, round = 0; i0 < have; i0 += kPickThreads, ++round) {
        const bool take = (takes >> round) & 1;
        const uint32_t b = __ballot_sync(0xffffffffu, take);
        const int at = upto + __popc(b & ((1u << lane) - 1));
        if (take && at < kPickThreads) list[at] = (u64)order_key(s.x[i0 + tid]) << 32 | s.index[i0 + tid];
        upto += __popc(b);
    }
    __syncthreads();
    const int n = *count;
    if (n > kPickThreads) return kTooMany;
    u64 *weights = list + kPickThreads, all;
    const u64 v = tid < n ? list[tid] : ~0ull;
    const float x = key_logit((uint32_t)(v >> 32));
    const double w = tid < n ? g.weight(x) : 0.0;
    const u64 units = tid < n ? to_units(w) : 0;
    weights[tid] = units;
    __syncthreads();
    // rank of this thread's element and the weight ahead of it, by looking at every other one
    int rank = 0;
    u64 before = 0;
    if (tid < (n + 31) / 32 * 32) {
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
            const bool ahead = list[j] < v;
            rank += ahead;
            before += ahead ? weights[j] : 0;
        }
    }
    // the lowest kept logit, and whether the list is sure to hold all above it
    auto sure = [&](bool kept) { return !(bound > -INFINITY) || !__syncthreads_or(kept && !(x >= bound)); };
    bool kept = tid < n && (!r.by_k || rank < r.k);
    if (r.by_k && !sure(kept)) return kNeedsMore;
    if (r.by_p && !by_p_late) {
        u64 mass = whole;
        if (r.by_k) prefix(kept ? units : 0, g.scratch, mass);
        const u64 target = min(max((u64)ceil(r.p * (double)mass), 1ull), mass);
        kept = kept && before < target;
        if (!sure(kept)) return kNeedsMore;
    }
    if (r.by_m) kept = kept && w >= r.m;
    const int number = __syncthreads_count(kept);
    u64 sum;
    const int slot = (int)prefix(kept ? 1 : 0, g.scratch, all);
    prefix(kept ? units : 0, g.scratch, sum);
    const u64 goal = min((u64)((double)r.u * (double)sum), sum - 1);
    // the kept ones: the weight of those with lower indices
    __syncthreads();
    if (kept) list[slot] = (u64)(uint32_t)v << 32 | tid;
    __syncthreads();
    if (tid < number) {
        const u64 me = list[tid], mine = weights[me & 511];
        u64 at = 0;
#pragma unroll 4
        for (int j = 0; j < number; ++j) {
            const u64 other = list[j];
            if (other < me) at += weights[other & 511];
        }
        if (at <= goal && at + mine > goal) answer(p, row, (int)(me >> 32), (float)((double)mine / (double)sum), number);
    }
    return kDone;
}

// `direct`: the vocabulary fits the list and there was no scan.
__global__ void __launch_bounds__(kPickThreads) pick_kernel(const Params p, int direct) {
    extern __shared__ __align__(16) unsigned char raw[];
    PickSmem& s = *reinterpret_cast<PickSmem*>(raw);
    const int row = blockIdx.x, tid = threadIdx.x;
    fill_table(s.tab);
    pdl_wait();
    pdl_launch_dependents();
    const Rule r = rule_of(p, row);
    const ChunkHead* heads = p.heads + (long long)row * p.chunks;
    const long long base = row * p.stride;
    static_assert(NEON_SAMPLER_MAX_VOCAB <= kChunk * kPickThreads, "a thread takes a head");
    static_assert(NEON_SAMPLER_MAX_VOCAB / kChunk <= kBins, "the histogram holds the chunks' list lengths");
    // the largest logit, the highest of the bounds, and a bound of all that is listed
    float top = -INFINITY, bound = -INFINITY, low = INFINITY;
    ChunkHead mine{-INFINITY, -INFINITY, 0, 0, 0.0, kRelative, 0};
    if (direct) {
        for (int i = tid; i < p.vocab; i += kPickThreads) {
            s.x[i] = load1(p, base + i);
            s.index[i] = i;
            top = fmaxf(top, s.x[i]);
        }
        low = kLowest;
    } else if (tid < p.chunks) {
        mine = heads[tid];
        top = mine.max;
        bound = mine.bound;
        if (mine.listed) low = fmaxf(mine.bound, kLowest);
    }
    float* fs = reinterpret_cast<float*>(s.scratch);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        bound = fmaxf(bound, __shfl_xor_sync(0xffffffffu, bound, o));
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    }
    if ((tid & 31) == 0) { fs[tid >> 5] = top; fs[32 + (tid >> 5)] = bound; fs[64 + (tid >> 5)] = low; }
    __syncthreads();
    top = fs[tid & 15];
    bound = fs[32 + (tid & 15)];
    low = fs[64 + (tid & 15)];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        bound = fmaxf(bound, __shfl_xor_sync(0xffffffffu, bound, o));
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    }
    __syncthreads();
    static_assert(kPickThreads == 512, "sixteen warps");
    if (tid == 0 && p.left) p.left[row] = 0;
    if (top == -INFINITY) {
        if (tid == 0) answer(p, row, -1, 0.f, 0);
        return;
    }
    const Weigher weight(top, r.c, s.tab);
    if (!direct && (r.greedy || !r.filters())) {
        // weights of the chunks, in order; greedily: the first chunk that has the maximum
        u64 w = r.greedy ? (u64)(mine.max == top) : 0ull, all;
        if (!r.greedy) w = chunk_units(mine, weight);
        const u64 run = prefix(w, s.scratch, all);
        const u64 target = r.greedy ? 0 : min((u64)((double)r.u * (double)all), all - 1);
        if (run <= target && run + w > target) {
            s.scratch[40] = tid;
            s.scratch[41] = target - run;
        }
        u64 n_valid;
        prefix(mine.valid, s.scratch, n_valid);
        const int i0 = (int)s.scratch[40] * kChunk;
        const u64 rest = s.scratch[41];
        // the token in it: two neighbouring elements a thread
        constexpr int kEach = kChunk / kPickThreads;
        u64 e[kEach], part = 0, have;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int i = i0 + tid * kEach + j;
            const float x = i < p.vocab ? load1(p, base + i) : -INFINITY;
            e[j] = r.greedy ? (u64)(x == top) : to_units(weight(x));
            part += e[j];
        }
        u64 at = prefix(part, s.scratch, have);
        const u64 goal = min(rest, have ? have - 1 : 0);  // the chunk's sum may differ from its elements' by their rounding
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            if (at <= goal && at + e[j] > goal)
                answer(p, row, i0 + tid * kEach + j, r.greedy ? 1.f : (float)((double)e[j] / (double)all), r.greedy ? 1 : (int)n_valid);
            at += e[j];
        }
        return;
    }
    const Group<1> g{s.hist, s.scratch, weight};
    auto one = [] { return 1ull; };
    if (r.greedy) {
        const Found f = first_key<1>(g, 0, p.vocab - 1, 0, true, [&](auto f) {
            for (int i = tid; i < p.vocab; i += kPickThreads) if (s.x[i] == top) f((uint32_t)i, one);
        });
        if (tid == 0) answer(p, row, (int)f.key, 1.f, 1);
        return;
    }
    u64 n64 = p.vocab, whole = 0;
    bool fits = true;
    if (direct) {
        if (r.by_p && !r.by_k) {
            u64 sum = 0;
            for (int i = tid; i < p.vocab; i += kPickThreads) sum += to_units(weight(s.x[i]));
            whole = g.total(sum, 0);
        }
    } else {
        // the listed elements, side by side
        const uint32_t at = (uint32_t)prefix(mine.listed, s.scratch, n64);
        prefix(chunk_units(mine, weight), s.scratch, whole);
        // (a bound above the largest: too many tokens share that for its stretch to list them, whatever other stretches list)
        fits = n64 > 0 && n64 <= kList && !(bound > top);
        if (fits) {
            uint32_t* starts = &s.hist[0][0];  // where each chunk's entries go, and how many they are
            if (tid < p.chunks) {
                starts[tid] = at;
                starts[kBins + tid] = (uint32_t)mine.listed;
            }
            __syncthreads();
            const uint2* lists = p.entries + (long long)row * p.chunks * kSlots;
            // a half warp per list, sixteen lists a round: most fit two loads
            const int half = tid >> 4, slot = tid & 15;
#pragma unroll 2
            for (int c = half; c < p.chunks; c += kPickThreads / 16) {
                const int to = starts[c], count = starts[kBins + c];
                uint2 v[2];
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (16 * h + slot < count) v[h] = lists[c * kSlots + 16 * h + slot];
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (16 * h + slot < count) {
                        s.x[to + 16 * h + slot] = __uint_as_float(v[h].x);
                        s.index[to + 16 * h + slot] = v[h].y;
                    }
                for (int e = 32 + slot; e < count; e += 16) {
                    const uint2 u = lists[c * kSlots + e];
                    s.x[to + e] = __uint_as_float(u.x);
                    s.index[to + e] = u.y;
                }
            }
            __syncthreads();
        }
    }
    if (fits) {
        const int n = (int)n64;
        Outcome outcome = r.filters() ? pick_few(g, s, p, row, r, n, whole, bound, low) : kTooMany;
        if (outcome == kTooMany) {
            auto each = [&](auto f) {
                for (int i = tid; i < n; i += kPickThreads)
                    if (s.x[i] > -INFINITY) f(s.x[i], s.index[i]);
            };
            Cut cut;
            const u64 have = direct && r.by_k ? g.total([&] { u64 c = 0; each([&](float, uint32_t) { ++c; }); return c; }(), 1) : n64;
            outcome = find_cut<1>(g, p, r, have, whole, bound, low, each, cut) ? kDone : kNeedsMore;
            if (outcome == kDone) {
                auto drawn = [&](float x, uint32_t i) { return cut.keeps(order_key(x), i) && (!r.by_m || weight(x) >= r.m); };
                u64 sum = 0, count = 0;
                each([&](float x, uint32_t i) { if (drawn(x, i)) { sum += to_units(weight(x)); ++count; } });
                sum = g.total(sum, 3);
                count = g.total(count, 4);
                const u64 goal = min((u64)((double)r.u * (double)sum), sum - 1);
                const Found f = first_key<1>(g, 0, p.vocab - 1, goal, true, [&](auto f) {
                    each([&](float x, uint32_t i) { if (drawn(x, i)) f(i, [&] { return to_units(weight(x)); }); });
                });
                if (tid == 0) answer(p, row, (int)f.key, (float)((double)f.at / (double)sum), (int)count);
            }
        }
        fits = outcome == kDone;
    }
    if (!fits && tid == 0) p.left[row] = 1;
}

// ---- whole ----------------------------------------------------------------------------------------------------------------
struct WholeSmem {
    uint32_t hist[3][kBins];
    u64 scratch[64];
    u64 parts[2][kPickThreads / 32];  // weights and counts of the warps' stretches
    uint16_t few[kFew];
    uint32_t n_few[4];
    double tab[kTable];
};

// Logits of a CTA: a whole number of four.
__host__ __device__ inline int whole_share(int vocab) { return (vocab + 4 * kClusterCtas - 1) / (4 * kClusterCtas) * 4; }

// Rows that pick left, one after the other on each cluster.  A CTA keeps its share of the row in shared memory, a warp's
// stretch of it is contiguous.
__global__ void __cluster_dims__(kClusterCtas, 1, 1) __launch_bounds__(kPickThreads) whole_kernel(const Params p) {
    extern __shared__ __align__(16) unsigned char raw[];
    WholeSmem& s = *reinterpret_cast<WholeSmem*>(raw);
    float* xs = reinterpret_cast<float*>(raw + sizeof(WholeSmem));
    constexpr int kWarps = kPickThreads / 32;
    const cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int share = whole_share(p.vocab), i0 = min(rank * share, p.vocab), n = min(share, p.vocab - i0);
    const int stretch = (share + kWarps - 1) / kWarps, w0 = min(warp * stretch, n), w1 = min(w0 + stretch, n);
    fill_table(s.tab);
    pdl_wait();
    for (int row = blockIdx.x / kClusterCtas; row < p.batch; row += gridDim.x / kClusterCtas) {
        if (!p.left[row]) continue;  // the same for the whole cluster
        const Rule r = rule_of(p, row);
        const ChunkHead* heads = p.heads + (long long)row * p.chunks;
        __syncthreads();
        float top = -INFINITY;
        const long long base = row * p.stride + i0;
        if (p.dtype == 0 && (reinterpret_cast<uintptr_t>(p.logits) + base * 4) % 16 == 0) {
            const float4* from = reinterpret_cast<const float4*>(static_cast<const float*>(p.logits) + base);
#pragma unroll 8
            for (int i = tid; i < n / 4; i += kPickThreads) {
                const float4 v = __ldcs(from + i);
                reinterpret_cast<float4*>(xs)[i] = make_float4(clean(v.x), clean(v.y), clean(v.z), clean(v.w));
            }
            if (tid < n % 4) xs[n / 4 * 4 + tid] = load1(p, base + n / 4 * 4 + tid);
        } else {
#pragma unroll 8
            for (int i = tid; i < n; i += kPickThreads) xs[i] = load1(p, base + i);
        }
        if (tid >= n % 4 && tid < 4 && n % 4) xs[n / 4 * 4 + tid] = -INFINITY;  // to a whole number of four
        ChunkHead mine{-INFINITY, -INFINITY, 0, 0, 0.0, kRelative, 0};
        if (tid < p.chunks) mine = heads[tid];
        top = mine.max;
        float* fs = reinterpret_cast<float*>(s.scratch);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (lane == 0) fs[warp] = top;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, fs[w]);
        __syncthreads();
        const Weigher weight(top, r.c, s.tab);
        const Group<kClusterCtas> g{s.hist, s.scratch, weight};
        u64 whole, have;
        prefix(chunk_units(mine, weight), s.scratch, whole);
        prefix(mine.valid, s.scratch, have);
        auto each = [&](auto f) {
#pragma unroll 2
            for (int i = tid; i < (n + 3) / 4; i += kPickThreads) {
                const float4 v = reinterpret_cast<const float4*>(xs)[i];
                if (v.x > -INFINITY) f(v.x, (uint32_t)(i0 + 4 * i));
                if (v.y > -INFINITY) f(v.y, (uint32_t)(i0 + 4 * i + 1));
                if (v.z > -INFINITY) f(v.z, (uint32_t)(i0 + 4 * i + 2));
                if (v.w > -INFINITY) f(v.w, (uint32_t)(i0 + 4 * i + 3));
            }
        };
        Cut cut;
        find_cut<kClusterCtas>(g, p, r, have, whole, -INFINITY, kLowest, each, cut, Few{s.few, s.n_few, xs, (uint32_t)i0});
        // by index: the warps' stretches, then the token in one of them
        auto units = [&](int i) -> u64 {
            const float x = xs[i];
            if (!(x > -INFINITY) || !cut.keeps(order_key(x), i0 + i)) return 0;
            const double w = weight(x);
            return !r.by_m || w >= r.m ? to_units(w) : 0;
        };
        u64 sum = 0, count = 0;
        const float cut_logit = cut.key == 0xffffffffu ? kLowest : key_logit(cut.key);
#pragma unroll 4
        for (int i = w0 + lane; i < w1; i += 32) {
            const float x = xs[i];
            if (!(x >= cut_logit) || !cut.keeps(order_key(x), i0 + i)) continue;
            const double w = weight(x);
            if (r.by_m && !(w >= r.m)) continue;
            sum += to_units(w);
            ++count;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            count += __shfl_xor_sync(0xffffffffu, count, o);
        }
        if (lane == 0) { s.parts[0][warp] = sum; s.parts[1][warp] = count; }
        cluster.sync();
        u64 part = 0, number = 0, all, kept;
        if (tid < kClusterCtas * kWarps) {
            const u64* theirs = cluster.map_shared_rank(&s.parts[0][0], tid / kWarps);
            part = theirs[tid % kWarps];
            number = theirs[kWarps + tid % kWarps];
        }
        const u64 before = prefix(part, s.scratch, all);
        const u64 goal = min((u64)((double)r.u * (double)all), all - 1);
        if (before <= goal && before + part > goal) {
            s.scratch[40] = tid;
            s.scratch[41] = goal - before;
        }
        prefix(number, s.scratch, kept);
        const int owner = (int)s.scratch[40];
        if (owner / kWarps == rank) {  // this CTA has the stretch: a few in a row to every thread
            const u64 rest = s.scratch[41];
            const int o0 = min(owner % kWarps * stretch, n), o1 = min(o0 + stretch, n), each_has = (stretch + kPickThreads - 1) / kPickThreads;
            const int t0 = min(o0 + tid * each_has, o1), t1 = min(t0 + each_has, o1);
            u64 have_units = 0, of_stretch;
            for (int i = t0; i < t1; ++i) have_units += units(i);
            u64 run = prefix(have_units, s.scratch, of_stretch);
            if (run <= rest && run + have_units > rest)
                for (int i = t0; i < t1; ++i) {
                    const u64 here = units(i);
                    if (run + here > rest) {
                        answer(p, row, i0 + i, (float)((double)here / (double)all), (int)kept);
                        break;
                    }
                    run += here;
                }
        }
        cluster.sync();  // the stretches' sums are read
    }
    cluster.sync();  // nobody leaves while others read its shared memory
}

}  // namespace sampler
}  // namespace neon
