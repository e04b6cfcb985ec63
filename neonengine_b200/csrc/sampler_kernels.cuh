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
// Cuts and token are found in the same way: "the first key at which a running sum (of ones or of weights) reaches a
// target" by histograms over ten bits of the key at a time - the key being the logit in descending order, or the index.
// Weights are integers of 2^-43 of the largest, so that sums depend on no order; a histogram keeps them as three words
// of 15 bits each per element, which shared memory can add atomically.
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
constexpr int kPickThreads = 512, kScanWarps = 4;
constexpr int kBins = 1024, kBinBits = 10;
constexpr int kWeightBits = 43;       // weights are multiples of 2^-43; a row's sum stays below 2^63
constexpr double kUnit = 8796093022208.0;  // 2^43
constexpr int kClusterCtas = 8;
constexpr float kLowest = -3.402823466e38f;  // the lowest that can be drawn
typedef unsigned long long u64;

struct ChunkHead {   // what a warp of the scan leaves about its logits
    float max, bound;   // largest; every logit >= bound is listed
    int listed, valid;  // entries; logits above -infinity
    double weight;      // relative to max
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
    double c;  // log2(e) / temperature
    int k;
    double p, m;
    float u;
    __device__ bool filters() const { return by_k || by_p || by_m; }
};
__device__ __forceinline__ Rule rule_of(const Params& p, int row) {
    Rule r;
    const float t = p.temperature ? p.temperature[row] : 1.f;
    r.greedy = !(t > 0.f);
    r.c = r.greedy ? 1.0 : 1.4426950408889634074 / (double)t;
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

__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : x + 0.f; }  // NaN is -infinity, -0 is 0
__device__ __forceinline__ float load1(const Params& p, long long i) {
    float x;
    if (p.dtype == 0) x = __ldg(static_cast<const float*>(p.logits) + i);
    else if (p.dtype == 1) x = __bfloat162float(static_cast<const __nv_bfloat16*>(p.logits)[i]);
    else x = __half2float(static_cast<const __half*>(p.logits)[i]);
    return clean(x);
}
// ascending keys for descending logits
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? b : ~b & 0x7fffffffu;
}
__device__ __forceinline__ float key_logit(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k : ~k & 0x7fffffffu); }

// 2^(j/128), j < 128
__device__ __forceinline__ void fill_table(double* tab) {
    for (int j = threadIdx.x; j < 128; j += blockDim.x) tab[j] = exp2(j / 128.0);
}
// exp of (x - top) / temperature, to 3e-12: a table of 2^(j/128) times a cubic on the remainder, whose next term is
// (ln 2 / 256)^4 / 24 = 2.2e-12
__device__ __forceinline__ double weight_of(float x, float top, double c, const double* tab) {
    const double kMagic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low word is the rounded integer
    if (x == top) return 1.0;
    const double t = ((double)x - (double)top) * c;
    if (!(t > -64.0)) return 0.0;
    const double kd = fma(t, 128.0, kMagic);
    const int k = __double2loint(kd);
    const double r = fma(kd - kMagic, -1.0 / 128.0, t);
    const double q = r * fma(r, fma(r, 0.055504108664821580, 0.24022650695910071), 0.69314718055994531);
    const double w = fma(tab[k & 127], q, tab[k & 127]);
    return __hiloint2double(__double2hiint(w) + ((k >> 7) << 20), __double2loint(w));
}
__device__ __forceinline__ u64 to_units(double w) {  // w <= 2^9, in 2^-43, rounded
    return (u64)(__double_as_longlong(fma(w, kUnit, 4503599627370496.0)) & 0xfffffffffffffll);
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

template <int DT>
__global__ void __launch_bounds__(kScanWarps * 32) scan_kernel(const Params p) {
    __shared__ double tab[128];
    const int lane = threadIdx.x & 31;
    pdl_wait();
    pdl_launch_dependents();
    fill_table(tab);
    __syncthreads();
    const long long task = (long long)blockIdx.x * kScanWarps + threadIdx.x / 32;
    const int row = (int)(task / p.chunks), chunk = (int)(task % p.chunks);
    if (row >= p.batch) return;
    const int i0 = chunk * kChunk, n = min(kChunk, p.vocab - i0);
    const long long base = row * p.stride + i0;
    float x[32];  // element 4 * (32 v + lane) + c is x[4 v + c]
    constexpr int kSize = DT == 0 ? 4 : 2;
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
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = clean(x[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const int e = 4 * (32 * (i / 4) + lane) + i % 4;
            x[i] = e < n ? load1(p, base + e) : -INFINITY;
        }
    }
    float top = x[0];
    int valid = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        top = fmaxf(top, x[i]);
        valid += x[i] > -INFINITY;
    }
    const Rule r = rule_of(p, row);
    ChunkHead head;
    float bound = INFINITY;
    if (!r.greedy && r.filters()) bound = __shfl_sync(0xffffffffu, warp_sorted(top), p.rank - 1);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    head.max = top;
    head.valid = __reduce_add_sync(0xffffffffu, valid);
    // the whole row's weight counts where nothing but top_p cuts it
    double sum = 0.0;
    if (!r.greedy && !r.by_k && (r.by_p || !r.by_m) && top > -INFINITY) {
#pragma unroll
        for (int i = 0; i < 32; ++i) sum += weight_of(x[i], top, r.c, tab);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    head.weight = sum;
    // the list
    int listed = 0;
    if (!r.greedy && r.filters()) {
        bound = fmaxf(bound, kLowest);  // -infinity is not listed
        int count = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) count += x[i] >= bound;
        if (__reduce_add_sync(0xffffffffu, count) > kSlots) {  // many equal ones: those above
            bound = bound < INFINITY ? nextafterf(bound, INFINITY) : bound;
            count = 0;
#pragma unroll
            for (int i = 0; i < 32; ++i) count += x[i] >= bound;
            if (__reduce_add_sync(0xffffffffu, count) > kSlots) bound = __int_as_float(0x7fc00000);  // none: nothing is >= NaN
        }
        uint2* list = p.entries + ((long long)row * p.chunks + chunk) * kSlots;
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
    if (lane == 0) p.heads[(long long)row * p.chunks + chunk] = head;
}

// ---- cuts and token among elements in shared memory ---------------------------------------------------------------------
// The elements of a row that CTAs of a group hold, and the histogram they share.
template <int C>
struct Group {
    uint32_t (*hist)[kBins];  // three words of a bin's sum
    u64* scratch;             // [64]
    const double* tab;
    float top;
    double c;
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
};

struct Found {
    uint32_t key;
    u64 before, at;  // sum of the keys before it, sum of the key itself
};

// The first key, ascending from klo to khi, at which the running sum reaches `target` (or exceeds it, with `beyond`);
// there has to be one.  Elements: visit(f) calls f(key, units) for each of this thread's that takes part.
template <int C, class Visit>
__device__ Found first_key(const Group<C>& g, uint32_t klo, uint32_t khi, u64 target, bool beyond, Visit visit) {
    Found f{klo, 0, 0};
    int shift = max(0, 32 - __clz(khi - klo) - kBinBits);
    if (khi == klo) shift = 0;
    while (true) {
        for (int i = threadIdx.x; i < 3 * kBins; i += blockDim.x) (&g.hist[0][0])[i] = 0;
        __syncthreads();
        visit([&](uint32_t key, u64 units) {
            if (key < klo || key > khi) return;
            const uint32_t b = (key - klo) >> shift;
            atomicAdd(&g.hist[0][b], (uint32_t)units & 0x7fffu);
            if (units >> 15) {
                atomicAdd(&g.hist[1][b], (uint32_t)(units >> 15) & 0x7fffu);
                if (units >> 30) atomicAdd(&g.hist[2][b], (uint32_t)(units >> 30));
            }
        });
        g.sync();
        // two neighbouring bins a thread, their running sums
        constexpr int kPer = kBins / kPickThreads;
        u64 bin[kPer], mine = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int b = threadIdx.x * kPer + j;
            bin[j] = 0;
            for (int r = 0; r < C; ++r) {
                const uint32_t* h = C == 1 ? &g.hist[0][0] : cg::this_cluster().map_shared_rank(&g.hist[0][0], r);
                bin[j] += (u64)h[b] + ((u64)h[kBins + b] << 15) + ((u64)h[2 * kBins + b] << 30);
            }
            mine += bin[j];
        }
        u64 run = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 v = __shfl_up_sync(0xffffffffu, run, o);
            if ((threadIdx.x & 31) >= o) run += v;
        }
        if ((threadIdx.x & 31) == 31) g.scratch[threadIdx.x >> 5] = run;
        __syncthreads();
        u64 start = f.before + run - mine;
        for (int w = 0; w < (int)(threadIdx.x >> 5); ++w) start += g.scratch[w];
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const u64 end = start + bin[j];
            const bool before_it = beyond ? start <= target : start < target, reached = beyond ? end > target : end >= target;
            if (before_it && reached && bin[j]) {  // one bin of all
                g.scratch[16] = threadIdx.x * kPer + j;
                g.scratch[17] = start;
                g.scratch[18] = bin[j];
            }
            start = end;
        }
        g.sync();  // also: everybody has read everybody's histogram
        const uint32_t b = (uint32_t)g.scratch[16];
        f.before = g.scratch[17];
        f.at = g.scratch[18];
        klo += b << shift;
        khi = min(khi, klo + ((1u << shift) - 1));
        f.key = klo;
        __syncthreads();
        if (shift == 0) return f;
        shift = max(0, shift - kBinBits);
    }
}

// Cuts and token of a row whose elements the group holds: each(f) calls f(logit, index) for this thread's.  whole_weight: of
// all tokens (used where top_p is the first cut).  bound: elements below it may be missing.  False: they are needed.
template <int C, class Each>
__device__ bool draw_row(const Group<C>& g, const Params& p, int row, const Rule& r, u64 whole_weight, float bound, float lowest, Each each) {
    uint32_t cut_key = 0xffffffffu, cut_index = 0xffffffffu;  // the last kept one
    auto kept = [&](float x, uint32_t i) {
        const uint32_t k = order_key(x);
        return k < cut_key || (k == cut_key && i <= cut_index);
    };
    auto units = [&](float x) { return to_units(weight_of(x, g.top, g.c, g.tab)); };
    // the last of `n` among the equal ones at a key
    auto cut_ties = [&](uint32_t key, u64 n) {
        return first_key<C>(g, 0, p.vocab - 1, n, false, [&](auto f) {
            each([&](float x, uint32_t i) { if (order_key(x) == key && kept(x, i)) f(i, 1); });
        }).key;
    };
    const uint32_t first = order_key(g.top), last = order_key(lowest);
    if (r.by_k) {
        const u64 have = g.total([&] { u64 n = 0; each([&](float, uint32_t) { ++n; }); return n; }(), 0);
        if (have > (u64)r.k) {
            const Found f = first_key<C>(g, first, last, r.k, false, [&](auto f) { each([&](float x, uint32_t) { f(order_key(x), 1); }); });
            if (!(key_logit(f.key) >= bound)) return false;
            const u64 n = r.k - f.before;
            const uint32_t ci = n < f.at ? cut_ties(f.key, n) : 0xffffffffu;
            cut_key = f.key;
            cut_index = ci;
        } else if (bound > -INFINITY) {
            return false;
        }
    }
    if (r.by_p) {
        u64 mass = whole_weight;
        if (r.by_k || whole_weight == 0)
            mass = g.total([&] { u64 s = 0; each([&](float x, uint32_t i) { if (kept(x, i)) s += units(x); }); return s; }(), 1);
        const u64 target = min(max((u64)ceil(r.p * (double)mass), 1ull), mass);
        bool all = false;
        if (!r.by_k && bound > -INFINITY) {  // does the list reach that far?
            const u64 have = g.total([&] { u64 s = 0; each([&](float x, uint32_t) { s += units(x); }); return s; }(), 2);
            if (have < target) return false;
        } else if (!r.by_k) {
            // rounding of the parts may leave the sum a few units short of `mass`
            const u64 have = g.total([&] { u64 s = 0; each([&](float x, uint32_t) { s += units(x); }); return s; }(), 2);
            all = have < target;
        }
        if (!all) {
            const Found f = first_key<C>(g, first, last, target, false, [&](auto f) {
                each([&](float x, uint32_t i) { if (kept(x, i)) f(order_key(x), units(x)); });
            });
            if (!(key_logit(f.key) >= bound)) return false;
            const u64 one = units(key_logit(f.key)), n = one ? (target - f.before + one - 1) / one : 1, ties = one ? f.at / one : 1;
            const uint32_t ci = n < ties ? cut_ties(f.key, n) : f.key == cut_key ? cut_index : 0xffffffffu;
            cut_key = f.key;
            cut_index = ci;
        }
    }
    if (r.by_m && !r.by_k && !r.by_p && bound > -INFINITY && !(weight_of(bound, g.top, g.c, g.tab) < r.m)) return false;
    auto drawn = [&](float x, uint32_t i) { return kept(x, i) && (!r.by_m || weight_of(x, g.top, g.c, g.tab) >= r.m); };
    u64 s = 0, n = 0;
    each([&](float x, uint32_t i) { if (drawn(x, i)) { s += units(x); ++n; } });
    s = g.total(s, 3);
    n = g.total(n, 4);
    const u64 target = min((u64)((double)r.u * (double)s), s - 1);
    const Found f = first_key<C>(g, 0, p.vocab - 1, target, true, [&](auto f) {
        each([&](float x, uint32_t i) { if (drawn(x, i)) f(i, units(x)); });
    });
    if (threadIdx.x == 0 && (C == 1 || cg::this_cluster().block_rank() == 0)) {
        p.tokens[row] = (int)f.key;
        if (p.probs) p.probs[row] = (float)((double)f.at / (double)s);
        if (p.kept) p.kept[row] = (int)n;
    }
    return true;
}

// ---- pick ---------------------------------------------------------------------------------------------------------------
struct PickSmem {
    uint32_t hist[3][kBins];
    u64 scratch[64];
    double tab[128];
    float x[kList];
    uint32_t index[kList];
};

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
    u64 before = 0;
    all = 0;
    for (int w = 0; w < (int)blockDim.x / 32; ++w) {
        if (w < warp) before += scratch[w];
        all += scratch[w];
    }
    return before + run - v;
}

// `direct`: the vocabulary fits the list and there was no scan.
__global__ void __launch_bounds__(kPickThreads) pick_kernel(const Params p, int direct) {
    extern __shared__ __align__(16) unsigned char raw[];
    PickSmem& s = *reinterpret_cast<PickSmem*>(raw);
    const int row = blockIdx.x, tid = threadIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    fill_table(s.tab);
    const Rule r = rule_of(p, row);
    const ChunkHead* heads = p.heads + (long long)row * p.chunks;
    const long long base = row * p.stride;
    static_assert(NEON_SAMPLER_MAX_VOCAB <= kChunk * kPickThreads, "a thread takes a head");
    static_assert(NEON_SAMPLER_MAX_VOCAB / kChunk <= kBins, "the histogram holds the chunks' list lengths");
    if (tid == 0 && p.left) p.left[row] = 0;
    // the largest logit, the highest of the bounds, and a bound of all that is listed
    float top = -INFINITY, bound = -INFINITY, low = INFINITY;
    ChunkHead mine{-INFINITY, -INFINITY, 0, 0, 0.0};
    if (direct) {
        for (int i = tid; i < p.vocab; i += kPickThreads) {
            s.x[i] = load1(p, base + i);
            s.index[i] = i;
            top = fmaxf(top, s.x[i]);
        }
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
    for (int w = 0; w < kPickThreads / 32; ++w) { top = fmaxf(top, fs[w]); bound = fmaxf(bound, fs[32 + w]); low = fminf(low, fs[64 + w]); }
    __syncthreads();
    auto answer = [&](int token, float prob, int kept) {
        p.tokens[row] = token;
        if (p.probs) p.probs[row] = prob;
        if (p.kept) p.kept[row] = kept;
    };
    if (top == -INFINITY) {
        if (tid == 0) answer(-1, 0.f, 0);
        return;
    }
    Group<1> g{s.hist, s.scratch, s.tab, top, r.c};
    if (direct) {
        auto each = [&](auto f) {
            for (int i = tid; i < p.vocab; i += kPickThreads)
                if (s.x[i] > -INFINITY) f(s.x[i], s.index[i]);
        };
        if (r.greedy) {
            const Found f = first_key<1>(g, 0, p.vocab - 1, 0, true, [&](auto f) { each([&](float x, uint32_t i) { if (x == top) f(i, 1); }); });
            if (tid == 0) answer((int)f.key, 1.f, 1);
            return;
        }
        draw_row<1>(g, p, row, r, 0, -INFINITY, kLowest, each);
        return;
    }
    if (r.greedy || !r.filters()) {
        // weights of the chunks, in order; greedily: the first chunk that has the maximum
        u64 w = r.greedy ? (u64)(mine.max == top) : 0ull, all;
        if (!r.greedy && mine.max > -INFINITY) w = (u64)(mine.weight * weight_of(mine.max, top, r.c, s.tab) * kUnit);
        const u64 run = prefix(w, s.scratch, all);
        const u64 target = r.greedy ? 0 : min((u64)((double)r.u * (double)all), all - 1);
        if (run <= target && run + w > target) {
            s.scratch[40] = tid;
            s.scratch[41] = target - run;
        }
        u64 n_valid;
        prefix(mine.valid, s.scratch, n_valid);
        const int chunk = (int)s.scratch[40], i0 = chunk * kChunk;
        const u64 rest = s.scratch[41];
        // the token in it: two neighbouring elements a thread
        constexpr int kEach = kChunk / kPickThreads;
        float x[kEach];
        u64 e[kEach], part = 0, have;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int i = i0 + tid * kEach + j;
            x[j] = i < p.vocab ? load1(p, base + i) : -INFINITY;
            e[j] = r.greedy ? (u64)(x[j] == top) : x[j] > -INFINITY ? to_units(weight_of(x[j], top, r.c, s.tab)) : 0;
            part += e[j];
        }
        u64 at = prefix(part, s.scratch, have);
        const u64 goal = min(rest, have ? have - 1 : 0);  // the chunk's sum may differ from its elements' by their rounding
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            if (at <= goal && at + e[j] > goal) answer(i0 + tid * kEach + j, r.greedy ? 1.f : (float)((double)e[j] / (double)all), r.greedy ? 1 : (int)n_valid);
            at += e[j];
        }
        return;
    }
    // the listed elements, side by side
    u64 n64, whole_all;
    const uint32_t at = (uint32_t)prefix(mine.listed, s.scratch, n64);
    prefix(mine.max > -INFINITY ? (u64)(mine.weight * weight_of(mine.max, top, r.c, s.tab) * kUnit) : 0ull, s.scratch, whole_all);
    const int n = (int)n64;
    bool fits = n <= kList;
    if (fits) {
        uint32_t* starts = &s.hist[0][0];  // where each chunk's entries go, and how many they are
        if (tid < p.chunks) {
            starts[tid] = at;
            starts[kBins + tid] = (uint32_t)mine.listed;
        }
        __syncthreads();
        const uint2* lists = p.entries + (long long)row * p.chunks * kSlots;
        for (int i = tid; i < p.chunks * kSlots; i += kPickThreads) {
            const int c = i / kSlots, e = i % kSlots;
            if (e < (int)starts[kBins + c]) {
                const uint2 v = lists[i];
                s.x[starts[c] + e] = __uint_as_float(v.x);
                s.index[starts[c] + e] = v.y;
            }
        }
        __syncthreads();
        auto each = [&](auto f) {
            for (int i = tid; i < n; i += kPickThreads) f(s.x[i], s.index[i]);
        };
        fits = n > 0 && draw_row<1>(g, p, row, r, whole_all, bound, low, each);
    }
    if (!fits && tid == 0) p.left[row] = 1;
}

// ---- whole ----------------------------------------------------------------------------------------------------------------
struct WholeSmem {
    uint32_t hist[3][kBins];
    u64 scratch[64];
    double tab[128];
};

// Rows that pick left, one after the other on each cluster.  A CTA keeps its share of the row in shared memory.
__global__ void __cluster_dims__(kClusterCtas, 1, 1) __launch_bounds__(kPickThreads) whole_kernel(const Params p) {
    extern __shared__ __align__(16) unsigned char raw[];
    WholeSmem& s = *reinterpret_cast<WholeSmem*>(raw);
    float* xs = reinterpret_cast<float*>(raw + sizeof(WholeSmem));
    const int rank = (int)cg::this_cluster().block_rank(), tid = threadIdx.x;
    const int share = (p.vocab + kClusterCtas - 1) / kClusterCtas, i0 = min(rank * share, p.vocab), n = min(share, p.vocab - i0);
    pdl_wait();
    fill_table(s.tab);
    for (int row = blockIdx.x / kClusterCtas; row < p.batch; row += gridDim.x / kClusterCtas) {
        if (!p.left[row]) continue;  // the same for the whole cluster
        const Rule r = rule_of(p, row);
        const ChunkHead* heads = p.heads + (long long)row * p.chunks;
        __syncthreads();
        float top = -INFINITY;
        for (int i = tid; i < n; i += kPickThreads) xs[i] = load1(p, row * p.stride + i0 + i);
        for (int c = tid; c < p.chunks; c += kPickThreads) top = fmaxf(top, heads[c].max);
        float* fs = reinterpret_cast<float*>(s.scratch);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if ((tid & 31) == 0) fs[tid >> 5] = top;
        __syncthreads();
        for (int w = 0; w < kPickThreads / 32; ++w) top = fmaxf(top, fs[w]);
        __syncthreads();
        Group<kClusterCtas> g{s.hist, s.scratch, s.tab, top, r.c};
        auto each = [&](auto f) {
            for (int i = tid; i < n; i += kPickThreads)
                if (xs[i] > -INFINITY) f(xs[i], (uint32_t)(i0 + i));
        };
        draw_row<kClusterCtas>(g, p, row, r, 0, -INFINITY, kLowest, each);
        g.sync();
    }
    cg::this_cluster().sync();  // nobody leaves while others read its shared memory
}

}  // namespace sampler
}  // namespace neon
