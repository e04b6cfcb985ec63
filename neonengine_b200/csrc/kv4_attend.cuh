// Attention over the 4-bit paged cache: few rows per key/value head (a decoding step, drafted tokens, short chunks).
//
// An item is (sequence, block of rows, key/value head): the G query heads that share the head times a few tokens, at most
// 8 * NT rows, against the 64-position steps that any of its rows sees.  All items' steps in a row are cut evenly over the
// CTAs of the grid and again over a CTA's warps, whatever the lengths are (they are device memory): a warp takes a contiguous
// run of steps and finishes the items that lie wholly in it.  Of others it leaves a partial result (maximum, sum,
// unnormalised output); the CTA folds its warps' and finishes what it has all of, merge_kernel folds the CTAs'.
//
// Per step a warp multiplies on mma.sync.m16n8k16 with positions (keys) and columns (values) as the 16 rows and the item's
// rows as the 8 columns: S^T = K Q^T, O^T += V^T P^T.  With G = 8 no row of a product is idle; tcgen05 would need 128 rows and a
// trip through tensor memory for the same few columns.  Codes become f16 by one conversion per two of them.
//   Keys keep their codes: each 32-column block has a sum of its own, and its scale is a factor of that sum (f32), so any
//   scale is exact.  Queries are f16, every row scaled by a power of two so that its largest value lies in [2^14, 2^15):
//   exact for bf16 and f16 down to 2^-28 of the largest.
//   Values: a pair of positions of one column is one f16x2 operand, multiplied by the two positions' scales relative to
//   the largest scale met so far (outputs are rescaled when it grows).  Where a step's scales lie more than 2^7 below it, its
//   values are added in f32, one position at a time (five times as long, and rare).
//   Probabilities are f16, relative to a level of their row: a group (the 64 or 32 positions weighed at once) whose largest would be
//   infinite raises it, to 2^8 below.  So a probability is rounded by 2^-12 of itself or by 2^-25, and the row's sum is 2^8 or more.  With value
//   scales 2^apart apart at most, n positions lose n * 2^(apart - 33) of the sum of weights times scales: 2^-10, once n * 2^apart is 2^23
//   (kCareful: 65536 positions of a warp's run at scales within 2^7).  From there on a group whose largest is below 1 lowers
//   the level, to 2^5 below it: then what a group loses is 2^-12 of its own, wherever the row's largest stands and whatever its value is.
//   Lowering ends where it takes the sum to 2^30; a group that needs more loses 2^-49 of the sum, and where scales lie further
//   apart than 2^24 it is added in f32.  Rescaling is off by 2^-22.
//   The softmax sum is one more product, with a row of ones.  Most steps need no exchange between lanes but one vote.
// Steps travel by bulk copies (one per page and head: a record is contiguous) into a ring per warp.
// What bounds it at G = 8: not the memory but issue slots and the conversions (two codes each, 64 lanes a clock and SM).  Measured with 64
// query and 8 key/value heads of 64: 64 sequences of 200 to 32768 positions 125 us for 476 MB, 3.8 TB/s (2.0 instructions a clock and SM;
// streaming the records alone 87 us); 8 sequences of 4096 16.2 us and one of 1500 9.3, where what counts is the chain of plan, page ids,
// copies, one or two steps, folding and the second launch.  24 sequences of 5 drafted tokens, 32 and 8 heads of 128, up to 6000 positions:
// 46 us, 1.0 instructions a clock and SM: latency, with eight warps at 255 registers.
#pragma once
#include "kv4_common.cuh"
#include "sm100_ptx.cuh"

namespace neon {
namespace kv4 {

constexpr int kStep = 64;             // positions of a step
constexpr float kNoMax = -1e30f;      // level before the first score
constexpr float kLog2e = 1.4426950408889634f;
// where (log2) the largest probability of a group may lie, as f16 pairs too, and where it is put when it does not
constexpr float kHigh = 15.5f, kLow = 0.f, kRaiseTo = 8.f, kLowerTo = 5.f;
constexpr uint32_t kHighest = 0x7bff7bffu, kLowest = 0x3c003c00u;  // (the largest f16; those below it by half a step round to it)
constexpr int kSpread = 7;         // how far (log2) a step's value scales may lie below the largest for f16 operands
constexpr int kCareful = 1 << 23;  // positions times how far the run's scales lie apart before small probabilities are looked after
constexpr int kMostSum = 30;       // (log2) how far lowering its level may take a row's sum
constexpr int kWide = 24;          // (log2) how far apart the run's scales may lie for what a group loses then not to count

constexpr int kMaxHeadRows = 1 << 26;        // rows times query heads a key/value head of a call
constexpr long long kMaxCtaUnits = 1 << 28;  // steps of a CTA: eight times as many are below 2^32 (and would take half a minute)

struct AttendParams {
    Batch b;
    Shape s;
    const uint8_t* cache;
    const void* q;
    long long q_stride;
    const uint16_t* sinks;
    int window, G, half;  // half: q and out are f16, else bf16
    float scale;
    void* out;
    float* part;  // partial results: [CTA][2] of CTAs, then [CTA][warp] of warps, each [R][D] outputs and [R][2] maxima and sums
    int grid, stages;
    int R;        // rows (tokens times G) of an item: 8 * NT
    uint32_t G_inverse;  // ceil(2^32 / G)
    // r / G for r < kMaxHeadRows: exact, as r * (G_inverse * G - 2^32) < 2^32
    __device__ __forceinline__ int token(int r) const { return G == 1 ? r : (int)__umulhi((uint32_t)r, G_inverse); }
    // first position that a row at `pos` may see (pos may be below 0, the window any number)
    __device__ __forceinline__ int first_seen(int pos) const { return window > 0 && pos >= window ? pos - window + 1 : 0; }
};

constexpr int kAttendWarps = 8;
constexpr long long kWaitCycles = 1000000000;  // half a second

// ---- the plan: how many steps each sequence has, before which unit it starts ------------------------------------
// Units are (sequence, key/value head, row block, step), in that order.
struct SeqPlan {
    int row0, n, len, pos0;      // first row, rows, positions, position of the first row
    int lo_step, steps, blocks;  // first step that any row sees, how many, row blocks
};

__device__ __forceinline__ SeqPlan plan_of(const AttendParams& p, int s) {
    SeqPlan r;
    const int2 sp = p.b.span(s);
    r.row0 = sp.x;
    r.n = sp.y;
    const int full = p.b.seq_lens[s];
    r.len = max(min(full, p.b.width * p.s.P), 0);
    r.pos0 = full - r.n;
    const int lo = p.first_seen(r.pos0);
    r.lo_step = lo / kStep;
    r.blocks = r.n > 0 ? (r.n * p.G + p.R - 1) >> (31 - __clz(p.R)) : 0;  // R is a power of two
    r.steps = r.n > 0 && r.len > lo ? (r.len + kStep - 1) / kStep - r.lo_step : 0;
    return r;
}

__device__ __forceinline__ long long units_of(const AttendParams& p, int s) {
    const SeqPlan r = plan_of(p, s);
    if (p.b.seq_lens[s] > p.b.width * p.s.P || (p.b.cu_q && p.b.cu_q[s + 1] < p.b.cu_q[s])) report(p.b.status, NEON_KV4_BAD_LENGTH);
    return (long long)p.s.nkv * r.blocks * r.steps;
}

// before[s] = units of the sequences before s, for s <= n; returns the units of a CTA.  The whole CTA takes part.
__device__ __forceinline__ long long scan_units(const AttendParams& p, long long* before) {
    if (p.b.n > 32) {
        for (int s = threadIdx.x; s < p.b.n; s += blockDim.x) before[s + 1] = units_of(p, s);
        __syncthreads();
    }
    if (threadIdx.x < 32) {
        long long carry = 0;
        for (int s0 = 0; s0 < p.b.n; s0 += 32) {
            const int s = s0 + threadIdx.x;
            long long v = s >= p.b.n ? 0 : p.b.n > 32 ? before[s + 1] : units_of(p, s);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long w = __shfl_up_sync(0xffffffffu, v, o);
                if (threadIdx.x >= o) v += w;
            }
            v += carry;
            if (s < p.b.n) before[s + 1] = v;
            carry = __shfl_sync(0xffffffffu, v, 31);
        }
        if (threadIdx.x == 0) before[0] = 0;
    }
    __syncthreads();
    // few units: a step for every warp of as many CTAs as that takes, so that little is left to merge
    const long long units = before[p.b.n];
    if (units <= 0x7fffffff) return max(((uint32_t)units + p.grid - 1) / p.grid, (uint32_t)kAttendWarps);
    return (units + p.grid - 1) / p.grid;
}

__device__ __forceinline__ int sequence_of(const long long* before, int n, long long unit) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (before[mid + 1] <= unit) lo = mid + 1; else hi = mid;
    }
    return lo;
}

// ---- one warp's work -------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8x8 matrix of 16-bit values, one row per four lanes, transposed
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t max_f16x2(uint32_t a, uint32_t b) {  // passes over NaN
    uint32_t d;
    asm("max.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t min_f16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("min.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^e for -126 <= e <= 127, 0 below, infinity above
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)min(max(e + 127, 0), 255) << 23); }

// floor(log2 x) of a positive x; 0 of infinities and NaN
__device__ __forceinline__ int log2_of(float x) {
    const int e = (int)(__float_as_uint(x) >> 23) - 127;
    return e < 128 ? e : 0;
}

__device__ __forceinline__ bool wait_bounded(uint64_t* bar, int parity) {
    if (sm100::mbar_test(bar, parity)) return true;
    const long long t0 = clock64();
    do {
        if (sm100::mbar_test(bar, parity)) return true;
    } while (clock64() - t0 < kWaitCycles);
    return false;
}

// out = acc / den as 16 bits, eight columns; den = 0: no position was seen
__device__ __forceinline__ void store_out(const AttendParams& p, long long at, const float (&x)[8]) {
    if (p.half) store8(static_cast<__half*>(p.out) + at, x);
    else store8(static_cast<__nv_bfloat16*>(p.out) + at, x);
}
__device__ __forceinline__ float inverse(float den) { return den > 0.f ? 1.f / den : (den == 0.f ? 0.f : den); }
__device__ __forceinline__ float sink_of(const AttendParams& p, int head, float m) {
    return p.sinks ? ex2(bf16_bits_to_float(p.sinks[head]) * kLog2e - m) : 0.f;
}

// Shared memory of a warp: the ring of steps, then the step's scales as operands, then the barriers.
//   ks f32 [64][D/32]   key scales
//   vs f16 [D/32][4 tiles][4][4]   value scales; the last index runs over positions t, t + 4, t + 8, t + 12 of a tile
// When its run is over, the ring holds its last partial result.
template <int D>
struct WarpSmem {
    static constexpr int kBlocks = D / 32, kRing = kStep * (D + D / 16), kKs = kStep * kBlocks * 4, kVs = kBlocks * kStep * 2;
    static constexpr int kMaxStages = 8;
    static __host__ __device__ constexpr int bytes(int stages) { return stages * kRing + kKs + kVs + kMaxStages * 8; }
};
struct Partial {  // a warp's unfinished item
    int there, starts, ends;  // whether it has the item's first, last step
    int row0, r0, rows, head;
    const float* data;        // [R][D] outputs, [R][2] maxima and sums
};
__host__ __device__ constexpr int plan_bytes(int n) { return (n + 2) / 2 * 16; }

template <int D, int P, int NT>
__global__ void __launch_bounds__(kAttendWarps * 32, (D == 64 && NT == 1) ? 2 : 1) attend_kernel(const AttendParams p) {
    using W = WarpSmem<D>;
    constexpr int NB = W::kBlocks, R = 8 * NT, kSlot = R * (D + 2);
    constexpr int kPages = kStep / P, kRec = P * (D + D / 16), kCodes = P * D / 2, kScales = P * D / 32;
    constexpr int TI = NT == 1 ? 4 : 2;      // 16-position tiles whose scores are held at once
    constexpr uint32_t kOnes = 0x3c003c00u;  // two f16 ones
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ Partial parts[2 * kAttendWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    long long* before = reinterpret_cast<long long*>(smem);
    unsigned char* mine = smem + plan_bytes(p.b.n) + warp * W::bytes(p.stages);
    float* ks = reinterpret_cast<float*>(mine + p.stages * W::kRing);
    __half* vs = reinterpret_cast<__half*>(mine + p.stages * W::kRing + W::kKs);
    uint64_t* full = reinterpret_cast<uint64_t*>(mine + p.stages * W::kRing + W::kKs + W::kVs);
    if (lane == 0)
        for (int i = 0; i < p.stages; ++i) sm100::mbar_init(&full[i], 1);
    if (lane < 2) parts[warp * 2 + lane].there = 0;
    sm100::fence_barrier_init();
    pdl_wait();
    pdl_launch_dependents();
    const long long share = scan_units(p, before), units = before[p.b.n];
    const long long cta_begin = min(blockIdx.x * share, units);
    const int cta_units = (int)(min(cta_begin + share, units) - cta_begin);
    const int run_begin = (int)((uint32_t)cta_units * warp / kAttendWarps), run_end = (int)((uint32_t)cta_units * (warp + 1) / kAttendWarps);
    const long long u_end = cta_begin + run_end;
    int left = run_end - run_begin, left_ahead = left;  // steps to multiply, to fetch
    auto block_of = [&](int i) { return (i >> 2) * 2 + (g >> 2); };  // column block of this lane's rows of output tile i
    bool timeout = false;

    if (left > 0) {
        struct Item { int s, head, block; };
        auto place = [&](Item& c, SeqPlan& q, long long unit) {  // returns the step
            c.s = sequence_of(before, p.b.n, unit);
            q = plan_of(p, c.s);
            const long long r = unit - before[c.s];
            if (r <= 0x7fffffff) {
                const uint32_t r32 = (uint32_t)r, item = r32 / (uint32_t)q.steps;
                c.head = q.blocks == 1 ? item : item / (uint32_t)q.blocks;
                c.block = item - c.head * q.blocks;
                return (int)(r32 - item * q.steps);
            }
            const long long item = r / q.steps;
            c.head = (int)(item / q.blocks);
            c.block = (int)(item % q.blocks);
            return (int)(r % q.steps);
        };
        auto next_item = [&](Item& c, SeqPlan& q, int units_left) {
            if (++c.block < q.blocks) return;
            c.block = 0;
            if (++c.head < p.s.nkv) return;
            if (units_left) place(c, q, u_end - units_left);
        };
        Item cur, ahead;
        SeqPlan q, qa;
        int step = place(cur, q, u_end - left);
        ahead = cur;
        qa = q;
        // ---- fetching: runs `stages` steps ahead ---------------------------------------------------------------------
        int a_page = (q.lo_step + step) * kPages, a_end = (q.lo_step + q.steps) * kPages;  // of the item that is fetched
        int id_base = -64, ids = -1;  // 32 page ids of its sequence, from id_base on
        uint32_t holes = 0;           // which pages of a stage are missing: four bits each
        auto fetch = [&](int stage) {
            if ((uint32_t)(a_page - id_base) >= 32u) {
                id_base = a_page;
                ids = -1;
                if ((a_page + lane) * P < qa.len) {
                    ids = p.b.table[ahead.s * p.b.table_stride + a_page + lane];
                    if (ids < 0 || ids >= p.b.n_pages) {
                        report(p.b.status, NEON_KV4_BAD_PAGE);
                        ids = -1;
                    }
                }
            }
            unsigned char* to = mine + stage * W::kRing;
            if constexpr (kPages == 1) {
                const int id = __shfl_sync(0xffffffffu, ids, a_page - id_base);
                if (lane == 0) {
                    sm100::mbar_expect_tx(&full[stage], id >= 0 ? kRec : 0);
                    if (id >= 0) sm100::bulk_load(to, p.cache + ((long long)id * p.s.nkv + ahead.head) * kRec, kRec, &full[stage]);
                }
                holes = id >= 0 ? holes & ~(15u << (4 * stage)) : holes | (1u << (4 * stage));
            } else {
                const int id = __shfl_sync(0xffffffffu, ids, a_page - id_base + (lane & (kPages - 1)));
                const uint32_t there = __ballot_sync(0xffffffffu, id >= 0) & ((1u << kPages) - 1);
                if (lane == 0) sm100::mbar_expect_tx(&full[stage], __popc(there) * kRec);
                __syncwarp();
                if (lane < kPages && id >= 0)
                    sm100::bulk_load(to + lane * kRec, p.cache + ((long long)id * p.s.nkv + ahead.head) * kRec, kRec, &full[stage]);
                holes = (holes & ~(15u << (4 * stage))) | ((there ^ ((1u << kPages) - 1)) << (4 * stage));
            }
            --left_ahead;
            a_page += kPages;
            if (a_page == a_end) {
                const int s = ahead.s;
                next_item(ahead, qa, left_ahead);
                a_page = qa.lo_step * kPages;
                a_end = a_page + qa.steps * kPages;
                if (ahead.s != s) id_base = -64;
            }
        };
        int stage = 0, phase = 0;
        bool started = false;

        while (left > 0) {
            // ---- an item: its queries --------------------------------------------------------------------------------
            const int r0 = cur.block * R, rows = min(R, q.n * p.G - r0);
            uint32_t qf[NT][NB][4];  // B operands: block, two k-steps of two registers
            float qs[NT][2];         // factor of the scores of columns 2t, 2t + 1
            uint4 raw[NT][NB];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int rr = r0 + min(j * 8 + g, rows - 1), token = p.token(rr);
                const uint16_t* src = static_cast<const uint16_t*>(p.q) + (q.row0 + token) * p.q_stride + (cur.head * p.G + rr - token * p.G) * D + t * 8;
#pragma unroll
                for (int b = 0; b < NB; ++b) raw[j][b] = *reinterpret_cast<const uint4*>(src + b * 32);
            }
            if (!started) {  // (the queries are on their way)
                for (int i = 0; i < p.stages && left_ahead > 0; ++i) fetch(i);
                started = true;
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float amax = 0.f, x[NB][8];
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    if (p.half) load8(reinterpret_cast<const __half*>(&raw[j][b]), x[b]);
                    else load8(reinterpret_cast<const __nv_bfloat16*>(&raw[j][b]), x[b]);
#pragma unroll
                    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[b][i]));
                }
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                const int e = (int)(__float_as_uint(amax) >> 23) - 127;  // floor(log2 amax); 128 for infinities
                const int up = amax > 0.f && e < 128 ? min(14 - e, 126) : 0;
                const float f = j * 8 + g < rows ? pow2i(up) : 0.f;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) qf[j][b][i] = f == 0.f ? 0u : pack2(x[b][2 * i] * f, x[b][2 * i + 1] * f, __half());
                const float product = p.scale * kLog2e * pow2i(-up), back = product == 0.f ? 1e-30f : product;  // (a scale of 0: all alike)
                qs[j][0] = __shfl_sync(0xffffffffu, back, 8 * t);
                qs[j][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
            }
            // what column c sees: positions above sees_lo(c), up to sees_hi(c)
            auto sees_hi = [&](int c) { return c < rows ? min(q.pos0 + p.token(r0 + c), q.len - 1) : -1; };
            auto sees_lo = [&](int c) { return p.first_seen(q.pos0 + p.token(r0 + c)) - 1; };
            const int pos_lo = q.pos0 + p.token(r0), pos_last = q.pos0 + p.token(r0 + rows - 1), pos_hi = min(pos_last, q.len - 1);
            const int first = p.first_seen(pos_lo);
            float o[NT][D / 16][4], l[NT][4], m[NT][2];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
                for (int i = 0; i < D / 16; ++i) o[j][i][0] = o[j][i][1] = o[j][i][2] = o[j][i][3] = 0.f;
                l[j][0] = l[j][1] = l[j][2] = l[j][3] = 0.f;
                m[j][0] = m[j][1] = kNoMax;
            }
            int ve[NB];          // largest value scale so far (its byte), per block
            int apart = kSpread;  // how far below it others were, at most
#pragma unroll
            for (int b = 0; b < NB; ++b) ve[b] = 0;
            const int n = min(q.steps - step, left);
            const bool starts = step == 0, ends = step + n == q.steps;
            // steps that any row sees a position of; steps of which every row sees every position
            const int see_begin = first / kStep, see_end = pos_hi < 0 ? 0 : pos_hi / kStep + 1;
            const int open_begin = (p.first_seen(pos_last) + kStep - 1) / kStep, open_end = (min(pos_lo, q.len - 1) + 1) >> 6;

            const int first_step = q.lo_step + step;
            int careful_from = first_step + (kCareful >> kSpread) / kStep;
            for (int at_step = first_step, end_step = at_step + n; at_step < end_step; ++at_step) {
                const int p0 = at_step * kStep;  // first position of the step
                if (!wait_bounded(&full[stage], phase)) {
                    timeout = true;
                    break;
                }
                const unsigned char* st = mine + stage * W::kRing;
                const uint32_t there = ~(holes >> (4 * stage)) & ((1u << kPages) - 1);
                const bool open = at_step >= open_begin && at_step < open_end && there == (1u << kPages) - 1;
                if (at_step >= see_begin && at_step < see_end) {
                    // ---- scales: lane l takes positions 2l and 2l + 1 -------------------------------------------------
                    int vb[NB][2];
                    uint32_t below = 0;  // the scales' distances from the largest, or'ed
                    {
                        const int q0 = 2 * lane, pg = q0 / P, in = q0 % P;
                        const unsigned char* sc = st + pg * kRec + 2 * kCodes + in * NB;
                        uint32_t kw[NB / 2], vw[NB / 2];  // four bytes: two positions of two blocks, or one of four
#pragma unroll
                        for (int i = 0; i < NB / 2; ++i) {
                            kw[i] = *reinterpret_cast<const uint32_t*>(sc + 4 * i);
                            vw[i] = *reinterpret_cast<const uint32_t*>(sc + kScales + 4 * i);
                        }
#pragma unroll
                        for (int i = 0; i < NB / 2; ++i) {
                            const float2 a = scales_to_f32(kw[i] & 0xffffu), c = scales_to_f32(kw[i] >> 16);
                            *reinterpret_cast<float4*>(ks + q0 * NB + 4 * i) = make_float4(a.x, a.y, c.x, c.y);
                        }
#pragma unroll
                        for (int b = 0; b < NB; ++b)
#pragma unroll
                            for (int i = 0; i < 2; ++i) vb[b][i] = (vw[(i * NB + b) / 4] >> (8 * ((i * NB + b) % 4))) & 255u;
                        if (!open) {
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const bool ok = ((there >> pg) & 1) && p0 + q0 + i <= pos_hi && p0 + q0 + i >= first;
#pragma unroll
                                for (int b = 0; b < NB; ++b) vb[b][i] = ok ? vb[b][i] : -1;
                            }
                        }
#pragma unroll
                        for (int b = 0; b < NB; ++b)
#pragma unroll
                            for (int i = 0; i < 2; ++i) below |= (uint32_t)(ve[b] - vb[b][i]);
                    }
                    bool plain = true;  // f16 operands do
                    if (__any_sync(0xffffffffu, below > (uint32_t)kSpread)) {  // (kSpread has all its bits set)
                        int grown = 0, under = 0;
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            for (int i = 0; i < 2; ++i) vb[b][i] = vb[b][i] > kTopScale && vb[b][i] < 255 ? kTopScale : vb[b][i];
                            int top = __reduce_max_sync(0xffffffffu, max(vb[b][0], vb[b][1]));
                            if (top == 255) {  // NaN blocks: no operand; the rows that see one become NaN
                                for (int i = 0; i < 2; ++i) {
                                    uint32_t bad = __ballot_sync(0xffffffffu, vb[b][i] == 255);
                                    if (vb[b][i] == 255) vb[b][i] = -1;
                                    for (; bad; bad &= bad - 1) {
                                        const int pos = p0 + 2 * (__ffs(bad) - 1) + i;
#pragma unroll
                                        for (int j = 0; j < NT; ++j)
#pragma unroll
                                            for (int c = 0; c < 2; ++c) {
                                                const int col = j * 8 + 2 * t + c;
                                                if (pos > sees_hi(col) || pos <= sees_lo(col)) continue;
#pragma unroll
                                                for (int w = 0; w < D / 16; ++w)
                                                    if (block_of(w) == b) o[j][w][c] = o[j][w][c + 2] = __uint_as_float(0x7fc00000u);
                                            }
                                    }
                                }
                                top = __reduce_max_sync(0xffffffffu, max(vb[b][0], vb[b][1]));
                            }
                            const int low = __reduce_min_sync(0xffffffffu, min(vb[b][0] < 0 ? 999 : vb[b][0], vb[b][1] < 0 ? 999 : vb[b][1]));
                            if (top > ve[b]) {
                                if (ve[b] > 0) grown = max(grown, top - ve[b]);
                                const float f = pow2i(ve[b] - top);
                                ve[b] = top;
#pragma unroll
                                for (int j = 0; j < NT; ++j)
#pragma unroll
                                    for (int i = 0; i < D / 16; ++i)
                                        if (block_of(i) == b) {
                                            o[j][i][0] *= f; o[j][i][1] *= f; o[j][i][2] *= f; o[j][i][3] *= f;
                                        }
                            }
                            under = max(under, ve[b] - low);
                        }
                        plain = under <= kSpread;
                        apart = max(apart + grown, under);
                        careful_from = first_step + (kCareful >> min(apart, 31)) / kStep;
                    }
                    // scales relative to the largest: 1 .. 2^-7 (anything finite where no row looks)
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int in = (2 * lane + i) & 15;
                            const int h = max(vb[b][i] - ve[b] + 15, 0) * 1024;
                            reinterpret_cast<uint16_t*>(vs)[((b * 4 + (lane >> 3)) * 4 + (in & 3)) * 4 + (in >> 2)] = (uint16_t)h;
                        }
                    __syncwarp();
                    // ---- scores: keys' rows g and g + 8 of a tile are its positions at and at + 8 ------------------------
                    const int at = (g & 1) * 4 + (g >> 1);
#pragma unroll 1
                    for (int i0 = 0; i0 < 4; i0 += TI) {
                        float sc[NT][TI][4];
#pragma unroll
                        for (int i = 0; i < TI; ++i) {
                            const int tile = 16 * (i0 + i);
                            const unsigned char* kt = st + (tile / P) * kRec + (tile % P + at) * (D / 2) + t * 4;
#pragma unroll
                            for (int b = 0; b < NB; ++b) {
                                uint32_t fa[4], fb[4];
                                codes_to_f16(*reinterpret_cast<const uint32_t*>(kt + b * 16), fa);
                                codes_to_f16(*reinterpret_cast<const uint32_t*>(kt + 8 * (D / 2) + b * 16), fb);
                                const float s0 = ks[(tile + at) * NB + b], s1 = ks[(tile + at + 8) * NB + b];
#pragma unroll
                                for (int j = 0; j < NT; ++j) {
                                    float acc[4] = {0.f, 0.f, 0.f, 0.f};
                                    mma_f16(acc, fa[0], fb[0], fa[1], fb[1], qf[j][b][0], qf[j][b][1]);
                                    mma_f16(acc, fa[2], fb[2], fa[3], fb[3], qf[j][b][2], qf[j][b][3]);
                                    sc[j][i][0] = b ? fmaf(acc[0], s0, sc[j][i][0]) : acc[0] * s0;
                                    sc[j][i][1] = b ? fmaf(acc[1], s0, sc[j][i][1]) : acc[1] * s0;
                                    sc[j][i][2] = b ? fmaf(acc[2], s1, sc[j][i][2]) : acc[2] * s1;
                                    sc[j][i][3] = b ? fmaf(acc[3], s1, sc[j][i][3]) : acc[3] * s1;
                                }
                            }
                        }
                        if (!open) {  // what a column does not see scores -infinity (columns' factors are never zero)
#pragma unroll
                            for (int j = 0; j < NT; ++j)
#pragma unroll
                                for (int c = 0; c < 2; ++c) {
                                    const int hi = sees_hi(j * 8 + 2 * t + c), lo = sees_lo(j * 8 + 2 * t + c);
                                    const float never = qs[j][c] > 0.f ? -INFINITY : INFINITY;
#pragma unroll
                                    for (int i = 0; i < TI; ++i)
#pragma unroll
                                        for (int h = 0; h < 2; ++h) {
                                            const int pos = p0 + 16 * (i0 + i) + at + 8 * h;
                                            if (!((there >> (16 * (i0 + i) / P)) & 1) || pos > hi || pos <= lo) sc[j][i][2 * h + c] = never;
                                        }
                                }
                        }
                        // ---- probabilities -----------------------------------------------------------------------------------
                        auto argument = [&](int j, int i, int c) { return fmaf(sc[j][i][c], qs[j][c & 1], -m[j][c & 1]); };
                        uint32_t pf[NT][TI][2], top = 0;
                        auto weigh = [&] {
                            top = 0;
#pragma unroll
                            for (int j = 0; j < NT; ++j)
#pragma unroll
                                for (int i = 0; i < TI; ++i)
#pragma unroll
                                    for (int h = 0; h < 2; ++h) {
                                        pf[j][i][h] = pack2(ex2(argument(j, i, 2 * h)), ex2(argument(j, i, 2 * h + 1)), __half());
                                        top = max_f16x2(top, pf[j][i][h]);
                                    }
                        };
                        weigh();
                        bool exact = !plain;  // values in f32
                        bool move = __any_sync(0xffffffffu, !__hble2(as_half2(top), as_half2(kHighest)));
                        const bool careful = at_step >= careful_from;
                        if (careful) {  // is the largest of each column large enough, too?
                            uint32_t least = kHighest;
#pragma unroll
                            for (int j = 0; j < NT; ++j) {
                                uint32_t most = 0;  // of each of two columns
#pragma unroll
                                for (int i = 0; i < TI; ++i) most = max_f16x2(most, max_f16x2(pf[j][i][0], pf[j][i][1]));
#pragma unroll
                                for (int off = 4; off < 32; off <<= 1) most = max_f16x2(most, __shfl_xor_sync(0xffffffffu, most, off));
                                least = min_f16x2(least, most);
                            }
                            move = move || __any_sync(0xffffffffu, !__hbge2(as_half2(least), as_half2(kLowest)));
                        }
                        if (move) {
                            bool lost = false;
                            float x[NT][2];  // the largest scores, in units of log 2
#pragma unroll
                            for (int j = 0; j < NT; ++j)
#pragma unroll
                                for (int c = 0; c < 2; ++c) {
                                    float factor = qs[j][c];
                                    x[j][c] = -INFINITY;
                                    asm volatile("" : "+f"(factor));  // keeps these products out of the steps that need none
#pragma unroll
                                    for (int i = 0; i < TI; ++i) x[j][c] = fmaxf(x[j][c], fmaxf(sc[j][i][c] * factor, sc[j][i][c + 2] * factor));
#pragma unroll
                                    for (int off = 4; off < 32; off <<= 1) x[j][c] = fmaxf(x[j][c], __shfl_xor_sync(0xffffffffu, x[j][c], off));
                                }
#pragma unroll
                            for (int j = 0; j < NT; ++j)
#pragma unroll
                                for (int c = 0; c < 2; ++c) {
                                    float now = x[j][c] > m[j][c] + kHigh ? x[j][c] - kRaiseTo : m[j][c];
                                    if (careful) {
                                        const bool low = x[j][c] < now + kLow && x[j][c] > -INFINITY;
                                        const float floor = now - (float)max(kMostSum - max(log2_of(l[j][c]), 0), 0);
                                        now = low ? fmaxf(x[j][c] - kLowerTo, floor) : now;
                                        lost = lost || (low && x[j][c] < now + kLow);
                                    }
                                    const float f = ex2(m[j][c] - now);
                                    m[j][c] = now;
                                    l[j][c] *= f;
#pragma unroll
                                    for (int i = 0; i < D / 16; ++i) { o[j][i][c] *= f; o[j][i][c + 2] *= f; }
                                }
                            weigh();
                            exact = exact || (apart > kWide && __any_sync(0xffffffffu, lost));
                        }
                        // ---- values ------------------------------------------------------------------------------------------
                        if (!exact) {
#pragma unroll
                            for (int i = 0; i < TI; ++i) {
                                const int tile = 16 * (i0 + i);
                                const unsigned char* vt = st + (tile / P) * kRec + kCodes + (tile % P + t) * (D / 2) + g * 4;
#pragma unroll
                                for (int j = 0; j < NT; ++j) {
                                    pf[j][i][0] = transpose8(pf[j][i][0]);
                                    pf[j][i][1] = transpose8(pf[j][i][1]);
                                    mma_f16(l[j], kOnes, kOnes, kOnes, kOnes, pf[j][i][0], pf[j][i][1]);
                                }
#pragma unroll
                                for (int w = 0; w < NB / 2; ++w) {  // words g and g + 8 of a position: columns 64 w + 8 g .. + 7
                                    const uint32_t v0 = *reinterpret_cast<const uint32_t*>(vt + w * 32), v1 = *reinterpret_cast<const uint32_t*>(vt + w * 32 + 4 * (D / 2));
                                    const uint32_t v2 = *reinterpret_cast<const uint32_t*>(vt + w * 32 + 8 * (D / 2)), v3 = *reinterpret_cast<const uint32_t*>(vt + w * 32 + 12 * (D / 2));
                                    const uint2 f = *reinterpret_cast<const uint2*>(vs + (((w * 2 + (g >> 2)) * 4 + i0 + i) * 4 + t) * 4);
                                    // bytes of (column, both positions): even columns, odd columns
                                    uint32_t ev[4], od[4], ev2[4], od2[4];
                                    codes_to_f16((v0 & 0x0f0f0f0fu) | ((v1 * 16) & 0xf0f0f0f0u), ev);
                                    codes_to_f16(((v0 >> 4) & 0x0f0f0f0fu) | (v1 & 0xf0f0f0f0u), od);
                                    codes_to_f16((v2 & 0x0f0f0f0fu) | ((v3 * 16) & 0xf0f0f0f0u), ev2);
                                    codes_to_f16(((v2 >> 4) & 0x0f0f0f0fu) | (v3 & 0xf0f0f0f0u), od2);
#pragma unroll
                                    for (int c = 0; c < 4; ++c) {
                                        const uint32_t a0 = mul_f16x2(ev[c], f.x), a1 = mul_f16x2(od[c], f.x), a2 = mul_f16x2(ev2[c], f.y), a3 = mul_f16x2(od2[c], f.y);
#pragma unroll
                                        for (int j = 0; j < NT; ++j) mma_f16(o[j][w * 4 + c], a0, a1, a2, a3, pf[j][i][0], pf[j][i][1]);
                                    }
                                }
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < TI; ++i)
#pragma unroll
                                for (int r = 0; r < 2; ++r) {
                                    float mine_p[NT][2];
#pragma unroll
                                    for (int j = 0; j < NT; ++j)
#pragma unroll
                                        for (int c = 0; c < 2; ++c) mine_p[j][c] = ex2(argument(j, i, 2 * r + c));
                                    for (int gg = 0; gg < 8; ++gg) {  // the position of row gg (+ 8) of the tile's scores
                                        const int pos = 16 * (i0 + i) + (gg & 1) * 4 + (gg >> 1) + 8 * r;
                                        const unsigned char* rp = st + (pos / P) * kRec;
                                        float w[NT][2];
#pragma unroll
                                        for (int j = 0; j < NT; ++j)
#pragma unroll
                                            for (int c = 0; c < 2; ++c) {
                                                w[j][c] = __shfl_sync(0xffffffffu, mine_p[j][c], gg * 4 + t);
                                                l[j][c] += w[j][c];
                                            }
#pragma unroll
                                        for (int h = 0; h < NB / 2; ++h) {
                                            const int blk = h * 2 + (g >> 2);
                                            int e = ve[0];
#pragma unroll
                                            for (int b = 1; b < NB; ++b) e = blk == b ? ve[b] : e;
                                            const int held = rp[2 * kCodes + kScales + (pos % P) * NB + blk];
                                            const int byte = held == 255 ? held : min(held, kTopScale);
                                            const float f = byte <= e ? pow2i(byte - e) : 0.f;  // above: seen by no row, or NaN
                                            uint32_t half2[4];
                                            codes_to_f16(*reinterpret_cast<const uint32_t*>(rp + kCodes + (pos % P) * (D / 2) + h * 32 + g * 4), half2);
#pragma unroll
                                            for (int x = 0; x < 4; ++x) {
                                                const float2 val = __half22float2(*reinterpret_cast<const __half2*>(&half2[x]));
#pragma unroll
                                                for (int j = 0; j < NT; ++j)
#pragma unroll
                                                    for (int c = 0; c < 2; ++c) {
                                                        o[j][h * 4 + x][c] = fmaf(w[j][c], val.x * f, o[j][h * 4 + x][c]);
                                                        o[j][h * 4 + x][c + 2] = fmaf(w[j][c], val.y * f, o[j][h * 4 + x][c + 2]);
                                                    }
                                            }
                                        }
                                    }
                                }
                        }
                    }
                }
                __syncwarp();  // the stage and the tables are read
                if (left_ahead > 0) fetch(stage);
                if (++stage == p.stages) { stage = 0; phase ^= 1; }
            }
            if (timeout) {
                report(p.b.status, NEON_KV4_TIMEOUT);
                for (int i = 1; i < p.stages; ++i)  // no copy may land after the CTA is gone
                    wait_bounded(&full[(stage + i) % p.stages], stage + i < p.stages ? phase : phase ^ 1);
                break;
            }
            left -= n;
            // ---- the item's result: finished, or in the ring (the run is over), or in global memory ------------------------
            float* slot = left == 0 ? reinterpret_cast<float*>(mine) : p.part + ((long long)p.grid * 2 + blockIdx.x * kAttendWarps + warp) * kSlot;
            const bool whole = starts && ends;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int col = j * 8 + 2 * t + c;
                    if (col >= rows) continue;
                    const int token = p.token(r0 + col), head = cur.head * p.G + r0 + col - token * p.G;
                    const float inv = whole ? inverse(l[j][c] + sink_of(p, head, m[j][c])) : 1.f;
                    if (!whole && g == 0) *reinterpret_cast<float2*>(slot + R * D + col * 2) = make_float2(m[j][c], l[j][c]);
#pragma unroll
                    for (int w = 0; w < NB / 2; ++w) {
                        const int blk = w * 2 + (g >> 2);
                        int e = ve[0];
#pragma unroll
                        for (int b = 1; b < NB; ++b) e = blk == b ? ve[b] : e;
                        const float f = pow2i(e - 127) * inv;
                        float x[8];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            x[2 * i] = o[j][w * 4 + i][c] * f;
                            x[2 * i + 1] = o[j][w * 4 + i][c + 2] * f;
                        }
                        if (whole) store_out(p, ((long long)(q.row0 + token) * p.s.nq + head) * D + w * 64 + g * 8, x);
                        else store8(slot + col * D + w * 64 + g * 8, x);
                    }
                }
            if (!whole && lane == 0) parts[warp * 2 + starts] = {1, starts, ends, q.row0, r0, rows, cur.head, slot};
            // to the next item
            step += n;
            if (step == q.steps) {
                step = 0;
                next_item(cur, q, left);
            }
        }
    }
    __syncthreads();
    // ---- the CTA's unfinished items: runs of its warps' partial results, in order.  A run ends with a part that has the
    // item's last step, or before one that has the next item's first.
    const Partial* part_of = &parts[lane & (2 * kAttendWarps - 1)];
    const uint32_t all = (1u << 2 * kAttendWarps) - 1, is = __ballot_sync(0xffffffffu, part_of->there) & all;
    const uint32_t first_of = __ballot_sync(0xffffffffu, part_of->there && part_of->starts) & all;
    const uint32_t last_of = __ballot_sync(0xffffffffu, part_of->there && part_of->ends) & all;
    for (uint32_t rest = is; rest;) {
        const int a = __ffs(rest) - 1;
        const uint32_t from = ~((1u << a) - 1), after = from & ~(1u << a);
        int end = 2 * kAttendWarps;
        if (last_of & from) end = min(end, __ffs(last_of & from));
        if (first_of & after) end = min(end, __ffs(first_of & after) - 1);
        const uint32_t members = is & from & ((1u << end) - 1);
        rest &= ~members;
        const Partial& f = parts[a];
        const bool starts = f.starts, ends = (last_of & members) != 0;
        float* slot = p.part + ((long long)blockIdx.x * 2 + starts) * kSlot;
        for (int i = threadIdx.x; i < f.rows * (D / 8); i += kAttendWarps * 32) {
            const int col = i / (D / 8), c8 = i % (D / 8) * 8;
            const float* src[kAttendWarps];
            float2 ml[kAttendWarps];
            float M = kNoMax;
            uint32_t todo = members;
#pragma unroll
            for (int k = 0; k < kAttendWarps; ++k) {
                src[k] = nullptr;
                ml[k] = make_float2(kNoMax, 0.f);
                if (todo) {
                    src[k] = parts[__ffs(todo) - 1].data;
                    todo &= todo - 1;
                    ml[k] = *reinterpret_cast<const float2*>(src[k] + R * D + col * 2);
                    M = fmaxf(M, ml[k].x);
                }
            }
            float den = 0.f, x[8] = {};
#pragma unroll
            for (int k = 0; k < kAttendWarps; ++k)
                if (src[k]) {
                    const float e = ex2(ml[k].x - M);
                    float v[8];
                    load8(src[k] + col * D + c8, v);
                    den = fmaf(ml[k].y, e, den);
#pragma unroll
                    for (int h = 0; h < 8; ++h) x[h] = fmaf(v[h], e, x[h]);
                }
            if (starts && ends) {
                const int token = p.token(f.r0 + col), head = f.head * p.G + f.r0 + col - token * p.G;
                const float inv = inverse(den + sink_of(p, head, M));
#pragma unroll
                for (int h = 0; h < 8; ++h) x[h] *= inv;
                store_out(p, ((long long)(f.row0 + token) * p.s.nq + head) * D + c8, x);
            } else {
                if (c8 == 0) *reinterpret_cast<float2*>(slot + R * D + col * 2) = make_float2(M, den);
                store8(slot + col * D + c8, x);
            }
        }
    }
}

// Folds the partial results of the items that more than one CTA took part in, and writes zeros where an item has no
// step.  One warp per row and query head; lanes take D/32 columns each.
template <int D>
__global__ void __launch_bounds__(256) merge_kernel(const AttendParams p) {
    constexpr int C = D / 32;
    extern __shared__ __align__(16) unsigned char smem[];
    long long* before = reinterpret_cast<long long*>(smem);
    const int lane = threadIdx.x & 31;
    const long long task = (long long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    const int row = (int)(task / p.s.nq), head = (int)(task % p.s.nq);
    // This kernel starts once every CTA of attend_kernel has found what ran before it complete, so the batch may be read
    // at once; the partial results only after pdl_wait().
    const long long share = scan_units(p, before);
    if (row >= p.b.rows) { pdl_wait(); return; }  // (every thread waits: this kernel is not over before attend_kernel is)
    // the row's sequence: the last whose first row is not behind it
    int s = row;
    if (p.b.cu_q) {
        int lo = 0, hi = p.b.n - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (p.b.cu_q[mid] <= row) lo = mid; else hi = mid - 1;
        }
        s = lo;
    }
    if (s >= p.b.n) { pdl_wait(); return; }
    const SeqPlan q = plan_of(p, s);
    if (row < q.row0 || row >= q.row0 + q.n) { pdl_wait(); return; }
    const int kvh = p.token(head), rr = (row - q.row0) * p.G + head - kvh * p.G, block = rr >> (31 - __clz(p.R)), col = rr & (p.R - 1);
    const long long at = ((long long)row * p.s.nq + head) * D + lane * C;
    auto put = [&](int i, float x) {
        if (p.half) static_cast<__half*>(p.out)[at + i] = __float2half_rn(x);
        else static_cast<__nv_bfloat16*>(p.out)[at + i] = __float2bfloat16_rn(x);
    };
    const long long u0 = before[s] + ((long long)kvh * q.blocks + block) * q.steps, u1 = u0 + q.steps;
    const int c0 = u0 <= 0x7fffffff && share <= 0x7fffffff ? (int)((uint32_t)u0 / (uint32_t)share) : (int)(u0 / share);
    const bool none = q.steps == 0, merge = !none && (c0 + 1) * share < u1;  // else one CTA had all of it and wrote the result
    // contributors: CTA c0, in which the item begins, with its second slot, then the following ones' first slots
    const long long slot = (long long)p.R * (D + 2);
    const float* base = p.part + c0 * 2 * slot;
    const int n = merge ? (uint64_t)(u1 - 1 - c0 * share) <= 0x7fffffff && share <= 0x7fffffff ? (int)((uint32_t)(u1 - 1 - c0 * share) / (uint32_t)share) + 1
                                                                                            : (int)((u1 - 1 - c0 * share) / share) + 1
                        : 0;
    pdl_wait();
    if (none) {  // zeros only now: what ran before attend_kernel may still have read the buffer
#pragma unroll
        for (int i = 0; i < C; ++i) put(i, 0.f);
    }
    if (!merge) return;
    float M = kNoMax, den = 0.f, acc[C] = {};
    for (int k0 = 0; k0 < n; k0 += 32) {
        const int k = k0 + lane;
        const float* src = base + (k == 0 ? slot : 2 * k * slot) + p.R * D + col * 2;
        const float m = k < n ? src[0] : kNoMax, l = k < n ? src[1] : 0.f;
        float now = fmaxf(M, m);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, o));
        const float f = k < n ? ex2(m - now) : 0.f, old = ex2(M - now);
        float part = l * f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
        den = den * old + part;
#pragma unroll
        for (int i = 0; i < C; ++i) acc[i] *= old;
        const int here = min(32, n - k0);
#pragma unroll 4
        for (int j = 0; j < here; ++j) {
            const float* from = base + (k0 + j == 0 ? slot : 2 * (k0 + j) * slot) + col * D + lane * C;
            const float w = __shfl_sync(0xffffffffu, f, j);
#pragma unroll
            for (int i = 0; i < C; ++i) acc[i] = fmaf(from[i], w, acc[i]);
        }
        M = now;
    }
    const float inv = inverse(den + sink_of(p, head, M));
#pragma unroll
    for (int i = 0; i < C; ++i) put(i, acc[i] * inv);
}

}  // namespace kv4
}  // namespace neon
