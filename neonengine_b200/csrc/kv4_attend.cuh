// Attention over the 4-bit paged cache: few rows per key/value head (a decoding step, drafted tokens, short chunks).
//
// An item is (sequence, block of rows, key/value head): the G query heads that share the head times a few tokens, at most
// 8 * NT rows, against the 64-position steps that any of its rows sees.  All items' steps in a row are cut evenly over the
// warps of the grid, whatever the lengths are (they are device memory): a warp takes a contiguous run of steps, finishes
// the items that lie wholly in its run and leaves a partial result (maximum, sum, unnormalised output) of the at most two
// that do not; merge_kernel folds those.
//
// Per step a warp multiplies on mma.sync.m16n8k16 with positions (keys) and columns (values) as the 16 rows and the item's
// rows as the 8 columns: S^T = K Q^T, O^T += V^T P^T.  With G = 8 no row of a product is idle; tcgen05 would need 128 rows and a
// trip through tensor memory for the same few columns.  Codes become f16 by one conversion per two of them.
//   Keys keep their codes: each 32-column block has a sum of its own, and its scale is a factor of that sum (f32), so any
//   scale is exact.  Queries are f16, every row scaled by a power of two so that its largest value lies in [2^14, 2^15):
//   exact for bf16 and f16 down to 2^-28 of the largest.
//   Values: a pair of positions of one column is one f16x2 operand, multiplied by the two positions' scales relative to
//   the largest scale met so far (outputs are rescaled when it grows).  Where scales lie further apart than 2^6, or grow
//   by more than 2^2, a probability that f16 rounds away could belong to a value that counts: such a step's values are
//   added in f32, one position at a time (five times as long, and rare), so no spread of scales loses anything.
//   Probabilities are rounded to f16 (2^-12), once; sums and statistics are f32.  The running maximum is raised only when a
//   score exceeds it by 2^8, so that most steps need no exchange between lanes.
// Steps travel by bulk copies (one per page and head: a record is contiguous) into a ring per warp.
#pragma once
#include "kv4_common.cuh"
#include "sm100_ptx.cuh"

namespace neon {
namespace kv4 {

constexpr int kStep = 64;             // positions of a step
constexpr float kNoMax = -1e30f;      // running maximum before the first score
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRaise = 8.f;         // how far (log2) a score may lie above the running maximum
constexpr int kSpread = 6, kGrowth = 2;  // how far (log2) value scales may lie below the largest, and the largest may grow, for f16 operands

struct AttendParams {
    Batch b;
    Shape s;
    const uint8_t* cache;
    const void* q;
    long long q_stride;
    const uint16_t* sinks;
    int window, G;
    float scale;
    void* out;
    float* part;      // [worker][2][8 * NT][2 + D]
    int workers;      // warps of the grid
    int stages;
    int row_blocks;   // rows (tokens times G) of an item: 8 * NT
};

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
    const int lo = p.window > 0 ? max(r.pos0 - p.window + 1, 0) : 0;
    r.lo_step = lo / kStep;
    r.blocks = r.n > 0 ? (r.n * p.G + p.row_blocks - 1) / p.row_blocks : 0;
    r.steps = r.n > 0 && r.len > lo ? (r.len + kStep - 1) / kStep - r.lo_step : 0;
    return r;
}

// before[s] = units of the sequences before s, for s <= n.  The whole CTA takes part; ends with a barrier.
__device__ __forceinline__ void scan_units(const AttendParams& p, long long* before) {
    for (int s = threadIdx.x; s < p.b.n; s += blockDim.x) {
        const SeqPlan r = plan_of(p, s);
        before[s + 1] = (long long)p.s.nkv * r.blocks * r.steps;
        if (p.b.seq_lens[s] > p.b.width * p.s.P || (p.b.cu_q && p.b.cu_q[s + 1] < p.b.cu_q[s])) report(p.b.status, NEON_KV4_BAD_LENGTH);
    }
    if (threadIdx.x == 0) before[0] = 0;
    __syncthreads();
    if (threadIdx.x < 32) {
        long long carry = 0;
        for (int s0 = 1; s0 <= p.b.n; s0 += 32) {
            const int s = s0 + threadIdx.x;
            long long v = s <= p.b.n ? before[s] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long w = __shfl_up_sync(0xffffffffu, v, o);
                if (threadIdx.x >= o) v += w;
            }
            v += carry;
            if (s <= p.b.n) before[s] = v;
            carry = __shfl_sync(0xffffffffu, v, 31);
        }
    }
    __syncthreads();
}

__device__ __forceinline__ long long worker_begin(long long units, int workers, int w) { return units * w / workers; }
__device__ __forceinline__ int worker_of(long long units, int workers, long long u) { return (int)(((u + 1) * workers - 1) / units); }

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
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^e for -126 <= e <= 127, 0 below, infinity above
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)min(max(e + 127, 0), 255) << 23); }

// Shared memory of a warp: the ring of steps, then the step's scales as operands, then the barriers.
//   ks f32 [64][D/32]   key scales
//   vs f16 [D/32][4 tiles][4][4]   value scales; the last index runs over positions t, t + 4, t + 8, t + 12 of a tile
template <int D>
struct WarpSmem {
    static constexpr int kBlocks = D / 32, kRing = kStep * (D + D / 16), kKs = kStep * kBlocks * 4, kVs = kBlocks * kStep * 2;
    static constexpr int kMaxStages = 8;
    static __host__ __device__ constexpr int bytes(int stages) { return stages * kRing + kKs + kVs + kMaxStages * 8; }
};

constexpr int kAttendWarps = 8;
constexpr long long kWaitCycles = 1000000000;  // half a second

__device__ __forceinline__ bool wait_bounded(uint64_t* bar, int parity) {
    if (sm100::mbar_test(bar, parity)) return true;
    const long long t0 = clock64();
    do {
        if (sm100::mbar_test(bar, parity)) return true;
    } while (clock64() - t0 < kWaitCycles);
    return false;
}

template <int D, int NT, class T>
__global__ void __launch_bounds__(kAttendWarps * 32, (D == 64 && NT <= 2) ? 2 : 1) attend_kernel(const AttendParams p) {
    using W = WarpSmem<D>;
    constexpr int NB = W::kBlocks, R = 8 * NT;
    extern __shared__ __align__(16) unsigned char smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    long long* before = reinterpret_cast<long long*>(smem);
    unsigned char* mine = smem + ((p.b.n + 2) / 2 * 16) + warp * W::bytes(p.stages);
    float* ks = reinterpret_cast<float*>(mine + p.stages * W::kRing);
    __half* vs = reinterpret_cast<__half*>(mine + p.stages * W::kRing + W::kKs);
    uint64_t* full = reinterpret_cast<uint64_t*>(mine + p.stages * W::kRing + W::kKs + W::kVs);
    if (lane == 0)
        for (int i = 0; i < p.stages; ++i) sm100::mbar_init(&full[i], 1);
    sm100::fence_barrier_init();
    pdl_wait();
    pdl_launch_dependents();
    scan_units(p, before);

    const long long units = before[p.b.n];
    // neighbouring workers on different SMs, so that few units spread over all of them
    const int worker = warp * gridDim.x + blockIdx.x;
    long long u = units ? worker_begin(units, p.workers, worker) : 0;
    const long long u_end = units ? worker_begin(units, p.workers, worker + 1) : 0;
    if (u >= u_end) return;

    const int P = p.s.P, lp = 31 - __clz(P), per_step = kStep / P, rec = p.s.record(), codes = p.s.codes(), scales = p.s.scales();
    // The unit that is fetched next: its sequence, head, block and step.
    auto seq_of = [&](long long unit) {
        int lo = 0, hi = p.b.n - 1;
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (before[mid + 1] <= unit) lo = mid + 1; else hi = mid;
        }
        return lo;
    };
    struct Cursor { int s, head, block, step; SeqPlan q; };
    auto place = [&](Cursor& c, long long unit) {
        c.s = seq_of(unit);
        c.q = plan_of(p, c.s);
        long long r = unit - before[c.s];
        c.step = (int)(r % c.q.steps);
        r /= c.q.steps;
        c.block = (int)(r % c.q.blocks);
        c.head = (int)(r / c.q.blocks);
    };
    auto advance = [&](Cursor& c, long long next) {  // to unit `next`, the one behind the cursor's
        if (++c.step < c.q.steps) return;
        c.step = 0;
        if (++c.block < c.q.blocks) return;
        c.block = 0;
        if (++c.head < p.s.nkv) return;
        if (next < u_end) place(c, next);
    };
    // Starts the copies of a unit's pages; returns a bit per page that is there.
    auto block_of = [&](int i) { return (i >> 2) * 2 + (g >> 2); };  // column block of this lane's rows of output tile i
    uint32_t valid = 0;  // four bits per stage
    auto fetch = [&](const Cursor& c, int stage) {
        const int first = (c.q.lo_step + c.step) * per_step;  // first page of the step
        int id = -1;
        if (lane < per_step && (first + lane) * P < c.q.len) {
            id = p.b.table[c.s * p.b.table_stride + first + lane];
            if (id < 0 || id >= p.b.n_pages) {
                report(p.b.status, NEON_KV4_BAD_PAGE);
                id = -1;
            }
        }
        const uint32_t there = __ballot_sync(0xffffffffu, id >= 0);
        if (lane == 0) sm100::mbar_expect_tx(&full[stage], __popc(there) * rec);
        __syncwarp();
        if (id >= 0)
            sm100::bulk_load(mine + stage * W::kRing + lane * rec, p.cache + ((long long)id * p.s.nkv + c.head) * rec, rec, &full[stage]);
        valid = (valid & ~(15u << (4 * stage))) | (there << (4 * stage));
    };

    Cursor ahead, cur;
    place(ahead, u);
    cur = ahead;
    long long u_ahead = u;
    for (int i = 0; i < p.stages && u_ahead < u_end; ++i) {
        fetch(ahead, i);
        ++u_ahead;
        advance(ahead, u_ahead);
    }
    int stage = 0, phase = 0;

    while (u < u_end) {
        // ---- an item: its queries --------------------------------------------------------------------------------
        const int r0 = cur.block * R, rows = min(R, cur.q.n * p.G - r0);
        uint32_t qf[NT][NB][4];   // B operands: block, two k-steps of two registers
        float qs[NT][2];          // factor of the scores of columns 2t, 2t + 1
        int hi[NT][2];            // last position that they see
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int r = j * 8 + g;
            float amax = 0.f, x[NB][8];
            if (r < rows) {
                const int rr = r0 + r;
                const T* src = static_cast<const T*>(p.q) + (cur.q.row0 + rr / p.G) * p.q_stride + (cur.head * p.G + rr % p.G) * D;
#pragma unroll
                for (int b = 0; b < NB; ++b) load8(src + b * 32 + t * 8, x[b]);
            } else {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[b][i] = 0.f;
            }
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[b][i]));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const int e = (int)(__float_as_uint(amax) >> 23) - 127;  // floor(log2 amax); 128 for infinities
            const int up = amax > 0.f && e < 128 ? min(14 - e, 126) : 0;
            const float f = pow2i(up);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
#pragma unroll
                for (int i = 0; i < 4; ++i) qf[j][b][i] = pack2(x[b][2 * i] * f, x[b][2 * i + 1] * f, __half());
            }
            const float back = p.scale * kLog2e * pow2i(-up);
            qs[j][0] = __shfl_sync(0xffffffffu, back, 8 * t);
            qs[j][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int c = j * 8 + 2 * t + i;
                hi[j][i] = c < rows ? min(cur.q.pos0 + (r0 + c) / p.G, cur.q.len - 1) : -1;
            }
        }
        const int pos_lo = cur.q.pos0 + r0 / p.G, pos_hi = min(cur.q.pos0 + (r0 + rows - 1) / p.G, cur.q.len - 1);
        float o[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[j][i][0] = o[j][i][1] = o[j][i][2] = o[j][i][3] = 0.f;
            m[j][0] = m[j][1] = kNoMax;
            l[j][0] = l[j][1] = 0.f;
        }
        int ve[NB];  // largest value scale so far (its byte), per block
#pragma unroll
        for (int b = 0; b < NB; ++b) ve[b] = 0;
        const int item_step0 = cur.step;
        const long long item_units = min((long long)(cur.q.steps - cur.step), u_end - u);
        const bool whole = item_step0 == 0 && item_units == cur.q.steps;
        const Cursor item = cur;

        for (int k = 0; k < (int)item_units; ++k) {
            const int p0 = (cur.q.lo_step + cur.step) * kStep;  // first position of the step
            if (!wait_bounded(&full[stage], phase)) {
                report(p.b.status, NEON_KV4_TIMEOUT);
                for (int i = 1; i < p.stages; ++i)  // no copy may land after the CTA is gone
                    wait_bounded(&full[(stage + i) % p.stages], stage + i < p.stages ? phase : phase ^ 1);
                return;
            }
            const unsigned char* st = mine + stage * W::kRing;
            const uint32_t there = (valid >> (4 * stage)) & 15u;
            // positions that a row of this item can see
            const int first = p.window > 0 ? max(pos_lo - p.window + 1, 0) : 0;
            // every position of the step is seen by every row
            const bool open = there == (1u << per_step) - 1 && p0 + kStep - 1 <= pos_lo && p0 + kStep <= cur.q.len &&
                              (p.window <= 0 || p0 > pos_hi - p.window);
            if (p0 <= pos_hi && p0 + kStep > first) {
                // ---- scales: lane l takes positions 2l and 2l + 1 ---------------------------------------------------
                int vmax[NB], vmin[NB], vb[NB][2];
                {
                    const int q0 = 2 * lane, pg = q0 >> lp, in = q0 & (P - 1);
                    const unsigned char* sc = st + pg * rec + 2 * codes + in * NB;
                    const bool ok0 = open || (((there >> pg) & 1) && p0 + q0 <= pos_hi && p0 + q0 >= first);
                    const bool ok1 = open || (((there >> pg) & 1) && p0 + q0 + 1 <= pos_hi && p0 + q0 + 1 >= first);
                    uint32_t kw[NB / 2], vw[NB / 2];  // four bytes: two positions of two blocks, or one of four
#pragma unroll
                    for (int i = 0; i < NB / 2; ++i) {
                        kw[i] = *reinterpret_cast<const uint32_t*>(sc + 4 * i);
                        vw[i] = *reinterpret_cast<const uint32_t*>(sc + scales + 4 * i);
                    }
#pragma unroll
                    for (int i = 0; i < NB / 2; ++i) {
                        const float2 a = scales_to_f32(kw[i] & 0xffffu), c = scales_to_f32(kw[i] >> 16);
                        *reinterpret_cast<float4*>(ks + q0 * NB + 4 * i) = make_float4(a.x, a.y, c.x, c.y);
                    }
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const int i0 = b, i1 = NB + b;  // byte of the two positions
                        vb[b][0] = ok0 ? (int)((vw[i0 / 4] >> (8 * (i0 % 4))) & 255u) : -1;
                        vb[b][1] = ok1 ? (int)((vw[i1 / 4] >> (8 * (i1 % 4))) & 255u) : -1;
                        vmax[b] = __reduce_max_sync(0xffffffffu, max(vb[b][0], vb[b][1]));
                        if (vmax[b] == 255) {  // NaN blocks: no operand; the rows that see one become NaN
                            for (int i = 0; i < 2; ++i) {
                                uint32_t bad = __ballot_sync(0xffffffffu, vb[b][i] == 255);
                                if (vb[b][i] == 255) vb[b][i] = -1;
                                for (; bad; bad &= bad - 1) {
                                    const int q = p0 + 2 * (__ffs(bad) - 1) + i;
#pragma unroll
                                    for (int j = 0; j < NT; ++j)
#pragma unroll
                                        for (int c = 0; c < 2; ++c) {
                                            const int own = cur.q.pos0 + (r0 + j * 8 + 2 * t + c) / p.G;
                                            if (q > hi[j][c] || (p.window > 0 && q <= own - p.window)) continue;
#pragma unroll
                                            for (int w = 0; w < D / 16; ++w)
                                                if (block_of(w) == b) o[j][w][c] = o[j][w][c + 2] = __uint_as_float(0x7fc00000u);
                                        }
                                }
                            }
                            vmax[b] = __reduce_max_sync(0xffffffffu, max(vb[b][0], vb[b][1]));
                        }
                        vmin[b] = __reduce_min_sync(0xffffffffu, min(vb[b][0] < 0 ? 999 : vb[b][0], vb[b][1] < 0 ? 999 : vb[b][1]));
                    }
                }
                bool plain = true;  // f16 operands do
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    if (vmax[b] > ve[b]) {
                        plain = plain && (ve[b] == 0 || vmax[b] - ve[b] <= kGrowth);
                        const float f = pow2i(ve[b] - vmax[b]);
                        ve[b] = vmax[b];
#pragma unroll
                        for (int j = 0; j < NT; ++j)
#pragma unroll
                            for (int i = 0; i < D / 16; ++i)
                                if (block_of(i) == b) {
                                    o[j][i][0] *= f; o[j][i][1] *= f; o[j][i][2] *= f; o[j][i][3] *= f;
                                }
                    }
                    plain = plain && ve[b] - vmin[b] <= kSpread;
                    // scales relative to the largest: 1 .. 2^-6
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int q = 2 * lane + i, in = q & 15;
                        const uint32_t h = vb[b][i] >= 0 ? (uint32_t)(15 - (ve[b] - vb[b][i])) << 10 : 0u;
                        reinterpret_cast<uint16_t*>(vs)[((b * 4 + (q >> 4)) * 4 + (in & 3)) * 4 + (in >> 2)] = (uint16_t)h;
                    }
                }
                __syncwarp();
                // ---- scores ------------------------------------------------------------------------------------------
                uint32_t pf[NT][4][2];  // probabilities as B operands
                float sc[NT][4][4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int tile = 16 * i, at = (g & 1) * 4 + (g >> 1);  // positions of rows g and g + 8 within the tile: at, at + 8
                    const unsigned char* kt = st + (tile >> lp) * rec + (tile & (P - 1)) * (D / 2);
                    float acc[NB][NT][4];
                    // the odd rows start with the other block: eight rows then cover all banks
                    uint32_t ka[NB], kb[NB];
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const int bb = b ^ (g & 1);
                        ka[b] = *reinterpret_cast<const uint32_t*>(kt + at * (D / 2) + bb * 16 + t * 4);
                        kb[b] = *reinterpret_cast<const uint32_t*>(kt + (at + 8) * (D / 2) + bb * 16 + t * 4);
                    }
#pragma unroll
                    for (int b = 0; b < NB; b += 2) {
                        const uint32_t x = ka[b], y = kb[b];
                        ka[b] = g & 1 ? ka[b + 1] : x;
                        ka[b + 1] = g & 1 ? x : ka[b + 1];
                        kb[b] = g & 1 ? kb[b + 1] : y;
                        kb[b + 1] = g & 1 ? y : kb[b + 1];
                    }
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        uint32_t fa[4], fb[4];
                        codes_to_f16(ka[b], fa);
                        codes_to_f16(kb[b], fb);
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            acc[b][j][0] = acc[b][j][1] = acc[b][j][2] = acc[b][j][3] = 0.f;
                            mma_f16(acc[b][j], fa[0], fb[0], fa[1], fb[1], qf[j][b][0], qf[j][b][1]);
                            mma_f16(acc[b][j], fa[2], fb[2], fa[3], fb[3], qf[j][b][2], qf[j][b][3]);
                        }
                    }
                    float s0[NB], s1[NB];
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        s0[b] = ks[(tile + at) * NB + b];
                        s1[b] = ks[(tile + at + 8) * NB + b];
                    }
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        float v[4] = {acc[0][j][0] * s0[0], acc[0][j][1] * s0[0], acc[0][j][2] * s1[0], acc[0][j][3] * s1[0]};
#pragma unroll
                        for (int b = 1; b < NB; ++b) {
                            v[0] = fmaf(acc[b][j][0], s0[b], v[0]);
                            v[1] = fmaf(acc[b][j][1], s0[b], v[1]);
                            v[2] = fmaf(acc[b][j][2], s1[b], v[2]);
                            v[3] = fmaf(acc[b][j][3], s1[b], v[3]);
                        }
#pragma unroll
                        for (int c = 0; c < 4; ++c) sc[j][i][c] = v[c] * qs[j][c & 1];
                    }
                    if (!open) {
                        const bool here = (there >> (tile >> lp)) & 1;
#pragma unroll
                        for (int j = 0; j < NT; ++j)
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                const int q = p0 + tile + at + (c >> 1) * 8, top = hi[j][c & 1];
                                const int own = top < 0 ? -1 : cur.q.pos0 + (r0 + j * 8 + 2 * t + (c & 1)) / p.G;
                                const bool seen = here && q <= top && (p.window <= 0 || q > own - p.window);
                                sc[j][i][c] = seen ? sc[j][i][c] : -INFINITY;
                            }
                    }
                }
                // ---- probabilities ---------------------------------------------------------------------------------------
                float top[NT][2];
                bool raise = false;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        top[j][c] = fmaxf(sc[j][0][c], sc[j][0][c + 2]);
#pragma unroll
                        for (int i = 1; i < 4; ++i) top[j][c] = fmaxf(top[j][c], fmaxf(sc[j][i][c], sc[j][i][c + 2]));
                        raise = raise || top[j][c] > m[j][c] + kRaise;
                    }
                }
                if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float x = top[j][c];
#pragma unroll
                            for (int off = 4; off < 32; off <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
                            const float now = fmaxf(m[j][c], x), f = ex2(m[j][c] - now);
                            m[j][c] = now;
                            l[j][c] *= f;
#pragma unroll
                            for (int i = 0; i < D / 16; ++i) { o[j][i][c] *= f; o[j][i][c + 2] *= f; }
                        }
                }
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            sc[j][i][c] = ex2(sc[j][i][c] - m[j][c & 1]);
                            l[j][c & 1] += sc[j][i][c];
                        }
                    }
                // ---- values ----------------------------------------------------------------------------------------------
                if (plain) {
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            pf[j][i][0] = transpose8(pack2(sc[j][i][0], sc[j][i][1], __half()));
                            pf[j][i][1] = transpose8(pack2(sc[j][i][2], sc[j][i][3], __half()));
                        }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int tile = 16 * i;
                        const unsigned char* vt = st + (tile >> lp) * rec + codes + ((tile & (P - 1)) + t) * (D / 2) + g * 4;
#pragma unroll
                        for (int w = 0; w < NB / 2; ++w) {  // words g and g + 8 of a position: columns 64 w + 8 g .. + 7
                            const uint32_t v0 = *reinterpret_cast<const uint32_t*>(vt + w * 32), v1 = *reinterpret_cast<const uint32_t*>(vt + w * 32 + 4 * (D / 2));
                            const uint32_t v2 = *reinterpret_cast<const uint32_t*>(vt + w * 32 + 8 * (D / 2)), v3 = *reinterpret_cast<const uint32_t*>(vt + w * 32 + 12 * (D / 2));
                            const uint2 f = *reinterpret_cast<const uint2*>(vs + (((w * 2 + (g >> 2)) * 4 + i) * 4 + t) * 4);
                            // bytes of (column, both positions): even columns, odd columns
                            uint32_t ev[4], od[4], ev2[4], od2[4];
                            codes_to_f16((v0 & 0x0f0f0f0fu) | ((v1 << 4) & 0xf0f0f0f0u), ev);
                            codes_to_f16(((v0 >> 4) & 0x0f0f0f0fu) | (v1 & 0xf0f0f0f0u), od);
                            codes_to_f16((v2 & 0x0f0f0f0fu) | ((v3 << 4) & 0xf0f0f0f0u), ev2);
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
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int r = 0; r < 2; ++r)
                            for (int gg = 0; gg < 8; ++gg) {  // the position of rows gg and gg + 8 of the tile's scores
                                const int q = 16 * i + (gg & 1) * 4 + (gg >> 1) + 8 * r;
                                const unsigned char* rp = st + (q >> lp) * rec;
                                float w[NT][2];
#pragma unroll
                                for (int j = 0; j < NT; ++j)
#pragma unroll
                                    for (int c = 0; c < 2; ++c) w[j][c] = __shfl_sync(0xffffffffu, sc[j][i][2 * r + c], gg * 4 + t);
#pragma unroll
                                for (int h = 0; h < NB / 2; ++h) {
                                    const int blk = h * 2 + (g >> 2);
                                    int e = ve[0];
#pragma unroll
                                    for (int b = 1; b < NB; ++b) e = blk == b ? ve[b] : e;
                                    const int byte = rp[2 * codes + scales + (q & (P - 1)) * NB + blk];
                                    const float f = byte <= e ? pow2i(byte - e) : 0.f;  // above: seen by no row, or NaN
                                    uint32_t half2[4];
                                    codes_to_f16(*reinterpret_cast<const uint32_t*>(rp + codes + (q & (P - 1)) * (D / 2) + h * 32 + g * 4), half2);
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
            __syncwarp();  // the stage and the tables are read
            ++u;
            advance(cur, u);
            if (u_ahead < u_end) {
                fetch(ahead, stage);
                ++u_ahead;
                advance(ahead, u_ahead);
            }
            if (++stage == p.stages) { stage = 0; phase ^= 1; }
        }
        // ---- the item's result -----------------------------------------------------------------------------------------
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) l[j][c] += __shfl_xor_sync(0xffffffffu, l[j][c], off);
                const int col = j * 8 + 2 * t + c;
                if (col >= rows) continue;
                const int rr = r0 + col, row = item.q.row0 + rr / p.G, head = item.head * p.G + rr % p.G;
                float inv = 1.f;
                if (whole) {
                    float den = l[j][c];
                    if (p.sinks) den += ex2(bf16_bits_to_float(p.sinks[head]) * kLog2e - m[j][c]);
                    inv = den > 0.f ? 1.f / den : (den == 0.f ? 0.f : den);
                }
                float* slot = p.part + (((long long)worker * 2 + (item_step0 == 0 ? 1 : 0)) * R + col) * (D + 2);
                if (!whole && g == 0) { slot[0] = m[j][c]; slot[1] = l[j][c]; }
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
                    if (whole) {
                        store8(static_cast<T*>(p.out) + ((long long)row * p.s.nq + head) * D + w * 64 + g * 8, x);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) *reinterpret_cast<float2*>(slot + 2 + w * 64 + g * 8 + 2 * i) = make_float2(x[2 * i], x[2 * i + 1]);
                    }
                }
            }
    }
}

// Folds the partial results of the items that more than one worker took part in, and writes zeros where an item has no
// step.  One warp per row and query head; lanes take D/32 columns each.
template <int D, class T>
__global__ void __launch_bounds__(256) merge_kernel(const AttendParams p) {
    constexpr int C = D / 32;
    extern __shared__ __align__(16) unsigned char smem[];
    long long* before = reinterpret_cast<long long*>(smem);
    pdl_wait();
    scan_units(p, before);
    const long long units = before[p.b.n];
    const int lane = threadIdx.x & 31, R = p.row_blocks;
    const long long task = (long long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    const int row = (int)(task / p.s.nq), head = (int)(task % p.s.nq);
    if (row >= p.b.rows) return;
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
    if (s >= p.b.n) return;
    const SeqPlan q = plan_of(p, s);
    if (row < q.row0 || row >= q.row0 + q.n) return;
    const int kvh = head / p.G, rr = (row - q.row0) * p.G + head % p.G, block = rr / p.row_blocks, col = rr % p.row_blocks;
    T* out = static_cast<T*>(p.out) + ((long long)row * p.s.nq + head) * D;
    if (q.steps == 0) {
#pragma unroll
        for (int i = 0; i < C; ++i) out[lane * C + i] = T(0.f);
        return;
    }
    const long long u0 = before[s] + ((long long)kvh * q.blocks + block) * q.steps, u1 = u0 + q.steps;
    {
        const int w = worker_of(units, p.workers, u0);
        if (worker_begin(units, p.workers, w + 1) >= u1) return;  // one worker had all of it and wrote the result
    }
    float M = kNoMax, den = 0.f, acc[C] = {};
    for (long long u = u0; u < u1;) {
        const int w = worker_of(units, p.workers, u);
        const float* slot = p.part + (((long long)w * 2 + (u == u0 ? 1 : 0)) * R + col) * (D + 2);
        const float m = slot[0], l = slot[1], now = fmaxf(M, m), a = ex2(M - now), b = ex2(m - now);
        den = den * a + l * b;
#pragma unroll
        for (int i = 0; i < C; ++i) acc[i] = acc[i] * a + slot[2 + lane * C + i] * b;
        M = now;
        u = worker_begin(units, p.workers, w + 1);
    }
    if (p.sinks) den += ex2(bf16_bits_to_float(p.sinks[head]) * kLog2e - M);
    const float inv = den > 0.f ? 1.f / den : (den == 0.f ? 0.f : den);
#pragma unroll
    for (int i = 0; i < C; ++i) out[lane * C + i] = T(acc[i] * inv);
}

}  // namespace kv4
}  // namespace neon
