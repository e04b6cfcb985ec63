// Attention over the 4-bit paged cache: chunks of prompts, on the tensor cores of a CTA (tcgen05).
//
// An item is (sequence, key/value head, 256 rows: 32 tokens at eight query heads a key/value head), as two tiles of 128 rows.  Per
// step of 64 positions:
//   copies    a warp brings each step's records (codes and scales) into shared memory, a bulk copy per page, four steps ahead;
//   unpacking four warps make two operands of them: bf16 keys [64 positions][64] and, transposed, tf32 values [64][64 positions];
//   products  one thread issues S = Q K^T (f32 in tensor memory, two buffers a tile), another O += P V with P read from tensor
//             memory: issuing takes as long as the products do, and neither waits behind the other's barriers;
//   softmax   two groups of four warps, one per tile, a row a thread: no exchange between threads.  P takes the place of S.
//             The output is rescaled (a trip through the registers) only when a step's probabilities, relative to the maximum so
//             far, reach 2^8.
// bf16 holds codes times any E8M0 scale exactly, and queries: f16 ones as the sum of two terms, with a product each.  The other
// product is tf32 because probabilities need more than bf16's 8 bits and f16 could not meet every scale of values; they are cut to
// tf32's 11 bits before they are summed, so that sum and output share the cut.
// What bounds it: neither pipe alone but the chain between them.  A step (256 rows, 64 positions) takes some 2400 clocks; the special
// function units need 1024 of them for its exponentials, the products 900 (tf32 runs at half the bf16 rate, and 64 columns make
// operands' reads from shared memory count), and some 5300 instructions go out, 0.55 a clock and scheduler.  Without the softmax's
// arithmetic a step takes 1700.  Two prompts' chunks of 2048 rows over up to 8192 positions, 64 and 8 heads: 692 us, 0.47 PFLOP/s.
#pragma once
#include "kv4_attend.cuh"

namespace neon {
namespace kv4 {

constexpr int kPreRows = 256, kPreStages = 3, kPreRaw = 4, kPreInfo = 8, kPreN = 64;
constexpr int kPreSoftmaxWarps = 8, kPreUnpackWarps = 4, kPreWarps = kPreSoftmaxWarps + kPreUnpackWarps + 3;
constexpr int kPreScoreWarp = kPreWarps - 3, kPreOutputWarp = kPreWarps - 2, kPreCopyWarp = kPreWarps - 1;

struct PrefillInfo {     // of a step
    uint32_t missing;    // pages that are not there
    uint32_t special;    // a value block is NaN:
    uint32_t nan[2][2];  // which, [block][position / 32]
};

struct PrefillSmem {
    unsigned char q[2][kPreRows * 128];               // [term][row][64 bf16], 128-byte swizzle
    unsigned char k[kPreStages][kStep * 128];         // [position][64 bf16]
    unsigned char v[kPreStages][2][kPreN * 128];      // [half of the positions][column][32 f32]
    unsigned char raw[kPreRaw][kStep * (64 + 4)];
    PrefillInfo info[kPreInfo];
    uint64_t raw_full[kPreRaw], raw_empty[kPreRaw], kv_full[kPreStages], kv_empty[kPreStages], s_full[2][2], p_full[2][2], pv_done[2][2], drained[2];
    uint32_t tmem;
    int abort, item[4];
};

// tensor memory columns: S (then P) of tile x, buffer b; O of tile x
__device__ __forceinline__ uint32_t col_s(int x, int b) { return x * 128 + b * 64; }
__device__ __forceinline__ uint32_t col_o(int x) { return 256 + x * kPreN; }

__device__ __forceinline__ void mma_bf16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_tf32_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// 32 columns of this warp's 32 lanes
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
          "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
          "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
          "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                   "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
// (the registers pass through the wait, so that nothing that uses them can come before it)
__device__ __forceinline__ void tmem_wait_load32(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                   "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                   "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 ::"memory");
}
__device__ __forceinline__ void tmem_wait_load16(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 ::"memory");
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Waits for a barrier's phase; false when that takes kWaitCycles, or when another wait of the CTA has already given up.  The
// hardware parks the warp for up to 4 us a try: 14 warps that probe in a loop would take a third of the issue slots.
__device__ __forceinline__ bool parked_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status) {
    const long long t0 = clock64();
    while (true) {
        uint32_t done;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(done) : "r"(sm100::smem_u32(bar)), "r"(parity), "r"(4000u) : "memory");
        if (done) return true;
        if (*abort_flag) return false;
        if (clock64() - t0 > kWaitCycles) {
            *abort_flag = 1;
            report(status, NEON_KV4_TIMEOUT);
            return false;
        }
    }
}

// 8 codes as f32, times a power of two
__device__ __forceinline__ void codes_to_f32(uint32_t w, float scale, float (&x)[8]) {
    uint32_t h[4];
    codes_to_f16(w, h);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        x[2 * i] = f.x * scale;
        x[2 * i + 1] = f.y * scale;
    }
}

template <int P>
__global__ void __launch_bounds__(kPreWarps * 32, 1) prefill_kernel(const AttendParams p) {
    constexpr int D = 64, kPages = kStep / P, kRec = P * (D + D / 16), kCodes = P * D / 2, kScales = P * D / 32;
    extern __shared__ unsigned char unaligned[];
    PrefillSmem& s = *reinterpret_cast<PrefillSmem*>(unaligned + (-sm100::smem_u32(unaligned) & 1023));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // ---- the item: the last tiles, which see the most, first --------------------------------------------------------------
    const int kvh = blockIdx.x % p.s.nkv, order = blockIdx.x / p.s.nkv;
    if (warp == 0) {
        int before = 0, found = -1, tile = 0;
        for (int s0 = 0; s0 < p.b.n; s0 += 32) {
            const int b = p.b.n - 1 - s0 - lane;  // sequences from the last on
            int tiles = 0;
            if (b >= 0) {
                tiles = (p.b.span(b).y * p.G + kPreRows - 1) / kPreRows;
                if (p.b.seq_lens[b] > p.b.width * P || (p.b.cu_q && p.b.cu_q[b + 1] < p.b.cu_q[b])) report(p.b.status, NEON_KV4_BAD_LENGTH);
            }
            int upto = tiles;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            upto += before;
            const uint32_t hit = __ballot_sync(0xffffffffu, order >= upto - tiles && order < upto);
            if (hit) {
                const int l = __ffs(hit) - 1;
                found = p.b.n - 1 - s0 - l;
                tile = __shfl_sync(0xffffffffu, upto, l) - 1 - order;  // the sequence's last tile first
                break;
            }
            before = __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) {
            s.item[0] = found;
            s.item[1] = tile;
            s.abort = 0;
        }
    }
    if (tid == 0) {
        for (int i = 0; i < kPreRaw; ++i) {
            sm100::mbar_init(&s.raw_full[i], 1);
            sm100::mbar_init(&s.raw_empty[i], 128);
        }
        for (int i = 0; i < kPreStages; ++i) {
            sm100::mbar_init(&s.kv_full[i], 128);
            sm100::mbar_init(&s.kv_empty[i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            sm100::mbar_init(&s.s_full[0][0] + i, 1);
            sm100::mbar_init(&s.p_full[0][0] + i, 128);
        }
        for (int i = 0; i < 4; ++i) sm100::mbar_init(&s.pv_done[0][0] + i, 1);
        for (int i = 0; i < 2; ++i) sm100::mbar_init(&s.drained[i], 1);
        sm100::fence_barrier_init();
    }
    if (tid < kPreInfo) s.info[tid] = {};
    __syncthreads();
    const int seq = s.item[0];
    if (seq < 0) return;
    AttendParams one = p;
    one.R = kPreRows;
    const SeqPlan q = plan_of(one, seq);
    const int r0 = s.item[1] * kPreRows, rows = min(kPreRows, q.n * p.G - r0);
    const int pos_lo = q.pos0 + p.token(r0), pos_hi = min(q.pos0 + p.token(r0 + rows - 1), q.len - 1);
    const int first = p.first_seen(pos_lo);
    const int step0 = first / kStep, n = pos_hi < first ? 0 : pos_hi / kStep + 1 - step0;
    // ---- queries, as bf16 terms -------------------------------------------------------------------------------------------
    const int tile = warp / 4;  // of a softmax warp
    const int rr = r0 + tid, token = p.token(min(rr, r0 + rows - 1)), head = kvh * p.G + min(rr, r0 + rows - 1) - token * p.G;
    if (tid < kPreRows) {
        const uint16_t* src = static_cast<const uint16_t*>(p.q) + (q.row0 + token) * p.q_stride + (long long)head * D;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            float x[8], y[8];
            if (p.half) load8(reinterpret_cast<const __half*>(src) + c * 8, x);
            else load8(reinterpret_cast<const __nv_bfloat16*>(src) + c * 8, x);
            const int at = tid * 128 + ((c ^ (tid & 7)) * 16);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = tid >= rows ? 0.f : p.scale < 0.f ? -x[i] : x[i];
                y[i] = x[i] - __bfloat162float(__float2bfloat16_rn(x[i]));
                if (x[i] - x[i] != 0.f) y[i] = 0.f;  // infinities have no second term
            }
            store8(reinterpret_cast<__nv_bfloat16*>(s.q[0] + at), x);
            if (p.half) store8(reinterpret_cast<__nv_bfloat16*>(s.q[1] + at), y);
        }
    }
    if (warp == kPreScoreWarp) sm100::tmem_alloc(&s.tmem, 512);
    sm100::fence_proxy_async();
    sm100::tc_fence_before();
    __syncthreads();
    sm100::tc_fence_after();
    const uint32_t tmem = s.tmem;
    // By a whole warp, which goes on or gives up as one; when a wait runs out, all others are called off.  A phase is told from the
    // one before by a bit, so every wait here is such that the phase before is known to be over and the one after cannot be
    // before this warp has gone on: barriers are one per buffer.
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (__all_sync(0xffffffffu, sm100::mbar_peek(bar, parity & 1))) return true;  // (a try that may park costs 200 clocks even then)
        return (bool)__all_sync(0xffffffffu, parked_wait(bar, parity & 1, &s.abort, p.b.status));
    };

    bool issue = false;  // this thread has issued products
    int fetched = 0;     // steps that were sent for
    if (n > 0 && warp < kPreSoftmaxWarps) {
        // ---- softmax: this thread's row ------------------------------------------------------------------------------------
        const int hi = tid < rows ? min(q.pos0 + token, q.len - 1) : -1, lo = p.first_seen(q.pos0 + token) - 1;
        const float positive = fabsf(p.scale) * kLog2e, qs = positive == 0.f ? 1e-30f : positive;
        const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);  // this warp's lanes: 32 * (warp % 4) in the upper half
        float m = kNoMax, l[4] = {0.f, 0.f, 0.f, 0.f};
        bool nan[2] = {false, false}, ok = true;
        for (int j = 0; j < n; ++j) {
            const int p0 = (step0 + j) * kStep, buf = j & 1;
            if (!wait(&s.s_full[tile][buf], j >> 1) || !wait(&s.kv_full[j % kPreStages], j / kPreStages)) { ok = false; break; }
            sm100::tc_fence_after();
            const PrefillInfo& info = s.info[j % kPreInfo];
            const uint32_t missing = info.missing;
            const bool masked = missing || p0 + kStep - 1 > hi || p0 <= lo;  // not every position is seen
            if (info.special)
#pragma unroll
                for (int b = 0; b < 2; ++b)
                    for (int h = 0; h < 2; ++h)
                        for (uint32_t bad = info.nan[b][h]; bad; bad &= bad - 1) {
                            const int pos = p0 + 32 * h + __ffs(bad) - 1;
                            nan[b] = nan[b] || (pos <= hi && pos > lo);
                        }
            uint32_t x[64];
            float sum[4], top;
            auto hide = [&](int from) {
                if (masked)
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (p0 + from + i > hi || p0 + from + i <= lo || ((missing >> ((from + i) / P)) & 1)) x[from + i] = 0xff800000u;
            };
            auto weigh = [&](int from) {
#pragma unroll
                for (int i = from; i < from + 32; ++i) {
                    x[i] = __float_as_uint(ex2(fmaf(__uint_as_float(x[i]), qs, -m))) & 0xffffe000u;  // tf32
                    sum[i & 3] += __uint_as_float(x[i]);
                }
            };
            // probabilities relative to the maximum so far, whose sum shows whether one is out of range
            auto read = [&](bool weighing) {
                tmem_load32(lanes + col_s(tile, buf), x);
                tmem_wait_load32(x);
                tmem_load32(lanes + col_s(tile, buf) + 32, x + 32);
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] = 0.f;
                hide(0);
                if (weighing) weigh(0);
                tmem_wait_load32(x + 32);
                hide(32);
                if (weighing) weigh(32);
            };
            read(j > 0);
            const bool out_of_range = j == 0 || !((sum[0] + sum[1]) + (sum[2] + sum[3]) < 256.f);
            if (__any_sync(0xffffffffu, out_of_range)) {
                if (j > 0) read(false);
                top = -INFINITY;
#pragma unroll
                for (int i = 0; i < 64; ++i) top = fmaxf(top, __uint_as_float(x[i]));
                const float now = out_of_range ? fmaxf(m, top * qs) : m, f = ex2(m - now);
                m = now;
#pragma unroll
                for (int i = 0; i < 4; ++i) l[i] *= f;
                if (j > 0) {
                    if (!wait(&s.pv_done[tile][buf ^ 1], (j - 1) >> 1)) { ok = false; break; }
                    sm100::tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < kPreN; c += 16) {
                        uint32_t o[16];
                        tmem_load16(lanes + col_o(tile) + c, o);
                        tmem_wait_load16(o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tmem_store16(lanes + col_o(tile) + c, o);
                    }
                    tmem_wait_store();
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] = 0.f;
                weigh(0);
                weigh(32);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) l[i] += sum[i];
            tmem_store32(lanes + col_s(tile, buf), x);
            tmem_store32(lanes + col_s(tile, buf) + 32, x + 32);
            tmem_wait_store();
            sm100::tc_fence_before();
            sm100::mbar_arrive(&s.p_full[tile][buf]);
        }
        if (ok && wait(&s.pv_done[tile][(n - 1) & 1], (n - 1) >> 1)) {
            sm100::tc_fence_after();
            const float inv = inverse((l[0] + l[1]) + (l[2] + l[3]) + sink_of(p, head, m));
#pragma unroll
            for (int c = 0; c < 64; c += 16) {
                uint32_t o[16];
                tmem_load16(lanes + col_o(tile) + c, o);
                tmem_wait_load16(o);
                if (tid < rows) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float y[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) y[i] = nan[c / 32] ? __uint_as_float(0x7fc00000u) : __uint_as_float(o[8 * h + i]) * inv;
                        store_out(p, ((long long)(q.row0 + token) * p.s.nq + head) * D + c + 8 * h, y);
                    }
                }
            }
        }
    } else if (n > 0 && warp < kPreSoftmaxWarps + kPreUnpackWarps) {
        // ---- unpacking -------------------------------------------------------------------------------------------------------
        const int t = tid & 127;
        for (int j = 0; j < n; ++j) {
            const int stage = j % kPreStages, p0 = (step0 + j) * kStep;
            if (!wait(&s.raw_full[j % kPreRaw], j / kPreRaw)) break;
            if (j >= kPreStages && !wait(&s.kv_empty[stage], j / kPreStages - 1)) break;
            const unsigned char* raw = s.raw[j % kPreRaw];
            PrefillInfo& info = s.info[j % kPreInfo];
            const uint32_t missing = info.missing;
            const bool whole = missing == 0 && p0 + kStep <= q.len;  // every position is there
            // keys: a position and half of its columns a thread.  Values: four positions and eight columns a thread.
            const int pos = t & 63, kb = t >> 6, group = (t & 7) + (t >> 6) * 8, word = (t >> 3) & 7, vb = word >> 2;
            auto live = [&](int at) { return whole || (!((missing >> (at / P)) & 1) && p0 + at < q.len); };
            const unsigned char *krec = raw + pos / P * kRec, *vrec = raw + group * 4 / P * kRec;  // (four positions lie in one page)
            uint4 kw = *reinterpret_cast<const uint4*>(krec + pos % P * (D / 2) + kb * 16);
            int kbyte = krec[2 * kCodes + pos % P * 2 + kb], vbyte[4];
            uint32_t vw[4];
            bool odd = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = (group * 4 + i) % P;
                vw[i] = *reinterpret_cast<const uint32_t*>(vrec + kCodes + at * (D / 2) + word * 4);
                vbyte[i] = vrec[2 * kCodes + kScales + at * 2 + vb];
                odd = odd || vbyte[i] > kTopScale;
            }
            sm100::mbar_arrive(&s.raw_empty[j % kPreRaw]);
            if (!whole) {
                if (!live(pos)) { kw = make_uint4(0u, 0u, 0u, 0u); kbyte = 0; }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!live(group * 4 + i)) { vw[i] = 0u; vbyte[i] = 0; }
            }
            if (odd)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (vbyte[i] == 255) {
                        if ((word & 3) == 0) {
                            atomicOr(&info.special, 1u);
                            atomicOr(&info.nan[vb][(group * 4 + i) / 32], 1u << ((group * 4 + i) % 32));
                        }
                        vbyte[i] = 0;
                        vw[i] = 0;
                    }
                    vbyte[i] = min(vbyte[i], kTopScale);
                }
            {
                const float scale = kbyte == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)min(kbyte, kTopScale) << 23);
                const uint32_t w[4] = {kw.x, kw.y, kw.z, kw.w};
                unsigned char* row = s.k[stage] + pos * 128;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float x[8];
                    codes_to_f32(w[c], scale, x);
                    store8(reinterpret_cast<__nv_bfloat16*>(row + (((4 * kb + c) ^ (pos & 7)) * 16)), x);
                }
            }
            {
                float x[4][8];
#pragma unroll
                for (int i = 0; i < 4; ++i) codes_to_f32(vw[i], __uint_as_float((uint32_t)vbyte[i] << 23), x[i]);
                unsigned char* base = s.v[stage][group >> 3] + word * 8 * 128;
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    *reinterpret_cast<float4*>(base + c * 128 + (((group & 7) ^ c) * 16)) = make_float4(x[0][c], x[1][c], x[2][c], x[3][c]);
            }
            sm100::fence_proxy_async();
            sm100::mbar_arrive(&s.kv_full[stage]);
        }
    } else if (n > 0 && warp == kPreCopyWarp) {
        // ---- copies ----------------------------------------------------------------------------------------------------------
        int id_base = -64, ids = -1;
        for (int j = 0; j < n; ++j, ++fetched) {
            const int page = (step0 + j) * kPages, stage = j % kPreRaw;
            if ((uint32_t)(page - id_base) >= 32u) {
                id_base = page;
                ids = -1;
                if ((page + lane) * P < q.len) {
                    ids = p.b.table[seq * p.b.table_stride + page + lane];
                    if (ids < 0 || ids >= p.b.n_pages) {
                        report(p.b.status, NEON_KV4_BAD_PAGE);
                        ids = -1;
                    }
                }
            }
            const int id = __shfl_sync(0xffffffffu, ids, page - id_base + (lane & (kPages - 1)));
            const uint32_t there = __ballot_sync(0xffffffffu, id >= 0) & ((1u << kPages) - 1);
            if (j >= kPreRaw && !wait(&s.raw_empty[stage], j / kPreRaw - 1)) break;
            PrefillInfo& info = s.info[j % kPreInfo];
            if (lane < 4) info.nan[lane / 2][lane % 2] = 0;
            __syncwarp();
            if (lane == 0) {
                info.missing = there ^ ((1u << kPages) - 1);
                info.special = 0;
                sm100::mbar_expect_tx(&s.raw_full[stage], __popc(there) * kRec);
            }
            __syncwarp();
            if (lane < kPages && id >= 0)
                sm100::bulk_load(s.raw[stage] + lane * kRec, p.cache + ((long long)id * p.s.nkv + kvh) * kRec, kRec, &s.raw_full[stage]);
        }
    } else if (n > 0 && warp == kPreScoreWarp) {
        // ---- scores ----------------------------------------------------------------------------------------------------------
        // f32 += bf16 * bf16; 128 rows, both operands K-major.  Descriptors differ by their start addresses (in 16 bytes) alone:
        // 2 for a k-step, a tile, a stage.
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((kStep / 8) << 17) | ((128u >> 4) << 24);
        const uint64_t dq = sm100::make_sw128_desc(sm100::smem_u32(s.q[0])), dk = sm100::make_sw128_desc(sm100::smem_u32(s.k[0]));
        constexpr uint32_t kTerm = kPreRows * 128 / 16, kTile = 128 * 128 / 16, kStageK = kStep * 128 / 16;
        issue = sm100::elect_one();
        bool ok = true;
        for (int j = 0; j < n && ok; ++j) {
            ok = wait(&s.kv_full[j % kPreStages], j / kPreStages);
            for (int x = 0; x < 2 && ok; ++x) {
                if (j >= 2) ok = wait(&s.pv_done[x][j & 1], (j - 2) >> 1);  // the probabilities of step j - 2 lie where these scores go
                if (!ok) break;
                sm100::tc_fence_after();
                if (issue) {
                    const uint64_t a = dq + x * kTile, b = dk + (uint32_t)(j % kPreStages) * kStageK;
                    const uint32_t d = tmem + col_s(x, j & 1);
#pragma unroll
                    for (int k = 0; k < 4; ++k) mma_bf16_ss(d, a + 2 * k, b + 2 * k, idesc, k > 0);
                    if (p.half)
#pragma unroll
                        for (int k = 0; k < 4; ++k) mma_bf16_ss(d, a + kTerm + 2 * k, b + 2 * k, idesc, 1);
                    sm100::tc_commit(&s.s_full[x][j & 1]);
                }
                __syncwarp();
            }
        }
    } else if (n > 0 && warp == kPreOutputWarp) {
        // ---- outputs: f32 += tf32 * tf32 -----------------------------------------------------------------------------------------
        const uint32_t idesc = (1u << 4) | (2u << 7) | (2u << 10) | ((kPreN / 8) << 17) | ((128u >> 4) << 24);
        const uint64_t dv = sm100::make_sw128_desc(sm100::smem_u32(s.v[0][0]));
        constexpr uint32_t kHalfV = kPreN * 128 / 16;
        issue = sm100::elect_one();
        bool ok = true;
        for (int j = 0; j < n && ok; ++j) {
            const int stage = j % kPreStages;
            ok = wait(&s.kv_full[stage], j / kPreStages);
            for (int x = 0; x < 2 && ok; ++x) {
                ok = wait(&s.p_full[x][j & 1], j >> 1);
                if (!ok) break;
                sm100::tc_fence_after();
                if (issue) {
                    const uint64_t b = dv + (uint32_t)stage * (2 * kHalfV);
                    const uint32_t d = tmem + col_o(x), a = tmem + col_s(x, j & 1);
#pragma unroll
                    for (int k = 0; k < 8; ++k) mma_tf32_ts(d, a + k * 8, b + k / 4 * kHalfV + k % 4 * 2, idesc, j > 0 || k > 0);
                    sm100::tc_commit(&s.pv_done[x][j & 1]);
                    if (x == 1) sm100::tc_commit(&s.kv_empty[stage]);
                }
                __syncwarp();
            }
        }
    }
    if (n == 0 && tid < rows)
        for (int c = 0; c < D; c += 8) {
            const float zero[8] = {};
            store_out(p, ((long long)(q.row0 + token) * p.s.nq + head) * D + c, zero);
        }
    sm100::tc_fence_before();
    __syncthreads();
    if (s.abort) {  // the same for the whole CTA: nobody waits any more.  What is under way has to end before shared and tensor memory go
        if (warp == kPreScoreWarp || warp == kPreOutputWarp) {
            uint64_t* done = &s.drained[warp == kPreOutputWarp];
            if (issue) sm100::tc_commit(done);
            __syncwarp();
            if (n > 0) wait_bounded(done, 0);
        } else if (warp == kPreCopyWarp) {
            for (int j = max(0, fetched - kPreRaw); j < fetched; ++j) wait_bounded(&s.raw_full[j % kPreRaw], (j / kPreRaw) & 1);
        }
        __syncthreads();
    }
    if (warp == kPreScoreWarp) sm100::tmem_dealloc(tmem, 512);
}

}  // namespace kv4
}  // namespace neon
