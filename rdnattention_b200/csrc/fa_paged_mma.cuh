// The many-rows kernel of the paged attention: row tiles of 128 on tcgen05.
//
// Trees of drafted tokens and chunks of prompts bring 17 to thousands of rows per KV
// head.  Per 64-key tile of head_dim 128 an SM receives 32 KB (about 1400 cycles of
// its share of the HBM bandwidth at 1.9 GHz), and 128 rows need 8192 exponentials (512
// cycles) and three products of 256 cycles (Q K^T for hi and for lo, P V), so one row
// tile per KV head is HBM-bound if the tensor pipe and the softmax overlap; more row
// tiles read the same keys again, partly from L2, and are bound on the SM.
//
//   warps 0..3, 4..7   two softmax groups (thread = row = TMEM lane); key tile i of
//                      the CTA goes to group i & 1
//   warp 8             TMA producer, as in the few-rows kernel (warp 9: none)
//   warps 10, 11       issue S = Q K^T and O += P V, each for every other tile
//
// TMEM (512 columns at head_dim 128): Q hi and lo as the A operand of S = Q K^T
// (hi + lo, see the few-rows kernel: a query in shared memory would be read again by
// every product and keep them at 48 cycles instead of 31 for 64 keys), four S (P over
// S in place, the A operand of O += P V), one O.  S = Q K^T runs up to four tiles ahead
// of the softmax, so the products of one tile and the exponentials of two others
// overlap.
//
// The groups share O and with it each row's reference maximum: tile i's group takes the
// reference that tile i - 1's left in shared memory (a token per warp pair orders
// them), and where its own maximum is more than 2^8 above it, waits for P V of tile
// i - 1, rescales O and leaves the new one.
//
// Measured (32 / 8 heads, head_dim 128): trees of 64 tokens in 16 ragged contexts of up to
// 8192, 100 to 105 us; 512 tokens of 2 prompts over 16384 slots, 353 to 371 us = 750 to 790
// TFLOP/s (half more with the products of lo) in short runs at 1.5 GHz, 437 us sustained at the
// 1.2 to 1.3 GHz that the power cap leaves.  There a tile takes about 1100 cycles, of which the
// tensor pipe is busy 768 (70 %) and the exponential unit 512 (48 %): the two groups' chains from
// scores to P take 2200 each (waits 300, reading the scores and their maximum 450, reference 150,
// exponentials to P 1100), and the products of a tile wait for them in turn.  A segment's start
// and end take about 10000 (lengths, positions, Q and the tables in turn; then O), which is why
// units lead the list by kLeadMma positions.
#pragma once

#include "fa_paged.cuh"

namespace rdna {
namespace paged {

template <int DP>
struct MmaLayout {
    static constexpr int NSW = 8;                       // softmax warps
    static constexpr int THREADS = 32 * (NSW + 4);
    // Registers: LAUNCH_REGS are the most that 12 warps can have each; a few move from the
    // other four warps, which need far fewer, to the softmax warps.
    static constexpr int LAUNCH_REGS = 168, SOFTMAX_REGS = 184, OTHER_REGS = 136;
    static_assert(NSW * SOFTMAX_REGS + 4 * OTHER_REGS <= (NSW + 4) * LAUNCH_REGS,
                  "register split exceeds the launch allocation");
    static constexpr int NBOX = DP / 64;
    static constexpr int BOX_BYTES = KT * 128;
    static constexpr int TILE = NBOX * BOX_BYTES;
    static constexpr int STAGE = 2 * TILE;
    static constexpr int NST = DP == 64 ? 12 : 6;  // 192 KB
    static constexpr int NSB = 4;  // S buffers
    static constexpr int RT = 128;
    static constexpr int NW = kMaxTree / 32;
    // barriers (8 bytes each): full [NST], empty [NST], then
    static constexpr int S_FULL = 2 * NST, P_FULL = S_FULL + NSB, PV_DONE = P_FULL + NSB,  // [NSB] each
        TOKEN = PV_DONE + NSB,                                                             // [2 groups][4 warps]
        O_FULL = TOKEN + 8, Q_FULL = O_FULL + 1, DRAIN = Q_FULL + 2, N_BARS = DRAIN + 2;  // Q_FULL [2 issuers]
    static constexpr int OFF_TMEM = 8 * N_BARS, OFF_ABORT = OFF_TMEM + 4, OFF_KEPT = OFF_ABORT + 4;
    static constexpr int OFF_RING = 1024;
    static constexpr int OFF_MASK = OFF_RING + NST * STAGE;  // [RT][NW], then [RT]
    static constexpr int OFF_M = OFF_MASK + RT * NW * 4 + RT * 4;  // [RT] reference maxima
    static constexpr int OFF_L = OFF_M + RT * 4;                   // [2][RT] row sums
    static constexpr int OFF_SEG = OFF_L + 2 * RT * 4;             // [NSW] Segment
    static constexpr int OFF_STAGE = OFF_SEG + NSW * 64;  // [NSW] 32 rows of 64 bytes (see row_chunk)
    static constexpr int STAGE_BYTES = 32 * 64;
    static constexpr int OFF_PRE = OFF_STAGE + NSW * STAGE_BYTES;
    static_assert(sizeof(Segment) <= 64, "a segment's slot");
    static constexpr int SMEM_BYTES = OFF_PRE + kMaxList * 4 + 1024;  // + alignment slack
    static_assert(SMEM_BYTES <= 232448, "shared memory of one CTA");
    // TMEM columns
    static constexpr int QHI = 0, QLO = DP / 2, S0 = DP, O0 = S0 + NSB * KT, TMEM_USED = O0 + DP;
    static constexpr int TMEM_COLS = 512;
    static_assert(TMEM_USED <= TMEM_COLS, "TMEM budget");
};

template <class E>
struct AbFormat;  // operand type code of the instruction descriptor
template <>
struct AbFormat<F16> {
    static constexpr uint32_t value = 0;
};
template <>
struct AbFormat<BF16> {
    static constexpr uint32_t value = 1;
};

// Row max of N values: 8 chains of three-input max.
template <int N>
__device__ __forceinline__ float row_max(const float* x) {
    float m[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) m[i] = fmaxf(x[i], x[i + 8]);
#pragma unroll
    for (int c = 16; c < N; c += 16)
#pragma unroll
        for (int i = 0; i < 8; ++i) m[i] = fmax3(m[i], x[c + i], x[c + 8 + i]);
    return fmax3(fmax3(m[0], m[1], m[2]), fmax3(m[3], m[4], m[5]), fmaxf(m[6], m[7]));
}

// 32 columns without waiting, and the wait that gives them (the registers pass through it, so
// that nothing reads them before).
__device__ __forceinline__ void tmem_ld_x32_begin(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld_x32_end(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

// A warp's exchange between rows held by lanes (TMEM) and rows in global memory: 32 rows of
// four 16-byte chunks, placed so that both orders of access are free of bank conflicts.
// Four lanes side by side take one row's 64 bytes of global memory; a lane on its own per
// row would touch 32 lines with every access (the query's load took 7000 cycles so).
__device__ __forceinline__ uint4* row_chunk(uint8_t* stage, int row, int c) {
    return reinterpret_cast<uint4*>(stage + row * 64 + ((c ^ (row >> 1 & 3)) << 4));
}

// Bits lo .. hi - 1 (clamped to 0 .. 64).
__device__ __forceinline__ uint64_t bits_between(int lo, int hi) {
    lo = max(lo, 0);
    hi = min(hi, 64);
    if (lo >= hi) return 0;
    return (hi == 64 ? ~0ull : (1ull << hi) - 1ull) & ~((1ull << lo) - 1ull);
}

// 64 mask bits of a row from drafted token `from` (may be negative) on; nw words.
__device__ __forceinline__ uint64_t draft_bits(const uint32_t* words, int nw, int from) {
    auto word = [&](int w) { return w >= 0 && w < nw ? words[w] : 0u; };
    const int w = from >> 5, sh = from & 31;  // (arithmetic shift: floor)
    const uint32_t a = word(w), b = word(w + 1), c = word(w + 2);
    const uint32_t lo = __funnelshift_r(a, b, sh), hi = __funnelshift_r(b, c, sh);
    return static_cast<uint64_t>(hi) << 32 | lo;
}

template <class E, int DP>
__global__ void __launch_bounds__(MmaLayout<DP>::THREADS, 1) fa_paged_mma_kernel(
    const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
    const __grid_constant__ AttnParams p) {
    using L = MmaLayout<DP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);  // (an offset keeps the address space known)
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t bars = smem_u32(smem);
    auto bar = [&](int i) { return bars + 8u * i; };
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_ABORT);
    const Abort ab{abort_flag};
    uint8_t* ring = smem + L::OFF_RING;
    int* pre = reinterpret_cast<int*>(smem + L::OFF_PRE);
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < L::NST; ++s) {
            mbar_init(bar(s), 1);
            mbar_init(bar(L::NST + s), 1);
        }
        for (int k = 0; k < L::NSB; ++k) {
            mbar_init(bar(L::S_FULL + k), 1);
            mbar_init(bar(L::P_FULL + k), 4);
            mbar_init(bar(L::PV_DONE + k), 1);
        }
        for (int k = 0; k < 8; ++k) mbar_init(bar(L::TOKEN + k), 1);
        mbar_init(bar(L::O_FULL), 1);
        mbar_init(bar(L::Q_FULL), L::NSW);
        mbar_init(bar(L::Q_FULL + 1), L::NSW);
        mbar_init(bar(L::DRAIN), 1);
        mbar_init(bar(L::DRAIN + 1), 1);
        fence_barrier_init();
        prefetch_tmap(&tmK);
        prefetch_tmap(&tmV);
    }
    warm_params(p);
    __syncthreads();
    grid_dependency_wait();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const Sched sched = make_sched(p, pre);
    if (sched.total == 0 || static_cast<int>(blockIdx.x) >= sched.ctas) {
        zero_empty_units(p, threadIdx.x, L::THREADS);
        return;
    }
    const int begin = cta_begin(sched, blockIdx.x), end = cta_begin(sched, blockIdx.x + 1);
    if (threadIdx.x == 0) {
        volatile int* k = reinterpret_cast<volatile int*>(smem + L::OFF_KEPT);
        k[0] = begin;
        k[1] = end;
        k[2] = sched.q;
        k[3] = sched.r;
    }
    if (warp == 0) {
        tmem_alloc(smem_u32(smem + L::OFF_TMEM), L::TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    // the producer needs no TMEM: it starts on the ring while the rest waits for it
    const bool producer = warp == L::NSW;
    if (!producer) named_bar_sync(2, L::THREADS - 32);
    tc_fence_after();
    const uint32_t tmem = producer ? 0 : *reinterpret_cast<volatile uint32_t*>(smem + L::OFF_TMEM);

    // (the softmax warps read these again where they need them: registers are for the scores)
    volatile int* const kept = reinterpret_cast<volatile int*>(smem + L::OFF_KEPT);

    int i0 = 0, e = 0;  // running tile number of the segment's first tile
    if (warp >= L::NSW) {
        regs_decrease<L::OTHER_REGS>();
        if (producer) {
            uint32_t filled = 0;
            int issued = -1;
            for (int pos = begin; pos < end;) {
                const Segment g = segment_at(p, pre, pos, end, e);
                if (!produce<L>(p, &tmK, &tmV, g, i0, bars, smem_u32(ring), filled, issued, ab, lane)) {
                    drain<L>(bars, filled, issued);
                    break;
                }
                i0 += g.count;
                pos = g.next;
            }
        } else if (warp >= L::NSW + 2) {
            // ------------------------------------------------------------ MMA issuers
            // Warp w issues both products of the tiles i with i & 1 == w: O += P V of tile i, then
            // S = Q K^T of tile i + 4 into the buffer that P V has just read (one thread's products
            // run in the order of their issue), so that one warp's waits fall into the other's
            // products.  The whole warp runs the loop and one elected lane issues: operands that are
            // the same in all lanes (the shuffles tell the compiler) stay in uniform registers, where
            // the MMA takes them; issued by a lane in a branch of its own, each cost 87 cycles.
            const int w = warp - (L::NSW + 2);
            constexpr uint32_t IDESC_QK = instr_desc(1u, AbFormat<E>::value, 0u, 128, KT);
            constexpr uint32_t IDESC_PV = instr_desc(1u, AbFormat<E>::value, 1u, 128, DP);
            const uint64_t kd = smem_desc(smem_u32(ring), 16, 1024, 2);
            const uint64_t vd = smem_desc(smem_u32(ring + L::TILE), L::BOX_BYTES, 1024, 2);
            const bool split = p.cos != nullptr;  // a query that is not turned has no lo
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            int seg = 0;
            bool ok = true;
            auto wait = [&](int i, int parity, int site) {
                ok = ok && __all_sync(0xffffffffu, mbar_wait(bar(i), parity, ab, site));
                return ok;
            };
            auto issue_qk = [&](int i) {
                const int s = i % L::NST, sb = i % L::NSB;
                if (!wait(s, i / L::NST & 1, 0x713)) return;
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t at = kd + (static_cast<uint32_t>(s * L::STAGE) >> 4);
                    const uint32_t tS = tm + L::S0 + sb * KT;
#pragma unroll
                    for (int kk = 0; kk < DP / 16; ++kk)
                        mma_f16_ts(tS, tm + L::QHI + kk * 8, at + ((kk / 4 * L::BOX_BYTES + kk % 4 * 32) >> 4), IDESC_QK,
                                   kk > 0);
                    if (split) {
#pragma unroll
                        for (int kk = 0; kk < DP / 16; ++kk)
                            mma_f16_ts(tS, tm + L::QLO + kk * 8, at + ((kk / 4 * L::BOX_BYTES + kk % 4 * 32) >> 4),
                                       IDESC_QK, 1);
                    }
                    tc_commit(bar(L::S_FULL + sb));
                }
                __syncwarp();
            };
            for (int pos = begin; pos < end && ok;) {
                const Segment g = segment_at(p, pre, pos, end, e);
                pos = g.next;
                if (g.count == 0) continue;
                const int behind = __shfl_sync(0xffffffffu, i0 + g.count, 0), start = __shfl_sync(0xffffffffu, i0, 0);
                const int first = start + ((w - start) & 1);
                // (signalled for segments with a tile of this warp only: no phase passes unseen)
                if (first < behind && !wait(L::Q_FULL + w, seg++ & 1, 0x711)) break;
                tc_fence_after();
                for (int i = first; i < behind && i < first + L::NSB; i += 2) issue_qk(i);
                for (int i = first; ok && i < behind; i += 2) {
                    const int s = i % L::NST, sb = i % L::NSB;
                    // both warps add to O: the tile before must have been added
                    if (!wait(L::P_FULL + sb, i / L::NSB & 1, 0x715)) break;
                    if (i > start && !wait(L::PV_DONE + (i - 1) % L::NSB, (i - 1) / L::NSB & 1, 0x712)) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t at = vd + (static_cast<uint32_t>(s * L::STAGE) >> 4);
#pragma unroll
                        for (int kk = 0; kk < KT / 16; ++kk)
                            mma_f16_ts(tm + L::O0, tm + L::S0 + sb * KT + kk * 8, at + ((kk * 16 * 128) >> 4), IDESC_PV,
                                       kk > 0 || i > start);
                        tc_commit(bar(L::NST + s));
                        tc_commit(bar(L::PV_DONE + sb));
                        if (i == behind - 1) tc_commit(bar(L::O_FULL));
                    }
                    __syncwarp();
                    if (i + L::NSB < behind) issue_qk(i + L::NSB);
                }
                i0 = behind;
            }
            // nothing of this warp's is in flight when the TMEM goes
            if (elect_one()) tc_commit(bar(L::DRAIN + w));
            mbar_wait_drain(bar(L::DRAIN + w), 0);
            __syncwarp();
        }
    } else {
        // ---------------------------------------------------------------- softmax
        regs_increase<L::SOFTMAX_REGS>();
        const int w = warp / 4, quad = warp % 4, lr = quad * 32 + lane;  // row of the tile
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        const uint32_t tO = tmem + lanes + L::O0;
        uint32_t* words = reinterpret_cast<uint32_t*>(smem + L::OFF_MASK);
        int* ctx_lo = reinterpret_cast<int*>(smem + L::OFF_MASK + L::RT * L::NW * 4);
        volatile float* ref = reinterpret_cast<volatile float*>(smem + L::OFF_M);
        float* sums = reinterpret_cast<float*>(smem + L::OFF_L);
        uint8_t* stage = smem + L::OFF_STAGE + warp * L::STAGE_BYTES;
        const int nw = (p.t.T + 31) / 32;
        const float sl2 = p.scale_log2;
        bool aborted = false;
        int seg = 0;  // segments so far
        auto wait = [&](int i, int parity, int site) {
            if (!aborted && !__all_sync(0xffffffffu, mbar_wait(bar(i), parity, ab, site))) aborted = true;
            return !aborted;
        };
        // each warp keeps its segment in shared memory
        Segment& g = reinterpret_cast<Segment*>(smem + L::OFF_SEG)[warp];
        if (lane == 0) {
            g.next = kept[0];
            g.e = 0;
        }
        __syncwarp();
        while (g.next < kept[1]) {
            {
                int from = g.e;
                const Segment found = segment_at(p, pre, g.next, kept[1], from);
                __syncwarp();
                if (lane == 0) g = found;
                __syncwarp();
            }
            if (g.count == 0) {
                __syncwarp();
                continue;
            }
            const int row0 = g.rt * p.RT, ta = p.by_G.div(row0), r = row0 + lr;
            const int qpos = row_position(p, g, r);
            {
                // the rows' Q, half of the columns each group, turned and split, into TMEM
#pragma unroll
                for (int c0 = 0; c0 < DP / 16; c0 += 4) {
                    uint4 hi[4], lo[4];
                    int pos[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) pos[k] = __shfl_sync(0xffffffffu, qpos, 8 * k + lane / 4);
                    load_q<E, 4, 8>(p, g, row0 + quad * 32 + lane / 4, pos, w * (DP / 16) + c0 + lane % 4, hi, lo);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        __syncwarp();
#pragma unroll
                        for (int k = 0; k < 4; ++k) *row_chunk(stage, 8 * k + lane / 4, lane % 4) = half ? lo[k] : hi[k];
                        __syncwarp();
                        uint4 mine[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) mine[k] = *row_chunk(stage, lane, k);
                        tmem_st_x16(tmem + lanes + (half ? L::QLO : L::QHI) + w * (DP / 4) + 4 * c0,
                                    reinterpret_cast<const uint32_t*>(mine));
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    for (int k = 0; k < 2; ++k)
                        if (((k - i0) & 1) < g.count) mbar_arrive(bar(L::Q_FULL + k));
            }
            if (p.mask != nullptr) {
                build_mask(p, g, words, threadIdx.x, 32 * L::NSW);
                named_bar_sync(1, 32 * L::NSW);
                if (p.window > 0) {
                    trim_mask(p, g, words, ctx_lo, threadIdx.x, 32 * L::NSW);
                    named_bar_sync(1, 32 * L::NSW);
                }
            }
            if (p.mask != nullptr && p.window > 0) {
                const int lo = first_seen(p, g, ctx_lo, lane);
                if (lane == 0) g.s.lo = lo;
                __syncwarp();
            }
            int rlo, rhi;
            row_limits(p, g, r, qpos, ctx_lo, rlo, rhi);
            const bool dead = rlo >= rhi;
            const int rw = dead ? 0 : (p.by_G.div(r) - ta) * nw;
            const bool idle = __all_sync(0xffffffffu, dead);  // no row of this warp sees a key
            // keys in [all_lo, all_hi) are seen by every row of the warp that sees any
            const int all_lo = __reduce_max_sync(0xffffffffu, dead ? 0 : rlo);
            int all_hi = __reduce_min_sync(0xffffffffu, dead ? INT_MAX : rhi);
            if (p.mask != nullptr) all_hi = min(all_hi, g.L);
            float m = -INFINITY, l = 0.f;
            const int behind = i0 + g.count, tile0 = g.s.t0 + g.first - i0, L0 = g.L;
            const int first = i0 + ((w - i0) & 1);
            for (int i = first; i < behind; i += 2) {
                const int sb = i % L::NSB;
                const uint32_t tS = tmem + lanes + L::S0 + sb * KT;
                // the scores, and the reference that the tile before left (the first tile of a segment
                // has none)
                if (!aborted) {
                    const bool here = mbar_wait(bar(L::S_FULL + sb), i / L::NSB & 1, ab, 0x701) &&
                                      (i == i0 || mbar_wait(bar(L::TOKEN + (w ^ 1) * 4 + quad), (i - 1) / 2 & 1, ab, 0x703));
                    if (!__all_sync(0xffffffffu, here)) aborted = true;
                }
                if (aborted) continue;
                tc_fence_after();
                // the first 32 scores stay in registers from the maximum to the exponentials, the last
                // 32 are read again behind the first exponentials (64 leave the compiler too few
                // registers); all reads are begun early
                float mx = -INFINITY;
                uint32_t raw[32], last[32];
                float *x = reinterpret_cast<float*>(raw), *y = reinterpret_cast<float*>(last);
                uint64_t see = ~0ull;
                bool edge = false;
                auto hide = [&](float* v, uint32_t bits) {
                    if (edge) {
#pragma unroll
                        for (int c = 0; c < 32; ++c)
                            if (!(bits >> c & 1u)) v[c] = -INFINITY;
                    }
                };
                int k0, valid;
                tile_keys(p, tile0 + i, k0, valid);
                if (!idle) {
                    tmem_ld_x32_begin(tS, raw);
                    tmem_ld_x32_begin(tS + 32, last);
                    edge = valid < KT || k0 < all_lo || k0 + KT > all_hi;
                    if (edge) {
                        see = bits_between(rlo - k0, min(rhi - k0, valid));
                        if (p.mask != nullptr && k0 + KT > L0)
                            see &= bits_between(0, L0 - k0) | draft_bits(words + rw, nw, k0 - L0);
                    }
                    tmem_ld_x32_end(raw);
                    tmem_ld_x32_end(last);
                    hide(x, static_cast<uint32_t>(see));
                    hide(y, static_cast<uint32_t>(see >> 32));
                    mx = fmaxf(row_max<32>(x), row_max<32>(y)) * sl2;
                }
                const float old = i > i0 ? ref[lr] : -INFINITY;
                float now = old;
                const bool grow = fmaxf(old, mx) > old + 8.f;
                if (grow) now = fmaxf(old, mx);
                if (__any_sync(0xffffffffu, grow) && i > i0) {
                    // O is rescaled only when a maximum grows by more than 2^8: the row's final 1 / l
                    // uses the same reference, and p stays below 2^8
                    if (!wait(L::PV_DONE + (i - 1) % L::NSB, (i - 1) / L::NSB & 1, 0x704)) continue;
                    tc_fence_after();
                    const float corr = grow ? ex2(old - now) : 1.f;
#pragma unroll 1
                    for (int c0 = 0; c0 < DP; c0 += 16) {
                        uint32_t o[16];
                        tmem_ld_x16(tO + c0, o);
#pragma unroll
                        for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * corr);
                        tmem_st_x16(tO + c0, o);
                    }
                    tmem_wait_st();
                    tc_fence_before();
                }
                ref[lr] = now;
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(L::TOKEN + w * 4 + quad));
                if (now != m) {
                    l *= ex2(m - now);  // (the other group may have moved it)
                    m = now;
                }
                __syncwarp();  // the TMEM accesses below are warp-wide
                if (!idle) {
                    // P is rounded to the cache's type, the operand type of the second product;
                    // the row sums take it unrounded
                    const float nm = m == -INFINITY ? 0.f : -m;
                    const uint64_t mul2 = f2(sl2, sl2), nm2 = f2(nm, nm);
                    uint64_t ls[4] = {0ull, 0ull, 0ull, 0ull};
                    auto exponentials = [&](const float* v, int c0) {
                        uint32_t pk[8];
#pragma unroll
                        for (int c = 0; c < 16; c += 2) {
                            float a0, a1;
                            f2_split(ffma2(f2(v[c], v[c + 1]), mul2, nm2), a0, a1);
                            const float p0 = ex2(a0), p1 = ex2(a1);
                            ls[(c >> 1) & 3] = fadd2(ls[(c >> 1) & 3], f2(p0, p1));
                            pk[c / 2] = E::pack(p0, p1);
                        }
                        tmem_st_x8(tS + c0 / 2, pk);  // (over scores that have been read)
                    };
                    exponentials(x, 0);
                    tmem_ld_x32_begin(tS + 32, last);
                    exponentials(x + 16, 16);
                    tmem_ld_x32_end(last);
                    hide(y, static_cast<uint32_t>(see >> 32));
                    exponentials(y, 32);
                    exponentials(y + 16, 48);
                    float s0, s1;
                    f2_split(fadd2(fadd2(ls[0], ls[1]), fadd2(ls[2], ls[3])), s0, s1);
                    l += s0 + s1;
                    tmem_wait_st();
                    tc_fence_before();
                }
                if (k0 < g.s.lo || k0 + KT > g.s.hi)
                    zero_unseen_v<DP>(ring + i % L::NST * L::STAGE + L::TILE, g.s.lo, g.s.hi, k0, quad * (KT / 4), KT / 4, lane, 32);
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(L::P_FULL + sb));
            }
            // ------------------------------------------------------------ epilogue
            wait(L::O_FULL, seg++ & 1, 0x702);
            tc_fence_after();
            // this group's sum against the segment's last reference
            {
                const int last = behind - 1;
                if ((last & 1) != w) wait(L::TOKEN + (w ^ 1) * 4 + quad, last / 2 & 1, 0x705);
                const float end_m = ref[lr];
                sums[w * L::RT + lr] = m == end_m ? l : l * ex2(m - end_m);
                m = end_m;
            }
            named_bar_sync(1, 32 * L::NSW);
            if (g.first == 0 && threadIdx.x == 0) describe_unit(p, Sched{0, 0, kept[2], kept[3]}, g, kept[0]);
            if (!aborted && !*abort_flag && !__all_sync(0xffffffffu, r >= p.rows)) {
                const float M = dead ? -INFINITY : m;
                const float lsum = dead ? 0.f : sums[lr] + sums[L::RT + lr];
                const bool whole = g.count == g.s.n;
                const float inv = whole ? (lsum == 0.f ? 0.f : 1.f / lsum) : 1.f;
                float* slot = partial_slot(p, segment_slot(g, kept[0]));
#pragma unroll 1
                for (int c0 = w * (DP / 2); c0 < (w + 1) * (DP / 2); c0 += 16) {
                    uint32_t raw[16];
                    __syncwarp();
                    tmem_ld_x16(tO + c0, raw);
                    float* o = reinterpret_cast<float*>(raw);
#pragma unroll
                    for (int k = 0; k < 16; ++k) o[k] = lsum == 0.f ? 0.f : o[k] * inv;
                    if (whole) {
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            *row_chunk(stage, lane, k) =
                                uint4{E::pack(o[8 * k], o[8 * k + 1]), E::pack(o[8 * k + 2], o[8 * k + 3]),
                                      E::pack(o[8 * k + 4], o[8 * k + 5]), E::pack(o[8 * k + 6], o[8 * k + 7])};
                        __syncwarp();
                        const int c = c0 + lane % 2 * 8;
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const int row = row0 + quad * 32 + 16 * k + lane / 2, t = p.by_G.div(row);
                            if (row < p.rows && c < p.D)
                                *reinterpret_cast<uint4*>(p.o + g.b * p.osb + (g.kvh * p.G + row - t * p.G) * p.osh +
                                                          t * p.oss + c) = *row_chunk(stage, 16 * k + lane / 2, lane % 2);
                        }
                    } else if (r < p.rows) {
#pragma unroll
                        for (int k = 0; k < 16; k += 4)
                            if (c0 + k < p.D)
                                reinterpret_cast<float4*>(slot)[(c0 + k) / 4 * p.RT + lr] =
                                    make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                    }
                }
                if (!whole && w == 0) {
                    slot[p.RT * p.D + lr] = M;
                    slot[p.RT * p.D + p.RT + lr] = lsum;
                }
            }
            tc_fence_before();
            named_bar_sync(1, 32 * L::NSW);  // Q, O, the mask and (m, l) areas are free again
            tc_fence_after();
            i0 = behind;
        }
        zero_empty_units(p, threadIdx.x, 32 * L::NSW);
    }
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, L::TMEM_COLS);
}

}  // namespace paged
}  // namespace rdna
