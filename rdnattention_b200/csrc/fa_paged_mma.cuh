// The many-rows kernel of the paged attention: row tiles of 128 on tcgen05.
//
// Trees of drafted tokens and chunks of prompts bring 17 to hundreds of rows per KV
// head.  Per 64-key tile of head_dim 128 an SM receives 32 KB (about 1340 cycles of
// its share of the HBM bandwidth), and 128 rows need 8192 exponentials (512 cycles)
// and three products of 128 cycles, so a tile of rows is HBM-bound as long as the
// softmax keeps up; more row tiles read the same keys again, mostly from L2.
//
//   warps 0..3, 4..7   two softmax groups (thread = row = TMEM lane); key tile i of
//                      the CTA goes to group i & 1
//   warps 8..11        producers (produce(), as in the few-rows kernel)
//   warp 12, warp 13   one lane issues S = Q K^T, one lane O += P V
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
#pragma once

#include "fa_paged.cuh"

namespace rdna {
namespace paged {

template <int DP>
struct MmaLayout {
    static constexpr int NPW = 4;
    static constexpr int NSW = 8;                       // softmax warps
    static constexpr int THREADS = 32 * (NSW + NPW + 4);
    static constexpr int NBOX = DP / 64;
    static constexpr int BOX_BYTES = KT * 128;
    static constexpr int TILE = NBOX * BOX_BYTES;
    static constexpr int STAGE = 2 * TILE;
    static constexpr int NST = 6;
    static constexpr int NSB = 4;  // S buffers
    static constexpr int RT = 128;
    static constexpr int NW = kMaxTree / 32;
    // barriers (8 bytes each): full [NST], empty [NST], then
    static constexpr int S_FULL = 2 * NST, P_FULL = S_FULL + NSB, PV_DONE = P_FULL + NSB,  // [NSB] each
        TOKEN = PV_DONE + NSB,                                                             // [2 groups][4 warps]
        O_FULL = TOKEN + 8, Q_FULL = O_FULL + 1, DRAIN = Q_FULL + 1, N_BARS = DRAIN + 2;
    static constexpr int OFF_TMEM = 8 * N_BARS, OFF_ABORT = OFF_TMEM + 4;
    static constexpr int OFF_RING = 1024;
    static constexpr int OFF_MASK = OFF_RING + NST * STAGE;  // [RT][NW], then [RT]
    static constexpr int OFF_M = OFF_MASK + RT * NW * 4 + RT * 4;  // [RT] reference maxima
    static constexpr int OFF_L = OFF_M + RT * 4;                   // [2][RT] row sums
    static constexpr int OFF_SEG = OFF_L + 2 * RT * 4;             // [NSW] Segment
    static constexpr int OFF_PRE = OFF_SEG + NSW * 64;
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

// Row max of 32 values: 8 chains of three-input max.
__device__ __forceinline__ float max32(const float* x) {
    float m[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) m[i] = fmax3(x[i], x[i + 8], x[i + 16]);
#pragma unroll
    for (int i = 0; i < 8; ++i) m[i] = fmaxf(m[i], x[i + 24]);
    return fmax3(fmax3(m[0], m[1], m[2]), fmax3(m[3], m[4], m[5]), fmaxf(m[6], m[7]));
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
__global__ void __launch_bounds__(MmaLayout<DP>::THREADS, 1) fa_paged_mma_kernel(const __grid_constant__ AttnParams p) {
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
            mbar_init(bar(s), 32 * L::NPW);
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
        mbar_init(bar(L::DRAIN), 1);
        mbar_init(bar(L::DRAIN + 1), 1);
        fence_barrier_init();
    }
    // columns behind head_dim are never copied: zero for good
    if (p.D < DP)
    for (int idx = threadIdx.x; idx < 2 * L::NST * KT * (DP / 8); idx += L::THREADS)
        if (idx % (DP / 8) * 8 >= p.D)
            *reinterpret_cast<uint4*>(ring + idx / (DP / 8) / KT * L::TILE +
                                      chunk_off(KT, idx / (DP / 8) % KT, idx % (DP / 8))) = uint4{0u, 0u, 0u, 0u};
    fence_proxy_async_smem();
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
    if (warp == 0) {
        tmem_alloc(smem_u32(smem + L::OFF_TMEM), L::TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    // the producers need no TMEM: they start on the ring while the rest waits for it
    const bool producer = warp >= L::NSW && warp < L::NSW + L::NPW;
    if (!producer) named_bar_sync(2, L::THREADS - 32 * L::NPW);
    tc_fence_after();
    const uint32_t tmem = producer ? 0 : *reinterpret_cast<volatile uint32_t*>(smem + L::OFF_TMEM);

    int i0 = 0, e = 0;  // running tile number of the segment's first tile
    if (producer) {
        for (int pos = begin; pos < end;) {
            const Segment g = segment_at(p, pre, pos, end, e);
            if (!produce<L>(p, g, i0, bars, smem_u32(ring), ab, threadIdx.x - 32 * L::NSW)) break;
            i0 += g.count;
            pos = g.next;
        }
        cp_async_wait_all();  // after an expired wait too, no copy outlives the CTA
    } else if (warp >= L::NSW + L::NPW) {
        // ------------------------------------------------------------ MMA issuers
        const int w = warp - (L::NSW + L::NPW);  // 0: S = Q K^T, 1: O += P V, others: idle
        if (w < 2) {
            constexpr uint32_t IDESC_QK = instr_desc(1u, AbFormat<E>::value, 0u, 128, KT);
            constexpr uint32_t IDESC_PV = instr_desc(1u, AbFormat<E>::value, 1u, 128, DP);
            const uint64_t kd = smem_desc(smem_u32(ring), 16, 1024, 2);
            const uint64_t vd = smem_desc(smem_u32(ring + L::TILE), L::BOX_BYTES, 1024, 2);
            const int halves = p.cos != nullptr ? 2 : 1;  // a query that is not turned has no lo
            int seg = 0, ok = 1;
            for (int pos = begin; pos < end && ok;) {
                const Segment g = segment_at(p, pre, pos, end, e);
                pos = g.next;
                if (g.count == 0) continue;
                if (lane == 0) {
                    if (w == 0) {
                        ok = mbar_wait(bar(L::Q_FULL), seg++ & 1, ab, 0x711);
                        tc_fence_after();
                    }
                    for (int i = i0; ok && i < i0 + g.count; ++i) {
                        const int s = i % L::NST, sb = i % L::NSB;
                        const uint32_t slot = static_cast<uint32_t>(s * L::STAGE) >> 4, tS = tmem + L::S0 + sb * KT;
                        if (w == 0) {
                            // the buffer's last P has been multiplied, the keys are there
                            ok = mbar_wait(bar(L::PV_DONE + sb), (i / L::NSB & 1) ^ 1, ab, 0x712) &&
                                 mbar_wait(bar(s), i / L::NST & 1, ab, 0x713);
                            if (!ok) break;
                            // the copies were written through the generic proxy, the products
                            // read through the async one
                            fence_proxy_async_smem();
                            tc_fence_after();
                            for (int half = 0; half < halves; ++half)
#pragma unroll
                                for (int kk = 0; kk < DP / 16; ++kk)
                                    mma_f16_ts(tS, tmem + (half ? L::QLO : L::QHI) + kk * 8,
                                               kd + slot +
                                                   static_cast<uint32_t>((kk / 4 * L::BOX_BYTES + kk % 4 * 32) >> 4),
                                               IDESC_QK, half > 0 || kk > 0);
                            tc_commit(bar(L::S_FULL + sb));
                        } else {
                            ok = mbar_wait(bar(s), i / L::NST & 1, ab, 0x714) &&
                                 mbar_wait(bar(L::P_FULL + sb), i / L::NSB & 1, ab, 0x715);
                            if (!ok) break;
                            fence_proxy_async_smem();
                            tc_fence_after();
#pragma unroll
                            for (int kk = 0; kk < KT / 16; ++kk)
                                mma_f16_ts(tmem + L::O0, tS + kk * 8, vd + slot + static_cast<uint32_t>((kk * 16 * 128) >> 4),
                                           IDESC_PV, kk > 0 || i > i0);
                            // (S of this tile came first: its keys have been read too)
                            tc_commit(bar(L::NST + s));
                            tc_commit(bar(L::PV_DONE + sb));
                            if (i == i0 + g.count - 1) tc_commit(bar(L::O_FULL));
                        }
                    }
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
                i0 += g.count;
            }
            if (lane == 0) {
                // nothing of this thread's is in flight when the TMEM goes
                tc_commit(bar(L::DRAIN + w));
                mbar_wait_drain(bar(L::DRAIN + w), 0);
            }
            __syncwarp();
        }
    } else {
        // ---------------------------------------------------------------- softmax
        const int w = warp / 4, quad = warp % 4, lr = quad * 32 + lane;  // row of the tile
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        const uint32_t tO = tmem + lanes + L::O0;
        uint32_t* words = reinterpret_cast<uint32_t*>(smem + L::OFF_MASK);
        int* ctx_lo = reinterpret_cast<int*>(smem + L::OFF_MASK + L::RT * L::NW * 4);
        volatile float* ref = reinterpret_cast<volatile float*>(smem + L::OFF_M);
        float* sums = reinterpret_cast<float*>(smem + L::OFF_L);
        const int nw = (p.t.T + 31) / 32;
        const float sl2 = p.scale_log2;
        bool aborted = false;
        int seg = 0;  // segments so far
        auto wait = [&](int i, int parity, int site) {
            if (!aborted && !__all_sync(0xffffffffu, mbar_wait(bar(i), parity, ab, site))) aborted = true;
            return !aborted;
        };
        for (int pos = begin; pos < end;) {
            // (each warp keeps its segment in shared memory: registers are for the scores)
            Segment& g = reinterpret_cast<Segment*>(smem + L::OFF_SEG)[warp];
            {
                const Segment found = segment_at(p, pre, pos, end, e);
                if (lane == 0) g = found;
                __syncwarp();
                pos = found.next;
            }
            if (g.count == 0) {
                __syncwarp();
                continue;
            }
            const int row0 = g.rt * p.RT, ta = p.by_G.div(row0), r = row0 + lr;
            {
                // this row's Q, half of the columns each group, turned and split, into TMEM
#pragma unroll 1
                for (int c0 = w * (DP / 16); c0 < (w + 1) * (DP / 16); c0 += 4) {
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint4 h, l;
                        load_q_chunk<E>(p, g, r, c0 + c, h, l);
                        hi[4 * c] = h.x;
                        hi[4 * c + 1] = h.y;
                        hi[4 * c + 2] = h.z;
                        hi[4 * c + 3] = h.w;
                        lo[4 * c] = l.x;
                        lo[4 * c + 1] = l.y;
                        lo[4 * c + 2] = l.z;
                        lo[4 * c + 3] = l.w;
                    }
                    __syncwarp();
                    tmem_st_x16(tmem + lanes + L::QHI + 4 * c0, hi);
                    tmem_st_x16(tmem + lanes + L::QLO + 4 * c0, lo);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(L::Q_FULL));
            }
            if (p.mask != nullptr) {
                build_mask(p, g, words, ctx_lo, threadIdx.x, 32 * L::NSW);
                named_bar_sync(1, 32 * L::NSW);
            }
            int rlo, rhi;
            row_limits(p, g, r, ta, ctx_lo, rlo, rhi);
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
                if (!wait(L::S_FULL + sb, i / L::NSB & 1, 0x701)) continue;
                tc_fence_after();
                // 32 scores at a time, so that the row fits the 128 registers of 512 threads: the
                // upper half for the maximum, then the lower half, which stays for its exponentials;
                // the upper half is read once more
                float mx = -INFINITY;
                uint32_t raw[32];
                float* x = reinterpret_cast<float*>(raw);
                uint32_t see[2] = {~0u, ~0u};
                bool edge = false;
                auto load_half = [&](int h) {
                    tmem_ld_x32(tS + 32 * h, raw);
                    if (edge) {
#pragma unroll
                        for (int c = 0; c < 32; ++c)
                            if (!(see[h] >> c & 1u)) x[c] = -INFINITY;
                    }
                };
                if (!idle) {
                    int k0, valid;
                    tile_keys(p, tile0 + i, k0, valid);
                    edge = valid < KT || k0 < all_lo || k0 + KT > all_hi;
                    if (edge) {
                        uint64_t bits = bits_between(rlo - k0, min(rhi - k0, valid));
                        if (p.mask != nullptr && k0 + KT > L0)
                            bits &= bits_between(0, L0 - k0) | draft_bits(words + rw, nw, k0 - L0);
                        see[0] = static_cast<uint32_t>(bits);
                        see[1] = static_cast<uint32_t>(bits >> 32);
                    }
                    load_half(1);
                    mx = max32(x);
                    load_half(0);
                    mx = fmaxf(mx, max32(x)) * sl2;
                }
                // the reference that the tile before left (the first tile of a segment has none)
                if (i > i0 && !wait(L::TOKEN + (w ^ 1) * 4 + quad, (i - 1) / 2 & 1, 0x703)) continue;
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
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (h == 1) load_half(1);
#pragma unroll
                        for (int c0 = 0; c0 < 32; c0 += 16) {
                            uint32_t pk[8];
#pragma unroll
                            for (int c = 0; c < 16; c += 2) {
                                float a0, a1;
                                f2_split(ffma2(f2(x[c0 + c], x[c0 + c + 1]), mul2, nm2), a0, a1);
                                const float p0 = ex2(a0), p1 = ex2(a1);
                                ls[(c >> 1) & 3] = fadd2(ls[(c >> 1) & 3], f2(p0, p1));
                                pk[c / 2] = E::pack(p0, p1);
                            }
                            // (columns whose scores have been read already)
                            tmem_st_x8(tS + 16 * h + c0 / 2, pk);
                        }
                    }
                    float s0, s1;
                    f2_split(fadd2(fadd2(ls[0], ls[1]), fadd2(ls[2], ls[3])), s0, s1);
                    l += s0 + s1;
                    tmem_wait_st();
                    tc_fence_before();
                }
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
            if (g.first == 0 && threadIdx.x == 0) describe_unit(p, sched, g, begin);
            if (!aborted && !*abort_flag && !__all_sync(0xffffffffu, r >= p.rows)) {
                const float M = dead ? -INFINITY : m;
                const float lsum = dead ? 0.f : sums[lr] + sums[L::RT + lr];
                const bool whole = g.count == g.s.n;
                const float inv = whole ? (lsum == 0.f ? 0.f : 1.f / lsum) : 1.f;
                float* slot = partial_slot(p, segment_slot(g, begin));
                const int t = p.by_G.div(r);
                uint16_t* out = p.o + g.b * p.osb + (g.kvh * p.G + r - t * p.G) * p.osh + t * p.oss;
                for (int c0 = w * (DP / 2); c0 < (w + 1) * (DP / 2); c0 += 32) {
                    uint32_t raw[32];
                    __syncwarp();
                    tmem_ld_x32(tO + c0, raw);
                    float o[32];
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = M == -INFINITY ? 0.f : __uint_as_float(raw[k]) * inv;
                    if (r < p.rows) {
#pragma unroll
                        for (int k = 0; k < 32; k += 8) {
                            if (c0 + k >= p.D) break;
                            if (whole) {
                                *reinterpret_cast<uint4*>(out + c0 + k) =
                                    uint4{E::pack(o[k], o[k + 1]), E::pack(o[k + 2], o[k + 3]),
                                          E::pack(o[k + 4], o[k + 5]), E::pack(o[k + 6], o[k + 7])};
                            } else {
                                float4* d = reinterpret_cast<float4*>(slot) + (c0 + k) / 4 * p.RT + lr;
                                d[0] = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                                d[p.RT] = make_float4(o[k + 4], o[k + 5], o[k + 6], o[k + 7]);
                            }
                        }
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
