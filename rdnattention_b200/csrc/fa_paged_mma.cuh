// The many-rows kernel of the paged attention: row tiles of 128 on tcgen05.
//
// Trees of drafted tokens and chunks of prompts bring 17 to hundreds of rows per KV
// head.  Per 64-key tile of head_dim 128 an SM receives 32 KB (about 1340 cycles of
// its share of the HBM bandwidth), and 128 rows need 8192 exponentials (512 cycles)
// and three products of 128 cycles, so a tile of rows is HBM-bound as long as the
// softmax keeps up; more row tiles read the same keys again, mostly from L2.
//
//   warps 0..3, 4..7   two softmax groups (thread = row = TMEM lane); key tile i of
//                      the CTA goes to group i & 1, each with its own S, O, m and l,
//                      so one group's softmax runs while the other's products do
//   warps 8..11        producers (produce(), as in the few-rows kernel)
//   warps 12, 13       one MMA-issuing lane for each group
//
// TMEM (512 columns at head_dim 128): Q hi and lo as the A operand of S = Q K^T
// (hi + lo, see the few-rows kernel: a query in shared memory would be read again by
// every product, 256 cycles each, and take 64 KB from the ring), S_0, S_1 (P over S
// in place, the A operand of O += P V), O_0, O_1.
// At the end of a segment the two groups' (O, m, l) join in the epilogue, each group
// taking half of the columns.
#pragma once

#include "fa_paged.cuh"

namespace rdna {
namespace paged {

template <int DP>
struct MmaLayout {
    static constexpr int NPW = 4;
    static constexpr int NSW = 8;                       // softmax warps
    static constexpr int THREADS = 32 * (NSW + NPW + 4);
    // Registers: launched with LAUNCH_REGS per thread (16 warps fill the register file),
    // moved to the softmax warps, which hold 64 scores each.
    static constexpr int LAUNCH_REGS = 128, SOFTMAX_REGS = 160, OTHER_REGS = 96;
    static_assert(NSW * SOFTMAX_REGS + (NPW + 4) * OTHER_REGS <= (NSW + NPW + 4) * LAUNCH_REGS,
                  "register split exceeds the launch allocation");
    static constexpr int NBOX = DP / 64;
    static constexpr int BOX_BYTES = KT * 128;
    static constexpr int TILE = NBOX * BOX_BYTES;
    static constexpr int STAGE = 2 * TILE;
    static constexpr int NST = 6;
    static_assert(NST % 2 == 0, "a ring slot belongs to one softmax group");
    static constexpr int RT = 128;
    static constexpr int NW = kMaxTree / 32;
    // barriers (8 bytes each): full [NST], empty [NST], then
    static constexpr int S_FULL = 2 * NST, P_FULL = S_FULL + 2, O_FULL = P_FULL + 2, Q_FULL = O_FULL + 2,
                         DRAIN = Q_FULL + 2, N_BARS = DRAIN + 2;
    static constexpr int OFF_TMEM = 8 * N_BARS, OFF_ABORT = OFF_TMEM + 4;
    static constexpr int OFF_RING = 1024;
    static constexpr int OFF_MASK = OFF_RING + NST * STAGE;  // [RT][NW + 2] (two words of padding), then [RT]
    static constexpr int OFF_ML = OFF_MASK + RT * NW * 4 + RT * 4;  // [2][RT] (m, l)
    static constexpr int OFF_SEG = OFF_ML + 2 * RT * 8;  // [NSW] Segment
    static constexpr int OFF_PRE = OFF_SEG + NSW * 64;
    static_assert(sizeof(Segment) <= 64, "a segment's slot");
    static constexpr int SMEM_BYTES = OFF_PRE + kMaxBatch * 4 + 1024;  // + alignment slack
    static_assert(SMEM_BYTES <= 232448, "shared memory of one CTA");
    // TMEM columns
    static constexpr int QHI = 0, QLO = DP / 2, S0 = DP, O0 = S0 + 2 * KT, TMEM_USED = O0 + 2 * DP;
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

// Row max of 64 values: 8 chains of three-input max.
__device__ __forceinline__ float max64(const float* x) {
    float m[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) m[i] = fmaxf(x[i], x[i + 8]);
#pragma unroll
    for (int c = 16; c < 64; c += 16)
#pragma unroll
        for (int i = 0; i < 8; ++i) m[i] = fmax3(m[i], x[c + i], x[c + 8 + i]);
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
        for (int w = 0; w < 2; ++w) {
            mbar_init(bar(L::S_FULL + w), 1);
            mbar_init(bar(L::P_FULL + w), 4);
            mbar_init(bar(L::O_FULL + w), 1);
            mbar_init(bar(L::Q_FULL + w), L::NSW);
            mbar_init(bar(L::DRAIN + w), 1);
        }
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

    int i0 = 0, b = 0;  // running tile number of the segment's first tile
    if (producer) {
        regs_decrease<L::OTHER_REGS>();
        for (int pos = begin; pos < end;) {
            const Segment g = segment_at(p, pre, pos, end, b);
            if (!produce<L>(p, g, i0, bars, smem_u32(ring), ab, threadIdx.x - 32 * L::NSW)) break;
            i0 += g.count;
            pos = g.next;
        }
        cp_async_wait_all();  // after an expired wait too, no copy outlives the CTA
    } else if (warp >= L::NSW + L::NPW) {
        // ------------------------------------------------------------ MMA issuers
        regs_decrease<L::OTHER_REGS>();
        const int w = warp - (L::NSW + L::NPW);
        if (w < 2) {
            constexpr uint32_t IDESC_QK = instr_desc(1u, AbFormat<E>::value, 0u, 128, KT);
            constexpr uint32_t IDESC_PV = instr_desc(1u, AbFormat<E>::value, 1u, 128, DP);
            const uint32_t tS = tmem + L::S0 + w * KT, tO = tmem + L::O0 + w * DP;
            const uint64_t kd = smem_desc(smem_u32(ring), 16, 1024, 2);
            const uint64_t vd = smem_desc(smem_u32(ring + L::TILE), L::BOX_BYTES, 1024, 2);
            int seg = 0, n = 0;  // segments with a tile of this group, and its tiles, so far
            int ok = 1;
            for (int pos = begin; pos < end && ok;) {
                const Segment g = segment_at(p, pre, pos, end, b);
                const int first = i0 + ((w - i0) & 1);
                if (lane == 0 && first < i0 + g.count) {
                    // (signalled only for segments with a tile of this group: no phase passes
                    // that this thread does not see)
                    ok = mbar_wait(bar(L::Q_FULL + w), seg++ & 1, ab, 0x711);
                    tc_fence_after();
                    for (int i = first; ok && i < i0 + g.count; i += 2, ++n) {
                        const int s = i % L::NST;
                        const uint32_t slot = static_cast<uint32_t>(s * L::STAGE) >> 4;
                        ok = mbar_wait(bar(s), i / L::NST & 1, ab, 0x712);
                        if (!ok) break;
                        // the copies were written through the generic proxy, the products read
                        // through the async one
                        fence_proxy_async_smem();
                        tc_fence_after();
#pragma unroll
                        for (int half = 0; half < 2; ++half)
#pragma unroll
                            for (int kk = 0; kk < DP / 16; ++kk)
                                mma_f16_ts(tS, tmem + (half ? L::QLO : L::QHI) + kk * 8,
                                           kd + slot + static_cast<uint32_t>((kk / 4 * L::BOX_BYTES + kk % 4 * 32) >> 4),
                                           IDESC_QK, half || kk > 0);
                        tc_commit(bar(L::S_FULL + w));
                        ok = mbar_wait(bar(L::P_FULL + w), n & 1, ab, 0x713);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll
                        for (int kk = 0; kk < KT / 16; ++kk)
                            mma_f16_ts(tO, tS + kk * 8, vd + slot + static_cast<uint32_t>((kk * 16 * 128) >> 4), IDESC_PV,
                                       kk > 0 || i > first);
                        tc_commit(bar(L::NST + s));
                        if (i + 2 >= i0 + g.count) tc_commit(bar(L::O_FULL + w));
                    }
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
                i0 += g.count;
                pos = g.next;
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
        regs_increase<L::SOFTMAX_REGS>();
        const int w = warp / 4, quad = warp % 4, lr = quad * 32 + lane;  // row of the tile
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        const uint32_t tS = tmem + lanes + L::S0 + w * KT, tO = tmem + lanes + L::O0;
        uint32_t* words = reinterpret_cast<uint32_t*>(smem + L::OFF_MASK);
        int* ctx_lo = reinterpret_cast<int*>(smem + L::OFF_MASK + L::RT * L::NW * 4);
        float2* ml = reinterpret_cast<float2*>(smem + L::OFF_ML);
        const int nw = (p.t.T + 31) / 32;
        const float sl2 = p.scale_log2;
        bool aborted = false;
        int n = 0, n_o = 0;  // tiles, and segments with a tile, of this group so far
        auto wait = [&](int i, int parity, int site) {
            if (!aborted && !__all_sync(0xffffffffu, mbar_wait(bar(i), parity, ab, site))) aborted = true;
            return !aborted;
        };
        for (int pos = begin; pos < end;) {
            // (each warp keeps its segment in shared memory: registers are for the scores)
            Segment& g = reinterpret_cast<Segment*>(smem + L::OFF_SEG)[warp];
            {
                const Segment found = segment_at(p, pre, pos, end, b);
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
                    tmem_st_x16(tmem + lanes + L::QHI + 4 * c0, hi);
                    tmem_st_x16(tmem + lanes + L::QLO + 4 * c0, lo);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    for (int k = 0; k < 2; ++k)
                        if (((k - i0) & 1) < g.count) mbar_arrive(bar(L::Q_FULL + k));
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
            for (int i = first; i < behind; i += 2, ++n) {
                if (!wait(L::S_FULL + w, n & 1, 0x701)) continue;
                if (!idle) {
                    tc_fence_after();
                    int k0, valid;
                    tile_keys(p, tile0 + i, k0, valid);
                    uint32_t raw[KT];
                    tmem_ld_x64(tS, raw);
                    float* x = reinterpret_cast<float*>(raw);
                    if (valid < KT || k0 < all_lo || k0 + KT > all_hi) {
                        uint64_t see = bits_between(rlo - k0, min(rhi - k0, valid));
                        if (p.mask != nullptr && k0 + KT > L0)
                            see &= bits_between(0, L0 - k0) | draft_bits(words + rw, nw, k0 - L0);
                        const uint32_t see0 = static_cast<uint32_t>(see), see1 = static_cast<uint32_t>(see >> 32);
#pragma unroll
                        for (int c = 0; c < 32; ++c) {
                            if (!(see0 >> c & 1u)) x[c] = -INFINITY;
                            if (!(see1 >> c & 1u)) x[32 + c] = -INFINITY;
                        }
                    }
                    const float mx = max64(x) * sl2;
                    // O is rescaled only when the maximum grows by more than 2^8: the row's final
                    // 1 / l uses the same reference, and p stays below 2^8
                    const bool grow = fmaxf(m, mx) > m + 8.f;
                    if (__any_sync(0xffffffffu, grow)) {
                        const float corr = grow ? ex2(m - fmaxf(m, mx)) : 1.f;
                        if (grow) {
                            m = fmaxf(m, mx);
                            l *= corr;
                        }
                        // (S of this tile was committed after the group's previous P V)
                        if (i > first)
#pragma unroll 1
                            for (int c0 = 0; c0 < DP; c0 += 16) {
                                uint32_t o[16];
                                tmem_ld_x16(tO + w * DP + c0, o);
#pragma unroll
                                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                                tmem_st_x16(tO + w * DP + c0, o);
                            }
                    }
                    // P is rounded to the cache's type, the operand type of the second product;
                    // the row sums take it unrounded
                    const float nm = m == -INFINITY ? 0.f : -m;
                    const uint64_t mul2 = f2(sl2, sl2), nm2 = f2(nm, nm);
                    uint64_t ls[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
                    for (int c0 = 0; c0 < KT; c0 += 16) {
                        uint32_t pk[8];
#pragma unroll
                        for (int c = 0; c < 16; c += 2) {
                            float a0, a1;
                            f2_split(ffma2(f2(x[c0 + c], x[c0 + c + 1]), mul2, nm2), a0, a1);
                            const float p0 = ex2(a0), p1 = ex2(a1);
                            ls[(c >> 1) & 3] = fadd2(ls[(c >> 1) & 3], f2(p0, p1));
                            pk[c / 2] = E::pack(p0, p1);
                        }
                        tmem_st_x8(tS + c0 / 2, pk);
                    }
                    float s0, s1;
                    f2_split(fadd2(fadd2(ls[0], ls[1]), fadd2(ls[2], ls[3])), s0, s1);
                    l += s0 + s1;
                    tmem_wait_st();
                    tc_fence_before();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(L::P_FULL + w));
            }
            // ------------------------------------------------------------ epilogue
            if (first < behind) wait(L::O_FULL + w, n_o++ & 1, 0x702);
            ml[w * L::RT + lr] = dead ? make_float2(-INFINITY, 0.f) : make_float2(m, l);
            tc_fence_before();
            named_bar_sync(1, 32 * L::NSW);
            tc_fence_after();
            if (g.first == 0 && threadIdx.x == 0) describe_unit(p, sched, g, begin);
            if (!aborted && !*abort_flag && !__all_sync(0xffffffffu, r >= p.rows)) {
                const float2 a = ml[lr], c = ml[L::RT + lr];
                const float M = fmaxf(a.x, c.x);
                const float fa = a.x == -INFINITY ? 0.f : ex2(a.x - M), fc = c.x == -INFINITY ? 0.f : ex2(c.x - M);
                const float lsum = fa * a.y + fc * c.y;
                const bool whole = g.count == g.s.n;
                const float inv = whole ? (lsum == 0.f ? 0.f : 1.f / lsum) : 1.f;
                float* slot = partial_slot(p, segment_slot(g, begin));
                const int t = p.by_G.div(r);
                uint16_t* out = p.o + g.b * p.osb + (g.kvh * p.G + r - t * p.G) * p.osh + t * p.oss;
                for (int c0 = w * (DP / 2); c0 < (w + 1) * (DP / 2); c0 += 32) {
                    uint32_t oa[32], oc[32];
                    tmem_ld_x32(tO + c0, oa);
                    tmem_ld_x32(tO + DP + c0, oc);
                    // (a group without a tile, or a row without a key, left its O undefined)
                    float o[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        o[e] = ((a.x == -INFINITY ? 0.f : fa * __uint_as_float(oa[e])) +
                                (c.x == -INFINITY ? 0.f : fc * __uint_as_float(oc[e]))) * inv;
                    if (r < p.rows) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            if (c0 + e >= p.D) break;
                            if (whole) {
                                *reinterpret_cast<uint4*>(out + c0 + e) =
                                    uint4{E::pack(o[e], o[e + 1]), E::pack(o[e + 2], o[e + 3]),
                                          E::pack(o[e + 4], o[e + 5]), E::pack(o[e + 6], o[e + 7])};
                            } else {
                                float4* d = reinterpret_cast<float4*>(slot) + (c0 + e) / 4 * p.RT + lr;
                                d[0] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                                d[p.RT] = make_float4(o[e + 4], o[e + 5], o[e + 6], o[e + 7]);
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
