// Attention of T new tokens per sequence over a paged KV cache (decode, chains
// of tokens, trees of drafted tokens).
//
// Rows: the G = H / Hkv query heads of a KV head times the T tokens, row r =
// (token r / G, head r % G), so every K/V byte serves the whole group.  What row
// (t, g) of sequence b sees, with L = cache_lens[b] and n = new_lens[b]:
//   chain  slots [0, L + t]
//   tree   slots [0, L) and the drafted slots L + u with mask[b][t][u], u < n
// and with a window w only the newest w of those: its drafted tokens (in index
// order, parents before children) first, then the newest of the context.
// Rows t >= n and rows that see nothing are written as zeros.
//
// Work: a unit = (sequence, KV head, tile of RT rows) times the key tiles that
// some row of it sees.  The tiles of all units form one list, and CTA c takes
// the c-th equal part of it: every CTA streams the same number of bytes whatever
// the lengths are, and the lengths stay on the device (a captured graph replays
// with new ones).  A unit that lies inside one CTA is finished there; the parts
// of the others go to a workspace as (O, m, l) in fp32 and the combine kernel
// joins them in list order, so results do not depend on timing.
#pragma once

#include <cuda.h>
#include <limits.h>
#include <math.h>

#include "paged.cuh"

namespace rdna {
namespace paged {

constexpr int kMaxTree = 256;          // drafted tokens under a mask
constexpr int kMaxBatch = 1024;        // sequences per launch (the host splits larger batches)
constexpr int kMinTiles = 4;           // tiles per CTA below which fewer CTAs take part

struct AttnParams {
    const uint16_t* q;
    uint16_t* o;
    int64_t qsb, qsh, qss, osb, osh, oss;
    Table t;
    const uint8_t* mask;  // [B][T][T] bool or null: chain
    int64_t msb, mst;
    const int* positions;  // [B][T] or null: cache_lens[b] + t
    const float *cos, *sin;
    int rope_rows;
    int B, H, Hkv, G, D;
    int rows;    // T * G
    int RT;      // rows per tile
    int n_rt;    // row tiles
    int KT;      // keys per tile
    int tpp;     // tiles per page (pages of at least KT slots), else 0: KT / P pages per tile
    int window;  // 0: none
    float scale_log2;
    float* ws;   // partials: 2 per CTA, each O [RT][D], m [RT], l [RT]
    int grid;    // CTAs of the attention kernel
};

// ---------------------------------------------------------------- the schedule
struct Span {
    int lo, hi;  // keys some row of the tile sees: [lo, hi)
    int t0, n;   // first key tile and their number
};

// Tile that holds key j.
__device__ __forceinline__ int tile_of(const AttnParams& p, int j) {
    if (p.tpp == 0) return j / p.KT;
    int page, row;
    p.t.split(j, page, row);
    return page * p.tpp + row / p.KT;
}

__device__ __forceinline__ Span row_tile_span(const AttnParams& p, int L, int n, int rt) {
    const int cap = p.t.cap();
    const int ta = rt * p.RT / p.G;  // tokens of the tile: [ta, tb]
    const int tb = min((min((rt + 1) * p.RT, p.rows) - 1) / p.G, n - 1);
    Span s{0, 0, 0, 0};
    if (ta >= n) return s;  // padding rows only
    s.hi = min(p.mask != nullptr ? L + n : L + tb + 1, cap);
    if (p.window > 0) s.lo = max(0, p.mask != nullptr ? L - p.window : L + ta + 1 - p.window);
    if (s.lo >= s.hi) return s;
    s.t0 = tile_of(p, s.lo);
    s.n = tile_of(p, s.hi - 1) + 1 - s.t0;
    return s;
}

// Tiles of one KV head of sequence b over all row tiles.
__device__ __forceinline__ int head_tiles(const AttnParams& p, int b) {
    const int L = p.t.len(b), n = p.t.news(b);
    int w = 0;
    for (int rt = 0; rt < p.n_rt; ++rt) w += row_tile_span(p, L, n, rt).n;
    return w;
}

// Fills pre[0 .. B] with the exclusive prefix sums of the sequences' tiles (all
// threads of the block; ends with a barrier).
__device__ __forceinline__ void schedule_prefix(const AttnParams& p, int* pre) {
    for (int b = threadIdx.x; b < p.B; b += blockDim.x) pre[b + 1] = head_tiles(p, b) * p.Hkv;
    __syncthreads();
    if (threadIdx.x < 32) {
        int carry = 0;
        for (int b0 = 0; b0 < p.B; b0 += 32) {
            const int b = b0 + threadIdx.x;
            int v = b < p.B ? pre[b + 1] : 0;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const int u = __shfl_up_sync(0xffffffffu, v, d);
                if (threadIdx.x >= d) v += u;
            }
            v += carry;
            if (b < p.B) pre[b + 1] = v;
            carry = __shfl_sync(0xffffffffu, v, 31);
        }
        if (threadIdx.x == 0) pre[0] = 0;
    }
    __syncthreads();
}

// CTAs that take part, and the first list position of CTA c.
__device__ __forceinline__ int active_ctas(const AttnParams& p, int total) {
    return min(p.grid, max(1, total / kMinTiles));
}
__device__ __forceinline__ int cta_begin(int c, int total, int ctas) {
    return static_cast<int>(static_cast<int64_t>(c) * total / ctas);
}
__device__ __forceinline__ int cta_of(int pos, int total, int ctas) {
    return static_cast<int>(((static_cast<int64_t>(pos) + 1) * ctas - 1) / total);
}

// One unit's share of a CTA: list positions [pos, pos + count) are the unit's
// tiles first .. first + count - 1.
struct Segment {
    int b, kvh, rt, L, n;
    Span s;
    int first, count;
};

__device__ __forceinline__ Segment segment_at(const AttnParams& p, const int* pre, int pos, int end, int& b) {
    while (pre[b + 1] <= pos) ++b;  // pos < total, so b stays below B
    Segment g;
    g.b = b;
    g.L = p.t.len(b);
    g.n = p.t.news(b);
    const int per_head = (pre[b + 1] - pre[b]) / p.Hkv;
    int off = pos - pre[b];
    g.kvh = off / per_head;
    off -= g.kvh * per_head;
    g.rt = 0;
    g.s = row_tile_span(p, g.L, g.n, 0);
    while (off >= g.s.n) {
        off -= g.s.n;
        ++g.rt;
        g.s = row_tile_span(p, g.L, g.n, g.rt);
    }
    g.first = off;
    g.count = min(g.s.n - off, end - pos);
    return g;
}

// First key of a tile and how many of its KT rows are keys (a page may end
// inside a tile; the rows behind its end are zero fill).
__device__ __forceinline__ void tile_keys(const AttnParams& p, int tile, int& k0, int& valid) {
    if (p.tpp == 0) {
        k0 = tile * p.KT;
        valid = p.KT;
    } else {
        const int page = tile / p.tpp, off = (tile - page * p.tpp) * p.KT;
        k0 = page * p.t.P + off;
        valid = min(p.KT, p.t.P - off);
    }
}

__device__ __forceinline__ float* partial_slot(const AttnParams& p, int slot) {
    return p.ws + static_cast<int64_t>(slot) * p.RT * (p.D + 2);
}

// Bits of the drafted tokens that the tokens of a row tile see: words[i * nw + w]
// for token ta + i, mask bytes to bits by ballot; then the window drops the
// lowest.  rlo_ctx[i] = first context slot token ta + i sees.  Threads
// tid .. of `nthreads` (whole warps) take part; the caller synchronises them.
__device__ __forceinline__ void build_mask(const AttnParams& p, const Segment& g, uint32_t* words, int* ctx_lo,
                                           int tid, int nthreads) {
    const int nw = (p.t.T + 31) / 32;
    const int ta = g.rt * p.RT / p.G;
    const int nt = min((min((g.rt + 1) * p.RT, p.rows) - 1) / p.G, g.n - 1) - ta + 1;
    const int lane = tid & 31;
    for (int i = tid / 32; i < nt; i += nthreads / 32) {
        const uint8_t* row = p.mask + g.b * p.msb + (ta + i) * p.mst;
        uint32_t mine = 0;  // lane w holds word w
        int seen = 0;
        for (int w = 0; w < nw; ++w) {
            const int u = 32 * w + lane;
            const uint32_t bits = __ballot_sync(0xffffffffu, u < g.n && row[u] != 0);
            seen += __popc(bits);
            if (lane == w) mine = bits;
        }
        int keep = seen;
        if (p.window > 0 && seen > p.window) {
            // drop the lowest seen - window bits
            int drop = seen - p.window;
            keep = p.window;
            for (int w = 0; w < nw; ++w) {
                uint32_t bits = __shfl_sync(0xffffffffu, mine, w);
                while (drop > 0 && bits != 0) {
                    bits &= bits - 1;
                    --drop;
                }
                if (lane == w) mine = bits;
            }
        }
        if (lane < nw) words[i * nw + lane] = mine;
        if (lane == 0) ctx_lo[i] = p.window > 0 ? max(0, g.L - (p.window - keep)) : 0;
    }
}

// ------------------------------------------------------------- the join kernel
// One warp per row of a split unit: O = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i
// over the CTAs that hold a part, in list order.  Units with no visible key get
// their zeros here; whole units were written by the attention kernel.
constexpr int kJoinWarps = 8;

template <class E>
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const __grid_constant__ AttnParams p) {
    __shared__ int pre[kMaxBatch + 1];
    grid_dependency_wait();
    schedule_prefix(p, pre);
    const int total = pre[p.B];
    const int ctas = active_ctas(p, total);
    const int groups = (p.RT + kJoinWarps - 1) / kJoinWarps;
    const int unit = blockIdx.x / groups;  // (b, kvh, rt)
    const int rt = unit % p.n_rt, kvh = unit / p.n_rt % p.Hkv, b = unit / p.n_rt / p.Hkv;
    const int lr = blockIdx.x % groups * kJoinWarps + threadIdx.x / 32;  // row of the tile
    const int r = rt * p.RT + lr;
    if (lr >= p.RT || r >= p.rows) return;
    const int L = p.t.len(b), n = p.t.news(b);
    int pos = pre[b], per_head = 0, before = 0, tiles = 0;
    for (int i = 0; i < p.n_rt; ++i) {
        const int w = row_tile_span(p, L, n, i).n;
        if (i < rt) before += w;
        if (i == rt) tiles = w;
        per_head += w;
    }
    pos += kvh * per_head + before;
    const int t = r / p.G, h = kvh * p.G + r % p.G;
    uint16_t* out = p.o + b * p.osb + h * p.osh + t * p.oss;
    const int lane = threadIdx.x & 31;
    if (tiles == 0) {
        for (int d = lane * 4; d < p.D; d += 128) *reinterpret_cast<uint2*>(out + d) = uint2{0u, 0u};
        return;
    }
    const int c0 = cta_of(pos, total, ctas), c1 = cta_of(pos + tiles - 1, total, ctas);
    if (c0 == c1) return;
    auto part = [&](int c) { return partial_slot(p, 2 * c + (pos <= cta_begin(c, total, ctas) ? 0 : 1)); };
    float M = -INFINITY;
    for (int c = c0; c <= c1; ++c) M = fmaxf(M, part(c)[p.RT * p.D + lr]);
    float l = 0.f;
    float4 o[2] = {};
    for (int c = c0; c <= c1; ++c) {
        const float* w = part(c);
        const float m = w[p.RT * p.D + lr];
        const float f = m == -INFINITY ? 0.f : ex2(m - M);
        l += f * w[p.RT * p.D + p.RT + lr];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int d = lane * 4 + 128 * i;
            if (d < p.D) {
                const float4 x = *reinterpret_cast<const float4*>(w + lr * p.D + d);
                o[i].x += f * x.x;
                o[i].y += f * x.y;
                o[i].z += f * x.z;
                o[i].w += f * x.w;
            }
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int d = lane * 4 + 128 * i;
        if (d < p.D)
            *reinterpret_cast<uint2*>(out + d) =
                uint2{E::pack(o[i].x * inv, o[i].y * inv), E::pack(o[i].z * inv, o[i].w * inv)};
    }
}

// -------------------------------------------------------- the few-rows kernel
// Up to 64 rows per tile as row groups of 16, each the M = 16 of m16n8k16.
//   warp 4       TMA producer: 32-key tiles of K and V through an NST-stage ring
//   warps 0..3   consumers, tile i -> warps of class i % (4 / NRG), one per row
//                group: S = Q K^T and O += P V on mma.sync with the online
//                softmax in registers
// The bound is HBM as long as the rows are few: per 32-key tile of head_dim 128
// a CTA moves 16 KB (about 670 cycles of its share of the bandwidth) and needs
// NRG * 128 MMAs on four schedulers.
constexpr int KT = 32;
constexpr int NCW = 4;
constexpr int THREADS = 32 * (NCW + 1);

template <int DP>
struct Layout {
    static constexpr int NBOX = DP / 64;  // 64-element boxes (128 B, SWIZZLE_128B)
    static constexpr int BOX_BYTES = KT * 128;
    static constexpr int TILE = NBOX * BOX_BYTES;
    static constexpr int STAGE = 2 * TILE;
    static constexpr int NST = DP <= 128 ? 8 : 4;
    static_assert(NST % NCW == 0, "each ring slot has one class of consumer warps");
    static constexpr int MAX_RG = DP <= 128 ? 4 : 2;
    static constexpr int RT = 16 * MAX_RG;
    static constexpr int PSTR = DP + 4;  // floats per partial row: O, m, l, padding
    static constexpr int OFF_RING = 1024;
    static constexpr int OFF_Q = OFF_RING + NST * STAGE;              // [RT][DP], swizzled like a K tile
    static constexpr int OFF_PART = OFF_Q + NBOX * RT * 128;          // [NCW][16][PSTR] fp32
    static constexpr int OFF_MASK = OFF_PART + NCW * 16 * PSTR * 4;   // [RT][kMaxTree / 32], then [RT]
    static constexpr int OFF_PRE = OFF_MASK + RT * (kMaxTree / 32) * 4 + RT * 4;
    static constexpr int SMEM_BYTES = OFF_PRE + (kMaxBatch + 1) * 4 + 1024;  // + alignment slack
    static_assert(SMEM_BYTES <= 232448, "shared memory of one CTA");
};

// Byte offset of 16-byte chunk c of row r in a tile of `rows` rows (64-element
// boxes one after the other, 128-byte swizzle).
__device__ __forceinline__ uint32_t chunk_off(int rows, int r, int c) {
    return static_cast<uint32_t>((c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <class E>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<F16>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<BF16>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Loads (and turns) one 16-byte chunk of row r of a row tile; zeros for rows
// that are padding or whose position lies outside the tables.
template <class E>
__device__ __forceinline__ uint4 load_q_chunk(const AttnParams& p, const Segment& g, int r, int ch) {
    const int t = r / p.G;
    if (r >= p.rows || t >= g.n || ch * 8 >= p.D) return uint4{0u, 0u, 0u, 0u};
    uint4 x = *reinterpret_cast<const uint4*>(p.q + g.b * p.qsb + (g.kvh * p.G + r % p.G) * p.qsh + t * p.qss + ch * 8);
    if (p.cos != nullptr) {
        const int pos = p.positions != nullptr ? p.positions[static_cast<int64_t>(g.b) * p.t.T + t] : g.L + t;
        if (static_cast<unsigned>(pos) >= static_cast<unsigned>(p.rope_rows)) return uint4{0u, 0u, 0u, 0u};
        const int64_t at = static_cast<int64_t>(pos) * (p.D / 2) + ch * 4;
        x = rotate4<E>(x, __ldg(reinterpret_cast<const float4*>(p.cos + at)),
                       __ldg(reinterpret_cast<const float4*>(p.sin + at)));
    }
    return x;
}

// Keys row r sees: [lo, hi), and with a mask the drafted slots from L on by bit.
// A row that is padding, or whose position lies outside the tables, sees none.
__device__ __forceinline__ void row_limits(const AttnParams& p, const Segment& g, int r, const int* ctx_lo, int& lo,
                                           int& hi) {
    const int t = r / p.G;
    bool ok = r < p.rows && t < g.n;
    if (ok && p.cos != nullptr) {
        const int pos = p.positions != nullptr ? p.positions[static_cast<int64_t>(g.b) * p.t.T + t] : g.L + t;
        ok = static_cast<unsigned>(pos) < static_cast<unsigned>(p.rope_rows);
    }
    if (!ok) {
        lo = 1;
        hi = 0;
    } else if (p.mask != nullptr) {
        lo = ctx_lo[t - g.rt * p.RT / p.G];
        hi = g.s.hi;
    } else {
        lo = p.window > 0 ? max(0, g.L + t + 1 - p.window) : 0;
        hi = min(g.L + t + 1, g.s.hi);
    }
}

template <class E, int DP>
__global__ void __launch_bounds__(THREADS, 1) fa_paged_kernel(const __grid_constant__ CUtensorMap tmK,
                                                              const __grid_constant__ CUtensorMap tmV,
                                                              const __grid_constant__ AttnParams p) {
    using L = Layout<DP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t bars = smem_u32(smem);
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (L::NST + s); };
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + 16 * L::NST);
    const Abort ab{abort_flag};
    uint8_t* ring = smem + L::OFF_RING;
    int* pre = reinterpret_cast<int*>(smem + L::OFF_PRE);

    const int NRG = p.RT / 16, NTG = NCW / NRG;
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < L::NST; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), NRG);
        }
        fence_barrier_init();
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    schedule_prefix(p, pre);  // its barriers also publish the mbarriers
    const int total = pre[p.B];
    const int ctas = active_ctas(p, total);
    if (total == 0 || static_cast<int>(blockIdx.x) >= ctas) return;
    const int begin = cta_begin(blockIdx.x, total, ctas), end = cta_begin(blockIdx.x + 1, total, ctas);

    if (warp == NCW) {
        // ------------------------------------------------------------ producer
        const uint64_t pol = policy_evict_first();
        const int box_rows = min(p.t.P, KT);
        const int ppt = p.tpp == 0 ? KT / p.t.P : 1;  // pages per tile
        int i = 0, b = 0;
        uint32_t filled = 0;  // slots that received a copy
        bool ok = true;
        for (int pos = begin; pos < end && ok;) {
            const Segment g = segment_at(p, pre, pos, end, b);
            const int* pages = p.t.pages + g.b * p.t.stride;
            int win = -1, ids = -1;  // 32 consecutive page table entries, one per lane
            for (int k = 0; k < g.count; ++k, ++i) {
                const int tile = g.s.t0 + g.first + k;
                const int lp0 = p.tpp == 0 ? tile * ppt : tile / p.tpp;
                const int row0 = p.tpp == 0 ? 0 : (tile - lp0 * p.tpp) * KT;
                if (lp0 / 32 != win) {
                    win = lp0 / 32;
                    const int e = win * 32 + lane;
                    ids = e < p.t.max_pages ? __ldg(pages + e) : -1;
                    if (static_cast<unsigned>(ids) >= static_cast<unsigned>(p.t.num_pages)) ids = -1;  // zero fill
                }
                const int s = i % L::NST, n = i / L::NST;
                if (lane == 0) ok = mbar_wait(empty_bar(s), (n & 1) ^ 1, ab, 0x601);
                ok = __shfl_sync(0xffffffffu, ok, 0);
                if (!ok) break;
                if (lane == 0) mbar_arrive_expect_tx(full_bar(s), L::STAGE);
                filled |= 1u << s;
                const uint32_t dst = smem_u32(ring + s * L::STAGE);
                for (int j = 0; j < ppt; ++j) {
                    const int page = __shfl_sync(0xffffffffu, ids, (lp0 + j) & 31);
                    if (lane == 0) {
                        const uint32_t d = dst + j * box_rows * 128;
#pragma unroll
                        for (int bx = 0; bx < L::NBOX; ++bx) {
                            tma_load_4d(d + bx * L::BOX_BYTES, &tmK, full_bar(s), bx * 64, row0, g.kvh, page, pol);
                            tma_load_4d(d + L::TILE + bx * L::BOX_BYTES, &tmV, full_bar(s), bx * 64, row0, g.kvh,
                                        page, pol);
                        }
                    }
                    __syncwarp();
                }
            }
            pos += g.count;
        }
        if (!ok && lane == 0) {
            // tile i was not issued; slot s last received tile j = the largest j < i with j % NST == s
            for (int s = 0; s < L::NST; ++s)
                if (filled >> s & 1u) {
                    const int j = (i - 1) - ((i - 1 - s) % L::NST + L::NST) % L::NST;
                    mbar_wait_drain(full_bar(s), (j / L::NST) & 1);
                }
        }
        __syncwarp();
        return;
    }

    // ---------------------------------------------------------------- consumers
    const int wrg = warp % NRG, wtg = warp / NRG;
    const int gq = lane >> 2, tq = lane & 3;
    uint32_t* words = reinterpret_cast<uint32_t*>(smem + L::OFF_MASK);
    int* ctx_lo = reinterpret_cast<int*>(smem + L::OFF_MASK + L::RT * (kMaxTree / 32) * 4);
    const int nw = (p.t.T + 31) / 32;
    const uint32_t qs = smem_u32(smem + L::OFF_Q);
    float* part = reinterpret_cast<float*>(smem + L::OFF_PART);
    const float sl2 = p.scale_log2;
    bool aborted = false;
    int i0 = 0, b = 0;  // running tile number of the segment's first tile
    for (int pos = begin; pos < end;) {
        const Segment g = segment_at(p, pre, pos, end, b);
        const int row0 = g.rt * p.RT;
        // Q of the row tile (rotated) into shared memory, and the mask bits
        for (int idx = threadIdx.x; idx < p.RT * (DP / 8); idx += 32 * NCW) {
            const int r = idx / (DP / 8), ch = idx % (DP / 8);
            *reinterpret_cast<uint4*>(smem + L::OFF_Q + chunk_off(p.RT, r, ch)) = load_q_chunk<E>(p, g, row0 + r, ch);
        }
        if (p.mask != nullptr) build_mask(p, g, words, ctx_lo, threadIdx.x, 32 * NCW);
        named_bar_sync(1, 32 * NCW);
        int rlo[2], rhi[2];
        const uint32_t* rw[2];
        for (int e = 0; e < 2; ++e) {
            const int r = row0 + wrg * 16 + gq + 8 * e;
            row_limits(p, g, r, ctx_lo, rlo[e], rhi[e]);
            rw[e] = words + (p.mask != nullptr && r < p.rows && r / p.G < g.n ? (r / p.G - row0 / p.G) * nw : 0);
        }
        // keys in [all_lo, all_hi) are seen by every row of the group that sees any; what the
        // others (padding, empty) add up there is dropped at the end of the segment
        const bool dead[2] = {rlo[0] >= rhi[0], rlo[1] >= rhi[1]};
        int all_lo = max(dead[0] ? 0 : rlo[0], dead[1] ? 0 : rlo[1]);
        int all_hi = min(dead[0] ? INT_MAX : rhi[0], dead[1] ? INT_MAX : rhi[1]);
        if (p.mask != nullptr) all_hi = min(all_hi, g.L);
        for (int d = 4; d < 32; d *= 2) {
            all_lo = max(all_lo, __shfl_xor_sync(0xffffffffu, all_lo, d));
            all_hi = min(all_hi, __shfl_xor_sync(0xffffffffu, all_hi, d));
        }
        uint32_t qa[DP <= 128 ? DP / 16 : 1][4];
        auto load_q = [&](int kk, uint32_t* a) {
            ldsm4(qs + chunk_off(p.RT, wrg * 16 + (lane & 15), 2 * kk + (lane >> 4)), a);
        };
        if constexpr (DP <= 128) {
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) load_q(kk, qa[kk]);
        }
        float oacc[DP / 8][4];
#pragma unroll
        for (int j = 0; j < DP / 8; ++j) oacc[j][0] = oacc[j][1] = oacc[j][2] = oacc[j][3] = 0.f;
        float m_run[2] = {-INFINITY, -INFINITY};
        float l_run[2] = {0.f, 0.f};

        // this warp's tiles of the segment: running numbers i with i % NTG == wtg
        for (int i = i0 + ((wtg - i0) % NTG + NTG) % NTG; i < i0 + g.count; i += NTG) {
            const int s = i % L::NST, n = i / L::NST;
            int k0, valid;
            tile_keys(p, g.s.t0 + g.first + (i - i0), k0, valid);
            bool ok = !aborted && mbar_wait(full_bar(s), n & 1, ab, 0x602);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {
                aborted = true;
                continue;
            }
            const uint32_t kb = smem_u32(ring + s * L::STAGE), vb = kb + L::TILE;
            const bool edge = valid < KT || k0 < all_lo || k0 + KT > all_hi;
            // slots no row of the unit sees may hold anything: V rows there become zeros (0 * NaN)
            const bool dirty = k0 < g.s.lo || k0 + KT > g.s.hi;
            if (dirty) {
                for (int idx = lane; idx < KT * (DP / 8); idx += 32) {
                    const int r = idx / (DP / 8);
                    if (k0 + r < g.s.lo || k0 + r >= g.s.hi)
                        *reinterpret_cast<uint4*>(ring + s * L::STAGE + L::TILE + chunk_off(KT, r, idx % (DP / 8))) =
                            uint4{0u, 0u, 0u, 0u};
                }
                __syncwarp();
            }
            float sc[4][4];
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) {
                uint32_t a_[4];
                if constexpr (DP > 128) load_q(kk, a_);
                const uint32_t* a = DP <= 128 ? qa[DP <= 128 ? kk : 0] : a_;
#pragma unroll
                for (int np = 0; np < 2; ++np) {
                    const int key = 16 * np + (lane & 7) + 8 * (lane >> 4), chunk = 2 * kk + (lane >> 3 & 1);
                    uint32_t bk[4];
                    ldsm4(kb + chunk_off(KT, key, chunk), bk);
                    mma16816<E>(sc[2 * np], a, bk[0], bk[1]);
                    mma16816<E>(sc[2 * np + 1], a, bk[2], bk[3]);
                }
            }
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int nt = 0; nt < 4; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = sc[nt][e] * sl2;
                    if (edge) {
                        const int ri = e >> 1, kr = 8 * nt + 2 * tq + (e & 1), key = k0 + kr;
                        bool see = kr < valid && key >= rlo[ri] && key < rhi[ri];
                        if (p.mask != nullptr && see && key >= g.L)
                            see = rw[ri][(key - g.L) >> 5] >> ((key - g.L) & 31) & 1u;
                        if (!see) v = -INFINITY;
                    }
                    sc[nt][e] = v;
                    mx[e >> 1] = fmaxf(mx[e >> 1], v);
                }
            float corr[2], mref[2];
#pragma unroll
            for (int ri = 0; ri < 2; ++ri) {
                mx[ri] = fmaxf(mx[ri], __shfl_xor_sync(0xffffffffu, mx[ri], 1));
                mx[ri] = fmaxf(mx[ri], __shfl_xor_sync(0xffffffffu, mx[ri], 2));
                const float mn = fmaxf(m_run[ri], mx[ri]);
                corr[ri] = mn == -INFINITY ? 1.f : ex2(m_run[ri] - mn);
                m_run[ri] = mn;
                mref[ri] = mn == -INFINITY ? 0.f : mn;
                l_run[ri] *= corr[ri];
            }
#pragma unroll
            for (int j = 0; j < DP / 8; ++j) {
                oacc[j][0] *= corr[0];
                oacc[j][1] *= corr[0];
                oacc[j][2] *= corr[1];
                oacc[j][3] *= corr[1];
            }
            // P is rounded to the cache's type, the operand type of the second product;
            // the row sums take it unrounded
            uint32_t pa[2][4];
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
                for (int h2 = 0; h2 < 2; ++h2) {
                    const int nt = 2 * k2 + h2;
                    const float p0 = ex2(sc[nt][0] - mref[0]), p1 = ex2(sc[nt][1] - mref[0]);
                    const float p2 = ex2(sc[nt][2] - mref[1]), p3 = ex2(sc[nt][3] - mref[1]);
                    l_run[0] += p0 + p1;
                    l_run[1] += p2 + p3;
                    pa[k2][2 * h2] = E::pack(p0, p1);
                    pa[k2][2 * h2 + 1] = E::pack(p2, p3);
                }
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
                for (int dp = 0; dp < DP / 16; ++dp) {
                    const int key = 16 * k2 + (lane & 15), chunk = 2 * dp + (lane >> 4);
                    uint32_t bv[4];
                    ldsm4_t(vb + chunk_off(KT, key, chunk), bv);
                    mma16816<E>(oacc[2 * dp], pa[k2], bv[0], bv[1]);
                    mma16816<E>(oacc[2 * dp + 1], pa[k2], bv[2], bv[3]);
                }
            if (dirty) fence_proxy_async_smem();  // the zeros before the slot's next copy
            __syncwarp();
            if (lane == 0) mbar_arrive(empty_bar(s));
        }
#pragma unroll
        for (int ri = 0; ri < 2; ++ri) {
            l_run[ri] += __shfl_xor_sync(0xffffffffu, l_run[ri], 1);
            l_run[ri] += __shfl_xor_sync(0xffffffffu, l_run[ri], 2);
        }
        // join the NTG warps of each row group in shared memory, then write the
        // rows out (a whole unit) or to the workspace (a part)
        float* wp = part + warp * 16 * L::PSTR;
#pragma unroll
        for (int ri = 0; ri < 2; ++ri) {
            float* row = wp + (gq + 8 * ri) * L::PSTR;
#pragma unroll
            for (int j = 0; j < DP / 8; ++j)
                *reinterpret_cast<float2*>(row + 8 * j + 2 * tq) =
                    dead[ri] ? make_float2(0.f, 0.f) : make_float2(oacc[j][2 * ri], oacc[j][2 * ri + 1]);
            if (tq == 0) {
                row[DP] = dead[ri] ? -INFINITY : m_run[ri];
                row[DP + 1] = dead[ri] ? 0.f : l_run[ri];
            }
        }
        named_bar_sync(1, 32 * NCW);
        const bool whole = g.count == g.s.n;
        float* slot = partial_slot(p, 2 * blockIdx.x + (pos - g.first <= begin ? 0 : 1));
        const int rows = min(p.RT, p.rows - row0);
        if (!*abort_flag) {
            for (int idx = threadIdx.x; idx < rows * (p.D / 8); idx += 32 * NCW) {
                const int lr = idx / (p.D / 8), c8 = idx % (p.D / 8);
                const float* row = part + (lr / 16) * 16 * L::PSTR + (lr % 16) * L::PSTR;
                float M = -INFINITY;
                for (int k = 0; k < NTG; ++k) M = fmaxf(M, row[k * NRG * 16 * L::PSTR + DP]);
                float o[8] = {}, l = 0.f;
                for (int k = 0; k < NTG; ++k) {
                    const float* x = row + k * NRG * 16 * L::PSTR;
                    const float f = x[DP] == -INFINITY ? 0.f : ex2(x[DP] - M);
                    l += f * x[DP + 1];
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[e] += f * x[8 * c8 + e];
                }
                if (whole) {
                    const float inv = l == 0.f ? 0.f : 1.f / l;
                    const int r = row0 + lr;
                    const uint4 v{E::pack(o[0] * inv, o[1] * inv), E::pack(o[2] * inv, o[3] * inv),
                                  E::pack(o[4] * inv, o[5] * inv), E::pack(o[6] * inv, o[7] * inv)};
                    *reinterpret_cast<uint4*>(p.o + g.b * p.osb + (g.kvh * p.G + r % p.G) * p.osh +
                                              (r / p.G) * p.oss + 8 * c8) = v;
                } else {
                    float4* d = reinterpret_cast<float4*>(slot + lr * p.D + 8 * c8);
                    d[0] = make_float4(o[0], o[1], o[2], o[3]);
                    d[1] = make_float4(o[4], o[5], o[6], o[7]);
                    if (c8 == 0) {
                        slot[p.RT * p.D + lr] = M;
                        slot[p.RT * p.D + p.RT + lr] = l;
                    }
                }
            }
        }
        named_bar_sync(1, 32 * NCW);  // the partials, Q and mask areas are free again
        i0 += g.count;
        pos += g.count;
    }
}

}  // namespace paged
}  // namespace rdna
