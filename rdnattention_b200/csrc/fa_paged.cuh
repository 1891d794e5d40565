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
// some row of it sees.  The tiles of all units, each unit's led by W positions for
// what starting a unit costs, form one list, and CTA c takes the c-th equal part of
// it (row tiles slowest, so that the CTAs that read the same keys for other rows do so
// at the same time and find them in L2): every CTA has the same time's work whatever
// the lengths are, and the lengths stay on the device (a captured graph replays with
// new ones).  A unit that lies inside one CTA is finished there; the parts
// of the others go to a workspace as (O, m, l) in fp32 and the join kernel adds
// them up in list order, so results do not depend on timing.
#pragma once

#include <cuda.h>
#include <limits.h>
#include <math.h>

#include "fa_decode.cuh"
#include "paged.cuh"

namespace rdna {
namespace paged {

constexpr int kMaxTree = 256;          // drafted tokens under a mask
constexpr int kMaxList = 2048;         // sequences x row tiles per launch (the host splits larger batches)
constexpr int KT = 64;                 // keys per tile
// AttnParams::W of the two kernels: about the tiles' worth of time that a segment's start and
// end take (ragged batch of 33: 157 us at 0, 112 at 4, 105 at 6, 107 at 8; trees of 64 tokens
// in 16 contexts: 104 us at 8, 102 at 12, 101 at 16; all at head_dim 128, other widths take the same).
constexpr int kLead = 6, kLeadMma = 12;

// n / d for n < 2^31 by a multiplication: with l = ceil(log2 d) and m =
// floor(2^(31 + l) / d) + 1, m d exceeds 2^(31 + l) by at most 2^l, so the error
// n (m d - 2^(31 + l)) / d 2^(31 + l) stays below 1 / d.
struct FastDiv {
    uint32_t d, m, l;
    void set(uint32_t div) {
        d = div;
        for (l = 0; (uint64_t(1) << l) < d; ++l) {
        }
        m = static_cast<uint32_t>((uint64_t(1) << (31 + l)) / d + 1);
    }
    __device__ __forceinline__ int div(int n) const {
        return l == 0 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), m) >> (l - 1));
    }
};

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
    FastDiv by_G, by_B;
    int rows;    // T * G
    int RT;      // rows per tile
    int n_rt;    // row tiles
    int tpp;     // key tiles per page (pages of at least KT slots), else 0: KT / P pages per tile
    FastDiv by_tpp;
    FastDiv by_P;
    int window;  // 0: none
    float scale_log2;  // |scale| log2 e (never 0: masked scores are -inf times it)
    uint32_t flip;     // 0x80008000 for a negative scale: the query's signs turn instead
    float* ws;   // partials: 2 per CTA, each O [D / 4][RT] float4, m [RT], l [RT]
    int2* units; // per unit (b, kvh, rt): first partial's slot, number of parts (0 or 1: nothing to join)
    int grid;    // CTAs of the attention kernel
    int W;       // list positions that a unit costs besides its tiles
    int join_shift;  // log2 of the join's rows per block
};

// Touches every line of the parameters once (one word per lane and 64 bytes), so that
// the constant-cache misses of a fresh launch overlap each other and the wait for the
// kernel before, instead of standing one by one in the way of the schedule.
__device__ __forceinline__ void warm_params(const AttnParams& p) {
    const int* w = reinterpret_cast<const int*>(&p);
    const int at = (threadIdx.x & 31) * 16;
    int v = w[at < static_cast<int>(sizeof(AttnParams) / 4) ? at : 0];
    asm volatile("" ::"r"(v));
}

// ---------------------------------------------------------------- the schedule
struct Span {
    int lo, hi;  // keys some row of the tile sees: [lo, hi)
    int t0, n;   // first key tile and their number
};

// Tile that holds key j.
__device__ __forceinline__ int tile_of(const AttnParams& p, int j) {
    if (p.tpp == 0) return j / KT;
    const int page = p.by_P.div(j);
    return page * p.tpp + (j - page * p.t.P) / KT;
}

__device__ __forceinline__ Span row_tile_span(const AttnParams& p, int L, int n, int rt) {
    const int cap = p.t.cap();
    const int ta = p.by_G.div(rt * p.RT);  // tokens of the tile: [ta, tb]
    const int tb = min(p.by_G.div(min((rt + 1) * p.RT, p.rows) - 1), n - 1);
    Span s{0, 0, 0, 0};
    if (ta >= n) return s;  // padding rows only
    s.hi = min(p.mask != nullptr ? L + n : L + tb + 1, cap);
    if (p.window > 0) s.lo = max(0, p.mask != nullptr ? L - p.window : L + ta + 1 - p.window);
    if (s.lo >= s.hi) return s;
    s.t0 = tile_of(p, s.lo);
    s.n = tile_of(p, s.hi - 1) + 1 - s.t0;
    return s;
}

// The list of a launch: entry e = rt * B + b, pre[e] (shared memory) = position behind it.
struct Sched {
    int total;  // positions of the launch
    int ctas;   // CTAs that take part
    int q, r;   // the first r of them take q + 1 positions, the others q
};

// Positions of an entry: all KV heads of a row tile of a sequence.
__device__ __forceinline__ int entry_cost(const AttnParams& p, int e) {
    const int rt = p.by_B.div(e), b = e - rt * p.B;
    const int tiles = row_tile_span(p, p.t.len(b), p.t.news(b), rt).n;
    return tiles > 0 ? (p.W + tiles) * p.Hkv : 0;
}

__device__ __forceinline__ int warp_scan(int v, int lane) {
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int u = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += u;
    }
    return v;
}

// All threads of the block.  Up to 32 entries every warp computes the whole list and
// writes the same values, so that no barrier stands between the lengths and the first
// key tile.
__device__ __forceinline__ Sched make_sched(const AttnParams& p, int* pre) {
    const int lane = threadIdx.x & 31, n = p.B * p.n_rt;
    Sched s;
    if (n <= 32) {
        const int v = warp_scan(lane < n ? entry_cost(p, lane) : 0, lane);
        if (lane < n) pre[lane] = v;
        s.total = __shfl_sync(0xffffffffu, v, 31);
        __syncwarp();
    } else {
        for (int e = threadIdx.x; e < n; e += blockDim.x) pre[e] = entry_cost(p, e);
        __syncthreads();
        if (threadIdx.x < 32) {
            int carry = 0;
            for (int e0 = 0; e0 < n; e0 += 32) {
                const int e = e0 + lane;
                const int v = warp_scan(e < n ? pre[e] : 0, lane) + carry;
                if (e < n) pre[e] = v;
                carry = __shfl_sync(0xffffffffu, v, 31);
            }
        }
        __syncthreads();
        s.total = pre[n - 1];
    }
    s.ctas = min(p.grid, max(1, s.total));
    s.q = s.total / s.ctas;
    s.r = s.total - s.q * s.ctas;
    return s;
}

__device__ __forceinline__ int cta_begin(const Sched& s, int c) { return c * s.q + min(c, s.r); }
// CTA that holds list position pos < total.
__device__ __forceinline__ int cta_of(const Sched& s, int pos) {
    const int wide = s.r * (s.q + 1);
    return pos < wide ? pos / (s.q + 1) : s.r + (pos - wide) / s.q;
}

// One unit's share of a CTA: its tiles first .. first + count - 1 (count may be 0: only
// the unit's lead lies in the CTA).
struct Segment {
    int b, kvh, rt, L, n;
    Span s;
    int first, count;
    int pos0;  // list position of the unit's tile 0
    int next;  // list position behind the segment
    int e;     // its list entry
};

// The segment at list position pos < total (a whole warp; e: an entry at or before it,
// kept from call to call).
__device__ __forceinline__ Segment segment_at(const AttnParams& p, const int* pre, int pos, int end, int& e) {
    const int lane = threadIdx.x & 31;
    for (;; e += 32) {
        const uint32_t past = __ballot_sync(0xffffffffu, e + lane < p.B * p.n_rt && pre[e + lane] > pos);
        if (past != 0) {
            e += __ffs(past) - 1;
            break;
        }
    }
    Segment g;
    g.e = e;
    g.rt = p.by_B.div(e);
    g.b = e - g.rt * p.B;
    g.L = p.t.len(g.b);
    g.n = p.t.news(g.b);
    g.s = row_tile_span(p, g.L, g.n, g.rt);
    int off = pos - (e > 0 ? pre[e - 1] : 0);
    g.kvh = off / (p.W + g.s.n);
    off -= g.kvh * (p.W + g.s.n);
    g.pos0 = pos - off + p.W;
    g.first = max(0, off - p.W);
    g.count = max(0, min(g.s.n - g.first, end - g.pos0 - g.first));
    g.next = min(g.pos0 + g.first + g.count, end);
    return g;
}

// First key of a tile and how many of its KT rows are keys (a page may end
// inside a tile; the rows behind its end are zero fill).
__device__ __forceinline__ void tile_keys(const AttnParams& p, int tile, int& k0, int& valid) {
    if (p.tpp == 0) {
        k0 = tile * KT;
        valid = KT;
    } else {
        const int page = p.by_tpp.div(tile), off = (tile - page * p.tpp) * KT;
        k0 = page * p.t.P + off;
        valid = min(KT, p.t.P - off);
    }
}

__device__ __forceinline__ float* partial_slot(const AttnParams& p, int slot) {
    return p.ws + static_cast<int64_t>(slot) * p.RT * (p.D + 2);
}
__device__ __forceinline__ int unit_index(const AttnParams& p, int b, int kvh, int rt) {
    return (b * p.Hkv + kvh) * p.n_rt + rt;
}
// The slot of a segment's partial: a CTA starts with at most one unit that began before it
// (or with it) and ends with at most one other that goes on.
__device__ __forceinline__ int segment_slot(const Segment& g, int begin) {
    return 2 * static_cast<int>(blockIdx.x) + (g.pos0 <= begin ? 0 : 1);
}
// What the join needs to know about a unit, from the CTA that holds its first tile.
__device__ __forceinline__ void describe_unit(const AttnParams& p, const Sched& sc, const Segment& g, int begin) {
    const int parts = g.count == g.s.n ? 1 : cta_of(sc, g.pos0 + g.s.n - 1) - static_cast<int>(blockIdx.x) + 1;
    p.units[unit_index(p, g.b, g.kvh, g.rt)] = make_int2(segment_slot(g, begin), parts);
}

// Row tiles that see no key belong to no CTA's list: their output rows are zeroed, and
// described, by CTA (b, rt) modulo the grid.  tid .. of nthreads threads.
__device__ __forceinline__ void zero_empty_units(const AttnParams& p, int tid, int nthreads) {
    for (int u = blockIdx.x; u < p.B * p.n_rt; u += gridDim.x) {
        const int b = u / p.n_rt, rt = u - b * p.n_rt;
        if (row_tile_span(p, p.t.len(b), p.t.news(b), rt).n > 0) continue;
        const int rows = min(p.RT, p.rows - rt * p.RT), nch = p.D / 8;
        for (int i = tid; i < p.Hkv * rows * nch; i += nthreads) {
            const int ch = i % nch, r = i / nch % rows, kvh = i / nch / rows, row = rt * p.RT + r;
            const int t = p.by_G.div(row), h = kvh * p.G + row - t * p.G;
            *reinterpret_cast<uint4*>(p.o + b * p.osb + h * p.osh + t * p.oss + ch * 8) = uint4{0u, 0u, 0u, 0u};
        }
        for (int kvh = tid; kvh < p.Hkv; kvh += nthreads) p.units[unit_index(p, b, kvh, rt)] = make_int2(0, 0);
    }
}

// Bits of the drafted tokens that the tokens of a row tile see: words[i * nw + w] for
// token ta + i, mask bytes to bits by ballot, four words' loads in flight.  Threads tid ..
// of `nthreads` (whole warps) take part; the caller synchronises them, and with a window
// calls trim_mask() then and synchronises again.
__device__ __forceinline__ int tile_tokens(const AttnParams& p, const Segment& g) {
    return min(p.by_G.div(min((g.rt + 1) * p.RT, p.rows) - 1), g.n - 1) - p.by_G.div(g.rt * p.RT) + 1;
}
__device__ __forceinline__ void build_mask(const AttnParams& p, const Segment& g, uint32_t* words, int tid,
                                           int nthreads) {
    const int nw = (p.t.T + 31) / 32, total = tile_tokens(p, g) * nw;
    const int lane = tid & 31, warps = nthreads / 32;
    const uint8_t* base = p.mask + g.b * p.msb + p.by_G.div(g.rt * p.RT) * p.mst;
    for (int j0 = tid / 32; j0 < total; j0 += 4 * warps) {
        uint32_t see[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int j = j0 + k * warps, i = j / nw, u = 32 * (j - i * nw) + lane;
            see[k] = j < total && u < g.n ? base[i * p.mst + u] : 0;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t bits = __ballot_sync(0xffffffffu, see[k] != 0);
            if (lane == 0 && j0 + k * warps < total) words[j0 + k * warps] = bits;
        }
    }
}
// The window: a token keeps its newest drafted tokens, at most w, and sees the newest w
// less those of the context, from ctx_lo[i] on.
__device__ __forceinline__ void trim_mask(const AttnParams& p, const Segment& g, uint32_t* words, int* ctx_lo, int tid,
                                          int nthreads) {
    const int nw = (p.t.T + 31) / 32, nt = tile_tokens(p, g);
    for (int i = tid; i < nt; i += nthreads) {
        int seen = 0;
        for (int w = 0; w < nw; ++w) seen += __popc(words[i * nw + w]);
        for (int w = 0, drop = seen - p.window; drop > 0; ++w) {
            uint32_t bits = words[i * nw + w];
            for (; drop > 0 && bits != 0; --drop) bits &= bits - 1;
            words[i * nw + w] = bits;
        }
        ctx_lo[i] = max(0, g.L - max(0, p.window - seen));
    }
}

// ------------------------------------------------------------- the join kernel
// O = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i over a split unit's parts, always in
// the same order.  A thread takes one row (lanes side by side, so the partials are read in
// runs of 64 or 256 bytes), 8 columns and every n-th part; the n shares of a block join in
// shared memory.  Bound by the latency of dependent reads (the unit, its parts) while
// there are few units of many parts: the WIDE form has blocks of 512 threads (n = 2 to 8 at
// head_dim 128), one for each SM at most, and eight parts' loads in flight.  With more units
// (of few parts then) the narrow form takes 16 rows with n = 1 and three parts in flight, four
// blocks on an SM (256 row tiles of 128 over 8192 keys: 9 us, wide 24 us).
constexpr int kJoinRows = 16, kJoinRowsWide = 4;  // rows of a block: 16; wide: 4, 8 or 16
constexpr int kJoinThreads = 512;

template <class E, bool WIDE>
__global__ void __launch_bounds__(kJoinThreads, WIDE ? 1 : 2) join_kernel(const __grid_constant__ AttnParams p) {
    extern __shared__ float joined[];  // [n - 1][10][width]
    constexpr int kJoinFlight = WIDE ? 8 : 3;
    const int rows = 1 << p.join_shift, groups = p.RT >> p.join_shift;
    const int unit = blockIdx.x / groups;
    const int width = rows * (p.D / 8), n = blockDim.x / width, split = threadIdx.x / width,
              tid = threadIdx.x - split * width;
    const int lr = blockIdx.x % groups * rows + (tid & (rows - 1));  // row of the tile
    const int c = (tid >> p.join_shift) * 8;                         // first column
    grid_dependency_wait();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int2 u = p.units[unit];
    const int rt = unit % p.n_rt, r = rt * p.RT + lr;
    if (u.y < 2) return;
    float M = -INFINITY, l = 0.f;
    float o[8] = {};
    auto add = [&](float m, float li, const float* x, float mx) {
        const float f = m == -INFINITY ? 0.f : ex2(m - mx);
        l += f * li;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] += f * x[e];
    };
    auto rescale = [&](float mx) {
        const float g = M == -INFINITY ? 0.f : ex2(M - mx);
        M = mx;
        l *= g;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] *= g;
    };
    for (int i0 = split; i0 < u.y; i0 += kJoinFlight * n) {
        float m[kJoinFlight], li[kJoinFlight], x[kJoinFlight][8];
        float mx = M;
#pragma unroll
        for (int k = 0; k < kJoinFlight; ++k) {
            const int i = i0 + k * n;
            m[k] = -INFINITY;
            li[k] = 0.f;
            if (i < u.y) {
                const float* w = partial_slot(p, i == 0 ? u.x : 2 * (u.x / 2 + i));
                m[k] = w[p.RT * p.D + lr];
                li[k] = w[p.RT * p.D + p.RT + lr];
                *reinterpret_cast<float4*>(x[k]) = *reinterpret_cast<const float4*>(w + (c / 4 * p.RT + lr) * 4);
                *reinterpret_cast<float4*>(x[k] + 4) = *reinterpret_cast<const float4*>(w + ((c / 4 + 1) * p.RT + lr) * 4);
            }
        }
#pragma unroll
        for (int k = 0; k < kJoinFlight; ++k) mx = fmaxf(mx, m[k]);
        rescale(mx);
#pragma unroll
        for (int k = 0; k < kJoinFlight; ++k)
            if (i0 + k * n < u.y) add(m[k], li[k], x[k], M);
    }
    if (split > 0) {
        float* s = joined + (split - 1) * 10 * width + tid;
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e * width] = o[e];
        s[8 * width] = M;
        s[9 * width] = l;
    }
    __syncthreads();
    if (split > 0 || r >= p.rows) return;
    for (int k = 1; k < n; ++k) {
        const float* s = joined + (k - 1) * 10 * width + tid;
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = s[e * width];
        const float m = s[8 * width];
        rescale(fmaxf(M, m));
        add(m, s[9 * width], x, M);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int kvh = unit / p.n_rt % p.Hkv, b = unit / p.n_rt / p.Hkv;
    const int t = p.by_G.div(r), h = kvh * p.G + r - t * p.G;
    *reinterpret_cast<uint4*>(p.o + b * p.osb + h * p.osh + t * p.oss + c) =
        uint4{E::pack(o[0] * inv, o[1] * inv), E::pack(o[2] * inv, o[3] * inv), E::pack(o[4] * inv, o[5] * inv),
              E::pack(o[6] * inv, o[7] * inv)};
}

// ------------------------------------------------------------- the cluster form
// A single sequence's heads are equally long, so an even split needs no list: a cluster of
// CTAs takes a unit, CTA `rank` the rank-th part of its tiles, and the parts are joined
// over distributed shared memory.  That saves the second launch and two trips through L2;
// the host's rule has the measurements.
__device__ __forceinline__ Segment cluster_segment(const AttnParams& p) {
    const int size = static_cast<int>(decode::cluster_size()), rank = static_cast<int>(decode::cluster_rank());
    const int unit = blockIdx.x / size;
    Segment g;
    g.rt = unit % p.n_rt;
    g.kvh = unit / p.n_rt % p.Hkv;
    g.b = unit / p.n_rt / p.Hkv;
    g.L = p.t.len(g.b);
    g.n = p.t.news(g.b);
    g.s = row_tile_span(p, g.L, g.n, g.rt);
    g.first = g.s.n * rank / size;
    g.count = g.s.n * (rank + 1) / size - g.first;
    g.pos0 = 0;
    g.next = 1;
    g.e = 0;
    return g;
}

__device__ __forceinline__ float4 ld_dsmem4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

// Joins the cluster's parts (at `part` in each CTA's shared memory: O [D / 4][RT] float4,
// m [RT], l [RT]) and writes the rows out; every thread of every CTA takes part.  A part that
// adds nothing has m = -inf and l = 0, and no O if its CTA had no tiles; scores that were all NaN
// leave m at -inf too, but a sum of NaN.
template <class E>
__device__ __forceinline__ void cluster_join(const AttnParams& p, const float* part, int tid, int nthreads) {
    decode::cluster_sync_all();
    const int size = static_cast<int>(decode::cluster_size()), rank = static_cast<int>(decode::cluster_rank());
    const int unit = blockIdx.x / size, rt = unit % p.n_rt, kvh = unit / p.n_rt % p.Hkv, b = unit / p.n_rt / p.Hkv;
    const uint32_t base = smem_u32(part);
    for (int i = rank * nthreads + tid; i < p.RT * (p.D / 4); i += size * nthreads) {
        const int lr = i & (p.RT - 1), c = i / p.RT, r = rt * p.RT + lr;
        if (r >= p.rows) continue;
        float M = -INFINITY, l = 0.f;
        float4 o{};
        for (int k0 = 0; k0 < size; k0 += 8) {
            float m[8], li[8];
            float4 x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                m[k] = -INFINITY;
                li[k] = 0.f;
                if (k0 + k < size) {
                    const uint32_t a = decode::map_to_rank(base, k0 + k);
                    m[k] = decode::ld_dsmem(a + 4 * (p.RT * p.D + lr));
                    li[k] = decode::ld_dsmem(a + 4 * (p.RT * p.D + p.RT + lr));
                    x[k] = ld_dsmem4(a + 16 * (c * p.RT + lr));
                }
            }
            float mx = M;
#pragma unroll
            for (int k = 0; k < 8; ++k) mx = fmaxf(mx, m[k]);
            const float g = M == -INFINITY ? 0.f : ex2(M - mx);
            M = mx;
            l *= g;
            o.x *= g;
            o.y *= g;
            o.z *= g;
            o.w *= g;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (m[k] != -INFINITY || li[k] != 0.f) {
                    const float f = m[k] == -INFINITY ? 0.f : ex2(m[k] - mx);
                    l += f * li[k];
                    o.x += f * x[k].x;
                    o.y += f * x[k].y;
                    o.z += f * x[k].z;
                    o.w += f * x[k].w;
                }
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int t = p.by_G.div(r);
        *reinterpret_cast<uint2*>(p.o + b * p.osb + (kvh * p.G + r - t * p.G) * p.osh + t * p.oss + 4 * c) =
            uint2{E::pack(o.x * inv, o.y * inv), E::pack(o.z * inv, o.w * inv)};
    }
    decode::cluster_sync_all();  // no CTA leaves while others read its part
}

// -------------------------------------------------------- the few-rows kernel
// Row groups of 16 (the M = 16 of m16n8k16), NRG of them per tile.
//   warps NCW..     prepare the next segment: turned queries, mask bits, rows' limits
//   last warp       TMA producer: 64-key tiles of K and V through an NST-stage ring
//   warps 0..NCW-1  consumers: the 32-key halves of the tiles go round the NCW /
//                   NRG warps of each row group: S = Q K^T and O += P V on mma.sync
//                   with the online softmax in registers
// Q is kept as the sum of two values of the cache's type, hi + lo (the rotated query
// in 32 bits splits into them but for 2^-22 / 2^-16 of it in fp16 / bf16), and both
// are multiplied with K: the bound is HBM, so the extra MMAs are free, and the
// scores are as exact as an fp32 product.
//
// Measured (head_dim 128): 64 sequences of 32768 slots, 8 KV heads of 8 query heads:
// 1.24 ms = 6.9 TB/s replayed on one input, 1.34 ms = 6.4 TB/s called over changing ones, 1.06 and
// 0.98 of the measured copy rate.  33 ragged sequences of up to 8192 slots, 32 / 8 heads, pages
// of 16: 106 to 111 us, 0.76 to 0.79 of the copy rate (what is missing are the segments' starts,
// four or five per CTA, and the join).
template <int DP>
struct Layout {
    static constexpr int NCW = DP <= 128 ? 8 : 4;
    // warps NCW .. that prepare segments; the last one of all is the producer
    static constexpr int NPREP = 3;
    static_assert(32 * NPREP % (DP / 8) == 0, "whole rows between a thread's chunks");
    static constexpr int THREADS = 32 * (NCW + NPREP + 1);
    static constexpr int NBOX = DP / 64;  // 64-element boxes (128 B, SWIZZLE_128B)
    static constexpr int BOX_BYTES = KT * 128;
    static constexpr int TILE = NBOX * BOX_BYTES;
    static constexpr int STAGE = 2 * TILE;
    static constexpr int NST = 512 / DP;  // 128 KB in flight
    // a slot's halves always go to the same warps, so no waiter is more than one phase behind
    static_assert(2 * NST % NCW == 0, "each ring slot has its own consumer warps");
    static constexpr int MAX_RT = DP <= 128 ? 16 : 32;
    static constexpr int PSTR = DP + 4;  // floats per partial row: O, m, l, padding
    static constexpr int OFF_RING = 1024;
    static constexpr int OFF_Q = OFF_RING + NST * STAGE;  // hi, lo: [RT][DP], swizzled like a K tile
    static constexpr int Q_BYTES = NBOX * MAX_RT * 128;
    // what a segment needs besides its tiles, NQ times (the producers fill the next one's)
    static constexpr int NQ = DP <= 128 ? 2 : 1;
    static constexpr bool ALIAS = DP > 128;               // the partials take Q's place
    static constexpr int OFF_PART = ALIAS ? OFF_Q : OFF_Q + NQ * 2 * Q_BYTES;  // [NCW][16][PSTR] fp32
    static constexpr int OFF_MASK = OFF_PART + NCW * 16 * PSTR * 4;  // [NQ] of: bits [RT][kMaxTree / 32], ctx_lo [RT],
    static constexpr int MASK_BYTES = MAX_RT * (kMaxTree / 32) * 4 + MAX_RT * 4 + MAX_RT * 8;  // limits [RT]
    static constexpr int OFF_PRE = OFF_MASK + NQ * MASK_BYTES;
    static constexpr int Q_FULL = 2 * NST, Q_EMPTY = Q_FULL + NQ, OFF_ABORT = 8 * (Q_EMPTY + NQ);  // barriers
    static constexpr int SMEM_BYTES = OFF_PRE + kMaxList * 4 + 1024;  // + alignment slack
    static_assert(!ALIAS || NCW * 16 * PSTR * 4 >= 2 * Q_BYTES, "Q fits below the partials");
    static_assert(SMEM_BYTES <= 232448, "shared memory of one CTA");
};

// Byte offset of 16-byte chunk c of row r in a tile of `rows` rows (64-element
// boxes one after the other, 128-byte swizzle).
__device__ __forceinline__ uint32_t chunk_off(int rows, int r, int c) {
    return static_cast<uint32_t>((c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// (With a memory clobber, unlike the dense decode kernel's: here the tile is also written by its reader.)
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
    decode::mma16816(c, a, b0, b1);
}
template <>
__device__ __forceinline__ void mma16816<BF16>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Position of row r, -1 for a row that sees nothing: padding, or a position outside the
// tables.  (Without tables the position does not matter.)
__device__ __forceinline__ int row_position(const AttnParams& p, const Segment& g, int r) {
    const int t = p.by_G.div(r);
    if (r >= p.rows || t >= g.n) return -1;
    if (p.cos == nullptr) return 0;
    const int pos = p.positions != nullptr ? p.positions[static_cast<int64_t>(g.b) * p.t.T + t] : g.L + t;
    return static_cast<unsigned>(pos) < static_cast<unsigned>(p.rope_rows) ? pos : -1;
}

// Loads chunk ch (16 bytes) of N rows of Q, r0, r0 + STEP, .. at positions pos[k], and turns
// them; hi + lo (see above).  Zeros for rows that see nothing.  All loads are issued before
// the first is used: one by one each would wait for two reads in turn.
template <class E, int N, int STEP>
__device__ __forceinline__ void load_q(const AttnParams& p, const Segment& g, int r0, const int* pos, int ch,
                                       uint4* hi, uint4* lo) {
    const uint16_t* base = p.q + g.b * p.qsb + g.kvh * p.G * p.qsh + ch * 8;
    const bool col = ch * 8 < p.D;
    float4 c[N], s[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int r = r0 + k * STEP, t = p.by_G.div(r);
        hi[k] = lo[k] = uint4{0u, 0u, 0u, 0u};
        if (pos[k] >= 0 && col) hi[k] = *reinterpret_cast<const uint4*>(base + (r - t * p.G) * p.qsh + t * p.qss);
    }
    if (p.cos != nullptr) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int64_t at = pos[k] >= 0 && col ? static_cast<int64_t>(pos[k]) * (p.D / 2) + ch * 4 : 0;
            c[k] = __ldg(reinterpret_cast<const float4*>(p.cos + at));
            s[k] = __ldg(reinterpret_cast<const float4*>(p.sin + at));
        }
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
        hi[k].x ^= p.flip;
        hi[k].y ^= p.flip;
        hi[k].z ^= p.flip;
        hi[k].w ^= p.flip;
    }
    if (p.cos != nullptr) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            turn_split<E>(hi[k].x, lo[k].x, c[k].x, s[k].x);
            turn_split<E>(hi[k].y, lo[k].y, c[k].y, s[k].y);
            turn_split<E>(hi[k].z, lo[k].z, c[k].z, s[k].z);
            turn_split<E>(hi[k].w, lo[k].w, c[k].w, s[k].w);
        }
    }
}

// Keys row r sees: [lo, hi), and with a mask the drafted slots from L on by bit.
__device__ __forceinline__ void row_limits(const AttnParams& p, const Segment& g, int r, int pos, const int* ctx_lo,
                                           int& lo, int& hi) {
    if (pos < 0) {
        lo = 1;
        hi = 0;
        return;
    }
    const int t = p.by_G.div(r);
    if (p.mask != nullptr) {
        lo = p.window > 0 ? ctx_lo[t - p.by_G.div(g.rt * p.RT)] : 0;
        hi = g.s.hi;
    } else {
        lo = p.window > 0 ? max(0, g.L + t + 1 - p.window) : 0;
        hi = min(g.L + t + 1, g.s.hi);
    }
}

// One lane of the (converged) warp, always the same.  The work it is elected for stays in a
// warp-uniform loop, and values that are the same in all lanes pass through a shuffle, so
// that the compiler keeps them in uniform registers, where TMA and MMA instructions take
// their operands: issued by `if (lane == 0)` a TMA box cost 180 cycles instead of 30 to 65
// and an MMA 87 instead of 38.
__device__ __forceinline__ bool elect_one() {
    uint32_t leader;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(leader)
        :
        : "memory");
    return leader != 0;
}
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// The producer's part of a segment (one warp): its tiles into the ring by TMA boxes of one
// page's rows (at most KT) x 64 columns; rows behind a page's end, columns behind head_dim
// and pages outside the cache are zero fill.  A copy alone reaches 6.7 TB/s with boxes of
// any height from 8 rows.  i: running tile number; `filled`, `issued`: for drain().  False
// when a wait expired.
template <class L>
__device__ __forceinline__ bool produce(const AttnParams& p, const CUtensorMap* tmK, const CUtensorMap* tmV,
                                        const Segment& g, int i, uint32_t bars, uint32_t ring, uint32_t& filled,
                                        int& issued, const Abort& ab, int lane) {
    // Keys that four or more row tiles read stay in L2 if they can; with fewer, what one CTA has
    // read is soon read by another or never again (32 / 8 heads, sustained, kept and evicted first: 512
    // tokens of 2 prompts over 16384 slots 437 and 479 us, 128 tokens 101 and 108, 96 tokens 84 and
    // 83; ragged trees of 64 tokens in 16 contexts 117 and 111).
    const uint64_t pol = p.n_rt >= 4 ? policy_evict_last() : policy_evict_first();
    const int ppt = uniform(p.tpp == 0 ? KT >> p.t.Pshift : 1), box = min(p.t.P, KT) * 128;  // pages per tile
    const int* pages = p.t.pages + g.b * p.t.stride;
    const int tile0 = g.s.t0 + g.first, count = uniform(g.count), kvh = uniform(g.kvh);
    i = uniform(i);
    int lp = uniform(p.tpp == 0 ? tile0 * ppt : p.by_tpp.div(tile0));  // logical page, first row in it
    int sub = uniform(p.tpp == 0 ? 0 : (tile0 - lp * p.tpp) * KT);
    int win = -1, ids = -1;  // 32 consecutive page table entries, one per lane
    for (int k = 0; k < count; ++k, ++i) {
        if (lp / 32 != win) {
            win = lp / 32;
            const int e = win * 32 + lane;
            ids = e < p.t.max_pages ? __ldg(pages + e) : -1;
            if (static_cast<unsigned>(ids) >= static_cast<unsigned>(p.t.num_pages)) ids = -1;  // zero fill
        }
        const int s = i % L::NST;
        const uint32_t full = bars + 8u * s, dst = ring + s * L::STAGE;
        if (!__all_sync(0xffffffffu, mbar_wait(bars + 8u * (L::NST + s), (i / L::NST & 1) ^ 1, ab, 0x601))) return false;
        filled |= 1u << s;
        issued = i;
        if (elect_one()) mbar_arrive_expect_tx(full, L::STAGE);
        __syncwarp();
        for (int j = 0; j < ppt; ++j) {
            const int page = uniform(__shfl_sync(0xffffffffu, ids, (lp + j) & 31));
            if (elect_one()) {
#pragma unroll
                for (int bx = 0; bx < L::NBOX; ++bx)
                    tma_load_4d(dst + bx * L::BOX_BYTES + j * box, tmK, full, bx * 64, sub, kvh, page, pol);
#pragma unroll
                for (int bx = 0; bx < L::NBOX; ++bx)
                    tma_load_4d(dst + L::TILE + bx * L::BOX_BYTES + j * box, tmV, full, bx * 64, sub, kvh, page, pol);
            }
            __syncwarp();
        }
        if (p.tpp == 0) {
            lp += ppt;
        } else if ((sub += KT) >= p.t.P) {
            sub = 0;
            ++lp;
        }
    }
    return true;
}

// After an expired wait: the copies in flight land before the CTA leaves.  Slot s last
// received tile j, the largest j <= issued with j % NST == s.
template <class L>
__device__ __forceinline__ void drain(uint32_t bars, uint32_t filled, int issued) {
    for (int s = 0; s < L::NST; ++s)
        if (filled >> s & 1u) {
            const int j = issued - ((issued - s) % L::NST + L::NST) % L::NST;
            mbar_wait_drain(bars + 8u * s, j / L::NST & 1);
        }
}

// First key that some row of the tile sees.  With a mask the window ends earlier than the
// span says, by the drafted tokens that even the row with the fewest sees (a whole warp; the
// mask is trimmed).
__device__ __forceinline__ int first_seen(const AttnParams& p, const Segment& g, const int* ctx_lo, int lane) {
    if (p.mask == nullptr || p.window <= 0) return g.s.lo;
    int lo = INT_MAX;
    for (int i = lane, nt = tile_tokens(p, g); i < nt; i += 32) lo = min(lo, ctx_lo[i]);
    return __reduce_min_sync(0xffffffffu, lo);
}

// Slots no row of the unit sees may hold anything (0 * NaN): zeros over the V rows of a tile
// whose keys k0 + r lie outside [lo, hi), rows r0 .. r0 + rows - 1, by n threads.
template <int DP>
__device__ __forceinline__ void zero_unseen_v(uint8_t* v, int lo, int hi, int k0, int r0, int rows, int tid, int n) {
    for (int idx = tid; idx < rows * (DP / 8); idx += n) {
        const int r = r0 + idx / (DP / 8);
        if (k0 + r < lo || k0 + r >= hi)
            *reinterpret_cast<uint4*>(v + chunk_off(KT, r, idx % (DP / 8))) = uint4{0u, 0u, 0u, 0u};
    }
    fence_proxy_async_smem();  // before the tensor core's reads, or the slot's next copy
}

template <class E, int DP, bool CLUSTER>
__global__ void __launch_bounds__(Layout<DP>::THREADS, 1) fa_paged_kernel(
    const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
    const __grid_constant__ AttnParams p) {
    using L = Layout<DP>;
    constexpr int NCW = L::NCW;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);  // (an offset keeps the address space known)
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t bars = smem_u32(smem);
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (L::NST + s); };
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_ABORT);
    const Abort ab{abort_flag};
    uint8_t* ring = smem + L::OFF_RING;
    int* pre = reinterpret_cast<int*>(smem + L::OFF_PRE);

    const int NRG = p.RT / 16, NTG = NCW / NRG;
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < L::NST; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), NRG * min(2, NTG));
        }
        for (int k = 0; k < L::NQ; ++k) {
            mbar_init(bars + 8u * (L::Q_FULL + k), 32 * L::NPREP);
            mbar_init(bars + 8u * (L::Q_EMPTY + k), 1);
        }
        fence_barrier_init();
        prefetch_tmap(&tmK);
        prefetch_tmap(&tmV);
    }
    warm_params(p);
    __syncthreads();
    grid_dependency_wait();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    Sched sched{};
    int begin = 0, end = 1;
    if constexpr (!CLUSTER) {
        sched = make_sched(p, pre);
        if (sched.total == 0 || static_cast<int>(blockIdx.x) >= sched.ctas) {
            zero_empty_units(p, threadIdx.x, L::THREADS);
            return;
        }
        begin = cta_begin(sched, blockIdx.x);
        end = cta_begin(sched, blockIdx.x + 1);
    }

    const int wrg = warp % NRG, wtg = warp / NRG;
    const int gq = lane >> 2, tq = lane & 3;
    const int nw = (p.t.T + 31) / 32;
    float* part = reinterpret_cast<float*>(smem + L::OFF_PART);
    const float sl2 = p.scale_log2;
    bool aborted = false;    // consumers: a wait expired
    uint32_t filled = 0;     // producer: slots that received a copy, last tile issued
    int issued = -1;
    int i0 = 0, e = 0, nseg = 0;  // running tile number of the segment's first tile; segments so far
    for (int pos = begin; pos < end;) {
        const Segment g = CLUSTER ? cluster_segment(p) : segment_at(p, pre, pos, end, e);
        pos = g.next;
        if (g.count == 0) {
            // (in a cluster: a part that adds nothing)
            if (CLUSTER && threadIdx.x < p.RT) {
                float* ml = reinterpret_cast<float*>(ring) + p.RT * p.D;
                ml[threadIdx.x] = -INFINITY;
                ml[p.RT + threadIdx.x] = 0.f;
            }
            continue;
        }
        const int row0 = g.rt * p.RT, ta = p.by_G.div(row0);
        const int qb = nseg % L::NQ, qn = nseg / L::NQ;
        ++nseg;
        uint8_t* qmem = smem + L::OFF_Q + qb * 2 * L::Q_BYTES;
        uint32_t* words = reinterpret_cast<uint32_t*>(smem + L::OFF_MASK + qb * L::MASK_BYTES);
        int* ctx_lo = reinterpret_cast<int*>(words + L::MAX_RT * (kMaxTree / 32));
        int2* limits = reinterpret_cast<int2*>(ctx_lo + L::MAX_RT);
        if (warp == NCW + L::NPREP) {
            if (!produce<L>(p, &tmK, &tmV, g, i0, bars, smem_u32(ring), filled, issued, ab, lane)) {
                drain<L>(bars, filled, issued);
                break;
            }
            i0 += g.count;
            continue;
        }
        if (warp >= NCW) {
            // Q of the row tile (turned, hi and lo), the mask bits and the rows' limits
            const int ptid = threadIdx.x - 32 * NCW;
            if (!__all_sync(0xffffffffu, mbar_wait(bars + 8u * (L::Q_EMPTY + qb), (qn & 1) ^ 1, ab, 0x603))) break;
            constexpr int STEP = 32 * L::NPREP / (DP / 8);  // rows between a thread's chunks
            for (int lr = ptid / (DP / 8); lr < p.RT; lr += 2 * STEP) {
                const int ch = ptid % (DP / 8);
                int pos[2];
                uint4 hi[2], lo[2];
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    pos[k] = lr + k * STEP < p.RT ? row_position(p, g, row0 + lr + k * STEP) : -1;
                load_q<E, 2, STEP>(p, g, row0 + lr, pos, ch, hi, lo);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (lr + k * STEP >= p.RT) continue;
                    *reinterpret_cast<uint4*>(qmem + chunk_off(p.RT, lr + k * STEP, ch)) = hi[k];
                    *reinterpret_cast<uint4*>(qmem + L::Q_BYTES + chunk_off(p.RT, lr + k * STEP, ch)) = lo[k];
                }
            }
            if (p.mask != nullptr) {
                build_mask(p, g, words, ptid, 32 * L::NPREP);
                if (p.window > 0) {
                    named_bar_sync(2, 32 * L::NPREP);
                    trim_mask(p, g, words, ctx_lo, ptid, 32 * L::NPREP);
                    named_bar_sync(2, 32 * L::NPREP);
                }
            }
            if (ptid < p.RT)
                row_limits(p, g, row0 + ptid, row_position(p, g, row0 + ptid), ctx_lo, limits[ptid].x, limits[ptid].y);
            mbar_arrive(bars + 8u * (L::Q_FULL + qb));
            continue;
        }
        // ------------------------------------------------------------ consumers
        if (!aborted && !__all_sync(0xffffffffu, mbar_wait(bars + 8u * (L::Q_FULL + qb), qn & 1, ab, 0x604)))
            aborted = true;
        const uint32_t qs = smem_u32(qmem);
        int rlo[2], rhi[2];
        const uint32_t* rw[2];
        for (int e = 0; e < 2; ++e) {
            const int lr = wrg * 16 + gq + 8 * e, t = p.by_G.div(row0 + lr);
            rlo[e] = limits[lr].x;
            rhi[e] = limits[lr].y;
            rw[e] = words + (rlo[e] < rhi[e] ? (t - ta) * nw : 0);
        }
        // keys in [all_lo, all_hi) are seen by every row of the group that sees any; what the
        // others (padding, empty) add up there is dropped at the end of the segment
        const bool dead[2] = {rlo[0] >= rhi[0], rlo[1] >= rhi[1]};
        int all_lo = max(dead[0] ? 0 : rlo[0], dead[1] ? 0 : rlo[1]);
        int all_hi = min(dead[0] ? INT_MAX : rhi[0], dead[1] ? INT_MAX : rhi[1]);
        if (p.mask != nullptr) all_hi = min(all_hi, g.L);
        all_lo = __reduce_max_sync(0xffffffffu, all_lo);
        all_hi = __reduce_min_sync(0xffffffffu, all_hi);
        const int seen_lo = first_seen(p, g, ctx_lo, lane);
        auto load_q = [&](int kk, int half, uint32_t* a) {
            ldsm4(qs + half * L::Q_BYTES + chunk_off(p.RT, wrg * 16 + (lane & 15), 2 * kk + (lane >> 4)), a);
        };
        float oacc[DP / 8][4];
#pragma unroll
        for (int j = 0; j < DP / 8; ++j) oacc[j][0] = oacc[j][1] = oacc[j][2] = oacc[j][3] = 0.f;
        float m_run[2] = {-INFINITY, -INFINITY};
        float l_run[2] = {0.f, 0.f};

        // this warp's halves of the segment: running numbers hh with hh % NTG == wtg
        for (int hh = 2 * i0 + ((wtg - 2 * i0) & (NTG - 1)); hh < 2 * (i0 + g.count); hh += NTG) {
            const int i = hh >> 1, s = i % L::NST, kh = (hh & 1) * 32;  // first key row of the half
            int k0, valid;
            tile_keys(p, g.s.t0 + g.first + (i - i0), k0, valid);
            k0 += kh;
            valid -= kh;
            bool ok = !aborted && mbar_wait(full_bar(s), i / L::NST & 1, ab, 0x602);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {
                aborted = true;
                continue;
            }
            // the last warp-half of a tile to finish frees its slot
            const bool last = NTG > 1 || (hh & 1);
            const bool none = valid <= 0 || k0 >= g.s.hi || k0 + 32 <= seen_lo;
            const uint32_t kb = smem_u32(ring) + s * L::STAGE, vb = kb + L::TILE;
            const bool edge = valid < 32 || k0 < all_lo || k0 + 32 > all_hi;
            const bool dirty = !none && (k0 < seen_lo || k0 + 32 > g.s.hi);
            if (dirty) {
                zero_unseen_v<DP>(ring + s * L::STAGE + L::TILE, seen_lo, g.s.hi, k0 - kh, kh, 32, lane, 32);
                __syncwarp();
            }
            if (!none) {
                float sc[4][4];
#pragma unroll
                for (int nt = 0; nt < 4; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
                // fragments of step kk + 1 load while step kk multiplies (Q's too: kept in
                // registers it would cost the eight warps their 168 registers each)
                const int krow = kh + (lane & 7) + 8 * (lane >> 4), kch = lane >> 3 & 1;
                uint32_t bk[2][2][4], al[2][4], ah[2][4];
                auto load_k = [&](int kk) {
                    ldsm4(kb + chunk_off(KT, krow, 2 * kk + kch), bk[kk & 1][0]);
                    ldsm4(kb + chunk_off(KT, krow + 16, 2 * kk + kch), bk[kk & 1][1]);
                    load_q(kk, 1, al[kk & 1]);
                    load_q(kk, 0, ah[kk & 1]);
                };
                load_k(0);
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk) {
                    if (kk + 1 < DP / 16) load_k(kk + 1);
#pragma unroll
                    for (int nt = 0; nt < 4; ++nt)
                        mma16816<E>(sc[nt], ah[kk & 1], bk[kk & 1][nt >> 1][2 * (nt & 1)], bk[kk & 1][nt >> 1][2 * (nt & 1) + 1]);
#pragma unroll
                    for (int nt = 0; nt < 4; ++nt)
                        mma16816<E>(sc[nt], al[kk & 1], bk[kk & 1][nt >> 1][2 * (nt & 1)],
                                    bk[kk & 1][nt >> 1][2 * (nt & 1) + 1]);
                }
                float mx[2] = {-INFINITY, -INFINITY};
                if (edge) {
#pragma unroll
                    for (int nt = 0; nt < 4; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int ri = e >> 1, kr = 8 * nt + 2 * tq + (e & 1), key = k0 + kr;
                            bool see = kr < valid && key >= rlo[ri] && key < rhi[ri];
                            if (p.mask != nullptr && see && key >= g.L)
                                see = rw[ri][(key - g.L) >> 5] >> ((key - g.L) & 31) & 1u;
                            if (!see) sc[nt][e] = -INFINITY;
                        }
                }
#pragma unroll
                for (int nt = 0; nt < 4; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[nt][e] *= sl2;
                        mx[e >> 1] = fmaxf(mx[e >> 1], sc[nt][e]);
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
                if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
                    for (int j = 0; j < DP / 8; ++j) {
                        oacc[j][0] *= corr[0];
                        oacc[j][1] *= corr[0];
                        oacc[j][2] *= corr[1];
                        oacc[j][3] *= corr[1];
                    }
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
                constexpr int VB = DP <= 128 ? 2 : 1;  // buffers: registers are short at 256
                uint32_t bv[VB][2][4];
                auto load_v = [&](int dp) {
#pragma unroll
                    for (int k2 = 0; k2 < 2; ++k2)
                        ldsm4_t(vb + chunk_off(KT, kh + 16 * k2 + (lane & 15), 2 * dp + (lane >> 4)), bv[dp % VB][k2]);
                };
                load_v(0);
#pragma unroll
                for (int dp = 0; dp < DP / 16; ++dp) {
                    if (VB > 1 && dp + 1 < DP / 16) load_v(dp + 1);
#pragma unroll
                    for (int k2 = 0; k2 < 2; ++k2) {
                        mma16816<E>(oacc[2 * dp], pa[k2], bv[dp % VB][k2][0], bv[dp % VB][k2][1]);
                        mma16816<E>(oacc[2 * dp + 1], pa[k2], bv[dp % VB][k2][2], bv[dp % VB][k2][3]);
                    }
                    if (VB == 1 && dp + 1 < DP / 16) load_v(dp + 1);
                }
            }
            __syncwarp();
            if (lane == 0 && last) mbar_arrive(empty_bar(s));
        }
#pragma unroll
        for (int ri = 0; ri < 2; ++ri) {
            l_run[ri] += __shfl_xor_sync(0xffffffffu, l_run[ri], 1);
            l_run[ri] += __shfl_xor_sync(0xffffffffu, l_run[ri], 2);
        }
        // join the NTG warps of each row group in shared memory, then write the
        // rows out (a whole unit) or to the workspace (a part)
        if constexpr (L::ALIAS) named_bar_sync(1, 32 * NCW);
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
        const bool whole = !CLUSTER && g.count == g.s.n;
        float* slot = CLUSTER ? reinterpret_cast<float*>(ring) : partial_slot(p, segment_slot(g, begin));
        if (!CLUSTER && g.first == 0 && threadIdx.x == 0) describe_unit(p, sched, g, begin);
        const int rows = min(p.RT, p.rows - row0);
        if (!*abort_flag) {
            // rows side by side: whole lines of the partial's [D / 4][RT] layout
            for (int idx = threadIdx.x; idx < p.RT * (DP / 4); idx += 32 * NCW) {
                const int lr = idx & (p.RT - 1), c = idx / p.RT * 4;
                if (c >= p.D || lr >= rows) continue;
                const float* row = part + ((lr / 16) * 16 + lr % 16) * L::PSTR;
                const int step = NRG * 16 * L::PSTR;
                float M = -INFINITY;
                for (int k = 0; k < NTG; ++k) M = fmaxf(M, row[k * step + DP]);
                float4 o{};
                float l = 0.f;
                for (int k = 0; k < NTG; ++k) {
                    const float* x = row + k * step;
                    const float f = x[DP] == -INFINITY ? 0.f : ex2(x[DP] - M);
                    const float4 v = *reinterpret_cast<const float4*>(x + c);
                    l += f * x[DP + 1];
                    o.x += f * v.x;
                    o.y += f * v.y;
                    o.z += f * v.z;
                    o.w += f * v.w;
                }
                if (whole) {
                    const float inv = l == 0.f ? 0.f : 1.f / l;
                    const int r = row0 + lr, t = p.by_G.div(r);
                    *reinterpret_cast<uint2*>(p.o + g.b * p.osb + (g.kvh * p.G + r - t * p.G) * p.osh + t * p.oss + c) =
                        uint2{E::pack(o.x * inv, o.y * inv), E::pack(o.z * inv, o.w * inv)};
                } else {
                    *reinterpret_cast<float4*>(slot + (c / 4 * p.RT + lr) * 4) = o;
                    if (c == 0) {
                        slot[p.RT * p.D + lr] = M;
                        slot[p.RT * p.D + p.RT + lr] = l;
                    }
                }
            }
        }
        named_bar_sync(1, 32 * NCW);  // the partials, Q and mask areas are free again
        if (threadIdx.x == 0) mbar_arrive(bars + 8u * (L::Q_EMPTY + qb));
        i0 += g.count;
    }
    if constexpr (CLUSTER) {
        __syncwarp();
        cluster_join<E>(p, reinterpret_cast<const float*>(ring), threadIdx.x, L::THREADS);
    } else if (warp < NCW) {
        zero_empty_units(p, threadIdx.x, 32 * NCW);
    }
}

}  // namespace paged
}  // namespace rdna
