// Paged KV cache: what its kernels share, and the two that only move rows
// (append with the position rotation, accept).
//
// Cache: K and V are [num_pages, Hkv, page_size, D] views (page / head / slot
// strides in elements, head_dim contiguous), fp16 or bf16.  Sequence b's token
// at slot s lives in row s % page_size of page table[b][s / page_size].  Keys
// are stored rotated, so a row keeps its value when it moves to another slot.
//
// Everything a call learns from device memory is checked where it is used,
// because the host cannot see it: lengths are clamped to [0, max_pages *
// page_size], a page outside [0, num_pages) is never written and reads as
// zeros, a token whose position lies outside the rotation tables is skipped.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "rope.cuh"
#include "sm100.cuh"

namespace rdna {
namespace paged {

using namespace sm100;

// Element types of the cache (rdna_paged_* `dtype`).
enum : int { DT_F16 = 0, DT_BF16 = 1 };

struct F16 {
    static __device__ __forceinline__ float2 unpack(uint32_t v) {
        return __half22float2(*reinterpret_cast<const __half2*>(&v));
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_half2(lo, hi); }
    // Values beyond the type's largest become that instead of an infinity.
    static __device__ __forceinline__ uint32_t pack_finite(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
};
struct BF16 {
    static __device__ __forceinline__ float2 unpack(uint32_t v) {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
    static __device__ __forceinline__ uint32_t pack_finite(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
};

// One interleaved pair turned by its angle, fp32 math with explicit roundings
// (the same bits in every kernel, the dense ones' function in fp16), rounded once to the element type.
template <class E>
__device__ __forceinline__ uint32_t rotate_pair(uint32_t v, float c, float s) {
    const float2 x = E::unpack(v);
    return E::pack(__fmaf_rn(x.x, c, -__fmul_rn(x.y, s)), __fmaf_rn(x.x, s, __fmul_rn(x.y, c)));
}
template <>
__device__ __forceinline__ uint32_t rotate_pair<F16>(uint32_t v, float c, float s) {
    return rope::rotate_pair(v, c, s);
}

// The same, as hi + lo: the rounded pair and what the rounding left, rounded again.  A turn can
// leave fp16's range by a factor of sqrt 2: hi is the largest value then, and lo holds the rest
// (an infinity or NaN stays one, in lo).
template <class E>
__device__ __forceinline__ void turn_split(uint32_t& hi, uint32_t& lo, float c, float s) {
    const float2 x = E::unpack(hi);
    const float a = __fmaf_rn(x.x, c, -__fmul_rn(x.y, s)), b = __fmaf_rn(x.x, s, __fmul_rn(x.y, c));
    hi = E::pack_finite(a, b);
    const float2 h = E::unpack(hi);
    lo = E::pack(a - h.x, b - h.y);
}

// 16 bytes = 4 pairs.
template <class E>
__device__ __forceinline__ uint4 rotate4(const uint4& x, const float4& c, const float4& s) {
    return uint4{rotate_pair<E>(x.x, c.x, s.x), rotate_pair<E>(x.y, c.y, s.y), rotate_pair<E>(x.z, c.z, s.z),
                 rotate_pair<E>(x.w, c.w, s.w)};
}

// The lengths and page table of a batch.
struct Table {
    const int* pages;       // [B][max_pages], rows `stride` apart
    const int* cache_lens;  // [B]: tokens in the cache before the new ones
    const int* new_lens;    // [B] or null: new tokens of each sequence (null: T)
    int64_t stride;
    int max_pages, num_pages;
    int P;      // slots per page
    int Pmask;  // P - 1 and log2 P when P is a power of two, else Pshift = -1
    int Pshift;
    int T;      // new tokens of each sequence in the (padded) batch

    __device__ __forceinline__ int cap() const { return max_pages * P; }  // the host checks that it fits
    __device__ __forceinline__ int len(int b) const { return min(max(cache_lens[b], 0), cap()); }
    __device__ __forceinline__ int news(int b) const {
        return new_lens == nullptr ? T : min(max(new_lens[b], 0), T);
    }
    __device__ __forceinline__ void split(int slot, int& page, int& row) const {
        if (Pshift >= 0) {
            page = slot >> Pshift;
            row = slot & Pmask;
        } else {
            page = slot / P;
            row = slot - page * P;
        }
    }
    // Physical page and row of a slot; false when there is none.
    __device__ __forceinline__ bool locate(int b, int64_t slot, int& page, int& row) const {
        if (slot < 0 || slot >= cap()) return false;
        int lp;
        split(static_cast<int>(slot), lp, row);
        page = pages[b * stride + lp];
        return static_cast<unsigned>(page) < static_cast<unsigned>(num_pages);
    }
};

struct Rows {  // [B, Hkv, T, D] view
    const uint16_t* p;
    int64_t sb, sh, ss;
};
struct Cache {  // [num_pages, Hkv, P, D] view, strides in bytes
    char* p;
    int64_t sh;
    uint32_t sp, ss;  // (32 bits: one multiply-add for each part of an address)

    __device__ __forceinline__ char* head(int h, int ch) const { return p + h * sh + ch * 16; }
    __device__ __forceinline__ char* at(char* head, int page, int row) const {
        return head + static_cast<uint64_t>(static_cast<uint32_t>(page)) * sp +
               static_cast<uint64_t>(static_cast<uint32_t>(row)) * ss;
    }
};

// ------------------------------------------------------------------- append
struct AppendParams {
    Rows k, v;
    Cache kc, vc;
    Table t;
    const int* positions;  // [B][T] or null: cache_lens[b] + t
    const float *cos, *sin;  // [rope_rows][D / 2] or null: K is stored as it is
    int rope_rows;
    int B, Hkv, D;
    int64_t n;  // B * Hkv * T * (D / 8) 16-byte chunks
};

// One 16-byte chunk of K and of V per thread: load, turn K, store.  K and V are
// read once; the rows of the tables and the page entries are read again for every
// head and sequence, from L2.  The chunk index runs fastest, then the token, so that
// both sides of the copy are contiguous within a page.  Bound by HBM: 4 prompts of 4096
// tokens, 8 heads of 128 (134 MB of rows and 2 MB of tables), 27.5 us over changing
// inputs = 0.76 of the measured copy rate, 25.2 us = 0.83 over the same; small calls by
// the latency of the length, page and row reads (2.4 us for one token).
template <class E>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ AppendParams p) {
    const int nch = p.D / 8;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= p.n) return;
    const int ch = static_cast<int>(i % nch);
    const int64_t bht = i / nch;
    const int t = static_cast<int>(bht % p.t.T);
    const int bh = static_cast<int>(bht / p.t.T);
    const int h = bh % p.Hkv, b = bh / p.Hkv;
    if (t >= p.t.news(b)) return;
    const int len = p.t.len(b);
    int page, row;
    if (!p.t.locate(b, static_cast<int64_t>(len) + t, page, row)) return;
    uint4 k = *reinterpret_cast<const uint4*>(p.k.p + b * p.k.sb + h * p.k.sh + t * p.k.ss + ch * 8);
    const uint4 v = *reinterpret_cast<const uint4*>(p.v.p + b * p.v.sb + h * p.v.sh + t * p.v.ss + ch * 8);
    if (p.cos != nullptr) {
        const int pos = p.positions != nullptr ? p.positions[static_cast<int64_t>(b) * p.t.T + t] : len + t;
        if (static_cast<unsigned>(pos) >= static_cast<unsigned>(p.rope_rows)) return;
        const int64_t at = static_cast<int64_t>(pos) * (p.D / 2) + ch * 4;
        k = rotate4<E>(k, __ldg(reinterpret_cast<const float4*>(p.cos + at)),
                       __ldg(reinterpret_cast<const float4*>(p.sin + at)));
    }
    *reinterpret_cast<uint4*>(p.kc.at(p.kc.head(h, ch), page, row)) = k;
    *reinterpret_cast<uint4*>(p.vc.at(p.vc.head(h, ch), page, row)) = v;
}

// ------------------------------------------------------------------- accept
constexpr int kMaxAccept = 256;

struct AcceptParams {
    Cache kc, vc;
    Table t;
    const int* accepted;      // [B][A]: drafted token that becomes the i-th accepted one
    const int* accepted_lens; // [B] or null: A
    int A, B, Hkv, D;
    int n;                    // 2 * Hkv * (D / 8) columns of 16 bytes per sequence
};

// Row len + i takes row len + accepted[i], all as they were before the call.  A thread
// owns one 16-byte column of one head of K or V and every row of it, so reading all its
// rows before it writes the first is enough: no two threads touch the same bytes.  The
// rows' places are worked out once per block; up to kAcceptRegs rows are held in registers,
// with every read in flight at once (the bound is the latency of three dependent reads:
// index, page table, row), more of them in shared memory.  One sequence with 4 tokens or
// 64 sequences with up to 9: 2.5 to 4 us.
constexpr int kAcceptRegs = 16;

template <bool REGS>
__global__ void accept_kernel(const __grid_constant__ AcceptParams p) {
    extern __shared__ uint4 stage[];
    __shared__ int2 from[kMaxAccept], to[kMaxAccept];  // page and row; page -1: nothing moves
    const int b = blockIdx.y;
    const int64_t len = p.t.len(b);
    const int n = p.accepted_lens == nullptr ? p.A : min(max(p.accepted_lens[b], 0), p.A);
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int a = p.accepted[static_cast<int64_t>(b) * p.A + i];
        int2 f{-1, 0}, t{-1, 0};
        const bool ok = a >= 0 && a != i && p.t.locate(b, len + a, f.x, f.y);
        if (!(p.t.locate(b, len + i, t.x, t.y) && ok)) f.x = -1;
        from[i] = f;
        to[i] = t;
    }
    __syncthreads();
    const int col = blockIdx.x * blockDim.x + threadIdx.x;
    if (col >= p.n) return;
    const int nch = p.D / 8;
    const int ch = col % nch, h = col / nch % p.Hkv;
    const Cache& c = col / nch / p.Hkv == 0 ? p.kc : p.vc;
    char* base = c.head(h, ch);
    if constexpr (REGS) {
        uint4 v[kAcceptRegs];
#pragma unroll
        for (int i = 0; i < kAcceptRegs; ++i)
            if (i < n && from[i].x >= 0) v[i] = *reinterpret_cast<const uint4*>(c.at(base, from[i].x, from[i].y));
#pragma unroll
        for (int i = 0; i < kAcceptRegs; ++i)
            if (i < n && from[i].x >= 0) *reinterpret_cast<uint4*>(c.at(base, to[i].x, to[i].y)) = v[i];
    } else {
        uint4* mine = stage + threadIdx.x;
#pragma unroll 4
        for (int i = 0; i < n; ++i)
            if (from[i].x >= 0) mine[i * blockDim.x] = *reinterpret_cast<const uint4*>(c.at(base, from[i].x, from[i].y));
        for (int i = 0; i < n; ++i)
            if (from[i].x >= 0) *reinterpret_cast<uint4*>(c.at(base, to[i].x, to[i].y)) = mine[i * blockDim.x];
    }
}

}  // namespace paged
}  // namespace rdna
