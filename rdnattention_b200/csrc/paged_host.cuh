// Host side of the paged KV-cache operators (included by forward.cu, the one
// translation unit that holds every kernel): checks, tensor maps, launches.
#pragma once

#include <algorithm>
#include <atomic>
#include <cmath>
#include <limits>
#include <type_traits>

namespace rdna {
namespace {

thread_local char g_err_paged[512] = {0};

int pfail(const char* msg) { return fail(g_err_paged, msg); }

bool p16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool p4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

// [n0, n1, n2, head_dim] view: strides positive multiples of 16 bytes on every axis longer than one.
const char* check_strides(int64_t s0, int64_t s1, int64_t s2, uint64_t n0, uint64_t n1, uint64_t n2) {
    const int64_t s[3] = {s0, s1, s2};
    const uint64_t n[3] = {n0, n1, n2};
    for (int i = 0; i < 3; ++i) {
        if (n[i] <= 1) continue;
        if (s[i] <= 0) return "strides must be positive";
        if (s[i] % 8 != 0) return "strides must be multiples of 16 bytes";
        if (s[i] >= (int64_t(1) << 39)) return "stride too large";  // 40 bits of bytes, a tensor map's limit
    }
    return nullptr;
}

// The sizes that a workspace query knows too.
const char* check_cache_sizes(const PagedCacheParams& c) {
    if (c.batchSize == 0 || c.numKvHeads == 0 || c.maxPages == 0)
        return "empty problem (batch_size, num_kv_heads, num_pages and max_pages must be > 0)";
    if (c.headDim < 32 || c.headDim > 256 || c.headDim % 32 != 0)
        return "unsupported head_dim (multiples of 32 from 32 to 256)";
    const bool pow2 = c.pageSize >= 8 && (c.pageSize & (c.pageSize - 1)) == 0;
    if (!pow2 && c.pageSize < 64) return "unsupported page_size (a power of two from 8 up, or any size from 64 up)";
    if (static_cast<uint64_t>(c.maxPages) * c.pageSize > (1u << 30)) return "max_pages * page_size exceeds 2^30";
    if (c.numKvHeads > 65535 || c.batchSize > (1u << 24)) return "too many heads or sequences";
    return nullptr;
}

const char* check_cache(const PagedCacheParams& c) {
    if (c.kCache == nullptr || c.vCache == nullptr || c.pageTable == nullptr || c.cacheLens == nullptr)
        return "null tensor pointer";
    if (c.dtype != paged::DT_F16 && c.dtype != paged::DT_BF16) return "dtype must be 0 (fp16) or 1 (bf16)";
    if (c.numPages == 0) return "empty problem (batch_size, num_kv_heads, num_pages and max_pages must be > 0)";
    if (const char* e = check_cache_sizes(c)) return e;
    if (c.numPages > INT32_MAX) return "too many pages";
    if (!p16(c.kCache) || !p16(c.vCache)) return "cache base pointers must be 16-byte aligned";
    if (!p4(c.pageTable) || !p4(c.cacheLens)) return "page_table and cache_lens must be 4-byte aligned";
    if (c.batchSize > 1 && c.tableStride < 0) return "strides must be positive";
    if (const char* e = check_strides(c.kcStrideP, c.kcStrideH, c.kcStrideS, c.numPages, c.numKvHeads, c.pageSize))
        return e;
    // the kernels hold the page and slot strides as 32 bits of bytes (one page has no stride)
    for (int64_t s : {c.kcStrideS, c.vcStrideS, c.numPages > 1 ? c.kcStrideP : 0, c.numPages > 1 ? c.vcStrideP : 0})
        if (s >= (int64_t(1) << 31)) return "cache page or slot stride too large";
    return check_strides(c.vcStrideP, c.vcStrideH, c.vcStrideS, c.numPages, c.numKvHeads, c.pageSize);
}

const char* check_rope(const void* cos, const void* sin, const void* positions, uint32_t rows) {
    if (!p4(positions)) return "positions must be 4-byte aligned";
    if (cos == nullptr && sin == nullptr) return nullptr;
    if (cos == nullptr || sin == nullptr) return "pass both rot_cos and rot_sin, or neither";
    if (!p16(cos) || !p16(sin)) return "rot_cos/rot_sin must be 16-byte aligned";
    if (rows == 0) return "the rotation tables have no rows";
    if (rows > INT32_MAX) return "too many rotation table rows";
    return nullptr;
}

paged::Table make_table(const PagedCacheParams& c, const void* new_lens, uint32_t T) {
    paged::Table t{};
    t.pages = static_cast<const int*>(c.pageTable);
    t.cache_lens = static_cast<const int*>(c.cacheLens);
    t.new_lens = static_cast<const int*>(new_lens);
    t.stride = c.tableStride;
    t.max_pages = static_cast<int>(c.maxPages);
    t.num_pages = static_cast<int>(c.numPages);
    t.P = static_cast<int>(c.pageSize);
    t.Pmask = t.P - 1;
    t.Pshift = -1;
    if ((t.P & t.Pmask) == 0)
        for (t.Pshift = 0; (1 << t.Pshift) < t.P; ++t.Pshift) {
        }
    t.T = static_cast<int>(T);
    return t;
}

paged::Cache cache_view(void* p, int64_t sp, int64_t sh, int64_t ss) {
    return paged::Cache{static_cast<char*>(p), 2 * sh, static_cast<uint32_t>(2 * sp), static_cast<uint32_t>(2 * ss)};
}

// What a launch needs to know of a device, asked for once: its SMs, and whether a kernel's
// attributes have been set there.
constexpr int kMaxPagedDevices = 64;

int current_device() {
    int dev = 0;
    cudaGetDevice(&dev);
    return dev >= 0 && dev < kMaxPagedDevices ? dev : -1;
}

int sm_count() {
    static std::atomic<int> known[kMaxPagedDevices];
    const int dev = current_device();
    int sms = dev >= 0 ? known[dev].load(std::memory_order_relaxed) : 0;
    if (sms == 0) {
        sms = 148;
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev >= 0 ? dev : 0);
        if (dev >= 0) known[dev].store(sms, std::memory_order_relaxed);
    }
    return sms;
}

template <auto K>
struct Kernel {
    static constexpr auto value = K;
};
constexpr int kMaxCluster = 16;
constexpr int kMaxPagedUnits = 74;  // (two CTAs for each of more do not fit 148 SMs)

// Lets `kern` use `smem` bytes on the current device.  regs != 0: the kernel moves registers
// between its warps and must have been given exactly that many per thread (an increase
// waits for registers the CTA has).
template <auto kern>
cudaError_t prepare_kernel(int smem, int regs, bool cluster = false) {
    static std::atomic<bool> done[kMaxPagedDevices];
    const int dev = current_device();
    if (dev >= 0 && done[dev].load(std::memory_order_acquire)) return cudaSuccess;
    cudaError_t ce = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (ce == cudaSuccess && regs != 0) {
        cudaFuncAttributes fa{};
        ce = cudaFuncGetAttributes(&fa, kern);
        if (ce == cudaSuccess && fa.numRegs != regs) ce = cudaErrorInvalidKernelImage;
    }
    if (ce == cudaSuccess && cluster) ce = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (ce == cudaSuccess && dev >= 0) done[dev].store(true, std::memory_order_release);
    return ce;
}

// Clusters of `size` CTAs that fit the current device at once (asked for once).
template <auto kern>
int max_clusters(int size, int threads, int smem) {
    static std::atomic<int> known[kMaxPagedDevices][kMaxCluster + 1];
    const int dev = current_device();
    int n = dev >= 0 ? known[dev][size].load(std::memory_order_relaxed) : 0;
    if (n == 0) {
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = size;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        cfg.gridDim = dim3(size);
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
            cudaGetLastError();
            n = 0;
        }
        if (dev >= 0) known[dev][size].store(n > 0 ? n : -1, std::memory_order_relaxed);
    }
    return n > 0 ? n : 0;
}

int launched() {
    const cudaError_t ce = cudaGetLastError();
    return ce == cudaSuccess ? 0 : fail(g_err_paged, "%s", cudaGetErrorString(ce));
}

// How a paged attention call is cut: rows per tile, key tiles per page.
struct PagedPlan {
    int dp;     // head_dim rounded up to the kernel's 64, 128 or 256
    bool mma;   // the tcgen05 kernel's row tiles of 128
    int RT, n_rt, tpp, grid, W;
    int64_t tiles;  // key tiles of a full page table
    int64_t step;   // sequences per launch; 0: the problem is too large
    size_t partials, bytes;  // workspace: bytes of the partials, in all
};

// Rows of a KV head within the kernels' 32 bits (either factor may be any 32-bit number).
bool rows_fit(uint32_t H, uint32_t Hkv, uint32_t T) { return H / Hkv <= (uint32_t(1) << 28) / std::max(T, 1u); }

PagedPlan paged_plan(const PagedAttentionParams& a) {
    const PagedCacheParams& c = a.c;
    PagedPlan f{};
    f.dp = c.headDim <= 64 ? 64 : c.headDim <= 128 ? 128 : 256;
    const int64_t rows = static_cast<int64_t>(a.numHeads / c.numKvHeads) * a.seqLen;
    f.mma = f.dp <= 128 && rows > 16;
    f.RT = f.mma ? 128 : f.dp <= 128 || rows <= 16 ? 16 : 32;
    f.n_rt = static_cast<int>((rows + f.RT - 1) / f.RT);
    const int64_t P = c.pageSize;
    f.tpp = P >= paged::KT ? static_cast<int>((P + paged::KT - 1) / paged::KT) : 0;
    f.tiles = f.tpp == 0 ? (c.maxPages * P + paged::KT - 1) / paged::KT : static_cast<int64_t>(c.maxPages) * f.tpp;
    f.grid = sm_count();
    f.W = f.mma ? paged::kLeadMma : paged::kLead;
    // units of a launch: at most kMaxList (sequence, row tile) pairs, and list positions of 32
    // bits (n_rt <= 2^11, so none of these products passes 64 bits)
    if (f.n_rt > paged::kMaxList) return f;
    const int64_t per_seq = (f.tiles + f.W) * f.n_rt * c.numKvHeads;
    const int64_t join_blocks =
        static_cast<int64_t>(c.numKvHeads) * f.n_rt * ((f.RT + paged::kJoinRows - 1) / paged::kJoinRows);
    f.step = std::min<int64_t>(INT32_MAX / std::max(per_seq, join_blocks), paged::kMaxList / f.n_rt);
    f.partials = align_up(static_cast<size_t>(2) * f.grid * f.RT * (c.headDim + 2) * sizeof(float));
    const int64_t seqs = std::min<int64_t>(c.batchSize, f.step);
    f.bytes = f.partials + align_up(static_cast<size_t>(seqs) * c.numKvHeads * f.n_rt * sizeof(int2));
    return f;
}

// The plan of a call, and which sizes no call takes: for the call and the workspace query alike.
// (Nothing is planned for seqLen 0.)
const char* plan_attention(const PagedAttentionParams& a, PagedPlan& f) {
    f = PagedPlan{};
    if (const char* e = check_cache_sizes(a.c)) return e;
    if (a.numHeads == 0 || a.numHeads % a.c.numKvHeads != 0)
        return "numHeads must be a positive multiple of numKvHeads";
    if (a.seqLen == 0) return nullptr;
    if (!rows_fit(a.numHeads, a.c.numKvHeads, a.seqLen)) return "sequence too long";
    f = paged_plan(a);
    return f.step == 0 ? "problem too large for one launch" : nullptr;
}

}  // namespace

int pagedAppend(const PagedAppendParams& a, void* stream) {
    if (const char* e = check_cache(a.c)) return pfail(e);
    if (a.key == nullptr || a.value == nullptr) return pfail("null tensor pointer");
    if (a.seqLen == 0) return 0;
    if (a.seqLen > (1u << 30)) return pfail("sequence too long");
    if (!p16(a.key) || !p16(a.value)) return pfail("tensor base pointers must be 16-byte aligned");
    if (!p4(a.newLens)) return pfail("new_lens must be 4-byte aligned");
    if (const char* e = check_strides(a.kStrideB, a.kStrideH, a.kStrideS, a.c.batchSize, a.c.numKvHeads, a.seqLen))
        return pfail(e);
    if (const char* e = check_strides(a.vStrideB, a.vStrideH, a.vStrideS, a.c.batchSize, a.c.numKvHeads, a.seqLen))
        return pfail(e);
    if (const char* e = check_rope(a.rotCos, a.rotSin, a.positions, a.ropeRows)) return pfail(e);
    paged::AppendParams p{};
    p.k = paged::Rows{static_cast<const uint16_t*>(a.key), a.kStrideB, a.kStrideH, a.kStrideS};
    p.v = paged::Rows{static_cast<const uint16_t*>(a.value), a.vStrideB, a.vStrideH, a.vStrideS};
    p.kc = cache_view(a.c.kCache, a.c.kcStrideP, a.c.kcStrideH, a.c.kcStrideS);
    p.vc = cache_view(a.c.vCache, a.c.vcStrideP, a.c.vcStrideH, a.c.vcStrideS);
    p.t = make_table(a.c, a.newLens, a.seqLen);
    p.positions = static_cast<const int*>(a.positions);
    p.cos = static_cast<const float*>(a.rotCos);
    p.sin = static_cast<const float*>(a.rotSin);
    p.rope_rows = static_cast<int>(a.ropeRows);
    p.B = static_cast<int>(a.c.batchSize);
    p.Hkv = static_cast<int>(a.c.numKvHeads);
    p.D = static_cast<int>(a.c.headDim);
    const int64_t heads = static_cast<int64_t>(p.B) * p.Hkv, chunks = static_cast<int64_t>(a.seqLen) * (p.D / 8);
    if (heads > INT32_MAX || heads > int64_t{INT32_MAX} * 256 / chunks) return pfail("problem too large for one launch");
    p.n = heads * chunks;
    const unsigned grid = static_cast<unsigned>((p.n + 255) / 256);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a.c.dtype == paged::DT_F16)
        paged::append_kernel<paged::F16><<<grid, 256, 0, st>>>(p);
    else
        paged::append_kernel<paged::BF16><<<grid, 256, 0, st>>>(p);
    return launched();
}

int pagedAccept(const PagedAcceptParams& a, void* stream) {
    if (const char* e = check_cache(a.c)) return pfail(e);
    if (a.maxAccepted == 0) return 0;
    if (a.accepted == nullptr) return pfail("null tensor pointer");
    if (a.maxAccepted > static_cast<uint32_t>(paged::kMaxAccept)) return pfail("more than 256 accepted tokens");
    if (!p4(a.accepted) || !p4(a.acceptedLens)) return pfail("accepted and accepted_lens must be 4-byte aligned");
    if (a.c.batchSize > 65535) return pfail("too many sequences for one launch");
    paged::AcceptParams p{};
    p.kc = cache_view(a.c.kCache, a.c.kcStrideP, a.c.kcStrideH, a.c.kcStrideS);
    p.vc = cache_view(a.c.vCache, a.c.vcStrideP, a.c.vcStrideH, a.c.vcStrideS);
    p.t = make_table(a.c, nullptr, 0);
    p.accepted = static_cast<const int*>(a.accepted);
    p.accepted_lens = static_cast<const int*>(a.acceptedLens);
    p.A = static_cast<int>(a.maxAccepted);
    p.B = static_cast<int>(a.c.batchSize);
    p.Hkv = static_cast<int>(a.c.numKvHeads);
    p.D = static_cast<int>(a.c.headDim);
    p.n = 2 * p.Hkv * (p.D / 8);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p.A <= paged::kAcceptRegs) {
        const dim3 grid((p.n + 127) / 128, p.B);
        paged::accept_kernel<true><<<grid, 128, 0, st>>>(p);
        return launched();
    }
    // threads x rows x 16 bytes of staging: 128 threads up to 96 rows, else 32
    const int threads = p.A <= 96 ? 128 : 32;
    const cudaError_t ce = prepare_kernel<paged::accept_kernel<false>>(196608, 0);
    if (ce != cudaSuccess) return fail(g_err_paged, "%s", cudaGetErrorString(ce));
    const dim3 grid((p.n + threads - 1) / threads, p.B);
    paged::accept_kernel<false><<<grid, threads, threads * p.A * 16, st>>>(p);
    return launched();
}

size_t pagedAttentionWorkspaceBytes(const PagedAttentionParams& a) {
    PagedPlan f;
    return plan_attention(a, f) != nullptr ? 0 : f.bytes;
}

int pagedAttention(const PagedAttentionParams& a, void* workspace, size_t workspace_bytes, void* stream) {
    const PagedCacheParams& c = a.c;
    if (const char* e = check_cache(c)) return pfail(e);
    if (a.q == nullptr || a.o == nullptr) return pfail("null tensor pointer");
    PagedPlan f;
    if (const char* e = plan_attention(a, f)) return pfail(e);
    if (a.seqLen == 0) return 0;
    if (a.treeMask != nullptr && a.seqLen > static_cast<uint32_t>(paged::kMaxTree))
        return pfail("tree_mask: more than 256 tokens");
    if (!p16(a.q) || !p16(a.o)) return pfail("tensor base pointers must be 16-byte aligned");
    if (!p4(a.newLens)) return pfail("new_lens must be 4-byte aligned");
    if (const char* e = check_strides(a.qStrideB, a.qStrideH, a.qStrideS, c.batchSize, a.numHeads, a.seqLen))
        return pfail(e);
    if (const char* e = check_strides(a.oStrideB, a.oStrideH, a.oStrideS, c.batchSize, a.numHeads, a.seqLen))
        return pfail(e);
    if (a.treeMask != nullptr && (a.maskStrideB < 0 || a.maskStrideT < 0)) return pfail("strides must be positive");
    if (const char* e = check_rope(a.rotCos, a.rotSin, a.positions, a.ropeRows)) return pfail(e);

    if (workspace == nullptr || workspace_bytes < f.bytes)
        return pfail("workspace missing or smaller than rdna_attention_paged_workspace_size()");
    if (reinterpret_cast<uintptr_t>(workspace) & (kWsAlign - 1)) return pfail("workspace must be 256-byte aligned");

    paged::AttnParams p{};
    p.q = static_cast<const uint16_t*>(a.q);
    p.o = static_cast<uint16_t*>(a.o);
    p.qsb = a.qStrideB;
    p.qsh = a.qStrideH;
    p.qss = a.qStrideS;
    p.osb = a.oStrideB;
    p.osh = a.oStrideH;
    p.oss = a.oStrideS;
    p.t = make_table(c, a.newLens, a.seqLen);
    p.mask = static_cast<const uint8_t*>(a.treeMask);
    p.msb = a.maskStrideB;
    p.mst = a.maskStrideT;
    p.positions = static_cast<const int*>(a.positions);
    p.cos = static_cast<const float*>(a.rotCos);
    p.sin = static_cast<const float*>(a.rotSin);
    p.rope_rows = static_cast<int>(a.ropeRows);
    p.H = static_cast<int>(a.numHeads);
    p.Hkv = static_cast<int>(c.numKvHeads);
    p.G = p.H / p.Hkv;
    p.D = static_cast<int>(c.headDim);
    p.rows = static_cast<int>(static_cast<uint32_t>(p.G) * a.seqLen);
    p.RT = f.RT;
    p.n_rt = f.n_rt;
    p.tpp = f.tpp;
    p.by_G.set(static_cast<uint32_t>(p.G));
    p.by_P.set(c.pageSize);
    p.by_tpp.set(f.tpp == 0 ? 1 : static_cast<uint32_t>(f.tpp));
    p.window = a.windowSize > 0 ? a.windowSize : 0;
    // (never 0, which times a masked score of -inf would be NaN: a scale of 0 becomes the smallest
    // normal number, and products of up to 1e30 give scores below 2e-8, which no weight shows)
    p.scale_log2 = std::max(std::fabs(a.scale) * 1.4426950408889634f, std::numeric_limits<float>::min());
    p.flip = a.scale < 0.f ? 0x80008000u : 0u;
    p.ws = static_cast<float*>(workspace);
    p.units = reinterpret_cast<int2*>(static_cast<char*>(workspace) + f.partials);
    p.grid = f.grid;
    p.W = f.W;

    CUtensorMap tmK, tmV;
    const uint32_t box_rows = std::min<uint32_t>(c.pageSize, paged::KT);
    const CUtensorMapDataType dt =
        c.dtype == paged::DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const View4 vk{c.kCache, {c.headDim, c.pageSize, c.numKvHeads, c.numPages}, {c.kcStrideS, c.kcStrideH, c.kcStrideP}};
    const View4 vv{c.vCache, {c.headDim, c.pageSize, c.numKvHeads, c.numPages}, {c.vcStrideS, c.vcStrideH, c.vcStrideP}};
    const char* e = nullptr;
    if ((e = make_map(&tmK, vk, dt, 2, 64, box_rows, CU_TENSOR_MAP_SWIZZLE_128B)) ||
        (e = make_map(&tmV, vv, dt, 2, 64, box_rows, CU_TENSOR_MAP_SWIZZLE_128B)))
        return pfail(e);

    cudaStream_t st = static_cast<cudaStream_t>(stream);
    for (int64_t b0 = 0; b0 < c.batchSize; b0 += f.step) {
        paged::AttnParams s = p;
        s.B = static_cast<int>(std::min<int64_t>(c.batchSize - b0, f.step));
        s.by_B.set(static_cast<uint32_t>(s.B));
        s.q += b0 * p.qsb;
        s.o += b0 * p.osb;
        s.t.pages += b0 * p.t.stride;
        s.t.cache_lens += b0;
        if (s.t.new_lens != nullptr) s.t.new_lens += b0;
        if (s.mask != nullptr) s.mask += b0 * p.msb;
        if (s.positions != nullptr) s.positions += b0 * a.seqLen;
        // Both kernels may start while the one before them on the stream ends: the
        // attention kernel waits for it before it reads or writes global memory, the join
        // waits for the attention kernel.
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        cfg.stream = st;
        cfg.gridDim = dim3(static_cast<unsigned>(f.grid));
        auto launch = [&](auto list, int threads, int smem, int regs) {
            constexpr auto kern = decltype(list)::value;
            cfg.blockDim = dim3(threads);
            cfg.dynamicSmemBytes = smem;
            cudaError_t ce = prepare_kernel<kern>(smem, regs);
            if (ce != cudaSuccess) return ce;
            return launch_timed(st, [&] { return cudaLaunchKernelEx(&cfg, kern, tmK, tmV, s); });
        };
        // The cluster form, where it fits; else the list.  It takes a single sequence's units,
        // each by the widest cluster of which enough fit the device at once (8 units: 10 CTAs
        // each, 4 or fewer: 16), and joins the parts itself.  One token at head_dim 128, cluster
        // and list: 1024 slots, 8 KV heads 9.2 and 12.3 us; 4096 slots, 8, 4 and 1 heads 12.0 and
        // 12.9, 11.1 and 14.0, 10.8 and 13.2; 8192 slots 14.6 and 15.4, 12.6 and 14.1, 12.2 and
        // 16.9.  Its CTAs are fewer, though, and the list is ahead from about 18 key tiles per
        // CTA on (16384 slots: 21.0 and 19.7, 16.4 and 16.7, 15.6 and 17.3; 32768: 34.5 and 29.8,
        // 24.6 and 21.1, 22.3 and 18.6).  The lengths are on the device, so the width of the page
        // table bounds the tiles: a short sequence in a wide table takes the list.
        bool joined = false;
        auto launch_cluster = [&](auto cluster, int threads, int smem) {
            constexpr auto kern = decltype(cluster)::value;
            const int units = p.Hkv * p.n_rt;
            if (c.batchSize != 1 || units > kMaxPagedUnits) return cudaSuccess;
            cudaError_t ce = prepare_kernel<kern>(smem, 0, true);
            if (ce != cudaSuccess) return ce;
            int size = kMaxCluster;
            while (size > 1 && units > max_clusters<kern>(size, threads, smem)) --size;
            if (size == 1 || f.tiles > 18 * size) return cudaSuccess;
            attr[1].id = cudaLaunchAttributeClusterDimension;
            attr[1].val.clusterDim.x = size;
            attr[1].val.clusterDim.y = 1;
            attr[1].val.clusterDim.z = 1;
            cfg.numAttrs = 2;
            cfg.gridDim = dim3(units * size);
            cfg.blockDim = dim3(threads);
            cfg.dynamicSmemBytes = smem;
            joined = true;
            return launch_timed(st, [&] { return cudaLaunchKernelEx(&cfg, kern, tmK, tmV, s); });
        };
        auto by_width = [&](auto E) {
            using T = decltype(E);
            auto few = [&](auto W) {
                constexpr int w = decltype(W)::value;
                using L = paged::Layout<w>;
                const cudaError_t ce =
                    launch_cluster(Kernel<paged::fa_paged_kernel<T, w, true>>{}, L::THREADS, L::SMEM_BYTES);
                if (ce != cudaSuccess || joined) return ce;
                return launch(Kernel<paged::fa_paged_kernel<T, w, false>>{}, L::THREADS, L::SMEM_BYTES, 0);
            };
            auto many = [&](auto W) {
                constexpr int w = decltype(W)::value;
                using L = paged::MmaLayout<w>;
                return launch(Kernel<paged::fa_paged_mma_kernel<T, w>>{}, L::THREADS, L::SMEM_BYTES, L::LAUNCH_REGS);
            };
            const std::integral_constant<int, 64> w64;
            const std::integral_constant<int, 128> w128;
            if (f.mma) return f.dp == 64 ? many(w64) : many(w128);
            return f.dp == 64 ? few(w64) : f.dp == 128 ? few(w128) : few(std::integral_constant<int, 256>{});
        };
        cudaError_t ce = c.dtype == paged::DT_F16 ? by_width(paged::F16{}) : by_width(paged::BF16{});
        if (ce == cudaSuccess) ce = cudaGetLastError();
        if (ce != cudaSuccess) return fail(g_err_paged, "%s", cudaGetErrorString(ce));
        if (joined) continue;
        cfg.numAttrs = 1;
        const int64_t join_rows = static_cast<int64_t>(s.B) * p.Hkv * p.n_rt * f.RT;
        const bool wide = join_rows <= static_cast<int64_t>(f.grid) * paged::kJoinRows;
        unsigned rows = wide ? paged::kJoinRowsWide : paged::kJoinRows;
        while (wide && join_rows > static_cast<int64_t>(f.grid) * rows) rows *= 2;
        for (s.join_shift = 0; (1u << s.join_shift) < rows; ++s.join_shift) {
        }
        const unsigned width = rows * (c.headDim / 8), shares = wide ? paged::kJoinThreads / width : 1;
        cfg.gridDim = dim3(static_cast<unsigned>(join_rows / rows));
        cfg.blockDim = dim3(shares * width);
        cfg.dynamicSmemBytes = (shares - 1) * 10 * width * sizeof(float);
        auto join = [&](auto E) {
            using T = decltype(E);
            return wide ? cudaLaunchKernelEx(&cfg, paged::join_kernel<T, true>, s)
                        : cudaLaunchKernelEx(&cfg, paged::join_kernel<T, false>, s);
        };
        ce = c.dtype == paged::DT_F16 ? join(paged::F16{}) : join(paged::BF16{});
        if (ce == cudaSuccess) ce = cudaGetLastError();
        if (ce != cudaSuccess) return fail(g_err_paged, "%s", cudaGetErrorString(ce));
    }
    return 0;
}

const char* lastErrorPaged() { return g_err_paged[0] ? g_err_paged : nullptr; }

}  // namespace rdna
