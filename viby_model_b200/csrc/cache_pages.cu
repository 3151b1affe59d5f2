// Pages of a cache of states: copy, fork, reorder, compact and clear, in place, for all tensors in one launch.
//
// A page is row i of every tensor.  Moves may chain and cross (beam search replaces every row by some parent's), so no
// page may be overwritten before every reader of it is done.  The bytes at one offset of a page only ever meet the bytes
// at the same offset of other pages: a CTA therefore takes a strip of a few hundred bytes of ALL moved pages of one
// tensor, loads it into shared memory, waits, and stores it.  No second buffer, no order between CTAs, and a page that
// stays costs nothing.  Bound by HBM: every moved byte is read once and written once.
//
// Every CTA works out the list of moves by itself from the index arrays (a few hundred entries, from L2) and then walks
// strips; that is cheaper than a launch of its own for the plan.
//
// Measured: compacting half of 512 pages of 6 layers of linear attention states of 4 heads of 160 x 160 in 122 to 133 us (4.7
// to 5.1 TB/s, 0.72 to 0.78 of a plain copy's rate); small moves are latency: three pages of 18 such layers forked in 10 us.
#include <algorithm>

#include "vc1d_common.cuh"
#include "vc1d_internal.h"

namespace vc1d {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTensors = VC1D_PAGES_MAX_TENSORS;
constexpr int kMaxPages = VC1D_PAGES_MAX_PAGES;
constexpr int kMaxEntries = VC1D_PAGES_MAX_ENTRIES;  // a thread's step past the last one stays within 32 bits

// Dynamic shared memory of a launch: the list of moves, and a staging area.  48 KB keep four CTAs on an SM; many pages take
// more, so that a strip is at least a 16-byte column of all of them.
constexpr int moves_bytes(int pages) { return (4 * pages + 15) & ~15; }
constexpr int staging_bytes(int pages) { return std::max(48 << 10, 16 * pages); }
constexpr int kMostShared = moves_bytes(kMaxPages) + staging_bytes(kMaxPages);

struct PTensor {
    char* base;
    long long page_bytes, stride;
    int unit;  // largest of 16, 8, 4, 2, 1 that divides base, page_bytes and stride
};

struct PParams {
    PTensor t[kMaxTensors];
    const void *source, *dst;
    const uint8_t* live;
    int32_t *new_index, *count;
    long long sum_page_bytes;
    int op, pages, n_tensors, n, wide_index;
    int stage_bytes;
};

__device__ __forceinline__ long long index_at(const void* p, int wide, int i) {
    return wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

__device__ __forceinline__ unsigned pack_move(int dst, int src) { return (unsigned)dst << 16 | (unsigned)src; }

// Sum over the threads before this one; `total` gets the sum over all.  Two barriers.
__device__ __forceinline__ int block_scan(int x, int* warp_sums, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inc = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += y;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += warp_sums[w];
        all += warp_sums[w];
    }
    *total = all;
    return before + inc - x;
}

// The holes below the number of live pages take, in order, the live pages from there on.
__device__ __forceinline__ int plan_compact(const PParams& p, unsigned* moves, int* warp_sums) {
    const int per = (p.pages + kThreads - 1) / kThreads;
    const int i0 = min(p.pages, (int)threadIdx.x * per), i1 = min(p.pages, i0 + per);
    int live = 0, total, n_holes, n_tails;
    for (int i = i0; i < i1; ++i) live += p.live[i] != 0;
    block_scan(live, warp_sums, &total);
    int holes = 0, tails = 0;
    for (int i = i0; i < i1; ++i) {
        const bool on = p.live[i] != 0;
        holes += !on && i < total;
        tails += on && i >= total;
    }
    int h = block_scan(holes, warp_sums, &n_holes), t = block_scan(tails, warp_sums, &n_tails);  // n_holes == n_tails
    unsigned short* half = reinterpret_cast<unsigned short*>(moves);  // [2 m] source, [2 m + 1] destination
    for (int i = i0; i < i1; ++i) {
        const bool on = p.live[i] != 0;
        if (!on && i < total) half[2 * h++ + 1] = (unsigned short)i;
        if (on && i >= total) half[2 * t++] = (unsigned short)i;
    }
    __syncthreads();
    if (blockIdx.x == 0) {
        for (int i = threadIdx.x; i < p.pages; i += kThreads) p.new_index[i] = p.live[i] == 0 ? -1 : i;
        __syncthreads();
        for (int m = threadIdx.x; m < n_holes; m += kThreads) p.new_index[moves[m] & 0xffffu] = (int)(moves[m] >> 16);
        if (threadIdx.x == 0) *p.count = total;
    }
    return n_holes;
}

template <typename U>
__device__ __forceinline__ void load_strip(const PTensor& t, long long off, int width, int lg, const unsigned* moves, int m, char* stage) {
    // stage: one row of 2^lg bytes per move
    const int per = (int)((1u << lg) / sizeof(U)), lgu = lg - (31 - __clz((int)sizeof(U)));
    for (int e = threadIdx.x; e < m * per; e += kThreads) {
        const int row = e >> lgu, at = (e & (per - 1)) * (int)sizeof(U);
        if (at >= width) continue;
        const char* g = t.base + (long long)(moves[row] & 0xffffu) * t.stride + off + at;
        char* s = stage + ((long long)row << lg) + at;
        if constexpr (sizeof(U) == 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(s)), "l"(g) : "memory");
        else
            *reinterpret_cast<U*>(s) = *reinterpret_cast<const U*>(g);
    }
}

template <typename U>
__device__ __forceinline__ void store_strip(const PTensor& t, long long off, int width, int lg, const unsigned* moves, int m, const char* stage,
                                            bool zero) {
    const int per = (int)((1u << lg) / sizeof(U)), lgu = lg - (31 - __clz((int)sizeof(U)));
    for (int e = threadIdx.x; e < m * per; e += kThreads) {
        const int row = e >> lgu, at = (e & (per - 1)) * (int)sizeof(U);
        if (at >= width) continue;
        U x{};
        if (!zero) x = *reinterpret_cast<const U*>(stage + ((long long)row << lg) + at);
        *reinterpret_cast<U*>(t.base + (long long)(moves[row] >> 16) * t.stride + off + at) = x;
    }
}

__global__ void __launch_bounds__(kThreads) k_pages(const __grid_constant__ PParams p) {
    extern __shared__ __align__(16) char smem[];
    __shared__ int warp_sums[kWarps];
    __shared__ int s_moves;
    __shared__ long long first[kMaxTensors + 1];  // first strip of each tensor
    unsigned* moves = reinterpret_cast<unsigned*>(smem);           // [pages]
    char* stage = smem + ((4 * (long long)p.pages + 15) & ~15LL);  // [stage_bytes]
    const int tid = threadIdx.x;

    if (tid == 0) s_moves = 0;
    __syncthreads();
    int m;
    if (p.op == VC1D_PAGES_COMPACT) {
        m = plan_compact(p, moves, warp_sums);
    } else if (p.op == VC1D_PAGES_REORDER) {
        for (int i = tid; i < p.pages; i += kThreads) {
            const long long s = index_at(p.source, p.wide_index, i);
            if (s >= 0 && s < p.pages && s != i) moves[atomicAdd(&s_moves, 1)] = pack_move(i, (int)s);
        }
        __syncthreads();
        m = s_moves;
    } else {
        // of equal destinations the lowest entry counts: its number, by page, in the staging area (4 bytes a page)
        int* winner = reinterpret_cast<int*>(stage);
        for (int i = tid; i < p.pages; i += kThreads) winner[i] = 0x7fffffff;
        __syncthreads();
        const bool copy = p.op == VC1D_PAGES_COPY;
        for (int i = tid; i < p.n; i += kThreads) {
            const long long d = index_at(p.dst, p.wide_index, i), s = copy ? index_at(p.source, p.wide_index, i) : 0;
            if (d >= 0 && d < p.pages && s >= 0 && s < p.pages) atomicMin(&winner[d], i);
        }
        __syncthreads();
        for (int d = tid; d < p.pages; d += kThreads) {
            const int i = winner[d];
            if (i == 0x7fffffff) continue;
            const int s = copy ? (int)index_at(p.source, p.wide_index, i) : -1;
            if (s != d) moves[atomicAdd(&s_moves, 1)] = pack_move(d, max(s, 0));
        }
        __syncthreads();
        m = s_moves;
    }
    if (m == 0) return;

    // Strips of 2^lg bytes: as wide as the staging area allows for m pages, but no wider than gives every CTA one.
    const long long fit = p.stage_bytes / m, share = p.sum_page_bytes / gridDim.x;
    int lg = 63 - __clzll(fit);
    while (lg > 7 && (1LL << lg) > share) --lg;
    if (tid == 0) {
        long long n = 0;
        for (int i = 0; i < p.n_tensors; ++i) {
            first[i] = n;
            n += (p.t[i].page_bytes + (1LL << lg) - 1) >> lg;
        }
        first[p.n_tensors] = n;
    }
    __syncthreads();
    const long long strips = first[p.n_tensors];
    const bool zero = p.op == VC1D_PAGES_FREE;
    for (long long strip = blockIdx.x; strip < strips; strip += gridDim.x) {
        int lo = 0, hi = p.n_tensors;  // the tensor with first[lo] <= strip < first[lo + 1]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            (first[mid] <= strip ? lo : hi) = mid;
        }
        const PTensor& t = p.t[lo];
        const long long off = (strip - first[lo]) << lg;
        const int width = (int)min(1LL << lg, t.page_bytes - off);
        if (!zero) {
            switch (t.unit) {
                case 16: load_strip<uint4>(t, off, width, lg, moves, m, stage); break;
                case 8: load_strip<uint2>(t, off, width, lg, moves, m, stage); break;
                case 4: load_strip<uint32_t>(t, off, width, lg, moves, m, stage); break;
                case 2: load_strip<uint16_t>(t, off, width, lg, moves, m, stage); break;
                default: load_strip<uint8_t>(t, off, width, lg, moves, m, stage); break;
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            __syncthreads();
        }
        switch (t.unit) {
            case 16: store_strip<uint4>(t, off, width, lg, moves, m, stage, zero); break;
            case 8: store_strip<uint2>(t, off, width, lg, moves, m, stage, zero); break;
            case 4: store_strip<uint32_t>(t, off, width, lg, moves, m, stage, zero); break;
            case 2: store_strip<uint16_t>(t, off, width, lg, moves, m, stage, zero); break;
            default: store_strip<uint8_t>(t, off, width, lg, moves, m, stage, zero); break;
        }
        __syncthreads();
    }
}

// Whether two sets of pages share a byte: exact when their strides agree (layers interleaved in one pool), else by extent.
bool overlap(const vc1d_page_tensor& a, const vc1d_page_tensor& b, int pages) {
    const char *a0 = static_cast<const char*>(a.base), *b0 = static_cast<const char*>(b.base);
    const char *a1 = a0 + (pages - 1) * a.stride_bytes + a.page_bytes, *b1 = b0 + (pages - 1) * b.stride_bytes + b.page_bytes;
    if (a1 <= b0 || b1 <= a0) return false;
    if (pages == 1 || a.stride_bytes != b.stride_bytes) return true;  // one page: any stride is allowed, 0 too
    const long long s = a.stride_bytes, d = (((b0 - a0) % s) + s) % s;  // b's pages start d bytes after a's, modulo the stride
    return d < a.page_bytes || d + b.page_bytes > s;
}

bool meet(const void* a, long long a_bytes, const void* b, long long b_bytes) {
    const char *x = static_cast<const char*>(a), *y = static_cast<const char*>(b);
    return a_bytes > 0 && b_bytes > 0 && x < y + b_bytes && y < x + a_bytes;
}

// Whether an array of the call lies among a tensor's pages: every CTA reads the index arrays while others already store.
bool inside(const vc1d_page_tensor& t, int pages, const void* p, long long bytes) {
    if (p == nullptr || bytes == 0) return false;
    const char *lo = static_cast<const char*>(p), *t0 = static_cast<const char*>(t.base);
    return lo < t0 + (pages - 1) * t.stride_bytes + t.page_bytes && t0 < lo + bytes;
}

}  // namespace
}  // namespace vc1d

extern "C" {

VC1D_API int vc1d_pages(const vc1d_pages_args* a, void* stream) {
    using namespace vc1d;
    if (a == nullptr) return VC1D_E_NULL;
    if (a->struct_size != sizeof(vc1d_pages_args)) return VC1D_E_STRUCT;
    if (a->op < VC1D_PAGES_REORDER || a->op > VC1D_PAGES_COMPACT) return VC1D_E_SHAPE;
    if (a->pages < 0 || a->n_tensors < 0 || a->n < 0) return VC1D_E_SHAPE;
    if (a->pages > kMaxPages || a->n_tensors > kMaxTensors || a->n > kMaxEntries) return VC1D_E_TOO_LARGE;
    const bool compact = a->op == VC1D_PAGES_COMPACT, listed = a->op == VC1D_PAGES_COPY || a->op == VC1D_PAGES_FREE;
    if (!compact && a->index_dtype != VC1D_I32 && a->index_dtype != VC1D_I64) return VC1D_E_DTYPE;
    if (compact && (a->count == nullptr || (a->pages > 0 && (a->live == nullptr || a->new_index == nullptr)))) return VC1D_E_NULL;
    if (!compact && (a->pages == 0 || a->n_tensors == 0 || (listed && a->n == 0))) return VC1D_OK;
    if (a->op == VC1D_PAGES_REORDER && a->source == nullptr) return VC1D_E_NULL;
    if (listed && a->dst == nullptr) return VC1D_E_NULL;
    if (a->op == VC1D_PAGES_COPY && a->source == nullptr) return VC1D_E_NULL;
    if (a->n_tensors > 0 && a->tensors == nullptr) return VC1D_E_NULL;
    // one CTA writes new_index and count while the others read live
    if (compact && (meet(a->new_index, 4LL * a->pages, a->live, a->pages) || meet(a->count, 4, a->live, a->pages) ||
                    meet(a->count, 4, a->new_index, 4LL * a->pages)))
        return VC1D_E_ALIAS;
    static thread_local PParams p;
    p.n_tensors = 0;
    p.sum_page_bytes = 0;
    for (int i = 0; i < a->n_tensors; ++i) {
        const vc1d_page_tensor& t = a->tensors[i];
        if (t.page_bytes < 0 || (a->pages > 1 && t.stride_bytes < t.page_bytes)) return VC1D_E_STRIDE;
        if (t.page_bytes == 0 || a->pages == 0) continue;
        if (t.base == nullptr) return VC1D_E_NULL;
        const long long ib = a->index_dtype == VC1D_I64 ? 8 : 4;
        if (compact ? inside(t, a->pages, a->live, a->pages) || inside(t, a->pages, a->new_index, 4LL * a->pages) || inside(t, a->pages, a->count, 4)
                    : (a->op != VC1D_PAGES_FREE && inside(t, a->pages, a->source, ib * (listed ? a->n : a->pages))) ||
                          (listed && inside(t, a->pages, a->dst, ib * a->n)))
            return VC1D_E_ALIAS;
        for (int j = 0; j < i; ++j)
            if (a->tensors[j].page_bytes > 0 && overlap(a->tensors[j], t, a->pages)) return VC1D_E_ALIAS;
        PTensor& d = p.t[p.n_tensors++];
        d.base = static_cast<char*>(t.base);
        d.page_bytes = t.page_bytes;
        d.stride = a->pages > 1 ? t.stride_bytes : t.page_bytes;
        const unsigned long long all = reinterpret_cast<uintptr_t>(t.base) | (unsigned long long)d.page_bytes | (unsigned long long)d.stride;
        d.unit = (int)std::min<unsigned long long>(16, all & (~all + 1));
        p.sum_page_bytes += d.page_bytes;
    }
    p.source = a->source;
    p.dst = a->dst;
    p.live = a->live;
    p.new_index = a->new_index;
    p.count = a->count;
    p.op = a->op;
    p.pages = a->pages;
    p.n = a->n;
    p.wide_index = a->index_dtype == VC1D_I64;
    p.stage_bytes = staging_bytes(a->pages);
    const int smem = moves_bytes(a->pages) + p.stage_bytes;
    // The limit belongs to the function, not to the host thread: always the largest, or a call with few pages would lower
    // it between another thread's call with many and its launch.
    cudaError_t e = cudaFuncSetAttribute(k_pages, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared);
    if (e != cudaSuccess) return (int)e;
    const int per_sm = std::max(1, std::min(4, (220 << 10) / (smem + 2048)));
    const long long most = std::max<long long>(1, p.sum_page_bytes / 128 + p.n_tensors);
    const unsigned grid = (unsigned)std::min<long long>(most, (long long)per_sm * sm_count());
    note_launch("pages");
    k_pages<<<grid, kThreads, smem, static_cast<cudaStream_t>(stream)>>>(p);
    return (int)cudaGetLastError();
}

VC1D_API uint32_t vc1d_sizeof_pages_args(void) { return (uint32_t)sizeof(vc1d_pages_args); }

}  // extern "C"
