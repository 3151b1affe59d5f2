// Linear attention on the fifth-generation tensor cores (bf16, channel stride 1, 16-byte aligned rows, dims a multiple of
// 8, at most 160 state rows).
//
// One CTA per SM owns one (row, head), a slab of 64 state columns and a part of the time axis, and walks its chunks of 128
// tokens.  Per chunk four products of tcgen05.mma, all with fp32 accumulators in TMEM:
//     P  = q k^T                    [128 queries x 128 keys]
//     KV = k^T (w v)                [state rows x 64]: what the chunk adds to the state; w v in three bf16 parts (24 bits)
//     Oi = q X                      [128 x 64]: from the state X before the chunk, rounded to bf16
//     Oa = bf16(decay P) v          [128 x 64]: P goes back to TMEM as the operand
// and o = decay Oi + Oa.  The fp32 state stays in registers (a thread per row) and takes each chunk's KV with an fp32
// multiply-add: the tensor cores never accumulate onto it, because they truncate where an fp32 add rounds.
// Sixteen warps, each group with its own part, chunk after chunk, linked by mbarriers only:
//     warps 0-3   decays of P, its operand, then the output
//     warps 4-7   the state: X = a^n X + KV, and its bf16 copy in shared memory   (rows 128-159: warp 14)
//     warps 8-11  the weighted values, split into three parts
//     warp 12     issues the products;  warps 13, 15  load tokens (cp.async: masked rows arrive as zeros, unread)
// While one chunk's P is being decayed, the next chunk's tokens arrive and the state runs ahead.
//
// Shared memory holds every operand as panels of 64 channels: rows of 128 bytes with the 16-byte units XORed by the row
// modulo 8 (the 128-byte swizzle of the matrix descriptors).  A panel serves as K-major (channels summed: q, k) and as
// MN-major operand (tokens summed: k^T, v, w v; state rows summed: X) alike, so nothing is transposed.
//
// Every wait is bounded.  When one expires the CTA notes it (the library's count of expired waits) and gives up.
#pragma once

#include "linear_attention.cuh"
#include "prefill_tma.cuh"

namespace vc1d {
namespace lin {
namespace tc {

using tma::fence_async_smem;
using tma::mbar_arrive;
using tma::mbar_init;
using tma::mbar_test;
using tma::smem_u32;

constexpr int kC = 128;               // tokens of a chunk
constexpr int kThreads = 512;
constexpr int kLoaders = 64;
constexpr int kPow = kC + 2;          // a^0 .. a^(kC + 1)
constexpr int kCols = 64;             // columns of a slab
constexpr int kPanel = kC * 128;      // bytes of a panel of 128 rows
constexpr unsigned kSpin = 1u << 22;  // polls of 64 ns and more

// TMEM columns
constexpr uint32_t kTmP = 0, kTmPb = 128, kTmOi = 192, kTmOa = 256, kTmKV = 320, kTmKV2 = 384, kTmCols = 512;

enum Bar { kFull, kPRaw, kPRdy, kVwRdy, kKvDone, kKvFree, kXRdy, kQxDone, kPvDone, kOFree, kBars };

struct Info {  // of a chunk's tokens; a ring of four
    unsigned valid[4], start[4];
    int n_all, run_all;
    int n_before[4], run_before[4];  // before each word
};

template <int ROWS>
struct Layout {
    static constexpr int kPanels = ROWS / 64 + (ROWS % 64 != 0);
    static constexpr int kStages = ROWS <= 128 ? 2 : 1;  // of q and k; v has two
    static constexpr int kQ = 0;
    static constexpr int kK = kQ + kStages * kPanels * kPanel;
    static constexpr int kV = kK + kStages * kPanels * kPanel;
    static constexpr int kW = kV + 2 * kPanel;
    static constexpr int kX = kW + 3 * kPanel;
    static constexpr int kPowers = kX + ROWS * 128;
    static constexpr int kAdd = kPowers + 8 * kPow;
    static constexpr int kInfo = kAdd + 4 * kC;
    static constexpr int kBar = (kInfo + 4 * (int)sizeof(Info) + 15) & ~15;
    static constexpr int kMisc = kBar + 8 * 2 * kBars;
    static constexpr int kBytes = kMisc + 16;
};

// ---- tcgen05 ----
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr & 0x3ffffu) >> 4) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(sbo >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// K-major: rows of 128 bytes, groups of 8 rows 1024 bytes apart.  MN-major: 64 elements of a row, the next 64 a panel
// further; 8 summed rows are 1024 bytes.
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) { return desc(addr, 16, 1024); }
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr) { return desc(addr, kPanel, 1024); }
__host__ __device__ constexpr uint32_t idesc(int n, bool a_mn, bool b_mn) {  // bf16 x bf16 -> fp32, 128 rows
    return 1u << 4 | 1u << 7 | 1u << 10 | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | (uint32_t)(n / 8) << 17 | (uint32_t)(128 / 16) << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t i, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a),
                 "l"(b), "r"(i), "r"((uint32_t)add)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t i, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a),
                 "l"(b), "r"(i), "r"((uint32_t)add)
                 : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_ld32(float (&r)[32], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
                 : "r"(addr));
}
__device__ __forceinline__ void tm_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
// barrier of `threads` threads that tells all of them whether all said yes
__device__ __forceinline__ bool all_of(int id, int threads, bool yes) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\tbarrier.cta.red.and.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r)
                 : "r"(id), "r"(threads), "r"((uint32_t)yes)
                 : "memory");
    return r != 0;
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// ROWS: state rows the kernel is built for (128 or 160).
template <int ROWS, bool STATES>
__global__ void __launch_bounds__(kThreads, 1) k_linear_tc(const __grid_constant__ Launch l, unsigned int* timeouts) {
    using L = Layout<ROWS>;
    using T = __nv_bfloat16;
    constexpr int NS = L::kStages;
    constexpr bool kSecond = ROWS > 128;  // warp 14 holds rows 128 and up
    extern __shared__ unsigned char raw[];
    // the swizzle goes by address: panels start at multiples of 1024
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    unsigned char* sm = raw + (base - smem_u32(raw));
    float* pw_hi = reinterpret_cast<float*>(sm + L::kPowers);
    float* pw_lo = pw_hi + kPow;
    float* add = reinterpret_cast<float*>(sm + L::kAdd);
    Info* infos = reinterpret_cast<Info*>(sm + L::kInfo);
    uint32_t* misc = reinterpret_cast<uint32_t*>(sm + L::kMisc);  // [0] TMEM address, [1] a wait expired
    volatile uint32_t* dead = misc + 1;

    const Run& r = l.run[blockIdx.z];
    const Common& c = l.c;
    const int slabs = (r.dv + kCols - 1) / kCols;
    const int slab = blockIdx.x % slabs, bh = blockIdx.x / slabs, seg = blockIdx.y;
    if (bh >= c.batch * c.heads) return;  // a run with fewer slabs than the launch's widest
    const int b = bh / c.heads, h = bh % c.heads;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int c0 = slab * kCols, cols = min(kCols, r.dv - c0);
    const int t_begin = seg * c.seg_chunks * kC;
    const int t_end = min(c.seqlen, t_begin + c.seg_chunks * kC);
    const int chunks = (t_end - t_begin + kC - 1) / kC;

    auto bar = [&](int kind, int chunk) { return base + L::kBar + 8 * (2 * kind + (chunk & 1)); };
    // Waits until the event of `kind` that belongs to `chunk` has happened.  Each kind has two barriers, for even and odd
    // chunks: nobody who waits is ever two chunks behind, so a phase cannot be missed.
    auto wait = [&](int kind, int chunk) {
        const uint32_t addr = bar(kind, chunk), parity = (uint32_t)(chunk >> 1) & 1u;
        for (unsigned i = 0; i < kSpin; ++i) {
            if (mbar_test(addr, parity)) return true;
            if (*dead) return false;
            if (i > 64) __nanosleep(64);
        }
        *dead = 1;
        atomicAdd(timeouts, 1u);
        return false;
    };

    // by a whole warp, with one answer for all of it
    auto wait_warp = [&](int kind, int chunk) { return (bool)__all_sync(0xffffffffu, wait(kind, chunk)); };

    for (int n = tid; n < kPow; n += kThreads) {
        const float d = c.log_decay[h];
        const double x = n == 0 ? 1.0 : exp((double)d * (double)n);
        const float hi = (float)x;
        const double lo = x - (double)hi;
        pw_hi[n] = hi;
        pw_lo[n] = (isfinite(hi) && lo == lo) ? (float)lo : 0.f;
    }
    for (int i = tid; i < L::kPowers / 16; i += kThreads) reinterpret_cast<uint4*>(sm)[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) {
        misc[1] = 0;
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(kFull, i), kLoaders);
            mbar_init(bar(kPRaw, i), 1);
            mbar_init(bar(kPRdy, i), 128);
            mbar_init(bar(kVwRdy, i), 128);
            mbar_init(bar(kKvDone, i), 1);
            mbar_init(bar(kKvFree, i), kSecond ? 160 : 128);
            mbar_init(bar(kXRdy, i), kSecond ? 160 : 128);
            mbar_init(bar(kQxDone, i), 1);
            mbar_init(bar(kPvDone, i), 1);
            mbar_init(bar(kOFree, i), 128);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(misc)), "n"(kTmCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_async_smem();  // the zeros, before any product reads them
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tm = misc[0];
    const uint32_t tm_lane = tm + ((uint32_t)(warp & 3) << 21);  // a warp reaches the 32 lanes of its place in its group

    // n and run of token i of a chunk, up to and with i
    auto count = [&](const Info& f, int i, int* n, int* run) {
        const int w = i >> 5;
        const unsigned upto = 0xffffffffu >> (31 - (i & 31));
        *n = f.n_before[w] + __popc(f.valid[w] & upto);
        *run = f.run_before[w] + __popc(f.start[w] & upto);
    };

    if (warp < 4) {
        // ------------------------------------------------------------------------------ decays of P, output
        const int row = tid;
        const long long obase = (long long)b * r.o.sb + (long long)h * r.o.sh;
        for (int ch = 0; !STATES && ch < chunks; ++ch) {
            if (!wait_warp(kFull, ch) || !wait_warp(kPRaw, ch)) break;
            fence_after();
            const Info& f = infos[ch & 3];
            int n_i, run_i;
            count(f, row, &n_i, &run_i);
            const int code = n_i + (run_i << 8);
            const bool ok = f.valid[warp] >> lane & 1u, from_x = run_i == 0;
            const float carry = pw_hi[max(n_i - r.shift, 0)] * r.s_carry;
            const bool plain = f.n_all == kC && f.run_all == 0;  // every token valid, one sequence
#pragma unroll 1
            for (int blk = 0; blk < 4; ++blk) {  // 32 keys
                uint32_t p[16];
                if (blk > warp) {  // later than all queries of this warp
#pragma unroll
                    for (int j = 0; j < 16; ++j) p[j] = 0;
                } else {
                    float x[32];
                    tm_ld32(x, tm_lane + kTmP + 32 * blk);
                    tm_wait_ld();
                    if (plain && blk < warp) {
                        // a^(row - key) as the product of a power per row and one per key, neither above 1 for a decay
                        const float own = pw_hi[row - 32 * blk - 31] * r.s_pair;
#pragma unroll
                        for (int j = 0; j < 32; ++j) x[j] *= own * pw_hi[31 - j];
                    } else if (plain) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) x[j] = j <= lane ? x[j] * (pw_hi[max(lane - j, 0)] * r.s_pair) : 0.f;
                    } else {
                        const unsigned vb = f.valid[blk], sb = f.start[blk];
                        int n = f.n_before[blk], run = f.run_before[blk];
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            n += vb >> j & 1u;
                            run += sb >> j & 1u;
                            const unsigned lag = (unsigned)(code - (n + (run << 8)));
                            x[j] = lag <= (unsigned)kC ? x[j] * (pw_hi[lag] * r.s_pair) : 0.f;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) p[j] = pack(x[2 * j], x[2 * j + 1]);
                }
                tm_st16(tm_lane + kTmPb + 16 * blk, p);
            }
            tm_wait_st();
            fence_before();
            mbar_arrive(bar(kPRdy, ch));
            if (!wait_warp(kPvDone, ch)) break;
            fence_after();
            const int t = t_begin + ch * kC + row;
            T* po = const_cast<T*>(static_cast<const T*>(r.o.p)) + obase + (long long)t * r.o.st + c0;
#pragma unroll 1
            for (int half = 0; half < 2; ++half) {
                float x[32], y[32];
                tm_ld32(x, tm_lane + kTmOi + 32 * half);
                tm_ld32(y, tm_lane + kTmOa + 32 * half);
                tm_wait_ld();
                if (half == 1) {
                    fence_before();
                    mbar_arrive(bar(kOFree, ch));
                }
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    // a later sequence takes nothing of X, infinities neither
                    const float o = from_x ? fmaf(x[j], carry, y[j]) : y[j];
                    x[j] = ok ? o : 0.f;
                }
                if (t < t_end) {
                    if (r.out_vec) {
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            if (32 * half + 8 * u < cols)
                                st_vec(po + 32 * half + 8 * u, make_uint4(pack(x[8 * u], x[8 * u + 1]), pack(x[8 * u + 2], x[8 * u + 3]),
                                                                          pack(x[8 * u + 4], x[8 * u + 5]), pack(x[8 * u + 6], x[8 * u + 7])));
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            const int col = 32 * half + j;
                            if (col < cols) {
                                const long long at = obase + (long long)t * r.o.st + (long long)(c0 + col) * r.o.sd;
                                if (r.out_f32)
                                    const_cast<float*>(static_cast<const float*>(r.o.p))[at] = x[j];
                                else
                                    const_cast<T*>(static_cast<const T*>(r.o.p))[at] = __float2bfloat16_rn(x[j]);
                            }
                        }
                    }
                }
            }
        }
    } else if (warp < 8 || (kSecond && warp == 14)) {
        // ------------------------------------------------------------------------------ state
        const int row = (warp == 14 ? 128 : 32 * (warp - 4)) + lane;
        const uint32_t kv = tm_lane + (warp == 14 ? kTmKV2 : kTmKV);
        float X[kCols];
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
            float x = 0.f;
            if (!STATES && row < r.da && j < cols) {
                if (seg > 0)
                    x = c.seg_state[blockIdx.z][((long long)(seg - 1) * c.batch * c.heads + bh) * ((long long)r.da * r.dv) + (long long)row * r.dv + c0 + j];
                else if (r.x0.p != nullptr)
                    x = r.x0.p[(long long)b * r.x0.sb + (long long)h * r.x0.sh + (long long)row * r.x0.sr + (long long)(c0 + j) * r.x0.sc];
            }
            X[j] = x;
        }
        auto store_x = [&]() {
            unsigned char* p = sm + L::kX + row * 128;
#pragma unroll
            for (int u = 0; u < 8; ++u)
                *reinterpret_cast<uint4*>(p + ((u ^ (row & 7)) << 4)) =
                    make_uint4(pack(X[8 * u], X[8 * u + 1]), pack(X[8 * u + 2], X[8 * u + 3]), pack(X[8 * u + 4], X[8 * u + 5]), pack(X[8 * u + 6], X[8 * u + 7]));
            fence_async_smem();
        };
        if (!STATES && chunks > 0) {
            store_x();
            mbar_arrive(bar(kXRdy, 0));
        }
        double seg_factor = 1.0;
        bool fine = true;
        for (int ch = 0; ch < chunks; ++ch) {
            if (!wait_warp(kFull, ch) || !wait_warp(kKvDone, ch)) {
                fine = false;
                break;
            }
            fence_after();
            const Info& f = infos[ch & 3];
            const float2 fac = make_float2(pw_hi[f.n_all], pw_lo[f.n_all]);
            const bool keep = f.run_all == 0;
            if (STATES) seg_factor = keep ? seg_factor * ((double)fac.x + (double)fac.y) : 0.0;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float x[32];
                tm_ld32(x, kv + 32 * half);
                tm_wait_ld();
                if (half == 1) {
                    fence_before();
                    mbar_arrive(bar(kKvFree, ch));
                }
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    float* s = X + 32 * half + j;
                    float2 y = make_float2(x[j], x[j + 1]);
                    if (keep) y = fma2(make_float2(s[0], s[1]), make_float2(fac.x, fac.x), fma2(make_float2(s[0], s[1]), make_float2(fac.y, fac.y), y));
                    s[0] = y.x;
                    s[1] = y.y;
                }
            }
            if (!STATES && ch + 1 < chunks) {
                if (!wait_warp(kQxDone, ch)) {  // this chunk's queries have read the copy
                    fine = false;
                    break;
                }
                store_x();
                mbar_arrive(bar(kXRdy, ch + 1));
            }
        }
        if (fine && row < r.da && (STATES || (seg == c.segments - 1 && r.xT.p != nullptr))) {
            float* dst = STATES ? c.seg_state[blockIdx.z] + ((long long)seg * c.batch * c.heads + bh) * ((long long)r.da * r.dv) + (long long)row * r.dv
                                : r.xT.p + (long long)b * r.xT.sb + (long long)h * r.xT.sh + (long long)row * r.xT.sr;
            const long long sc = STATES ? 1 : r.xT.sc;
#pragma unroll
            for (int j = 0; j < kCols; ++j)
                if (j < cols) dst[(long long)(c0 + j) * sc] = X[j];
            if (STATES && slab == 0 && row == 0) {
                const float hi = (float)seg_factor;
                c.seg_factor[blockIdx.z][(long long)seg * c.batch * c.heads + bh] = make_float2(hi, (float)(seg_factor - (double)hi));
            }
        }
    } else if (warp < 12) {
        // ------------------------------------------------------------------------------ weighted values
        const int me = tid - 256;
        for (int ch = 0; ch < chunks; ++ch) {
            const bool ok = wait(kFull, ch) && (ch == 0 || wait(kKvDone, ch - 1));
            if (!all_of(1, 128, ok)) break;  // the weights of the chunk before are no longer read
            const Info& f = infos[ch & 3];
            {
                int n, run;
                count(f, me, &n, &run);
                add[me] = run == f.run_all ? pw_hi[f.n_all - n + r.shift] * r.s_add : 0.f;
                asm volatile("bar.sync 1, 128;" ::: "memory");
            }
            const unsigned char* v = sm + L::kV + (ch & 1) * kPanel;
            unsigned char* w = sm + L::kW;
            const int at = ((me & 7) ^ (me >> 3 & 7)) << 4;  // rows 16 apart have the same swizzle
#pragma unroll 2
            for (int i = 0; i < 8; ++i) {
                const int tok = (me >> 3) + 16 * i;
                const uint4 in = *reinterpret_cast<const uint4*>(v + tok * 128 + at);
                const float2 wt = make_float2(add[tok], add[tok]);
                const uint32_t e[4] = {in.x, in.y, in.z, in.w};
                uint32_t part[3][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float2 x = mul2(make_float2(__uint_as_float(e[j] << 16), __uint_as_float(e[j] & 0xffff0000u)), wt);
                    // three parts cut off the top, eight bits each: nothing of the 24 is lost
#pragma unroll
                    for (int p = 0; p < 3; ++p) {
                        part[p][j] = __byte_perm(__float_as_uint(x.x), __float_as_uint(x.y), 0x7632);
                        if (p < 2)
                            x = fma2(make_float2(__uint_as_float(__float_as_uint(x.x) & 0xffff0000u), __uint_as_float(__float_as_uint(x.y) & 0xffff0000u)),
                                     make_float2(-1.f, -1.f), x);
                    }
                }
#pragma unroll
                for (int p = 0; p < 3; ++p)
                    *reinterpret_cast<uint4*>(w + p * kPanel + tok * 128 + at) = make_uint4(part[p][0], part[p][1], part[p][2], part[p][3]);
            }
            fence_async_smem();
            mbar_arrive(bar(kVwRdy, ch));
        }
    } else if (warp == 12) {
        // ------------------------------------------------------------------------------ products
        if (lane == 0) {
            const int steps = (r.da + 15) / 16;
            const uint32_t q0 = base + L::kQ, k0 = base + L::kK, v0 = base + L::kV, w0 = base + L::kW, x0 = base + L::kX;
            for (int ch = 0; ch < chunks; ++ch) {
                const uint32_t q = q0 + (ch % NS) * L::kPanels * kPanel, k = k0 + (ch % NS) * L::kPanels * kPanel, v = v0 + (ch & 1) * kPanel;
                if (!wait(kFull, ch)) break;
                fence_after();
                if (!STATES) {
                    for (int s = 0; s < steps; ++s) {
                        const uint32_t off = (s >> 2) * kPanel + (s & 3) * 32;
                        mma_ss(tm + kTmP, desc_k(q + off), desc_k(k + off), idesc(128, false, false), s > 0);
                    }
                    commit(bar(kPRaw, ch));
                }
                if (!wait(kVwRdy, ch) || (ch > 0 && !wait(kKvFree, ch - 1))) break;
                fence_after();
#pragma unroll 1
                for (int tile = 0; tile < (kSecond ? 2 : 1); ++tile)  // rows 0-127; 64-191, of which 128-159 are used
#pragma unroll 1
                    for (int p = 2; p >= 0; --p)
                        for (int s = 0; s < kC / 16; ++s)
                            mma_ss(tm + (tile ? kTmKV2 : kTmKV), desc_mn(k + tile * kPanel + s * 2048), desc_mn(w0 + p * kPanel + s * 2048),
                                   idesc(64, true, true), p < 2 || s > 0);
                commit(bar(kKvDone, ch));
                if (!STATES) {
                    if (!wait(kXRdy, ch) || (ch > 0 && !wait(kOFree, ch - 1))) break;
                    fence_after();
                    for (int s = 0; s < steps; ++s)
                        mma_ss(tm + kTmOi, desc_k(q + (s >> 2) * kPanel + (s & 3) * 32), desc_mn(x0 + s * 2048), idesc(64, false, true), s > 0);
                    commit(bar(kQxDone, ch));
                    if (!wait(kPRdy, ch)) break;
                    fence_after();
                    for (int s = 0; s < kC / 16; ++s) mma_ts(tm + kTmOa, tm + kTmPb + 8 * s, desc_mn(v + s * 2048), idesc(64, false, true), s > 0);
                    commit(bar(kPvDone, ch));
                }
            }
        }
        __syncwarp();
    } else if (warp != 14) {
        // ------------------------------------------------------------------------------ tokens
        const int me = (warp == 13 ? 0 : 32) + lane;
        const T* pa = static_cast<const T*>(r.a.p) + (long long)b * r.a.sb + (long long)(h / r.a.group) * r.a.sh;
        const T* pk = static_cast<const T*>(r.k.p) + (long long)b * r.k.sb + (long long)(h / r.k.group) * r.k.sh;
        const T* pv = static_cast<const T*>(r.v.p) + (long long)b * r.v.sb + (long long)(h / r.v.group) * r.v.sh + c0;
        auto fill_info = [&](int ch) {  // by one warp
            Info* f = infos + (ch & 3);
            const int t0 = t_begin + ch * kC;
            int n = 0, run = 0;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int t = t0 + 32 * w + lane;
                const long long at = r.reverse ? c.seqlen - 1 - t : t;
                bool v = t < t_end, s = false;
                if (v && c.mask != nullptr) v = mask_valid(c.mask, c.mask_dtype, (long long)b * c.mask_sb + at * c.mask_st);
                if (t < t_end && c.seq_idx != nullptr && t > 0) {
                    const int32_t* p = c.seq_idx + (long long)b * c.seq_sb + at * c.seq_st;
                    s = p[0] != (r.reverse ? p[c.seq_st] : p[-c.seq_st]);
                }
                const unsigned vb = __ballot_sync(0xffffffffu, v), sb = __ballot_sync(0xffffffffu, s);
                if (lane == 0) {
                    f->valid[w] = vb;
                    f->start[w] = sb;
                    f->n_before[w] = n;
                    f->run_before[w] = run;
                }
                n += __popc(vb);
                run += __popc(sb);
            }
            if (lane == 0) {
                f->n_all = n;
                f->run_all = run;
            }
        };
        // 16-byte pieces: a thread has the pieces `me & 7` of every eighth row of a panel
        auto load_panel = [&](const Info& f, const T* src, long long st, bool has, uint32_t dst) {
            const int u = me & 7;
#pragma unroll 4
            for (int row = me >> 3; row < kC; row += kLoaders / 8) {
                const bool ok = f.valid[row >> 5] >> (row & 31) & 1u;
                if (has) cp16(dst + row * 128 + ((u ^ (row & 7)) << 4), ok ? src + row * st + u * 8 : src, ok);
            }
        };
        if (warp == 13 && chunks > 0) fill_info(0);
        for (int ch = 0; ch < chunks; ++ch) {
            bool ok = ch < NS || (wait(kKvDone, ch - NS) && (STATES || wait(kQxDone, ch - NS)));
            ok = ok && (ch < 2 || (wait(kKvDone, ch - 2) && wait(kKvFree, ch - 2) && (STATES || wait(kPvDone, ch - 2))));
            if (!all_of(2, kLoaders, ok)) break;  // this chunk's info is there
            const Info& f = infos[ch & 3];
            const long long t0 = t_begin + ch * kC;
            for (int p = 0; p < L::kPanels; ++p) {
                const bool has = p * 64 + (me & 7) * 8 < r.da;
                load_panel(f, pk + t0 * r.k.st + p * 64, r.k.st, has, base + L::kK + ((ch % NS) * L::kPanels + p) * kPanel);
                if (!STATES) load_panel(f, pa + t0 * r.a.st + p * 64, r.a.st, has, base + L::kQ + ((ch % NS) * L::kPanels + p) * kPanel);
            }
            load_panel(f, pv + t0 * r.v.st, r.v.st, (me & 7) * 8 < cols, base + L::kV + (ch & 1) * kPanel);
            if (warp == 13 && ch + 1 < chunks) fill_info(ch + 1);
            asm volatile("cp.async.wait_all;" ::: "memory");
            fence_async_smem();
            mbar_arrive(bar(kFull, ch));
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    if (warp == 12) {
        fence_after();
        if (*dead && lane == 0) {
            // products may still be under way: they end by themselves, and TMEM has to outlive them
            mbar_init(base + L::kBar, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            commit(base + L::kBar);
            for (unsigned i = 0; i < kSpin && !mbar_test(base + L::kBar, 0); ++i) __nanosleep(64);
        }
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "n"(kTmCols));
    }
}

template <int ROWS, bool STATES>
cudaError_t launch(const Launch& l, unsigned int* timeouts, cudaStream_t s) {
    constexpr int smem = Layout<ROWS>::kBytes + 1008;  // and what aligning the panels takes
    static_assert(smem <= 232448, "shared memory of an SM");
    int slabs = 0;
    for (int i = 0; i < l.runs; ++i) slabs = max(slabs, (l.run[i].dv + kCols - 1) / kCols);
    auto kernel = k_linear_tc<ROWS, STATES>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned)(l.c.batch * l.c.heads * slabs), STATES ? l.c.segments - 1 : l.c.segments, l.runs);
    note_launch(STATES ? "linear_tc_states" : "linear_tc");
    kernel<<<grid, kThreads, smem, s>>>(l, timeouts);
    return cudaGetLastError();
}

}  // namespace tc
}  // namespace lin
}  // namespace vc1d
