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
// Six groups of four warps, each with its own part, chunk after chunk, linked by mbarriers only:
//     warps 0-3    decays of P and its operand for the keys 0-63, then the columns 0-31 of the output
//     warps 4-7    the state: X = a^n X + KV, and its bf16 copy in shared memory   (rows 128-159: warp 22)
//     warps 8-15   the weighted values, split into three parts
//     warps 16-19  the same for the keys 64-127 and the columns 32-63
//     warp 20      issues the products
//     warp 21      brings tokens in by TMA (the 128-byte swizzle and the zeros past the last token are the copy's)
//     warp 23      says which tokens of a chunk count; where there is a mask, clears the rows of masked ones, whatever they
//                  hold, and hands the chunk over
// The parts are short programs of a few hundred instructions at five or so cycles each, so it is the longest part that
// sets the pace: that is why there are so many, and twice the warps for the weighted values.
// While one chunk's P is being decayed, the next chunk's tokens arrive and the state runs ahead.
//
// What bounds it: shared memory and the chain of a chunk.  A chunk of 128 state rows moves some 440 KB through shared memory
// (KV reads k^T three times, once for each part), 3400 cycles of the 5300 that a chunk takes; with 160 rows it is 620 KB,
// 4900 of 7200 to 9000.  The tensor cores work for less than a third of the time, HBM for a sixth.  Launches of a captured
// graph: 8 x 1024 tokens of 16 heads of 128 64 us (the warp-level kernel: 123); 64 x 1024 of 4 heads of 128 118 us, of 160
// 224 us; 65536 tokens of 16 heads of 128, three launches, 620 us, 0.26 of the rate that memory would allow.  80 registers
// a thread leave spills of 88 bytes (128 rows) and 184 (160 rows), none where only states are wanted.
// Measured and not taken: a second warp that issues products, weighing in two halves, a second buffer of keys for 160
// rows (their last 32 channels as half a panel).  On one and the same GPU together 631 us instead of 637 for the last of
// these, but 1069 instead of 996 for a training step of heads of 160, because the warp that clears masked rows then also
// asks for tokens.
//
// Shared memory holds every operand as panels of 64 channels: rows of 128 bytes with the 16-byte units XORed by the row
// modulo 8 (the 128-byte swizzle of the matrix descriptors).  A panel serves as K-major (channels summed: q, k) and as
// MN-major operand (tokens summed: k^T, v, w v; state rows summed: X) alike, so nothing is transposed.  A run from the last
// token to the first takes its chunks from the end and keeps the tokens of a chunk in their natural order; only the
// powers of the decay know the direction.
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
constexpr int kThreads = 768;
constexpr int kSmallRegs = 64, kLargeRegs = 112;  // four groups and two: six times the 80 of the launch
constexpr int kRegisterShare = 4 * 128 * kSmallRegs + 2 * 128 * kLargeRegs;
static_assert(kRegisterShare <= 65536, "registers of an SM");
constexpr int kWeighers = 256;
constexpr int kWholeChunks = 4096;  // chunks that are looked over beforehand; later ones count as not whole
constexpr int kPow = kC + 2;          // a^0 .. a^(kC + 1)
constexpr int kCols = 64;             // columns of a slab
constexpr int kPanel = kC * 128;      // bytes of a panel of 128 rows

// Polls after which a wait gives up: about a second, where a chunk takes microseconds.  A poll that fails takes 1.6 us and more:
// try_wait itself waits (1.5 us measured), and a sleep of 64 ns follows.  A constant: as an argument it costs spills.
constexpr unsigned kMaxPolls = 1u << 18;

// TMEM columns
// P has two buffers, for even and odd chunks, so that the next chunk's products need not wait for this one's decays.  The
// operand made from P takes P's place: keys 0-63 in columns 0-31, keys 64-127 in columns 64-95, each over products that
// the warps which write it have read themselves.
constexpr uint32_t kTmP = 0, kTmOi = 256, kTmOa = 320, kTmKV = 384, kTmKV2 = 448, kTmCols = 512;
__host__ __device__ constexpr uint32_t operand_column(int blk) { return (blk >> 1) * 64 + (blk & 1) * 16; }  // of 32 keys

enum Bar { kTmaQ, kTmaK, kTmaV, kQFull, kKFull, kVFull, kPRaw, kPRdy, kVwRdy, kKvDone, kKvFree, kXRdy, kQxDone, kPvDone, kOFree, kBars };

struct Info {  // of a chunk's tokens, bit i of word i / 32 for token i; a ring of four
    unsigned valid[4], start[4];
    int n_all, run_all;
    int n_before[4], run_before[4];  // in the words below
};
struct Maps {
    CUtensorMap a, k, v;
};
struct AllMaps {
    Maps run[kMaxRuns];
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
    static constexpr int kBlock = kX + ROWS * 128;
    static constexpr int kPowers = kBlock + 256;  // 32 zeros before them
    static constexpr int kAdd = kPowers + 8 * kPow;
    static constexpr int kWhole = kAdd + 4 * kC;  // bit per chunk: no token is masked
    static constexpr int kInfo = kWhole + kWholeChunks / 8;
    static constexpr int kBar = (kInfo + 4 * (int)sizeof(Info) + 15) & ~15;
    static constexpr int kMisc = kBar + 8 * 2 * kBars;
    static constexpr int kBytes = kMisc + 32;
};

// ---- tcgen05 ----
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr & 0x3ffffu) >> 4) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(sbo >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// the same matrix `bytes` further
__device__ __forceinline__ uint64_t at(uint64_t d, uint32_t bytes) { return d + (bytes >> 4); }
// K-major: rows of 128 bytes, groups of 8 rows 1024 bytes apart.  MN-major: 64 elements of a row, the next 64 a panel
// further; 8 summed rows are 1024 bytes.
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) { return desc(addr, 16, 1024); }
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr) { return desc(addr, kPanel, 1024); }
__host__ __device__ constexpr uint32_t idesc(int n, bool a_mn, bool b_mn) {  // bf16 x bf16 -> fp32, 128 rows
    return 1u << 4 | 1u << 7 | 1u << 10 | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | (uint32_t)(n / 8) << 17 | (uint32_t)(128 / 16) << 24;
}
// Called by a whole warp, with one lane that issues: descriptors then come from the warp's uniform registers, without a
// move from a lane's registers for every operand (a thread of its own took twice as long to issue a product).
__device__ __forceinline__ bool elect_lane() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ void mma_ss(bool leader, uint32_t d, uint64_t a, uint64_t b, uint32_t i, bool add) {
    if (leader)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a),
                     "l"(b), "r"(i), "r"((uint32_t)add)
                     : "memory");
}
__device__ __forceinline__ void mma_ts(bool leader, uint32_t d, uint32_t a, uint64_t b, uint32_t i, bool add) {
    if (leader)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a),
                     "l"(b), "r"(i), "r"((uint32_t)add)
                     : "memory");
}
// after the products that the same lane has issued
__device__ __forceinline__ void commit(bool leader, uint32_t bar) {
    if (leader) asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
// The loaded values pass through the wait, so that no use of them can be scheduled before it.
__device__ __forceinline__ void tm_wait_ld(float (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]), "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tm_wait_ld(float (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]), "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]), "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]), "+f"(r[23]), "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_ld32(float (&r)[32], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
                 : "r"(addr));
}
__device__ __forceinline__ void tm_ld16(float (&r)[16], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
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
__device__ __forceinline__ void few_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kSmallRegs)); }
__device__ __forceinline__ void many_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kLargeRegs)); }
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map),
                 "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// A bounded wait.
__device__ __forceinline__ bool poll(uint32_t addr, uint32_t parity, volatile uint32_t* dead, unsigned int* timeouts) {
#pragma unroll 1
    for (unsigned i = 0; i < kMaxPolls; ++i) {
        if (mbar_test(addr, parity)) return true;
        if (*dead) return false;
        if (i > 64) __nanosleep(64);
    }
    *dead = 1;
    atomicAdd(timeouts, 1u);
    return false;
}

// ROWS: state rows the kernel is built for (128 or 160).  REV: tokens run from the last to the first; a constant, because
// the hot code of all parts together has to stay in the SM's instruction cache.
template <int ROWS, bool STATES, bool REV>
__global__ void __launch_bounds__(kThreads, 1) k_linear_tc(const __grid_constant__ Launch l, const __grid_constant__ AllMaps maps, unsigned int* timeouts) {
    using L = Layout<ROWS>;
    using T = __nv_bfloat16;
    constexpr int NS = L::kStages;
    constexpr bool kSecond = ROWS > 128;  // warp 22 holds rows 128 and up
    extern __shared__ __align__(1024) unsigned char sm[];  // the swizzle goes by address: panels start at multiples of 1024
    const uint32_t base = smem_u32(sm);
    float* block = reinterpret_cast<float*>(sm + L::kBlock);  // a^31 .. a^0; a^0 .. a^31 in a reversed run
    float* pw_hi = reinterpret_cast<float*>(sm + L::kPowers);
    float* pw_lo = pw_hi + kPow;
    float* add = reinterpret_cast<float*>(sm + L::kAdd);
    Info* infos = reinterpret_cast<Info*>(sm + L::kInfo);
    uint32_t* misc = reinterpret_cast<uint32_t*>(sm + L::kMisc);  // [0] TMEM address, [1] a wait expired, [2-3] a last barrier, [4-6] chunks asked for, [7] chunks announced
    volatile uint32_t* dead = misc + 1;

    const Run& r = l.run[blockIdx.z];
    const Common& c = l.c;
    const int slabs = (r.dv + kCols - 1) / kCols;
    const int slab = blockIdx.x % slabs, bh = blockIdx.x / slabs, seg = blockIdx.y;
    if (bh >= c.batch * c.heads) return;  // a run with fewer slabs than the launch's widest
    if ((base & 1023u) != 0) {  // cannot be: the array says so
        if (threadIdx.x == 0) atomicAdd(timeouts, 1u);
        return;
    }
    const int b = bh / c.heads, h = bh % c.heads;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int c0 = slab * kCols, cols = min(kCols, r.dv - c0);
    constexpr bool rev = REV;
    // tokens in the run's order; a chunk's first token in natural order, negative where the last chunk of a reversed run
    // reaches past the first token
    const int t_begin = seg * c.seg_chunks * kC;
    const int t_end = min(c.seqlen, t_begin + c.seg_chunks * kC);
    int chunks = (t_end - t_begin + kC - 1) / kC, skipped = 0;  // padding at either end is not walked
    auto first_token = [&](int ch) { return rev ? c.seqlen - t_begin - (skipped + ch + 1) * kC : t_begin + (skipped + ch) * kC; };

    // the weighted values of a chunk; where no queries are needed their buffers hold those of every other chunk
    auto weighted = [&](int ch) { return STATES && (ch & 1) ? L::kQ : L::kW; };
    unsigned* whole = reinterpret_cast<unsigned*>(sm + L::kWhole);
    // whether rows of the chunk may have to be cleared: the copy then reports to the warp that does so
    auto to_clear = [&](int ch) { return c.mask != nullptr && !(skipped + ch < kWholeChunks && (whole[(skipped + ch) >> 5] >> ((skipped + ch) & 31) & 1u)); };
    auto bar = [&](int kind, int chunk) { return base + L::kBar + 8 * (2 * kind + (chunk & 1)); };
    // Waits until the event of `kind` that belongs to `chunk` has happened.  Each kind has two barriers, for even and odd
    // chunks: nobody who waits is ever two chunks behind, so a phase cannot be missed.
    auto wait = [&](int kind, int chunk) { return poll(bar(kind, chunk), (uint32_t)(chunk >> 1) & 1u, dead, timeouts); };
    // by a whole warp, with one answer for all of it
    auto wait_warp = [&](int kind, int chunk) { return (bool)__all_sync(0xffffffffu, wait(kind, chunk)); };

    for (int n = tid; n < kPow; n += kThreads) {
        const float d = c.log_decay[h];
        const double x = n == 0 ? 1.0 : exp((double)d * (double)n);
        const float hi = (float)x;
        const double lo = x - (double)hi;
        pw_hi[n] = hi;
        pw_lo[n] = (isfinite(hi) && lo == lo) ? (float)lo : 0.f;
        if (n < 32) block[rev ? n : 31 - n] = hi, pw_hi[n - 32] = 0.f;
    }
    // panels of k that the head does not reach are read as rows of the state all the same; every other byte is written first
    for (int p = (r.da + 63) / 64; p < L::kPanels; ++p)
        for (int i = tid; i < NS * kPanel / 16; i += kThreads)
            *reinterpret_cast<uint4*>(sm + L::kK + (i / (kPanel / 16) * L::kPanels + p) * kPanel + i % (kPanel / 16) * 16) = make_uint4(0, 0, 0, 0);
    if (tid == 0) {
        misc[1] = misc[4] = misc[5] = misc[6] = misc[7] = 0;
        for (int i = 0; i < 2; ++i) {
            for (int x = 0; x < 3; ++x) {
                mbar_init(bar(kTmaQ + x, i), 1);
                mbar_init(bar(kQFull + x, i), kQFull + x == kVFull ? 2 : 1);  // values: and the chunk's info
            }
            mbar_init(bar(kPRaw, i), 2);   // the products, and the chunk's info
            mbar_init(bar(kPRdy, i), 256);
            mbar_init(bar(kVwRdy, i), kWeighers);
            mbar_init(bar(kKvDone, i), 2);
            mbar_init(bar(kKvFree, i), kSecond ? 160 : 128);
            mbar_init(bar(kXRdy, i), kSecond ? 160 : 128);
            mbar_init(bar(kQxDone, i), 1);
            mbar_init(bar(kPvDone, i), 1);
            mbar_init(bar(kOFree, i), 256);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 20) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(misc)), "n"(kTmCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_async_smem();  // the zeros, before any product reads them
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tm = misc[0];
    if (c.mask != nullptr && chunks > 0) {
        // chunks between the first and the last valid token, in the run's order; the outputs of the others are zeros
        int* range = reinterpret_cast<int*>(add);
        if (tid == 0) range[0] = chunks, range[1] = -1;
        for (int i = tid; i < kWholeChunks / 32; i += kThreads) whole[i] = 0;
        __syncthreads();
        for (int ch = warp; ch < chunks; ch += kThreads / 32) {
            int n = 0;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int i = t_begin + ch * kC + 32 * w + lane;
                const bool v = i < t_end && mask_valid(c.mask, c.mask_dtype, (long long)b * c.mask_sb + (long long)(rev ? c.seqlen - 1 - i : i) * c.mask_st);
                n += __popc(__ballot_sync(0xffffffffu, v));
            }
            if (lane == 0 && n > 0) {
                atomicMin(&range[0], ch);
                atomicMax(&range[1], ch);
                if (n == kC && ch < kWholeChunks) atomicOr(&whole[ch >> 5], 1u << (ch & 31));
            }
        }
        __syncthreads();
        const int lo = range[0], hi = range[1];
        __syncthreads();  // the array gets its own use
        if (!STATES) {
            const int eb = r.out_f32 ? 4 : 2, before = max(0, min(t_end, t_begin + lo * kC) - t_begin), after = hi < 0 ? t_end : min(t_end, t_begin + (hi + 1) * kC);
            char* o = const_cast<char*>(static_cast<const char*>(r.o.p)) + ((long long)b * r.o.sb + (long long)h * r.o.sh + (long long)c0 * r.o.sd) * eb;
            const long long n = (long long)(before + t_end - after) * kCols;  // 2^25 padded tokens pass 31 bits
            for (long long i = tid; i < n; i += kThreads) {
                const int row = (int)(i / kCols), col = (int)(i % kCols), at = row < before ? t_begin + row : after + row - before;
                if (col >= cols) continue;
                char* q = o + ((long long)(rev ? c.seqlen - 1 - at : at) * r.o.st + col * r.o.sd) * eb;
                if (r.out_f32)
                    *reinterpret_cast<float*>(q) = 0.f;
                else
                    *reinterpret_cast<T*>(q) = __float2bfloat16_rn(0.f);
            }
        }
        skipped = hi < 0 ? 0 : lo;
        chunks = hi < 0 ? 0 : hi - lo + 1;
    }
    const uint32_t tm_lane = tm + ((uint32_t)(warp & 3) << 21);  // a warp reaches the 32 lanes of its place in its group

    // Valid tokens and sequence starts of a chunk up to and with token i, in the run's order.
    auto count = [&](const Info& f, int i, int* n, int* run) {
        const int w = i >> 5;
        const unsigned upto = 0xffffffffu >> (31 - (i & 31)), below = upto >> 1;
        *n = rev ? f.n_all - f.n_before[w] - __popc(f.valid[w] & below) : f.n_before[w] + __popc(f.valid[w] & upto);
        *run = rev ? f.run_all - f.run_before[w] - __popc(f.start[w] & below) : f.run_before[w] + __popc(f.start[w] & upto);
    };

    // The part of the warps that hold the state, a thread per row; its sums are in the TMEM columns from `column` on.
    auto state = [&](int row, uint32_t column) {
        const uint32_t kv = tm_lane + column;
        float X[kCols];
        {
            const float* src = nullptr;
            long long step = 1;
            if (!STATES && row < r.da) {
                if (seg > 0) {
                    src = c.seg_state[blockIdx.z] + ((long long)(seg - 1) * c.batch * c.heads + bh) * ((long long)r.da * r.dv) + (long long)row * r.dv + c0;
                } else if (r.x0.p != nullptr) {
                    src = r.x0.p + (long long)b * r.x0.sb + (long long)h * r.x0.sh + (long long)row * r.x0.sr + (long long)c0 * r.x0.sc;
                    step = r.x0.sc;
                }
            }
            const int n = src == nullptr ? 0 : cols;
            if (step == 1 && (reinterpret_cast<uintptr_t>(src) & 15u) == 0) {
#pragma unroll
                for (int j = 0; j < kCols; j += 4) {
                    const float4 x = j < n ? *reinterpret_cast<const float4*>(src + j) : make_float4(0.f, 0.f, 0.f, 0.f);
                    X[j] = x.x, X[j + 1] = x.y, X[j + 2] = x.z, X[j + 3] = x.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < kCols; ++j) {
                    X[j] = j < n ? *src : 0.f;
                    src += step;
                }
            }
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
#pragma unroll 1
        for (int ch = 0; ch < chunks; ++ch) {
            if (!wait_warp(kKvDone, ch)) {
                fine = false;
                break;
            }
            fence_after();
            const Info& f = infos[ch & 3];
            const float2 fac = make_float2(pw_hi[f.n_all], pw_lo[f.n_all]);
            const bool keep = f.run_all == 0;
            if (STATES) seg_factor = keep ? seg_factor * ((double)fac.x + (double)fac.y) : 0.0;
#pragma unroll
            for (int j0 = 0; j0 < kCols; j0 += 16) {
                float x[16];
                tm_ld16(x, kv + j0);
                tm_wait_ld(x);
                if (j0 + 16 == kCols) {
                    fence_before();
                    mbar_arrive(bar(kKvFree, ch));
                }
#pragma unroll
                for (int j = 0; j < 16; j += 2) {
                    float* s = X + j0 + j;
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
            dst += c0 * sc;
            if (sc == 1 && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
#pragma unroll
                for (int j = 0; j < kCols; j += 4)
                    if (j < cols) *reinterpret_cast<float4*>(dst + j) = make_float4(X[j], X[j + 1], X[j + 2], X[j + 3]);
            } else {
#pragma unroll
                for (int j = 0; j < kCols; ++j) {
                    if (j < cols) *dst = X[j];
                    dst += sc;
                }
            }
            if (STATES && slab == 0 && row == 0) {
                const float hi = (float)seg_factor;
                c.seg_factor[blockIdx.z][(long long)seg * c.batch * c.heads + bh] = make_float2(hi, (float)(seg_factor - (double)hi));
            }
        }
    };

    if (warp < 4 || (warp >= 16 && warp < 20)) {
        // ------------------------------------------------------------------------------ decays of P, outputs
        few_registers();
        const int half = warp >> 4, place = warp & 3, row = 32 * place + lane;
        const long long obase = (long long)b * r.o.sb + (long long)h * r.o.sh;
#pragma unroll 1
        for (int ch = 0; !STATES && ch < chunks; ++ch) {
            if (!wait_warp(kPRaw, ch)) break;
            fence_after();
            const uint32_t tm_p = tm_lane + kTmP + (ch & 1) * 128;
            const Info& f = infos[ch & 3];
            int n_i, run_i;
            count(f, row, &n_i, &run_i);
            const bool plain = f.n_all == kC && f.run_all == 0;  // every token valid, one sequence
#pragma unroll 1
            for (int blk = 2 * half; blk < 2 * half + 2; ++blk) {  // 32 keys
                uint32_t p[16];
                if (rev ? blk < place : blk > place) {  // later than all queries of this warp
#pragma unroll
                    for (int j = 0; j < 16; ++j) p[j] = 0;
                } else {
                    float x[32];
                    tm_ld32(x, tm_p + 32 * blk);
                    tm_wait_ld(x);
                    if (plain && blk != place) {
                        // a^|row - key| as the product of a power per row and one per key, neither above 1 for a decay
                        const float own = pw_hi[rev ? 32 * blk - row : row - 32 * blk - 31] * r.s_pair;
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const float4 w = *reinterpret_cast<const float4*>(block + j);
                            const float2 y = mul2(make_float2(x[j], x[j + 1]), mul2(make_float2(own, own), make_float2(w.x, w.y)));
                            const float2 z = mul2(make_float2(x[j + 2], x[j + 3]), mul2(make_float2(own, own), make_float2(w.z, w.w)));
                            p[j / 2] = pack(y.x, y.y);
                            p[j / 2 + 1] = pack(z.x, z.y);
                        }
                    } else if (plain) {
                        const float* pz = pw_hi + (rev ? -lane : lane);  // 32 zeros lie before the powers, for later tokens
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            const float y = x[j] * (pz[rev ? j : -j] * r.s_pair);
                            x[j] = (rev ? j >= lane : j <= lane) ? y : 0.f;  // whatever they hold
                        }
#pragma unroll
                        for (int j = 0; j < 16; ++j) p[j] = pack(x[2 * j], x[2 * j + 1]);
                    } else {
                        const int code = n_i + (run_i << 8);
                        const unsigned vb = f.valid[blk], sb = f.start[blk];
                        int n = f.n_before[blk], run = f.run_before[blk];
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            const int n0 = n, run0 = run;
                            n += vb >> j & 1u;
                            run += sb >> j & 1u;
                            const unsigned lag = (unsigned)(code - (rev ? f.n_all - n0 + ((f.run_all - run0) << 8) : n + (run << 8)));
                            x[j] = lag <= (unsigned)kC ? x[j] * (pw_hi[lag] * r.s_pair) : 0.f;
                        }
#pragma unroll
                        for (int j = 0; j < 16; ++j) p[j] = pack(x[2 * j], x[2 * j + 1]);
                    }
                }
                tm_st16(tm_p + operand_column(blk), p);
            }
            tm_wait_st();
            fence_before();
            mbar_arrive(bar(kPRdy, ch));
            if (!wait_warp(kPvDone, ch)) break;
            fence_after();
            const bool ok = f.valid[place] >> lane & 1u, from_x = run_i == 0;
            const float carry = pw_hi[max(n_i - r.shift, 0)] * r.s_carry;
            const int t = first_token(ch) + row;
            T* po = const_cast<T*>(static_cast<const T*>(r.o.p)) + obase + (long long)t * r.o.st + c0;
#pragma unroll 1
            for (int j0 = 32 * half; j0 < 32 * half + 32; j0 += 16) {
                float x[16], y[16];
                tm_ld16(x, tm_lane + kTmOi + j0);
                tm_ld16(y, tm_lane + kTmOa + j0);
                tm_wait_ld(x);
                tm_wait_ld(y);
                if (j0 & 16) {
                    fence_before();
                    mbar_arrive(bar(kOFree, ch));
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    // a later sequence takes nothing of X, infinities neither
                    const float o = from_x ? fmaf(x[j], carry, y[j]) : y[j];
                    x[j] = ok ? o : 0.f;
                }
                if (t >= 0 && t < c.seqlen) {
                    if (r.out_vec && r.out_f32) {
                        float* q = reinterpret_cast<float*>(const_cast<void*>(r.o.p)) + obase + (long long)t * r.o.st + c0 + j0;
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            if (j0 + 4 * u < cols) *reinterpret_cast<float4*>(q + 4 * u) = make_float4(x[4 * u], x[4 * u + 1], x[4 * u + 2], x[4 * u + 3]);
                    } else if (r.out_vec) {
#pragma unroll
                        for (int u = 0; u < 2; ++u)
                            if (j0 + 8 * u < cols)
                                st_vec(po + j0 + 8 * u, make_uint4(pack(x[8 * u], x[8 * u + 1]), pack(x[8 * u + 2], x[8 * u + 3]),
                                                                   pack(x[8 * u + 4], x[8 * u + 5]), pack(x[8 * u + 6], x[8 * u + 7])));
                    } else {
                        const int eb = r.out_f32 ? 4 : 2;
                        char* q = const_cast<char*>(static_cast<const char*>(r.o.p)) + (obase + (long long)t * r.o.st + (c0 + j0) * r.o.sd) * eb;
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            if (j0 + j < cols) {
                                if (r.out_f32)
                                    *reinterpret_cast<float*>(q) = x[j];
                                else
                                    *reinterpret_cast<T*>(q) = __float2bfloat16_rn(x[j]);
                            }
                            q += r.o.sd * eb;
                        }
                    }
                }
            }
        }
    } else if (warp < 8) {
        many_registers();
        state(32 * (warp - 4) + lane, kTmKV);
    } else if (warp < 16) {
        // ------------------------------------------------------------------------------ weighted values
        few_registers();
        const int me = tid - 256;
#pragma unroll 1
        for (int ch = 0; ch < chunks; ++ch) {
            constexpr int kBack = STATES ? 2 : 1;  // buffers
            const bool ok = wait(kVFull, ch) && (ch < kBack || wait(kKvDone, ch - kBack));
            if (!all_of(1, kWeighers, ok)) break;  // the weights of the chunk before are no longer read
            const Info& f = infos[ch & 3];
            if (me < kC) {
                int n, run;
                count(f, me, &n, &run);
                add[me] = run == f.run_all ? pw_hi[f.n_all - n + r.shift] * r.s_add : 0.f;
            }
            asm volatile("bar.sync 1, %0;" ::"n"(kWeighers) : "memory");
            const unsigned char* v = sm + L::kV + (ch & 1) * kPanel;
            unsigned char* w = sm + weighted(ch);
            const int at = ((me & 7) ^ (me >> 3 & 7)) << 4;  // rows 32 apart have the same swizzle
#pragma unroll 2
            for (int i = 0; i < kC * 8 / kWeighers; ++i) {
                const int tok = (me >> 3) + kWeighers / 8 * i;
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
    } else {
        many_registers();  // the same instruction for the four warps of the group
        // ------------------------------------------------------------------------------ products
        if (warp == 20) {
            const bool leader = elect_lane();
            const int steps = (r.da + 15) / 16;
            const uint32_t q0 = base + L::kQ, k0 = base + L::kK, v0 = base + L::kV, x0 = base + L::kX;
            auto products_of_keys = [&](int ch) {  // P of a chunk
                if (!wait_warp(kKFull, ch) || !wait_warp(kQFull, ch)) return false;
                fence_after();
                const uint64_t dq = desc_k(q0 + (ch % NS) * L::kPanels * kPanel), dk = desc_k(k0 + (ch % NS) * L::kPanels * kPanel);
                const uint32_t d = tm + kTmP + (ch & 1) * 128;
#pragma unroll
                for (int s = 0; s < ROWS / 16; ++s)
                    if (s < steps) mma_ss(leader, d, at(dq, (s >> 2) * kPanel + (s & 3) * 32), at(dk, (s >> 2) * kPanel + (s & 3) * 32), idesc(128, false, false), s > 0);
                commit(leader, bar(kPRaw, ch));
                return true;
            };
            bool going = STATES || NS == 1 || chunks == 0 || products_of_keys(0);
#pragma unroll 1
            for (int ch = 0; going && ch < chunks; ++ch) {
                const uint32_t q = q0 + (ch % NS) * L::kPanels * kPanel, k = k0 + (ch % NS) * L::kPanels * kPanel, v = v0 + (ch & 1) * kPanel;
                if (!wait_warp(kKFull, ch) || !wait_warp(kVwRdy, ch) || (ch > 0 && !wait_warp(kKvFree, ch - 1))) break;
                fence_after();
#pragma unroll 1
                for (int tile = 0; tile < (kSecond ? 2 : 1); ++tile) {  // rows 0-127; 64-191, of which 128-159 are used
                    const uint64_t dk = desc_mn(k + tile * kPanel);
                    uint64_t dw = desc_mn(base + weighted(ch) + 2 * kPanel);
#pragma unroll 1
                    for (int p = 2; p >= 0; --p) {
#pragma unroll
                        for (int s = 0; s < kC / 16; ++s) mma_ss(leader, tm + (tile ? kTmKV2 : kTmKV), at(dk, s * 2048), at(dw, s * 2048), idesc(kCols, true, true), p < 2 || s > 0);
                        dw -= kPanel >> 4;
                    }
                }
                commit(leader, bar(kKvDone, ch));
                if (!STATES) {
                    // with one buffer of keys the state's products go first: theirs is the longer way to the next chunk
                    if (NS == 1 && !products_of_keys(ch)) break;
                    if (!wait_warp(kXRdy, ch) || (ch > 0 && !wait_warp(kOFree, ch - 1))) break;
                    fence_after();
                    const uint64_t dq = desc_k(q), dx = desc_mn(x0), dv = desc_mn(v);
#pragma unroll
                    for (int s = 0; s < ROWS / 16; ++s)
                        if (s < steps) mma_ss(leader, tm + kTmOi, at(dq, (s >> 2) * kPanel + (s & 3) * 32), at(dx, s * 2048), idesc(kCols, false, true), s > 0);
                    commit(leader, bar(kQxDone, ch));
                    // the next chunk's products fill the time that this one's decays take
                    if (NS == 2 && ch + 1 < chunks && !products_of_keys(ch + 1)) break;
                    if (!wait_warp(kPRdy, ch)) break;
                    fence_after();
#pragma unroll
                    for (int s = 0; s < kC / 16; ++s)
                        mma_ts(leader, tm + kTmOa, tm + kTmP + (ch & 1) * 128 + operand_column(s >> 1) + 8 * (s & 1), at(dv, s * 2048), idesc(kCols, false, true), s > 0);
                    commit(leader, bar(kPvDone, ch));
                }
            }
        }
        if (kSecond && warp == 22) state(128 + lane, kTmKV2);
        // ------------------------------------------------------------------------------ tokens
        const Maps& m = maps.run[blockIdx.z];
        const int panels = (r.da + 63) / 64;
        const bool leader = elect_lane();
        if (warp == 21 && leader) {
            tma::prefetch_tensormap(&m.k);
            tma::prefetch_tensormap(&m.v);
            if (!STATES) tma::prefetch_tensormap(&m.a);
        }
        const int head_a = h / r.a.group, head_k = h / r.k.group, head_v = h / r.v.group;
#pragma unroll 1
        for (int ch = 0; warp == 21 && ch < chunks; ++ch) {
            const int t0 = first_token(ch);
            const int hand_over = to_clear(ch) ? kTmaQ : kQFull;
            auto ask = [&](const CUtensorMap* map, int what, int n_panels, int c_first, int head, uint32_t to) {
                const uint32_t done = bar(hand_over + what, ch);
                if (leader) {
                    tma::mbar_arrive_expect_tx(done, n_panels * kPanel);
                    tma_load_4d(to, map, c_first, t0, head, b, done);
                }
#pragma unroll
                for (int p = 1; p < L::kPanels; ++p)
                    if (leader && p < n_panels) tma_load_4d(to + p * kPanel, map, c_first + p * 64, t0, head, b, done);
                if (leader) {
                    // the other barrier goes through its phase of this chunk too: phases are counted in chunks
                    if (hand_over == kQFull && c.mask != nullptr) mbar_arrive(bar(kTmaQ + what, ch));
                    misc[4 + what] = ch + 1;
                }
            };
            auto all = [&](bool ok) { return (bool)__all_sync(0xffffffffu, ok); };
            auto ask_values = [&]() {
                if (!all(ch < 2 || STATES || wait(kPvDone, ch - 2))) return false;
                ask(&m.v, 2, 1, c0, head_v, base + L::kV + (ch & 1) * kPanel);
                return true;
            };
            // Values have two buffers, keys and queries as many as fit.  Each is asked for when its own is free: with two of
            // each, keys first; with one, values, because the next chunk's wait for nothing else.
            if (!all(ch < 2 || (wait(kKvDone, ch - 2) && wait(kKvFree, ch - 2) && (STATES || wait(kPRaw, ch - 2))))) break;
            if (NS == 1) {
                if (!ask_values()) break;
                if (!all(ch < 1 || (wait(kKvDone, ch - 1) && (STATES || wait(kPRaw, ch - 1))))) break;
            }
            ask(&m.k, 1, panels, 0, head_k, base + L::kK + (ch % NS) * L::kPanels * kPanel);
            if (!STATES) {
                if (!all(ch < NS || wait(kQxDone, ch - NS))) break;
                ask(&m.a, 0, panels, 0, head_a, base + L::kQ + (ch % NS) * L::kPanels * kPanel);
            }
            if (NS == 2 && !ask_values()) break;
            __syncwarp();
        }
#pragma unroll 1
        for (int ch = 0; warp == 23 && ch < chunks; ++ch) {
            if (ch + 1 == c.test_expire) break;  // the self-test's missing chunk
            // nobody looks at the chunk before the last but one any more
            if (ch >= 2 && !(wait_warp(kKvFree, ch - 2) && (STATES || wait_warp(kPvDone, ch - 2)))) break;
            const int t0 = first_token(ch);
            // the tokens of the chunk that count, and the sequence starts in the run's order
            Info* f = infos + (ch & 3);
            int n = 0, run = 0;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int t = t0 + 32 * w + lane;
                bool v = t >= 0 && t < c.seqlen, s = false;
                if (v && c.seq_idx != nullptr && (rev ? t + 1 < c.seqlen : t > 0)) {
                    const int32_t* p = c.seq_idx + (long long)b * c.seq_sb + (long long)t * c.seq_st;
                    s = p[0] != (rev ? p[c.seq_st] : p[-c.seq_st]);
                }
                if (v && c.mask != nullptr) v = mask_valid(c.mask, c.mask_dtype, (long long)b * c.mask_sb + (long long)t * c.mask_st);
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
            __syncwarp();
            if (leader) {  // for those who wait for the products or the values
                if (!STATES) mbar_arrive(bar(kPRaw, ch));
                mbar_arrive(bar(kKvDone, ch));
                mbar_arrive(bar(kVFull, ch));
                misc[7] = ch + 1;
            }
            if (!to_clear(ch)) continue;
            bool ok = true;
#pragma unroll 1
            for (int turn = 0; turn < (STATES ? 2 : 3); ++turn) {  // in the order they are asked for
                const int what = NS == 1 ? 2 - turn : (STATES ? 1 + turn : (turn + 1) % 3);  // 2: values, 1: keys, 0: queries
                ok = wait_warp(kTmaQ + what, ch);
                if (!ok) break;
                {
                    unsigned char* to = sm + (what == 2 ? L::kV + (ch & 1) * kPanel : (what == 1 ? L::kK : L::kQ) + (ch % NS) * L::kPanels * kPanel);
                    for (int row = lane >> 3; row < kC; row += 4) {  // eight lanes to a row
                        if (f->valid[row >> 5] >> (row & 31) & 1u) continue;
                        for (int p = 0; p < (what == 2 ? 1 : panels); ++p)
                            *reinterpret_cast<uint4*>(to + p * kPanel + row * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fence_async_smem();
                }
                __syncwarp();
                if (leader) mbar_arrive(bar(kQFull + what, ch));
            }
            if (!ok) break;
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == 20) {
        fence_after();
        const bool issuer = elect_lane();  // a commit speaks for the products of its own thread only
        if (*dead && issuer) {
            // products and copies may still be under way: they end by themselves, and TMEM and shared memory have to
            // outlive them.  A barrier of its own for the products; the copies' barriers for the copies.  That of the values
            // also wants the chunk's announcement, which may never have come.
            const uint32_t last = base + L::kMisc + 8;
            mbar_init(last, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            commit(true, last);
            for (unsigned i = 0; i < kMaxPolls && !mbar_test(last, 0); ++i) __nanosleep(64);
            for (int what = 0; what < 3; ++what) {
                const int asked = misc[4 + what];
                for (int ch = max(0, asked - 2); ch < asked; ++ch) {
                    if (what == 2 && ch >= (int)misc[7] && !to_clear(ch)) mbar_arrive(bar(kVFull, ch));
                    for (unsigned i = 0; i < kMaxPolls && !mbar_test(bar((to_clear(ch) ? kTmaQ : kQFull) + what, ch), (uint32_t)(ch >> 1) & 1u); ++i) __nanosleep(64);
                }
            }
        }
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "n"(kTmCols));
    }
}

// The tensor map of rows as [batch, head, token, channel] with boxes of 64 channels x 128 tokens.
inline bool encode(CUtensorMap* map, const Rows& r, int batch, int heads, int seqlen, int dim) {
    tma::EncodeFn enc = tma::encode_fn();
    if (enc == nullptr) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)dim, (cuuint64_t)seqlen, (cuuint64_t)(heads / r.group), (cuuint64_t)batch};
    cuuint64_t st[3] = {2 * (cuuint64_t)r.st, 2 * (cuuint64_t)r.sh, 2 * (cuuint64_t)r.sb};
    for (int i = 0; i < 3; ++i)
        if (dims[i + 1] == 1) st[i] = 1024;  // an extent of 1 makes its stride irrelevant, but the encoder wants a legal one
    const cuuint32_t box[4] = {64, kC, 1, 1}, step[4] = {1, 1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(r.p), dims, st, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// rows whose tokens run backwards, in natural order again
inline Rows natural(Rows r, int seqlen, int eb) {
    r.p = static_cast<const char*>(r.p) + (long long)(seqlen - 1) * r.st * eb;
    r.st = -r.st;
    return r;
}

template <int ROWS, bool STATES, bool REV>
cudaError_t launch(const Launch& given, unsigned int* timeouts, cudaStream_t s) {
    constexpr int smem = Layout<ROWS>::kBytes;
    static_assert(smem <= 232448, "shared memory of an SM");
    Launch l = given;
    AllMaps maps;
    int slabs = 0;
    for (int i = 0; i < l.runs; ++i) {
        Run& r = l.run[i];
        if (r.reverse) {
            r.a = natural(r.a, l.c.seqlen, 2);
            r.k = natural(r.k, l.c.seqlen, 2);
            r.v = natural(r.v, l.c.seqlen, 2);
            r.o = natural(r.o, l.c.seqlen, r.out_f32 ? 4 : 2);
        }
        slabs = max(slabs, (r.dv + kCols - 1) / kCols);
        Maps& m = maps.run[i];
        if (!(encode(&m.a, r.a, l.c.batch, l.c.heads, l.c.seqlen, r.da) && encode(&m.k, r.k, l.c.batch, l.c.heads, l.c.seqlen, r.da) &&
              encode(&m.v, r.v, l.c.batch, l.c.heads, l.c.seqlen, r.dv)))
            return cudaErrorNotSupported;
    }
    auto kernel = k_linear_tc<ROWS, STATES, REV>;
    static std::atomic<bool> fits{false};
    cudaError_t e = check_registers(kernel, kThreads, kRegisterShare, fits);
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned)(l.c.batch * l.c.heads * slabs), STATES ? l.c.segments - 1 : l.c.segments, l.runs);
    note_launch(STATES ? "linear_tc_states" : "linear_tc");
    kernel<<<grid, kThreads, smem, s>>>(l, maps, timeouts);
    return cudaGetLastError();
}

}  // namespace tc
}  // namespace lin
}  // namespace vc1d
