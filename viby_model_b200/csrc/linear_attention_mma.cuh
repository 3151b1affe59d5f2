// Linear attention on the tensor cores (16-bit types, channel stride 1, 16-byte aligned rows, head dims a multiple of 8).
//
// One CTA of eight warps owns one (row, head), a slab of BV state columns and a part of the time axis, and walks its
// chunks of 64 tokens with one barrier each.  Four warps compute outputs, four roll the state on; the fp32 state stays in
// the latter's registers for the whole walk (warp w holds the 16-row blocks w, w + 4, ... of the slab).  Per chunk:
//     output warp, 16 queries:  P = q k^T and O = q X in one pass over q's fragments (keys later than the warp's
//                               queries are skipped);  O = decay O + (decay P) v, P going from accumulators to operands
//     state warp:               X = a^n X + (w k)^T v, k^T straight from shared memory, weighted and split in registers;
//                               the rounded X that the next chunk's queries read goes to the other of two buffers
// k and v of the next chunk are in flight meanwhile (two buffers); an output warp refills its own rows of q as soon as it
// has read them, and its part of the output passes through these rows.  Two CTAs share an SM: sixteen warps, four chains of
// dependent work per scheduler (eight warps that did both in turn, four per CTA, took twice as long).  The warps' shares
// of the registers are unequal: setmaxnreg.
//
// Roundings.  The state that the queries read and the products inside a chunk are rounded to the I/O type, as operands
// of the second product: each term of an output meets one such rounding, of the size of the output's own.  The state
// itself is fp32 in every respect: the weighted keys are split into three bf16 parts (24 bits), fp16 ones into two tf32
// parts (22 bits, and no trouble with fp16's range), and a chunk's sum is formed from zero and then added to the state,
// because the tensor cores truncate where an fp32 add rounds: thousands of accumulations onto one long-lived state would
// all err towards zero.  fp16's range: the rounded state and the products are scaled by powers of two (per CTA, per query)
// around their maximum.
//
// What bounds it: mma.sync itself, and the parts of the state's products.  8 x 1024 tokens of 16 heads of 128: 123 us in bf16,
// 143 us in fp16 (tcgen05, bf16: 64).  Spills, all of them small (bytes stored, bf16 / fp16): 160 x 80 rows 360 / 236, 256
// rows 96 / 108, 128 rows 20 / 132; those of 256 rows come from the test for chunks without a token: 1 to 2 % for dense
// prompts, while padded ones are 2 to 5 % faster by it.
#pragma once

#include "linear_attention.cuh"

namespace vc1d {
namespace lin {
namespace mma {

constexpr int kWarps = 4;             // of each kind
constexpr int kThreads = 2 * 32 * kWarps;
constexpr int kPad = 8;               // zeros before the table of decays of pairs
constexpr int kSms = 148;             // of a B200; with another count the schedulers' loads are less even, no more

struct Info {  // of a chunk's tokens, by one warp two chunks ahead
    float carry[kChunk];   // a^{n_i} for tokens of the sequence that the chunk starts in, else 0
    float add[kChunk];     // weight of the token's key in the state after the chunk
    uint16_t code[kChunk]; // n_i + (run_i << 8): as ChunkInfo::code, 16 bits wide
    unsigned valid[2];
    int n_all, run_all;
};

template <int DAP, int BV>
struct Layout {
    // rows padded by 16 bytes: 8 consecutive rows start in 8 different 16-byte bank groups, as ldmatrix wants them
    static constexpr int kStrideA = DAP + 8, kStrideV = BV + 8;
    // the 160 x 80 variant has its state rows unpadded (two-way conflicts) and once only (a barrier more): two CTAs just
    // fit an SM
    static constexpr bool kOneX = BV == 80;
    static constexpr int kStrideX = kOneX ? BV : BV + 8;
    static constexpr int kQ = 0;
    static constexpr int kK = kQ + kChunk * kStrideA;
    static constexpr int kV = kK + 2 * kChunk * kStrideA;
    static constexpr int kX = kV + 2 * kChunk * kStrideV;
    static constexpr int kEnd = kX + (kOneX ? 1 : 2) * DAP * kStrideX;  // 16-bit elements
    static constexpr int kBytes = 2 * kEnd + 3 * (int)sizeof(Info) + 4 * (3 * kPowers + kPad) + 4 * 2 * kWarps;
};
// Registers per thread of output and state warps, out of the 65536 / (2 * 256) that two CTAs leave for each: the sum of
// both shares is that of the launch.  256 rows have a CTA per SM and need no shares.
template <int DAP>
struct Registers {
    static constexpr bool kShares = DAP <= 160 && DAP > 64;
    static constexpr int kOut = DAP == 160 ? 88 : 104, kState = 256 - kOut;
    static constexpr int kShare = kThreads / 2 * (kOut + kState);
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void stsm4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ void mma_tf32(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int DT>
struct Half;
template <>
struct Half<VC1D_BF16> {
    __device__ __forceinline__ static void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    __device__ __forceinline__ static uint32_t pack(float lo, float hi) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    __device__ __forceinline__ static float lo(uint32_t v) { return __uint_as_float(v << 16); }
    __device__ __forceinline__ static float hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
};
template <>
struct Half<VC1D_F16> {
    __device__ __forceinline__ static void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    __device__ __forceinline__ static uint32_t pack(float lo, float hi) {
        const __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    __device__ __forceinline__ static float lo(uint32_t v) { return __half2float(__ushort_as_half((unsigned short)(v & 0xffffu))); }
    __device__ __forceinline__ static float hi(uint32_t v) { return __half2float(__ushort_as_half((unsigned short)(v >> 16))); }
};

__device__ __forceinline__ uint32_t to_tf32(float x) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
    return r & 0xffffe000u;
}

// 2^k that brings x (>= 0) to [2^13, 2^14), and its inverse; 1 for 0, infinities and NaN.  x below 2^least counts as 2^least.
__device__ __forceinline__ void scale_around(float x, int least, float* up, float* down) {
    int e = (int)(__float_as_uint(x) >> 23) - 127;
    if (x == 0.f || e == 128) e = 13;
    e = max(least, min(113, e));
    *up = __uint_as_float((unsigned)(127 + 13 - e) << 23);
    *down = __uint_as_float((unsigned)(127 - 13 + e) << 23);
}

// DAP: rows of the state, padded; BV: columns of a slab.
template <int DT, int DAP, int BV, bool STATES>
__global__ void __launch_bounds__(kThreads, DAP == 256 ? 1 : 2) k_linear_mma(const __grid_constant__ Launch l) {
    using E = Elem<DT>;
    using T = typename E::type;
    using Hf = Half<DT>;
    using L = Layout<DAP, BV>;
    constexpr int kBlocks = DAP / 16;                       // 16-row blocks of the state
    constexpr int kMine = (kBlocks + kWarps - 1) / kWarps;  // at most so many of them per state warp
    constexpr int kN = BV / 8;                              // 8-column tiles of a slab
    constexpr int kUnitsA = DAP / 8, kUnitsV = BV / 8;      // 16-byte units of a row
    constexpr bool kF16 = DT == VC1D_F16;

    extern __shared__ __align__(16) unsigned char raw[];
    T* sm = reinterpret_cast<T*>(raw);
    Info* infos = reinterpret_cast<Info*>(raw + 2 * L::kEnd);
    float* pw_hi = reinterpret_cast<float*>(raw + 2 * L::kEnd + 3 * sizeof(Info));
    float* pw_lo = pw_hi + kPowers;
    float* pairs = pw_lo + kPowers + kPad;  // [-kPad .. kPowers): s_pair a^lag, 0 for negative lags
    float* warp_max = pairs + kPowers;      // [2][kWarps], by chunk (fp16)

    const Run& r = l.run[blockIdx.z];
    const Common& c = l.c;
    const int slabs = (r.dv + BV - 1) / BV;
    const int slab = blockIdx.x % slabs, bh = blockIdx.x / slabs, seg = blockIdx.y;
    if (bh >= c.batch * c.heads) return;  // a run with fewer slabs than the launch's widest
    const int b = bh / c.heads, h = bh % c.heads;
    const int tid = threadIdx.x, lane = tid & 31, warp = (tid >> 5) & 3;
    const bool state_warp = tid >= kThreads / 2;
    const int g = lane >> 2, t4 = lane & 3;
    const int c0 = slab * BV, cols = min(BV, r.dv - c0);

    for (int n = tid; n < kPowers; n += kThreads) {
        const float d = c.log_decay[h];
        const double x = n == 0 ? 1.0 : exp((double)d * (double)n);
        const float hi = (float)x;
        const double lo = x - (double)hi;
        pw_hi[n] = hi;
        pw_lo[n] = (isfinite(hi) && lo == lo) ? (float)lo : 0.f;
        pairs[n] = hi * r.s_pair;
    }
    if (tid < kPad) pairs[tid - kPad] = 0.f;
    for (int i = tid; i < L::kEnd / 8; i += kThreads) reinterpret_cast<uint4*>(sm)[i] = make_uint4(0, 0, 0, 0);

    const int t_begin = seg * c.seg_chunks * kChunk;
    const int t_end = min(c.seqlen, t_begin + c.seg_chunks * kChunk);
    const int chunks = (t_end - t_begin + kChunk - 1) / kChunk;
    const T* pa = static_cast<const T*>(r.a.p) + (long long)b * r.a.sb + (long long)(h / r.a.group) * r.a.sh;
    const T* pk = static_cast<const T*>(r.k.p) + (long long)b * r.k.sb + (long long)(h / r.k.group) * r.k.sh;
    const T* pv = static_cast<const T*>(r.v.p) + (long long)b * r.v.sb + (long long)(h / r.v.group) * r.v.sh + c0;
    const int ua = r.da / 8, uv = cols / 8;  // units that hold data
    __syncthreads();  // shared memory is zero, the powers are there

    auto fill_info = [&](int chunk) {  // by one warp
        Info* f = infos + chunk % 3;
        const int t0 = t_begin + chunk * kChunk;
        unsigned ok[2], start[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int t = t0 + 32 * half + lane;
            const long long at = r.reverse ? c.seqlen - 1 - t : t;
            bool v = t < t_end, s = false;
            if (v && c.mask != nullptr) v = mask_valid(c.mask, c.mask_dtype, (long long)b * c.mask_sb + at * c.mask_st);
            if (t < t_end && c.seq_idx != nullptr && t > 0) {
                const int32_t* p = c.seq_idx + (long long)b * c.seq_sb + at * c.seq_st;
                s = p[0] != (r.reverse ? p[c.seq_st] : p[-c.seq_st]);
            }
            ok[half] = __ballot_sync(0xffffffffu, v);
            start[half] = __ballot_sync(0xffffffffu, s);
        }
        const unsigned upto = 0xffffffffu >> (31 - lane);
        const int n0 = __popc(ok[0]), r0 = __popc(start[0]);
        const int n_all = n0 + __popc(ok[1]), run_all = r0 + __popc(start[1]);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int n = (half ? n0 : 0) + __popc(ok[half] & upto), run = (half ? r0 : 0) + __popc(start[half] & upto);
            f->code[32 * half + lane] = (uint16_t)(n + (run << 8));
            f->carry[32 * half + lane] = run == 0 ? pw_hi[max(n - r.shift, 0)] * r.s_carry : 0.f;
            f->add[32 * half + lane] = run == run_all ? pw_hi[n_all - n + r.shift] * r.s_add : 0.f;
        }
        if (lane == 0) {
            f->valid[0] = ok[0];
            f->valid[1] = ok[1];
            f->n_all = n_all;
            f->run_all = run_all;
        }
    };
    // 16-byte pieces of 64 rows, dealt out to the CTA; rows of masked tokens arrive as zeros without being read
    auto load_rows = [&](const Info* f, const T* src, long long st, int units, int used, uint32_t dst, int stride, int lanes, int at0, int first) {
        int row = first / units, u = first % units;
        const int row_step = lanes / units, u_step = lanes % units;
        for (int n = at0; row < n;) {
            if (u < used) {
                const bool ok = f->valid[row >> 5] >> (row & 31) & 1u;
                cp16(dst + 2 * (row * stride + u * 8), ok ? src + row * st + u * 8 : src, ok);
            }
            row += row_step;
            u += u_step;
            if (u >= units) u -= units, ++row;
        }
    };
    auto load_kv = [&](int chunk) {
        const Info* f = infos + chunk % 3;
        const long long t0 = t_begin + chunk * kChunk;
        const int buf = chunk & 1;
        load_rows(f, pk + t0 * r.k.st, r.k.st, kUnitsA, ua, smem_u32(sm + L::kK + buf * kChunk * L::kStrideA), L::kStrideA, kThreads, kChunk, tid);
        load_rows(f, pv + t0 * r.v.st, r.v.st, kUnitsV, uv, smem_u32(sm + L::kV + buf * kChunk * L::kStrideV), L::kStrideV, kThreads, kChunk, tid);
    };

    if (chunks > 0) {
        if (tid < 32) fill_info(0);
        if (tid >= 32 && tid < 64 && chunks > 1) fill_info(1);
        __syncthreads();
        load_kv(0);
    }

    if (!state_warp) {
        // ------------------------------------------------------------------------------------------- outputs
        if constexpr (Registers<DAP>::kShares) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Registers<DAP>::kOut));
        // The later a warp's queries are, the more keys they see.  Every other wave of CTAs deals the 16-row groups out in
        // reverse, so that the two CTAs of an SM load its four schedulers alike.
        const int grp = ((blockIdx.x / kSms) & 1) ? kWarps - 1 - warp : warp;
        T* sq = sm + L::kQ + grp * 16 * L::kStrideA;  // this warp's rows of q
        auto load_q = [&](int chunk) {
            const Info* f = infos + chunk % 3;
            const long long t0 = t_begin + chunk * kChunk;
            // units past the head's end are cleared too: the output passes through these rows
            const uint32_t d = smem_u32(sm + L::kQ);
            int row = grp * 16 + lane / kUnitsA, u = lane % kUnitsA;
            for (; row < grp * 16 + 16;) {
                const bool ok = u < ua && (f->valid[row >> 5] >> (row & 31) & 1u);
                cp16(d + 2 * (row * L::kStrideA + u * 8), ok ? pa + (t0 + row) * r.a.st + u * 8 : pa, ok);
                row += 32 / kUnitsA;
                u += 32 % kUnitsA;
                if (u >= kUnitsA) u -= kUnitsA, ++row;
            }
        };
        // The output of this warp's 16 queries of a chunk.  Loops stay rolled where registers allow it: the code of both
        // kinds of warps has to stay in the instruction caches (a copy per group of queries, all unrolled, ran at the same
        // speed as eight warps less: two thirds of the warps' time went into waiting for instructions).
        auto outputs = [&](int chunk) {
            // key tiles of one pass: with 80 columns the products of 32 keys at a time, for want of registers
            constexpr int kPass = BV == 80 ? 2 : 4;
            const Info& f = infos[chunk % 3];
            const T* sk = sm + L::kK + (chunk & 1) * kChunk * L::kStrideA;
            const T* sv = sm + L::kV + (chunk & 1) * kChunk * L::kStrideV;
            const T* sx = sm + L::kX + (L::kOneX ? 0 : (chunk & 1) * DAP * L::kStrideX);
            const uint32_t aq = smem_u32(sq + (lane & 15) * L::kStrideA + (lane >> 4) * 8);
            const uint32_t bk = smem_u32(sk + ((lane & 7) + (lane >> 4) * 8) * L::kStrideA + (lane >> 3 & 1) * 8);
            const uint32_t bx = smem_u32(sx + ((lane & 7) + (lane >> 3 & 1) * 8) * L::kStrideX + (lane >> 4) * 8);
            const uint32_t bv = smem_u32(sv + ((lane & 7) + (lane >> 3 & 1) * 8) * L::kStrideV + (lane >> 4) * 8);
            const int i0 = grp * 16 + g;
            const bool plain = f.n_all == kChunk && f.run_all == 0;  // every token valid, one sequence
            float O[kN][4];
#pragma unroll
            for (int n = 0; n < kN; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) O[n][e] = 0.f;
            float down0 = 1.f, down1 = 1.f;  // fp16: what the sums have to be multiplied by
#pragma unroll
            for (int pass = 0; pass < 4 / kPass; ++pass) {
                if (pass * kPass > grp) break;
                // ---- P = q k^T, and O = q X on the first pass ----
                constexpr int kTiles = 2 * kPass;
                float P[kTiles][4];
#pragma unroll
                for (int n = 0; n < kTiles; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) P[n][e] = 0.f;
#pragma unroll 1
                for (int kk = 0; kk < kBlocks; ++kk) {
                    uint32_t a[4];
                    ldsm4(a, aq + 2 * (kk * 16));
#pragma unroll
                    for (int j = 0; j < kPass; ++j) {
                        if (pass * kPass + j <= grp) {
                            uint32_t kb[4];
                            ldsm4(kb, bk + 2 * ((pass * kPass + j) * 16 * L::kStrideA + kk * 16));
                            Hf::mma(P[2 * j], a, kb[0], kb[1]);
                            Hf::mma(P[2 * j + 1], a, kb[2], kb[3]);
                        }
                    }
                    if (pass == 0) {
#pragma unroll
                        for (int n = 0; n < kN; n += 2) {
                            uint32_t xb[4];
                            ldsm4t(xb, bx + 2 * (kk * 16 * L::kStrideX + n * 8));
                            Hf::mma(O[n], a, xb[0], xb[1]);
                            Hf::mma(O[n + 1], a, xb[2], xb[3]);
                        }
                    }
                }
                if (L::kOneX && pass == 0) asm volatile("bar.arrive 1, %0;" ::"n"(kThreads) : "memory");  // X has been read
                // ---- decays ----
                if (plain) {
                    const float* pz = pairs + g - 2 * t4;  // lag of row g and key 2 t4 of a tile at distance 0
#pragma unroll
                    for (int n = 0; n < kTiles; ++n) {
                        const int tile = pass * kTiles + n;
                        const int d = 8 * (2 * grp - tile);  // tiles of later keys hold zeros
                        P[n][0] *= d >= 0 ? pz[d] : 0.f;
                        P[n][1] *= d >= 0 ? pz[d - 1] : 0.f;
                        P[n][2] *= d >= -8 ? pz[d + 8] : 0.f;
                        P[n][3] *= d >= -8 ? pz[d + 7] : 0.f;
                    }
                } else {
                    const int code0 = f.code[i0], code1 = f.code[i0 + 8];
#pragma unroll
                    for (int n = 0; n < kTiles; ++n) {
                        const int tile = pass * kTiles + n;
                        if (tile <= 2 * grp + 1) {
                            const uint32_t cj = *reinterpret_cast<const uint32_t*>(f.code + tile * 8 + 2 * t4);
                            const int ca = (int)(cj & 0xffffu), cb = (int)(cj >> 16);
                            const unsigned l00 = (unsigned)(code0 - ca), l01 = (unsigned)(code0 - cb);
                            const unsigned l10 = (unsigned)(code1 - ca), l11 = (unsigned)(code1 - cb);
                            P[n][0] = l00 <= kChunk ? P[n][0] * pairs[l00] : 0.f;
                            P[n][1] = l01 <= kChunk ? P[n][1] * pairs[l01] : 0.f;
                            P[n][2] = l10 <= kChunk ? P[n][2] * pairs[l10] : 0.f;
                            P[n][3] = l11 <= kChunk ? P[n][3] * pairs[l11] : 0.f;
                        }
                    }
                }
                float f0 = 1.f, f1 = 1.f;
                bool in0 = true, in1 = true;
                if (pass == 0) {
                    f0 = f.carry[i0], f1 = f.carry[i0 + 8];
                    // a later sequence takes nothing of X, infinities neither
                    in0 = (f.code[i0] >> 8) == 0, in1 = (f.code[i0 + 8] >> 8) == 0;
                    if constexpr (kF16) {
                        const float* own = warp_max + (chunk & 1) * kWarps;
                        float m = own[0], up, x_down;
#pragma unroll
                        for (int w = 1; w < kWarps; ++w) m = fmaxf(m, own[w]);
                        scale_around(m, -100, &up, &x_down);
                        f0 *= x_down;
                        f1 *= x_down;
                    }
                }
                if constexpr (kF16) {
                    float m0 = 0.f, m1 = 0.f, up0, up1, old0 = down0, old1 = down1;
#pragma unroll
                    for (int n = 0; n < kTiles; ++n) {
                        m0 = fmaxf(m0, fmaxf(fabsf(P[n][0]), fabsf(P[n][1])));
                        m1 = fmaxf(m1, fmaxf(fabsf(P[n][2]), fabsf(P[n][3])));
                    }
#pragma unroll
                    for (int d = 1; d < 4; d <<= 1) {
                        m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, d));
                        m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, d));
                    }
                    // products below 2^-20 reach fp16 outputs as less than its smallest step, so they need no larger factor,
                    // which what the state adds to this accumulator would have to bear too
                    scale_around(m0, -20, &up0, &down0);
                    scale_around(m1, -20, &up1, &down1);
                    f0 *= old0 * up0;
                    f1 *= old1 * up1;
#pragma unroll
                    for (int n = 0; n < kTiles; ++n) {
                        P[n][0] *= up0, P[n][1] *= up0;
                        P[n][2] *= up1, P[n][3] *= up1;
                    }
                }
                if (pass == 0 || kF16) {
#pragma unroll
                    for (int n = 0; n < kN; ++n) {
                        O[n][0] = in0 ? O[n][0] * f0 : 0.f, O[n][1] = in0 ? O[n][1] * f0 : 0.f;
                        O[n][2] = in1 ? O[n][2] * f1 : 0.f, O[n][3] = in1 ? O[n][3] * f1 : 0.f;
                    }
                }
                // ---- O += P v ----
#pragma unroll
                for (int j = 0; j < kPass; ++j) {
                    const int kk = pass * kPass + j;
                    if (kk <= grp) {
                        const uint32_t a[4] = {Hf::pack(P[2 * j][0], P[2 * j][1]), Hf::pack(P[2 * j][2], P[2 * j][3]),
                                               Hf::pack(P[2 * j + 1][0], P[2 * j + 1][1]), Hf::pack(P[2 * j + 1][2], P[2 * j + 1][3])};
#pragma unroll
                        for (int n = 0; n < kN; n += 2) {
                            uint32_t vb[4];
                            ldsm4t(vb, bv + 2 * (kk * 16 * L::kStrideV + n * 8));
                            Hf::mma(O[n], a, vb[0], vb[1]);
                            Hf::mma(O[n + 1], a, vb[2], vb[3]);
                        }
                    }
                }
            }
            // ---- out ----
            const bool ok0 = f.valid[i0 >> 5] >> (i0 & 31) & 1u, ok1 = f.valid[(i0 + 8) >> 5] >> ((i0 + 8) & 31) & 1u;
#pragma unroll
            for (int n = 0; n < kN; ++n) {
                O[n][0] = ok0 ? O[n][0] * down0 : 0.f, O[n][1] = ok0 ? O[n][1] * down0 : 0.f;
                O[n][2] = ok1 ? O[n][2] * down1 : 0.f, O[n][3] = ok1 ? O[n][3] * down1 : 0.f;
            }
            const int t0 = t_begin + chunk * kChunk + grp * 16;
            const long long obase = (long long)b * r.o.sb + (long long)h * r.o.sh;
            __syncwarp();  // every lane has read its fragments of q
            if (r.out_vec && !r.out_f32) {
#pragma unroll
                for (int n = 0; n < kN; n += 2)
                    stsm4(aq + 2 * (n * 8), Hf::pack(O[n][0], O[n][1]), Hf::pack(O[n][2], O[n][3]), Hf::pack(O[n + 1][0], O[n + 1][1]),
                          Hf::pack(O[n + 1][2], O[n + 1][3]));
                __syncwarp();
                T* po = const_cast<T*>(static_cast<const T*>(r.o.p)) + obase + c0;
#pragma unroll
                for (int i = lane; i < 16 * kUnitsV; i += 32) {
                    const int row = i / kUnitsV, u = i % kUnitsV;
                    if (u < uv && t0 + row < t_end)
                        st_vec(po + (long long)(t0 + row) * r.o.st + u * 8, *reinterpret_cast<const uint4*>(sq + row * L::kStrideA + u * 8));
                }
                __syncwarp();
            } else {
#pragma unroll
                for (int n = 0; n < kN; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int t = t0 + g + (e >> 1) * 8, col = n * 8 + 2 * t4 + (e & 1);
                        if (t < t_end && col < cols) {
                            const long long at = obase + (long long)t * r.o.st + (long long)(c0 + col) * r.o.sd;
                            if (r.out_f32)
                                const_cast<float*>(static_cast<const float*>(r.o.p))[at] = O[n][e];
                            else
                                const_cast<T*>(static_cast<const T*>(r.o.p))[at] = E::from_float(O[n][e]);
                        }
                    }
            }
        };
        if (!STATES && chunks > 0) load_q(0);
        cp_commit();
        for (int chunk = 0; chunk < chunks; ++chunk) {
            cp_wait();
            __syncthreads();  // this chunk's tokens and the rounded state are there; the other buffers are free
            if (chunk + 1 < chunks) load_kv(chunk + 1);
            cp_commit();
            if (chunk + 2 < chunks && warp == (chunk & 3)) fill_info(chunk + 2);
            if (!STATES) {
                outputs(chunk);
                if (chunk + 1 < chunks) load_q(chunk + 1);
                cp_commit();
            }
        }
        return;
    }

    // ----------------------------------------------------------------------------------------------- state
    if constexpr (Registers<DAP>::kShares) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Registers<DAP>::kState));
    float X[kMine][kN][4];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const int blk = warp + kWarps * i;
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = blk * 16 + g + (e >> 1) * 8, col = n * 8 + 2 * t4 + (e & 1);
                float x = 0.f;
                if (!STATES && blk < kBlocks && row < r.da && col < cols) {
                    if (seg > 0)
                        x = c.seg_state[blockIdx.z][((long long)(seg - 1) * c.batch * c.heads + bh) * ((long long)r.da * r.dv) +
                                                    (long long)row * r.dv + c0 + col];
                    else if (r.x0.p != nullptr)
                        x = r.x0.p[(long long)b * r.x0.sb + (long long)h * r.x0.sh + (long long)row * r.x0.sr + (long long)(c0 + col) * r.x0.sc];
                }
                X[i][n][e] = x;
            }
    }
    // Rounds X into the buffer of `chunk`.  fp16: scaled by a power of two around the largest magnitude of the slab.
    auto store_x = [&](int chunk) {
        float up = 1.f;
        if constexpr (kF16) {
            float m = 0.f, down;
#pragma unroll
            for (int i = 0; i < kMine; ++i)
#pragma unroll
                for (int n = 0; n < kN; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(X[i][n][e]));
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
            float* own = warp_max + (chunk & 1) * kWarps;
            if (lane == 0) own[warp] = m;
            asm volatile("bar.sync 2, %0;" ::"n"(kThreads / 2) : "memory");
            m = own[0];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) m = fmaxf(m, own[w]);
            scale_around(m, -100, &up, &down);
        }
        T* sx = sm + L::kX + (L::kOneX ? 0 : (chunk & 1) * DAP * L::kStrideX);
        const uint32_t at = smem_u32(sx + (lane & 15) * L::kStrideX + (lane >> 4) * 8);
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int blk = warp + kWarps * i;
            if (blk < kBlocks) {
#pragma unroll
                for (int n = 0; n < kN; n += 2)
                    stsm4(at + 2 * (blk * 16 * L::kStrideX + n * 8), Hf::pack(X[i][n][0] * up, X[i][n][1] * up),
                          Hf::pack(X[i][n][2] * up, X[i][n][3] * up), Hf::pack(X[i][n + 1][0] * up, X[i][n + 1][1] * up),
                          Hf::pack(X[i][n + 1][2] * up, X[i][n + 1][3] * up));
            }
        }
    };
    if (!STATES && chunks > 0) store_x(0);
    cp_commit();
    double seg_factor = 1.0;
    const bool want_last = STATES || seg < c.segments - 1 || r.xT.p != nullptr;

    for (int chunk = 0; chunk < chunks; ++chunk) {
        cp_wait();
        __syncthreads();
        if (chunk + 1 < chunks) load_kv(chunk + 1);
        cp_commit();
        const bool more = chunk + 1 < chunks;
        // without a token the state stays, whatever it holds: not even times 1 + 0
        if ((more || want_last) && infos[chunk % 3].n_all != 0) {
            const Info& f = infos[chunk % 3];
            const T* sk = sm + L::kK + (chunk & 1) * kChunk * L::kStrideA;
            const T* sv = sm + L::kV + (chunk & 1) * kChunk * L::kStrideV;
            const float2 fac = make_float2(pw_hi[f.n_all], pw_lo[f.n_all]);
            const bool keep = f.run_all == 0;
            if (STATES) seg_factor = keep ? seg_factor * ((double)fac.x + (double)fac.y) : 0.0;
            const uint32_t ak = smem_u32(sk + ((lane & 7) + (lane >> 4) * 8) * L::kStrideA + (lane >> 3 & 1) * 8);
            const uint32_t bv = smem_u32(sv + ((lane & 7) + (lane >> 3 & 1) * 8) * L::kStrideV + (lane >> 4) * 8);
            // column tiles whose sums are formed at once: all, or, for want of registers, 48 and 32 columns
            constexpr int kGroup = BV == 80 ? 6 : kN;
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const int blk = warp + kWarps * i;
                if (blk >= kBlocks) continue;
#pragma unroll
                for (int n0 = 0; n0 < kN; n0 += kGroup) {
                    constexpr int kMost = kGroup;
                    const int tiles = kN - n0 < kMost ? kN - n0 : kMost;  // a constant once unrolled
                    float acc[kMost][4] = {};
#pragma unroll 1
                    for (int kk = 0; kk < 4; ++kk) {
                        uint32_t kf[4], A[kF16 ? 16 : 12];
                        ldsm4t(kf, ak + 2 * (kk * 16 * L::kStrideA + blk * 16));
                        const float2 w0 = *reinterpret_cast<const float2*>(f.add + kk * 16 + 2 * t4);
                        const float2 w1 = *reinterpret_cast<const float2*>(f.add + kk * 16 + 8 + 2 * t4);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float2 x = mul2(make_float2(Hf::lo(kf[e]), Hf::hi(kf[e])), e < 2 ? w0 : w1);
                            if constexpr (kF16) {
                                // keys 2t go to the first, 2t + 1 to the second half of a step of eight
                                const int at = (e >> 1) * 8 + (e & 1);
                                A[at] = to_tf32(x.x);
                                A[at + 2] = to_tf32(x.y);
                                A[at + 4] = to_tf32(x.x - __uint_as_float(A[at]));
                                A[at + 6] = to_tf32(x.y - __uint_as_float(A[at + 2]));
                            } else {
                                // three parts cut off the top, eight bits each: nothing of the 24 is lost
#pragma unroll
                                for (int p = 0; p < 3; ++p) {
                                    A[4 * p + e] = __byte_perm(__float_as_uint(x.x), __float_as_uint(x.y), 0x7632);
                                    if (p < 2)
                                        x = fma2(make_float2(__uint_as_float(__float_as_uint(x.x) & 0xffff0000u), __uint_as_float(__float_as_uint(x.y) & 0xffff0000u)),
                                                 make_float2(-1.f, -1.f), x);
                                }
                            }
                        }
#pragma unroll
                        for (int j = 0; j < kMost; j += 2) {
                            if (j >= tiles) break;
                            uint32_t vb[4];
                            ldsm4t(vb, bv + 2 * (kk * 16 * L::kStrideV + (n0 + j) * 8));
                            if constexpr (kF16) {
#pragma unroll
                                for (int m = 0; m < 2; ++m) {
                                    const uint32_t x0 = __float_as_uint(Hf::lo(vb[2 * m])), x1 = __float_as_uint(Hf::hi(vb[2 * m]));
                                    const uint32_t y0 = __float_as_uint(Hf::lo(vb[2 * m + 1])), y1 = __float_as_uint(Hf::hi(vb[2 * m + 1]));
                                    mma_tf32(acc[j + m], A[4], A[5], A[6], A[7], x0, x1);
                                    mma_tf32(acc[j + m], A[12], A[13], A[14], A[15], y0, y1);
                                    mma_tf32(acc[j + m], A[0], A[1], A[2], A[3], x0, x1);
                                    mma_tf32(acc[j + m], A[8], A[9], A[10], A[11], y0, y1);
                                }
                            } else {
#pragma unroll
                                for (int p = 2; p >= 0; --p) {
                                    const uint32_t a[4] = {A[4 * p], A[4 * p + 1], A[4 * p + 2], A[4 * p + 3]};
                                    Hf::mma(acc[j], a, vb[0], vb[1]);
                                    Hf::mma(acc[j + 1], a, vb[2], vb[3]);
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int j = 0; j < kMost; ++j) {
                        if (j >= tiles) break;
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            float* x = X[i][n0 + j] + e;
                            float2 y = make_float2(acc[j][e], acc[j][e + 1]);
                            if (keep) y = fma2(make_float2(x[0], x[1]), make_float2(fac.x, fac.x), fma2(make_float2(x[0], x[1]), make_float2(fac.y, fac.y), y));
                            x[0] = y.x;
                            x[1] = y.y;
                        }
                    }
                }
            }
        }
        if (!STATES) {
            if (L::kOneX) asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");  // the queries have read this chunk's X
            if (more) store_x(chunk + 1);
        }
    }

    // ---- the state after the last token ----
    const bool write_final = !STATES && seg == c.segments - 1 && r.xT.p != nullptr;
    if (STATES || write_final) {
        float* dst = STATES ? c.seg_state[blockIdx.z] + ((long long)seg * c.batch * c.heads + bh) * ((long long)r.da * r.dv)
                            : r.xT.p + (long long)b * r.xT.sb + (long long)h * r.xT.sh;
        const long long sr = STATES ? r.dv : r.xT.sr, sc = STATES ? 1 : r.xT.sc;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int blk = warp + kWarps * i;
#pragma unroll
            for (int n = 0; n < kN; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int row = blk * 16 + g + (e >> 1) * 8, col = n * 8 + 2 * t4 + (e & 1);
                    if (blk < kBlocks && row < r.da && col < cols) dst[(long long)row * sr + (long long)(c0 + col) * sc] = X[i][n][e];
                }
        }
        if (STATES && slab == 0 && tid == kThreads / 2) {
            const float hi = (float)seg_factor;
            c.seg_factor[blockIdx.z][(long long)seg * c.batch * c.heads + bh] = make_float2(hi, (float)(seg_factor - (double)hi));
        }
    }
}

template <int DT, int DAP, int BV, bool STATES>
cudaError_t launch(const Launch& l, cudaStream_t s) {
    constexpr int smem = Layout<DAP, BV>::kBytes;
    int slabs = 0;
    for (int i = 0; i < l.runs; ++i) slabs = max(slabs, (l.run[i].dv + BV - 1) / BV);
    auto kernel = k_linear_mma<DT, DAP, BV, STATES>;
    if constexpr (Registers<DAP>::kShares) {
        static std::atomic<bool> fits{false};
        const cudaError_t r = check_registers(kernel, kThreads, Registers<DAP>::kShare, fits);
        if (r != cudaSuccess) return r;
    }
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned)(l.c.batch * l.c.heads * slabs), STATES ? l.c.segments - 1 : l.c.segments, l.runs);
    note_launch(STATES ? "linear_mma_states" : "linear_mma");
    kernel<<<grid, kThreads, smem, s>>>(l);
    return cudaGetLastError();
}

template <int DT>
cudaError_t launch_type(const Launch& l, bool states, cudaStream_t s) {
    switch (mma_rows(l)) {
        case 64: return states ? launch<DT, 64, 64, true>(l, s) : launch<DT, 64, 64, false>(l, s);
        case 128: return states ? launch<DT, 128, 64, true>(l, s) : launch<DT, 128, 64, false>(l, s);
        case 160: return states ? launch<DT, 160, 80, true>(l, s) : launch<DT, 160, 80, false>(l, s);
        default: return states ? launch<DT, 256, 64, true>(l, s) : launch<DT, 256, 64, false>(l, s);
    }
}

}  // namespace mma
}  // namespace lin
}  // namespace vc1d
