// Linear attention with a fixed decay for each head: what the kernels of the operator share.
//
// With a = exp(log_decay[h]) and n_i the number of valid tokens up to and with token i:
//     S_t = a S_{t-1} + k_t v_t^T,     o_t = scale * q_t^T S_t          (a masked token leaves S alone, o_t = 0)
// A chunk of C tokens that starts from the state X needs no step-by-step recurrence:
//     o_i = scale * [ a^{n_i} q_i X + sum_{j<=i} a^{n_i - n_j} (q_i . k_j) v_j ]        (n counted inside the chunk)
//     X' = a^{n_C} X + sum_j a^{n_C - n_j} k_j v_j^T
//
// Every pass of the operator is one "run" of that chunk recurrence over (a, k, v) -> out:
//     forward   (q,  k,  v) -> o    tokens in order,  state [Dk, Dv]
//     dq        (do, v,  k) -> dq   tokens in order,  state [Dv, Dk] (the forward's, transposed)
//     dk        (v,  do, q) -> dk   last token first, state [Dv, Dk] (gradient of S, transposed)
//     dv        (k,  q, do) -> dv   last token first, state [Dk, Dv] (gradient of S)
// In the backward direction the state that enters a chunk is a * dS, so that the gradient of the final state enters
// as it is and the gradient of the initial state leaves as it is; the powers then shift by one (`shift` below).
#pragma once

#include <atomic>
#include <cstdlib>

#include "vc1d_common.cuh"
#include "vc1d_internal.h"

namespace vc1d {
namespace lin {

constexpr int kChunk = 64;             // tokens of a chunk
constexpr int kMaxDim = 256;           // largest head dimension
constexpr int kPowers = kChunk + 2;    // a^0 .. a^(kChunk + 1)
constexpr int kMaxSegments = 64;

struct Rows {  // [batch, token, head, channel], element strides; token stride negative when time runs backwards
    const void* p;
    long long sb, st, sh, sd;
    int group;  // head h reads head h / group
};

struct State {  // [batch, head, row, column] fp32
    float* p;
    long long sb, sh, sr, sc;
};

struct Run {
    Rows a, k, v, o;  // o.p is written
    State x0, xT;     // state before the first and after the last token; p may be NULL
    int da, dv;       // channels of a and k (rows of the state), channels of v and out (its columns)
    int out_f32;      // out holds fp32 (partial sums of shared heads), else the I/O type
    int out_vec;      // out takes 16-byte stores (tensor-core kernel)
    int reverse;      // tokens run from the last to the first (the strides of a, k, v, o already say so)
    int shift;        // 1 in the backward direction
    float s_pair, s_carry, s_add;  // factors on the products inside a chunk, on a X, and on what enters the state
};

struct Common {
    const float* log_decay;
    const void* mask;           // [batch, token]; NULL = every token is valid
    const int32_t* seq_idx;     // [batch, token]; NULL = one sequence
    long long mask_sb, mask_st, seq_sb, seq_st;
    int mask_dtype;
    int batch, heads, seqlen;
    int segments;               // time is split into this many parts of seg_chunks chunks
    int seg_chunks;
    int test_expire;            // self-test: the chunk, counted from 1, that kTc withholds; 0 = none
    // workspace of a split launch, per run: [segments - 1][batch * heads][da * dv] states, then factors (hi, lo)
    float* seg_state[3];
    float2* seg_factor[3];
};

constexpr int kMaxRuns = 3;
struct Launch {
    Common c;
    Run run[kMaxRuns];
    int runs;
};

__device__ __forceinline__ bool mask_valid(const void* mask, int dtype, long long at) {
    switch (dtype) {
        case VC1D_U8: return static_cast<const uint8_t*>(mask)[at] != 0;
        case VC1D_I32: return static_cast<const int32_t*>(mask)[at] != 0;
        case VC1D_I64: return static_cast<const int64_t*>(mask)[at] != 0;
        case VC1D_F32: return static_cast<const float*>(mask)[at] != 0.f;
        // bf16 and fp16: any bit apart from the sign
        default: return (static_cast<const uint16_t*>(mask)[at] & 0x7fffu) != 0;
    }
}

// What a chunk needs to know about its tokens.  code[i] = n_i + (run_i << 16), where n_i counts the valid tokens up to
// and with i and run_i the sequence starts up to and with i (packed rows).  For two tokens i, j of a chunk,
// (unsigned)(code[i] - code[j]) <= kChunk exactly when j is not later than i among the valid tokens and of the same
// sequence; the difference then is the power of the decay.  Rows of masked tokens count as zeros, so theirs does not matter.
struct ChunkInfo {
    int code[kChunk];
    unsigned valid[2];  // bit i % 32 of word i / 32
    int n_all;          // valid tokens
    int run_all;        // sequence starts
};

// One warp fills the info of the chunk that starts at token t0 (in the run's own order).  Tokens from t_end on are masked.
__device__ __forceinline__ void chunk_info(const Common& c, bool reverse, int b, int t0, int t_end, ChunkInfo* info) {
    const int lane = threadIdx.x & 31;
    unsigned ok[2], start[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int t = t0 + 32 * half + lane;
        const long long at = reverse ? c.seqlen - 1 - t : t;
        bool v = t < t_end, s = false;
        if (v && c.mask != nullptr) v = mask_valid(c.mask, c.mask_dtype, (long long)b * c.mask_sb + at * c.mask_st);
        if (t < t_end && c.seq_idx != nullptr && t > 0) {
            const int32_t* p = c.seq_idx + (long long)b * c.seq_sb + at * c.seq_st;
            s = p[0] != (reverse ? p[c.seq_st] : p[-c.seq_st]);
        }
        ok[half] = __ballot_sync(0xffffffffu, v);
        start[half] = __ballot_sync(0xffffffffu, s);
    }
    const unsigned upto = 0xffffffffu >> (31 - lane);
    const int n0 = __popc(ok[0]), r0 = __popc(start[0]);
    info->code[lane] = __popc(ok[0] & upto) + (__popc(start[0] & upto) << 16);
    info->code[lane + 32] = n0 + __popc(ok[1] & upto) + ((r0 + __popc(start[1] & upto)) << 16);
    if (lane == 0) {
        info->valid[0] = ok[0];
        info->valid[1] = ok[1];
        info->n_all = n0 + __popc(ok[1]);
        info->run_all = r0 + __popc(start[1]);
    }
}

// a^n for n = 0 .. kPowers - 1 as the sum of two floats.  The factor that a long-lived state meets once per chunk is
// applied with both parts: its rounding to one float (2^-25 relative) would repeat with the same sign at every chunk.
// n = 0 is exactly 1 also for log_decay = -inf.
__device__ __forceinline__ void fill_powers(float2* pw, float log_decay, int tid, int threads) {
    for (int n = tid; n < kPowers; n += threads) {
        const double x = n == 0 ? 1.0 : exp((double)log_decay * (double)n);
        const float hi = (float)x;
        const double lo = x - (double)hi;
        pw[n] = make_float2(hi, (isfinite(hi) && lo == lo) ? (float)lo : 0.f);
    }
}

// ---- host: checks of arguments ----
inline bool is_io_dtype(int dt) { return dt == VC1D_F32 || dt == VC1D_BF16 || dt == VC1D_F16; }
inline bool is_mask_dtype(int dt) { return is_io_dtype(dt) || dt == VC1D_U8 || dt == VC1D_I32 || dt == VC1D_I64; }

struct Range {
    const char *lo, *hi;
};
template <int D>
Range extent(const void* base, int eb, const int (&n)[D], const int64_t (&s)[D]) {
    long long lo = 0, hi = 0;
    for (int i = 0; i < D; ++i) {
        const long long span = (long long)(n[i] - 1) * s[i];
        (span < 0 ? lo : hi) += span;
    }
    const char* b = static_cast<const char*>(base);
    return {b + lo * eb, b + (hi + 1) * eb};
}
inline bool overlap(const Range& a, const Range& b) { return a.lo < b.hi && b.lo < a.hi; }
// Memory that a call reads and memory that it writes: what is written may overlap nothing else, the decays, masks and
// sequence numbers included, because some CTAs read them while others already store.
struct Touched {
    Range read[12], written[4];
    int reads = 0, writes = 0;
    void reads_from(const Range& r) { read[reads++] = r; }
    void writes_to(const Range& r) { written[writes++] = r; }
    bool clash() const {
        for (int i = 0; i < writes; ++i) {
            for (int j = 0; j < reads; ++j)
                if (overlap(written[i], read[j])) return true;
            for (int j = 0; j < i; ++j)
                if (overlap(written[i], written[j])) return true;
        }
        return false;
    }
};
// A written tensor gives every element a place of its own: each stride passes the whole extent of the axes with smaller ones
// (no stride 0, no windows that overlap).
template <int D>
bool writable(const int (&n)[D], const int64_t (&s)[D]) {
    int axis[D], used = 0;
    for (int i = 0; i < D; ++i) {
        if (n[i] == 0) return true;
        if (n[i] == 1) continue;
        int at = used++;
        for (; at > 0 && std::llabs(s[axis[at - 1]]) > std::llabs(s[i]); --at) axis[at] = axis[at - 1];
        axis[at] = i;
    }
    long long span = 0;
    for (int i = 0; i < used; ++i) {
        const long long stride = std::llabs(s[axis[i]]);
        if (stride <= span) return false;
        span += (long long)(n[axis[i]] - 1) * stride;
    }
    return true;
}

// Kernels whose warps have unequal shares of the registers (setmaxnreg).  A share that is raised waits, without any limit, until
// the other warps have given up enough of what the CTA was launched with: `share` is what all warps together ask for.
constexpr bool shares_fit(int regs_per_thread, int threads, int share) { return (regs_per_thread + 7) / 8 * 8 * threads >= share; }
static_assert(shares_fit(80, 768, 61440) && shares_fit(73, 768, 61440) && !shares_fit(72, 768, 61440) && !shares_fit(120, 256, 32768));

// Refuses a launch whose compiled kernel has not the registers that its shares add up to; asked for until it was found once.
template <typename Kernel>
cudaError_t check_registers(Kernel* kernel, int threads, int share, std::atomic<bool>& fits) {
    if (fits.load(std::memory_order_relaxed)) return cudaSuccess;
    cudaFuncAttributes at{};
    cudaError_t e = cudaFuncGetAttributes(&at, kernel);
    if (e == cudaSuccess && !shares_fit(at.numRegs, threads, share)) e = cudaErrorLaunchOutOfResources;
    if (e == cudaSuccess) fits.store(true, std::memory_order_relaxed);
    return e;
}

// The kernels.  kMma: warp-level products, 16-bit types, any head.  kTc: tcgen05, bf16, heads up to 160.
enum Kind { kSimt, kMma, kTc };

inline int largest_rows(const Launch& l) {
    int da = 0;
    for (int i = 0; i < l.runs; ++i) da = l.run[i].da > da ? l.run[i].da : da;
    return da;
}
// Rows of the state that kMma is compiled for; columns of a slab; tokens of a chunk; CTAs that share an SM.  160 rows
// (Viby's heads) have a kMma variant of their own with slabs of 80: half of 160 columns, and two CTAs per SM.
inline int mma_rows(const Launch& l) {
    const int da = largest_rows(l);
    return da <= 64 ? 64 : da <= 128 ? 128 : da <= 160 ? 160 : 256;
}
inline int slab_of(const Launch& l, Kind k) { return k == kMma && mma_rows(l) == 160 ? 80 : 64; }
inline int chunk_of(Kind k) { return k == kTc ? 128 : kChunk; }
inline int ctas_per_sm(const Launch& l, Kind k) { return (k == kMma && mma_rows(l) <= 160) || (k == kSimt && largest_rows(l) <= 96) ? 2 : 1; }

}  // namespace lin

// Launchers.
// states_only: no outputs; part s of the time axis leaves its own state and total factor in the workspace.
cudaError_t launch_linear_simt(const lin::Launch& l, int dtype, bool states_only, cudaStream_t s);
// 16-bit types only; a, k, v with channel stride 1, 16-byte aligned rows, dims a multiple of 8 (lin::mma_fits).
cudaError_t launch_linear_mma_bf16(const lin::Launch& l, bool states_only, cudaStream_t s);
cudaError_t launch_linear_mma_f16(const lin::Launch& l, bool states_only, cudaStream_t s);
// bf16, as above and at most 160 state rows in every run.
cudaError_t launch_linear_tc(const lin::Launch& l, bool states_only, cudaStream_t s);
// Packed rows, after the outputs: replaces what bad values of one sequence left in the others.
cudaError_t launch_linear_isolate(const lin::Launch& l, int dtype, cudaStream_t s);

}  // namespace vc1d
