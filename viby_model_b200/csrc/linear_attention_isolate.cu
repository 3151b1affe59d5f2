// Packed rows: keeps the infinities and NaN of one sequence out of the others.
//
// The kernels take a chunk's products at once: a pair of tokens of different sequences, or of a query and a later key, has the
// weight 0, and 0 times a value that is not finite is NaN.  So a bad value of one request would reach its neighbours in the
// chunk, and through the state all of the request that follows.  What it leaves there is always NaN, never infinity, and it is
// rare: this kernel looks the outputs over and, where a token has a NaN although no key or value of its own sequence up to
// it is to blame, runs the recurrence for it as it is written,
//     Y_t = a Y_{t-1} + s k_t v_t^T,   o_t = q_t^T Y_t     from the sequence's first token,
// and replaces the NaN.  All other outputs stay as they are.
//
// It need not read all outputs.  A bad value in a chunk shows in the chunk's last token (as an infinity where that is of the same
// sequence, else as the NaN that 0 times it is), a bad state in all tokens of the sequence that the chunk starts in: the
// last token of every 64 (both lengths of chunks end there) and of every sequence tell.
//
// Bound by its launch and its latency.  A CTA takes 256 tokens of one (row, head, slab of 64 columns).  24567 tokens of 8 heads of
// 64: 6 us (bf16) to 10 us (fp16) behind main kernels of 81 and 102; 300 tokens: 3 us.  1024 tokens a CTA, or more CTAs an SM
// for fewer registers, took the same.  The recurrence costs about two microseconds a token, behind a bad value only.
#include "linear_attention.cuh"

namespace vc1d {
namespace lin {
namespace {

constexpr int kThreads = 256;
constexpr int kPart = kThreads;  // tokens of a CTA
constexpr int kSlab = 64;
constexpr int kGroups = kThreads / kSlab;
constexpr int kRowsEach = kMaxDim / kGroups;  // state rows of a thread

__device__ __forceinline__ bool is_nan(float x) { return x != x; }
__device__ __forceinline__ bool is_nan(__nv_bfloat16 x) { return (__bfloat16_as_ushort(x) & 0x7fffu) > 0x7f80u; }
__device__ __forceinline__ bool is_nan(__half x) { return (__half_as_ushort(x) & 0x7fffu) > 0x7c00u; }

// This thread's share of the rows first .. last - 1 (at most kPart): 16 bytes of every so many rows, all a few of them asked for at once.
template <typename O>
__device__ __forceinline__ bool nan_in_rows(const O* o, long long stride, int first, int last, int cols) {
    constexpr int kPer = 16 / (int)sizeof(O), kAcross = kSlab / kPer, kDown = kThreads / kAcross, kSteps = kPart / kDown, kBatch = 8;
    const int at = (int)threadIdx.x % kAcross * kPer, row = first + (int)threadIdx.x / kAcross;
    if (at >= cols) return false;
    bool bad = false;
#pragma unroll
    for (int s0 = 0; s0 < kSteps; s0 += kBatch) {
        uint4 x[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int t = row + (s0 + i) * kDown;
            x[i] = t < last ? *reinterpret_cast<const uint4*>(o + (long long)t * stride + at) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const O* y = reinterpret_cast<const O*>(&x[i]);
#pragma unroll
            for (int j = 0; j < kPer; ++j) bad |= is_nan(y[j]);
        }
    }
    return bad;
}

template <int DT>
__global__ void __launch_bounds__(kThreads, 2) k_linear_isolate(const __grid_constant__ Launch l, int pieces, int slabs_most) {
    using E = Elem<DT>;
    using T = typename E::type;
    __shared__ float key[kMaxDim], query[kMaxDim], sums[kGroups][kSlab];
    __shared__ int found;
    griddep_wait();
    const Run& r = l.run[blockIdx.z];
    const Common& c = l.c;
    const int tid = threadIdx.x, slabs = (r.dv + kSlab - 1) / kSlab;

    for (int piece = blockIdx.y; piece < pieces; piece += gridDim.y) {  // row, head and slab
        const int slab = piece % slabs_most, bh = piece / slabs_most;
        if (slab >= slabs) continue;  // a run with fewer slabs than the launch's widest
        const int b = bh / c.heads, h = bh % c.heads, c0 = slab * kSlab, cols = min(kSlab, r.dv - c0);
        const int i0 = blockIdx.x * kPart, i1 = min(c.seqlen, i0 + kPart);  // tokens in the run's order
        const T* pa = static_cast<const T*>(r.a.p) + (long long)b * r.a.sb + (long long)(h / r.a.group) * r.a.sh;
        const T* pk = static_cast<const T*>(r.k.p) + (long long)b * r.k.sb + (long long)(h / r.k.group) * r.k.sh;
        const T* pv = static_cast<const T*>(r.v.p) + (long long)b * r.v.sb + (long long)(h / r.v.group) * r.v.sh + (long long)c0 * r.v.sd;
        const long long out0 = (long long)b * r.o.sb + (long long)h * r.o.sh + (long long)c0 * r.o.sd;
        float* o32 = static_cast<float*>(const_cast<void*>(r.o.p));
        T* o16 = static_cast<T*>(const_cast<void*>(r.o.p));
        auto output = [&](int i, int col) {
            const long long at = out0 + (long long)i * r.o.st + (long long)col * r.o.sd;
            return r.out_f32 ? o32[at] : E::to_float(o16[at]);
        };
        auto out_is_nan = [&](int i, int col) { return is_nan(output(i, col)); };
        // whether any output of the tokens first .. last - 1 is NaN; one answer for the CTA
        auto nan_among = [&](int first, int last) {
            bool bad = false;
            if (r.out_vec && r.dv % 8 == 0) {
                bad = r.out_f32 ? nan_in_rows<float>(o32 + out0, r.o.st, first, last, cols) : nan_in_rows<T>(o16 + out0, r.o.st, first, last, cols);
            } else {
                for (int e = tid; e < (last - first) * cols; e += kThreads) bad |= out_is_nan(first + e / cols, e % cols);
            }
            return __syncthreads_or(bad) != 0;
        };
        auto starts = [&](int i) {  // whether a sequence starts at token i
            if (i == 0) return true;
            const long long at = r.reverse ? c.seqlen - 1 - i : i;
            const int32_t* p = c.seq_idx + (long long)b * c.seq_sb + at * c.seq_st;
            return p[0] != (r.reverse ? p[c.seq_st] : p[-c.seq_st]);
        };
        {
            const int i = i0 + tid, lane = tid & 31;
            unsigned tell = __ballot_sync(0xffffffffu, i < i1 && ((i & (kChunk - 1)) == kChunk - 1 || i == c.seqlen - 1 || starts(i + 1)));
            bool bad = false;
            while (tell != 0) {  // four tokens' rows at once
                float x[4][2];
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const int t = tell != 0 ? i - lane + __ffs(tell) - 1 : -1;
                    tell &= tell - 1;
                    x[n][0] = t >= 0 && lane < cols ? output(t, lane) : 0.f;
                    x[n][1] = t >= 0 && lane + 32 < cols ? output(t, lane + 32) : 0.f;
                }
#pragma unroll
                for (int n = 0; n < 4; ++n) bad |= !isfinite(x[n][0]) | !isfinite(x[n][1]);
            }
            if (!__syncthreads_or(bad) || !nan_among(i0, i1)) continue;
        }
        for (int p0 = i0, p1; p0 < i1; p0 = p1) {  // the sequences of the part
            __syncthreads();
            if (tid == 0) found = i1;
            __syncthreads();
            const int next = p0 + 1 + tid;
            if (next < i1 && starts(next)) atomicMin(&found, next);
            __syncthreads();
            p1 = found;
            if (!nan_among(p0, p1)) continue;
            int first = p0;  // of the sequence
            for (int hi = p0; p0 == i0; hi -= kThreads) {
                __syncthreads();
                if (tid == 0) found = -1;
                __syncthreads();
                if (hi - tid >= 0 && starts(hi - tid)) atomicMax(&found, hi - tid);
                __syncthreads();
                first = found;
                if (first >= 0) break;
            }
            // A bad state is in every token of the sequence from there on.  The part where that begins goes on through the others
            // (below): one walk for each sequence, however long.
            if (first < i0 && nan_among(i0 - 1, i0) && nan_among(i0, i0 + 1)) continue;
            // the sequence's first token with a key, or a value of this slab, that is not finite
            int end = p1;
            // (a token a warp at first: where all is bad that is enough)
            for (int t0 = first, each = 1; t0 < p1 && end == p1; t0 += kThreads / 32 * each, each = 32) {
                int worst = p1;
                for (int t = min(p1, t0 + (tid >> 5) * each + each) - 1; t >= t0 + (tid >> 5) * each; --t) {
                    bool bad = false;
                    for (int d = tid & 31; d < r.da; d += 32) bad |= !isfinite(E::to_float(pk[(long long)t * r.k.st + d * r.k.sd]));
                    for (int d = tid & 31; d < cols; d += 32) bad |= !isfinite(E::to_float(pv[(long long)t * r.v.st + d * r.v.sd]));
                    if (bad) worst = t;
                }
                __syncthreads();
                if (tid == 0) found = p1;
                __syncthreads();
                if (worst < p1) atomicMin(&found, worst);
                __syncthreads();
                end = found;
            }
            if (end <= p0 || !nan_among(p0, end)) continue;

            const int col = tid % kSlab, group = tid / kSlab;
            const double e = exp((double)c.log_decay[h]);
            const float hi = (float)e, lo = isfinite(hi) ? (float)(e - (double)hi) : 0.f;
            float Y[kRowsEach] = {};
            static_assert(kThreads == kMaxDim, "a thread per channel of a key");
            // a token's values as they are, asked for a token ahead
            T k_t = E::from_float(0.f), q_t = k_t, v_t = k_t, o_t = k_t;
            float o_t32 = 0.f;
            int id_t = 0, id_before = 0;
            auto ask = [&](int t) {
                if (tid < r.da) k_t = pk[(long long)t * r.k.st + tid * r.k.sd];
                if (tid < r.da && t >= p0) q_t = pa[(long long)t * r.a.st + tid * r.a.sd];
                if (col < cols) v_t = pv[(long long)t * r.v.st + col * r.v.sd];
                if (t >= p0 && tid < cols) {
                    const long long at = out0 + (long long)t * r.o.st + (long long)tid * r.o.sd;
                    if (r.out_f32)
                        o_t32 = o32[at];
                    else
                        o_t = o16[at];
                }
                if (t >= i1) {
                    const int32_t* p = c.seq_idx + (long long)b * c.seq_sb + (r.reverse ? c.seqlen - 1 - t : t) * c.seq_st;
                    id_t = p[0], id_before = r.reverse ? p[c.seq_st] : p[-c.seq_st];
                }
            };
            ask(first);
            for (int t = first; t < end; ++t) {
                __syncthreads();  // key, query and sums have been read
                const float k_now = E::to_float(k_t), v_now = E::to_float(v_t), v = v_now * r.s_pair;
                key[tid] = k_now;
                query[tid] = E::to_float(q_t);
                const bool replace = tid < cols && (r.out_f32 ? is_nan(o_t32) : is_nan(o_t));
                // in the parts that follow the sequence may end or have a bad value of its own
                if (__syncthreads_or((id_t != id_before) | !isfinite(k_now) | !isfinite(v_now))) break;
                if (t + 1 < end) ask(t + 1);
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < kRowsEach; ++i) {
                    const int row = i * kGroups + group;
                    if (i % 8 == 0 && i * kGroups >= r.da) break;  // channels from r.da on are zeros
                    Y[i] = fmaf(Y[i], hi, fmaf(Y[i], lo, key[row] * v));
                    sum = fmaf(query[row], Y[i], sum);
                }
                if (t < p0) continue;
                sums[group][col] = sum;
                __syncthreads();
                if (replace) {
                    float x = 0.f;
#pragma unroll
                    for (int g = 0; g < kGroups; ++g) x += sums[g][tid];
                    const long long at = out0 + (long long)t * r.o.st + (long long)tid * r.o.sd;
                    if (r.out_f32)
                        o32[at] = x;
                    else
                        o16[at] = E::from_float(x);
                }
                if (t + 1 == end && end % kPart == 0 && end < c.seqlen && nan_among(end, end + 1)) {
                    ask(end);
                    end = min(c.seqlen, end + kPart);
                }
            }
        }
    }
}

}  // namespace
}  // namespace lin

cudaError_t launch_linear_isolate(const lin::Launch& l, int dtype, cudaStream_t s) {
    using namespace lin;
    int slabs = 0;
    for (int i = 0; i < l.runs; ++i) slabs = max(slabs, (l.run[i].dv + kSlab - 1) / kSlab);
    const int pieces = l.c.batch * l.c.heads * slabs;  // fits: checked with the arguments
    // a programmatic dependent of the main kernel: its launch does not wait for that one to drain
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((l.c.seqlen + kPart - 1) / kPart, pieces < 65535 ? pieces : 65535, l.runs);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    switch (dtype) {
        case VC1D_F32: return cudaLaunchKernelEx(&cfg, k_linear_isolate<VC1D_F32>, l, pieces, slabs);
        case VC1D_BF16: return cudaLaunchKernelEx(&cfg, k_linear_isolate<VC1D_BF16>, l, pieces, slabs);
        default: return cudaLaunchKernelEx(&cfg, k_linear_isolate<VC1D_F16>, l, pieces, slabs);
    }
}

}  // namespace vc1d
