// One token of linear attention against the fp32 state (decode):
//     S <- a S + k v^T (in place),   o = scale * q^T S
// The state is read and written once and everything else is small, so the call is bound by 8 bytes of HBM traffic per
// state element.  A CTA owns a slab of columns of one (row, head): a row of the slab is 8 or 16 lanes of 16 bytes, and
// every thread has up to eight rows in flight, asked for together with the keys and queries that go with them.  Wide slabs
// where there are CTAs enough to fill the GPU several times over (fewer, longer CTAs), narrow ones else.  The sum over
// the rows of S is finished with shuffles and one exchange through shared memory.
//
// Measured: 256 requests of 16 heads of 128 x 128 in 100 us (5.3 TB/s, 0.80 of a plain copy's rate, which is what a read
// and write of the same lines reaches here); one request of 4 heads of 160 x 160 in 4 us, which is launch and latency.
#include "linear_attention.cuh"

namespace vc1d {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = VC1D_LINEAR_MAX_DIM;

struct LUParams {
    const void *q, *k, *v, *mask;
    void* out;
    float* state;
    const float* log_decay;
    long long q_s[3], k_s[3], v_s[3], o_s[3], s_s[4], mask_s;
    int heads, group_k, group_v, da, dv, slabs, mask_dtype;
    float scale;
};

// VEC: columns per thread.  4: state rows of 16-byte aligned float4; 1: any strides.  ACROSS: threads along the columns.
template <int DT, int VEC, int ACROSS>
__global__ void __launch_bounds__(kThreads) k_linear_update(const __grid_constant__ LUParams p) {
    using E = Elem<DT>;
    using T = typename E::type;
    constexpr int kCols = ACROSS * VEC;
    constexpr int kRows = kThreads / ACROSS;   // rows in flight per step
    constexpr int kSteps = kMaxDim / kRows;    // steps of the largest head
    constexpr int kBatch = 8;                  // rows in flight per thread
    __shared__ float part[kThreads / 32][kCols];

    const int slab = blockIdx.x % p.slabs;
    const long long bh = blockIdx.x / p.slabs;
    const long long b = bh / p.heads;
    const int h = (int)(bh % p.heads);
    const int tid = threadIdx.x, lane = tid & 31;
    const int col = slab * kCols + (tid % ACROSS) * VEC, row0 = tid / ACROSS;
    const bool in = col < p.dv;
    T* out = static_cast<T*>(p.out) + b * p.o_s[0] + h * p.o_s[1];

    if (p.mask != nullptr && !lin::mask_valid(p.mask, p.mask_dtype, b * p.mask_s)) {
        if (tid < kCols && slab * kCols + tid < p.dv) out[(long long)(slab * kCols + tid) * p.o_s[2]] = E::from_float(0.f);
        return;
    }
    float* s = p.state + b * p.s_s[0] + h * p.s_s[1];
    const T* q = static_cast<const T*>(p.q) + b * p.q_s[0] + h * p.q_s[1];
    const T* k = static_cast<const T*>(p.k) + b * p.k_s[0] + (h / p.group_k) * p.k_s[1];
    const T* v = static_cast<const T*>(p.v) + b * p.v_s[0] + (h / p.group_v) * p.v_s[1];

    float acc[VEC] = {}, vv[VEC] = {};
    float2 a = make_float2(0.f, 0.f);
#pragma unroll
    for (int step0 = 0; step0 < kSteps; step0 += kBatch) {
        if (step0 > 0 && step0 * kRows >= p.da) break;
        float x[kBatch][VEC], kk[kBatch], qq[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int row = row0 + (step0 + i) * kRows;
            if (step0 + i < kSteps && in && row < p.da) {
                if constexpr (VEC == 4) {
                    const float4 f = __ldcs(reinterpret_cast<const float4*>(s + row * p.s_s[2] + col));
                    x[i][0] = f.x, x[i][1] = f.y, x[i][2] = f.z, x[i][3] = f.w;
                } else {
                    x[i][0] = s[row * p.s_s[2] + col * p.s_s[3]];
                }
                kk[i] = E::to_float(k[row * p.k_s[2]]);
                qq[i] = E::to_float(q[row * p.q_s[2]]);
            }
        }
        if (step0 == 0) {
            if (in) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) vv[j] = E::to_float(v[(long long)(col + j) * p.v_s[2]]);
            }
            // the decay in two floats: its rounding to one would repeat with the same sign at every token
            if (lane == 0) {
                const double e = exp((double)p.log_decay[h]);
                a.x = (float)e;
                const double lo = e - (double)a.x;
                a.y = (isfinite(a.x) && lo == lo) ? (float)lo : 0.f;
            }
            a.x = __shfl_sync(0xffffffffu, a.x, 0);
            a.y = __shfl_sync(0xffffffffu, a.y, 0);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int row = row0 + (step0 + i) * kRows;
            if (step0 + i < kSteps && in && row < p.da) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    x[i][j] = fmaf(x[i][j], a.x, fmaf(x[i][j], a.y, kk[i] * vv[j]));
                    acc[j] = fmaf(qq[i], x[i][j], acc[j]);
                }
                if constexpr (VEC == 4)
                    __stcs(reinterpret_cast<float4*>(s + row * p.s_s[2] + col), make_float4(x[i][0], x[i][1], x[i][2], x[i][3]));
                else
                    s[row * p.s_s[2] + col * p.s_s[3]] = x[i][0];
            }
        }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
#pragma unroll
        for (int m = ACROSS; m < 32; m <<= 1) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], m);
        if (lane < ACROSS) part[tid / 32][lane * VEC + j] = acc[j];
    }
    __syncthreads();
    if (tid < kCols && slab * kCols + tid < p.dv) {
        float o = 0.f;
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) o += part[w][tid];
        out[(long long)(slab * kCols + tid) * p.o_s[2]] = E::from_float(o * p.scale);
    }
}

template <int DT>
cudaError_t launch(LUParams p, bool vec, long long heads, cudaStream_t s) {
    // wide slabs from four CTAs per SM on: 256 requests x 16 heads of 128 x 128
    const long long wide = heads * ((p.dv + 63) / 64);
    const bool is_wide = vec && wide >= 4LL * sm_count();
    const int cols = is_wide ? 64 : 32;
    p.slabs = (p.dv + cols - 1) / cols;
    const unsigned blocks = (unsigned)(heads * p.slabs);
    note_launch("linear_update");
    if (is_wide)
        k_linear_update<DT, 4, 16><<<blocks, kThreads, 0, s>>>(p);
    else if (vec)
        k_linear_update<DT, 4, 8><<<blocks, kThreads, 0, s>>>(p);
    else
        k_linear_update<DT, 1, 32><<<blocks, kThreads, 0, s>>>(p);
    return cudaGetLastError();
}

}  // namespace
}  // namespace vc1d

extern "C" {

VC1D_API int vc1d_linear_update(const vc1d_linear_update_args* a, void* stream) {
    using namespace vc1d;
    if (a == nullptr) return VC1D_E_NULL;
    if (a->struct_size != sizeof(vc1d_linear_update_args)) return VC1D_E_STRUCT;
    if (!lin::is_io_dtype(a->dtype)) return VC1D_E_DTYPE;
    if (a->mask != nullptr && !lin::is_mask_dtype(a->mask_dtype)) return VC1D_E_DTYPE;
    if (a->batch < 0 || a->heads < 1 || a->heads_k < 1 || a->heads_v < 1 || a->dim_k < 1 || a->dim_v < 1) return VC1D_E_SHAPE;
    if (a->heads % a->heads_k != 0 || a->heads % a->heads_v != 0) return VC1D_E_SHAPE;
    if (a->dim_k > kMaxDim || a->dim_v > kMaxDim) return VC1D_E_TOO_LARGE;
    const long long heads = (long long)a->batch * a->heads;
    if (heads * (kMaxDim / 32) > 0x7fffffffLL) return VC1D_E_TOO_LARGE;
    if (heads == 0) return VC1D_OK;
    if (a->q == nullptr || a->k == nullptr || a->v == nullptr || a->out == nullptr || a->state == nullptr || a->log_decay == nullptr)
        return VC1D_E_NULL;
    const int n_q[3] = {a->batch, a->heads, a->dim_k}, n_k[3] = {a->batch, a->heads_k, a->dim_k}, n_v[3] = {a->batch, a->heads_v, a->dim_v},
              n_o[3] = {a->batch, a->heads, a->dim_v}, n_s[4] = {a->batch, a->heads, a->dim_k, a->dim_v};
    if (!lin::writable(n_o, a->out_strides) || !lin::writable(n_s, a->state_strides)) return VC1D_E_STRIDE;
    const int eb = elem_bytes(a->dtype), n_h[1] = {a->heads}, n_b[1] = {a->batch};
    const int64_t one[1] = {1}, mask_stride[1] = {a->mask_stride};
    lin::Touched t;
    t.reads_from(lin::extent(a->q, eb, n_q, a->q_strides));
    t.reads_from(lin::extent(a->k, eb, n_k, a->k_strides));
    t.reads_from(lin::extent(a->v, eb, n_v, a->v_strides));
    t.reads_from(lin::extent(a->log_decay, 4, n_h, one));
    if (a->mask != nullptr) t.reads_from(lin::extent(a->mask, elem_bytes(a->mask_dtype), n_b, mask_stride));
    t.writes_to(lin::extent(a->out, eb, n_o, a->out_strides));
    t.writes_to(lin::extent(a->state, 4, n_s, a->state_strides));
    if (t.clash()) return VC1D_E_ALIAS;
    LUParams p{};
    p.q = a->q;
    p.k = a->k;
    p.v = a->v;
    p.mask = a->mask;
    p.out = a->out;
    p.state = a->state;
    p.log_decay = a->log_decay;
    for (int i = 0; i < 3; ++i) {
        p.q_s[i] = a->q_strides[i];
        p.k_s[i] = a->k_strides[i];
        p.v_s[i] = a->v_strides[i];
        p.o_s[i] = a->out_strides[i];
    }
    for (int i = 0; i < 4; ++i) p.s_s[i] = a->state_strides[i];
    p.mask_s = a->mask_stride;
    p.mask_dtype = a->mask_dtype;
    p.heads = a->heads;
    p.group_k = a->heads / a->heads_k;
    p.group_v = a->heads / a->heads_v;
    p.da = a->dim_k;
    p.dv = a->dim_v;
    p.scale = a->scale;
    const bool vec = a->state_strides[3] == 1 && a->dim_v % 4 == 0 && a->state_strides[0] % 4 == 0 && a->state_strides[1] % 4 == 0 &&
                     a->state_strides[2] % 4 == 0 && (reinterpret_cast<uintptr_t>(a->state) & 15u) == 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (a->dtype) {
        case VC1D_F32: return (int)launch<VC1D_F32>(p, vec, heads, s);
        case VC1D_BF16: return (int)launch<VC1D_BF16>(p, vec, heads, s);
        default: return (int)launch<VC1D_F16>(p, vec, heads, s);
    }
}

VC1D_API uint32_t vc1d_sizeof_linear_update_args(void) { return (uint32_t)sizeof(vc1d_linear_update_args); }

}  // extern "C"
