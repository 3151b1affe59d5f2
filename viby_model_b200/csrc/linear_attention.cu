// Linear attention: checks of arguments, how the time axis is split, and the runs that make up a forward or backward
// pass (linear_attention.cuh).  The products live in linear_attention_simt.cu, linear_attention_mma.cuh and
// linear_attention_tc.cuh.
#include <algorithm>

#include "linear_attention.cuh"

namespace vc1d {
namespace lin {
namespace {

// Joins the parts of the time axis: part s left its own state (from zero) and its total factor f_s; the state that
// part s + 1 starts from is f_s * (the one that part s started from) + that.  Written over the parts' own states.
__global__ void __launch_bounds__(256) k_linear_join(const __grid_constant__ Launch l) {
    const Run& r = l.run[blockIdx.y];
    const Common& c = l.c;
    const long long per = (long long)r.da * r.dv, all = (long long)c.batch * c.heads * per;
    float* state = c.seg_state[blockIdx.y];
    const float2* factor = c.seg_factor[blockIdx.y];
    const int parts = c.segments - 1, bhs = c.batch * c.heads;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (long long)gridDim.x * blockDim.x) {
        const int bh = (int)(i / per);
        float x = 0.f;
        if (r.x0.p != nullptr) {
            const int e = (int)(i % per), row = e / r.dv, col = e % r.dv;
            x = r.x0.p[(long long)(bh / c.heads) * r.x0.sb + (long long)(bh % c.heads) * r.x0.sh + (long long)row * r.x0.sr +
                       (long long)col * r.x0.sc];
        }
        for (int s0 = 0; s0 < parts; s0 += 8) {  // eight loads in flight
            float z[8];
            float2 f[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (s0 + j < parts) {
                    z[j] = state[(s0 + j) * all + i];
                    f[j] = factor[(long long)(s0 + j) * bhs + bh];
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (s0 + j < parts) {
                    // factor 0 is a sequence that ended inside the part: whatever came before is gone, infinities too
                    // a second half of 0 (a part without a token: the factor 1) adds nothing, where infinity * 0 would
                    x = f[j].x == 0.f ? z[j] : fmaf(x, f[j].x, f[j].y == 0.f ? z[j] : fmaf(x, f[j].y, z[j]));
                    state[(s0 + j) * all + i] = x;
                }
            }
        }
    }
}

// Gradients of shared heads: out[b, t, g, d] = sum over the heads of group g of part[b, t, h, d], in order of h.  A thread
// has four channels of one (b, t, g); bound by reading the partial sums once.
template <int DT>
__global__ void __launch_bounds__(256) k_linear_sum_heads(const float* part, Rows out, int heads, int seqlen, int dim, long long n) {
    using T = typename Elem<DT>::type;
    const int groups = heads / out.group, quads = (dim + 3) / 4;
    const bool whole = dim % 4 == 0;  // rows of partial sums are 16-byte aligned
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        const int d = (int)(i % quads) * 4;
        long long rest = i / quads;
        const int g = (int)(rest % groups);
        rest /= groups;
        const long long t = rest % seqlen, b = rest / seqlen;
        const float* p = part + ((b * seqlen + t) * heads + (long long)g * out.group) * dim + d;
        float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int j = 0; j < out.group; ++j, p += dim) {
            if (whole) {
                const float4 v = __ldcs(reinterpret_cast<const float4*>(p));
                x[0] += v.x, x[1] += v.y, x[2] += v.z, x[3] += v.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < dim) x[e] += p[e];
            }
        }
        T* o = static_cast<T*>(const_cast<void*>(out.p)) + b * out.sb + t * out.st + g * out.sh + d * out.sd;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < dim) o[e * out.sd] = Elem<DT>::from_float(x[e]);
    }
}

struct Shape {
    int q[4], k[4], v[4], o[4], s[4];
};
Shape shape_of(const vc1d_linear_args& a) {
    return {{a.batch, a.seqlen, a.heads, a.dim_k},
            {a.batch, a.seqlen, a.heads_k, a.dim_k},
            {a.batch, a.seqlen, a.heads_v, a.dim_v},
            {a.batch, a.seqlen, a.heads, a.dim_v},
            {a.batch, a.heads, a.dim_k, a.dim_v}};
}

int check(const vc1d_linear_args* a) {
    if (a == nullptr) return VC1D_E_NULL;
    if (a->struct_size != sizeof(vc1d_linear_args)) return VC1D_E_STRUCT;
    if (!is_io_dtype(a->dtype)) return VC1D_E_DTYPE;
    if (a->mask != nullptr && !is_mask_dtype(a->mask_dtype)) return VC1D_E_DTYPE;
    if (a->batch < 0 || a->seqlen < 0 || a->heads < 1 || a->heads_k < 1 || a->heads_v < 1 || a->dim_k < 1 || a->dim_v < 1)
        return VC1D_E_SHAPE;
    if (a->heads % a->heads_k != 0 || a->heads % a->heads_v != 0) return VC1D_E_SHAPE;
    if (a->kernel < VC1D_LINEAR_AUTO || a->kernel > VC1D_LINEAR_TC || a->segments < 0 || a->segments > kMaxSegments) return VC1D_E_SHAPE;
    if (a->dim_k > kMaxDim || a->dim_v > kMaxDim || a->seqlen > (1 << 30)) return VC1D_E_TOO_LARGE;
    if ((long long)a->batch * a->heads * (kMaxDim / 16) > 0x7fffffffLL) return VC1D_E_TOO_LARGE;
    if (a->seq_idx != nullptr && (a->mask != nullptr || a->initial_state != nullptr || a->final_state != nullptr)) return VC1D_E_SHAPE;
    return VC1D_OK;
}

// What every pass reads: the decays, the initial state, and with tokens q, k, v, the mask and the sequence numbers.
Touched inputs(const vc1d_linear_args& a) {
    const Shape n = shape_of(a);
    const int eb = elem_bytes(a.dtype), n_bt[2] = {a.batch, a.seqlen}, n_h[1] = {a.heads};
    const int64_t one[1] = {1};
    Touched t;
    t.reads_from(extent(a.log_decay, 4, n_h, one));
    if (a.initial_state != nullptr) t.reads_from(extent(a.initial_state, 4, n.s, a.initial_strides));
    if (a.seqlen == 0) return t;
    t.reads_from(extent(a.q, eb, n.q, a.q_strides));
    t.reads_from(extent(a.k, eb, n.k, a.k_strides));
    t.reads_from(extent(a.v, eb, n.v, a.v_strides));
    if (a.mask != nullptr) t.reads_from(extent(a.mask, elem_bytes(a.mask_dtype), n_bt, a.mask_strides));
    if (a.seq_idx != nullptr) t.reads_from(extent(a.seq_idx, 4, n_bt, a.seq_strides));
    return t;
}

int check_forward(const vc1d_linear_args* a) {
    const int st = check(a);
    if (st != VC1D_OK) return st;
    if (a->batch == 0) return VC1D_OK;
    if (a->log_decay == nullptr) return VC1D_E_NULL;
    const Shape n = shape_of(*a);
    Touched t = inputs(*a);
    if (a->seqlen > 0) {
        if (a->q == nullptr || a->k == nullptr || a->v == nullptr || a->out == nullptr) return VC1D_E_NULL;
        if (!writable(n.o, a->out_strides)) return VC1D_E_STRIDE;
        t.writes_to(extent(a->out, elem_bytes(a->dtype), n.o, a->out_strides));
    }
    if (a->final_state != nullptr) {
        if (!writable(n.s, a->final_strides)) return VC1D_E_STRIDE;
        t.writes_to(extent(a->final_state, 4, n.s, a->final_strides));
    }
    return t.clash() ? VC1D_E_ALIAS : VC1D_OK;
}

Rows rows(const void* p, const int64_t (&s)[4], int group) { return {p, s[0], s[1], s[2], s[3], group}; }
State state(const float* p, const int64_t (&s)[4], bool transposed) {
    return {const_cast<float*>(p), s[0], s[1], transposed ? s[3] : s[2], transposed ? s[2] : s[3]};
}
// the same rows from the last token to the first
Rows reversed(Rows r, int seqlen, int eb) {
    r.p = static_cast<const char*>(r.p) + (long long)(seqlen - 1) * r.st * eb;
    r.st = -r.st;
    return r;
}

Common common_of(const vc1d_linear_args& a) {
    Common c{};
    c.log_decay = a.log_decay;
    c.mask = a.mask;
    c.mask_dtype = a.mask_dtype;
    c.mask_sb = a.mask_strides[0];
    c.mask_st = a.mask_strides[1];
    c.seq_idx = a.seq_idx;
    c.seq_sb = a.seq_strides[0];
    c.seq_st = a.seq_strides[1];
    c.batch = a.batch;
    c.heads = a.heads;
    c.seqlen = a.seqlen;
    c.test_expire = a.test_expire;
    return c;
}

constexpr long long align16(long long n) { return (n + 15) & ~15LL; }

long long split_bytes(const Launch& l, int segments) {
    long long n = 0;
    if (segments > 1)
        for (int i = 0; i < l.runs; ++i)
            n += align16(4LL * (segments - 1) * l.c.batch * l.c.heads * l.run[i].da * l.run[i].dv) + align16(8LL * (segments - 1) * l.c.batch * l.c.heads);
    return n;
}

bool vector_rows(const Rows& r, int eb) {
    const int per = 16 / eb;
    return r.sd == 1 && r.sb % per == 0 && r.st % per == 0 && r.sh % per == 0 && (reinterpret_cast<uintptr_t>(r.p) & 15u) == 0;
}
bool mma_fits(const Launch& l, int dtype) {
    if (dtype == VC1D_F32) return false;
    for (int i = 0; i < l.runs; ++i) {
        const Run& r = l.run[i];
        if (r.da % 8 != 0 || r.dv % 8 != 0 || !vector_rows(r.a, 2) || !vector_rows(r.k, 2) || !vector_rows(r.v, 2)) return false;
    }
    return true;
}
// Tensor maps have no zero strides (broadcast inputs) and none of 2^40 bytes.
bool tma_fits(const Launch& l) {
    if (!tma_available()) return false;
    for (int i = 0; i < l.runs; ++i) {
        const Run& r = l.run[i];
        for (const Rows* x : {&r.a, &r.k, &r.v}) {
            const long long st = x->st < 0 ? -x->st : x->st, most = 1LL << 38;
            if ((l.c.seqlen > 1 && (st == 0 || st > most)) || (l.c.heads / x->group > 1 && (x->sh <= 0 || x->sh > most)) ||
                (l.c.batch > 1 && (x->sb <= 0 || x->sb > most)))
                return false;
            if ((x->st < 0) != (r.reverse != 0) && l.c.seqlen > 1) return false;
        }
    }
    return true;
}
Kind pick(const Launch& l, int dtype, int kernel) {
    if (l.c.seqlen == 0) return kSimt;  // copies the state; there is nothing to make tensor maps of
    if (kernel == VC1D_LINEAR_SIMT || !mma_fits(l, dtype)) return kSimt;
    return kernel != VC1D_LINEAR_MMA && dtype == VC1D_BF16 && largest_rows(l) <= 160 && tma_fits(l) ? kTc : kMma;
}

// whether the kernel that the caller names takes this launch
bool kernel_fits(const Launch& l, int dtype, int kernel) {
    return kernel == VC1D_LINEAR_AUTO || kernel == VC1D_LINEAR_SIMT || pick(l, dtype, kernel) == (kernel == VC1D_LINEAR_TC ? kTc : kMma);
}

// Parts of the time axis.
int plan_launch(const Launch& l, int dtype, int kernel, int wanted) {
    const Kind kind = pick(l, dtype, kernel);
    const int slab = slab_of(l, kind), chunks = (l.c.seqlen + chunk_of(kind) - 1) / chunk_of(kind);
    long long ctas = 0;
    for (int i = 0; i < l.runs; ++i) ctas += (long long)l.c.batch * l.c.heads * ((l.run[i].dv + slab - 1) / slab);
    int n = wanted;
    if (n == 0) {
        // Time in units of a chunk: waves of CTAs, each of them its chunks and a start-up of one and a half; a split adds
        // the pass over keys and values that finds the parts' states (0.4 of a chunk's work) and the join.  Against 15 other
        // counts from 1 to 64 the choice is the fastest or within 1 % of it for nine shapes of all kernels (1000 to 24567 tokens
        // on the tensor cores, 777 and 4000 in fp32), and 2 % behind for 65536 tokens of 16 heads of 128 (619 us, 605 with 4).
        const long long slots = (long long)ctas_per_sm(l, kind) * sm_count();
        double best = 0;
        for (int m = 1; m <= std::min(kMaxSegments, std::max(1, chunks)); ++m) {
            const double per = (chunks + m - 1) / m;
            double t = (double)((ctas * m + slots - 1) / slots) * (per + 1.5);
            if (m > 1) t += (double)((ctas * (m - 1) + slots - 1) / slots) * (0.4 * per + 1.5) + 1.5;
            if (m == 1 || t < best) best = t, n = m;
        }
    }
    n = std::max(1, std::min({n, kMaxSegments, chunks}));
    const int per = (chunks + n - 1) / n;
    return per > 0 ? std::max(1, (chunks + per - 1) / per) : 1;  // no part is empty
}

cudaError_t launch_one(const Launch& l, int dtype, Kind kind, bool states_only, cudaStream_t s) {
    if (kind == kSimt) return launch_linear_simt(l, dtype, states_only, s);
    if (kind == kTc) return launch_linear_tc(l, states_only, s);
    return dtype == VC1D_BF16 ? launch_linear_mma_bf16(l, states_only, s) : launch_linear_mma_f16(l, states_only, s);
}

// Enqueues the runs of `l`, split along time if the workspace allows it.
cudaError_t enqueue(Launch& l, int dtype, int kernel, int segments, char* ws, long long ws_bytes, cudaStream_t s) {
    Kind kind = pick(l, dtype, kernel);
    for (int i = 0; i < l.runs; ++i) l.run[i].out_vec = vector_rows(l.run[i].o, l.run[i].out_f32 ? 4 : elem_bytes(dtype));
    if (segments > 1 && (ws == nullptr || ws_bytes < split_bytes(l, segments))) segments = 1;
    const int chunks = (l.c.seqlen + chunk_of(kind) - 1) / chunk_of(kind);
    l.c.segments = segments;
    l.c.seg_chunks = std::max(1, (chunks + segments - 1) / segments);
    if (segments > 1) {
        for (int i = 0; i < l.runs; ++i) {
            const long long bh = (long long)l.c.batch * l.c.heads;
            l.c.seg_state[i] = reinterpret_cast<float*>(ws);
            ws += align16(4LL * (segments - 1) * bh * l.run[i].da * l.run[i].dv);
            l.c.seg_factor[i] = reinterpret_cast<float2*>(ws);
            ws += align16(8LL * (segments - 1) * bh);
        }
        cudaError_t e = launch_one(l, dtype, kind, true, s);
        if (e != cudaSuccess) return e;
        long long most = 0;
        for (int i = 0; i < l.runs; ++i) most = std::max(most, (long long)l.c.batch * l.c.heads * l.run[i].da * l.run[i].dv);
        const dim3 grid((unsigned)std::min<long long>((most + 255) / 256, 16LL * sm_count()), l.runs);
        note_launch("linear_join");
        k_linear_join<<<grid, 256, 0, s>>>(l);
        e = cudaGetLastError();
        if (e != cudaSuccess) return e;
    }
    const bool packed = l.c.seq_idx != nullptr && l.c.seqlen > 0;
    if (packed) note_launch("linear_isolate");  // counted here: the name that stays is the main kernel's
    cudaError_t e = launch_one(l, dtype, kind, false, s);
    return e == cudaSuccess && packed ? launch_linear_isolate(l, dtype, s) : e;
}

Launch forward_launch(const vc1d_linear_args& a) {
    Launch l{};
    l.c = common_of(a);
    l.runs = 1;
    Run& r = l.run[0];
    r.a = rows(a.q, a.q_strides, 1);
    r.k = rows(a.k, a.k_strides, a.heads / a.heads_k);
    r.v = rows(a.v, a.v_strides, a.heads / a.heads_v);
    r.o = rows(a.out, a.out_strides, 1);
    r.x0 = state(a.initial_state, a.initial_strides, false);
    r.xT = state(a.final_state, a.final_strides, false);
    r.da = a.dim_k;
    r.dv = a.dim_v;
    r.s_pair = r.s_carry = a.scale;
    r.s_add = 1.f;
    return l;
}

int check_backward(const vc1d_linear_bwd_args* a) {
    if (a == nullptr) return VC1D_E_NULL;
    if (a->struct_size != sizeof(vc1d_linear_bwd_args)) return VC1D_E_STRUCT;
    vc1d_linear_args f = a->f;
    f.final_state = nullptr;
    const int st = check(&f);
    if (st != VC1D_OK) return st;
    if (a->segments < 0 || a->segments > kMaxSegments) return VC1D_E_SHAPE;
    if (f.seq_idx != nullptr && (a->dfinal != nullptr || a->dinitial != nullptr)) return VC1D_E_SHAPE;
    if (f.batch == 0) return VC1D_OK;
    if (f.log_decay == nullptr) return VC1D_E_NULL;
    const Shape n = shape_of(f);
    const int eb = elem_bytes(f.dtype);
    Touched t = inputs(f);
    if (a->dfinal != nullptr) t.reads_from(extent(a->dfinal, 4, n.s, a->dfinal_strides));
    if (f.seqlen > 0) {
        if (f.q == nullptr || f.k == nullptr || f.v == nullptr || a->dout == nullptr || a->dq == nullptr || a->dk == nullptr || a->dv == nullptr)
            return VC1D_E_NULL;
        if (!writable(n.q, a->dq_strides) || !writable(n.k, a->dk_strides) || !writable(n.v, a->dv_strides)) return VC1D_E_STRIDE;
        t.reads_from(extent(a->dout, eb, n.o, a->dout_strides));
        t.writes_to(extent(a->dq, eb, n.q, a->dq_strides));
        t.writes_to(extent(a->dk, eb, n.k, a->dk_strides));
        t.writes_to(extent(a->dv, eb, n.v, a->dv_strides));
    }
    if (a->dinitial != nullptr) {
        if (!writable(n.s, a->dinitial_strides)) return VC1D_E_STRIDE;
        t.writes_to(extent(a->dinitial, 4, n.s, a->dinitial_strides));
    }
    return t.clash() ? VC1D_E_ALIAS : VC1D_OK;
}

// dq: tokens in order.  Then dk and dv: tokens from the last to the first.
void backward_launches(const vc1d_linear_bwd_args& a, Launch* fwd, Launch* rev, float* part_k, float* part_v) {
    const vc1d_linear_args& f = a.f;
    const int eb = elem_bytes(f.dtype), T = f.seqlen, gk = f.heads / f.heads_k, gv = f.heads / f.heads_v;
    const Rows q = rows(f.q, f.q_strides, 1), k = rows(f.k, f.k_strides, gk), v = rows(f.v, f.v_strides, gv),
               g = rows(a.dout, a.dout_strides, 1);
    *fwd = Launch{};
    fwd->c = common_of(f);
    fwd->runs = 1;
    Run& dq = fwd->run[0];
    dq.a = g;
    dq.k = v;
    dq.v = k;
    dq.o = rows(a.dq, a.dq_strides, 1);
    dq.x0 = state(f.initial_state, f.initial_strides, true);
    dq.da = f.dim_v;
    dq.dv = f.dim_k;
    dq.s_pair = dq.s_carry = f.scale;
    dq.s_add = 1.f;

    *rev = Launch{};
    rev->c = common_of(f);
    rev->runs = 2;
    Run& dk = rev->run[0];
    Run& dv = rev->run[1];
    dk.a = reversed(v, T, eb);
    dk.k = reversed(g, T, eb);
    dk.v = reversed(q, T, eb);
    dk.da = f.dim_v;
    dk.dv = f.dim_k;
    dk.x0 = state(a.dfinal, a.dfinal_strides, true);
    dv.a = reversed(k, T, eb);
    dv.k = reversed(q, T, eb);
    dv.v = reversed(g, T, eb);
    dv.da = f.dim_k;
    dv.dv = f.dim_v;
    dv.x0 = state(a.dfinal, a.dfinal_strides, false);
    dv.xT = state(a.dinitial, a.dinitial_strides, false);
    const int64_t pk[4] = {(int64_t)T * f.heads * f.dim_k, (int64_t)f.heads * f.dim_k, f.dim_k, 1};
    const int64_t pv[4] = {(int64_t)T * f.heads * f.dim_v, (int64_t)f.heads * f.dim_v, f.dim_v, 1};
    dk.out_f32 = gk > 1;
    dv.out_f32 = gv > 1;
    dk.o = gk > 1 ? reversed(rows(part_k, pk, 1), T, 4) : reversed(rows(a.dk, a.dk_strides, 1), T, eb);
    dv.o = gv > 1 ? reversed(rows(part_v, pv, 1), T, 4) : reversed(rows(a.dv, a.dv_strides, 1), T, eb);
    for (Run* r : {&dk, &dv}) {
        r->reverse = r->shift = 1;
        r->s_pair = r->s_add = f.scale;  // the state holds scaled sums, so that the final state's gradient enters as it is
        r->s_carry = 1.f;
    }
}

long long part_bytes(const vc1d_linear_args& f, int heads_x, int dim) {
    return heads_x == f.heads ? 0 : align16(4LL * f.batch * f.seqlen * f.heads * dim);
}

cudaError_t sum_heads(int dtype, const float* part, const Rows& out, const vc1d_linear_args& f, int dim, cudaStream_t s) {
    const long long n = (long long)f.batch * f.seqlen * (f.heads / out.group) * ((dim + 3) / 4);
    const int grid = (int)std::min<long long>((n + 255) / 256, 32LL * sm_count());
    note_launch("linear_sum_heads");
    switch (dtype) {
        case VC1D_F32: k_linear_sum_heads<VC1D_F32><<<grid, 256, 0, s>>>(part, out, f.heads, f.seqlen, dim, n); break;
        case VC1D_BF16: k_linear_sum_heads<VC1D_BF16><<<grid, 256, 0, s>>>(part, out, f.heads, f.seqlen, dim, n); break;
        default: k_linear_sum_heads<VC1D_F16><<<grid, 256, 0, s>>>(part, out, f.heads, f.seqlen, dim, n); break;
    }
    return cudaGetLastError();
}

}  // namespace
}  // namespace lin
}  // namespace vc1d

extern "C" {

VC1D_API int vc1d_linear(const vc1d_linear_args* a, void* stream) {
    using namespace vc1d;
    const int st = lin::check_forward(a);
    if (st != VC1D_OK || a->batch == 0) return st;
    if (a->seqlen == 0 && a->final_state == nullptr) return VC1D_OK;
    if ((reinterpret_cast<uintptr_t>(a->workspace) & 15u) != 0) return VC1D_E_STRIDE;
    lin::Launch l = lin::forward_launch(*a);
    if (a->seqlen > 0 && !lin::kernel_fits(l, a->dtype, a->kernel)) return VC1D_E_STRIDE;
    return (int)lin::enqueue(l, a->dtype, a->kernel, lin::plan_launch(l, a->dtype, a->kernel, a->segments), static_cast<char*>(a->workspace), a->workspace_bytes,
                             static_cast<cudaStream_t>(stream));
}

VC1D_API int64_t vc1d_linear_workspace(const vc1d_linear_args* a) {
    using namespace vc1d;
    const int st = lin::check(a);
    if (st != VC1D_OK) return st;
    if (a->batch == 0 || a->seqlen == 0) return 0;
    const lin::Launch l = lin::forward_launch(*a);
    return lin::split_bytes(l, lin::plan_launch(l, a->dtype, a->kernel, a->segments));
}

VC1D_API int vc1d_linear_bwd(const vc1d_linear_bwd_args* a, void* stream) {
    using namespace vc1d;
    const int st = lin::check_backward(a);
    if (st != VC1D_OK || a->f.batch == 0) return st;
    if (a->f.seqlen == 0 && a->dinitial == nullptr) return VC1D_OK;
    if ((reinterpret_cast<uintptr_t>(a->workspace) & 15u) != 0) return VC1D_E_STRIDE;
    const vc1d_linear_args& f = a->f;
    const long long bk = lin::part_bytes(f, f.heads_k, f.dim_k), bv = lin::part_bytes(f, f.heads_v, f.dim_v);
    if (bk + bv > 0 && (a->workspace == nullptr || a->workspace_bytes < bk + bv)) return VC1D_E_NULL;
    char* ws = static_cast<char*>(a->workspace);
    float *part_k = reinterpret_cast<float*>(ws), *part_v = reinterpret_cast<float*>(ws + bk);
    char* split = ws == nullptr ? nullptr : ws + bk + bv;
    const long long left = a->workspace_bytes - bk - bv;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    lin::Launch fwd, rev;
    lin::backward_launches(*a, &fwd, &rev, part_k, part_v);
    if (f.seqlen > 0 && !(lin::kernel_fits(fwd, f.dtype, f.kernel) && lin::kernel_fits(rev, f.dtype, f.kernel))) return VC1D_E_STRIDE;
    cudaError_t e = cudaSuccess;
    // the two launches follow each other on the stream, so they use the same workspace
    if (f.seqlen > 0) e = lin::enqueue(fwd, f.dtype, f.kernel, lin::plan_launch(fwd, f.dtype, f.kernel, a->segments), split, left, s);
    if (e == cudaSuccess) e = lin::enqueue(rev, f.dtype, f.kernel, lin::plan_launch(rev, f.dtype, f.kernel, a->segments), split, left, s);
    if (e == cudaSuccess && bk > 0)
        e = lin::sum_heads(f.dtype, part_k, lin::rows(a->dk, a->dk_strides, f.heads / f.heads_k), f, f.dim_k, s);
    if (e == cudaSuccess && bv > 0)
        e = lin::sum_heads(f.dtype, part_v, lin::rows(a->dv, a->dv_strides, f.heads / f.heads_v), f, f.dim_v, s);
    return (int)e;
}

VC1D_API int64_t vc1d_linear_bwd_workspace(const vc1d_linear_bwd_args* a) {
    using namespace vc1d;
    if (a == nullptr) return VC1D_E_NULL;
    if (a->struct_size != sizeof(vc1d_linear_bwd_args)) return VC1D_E_STRUCT;
    vc1d_linear_args f = a->f;
    f.final_state = nullptr;
    const int st = lin::check(&f);
    if (st != VC1D_OK) return st;
    if (f.batch == 0 || f.seqlen == 0) return 0;
    lin::Launch fwd, rev;
    lin::backward_launches(*a, &fwd, &rev, nullptr, nullptr);
    return lin::part_bytes(f, f.heads_k, f.dim_k) + lin::part_bytes(f, f.heads_v, f.dim_v) +
           std::max(lin::split_bytes(fwd, lin::plan_launch(fwd, f.dtype, f.kernel, a->segments)), lin::split_bytes(rev, lin::plan_launch(rev, f.dtype, f.kernel, a->segments)));
}

VC1D_API uint32_t vc1d_sizeof_linear_args(void) { return (uint32_t)sizeof(vc1d_linear_args); }
VC1D_API uint32_t vc1d_sizeof_linear_bwd_args(void) { return (uint32_t)sizeof(vc1d_linear_bwd_args); }

}  // extern "C"
