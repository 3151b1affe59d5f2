// Linear attention on the fp32 pipes: any strides, every type, head dimensions up to 256.  Takes fp32 tensors and the
// layouts that the tensor-core kernel cannot load.
//
// One CTA of 256 threads owns one (row, head, slab of 64 state columns, part of the time axis) and walks its chunks of
// 64 tokens.  q, k, v (converted to fp32), the state slab and the 64 x 64 products sit in shared memory; every product
// is a register tile of 4 x 4 outputs per thread, fed by 128-bit shared loads (8 of them per 64 multiply-adds).
//
// Bound by those shared loads and by latency: a forward and backward pass over 3 x 777 tokens of 6 heads of 72 and 88 takes
// 410 us in fp32, where memory would allow 2.5: 18 (row, head) pairs and two slabs for 148 SMs, so that the time axis is split
// and every part computed twice over, once for its state.
#include "linear_attention.cuh"

namespace vc1d {
namespace lin {
namespace {

constexpr int kThreads = 256;
constexpr int kSlab = 64;  // state columns of a CTA

__device__ __forceinline__ float4 ld4(const float* p) { return *reinterpret_cast<const float4*>(p); }

__device__ __forceinline__ void tile_fma(float (&acc)[4][4], const float4 (&a)[4], const float4 (&b)[4]) {
    // acc[i][j] += a_i . (b_0..3)[j]: four steps of the summed index at once, b rows are steps
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x[4] = {a[i].x, a[i].y, a[i].z, a[i].w};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            acc[i][0] = fmaf(x[s], b[s].x, acc[i][0]);
            acc[i][1] = fmaf(x[s], b[s].y, acc[i][1]);
            acc[i][2] = fmaf(x[s], b[s].z, acc[i][2]);
            acc[i][3] = fmaf(x[s], b[s].w, acc[i][3]);
        }
    }
}

template <int DT, bool STATES>
__global__ void __launch_bounds__(kThreads, 2) k_linear_simt(const __grid_constant__ Launch l) {
    using E = Elem<DT>;
    using T = typename E::type;
    extern __shared__ __align__(16) float sm[];
    __shared__ ChunkInfo info;
    __shared__ float2 pw[kPowers];
    __shared__ float add[kChunk];

    const Run& r = l.run[blockIdx.z];
    const Common& c = l.c;
    const int slabs = (r.dv + kSlab - 1) / kSlab;
    const int seg = blockIdx.y;
    const int slab = blockIdx.x % slabs;
    const int bh = blockIdx.x / slabs;
    if (bh >= c.batch * c.heads) return;  // a run with fewer slabs than the launch's widest
    const int b = bh / c.heads, h = bh % c.heads;
    const int tid = threadIdx.x;
    const int dap = (r.da + 3) & ~3;  // rows padded with zeros to a multiple of four
    const int rs = dap + 4;           // row stride of a and k: 16-byte rows on different banks
    const int c0 = slab * kSlab;
    const int cols = min(kSlab, r.dv - c0);

    float* sa = sm;                    // [64][rs]
    float* sp = sa;                    // [64][64 + 4] products of a and k, once a is no longer read
    float* sk = sa + kChunk * max(rs, kChunk + 4);  // [64][rs]
    float* sv = sk + kChunk * rs;      // [64][64]
    float* sx = sv + kChunk * kSlab;   // [dap][64] state

    fill_powers(pw, c.log_decay[h], tid, kThreads);
    {
        const bool from_seg = !STATES && seg > 0;
        for (int i = tid; i < dap * kSlab; i += kThreads) {
            const int row = i / kSlab, col = i % kSlab;
            float x = 0.f;
            if (row < r.da && col < cols) {
                if (from_seg)
                    x = c.seg_state[blockIdx.z][((long long)(seg - 1) * c.batch * c.heads + bh) * ((long long)r.da * r.dv) +
                                                (long long)row * r.dv + c0 + col];
                else if (!STATES && r.x0.p != nullptr)
                    x = r.x0.p[(long long)b * r.x0.sb + (long long)h * r.x0.sh + (long long)row * r.x0.sr +
                               (long long)(c0 + col) * r.x0.sc];
            }
            sx[i] = x;
        }
    }
    const int t_begin = seg * c.seg_chunks * kChunk;
    const int t_end = min(c.seqlen, t_begin + c.seg_chunks * kChunk);
    const T* pa = static_cast<const T*>(r.a.p) + (long long)b * r.a.sb + (long long)(h / r.a.group) * r.a.sh;
    const T* pk = static_cast<const T*>(r.k.p) + (long long)b * r.k.sb + (long long)(h / r.k.group) * r.k.sh;
    const T* pv = static_cast<const T*>(r.v.p) + (long long)b * r.v.sb + (long long)(h / r.v.group) * r.v.sh;

    auto wide_rows = [&](const T* p, const Rows& x, int channels) {
        return DT == VC1D_F32 && x.sd == 1 && channels % 4 == 0 && x.st % 4 == 0 && (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
    };
    const bool wide_a = wide_rows(pa, r.a, r.da), wide_k = wide_rows(pk, r.k, r.da), wide_v = wide_rows(pv + (long long)c0 * r.v.sd, r.v, cols);

    const int ti = (tid / 16) * 4, tj = (tid % 16) * 4;  // this thread's 4 x 4 tile of a 64 x 64 product
    double seg_factor = 1.0;

    for (int t0 = t_begin; t0 < t_end; t0 += kChunk) {
        __syncthreads();  // the tiles of the chunk before are no longer read
        if (tid < 32) chunk_info(c, r.reverse, b, t0, t_end, &info);
        __syncthreads();
        // a warp per row: rows of masked tokens and channels past the head's end become zeros, unread
        auto fetch = [&](const T* src, long long st, long long sd, int channels, int padded, float* dst, int stride, bool wide) {
#pragma unroll 2
            for (int row = tid >> 5; row < kChunk; row += kThreads / 32) {
                const bool ok = info.valid[row >> 5] >> (row & 31) & 1u;
                const T* p = src + (long long)(t0 + row) * st;
                if (wide) {  // fp32, channel stride 1, 16-byte aligned rows
                    for (int d = (tid & 31) * 4; d < padded; d += 128) {
                        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (ok && d < channels) x = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + d));
                        *reinterpret_cast<float4*>(dst + row * stride + d) = x;
                    }
                } else {
                    for (int d = tid & 31; d < padded; d += 32) dst[row * stride + d] = ok && d < channels ? E::to_float(p[d * sd]) : 0.f;
                }
            }
        };
        if (!STATES) fetch(pa, r.a.st, r.a.sd, r.da, dap, sa, rs, wide_a);
        fetch(pk, r.k.st, r.k.sd, r.da, dap, sk, rs, wide_k);
        fetch(pv + (long long)c0 * r.v.sd, r.v.st, r.v.sd, cols, kSlab, sv, kSlab, wide_v);
        if (tid < kChunk) {  // what a token's key weighs in the state after the chunk
            const int code = info.code[tid];
            add[tid] = (code >> 16) == info.run_all ? pw[info.n_all - (code & 0xffff) + r.shift].x * r.s_add : 0.f;
        }
        __syncthreads();
        const int n_all = info.n_all, run_all = info.run_all;
        if (!STATES) {
            float acc[4][4] = {};
            if (tj <= ti + 3) {  // tiles above the diagonal hold only later tokens
                for (int d = 0; d < dap; d += 4) {
                    float4 x[4], y[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[i] = ld4(sa + (ti + i) * rs + d);
                        y[i] = ld4(sk + (tj + i) * rs + d);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            acc[i][j] = fmaf(x[i].x, y[j].x, fmaf(x[i].y, y[j].y, fmaf(x[i].z, y[j].z, fmaf(x[i].w, y[j].w, acc[i][j]))));
                }
            }
            // a X, then the row's power of the decay, then the products inside the chunk
            float out[4][4] = {};
            for (int d = 0; d < dap; d += 4) {
                float4 x[4], y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = ld4(sa + (ti + i) * rs + d);
                    y[i] = ld4(sx + (d + i) * kSlab + tj);
                }
                tile_fma(out, x, y);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int code = info.code[ti + i];
                const float f = (code >> 16) == 0 ? pw[max(code - r.shift, 0)].x * r.s_carry : 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) out[i][j] = (code >> 16) == 0 ? out[i][j] * f : 0.f;
            }
            __syncthreads();  // a has been read by all
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float4 p;
                float* pp = &p.x;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned lag = (unsigned)(info.code[ti + i] - info.code[tj + j]);
                    pp[j] = lag <= (unsigned)kChunk ? acc[i][j] * (pw[lag].x * r.s_pair) : 0.f;
                }
                *reinterpret_cast<float4*>(sp + (ti + i) * (kChunk + 4) + tj) = p;
            }
            __syncthreads();
            for (int j = 0; j < ti + 4; j += 4) {
                float4 x[4], y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = ld4(sp + (ti + i) * (kChunk + 4) + j);
                    y[i] = ld4(sv + (j + i) * kSlab + tj);
                }
                tile_fma(out, x, y);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = t0 + ti + i;
                if (t >= t_end) continue;
                const bool ok = info.valid[(ti + i) >> 5] >> ((ti + i) & 31) & 1u;
                const long long base = (long long)b * r.o.sb + (long long)t * r.o.st + (long long)h * r.o.sh;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (tj + j >= cols) continue;
                    const long long at = base + (long long)(c0 + tj + j) * r.o.sd;
                    if (r.out_f32)
                        const_cast<float*>(static_cast<const float*>(r.o.p))[at] = ok ? out[i][j] : 0.f;
                    else
                        const_cast<T*>(static_cast<const T*>(r.o.p))[at] = E::from_float(ok ? out[i][j] : 0.f);
                }
            }
        }
        // the state: X' = a^{n_C} X + sum_j w_j k_j v_j^T
        __syncthreads();  // the queries have read it
        const float2 f = pw[n_all];
        // without a token the state stays, whatever it holds: not even times 1 + 0
        for (int i0 = n_all == 0 ? dap : tid / 16 * 4; i0 < dap; i0 += kThreads / 16 * 4) {
            float acc[4][4] = {};
#pragma unroll 4
            for (int j = 0; j < kChunk; ++j) {
                const float4 x = ld4(sk + j * rs + i0), y = ld4(sv + j * kSlab + tj);
                const float w = add[j];
                const float xs[4] = {x.x * w, x.y * w, x.z * w, x.w * w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    acc[i][0] = fmaf(xs[i], y.x, acc[i][0]);
                    acc[i][1] = fmaf(xs[i], y.y, acc[i][1]);
                    acc[i][2] = fmaf(xs[i], y.z, acc[i][2]);
                    acc[i][3] = fmaf(xs[i], y.w, acc[i][3]);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float* px = sx + (i0 + i) * kSlab + tj;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    px[j] = run_all == 0 ? fmaf(px[j], f.x, fmaf(px[j], f.y, acc[i][j])) : acc[i][j];
            }
        }
        if (STATES) seg_factor = run_all == 0 ? seg_factor * ((double)f.x + (double)f.y) : 0.0;
    }
    __syncthreads();
    if (STATES) {
        float* dst = c.seg_state[blockIdx.z] + ((long long)seg * c.batch * c.heads + bh) * ((long long)r.da * r.dv);
        for (int i = tid; i < r.da * kSlab; i += kThreads) {
            const int row = i / kSlab, col = i % kSlab;
            if (col < cols) dst[(long long)row * r.dv + c0 + col] = sx[row * kSlab + col];
        }
        if (slab == 0 && tid == 0) {
            const float hi = (float)seg_factor;
            c.seg_factor[blockIdx.z][(long long)seg * c.batch * c.heads + bh] = make_float2(hi, (float)(seg_factor - (double)hi));
        }
    } else if (seg == c.segments - 1 && r.xT.p != nullptr) {
        for (int i = tid; i < r.da * kSlab; i += kThreads) {
            const int row = i / kSlab, col = i % kSlab;
            if (col < cols)
                r.xT.p[(long long)b * r.xT.sb + (long long)h * r.xT.sh + (long long)row * r.xT.sr + (long long)(c0 + col) * r.xT.sc] =
                    sx[row * kSlab + col];
        }
    }
}

// Dynamic shared memory of a CTA whose state has `da` rows (a multiple of four).
constexpr int shared_bytes(int da) {
    return 4 * (kChunk * ((da > kChunk ? da : kChunk) + 4) + kChunk * (da + 4) + kChunk * kSlab + da * kSlab);
}
static_assert(shared_bytes(kMaxDim) + 4096 <= 232448, "shared memory of a CTA");

template <int DT, bool STATES>
cudaError_t launch(const Launch& l, cudaStream_t s) {
    int da = 0, slabs = 0;
    for (int i = 0; i < l.runs; ++i) {
        da = max(da, (l.run[i].da + 3) & ~3);
        slabs = max(slabs, (l.run[i].dv + kSlab - 1) / kSlab);
    }
    const int smem = shared_bytes(da);
    const long long blocks = (long long)l.c.batch * l.c.heads * slabs;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    // The limit belongs to the function, not to the host thread: always that of the largest heads, or a call with small ones
    // would lower it between another thread's call and its launch.
    cudaError_t e = cudaFuncSetAttribute(k_linear_simt<DT, STATES>, cudaFuncAttributeMaxDynamicSharedMemorySize, shared_bytes(kMaxDim));
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned)blocks, STATES ? l.c.segments - 1 : l.c.segments, l.runs);
    note_launch(STATES ? "linear_simt_states" : "linear_simt");
    k_linear_simt<DT, STATES><<<grid, kThreads, smem, s>>>(l);
    return cudaGetLastError();
}

template <bool STATES>
cudaError_t launch_dt(const Launch& l, int dtype, cudaStream_t s) {
    switch (dtype) {
        case VC1D_F32: return launch<VC1D_F32, STATES>(l, s);
        case VC1D_BF16: return launch<VC1D_BF16, STATES>(l, s);
        default: return launch<VC1D_F16, STATES>(l, s);
    }
}

}  // namespace
}  // namespace lin

cudaError_t launch_linear_simt(const lin::Launch& l, int dtype, bool states_only, cudaStream_t s) {
    return states_only ? lin::launch_dt<true>(l, dtype, s) : lin::launch_dt<false>(l, dtype, s);
}

}  // namespace vc1d
