// gx_norm.cu — the norms around a block, with its gate and residual scale:
//
//   before:  h = x / sqrt(mean(x^2) + eps) * w,                      gate = gate_w . h
//   after:   v = y / sqrt(mean(y^2) + eps) * post   (or y itself)
//            r = res_scale * res + block_scale * gate * v            gate: 1, sigmoid per token or per element
//            res_out = r,  out = r / sqrt(mean(r^2) + eps) * next,   next_gate = next_gate_w . out
//
// Bound by reading and writing every row once. A group of G threads takes a row and holds it in
// registers from the first read to the last write, 8 values in each of up to VPT vectors a thread; the
// weights come through L1, which the streamed rows do not pass (16 CTAs and more on an SM share them).
// Sums meet by shuffles, and across warps once in shared memory.
//
// Measured: 16384 rows of 4096 (bf16 in and out) 42 us, 98 % of the copy bandwidth; 4067 rows of 2048
// with a gate per element, the residual and the next norm 27 us, 85 %; one row of 2048 the cost of a launch.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>


#include "../../include/gyro_moe.h"
#include "gx_dense.cuh"
#include "gx_device.cuh"
#include "gx_internal.h"

namespace gx {

using namespace dense;

namespace {

constexpr int kNormThreads = 256;    // of the long-row kernels
constexpr int kNormRowMax = 16384;   // longest row held in registers: 512 threads of 4 vectors

__device__ __forceinline__ void store_act(void *p, int bf16, size_t i, float v) {
    if (bf16) reinterpret_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
    else reinterpret_cast<float *>(p)[i] = v;
}

// 1 / (1 + e^-x) in 10 instructions (expf and a division take four times as many, which bounds the kernel that
// gates every element): 2^t with the rounding of t = -x log2 e put back, off by at most 8 units of 2^-24 (4 of the
// power of two, 2 of the reciprocal, 1 of each sum). From -88 down, where 2^t would pass the f32 range and its
// correction with it, x counts as -88: the reciprocal of 2^126.96 is below the smallest normal number, and 0. From
// 10^4 up (and at Inf, whose remainder would be a NaN) it is 1. A NaN stays one.
__device__ __forceinline__ float sigmoid(float x) {
    constexpr float l2e = 1.44269504088896341f, l2e_rest = (float)(1.44269504088896341 - (double)1.44269504088896341f);
    asm("min.NaN.f32 %0, %0, 0f461c4000;\n max.NaN.f32 %0, %0, 0fc2b00000;" : "+f"(x));  // 10^4, -88
    const float t = -x * l2e, rest = fmaf(-x, l2e_rest, fmaf(-x, l2e, -t));
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    e = fmaf(e, rest * 0.693147180559945309f, e);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return r;
}

__device__ __forceinline__ float block_sum(float v, float *red) {
    v = warp_sum(v);
    __syncthreads();  // red may still be read from the sum before
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kNormThreads / 32; ++w) t += red[w];
    return t;
}

// ---- rows too long for registers: read again for each step -----------------------------------------
__global__ void __launch_bounds__(kNormThreads) norm_long_kernel(NormArgs a) {
    __shared__ float red[kNormThreads / 32];
    pdl_launch_dependents();
    pdl_wait();
    const size_t t = blockIdx.x;
    float ss = 0.f;
    for (int i = threadIdx.x; i < a.E; i += kNormThreads) {
        const float v = load_act(a.x, a.x_bf16, t * a.ldx + i);
        ss = fmaf(v, v, ss);
    }
    const float scale = 1.0f / sqrtf(block_sum(ss, red) / (float)a.E + a.eps);
    float g = 0.f;
    for (int i = threadIdx.x; i < a.E; i += kNormThreads) {
        const float h = load_act(a.x, a.x_bf16, t * a.ldx + i) * scale * (a.w ? a.w[i] : 1.f);
        store_act(a.y, a.y_bf16, t * a.ldy + i, h);
        if (a.gate_w) g = fmaf(a.gate_w[i], h, g);
    }
    if (a.gate_w) {
        g = block_sum(g, red);
        if (threadIdx.x == 0) a.gate[t] = g;
    }
}

__device__ __forceinline__ float residual_value(const ResidualArgs &a, size_t t, int i, float yscale, float tgate) {
    float v = load_act(a.y, a.y_bf16, t * a.ldy + i) * yscale;
    if (a.post) v *= a.post[i];
    if (a.gate_kind == GX_GATE_ELEMENT) v *= sigmoid(load_act(a.gate, a.gate_bf16, t * a.ldg + i));
    return a.res_scale * load_act(a.res, a.res_bf16, t * a.ldr + i) + a.block_scale * tgate * v;
}

__global__ void __launch_bounds__(kNormThreads) residual_long_kernel(ResidualArgs a) {
    __shared__ float red[kNormThreads / 32];
    pdl_launch_dependents();
    pdl_wait();
    const size_t t = blockIdx.x;
    float yscale = 1.f;
    if (a.post_norm) {
        float ss = 0.f;
        for (int i = threadIdx.x; i < a.E; i += kNormThreads) {
            const float v = load_act(a.y, a.y_bf16, t * a.ldy + i);
            ss = fmaf(v, v, ss);
        }
        yscale = 1.0f / sqrtf(block_sum(ss, red) / (float)a.E + a.eps);
    }
    const float tgate = a.gate_kind == GX_GATE_TOKEN ? sigmoid(reinterpret_cast<const float *>(a.gate)[t]) : 1.f;
    // The sum of squares first: res_out may be res, so r is computed again before it is stored.
    float ss = 0.f;
    if (a.out)
        for (int i = threadIdx.x; i < a.E; i += kNormThreads) {
            const float r = residual_value(a, t, i, yscale, tgate);
            ss = fmaf(r, r, ss);
        }
    const float rscale = a.out ? 1.0f / sqrtf(block_sum(ss, red) / (float)a.E + a.next_eps) : 0.f;
    float g = 0.f;
    for (int i = threadIdx.x; i < a.E; i += kNormThreads) {
        const float r = residual_value(a, t, i, yscale, tgate);
        store_act(a.res_out, a.res_bf16, t * a.ldro + i, r);
        if (a.out) {
            const float h = r * rscale * (a.next ? a.next[i] : 1.f);
            store_act(a.out, a.out_bf16, t * a.ldo + i, h);
            if (a.next_gate_w) g = fmaf(a.next_gate_w[i], h, g);
        }
    }
    if (a.out && a.next_gate_w) {
        g = block_sum(g, red);
        if (threadIdx.x == 0) a.next_gate[t] = g;
    }
}

// ---- rows held in registers --------------------------------------------------------------------
// Thread l of a row's G has the elements (k G + l) 8 + j (VEC: 16-byte accesses; the width is a
// multiple of 8 and every row aligned) or (8 k + j) G + l. (Kernels for each combination of
// encodings were no faster.)
template <int VPT, bool VEC>
struct Row {
    int G, l, E;
    __device__ __forceinline__ int at(int k, int j) const { return VEC ? (k * G + l) * 8 + j : (8 * k + j) * G + l; }
    __device__ __forceinline__ void load(const void *p, int bf16, size_t base, float (&v)[VPT][8]) const {
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[k][j] = 0.f;
            if constexpr (VEC) {
                const int i = at(k, 0);
                if (i >= E) continue;
                if (bf16) {
                    const uint4 q = __ldcs(reinterpret_cast<const uint4 *>(reinterpret_cast<const __nv_bfloat16 *>(p) + base + i));
                    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        v[k][2 * j] = __uint_as_float(w[j] << 16);
                        v[k][2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
                    }
                } else {
                    const float4 *f = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p) + base + i);
                    const float4 a = __ldcs(f), b = __ldcs(f + 1);
                    v[k][0] = a.x; v[k][1] = a.y; v[k][2] = a.z; v[k][3] = a.w;
                    v[k][4] = b.x; v[k][5] = b.y; v[k][6] = b.z; v[k][7] = b.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (at(k, j) < E) v[k][j] = load_act(p, bf16, base + at(k, j));
            }
        }
    }
    __device__ __forceinline__ void store(void *p, int bf16, size_t base, const float (&v)[VPT][8]) const {
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            if constexpr (VEC) {
                const int i = at(k, 0);
                if (i >= E) continue;
                if (bf16) {
                    uint32_t w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const __nv_bfloat162 h = __floats2bfloat162_rn(v[k][2 * j], v[k][2 * j + 1]);
                        w[j] = *reinterpret_cast<const uint32_t *>(&h);
                    }
                    *reinterpret_cast<uint4 *>(reinterpret_cast<__nv_bfloat16 *>(p) + base + i) = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
                    float4 *f = reinterpret_cast<float4 *>(reinterpret_cast<float *>(p) + base + i);
                    f[0] = make_float4(v[k][0], v[k][1], v[k][2], v[k][3]);
                    f[1] = make_float4(v[k][4], v[k][5], v[k][6], v[k][7]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (at(k, j) < E) store_act(p, bf16, base + at(k, j), v[k][j]);
            }
        }
    }
    // weights of vector k (1 where there are none)
    __device__ __forceinline__ void weights(const float *w, int k, float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 1.f;
        if (!w) return;
        if constexpr (VEC) {
            const int i = at(k, 0);
            if (i >= E) return;
            const float4 a = __ldg(reinterpret_cast<const float4 *>(w + i)), b = __ldg(reinterpret_cast<const float4 *>(w + i) + 1);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (at(k, j) < E) v[j] = __ldg(w + at(k, j));
        }
    }
};

// Sum over a row's threads; red: a place of its own for each sum of a kernel.
__device__ __forceinline__ float row_sum(float v, int G, float *red) {
    v = warp_sum(v);
    if (G == 32) return v;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.f;
    for (int w = 0; w < G / 32; ++w) t += red[w];
    return t;
}

template <int VPT>
__device__ __forceinline__ float square_sum(const float (&v)[VPT][8]) {
    float ss[VPT];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        ss[k] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss[k] = fmaf(v[k][j], v[k][j], ss[k]);
    }
#pragma unroll
    for (int k = 1; k < VPT; ++k) ss[0] += ss[k];
    return ss[0];
}

template <int VPT, bool VEC>
__global__ void __launch_bounds__(512) norm_row_kernel(NormArgs a, int G) {
    __shared__ float red[2][32];
    pdl_launch_dependents();
    const size_t t = (size_t)blockIdx.x * (blockDim.x / G) + threadIdx.x / G;
    if (t >= (size_t)a.n_tok) return;  // whole warps: G is 32 where a CTA has more than one row
    const Row<VPT, VEC> row{G, (int)(threadIdx.x % G), a.E};
    pdl_wait();
    float v[VPT][8];
    row.load(a.x, a.x_bf16, t * a.ldx, v);
    const float scale = 1.0f / sqrtf(row_sum(square_sum(v), G, red[0]) / (float)a.E + a.eps);
    float g = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        float w[8];
        row.weights(a.w, k, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[k][j] = v[k][j] * scale * w[j];
        if (a.gate_w) {
            row.weights(a.gate_w, k, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) g = fmaf(w[j], v[k][j], g);
        }
    }
    row.store(a.y, a.y_bf16, t * a.ldy, v);
    if (a.gate_w) {
        g = row_sum(g, G, red[1]);
        if (row.l == 0) a.gate[t] = g;
    }
}

// Many rows of G * 8 * VPT values exactly, 16-byte accesses, no gate: each CTA walks over rows with its
// weights in registers and the next row already on its way.
template <int VPT, bool XB, bool YB>
__global__ void __launch_bounds__(512, 2) norm_stream_kernel(NormArgs a) {
    __shared__ float red[2][32];
    constexpr int Q = XB ? 1 : 2;  // 16-byte words of 8 values
    const int G = blockDim.x, l = threadIdx.x;
    pdl_launch_dependents();
    pdl_wait();
    uint4 raw[VPT][Q];
    auto fetch = [&](size_t t) {
#pragma unroll
        for (int k = 0; k < VPT; ++k)
#pragma unroll
            for (int q = 0; q < Q; ++q)
                raw[k][q] = __ldcs(reinterpret_cast<const uint4 *>(reinterpret_cast<const uint8_t *>(a.x) + t * a.ldx * (XB ? 2 : 4)) +
                                   (k * G + l) * Q + q);
    };
    size_t t = blockIdx.x;
    fetch(t);
    float w[VPT][8];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[k][j] = 1.f;
        if (a.w) {
            const float4 *p = reinterpret_cast<const float4 *>(a.w) + (k * G + l) * 2;
            const float4 u = __ldg(p), v = __ldg(p + 1);
            w[k][0] = u.x; w[k][1] = u.y; w[k][2] = u.z; w[k][3] = u.w;
            w[k][4] = v.x; w[k][5] = v.y; w[k][6] = v.z; w[k][7] = v.w;
        }
    }
    const float mean = 1.0f / (float)a.E;
    for (int parity = 0; t < (size_t)a.n_tok; t += gridDim.x, parity ^= 1) {
        float v[VPT][8];
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const uint32_t *u = reinterpret_cast<const uint32_t *>(&raw[k][0]);
#pragma unroll
            for (int j = 0; j < 4 * Q; ++j) {
                if constexpr (XB) {
                    v[k][2 * j] = __uint_as_float(u[j] << 16);
                    v[k][2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
                } else {
                    v[k][j] = __uint_as_float(u[j]);
                }
            }
        }
        if (t + gridDim.x < (size_t)a.n_tok) fetch(t + gridDim.x);
        // two places for the sums in turn: one barrier a row
        const float ss = row_sum(square_sum(v), G, red[parity]);
        const float scale = 1.0f / sqrtf(fmaf(ss, mean, a.eps));
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[k][j] = v[k][j] * scale * w[k][j];
            if constexpr (YB) {
                uint32_t o[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(v[k][2 * j], v[k][2 * j + 1]);
                    o[j] = *reinterpret_cast<const uint32_t *>(&h);
                }
                reinterpret_cast<uint4 *>(reinterpret_cast<__nv_bfloat16 *>(a.y) + t * a.ldy)[k * G + l] = make_uint4(o[0], o[1], o[2], o[3]);
            } else {
                float4 *f = reinterpret_cast<float4 *>(reinterpret_cast<float *>(a.y) + t * a.ldy) + (k * G + l) * 2;
                f[0] = make_float4(v[k][0], v[k][1], v[k][2], v[k][3]);
                f[1] = make_float4(v[k][4], v[k][5], v[k][6], v[k][7]);
            }
        }
    }
}

template <int VPT, bool VEC>
__global__ void __launch_bounds__(512) residual_row_kernel(ResidualArgs a, int G) {
    __shared__ float red[3][32];
    pdl_launch_dependents();
    const size_t t = (size_t)blockIdx.x * (blockDim.x / G) + threadIdx.x / G;
    if (t >= (size_t)a.n_tok) return;
    const Row<VPT, VEC> row{G, (int)(threadIdx.x % G), a.E};
    pdl_wait();
    float v[VPT][8], r[VPT][8], e[VPT][8];
    row.load(a.y, a.y_bf16, t * a.ldy, v);
    row.load(a.res, a.res_bf16, t * a.ldr, r);
    if (a.gate_kind == GX_GATE_ELEMENT) row.load(a.gate, a.gate_bf16, t * a.ldg, e);
    float tgate = a.block_scale;
    if (a.gate_kind == GX_GATE_TOKEN) tgate *= sigmoid(reinterpret_cast<const float *>(a.gate)[t]);
    float yscale = 1.f;
    if (a.post_norm) yscale = 1.0f / sqrtf(row_sum(square_sum(v), G, red[0]) / (float)a.E + a.eps);
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        float w[8];
        row.weights(a.post, k, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float x = v[k][j] * yscale * w[j];
            if (a.gate_kind == GX_GATE_ELEMENT) x *= sigmoid(e[k][j]);
            r[k][j] = a.res_scale * r[k][j] + tgate * x;
        }
    }
    row.store(a.res_out, a.res_bf16, t * a.ldro, r);
    if (!a.out) return;
    const float rscale = 1.0f / sqrtf(row_sum(square_sum(r), G, red[1]) / (float)a.E + a.next_eps);
    float g = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        float w[8];
        row.weights(a.next, k, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) r[k][j] = r[k][j] * rscale * w[j];
        if (a.next_gate_w) {
            row.weights(a.next_gate_w, k, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) g = fmaf(w[j], r[k][j], g);
        }
    }
    row.store(a.out, a.out_bf16, t * a.ldo, r);
    if (a.next_gate_w) {
        g = row_sum(g, G, red[2]);
        if (row.l == 0) a.next_gate[t] = g;
    }
}

// Whether rows of E elements at stride ld can be accessed 16 bytes at a time.
bool vec_rows(const void *p, int bf16, long long ld) {
    return !p || (((uintptr_t)p & 15) == 0 && ld * (bf16 ? 2 : 4) % 16 == 0);
}
bool vec_words(const float *p) { return ((uintptr_t)p & 15) == 0; }

// Threads of a row, and rows of a CTA: rows of up to 512 values take one warp each, 8 in a CTA.
struct Shape {
    int G, block, grid;
};
Shape row_shape(int E, int n_tok, int vpt) {
    Shape s;
    const int lanes = (E + 8 * vpt - 1) / (8 * vpt);
    s.G = (lanes + 31) / 32 * 32;
    const int rows = s.G == 32 ? 8 : 1;
    s.block = s.G * rows;
    s.grid = (n_tok + rows - 1) / rows;
    return s;
}

// The vectors of a thread: two; four for rows beyond 8192; one while the rows are fewer than the SMs and
// latency is what counts.
int row_vectors(int E, int n_tok, int sm_count) { return n_tok < sm_count && E <= 4096 ? 1 : E <= 8192 ? 2 : 4; }

template <int VPT>
cudaError_t launch_norm_row(const NormArgs &a, bool vec, cudaStream_t s) {
    const Shape p = row_shape(a.E, a.n_tok, VPT);
    auto *k = vec ? norm_row_kernel<VPT, true> : norm_row_kernel<VPT, false>;
    return launch_chain_pdl(true, k, dim3((unsigned)p.grid), dim3((unsigned)p.block), 0, s, a, p.G);
}

template <int VPT>
cudaError_t launch_residual_row(const ResidualArgs &a, bool vec, cudaStream_t s) {
    const Shape p = row_shape(a.E, a.n_tok, VPT);
    auto *k = vec ? residual_row_kernel<VPT, true> : residual_row_kernel<VPT, false>;
    return launch_chain_pdl(true, k, dim3((unsigned)p.grid), dim3((unsigned)p.block), 0, s, a, p.G);
}

}  // namespace

cudaError_t launch_norm(const NormArgs &a, int sm_count, cudaStream_t s) {
    if (a.n_tok <= 0) return cudaSuccess;
    if (a.E > kNormRowMax)
        return launch_chain_pdl(true, norm_long_kernel, dim3((unsigned)a.n_tok), dim3(kNormThreads), 0, s, a);
    const bool vec = a.E % 8 == 0 && vec_rows(a.x, a.x_bf16, a.ldx) && vec_rows(a.y, a.y_bf16, a.ldy) && vec_words(a.w) &&
                     vec_words(a.gate_w);
    // Enough rows for every CTA to walk over several, in the widths that fill its threads (64 threads and
    // more of two vectors).
    const int G = a.E / 16, resident = sm_count * (1024 / (G ? G : 1));
    if (vec && !a.gate_w && a.E % 512 == 0 && a.E >= 1024 && a.E <= 8192 && a.n_tok >= 4 * resident) {
        auto *k = a.x_bf16 ? (a.y_bf16 ? norm_stream_kernel<2, true, true> : norm_stream_kernel<2, true, false>)
                           : (a.y_bf16 ? norm_stream_kernel<2, false, true> : norm_stream_kernel<2, false, false>);
        return launch_chain_pdl(true, k, dim3((unsigned)resident), dim3((unsigned)G), 0, s, a);
    }
    switch (row_vectors(a.E, a.n_tok, sm_count)) {
        case 1: return launch_norm_row<1>(a, vec, s);
        case 2: return launch_norm_row<2>(a, vec, s);
        default: return launch_norm_row<4>(a, vec, s);
    }
}

cudaError_t launch_norm_residual(const ResidualArgs &a, int sm_count, cudaStream_t s) {
    if (a.n_tok <= 0) return cudaSuccess;
    if (a.E > kNormRowMax)
        return launch_chain_pdl(true, residual_long_kernel, dim3((unsigned)a.n_tok), dim3(kNormThreads), 0, s, a);
    const bool vec = a.E % 8 == 0 && vec_rows(a.y, a.y_bf16, a.ldy) && vec_rows(a.res, a.res_bf16, a.ldr) &&
                     vec_rows(a.res_out, a.res_bf16, a.ldro) && vec_rows(a.out, a.out_bf16, a.ldo) &&
                     (a.gate_kind != GX_GATE_ELEMENT || vec_rows(a.gate, a.gate_bf16, a.ldg)) && vec_words(a.post) &&
                     vec_words(a.next) && vec_words(a.next_gate_w);
    switch (row_vectors(a.E, a.n_tok, sm_count)) {
        case 1: return launch_residual_row<1>(a, vec, s);
        case 2: return launch_residual_row<2>(a, vec, s);
        default: return launch_residual_row<4>(a, vec, s);
    }
}

}  // namespace gx
