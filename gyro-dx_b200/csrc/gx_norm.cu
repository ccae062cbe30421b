// gx_norm.cu — the norms around a block, with its gate and residual scale:
//
//   before:  h = x / sqrt(mean(x^2) + eps) * w,                      gate = gate_w . h
//   after:   v = y / sqrt(mean(y^2) + eps) * post   (or y itself)
//            r = res_scale * res + block_scale * gate * v            gate: 1, sigmoid per token or per element
//            res_out = r,  out = r / sqrt(mean(r^2) + eps) * next,   next_gate = next_gate_w . out
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

constexpr int kNormThreads = 256;

__device__ __forceinline__ void store_act(void *p, int bf16, size_t i, float v) {
    if (bf16) reinterpret_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
    else reinterpret_cast<float *>(p)[i] = v;
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

__global__ void __launch_bounds__(kNormThreads) norm_kernel(NormArgs a) {
    __shared__ float red[kNormThreads / 32];
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
    if (a.gate_kind == GX_GATE_ELEMENT) v *= sigmoid_ref(load_act(a.gate, a.gate_bf16, t * a.ldg + i));
    return a.res_scale * load_act(a.res, a.res_bf16, t * a.ldr + i) + a.block_scale * tgate * v;
}

__global__ void __launch_bounds__(kNormThreads) norm_residual_kernel(ResidualArgs a) {
    __shared__ float red[kNormThreads / 32];
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
    const float tgate = a.gate_kind == GX_GATE_TOKEN ? sigmoid_ref(reinterpret_cast<const float *>(a.gate)[t]) : 1.f;
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

}  // namespace

cudaError_t launch_norm(const NormArgs &a, cudaStream_t s) {
    if (a.n_tok <= 0) return cudaSuccess;
    norm_kernel<<<a.n_tok, kNormThreads, 0, s>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_norm_residual(const ResidualArgs &a, cudaStream_t s) {
    if (a.n_tok <= 0) return cudaSuccess;
    norm_residual_kernel<<<a.n_tok, kNormThreads, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace gx
