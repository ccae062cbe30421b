// gx_logprobs.cu — log probabilities of given tokens over rows of logits, with the entropy, the
// given token's rank and the likeliest alternatives. With z = scale * x, m = max z, s = sum e^(z-m):
//
//   logprob = (z_t - m) - ln s,   entropy = ln s - (sum e^(z-m) (z-m)) / s,
//   rank = 1 + #{x > x_t},        the n_top largest x, equal ones by rising id.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include "../../include/gyro_moe.h"
#include "gx_dense.cuh"
#include "gx_device.cuh"
#include "gx_internal.h"

namespace gx {

using namespace dense;

namespace {

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;

// A logit and its id as one key that orders by value, then by lower id; a NaN lies below -Inf and
// -0 equals 0. No key of a logit is 0.
__device__ __forceinline__ uint64_t logit_key(float x, uint32_t id) {
    uint32_t u = __float_as_uint(x + 0.0f);
    u = (u >> 31) ? ~u : u | 0x80000000u;
    if (isnan(x)) u = 1u;
    return ((uint64_t)u << 32) | (0xffffffffu - id);
}

template <typename T, typename F>
__device__ __forceinline__ T block_reduce(T v, T *red, F f) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < kLpWarps; ++w) v = f(v, red[w]);
    return v;
}

__device__ __forceinline__ float max_nan(float a, float b) { return isnan(a) || isnan(b) ? CUDART_NAN_F : fmaxf(a, b); }

__global__ void __launch_bounds__(kLpThreads) logprobs_kernel(LogprobsArgs a) {
    __shared__ float redf[kLpWarps];
    __shared__ unsigned redu[kLpWarps];
    __shared__ unsigned long long redk[kLpWarps];
    const size_t r = blockIdx.x, base = r * (size_t)a.stride;
    const uint32_t V = (uint32_t)a.n_vocab;
    auto add = [](auto p, auto q) { return p + q; };
    float m = -CUDART_INF_F;
    for (uint32_t i = threadIdx.x; i < V; i += kLpThreads) m = max_nan(m, load_act(a.logits, a.bf16, base + i));
    m = block_reduce(m, redf, [](float p, float q) { return max_nan(p, q); });
    const uint32_t tok = a.tokens ? a.tokens[r] : GX_NO_TOKEN;
    const bool has = tok < V;
    const float xt = has ? load_act(a.logits, a.bf16, base + tok) : 0.f;
    const float xt_cmp = isnan(xt) ? -CUDART_INF_F : xt;
    float s = 0.f, et = 0.f;
    unsigned above = 0;
    for (uint32_t i = threadIdx.x; i < V; i += kLpThreads) {
        const float x = load_act(a.logits, a.bf16, base + i);
        const float t = x == m && !isinf(x) ? 0.f : m == -CUDART_INF_F ? 0.f : (x - m) * a.scale;
        const float e = expf(t);
        s += e;
        if (e > 0.f) et = fmaf(e, t, et);
        if (isnan(e)) et = e;
        above += isnan(xt) ? !isnan(x) : x > xt_cmp;
    }
    s = block_reduce(s, redf, add);
    et = block_reduce(et, redf, add);
    above = block_reduce(above, redu, add);
    const float ls = logf(s);
    // halves, so that a difference beyond the f32 range that the scale brings back is not lost
    auto lp = [&](float x) { return (m == -CUDART_INF_F ? 0.f : (0.5f * x - 0.5f * m) * (2.f * a.scale)) - ls; };
    if (threadIdx.x == 0) {
        const bool bad = a.tokens && !has && tok != GX_NO_TOKEN;
        if (bad) atomicExch(a.err, KERR_BOUNDS);
        if (a.logprob) a.logprob[r] = has ? lp(xt) : bad ? CUDART_NAN_F : 0.f;
        if (a.rank) a.rank[r] = has ? above + 1 : 0;
        if (a.entropy) a.entropy[r] = ls - et / s;
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < a.n_top; ++k) {
        unsigned long long best = 0;
        for (uint32_t i = threadIdx.x; i < V; i += kLpThreads) {
            const unsigned long long key = logit_key(load_act(a.logits, a.bf16, base + i), i);
            if (key < last && key > best) best = key;
        }
        best = block_reduce(best, redk, [](unsigned long long p, unsigned long long q) { return p > q ? p : q; });
        last = best;
        if (threadIdx.x == 0) {
            const uint32_t id = 0xffffffffu - (uint32_t)best;
            if (a.top_ids) a.top_ids[r * a.n_top + k] = id;
            if (a.top_logprobs) a.top_logprobs[r * a.n_top + k] = lp(load_act(a.logits, a.bf16, base + id));
        }
    }
}

}  // namespace

cudaError_t launch_logprobs(const LogprobsArgs &a, int sm_count, cudaStream_t s) {
    if (a.n_rows <= 0) return cudaSuccess;
    logprobs_kernel<<<a.n_rows, kLpThreads, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace gx
