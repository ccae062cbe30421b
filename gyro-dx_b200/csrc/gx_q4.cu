// gx_q4.cu — matrix-vector products with 4-bit weights and group scales (GGUF Q4_0 and Q4_1):
//
//   y[t][r] = sum over groups of 32 columns of  d * sum_c (q - 8) x[t][c]        (Q4_0)
//                                               d * sum_c q x[t][c] + m * sum_c x[t][c]   (Q4_1)
//
// with fp16 d and m per group and 4-bit q.
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

constexpr int kQ4Warps = 4;
constexpr int kQ4Tok = 8;

__device__ __forceinline__ void store_act(void *p, int bf16, size_t i, float v) {
    if (bf16) reinterpret_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
    else reinterpret_cast<float *>(p)[i] = v;
}

// One warp per row, a lane per group of 32 columns, up to 8 tokens at a time, f32 sums.
__global__ void __launch_bounds__(kQ4Warps * 32) q4_rows_kernel(Q4Args a) {
    const int r = blockIdx.x * kQ4Warps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (r >= a.rows) return;
    const int NG = a.cols / 32, gb = a.type == GX_Q4_0 ? 18 : 20;
    const uint8_t *row = a.w + (size_t)r * NG * gb;
    for (int t0 = 0; t0 < a.n_tok; t0 += kQ4Tok) {
        const int nt = min(kQ4Tok, a.n_tok - t0);
        float acc[kQ4Tok];
#pragma unroll
        for (int t = 0; t < kQ4Tok; ++t) acc[t] = 0.f;
        for (int g = lane; g < NG; g += 32) {
            const uint8_t *b = row + (size_t)g * gb;
            const float d = __half2float(*reinterpret_cast<const __half *>(b));
            const float m = a.type == GX_Q4_0 ? -8.f * d : __half2float(*reinterpret_cast<const __half *>(b + 2));
            const uint8_t *q = b + gb - 16;
#pragma unroll
            for (int t = 0; t < kQ4Tok; ++t) {
                if (t >= nt) break;
                const size_t base = (size_t)(t0 + t) * a.ldx + (size_t)g * 32;
                float qx = 0.f, sx = 0.f;
                for (int j = 0; j < 16; ++j) {
                    const float x0 = load_act(a.x, a.x_bf16, base + j), x1 = load_act(a.x, a.x_bf16, base + j + 16);
                    qx = fmaf((float)(q[j] & 15), x0, fmaf((float)(q[j] >> 4), x1, qx));
                    sx += x0 + x1;
                }
                acc[t] = fmaf(d, qx, fmaf(m, sx, acc[t])) + (sx - sx);  // Inf and NaN activations: NaN
            }
        }
#pragma unroll
        for (int t = 0; t < kQ4Tok; ++t) {
            if (t >= nt) break;
            const float s = warp_sum(acc[t]);
            if (lane == 0) store_act(a.y, a.y_bf16, (size_t)(t0 + t) * a.ldy + r, s);
        }
    }
}

}  // namespace

uint64_t q4_row_bytes(uint32_t type, uint64_t cols) {
    if ((type != GX_Q4_0 && type != GX_Q4_1) || cols % 32) return 0;
    return cols / 32 * (type == GX_Q4_0 ? 18 : 20);
}

uint64_t q4_bytes(uint32_t type, uint64_t rows, uint64_t cols) { return rows * q4_row_bytes(type, cols); }

cudaError_t launch_q4_repack(uint32_t type, const uint8_t *raw, uint32_t rows, uint32_t cols, uint8_t *w,
                             cudaStream_t s) {
    return cudaMemcpyAsync(w, raw, q4_bytes(type, rows, cols), cudaMemcpyDeviceToDevice, s);
}

cudaError_t launch_q4_linear(const Q4Args &a, int sm_count, cudaStream_t s) {
    if (a.n_tok <= 0 || a.rows <= 0) return cudaSuccess;
    q4_rows_kernel<<<(a.rows + kQ4Warps - 1) / kQ4Warps, kQ4Warps * 32, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace gx
