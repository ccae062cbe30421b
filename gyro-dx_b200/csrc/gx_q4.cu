// gx_q4.cu — matrix-vector products with 4-bit weights and group scales (GGUF Q4_0 and Q4_1):
//
//   y[t][r] = sum over groups of 32 columns of  d * (sum_c q x[t][c] - 8 sum_c x[t][c])       (Q4_0)
//                                               d *  sum_c q x[t][c] + m sum_c x[t][c]        (Q4_1)
//
// with fp16 d and m per group and 4-bit q.
//
// The sums over a group run on the tensor cores (mma.sync m16n8k16, f32 accumulation) on the integers
// q - 8 (Q4_1: q), which f16 holds exactly, and d meets the group's sum in f32, so no weight is ever
// rounded. A code in the low bits of an f16 under the exponent of 1024 is 1024 + q, four bits higher
// 1024 + 16 q: one shift, four and-ors and four half2 operations turn a word of 8 codes into its four
// A registers. (Codes as f16 subnormals need no arithmetic at all, but the product then aligns its
// terms by the subnormals' exponent and loses their leading zeros: 2e-6 to 4e-6 relative error
// measured, against 1e-7.)
//
// Activations become f16 fragments in shared memory once per CTA: each unit of 128 columns of a token
// is scaled by a power of two that brings its largest value to 2^14..2^15; an f32 value is split into
// two f16 (22 bits, two columns of the product), a bf16 value fits one.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>

#include "../../include/gyro_moe.h"
#include "gx_dense.cuh"
#include "gx_device.cuh"
#include "gx_internal.h"

namespace gx {

using namespace dense;

namespace {

// ---- device layout ---------------------------------------------------------------------------
// Units of 16 rows x 128 columns (4 groups), ordered [row tile][unit]; rows and columns past the
// matrix have zero scales. Lane l = 4 g + q of a warp owns rows g and g + 8 and, in each group, the
// columns 8 q .. 8 q + 7, the k-slices its A registers hold:
//   [32 lanes][4 groups] words of row g     code of column 8 q + i in bits 4 i .. 4 i + 3
//   [32 lanes][4 groups] words of row g + 8
//   [8 g][4 groups][row g, row g + 8] fp16 d
//   [8 g][4 groups][row g, row g + 8] fp16 m   (Q4_1)
constexpr int kUnitCols = 128, kTileRows = 16;
__host__ __device__ constexpr int unit_bytes(uint32_t type) { return type == GX_Q4_0 ? 1152 : 1280; }

__device__ __forceinline__ void store_act(void *p, int bf16, size_t i, float v) {
    if (bf16) reinterpret_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
    else reinterpret_cast<float *>(p)[i] = v;
}

// One thread per (row of the padded matrix, group): 4 words and the scales of a group.
__global__ void __launch_bounds__(256) q4_repack_kernel(uint32_t type, const uint8_t *raw, int rows, int cols,
                                                        uint8_t *w, long long n) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int NG = (cols + kUnitCols - 1) / kUnitCols * 4;
    const long long row = i / NG;
    const int grp = (int)(i % NG), g = (int)(row & 7), hi = (int)(row >> 3) & 1, j = grp & 3;
    uint8_t *u = w + ((row / kTileRows) * (NG / 4) + grp / 4) * unit_bytes(type);
    uint32_t words[4] = {0u, 0u, 0u, 0u};
    uint16_t d = 0, m = 0;
    if (row < rows && grp < cols / 32) {
        const int gb = type == GX_Q4_0 ? 18 : 20;
        const uint16_t *b = reinterpret_cast<const uint16_t *>(raw + (row * (cols / 32) + grp) * gb);
        d = b[0];
        if (type == GX_Q4_1) m = b[1];
        b += gb / 2 - 8;
        for (int k = 0; k < 8; ++k) {  // bytes 2k, 2k+1: columns 2k, 2k+1 (low halves) and 2k+16, 2k+17
            const uint32_t v = b[k];
            const int q = k >> 2, s = 8 * (k & 3);
            words[q] |= ((v & 15u) | ((v >> 4) & 0xf0u)) << s;
            words[q + 2] |= (((v >> 4) & 15u) | ((v >> 8) & 0xf0u)) << s;
        }
    }
    uint32_t *codes = reinterpret_cast<uint32_t *>(u + 512 * hi);
    for (int q = 0; q < 4; ++q) codes[(4 * g + q) * 4 + j] = words[q];
    reinterpret_cast<uint16_t *>(u + 1024)[(g * 4 + j) * 2 + hi] = d;
    if (type == GX_Q4_1) reinterpret_cast<uint16_t *>(u + 1152)[(g * 4 + j) * 2 + hi] = m;
}

// ---- few tokens: a GEMV on mma.sync ------------------------------------------------------------
__device__ __forceinline__ float half_value(uint32_t w, int hi) {
    const __half2 h = *reinterpret_cast<const __half2 *>(&w);
    return hi ? __high2float(h) : __low2float(h);
}

// A lane's part of a unit: the words of its two rows, and the scales (row g in the low half, row g + 8
// in the high one) of the groups whose sums it holds.
template <uint32_t TYPE, int SETS>
struct Unit {
    uint4 c0, c1;
    uint32_t d[SETS], m[SETS];
};
// p: the lane's words of row g; its scales lie scale bytes after them.
template <uint32_t TYPE, int SETS>
__device__ __forceinline__ void load_unit(Unit<TYPE, SETS> &u, const uint8_t *p, int scale) {
    u.c0 = __ldcs(reinterpret_cast<const uint4 *>(p));
    u.c1 = __ldcs(reinterpret_cast<const uint4 *>(p + 512));
    auto scales = [&](uint32_t (&d)[SETS], const uint8_t *at) {
        if constexpr (SETS == 4) {
            const uint4 v = __ldcs(reinterpret_cast<const uint4 *>(at));
            d[0] = v.x;
            d[1] = v.y;
            d[2] = v.z;
            d[3] = v.w;
        } else {
#pragma unroll
            for (int s = 0; s < SETS; ++s) d[s] = __ldcs(reinterpret_cast<const uint32_t *>(at + s * 8));
        }
    };
    scales(u.d, p + scale);
    if constexpr (TYPE == GX_Q4_1) scales(u.m, p + scale + 128);
}

// The 8 scaled values of columns 8 q .. of a group as the fragment of token t (column t in bf16; 2 t
// and 2 t + 1, the upper and lower part, in f32).
template <bool XB>
__device__ __forceinline__ void put_fragment(uint8_t *group, int t, int q, const float (&v)[8]) {
    auto put = [&](int c, const float (&x)[8]) {
        *reinterpret_cast<uint4 *>(group + ((size_t)c * 4 + q) * 16) =
            make_uint4(pack_half2(x[0], x[4]), pack_half2(x[2], x[6]), pack_half2(x[1], x[5]), pack_half2(x[3], x[7]));
    };
    if constexpr (XB) {
        put(t, v);
    } else {
        float hi[8], lo[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) split_hilo(v[k], hi[k], lo[k]);
        put(2 * t, hi);
        put(2 * t + 1, lo);
    }
}

// The product of a group's first half on nothing (mma16816 adds the second to it).
__device__ __forceinline__ void mma16816_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// The product of a group: both halves of its 32 columns, on nothing.
__device__ __forceinline__ void mma_group(float (&d)[4], const uint32_t (&a0)[4], const uint32_t (&a1)[4], const uint4 &b) {
    asm("{\n"
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%12,%13}, {%16,%16,%16,%16};\n"
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%8,%9,%10,%11}, {%14,%15}, {%0,%1,%2,%3};\n"
        "}\n"
        : "=&f"(d[0]), "=&f"(d[1]), "=&f"(d[2]), "=&f"(d[3])
        : "r"(a0[0]), "r"(a0[1]), "r"(a0[2]), "r"(a0[3]), "r"(a1[0]), "r"(a1[1]), "r"(a1[2]), "r"(a1[3]), "r"(b.x), "r"(b.y),
          "r"(b.z), "r"(b.w), "f"(0.f));
}

// The A registers of 8 codes of row g (r0) and of row g + 8 (r1): columns (0,4) (2,6) of each in a0,
// (1,5) (3,7) in a1.
template <uint32_t TYPE>
__device__ __forceinline__ void code_fragments(uint32_t r0, uint32_t r1, uint32_t (&a0)[4], uint32_t (&a1)[4]) {
    constexpr float off = TYPE == GX_Q4_0 ? 8.f : 0.f;
    const __half2 sub = __float2half2_rn(-1024.f - off), mul = __float2half2_rn(0.0625f), sub16 = __float2half2_rn(-64.f - off);
    auto and_or = [](uint32_t v, uint32_t mask) {  // (v & mask) | 0x64006400
        uint32_t h;
        asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(h) : "r"(v), "r"(mask), "r"(0x64006400u));
        return h;
    };
    auto low = [&](uint32_t v) {
        const uint32_t h = and_or(v, 0x000f000fu);
        const __half2 r = __hadd2(*reinterpret_cast<const __half2 *>(&h), sub);
        return *reinterpret_cast<const uint32_t *>(&r);
    };
    auto high = [&](uint32_t v) {
        const uint32_t h = and_or(v, 0x00f000f0u);
        const __half2 r = __hfma2(*reinterpret_cast<const __half2 *>(&h), mul, sub16);
        return *reinterpret_cast<const uint32_t *>(&r);
    };
    a0[0] = low(r0);
    a0[1] = low(r1);
    a0[2] = low(r0 >> 8);
    a0[3] = low(r1 >> 8);
    a1[0] = high(r0);
    a1[1] = high(r1);
    a1[2] = high(r0 >> 8);
    a1[3] = high(r1 >> 8);
}

// One token's 8 columns of a unit of a CTA's range: its values (0 past the matrix), and the largest
// magnitude of the unit by its bits (16 lanes hold a unit; an Inf or NaN has the largest exponent).
template <bool XB>
__device__ __forceinline__ uint32_t load_cell(const Q4Args &a, int t, int col, bool on, bool vec, float (&v)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = 0.f;
    if (on && col < a.cols) {  // cols is a multiple of 32: a cell is inside or outside
        const size_t at = (size_t)t * a.ldx + col;
        if (vec) load_x8(a.x, XB, at, v);
        else {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = load_act(a.x, XB, at + k);
        }
    }
    uint32_t big = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) big = max(big, __float_as_uint(v[k]) & 0x7fffffffu);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, o));
    return big;
}
template <typename T>
__device__ __forceinline__ T quad_sum(T v) {
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// Two ways to multiply a unit by few tokens. Each stages the activations of a CTA's units in shared
// memory, a block of BYTES per unit, and gives a lane's part of the sums of rows g and g + 8.
//
// Ints: one or two tokens on the integer tensor cores. Here the arithmetic around the product is what
// costs, and codes are integers already: two ands and a shift turn a word of 8 into A registers
// of m16n8k32 (u8), a third of the work of the f16 form. A value becomes a whole number of 2^-29 of its
// unit's power of two (30 bits), its four signed base-256 digits four columns of the product, exact in
// 32 bits; -8 sum of digits is the initial accumulator, under an offset (2^23 + 2^22 as f32 bits) that
// makes the result a float by itself. One token's 4 columns leave 4 free: two groups share an
// accumulator, the fragment of each being zero in the columns of the other.
template <uint32_t TYPE, bool XB, int T>
struct Ints {
    static constexpr int TOK = T, NA = 2, SETS = T == 1 ? 2 : 4, kDepth = T == 1 ? 5 : 4;  // units in flight
    static constexpr int CTAS(int W) { return W == 16 ? 1 : 2; }                       // resident on an SM
    // [4 groups][T tokens][4 digits][4 q] 8 B: the digit of columns (0 2 4 6) and (1 3 5 7) of 8 q ..
    static constexpr int GROUP = T * 128, ZERO = 4 * GROUP;       // T == 1: 32 B of zeros
    static constexpr int INIT = ZERO + (T == 1 ? 32 : 0);         // Q4_0: [group][token][digit pair] int4 accumulators
    static constexpr int SUM = INIT;                              // Q4_1: [group][token][digit pair] float: sum x, 0
    static constexpr int INV = TYPE == GX_Q4_0 ? INIT + T * 128 : SUM + T * 32;  // [token] float: 2^24 units of the numbers
    static constexpr int BYTES = (INV + T * 4 + 15) / 16 * 16;
    static constexpr uint32_t kOffset = 0x4b400000u;              // 2^23 + 2^22 as a float

    int at[4];       // the lane's fragment in each group
    float w0, w1;    // weights of the digits that its accumulator columns hold
    float acc[NA];   // rows g and g + 8; T == 2: token q >> 1

    __device__ __forceinline__ void init(int lane, int nt) {
        const int g = lane >> 2, q = lane & 3;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            at[j] = T == 2 ? j * GROUP + ((g >> 2) < nt ? g : (g & 3)) * 32 + q * 8
                           : (g >> 2 == (j & 1) ? j * GROUP + (g & 3) * 32 : ZERO) + q * 8;
        w0 = (q & 1) ? 0x1p-16f : 1.f;
        w1 = (q & 1) ? 0x1p-24f : 0x1p-8f;
    }
    static __device__ __forceinline__ int scale_offset(int lane) {
        return T == 1 ? (lane >> 1) * 4 + (lane >> 2) * 8 : (lane >> 2) * 16;
    }
    static __device__ void stage(const Q4Args &a, int t0, int nt, int u0, int nu, uint8_t *smem, bool vec, int tid, int nthreads) {
        const int cells = nu * 16, total = nt * cells;
        for (int base = 0; base < total; base += nthreads) {
            const int i = base + tid;
            const bool on = i < total;
            const int t = on ? i / cells : 0, cell = on ? i % cells : 0, q = cell & 3, j = (cell >> 2) & 3;
            float v[8];
            const uint32_t big = load_cell<XB>(a, t0 + t, u0 * kUnitCols + cell * 8, on, vec, v), e = big >> 23;
            // 2^k with the unit's largest value below 2^30, as two factors: it may pass the f32 range
            const int k = 29 + 127 - (int)max(min(e, 254u), 1u), k1 = k / 2, k2 = k - k1;
            const float s1 = __uint_as_float((uint32_t)(127 + k1) << 23), s2 = __uint_as_float((uint32_t)(127 + k2) << 23);
            uint32_t b[8];
            float fs = 0.f;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const float x = e == 255u ? 0.f : v[c] * s1 * s2;
                b[c] = ((uint32_t)__float2int_rn(x) + 0x00808080u) ^ 0x00808080u;  // signed digits, byte by byte
                fs += v[c];
            }
            uint32_t w[2][4];  // [half of the columns][digit, most significant first]
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t lo01 = __byte_perm(b[h], b[h + 2], 0x5140), hi01 = __byte_perm(b[h], b[h + 2], 0x7362);
                const uint32_t lo23 = __byte_perm(b[h + 4], b[h + 6], 0x5140), hi23 = __byte_perm(b[h + 4], b[h + 6], 0x7362);
                w[h][3] = __byte_perm(lo01, lo23, 0x5410);
                w[h][2] = __byte_perm(lo01, lo23, 0x7632);
                w[h][1] = __byte_perm(hi01, hi23, 0x5410);
                w[h][0] = __byte_perm(hi01, hi23, 0x7632);
            }
            int ds[4];
#pragma unroll
            for (int d = 0; d < 4; ++d) ds[d] = __dp4a((int)w[0][d], 0x01010101, __dp4a((int)w[1][d], 0x01010101, 0));
            if constexpr (TYPE == GX_Q4_0) {
#pragma unroll
                for (int d = 0; d < 4; ++d) ds[d] = (int)kOffset - 8 * quad_sum(ds[d]);
            } else {
                fs = quad_sum(fs);
            }
            if (!on) continue;
            uint8_t *u = smem + (cell >> 4) * BYTES;
#pragma unroll
            for (int d = 0; d < 4; ++d)
                *reinterpret_cast<uint2 *>(u + j * GROUP + (t * 4 + d) * 32 + q * 8) = make_uint2(w[0][d], w[1][d]);
            if (q == 0) {
                if constexpr (TYPE == GX_Q4_0) {
                    int4 *n = reinterpret_cast<int4 *>(u + INIT) + (j * T + t) * 2;
                    n[0] = make_int4(ds[0], ds[1], ds[0], ds[1]);
                    n[1] = make_int4(ds[2], ds[3], ds[2], ds[3]);
                } else {
                    reinterpret_cast<float2 *>(u + SUM)[j * T + t] = make_float2(fs, 0.f);
                }
            }
            if ((cell & 15) == 0) {
                reinterpret_cast<float *>(u + INV)[t] =
                    e == 255u ? __uint_as_float(0x7fffffffu)
                              : __uint_as_float((uint32_t)(151 - k1) << 23) * __uint_as_float((uint32_t)(127 - k2) << 23);
                if constexpr (T == 1) {
                    reinterpret_cast<uint4 *>(u + ZERO)[0] = make_uint4(0u, 0u, 0u, 0u);
                    reinterpret_cast<uint4 *>(u + ZERO)[1] = make_uint4(0u, 0u, 0u, 0u);
                }
            }
        }
    }
    __device__ __forceinline__ void unit(const Unit<TYPE, SETS> &u, const uint8_t *x, int lane) {
        const int q = lane & 3;
        const uint32_t c0[4] = {u.c0.x, u.c0.y, u.c0.z, u.c0.w}, c1[4] = {u.c1.x, u.c1.y, u.c1.z, u.c1.w};
        const float inv = reinterpret_cast<const float *>(x + INV)[T == 1 ? 0 : q >> 1], v0 = inv * w0, v1 = inv * w1;
        int4 c;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            constexpr uint32_t M = 0x0f0f0f0fu;
            const uint32_t a[4] = {c0[j] & M, c1[j] & M, (c0[j] >> 4) & M, (c1[j] >> 4) & M};
            const bool first = T == 2 || (j & 1) == 0, last = T == 2 || (j & 1) == 1;
            const int set = T == 2 ? j : j >> 1;
            const int row = set * 4 + q;  // [group][token][digit pair] of the lane's columns
            if (first) {
                if constexpr (TYPE == GX_Q4_0) c = reinterpret_cast<const int4 *>(x + INIT)[row];
                else c = make_int4(kOffset, kOffset, kOffset, kOffset);
            }
            const uint2 b = *reinterpret_cast<const uint2 *>(x + at[j]);
            asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                : "+r"(c.x), "+r"(c.y), "+r"(c.z), "+r"(c.w)
                : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
            if (!last) continue;
            constexpr float off = 12582912.f;
            const float f0 = __int_as_float(c.x) - off, f1 = __int_as_float(c.y) - off;
            const float f2 = __int_as_float(c.z) - off, f3 = __int_as_float(c.w) - off;
            acc[0] = fmaf(half_value(u.d[set], 0), fmaf(f1, v1, f0 * v0), acc[0]);
            acc[1] = fmaf(half_value(u.d[set], 1), fmaf(f3, v1, f2 * v0), acc[1]);
            if constexpr (TYPE == GX_Q4_1) {
                const float sx = reinterpret_cast<const float *>(x + SUM)[row];
                acc[0] = fmaf(half_value(u.m[set], 0), sx, acc[0]);
                acc[1] = fmaf(half_value(u.m[set], 1), sx, acc[1]);
            }
        }
    }
    __device__ __forceinline__ void put(float *dst, int lane) {  // [token][16 rows]
        const int g = lane >> 2, q = lane & 3;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            acc[k] += __shfl_xor_sync(0xffffffffu, acc[k], 1);
            if (T == 1) acc[k] += __shfl_xor_sync(0xffffffffu, acc[k], 2);
        }
        if (T == 1 ? q == 0 : (q & 1) == 0) {
            dst[(q >> 1) * 16 + g] = acc[0];
            dst[(q >> 1) * 16 + g + 8] = acc[1];
        }
    }
    __device__ __forceinline__ void clear() { acc[0] = acc[1] = 0.f; }
};

// Halves: more tokens, P product columns of f16: a token takes one in bf16 and two in f32 (its upper
// and lower part). P = 4 leaves columns free, which a second group takes as in Ints.
template <uint32_t TYPE, bool XB, int P>
struct Halves {
    static constexpr int NT = P <= 8 ? 1 : P / 8, GPC = P < 8 ? 8 / P : 1, SETS = 4 / GPC, ATS = GPC > 1 ? 4 : NT;
    static constexpr int TOK = XB ? P : P / 2, NA = XB ? 4 : 2, kDepth = TYPE == GX_Q4_0 || P < 8 ? 3 : 2;
    static constexpr int CTAS(int W) { return W == 16 ? 1 : P <= 8 ? 3 : 2; }
    // [4 groups][P columns][4 q] 16 B: x of columns (0,4) (2,6) (1,5) (3,7) of 8 q ..
    static constexpr int GROUP = P * 64, ZERO = 4 * GROUP;        // GPC > 1: 64 B of zeros
    static constexpr int SUM = ZERO + (GPC > 1 ? 64 : 0);         // Q4_1: [group][token] float: sum x
    static constexpr int INV = SUM + (TYPE == GX_Q4_1 ? 4 * TOK * 4 : 0);  // [token] float: 1 / scale
    static constexpr int BYTES = (INV + TOK * 4 + 15) / 16 * 16;

    int at[ATS];          // the lane's fragment in each tile of a group; GPC > 1: in each group
    float acc[NT][NA];    // XB: (row g, token c), (g, c + 1), (g + 8, c), (g + 8, c + 1), c = 8 n + 2 q mod P;
                          // f32: (row g, token c / 2), (row g + 8, token c / 2)

    __device__ __forceinline__ void init(int lane, int nt) {
        // Columns without a token read the first one's fragment where nothing is stored of their sums,
        // and the zeros where a column's sums meet those of others.
        const int g = lane >> 2, q = lane & 3, live = XB ? nt : 2 * nt;
#pragma unroll
        for (int k = 0; k < ATS; ++k) {
            if constexpr (GPC > 1) at[k] = (g / P == k % GPC && g % P < live ? k * GROUP + g % P * 64 : ZERO) + q * 16;
            else at[k] = (8 * k + g < live ? 8 * k + g : 0) * 64 + q * 16;
        }
    }
    static __device__ __forceinline__ int scale_offset(int lane) {
        return P == 4 ? (lane >> 1) * 4 + (lane >> 2) * 8 : (lane >> 2) * 16;
    }
    static __device__ void stage(const Q4Args &a, int t0, int nt, int u0, int nu, uint8_t *smem, bool vec, int tid, int nthreads) {
        const int cells = nu * 16, total = nt * cells;
        for (int base = 0; base < total; base += nthreads) {
            const int i = base + tid;
            const bool on = i < total;
            const int t = on ? i / cells : 0, cell = on ? i % cells : 0, q = cell & 3, j = (cell >> 2) & 3;
            float v[8];
            const uint32_t e = load_cell<XB>(a, t0 + t, u0 * kUnitCols + cell * 8, on, vec, v) >> 23, se = min(268u - e, 247u);
            const float s = __uint_as_float(se << 23);
            float ss = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                v[k] = e == 255u ? __uint_as_float(0x7fffffffu) : v[k] * s;
                ss += v[k];
            }
            if constexpr (TYPE == GX_Q4_1) ss = quad_sum(ss);
            if (!on) continue;
            uint8_t *u = smem + (cell >> 4) * BYTES;
            put_fragment<XB>(u + j * GROUP, t, q, v);
            if (TYPE == GX_Q4_1 && q == 0) reinterpret_cast<float *>(u + SUM)[j * TOK + t] = ss;
            if ((cell & 15) == 0) reinterpret_cast<float *>(u + INV)[t] = __uint_as_float((254u - se) << 23);
            if (GPC > 1 && (cell & 12) == 0) reinterpret_cast<uint4 *>(u + ZERO)[q] = make_uint4(0u, 0u, 0u, 0u);
        }
    }
    __device__ __forceinline__ void unit(const Unit<TYPE, SETS> &u, const uint8_t *x, int lane) {
        const int q = lane & 3;
        const uint32_t c0[4] = {u.c0.x, u.c0.y, u.c0.z, u.c0.w}, c1[4] = {u.c1.x, u.c1.y, u.c1.z, u.c1.w};
        float part[NT][NA], c[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < NA; ++k) part[n][k] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t a0[4], a1[4];
            code_fragments<TYPE>(c0[j], c1[j], a0, a1);
            const int jj = j % GPC, set = j / GPC;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint4 b = *reinterpret_cast<const uint4 *>(x + (GPC > 1 ? at[j] : j * GROUP + at[n]));
                if (jj == 0) mma16816_first(c[n], a0, b.x, b.y);
                else mma16816(c[n], a0, b.x, b.y);
                mma16816(c[n], a1, b.z, b.w);
            }
            if (jj != GPC - 1) continue;
            const float d0 = half_value(u.d[set], 0), d1 = half_value(u.d[set], 1);
            const float *sum = reinterpret_cast<const float *>(x + SUM) + (set * GPC + (2 * q) / P) * TOK;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int col = 8 * n + (2 * q) % P;
                if constexpr (XB) {
                    part[n][0] = fmaf(d0, c[n][0], part[n][0]);
                    part[n][1] = fmaf(d0, c[n][1], part[n][1]);
                    part[n][2] = fmaf(d1, c[n][2], part[n][2]);
                    part[n][3] = fmaf(d1, c[n][3], part[n][3]);
                    if constexpr (TYPE == GX_Q4_1) {
                        const float2 sx = *reinterpret_cast<const float2 *>(sum + col);
                        const float m0 = half_value(u.m[set], 0), m1 = half_value(u.m[set], 1);
                        part[n][0] = fmaf(m0, sx.x, part[n][0]);
                        part[n][1] = fmaf(m0, sx.y, part[n][1]);
                        part[n][2] = fmaf(m1, sx.x, part[n][2]);
                        part[n][3] = fmaf(m1, sx.y, part[n][3]);
                    }
                } else {
                    part[n][0] = fmaf(d0, c[n][0] + c[n][1], part[n][0]);
                    part[n][1] = fmaf(d1, c[n][2] + c[n][3], part[n][1]);
                    if constexpr (TYPE == GX_Q4_1) {
                        part[n][0] = fmaf(half_value(u.m[set], 0), sum[col / 2], part[n][0]);
                        part[n][1] = fmaf(half_value(u.m[set], 1), sum[col / 2], part[n][1]);
                    }
                }
            }
        }
        const float *inv = reinterpret_cast<const float *>(x + INV);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int col = 8 * n + (2 * q) % P;
            if constexpr (XB) {
                const float2 iv = *reinterpret_cast<const float2 *>(inv + col);
                acc[n][0] = fmaf(part[n][0], iv.x, acc[n][0]);
                acc[n][1] = fmaf(part[n][1], iv.y, acc[n][1]);
                acc[n][2] = fmaf(part[n][2], iv.x, acc[n][2]);
                acc[n][3] = fmaf(part[n][3], iv.y, acc[n][3]);
            } else {
                acc[n][0] = fmaf(part[n][0], inv[col / 2], acc[n][0]);
                acc[n][1] = fmaf(part[n][1], inv[col / 2], acc[n][1]);
            }
        }
    }
    __device__ __forceinline__ void put(float *dst, int lane) {
        const int g = lane >> 2, q = lane & 3;
        if constexpr (GPC > 1) {  // P == 4: lanes q and q + 2 hold two groups of the same tokens
#pragma unroll
            for (int k = 0; k < NA; ++k) acc[0][k] += __shfl_xor_sync(0xffffffffu, acc[0][k], 2);
            if (q >= P / 2) return;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int col = 8 * n + 2 * q;
            if constexpr (XB) {
                dst[col * 16 + g] = acc[n][0];
                dst[(col + 1) * 16 + g] = acc[n][1];
                dst[col * 16 + g + 8] = acc[n][2];
                dst[(col + 1) * 16 + g + 8] = acc[n][3];
            } else {
                dst[col / 2 * 16 + g] = acc[n][0];
                dst[col / 2 * 16 + g + 8] = acc[n][1];
            }
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < NA; ++k) acc[n][k] = 0.f;
    }
};

constexpr int kMaxSmem = 227 * 1024, kStaticSmem = 1024;  // of a CTA; what of it is not dynamic, at most

// Lets a kernel use all of it, once per device (a call for every launch costs 0.5 us).
struct SmemLimit {
    std::atomic<uint64_t> done{0};
    template <typename K>
    cudaError_t raise(K *k) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess || (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1))) return e;
        e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem - kStaticSmem);
        if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
        return e;
    }
};

struct GemvPlan {
    int RT, KT;      // row tiles, units in a row
    int S;           // CTAs of a cluster that split the columns
    int WK;          // warps of a CTA that split its columns; W / WK row tiles at a time
    int t0, nt;      // tokens of this launch
    int vec;         // activations can be read 16 bytes at a time
    int red_off;
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(const float *p, uint32_t rank) {
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

__device__ __forceinline__ float4 ld_cluster4(const float *p, uint32_t rank) {
    uint32_t at;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}

// Row tiles go to groups of WK warps, in turn over the grid; the warps of a group take the units of
// a row tile in turn, with kDepth units in flight in registers across row tiles, and add their parts
// in shared memory. With S > 1 each cluster has one pass of row tiles, its CTAs take S ranges of the
// units, and rank 0 adds their parts.
template <uint32_t TYPE, class M, int W>
__global__ void __launch_bounds__(W * 32, M::CTAS(W)) q4_gemv_kernel(Q4Args a, GemvPlan p) {
    constexpr int kDepth = M::kDepth, RED = kTileRows * M::TOK;
    extern __shared__ __align__(16) uint8_t smem[];
    float *red = reinterpret_cast<float *>(smem + p.red_off);  // [2][W][RED]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = p.S > 1 ? (int)cluster_rank() : 0;
    const int u0 = (int)((long long)p.KT * rank / p.S), u1 = (int)((long long)p.KT * (rank + 1) / p.S), nu = u1 - u0;
    const int groups = W / p.WK, wg = warp / p.WK, wk = warp % p.WK;
    const int step = (int)(gridDim.x / p.S) * groups;
    const int rt0 = (int)(blockIdx.x / p.S) * groups + wg;

    // cursor of the loads: the next unit of this warp, units left of its row tile, row tiles left
    constexpr int UB = unit_bytes(TYPE);
    const bool idle = wk >= nu;  // more warps than units: this one only takes part in the sums
    const int per = idle ? 0 : (nu - wk + p.WK - 1) / p.WK, scale = 1024 + M::scale_offset(lane) - lane * 16;
    const uint8_t *lp = a.w + ((size_t)rt0 * p.KT + u0 + wk) * UB + lane * 16;
    int lleft = per, ltiles = rt0 < p.RT && !idle ? (p.RT - rt0 + step - 1) / step : 0;
    const int unit_step = p.WK * UB;
    const long long tile_step = (long long)step * p.KT * UB - (long long)(per - 1) * unit_step;
    Unit<TYPE, M::SETS> buf[kDepth];
    auto fetch = [&](Unit<TYPE, M::SETS> &u) {
        if (ltiles > 0) {
            load_unit(u, lp, scale);
            if (--lleft == 0) {
                lleft = per;
                --ltiles;
                lp += tile_step;
            } else {
                lp += unit_step;
            }
        }
    };
#pragma unroll
    for (int k = 0; k < kDepth; ++k) fetch(buf[k]);
    pdl_launch_dependents();
    pdl_wait();  // the weights never change; the activations may come from the kernel before
    M::stage(a, p.t0, p.nt, u0, nu, smem, p.vec != 0, tid, W * 32);
    __syncthreads();

    M m;
    m.init(lane, p.nt);
    m.clear();
    int rt = rt0, left = per, parity = 0;
    const uint8_t *x = smem + wk * M::BYTES;  // the activations of the next unit
    auto finish = [&]() {  // the row tile rt is complete in this warp
        float *mine = red + (size_t)(parity * W + warp) * RED;
        m.put(mine, lane);
        if (p.WK > 1) {
            asm volatile("bar.sync %0, %1;" ::"r"(1 + wg), "r"(32 * p.WK) : "memory");
        } else {
            __syncwarp();
        }
        const float *all = red + (size_t)(parity * W + wg * p.WK) * RED;
        float *keep = red + (size_t)(parity * W + wg * p.WK) * RED;
        for (int i = wk * 32 + lane; i < 16 * p.nt; i += 32 * p.WK) {
            float s = all[i];
            for (int k = 1; k < p.WK; ++k) s += all[(size_t)k * RED + i];
            if (p.S > 1) keep[i] = s;
            else if (rt * 16 + (i & 15) < a.rows)
                store_act(a.y, a.y_bf16, (size_t)(p.t0 + (i >> 4)) * a.ldy + rt * 16 + (i & 15), s);
        }
        if (p.WK == 1) __syncwarp();
        parity ^= 1;
        rt += step;
        m.clear();
    };
    if (idle) {
        while (rt < p.RT) finish();
    }
    while (rt < p.RT) {
#pragma unroll
        for (int k = 0; k < kDepth; ++k) {
            if (rt >= p.RT) break;
            m.unit(buf[k], x, lane);
            fetch(buf[k]);
            x += p.WK * M::BYTES;
            if (--left == 0) {
                finish();
                left = per;
                x = smem + wk * M::BYTES;
            }
        }
    }
    if (p.S > 1) {  // one pass: the sums lie in parity 0
        cluster_sync_all();
        if (rank == 0 && rt0 < p.RT) {
            const float *all = red + (size_t)(wg * p.WK) * RED;
            for (int i = wk * 32 + lane; i < 16 * p.nt; i += 32 * p.WK) {
                float s = all[i];
                for (int r = 1; r < p.S; ++r) s += ld_cluster(all + i, (uint32_t)r);
                if (rt0 * 16 + (i & 15) < a.rows)
                    store_act(a.y, a.y_bf16, (size_t)(p.t0 + (i >> 4)) * a.ldy + rt0 * 16 + (i & 15), s);
            }
        }
        cluster_sync_all();  // no CTA leaves while its part is read
    }
}

template <uint32_t TYPE, class M, int W>
cudaError_t launch_gemv_w(const Q4Args &a, GemvPlan p, int smem, int grid, cudaStream_t s) {
    auto *k = q4_gemv_kernel<TYPE, M, W>;
    static SmemLimit limit;
    const cudaError_t e = limit.raise(k);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(W * 32);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)p.S;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.S > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, k, a, p);
}

template <uint32_t TYPE, bool XB, class M>
cudaError_t launch_gemv(const Q4Args &a, int t0, int nt, int sm_count, cudaStream_t s) {
    GemvPlan p{};
    p.RT = (a.rows + kTileRows - 1) / kTileRows;
    p.KT = (a.cols + kUnitCols - 1) / kUnitCols;
    p.t0 = t0;
    p.nt = nt;
    const size_t esz = XB ? 2 : 4;
    p.vec = ((uintptr_t)a.x & 15) == 0 && (a.ldx * esz) % 16 == 0;
    // Enough warps for 16 on every SM: first the warps of a CTA split a row's units (down to two
    // units a warp), then the CTAs of a cluster do.
    const long long want = 16ll * sm_count;
    p.S = 1;
    p.WK = 1;
    while (p.WK < 8 && (long long)p.RT * p.WK < want && p.KT >= 4 * p.WK) p.WK *= 2;
    while (p.S < 8 && (long long)p.RT * p.WK * p.S < want && p.KT >= 4 * p.WK * p.S) p.S *= 2;
    // the activations of a CTA's units have to fit
    while (p.S < 8 && (long long)((p.KT + p.S - 1) / p.S) * M::BYTES > 100 * 1024) p.S *= 2;
    const int xbytes = (p.KT + p.S - 1) / p.S * M::BYTES;
    const bool wide = xbytes > 56 * 1024;  // few CTAs fit an SM: 16 warps each instead of 8
    const int W = wide ? 16 : 8;
    p.red_off = xbytes;
    const int smem = p.red_off + 2 * W * kTileRows * M::TOK * 4;
    if (smem > kMaxSmem - kStaticSmem) return cudaErrorInvalidValue;
    const int groups = W / p.WK, need = (p.RT + groups - 1) / groups;
    const int resident = sm_count * M::CTAS(W);
    const int grid = p.S > 1 ? need * p.S : need < resident ? need : resident;
    return wide ? launch_gemv_w<TYPE, M, 16>(a, p, smem, grid, s) : launch_gemv_w<TYPE, M, 8>(a, p, smem, grid, s);
}

// ---- more tokens: a tiled product on mma.sync ---------------------------------------------------
// The activations are packed once per call (q4_pack_kernel) into the same fragments, at one scale per
// token, in a workspace of the context: [unit][4 groups][COLS columns][4 q] 16 B, then the group sums
// [4 groups][TOK tokens] of the unit; the tokens' inverse scales stand before the first unit. (A scale and
// a CTA per token and range of units packs no faster, and the product then waits 2 us longer for it.)
constexpr int kQ4InvBytes = 64 * 4;

struct GemmPlan {
    int RT, KT;
    int WM, WK;      // warps: row tiles of a CTA, and splits of its units
    int S;           // CTAs of a cluster that split the units
    int vec;
};

constexpr int kPackThreads = 512;

// One CTA per token.
template <uint32_t TYPE, bool XB>
__global__ void __launch_bounds__(kPackThreads) q4_pack_kernel(Q4Args a, uint8_t *ws, int KT, int cols_padded, int vec) {
    __shared__ uint32_t red[kPackThreads / 32];
    const int t = blockIdx.x, tid = threadIdx.x, cells = KT * 16;
    const int tok_padded = XB ? cols_padded : cols_padded / 2;
    const size_t unit = (size_t)cols_padded * 256 + (size_t)tok_padded * 16;
    pdl_launch_dependents();
    pdl_wait();
    auto load = [&](int cell, float (&v)[8]) {
        const int col = cell * 8;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = 0.f;
        if (cell < cells && col < a.cols) {
            const size_t at = (size_t)t * a.ldx + col;
            if (vec) load_x8(a.x, XB, at, v);
            else {
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = load_act(a.x, XB, at + k);
            }
        }
    };
    float first[8];
    load(tid, first);
    uint32_t big = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) big = max(big, __float_as_uint(first[k]) & 0x7fffffffu);
    for (int cell = tid + kPackThreads; cell < cells; cell += kPackThreads) {
        float v[8];
        load(cell, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) big = max(big, __float_as_uint(v[k]) & 0x7fffffffu);
    }
    big = __reduce_max_sync(0xffffffffu, big);
    if ((tid & 31) == 0) red[tid >> 5] = big;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kPackThreads / 32; ++w) big = max(big, red[w]);
    const uint32_t e = big >> 23, se = min(268u - e, 247u);
    const float s = __uint_as_float(se << 23);
    if (tid == 0) reinterpret_cast<float *>(ws)[t] = __uint_as_float((254u - se) << 23);
    uint8_t *units = ws + kQ4InvBytes;
    for (int base = 0; base < cells; base += kPackThreads) {  // cells is a multiple of 16: quads stay together
        const int cell = base + tid;
        float v[8];
        if (base == 0) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = first[k];
        } else {
            load(cell, v);
        }
        float ss = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            v[k] = e == 255u ? __uint_as_float(0x7fffffffu) : v[k] * s;
            ss += v[k];
        }
        if constexpr (TYPE == GX_Q4_1) ss = quad_sum(ss);
        if (cell >= cells) continue;
        const int q = cell & 3, j = (cell >> 2) & 3;
        uint8_t *u = units + (size_t)(cell >> 4) * unit;
        put_fragment<XB>(u + (size_t)j * cols_padded * 64, t, q, v);
        if (TYPE == GX_Q4_1 && q == 0) reinterpret_cast<float *>(u + (size_t)cols_padded * 256)[j * tok_padded + t] = ss;
    }
}

constexpr int kGemmWarps = 8;
constexpr int gemm_stages(int MT) { return MT == 2 ? 3 : 2; }

// acc += d * c, both halves in one instruction.
__device__ __forceinline__ void fma2(float2 &acc, float d, float2 c) {
    asm("{\n.reg .b64 a, b, d;\n"
        "mov.b64 a, {%0, %1};\nmov.b64 d, {%2, %2};\nmov.b64 b, {%3, %4};\n"
        "fma.rn.f32x2 a, d, b, a;\nmov.b64 {%0, %1}, a;\n}"
        : "+f"(acc.x), "+f"(acc.y)
        : "f"(d), "f"(c.x), "f"(c.y));
}
__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// A CTA takes WM row tiles by all tokens over its range of units: warp (wk, wm) one row tile of every
// WK-th unit, NB product tiles wide, so that a code is unpacked once. Codes and fragments come by bulk
// copies through a ring of shared-memory stages of WK units; the parts are added over wk and the
// cluster's CTAs at the end.
template <uint32_t TYPE, bool XB, int NB, int MT>
__global__ void __launch_bounds__(kGemmWarps * 32, 2) q4_gemm_kernel(Q4Args a, const uint8_t *ws, GemmPlan p) {
    constexpr int UB = unit_bytes(TYPE), COLS = 8 * NB, TOK = XB ? COLS : COLS / 2;
    constexpr int BU = COLS * 256 + TOK * 16;  // a unit's fragments and sums
    constexpr int kGemmStages = gemm_stages(MT);
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[kGemmStages], empty[kGemmStages];  // a stage has come; all warps have read it
    __shared__ float inv[64];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
    const int wm = warp % p.WM, wk = warp / p.WM;
    const int unit_stage = BU + MT * p.WM * UB, stage_bytes = p.WK * unit_stage;
    const int rank = p.S > 1 ? (int)cluster_rank() : 0;
    const int u0 = (int)((long long)p.KT * rank / p.S), u1 = (int)((long long)p.KT * (rank + 1) / p.S), nu = u1 - u0;
    const int rt0 = (int)(blockIdx.x / p.S) * p.WM * MT, iters = (nu + p.WK - 1) / p.WK;
    const int tiles = min(p.WM * MT, p.RT - rt0);
    const uint8_t *units = ws + kQ4InvBytes;

    auto copy_codes = [&](int it) {  // and the bytes that the stage waits for
        const int n = min(p.WK, nu - it * p.WK);
        mbar_expect_tx(&bars[it % kGemmStages], (uint32_t)(n * (BU + tiles * UB)));
        for (int k = 0; k < n; ++k)
            for (int t = 0; t < tiles; ++t)
                bulk_g2s(smem + (it % kGemmStages) * stage_bytes + k * unit_stage + BU + t * UB,
                         a.w + ((size_t)(rt0 + t) * p.KT + u0 + it * p.WK + k) * UB, UB, &bars[it % kGemmStages]);
    };
    auto copy_frags = [&](int it) {
        const int n = min(p.WK, nu - it * p.WK);
        for (int k = 0; k < n; ++k)
            bulk_g2s(smem + (it % kGemmStages) * stage_bytes + k * unit_stage, units + (size_t)(u0 + it * p.WK + k) * BU, BU,
                     &bars[it % kGemmStages]);
    };
    if (tid == 0) {
        for (int i = 0; i < kGemmStages; ++i) {
            mbar_init(&bars[i], 1);
            mbar_init(&empty[i], kGemmWarps);
        }
        fence_barrier_init();
        // the weights never change: they may be fetched before the activations are packed
        for (int i = 0; i < kGemmStages && i < iters; ++i) copy_codes(i);
    }
    __syncthreads();
    pdl_launch_dependents();
    pdl_wait();
    if (tid == 0)
        for (int i = 0; i < kGemmStages && i < iters; ++i) copy_frags(i);
    if (tid < 64) inv[tid] = tid < a.n_tok ? reinterpret_cast<const float *>(ws)[tid] : 0.f;

    // sums of (row g; row g + 8) of columns 2 q and 2 q + 1: two tokens in bf16, the parts of one in f32
    float2 acc[MT][NB][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NB; ++n) acc[m][n][0] = acc[m][n][1] = make_float2(0.f, 0.f);
    bool ok = true;  // an expired wait is reported and ends the warp's loop
    int copied = min(iters, kGemmStages);
    for (int it = 0; it < iters; ++it) {
        ok = mbar_wait(&bars[it % kGemmStages], (uint32_t)(it / kGemmStages & 1), a.err);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (it * p.WK + wk < nu && wm * MT < tiles) {
            const uint8_t *st = smem + (it % kGemmStages) * stage_bytes + wk * unit_stage;
            const float *sums = reinterpret_cast<const float *>(st + COLS * 256);
            const uint8_t *t = st + BU + wm * MT * UB;  // a tile past the matrix holds what was there: nothing of it is stored
            const uint32_t *codes = reinterpret_cast<const uint32_t *>(t) + lane * 4;
            const uint32_t *scales = reinterpret_cast<const uint32_t *>(t + 1024) + g * 4;
#pragma unroll 1
            for (int j = 0; j < 4; ++j) {
                uint32_t a0[MT][4], a1[MT][4], mw[MT];
                float d0[MT], d1[MT];
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    code_fragments<TYPE>(codes[m * (UB / 4) + j], codes[m * (UB / 4) + j + 128], a0[m], a1[m]);
                    d0[m] = half_value(scales[m * (UB / 4) + j], 0);
                    d1[m] = half_value(scales[m * (UB / 4) + j], 1);
                    if constexpr (TYPE == GX_Q4_1) mw[m] = scales[m * (UB / 4) + j + 32];
                }
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    const uint4 b = *reinterpret_cast<const uint4 *>(st + ((j * COLS + 8 * n) * 4 + lane) * 16);
                    float2 sx = make_float2(0.f, 0.f);
                    if constexpr (TYPE == GX_Q4_1) {
                        if constexpr (XB) sx = *reinterpret_cast<const float2 *>(sums + j * TOK + 8 * n + 2 * q);
                        else sx.x = sums[j * TOK + 4 * n + q];
                    }
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        float c[4];
                        mma_group(c, a0[m], a1[m], b);
                        fma2(acc[m][n][0], d0[m], make_float2(c[0], c[1]));
                        fma2(acc[m][n][1], d1[m], make_float2(c[2], c[3]));
                        if constexpr (TYPE == GX_Q4_1) {
                            fma2(acc[m][n][0], half_value(mw[m], 0), sx);
                            fma2(acc[m][n][1], half_value(mw[m], 1), sx);
                        }
                    }
                }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[it % kGemmStages]);
        // the first warp refills the stage of the step before, which the others have likely left by now
        if (tid == 0 && it > 0 && copied < iters && ok) {
            ok = mbar_wait(&empty[(it - 1) % kGemmStages], (uint32_t)((it - 1) / kGemmStages & 1), a.err);
            if (ok) {
                copy_codes(copied);
                copy_frags(copied);
                ++copied;
            }
        }
    }
    if (!__syncthreads_and(ok) && tid == 0)  // no copy may outlive the CTA
        for (int it = copied > kGemmStages ? copied - kGemmStages : 0; it < copied; ++it)
            mbar_wait(&bars[it % kGemmStages], (uint32_t)(it / kGemmStages & 1), nullptr);
    __syncthreads();
    // parts [WK][TOK][rows + 8] over the stages
    const int rows = MT * p.WM * 16, ld = rows + 8, part = TOK * ld;
    float *mine = reinterpret_cast<float *>(smem) + wk * part;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const int t = XB ? 8 * n + 2 * q : 4 * n + q;
        const float i0 = inv[t], i1 = XB ? inv[t + 1] : 0.f;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int r = (wm * MT + m) * 16 + g;
            if constexpr (XB) {
                mine[t * ld + r] = acc[m][n][0].x * i0;
                mine[(t + 1) * ld + r] = acc[m][n][0].y * i1;
                mine[t * ld + r + 8] = acc[m][n][1].x * i0;
                mine[(t + 1) * ld + r + 8] = acc[m][n][1].y * i1;
            } else {
                mine[t * ld + r] = (acc[m][n][0].x + acc[m][n][0].y) * i0;
                mine[t * ld + r + 8] = (acc[m][n][1].x + acc[m][n][1].y) * i0;
            }
        }
    }
    if (p.S > 1) cluster_sync_all();
    else __syncthreads();
    // the CTAs of a cluster share the sums out, four rows of a token to a thread
    const float *all = reinterpret_cast<const float *>(smem);
    for (int i = rank * kGemmWarps * 32 + tid; i < a.n_tok * rows / 4; i += p.S * kGemmWarps * 32) {
        const int t = i / (rows / 4), r = (i - t * (rows / 4)) * 4, row = rt0 * 16 + r;
        if (row >= a.rows) continue;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k = 0; k < p.WK; ++k) {
            const float *at = all + k * part + t * ld + r;
            float4 v[8];  // all parts on their way before the first is added
#pragma unroll
            for (int c = 0; c < 8; ++c)
                if (c < p.S) v[c] = p.S > 1 ? ld_cluster4(at, (uint32_t)c) : *reinterpret_cast<const float4 *>(at);
#pragma unroll
            for (int c = 0; c < 8; ++c)
                if (c < p.S) {
                    s.x += v[c].x;
                    s.y += v[c].y;
                    s.z += v[c].z;
                    s.w += v[c].w;
                }
        }
        const size_t o = (size_t)t * a.ldy + row;
        const float out[4] = {s.x, s.y, s.z, s.w};
        for (int k = 0; k < 4 && row + k < a.rows; ++k) store_act(a.y, a.y_bf16, o + k, out[k]);
    }
    if (p.S > 1) cluster_sync_all();  // no CTA leaves while its parts are read
}

template <uint32_t TYPE, bool XB, int NB, int MT>
cudaError_t launch_gemm_mt(const Q4Args &a, uint8_t *ws, int sm_count, cudaStream_t s) {
    constexpr int COLS = 8 * NB, TOK = XB ? COLS : COLS / 2, BU = COLS * 256 + TOK * 16;
    GemmPlan p{};
    p.RT = (a.rows + kTileRows - 1) / kTileRows;
    p.KT = (a.cols + kUnitCols - 1) / kUnitCols;
    p.WM = kGemmWarps;
    p.WK = p.S = 1;
    // CTAs for one and a half on every SM: first the CTAs of a cluster split the units (down to two units
    // a CTA), then fewer row tiles and more splits in a CTA.
    auto ctas = [&] { return (p.RT + MT * p.WM - 1) / (MT * p.WM) * p.S; };
    auto ring = [&](int wm, int wk) { return gemm_stages(MT) * wk * (BU + MT * wm * unit_bytes(TYPE)); };
    while (p.S < 8 && ctas() < sm_count * 3 / 2 && p.KT >= 4 * p.S) p.S *= 2;
    while (p.WM > 1 && ctas() < sm_count * 3 / 2 && p.KT >= 4 * p.S * p.WK && ring(p.WM / 2, p.WK * 2) <= kMaxSmem / 2) {
        p.WM /= 2;
        p.WK *= 2;
    }
    const int parts = p.WK * TOK * (MT * p.WM * 16 + 8) * 4;
    const int smem = ring(p.WM, p.WK) > parts ? ring(p.WM, p.WK) : parts;
    if (smem > kMaxSmem - kStaticSmem) return cudaErrorInvalidValue;
    p.vec = ((uintptr_t)a.x & 15) == 0 && a.ldx * (XB ? 2 : 4) % 16 == 0;
    cudaError_t e = launch_chain_pdl(true, q4_pack_kernel<TYPE, XB>, dim3((unsigned)a.n_tok), dim3(kPackThreads), 0, s, a, ws,
                                     p.KT, COLS, p.vec);
    if (e != cudaSuccess) return e;
    auto *k = q4_gemm_kernel<TYPE, XB, NB, MT>;
    static SmemLimit limit;
    e = limit.raise(k);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas());
    cfg.blockDim = dim3(kGemmWarps * 32);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)p.S;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.S > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, k, a, (const uint8_t *)ws, p);
}

template <uint32_t TYPE, bool XB, int NB>
cudaError_t launch_gemm(const Q4Args &a, uint8_t *ws, int sm_count, cudaStream_t s) {
    if constexpr (NB <= 8) {  // two row tiles by more columns do not fit the registers
        if (a.rows >= 4096) return launch_gemm_mt<TYPE, XB, NB, 2>(a, ws, sm_count, s);
    }
    return launch_gemm_mt<TYPE, XB, NB, 1>(a, ws, sm_count, s);
}

template <uint32_t TYPE, bool XB>
cudaError_t launch_tokens(const Q4Args &a, uint8_t *ws, int sm_count, cudaStream_t s) {
    constexpr int T1 = XB ? 8 : 4;
    if (a.n_tok > 2 * T1) {  // up to 64 tokens: 8 product tiles in bf16, 16 in f32
        const int tiles = (a.n_tok + T1 - 1) / T1;
        if (tiles <= 4) return launch_gemm<TYPE, XB, 4>(a, ws, sm_count, s);
        if (tiles <= 6) return launch_gemm<TYPE, XB, 6>(a, ws, sm_count, s);
        if (tiles <= 8) return launch_gemm<TYPE, XB, 8>(a, ws, sm_count, s);
        if constexpr (!XB) {
            if (tiles <= 12) return launch_gemm<TYPE, XB, 12>(a, ws, sm_count, s);
            return launch_gemm<TYPE, XB, 16>(a, ws, sm_count, s);
        }
    }
    // 16 columns where their activations fit the cluster's shared memory, else 8 at a time
    const int KT = (a.cols + kUnitCols - 1) / kUnitCols;
    const int most = ((KT + 7) / 8) * Halves<TYPE, XB, 16>::BYTES <= 160 * 1024 ? 2 * T1 : T1;
    for (int t0 = 0; t0 < a.n_tok; t0 += most) {
        const int nt = a.n_tok - t0 < most ? a.n_tok - t0 : most, cols = XB ? nt : 2 * nt;
        const cudaError_t e = nt == 1     ? launch_gemv<TYPE, XB, Ints<TYPE, XB, 1>>(a, t0, nt, sm_count, s)
                              : nt == 2   ? launch_gemv<TYPE, XB, Ints<TYPE, XB, 2>>(a, t0, nt, sm_count, s)
                              : cols <= 4 ? launch_gemv<TYPE, XB, Halves<TYPE, XB, 4>>(a, t0, nt, sm_count, s)
                              : cols <= 8 ? launch_gemv<TYPE, XB, Halves<TYPE, XB, 8>>(a, t0, nt, sm_count, s)
                                          : launch_gemv<TYPE, XB, Halves<TYPE, XB, 16>>(a, t0, nt, sm_count, s);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

uint64_t padded_units(uint64_t rows, uint64_t cols) {
    return (rows + kTileRows - 1) / kTileRows * ((cols + kUnitCols - 1) / kUnitCols);
}

}  // namespace

uint64_t q4_row_bytes(uint32_t type, uint64_t cols) {
    if ((type != GX_Q4_0 && type != GX_Q4_1) || cols % 32) return 0;
    return cols / 32 * (type == GX_Q4_0 ? 18 : 20);
}

uint64_t q4_bytes(uint32_t type, uint64_t rows, uint64_t cols) { return padded_units(rows, cols) * unit_bytes(type); }

cudaError_t launch_q4_repack(uint32_t type, const uint8_t *raw, uint32_t rows, uint32_t cols, uint8_t *w,
                             cudaStream_t s) {
    const long long n = (long long)padded_units(rows, cols) * kTileRows * 4;
    const long long blocks = (n + 255) / 256;
    if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
    q4_repack_kernel<<<(unsigned)blocks, 256, 0, s>>>(type, raw, (int)rows, (int)cols, w, n);
    return cudaGetLastError();
}

uint64_t q4_workspace_bytes(uint64_t cols) {
    // 64 tokens in f32: 128 product columns of 64 B in each of a unit's groups, and 64 sums
    return kQ4InvBytes + (cols + kUnitCols - 1) / kUnitCols * (4 * (128 * 64 + 64 * 4));
}

cudaError_t launch_q4_linear(const Q4Args &a, uint8_t *ws, int sm_count, cudaStream_t s) {
    if (a.n_tok <= 0 || a.rows <= 0) return cudaSuccess;
    if (a.type == GX_Q4_0)
        return a.x_bf16 ? launch_tokens<GX_Q4_0, true>(a, ws, sm_count, s) : launch_tokens<GX_Q4_0, false>(a, ws, sm_count, s);
    return a.x_bf16 ? launch_tokens<GX_Q4_1, true>(a, ws, sm_count, s) : launch_tokens<GX_Q4_1, false>(a, ws, sm_count, s);
}

}  // namespace gx
