// gx_q4.cu — matrix-vector products with 4-bit weights and group scales (GGUF Q4_0 and Q4_1):
//
//   y[t][r] = sum over groups of 32 columns of  d * (sum_c q x[t][c] - 8 sum_c x[t][c])       (Q4_0)
//                                               d *  sum_c q x[t][c] + m sum_c x[t][c]        (Q4_1)
//
// with fp16 d and m per group and 4-bit q.
//
// Up to 16 product columns are a GEMV, more a product on tcgen05 (each below). In the GEMV the sums over a
// group run on mma.sync on the integers q - 8 (Q4_1: q), which f16 and 8-bit integers hold exactly, and d meets
// the group's sum in f32, so no weight is ever rounded. A code in the low bits of an f16 under the exponent of
// 1024 is 1024 + q, four bits higher 1024 + 16 q: one shift, four and-ors and four half2 operations turn a word
// of 8 codes into its four A registers. (Codes as f16 subnormals need no arithmetic at all, but the product then
// aligns its terms by the subnormals' exponent and loses their leading zeros: 2e-6 to 4e-6 relative error
// measured, against 1e-7.) Its activations become fragments in shared memory once per CTA: each unit of 128
// columns of a token is scaled by a power of two that brings its largest value to 2^14..2^15; an f32 value is
// split into two f16 (22 bits, two columns of the product), a bf16 value fits one.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>

#include "../../include/gyro_moe.h"
#include "gx_dense.cuh"
#include "gx_device.cuh"
#include "gx_internal.h"
#include "gx_q4_tc.h"
#include "gx_umma.cuh"

namespace gx {

using namespace dense;

namespace {

// ---- device layout ---------------------------------------------------------------------------
// Units of 16 rows x 128 columns (4 groups), ordered [block of 8 row tiles][unit][row tile], so that one
// bulk copy brings the codes of up to 128 rows; rows and columns past the matrix have zero scales. Lane l = 4 g + q of a warp owns rows g and g + 8 and, in each group, the
// columns 8 q .. 8 q + 7, the k-slices its A registers hold:
//   [32 lanes][4 groups] words of row g     code of column 8 q + i in bits 4 i .. 4 i + 3
//   [32 lanes][4 groups] words of row g + 8
//   [8 g][4 groups][row g, row g + 8] fp16 d
//   [8 g][4 groups][row g, row g + 8] fp16 m   (Q4_1)
constexpr int kUnitCols = 128, kTileRows = 16, kBlockTiles = 8;
// Number of the unit u of the row tile rt, of KT units in a row.
__host__ __device__ constexpr long long unit_index(long long rt, int u, int KT) {
    return (rt / kBlockTiles * KT + u) * kBlockTiles + rt % kBlockTiles;
}

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
    uint8_t *u = w + unit_index(row / kTileRows, grp / 4, NG / 4) * q4_unit_bytes(type);
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
    static constexpr int SUM = INIT;                              // Q4_1: [group][token][digit pair] float: sum x in kUnit, 0
    static constexpr int INV = TYPE == GX_Q4_0 ? INIT + T * 128 : SUM + T * 32;  // [token] float: 2^24 units of the numbers
    static constexpr int BYTES = (INV + T * 4 + 15) / 16 * 16;
    static constexpr uint32_t kOffset = 0x4b400000u;              // 2^23 + 2^22 as a float
    // Of the lane's sums: with Q4_1 in 32nds, since sum x of a group may pass the f32 range where m sum x does not.
    static constexpr float kUnit = TYPE == GX_Q4_1 ? 0x1p-5f : 1.f;

    int at[4];       // the lane's fragment in each group
    float acc[NA];   // rows g and g + 8; T == 2: token q >> 1; odd lanes hold the lower two digits, 2^16 times

    __device__ __forceinline__ void init(int lane, int nt) {
        const int g = lane >> 2, q = lane & 3;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            at[j] = T == 2 ? j * GROUP + ((g >> 2) < nt ? g : (g & 3)) * 32 + q * 8
                           : (g >> 2 == (j & 1) ? j * GROUP + (g & 3) * 32 : ZERO) + q * 8;
    }
    static __device__ __forceinline__ int scale_offset(int lane) {
        return T == 1 ? (lane >> 1) * 4 + (lane >> 2) * 8 : (lane >> 2) * 16;
    }
    static __device__ void stage(const Q4Args &a, int u0, int nu, uint8_t *smem, bool vec, int tid, int nthreads) {
        const int cells = nu * 16, total = a.n_tok * cells;
        for (int base = 0; base < total; base += nthreads) {
            const int i = base + tid;
            const bool on = i < total;
            const int t = on ? i / cells : 0, cell = on ? i % cells : 0, q = cell & 3, j = (cell >> 2) & 3;
            float v[8];
            const uint32_t big = load_cell<XB>(a, t, u0 * kUnitCols + cell * 8, on, vec, v), e = big >> 23;
            // 2^k with the unit's largest value below 2^30, as two factors: it may pass the f32 range
            const int k = 29 + 127 - (int)max(min(e, 254u), 1u), k1 = k / 2, k2 = k - k1;
            const float s1 = __uint_as_float((uint32_t)(127 + k1) << 23), s2 = __uint_as_float((uint32_t)(127 + k2) << 23);
            uint32_t b[8];
            float fs = 0.f;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const float x = e == 255u ? 0.f : v[c] * s1 * s2;
                b[c] = ((uint32_t)__float2int_rn(x) + 0x00808080u) ^ 0x00808080u;  // signed digits, byte by byte
                fs = fmaf(v[c], kUnit, fs);
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
                              : __uint_as_float((uint32_t)(151 - k1) << 23) * __uint_as_float((uint32_t)(127 - k2) << 23) * kUnit;
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
        const float inv = reinterpret_cast<const float *>(x + INV)[T == 1 ? 0 : q >> 1];
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
            // d before the unit's power of two: the sum of x by codes alone may pass the f32 range
            acc[0] = fmaf(half_value(u.d[set], 0) * fmaf(f1, 0x1p-8f, f0), inv, acc[0]);
            acc[1] = fmaf(half_value(u.d[set], 1) * fmaf(f3, 0x1p-8f, f2), inv, acc[1]);
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
            acc[k] *= (q & 1) ? 0x1p-16f / kUnit : 1.f / kUnit;
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
    static __device__ void stage(const Q4Args &a, int u0, int nu, uint8_t *smem, bool vec, int tid, int nthreads) {
        const int cells = nu * 16, total = a.n_tok * cells;
        for (int base = 0; base < total; base += nthreads) {
            const int i = base + tid;
            const bool on = i < total;
            const int t = on ? i / cells : 0, cell = on ? i % cells : 0, q = cell & 3, j = (cell >> 2) & 3;
            float v[8];
            const uint32_t e = load_cell<XB>(a, t, u0 * kUnitCols + cell * 8, on, vec, v) >> 23, se = min(268u - e, 247u);
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

constexpr int kStaticSmem = 1024;  // of a CTA, what is not dynamic, at most

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
    int vec;         // activations can be read 16 bytes at a time
    int red_off;
};

__device__ __forceinline__ uint32_t pack_bf2(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
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

    // cursor of the loads: the next unit of this warp, units left of its row tile, the row tile
    constexpr int UB = q4_unit_bytes(TYPE);
    const bool idle = wk >= nu;  // more warps than units: this one only takes part in the sums
    const int per = idle ? 0 : (nu - wk + p.WK - 1) / p.WK, scale = 1024 + M::scale_offset(lane) - lane * 16;
    auto tile_at = [&](int rt) { return a.w + unit_index(rt, u0 + wk, p.KT) * UB + lane * 16; };
    const uint8_t *lp = tile_at(rt0);
    int lleft = per, lrt = idle ? p.RT : rt0;
    const int unit_step = p.WK * kBlockTiles * UB;
    Unit<TYPE, M::SETS> buf[kDepth];
    auto fetch = [&](Unit<TYPE, M::SETS> &u) {
        if (lrt < p.RT) {
            load_unit(u, lp, scale);
            if (--lleft == 0) {
                lleft = per;
                lrt += step;
                lp = tile_at(lrt);
            } else {
                lp += unit_step;
            }
        }
    };
#pragma unroll
    for (int k = 0; k < kDepth; ++k) fetch(buf[k]);
    pdl_launch_dependents();
    pdl_wait();  // the weights never change; the activations may come from the kernel before
    M::stage(a, u0, nu, smem, p.vec != 0, tid, W * 32);
    __syncthreads();

    M m;
    m.init(lane, a.n_tok);
    m.clear();
    int rt = rt0, left = per, parity = 0;
    const uint8_t *x = smem + wk * M::BYTES;  // the activations of the next unit
    auto finish = [&]() {  // the row tile rt is complete in this warp
        float *mine = red + (size_t)(parity * W + warp) * RED;
        m.put(mine, lane);
        if (p.WK > 1) named_sync(1 + wg, 32 * p.WK);
        else __syncwarp();
        const float *all = red + (size_t)(parity * W + wg * p.WK) * RED;
        float *keep = red + (size_t)(parity * W + wg * p.WK) * RED;
        for (int i = wk * 32 + lane; i < 16 * a.n_tok; i += 32 * p.WK) {
            float s = all[i];
            for (int k = 1; k < p.WK; ++k) s += all[(size_t)k * RED + i];
            if (p.S > 1) keep[i] = s;
            else if (rt * 16 + (i & 15) < a.rows)
                store_act(a.y, a.y_bf16, (size_t)(i >> 4) * a.ldy + rt * 16 + (i & 15), s);
        }
        __syncwarp();  // the product of the next unit takes a whole warp
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
            for (int i = wk * 32 + lane; i < 16 * a.n_tok; i += 32 * p.WK) {
                float s = all[i];
                for (int r = 1; r < p.S; ++r) s += ld_cluster(all + i, (uint32_t)r);
                if (rt0 * 16 + (i & 15) < a.rows)
                    store_act(a.y, a.y_bf16, (size_t)(i >> 4) * a.ldy + rt0 * 16 + (i & 15), s);
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
cudaError_t launch_gemv(const Q4Args &a, int sm_count, cudaStream_t s) {
    GemvPlan p{};
    p.RT = (a.rows + kTileRows - 1) / kTileRows;
    p.KT = (a.cols + kUnitCols - 1) / kUnitCols;
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

// ---- more tokens: a product on tcgen05 ----------------------------------------------------------
// D[128 rows][N] = sum over the columns of w x, in an accumulator in tensor memory. That asks for weights
// that the tensor core can take as they are: d (q - 8) has up to 15 significant bits, and two bf16 hold it
// exactly (Split). Decoder warps write both parts into tensor memory, a lane a row, as A; the packed
// activations are B in shared memory, one column a token in bf16 and three in f32 (8 bits each, all 24).
// No weight and no activation is rounded.
//
// (With d applied to each group's sum afterwards, as in the GEMV, the product needs an accumulator a group,
// read back by warps that multiply: 42 us alone on a stream, 64 bf16 tokens by 8192 x 8192, and 48 to 62 on
// mma.sync; this one takes 28.7.)
//
// What bounds it: the chain of one unit (128 columns) in the issuing thread, three waits, 16 MMAs and three
// commits, more than 0.5 us; the MMAs at their full rate would take 0.15 us, the codes' bytes 0.18. So a unit has
// one full and one empty barrier for its weights, its codes come by one bulk copy (a copy for each of its 8
// row tiles kept the copying thread 0.9 us a unit), and one thread runs the issue loop by itself (a whole
// warp with an elected lane took 4 us more, measured with one accumulator over all units).
//
// Warps: 0 copies, 1 tensor memory and MMA issue, then sets of four decoders that take units in turn, and four
// that read the sums. Three sets: 28.7 us, two: 29.2 (8192 x 8192, 64 bf16 tokens).
constexpr int kTcRows = kTileRows * kBlockTiles;
// An accumulator takes one unit and is then read and added in registers. The tensor core cuts its sum off after each
// of a unit's 16 MMAs, always towards zero. Relative error in the 2-norm before the results are rounded (64 bf16 tokens
// by 8192 x 8192, Q4_0 and Q4_1; a product of the unpacked weights in f32 has 1.5e-6), and time with bf16 results:
//   one unit 1.3e-7, 2.4e-7, 28.7 us;  four 6.2e-7, 8.6e-7, 28.0;  sixteen 2.7e-6, 3.6e-6, 27.7
// (64 f32 tokens: 57.9, 45.9, 43.2 us). Sixteen would do for bf16 results, but put twice as many of them on the other
// side of a rounding's border as the product in f32 does; with one, a bf16 result is the f32 result rounded.
constexpr int kQ4InvBytes = 64 * 4;  // of a workspace: the tokens' inverse scales, before the first unit
constexpr int kPackThreads = 512;

// One CTA per token: its values at the power of two that brings the largest to 2^14..2^15 (a token with an
// Inf or NaN is all NaN), in bf16 parts.
template <uint32_t TYPE, bool XB, int TP>
__global__ void __launch_bounds__(kPackThreads) q4_pack_kernel(Q4Args a, uint8_t *ws, int KT, int vec) {
    using C = Tc<TYPE, XB, TP>;
    __shared__ uint32_t red[kPackThreads / 32];
    const int t = blockIdx.x, tid = threadIdx.x, cells = KT * 16;
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
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = e == 255u ? __uint_as_float(0x7fffffffu) : v[k] * s;
        const int q = cell & 3, j = (cell >> 2) & 3;
        uint8_t *u = units + (size_t)(cell >> 4) * C::BU;
#pragma unroll
        for (int piece = 0; piece < (XB ? 1 : 3); ++piece) {
            const int row = piece * TP + t;
            uint8_t *at = u + (row >> 3) * 1024 + (row & 7) * 128;
            float x[8], ss = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                x[k] = __bfloat162float(__float2bfloat16_rn(v[k]));
                v[k] -= x[k];
                ss += x[k];
            }
            if constexpr (TYPE == GX_Q4_1) ss = quad_sum(ss);
            if (cell >= cells) continue;
            *reinterpret_cast<uint4 *>(at + (j >> 1) * C::N * 128 + (((4 * (j & 1) + q) ^ (row & 7)) << 4)) =
                make_uint4(pack_bf2(x[0], x[4]), pack_bf2(x[1], x[5]), pack_bf2(x[2], x[6]), pack_bf2(x[3], x[7]));
            if (TYPE == GX_Q4_1 && q == 0) {
                const float s1 = __bfloat162float(__float2bfloat16_rn(ss)), s2 = __bfloat162float(__float2bfloat16_rn(ss - s1));
                const float s3 = ss - s1 - s2;
                *reinterpret_cast<uint4 *>(at + 2 * C::N * 128 + ((j ^ (row & 7)) << 4)) =
                    make_uint4(pack_bf2(s1, s2), pack_bf2(s3, s1), pack_bf2(s2, s3), 0u);
            }
        }
    }
}

// The weights of a group as two bf16 each, exactly.
//
// Q4_0: d = d1 + d2, d1 of 5 significant bits (nearest), so d2 has 5 too, and (q - 8) d1, (q - 8) d2 have 8. A
// code in bits 3 .. 6 under the exponent of 128 is 8 (16 + q), and (q - 8) d1 = 8 (16 + q) d1 / 8 - 24 d1 with
// all of it in bf16: one instruction for two weights and each part.
//
// Q4_1: q has 4 bits, which leaves none. d1 of 8 bits, d2 the last 3; hi = bf16(q d1), and lo = q d - hi has 7
// bits at most. Its negative comes out of two multiply-adds, and the product subtracts it.
template <uint32_t TYPE>
struct Split {
    __nv_bfloat162 a, b, c, d;
    __device__ __forceinline__ explicit Split(float scale) {
        if constexpr (TYPE == GX_Q4_0) {
            const float d1 = __uint_as_float((__float_as_uint(scale) + 0x40000u) & 0xfff80000u), d2 = scale - d1;
            a = __float2bfloat162_rn(d1 * 0.125f);
            b = __float2bfloat162_rn(d1 * -24.f);
            c = __float2bfloat162_rn(d2 * 0.125f);
            d = __float2bfloat162_rn(d2 * -24.f);
        } else {
            a = __float2bfloat162_rn(scale);
            const float d1 = __low2float(a);
            b = __float2bfloat162_rn(-d1);
            c = __float2bfloat162_rn(d1 - scale);
        }
    }
    // Codes k and k + 4 of a word.
    __device__ __forceinline__ void pair(uint32_t word, int k, uint32_t &hi, uint32_t &lo) const {
        constexpr int at = TYPE == GX_Q4_0 ? 3 : 0;  // bit of the code
        const int right = 4 * k - at;
        uint32_t v;
        asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(v) : "r"(right < 0 ? word << -right : word >> right), "r"(0x000f000fu << at), "r"(0x43004300u));
        const __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162 *>(&v);
        __nv_bfloat162 h, l;
        if constexpr (TYPE == GX_Q4_0) {
            h = __hfma2(x, a, b);
            l = __hfma2(x, c, d);
        } else {
            const __nv_bfloat162 q = __hadd2(x, __float2bfloat162_rn(-128.f));
            h = __hmul2(q, a);
            l = __hfma2(q, c, __hfma2(q, b, h));
        }
        hi = *reinterpret_cast<const uint32_t *>(&h);
        lo = *reinterpret_cast<const uint32_t *>(&l);
    }
};

struct TcPlan {
    int RT, KT, blocks, S;
};

template <uint32_t TYPE, bool XB, int TP>
__global__ void __launch_bounds__((Tc<TYPE, XB, TP>::THREADS), 1) q4_tc_kernel(Q4Args a, const uint8_t *ws, TcPlan p) {
    using C = Tc<TYPE, XB, TP>;
    constexpr int UB = q4_unit_bytes(TYPE), XS = C::XS, AS = C::AS;
    extern __shared__ __align__(1024) uint8_t tc_raw[];
    __shared__ float inv[64];
    uint8_t *sm = reinterpret_cast<uint8_t *>(((uintptr_t)tc_raw + 1023) & ~(uintptr_t)1023);
    float *red = reinterpret_cast<float *>(sm);  // [TP][128] f32: a cluster's parts, when the stages are done
    uint64_t *full_x = reinterpret_cast<uint64_t *>(sm + C::BARS), *empty_x = full_x + XS;
    uint64_t *full_a = empty_x + XS, *empty_a = full_a + AS;
    uint64_t *full_d = empty_a + AS, *empty_d = full_d + 2, *done = empty_d + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(done + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = p.S > 1 ? (int)cluster_rank() : 0;
    const int u0 = (int)((long long)p.KT * rank / p.S), nu = (int)((long long)p.KT * (rank + 1) / p.S) - u0;
    // row blocks of this CTA: with S > 1 one, else every gridDim.x-th
    const int first = (int)blockIdx.x / p.S, step = (int)gridDim.x / p.S, items = first < p.blocks ? (p.blocks - first + step - 1) / step : 0;
    if (tid == 0) {
        for (int i = 0; i < XS; ++i) {
            mbar_init(&full_x[i], 1);
            mbar_init(&empty_x[i], 1);
        }
        for (int i = 0; i < AS; ++i) {
            mbar_init(&full_a[i], 4);
            mbar_init(&empty_a[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&full_d[i], 1);
            mbar_init(&empty_d[i], 4);
        }
        mbar_init(done, 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    pdl_launch_dependents();
    if (warp == 1) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t a_cols = tmem + (uint32_t)(C::SLOTS * C::SLOT);
    // An expired wait is reported and ends every role of the CTA.
    auto wait = [&](uint64_t *bar, uint32_t parity) -> bool {
        if (mbar_try_wait(bar, parity)) return true;
        if (*abort_flag) return false;
        if (mbar_wait(bar, parity, a.err)) return true;
        *abort_flag = 1;
        return false;
    };
    auto wait_all = [&](uint64_t *bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)); };
    const int total = items * nu;  // units, item by item
    // No bounded wait starts before the activations can be packed, however long the kernel before takes.
    if (warp != 0) pdl_wait();

    if (warp == 0) {
        if (lane == 0) {
            int block = first, u = 0;  // of the next codes
            auto codes = [&](int st) {
                mbar_expect_tx(&full_x[st], (uint32_t)C::STAGE);
                bulk_g2s(sm + st * C::STAGE + C::BU, a.w + unit_index(block * kBlockTiles, u0 + u, p.KT) * UB, kBlockTiles * UB,
                         &full_x[st]);
                if (++u == nu) {
                    u = 0;
                    block += step;
                }
            };
            // the weights never change: they are fetched before the activations are packed
            for (int n = 0; n < XS && n < total; ++n) codes(n);
            pdl_wait();
            for (int n = 0, v = 0; n < total; ++n) {
                const int st = n % XS;
                if (n >= XS) {
                    if (!wait(&empty_x[st], (uint32_t)(n / XS & 1) ^ 1u)) break;
                    codes(st);
                }
                bulk_g2s(sm + st * C::STAGE, ws + kQ4InvBytes + (size_t)(u0 + v) * C::BU, C::BU, &full_x[st]);
                v = v + 1 == nu ? 0 : v + 1;
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {
        constexpr uint32_t idesc = f16_idesc(kTcRows, C::N) | (1u << 7) | (1u << 10);  // A and B are bf16
        constexpr uint32_t idesc_lo = TYPE == GX_Q4_1 ? idesc | (1u << 13) : idesc;     // A negated
        bool ok = true;
        for (int n = 0; ok && n < total; ++n) {
            const int sx = n % XS, sa = n % AS, slot = n % C::SLOTS;
            const uint32_t dst = tmem + (uint32_t)(slot * C::SLOT);
            ok = wait(&empty_d[slot], (uint32_t)(n / C::SLOTS & 1) ^ 1u);
            ok = ok && wait(&full_x[sx], (uint32_t)(n / XS & 1)) && wait(&full_a[sa], (uint32_t)(n / AS & 1));
            if (!ok) break;
            tc_fence_after();
            const uint64_t xd = sw128_desc(smem_u32(sm + sx * C::STAGE));
            const uint32_t at = a_cols + (uint32_t)(C::AC * sa);
            // k-step k: half k / 4 of the unit, 32 bytes further in every 128-byte row. The small parts come first,
            // and m before the codes that it offsets: what an MMA cuts off goes by the sum so far.
            auto step_b = [&](int k) { return xd + (uint64_t)((k >> 2) * (C::N * 128 >> 4) + 2 * (k & 3)); };
#pragma unroll
            for (int k = 0; k < 8; ++k) umma_f16_ts(dst, at + 64u + 8u * k, step_b(k), idesc_lo, k > 0);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (TYPE == GX_Q4_1 && k % 4 == 0) umma_f16_ts(dst, at + 128u + 2u * k, step_b(8 + k / 4), idesc, 1u);
                umma_f16_ts(dst, at + 8u * k, step_b(k), idesc, 1u);
            }
            umma_commit(&empty_a[sa]);
            umma_commit(&empty_x[sx]);
            umma_commit(&full_d[slot]);
        }
        // all issued MMAs complete before TMEM is released
        umma_commit(done);
        mbar_wait(done, 0, nullptr);
        }
        __syncwarp();
    } else if (warp < 2 + 4 * C::SETS) {
        // decoders: row i of the block
        const int set = (warp - 2) >> 2, lg = warp & 3, i = 32 * lg + lane, r = i & 15, rot = (r >> 1) & 3, sh = r & 8 ? 16 : 0;
        for (int n = set; n < total; n += C::SETS) {
            const int sx = n % XS, sa = n % AS;
            if (C::FREE_FIRST && !wait_all(&empty_a[sa], (uint32_t)(n / AS & 1) ^ 1u)) break;
            if (!wait_all(&full_x[sx], (uint32_t)(n / XS & 1))) break;
            // 64 bytes of the row's codes: word j of 16-byte part q are columns 8 q .. of group j. The lanes
            // start at different parts, so that 8 of them read all banks.
            const uint8_t *tile = sm + sx * C::STAGE + C::BU + (i >> 4) * UB;
            const uint4 *w = reinterpret_cast<const uint4 *>(tile + (r >> 3) * 512 + (r & 7) * 64);
            uint4 c[4] = {w[rot], w[(rot + 1) & 3], w[(rot + 2) & 3], w[(rot + 3) & 3]};  // parts rot, rot + 1, ..
            const uint4 d4 = reinterpret_cast<const uint4 *>(tile + 1024)[r & 7];
            uint4 m4 = make_uint4(0u, 0u, 0u, 0u);
            if constexpr (TYPE == GX_Q4_1) m4 = reinterpret_cast<const uint4 *>(tile + 1152)[r & 7];
            auto sel = [](bool p, uint4 x, uint4 y) { return make_uint4(p ? x.x : y.x, p ? x.y : y.y, p ? x.z : y.z, p ? x.w : y.w); };
            {
                const bool odd = rot & 1, two = rot & 2;
                const uint4 e[4] = {sel(odd, c[3], c[0]), sel(odd, c[0], c[1]), sel(odd, c[1], c[2]), sel(odd, c[2], c[3])};
                c[0] = sel(two, e[2], e[0]);
                c[1] = sel(two, e[3], e[1]);
                c[2] = sel(two, e[0], e[2]);
                c[3] = sel(two, e[1], e[3]);
            }
            if (!C::FREE_FIRST && !wait_all(&empty_a[sa], (uint32_t)(n / AS & 1) ^ 1u)) break;
            tc_fence_after();
            const uint32_t at = a_cols + ((uint32_t)(32 * lg) << 16) + (uint32_t)(C::AC * sa);
            uint32_t mv[16];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                auto group = [g](const uint4 &v) { return g == 0 ? v.x : g == 1 ? v.y : g == 2 ? v.z : v.w; };
                const Split<TYPE> split(half_value(group(d4) >> sh, 0));
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int k = 0; k < 4; ++k) split.pair(group(c[q]), k, hi[4 * q + k], lo[4 * q + k]);
                tmem_st16(at + 16u * g, hi);
                tmem_st16(at + 64u + 16u * g, lo);
                if constexpr (TYPE == GX_Q4_1) {
                    const float f = half_value(group(m4) >> sh, 0), m1 = __bfloat162float(__float2bfloat16_rn(f)), m2 = f - m1;
                    mv[4 * g] = pack_bf2(m1, m1);
                    mv[4 * g + 1] = pack_bf2(m1, m2);
                    mv[4 * g + 2] = pack_bf2(m2, m2);
                    mv[4 * g + 3] = 0u;
                }
            }
            if constexpr (TYPE == GX_Q4_1) tmem_st16(at + 128u, mv);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full_a[sa]);
        }
    } else {
        const int lg = warp & 3, i = 32 * lg + lane;
        for (int t = i; t < TP; t += kTcRows) inv[t] = t < a.n_tok ? __ldcg(reinterpret_cast<const float *>(ws) + t) : 0.f;
        named_sync(1, 128);
        bool ok = true;
        for (int item = 0, n = 0; ok && item < items; ++item) {
            const int row = (first + item * step) * kTcRows + i;
            float acc[TP];
#pragma unroll
            for (int t = 0; t < TP; ++t) acc[t] = 0.f;
            for (int u = 0; u < nu; ++u, ++n) {
                const int slot = n % C::SLOTS;
                ok = wait_all(&full_d[slot], (uint32_t)(n / C::SLOTS & 1));
                if (!ok) break;
                tc_fence_after();
                const uint32_t at = tmem + ((uint32_t)(32 * lg) << 16) + (uint32_t)(slot * C::SLOT);
#pragma unroll
                for (int t0 = 0; t0 < C::N; t0 += 16) {  // in f32 the parts of a token lie TP apart
                    uint32_t v[16];
                    tmem_ld16(at + (uint32_t)t0, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 16; ++k) acc[(t0 + k) % TP] += __uint_as_float(v[k]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty_d[slot]);
            }
            if (!ok) break;
#pragma unroll
            for (int t = 0; t < TP; ++t) {
                if (t >= a.n_tok) break;
                const float y = acc[t] * inv[t];
                if (p.S > 1) red[t * kTcRows + i] = y;
                else if (row < a.rows) store_act(a.y, a.y_bf16, (size_t)t * a.ldy + row, y);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    if (warp == 0 && lane == 0 && *abort_flag) {  // no copy may outlive the CTA: at most one a stage is under way
        for (int i = 0; i < XS; ++i)
            for (uint32_t parity = 0; parity < 2; ++parity) mbar_wait(&full_x[i], parity, nullptr);
    }
    if (p.S > 1) {
        cluster_sync_all();
        // the CTAs of a cluster divide the sums among them, four rows of a token to a thread
        for (int j = rank * C::THREADS + tid; j < a.n_tok * (kTcRows / 4); j += p.S * C::THREADS) {
            const int t = j / (kTcRows / 4), r = j % (kTcRows / 4) * 4, row = first * kTcRows + r;
            if (row >= a.rows) continue;
            const float *at = red + t * kTcRows + r;
            float4 v[8];  // all parts on their way before the first is added
#pragma unroll
            for (int c = 0; c < 8; ++c)
                if (c < p.S) v[c] = ld_cluster4(at, (uint32_t)c);
            float4 s = v[0];
#pragma unroll
            for (int c = 1; c < 8; ++c)
                if (c < p.S) {
                    s.x += v[c].x;
                    s.y += v[c].y;
                    s.z += v[c].z;
                    s.w += v[c].w;
                }
            const float out[4] = {s.x, s.y, s.z, s.w};
            for (int k = 0; k < 4 && row + k < a.rows; ++k) store_act(a.y, a.y_bf16, (size_t)t * a.ldy + row + k, out[k]);
        }
        cluster_sync_all();  // no CTA leaves while its part is read
    }
}

template <uint32_t TYPE, bool XB, int TP>
cudaError_t launch_tc(const Q4Args &a, uint8_t *ws, int sm_count, cudaStream_t s) {
    using C = Tc<TYPE, XB, TP>;
    TcPlan p{};
    p.RT = (a.rows + kTileRows - 1) / kTileRows;
    p.KT = (a.cols + kUnitCols - 1) / kUnitCols;
    p.blocks = (p.RT + 7) / 8;
    // One CTA an SM. Where row blocks leave SMs idle, the CTAs of a cluster split the units (down to two a
    // CTA). 148 SMs take 130 to 135 CTAs at once in clusters of 3 to 6, but 120 in clusters of 8: 16 row blocks
    // of 8192 columns by 64 tokens took 25.5 us with 8 (two waves), 16.2 with 6.
    p.S = 1;
    for (int c = 2; c <= 6; ++c)
        if (p.blocks * c <= (c == 2 ? sm_count : sm_count * 7 / 8) && p.KT >= 2 * c) p.S = c;
    const int vec = ((uintptr_t)a.x & 15) == 0 && a.ldx * (XB ? 2 : 4) % 16 == 0;
    cudaError_t e = launch_chain_pdl(true, q4_pack_kernel<TYPE, XB, TP>, dim3((unsigned)a.n_tok), dim3(kPackThreads), 0, s, a, ws,
                                     p.KT, vec);
    if (e != cudaSuccess) return e;
    auto *k = q4_tc_kernel<TYPE, XB, TP>;
    static SmemLimit limit;
    e = limit.raise(k);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.S > 1 ? p.blocks * p.S : p.blocks < sm_count ? p.blocks : sm_count));
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::BYTES;
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

// The GEMV takes up to 16 product columns (a token is one in bf16, two in f32), but every CTA stages the
// activations for itself, which from 48 K of them costs more than the product's two launches: 8192 x 8192 by 3, 5,
// 8 tokens of f32 take 28.2, 51.5, 57.3 us there and 24.0, 24.3, 24.6 here; 8192 x 2048 takes 6.8, 6.4, 7.0 there and
// 10.4, 10.6, 10.7 here. One and two tokens (Ints) are always the GEMV's: 8192 x 8192 11.7 and 12.8 us.
template <uint32_t TYPE, bool XB>
cudaError_t launch_tokens(const Q4Args &a, uint8_t *ws, int sm_count, cudaStream_t s) {
    const int n = a.n_tok, columns = XB ? n : 2 * n;
    if (n == 1) return launch_gemv<TYPE, XB, Ints<TYPE, XB, 1>>(a, sm_count, s);
    if (n == 2) return launch_gemv<TYPE, XB, Ints<TYPE, XB, 2>>(a, sm_count, s);
    if (columns <= 16 && (long long)columns * a.cols < 48 * 1024) {
        if constexpr (XB) {
            if (columns <= 4) return launch_gemv<TYPE, XB, Halves<TYPE, XB, 4>>(a, sm_count, s);
        }
        if (columns <= 8) return launch_gemv<TYPE, XB, Halves<TYPE, XB, 8>>(a, sm_count, s);
        return launch_gemv<TYPE, XB, Halves<TYPE, XB, 16>>(a, sm_count, s);
    }
    if (n <= 16) return launch_tc<TYPE, XB, 16>(a, ws, sm_count, s);
    if (n <= 32) return launch_tc<TYPE, XB, 32>(a, ws, sm_count, s);
    return launch_tc<TYPE, XB, 64>(a, ws, sm_count, s);
}

uint64_t padded_units(uint64_t rows, uint64_t cols) {
    constexpr uint64_t block = kTileRows * kBlockTiles;
    return (rows + block - 1) / block * kBlockTiles * ((cols + kUnitCols - 1) / kUnitCols);
}

}  // namespace

uint64_t q4_row_bytes(uint32_t type, uint64_t cols) {
    if ((type != GX_Q4_0 && type != GX_Q4_1) || cols % 32) return 0;
    return cols / 32 * (type == GX_Q4_0 ? 18 : 20);
}

uint64_t q4_bytes(uint32_t type, uint64_t rows, uint64_t cols) { return padded_units(rows, cols) * q4_unit_bytes(type); }

cudaError_t launch_q4_repack(uint32_t type, const uint8_t *raw, uint32_t rows, uint32_t cols, uint8_t *w,
                             cudaStream_t s) {
    const long long n = (long long)padded_units(rows, cols) * kTileRows * 4;
    const long long blocks = (n + 255) / 256;
    if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
    q4_repack_kernel<<<(unsigned)blocks, 256, 0, s>>>(type, raw, (int)rows, (int)cols, w, n);
    return cudaGetLastError();
}

uint64_t q4_workspace_bytes(uint64_t cols) {
    return kQ4InvBytes + (cols + kUnitCols - 1) / kUnitCols * Tc<GX_Q4_1, false, 64>::BU;
}

cudaError_t launch_q4_linear(const Q4Args &a, uint8_t *ws, int sm_count, cudaStream_t s) {
    if (a.n_tok <= 0 || a.rows <= 0) return cudaSuccess;
    if (a.type == GX_Q4_0)
        return a.x_bf16 ? launch_tokens<GX_Q4_0, true>(a, ws, sm_count, s) : launch_tokens<GX_Q4_0, false>(a, ws, sm_count, s);
    return a.x_bf16 ? launch_tokens<GX_Q4_1, true>(a, ws, sm_count, s) : launch_tokens<GX_Q4_1, false>(a, ws, sm_count, s);
}

}  // namespace gx
