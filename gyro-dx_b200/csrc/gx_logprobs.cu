// gx_logprobs.cu — log probabilities of given tokens over rows of logits, with the entropy, the
// given token's rank and the likeliest alternatives. With t = scale (x - ref), s = sum e^t:
//
//   logprob = t_token - ln s,   entropy = ln s - (sum e^t t) / s,
//   rank = 1 + #{x > x_token},  the n_top largest x, equal ones by rising id.
//
// Bound by reading the logits once, 10 instructions a logit. A cluster of CTAs takes a row, each CTA a
// slice that its threads stream through registers, four 16-byte words ahead. The reference ref need not be
// the maximum, only near it: it is that of the slice's first words, and a thread that meets a logit more
// than 2^8 times as likely moves on to a new one. (It is always a logit of the row: either the largest, and s >= 1
// and all t <= 0 exactly, or one that weighs 2^-8 of it, and no probability is within roundings of 1. So no log
// probability comes out above 0 and no entropy below.) Each lane's maximum in the first words also gives a
// floor for the top, so that few logits are candidates; those enter the warp's sorted list, a key in a
// lane. The lists and sums meet in shared memory, then in that of the cluster's first CTA. Nothing
// depends on the order in which threads run.
//
// Measured: 1500 rows of 131073 f32 139 to 149 us, 82 to 87 % of the copy bandwidth; 64 rows of 150001 bf16 12.4 us
// (1.5 TB/s: starting clusters and merging their lists takes half of it); one row of 32000 7 us, a launch
// and the two passes over its cluster's lists.
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
constexpr int kLpAhead = 4;       // 16-byte words of a thread in flight
constexpr int kLpMaxCluster = 16;

typedef unsigned long long u64;

// A logit and its id as one key that orders by value, then by lower id; a NaN lies below -Inf and
// -0 equals 0. No key of a logit is 0.
__device__ __forceinline__ u64 logit_key(float x, uint32_t id) {
    uint32_t u = __float_as_uint(x + 0.0f);
    u = (u >> 31) ? ~u : u | 0x80000000u;
    if (isnan(x)) u = 1u;
    return ((u64)u << 32) | (0xffffffffu - id);
}
__device__ __forceinline__ uint32_t key_id(u64 key) { return 0xffffffffu - (uint32_t)key; }
__device__ __forceinline__ float key_value(u64 key) {
    const uint32_t u = (uint32_t)(key >> 32);
    if (u == 1u) return CUDART_NAN_F;
    return __uint_as_float((u >> 31) ? u & 0x7fffffffu : ~u);
}

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// A warp's n_top best keys so far, the lane's rank among them in falling order (0: none yet).
__device__ __forceinline__ void warp_insert(u64 &list, u64 key, int lane) {
    // lanes whose key is better keep it; the first that is not takes the new one, the rest move up
    const u64 up = __shfl_up_sync(0xffffffffu, list, 1);
    if (list < key) list = (lane > 0 && up < key) ? up : key;
}

// What a CTA hands to the first one of its cluster.
struct Part {
    float ref, s, et;
    unsigned above;
    u64 top[kMaxTop];
};

template <typename T>
struct Vec;
template <>
struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void get(uint4 q, float (&v)[4]) {
        v[0] = __uint_as_float(q.x);
        v[1] = __uint_as_float(q.y);
        v[2] = __uint_as_float(q.z);
        v[3] = __uint_as_float(q.w);
    }
    static __device__ __forceinline__ float pick(const uint4 &q, int k) {
        return __uint_as_float(k < 2 ? (k < 1 ? q.x : q.y) : (k < 3 ? q.z : q.w));
    }
};
template <>
struct Vec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(uint4 q, float (&v)[8]) {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[2 * j] = __uint_as_float(w[j] << 16);
            v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ float pick(const uint4 &q, int k) {
        const uint32_t w = k < 4 ? (k < 2 ? q.x : q.y) : (k < 6 ? q.z : q.w);
        return __uint_as_float((k & 1) ? w & 0xffff0000u : w << 16);
    }
};
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }

__device__ __forceinline__ uint32_t peer_addr(const void *p, uint32_t rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    return at;
}
__device__ __forceinline__ void st_peer(uint32_t at, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
__device__ __forceinline__ void st_peer(uint32_t at, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory");
}
// The best 32 keys of two falling lists, a key in a lane, as a falling list: one against the other
// reversed leaves the best 32 in a bitonic order, which five exchanges sort.
__device__ __forceinline__ u64 merge_lists(u64 a, u64 b, int lane) {
    b = __shfl_sync(0xffffffffu, b, 31 - lane);
    u64 k = a > b ? a : b;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        const u64 o = __shfl_xor_sync(0xffffffffu, k, d);
        k = ((lane & d) == 0) == (k > o) ? k : o;
    }
    return k;
}
// n lists (a power of two, at most 16) in shared memory, [n][32]: the merged list in warp 0. All threads.
__device__ __forceinline__ u64 merge_all(u64 (*lists)[32], int n, int warp, int lane) {
    u64 k = warp < n ? lists[warp][lane] : 0;
    for (int h = n / 2; h > 0; h /= 2) {
        if (warp < h) {
            k = merge_lists(k, lists[warp + h][lane], lane);
            lists[warp][lane] = k;
        }
        __syncthreads();
    }
    return k;
}

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ __nv_bfloat162 as_bf2(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162 *>(&w); }
// What is read past a slice: masked tokens.
template <typename T>
__device__ __forceinline__ uint4 masked_word() {
    const uint32_t w = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
    return make_uint4(w, w, w, w);
}
// The largest of a vector without NaN.
template <typename T>
__device__ __forceinline__ float vec_max(uint4 q);
template <>
__device__ __forceinline__ float vec_max<float>(uint4 q) {
    return fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
}
template <>
__device__ __forceinline__ float vec_max<__nv_bfloat16>(uint4 q) {
    const __nv_bfloat162 m = __hmax2(__hmax2(as_bf2(q.x), as_bf2(q.y)), __hmax2(as_bf2(q.z), as_bf2(q.w)));
    return fmaxf(__low2float(m), __high2float(m));
}

// An order of floats as unsigned numbers, for a warp's maximum in one instruction (-0 below 0 here; NaN
// does not occur).
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x);
    return (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float((u >> 31) ? u & 0x7fffffffu : ~u); }

// Sums relative to one reference, moved to another: a part with no weight there (masked tokens, or 2^-126
// of the whole) counts nothing.
__device__ __forceinline__ void move_sums(float &s, float &et, float from, float to, float c2) {
    const float d = from == to ? 0.f : fmaxf((from - to) * c2, -200.f), w = ex2(d);
    et = w * fmaf(s, d, et);
    s *= w;
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kLpThreads, 4) logprobs_kernel(LogprobsArgs a, int C, int slice) {
    constexpr int N = Vec<T>::N, SZ = (int)sizeof(T);
    __shared__ float redf[4][kLpWarps];
    __shared__ unsigned redu[kLpWarps];
    __shared__ u64 lists[kLpMaxCluster][32];  // of the warps, then of the cluster's CTAs
    __shared__ Part parts[kLpMaxCluster];
    static_assert(kLpMaxCluster >= kLpWarps && kMaxTop == 32, "a list is a warp wide");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = C > 1 ? (int)cluster_rank() : 0;
    const size_t r = blockIdx.x / C;
    const int V = a.n_vocab;
    // this CTA's logits [i0, i1) of the row: 16-byte words in the middle, single logits at the ends
    const T *row = reinterpret_cast<const T *>(a.logits) + r * (size_t)a.stride;
    const int i0 = min(V, rank * slice), i1 = min(V, i0 + slice), n = i1 - i0;
    const T *src = row + i0;
    const int head = min(n, (int)((16 - ((uintptr_t)src & 15)) & 15) / SZ);
    const int words = (n - head) / N, tail0 = head + words * N;
    const uint4 *word = reinterpret_cast<const uint4 *>(src + head);
    if (C > 1) cluster_arrive_relaxed();
    pdl_launch_dependents();
    pdl_wait();
    uint4 next[kLpAhead];
#pragma unroll
    for (int j = 0; j < kLpAhead; ++j) {
        const int w = j * kLpThreads + tid;
        next[j] = w < words ? __ldcs(word + w) : masked_word<T>();
    }
    // the slice's ends, one logit a thread (fewer than 2 N of them)
    const int ends = n - words * N;
    const int end_i = tid < head ? tid : tail0 + tid - head;
    const bool has_end = tid < ends;
    const float end_x = has_end ? to_f(src[end_i]) : -CUDART_INF_F;
    const uint32_t tok = a.tokens ? a.tokens[r] : GX_NO_TOKEN;
    const bool has = tok < (uint32_t)V;
    const float xt = has ? to_f(row[tok]) : CUDART_INF_F;
    const bool xt_nan = isnan(xt);
    const float mark = xt_nan ? CUDART_INF_F : xt;  // logits above this one are counted (above a NaN: all of them)

    // the reference, and the floor of the candidates, from the first words
    float own = vec_max<T>(next[0]);
#pragma unroll
    for (int j = 1; j < kLpAhead; ++j) own = fmaxf(own, vec_max<T>(next[j]));
    if (isnan(own)) own = -CUDART_INF_F;
    uint32_t o = ordered(own), t = __reduce_max_sync(0xffffffffu, o);
    if (lane == 0) redf[0][warp] = unordered(t);
    if (TOP) {
        // The k-th largest of the lanes' maxima, k = n_top / 8 rounded up: each maximum is a logit of its
        // own, so the least of the 8 warps' values is a floor that at least n_top logits reach.
        for (int k = (a.n_top + kLpWarps - 1) / kLpWarps; k > 1; --k) {
            if (lane == __ffs(__ballot_sync(0xffffffffu, o == t)) - 1) o = 0;
            t = __reduce_max_sync(0xffffffffu, o);
        }
        if (lane == 0) redf[1][warp] = unordered(t);
    }
    __syncthreads();
    float ref = redf[0][0], floor = TOP ? redf[1][0] : 0.f;
#pragma unroll
    for (int w = 1; w < kLpWarps; ++w) {
        ref = fmaxf(ref, redf[0][w]);
        if (TOP) floor = fminf(floor, redf[1][w]);
    }
    ref = fmaxf(ref, -3.402823466e38f);  // a finite one where the first words are masked

    const float c2 = a.scale * CUDART_L2E_F, reach = 8.f / c2;  // t below in units of ln 2
    float s = 0.f, et = 0.f, limit = ref + reach;
    unsigned above = 0;
    u64 list = 0, worst = 0;   // the warp's best keys by lane, its n_top-th
    auto sum = [&](float x) {
        const float d = max_nan((x - ref) * c2, -200.f);  // e^t is 0 there, and 0 * t stays 0; a NaN shows in s
        const float e = ex2(d);
        s += e;
        et = fmaf(e, d, et);
    };
    auto reach_for = [&](float x) {  // a new reference for a logit far above
        if (x > limit) {
            move_sums(s, et, ref, x, c2);
            ref = x;
            limit = ref + reach;
        }
    };
    auto offer = [&](u64 key) {  // one key of each lane, 0 for none
        unsigned who = __ballot_sync(0xffffffffu, key > worst);
        while (who) {
            const int l = __ffs(who) - 1;
            const u64 k = __shfl_sync(0xffffffffu, key, l);
            warp_insert(list, k, lane);
            worst = __shfl_sync(0xffffffffu, list, a.n_top - 1);
            who = (who & (who - 1)) & __ballot_sync(0xffffffffu, key > worst);
        }
    };
    // From step to step a warp meets its logits by rising id, so once its list is full only a larger value
    // enters it: a logit above gate (before that, one at the floor too).
    const float below = floor == 0.f ? -1.401298464e-45f : unordered(ordered(floor) - 1u);
    float gate = floor == -CUDART_INF_F ? floor : below;
    bool any_enters = TOP && floor == -CUDART_INF_F;  // masked tokens too, while the list is not full
    for (int w0 = tid; w0 - tid < words; w0 += kLpAhead * kLpThreads) {
        const bool inside = w0 - tid + 2 * kLpAhead * kLpThreads <= words;  // the next words all lie in the slice
        unsigned hits = 0;  // words of the warp with candidates
#pragma unroll
        for (int j = 0; j < kLpAhead; ++j) {
            const int ahead = w0 + (j + kLpAhead) * kLpThreads;
            float v[N];
            Vec<T>::get(next[j], v);
            const float top = vec_max<T>(next[j]);
            if (__any_sync(0xffffffffu, top > limit)) reach_for(top);
            if (TOP) hits |= __any_sync(0xffffffffu, top > gate) ? 1u << j : 0u;
#pragma unroll
            for (int k = 0; k < N; ++k) sum(v[k]);
            if (__any_sync(0xffffffffu, top > mark)) {
#pragma unroll
                for (int k = 0; k < N; ++k) above += v[k] > mark;
            }
            if (inside) next[j] = __ldcs(word + ahead);
            else next[j] = ahead < words ? __ldcs(word + ahead) : masked_word<T>();
        }
        if (TOP) {
            if (any_enters) hits = (1u << kLpAhead) - 1u;
            while (hits) {  // rare: the words are read again, so that this code stands once
                const int w = w0 + (__ffs(hits) - 1) * kLpThreads;
                hits &= hits - 1;
                const uint4 q = w < words ? word[w] : masked_word<T>();
                float v[N];
                Vec<T>::get(q, v);
                unsigned mine = 0;  // the lane's candidates in the word
#pragma unroll
                for (int k = 0; k < N; ++k) mine |= v[k] > gate || any_enters ? 1u << k : 0u;
                if (w >= words) mine = 0;
                while (__any_sync(0xffffffffu, mine != 0)) {  // one of each lane
                    const int k = __ffs(mine) - 1;
                    mine &= mine - 1;
                    offer(k >= 0 ? logit_key(Vec<T>::pick(q, k), (uint32_t)(i0 + head + w * N + k)) : 0);
                }
                if (worst != 0) {
                    gate = fmaxf(gate, key_value(worst));
                    any_enters = false;
                }
            }
        }
    }
    if (has_end) {
        reach_for(end_x);
        sum(end_x);
        above += end_x > mark;
    }
    if (TOP && warp == 0) offer(has_end ? logit_key(end_x, (uint32_t)(i0 + end_i)) : 0);
    // A NaN lies below every number: where there is one (or +Inf, whose sums are NaN too), the counts and
    // the list are made again the slow way.
    if (xt_nan && tid == 0) above = (unsigned)n;
    if (__syncthreads_or(isnan(s))) {
        auto count = [&](float x) { above += xt_nan ? !isnan(x) : x > xt; };
        above = 0;
        list = worst = 0;
        for (int w0 = warp * 32; w0 < words; w0 += kLpThreads) {
            const bool on = w0 + lane < words;
            const uint4 q = on ? word[w0 + lane] : masked_word<T>();
#pragma unroll 1
            for (int k = 0; k < N; ++k) {
                const float x = Vec<T>::pick(q, k);
                if (on) count(x);
                if (TOP) offer(on ? logit_key(x, (uint32_t)(i0 + head + (w0 + lane) * N + k)) : 0);
            }
        }
        if (has_end) count(end_x);
        if (TOP && warp == 0) offer(has_end ? logit_key(end_x, (uint32_t)(i0 + end_i)) : 0);
        s = CUDART_NAN_F;
    }
    {
        float m = ref;
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
        move_sums(s, et, ref, m, c2);
        ref = m;
    }
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, k);
        et += __shfl_xor_sync(0xffffffffu, et, k);
    }
    above = __reduce_add_sync(0xffffffffu, above);
    if (lane == 0) {
        redf[0][warp] = ref;
        redf[2][warp] = s;
        redf[3][warp] = et;
        redu[warp] = above;
    }
    if (TOP) lists[warp][lane] = list;
    __syncthreads();
    u64 best = TOP ? merge_all(lists, kLpWarps, warp, lane) : 0;
    // into the first CTA's parts
    if (C > 1) cluster_wait();
    if (warp == 0) {
        // the warps' sums, one in a lane
        float m = lane < kLpWarps ? redf[0][lane] : -CUDART_INF_F, ss = lane < kLpWarps ? redf[2][lane] : 0.f;
        float te = lane < kLpWarps ? redf[3][lane] : 0.f, to = m;
        unsigned ab = lane < kLpWarps ? redu[lane] : 0;
#pragma unroll
        for (int k = 4; k > 0; k >>= 1) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, k));
        to = __shfl_sync(0xffffffffu, to, 0);
        move_sums(ss, te, m, to, c2);
#pragma unroll
        for (int k = 4; k > 0; k >>= 1) {
            ss += __shfl_xor_sync(0xffffffffu, ss, k);
            te += __shfl_xor_sync(0xffffffffu, te, k);
        }
        ab = __reduce_add_sync(0xffffffffu, ab);
        if (C > 1) {
            const uint32_t at = peer_addr(&parts[rank], 0u);
            if (lane == 0) {
                st_peer(at + (uint32_t)offsetof(Part, ref), __float_as_uint(to));
                st_peer(at + (uint32_t)offsetof(Part, s), __float_as_uint(ss));
                st_peer(at + (uint32_t)offsetof(Part, et), __float_as_uint(te));
                st_peer(at + (uint32_t)offsetof(Part, above), ab);
            }
            if (TOP) st_peer(at + (uint32_t)offsetof(Part, top) + 8u * lane, best);
        } else if (lane == 0) {
            parts[0].ref = to;
            parts[0].s = ss;
            parts[0].et = te;
            parts[0].above = ab;
        }
    }
    if (C > 1) cluster_sync_all();
    else __syncthreads();
    if (rank != 0) return;
    // the row: every thread computes the same totals
    float M = parts[0].ref;
    for (int c = 1; c < C; ++c) M = fmaxf(M, parts[c].ref);
    float S = 0.f, ET = 0.f;
    unsigned AB = 0;
    for (int c = 0; c < C; ++c) {
        float ss = parts[c].s, te = parts[c].et;
        move_sums(ss, te, parts[c].ref, M, c2);
        S += ss;
        ET += te;
        AB += parts[c].above;
    }
    const bool flat = S == 0.f;  // every token masked: a row of equal logits
    if (flat) S = (float)V;
    if (isinf(S)) S = CUDART_NAN_F;
    const float ls = logf(S);
    // halves, so that a difference beyond the f32 range that the scale brings back is not lost
    auto lp = [&](float x) { return (flat ? 0.f : (0.5f * x - 0.5f * M) * (2.f * a.scale)) - ls; };
    if (tid == 0) {
        const bool bad = a.tokens && !has && tok != GX_NO_TOKEN;
        if (bad) atomicExch(a.err, KERR_BOUNDS);
        if (a.logprob) a.logprob[r] = has ? lp(xt) : bad ? CUDART_NAN_F : 0.f;
        if (a.rank) a.rank[r] = has ? AB + 1 : 0;
        if (a.entropy) a.entropy[r] = ls - ET / S * CUDART_LN2_F;
    }
    if (TOP) {
        if (C > 1) {
            for (int c = warp; c < C; c += kLpWarps) lists[c][lane] = parts[c].top[lane];
            __syncthreads();
            best = merge_all(lists, C, warp, lane);
        }
        if (tid < a.n_top) {
            if (a.top_ids) a.top_ids[r * a.n_top + tid] = key_id(best);
            if (a.top_logprobs) a.top_logprobs[r * a.n_top + tid] = lp(key_value(best));
        }
    }
}

template <typename T, bool TOP>
cudaError_t launch_lp(const LogprobsArgs &a, int sm_count, cudaStream_t s) {
    auto *k = logprobs_kernel<T, TOP>;
    constexpr int N = Vec<T>::N;
    // CTAs for every row until every SM has one, in slices of at least 16 KB: a CTA's floor, lists and
    // merges cost as much as some 16 KB of logits (64 rows of 150001 in bf16: 35 us in 16 CTAs a row, 20 in
    // 8, 12.7 in 4, 14.7 in 2)
    int C = 1;
    auto bytes = [&] { return (long long)a.n_vocab / C * (long long)sizeof(T); };
    while (C < kLpMaxCluster && (long long)a.n_rows * C < sm_count && bytes() >= 32 * 1024) C *= 2;
    if ((long long)a.n_rows * C > 0x7fffffffll) return cudaErrorInvalidValue;
    const int slice = ((a.n_vocab + C - 1) / C + N - 1) / N * N;
    if (C > 8) {
        const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.n_rows * C));
    cfg.blockDim = dim3(kLpThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)C;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = C > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, k, a, C, slice);
}

}  // namespace

cudaError_t launch_logprobs(const LogprobsArgs &a, int sm_count, cudaStream_t s) {
    if (a.n_rows <= 0) return cudaSuccess;
    if (a.bf16)
        return a.n_top ? launch_lp<__nv_bfloat16, true>(a, sm_count, s) : launch_lp<__nv_bfloat16, false>(a, sm_count, s);
    return a.n_top ? launch_lp<float, true>(a, sm_count, s) : launch_lp<float, false>(a, sm_count, s);
}

}  // namespace gx
