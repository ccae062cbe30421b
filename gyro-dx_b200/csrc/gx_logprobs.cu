// gx_logprobs.cu — log probabilities of given tokens over rows of logits, with the entropy, the
// given token's rank and the likeliest alternatives. With m = max x, t = scale (x - m), s = sum e^t:
//
//   logprob = t_token - ln s,   entropy = ln s - (sum e^t t) / s,
//   rank = 1 + #{x > x_token},  the n_top largest x, equal ones by rising id.
//
// Bound by reading the logits once. A cluster of CTAs takes a row, each CTA a slice that it keeps in
// shared memory: bulk copies bring it in chunks, and each chunk is scanned for its maximum as it
// arrives. With the maximum known a second pass over shared memory sums e^t and e^t t, counts the
// logits above the given one and picks candidates for the top: each thread's own maximum is known
// too, and gives a floor that few logits pass. The CTAs' results meet
// in the first one's shared memory. Nothing depends on the order in which threads run.
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
constexpr int kLpChunks = 4;      // bulk copies of a slice
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
    float m, s, et;
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
};
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }

__device__ __forceinline__ uint32_t lp_cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
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
__device__ __forceinline__ void lp_cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}

// The n_top best of n keys in shared memory (distinct, 0 for none), in falling order, into out: a key's
// place is the number of better ones.
__device__ __forceinline__ void rank_keys(const u64 *keys, int n, int n_top, u64 *out, int tid) {
    for (int i = tid; i < n; i += kLpThreads) {
        const u64 k = keys[i];
        if (k == 0) continue;
        int place = 0;
        for (int j = 0; j < n; ++j) place += keys[j] > k;
        if (place < n_top) out[place] = k;
    }
}

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Running maximum of a thread over vectors, NaN included.
template <typename T>
struct RunMax;
template <>
struct RunMax<float> {
    float m;
    __device__ __forceinline__ RunMax() { m = -CUDART_INF_F; }
    __device__ __forceinline__ void add(uint4 q) {
        m = max_nan(max_nan(m, max_nan(__uint_as_float(q.x), __uint_as_float(q.y))),
                    max_nan(__uint_as_float(q.z), __uint_as_float(q.w)));
    }
    __device__ __forceinline__ float get() const { return m; }
};
__device__ __forceinline__ __nv_bfloat162 as_bf2(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162 *>(&w); }
template <>
struct RunMax<__nv_bfloat16> {
    __nv_bfloat162 m;
    __device__ __forceinline__ RunMax() { m = __floats2bfloat162_rn(-CUDART_INF_F, -CUDART_INF_F); }
    __device__ __forceinline__ void add(uint4 q) {
        m = __hmax2_nan(m, __hmax2_nan(__hmax2_nan(as_bf2(q.x), as_bf2(q.y)), __hmax2_nan(as_bf2(q.z), as_bf2(q.w))));
    }
    __device__ __forceinline__ float get() const { return max_nan(__low2float(m), __high2float(m)); }
};
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

template <typename T, bool TOP>
__global__ void __launch_bounds__(kLpThreads) logprobs_kernel(LogprobsArgs a, int C, int slice) {
    constexpr int N = Vec<T>::N, SZ = (int)sizeof(T);
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[kLpChunks];
    __shared__ float redf[4][kLpWarps];
    __shared__ unsigned redu[kLpWarps], counts[kLpWarps];
    __shared__ u64 lists[kLpWarps * kMaxTop];
    __shared__ u64 best[kMaxTop];
    __shared__ Part parts[kLpMaxCluster];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = C > 1 ? (int)lp_cluster_rank() : 0;
    const size_t r = blockIdx.x / C;
    const int V = a.n_vocab;
    // this CTA's logits [i0, i1) of the row: 16-byte words in the middle, single logits at the ends
    const T *row = reinterpret_cast<const T *>(a.logits) + r * (size_t)a.stride;
    const int i0 = min(V, rank * slice), i1 = min(V, i0 + slice), n = i1 - i0;
    const T *src = row + i0;
    const int head = min(n, (int)((16 - ((uintptr_t)src & 15)) & 15) / SZ);
    const int words = (n - head) / N, tail0 = head + words * N;
    uint4 *buf = reinterpret_cast<uint4 *>(smem);
    const int per = (words + kLpChunks - 1) / kLpChunks;
    if (tid == 0) {
#pragma unroll
        for (int c = 0; c < kLpChunks; ++c) mbar_init(&bars[c], 1);
        fence_barrier_init();
        pdl_wait();
#pragma unroll
        for (int c = 0; c < kLpChunks; ++c) {
            const int w0 = c * per, w1 = min(words, w0 + per);
            if (w0 >= w1) continue;
            mbar_expect_tx(&bars[c], (uint32_t)(w1 - w0) * 16u);
            bulk_g2s(buf + w0, reinterpret_cast<const uint4 *>(src + head) + w0, (uint32_t)(w1 - w0) * 16u, &bars[c]);
        }
    }
    __syncthreads();
    if (C > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // this CTA has started
    pdl_launch_dependents();
    pdl_wait();
    // the slice's ends, one logit a thread (fewer than 2 N of them)
    const int ends = n - words * N;
    const int end_i = tid < head ? tid : tail0 + tid - head;
    const bool has_end = tid < ends;
    const float end_x = has_end ? to_f(src[end_i]) : -CUDART_INF_F;
    const uint32_t tok = a.tokens ? a.tokens[r] : GX_NO_TOKEN;
    const bool has = tok < (uint32_t)V;
    const float xt = has ? to_f(row[tok]) : CUDART_INF_F;

    // pass 1, chunk by chunk: the thread's maximum
    RunMax<T> run;
    bool ok = true;
#pragma unroll
    for (int c = 0; c < kLpChunks; ++c) {
        const int w0 = c * per, w1 = min(words, w0 + per);
        if (w0 >= w1) continue;
        ok = ok && mbar_wait(&bars[c], 0u, a.err);
        if (!ok) continue;
#pragma unroll 4
        for (int w = w0 + tid; w < w1; w += kLpThreads) run.add(buf[w]);
    }
    ok = __syncthreads_and(ok);
    if (!ok && tid == 0) {  // an expired wait is reported; no copy may outlive the CTA
        for (int c = 0; c < kLpChunks; ++c)
            if (c * per < words) mbar_wait(&bars[c], 0u, nullptr);
    }
    const float own = max_nan(run.get(), end_x);
    float m = own;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) redf[0][warp] = m;
    if (TOP) {
        // The k-th largest of the lanes' maxima, k = n_top / 8 rounded up: each maximum is a logit of its
        // own, so the least of the 8 warps' values is a floor that at least n_top logits reach.
        uint32_t o = isnan(own) ? ordered(-CUDART_INF_F) : ordered(own), t = 0;
        for (int k = (a.n_top + kLpWarps - 1) / kLpWarps; k > 0; --k) {
            t = __reduce_max_sync(0xffffffffu, o);
            const unsigned who = __ballot_sync(0xffffffffu, o == t);
            if (lane == __ffs(who) - 1) o = 0;
        }
        if (lane == 0) redf[1][warp] = unordered(t);
    }
    __syncthreads();
    m = redf[0][0];
    float floor = TOP ? redf[1][0] : 0.f;
#pragma unroll
    for (int w = 1; w < kLpWarps; ++w) {
        m = max_nan(m, redf[0][w]);
        if (TOP) floor = fminf(floor, redf[1][w]);
    }
    const bool has_nan = isnan(m);

    // pass 2
    const bool flat = m == -CUDART_INF_F;  // every token masked: a row of equal logits
    const float c2 = a.scale * CUDART_L2E_F;
    float s = 0.f, et = 0.f;
    unsigned above = 0;
    u64 list = 0, worst = 0;   // the warp's best keys by lane, its n_top-th
    auto sums = [&](float x) {
        const float t = flat ? 0.f : fmaxf((x - m) * c2, -200.f);  // e^t is 0 there, and 0 * t stays 0
        const float e = ex2(t);
        s += e;
        et = fmaf(e, t, et);
    };
    // logits above the given one; NaN lies below all others
    auto count = [&](float x) { above += isnan(xt) ? !isnan(x) : x > xt; };
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
    if (has_end) {
        sums(end_x);
        count(end_x);
    }
    if (TOP) offer(has_end ? logit_key(end_x, (uint32_t)(i0 + end_i)) : 0);
    float least = worst ? key_value(worst) : -CUDART_INF_F;  // value of the n_top-th key
    if (isnan(least)) least = -CUDART_INF_F;
    for (int w0 = warp * 32; w0 < words; w0 += kLpThreads) {
        const int w = w0 + lane;
        const bool on = ok && w < words;
        float v[N], top = -CUDART_INF_F;
        if (on) {
            const uint4 q = buf[w];
            Vec<T>::get(q, v);
            top = vec_max<T>(q);
#pragma unroll
            for (int k = 0; k < N; ++k) sums(v[k]);
            if (top > xt || isnan(xt)) {
#pragma unroll
                for (int k = 0; k < N; ++k) count(v[k]);
            }
        }
        if (TOP) {
            const bool cand = on && (has_nan || (top >= floor && top >= least));
            if (__any_sync(0xffffffffu, cand)) {
#pragma unroll
                for (int k = 0; k < N; ++k) offer(cand ? logit_key(v[k], (uint32_t)(i0 + head + w * N + k)) : 0);
                least = worst ? key_value(worst) : -CUDART_INF_F;
                if (isnan(least)) least = -CUDART_INF_F;
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        et += __shfl_xor_sync(0xffffffffu, et, o);
        above += __shfl_xor_sync(0xffffffffu, above, o);
    }
    if (lane == 0) {
        redf[2][warp] = s;
        redf[3][warp] = et;
        redu[warp] = above;
    }
    if (TOP) {
        const unsigned mine = __ballot_sync(0xffffffffu, lane < a.n_top && list != 0);
        if (lane == 0) counts[warp] = __popc(mine);
        if (tid < kMaxTop) best[tid] = 0;
    }
    __syncthreads();
    if (TOP) {
        int at = 0, all = 0;
#pragma unroll
        for (int w = 0; w < kLpWarps; ++w) {
            at += w < warp ? (int)counts[w] : 0;
            all += (int)counts[w];
        }
        if (lane < (int)counts[warp]) lists[at + lane] = list;
        __syncthreads();
        rank_keys(lists, all, a.n_top, best, tid);
        __syncthreads();
    }
    // into the first CTA's parts
    if (C > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (warp == 0) {
        float ss = 0.f, te = 0.f;
        unsigned ab = 0;
#pragma unroll
        for (int w = 0; w < kLpWarps; ++w) {
            ss += redf[2][w];
            te += redf[3][w];
            ab += redu[w];
        }
        if (C > 1) {
            const uint32_t at = peer_addr(&parts[rank], 0u);
            if (lane == 0) {
                st_peer(at + (uint32_t)offsetof(Part, m), __float_as_uint(m));
                st_peer(at + (uint32_t)offsetof(Part, s), __float_as_uint(ss));
                st_peer(at + (uint32_t)offsetof(Part, et), __float_as_uint(te));
                st_peer(at + (uint32_t)offsetof(Part, above), ab);
            }
            if (TOP && lane < a.n_top) st_peer(at + (uint32_t)offsetof(Part, top) + 8u * lane, best[lane]);
        } else if (lane == 0) {
            parts[0].m = m;
            parts[0].s = ss;
            parts[0].et = te;
            parts[0].above = ab;
        }
    }
    if (C > 1) lp_cluster_sync();
    else __syncthreads();
    if (rank != 0) return;
    // the row: every thread computes the same totals
    float M = parts[0].m;
    for (int c = 1; c < C; ++c) M = max_nan(M, parts[c].m);
    float S = 0.f, ET = 0.f;
    unsigned AB = 0;
    for (int c = 0; c < C; ++c) {
        // a part's sums are relative to its own maximum; one of masked tokens only has no weight in a row
        // that has others
        const float pm = parts[c].m, t = pm == M ? 0.f : fmaxf((pm - M) * c2, -200.f), w = pm == M ? 1.f : ex2(t);
        S = fmaf(parts[c].s, w, S);
        ET = fmaf(w, fmaf(parts[c].s, t, parts[c].et), ET);
        AB += parts[c].above;
    }
    if (isnan(M) || M == CUDART_INF_F) S = CUDART_NAN_F;
    const float ls = logf(S);
    // halves, so that a difference beyond the f32 range that the scale brings back is not lost
    auto lp = [&](float x) { return (M == -CUDART_INF_F ? 0.f : (0.5f * x - 0.5f * M) * (2.f * a.scale)) - ls; };
    if (tid == 0) {
        const bool bad = a.tokens && !has && tok != GX_NO_TOKEN;
        if (bad) atomicExch(a.err, KERR_BOUNDS);
        if (a.logprob) a.logprob[r] = has ? lp(xt) : bad ? CUDART_NAN_F : 0.f;
        if (a.rank) a.rank[r] = has ? AB + 1 : 0;
        if (a.entropy) a.entropy[r] = ls - ET / S * CUDART_LN2_F;
    }
    if (TOP) {
        if (C > 1) {
            u64 *all = reinterpret_cast<u64 *>(smem);  // the slice is no longer needed
            for (int i = tid; i < C * a.n_top; i += kLpThreads) all[i] = parts[i / a.n_top].top[i % a.n_top];
            __syncthreads();
            rank_keys(all, C * a.n_top, a.n_top, best, tid);
            __syncthreads();
        }
        if (tid < a.n_top) {
            if (a.top_ids) a.top_ids[r * a.n_top + tid] = key_id(best[tid]);
            if (a.top_logprobs) a.top_logprobs[r * a.n_top + tid] = lp(key_value(best[tid]));
        }
    }
}

template <typename T, bool TOP>
cudaError_t launch_lp(const LogprobsArgs &a, int sm_count, cudaStream_t s) {
    auto *k = logprobs_kernel<T, TOP>;
    constexpr int N = Vec<T>::N;
    // Slices of at most 56 KB, so that three CTAs overlap on an SM; while the rows leave SMs idle, down to
    // 8 KB.
    int C = 1;
    auto bytes = [&] { return (((long long)a.n_vocab + C - 1) / C + N) * (long long)sizeof(T); };
    while (C < kLpMaxCluster && bytes() > 56 * 1024) C *= 2;
    while (C < kLpMaxCluster && (long long)a.n_rows * C < sm_count && bytes() > 8 * 1024) C *= 2;
    if ((long long)a.n_rows * C > 0x7fffffffll) return cudaErrorInvalidValue;
    const int slice = ((a.n_vocab + C - 1) / C + N - 1) / N * N;
    int smem = slice * (int)sizeof(T);
    if (smem < C * kMaxTop * 8) smem = C * kMaxTop * 8;
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess && C > 8) e = cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.n_rows * C));
    cfg.blockDim = dim3(kLpThreads);
    cfg.dynamicSmemBytes = (size_t)smem;
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
