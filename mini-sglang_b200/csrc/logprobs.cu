// Log probabilities of given tokens, the entropy of every row and its most probable tokens, in one pass over the logits.
//
// Of a row x of V logits, with m = max x, s = sum e^(x_j - m) and t = sum e^(x_j - m) (x_j - m):
//
//     log p_j = (x_j - m) - log s            entropy = log s - t / s
//
// m, s and t are kept per thread in float32 and moved together: where m grows by d, s becomes s e^-d and t becomes
// (t - d s) e^-d.  The best `top` tokens are kept per warp, one a lane and in order, as 64-bit keys of the value's bits (made to
// sort as whole numbers) above the complement of the index: all keys differ, so the order is total (among equal logits the lower
// index comes first) and no schedule of the warps can change the outcome.  A warp looks closer at a stretch of values only where
// one reaches the weakest key that any warp of the block keeps, which of random values few do after the first stretches.
//
// A row is read by a cluster of C blocks, whose first merges the others' sums and keys out of their shared memory: no scratch memory,
// no counters, one launch.
//
// A logit of -inf adds nothing.  A row with a NaN, with +inf or with nothing but -inf has NaN in all its probabilities, as the
// formula has; its top tokens are those of the highest numbers (a NaN is none).  A token outside the vocabulary gets NaN.
#include <cooperative_groups.h>
#include "common.cuh"

namespace cg = cooperative_groups;

constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32, LP_MAX_TOP = 32, LP_UNROLL = 4;

__device__ __forceinline__ unsigned lp_order(float v) {            // sorts as v does; -0 as +0
    const unsigned b = __float_as_uint(v + 0.f);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float lp_value(unsigned o) { return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ unsigned long long lp_key(float v, int j) { return ((unsigned long long)lp_order(v) << 32) | (0xffffffffu - (unsigned)j); }

__device__ __forceinline__ float lp_exp2(float x) {                // 2^x; what underflows is 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

struct LpSums { float m, s, t; };
// e^d is 0 from here on down; d itself is cut there, since d s may leave the range (a masked part of the type's lowest values) and t e^d be 0 x inf
__device__ __forceinline__ float lp_shift(float d) { return d < -200.f ? -200.f : d; }
__device__ __forceinline__ LpSums lp_join(LpSums a, LpSums b) {
    const float m = fmaxf(a.m, b.m), mu = m == -INFINITY ? 0.f : m;
    // (a part that saw nothing has s = t = 0 and m = -inf: its shift is taken as 0)
    const float da = a.m == -INFINITY ? 0.f : lp_shift(a.m - mu), db = b.m == -INFINITY ? 0.f : lp_shift(b.m - mu);
    const float fa = expf(da), fb = expf(db);
    return LpSums{m, a.s * fa + b.s * fb, (a.t + a.s * da) * fa + (b.t + b.s * db) * fb};
}

// a warp's keys: lane i holds the i-th best (0: none yet)
struct LpBest {
    unsigned long long mine, weakest;                // weakest: of the first `top` lanes
    __device__ __forceinline__ void put(unsigned long long key, int top, int lane) {         // the same key in all lanes, above `weakest`
        const int at = __popc(__ballot_sync(0xffffffffu, mine > key));
        const unsigned long long up = __shfl_up_sync(0xffffffffu, mine, 1);
        if (lane > at) mine = up;
        if (lane == at) mine = key;
        weakest = __shfl_sync(0xffffffffu, mine, top - 1);
    }
    __device__ __forceinline__ void offer(unsigned long long key, int top, int lane) {       // a key a lane (0: none)
        unsigned who = __ballot_sync(0xffffffffu, key > weakest);
        while (who) {
            const int src = __ffs(who) - 1;
            const unsigned long long k = __shfl_sync(0xffffffffu, key, src);
            if (k > weakest) put(k, top, lane);
            who &= who - 1;
        }
    }
};

template <typename T> struct LpVec;
template <> struct LpVec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void split(const uint4& v, float (&x)[4]) {
        x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
    }
};
template <> struct LpVec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void split(const uint4& v, float (&x)[8]) {
        const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
};

struct LpPart {                                      // what a block hands to the first of its cluster
    LpSums sums;
    unsigned long long best[LP_MAX_TOP];
};

template <typename T, bool TOP>
__global__ void __launch_bounds__(LP_THREADS) token_logprobs_kernel(const T* __restrict__ logits, long long row_stride, int V, const int* __restrict__ tokens,
                                                                    int top, float* __restrict__ lp_out, float* __restrict__ entropy_out,
                                                                    float* __restrict__ top_lp, int* __restrict__ top_id, int C) {
    constexpr int N = LpVec<T>::N, U = LP_UNROLL;
    __shared__ LpPart part;
    __shared__ LpSums warp_sums[LP_WARPS];
    __shared__ unsigned long long warp_best[LP_WARPS][LP_MAX_TOP];
    __shared__ unsigned sh_weakest;                  // a lower bound of the block's weakest kept value (as lp_order)
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / C, rank = blockIdx.x - row * C;
    const T* x = logits + (size_t)row * row_stride;
    if (tid == 0) sh_weakest = 0u;
    pdl_launch_dependents();
    pdl_wait();
    pdl_after_wait();
    __syncthreads();

    // this block's share [j0, j1) and within it the stretch [a, b) of whole aligned vectors
    const int per = (((V + C - 1) / C) + 7) & ~7;
    const int j0 = min(V, rank * per), j1 = min(V, j0 + per);
    const int lead = (int)((16 - ((uintptr_t)(x + j0) & 15)) & 15) / (int)sizeof(T);
    const int a = min(j1, j0 + lead), n_vec = (j1 - a) / N, b = a + n_vec * N;

    LpSums sum{-INFINITY, 0.f, 0.f};
    LpBest best{0ull, 0ull};
    auto add = [&](const float* v, int n) {
        float mx = v[0];
#pragma unroll
        for (int i = 1; i < n; ++i) mx = fmaxf(mx, v[i]);
        if (mx > sum.m) {
            const float d = sum.m == -INFINITY ? 0.f : lp_shift(sum.m - mx), f = expf(d);
            sum.t = (sum.t + sum.s * d) * f;
            sum.s *= f;
            sum.m = mx;
        }
        const float mu = sum.m == -INFINITY ? 0.f : sum.m;
        float s = 0.f, t = 0.f;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float d = v[i] - mu, e = lp_exp2(d * 1.4426950408889634f);
            s += e;
            t = fmaf(e, fmaxf(d, -1e30f), t);        // (0 x -inf would be NaN)
        }
        sum.s += s;
        sum.t += t;
        return mx;
    };
    auto weakest_value = [&]() {                     // values below it cannot be among the block's best
        const unsigned w = *reinterpret_cast<volatile unsigned*>(&sh_weakest);
        return w == 0u ? -INFINITY : lp_value(w);
    };
    auto publish = [&]() {
        const unsigned w = (unsigned)(best.weakest >> 32);
        if (lane == 0 && w > *reinterpret_cast<volatile unsigned*>(&sh_weakest)) atomicMax(&sh_weakest, w);
    };

    {   // the ends that are no whole vectors: up to N - 1 values on either side
        const int j = warp == 0 ? (lane < 16 ? j0 + lane : b + lane - 16) : j1;
        const bool there = warp == 0 && (lane < 16 ? j < a : j < j1);
        const float v[1] = {there ? to_f32<T>(x[j]) : -INFINITY};
        if (warp == 0) {
            add(v, 1);
            if (TOP) best.offer(there && v[0] == v[0] ? lp_key(v[0], j) : 0ull, top, lane);
        }
    }
    const uint4* src = reinterpret_cast<const uint4*>(x + a);
    for (int base = 0; base < n_vec; base += LP_THREADS * U) {
        uint4 raw[U];
        const bool full = base + LP_THREADS * U <= n_vec;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = base + u * LP_THREADS + tid;
            if (full || i < n_vec) raw[u] = __ldg(src + i);
        }
        float v[U * N];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float w[N];
            LpVec<T>::split(raw[u], w);
            const bool there = full || base + u * LP_THREADS + tid < n_vec;
#pragma unroll
            for (int e = 0; e < N; ++e) v[u * N + e] = there ? w[e] : -INFINITY;
        }
        const float mx = add(v, U * N);
        if (TOP) {
            const float least = weakest_value();
            if (__any_sync(0xffffffffu, mx >= least)) {
#pragma unroll
                for (int i = 0; i < U * N; ++i) {
                    const int at = base + (i / N) * LP_THREADS + tid;
                    const bool there = (full || at < n_vec) && v[i] >= least;
                    if (__any_sync(0xffffffffu, there)) best.offer(there ? lp_key(v[i], a + at * N + i % N) : 0ull, top, lane);
                }
                publish();
            }
        }
    }

    // ---- the block's warps, then the cluster's blocks
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const LpSums other{__shfl_xor_sync(0xffffffffu, sum.m, o), __shfl_xor_sync(0xffffffffu, sum.s, o), __shfl_xor_sync(0xffffffffu, sum.t, o)};
        sum = lp_join(sum, other);
    }
    if (lane == 0) warp_sums[warp] = sum;
    if (TOP) warp_best[warp][lane] = lane < top ? best.mine : 0ull;
    __syncthreads();
    if (warp == 0) {
        LpSums all = warp_sums[0];
        for (int w = 1; w < LP_WARPS; ++w) all = lp_join(all, warp_sums[w]);
        if (TOP)
            for (int w = 1; w < LP_WARPS; ++w) best.offer(warp_best[w][lane], top, lane);
        sum = all;
        if (lane == 0) part.sums = sum;
        if (TOP) part.best[lane] = lane < top ? best.mine : 0ull;
    }
    if (C > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        if (rank == 0 && warp == 0) {
            for (int r = 1; r < C; ++r) {
                const LpPart* other = cluster.map_shared_rank(&part, r);
                sum = lp_join(sum, other->sums);
                if (TOP) best.offer(other->best[lane], top, lane);
            }
        }
        cluster.sync();                              // nobody leaves while its shared memory is read
    }
    if (rank != 0 || warp != 0) return;
    const float log_s = logf(sum.s);
    if (lane == 0) {
        const int tok = tokens[row];
        const float given = tok >= 0 && tok < V ? to_f32<T>(x[tok]) : __int_as_float(0x7fc00000);
        lp_out[row] = (given - sum.m) - log_s;
        entropy_out[row] = log_s - sum.t / sum.s;
    }
    if (TOP && lane < top) {
        const bool any = best.mine != 0ull;
        top_lp[(size_t)row * top + lane] = any ? (lp_value((unsigned)(best.mine >> 32)) - sum.m) - log_s : __int_as_float(0x7fc00000);
        top_id[(size_t)row * top + lane] = any ? (int)(0xffffffffu - (unsigned)best.mine) : -1;
    }
}

template <typename T>
static int lp_launch(const void* logits, int rows, int V, long long row_stride, const int* tokens, int top, float* lp, float* entropy, float* top_lp,
                     int* top_id, int C, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows * (unsigned)C);
    cfg.blockDim = dim3(LP_THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = msgl_pdl_enabled() ? 2 : 1;
    if (top > 0) cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, true>, (const T*)logits, row_stride, V, tokens, top, lp, entropy, top_lp, top_id, C);
    else cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, false>, (const T*)logits, row_stride, V, tokens, top, lp, entropy, top_lp, top_id, C);
    return msgl_check_launch();
}

// blocks: how many blocks share a row (1, 2, 4 or 8: a portable cluster).  lp, entropy: [rows]; top_lp, top_id: [rows, top].
MSGL_API int msgl_token_logprobs(const void* logits, int rows, int vocab, long long row_stride, const int* tokens, int top, float* lp, float* entropy,
                                 float* top_lp, int* top_id, int blocks, int dtype, cudaStream_t stream) {
    if (rows <= 0) return MSGL_OK;
    if (vocab <= 0 || top < 0 || top > LP_MAX_TOP || top > vocab || (long long)rows * blocks > 0x7fffffffLL) return MSGL_ERR_SIZE;
    if (blocks != 1 && blocks != 2 && blocks != 4 && blocks != 8) return MSGL_ERR_SIZE;
    if (tokens == nullptr || (top > 0 && (top_lp == nullptr || top_id == nullptr))) return MSGL_ERR_SIZE;
    if (dtype == MSGL_F32) return lp_launch<float>(logits, rows, vocab, row_stride, tokens, top, lp, entropy, top_lp, top_id, blocks, stream);
    if (dtype == MSGL_BF16) return lp_launch<__nv_bfloat16>(logits, rows, vocab, row_stride, tokens, top, lp, entropy, top_lp, top_id, blocks, stream);
    return MSGL_ERR_DTYPE;
}
