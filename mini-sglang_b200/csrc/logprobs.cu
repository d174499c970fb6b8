// Log probabilities of given tokens, the entropy of every row and its most probable tokens, in one pass over the logits.
//
// Of a row x of V logits, with m = max x, s = sum e^(x_j - m) and t = sum e^(x_j - m) (x_j - m):
//
//     log p_j = (x_j - m) - log s            entropy = log s - t / s
//
// m, s and t are float32 and kept per thread; where m grows by d, s becomes s e^-d and t becomes (t - d s) e^-d.
//
// The most probable tokens are kept as 64-bit keys, the value's bits made to sort as whole numbers above the complement of the index: all
// keys differ, so the order is total (among equal logits the lower index comes first) and no schedule can change the outcome.  Every warp
// puts candidates into shared memory by itself: values above the block's `least`.  That is at first about the top-th largest of the
// threads' maxima in the block's first stretch (found bit by bit, with a count of the block a bit), which about `top` values of a stretch
// of random ones reach; after stretches 2, 4, 8, ... the block merges what the warps have found with its best so far, by counting for
// each how many are greater, and the weakest of the best becomes `least`.  So few stretches hold a candidate, and no barrier stands in
// those between.
//
// A row is read by a cluster of C blocks, whose first merges the others' sums and keys out of their shared memory: no scratch memory,
// no counters, one launch.
//
// Many rows are bound by their bytes, or by the instructions of a value where these are few bytes: 2,048 rows of 151,936 in float32 take 184 us without top tokens (6.8 TB/s), 198 with
// five, 205 with twenty, in bfloat16 153 with five (4.1 TB/s; some ten instructions a value).  Values go in pairs through the packed float32
// instructions, and the next stretch is asked for before the present one is worked on.  Few rows are bound by latency: one row with twenty takes
// 10.8 us (4.5 without): the launch, the first bound (1.2), eight blocks' share of the row, two merges and the cluster's two barriers follow on one another.
//
// A logit of -inf adds nothing.  A row with a NaN, with +inf or with nothing but -inf has NaN in all its probabilities, as the
// formula has; its top tokens are those of the highest numbers (a NaN is none).  A token outside the vocabulary gets NaN.
#include <cooperative_groups.h>
#include "common.cuh"

namespace cg = cooperative_groups;

constexpr int LP_MAX_TOP = 32, LP_PER = 16;      // values of a thread and stretch
constexpr int LP_ROOM = 128;                         // candidates that a warp has room for
constexpr int LP_REST = 4;                           // stretches that have to be left for a merge to pay
constexpr float LP_LOG2E = 1.4426950408889634f;

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
__device__ __forceinline__ float lp_exp(float x) { return lp_exp2(x * LP_LOG2E); }

// two float32 values in one 64-bit register, for the packed float32 instructions of sm_100
__device__ __forceinline__ unsigned long long lp_pack(float lo, float hi) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 lp_unpack(unsigned long long v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ unsigned long long lp_add2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long lp_mul2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long lp_fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

struct LpSums {
    float m, s, t;                                   // m: -inf where no number above it was seen (s = t = 0 then)
    // e^d is 0 from -200 on down; d itself is cut there, since d s may leave the range (a masked part of the type's lowest values) and t e^d be 0 x inf
    __device__ __forceinline__ void move(float to) {
        const float d = m == -INFINITY ? 0.f : fmaxf(m - to, -200.f), f = lp_exp(d);
        t = fmaf(s, d, t) * f;
        s *= f;
        m = to;
    }
};
// the sums of a warp's lanes, to all of them: the maximum first, so that every lane moves once
__device__ __forceinline__ LpSums lp_warp_join(LpSums a) {
    float to = a.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, o));
    a.move(to);                                      // (all -inf: to is -inf as a.m is, and nothing changes)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
        a.t += __shfl_xor_sync(0xffffffffu, a.t, o);
    }
    return a;
}

template <typename T> struct LpVec;
template <> struct LpVec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void split(const uint4& v, float* x) {
        x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
    }
};
template <> struct LpVec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void split(const uint4& v, float* x) {
        const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
};

// found[0 .. n) -> its best `top` in order, by a warp, or by a whole block; best: room for `top`
template <bool BLOCK>
__device__ __forceinline__ void lp_cut(unsigned long long* found, int n, int top, unsigned long long* best) {
    const int me = BLOCK ? (int)threadIdx.x : (int)(threadIdx.x & 31), size = BLOCK ? (int)blockDim.x : 32;
    auto sync = [&]() { if (BLOCK) __syncthreads(); else __syncwarp(); };
    sync();
#pragma unroll 1
    for (int i = me; i < n; i += size) {
        const unsigned long long key = found[i];
        int above = 0, j = 0;
#pragma unroll 4
        for (; j + 2 <= n; j += 2) {                 // two keys a load
            const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(found + j);
            above += (w.x > key ? 1 : 0) + (w.y > key ? 1 : 0);
        }
        if (j < n) above += found[j] > key ? 1 : 0;
        if (above < top) best[above] = key;
    }
    sync();
#pragma unroll 1
    for (int i = me; i < min(n, top); i += size) found[i] = best[i];
    sync();
}

template <typename T, bool TOP, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
token_logprobs_kernel(const T* __restrict__ logits, long long row_stride, int V, const int* __restrict__ tokens, int top, float* __restrict__ lp_out,
                      float* __restrict__ entropy_out, float* __restrict__ top_lp, int* __restrict__ top_id, int C) {
    constexpr int N = LpVec<T>::N, U = LP_PER / N, WARPS = THREADS / 32;
    constexpr unsigned ALL = 0xffffffffu;
    __shared__ __align__(16) unsigned long long found[TOP ? WARPS : 1][TOP ? LP_ROOM : 2];     // each warp's candidates
    __shared__ __align__(16) unsigned long long merged[TOP ? WARPS * LP_ROOM + LP_MAX_TOP : 2];      // the block's best in order, then what joins them
    __shared__ unsigned long long best_of[TOP ? WARPS : 1][TOP ? LP_MAX_TOP : 1];
    __shared__ LpSums warp_sums[WARPS], block_sums;
    __shared__ int sh_merged;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / C, rank = blockIdx.x - row * C;
    const T* x = logits + (size_t)row * row_stride;
    if (tid == 0) sh_merged = 0;
    pdl_launch_dependents();
    pdl_wait();
    pdl_after_wait();

    // this block's share [j0, j1) and within it the stretch [a, b) of whole aligned vectors
    const int per = (((V + C - 1) / C) + 7) & ~7;
    const int j0 = min(V, rank * per), j1 = min(V, j0 + per);
    const int lead = (int)((16 - ((uintptr_t)(x + j0) & 15)) & 15) / (int)sizeof(T);
    const int a = min(j1, j0 + lead), n_vec = (j1 - a) / N, b = a + n_vec * N;

    LpSums sum{-INFINITY, 0.f, 0.f};
    // A value counts if its key is above `weakest`.  Of a later stretch that is: above `least`, since what stands behind these has lower indices; all numbers
    // count as long as not `full`.
    unsigned long long weakest = 0ull;
    float least = -INFINITY;
    bool full = false;
    int held = 0, n_best = 0;                        // this warp's candidates, the block's best
    unsigned long long* mine = found[TOP ? warp : 0];
    auto raise = [&](unsigned long long key) { weakest = key; least = lp_value((unsigned)(key >> 32)); full = true; };
    auto merge = [&]() {                             // all threads
        __syncthreads();
        for (int i0 = 0; i0 < held; i0 += 32) {
            const unsigned long long key = i0 + lane < held ? mine[i0 + lane] : 0ull;
            const bool in = key != 0ull && key >= weakest;         // (a warp that ran out of room has its own weakest among them)
            const unsigned who = __ballot_sync(ALL, in);
            int at = 0;
            if (lane == 0) at = atomicAdd(&sh_merged, __popc(who));
            at = __shfl_sync(ALL, at, 0);
            if (in) merged[at + __popc(who & ((1u << lane) - 1u))] = key;
        }
        held = 0;
        __syncthreads();
        const int n = sh_merged;
        lp_cut<true>(merged, n, top, best_of[0]);
        n_best = min(n, top);
        if (tid == 0) sh_merged = n_best;
        if (n_best == top) raise(merged[top - 1]);
    };
    auto put = [&](bool in, float v, int j) {        // a value a lane
        const unsigned long long key = lp_key(v, j);
        in = in && v == v && key > weakest;
        unsigned who = __ballot_sync(ALL, in);
        if (held + __popc(who) > LP_ROOM) {
            lp_cut<false>(mine, held, top, best_of[TOP ? warp : 0]);
            held = top;
            raise(mine[top - 1]);
            in = in && key > weakest;
            who = __ballot_sync(ALL, in);
        }
        if (in) mine[held + __popc(who & ((1u << lane) - 1u))] = key;
        held += __popc(who);
    };
    const uint4* src = reinterpret_cast<const uint4*>(x + a);
    uint4 next[U];
    auto ask = [&](int base) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = base + u * THREADS + tid;
            if (i < n_vec) next[u] = __ldg(src + i);
        }
    };
    ask(0);
    for (int base = 0; base < n_vec; base += THREADS * U) {
        const bool whole = base + THREADS * U <= n_vec;
        float v[LP_PER];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            LpVec<T>::split(next[u], v + u * N);
            if (!whole && base + u * THREADS + tid >= n_vec)
#pragma unroll
                for (int e = 0; e < N; ++e) v[u * N + e] = -INFINITY;
        }
        ask(base + THREADS * U);
        float mx = v[0];
#pragma unroll
        for (int i = 1; i < LP_PER; ++i) mx = fmaxf(mx, v[i]);
        if (mx > sum.m) sum.move(mx);
        {
            const float m = sum.m == -INFINITY ? 0.f : sum.m;
            const unsigned long long m2 = lp_pack(-m, -m), c2 = lp_pack(LP_LOG2E, LP_LOG2E);
            unsigned long long s2 = 0ull, t2 = 0ull;               // (0.f, 0.f)
#pragma unroll
            for (int i = 0; i < LP_PER; i += 2) {
                const unsigned long long d = lp_add2(lp_pack(v[i], v[i + 1]), m2);
                const float2 y = lp_unpack(lp_mul2(d, c2));
                const unsigned long long e = lp_pack(lp_exp2(y.x), lp_exp2(y.y));
                s2 = lp_add2(s2, e);
                t2 = lp_fma2(e, d, t2);
            }
            const float2 s = lp_unpack(s2);
            const float2 t = lp_unpack(t2);
            float add_t = t.x + t.y;
            if (add_t != add_t) {                    // 0 x -inf somewhere, or a NaN: again, with -inf counted as nothing
                add_t = 0.f;
#pragma unroll
                for (int i = 0; i < LP_PER; ++i) add_t = fmaf(lp_exp(v[i] - m), fmaxf(v[i] - m, -1e30f), add_t);
            }
            sum.s += s.x + s.y;
            sum.t += add_t;
        }
        if (TOP) {
            const bool first = base == 0;
            if (first) {                             // the highest number that `top` threads' maxima reach, to 16 bits
                const unsigned o = mx == mx ? lp_order(mx) : 0u;
                unsigned bound = 0u;
                for (unsigned bit = 0x80000000u; bit >= 0x10000u; bit >>= 1)
                    if (__syncthreads_count(o >= (bound | bit)) >= top) bound |= bit;
                full = bound > lp_order(-INFINITY);
                if (full) least = lp_value(bound);
            }
            if (__any_sync(ALL, full && !first ? mx > least : mx >= least)) {
                auto index = [&](int i) { return a + (base + (i / N) * THREADS + tid) * N + i % N; };
                auto from = [&](float least_wanted) {    // this lane's values that reach it, a bit each
                    unsigned bits = 0u;
#pragma unroll
                    for (int i = 0; i < LP_PER; ++i) bits |= v[i] >= least_wanted ? 1u << i : 0u;
                    return bits;
                };
                unsigned there = ~0u;
                if (!whole) {
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (base + u * THREADS + tid >= n_vec) there &= ~(((1u << N) - 1u) << (u * N));
                }
                unsigned bits = from(least) & there;
                while (__any_sync(ALL, bits != 0u)) {    // a value a lane and round; few of both
                    const int at = __ffs(bits) - 1;
                    float w = v[0];
#pragma unroll
                    for (int i = 1; i < LP_PER; ++i) w = at == i ? v[i] : w;
                    put(bits != 0u, w, index(max(at, 0)));
                    bits &= bits - 1u;
                }
            }
            // (the numbers of stretches are the same for all threads)
            const int done = base / (THREADS * U) + 1;
            if (done > 1 && (done & (done - 1)) == 0 && base + (1 + LP_REST) * THREADS * U < n_vec) merge();
        }
    }
    if (warp == 0) {                                 // the ends that are no whole vectors: up to N - 1 values on either side
        const int j = lane < 16 ? j0 + lane : b + lane - 16;
        const bool there = j < (lane < 16 ? a : j1);
        const float v = there ? to_f32<T>(x[j]) : -INFINITY;
        if (v > sum.m) sum.move(v);
        const float d = v - (sum.m == -INFINITY ? 0.f : sum.m), e = lp_exp(d);
        sum.s += e;
        sum.t = fmaf(e, fmaxf(d, -1e30f), sum.t);    // (0 x -inf would be NaN)
        if (TOP) put(there, v, j);
    }

    // ---- the block's warps, then the cluster's blocks
    sum = lp_warp_join(sum);
    if (lane == 0) warp_sums[warp] = sum;
    if (TOP) merge();
    __syncthreads();
    if (warp == 0) {
        sum = lp_warp_join(lane < WARPS ? warp_sums[lane] : LpSums{-INFINITY, 0.f, 0.f});
        if (lane == 0) block_sums = sum;
    }
    if (C > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        if (rank == 0) {
            if (TOP) {                               // the others' best behind this block's own
                const int r = warp, i = lane;                // (32 at most)
                held = r > 0 && r < C ? *cluster.map_shared_rank(&sh_merged, r) : 0;
                if (i < held) mine[i] = cluster.map_shared_rank(merged, r)[i];
                merge();
            }
            if (warp == 0) sum = lp_warp_join(lane < C ? *cluster.map_shared_rank(&block_sums, lane) : LpSums{-INFINITY, 0.f, 0.f});
        }
        cluster.sync();                              // nobody leaves while its shared memory is read
    }
    if (rank != 0 || warp != 0) return;
    const float log_s = logf(sum.s);
    const float none = __int_as_float(0x7fc00000);
    if (lane == 0) {
        const int tok = tokens[row];
        lp_out[row] = tok >= 0 && tok < V ? (to_f32<T>(x[tok]) - sum.m) - log_s : none;
        entropy_out[row] = log_s - sum.t / sum.s;
    }
    if (TOP && lane < top) {
        const unsigned long long key = lane < n_best ? merged[lane] : 0ull;
        top_lp[(size_t)row * top + lane] = key ? (lp_value((unsigned)(key >> 32)) - sum.m) - log_s : none;
        top_id[(size_t)row * top + lane] = key ? (int)(0xffffffffu - (unsigned)key) : -1;
    }
}

template <typename T, int THREADS>
static int lp_launch(const void* logits, int rows, int V, long long row_stride, const int* tokens, int top, float* lp, float* entropy, float* top_lp,
                     int* top_id, int C, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows * (unsigned)C);
    cfg.blockDim = dim3(THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = msgl_pdl_enabled() ? 2 : 1;
    if (top > 0) cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, true, THREADS>, (const T*)logits, row_stride, V, tokens, top, lp, entropy, top_lp, top_id, C);
    else cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, false, THREADS>, (const T*)logits, row_stride, V, tokens, top, lp, entropy, top_lp, top_id, C);
    return msgl_check_launch();
}

// blocks: how many blocks share a row (1, 2, 4 or 8: a portable cluster); large: blocks of 512 threads, not of 256.  lp, entropy: [rows]; top_lp, top_id: [rows, top].
MSGL_API int msgl_token_logprobs(const void* logits, int rows, int vocab, long long row_stride, const int* tokens, int top, float* lp, float* entropy,
                                 float* top_lp, int* top_id, int blocks, int large, int dtype, cudaStream_t stream) {
    if (rows <= 0) return MSGL_OK;
    if (vocab <= 0 || top < 0 || top > LP_MAX_TOP || top > vocab || (long long)rows * blocks > 0x7fffffffLL) return MSGL_ERR_SIZE;
    if (blocks != 1 && blocks != 2 && blocks != 4 && blocks != 8) return MSGL_ERR_SIZE;
    if (tokens == nullptr || (top > 0 && (top_lp == nullptr || top_id == nullptr))) return MSGL_ERR_SIZE;
#define MSGL_LP(T, THREADS) lp_launch<T, THREADS>(logits, rows, vocab, row_stride, tokens, top, lp, entropy, top_lp, top_id, blocks, stream)
    if (dtype == MSGL_F32) return large ? MSGL_LP(float, 512) : MSGL_LP(float, 256);
    if (dtype == MSGL_BF16) return large ? MSGL_LP(__nv_bfloat16, 512) : MSGL_LP(__nv_bfloat16, 256);
#undef MSGL_LP
    return MSGL_ERR_DTYPE;
}
