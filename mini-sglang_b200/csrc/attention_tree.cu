// Attention for trees of drafted tokens over the paged cache.
//
// Request r brings n = q_start[r + 1] - q_start[r] drafts whose keys and values are the last n of its kv_len[r] cached ones.  A draft sees
// every key before them and of the drafts those whose bits are set in its mask row (its ancestors and itself, as draft_plan makes them, or
// any other set):
//
//     o_i = sum_j p_ij v_j,   p_i = softmax over the keys that i sees of scale q_i k_j;   a draft that sees none gets 0
//
// What a draft does not see counts for nothing, whatever its key and value hold.  Query head h reads kv head h / G, G = n_q / n_kv.  The
// cache is [page][kv head][slot][d]; the key at place i of request r lies in page block_table[r][i / P], slot i % P.
//
// Work.  A row is a (draft, head of the group) pair, so all rows of a kv head share its keys.  An item is up to ROWS rows of one request
// under one kv head; its keys are cut into tiles of KT.  All items are laid end to end, an item as long as its tiles and TREE_HEAD
// more (what it costs beside them), and cut into one equal run a block: every block works out its run from the
// requests' lengths by itself, so the host knows none of them and a captured launch serves any.  A block that has a whole item writes
// its rows; of one that is cut every block leaves float32 partial sums with their maximum and sum of weights, and a second launch joins
// them in the order of the keys.  What a small launch takes, at 8 drafts behind 1,000 keys (32 query heads on 8) 12.2 us: 1.8 until the work is cut, 1.5 for a
// page's number and its copy's start, 2.5 for a tile, 1.8 to the last store, 1 to the join's start and 2 in it.
#include "common.cuh"
#include <math.h>

__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ float fast_exp2(float x) {          // 2^x by the special-function unit (relative error about 2^-22; -inf gives 0)
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<unsigned*>(&v);
}

struct TreeRecord {               // the cut item whose first piece a block has
    int pieces;                   // 0: it has none
    int rows, tok0, row0, kvh;    // rows of the item, the first of them among the request's under the kv head, the request's first draft
    int pad[3];
};

struct TreeParams {
    const void* q;                // [T, n_q, d]
    void* out;
    const void* k_cache;          // [pages, n_kv, page_size, d]
    const void* v_cache;
    const int* q_start;           // [B + 1]
    const int* kv_len;            // [B]
    const int* table;             // [B, table_width], rows table_stride apart
    const unsigned* mask;         // [T, words]
    // Partial results, by four columns and then by rows: what a warp's 32 rows write or read of one column lies side by side (row by row, 64 drafts of
    // one request behind 4,096 keys spent 6 us on writing them and 7 on the join).
    float* part_o;                // [2 * blocks][ceil(d / 4)][ROWS][4]
    float* part_ml;               // [2 * blocks][ROWS][2]  (maximum in log2 units, sum of the weights)
    struct TreeRecord* record;    // [blocks]
    int B, T, n_q, n_kv, G, d, page_size, page_shift, table_stride, table_width, words;
    long long pages;
    float scale_log2;             // scale * log2(e)
    int max_draft;                // most drafts of a request
    int vectors;                  // rows of the caches are whole 16 bytes, on 16-byte boundaries
};

// ---------------------------------------------------------------------------------------
// the cut of the work
// ---------------------------------------------------------------------------------------
constexpr int TREE_HEAD = 1;      // what an item costs beside its tiles, in tiles
constexpr int TREE_SHARE = TREE_HEAD + 1;      // a block's run is no shorter: so no piece of an item is empty and none lies in more than its blocks

struct TreeSegment {              // tiles [t_lo, t_hi) of one item
    int r, kvh, row0, rows;       // row0: first row of the item among the request's n * G under the kv head
    int tok0, n, kv, base;        // the request's first draft in the stream, its drafts, its keys, those before the drafts
    int t_lo, t_hi, tiles;
};

struct TreeWalkState { int whole, rest, x_lo, x_hi, start, blocks, r, item; };      // (a walk put aside)
struct TreeStart {                // what the block's walkers start with: the first segment, and the walk behind it
    TreeWalkState walk;
    TreeSegment first;
    int work;
};

template <int ROWS, int KT>
struct TreeWalk {
    const TreeParams& p;
    int blocks;                   // in use
    int whole, rest;              // the work's length (the host has seen to it that it fits) over them, and what is left
    int x_lo, x_hi;               // this block's run
    int r = 0, item = 0;
    int start = 0;                // where the request's first item starts

    __device__ __forceinline__ TreeWalk(const TreeParams& q) : p(q) {}
    __device__ __forceinline__ void store(TreeWalkState& s) const { s.whole = whole; s.rest = rest; s.x_lo = x_lo; s.x_hi = x_hi; s.start = start; s.blocks = blocks; s.r = r; s.item = item; }
    __device__ __forceinline__ void load(const TreeWalkState& s) { whole = s.whole; rest = s.rest; x_lo = s.x_lo; x_hi = s.x_hi; start = s.start; blocks = s.blocks; r = s.r; item = s.item; }
    struct Request { int tok0, n, kv, base, tiles, groups, items; };      // groups: items under a kv head
    __device__ __forceinline__ Request request(int i) const {
        Request w;
        w.tok0 = min(max(p.q_start[i], 0), p.T);
        const int brought = min(max(p.q_start[i + 1], w.tok0), p.T) - w.tok0;
        w.n = min(brought, p.max_draft);             // (drafts beyond the host's bound have no rows; their keys are the last ones all the same)
        w.kv = (int)min((long long)max(p.kv_len[i], 0), (long long)p.table_width * p.page_size);
        w.base = w.kv - brought;
        w.tiles = max(1, (w.kv + KT - 1) / KT);
        w.groups = (w.n * p.G + ROWS - 1) / ROWS;
        w.items = p.n_kv * w.groups;
        return w;
    }
    // floor(a / b) of whole numbers below 2^24, by the reciprocal: one thread finds the first segment for all, and waits for every division
    static __device__ __forceinline__ int quotient(int a, int b) {
        int q = (int)(__fdividef((float)a, (float)b));
        q -= q * b > a ? 1 : 0;
        return q + (a - q * b >= b ? 1 : 0);
    }
    __device__ __forceinline__ int cut_at(int k) const { return whole * k + quotient(rest * k, blocks); }      // floor(total k / blocks); (k and rest: some hundreds)
    // the tile that a cut at x falls on, in an item that starts at `s`
    __device__ __forceinline__ int tile_at(int x, int s, int tiles) const {
        return min(max(x - s - TREE_HEAD, 0), tiles);
    }
    // All threads of the block: the run of block j of nb; false: it has none.  The thread whose request the run starts in finds the first segment for all:
    // every further look at the lengths would be a wait for memory (walking from its start each by itself took the warps 2 us longer).
    __device__ __forceinline__ bool begin(int j, int nb, TreeStart& to) {
        __shared__ int sums[32];
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n_warps = blockDim.x >> 5;
        const int per = (p.B + blockDim.x - 1) / blockDim.x, i0 = min(p.B, tid * per), i1 = min(p.B, i0 + per);
        int mine = 0;
        Request w = {};                              // the thread's last request: where each has one, it is not looked at again
        for (int i = i0; i < i1; ++i) { w = request(i); mine += w.items * (w.tiles + TREE_HEAD); }
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += v; }
        if (lane == 31) sums[warp] = upto;
        if (tid == 0) to.work = 0;
        __syncthreads();
        int before = upto - mine, total = 0;
        const int warps = per == 1 ? (p.B + 31) >> 5 : n_warps;          // that have any
        for (int k = 0; k < warps; ++k) { if (k < warp) before += sums[k]; total += sums[k]; }
        blocks = max(1, min(nb, total / TREE_SHARE));
        if (total == 0 || j >= blocks) return false;
        whole = total / blocks;
        rest = total - whole * blocks;
        x_lo = cut_at(j);
        x_hi = cut_at(j + 1);
        if (x_lo >= before && x_lo < before + mine) {
            start = before;
            r = i0;
            if (per > 1)
                for (;; ++r) {
                    w = request(r);
                    const int len = w.items * (w.tiles + TREE_HEAD);
                    if (x_lo < start + len || r + 1 >= i1) break;
                    start += len;
                }
            item = (x_lo - start) / (w.tiles + TREE_HEAD);
            // (a run is long enough to hold a tile of the item that it starts in)
            const int s = start + item * (w.tiles + TREE_HEAD), e = s + w.tiles + TREE_HEAD;
            to.first = segment(w, x_lo > s ? tile_at(x_lo, s, w.tiles) : 0, x_hi < e ? tile_at(x_hi, s, w.tiles) : w.tiles);
            ++item;
            to.work = 1;
            store(to.walk);
        }
        __syncthreads();
        load(to.walk);
        return to.work != 0;
    }
    // tiles [lo, hi) of item `item` of request r, which is w
    __device__ __forceinline__ TreeSegment segment(const Request& w, int lo, int hi) const {
        const int kvh = w.groups == 1 ? item : item / w.groups, row0 = (item - kvh * w.groups) * ROWS;
        return TreeSegment{r, kvh, row0, min(ROWS, w.n * p.G - row0), w.tok0, w.n, w.kv, w.base, lo, hi, w.tiles};
    }
    // the next segment of the run; false: it is done
    __device__ __forceinline__ bool next(TreeSegment& g) {
        while (r < p.B) {
            const Request w = request(r);
            const int len = w.tiles + TREE_HEAD;
            for (; item < w.items; ++item) {
                const int s = start + item * len;
                if (s >= x_hi) return false;
                const int lo = x_lo > s ? tile_at(x_lo, s, w.tiles) : 0, hi = x_hi < s + len ? tile_at(x_hi, s, w.tiles) : w.tiles;
                if (lo >= hi) continue;
                g = segment(w, lo, hi);
                ++item;
                return true;
            }
            start += w.items * len;
            item = 0;
            ++r;
        }
        return false;
    }
    // pieces of the item whose first piece `g` is, in block j
    __device__ __forceinline__ int pieces(const TreeSegment& g, int j) const {
        const int s = start + (item - 1) * (g.tiles + TREE_HEAD), e = s + g.tiles + TREE_HEAD;
        int k = j + 1;
        while (k < blocks) {
            const int x = cut_at(k + 1);
            ++k;
            if (x >= e || tile_at(x, s, g.tiles) >= g.tiles) break;
        }
        return k - j;
    }
};

// 32 keys from key0 on, a bit each: does the draft with mask row `row` see them?  (all before base; none from kv on)
__device__ __forceinline__ unsigned tree_seen(const unsigned* row, int words, int key0, int base, int kv) {
    const int d0 = key0 - base;
    unsigned m;
    if (d0 <= -32) m = ~0u;
    else if (d0 < 0) m = (words > 0 ? row[0] << -d0 : 0u) | ((1u << -d0) - 1u);
    else {
        const int w = d0 >> 5, s = d0 & 31;
        m = w < words ? row[w] >> s : 0u;
        if (s > 0 && w + 1 < words) m |= row[w + 1] << (32 - s);
    }
    const int left = kv - key0;
    return left >= 32 ? m : left <= 0 ? 0u : m & ((1u << left) - 1u);
}

__device__ __forceinline__ int tree_page(const TreeParams& p, int key) { return p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size; }

struct TreeYes { static constexpr bool value = true; };
struct TreeNo { static constexpr bool value = false; };
template <typename T> struct TsVec;                  // 16 bytes of a row; MOST: of them one of eight threads has for 128 columns
template <> struct TsVec<float> {
    static constexpr int N = 4, MOST = 4;
    static __device__ __forceinline__ void store(float* to, const uint4& v) { *reinterpret_cast<uint4*>(to) = v; }
};
template <> struct TsVec<__nv_bfloat16> {
    static constexpr int N = 8, MOST = 2;
    static __device__ __forceinline__ void store(float* to, const uint4& v) {
        *reinterpret_cast<uint4*>(to) = make_uint4(v.x << 16, v.x & 0xffff0000u, v.y << 16, v.y & 0xffff0000u);
        *reinterpret_cast<uint4*>(to + 4) = make_uint4(v.z << 16, v.z & 0xffff0000u, v.w << 16, v.w & 0xffff0000u);
    }
};

// ---------------------------------------------------------------------------------------
// Head sizes up to 128 and some work, any page size, float32 or bfloat16 data, float32 arithmetic: 64 rows a block, tiles of 64 keys, two blocks an SM.
//
// Warp w owns rows 16 (w / 2) .. + 15 and, of the scores, half of the keys, of O, half of the columns.  A thread has four rows (every fourth) against four
// keys (every eighth) and then against eight columns: eight loads of 16 bytes for 64 multiply-adds, three for 32, and no two lanes meet a
// bank.  The two warps of a row meet over its maximum.  P takes the place of the keys, key by key, a thread's four rows side by side.  A tile takes an SM 18,700
// cycles (2 requests of 64 drafts behind 4,000 keys, 40 query heads on 8: 344 us, 30 TFLOP/s), of which shared memory's 128 bytes a cycle account for 14,300 and the
// multiply-adds for 8,200; eight rows a thread, which takes a third off the first, leaves too few warps to hide its latency (342 us).  A key that a row does not see
// has the weight -1, which the product leaves out: its value may be anything.
// ---------------------------------------------------------------------------------------
constexpr int TF_ROWS = 64, TF_KT = 64, TF_D = 128, TF_THREADS = 256, TF_PITCH = TF_D + 4, TF_PPITCH = TF_ROWS + 4;
constexpr size_t TF_SMEM = (size_t)(TF_ROWS + 2 * TF_KT) * TF_PITCH * sizeof(float);
static_assert(TF_PPITCH <= TF_PITCH, "P lies over the keys");

__device__ __forceinline__ void tf_cp_async16(float* to, const void* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_u32(to)), "l"(from), "r"(there ? 16 : 0));
}

template <typename T>
__global__ void __launch_bounds__(TF_THREADS, 2) tree_tile_kernel(const TreeParams p) {
    extern __shared__ __align__(16) float tf_smem[];
    __shared__ float sh_max[2][TF_ROWS], sh_sum[2][TF_ROWS];
    __shared__ TreeStart begun;
    float* Qs = tf_smem;                             // [64][pitch]; columns from d on are zero, in all three
    float* Ks = Qs + TF_ROWS * TF_PITCH;
    float* Vs = Ks + TF_KT * TF_PITCH;
    float* Ps = Ks;                                  // [64 keys][64 rows + 4]
    const int d = p.d, d4 = (d + 3) >> 2, G = p.G, j = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, side = warp & 1, rg = lane >> 3, kg = lane & 7, row_base = (warp >> 1) * 16;
    pdl_launch_dependents();
    pdl_wait();
    pdl_after_wait();
    TreeWalk<TF_ROWS, TF_KT> walk(p);
    TreeRecord record = {};
    if (walk.begin(j, gridDim.x, begun)) {
        for (int i = tid; i < (TF_ROWS + 2 * TF_KT) * TF_PITCH; i += TF_THREADS) tf_smem[i] = 0.f;
        TreeSegment g = begun.first;
        for (bool more = true; more; more = walk.next(g)) {
            __syncthreads();                         // the segment before has been read
            const int my_key = tid >> 2, sub = tid & 3;
            {
                const int rr = g.row0 + my_key;
                const T* src = reinterpret_cast<const T*>(p.q) + ((size_t)(g.tok0 + rr / G) * p.n_q + (size_t)g.kvh * G + rr % G) * d;
                for (int c = sub; c < d; c += 4) Qs[my_key * TF_PITCH + c] = my_key < g.rows ? to_f32<T>(src[c]) : 0.f;
            }
            float o[4][8], m_run[4], l_run[4];
            const unsigned* row_mask[4];
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                m_run[a] = -INFINITY;
                l_run[a] = 0.f;
                row_mask[a] = p.mask + (size_t)(g.tok0 + (g.row0 + min(row_base + rg + 4 * a, g.rows - 1)) / G) * p.words;
#pragma unroll
                for (int c = 0; c < 8; ++c) o[a][c] = 0.f;
            }
            const bool busy = row_base < g.rows;     // whether the warp has rows
            for (int t = g.t_lo; t < g.t_hi; ++t) {
                const int key0 = t * TF_KT;
                __syncthreads();                     // the tile before has been read
                {
                    const int key = key0 + my_key;
                    long long at = -1;               // element offset of the key's row
                    if (key < g.kv) {
                        const int pi = tree_page(p, key), id = p.table[(size_t)g.r * p.table_stride + pi];
                        if (id >= 0 && id < p.pages) at = (((long long)id * p.n_kv + g.kvh) * p.page_size + (key - pi * p.page_size)) * d;
                    }
                    const T* k = reinterpret_cast<const T*>(p.k_cache) + max(at, 0ll);
                    const T* v = reinterpret_cast<const T*>(p.v_cache) + max(at, 0ll);
                    float* to_k = Ks + my_key * TF_PITCH;
                    float* to_v = Vs + my_key * TF_PITCH;
                    constexpr int N = TsVec<T>::N;
                    // (P lay over the keys: what is no head element has to be zero again)
                    for (int c = d + sub; c < TF_PITCH; c += 4) to_k[c] = 0.f;
                    if (p.vectors && sizeof(T) == 4) {
#pragma unroll 8
                        for (int c = sub * N; c < d; c += 4 * N) {
                            tf_cp_async16(to_k + c, k + c, at >= 0);
                            tf_cp_async16(to_v + c, v + c, at >= 0);
                        }
                        asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;\n" ::: "memory");
                    } else if (p.vectors) {
                        uint4 raw[2][TF_D / (4 * N)];
#pragma unroll
                        for (int i = 0; i < TF_D / (4 * N); ++i) {
                            const int c = (sub + 4 * i) * N;
                            const bool there = at >= 0 && c < d;
                            raw[0][i] = there ? *reinterpret_cast<const uint4*>(k + c) : make_uint4(0u, 0u, 0u, 0u);
                            raw[1][i] = there ? *reinterpret_cast<const uint4*>(v + c) : make_uint4(0u, 0u, 0u, 0u);
                        }
#pragma unroll
                        for (int i = 0; i < TF_D / (4 * N); ++i) {
                            const int c = (sub + 4 * i) * N;
                            if (c >= d) continue;
                            TsVec<T>::store(to_k + c, raw[0][i]);
                            TsVec<T>::store(to_v + c, raw[1][i]);
                        }
                    } else {
                        for (int c = sub; c < d; c += 4) {
                            to_k[c] = at >= 0 ? to_f32<T>(k[c]) : 0.f;
                            to_v[c] = at >= 0 ? to_f32<T>(v[c]) : 0.f;
                        }
                    }
                }
                __syncthreads();
                float s[4][4];
#pragma unroll
                for (int a = 0; a < 4; ++a) s[a][0] = s[a][1] = s[a][2] = s[a][3] = 0.f;
                const bool ends = key0 + TF_KT > g.base;
                if (busy) {
                    const float* q0 = Qs + (row_base + rg) * TF_PITCH;
                    const float* k0 = Ks + (32 * side + kg) * TF_PITCH;
#pragma unroll 2
                    for (int c = 0; c < 4 * d4; c += 4) {
                        float4 q4[4], k4[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            q4[i] = *reinterpret_cast<const float4*>(q0 + 4 * i * TF_PITCH + c);
                            k4[i] = *reinterpret_cast<const float4*>(k0 + 8 * i * TF_PITCH + c);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e)          // (sixteen sums between two terms of one)
#pragma unroll
                            for (int a = 0; a < 4; ++a)
#pragma unroll
                                for (int b = 0; b < 4; ++b)
                                    s[a][b] = fmaf(e == 0 ? q4[a].x : e == 1 ? q4[a].y : e == 2 ? q4[a].z : q4[a].w, e == 0 ? k4[b].x : e == 1 ? k4[b].y : e == 2 ? k4[b].z : k4[b].w, s[a][b]);
                    }
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        const unsigned seen = ends ? tree_seen(row_mask[a], p.words, key0 + 32 * side, g.base, g.kv) : ~0u;
                        float mx = -INFINITY;
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            s[a][b] = seen >> (kg + 8 * b) & 1u ? s[a][b] * p.scale_log2 : -INFINITY;
                            mx = fmaxf(mx, s[a][b]);
                        }
#pragma unroll
                        for (int w = 1; w < 8; w <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
                        if (kg == 0) sh_max[side][row_base + rg + 4 * a] = mx;
                    }
                }
                __syncthreads();                     // the keys have been read, the maxima are there
                if (busy) {
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        const int row = row_base + rg + 4 * a;
                        const float mx = fmaxf(m_run[a], fmaxf(sh_max[0][row], sh_max[1][row])), mu = mx == -INFINITY ? 0.f : mx, f = fast_exp2(m_run[a] - mu);
                        const unsigned seen = ends ? tree_seen(row_mask[a], p.words, key0 + 32 * side, g.base, g.kv) : ~0u;
                        m_run[a] = mx;
                        float sum = 0.f;
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            const float e = fast_exp2(s[a][b] - mu);
                            sum += e;
                            s[a][b] = seen >> (kg + 8 * b) & 1u ? e : -1.f;
                        }
                        l_run[a] = fmaf(l_run[a], f, sum);       // this thread's keys alone
#pragma unroll
                        for (int c = 0; c < 8; ++c) o[a][c] *= f;
                    }
#pragma unroll
                    for (int b = 0; b < 4; ++b)
                        *reinterpret_cast<float4*>(Ps + (32 * side + kg + 8 * b) * TF_PPITCH + row_base + 4 * rg) = make_float4(s[0][b], s[1][b], s[2][b], s[3][b]);
                }
                __syncthreads();
                if (busy) {
                    auto product = [&](auto guarded) {
#pragma unroll 4
                        for (int key = 0; key < TF_KT; ++key) {
                            const float4 w4 = *reinterpret_cast<const float4*>(Ps + key * TF_PPITCH + row_base + 4 * rg);
                            const float4 va = *reinterpret_cast<const float4*>(Vs + key * TF_PITCH + 64 * side + 4 * kg);
                            const float4 vb = *reinterpret_cast<const float4*>(Vs + key * TF_PITCH + 64 * side + 4 * kg + 32);
                            const float w[4] = {w4.x, w4.y, w4.z, w4.w}, v[8] = {va.x, va.y, va.z, va.w, vb.x, vb.y, vb.z, vb.w};
#pragma unroll
                            for (int a = 0; a < 4; ++a) {
                                if (decltype(guarded)::value && w[a] < 0.f) continue;
#pragma unroll
                                for (int c = 0; c < 8; ++c) o[a][c] = fmaf(w[a], v[c], o[a][c]);
                            }
                        }
                    };
                    if (ends) product(TreeYes());
                    else product(TreeNo());
                }
            }
            // ---- the segment's end
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                float l = l_run[a];
#pragma unroll
                for (int w = 1; w < 8; w <<= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
                if (kg == 0) sh_sum[side][row_base + rg + 4 * a] = l;
            }
            __syncthreads();
            const bool whole = g.t_lo == 0 && g.t_hi == g.tiles;
            const int slot = 2 * j + (g.t_lo == 0 ? 1 : 0);
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const int row = row_base + rg + 4 * a;
                if (row >= g.rows) continue;
                const float l = sh_sum[0][row] + sh_sum[1][row];
                if (whole) {
                    const int rr = g.row0 + row;
                    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
                    T* dst = reinterpret_cast<T*>(p.out) + ((size_t)(g.tok0 + rr / G) * p.n_q + (size_t)g.kvh * G + rr % G) * d;
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const int col = 64 * side + 4 * kg + (c >> 2) * 32 + (c & 3);
                        if (col < d) dst[col] = from_f32<T>(o[a][c] * inv);
                    }
                } else {
                    float4* dst = reinterpret_cast<float4*>(p.part_o) + (size_t)slot * d4 * TF_ROWS + row;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (16 * side + kg + 8 * h < d4) dst[(16 * side + kg + 8 * h) * TF_ROWS] = make_float4(o[a][4 * h], o[a][4 * h + 1], o[a][4 * h + 2], o[a][4 * h + 3]);
                    if (side == 0 && kg == 0) *reinterpret_cast<float2*>(p.part_ml + ((size_t)slot * TF_ROWS + row) * 2) = make_float2(m_run[a], l);
                }
            }
            if (!whole && g.t_lo == 0) record = TreeRecord{walk.pieces(g, j), g.rows, g.tok0, g.row0, g.kvh, {0, 0, 0}};
        }
    }
    if (tid == 0) p.record[j] = record;
}

// ---------------------------------------------------------------------------------------
// Head sizes up to 512, any page size, float32 or bfloat16 data, float32 arithmetic: 32 rows a block, tiles of 32 keys.
//
// Warp w owns rows 4 w .. 4 w + 3.  Scores: lane = key, four rows a lane, K rows of odd 16-byte pitch, so that a warp's loads of them
// meet no bank twice; P^T goes to shared memory (four rows a key side by side) and O is four rows x 4 CB columns a lane.  Bound by what
// shared memory delivers (five loads of 16 bytes for sixteen multiply-adds of the scores, two of O's), its steps are shorter than those of the kernel above.
// float32, head size 128, this one / that one, us: groups of four, 1 request of 32 drafts behind 500 keys 26 / 49, 8 of 20 behind 100 40 / 41, 16 of 30 behind 300
// 151 / 131, 2 of 12 behind 6,000 152 / 117, 4 of 26 behind 1,500 158 / 123; of two, 4 of 26 behind 1,500 86 / 72, 1 of 64 behind 2,000 66 / 56, 8 of 40 behind 500 (80 rows,
// of 96 and of 128) 95 / 104; of five, 2 of 64 behind 4,000 475 / 344.  So it stands where there are no more than 32 rows, fewer than three tiles of the other an
// SM, or where these are more than a third of its own tiles (as far as the host knows: the table's width; a table of some thousand keys a request whose
// requests are short goes to that one all the same: 4 of 26 behind 200 26 / 49, groups of four, 2 of 12 behind 600 31 / 47, 8 of 20 behind 100 40 / 40, 16 of 30 behind 100, groups of two, 49 / 56).
// bfloat16 heads other than the tensor cores' (4 requests behind 4,000 keys, 16 heads on 4; us, 8 / 32 drafts): heads of 96 52 / 116, of 192 88 / 289, of 256 106 / 349 (keys and values alone
// 4, 8 and 10); rows of 320 that are key and value of 16 heads at once, 1 request 56 / 143, 16 requests 538 / 2,071 (6): multiply-adds at 0.2 to 0.37 of their rate, and keys read again for every 32 rows.
// ---------------------------------------------------------------------------------------
constexpr int TS_ROWS = 32, TS_KT = 32, TS_THREADS = 256;

template <typename T, int CB>
__global__ void __launch_bounds__(TS_THREADS, CB <= 2 ? 2 : 1) tree_simt_kernel(const TreeParams p) {
    extern __shared__ __align__(16) float ts_smem[];
    const int d = p.d, pitch = CB * 128 + 4, d4 = (d + 3) >> 2;
    float* Qs = ts_smem;                             // [32][pitch]; columns from d on are zero
    float* Ks = Qs + TS_ROWS * pitch;                // [32][pitch]
    float* Vs = Ks + TS_KT * pitch;                  // [32][pitch]
    float* Ps = Vs + TS_KT * pitch;                  // [8 warps][32 keys][4 rows]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, j = blockIdx.x;
    const int G = p.G;
    pdl_launch_dependents();
    pdl_wait();
    pdl_after_wait();
    TreeWalk<TS_ROWS, TS_KT> walk(p);
    TreeRecord record = {};
    __shared__ TreeStart begun;
    if (walk.begin(j, gridDim.x, begun)) {
        for (int i = tid; i < (TS_ROWS + 2 * TS_KT) * pitch; i += TS_THREADS) ts_smem[i] = 0.f;      // (what lies from d on stays zero)
        TreeSegment g = begun.first;
        for (bool more = true; more; more = walk.next(g)) {
            const T* q = reinterpret_cast<const T*>(p.q);
            __syncthreads();                         // the segment before has been read
            {
                const int row = tid >> 3, rr = g.row0 + row;
                const T* src = q + ((size_t)(g.tok0 + rr / G) * p.n_q + (size_t)g.kvh * G + rr % G) * d;
                for (int c = tid & 7; c < d; c += 8) Qs[row * pitch + c] = row < g.rows ? to_f32<T>(src[c]) : 0.f;
            }
            float o[4][CB][4], m_run[4], l_run[4];
            const unsigned* row_mask[4];
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                m_run[a] = -INFINITY;
                l_run[a] = 0.f;
                const int row = min(4 * warp + a, g.rows - 1);
                row_mask[a] = p.mask + (size_t)(g.tok0 + (g.row0 + row) / G) * p.words;
#pragma unroll
                for (int b = 0; b < CB; ++b) o[a][b][0] = o[a][b][1] = o[a][b][2] = o[a][b][3] = 0.f;
            }
            // a thread fetches pieces of one key and its value, eight threads a key: 16 bytes at a time where the rows are made of them, the next tile's while
            // this one is worked on (head sizes up to 128)
            const int my_key = tid >> 3, sub = tid & 7;
            uint4 raw_k[TsVec<T>::MOST * CB], raw_v[TsVec<T>::MOST * CB];
            auto place = [&](int key) -> long long {         // element offset of the key's row, or -1
                if (key >= g.kv) return -1;
                const int pi = tree_page(p, key), id = p.table[(size_t)g.r * p.table_stride + pi];
                return id >= 0 && id < p.pages ? (((long long)id * p.n_kv + g.kvh) * p.page_size + (key - pi * p.page_size)) * d : -1;
            };
            auto fetch = [&](int t) {
                const long long at = place(t * TS_KT + my_key);
#pragma unroll
                for (int i = 0; i < TsVec<T>::MOST * CB; ++i) {
                    const int c = (sub + 8 * i) * TsVec<T>::N;
                    const bool there = at >= 0 && c < d;
                    raw_k[i] = there ? *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.k_cache) + at + c) : make_uint4(0u, 0u, 0u, 0u);
                    raw_v[i] = there ? *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.v_cache) + at + c) : make_uint4(0u, 0u, 0u, 0u);
                }
            };
            auto put_down = [&]() {
#pragma unroll
                for (int i = 0; i < TsVec<T>::MOST * CB; ++i) {
                    const int c = (sub + 8 * i) * TsVec<T>::N;
                    if (c >= d) continue;
                    TsVec<T>::store(Ks + my_key * pitch + c, raw_k[i]);
                    TsVec<T>::store(Vs + my_key * pitch + c, raw_v[i]);
                }
            };
            if (p.vectors && CB == 1) fetch(g.t_lo);
            for (int t = g.t_lo; t < g.t_hi; ++t) {
                const int key0 = t * TS_KT;
                __syncthreads();                     // the tile before has been read (and Q written)
                if (p.vectors) {
                    if (CB > 1) fetch(t);
                    put_down();
                } else {
                    const long long at = place(key0 + my_key);
                    for (int c = sub; c < d; c += 8) {
                        Ks[my_key * pitch + c] = at >= 0 ? to_f32<T>(reinterpret_cast<const T*>(p.k_cache)[at + c]) : 0.f;
                        Vs[my_key * pitch + c] = at >= 0 ? to_f32<T>(reinterpret_cast<const T*>(p.v_cache)[at + c]) : 0.f;
                    }
                }
                __syncthreads();
                if (p.vectors && CB == 1 && t + 1 < g.t_hi) fetch(t + 1);
                if (4 * warp >= g.rows) continue;    // (no row of this warp)
                float s[4] = {0.f, 0.f, 0.f, 0.f};
                for (int c = 0; c < d4; ++c) {
                    const float4 k4 = *reinterpret_cast<const float4*>(Ks + lane * pitch + 4 * c);
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        const float4 q4 = *reinterpret_cast<const float4*>(Qs + (4 * warp + a) * pitch + 4 * c);
                        s[a] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, s[a]))));
                    }
                }
                const bool ends = key0 + TS_KT > g.base;
                float w[4];
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    const unsigned seen = ends ? tree_seen(row_mask[a], p.words, key0, g.base, g.kv) : ~0u;
                    const bool in = seen >> lane & 1u;
                    s[a] = in ? s[a] * p.scale_log2 : -INFINITY;
                    const float mx = fmaxf(m_run[a], warp_max(s[a])), mu = mx == -INFINITY ? 0.f : mx;
                    const float f = fast_exp2(m_run[a] - mu), e = fast_exp2(s[a] - mu);
                    m_run[a] = mx;
                    l_run[a] = fmaf(l_run[a], f, e);             // this lane's keys alone
                    w[a] = in ? e : -1.f;
#pragma unroll
                    for (int b = 0; b < CB; ++b) { o[a][b][0] *= f; o[a][b][1] *= f; o[a][b][2] *= f; o[a][b][3] *= f; }
                }
                float* P = Ps + warp * TS_KT * 4;
                *reinterpret_cast<float4*>(P + lane * 4) = make_float4(w[0], w[1], w[2], w[3]);
                __syncwarp();
                auto product = [&](auto guarded) {
#pragma unroll 4
                    for (int key = 0; key < TS_KT; ++key) {
                        const float4 w4 = *reinterpret_cast<const float4*>(P + key * 4);
                        const float ww[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                        for (int b = 0; b < CB; ++b) {
                            const float4 v4 = *reinterpret_cast<const float4*>(Vs + key * pitch + b * 128 + lane * 4);
#pragma unroll
                            for (int a = 0; a < 4; ++a) {
                                if (decltype(guarded)::value && ww[a] < 0.f) continue;
                                o[a][b][0] = fmaf(ww[a], v4.x, o[a][b][0]); o[a][b][1] = fmaf(ww[a], v4.y, o[a][b][1]);
                                o[a][b][2] = fmaf(ww[a], v4.z, o[a][b][2]); o[a][b][3] = fmaf(ww[a], v4.w, o[a][b][3]);
                            }
                        }
                    }
                };
                if (ends) product(TreeYes());
                else product(TreeNo());
                __syncwarp();
            }
            const bool whole = g.t_lo == 0 && g.t_hi == g.tiles;
            const int slot = 2 * j + (g.t_lo == 0 ? 1 : 0);
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const int row = 4 * warp + a;
                if (row >= g.rows) continue;
                const float l = warp_sum(l_run[a]);
                if (whole) {
                    const int rr = g.row0 + row;
                    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
                    T* dst = reinterpret_cast<T*>(p.out) + ((size_t)(g.tok0 + rr / G) * p.n_q + (size_t)g.kvh * G + rr % G) * d;
#pragma unroll
                    for (int b = 0; b < CB; ++b)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (b * 128 + lane * 4 + e < d) dst[b * 128 + lane * 4 + e] = from_f32<T>(o[a][b][e] * inv);
                } else {
                    float4* dst = reinterpret_cast<float4*>(p.part_o) + (size_t)slot * d4 * TS_ROWS + row;
#pragma unroll
                    for (int b = 0; b < CB; ++b)
                        if (b * 32 + lane < d4) dst[(b * 32 + lane) * TS_ROWS] = make_float4(o[a][b][0], o[a][b][1], o[a][b][2], o[a][b][3]);
                    if (lane == 0) *reinterpret_cast<float2*>(p.part_ml + ((size_t)slot * TS_ROWS + row) * 2) = make_float2(m_run[a], l);
                }
            }
            if (!whole && g.t_lo == 0) record = TreeRecord{walk.pieces(g, j), g.rows, g.tok0, g.row0, g.kvh, {0, 0, 0}};
        }
    }
    if (tid == 0) p.record[j] = record;
}

// ---------------------------------------------------------------------------------------
// The pieces of cut items, joined in the order of the keys.  A warp takes 32 rows, a lane each, and TJ_C fours of columns of the item whose first piece
// block j has.  Bound by latency: a record, the pieces' maxima, then their rows, TJ_K pieces and so 24 loads of 512 bytes of a warp at a time.
// ---------------------------------------------------------------------------------------
constexpr int TJ_WARPS = 4;


template <typename T, int ROWS, int TJ_C, int TJ_K>
__global__ void __launch_bounds__(TJ_WARPS * 32) tree_join_kernel(const TreeParams p) {
    static_assert(TJ_C % 2 == 0, "16 bytes of bfloat16 are two fours of columns");
    const int lane = threadIdx.x & 31, j = blockIdx.x, d4 = (p.d + 3) >> 2, n_cols = (d4 + TJ_C - 1) / TJ_C, task = blockIdx.y * TJ_WARPS + (threadIdx.x >> 5);
    const int row = task / n_cols * 32 + lane, c0 = task % n_cols * TJ_C;       // of the item; in fours of columns
    pdl_wait();
    pdl_small();
    const int4 rec = *reinterpret_cast<const int4*>(p.record + j);           // pieces, rows, first draft, first row
    const int pieces = rec.x, kvh = p.record[j].kvh;
    if (pieces == 0 || row >= rec.y) return;
    const int G = p.G, d = p.d, rr = rec.w + row, tok0 = rec.z;
    auto slot = [&](int k) { return (size_t)(2 * (j + k) + (k == 0 ? 1 : 0)); };
    auto ml_of = [&](int k) { return *reinterpret_cast<const float2*>(p.part_ml + (slot(k) * ROWS + row) * 2); };
    float M = -INFINITY, L = 0.f;
    float4 acc[TJ_C];
#pragma unroll
    for (int c = 0; c < TJ_C; ++c) acc[c] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = 0; k0 < pieces; k0 += TJ_K) {      // TJ_K pieces at a time: their maxima and rows are all asked for at once
        float2 ml[TJ_K];
        float4 v[TJ_K][TJ_C];
#pragma unroll
        for (int k = 0; k < TJ_K; ++k) {
            const bool there = k0 + k < pieces;
            ml[k] = there ? ml_of(k0 + k) : make_float2(-INFINITY, 0.f);
            const float4* src = reinterpret_cast<const float4*>(p.part_o) + slot(k0 + k) * d4 * ROWS + row;
#pragma unroll
            for (int c = 0; c < TJ_C; ++c) v[k][c] = there && c0 + c < d4 ? src[(c0 + c) * ROWS] : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float mx = M;
#pragma unroll
        for (int k = 0; k < TJ_K; ++k) mx = fmaxf(mx, ml[k].x);
        const float mu = mx == -INFINITY ? 0.f : mx, f = fast_exp2(M - mu);
        M = mx;
        L *= f;
#pragma unroll
        for (int c = 0; c < TJ_C; ++c) { acc[c].x *= f; acc[c].y *= f; acc[c].z *= f; acc[c].w *= f; }
#pragma unroll
        for (int k = 0; k < TJ_K; ++k) {
            const float w = fast_exp2(ml[k].x - mu);
            L = fmaf(w, ml[k].y, L);
#pragma unroll
            for (int c = 0; c < TJ_C; ++c) {
                acc[c].x = fmaf(w, v[k][c].x, acc[c].x); acc[c].y = fmaf(w, v[k][c].y, acc[c].y);
                acc[c].z = fmaf(w, v[k][c].z, acc[c].z); acc[c].w = fmaf(w, v[k][c].w, acc[c].w);
            }
        }
    }
    const float inv = L > 0.f ? 1.f / L : (L == L ? 0.f : L);
    T* dst = reinterpret_cast<T*>(p.out) + ((size_t)(tok0 + rr / G) * p.n_q + (size_t)kvh * G + rr % G) * d + c0 * 4;
    if (sizeof(T) == 2 && (d & 7) == 0 && ((uintptr_t)p.out & 15) == 0) {
#pragma unroll
        for (int c = 0; c < TJ_C; c += 2)
            if (c0 + c < d4)
                *reinterpret_cast<uint4*>(dst + c * 4) = make_uint4(pack_bf16(acc[c].x * inv, acc[c].y * inv), pack_bf16(acc[c].z * inv, acc[c].w * inv),
                                                                    pack_bf16(acc[c + 1].x * inv, acc[c + 1].y * inv), pack_bf16(acc[c + 1].z * inv, acc[c + 1].w * inv));
        return;
    }
#pragma unroll
    for (int c = 0; c < TJ_C; ++c) {
        const float x[4] = {acc[c].x, acc[c].y, acc[c].z, acc[c].w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if ((c0 + c) * 4 + e < d) dst[c * 4 + e] = from_f32<T>(x[e] * inv);
    }
}
// Eight columns a warp and twelve pieces at a time where there are some pieces an item, or few warps anyhow (whole calls in bfloat16, 32 query heads on 8: 8 drafts
// behind 4,096 keys 16.1 us against 19.9 with sixteen columns and six pieces, 64 drafts 26.5 against 28.0); with two or three pieces of many rows that
// is more blocks than it helps (8 requests of 32 drafts behind 1,000 keys 28.2 against 26.2).
template <typename T, int ROWS, int KT>
static void tree_join(const TreeParams& p, int blocks, int max_rows, cudaStream_t stream) {
    if ((long long)p.table_width * p.page_size <= KT) return;        // one tile at most: nothing is cut
    const long long items = (long long)p.B * p.n_kv * ((max_rows + ROWS - 1) / ROWS);
    const bool narrow = max_rows <= 32 || 4 * items <= blocks;
    const int columns = narrow ? 8 : 16, tasks = ((max_rows < ROWS ? max_rows : ROWS) + 31) / 32 * ((p.d + columns - 1) / columns);
    const dim3 grid(blocks, (tasks + TJ_WARPS - 1) / TJ_WARPS);
    if (narrow) msgl_launch_pdl(tree_join_kernel<T, ROWS, 2, 12>, grid, dim3(TJ_WARPS * 32), 0, stream, p);
    else msgl_launch_pdl(tree_join_kernel<T, ROWS, 4, 6>, grid, dim3(TJ_WARPS * 32), 0, stream, p);
}

#include "attention_tree_tc.cuh"

static int tree_blocks_per_sm(int d) { return d <= 256 ? 2 : 1; }         // of the kernels without tensor cores
static size_t tree_simt_smem(int cb) { return ((size_t)(TS_ROWS + 2 * TS_KT) * (cb * 128 + 4) + 8 * TS_KT * 4) * sizeof(float); }

// Whether the tensor cores take a launch: bfloat16, head sizes 64 and 128, pages that TMA can fetch, a cache whose rows a coordinate can name.
MSGL_API int msgl_tree_attention_tensor(int d, int page_size, long long cache_rows, int dtype) {
    return dtype == MSGL_BF16 && (d == 64 || d == 128) && page_size >= 8 && (page_size & (page_size - 1)) == 0 && cache_rows < 0x7fffffffLL - 4096 && tc_encoder() != nullptr;
}
// The kernels: 32 rows a block, 64 rows a block, tensor cores.
enum { TREE_SIMT = 0, TREE_TILE = 1, TREE_TC = 2 };
// Blocks of a launch and rows of an item, for the sizes of the scratch memory: part_o [2 * blocks][ceil(d / 4)][rows][4], part_ml [2 * blocks][rows][2] float32, record [blocks][8] int32.
MSGL_API int msgl_tree_attention_blocks(int d, int kind) { return msgl_sm_count() * (kind == TREE_TC ? 1 : tree_blocks_per_sm(d)); }
MSGL_API int msgl_tree_attention_rows(int kind) { return kind == TREE_TC ? TT_ROWS : kind == TREE_TILE ? TF_ROWS : TS_ROWS; }

template <typename T, int CB>
static int tree_simt_launch(const TreeParams& p, int blocks, int max_rows, cudaStream_t stream) {
    static MsglOncePerDevice attr_set;
    if (attr_set.due()) {
        if (cudaFuncSetAttribute(tree_simt_kernel<T, CB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)tree_simt_smem(CB)) != cudaSuccess) return msgl_check_launch();
        attr_set.mark();
    }
    msgl_launch_pdl(tree_simt_kernel<T, CB>, dim3(blocks), dim3(TS_THREADS), tree_simt_smem(CB), stream, p);
    tree_join<T, TS_ROWS, TS_KT>(p, blocks, max_rows, stream);
    return msgl_check_launch();
}

template <typename T>
static int tree_tile_launch(const TreeParams& p, int blocks, int max_rows, cudaStream_t stream) {
    static MsglOncePerDevice attr_set;
    if (attr_set.due()) {
        if (cudaFuncSetAttribute(tree_tile_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)TF_SMEM) != cudaSuccess) return msgl_check_launch();
        attr_set.mark();
    }
    msgl_launch_pdl(tree_tile_kernel<T>, dim3(blocks), dim3(TF_THREADS), TF_SMEM, stream, p);
    tree_join<T, TF_ROWS, TF_KT>(p, blocks, max_rows, stream);
    return msgl_check_launch();
}

template <int D>
static int tree_tc_launch(const TreeParams& p, int* status, int blocks, int max_rows, cudaStream_t stream) {
    static MsglOncePerDevice attr_set;
    if (attr_set.due()) {
        if (cudaFuncSetAttribute(tree_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)TreeTc<D>::ALLOC) != cudaSuccess) return msgl_check_launch();
        attr_set.mark();
    }
    const int box = p.page_size < 128 ? p.page_size : 128;
    const long long rows = p.pages * p.n_kv * p.page_size;
    CUtensorMap kmap, vmap;
    if (!tc_matrix_map(p.k_cache, rows, D, (long long)D * 2, box, &kmap) || !tc_matrix_map(p.v_cache, rows, D, (long long)D * 2, box, &vmap)) return MSGL_ERR_SIZE;
    msgl_launch_pdl(tree_tc_kernel<D>, dim3(blocks), dim3(TT_THREADS), TreeTc<D>::ALLOC, stream, p, status, kmap, vmap, box);
    tree_join<__nv_bfloat16, TT_ROWS, TT_KT>(p, blocks, max_rows, stream);
    return msgl_check_launch();
}

// kind: the kernel (of the tensor cores, status points at the status word); max_draft: the most drafts that a request has.
MSGL_API int msgl_tree_attention(const void* q, void* out, const void* k_cache, const void* v_cache, const int* q_start, const int* kv_len, const int* table,
                                 const void* mask, int B, int T, int n_q, int n_kv, int d, int page_size, int table_stride, int table_width, int words,
                                 long long pages, float scale, float* part_o, float* part_ml, int* record, int blocks, int max_draft, int kind, int* status,
                                 int dtype, cudaStream_t stream) {
    if (B <= 0 || T <= 0) return MSGL_OK;
    if (n_kv <= 0 || n_q <= 0 || n_q % n_kv || d < 1 || d > 512 || page_size < 1 || table_width < 1 || words < 1 || blocks < 1 || pages < 0 || max_draft < 1) return MSGL_ERR_SIZE;
    const int max_rows = max_draft < T ? max_draft * (n_q / n_kv) : T * (n_q / n_kv);            // most rows of a request under a kv head
    if ((long long)table_width * page_size > 0x7fffffffLL - 1024 || (long long)T * (n_q / n_kv) > 0x7fffffffLL / 2) return MSGL_ERR_SIZE;
    // the length of the work, in whole numbers of 32 bits: at most this many tiles and heads of items
    if ((long long)B * n_kv * ((long long)max_rows / TS_ROWS + 1) * ((long long)table_width * page_size / TS_KT + 1 + TREE_HEAD) > 0x7fffffffLL) return MSGL_ERR_SIZE;
    if (((uintptr_t)part_o | (uintptr_t)record) & 15 || (uintptr_t)part_ml & 7) return MSGL_ERR_ALIGN;
    TreeParams p;
    p.q = q; p.out = out; p.k_cache = k_cache; p.v_cache = v_cache; p.q_start = q_start; p.kv_len = kv_len; p.table = table; p.mask = (const unsigned*)mask;
    p.part_o = part_o; p.part_ml = part_ml; p.record = (TreeRecord*)record;
    p.B = B; p.T = T; p.n_q = n_q; p.n_kv = n_kv; p.G = n_q / n_kv; p.d = d; p.page_size = page_size; p.table_stride = table_stride; p.table_width = table_width; p.words = words;
    p.pages = pages; p.max_draft = max_draft;
    p.page_shift = -1;
    if ((page_size & (page_size - 1)) == 0) { int sh = 0; while ((1 << sh) < page_size) ++sh; p.page_shift = sh; }
    p.scale_log2 = scale * 1.4426950408889634f;
    p.vectors = (((uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)(d * (dtype == MSGL_F32 ? 4 : 2))) & 15) == 0;
    if (kind == TREE_TC) {
        if (status == nullptr || pages < 1 || !msgl_tree_attention_tensor(d, page_size, pages * n_kv * page_size, dtype)) return MSGL_ERR_SIZE;
        if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) return MSGL_ERR_ALIGN;
        return d == 128 ? tree_tc_launch<128>(p, status, blocks, max_rows, stream) : tree_tc_launch<64>(p, status, blocks, max_rows, stream);
    }
    if (kind == TREE_TILE && d > TF_D) return MSGL_ERR_SIZE;
#define MSGL_TREE(T) (kind == TREE_TILE ? tree_tile_launch<T>(p, blocks, max_rows, stream) : d <= 128 ? tree_simt_launch<T, 1>(p, blocks, max_rows, stream) : d <= 256 ? tree_simt_launch<T, 2>(p, blocks, max_rows, stream) : tree_simt_launch<T, 4>(p, blocks, max_rows, stream))
    if (dtype == MSGL_F32) return MSGL_TREE(float);
    if (dtype == MSGL_BF16) return MSGL_TREE(__nv_bfloat16);
#undef MSGL_TREE
    return MSGL_ERR_DTYPE;
}
