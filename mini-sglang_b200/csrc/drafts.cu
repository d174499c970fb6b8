// The bookkeeping of a step that verifies drafted tokens: the fields of the step, and the path that the model agrees with.
//
// A request brings n drafts behind its `cached` tokens.  Draft 0 is the newest accepted token; the parent of draft i > 0 is an earlier
// draft (an index within the request; anything else counts as none, so a bad parent can neither loop nor read out of range).  Draft i
// is written to the cache at place cached + i, whatever its depth; its position is cached + (number of its ancestors).
#include "common.cuh"

constexpr int DR_MAX = 256, DR_WORDS = DR_MAX / 32;

// ---------------------------------------------------------------------------------------
// The fields of the step, a block a request.  Ancestors by pointer doubling: every draft holds a set of bits (itself) and a pointer (its
// parent); in a round it takes over the set its pointer points at and that draft's pointer, so a chain of 256 is done in eight rounds.
// Bound by latency: lengths, parents, table entries and the rounds follow on one another.  8 drafts of one request take 2.9 us, 64 of each of
// 256 requests 4.1 (launch included).
// ---------------------------------------------------------------------------------------
__global__ void __launch_bounds__(DR_MAX) draft_plan_kernel(const int* __restrict__ parents, int T, const int* __restrict__ lens, const int* __restrict__ cached,
                                                            int B, const int* __restrict__ table, int table_stride, int table_width, int page_size,
                                                            int max_draft, int words, int* __restrict__ q_start, int* __restrict__ kv_len,
                                                            int* __restrict__ positions, int* __restrict__ token_req, int* __restrict__ out_loc,
                                                            unsigned* __restrict__ mask) {
    __shared__ unsigned bits[2][DR_MAX * DR_WORDS];
    __shared__ int up[2][DR_MAX];
    __shared__ int warp_sum[DR_MAX / 32];
    const int r = blockIdx.x, tid = threadIdx.x, n_threads = blockDim.x;
    pdl_launch_dependents();
    pdl_wait();
    pdl_after_wait();
    auto length = [&](int i) { return min(max(lens[i], 0), max_draft); };
    int before = 0;
    for (int i = tid; i < r; i += n_threads) before += length(i);
    before = __reduce_add_sync(0xffffffffu, before);
    if ((tid & 31) == 0) warp_sum[tid >> 5] = before;
    __syncthreads();
    before = 0;
    for (int w = 0; w < n_threads / 32; ++w) before += warp_sum[w];
    const int start = min(before, T), n = min(length(r), T - start), base = min(max(cached[r], 0), 0x7fffffff - DR_MAX);
    if (tid == 0) {
        q_start[r] = start;
        kv_len[r] = base + n;
        if (r == B - 1) q_start[B] = start + n;
    }
    if (tid < n) {
        const int p = parents[start + tid];
        up[0][tid] = p >= 0 && p < tid ? p : -1;
        for (int w = 0; w < words; ++w) bits[0][tid * words + w] = w == (tid >> 5) ? 1u << (tid & 31) : 0u;
    }
    int at = 0;
    __syncthreads();
    for (;;) {                                       // at most log2(256) rounds: a pointer's distance doubles
        const int p = tid < n ? up[at][tid] : -1;
        if (!__syncthreads_or(p >= 0)) break;
        if (tid < n) {
            for (int w = 0; w < words; ++w) bits[at ^ 1][tid * words + w] = bits[at][tid * words + w] | (p >= 0 ? bits[at][p * words + w] : 0u);
            up[at ^ 1][tid] = p >= 0 ? up[at][p] : -1;
        }
        at ^= 1;
        __syncthreads();
    }
    if (tid < n) {
        const int t = start + tid, place = base + tid, page = place / page_size;
        int depth = -1;
        for (int w = 0; w < words; ++w) {
            const unsigned b = bits[at][tid * words + w];
            mask[(size_t)t * words + w] = b;
            depth += __popc(b);
        }
        positions[t] = base + depth;
        token_req[t] = r;
        const int id = page < table_width ? table[(size_t)r * table_stride + page] : -1;
        const long long slot = (long long)id * page_size + (place - page * page_size);
        out_loc[t] = id >= 0 && slot <= 0x7fffffffLL ? (int)slot : 0;          // (a negative slot would be written to in front of the caches)
    }
    if (r == B - 1) {                                // rows behind the last draft: position 0 on the page for padding, nothing seen
        for (int t = start + n + tid; t < T; t += n_threads) {
            positions[t] = 0;
            token_req[t] = 0;
            out_loc[t] = 0;
            for (int w = 0; w < words; ++w) mask[(size_t)t * words + w] = 0u;
        }
    }
}

// parents [T], lens and cached [B], table [B, table_width] (rows table_stride apart) -> q_start [B + 1], kv_len [B], positions, token_req
// and out_loc [T], mask [T, words] (bit i of a row: its request's draft i is the row's draft or one of its ancestors).
MSGL_API int msgl_draft_plan(const int* parents, int T, const int* lens, const int* cached, int B, const int* table, int table_stride, int table_width,
                             int page_size, int max_draft, int words, int* q_start, int* kv_len, int* positions, int* token_req, int* out_loc,
                             void* mask, cudaStream_t stream) {
    if (B <= 0) return MSGL_OK;
    if (T < 0 || page_size < 1 || table_width < 1 || max_draft < 1 || max_draft > DR_MAX || words != (max_draft + 31) / 32) return MSGL_ERR_SIZE;
    msgl_launch_pdl(draft_plan_kernel, dim3(B), dim3(words * 32), 0, stream, parents, T, lens, cached, B, table, table_stride, table_width, page_size,
                    max_draft, words, q_start, kv_len, positions, token_req, out_loc, (unsigned*)mask);
    return msgl_check_launch();
}

// ---------------------------------------------------------------------------------------
// The accepted path: from draft 0 on to the child whose token is the one that the model put after its parent (the first such child), as
// far as there is one.  Every block walks its request's tree by itself; the blocks along y then move the path's rows of their caches to
// the places behind the cached tokens.
//
// Row path[i] goes to place i <= path[i], in ascending order of i: a thread owns a 16-byte column of all rows, loads DR_BATCH of them
// and stores them, so no row is overwritten before it was read (a later row's source lies behind all earlier targets).
// Bound by latency for small batches (8 drafts, the 56 caches of 28 layers: 2.7 us), else by the rows' bytes (64 requests of 61 drafts, 8 caches of
// 8 heads, 6.4 MB: 4.2 us, 1.5 TB/s).
// ---------------------------------------------------------------------------------------
constexpr int DR_CACHES = 128, DR_BATCH = 8, DR_COPY_THREADS = 256;
struct DraftCaches { void* p[DR_CACHES]; };

template <typename U>
__global__ void __launch_bounds__(DR_COPY_THREADS) draft_accept_kernel(const int* __restrict__ tokens, const int* __restrict__ parents,
                                                                       const int* __restrict__ following, const int* __restrict__ q_start, int T, int max_draft,
                                                                       int* __restrict__ kept_out, int* __restrict__ path_out, int* __restrict__ token_out,
                                                                       const int* __restrict__ kv_len, const int* __restrict__ table, int table_stride,
                                                                       int table_width, int page_size, long long pages, int n_kv, int row_units, int n_caches,
                                                                       const __grid_constant__ DraftCaches caches) {
    __shared__ int child[DR_MAX], path[DR_MAX], next[DR_MAX];
    __shared__ int2 from[DR_MAX], to[DR_MAX];        // page, row within it
    __shared__ int sh_kept, sh_first;
    const int r = blockIdx.x, tid = threadIdx.x;
    pdl_launch_dependents();
    pdl_wait();
    pdl_after_wait();
    const int start = min(max(q_start[r], 0), T), brought = min(max(q_start[r + 1] - start, 0), T - start), n = min(brought, max_draft);
    int tok = 0, up = -1;
    child[tid] = DR_MAX;
    if (tid < n) {
        next[tid] = following[start + tid];
        tok = tokens[start + tid];
        up = parents[start + tid];
    }
    __syncthreads();
    if (tid < n && up >= 0 && up < tid && tok == next[up]) atomicMin(&child[up], tid);       // the lowest index, in whatever order they come
    __syncthreads();
    if (tid == 0) {
        int kept = 0, first = DR_MAX;                // first: the first of the path that has to move
        for (int at = 0; at < n; at = child[at]) {
            if (at != kept && first == DR_MAX) first = kept;
            path[kept++] = at;
        }
        sh_kept = kept;
        sh_first = first;
    }
    __syncthreads();
    const int kept = sh_kept, first = sh_first;
    if (kept_out != nullptr && blockIdx.y == 0) {
        if (tid == 0) kept_out[r] = kept;
        if (tid < max_draft) {
            path_out[(size_t)r * max_draft + tid] = tid < kept ? path[tid] : -1;
            token_out[(size_t)r * max_draft + tid] = tid < kept ? next[path[tid]] : -1;
        }
    }
    if (n_caches == 0 || first >= kept) return;
    const int base = kv_len[r] - brought;
    auto place = [&](int i) {
        const int at = base + i, page = at / page_size;
        if (at < 0 || page >= table_width) return make_int2(-1, 0);
        const int id = table[(size_t)r * table_stride + page];
        return make_int2(id >= 0 && id < pages ? id : -1, at - page * page_size);
    };
    if (tid >= first && tid < kept) { from[tid] = place(path[tid]); to[tid] = place(tid); }
    __syncthreads();
    // a (cache, head, unit of a row) a thread, all rows of the path in order
    const int columns = n_kv * row_units, all = n_caches * columns;
    for (int c = blockIdx.y * DR_COPY_THREADS + tid; c < all; c += gridDim.y * DR_COPY_THREADS) {
        const int which = c / columns, in = c - which * columns, h = in / row_units, u = in - h * row_units;
        U* cache = reinterpret_cast<U*>(caches.p[which]);
        auto unit = [&](int2 w) { return cache + (((size_t)w.x * n_kv + h) * page_size + w.y) * row_units + u; };
        for (int i0 = first; i0 < kept; i0 += DR_BATCH) {
            U v[DR_BATCH];
#pragma unroll
            for (int k = 0; k < DR_BATCH; ++k)
                if (i0 + k < kept && from[i0 + k].x >= 0) v[k] = *unit(from[i0 + k]);
#pragma unroll
            for (int k = 0; k < DR_BATCH; ++k)
                if (i0 + k < kept && from[i0 + k].x >= 0 && to[i0 + k].x >= 0) *unit(to[i0 + k]) = v[k];
        }
    }
}

// tokens, parents, following [T]; q_start [B + 1] -> kept [B], path and token [B, max_draft] (-1 behind the path; none is written where
// kept is null).  caches: n_caches arrays [pages, n_kv, page_size, row_bytes], with kv_len [B] and table [B, table_width].
// blocks_y: blocks of a request.
MSGL_API int msgl_draft_accept(const int* tokens, const int* parents, const int* following, const int* q_start, int B, int T, int max_draft, int* kept, int* path,
                               int* token, const int* kv_len, const int* table, int table_stride, int table_width, int page_size, long long pages, int n_kv,
                               int row_bytes, void* const* caches, int n_caches, int blocks_y, cudaStream_t stream) {
    if (B <= 0) return MSGL_OK;
    if (T < 0 || max_draft < 1 || max_draft > DR_MAX || n_caches < 0 || n_caches > DR_CACHES || blocks_y < 1 || blocks_y > 65535) return MSGL_ERR_SIZE;
    if (n_caches > 0 && (kv_len == nullptr || table == nullptr || page_size < 1 || table_width < 1 || n_kv < 1 || row_bytes < 2 || row_bytes % 2)) return MSGL_ERR_SIZE;
    DraftCaches c = {};
    uintptr_t bits = (uintptr_t)row_bytes;
    for (int i = 0; i < n_caches; ++i) { c.p[i] = caches[i]; bits |= (uintptr_t)caches[i]; }
    const int unit = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 2;
    if (bits % 2) return MSGL_ERR_ALIGN;
    const int units = row_bytes / unit;
    if ((long long)n_caches * n_kv * units + (long long)blocks_y * DR_COPY_THREADS > 0x7fffffffLL) return MSGL_ERR_SIZE;      // (a thread's counter steps once past the last column)
#define MSGL_ACCEPT(U)                                                                                                                                          \
    msgl_launch_pdl(draft_accept_kernel<U>, dim3(B, blocks_y), dim3(DR_COPY_THREADS), 0, stream, tokens, parents, following, q_start, T, max_draft, kept, path,   \
                    token, kv_len, table, table_stride, table_width, page_size, pages, n_kv, units, n_caches, c)
    if (unit == 16) MSGL_ACCEPT(uint4);
    else if (unit == 4) MSGL_ACCEPT(unsigned);
    else MSGL_ACCEPT(unsigned short);
#undef MSGL_ACCEPT
    return msgl_check_launch();
}
