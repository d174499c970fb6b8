// Attention over a cache in 4 bits on the tensor cores: bfloat16, head sizes 64 and 128, requests that bring few tokens.
//
// A segment is up to 8 rows (token, query head) of one request under one kv head, and its keys in units of 32.  The units of all segments are dealt out
// over one block an SM: every block works out from the requests' lengths alone which are its own.
//   * few keys: a segment of u units has max(1, u / PIECE) equal pieces, a block a piece (or a block a whole segment, where that is nearly even);
//   * many short segments: a warp takes whole segments;
//   * otherwise the units of all segments, each with HEAD units ahead for what a segment costs beside its keys, are laid end to end and cut into runs of
//     equal length; a cut within SNAP units of a segment's edge moves onto the edge.
// Pieces of a segment lie in consecutive blocks.  A segment within one block is written out by it; of the others every block leaves its partial result
// in scratch memory, and the one that raises the segment's counter to its number of pieces merges them in the order of the keys and clears the counter.
//
// Mathematics.  A code c enters the products as u = 1 + c / 16, which is exact in bfloat16 with the code in the top four bits of the fraction: a shift and
// a masked "or" make two elements of a word at once.  With a key's step and base,
//     q k = 16 step (sum q u - sum q) + base sum q                 (the accumulator starts at -sum q, and the rest is one multiplication and one addition a score)
//     o   = sum_j p_j (base_j + step_j c_j) = sum_j w_j u_j + sum_j (p_j base_j - w_j),   w_j = bf16(16 p_j step_j)
// where the rounded w_j stands in both sums, so that the offset of u cancels whatever w_j was rounded to; its rounding counts by the code alone.
// Scores, p, sums and outputs are float32.  S^T = K Q^T with keys on the M dimension, the head's elements permuted so that a lane reads 16 bytes
// of a row; P goes through movmatrix; V^T fragments come by ldmatrix.trans on 16-bit columns, four codes of two neighbouring keys a register.  The
// exponentials' reference moves only where a score lies KR_LAZY above it.
#pragma once

constexpr float KR_LAZY = 8.f;
constexpr int KR_KEYS = 32;          // keys of a unit
constexpr int KR_MAX_B = 256;        // requests of a launch, a thread each
constexpr int KR_PIECE = 8;          // units of a piece at least, where segments are cut by themselves
constexpr int KR_SNAP = 3;           // a cut this close to a segment's edge moves onto it
constexpr int KR_HEAD = 3;           // what a segment costs beside its units, in units
constexpr int KR_WARP_UNITS = 8;     // longest segment where a warp takes whole segments

struct Kv4Runs {
    const __nv_bfloat16* q; __nv_bfloat16* out;
    const unsigned char* k; const unsigned char* v; const uint2* steps;
    const int* q_start; const int* kv_len; const int* block_table;
    float* part_o;                   // [2 * blocks][8][D]
    float* part_ml;                  // [2 * blocks][8][2]
    int* count;                      // a word a segment, zero before and after
    long long bt_stride;
    int B, T, n_q, n_kv, page_size, page_shift, pages, bt_width, window, max_q;
    float scale;
};

__device__ __forceinline__ unsigned kr_smem(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void kr_cp16(unsigned s, const void* g, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(s), "l"(g), "r"(there ? 16 : 0));
}
__device__ __forceinline__ void kr_cp8(unsigned s, const void* g, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;\n" ::"r"(s), "l"(g), "r"(there ? 8 : 0));
}
__device__ __forceinline__ void kr_commit() { asm volatile("cp.async.commit_group;\n"); }
template <int N> __device__ __forceinline__ void kr_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N)); }
__device__ __forceinline__ float kr_exp2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ unsigned kr_pack(float lo, float hi) {
    unsigned r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ unsigned kr_trans(unsigned v) {
    unsigned r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void kr_mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// codes I of both halves of a word as 1 + c / 16 in bfloat16
template <int I> __device__ __forceinline__ unsigned kr_unit(unsigned w) {
    const unsigned s = I == 0 ? w << 3 : w >> (4 * I - 3);
    return (s & 0x00780078u) | 0x3f803f80u;
}

template <int D, int NW, int ST>
constexpr size_t kr_smem_bytes() {
    return (size_t)NW * ST * (KR_KEYS * (D + 8)) + (size_t)NW * 8 * (D + 4) * 4 + (size_t)NW * 8 * 2 * 4 + (8 * KR_MAX_B + 4) * 4;
}

struct KrCursor {
    int r, s, kvh, tile, c0, u;      // request, its segment, kv head and tile of rows; first unit of the segment among all, units
};

template <int D, int NW, int ST>
__global__ void __launch_bounds__(NW * 32, 1) kv4_attn_runs_kernel(const Kv4Runs p) {
    extern __shared__ __align__(128) unsigned char kr_sh[];
    constexpr int ROW = D / 2, KV_BYTES = KR_KEYS * ROW, STAGE = 2 * KV_BYTES + KR_KEYS * 8, OLD = D + 4, THREADS = NW * 32;
    constexpr int CH = ROW / 16;                          // 16-byte chunks of a row
    constexpr int SW = CH == 4 ? 1 : 2;                   // chunk c of row r lies at c ^ (r >> SW & CH - 1): eight rows' chunks c are eight different 16-byte columns
    constexpr int QW = D / 32;                            // words of codes of a key row a lane
    static_assert(D == 64 || D == 128, "lanes read 8 or 16 bytes of a key row");
    float* Om = reinterpret_cast<float*>(kr_sh + (size_t)NW * ST * STAGE);      // [NW][8][OLD]
    float* Mm = Om + NW * 8 * OLD;                        // [NW][8]
    float* Lm = Mm + NW * 8;                              // [NW][8]
    int* pre_u = reinterpret_cast<int*>(Lm + NW * 8);     // [B + 1] units of all segments of the requests before
    int* pre_s = pre_u + KR_MAX_B + 1;                    // [B + 1] segments of the requests before
    int* units = pre_s + KR_MAX_B + 1;                    // per request: units of a segment, first unit, keys, first token, tokens, last position + 1
    int* first = units + KR_MAX_B;
    int* keys = first + KR_MAX_B;
    int* token = keys + KR_MAX_B;
    int* tokens = token + KR_MAX_B;
    int* ends = tokens + KR_MAX_B;
    __shared__ int4 sh_sum[NW];
    __shared__ int2 sh_run;
    __shared__ int4 sh_seg;                               // request, its segment, (by_piece) pieces of the segment, this block's
    __shared__ int sh_last;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int G = p.n_q / p.n_kv, NB = (int)gridDim.x, j = (int)blockIdx.x;
    pdl_wait();

    // ---- the requests, their units, segments and pieces, and the sums over those before; a request a thread
    int my_u = 0, my_segs = 0, my_pc = 0;
    if (tid < p.B) {
        const int t0 = p.q_start != nullptr ? p.q_start[tid] : tid, n = p.q_start != nullptr ? p.q_start[tid + 1] - t0 : 1, len = p.kv_len[tid];
        const int kv = max(min(len, p.bt_width * p.page_size), 0), f = (p.window > 0 ? max(len - n - p.window + 1, 0) : 0) / KR_KEYS;
        if (n >= 1 && n <= p.max_q && t0 >= 0 && t0 + n <= p.T) {
            my_u = max((kv + KR_KEYS - 1) / KR_KEYS - f, 1);
            my_segs = p.n_kv * ((n * G + 7) >> 3);
            my_pc = max(1, my_u / KR_PIECE);
        }
        units[tid] = my_u; first[tid] = f; keys[tid] = kv; token[tid] = t0; tokens[tid] = n; ends[tid] = len;
    }
    int at_u = my_u * my_segs, at_s = my_segs, at_p = my_pc * my_segs;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, at_u, o), b = __shfl_up_sync(0xffffffffu, at_s, o), c = __shfl_up_sync(0xffffffffu, at_p, o);
        if (lane >= o) { at_u += a; at_s += b; at_p += c; }
    }
    const int most = __reduce_max_sync(0xffffffffu, my_u);
    if (lane == 31) sh_sum[warp] = make_int4(at_u, at_s, at_p, most);
    __syncthreads();
    int U = 0, S = 0, pieces_all = 0, longest = 0;
    at_u -= my_u * my_segs; at_s -= my_segs; at_p -= my_pc * my_segs;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        const int4 x = sh_sum[w];
        if (w < warp) { at_u += x.x; at_s += x.y; at_p += x.z; }
        U += x.x; S += x.y; pieces_all += x.z;
        longest = max(longest, x.w);
    }
    if (tid < p.B) { pre_u[tid] = at_u; pre_s[tid] = at_s; }
    if (tid == 0) { pre_u[p.B] = U; pre_s[p.B] = S; sh_run = make_int2(0, 0); }
    if (S == 0) return;
    if (pieces_all > NB && S <= NB && 3ll * longest * NB <= 4ll * U) {        // a block a segment is nearly even, and nothing is left to merge
        pieces_all = S;
        at_p = at_s;
        my_pc = my_segs > 0 ? 1 : 0;
    }
    const bool by_piece = pieces_all <= NB;
    const bool by_warp = !by_piece && longest <= KR_WARP_UNITS && (8ll * longest + 6) * NB < 11ll * S;

    // ---- this block's run of units [lo, hi) of the segments laid end to end, and the segment it starts in
    const long long V = U + (long long)KR_HEAD * S;
    __syncthreads();
    if (by_piece) {
        const int in_r = j - at_p;
        if (in_r >= 0 && in_r < my_pc * my_segs) {
            const int s = in_r / my_pc, piece = in_r - s * my_pc, c0 = at_u + s * my_u;
            sh_seg = make_int4(tid, s, my_pc, piece);
            sh_run = make_int2(c0 + (int)((long long)my_u * piece / my_pc), c0 + (int)((long long)my_u * (piece + 1) / my_pc));
        }
    } else if (!by_warp) {
        // the thread whose request holds the raw cut floor(V i / NB) finds the cut: a segment's edge or a unit within it
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int i = j + e;
            if (i == NB && tid == 0) sh_run.y = U;
            const long long in_r = V * i / NB - (at_u + (long long)KR_HEAD * at_s);
            if (in_r >= 0 && in_r < (long long)(my_u + KR_HEAD) * my_segs) {
                const int s = (int)in_r / (my_u + KR_HEAD), off = (int)in_r - s * (my_u + KR_HEAD) - KR_HEAD;
                const int unit = off <= KR_SNAP ? 0 : my_u - off <= KR_SNAP ? my_u : off, x = at_u + s * my_u + unit;
                if (e == 1) { sh_run.y = x; continue; }
                sh_run.x = x;
                sh_seg = make_int4(tid, unit == my_u ? s + 1 : s, 1, 0);      // a cut at the end: the run starts with the segment behind
            }
        }
    }
    __syncthreads();
    auto settle = [&](KrCursor& c) {                      // from a request's end to the next segment; there is one
        while (c.s >= pre_s[c.r + 1] - pre_s[c.r]) { ++c.r; c.s = 0; }
        c.u = units[c.r];
        const int tiles = (tokens[c.r] * G + 7) >> 3;
        c.kvh = c.s / tiles;
        c.tile = c.s - c.kvh * tiles;
        c.c0 = pre_u[c.r] + c.s * c.u;
    };
    int lo, hi, seg_pieces = 1, piece = 0;
    KrCursor seg;
    if (by_warp) {                                        // segments [s0, s1) in order are this warp's
        const int idx = warp * NB + j, W = NB * NW, s0 = (int)((long long)S * idx / W), s1 = (int)((long long)S * (idx + 1) / W);
        if (s0 >= s1) return;                             // (no barrier of the block lies behind)
        auto find = [&](int s, KrCursor& c) {             // the request of segment s
            int a = 0, b = p.B;                           // pre_s[a] <= s < pre_s[b]
            while (b - a > 1) {
                const int m = (a + b) >> 1;
                if (pre_s[m] <= s) a = m; else b = m;
            }
            c.r = a;
            c.s = s - pre_s[a];
            settle(c);
        };
        find(s1 - 1, seg);
        hi = seg.c0 + seg.u;
        find(s0, seg);
        lo = seg.c0;
    } else {
        lo = sh_run.x; hi = sh_run.y;
        if (lo >= hi) return;
        seg_pieces = sh_seg.z; piece = sh_seg.w;
        seg.r = sh_seg.x; seg.s = sh_seg.y;
        settle(seg);
    }
    // the warp's units: x0, x0 + step, ... below hi
    const int step = by_warp ? 1 : NW, x0 = by_warp ? lo : lo + warp, n_my = hi > x0 ? (hi - x0 + step - 1) / step : 0;
    const unsigned ring = kr_smem(kr_sh) + (unsigned)warp * ST * STAGE;

    // ---- the warp's loader: a lane knows the row of key `lane` of the unit that is asked for next, its page looked up a unit before
    KrCursor ld = seg;
    auto row_of = [&](int i) -> unsigned {
        if (i >= n_my) return 0xffffffffu;
        const int x = x0 + i * step;
        while (x >= ld.c0 + ld.u) { ++ld.s; settle(ld); }
        const int key = (x - ld.c0 + first[ld.r]) * KR_KEYS + lane;
        if (key >= keys[ld.r]) return 0xffffffffu;
        const int at = p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size;
        const int page = p.block_table[ld.r * p.bt_stride + at];
        return page >= 0 && page < p.pages ? ((unsigned)page * p.n_kv + ld.kvh) * p.page_size + (key - at * p.page_size) : 0xffffffffu;
    };
    auto load = [&](int i, unsigned row) {
        const unsigned st = ring + (unsigned)(i % ST) * STAGE;
#pragma unroll
        for (int m = 0; m < CH; ++m) {                    // 32 rows of CH chunks: CH a lane
            const int r = m * (32 / CH) + lane / CH, c = lane % CH;
            const unsigned src = __shfl_sync(0xffffffffu, row, r), dst = st + r * ROW + ((c ^ ((r >> SW) & (CH - 1))) << 4);
            const bool there = src != 0xffffffffu;
            const size_t off = there ? (size_t)src * ROW + c * 16 : 0;
            kr_cp16(dst, p.k + off, there);
            kr_cp16(dst + KV_BYTES, p.v + off, there);
        }
        const bool there = row != 0xffffffffu;
        kr_cp8(st + 2 * KV_BYTES + lane * 8, p.steps + (there ? row : 0u), there);
    };
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) {
        const unsigned row = row_of(i);
        if (i < n_my) load(i, row);
        kr_commit();
    }
    unsigned next = row_of(ST - 1);

    // Q as B operand: lane (g, t) holds row g's elements e, e + 4 of each of its words of eight, e = 0..3
    unsigned qf[QW][4];
    float qsum[2];                                        // of rows 2 t and 2 t + 1
    int c_end[2], c_from[2];                              // of these rows: the last key seen + 1, the first
    int all_end = 0, all_from = 0;                        // keys below all_end and from all_from on are seen by every row
    auto load_q = [&](const KrCursor& c) {
        const int n = tokens[c.r] * G, row = c.tile * 8 + g;
        const bool there = row < n;
        const int tok = row / G;
        const __nv_bfloat16* src = p.q + ((size_t)(token[c.r] + (there ? tok : 0)) * p.n_q + (size_t)c.kvh * G + (there ? row - tok * G : 0)) * D + t * (D / 4);
#pragma unroll
        for (int w = 0; w < QW; ++w) {
            const uint4 x = there ? *reinterpret_cast<const uint4*>(src + 8 * w) : make_uint4(0u, 0u, 0u, 0u);      // elements 01 23 45 67
            qf[w][0] = __byte_perm(x.x, x.z, 0x5410);
            qf[w][1] = __byte_perm(x.x, x.z, 0x7632);
            qf[w][2] = __byte_perm(x.y, x.w, 0x5410);
            qf[w][3] = __byte_perm(x.y, x.w, 0x7632);
        }
        float one[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < QW; ++w) {
            kr_mma(one, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u, qf[w][0], qf[w][1]);
            kr_mma(one, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u, qf[w][2], qf[w][3]);
        }
        qsum[0] = one[0]; qsum[1] = one[1];
        const int p0 = ends[c.r] - tokens[c.r], kv = keys[c.r];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int pos = p0 + min(c.tile * 8 + 2 * t + e, n - 1) / G;
            c_end[e] = min(pos + 1, kv);
            c_from[e] = p.window > 0 ? pos - p.window + 1 : 0;
        }
        all_end = min(p0 + c.tile * 8 / G + 1, kv);
        all_from = p.window > 0 ? p0 + min(c.tile * 8 + 7, n - 1) / G - p.window + 1 : 0;
    };
    load_q(seg);
    const float sc = p.scale * 1.4426950408889634f;
    int i = 0;
    bool first_segment = true;
    for (int begin = lo; begin < hi;) {
        const int end = min(hi, seg.c0 + seg.u);
        float o[D / 16][4];
#pragma unroll
        for (int mt = 0; mt < D / 16; ++mt) o[mt][0] = o[mt][1] = o[mt][2] = o[mt][3] = 0.f;
        float m_c[2] = {-INFINITY, -INFINITY}, l_c[2] = {0.f, 0.f}, z_c[2] = {0.f, 0.f};

        for (; i < n_my; ++i) {
            const int x = x0 + i * step;
            if (x >= end) break;
            kr_wait<ST - 2>();
            __syncwarp();                     // unit i has come for all lanes, and all have left the stage that is filled next
            if (i + ST - 1 < n_my) load(i + ST - 1, next);
            kr_commit();
            next = row_of(i + ST);
            const unsigned st = ring + (unsigned)(i % ST) * STAGE;
            const int key0 = (x - seg.c0 + first[seg.r]) * KR_KEYS;
            // ---- S^T = K Q^T, 16 keys a time
            float v[2][4];
            uint2 row_st[2][2];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const int r = 16 * m + g;
                unsigned kl[QW], kh[QW];
                if constexpr (D == 128) {
                    const unsigned a = st + r * ROW + ((t ^ ((r >> SW) & 3)) << 4);      // (row r + 8 has the same permutation)
                    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(kl[0]), "=r"(kl[1]), "=r"(kl[QW - 2]), "=r"(kl[QW - 1]) : "r"(a));
                    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(kh[0]), "=r"(kh[1]), "=r"(kh[QW - 2]), "=r"(kh[QW - 1]) : "r"(a + 8 * ROW));
                } else {
                    const unsigned a = st + r * ROW + (((t >> 1) ^ ((r >> SW) & 1)) << 4) + (t & 1) * 8;
                    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(kl[0]), "=r"(kl[1]) : "r"(a));
                    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(kh[0]), "=r"(kh[1]) : "r"(a + 8 * ROW));
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(row_st[m][h].x), "=r"(row_st[m][h].y) : "r"(st + 2 * KV_BYTES + (r + 8 * h) * 8));
                float s[4] = {-qsum[0], -qsum[1], -qsum[0], -qsum[1]}, s2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < QW; ++w) {
                    kr_mma(s, kr_unit<0>(kl[w]), kr_unit<0>(kh[w]), kr_unit<1>(kl[w]), kr_unit<1>(kh[w]), qf[w][0], qf[w][1]);
                    kr_mma(s2, kr_unit<2>(kl[w]), kr_unit<2>(kh[w]), kr_unit<3>(kl[w]), kr_unit<3>(kh[w]), qf[w][2], qf[w][3]);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float a = bf16_of(row_st[m][h].x & 0xffffu) * (16.f * sc), b = bf16_of(row_st[m][h].x >> 16) * sc;
#pragma unroll
                    for (int e = 0; e < 2; ++e) v[m][2 * h + e] = fmaf(a, s[2 * h + e] + s2[2 * h + e], b * qsum[e]);
                }
            }
            const bool edge = key0 + KR_KEYS > all_end || key0 < all_from;
            unsigned hidden = 0;                          // bit 4 m + e: value e of part m is a key that its row does not see
            if (edge) {
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = key0 + 16 * m + g + ((e & 2) ? 8 : 0);
                        if (key >= c_end[e & 1] || key < c_from[e & 1]) { v[m][e] = -INFINITY; hidden |= 1u << (4 * m + e); }
                    }
            }
            bool behind = false;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) behind = behind || v[m][e] > m_c[e & 1] + KR_LAZY;
            if (__any_sync(0xffffffffu, behind)) {
                float alpha[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float mx = fmaxf(fmaxf(v[0][e], v[0][e + 2]), fmaxf(v[1][e], v[1][e + 2]));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    const float mn = fmaxf(m_c[e], mx), mu = mn == -INFINITY ? 0.f : mn;
                    alpha[e] = kr_exp2(m_c[e] - mu);
                    m_c[e] = mn;
                    l_c[e] *= alpha[e];
                    z_c[e] *= alpha[e];
                }
#pragma unroll
                for (int mt = 0; mt < D / 16; ++mt) {
                    o[mt][0] *= alpha[0]; o[mt][1] *= alpha[1];
                    o[mt][2] *= alpha[0]; o[mt][3] *= alpha[1];
                }
            }
            // ---- weights of the codes, and what the bases add
            unsigned pb[2][2];
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float step16 = 16.f * bf16_of(row_st[m][h].y & 0xffffu), base = bf16_of(row_st[m][h].y >> 16);
                    float pr[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float mu = m_c[e] == -INFINITY ? 0.f : m_c[e];
                        pr[e] = kr_exp2(v[m][2 * h + e] - mu);
                        l_c[e] += pr[e];
                    }
                    const unsigned w = kr_pack(pr[0] * step16, pr[1] * step16);
                    const float w0 = __uint_as_float(w << 16), w1 = __uint_as_float(w & 0xffff0000u);
                    if (edge) {                           // a key that a row does not see counts for nothing, whatever it holds
                        z_c[0] += ((hidden >> (4 * m + 2 * h)) & 1u ? 0.f : pr[0] * base) - w0;
                        z_c[1] += ((hidden >> (4 * m + 2 * h + 1)) & 1u ? 0.f : pr[1] * base) - w1;
                    } else {
                        z_c[0] += fmaf(pr[0], base, -w0);
                        z_c[1] += fmaf(pr[1], base, -w1);
                    }
                    pb[m][h] = kr_trans(w);
                }
            // ---- O^T += U^T W^T
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const int r = 16 * m + (lane & 15);       // matrices: keys 0-7 and 8-15 of two neighbouring chunks
#pragma unroll
                for (int c2 = 0; c2 < CH / 2; ++c2) {
                    unsigned a[4];
                    const unsigned va = st + KV_BYTES + r * ROW + (((2 * c2 + (lane >> 4)) ^ ((r >> SW) & (CH - 1))) << 4);
                    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]) : "r"(va));
#pragma unroll
                    for (int h = 0; h < 2; ++h) {         // 32 elements: lane g has codes 4 g .. 4 g + 3 of keys 2 t, 2 t + 1
                        const unsigned lo8 = a[2 * h], hi8 = a[2 * h + 1];
                        kr_mma(o[4 * c2 + 2 * h], kr_unit<0>(lo8), kr_unit<1>(lo8), kr_unit<0>(hi8), kr_unit<1>(hi8), pb[m][0], pb[m][1]);
                        kr_mma(o[4 * c2 + 2 * h + 1], kr_unit<2>(lo8), kr_unit<3>(lo8), kr_unit<2>(hi8), kr_unit<3>(hi8), pb[m][0], pb[m][1]);
                    }
                }
            }
        }
        // ---- the warps' results through shared memory, added in warp order
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
                l_c[e] += __shfl_xor_sync(0xffffffffu, l_c[e], d);
                z_c[e] += __shfl_xor_sync(0xffffffffu, z_c[e], d);
            }
        const KrCursor now = seg;
        if (end >= hi) pdl_late();
        else { ++seg.s; settle(seg); load_q(seg); }       // the next segment's
        if (by_warp) __syncwarp();
        else if (!first_segment) __syncthreads();         // the segment before has been read
        first_segment = false;
#pragma unroll
        for (int mt = 0; mt < D / 16; ++mt)               // columns of o[2 x + y]: elements 32 (x / 1) ... : chunk mt / 2, elements 4 g + 2 (mt & 1) and the next
#pragma unroll
            for (int e = 0; e < 2; ++e)
                *reinterpret_cast<float2*>(Om + (warp * 8 + 2 * t + e) * OLD + (mt >> 1) * 32 + 4 * g + 2 * (mt & 1)) = make_float2(o[mt][e] + z_c[e], o[mt][e + 2] + z_c[e]);
        if (g == 0) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                Mm[warp * 8 + 2 * t + e] = m_c[e];
                Lm[warp * 8 + 2 * t + e] = l_c[e];
            }
        }
        const int row0 = now.tile * 8, n_rows = min(8, tokens[now.r] * G - row0);
        auto out_row = [&](int c) -> __nv_bfloat16* {
            const int tok = (row0 + c) / G;
            return p.out + ((size_t)(token[now.r] + tok) * p.n_q + (size_t)now.kvh * G + (row0 + c - tok * G)) * D;
        };
        auto put4 = [&](int c, int col, float4 x, float L) {
            const float inv = L != 0.f ? 1.f / L : 0.f;
            *reinterpret_cast<uint2*>(out_row(c) + col) = make_uint2(kr_pack(x.x * inv, x.y * inv), kr_pack(x.z * inv, x.w * inv));
        };
        constexpr int COLS = D / 4;                       // pieces of four elements a row
        if (by_warp) {
            __syncwarp();
            for (int idx = lane; idx < n_rows * COLS; idx += 32) {
                const int c = idx / COLS, col = idx % COLS * 4;
                put4(c, col, *reinterpret_cast<const float4*>(Om + (warp * 8 + c) * OLD + col), Lm[warp * 8 + c]);
            }
        } else {
            int pieces = seg_pieces, mine = piece;        // pieces of this segment, this block's among them
            if (!by_piece) {
                pieces = 1; mine = 0;
                if (begin > now.c0 || end < now.c0 + now.u) {      // the cuts inside are those of c + SNAP < floor(V i / NB) < c + u - SNAP; piece k in block first_cut - 1 + k
                    const long long c = now.c0 + (long long)KR_HEAD * (pre_s[now.r] + now.s + 1);
                    const int first_cut = (int)(((c + KR_SNAP + 1) * NB + V - 1) / V), last_cut = (int)(((c + now.u - KR_SNAP) * NB + V - 1) / V) - 1;
                    pieces = last_cut - first_cut + 2;
                    mine = j - (first_cut - 1);
                }
            }
            __syncthreads();
            const int slot = 2 * j + (mine == 0 ? 1 : 0);      // a run has at most one segment's first piece (its end) and one's later one (its start)
            for (int idx = tid; idx < n_rows * COLS; idx += THREADS) {
                const int c = idx / COLS, col = idx % COLS * 4;
                float M = -INFINITY;
#pragma unroll
                for (int w = 0; w < NW; ++w) M = fmaxf(M, Mm[w * 8 + c]);
                const float Mu = M == -INFINITY ? 0.f : M;
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                float L = 0.f;
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    const float f = kr_exp2(Mm[w * 8 + c] - Mu);
                    const float4 ov = *reinterpret_cast<const float4*>(Om + (w * 8 + c) * OLD + col);
                    acc.x = fmaf(f, ov.x, acc.x); acc.y = fmaf(f, ov.y, acc.y);
                    acc.z = fmaf(f, ov.z, acc.z); acc.w = fmaf(f, ov.w, acc.w);
                    L += f * Lm[w * 8 + c];
                }
                if (pieces == 1) {
                    put4(c, col, acc, L);
                } else {
                    *reinterpret_cast<float4*>(p.part_o + ((size_t)slot * 8 + c) * D + col) = acc;
                    if (col == 0) *reinterpret_cast<float2*>(p.part_ml + ((size_t)slot * 8 + c) * 2) = make_float2(M, L);
                }
            }
            if (pieces > 1) {
                __syncthreads();
                int* count = p.count + pre_s[now.r] + now.s;
                if (tid == 0) {                           // the fence behind the barrier covers what the block's other threads wrote
                    __threadfence();
                    sh_last = atomicAdd(count, 1) == pieces - 1;
                    __threadfence();
                }
                __syncthreads();
                if (sh_last) {                            // all pieces are there: merged in the order of the keys
                    const int b0 = j - mine;              // the block of piece 0
                    if (tid == 0) *count = 0;
                    for (int idx = tid; idx < n_rows * COLS; idx += THREADS) {
                        const int c = idx / COLS, col = idx % COLS * 4;
                        auto row_at = [&](int k) -> size_t { return (size_t)(2 * (b0 + k) + (k == 0 ? 1 : 0)) * 8 + c; };
                        float M = -INFINITY, L = 0.f;
                        for (int k = 0; k < pieces; ++k) M = fmaxf(M, __ldcg(p.part_ml + row_at(k) * 2));
                        const float Mu = M == -INFINITY ? 0.f : M;
                        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                        for (int k = 0; k < pieces; ++k) {
                            const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml + row_at(k) * 2));
                            const float4 ov = __ldcg(reinterpret_cast<const float4*>(p.part_o + row_at(k) * D + col));
                            const float f = kr_exp2(ml.x - Mu);
                            L = fmaf(f, ml.y, L);
                            acc.x = fmaf(f, ov.x, acc.x); acc.y = fmaf(f, ov.y, acc.y);
                            acc.z = fmaf(f, ov.z, acc.z); acc.w = fmaf(f, ov.w, acc.w);
                        }
                        put4(c, col, acc, L);
                    }
                }
            }
        }
        begin = end;
    }
    kr_wait<0>();
}

constexpr int KR_NW = 8, KR_ST = 4;

// Requests with 1 .. max_q tokens; q_start null: request r has token r.  count: a word for every 8 rows of a request under a kv head, zero before and after.
MSGL_API int msgl_kv4_attention_runs(const void* q, void* out, const void* k, const void* v, const void* steps, const int* q_start, const int* kv_len, const int* block_table,
                                     long long bt_stride, int bt_width, float* part_o, float* part_ml, int* count, int blocks, int B, int T, int n_q, int n_kv, int d,
                                     int page_size, int pages, int window, int max_q, float scale, cudaStream_t stream) {
    if (B <= 0 || T <= 0) return MSGL_OK;
    if ((d != 64 && d != 128) || B > KR_MAX_B || n_kv < 1 || n_q < 1 || n_q % n_kv || page_size < 1 || pages < 1 || bt_width < 1 || max_q < 1 || blocks < 1 || blocks > 4096 ||
        (long long)bt_width * page_size > 0x3fffffffLL || (long long)pages * n_kv * page_size >= 0xffffffffLL || part_o == nullptr || part_ml == nullptr || count == nullptr)
        return MSGL_ERR_SIZE;
    const long long tiles = ((long long)max_q * (n_q / n_kv) + 7) / 8, most = (long long)B * n_kv * tiles;
    if (most * (((long long)bt_width * page_size + KR_KEYS - 1) / KR_KEYS + KR_HEAD + 1) >= (1LL << 31)) return MSGL_ERR_SIZE;
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k | (uintptr_t)v | (uintptr_t)steps | (uintptr_t)part_o | (uintptr_t)part_ml) & 15) return MSGL_ERR_ALIGN;
    static MsglOncePerDevice attr_set;
    if (attr_set.due()) {
        if (cudaFuncSetAttribute(kv4_attn_runs_kernel<64, KR_NW, KR_ST>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kr_smem_bytes<64, KR_NW, KR_ST>()) != cudaSuccess ||
            cudaFuncSetAttribute(kv4_attn_runs_kernel<128, KR_NW, KR_ST>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kr_smem_bytes<128, KR_NW, KR_ST>()) != cudaSuccess)
            return msgl_check_launch();
        attr_set.mark();
    }
    Kv4Runs p = {(const __nv_bfloat16*)q, (__nv_bfloat16*)out, (const unsigned char*)k, (const unsigned char*)v, (const uint2*)steps, q_start, kv_len, block_table, part_o,
                 part_ml, count, bt_stride, B, T, n_q, n_kv, page_size, -1, pages, bt_width, window, max_q, scale};
    if ((page_size & (page_size - 1)) == 0) { p.page_shift = 0; while ((1 << p.page_shift) < page_size) ++p.page_shift; }
    if (d == 64) msgl_launch_pdl(kv4_attn_runs_kernel<64, KR_NW, KR_ST>, dim3(blocks), dim3(KR_NW * 32), kr_smem_bytes<64, KR_NW, KR_ST>(), stream, p);
    else msgl_launch_pdl(kv4_attn_runs_kernel<128, KR_NW, KR_ST>, dim3(blocks), dim3(KR_NW * 32), kr_smem_bytes<128, KR_NW, KR_ST>(), stream, p);
    return msgl_check_launch();
}
