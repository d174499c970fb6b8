// Attention for trees of drafted tokens on the 5th-generation tensor cores: bfloat16, head sizes 64 and 128, pages that TMA can fetch.
//
// A block, alone on its SM, walks its run of segments (attention_tree.cu): up to 256 rows -- (draft, head of the group) pairs of one kv head --
// against tiles of 128 keys.
//
//     S = Q K^T     tcgen05.mma 128 x 128 x 16, operands in shared memory, accumulator in tensor memory
//     softmax       two threads a row (TMEM lane), 64 scores each in registers; P, rounded to bfloat16 (by up to half a step, 2^-8 of each weight;
//                   the sum of the weights is taken before), goes back over the columns that each thread's scores had
//     O += P V      tcgen05.mma 128 x D x 16, P from tensor memory, V from shared memory as it lies in the cache
//
// The products of a tile keep the tensor core about as busy as its exponentials the special-function units, and one follows the other for
// any one tile.  So there are always two softmax groups, A and B, with scores and accumulators of their own, and the issuer alternates
// between them:  S_A  S_B  P V_A  S_A  P V_B  S_B ...  What differs is what they share:
//
//     more than 128 rows    A has rows 0 .. 127, B the others; both see every key tile
//     up to 128 rows        both have the same rows, A the even key tiles of the segment, B the odd ones; the two results are joined at the end
//
// so few rows, where the stream of keys is the bound, still have two tiles in work and two on their way.
//
// Keys come by TMA (a page of a kv head is a run of rows of the cache taken as one matrix), a lane a page, into rings of ST tiles of keys
// and of values; the loaders run ahead across the segments.  Of the tiles that hold drafts the values are looked at: rows behind the last
// key are cleared (free slots may hold anything), and elements that are no numbers are cleared and remembered, since 0 x inf would reach
// drafts that do not see them; the drafts that do see them get them back at the end.
//
// The exponentials' reference m need not be a row's maximum: it moves where a tile's maximum is 2^8 above it, and O is scaled in tensor
// memory then.  The two threads of a row meet once a tile, over the maximum, so they move alike.
//
// Bound, at 32 query heads on 8 kv heads of 128: up to 128 rows by the stream of keys and values (37 requests behind 8,192 keys: 1 draft 191 us, 6.5 TB/s, 8 drafts 196, 16 drafts 205, 32
// drafts 218, 5.7 TB/s); beyond by a tile's chain from scores over P to P V (64 drafts 330 to 350 us, some 900 TFLOP/s).  There a tile of 256 rows takes
// 3,700 to 3,900 cycles, 2,048 of them in the tensor core, 2,048 in the exponentials: scores come 710 cycles after their first product was issued, 950 beside the
// other group's work (Q and K out of shared memory take all of its 128 bytes a cycle), the softmax takes 2,100, the issuer sees P 300 later.
//
// Every wait is bounded; a block that gives up sets the status word, waits for its copies, frees its tensor memory and returns.
//
// Warps: 0-7 softmax A, 8-15 softmax B (all also fetch Q), 16 keys, 17 values, 18 issuer.  A softmax warp w works on TMEM lanes 32 (w % 4) .., and
// on the half (w / 4) % 2 of a tile's keys and of O's columns.  With one thread a row and 128 scores each a tile of 256 rows took 2.7 us, half
// of it waiting for the next scores: the softmax of a tile is what its successor waits for, and so it is spread over twice the warps.
// What the softmax warps know of their segments stands in shared memory: there is no register for it.
#pragma once
#include "tc_common.cuh"

constexpr int TT_ROWS = 256, TT_KT = 128, TT_THREADS = 608, TT_SOFT = 512;
constexpr unsigned TT_HALF = 128u * 128u;            // 128 rows of 64 columns, 128-byte swizzle: 16 KB
constexpr int TT_BAD = 8;                            // segments whose non-numbers are remembered: more than the loaders run ahead

template <int D> struct TreeTc {
    static constexpr int H = D / 64, ST = D == 128 ? 2 : 4;                                       // halves of a row, stages of a ring
    static constexpr unsigned TILE = H * TT_HALF;
    static constexpr unsigned SMEM = 2u * TILE + 2u * ST * TILE;                                  // Q_A, Q_B, keys, values
    static constexpr unsigned ALLOC = SMEM + 1024u + 512u + 1280u * 4u;                           // barriers, scalars and exchange ahead, alignment
};

// two float32 values in one 64-bit register, for the packed float32 instructions of sm_100
__device__ __forceinline__ unsigned long long tt_pack(float lo, float hi) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void tt_unpack(unsigned long long v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;\n" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ unsigned long long tt_fma(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ unsigned long long tt_add(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ void tt_cp_async16(unsigned s, const void* gmem, bool valid) {
    const int n = valid ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(s), "l"(gmem), "r"(n));
}
// byte offset of (row, 16-byte chunk c) in a swizzled tile
__device__ __forceinline__ unsigned tt_off(int row, int c) {
    return (unsigned)(c >> 3) * TT_HALF + (unsigned)row * 128u + (unsigned)(((c & 7) ^ (row & 7)) << 4);
}
__device__ __forceinline__ unsigned tt_nonfinite(unsigned w) {               // two bfloat16: the bits of those that are inf or NaN
    return ((w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
}

// The products are issued by a whole warp, converged, one lane of which is elected: what they take then stands in uniform registers.  From a branch of
// a single lane every operand had to be moved there by itself, and a 128 x 128 x 16 product (64 cycles) took 118.
__device__ __forceinline__ unsigned tt_elect() {
    unsigned leader;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(leader));
    return leader;
}
__device__ __forceinline__ void tt_mma(unsigned leader, unsigned d_tmem, unsigned long long a_desc, unsigned long long b_desc, unsigned idesc, unsigned accumulate) {
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\n"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(leader) : "memory");
}
__device__ __forceinline__ void tt_mma_ta(unsigned leader, unsigned d_tmem, unsigned a_tmem, unsigned long long b_desc, unsigned idesc, unsigned accumulate) {
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\n"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
                 ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(leader) : "memory");
}
__device__ __forceinline__ void tt_commit(unsigned leader, unsigned bar) {
    asm volatile("{\n.reg .pred q;\nsetp.ne.b32 q, %1, 0;\n@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar), "r"(leader) : "memory");
}

// tma_box: rows of a TMA box, min(page_size, 128)
template <int D>
__global__ void __launch_bounds__(TT_THREADS, 1) tree_tc_kernel(const TreeParams p, int* status, const __grid_constant__ CUtensorMap kmap,
                                                                const __grid_constant__ CUtensorMap vmap, int tma_box) {
    using C = TreeTc<D>;
    constexpr int ST = C::ST, H = C::H;
    extern __shared__ __align__(16) unsigned char tt_smem[];
    // ahead of the tiles: barriers, scalars, the non-numbers' words, what the rows' threads exchange
    unsigned& tmem_base_s = *reinterpret_cast<unsigned*>(tt_smem + 248);
    unsigned* bad_words = reinterpret_cast<unsigned*>(tt_smem + 256);                     // [TT_BAD][8]
    float* exchange = reinterpret_cast<float*>(tt_smem + 512);                            // [2 groups][2 halves][128] maxima, the same of sums, [2][128] references
    __shared__ TreeSegment sh_seg[2];                // the softmax groups' segment and the one after it
    __shared__ int sh_more[2];                        // 0: there is none; the rows of Q to write for it
    __shared__ TreeWalkState sh_walk;                 // their walk
    __shared__ TreeStart begun;
    __shared__ TreeRecord sh_record;                 // (thread 0's; there is no register for it either)
    const unsigned smem_base = smem_u32(tt_smem);
    const unsigned smem0 = (smem_base + 512u + 1280u * 4u + 1023u) & ~1023u;
    const unsigned q_s = smem0, k_s = q_s + 2u * C::TILE, v_s = k_s + ST * C::TILE;
    auto bar_s = [&](int x) { return smem_base + 8u * x; };                  // S_X is in TMEM (tensor core commits)
    // P_X's first 32 of every 64 keys are in TMEM and O_X is rescaled, and the others are there as well (8 softmax warps each)
    auto bar_p = [&](int x, int part) { return smem_base + (part ? 192u : 16u) + 8u * x; };
    auto bar_o = [&](int x) { return smem_base + 32u + 8u * x; };            // P V_X is done (tensor core commits)
    const unsigned bar_q = smem_base + 48u, bar_vt = smem_base + 56u;        // the segment's Q is there (512 threads); a V tile that is looked at has come
    auto bar_kf = [&](int st) { return smem_base + 64u + 8u * st; };         // stage holds a tile of keys (TMA bytes)
    auto bar_kr = [&](int st) { return smem_base + 96u + 8u * st; };         // it has been read
    auto bar_vf = [&](int st) { return smem_base + 128u + 8u * st; };
    auto bar_vr = [&](int st) { return smem_base + 160u + 8u * st; };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, j = blockIdx.x;
    const int G = p.G;

    if (tid == 0) {
        sh_record = TreeRecord{};
        for (int x = 0; x < 2; ++x) { tc_mbar_init(bar_s(x), 1); tc_mbar_init(bar_p(x, 0), 8); tc_mbar_init(bar_p(x, 1), 8); tc_mbar_init(bar_o(x), 1); }
        for (int st = 0; st < ST; ++st) { tc_mbar_init(bar_kf(st), 1); tc_mbar_init(bar_kr(st), 1); tc_mbar_init(bar_vf(st), 1); tc_mbar_init(bar_vr(st), 1); }
        tc_mbar_init(bar_q, TT_SOFT); tc_mbar_init(bar_vt, 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (tid == 32) {
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&kmap) : "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&vmap) : "memory");
    }
    pdl_launch_dependents();
    pdl_wait();
    pdl_after_wait();
    const int gave_up = *reinterpret_cast<volatile int*>(status);           // (on its way while the work is cut)
    if (warp == 18) {            // all 512 columns of tensor memory: S_A | S_B | O_A | O_B (behind the wait: a kernel ahead of this one may want some)
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(&tmem_base_s)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    tc_fence_before();
    TreeWalk<TT_ROWS, TT_KT> walk(p);
    const bool mine = walk.begin(j, gridDim.x, begun) && smem0 + C::SMEM <= smem_base + C::ALLOC;
    const bool work = __syncthreads_or(gave_up != 0) == 0 && mine;           // (an earlier block gave up: do not pile up)
    tc_fence_after();
    const unsigned tmem = tmem_base_s;
    int fail = 0;

    if (!work) {
        if (tid == 0 && smem0 + C::SMEM > smem_base + C::ALLOC) atomicExch(status, 2);      // allocation not aligned as assumed
    } else if (warp == 16 || warp == 17) {
        // =========================== loaders: lane b brings box b
        const bool is_k = warp == 16;
        const CUtensorMap* map = is_k ? &kmap : &vmap;
        const int n_box = TT_KT / tma_box;
        unsigned vt_phase = 0, count = 0, seg = 0;
        // Values that are looked at: clears the rows behind the last key and what is no number, once the tile has come.  Put off until the next tile's pages are known.
        int due = -1, due_key0 = 0, due_base = 0, due_kv = 0;                        // the stage of such a tile
        unsigned due_seg = 0;
        auto look = [&]() {
            const int st = due;
            due = -1;
            if (__any_sync(0xffffffffu, !tc_mbar_wait(bar_vt, vt_phase))) return false;
            vt_phase ^= 1u;
            const unsigned dst_tile = v_s + (unsigned)st * C::TILE;
            auto chunk_at = [&](int row, int c) { return dst_tile + tt_off(row, c); };
            const int end = min(max(due_kv - due_key0, 0), TT_KT);           // rows that hold keys
            for (int i = lane; i < (TT_KT - end) * H * 8; i += 32)
                asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};\n" ::"r"(chunk_at(end + i / (H * 8), i % (H * 8))), "r"(0u) : "memory");
            const int first = min(max(due_base - due_key0, 0), end);         // the drafts among them
            for (int i = lane; i < (end - first) * H * 8; i += 32) {
                const int row = first + i / (H * 8);
                const unsigned a = chunk_at(row, i % (H * 8));
                uint4 v;
                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
                const unsigned bx = tt_nonfinite(v.x), by = tt_nonfinite(v.y), bz = tt_nonfinite(v.z), bw = tt_nonfinite(v.w);
                if ((bx | by | bz | bw) != 0u) {
                    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};\n" ::"r"(a), "r"(v.x & ~bx), "r"(v.y & ~by), "r"(v.z & ~bz), "r"(v.w & ~bw) : "memory");
                    const int draft = due_key0 + row - due_base;
                    if (draft >= 0 && draft < 256) atomicOr(&bad_words[(due_seg % TT_BAD) * 8 + (draft >> 5)], 1u << (draft & 31));
                }
            }
            tc_fence_async_smem();
            __syncwarp();
            if (lane == 0) tc_mbar_arrive(bar_vf(st));
            return true;
        };
        TreeSegment g = begun.first;
        for (bool more = true; !fail && more; more = walk.next(g), ++seg) {
            const int* bt = p.table + (size_t)g.r * p.table_stride;
            if (!is_k) { if (lane < 8) bad_words[(seg % TT_BAD) * 8 + lane] = 0u; __syncwarp(); }
            for (int t = g.t_lo; t < g.t_hi; ++t, ++count) {
                const int st = count % ST, key0 = t * TT_KT, key_b = key0 + lane * tma_box;
                int y = -1;                          // (a box that is not fetched)
                if (lane < n_box && key_b < g.kv) {
                    const int pi = tree_page(p, key_b), id = bt[pi];
                    // a page outside the cache: rows ahead of the matrix, which TMA reads as zeros
                    y = id >= 0 && id < p.pages ? (int)(((long long)id * p.n_kv + g.kvh) * p.page_size) + (key_b - pi * p.page_size) : -1024;
                }
                const unsigned n_act = __popc(__ballot_sync(0xffffffffu, y != -1));
                const bool looked_at = !is_k && key0 + TT_KT > g.base;
                if (due >= 0 && !look()) { fail = 1; break; }
                if (count >= ST && __any_sync(0xffffffffu, !tc_mbar_wait(is_k ? bar_kr(st) : bar_vr(st), (count / ST - 1) & 1))) { fail = 1; break; }
                const unsigned bar = looked_at ? bar_vt : (is_k ? bar_kf(st) : bar_vf(st)), dst_tile = (is_k ? k_s : v_s) + (unsigned)st * C::TILE;
                if (lane == 0) tc_mbar_expect_tx(bar, n_act * H * (unsigned)tma_box * 128u);
                __syncwarp();
                if (y != -1) {
                    const unsigned dst = dst_tile + (unsigned)(lane * tma_box) * 128u;
#pragma unroll
                    for (int h = 0; h < H; ++h) tc_tma_load(dst + h * TT_HALF, map, 64 * h, y, bar);
                }
                if (looked_at) { due = st; due_key0 = key0; due_base = g.base; due_kv = g.kv; due_seg = seg; }
            }
        }
        if (!fail && due >= 0 && !look()) fail = 1;
        // nobody leaves with copies under way (values that are looked at have been waited for above)
        for (unsigned c = count > ST ? count - ST : 0; c < count; ++c) tc_mbar_wait(is_k ? bar_kf(c % ST) : bar_vf(c % ST), (c / ST) & 1);
    } else if (warp == 18) {
        // =========================== issuer
        const unsigned idesc_s = tc_idesc(false, TT_KT), idesc_o = tc_idesc(true, D), leader = tt_elect();
        // descriptors of the first tiles; others are a number of 16-byte units further in the address field
        const unsigned long long dq = tc_desc(q_s, 16, 1024), dk = tc_desc(k_s, 16, 1024), dv = tc_desc(v_s, TT_HALF, 1024);
        constexpr unsigned step = C::TILE >> 4;
        const unsigned tm = __shfl_sync(0xffffffffu, tmem, 0);
        unsigned count = 0, seg = 0, phase_p[2] = {0u, 0u};                           // tiles before this segment
        TreeSegment g = begun.first;
        auto wait = [&](unsigned bar, unsigned parity) { return __all_sync(0xffffffffu, tc_mbar_wait(bar, parity)) != 0; };
        bool ok = true;
        for (bool more = true; ok && more; more = walk.next(g), ++seg) {
            const bool dual = __shfl_sync(0xffffffffu, g.rows, 0) > 128;
            const int tiles = __shfl_sync(0xffffffffu, g.t_hi - g.t_lo, 0), steps = dual ? 2 * tiles : tiles;
            auto tile_of = [&](int s) { return count + (dual ? s >> 1 : s); };
            auto issue_o = [&](int s) {                               // O_X += P_X V
                const int x = s & 1;
                const unsigned c = tile_of(s), st = c % ST;
                if (!dual || x == 0) ok = wait(bar_vf(st), (c / ST) & 1);
                const unsigned long long dv_st = dv + st * step;
                const unsigned t_o = tm + 256u + (unsigned)x * 128u, t_p = tm + (unsigned)x * 128u;
                // in two parts, as P comes: of both halves of the keys the first two sixteens, then the others
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    if (ok) ok = wait(bar_p(x, part), phase_p[x]);
                    if (!ok) return;
                    tc_fence_after();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int kk = (i >> 1) * 4 + part * 2 + (i & 1);
                        tt_mma_ta(leader, t_o, t_p + (kk >> 2) * 64u + (kk & 3) * 8u, dv_st + kk * (2048u >> 4), idesc_o, part + i > 0 ? 1u : s < 2 ? 0u : 1u);
                    }
                }
                phase_p[x] ^= 1u;
                tt_commit(leader, bar_o(x));
                if (!dual || x == 1) tt_commit(leader, bar_vr(st));
            };
            ok = wait(bar_q, seg & 1);
            tc_fence_async_smem();                    // Q came by plain copies (keys and values by TMA; the values that are looked at are fenced where they are written)
            for (int s = 0; s < steps && ok; ++s) {
                const int x = s & 1;
                const unsigned c = tile_of(s), st = c % ST;
                if (!dual || x == 0) ok = wait(bar_kf(st), (c / ST) & 1);
                if (!ok) break;
                tc_fence_after();
                const unsigned long long dq_x = dq + (dual && x ? step : 0u), dk_st = dk + st * step;
                const unsigned t_s = tm + (unsigned)x * 128u;
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const unsigned at = (kk >> 2) * (TT_HALF >> 4) + (kk & 3) * 2u;
                    tt_mma(leader, t_s, dq_x + at, dk_st + at, idesc_s, kk > 0 ? 1u : 0u);
                }
                tt_commit(leader, bar_s(x));
                if (!dual || x == 1) tt_commit(leader, bar_kr(st));
                if (s >= 1) issue_o(s - 1);
            }
            if (ok) issue_o(steps - 1);
            count += tiles;
        }
        if (!ok) fail = 1;
    } else if (warp < 16) {
        // =========================== softmax: group x, half of the columns; TMEM lane lane_row
        const int x = warp >> 3, half = (warp >> 2) & 1, lane_row = tid & 127;
        const unsigned lane_sel = (unsigned)((warp & 3) * 32) << 16;
        const unsigned ts = tmem + (unsigned)x * 128u + lane_sel, to = tmem + 256u + (unsigned)x * 128u + lane_sel;
        float* const ex_max = exchange + x * 256, * const ex_sum = exchange + 512, * const ex_ref = exchange + 1024;
        const int pair = 2 + x * 4 + (warp & 3);     // the barrier of the two warps of these rows
        unsigned phase_s = 0, phase_o = 0, seg = 0;
        const float sc = p.scale_log2;
        // before: of the segment ahead (of none: 256)
        auto rows_to_write = [](int rows, int before) { return max(rows, rows <= 128 ? min(before, 128) : before > 128 ? before : 256); };
        auto find = [&](unsigned s) {                // (one thread)
            walk.load(sh_walk);
            TreeSegment w;
            const bool more = walk.next(w);
            sh_more[s & 1] = more ? rows_to_write(w.rows, sh_seg[(s - 1) & 1].rows) : 0;
            if (more) sh_seg[s & 1] = w;
            walk.store(sh_walk);
        };
        // 16-byte chunks over all softmax threads.  Rows without a query are zero, which spares the tensor cores' power; only those are written that held one for the
        // segment before (all of them each time took a segment 0.8 us).  (An item's rows are below 2^24: divided by way of the reciprocal.)
        auto load_q = [&](const TreeSegment& w, int upto) {
            const __nv_bfloat16* qg = reinterpret_cast<const __nv_bfloat16*>(p.q);
            for (int i = tid; i < upto * H * 8; i += TT_SOFT) {
                const int row = i / (H * 8), c = i % (H * 8), rr = w.row0 + row, draft = walk.quotient(rr, G);
                const bool valid = row < w.rows;
                tt_cp_async16(q_s + (unsigned)(row >> 7) * C::TILE + tt_off(row & 127, c),
                              valid ? qg + ((size_t)(w.tok0 + draft) * p.n_q + (size_t)w.kvh * G + (rr - draft * G)) * D + c * 8 : qg, valid);
            }
            tc_cp_async_arrive(bar_q);
        };
        load_q(begun.first, rows_to_write(begun.first.rows, TT_ROWS));
        if (tid == 0) { sh_seg[0] = begun.first; sh_more[0] = 1; sh_walk = begun.walk; }
        asm volatile("bar.sync 1, 512;\n" ::: "memory");
        for (; *reinterpret_cast<volatile int*>(&sh_more[seg & 1]) != 0; ++seg) {
            const TreeSegment& g = sh_seg[seg & 1];
            const bool dual = g.rows > 128;
            const bool cut = g.t_lo != 0 || g.t_hi != g.tiles;
            if (tid == TT_SOFT - 32) {               // (of the last warp: with few rows it has nothing else to do, and the first has all)
                if (cut && g.t_lo == 0) {
                    walk.load(sh_walk);
                    sh_record = TreeRecord{walk.pieces(g, j), g.rows, g.tok0, g.row0, g.kvh, {0, 0, 0}};
                }
                find(seg + 1);                       // (the segment before the present one has been left by all)
            }

            const int tiles = g.t_hi - g.t_lo, n_mine = dual ? tiles : (tiles + 1 - x) >> 1;
            const int row = dual ? x * 128 + lane_row : lane_row, rr = g.row0 + row;
            const bool valid = row < g.rows, active = row - lane < g.rows;               // whether the row, and any of the warp's, exists
            const int tok = g.tok0 + (valid ? walk.quotient(rr, G) : 0);
            float m_run = -INFINITY, l_run = 0.f;    // of the row; of this thread's half of the keys
            if (!active)                             // (P of rows that do not exist may be anything)
                for (int it = 0; it < n_mine; ++it) {
                    if (!fail && __any_sync(0xffffffffu, !tc_mbar_wait(bar_s(x), phase_s))) fail = 1;
                    phase_s ^= 1u;
                    if (lane == 0) { tc_mbar_arrive(bar_p(x, 0)); tc_mbar_arrive(bar_p(x, 1)); }
                }
            else for (int it = 0; it < n_mine; ++it) {          // (a warp that gave up goes on to meet its partner)
                if (!fail && __any_sync(0xffffffffu, !tc_mbar_wait(bar_s(x), phase_s))) fail = 1;
                phase_s ^= 1u;
                tc_fence_after();
                const int key0 = (g.t_lo + (dual ? it : 2 * it + x)) * TT_KT + 64 * half;
                float s0[32], s1[32];
                tc_ld32(ts + 64 * half, s0); tc_ld32(ts + 64 * half + 32, s1);
                tc_wait_ld(s0); tc_wait_ld(s1);
                unsigned seen1 = ~0u;
                auto hide = [&](float (&sv)[32], unsigned seen) {
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (!(seen >> e & 1u)) sv[e] = -INFINITY;
                };
                if (key0 + 64 > g.base) {
                    const unsigned* row_mask = p.mask + (size_t)tok * p.words;
                    hide(s0, tree_seen(row_mask, p.words, key0, g.base, g.kv));
                    seen1 = tree_seen(row_mask, p.words, key0 + 32, g.base, g.kv);
                    hide(s1, seen1);
                }
                float c4[4];                     // (maxima of three: one instruction)
#pragma unroll
                for (int e = 0; e < 4; ++e) c4[e] = fmaxf(s0[e], s1[e]);
#pragma unroll
                for (int e = 4; e < 32; ++e) c4[e & 3] = fmaxf(fmaxf(c4[e & 3], s0[e]), s1[e]);
                const float mine = fmaxf(fmaxf(c4[0], c4[1]), fmaxf(c4[2], c4[3])) * sc;
                ex_max[half * 128 + lane_row] = mine;
                asm volatile("bar.sync %0, 64;\n" ::"r"(pair) : "memory");
                const float mx = fmaxf(mine, ex_max[(1 - half) * 128 + lane_row]);
                const bool move = mx > m_run + 8.f || (m_run == -INFINITY && mx > -INFINITY);
                if (__any_sync(0xffffffffu, move)) {
                    const float a = move ? fast_exp2(m_run - mx) : 1.f;              // 0 for the first
                    if (move) { m_run = mx; l_run *= a; }
                    if (it >= 1) {               // (P V of this group's tile before is done: this S was issued after it)
#pragma unroll 1
                        for (int cb = half * (D / 32); cb < (half + 1) * (D / 32); ++cb) {
                            unsigned v0[16];
                            tc_ld16(to + cb * 16, v0);
                            tc_wait_ld16(v0);
#pragma unroll
                            for (int e = 0; e < 16; ++e) v0[e] = __float_as_uint(__uint_as_float(v0[e]) * a);
                            tc_st16(to + cb * 16, v0);
                        }
                    }
                }
                const float mu = m_run == -INFINITY ? 0.f : m_run;
                const unsigned long long sc2 = tt_pack(sc, sc), nmu2 = tt_pack(-mu, -mu);
                unsigned long long sum2[4] = {0ull, 0ull, 0ull, 0ull};               // (0.f, 0.f)
                auto expo = [&](const float (&sv)[32], int cb) {
                    unsigned pk[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        float x0, x1;
                        tt_unpack(tt_fma(tt_pack(sv[e], sv[e + 1]), sc2, nmu2), x0, x1);
                        const float e0 = fast_exp2(x0), e1 = fast_exp2(x1);
                        sum2[(e >> 1) & 3] = tt_add(sum2[(e >> 1) & 3], tt_pack(e0, e1));
                        pk[e >> 1] = pack_bf16(e0, e1);
                    }
                    tc_st16(ts + 64 * half + cb * 16, pk);
                };
                expo(s0, 0);
                tc_ld32(ts + 64 * half + 32, s1);            // (read again: kept, they would push others out of the registers)
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) tc_mbar_arrive(bar_p(x, 0));
                tc_wait_ld(s1);
                if (seen1 != ~0u) hide(s1, seen1);
                expo(s1, 1);
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) tc_mbar_arrive(bar_p(x, 1));
                float lo, hi;
                tt_unpack(tt_add(tt_add(sum2[0], sum2[1]), tt_add(sum2[2], sum2[3])), lo, hi);
                l_run += lo + hi;
            }
            // ---- the segment's end
            if (n_mine > 0) {
                if (!fail && __any_sync(0xffffffffu, !tc_mbar_wait(bar_o(x), (phase_o + n_mine - 1) & 1))) fail = 1;
                phase_o += n_mine;
                tc_fence_after();
            }
            // the row's halves and, where both groups have it, the groups' results; both groups meet here, also where one of them has given up
            ex_sum[(x * 2 + half) * 128 + lane_row] = l_run;
            if (half == 0) ex_ref[x * 128 + lane_row] = m_run;
            tc_fence_before();
            asm volatile("bar.sync 1, 512;\n" ::: "memory");
            tc_fence_after();
            // both groups have seen the last of this segment's scores, so Q is free: the next segment's comes while this one's rows are written, and its first
            // scores are made meanwhile
            if (const int upto = *reinterpret_cast<volatile int*>(&sh_more[(seg + 1) & 1])) load_q(sh_seg[(seg + 1) & 1], upto);
            float fa = 1.f, fb = 0.f, m_all = m_run, l_all;                              // factors of O_A and O_B (dual: of the group's own alone)
            if (dual) {
                l_all = ex_sum[x * 256 + lane_row] + ex_sum[x * 256 + 128 + lane_row];
            } else {
                const float ma = ex_ref[lane_row], mb = ex_ref[128 + lane_row];
                m_all = fmaxf(ma, mb);
                const float mu = m_all == -INFINITY ? 0.f : m_all;
                fa = fast_exp2(ma - mu);
                fb = fast_exp2(mb - mu);
                l_all = (ex_sum[lane_row] + ex_sum[128 + lane_row]) * fa + (ex_sum[256 + lane_row] + ex_sum[384 + lane_row]) * fb;
            }
            if (active && !fail) {
                const bool whole = !cut;
                const unsigned* row_mask = p.mask + (size_t)tok * p.words;
                const float inv = whole ? (l_all > 0.f ? 1.f / l_all : (l_all == l_all ? 0.f : l_all)) : 1.f;
                const unsigned* bad = bad_words + (seg % TT_BAD) * 8;
                unsigned any_bad = 0u;
#pragma unroll
                for (int w = 0; w < 8; ++w) any_bad |= *reinterpret_cast<const volatile unsigned*>(bad + w);
                const int slot = 2 * j + (g.t_lo == 0 ? 1 : 0);
                // blocks of 32 columns: two threads a row share them out, or four
                const int cb0 = dual ? half * (D / 64) : D == 128 ? 2 * x + half : x, cb1 = dual ? cb0 + D / 64 : D == 128 || half == 0 ? cb0 + 1 : cb0;
                const bool two = !dual && tiles > 1;
                __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(p.out) + ((size_t)tok * p.n_q + (size_t)g.kvh * G + (valid ? rr - (tok - g.tok0) * G : 0)) * D;
                float4* part = reinterpret_cast<float4*>(p.part_o) + (size_t)slot * (D / 4) * TT_ROWS + row;
                const unsigned t_own = dual ? to : tmem + 256u + lane_sel, t_other = tmem + 384u + lane_sel;
#pragma unroll 1
                for (int cb = cb0; cb < cb1; ++cb) {
                    float v[32];
                    tc_ld32(t_own + cb * 32, v);
                    tc_wait_ld(v);
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[e] *= fa;
                    if (two) {
                        float u[32];
                        tc_ld32(t_other + cb * 32, u);
                        tc_wait_ld(u);
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = fmaf(u[e], fb, v[e]);
                    }
                    if (any_bad != 0u && valid) {    // what was taken out of the values of drafts that this row sees
                        for (int w = 0; w < 8; ++w)
                            for (unsigned left = w < p.words ? row_mask[w] & *reinterpret_cast<const volatile unsigned*>(bad + w) : 0u; left; left &= left - 1u) {
                                const int key = g.base + 32 * w + __ffs(left) - 1, pi = tree_page(p, key);
                                const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(p.v_cache) +
                                    (((size_t)p.table[(size_t)g.r * p.table_stride + pi] * p.n_kv + g.kvh) * p.page_size + (key - pi * p.page_size)) * D + cb * 32;
#pragma unroll
                                for (int e = 0; e < 32; ++e) {
                                    const float f = __bfloat162float(src[e]);
                                    if (!(fabsf(f) < INFINITY)) v[e] += f;
                                }
                            }
                    }
                    if (valid && whole) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8)
                            *reinterpret_cast<uint4*>(dst + cb * 32 + e) = make_uint4(pack_bf16(v[e] * inv, v[e + 1] * inv), pack_bf16(v[e + 2] * inv, v[e + 3] * inv),
                                                                                      pack_bf16(v[e + 4] * inv, v[e + 5] * inv), pack_bf16(v[e + 6] * inv, v[e + 7] * inv));
                    } else if (valid) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4) part[(cb * 8 + e / 4) * TT_ROWS] = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
                    }
                }
                if (valid && !whole && half == 0 && (dual || x == 0)) *reinterpret_cast<float2*>(p.part_ml + ((size_t)slot * TT_ROWS + row) * 2) = make_float2(m_all, l_all);
            }
            tc_fence_before();
            asm volatile("bar.sync 1, 512;\n" ::: "memory");                 // the exchange and both accumulators are free
        }
    }
    if (tid == 0) p.record[j] = sh_record;
    pdl_late();
    tc_fence_before();
    const bool failed = __syncthreads_or(fail) != 0;
    tc_fence_after();
    if (failed && tid == 0) atomicExch(status, 1);
    if (warp == 18) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
}
