// Attention over a cache in 4 bits on the tensor cores: bfloat16, head sizes 64 and 128, requests that bring few tokens.
//
// A segment is up to 8 rows (token, query head) of one request under one kv head, and its keys in units of 32.  The units of all segments are dealt out
// over the warps of one block an SM; every warp works out from the requests' lengths alone which are its own, and goes through them by itself.
//   * few keys: a segment of u units has u / PIECE equal pieces (one up to ALONE units), a block a piece (or a block a whole segment, where that is nearly even), and a piece's
//     units are dealt out over the block's warps;
//   * otherwise the units of all segments, each with HEAD units ahead for what a segment costs beside its keys, are laid end to end and cut into as many runs of
//     equal length as there are warps.
// A segment within one warp's run is written out by it.  Of the others a warp leaves its part (it has at most two: one that its run starts with, and its last) in
// shared memory; behind the only barrier after the cut, parts of one segment are added in the order of the keys.  Where other blocks hold parts too, the
// sum goes to scratch memory, and the block that raises the segment's counter to the number of blocks adds them up and clears the counter.
//
// Mathematics.  A code c enters the products as a float16 number without a shift of its exponent: four bits at the bottom of the fraction are the subnormal
// c 2^-24, four bits above them 16 c 2^-24, both exact, so one "and" makes two elements of a word and every second pair takes no shift.  What the places differ by
// is put right in Q (elements that meet 16 c are divided by 16) and in rows of O at the end.  Of the values a byte goes in whole, as c + 16 c' 2^-24, beside its upper
// code alone, and the sums are told apart at the end: the upper bytes then take no masks (four operations eight codes instead of five).  With a key's step and base and q^ = q 2^e (e a row's
// own: |q^| < 2^15, exact unless it is 2^-29 of the row's largest element),
//     q k = step 2^(24 - e) sum q^ (c 2^-24) + base sum q
//     o   = sum_j p_j (base_j + step_j c_j) = 2^24 / F sum_j w_j (c_j 2^-24) + sum_j p_j base_j,   w_j = float16(p_j step_j F)
// F is a power of two of the warp's own that keeps step F <= 64 (p is at most 2^8, see KR_LAZY): where a unit brings a larger step, F and the sums are scaled down.
// That step may be of a key which a row does not see or gives no weight.  A row whose largest weight p step F then lies below KR_FLOOR takes its exponentials' reference g powers of two
// below its largest score: its p are up to 2^g and its w large enough again.  All sums of a row are against the same reference, so nothing else changes, but that every unit is
// looked at while g > 0.  w keeps 11 bits; below 2^-8 of the row's largest weight (2^-20 where steps are alike) it loses them one by one, and so it does where an unseen step
// is more than KR_LIFT powers of two above those that count.  64 requests of up to 16,000 keys take 0.7 % longer for it (with a factor a row, and weights looked at in every unit
// whose steps grow, 4 %); with g > 0 for all rows 64 of 8,000 take 124 us instead of 104.  So KR_FLOOR leaves g at 0 where a first key has nearly all weight and a value 1/500 of the
// others' size (2^-3 did not).  The tensor core cuts its sums off rather than rounding them, and those of codes from
// 0 up grow all the way while what they leave beside the bases is small (a mean of 16,000 values came out 1 % off); so every unit takes the middles of the codes times
// its weights out of all sums by one more product, and they are added back at the end from float32 sums of their own.
// Scores, p, sums and outputs are float32.  S^T = K Q^T with keys on the M dimension, the head's elements permuted so that a lane reads 16 bytes
// of a row; P goes through movmatrix; V^T fragments come by ldmatrix.trans on 16-bit columns, four codes of two neighbouring keys a register.  The
// exponentials' reference moves only where a score lies KR_LAZY above it.
//
// What bounds it.  Where there is work for all SMs, the operations of a unit: 500 instructions a warp for 4.3 KB, 144 of them to take codes apart, on a pipe that takes half an instruction a
// cycle; 64 requests of up to 16,000 keys (32 heads on 8, 794 MB) 142 us, 5.6 TB/s, 0.86 of copy.  With nine copies a lane for every unit whose sizes are looked at one by one it took 152, with
// selects for hidden keys in the inner loop 3 us more.  12 warps at 160 registers and three units a ring 141, 16 at 128 and two 145, 14 164, 8 with four 179 (before the last steps).  Few keys:
// latency; 1 request of 1,000 keys 10.5 us: 1.5 until the warps know their units, 1.4 for pages and queries, 2.5 for two units, 3 to add up and write.  16 requests of up to 4,096 keys 22.6 us
// (floor 8.4).
// A block that handed units to its warps in turn, with a barrier and a merge a segment, took 195 us for the first case and 58 where this takes 32 (123 requests of up to 777 keys, 64 heads).  bfloat16 codes
// 1 + c / 16 took 275 (two operations more a pair).  16 rows a segment, two products for every pair of codes, halve the codes' work but leave registers for 8 warps: 8 requests
// of 32 tokens behind 8,000 keys 200 -> 177, 12 of 5 tokens behind 2,000 26 -> 30: not kept.
#pragma once
#include <type_traits>

constexpr float KR_LAZY = 8.f;
constexpr int KR_FLOOR = -6, KR_LIFT = 100;      // powers of two: where a row's largest weight lies at least; how far its reference goes below its largest score at most
constexpr int KR_KEYS = 32;          // keys of a unit
constexpr int KR_MAX_B = 256;        // requests of a launch, a thread each
constexpr int KR_PIECE = 16;         // units of a block's piece at least, where segments are cut by themselves ...
constexpr int KR_ALONE = 48;         // ... and none of up to this many units is (32 units, 1 request of 1,000 keys: whole 10.1 us, in two pieces 10.8)
constexpr int KR_HEAD = 2;           // what a segment costs beside its units, in units (1: 12 of 5 tokens 26.4 us instead of 25.7; 3 and 4 are behind)

struct Kv4Runs {
    const __nv_bfloat16* q; __nv_bfloat16* out;
    const unsigned char* k; const unsigned char* v; const uint2* steps;
    const int* q_start; const int* kv_len; const int* block_table;
    float* part_o;                   // [2 * blocks][8][D]
    float* part_ml;                  // [2 * blocks][8][2]
    int* count;                      // a word a segment, zero before and after
    long long bt_stride;
    int B, T, n_q, n_kv, page_size, page_shift, pages, bt_width, window, max_q;
    int ahead;                       // what was written before the launch ahead of this one: 1: kv_len, q_start and block_table, which are read before it is waited for;
                                     // 2: all that is read here: it is waited for at the end
    float scale;
};

__device__ __forceinline__ unsigned kr_smem(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
// copies of 16 and 8 bytes; ZERO: or of that many zeros (there = false).  Offsets are compile-time numbers, so that they cost no additions
template <int S, int G, bool ZERO> __device__ __forceinline__ void kr_cp16(unsigned s, const void* g, bool there) {
    if (ZERO) asm volatile("{\n.reg .pred p;\nsetp.eq.u32 p, %2, 0;\ncp.async.cg.shared.global [%0 + %3], [%1 + %4], 16, p;\n}\n" ::"r"(s), "l"(g), "r"((unsigned)there), "n"(S), "n"(G));
    else asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %3], 16;\n" ::"r"(s), "l"(g), "n"(S), "n"(G));
}
template <bool ZERO> __device__ __forceinline__ void kr_cp8(unsigned s, const void* g, bool there) {
    if (ZERO) asm volatile("{\n.reg .pred p;\nsetp.eq.u32 p, %2, 0;\ncp.async.ca.shared.global [%0], [%1], 8, p;\n}\n" ::"r"(s), "l"(g), "r"((unsigned)there));
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n" ::"r"(s), "l"(g));
}
// f(0), f(1), ... with the number as a constant
template <int N, int I = 0, typename F> __device__ __forceinline__ void kr_each(F f) {
    if constexpr (I < N) { f(std::integral_constant<int, I>{}); kr_each<N, I + 1>(f); }
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
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void kr_mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// shared memory at an address and a compile-time offset
template <int O> __device__ __forceinline__ void kr_lds4(unsigned a, unsigned& x, unsigned& y, unsigned& z, unsigned& w) {
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4 + %5];\n" : "=r"(x), "=r"(y), "=r"(z), "=r"(w) : "r"(a), "n"(O));
}
template <int O> __device__ __forceinline__ void kr_lds2(unsigned a, unsigned& x, unsigned& y) {
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2 + %3];\n" : "=r"(x), "=r"(y) : "r"(a), "n"(O));
}
template <int O> __device__ __forceinline__ void kr_ldsm_t(unsigned a, unsigned (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4 + %5];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a), "n"(O));
}
// with an accumulator of zeros
__device__ __forceinline__ void kr_mma0(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// two floats to float16
__device__ __forceinline__ unsigned kr_half2(float lo, float hi) {
    unsigned r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// two rows of A (words wl, wh) times Q: elements 0 4, 1 5 (16 times their codes), 2 6, 3 7 (likewise) of the words
constexpr unsigned KR_LOW = 0x000f000fu, KR_HIGH = 0x00f000f0u, KR_BYTE = 0x00ff00ffu;
constexpr unsigned KR_MID_BYTE = 0x80808080u, KR_MID_HIGH = 0x80788078u;      // -128 and -120, about the middles of a byte and of its upper code, as float16 subnormals

__device__ __forceinline__ int kr_pieces(int u) { return u <= KR_ALONE ? 1 : u / KR_PIECE; }

struct KrCursor {
    int r, s, kvh, tile, c0, u;      // request, its segment, kv head and tile of rows; first unit of the segment among all, units
    unsigned key0;                   // (unit among all) * KR_KEYS + key0 is the unit's first key, modulo 2^32
    int keys;                        // of the request
};

template <int D, int NW, int ST>
constexpr size_t kr_smem_bytes() {
    return (size_t)NW * ST * (KR_KEYS * (D + 8)) + (size_t)NW * 8 * (D + 4) * 4 + (size_t)NW * 2 * (16 + 1) * 4 + (8 * KR_MAX_B + 4) * 4 + (size_t)NW * 16 * 4;
}

template <int D, int NW, int ST, bool WHOLE>
__global__ void __launch_bounds__(NW * 32, 1) kv4_attn_runs_kernel(const Kv4Runs p) {
    extern __shared__ __align__(128) unsigned char kr_sh[];
    constexpr int ROW = D / 2, KV_BYTES = KR_KEYS * ROW, STAGE = 2 * KV_BYTES + KR_KEYS * 8, OLD = D + 4;
    constexpr int CH = ROW / 16;                          // 16-byte chunks of a row
    constexpr int SW = CH == 4 ? 1 : 2;                   // chunk c of row r lies at c ^ (r >> SW & CH - 1): eight rows' chunks c are eight different 16-byte columns
    constexpr int QW = D / 32;                            // words of codes of a key row a lane
    static_assert(D == 64 || D == 128, "lanes read 8 or 16 bytes of a key row");
    static_assert(ST * STAGE >= 8 * OLD * 4, "a warp's last result lies where its ring was");
    float* firsts = reinterpret_cast<float*>(kr_sh + (size_t)NW * ST * STAGE);      // [NW][8][OLD] results that a run starts with
    float* slot_ml = firsts + NW * 8 * OLD;               // [NW][2][8][2] maxima and sums of a warp's first and last result
    int* slot_seg = reinterpret_cast<int*>(slot_ml + NW * 32);      // [NW][2] their segments, -1: none
    int* pre_u = slot_seg + NW * 2;                       // [B + 1] units of all segments of the requests before
    int* pre_s = pre_u + KR_MAX_B + 1;                    // [B + 1] segments of the requests before
    int* units = pre_s + KR_MAX_B + 1;                    // per request: units of a segment, first unit, keys, first token, tokens, keys with those beyond the table
    int* first = units + KR_MAX_B;
    int* keys = first + KR_MAX_B;
    int* token = keys + KR_MAX_B;
    int* tokens = token + KR_MAX_B;
    int* ends = tokens + KR_MAX_B;
    float* lifts = reinterpret_cast<float*>(ends + KR_MAX_B + 2) + (threadIdx.x >> 5) * 16;      // [8][2] a warp's rows: largest p step (p against the largest score), g; since the first key
    __shared__ int sh_all[4];                             // units and segments of all requests; whether segments are cut by themselves; (by_piece) blocks of this block's segment
    __shared__ int sh_mine;                               // by_piece: this block's number among them
    __shared__ int sh_x[NW + 1], sh_r[NW + 1], sh_s[NW + 1];      // the warps' runs: where they start among all units, the request, its segment
    __shared__ int sh_last[2];

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int G = p.n_q / p.n_kv, NB = (int)gridDim.x, j = (int)blockIdx.x, W = NB * NW;      // W: warps of the launch
    if (p.ahead == 0) pdl_wait();
    auto leave = [&]() { if (p.ahead != 0) pdl_wait(); };      // (whoever waits for this kernel counts on the one before it as well)

    // ---- the requests, a thread each; then one warp sums up their units, segments and pieces, neighbouring requests a lane, and cuts.  (Short code: it runs once, from a
    // cold instruction cache.)
    static_assert(NW * 32 >= KR_MAX_B || NW * 64 >= KR_MAX_B, "one or two requests a thread");
#pragma unroll 1
    for (int r = tid; r < p.B; r += NW * 32) {
        const int t0 = p.q_start != nullptr ? p.q_start[r] : r, n = p.q_start != nullptr ? p.q_start[r + 1] - t0 : 1, len = max(p.kv_len[r], 0);
        const int kv = max(min(len, p.bt_width * p.page_size), 0), f = (p.window > 0 ? max(len - n - p.window + 1, 0) : 0) / KR_KEYS;
        const bool taken = n >= 1 && n <= p.max_q && t0 >= 0 && t0 + n <= p.T;
        units[r] = taken ? max((kv + KR_KEYS - 1) / KR_KEYS - f, 1) : 0;
        pre_s[r] = taken ? p.n_kv * ((n * G + 7) >> 3) : 0;      // (its own segments, until they are summed up)
        first[r] = f; keys[r] = kv; token[r] = t0; tokens[r] = n; ends[r] = len;
    }
    if (lane < 2) slot_seg[2 * warp + lane] = -1;
    if (tid <= NW) sh_x[tid] = 0;
    if (tid == 0) sh_all[3] = 1;                          // (ahead of the barrier: the lane that finds the block's piece writes over it)
    __syncthreads();
    if (warp == 0) {
        const int per = (p.B + 31) >> 5, r0 = lane * per, r1 = min(r0 + per, p.B);
        int U = 0, S = 0, P = 0, longest = 0;
#pragma unroll 1
        for (int r = r0; r < r1; ++r) {
            const int u = units[r], segs = pre_s[r];
            U += u * segs;
            S += segs;
            P += kr_pieces(u) * segs;
            longest = max(longest, u);
        }
        int at_u = -U, at_s = -S, at_p = -P;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, U, o), y = __shfl_up_sync(0xffffffffu, S, o), z = __shfl_up_sync(0xffffffffu, P, o);
            if (lane >= o) { U += x; S += y; P += z; }
        }
        at_u += U; at_s += S; at_p += P;
        U = __shfl_sync(0xffffffffu, U, 31); S = __shfl_sync(0xffffffffu, S, 31); P = __shfl_sync(0xffffffffu, P, 31);
        longest = __reduce_max_sync(0xffffffffu, longest);
        const bool whole = P > NB && S <= NB && 3ll * longest * NB <= 4ll * U;      // a block a segment is nearly even, and nothing is left to merge
        const bool by_piece = whole || P <= NB;
        if (whole) at_p = at_s;
        if (lane == 0) { sh_all[0] = U; sh_all[1] = S; sh_all[2] = by_piece; pre_u[p.B] = U; pre_s[p.B] = S; }
#pragma unroll 1
        for (int r = r0; r < r1; ++r) {
            const int u = units[r], segs = pre_s[r], pc = whole ? 1 : kr_pieces(u), in_r = j - at_p;
            pre_u[r] = at_u; pre_s[r] = at_s;
            if (by_piece && in_r >= 0 && in_r < pc * segs) {      // the block's piece, dealt out over its warps
                const int s = in_r / pc, piece = in_r - s * pc, a = (int)((long long)u * piece / pc), n = (int)((long long)u * (piece + 1) / pc) - a;
                sh_all[3] = pc;
                sh_mine = piece;
#pragma unroll 1
                for (int w = 0; w <= NW; ++w) { sh_x[w] = at_u + s * u + a + n * w / NW; sh_r[w] = r; sh_s[w] = s; }
            }
            at_u += u * segs; at_s += segs; at_p += pc * segs;
        }
        __syncwarp();
        if (!by_piece && lane <= NW) {
            // cut i = floor(V i / W) falls into a request (the last whose V-sum before it is no larger), there into a segment, there onto a unit; a cut a lane
            const int V = U + KR_HEAD * S, V_per = V / W, i = j * NW + lane;
            int x = U;
            if (i < W) {
                const int raw = i * V_per + (int)((unsigned)i * (unsigned)(V - V_per * W) / (unsigned)W);
                int a = 0, b = p.B;
#pragma unroll 1
                while (b - a > 1) {
                    const int m = (a + b) >> 1;
                    if (pre_u[m] + KR_HEAD * pre_s[m] <= raw) a = m; else b = m;
                }
                const int un = units[a], in_r = raw - pre_u[a] - KR_HEAD * pre_s[a];      // (requests without segments lie ahead of one with the same sum)
                int s = in_r / (un + KR_HEAD);
                const int off = in_r - s * (un + KR_HEAD) - KR_HEAD, unit = max(off, 0);
                x = pre_u[a] + s * un + unit;
                sh_r[lane] = a;
                sh_s[lane] = s;
            }
            sh_x[lane] = x;
        }
    }
    static_assert(2 * NW <= 32, "a lane a cut, and later a part");
    __syncthreads();

    // ---- this warp's run of units [lo, hi) of the segments laid end to end, and the segment it starts in
    const bool by_piece = sh_all[2];
    if (sh_x[0] >= sh_x[NW]) { leave(); return; }         // (the whole block)
    auto settle = [&](KrCursor& c) {                      // from a request's end to the next segment; there is one
        while (c.s >= pre_s[c.r + 1] - pre_s[c.r]) { ++c.r; c.s = 0; }
        c.u = units[c.r];
        const int tiles = (tokens[c.r] * G + 7) >> 3;
        c.kvh = c.s;
        c.tile = 0;
        if (tiles > 1) { c.kvh = c.s / tiles; c.tile = c.s - c.kvh * tiles; }
        c.c0 = pre_u[c.r] + c.s * c.u;
        c.key0 = (unsigned)(first[c.r] - c.c0) * KR_KEYS;
        c.keys = keys[c.r];
    };
    const int lo = sh_x[warp], hi = sh_x[warp + 1];
    KrCursor seg;
    seg.r = sh_r[warp]; seg.s = sh_s[warp];
    const int n_my = max(hi - lo, 0);
    const unsigned ring = kr_smem(kr_sh) + (unsigned)warp * ST * STAGE;
    if (n_my > 0) {
        settle(seg);

        // ---- the warp's loader.  WHOLE: a page is a power of two of 16 keys or more, and all lanes know where the unit's two runs of 16 lie (rows behind the request's last
        // key are copied as they are, and hidden); else a lane knows the row of key `lane`.  The pages are looked up a unit before they are asked for.
        KrCursor ld = seg;
        const int* ld_table = p.block_table + ld.r * p.bt_stride;
        struct Place { int page0, page1, add0, add1; };      // row: page * n_kv * page_size + add
        const int page_rows = p.n_kv * p.page_size;
        auto look_up = [&](int key, int& page, int& add) {
            page = -1;
            if (key >= ld.keys) return;
            const int at = WHOLE ? key >> p.page_shift : key / p.page_size;
            add = ld.kvh * p.page_size + (WHOLE ? key & (p.page_size - 1) : key - at * p.page_size);
            page = ld_table[at];
        };
        auto place_of = [&](int x) -> Place {
            Place w = {-1, -1, 0, 0};
            if (x >= hi) return w;
            if (x >= ld.c0 + ld.u) {
                do { ++ld.s; settle(ld); } while (x >= ld.c0 + ld.u);
                ld_table = p.block_table + ld.r * p.bt_stride;
            }
            const int key = (int)((unsigned)x * KR_KEYS + ld.key0);
            look_up(WHOLE ? key : key + lane, w.page0, w.add0);
            if (WHOLE) look_up(key + 16, w.page1, w.add1);
            return w;
        };
        constexpr int PER = 32 / CH;                      // rows that a copy of the warp takes: CH copies a unit
        const int l_row = lane / CH, l_ch = lane % CH;
        const unsigned l_dst = ring + l_row * ROW + ((l_ch ^ ((l_row >> SW) & (CH - 1))) << 4);
        static_assert(PER % (CH << SW) == 0, "one place for all copies");
        const unsigned char *k_lane = p.k + lane * 16, *v_lane = p.v + lane * 16;
        auto load = [&](unsigned st, const Place& w) {    // st: the stage's offset in the ring
            if (WHOLE) {
                const bool t0 = (unsigned)w.page0 < (unsigned)p.pages, t1 = (unsigned)w.page1 < (unsigned)p.pages;
                const unsigned r0 = t0 ? (unsigned)w.page0 * page_rows + w.add0 : 0u, r1 = t1 ? (unsigned)w.page1 * page_rows + w.add1 : 0u;
                const unsigned char *k0 = k_lane + (size_t)r0 * ROW, *v0 = v_lane + (size_t)r0 * ROW, *k1 = k_lane + (size_t)r1 * ROW, *v1 = v_lane + (size_t)r1 * ROW;
                const bool up = lane & 16;
                const uint2* s0 = p.steps + ((up ? r1 : r0) + (lane & 15));
                auto copy = [&](auto zero) {
                    constexpr bool ZERO = zero.value;
                    kr_each<CH>([&](auto m) {
                        constexpr int R = m.value * PER, H = R / 16, S = R * ROW, O = (R - 16 * H) * ROW;
                        kr_cp16<S, O, ZERO>(l_dst + st, H ? k1 : k0, H ? t1 : t0);
                        kr_cp16<S + KV_BYTES, O, ZERO>(l_dst + st, H ? v1 : v0, H ? t1 : t0);
                    });
                    kr_cp8<ZERO>(ring + st + 2 * KV_BYTES + lane * 8, s0, up ? t1 : t0);
                };
                if (t0 && t1) copy(std::false_type{});
                else copy(std::true_type{});
            } else {
                const unsigned row = (unsigned)w.page0 < (unsigned)p.pages ? (unsigned)w.page0 * page_rows + w.add0 : 0xffffffffu;
                kr_each<CH>([&](auto m) {
                    constexpr int S = m.value * PER * ROW;
                    const unsigned src = __shfl_sync(0xffffffffu, row, m.value * PER + l_row);
                    const size_t off = src != 0xffffffffu ? (size_t)src * ROW + l_ch * 16 : 0;
                    kr_cp16<S, 0, true>(l_dst + st, p.k + off, src != 0xffffffffu);
                    kr_cp16<S + KV_BYTES, 0, true>(l_dst + st, p.v + off, src != 0xffffffffu);
                });
                kr_cp8<true>(ring + st + 2 * KV_BYTES + lane * 8, p.steps + (row != 0xffffffffu ? row : 0u), row != 0xffffffffu);
            }
        };

        // Q as B operand: lane (g, t) holds row g's elements e, e + 4 of each of its words of eight, e = 0..3
        const float sc = p.scale * 1.4426950408889634f;
        unsigned qf[QW][4];
        float q_base[2], q_step[2];                       // of rows 2 t and 2 t + 1: what a key's base and its step times the accumulated sum count in a score (log2 units)
        int c_end[2], c_from[2];                          // of these rows: the last key seen + 1, the first
        int all_end = 0, all_from = 0;                    // keys below all_end and from all_from on are seen by every row
        uint4 x_q[QW];                                    // the queries as they come
        auto fetch_q = [&](const KrCursor& c) {
            const int row = c.tile * 8 + g;
            const bool there = row < tokens[c.r] * G;
            const int tok = row / G;
            const __nv_bfloat16* src = p.q + ((size_t)(token[c.r] + (there ? tok : 0)) * p.n_q + (size_t)c.kvh * G + (there ? row - tok * G : 0)) * D + t * (D / 4);
#pragma unroll
            for (int w = 0; w < QW; ++w) x_q[w] = there ? *reinterpret_cast<const uint4*>(src + 8 * w) : make_uint4(0u, 0u, 0u, 0u);
        };
        auto take_q = [&](const KrCursor& c) {
            const int n = tokens[c.r] * G;
            float sum = 0.f, top = 0.f;
#pragma unroll
            for (int w = 0; w < QW; ++w) {
                const unsigned y[4] = {x_q[w].x, x_q[w].y, x_q[w].z, x_q[w].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float a = __uint_as_float(y[e] << 16), b = __uint_as_float(y[e] & 0xffff0000u);
                    sum += a + b;
                    top = fmaxf(top, fmaxf(fabsf(a), fabsf(b)));
                }
            }
#pragma unroll
            for (int d = 1; d < 4; d <<= 1) {
                sum += __shfl_xor_sync(0xffffffffu, sum, d);
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            }
            const int e2 = min(max(14 - ((int)(__float_as_uint(top) >> 23) - 127), -100), 100);      // top 2^e2 lies in [2^14, 2^15)
            const float up = __uint_as_float((unsigned)(127 + e2) << 23), up16 = up * 0.0625f, down = __uint_as_float((unsigned)(127 - e2) << 23) * 16777216.f;
#pragma unroll
            for (int w = 0; w < QW; ++w) {                // elements 01 23 45 67
                const unsigned y[4] = {x_q[w].x, x_q[w].y, x_q[w].z, x_q[w].w};
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    qf[w][2 * e] = kr_half2(__uint_as_float(y[e] << 16) * up, __uint_as_float(y[e + 2] << 16) * up);
                    qf[w][2 * e + 1] = kr_half2(__uint_as_float(y[e] & 0xffff0000u) * up16, __uint_as_float(y[e + 2] & 0xffff0000u) * up16);
                }
            }
            const int p0 = ends[c.r] - tokens[c.r], kv = keys[c.r];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                q_base[e] = __shfl_sync(0xffffffffu, sum, (2 * t + e) * 4) * sc;
                q_step[e] = __shfl_sync(0xffffffffu, down, (2 * t + e) * 4) * sc;
                const int pos = p0 + min(c.tile * 8 + 2 * t + e, n - 1) / G;
                c_end[e] = min(pos + 1, kv);
                c_from[e] = p.window > 0 ? pos - p.window + 1 : 0;
            }
            all_end = min(p0 + c.tile * 8 / G + 1, kv);
            all_from = p.window > 0 ? p0 + min(c.tile * 8 + 7, n - 1) / G - p.window + 1 : 0;
        };
        if (p.ahead != 1) fetch_q(seg);
        Place next;
        {
            Place w[ST - 1];
#pragma unroll
            for (int i = 0; i < ST - 1; ++i) w[i] = place_of(lo + i);
            next = place_of(lo + ST - 1);
            if (p.ahead == 1) { pdl_wait(); fetch_q(seg); }
#pragma unroll
            for (int i = 0; i < ST - 1; ++i) {
                if (i < n_my) load(i * STAGE, w[i]);
                kr_commit();
            }
        }
        take_q(seg);
        // where this lane reads in a stage: its key rows, its rows' steps, its matrix rows of the values (of two chunk pairs)
        const unsigned at_k = ring + (D == 128 ? g * ROW + ((t ^ ((g >> SW) & 3)) << 4) : g * ROW + (((t >> 1) ^ ((g >> SW) & 1)) << 4) + (t & 1) * 8);
        const unsigned at_s = ring + 2 * KV_BYTES + g * 8;
        const unsigned at_v = ring + KV_BYTES + (lane & 15) * ROW + (((lane >> 4) ^ (((lane & 15) >> SW) & (CH - 1))) << 4);
        unsigned st = 0, st_load = (ST - 1) * STAGE;      // offsets of the stage that is worked on and of the one that is filled
        for (int x = lo; x < hi;) {
            const int begin = x, end = min(hi, seg.c0 + seg.u);
            float o[D / 16][4];
#pragma unroll
            for (int mt = 0; mt < D / 16; ++mt) o[mt][0] = o[mt][1] = o[mt][2] = o[mt][3] = 0.f;
            float m_c[2] = {-INFINITY, -INFINITY}, mu_c[2] = {0.f, 0.f}, l_c[2] = {0.f, 0.f}, z_c[2] = {0.f, 0.f};      // mu_c: the exponentials' reference (m_c, or 0 before a key)
            float lim_c[2] = {-INFINITY, -INFINITY};      // how far above it a score may lie (a first key lies above any)
            float F = 0.f;                                // 0: no step seen yet
            float mid[4] = {0.f, 0.f, 0.f, 0.f};          // what the middles of the codes have been taken out by (KR_MID), rows and columns as o's

            for (; x < end; ++x) {
                kr_wait<ST - 2>();
                __syncwarp();                             // the unit has come for all lanes, and all have left the stage that is filled next
                if (x + ST - 1 < hi) load(st_load, next);
                kr_commit();
                next = place_of(x + ST);
                const int key0 = (int)((unsigned)x * KR_KEYS + seg.key0);
                // ---- S^T = K Q^T, 16 keys a time; v: scores less their reference, log2 units
                float v[2][4], s[2][2][4];
                uint2 row_st[2][2];
                unsigned kl[2][QW], kh[2][QW];
                kr_each<2>([&](auto mm) {
                    constexpr int m = mm.value;
                    if constexpr (D == 128) {
                        kr_lds4<16 * m * ROW>(at_k + st, kl[m][0], kl[m][1], kl[m][QW - 2], kl[m][QW - 1]);
                        kr_lds4<(16 * m + 8) * ROW>(at_k + st, kh[m][0], kh[m][1], kh[m][QW - 2], kh[m][QW - 1]);
                    } else {
                        kr_lds2<16 * m * ROW>(at_k + st, kl[m][0], kl[m][1]);
                        kr_lds2<(16 * m + 8) * ROW>(at_k + st, kh[m][0], kh[m][1]);
                    }
                });
                kr_each<2>([&](auto mm) {
                    constexpr int m = mm.value;
                    kr_lds2<128 * m>(at_s + st, row_st[m][0].x, row_st[m][0].y);
                    kr_lds2<128 * m + 64>(at_s + st, row_st[m][1].x, row_st[m][1].y);
                });
#pragma unroll
                for (int w = 0; w < QW; ++w)              // four chains side by side
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        const unsigned l = kl[m][w], u = kh[m][w], l8 = l >> 8, u8 = u >> 8;
                        if (w == 0) {
                            kr_mma0(s[m][0], l & KR_LOW, u & KR_LOW, l & KR_HIGH, u & KR_HIGH, qf[w][0], qf[w][1]);
                            kr_mma0(s[m][1], l8 & KR_LOW, u8 & KR_LOW, l8 & KR_HIGH, u8 & KR_HIGH, qf[w][2], qf[w][3]);
                        } else {
                            kr_mma(s[m][0], l & KR_LOW, u & KR_LOW, l & KR_HIGH, u & KR_HIGH, qf[w][0], qf[w][1]);
                            kr_mma(s[m][1], l8 & KR_LOW, u8 & KR_LOW, l8 & KR_HIGH, u8 & KR_HIGH, qf[w][2], qf[w][3]);
                        }
                    }
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float a = __uint_as_float(row_st[m][h].x << 16), b = __uint_as_float(row_st[m][h].x & 0xffff0000u);
#pragma unroll
                        for (int e = 0; e < 2; ++e) v[m][2 * h + e] = fmaf(a * q_step[e], s[m][0][2 * h + e] + s[m][1][2 * h + e], fmaf(b, q_base[e], -mu_c[e]));
                    }
                if (key0 + KR_KEYS > all_end || key0 < all_from) {      // keys that some row does not see
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int key = key0 + 16 * m + 8 * h + g;
                            // a value row that is no number shows through the scores of those who see it, and counts for nothing elsewhere; nor does what lies behind the last key
                            const unsigned y = row_st[m][h].y;
                            const bool number = (y & 0x7f800000u) != 0x7f800000u && (y & 0x7f80u) != 0x7f80u;
                            if (!number || key >= seg.keys) row_st[m][h].y = 0u;
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                if (!number) v[m][2 * h + e] = CUDART_NAN_F;
                                if (key >= c_end[e] || key < c_from[e]) v[m][2 * h + e] = -INFINITY;
                            }
                        }
                }
                float st_f[2][2];                         // values' steps times F
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int h = 0; h < 2; ++h) st_f[m][h] = __uint_as_float(row_st[m][h].y << 16) * F;
                // how far the largest score lies above its reference, and the largest step
                const float above[2] = {fmaxf(fmaxf(v[0][0], v[0][2]), fmaxf(v[1][0], v[1][2])), fmaxf(fmaxf(v[0][1], v[0][3]), fmaxf(v[1][1], v[1][3]))};
                const float most_step = fmaxf(fmaxf(st_f[0][0], st_f[0][1]), fmaxf(st_f[1][0], st_f[1][1]));
                if (__any_sync(0xffffffffu, above[0] > lim_c[0] || above[1] > lim_c[1] || most_step > 64.f)) {
                    float alpha[2];
                    // the largest step of the unit, to the power of two above it
                    float step = 0.f;
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int h = 0; h < 2; ++h) step = fmaxf(step, __uint_as_float(row_st[m][h].y << 16));
                    const unsigned bits = __reduce_max_sync(0xffffffffu, __float_as_uint(step));
                    const float f = 64.f / fminf(fmaxf(__uint_as_float((bits + 0x007fffffu) & 0x7f800000u), 0x1p-100f), 0x1p127f), down = F == 0.f || f >= F ? 1.f : f / F;
                    if (F == 0.f || f < F) F = f;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mx = above[e];
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        float* lift = lifts + 4 * t + 2 * e;
                        const bool first = m_c[e] == -INFINITY;
                        const float old = m_c[e] + (first ? 0.f : lift[1]), mn = fmaxf(old, mx + mu_c[e]), at = mn == -INFINITY ? 0.f : mn;
                        float top = 0.f;                  // the unit's largest p step
#pragma unroll
                        for (int m = 0; m < 2; ++m)
#pragma unroll
                            for (int h = 0; h < 2; ++h) top = fmaxf(top, kr_exp2(v[m][2 * h + e] + (mu_c[e] - at)) * __uint_as_float(row_st[m][h].y << 16));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        if (!first) top = fmaxf(top, lift[0] * kr_exp2(old - at));
                        const int g = top > 0.f ? min(max(KR_FLOOR + 127 - (int)(__float_as_uint(top * F) >> 23), 0), KR_LIFT) : 0;
                        const float mu = at - (float)g;
                        __syncwarp();                     // (eight lanes have the same rows)
                        lift[0] = top;
                        lift[1] = (float)g;
                        alpha[e] = kr_exp2(m_c[e] - mu);
#pragma unroll
                        for (int m = 0; m < 2; ++m) { v[m][e] -= mu - mu_c[e]; v[m][e + 2] -= mu - mu_c[e]; }
                        m_c[e] = mn == -INFINITY ? -INFINITY : mu;
                        mu_c[e] = mu;
                        l_c[e] *= alpha[e];
                        z_c[e] *= alpha[e];
                        alpha[e] *= down;
                        mid[e] *= alpha[e];
                        mid[e + 2] *= alpha[e];
                        lim_c[e] = mn == -INFINITY || g > 0 ? -INFINITY : KR_LAZY;
                    }
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int h = 0; h < 2; ++h) st_f[m][h] = __uint_as_float(row_st[m][h].y << 16) * F;
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
                        const float base = __uint_as_float(row_st[m][h].y & 0xffff0000u);
                        const float p0 = kr_exp2(v[m][2 * h]), p1 = kr_exp2(v[m][2 * h + 1]);
                        l_c[0] += p0;
                        l_c[1] += p1;
                        z_c[0] = fmaf(p0, base, z_c[0]);
                        z_c[1] = fmaf(p1, base, z_c[1]);
                        pb[m][h] = kr_trans(kr_half2(p0 * st_f[m][h], p1 * st_f[m][h]));
                    }
                // ---- the middles of the codes times the weights, out of all sums (the same for every element)
                float d_mid[4];
                kr_mma0(d_mid, KR_MID_BYTE, KR_MID_HIGH, KR_MID_BYTE, KR_MID_HIGH, pb[0][0], pb[0][1]);
                kr_mma(d_mid, KR_MID_BYTE, KR_MID_HIGH, KR_MID_BYTE, KR_MID_HIGH, pb[1][0], pb[1][1]);
                const F2 d_even = f2(d_mid[0], d_mid[1]), d_odd = f2(d_mid[2], d_mid[3]);
                auto put = [&](float (&x)[4]) {
                    f2_get(f2_add(f2(x[0], x[1]), d_even), x[0], x[1]);
                    f2_get(f2_add(f2(x[2], x[3]), d_odd), x[2], x[3]);
                };
                put(mid);
#pragma unroll
                for (int mt = 0; mt < D / 16; ++mt) put(o[mt]);
                // ---- O^T += C^T W^T; matrices: keys 0-7 and 8-15 of two neighbouring chunks.  Lane g gets codes 4 g .. 4 g + 3 of keys 2 t, 2 t + 1 of a chunk
                kr_each<2>([&](auto mm) {
                    constexpr int m = mm.value;
                    kr_each<CH / 2>([&](auto cc) {
                        constexpr int c2 = cc.value;
                        unsigned a[4];
                        kr_ldsm_t<16 * m * ROW>((at_v ^ (32 * c2)) + st, a);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const unsigned a_lo = a[2 * h], a_hi = a[2 * h + 1], b_lo = __byte_perm(a_lo, 0u, 0x4341), b_hi = __byte_perm(a_hi, 0u, 0x4341);
                            kr_mma(o[4 * c2 + 2 * h], a_lo & KR_BYTE, a_lo & KR_HIGH, a_hi & KR_BYTE, a_hi & KR_HIGH, pb[m][0], pb[m][1]);
                            kr_mma(o[4 * c2 + 2 * h + 1], b_lo, b_lo & KR_HIGH, b_hi, b_hi & KR_HIGH, pb[m][0], pb[m][1]);
                        }
                    });
                });
                st = st == (ST - 1) * STAGE ? 0 : st + STAGE;
                st_load = st_load == (ST - 1) * STAGE ? 0 : st_load + STAGE;
            }
            // ---- the segment's result, or this warp's part of it
            const KrCursor now = seg;
            const float of = F > 0.f ? 1.f / F : 0.f, of16 = of * 0.0625f;
            constexpr float UP = 16777216.f;              // (by itself: UP / F is beyond float32 for steps above 2^109)
#pragma unroll
            for (int mt = 0; mt < D / 16; ++mt) {         // even elements come with 16 times the odd one behind them
                o[mt][0] = (o[mt][0] - o[mt][2]) * UP; o[mt][1] = (o[mt][1] - o[mt][3]) * UP;
                o[mt][2] *= UP; o[mt][3] *= UP;
            }
            const float even[2] = {(mid[0] - mid[2]) * UP, (mid[1] - mid[3]) * UP}, odd[2] = {mid[2] * UP, mid[3] * UP};
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    l_c[e] += __shfl_xor_sync(0xffffffffu, l_c[e], d);
                    z_c[e] += __shfl_xor_sync(0xffffffffu, z_c[e], d);
                }
            if (begin == now.c0 && end == now.c0 + now.u) {      // all of it: rows 2 t and 2 t + 1, elements 4 g .. 4 g + 3 of every chunk
                const int n = tokens[now.r] * G;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = now.tile * 8 + 2 * t + e;
                    if (row >= n) continue;
                    const int tok = row / G;
                    __nv_bfloat16* dst = p.out + ((size_t)(token[now.r] + tok) * p.n_q + (size_t)now.kvh * G + (row - tok * G)) * D + 4 * g;
                    const float inv = l_c[e] != 0.f ? 1.f / l_c[e] : 0.f, a = of * inv, b = of16 * inv, z0 = fmaf(-even[e], of, z_c[e]) * inv, z1 = fmaf(-odd[e], of16, z_c[e]) * inv;
#pragma unroll
                    for (int c = 0; c < CH; ++c)
                        *reinterpret_cast<uint2*>(dst + 32 * c) = make_uint2(kr_pack(fmaf(o[2 * c][e], a, z0), fmaf(o[2 * c][e + 2], b, z1)),
                                                                             kr_pack(fmaf(o[2 * c + 1][e], a, z0), fmaf(o[2 * c + 1][e + 2], b, z1)));
                }
            } else {
                const int slot = end == hi ? 1 : 0;
                if (slot) { kr_wait<0>(); __syncwarp(); }      // the ring has been read
                float* to = slot ? reinterpret_cast<float*>(kr_sh + (size_t)warp * ST * STAGE) : firsts + warp * 8 * OLD;
#pragma unroll
                for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        *reinterpret_cast<float2*>(to + (2 * t + e) * OLD + (mt >> 1) * 32 + 4 * g + 2 * (mt & 1)) = make_float2(fmaf(o[mt][e], of, fmaf(-even[e], of, z_c[e])), fmaf(o[mt][e + 2], of16, fmaf(-odd[e], of16, z_c[e])));
                if (g == 0)
#pragma unroll
                    for (int e = 0; e < 2; ++e) *reinterpret_cast<float2*>(slot_ml + ((2 * warp + slot) * 8 + 2 * t + e) * 2) = make_float2(m_c[e], l_c[e]);
                if (lane == 0) slot_seg[2 * warp + slot] = pre_s[now.r] + now.s;
            }
            if (end < hi) { ++seg.s; settle(seg); fetch_q(seg); take_q(seg); }
        }
        kr_wait<0>();
    }
    pdl_late();
    __syncthreads();

    // ---- the block's parts of segments, in the order of their keys: neighbours of one segment are a group, added in that order.  A lane knows a slot, and
    // the lane of a group's first slot its segment
    const int of_slot = lane < 2 * NW ? slot_seg[lane] : -1;
    const unsigned there = __ballot_sync(0xffffffffu, of_slot >= 0);
    if (there == 0) { leave(); return; }                  // (all warps see the same)
    const unsigned under = there & ((1u << lane) - 1u);
    const int before = __shfl_sync(0xffffffffu, of_slot, 31 - __clz(under | 1u));
    const bool leads = of_slot >= 0 && (under == 0 || before != of_slot);
    const unsigned starts = __ballot_sync(0xffffffffu, leads);
    int pieces = 0, mine = 0, n_rows = 0, row0 = 0, at_token = 0, at_head = 0;      // blocks that hold parts of the segment, this one among them; its rows
    if (leads) {
        int a = 0, b = p.B;                               // the segment's request
        while (b - a > 1) {
            const int m = (a + b) >> 1;
            if (pre_s[m] <= of_slot) a = m; else b = m;
        }
        const int s = of_slot - pre_s[a], tiles = (tokens[a] * G + 7) >> 3, kvh = s / tiles;
        row0 = (s - kvh * tiles) * 8;
        n_rows = min(8, tokens[a] * G - row0);
        at_token = token[a];
        at_head = kvh * G;
        pieces = sh_all[3];
        mine = sh_mine;
        if (!by_piece) {                                  // the cuts inside are those of c < floor(V i / W) < c + u; part k lies in warp first_cut - 1 + k
            const long long at = pre_u[a] + (long long)s * units[a] + (long long)KR_HEAD * (of_slot + 1);
            const int V = sh_all[0] + KR_HEAD * sh_all[1];
            const int first_cut = (int)(((at + 1) * W + V - 1) / V), last_cut = (int)(((at + units[a]) * W + V - 1) / V) - 1;
            const int b0 = (first_cut - 1) / NW;
            pieces = last_cut / NW - b0 + 1;
            mine = j - b0;
        }
    }
    constexpr int COLS = D / 4;                           // pieces of four elements a row
    int sum_rows = n_rows;                                // rows of the groups before
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, sum_rows, o);
        if (lane >= o) sum_rows += x;
    }
    const int all_rows = __shfl_sync(0xffffffffu, sum_rows, 31);
    sum_rows -= n_rows;
    auto out_row = [&](int lead, int row) -> __nv_bfloat16* {
        const int r = __shfl_sync(0xffffffffu, row0, lead) + row, tok = r / G;
        return p.out + ((size_t)(__shfl_sync(0xffffffffu, at_token, lead) + tok) * p.n_q + (__shfl_sync(0xffffffffu, at_head, lead) + r - tok * G)) * D + 4 * lane;
    };
    for (int task = warp; task < all_rows; task += NW) {  // a row a warp
        const int lead = 31 - __clz(__ballot_sync(0xffffffffu, leads && sum_rows <= task)), row = task - __shfl_sync(0xffffffffu, sum_rows, lead);
        const unsigned above = starts & ~((2u << lead) - 1u), group = there & ~((1u << lead) - 1u) & (above ? (above & (0u - above)) - 1u : 0xffffffffu);
        const bool in = group >> lane & 1u;
        const float2 ml = in ? *reinterpret_cast<const float2*>(slot_ml + (lane * 8 + row) * 2) : make_float2(-INFINITY, 0.f);
        const float M = warp_max(ml.x), Mu = M == -INFINITY ? 0.f : M, f = in ? kr_exp2(ml.x - Mu) : 0.f, L = warp_sum(f * ml.y);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (unsigned rest = group; rest; rest &= rest - 1) {
            const int k = __ffs(rest) - 1;
            const float w = __shfl_sync(0xffffffffu, f, k);
            const float* from = (k & 1 ? reinterpret_cast<const float*>(kr_sh + (size_t)(k >> 1) * ST * STAGE) : firsts + (k >> 1) * 8 * OLD) + row * OLD;
            if (lane < COLS) {
                const float4 x = *reinterpret_cast<const float4*>(from + 4 * lane);
                acc.x = fmaf(w, x.x, acc.x); acc.y = fmaf(w, x.y, acc.y);
                acc.z = fmaf(w, x.z, acc.z); acc.w = fmaf(w, x.w, acc.w);
            }
        }
        __nv_bfloat16* dst = out_row(lead, row);
        const bool alone = __shfl_sync(0xffffffffu, pieces, lead) == 1;
        const int out_slot = 2 * j + (__shfl_sync(0xffffffffu, mine, lead) == 0 ? 1 : 0);
        if (lane >= COLS) continue;
        if (alone) {
            const float inv = L != 0.f ? 1.f / L : 0.f;
            *reinterpret_cast<uint2*>(dst) = make_uint2(kr_pack(acc.x * inv, acc.y * inv), kr_pack(acc.z * inv, acc.w * inv));
        } else {
            *reinterpret_cast<float4*>(p.part_o + ((size_t)out_slot * 8 + row) * D + 4 * lane) = acc;
            if (lane == 0) *reinterpret_cast<float2*>(p.part_ml + ((size_t)out_slot * 8 + row) * 2) = make_float2(M, L);
        }
    }
    // segments that other blocks hold parts of as well: one from before, one that goes on
    const unsigned open = __ballot_sync(0xffffffffu, pieces > 1);
    if (open == 0) { leave(); return; }
    __syncthreads();
    if (warp == 0) {                                      // the fence behind the barrier covers what the block's other threads wrote
        if (pieces > 1) {
            __threadfence();
            sh_last[open & ((1u << lane) - 1u) ? 1 : 0] = atomicAdd(p.count + of_slot, 1) == pieces - 1;
            __threadfence();
        }
    }
    __syncthreads();
#pragma unroll 1
    for (int q = 0; q < __popc(open); ++q) {
        if (!sh_last[q]) continue;                        // the last block of a segment: all parts are there, and are merged in the order of the keys
        const int lead = q == 0 ? __ffs(open) - 1 : 31 - __clz(open);
        const int n = __shfl_sync(0xffffffffu, pieces, lead), b0 = j - __shfl_sync(0xffffffffu, mine, lead), rows = __shfl_sync(0xffffffffu, n_rows, lead);      // b0: the block of part 0
        if (tid == lead) p.count[of_slot] = 0;
        for (int row = warp; row < rows; row += NW) {
            auto at = [&](int k) -> size_t { return (size_t)(2 * (b0 + k) + (k == 0 ? 1 : 0)) * 8 + row; };
            float2 ml = lane < n ? __ldcg(reinterpret_cast<const float2*>(p.part_ml + at(lane) * 2)) : make_float2(-INFINITY, 0.f);
            float M = ml.x;
            for (int k = lane + 32; k < n; k += 32) M = fmaxf(M, __ldcg(p.part_ml + at(k) * 2));
            M = warp_max(M);
            const float Mu = M == -INFINITY ? 0.f : M;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            float L = 0.f;
            for (int k0 = 0; k0 < n; k0 += 32) {
                if (k0 > 0) ml = k0 + lane < n ? __ldcg(reinterpret_cast<const float2*>(p.part_ml + at(k0 + lane) * 2)) : make_float2(-INFINITY, 0.f);
                const float w = kr_exp2(ml.x - Mu);
                L = fmaf(w, ml.y, L);
                const int m = min(n - k0, 32);
#pragma unroll 4
                for (int k = 0; k < m; ++k) {
                    const float f = __shfl_sync(0xffffffffu, w, k);
                    if (lane < COLS) {
                        const float4 x = __ldcg(reinterpret_cast<const float4*>(p.part_o + at(k0 + k) * D + 4 * lane));
                        acc.x = fmaf(f, x.x, acc.x); acc.y = fmaf(f, x.y, acc.y);
                        acc.z = fmaf(f, x.z, acc.z); acc.w = fmaf(f, x.w, acc.w);
                    }
                }
            }
            L = warp_sum(L);
            __nv_bfloat16* dst = out_row(lead, row);
            const float inv = L != 0.f ? 1.f / L : 0.f;
            if (lane < COLS) *reinterpret_cast<uint2*>(dst) = make_uint2(kr_pack(acc.x * inv, acc.y * inv), kr_pack(acc.z * inv, acc.w * inv));
        }
    }
    leave();
}

constexpr int KR_NW = 12, KR_ST = 3;      // warps of a block, units of a warp's ring

// Requests with 1 .. max_q tokens; q_start null: request r has token r.  count: a word for every 8 rows of a request under a kv head, zero before and after.
struct Kv4RunsArgs {
    long long q, out, k, v, steps, q_start, kv_len, block_table, bt_stride, bt_width, part_o, part_ml, count, blocks, B, T, n_q, n_kv, d, page_size, pages, window, max_q, ahead, stream;
    double scale;
};

MSGL_API int msgl_kv4_attention_runs(const Kv4RunsArgs* x) {
    const void *q = (const void*)x->q, *k = (const void*)x->k, *v = (const void*)x->v, *steps = (const void*)x->steps;
    void* out = (void*)x->out;
    const int *q_start = (const int*)x->q_start, *kv_len = (const int*)x->kv_len, *block_table = (const int*)x->block_table;
    float *part_o = (float*)x->part_o, *part_ml = (float*)x->part_ml;
    int* count = (int*)x->count;
    const long long bt_stride = x->bt_stride;
    const int bt_width = (int)x->bt_width, blocks = (int)x->blocks, B = (int)x->B, T = (int)x->T, n_q = (int)x->n_q, n_kv = (int)x->n_kv, d = (int)x->d, page_size = (int)x->page_size,
              pages = (int)x->pages, window = (int)x->window, max_q = (int)x->max_q;
    const float scale = (float)x->scale;
    cudaStream_t stream = (cudaStream_t)x->stream;
    if (B <= 0 || T <= 0) return MSGL_OK;
    if ((d != 64 && d != 128) || B > KR_MAX_B || n_kv < 1 || n_q < 1 || n_q % n_kv || page_size < 1 || pages < 1 || bt_width < 1 || max_q < 1 || blocks < 1 || blocks > 4096 ||
        (long long)bt_width * page_size > 0x3fffffffLL || (long long)pages * n_kv * page_size >= 0xffffffffLL || part_o == nullptr || part_ml == nullptr || count == nullptr)
        return MSGL_ERR_SIZE;
    const long long tiles = ((long long)max_q * (n_q / n_kv) + 7) / 8, most = (long long)B * n_kv * tiles;
    if (most * (((long long)bt_width * page_size + KR_KEYS - 1) / KR_KEYS + KR_HEAD + 1) >= (1LL << 31)) return MSGL_ERR_SIZE;
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k | (uintptr_t)v | (uintptr_t)steps | (uintptr_t)part_o | (uintptr_t)part_ml) & 15) return MSGL_ERR_ALIGN;
    static MsglOncePerDevice attr_set;
#define KR_EACH(DO) DO(64, true) DO(64, false) DO(128, true) DO(128, false)
    if (attr_set.due()) {
#define KR_SET(DD, WW) if (cudaFuncSetAttribute(kv4_attn_runs_kernel<DD, KR_NW, KR_ST, WW>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kr_smem_bytes<DD, KR_NW, KR_ST>()) != cudaSuccess) return msgl_check_launch();
        KR_EACH(KR_SET)
#undef KR_SET
        attr_set.mark();
    }
    Kv4Runs p = {(const __nv_bfloat16*)q, (__nv_bfloat16*)out, (const unsigned char*)k, (const unsigned char*)v, (const uint2*)steps, q_start, kv_len, block_table, part_o,
                 part_ml, count, bt_stride, B, T, n_q, n_kv, page_size, -1, pages, bt_width, window, max_q, (int)x->ahead, scale};
    if ((page_size & (page_size - 1)) == 0) { p.page_shift = 0; while ((1 << p.page_shift) < page_size) ++p.page_shift; }
    const bool whole = page_size >= 16 && p.page_shift >= 0;
#define KR_GO(DD, WW) if (d == DD && whole == WW) msgl_launch_pdl(kv4_attn_runs_kernel<DD, KR_NW, KR_ST, WW>, dim3(blocks), dim3(KR_NW * 32), kr_smem_bytes<DD, KR_NW, KR_ST>(), stream, p);
    KR_EACH(KR_GO)
#undef KR_GO
#undef KR_EACH
    return msgl_check_launch();
}
