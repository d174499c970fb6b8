// A paged key/value cache held in 4 bits: appending to it, reading pages back, attention over it.
//
// A row is one token's key or value under one kv head: d codes c in 0..15, two to a byte (the even element in the low half), and two
// bfloat16 numbers, a step and a base; an element stands for base + c * step, summed in float32 (the product of a 4-bit and an 8-bit
// number is exact).  Arrays: k, v [pages][kv heads][page][d / 2] bytes, steps [pages][kv heads][page][4] = k step, k base, v step, v base.
// 68 bytes a row of 128 where bfloat16 takes 256.
//
// A row x becomes: base = bf16(min x), step = bf16((max x - base) / 15), c = rint((x - base) / step) within 0..15.  Codes are made against
// the step and base as they are kept, so their rounding costs no more than the code's own half step.  The base is the least element (not a
// midpoint), since that is exact for bfloat16 rows.  A row without width (step below 2^-100) has step 0; one with an infinite element or a NaN, or
// wider than bfloat16 reaches, stands for NaN throughout, so that it shows in every result that it enters.
//
//   kv4_append_vec_kernel / kv4_append_kernel   norm, rotation, codes, q            (bound by bytes)
//   kv4_restore_kernel                          rows back to bfloat16 or float32    (bound by bytes)
//   kv4_attn_any_kernel                         attention, any head size and type   (float32 arithmetic)
//   kv4_attn_runs_kernel (kv4_runs.cuh)         attention on mma, bfloat16, head sizes 64 and 128
#include "common.cuh"
#include <float.h>
#include <math_constants.h>

constexpr int KV4_MAX_D = 512;

__device__ __forceinline__ float bf16_of(unsigned short b) { return __uint_as_float((unsigned)b << 16); }

// min and max that keep a NaN
__device__ __forceinline__ float min_nan(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float min_nan(float a, float b, float c) { float r; asm("min.NaN.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }
__device__ __forceinline__ float max_nan(float a, float b, float c) { float r; asm("max.NaN.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }

// pairs of floats in the packed instructions of sm_100 (a product and a sum of it may become one operation, so what has to be rounded apart is not written with these)
typedef unsigned long long F2;
__device__ __forceinline__ F2 f2(float a, float b) { F2 r; asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ F2 f2(float a) { return f2(a, a); }
__device__ __forceinline__ void f2_get(F2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;\n" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ F2 f2_mul(F2 a, F2 b) { F2 r; asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ F2 f2_add(F2 a, F2 b) { F2 r; asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) { F2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }

struct Kv4Scale {
    float base, step, inv;
    unsigned bits;                  // step in the low half, base in the high one, as they are kept
    __device__ __forceinline__ Kv4Scale(float lo, float hi) {
        __nv_bfloat16 b = __float2bfloat16_rn(lo), s = __float2bfloat16_rn(__fmul_rn(__fsub_rn(hi, __bfloat162float(b)), 1.f / 15.f));
        base = __bfloat162float(b);
        step = __bfloat162float(s);
        if (!(fabsf(base) <= FLT_MAX) || !(fabsf(step) <= FLT_MAX)) { base = CUDART_NAN_F; step = 0.f; }
        else if (!(step >= 0x1p-100f)) step = 0.f;
        inv = step > 0.f ? __fdiv_rn(1.f, step) : 0.f;
        bits = (unsigned)__bfloat16_as_ushort(__float2bfloat16_rn(step)) | ((unsigned)__bfloat16_as_ushort(__float2bfloat16_rn(base)) << 16);
    }
    // The codes of eight elements as one word.  A code is the whole number next to the quotient (x - base) / step, an even one where that lies half way between two, so the
    // quotient has to be right to its last bit there: c = rint(y) of y = (x - base) inv leaves the exact remainder r = (x - base) - c step, and c + r inv is the quotient rounded
    // once (but for one in 2^24 of those next to a half, either of whose codes is as near).  Adding 1.5 2^23 rounds to whole numbers and leaves them in the low bits.
    __device__ __forceinline__ unsigned codes(const F2 (&x)[4]) const {
        const F2 whole = f2(12582912.f), minus = f2(-12582912.f), nb = f2(-base), ns = f2(-step), iv = f2(inv);
        unsigned word = 0;
        if (!(step > 0.f)) return 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const F2 d = f2_add(x[i], nb), c = f2_add(f2_add(f2_mul(d, iv), whole), minus), q = f2_fma(f2_fma(c, ns, d), iv, c);
            float a, b;
            f2_get(q, a, b);
            a = fminf(fmaxf(a, 0.f), 15.f);
            b = fminf(fmaxf(b, 0.f), 15.f);
            f2_get(f2_add(f2(a, b), whole), a, b);
            word += ((__float_as_uint(a) - 0x4b400000u) << (8 * i)) + ((__float_as_uint(b) - 0x4b400000u) << (8 * i + 4));
        }
        return word;
    }
};

// x * inv * w and the rotation in separately rounded operations, so that the codes are those of the written formula whichever kernel makes them
__device__ __forceinline__ float rot_sub(float a, float c, float b, float s) { return __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s)); }
__device__ __forceinline__ float rot_add(float a, float s, float b, float c) { return __fadd_rn(__fmul_rn(a, s), __fmul_rn(b, c)); }
// The squares are summed in 64 bits: a code next to a border must not hang on the order of a sum (the same token gives the same row in a step of any make-up).
__device__ __forceinline__ float inv_rms(double ss, int d, float eps) { return __fdiv_rn(1.f, __fsqrt_rn(__fadd_rn((float)(ss / (double)d), eps))); }
template <typename T> __device__ __forceinline__ double square(float x) { return sizeof(T) == 2 ? (double)(x * x) : (double)x * (double)x; }      // (a bfloat16's square is exact in float32)

struct Kv4Append {
    const void* qkv; long long stride;                    // [T] rows of (n_q + 2 n_kv) d elements
    const int* positions; const int* out_loc;
    const void* qw; const void* kw; int w_f32; float eps;
    const float* table; int rot, max_pos, interleaved;
    void* q_out;
    unsigned char* k; unsigned char* v; unsigned* steps;  // steps: two words a row, keys' and values'
    long long slots;                                      // of the cache: page numbers beyond are left out
    int page_size, n_q, n_kv, d, T;
    int early;                                            // the next launch may start while this one waits for the one ahead
    int parts;                                            // parts that a token's heads are dealt out over
    unsigned magic; int less, shift;                      // a quotient by it: (h + ((x - h) >> less)) >> shift with h = x magic >> 32 (Granlund and Montgomery)
    __device__ __forceinline__ long long row_of_slot(int slot, int kvh) const {      // -1: nowhere
        if (slot < 0 || slot >= slots) return -1;
        const int page = slot / page_size;
        return ((long long)page * n_kv + kvh) * page_size + (slot - page * page_size);
    }
};

// Any head size in steps of 8, partial and pairwise rotations: a warp a head of a token.
template <typename T>
__global__ void kv4_append_kernel(const Kv4Append p) {
    extern __shared__ float kv4_sh[];
    const int lane = threadIdx.x & 31, n_heads = p.n_q + 2 * p.n_kv, d = p.d;
    const long long unit = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    float* hv = kv4_sh + (size_t)(threadIdx.x >> 5) * d;
    pdl_wait();
    pdl_small();
    if (unit >= (long long)p.T * n_heads) return;
    const int t = (int)(unit / n_heads), head = (int)(unit - (long long)t * n_heads);
    const bool is_q = head < p.n_q, is_k = !is_q && head < p.n_q + p.n_kv;
    const T* src = reinterpret_cast<const T*>(p.qkv) + (size_t)t * p.stride + (size_t)head * d;
    const void* nw = is_q ? p.qw : (is_k ? p.kw : nullptr);
    double ss = 0.0;
    for (int i = lane; i < d; i += 32) {
        const float x = to_f32<T>(src[i]);
        hv[i] = x;
        ss += square<T>(x);
    }
    if (nw != nullptr) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float inv = inv_rms(ss, d, p.eps);
        for (int i = lane; i < d; i += 32) hv[i] = __fmul_rn(__fmul_rn(hv[i], inv), load_weight(nw, i, p.w_f32));
    }
    __syncwarp();
    const int rot = (is_q || is_k) && p.table != nullptr ? p.rot : 0, half = rot >> 1;
    int pos = rot ? p.positions[t] : 0;
    pos = pos < 0 ? 0 : (pos >= p.max_pos ? p.max_pos - 1 : pos);
    const float* cs = p.table + (size_t)pos * rot;
    auto turned = [&](int i) -> float {
        if (i >= rot) return hv[i];
        if (p.interleaved) {
            const int a = i >> 1;
            return (i & 1) ? rot_add(hv[i - 1], cs[half + a], hv[i], cs[a]) : rot_sub(hv[i], cs[a], hv[i + 1], cs[half + a]);
        }
        return i < half ? rot_sub(hv[i], cs[i], hv[i + half], cs[half + i]) : rot_add(hv[i - half], cs[i], hv[i], cs[i - half]);
    };
    if (is_q) {
        T* dst = reinterpret_cast<T*>(p.q_out) + ((size_t)t * p.n_q + head) * d;
        for (int i = lane; i < d; i += 32) dst[i] = from_f32<T>(turned(i));
        return;
    }
    // eight neighbouring elements a lane: a word of codes
    float x[KV4_MAX_D / 256][8], lo = CUDART_INF_F, hi = -CUDART_INF_F;
#pragma unroll
    for (int j = 0; j < KV4_MAX_D / 256; ++j) {
        const int w = lane + 32 * j;
        if (8 * w >= d) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[j][e] = turned(8 * w + e);
            lo = min_nan(lo, x[j][e]);
            hi = max_nan(hi, x[j][e]);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const Kv4Scale sc(lo, hi);
    const long long row = p.row_of_slot(p.out_loc[t], is_k ? head - p.n_q : head - p.n_q - p.n_kv);
    if (row < 0) return;
    unsigned* dst = reinterpret_cast<unsigned*>((is_k ? p.k : p.v) + row * (d >> 1));
#pragma unroll
    for (int j = 0; j < KV4_MAX_D / 256; ++j) {
        const int w = lane + 32 * j;
        if (8 * w >= d) continue;
        const F2 y[4] = {f2(x[j][0], x[j][1]), f2(x[j][2], x[j][3]), f2(x[j][4], x[j][5]), f2(x[j][6], x[j][7])};
        dst[w] = sc.codes(y);
    }
    if (lane == 0) p.steps[2 * row + (is_k ? 0 : 1)] = sc.bits;
}

// Head sizes 32, 64, 128, 256 whose rotation (if any) covers the whole head in halves: L = d / 16 lanes work on one head of a token, a lane on eight
// elements of the lower half and the eight that they are rotated with, so that every copy is 16 bytes, every word of codes one lane's, and only the sum
// and the extremes take shuffles.  All that a lane reads but the weights is asked for before it works on any of it.
// Bound by its operations and by how few warps wait on memory meanwhile.  Where there is much to do, lanes therefore go through several heads of their token (LOOP): the cosines, the slot and its
// page are looked up once, and the next head is asked for while they work on one.  8,192 tokens of 32 + 8 heads (176 MB, floor 27 us) 40 us, 4.4 TB/s; with one head
// a lane 50.4 (330 instructions a warp of four heads), the 16-bit cache's kernel 46.7; 16,000 tokens 79 and 93.5.  The loop's registers leave 28 warps an SM for 36, so that up to KV4_APPEND_ROUNDS times
// what runs at a time one head a lane is quicker (1,500 tokens 9.9 us and 11.0, 400 3.9 and 5.1; level at 2,500); where all run at once the loop's kernel is again, without its loop (1 token 2.35 and 2.5; 128 2.9;
// the 16-bit cache's kernel 1.5, 2.0).  Blocks of 256 threads 59 (where these took 52), scalar arithmetic and a division an element 65; the next head not asked for ahead 48 (where these took 41).
constexpr int KV4_APPEND_THREADS = 128;
constexpr int KV4_APPEND_ROUNDS = 4;      // one head a lane up to so many times what runs at a time
template <typename T, bool LOOP> constexpr int KV4_APPEND_BLOCKS = !LOOP ? 9 : sizeof(T) == 2 ? 7 : 6;      // an SM: 56, 72 and 80 registers a thread
__device__ __forceinline__ void kv4_weights(const void* w, int at, int f32, F2 (&out)[4]) {      // eight of them, 16 bytes a load
    if (f32) {
        const ulonglong2* p = reinterpret_cast<const ulonglong2*>(reinterpret_cast<const float*>(w) + at);
        const ulonglong2 a = p[0], b = p[1];
        out[0] = a.x; out[1] = a.y; out[2] = b.x; out[3] = b.y;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(w) + at);
        const unsigned y[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = f2(__uint_as_float(y[i] << 16), __uint_as_float(y[i] & 0xffff0000u));
    }
}

// 8 elements of either half of the rotation, asked for
template <typename T, int L>
__device__ __forceinline__ void kv4_append_ask(const T* src, uint4 (&raw)[2][sizeof(T) / 2]) {
    constexpr int V = 16 / sizeof(T);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int k = 0; k < sizeof(T) / 2; ++k) raw[h][k] = *reinterpret_cast<const uint4*>(src + h * 8 * L + k * V);
}
// cosines and sines of the lower half's elements at a position
template <int L>
__device__ __forceinline__ void kv4_append_angles(const Kv4Append& p, int pos, int l, F2 (&ang)[8]) {
    pos = pos < 0 ? 0 : (pos >= p.max_pos ? p.max_pos - 1 : pos);
    const ulonglong2* cs = reinterpret_cast<const ulonglong2*>(p.table + (size_t)pos * (16 * L) + 8 * l);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const ulonglong2 a = cs[(k & 1) + (k >> 1) * (8 * L / 4)];
        ang[2 * k] = a.x;
        ang[2 * k + 1] = a.y;
    }
}
// one head of a token; row_of(kv head): its row in the cache, -1: nowhere
template <typename T, int L, typename Row>
__device__ __forceinline__ void kv4_append_head(const Kv4Append& p, const uint4 (&raw)[2][sizeof(T) / 2], const F2 (&ang)[8], int l, int token, int head, Row row_of) {
    constexpr int d = 16 * L, half = 8 * L, V = 16 / sizeof(T), N = 8 / V;          // elements of a 16-byte piece, pieces of eight elements
    const bool is_q = head < p.n_q, is_k = !is_q && head < p.n_q + p.n_kv, turns = (is_q || is_k) && p.table != nullptr;
    const void* nw = is_q ? p.qw : (is_k ? p.kw : nullptr);
    const unsigned group = (unsigned)(((1ull << L) - 1) << (threadIdx.x & 31 & ~(L - 1)));
    F2 x[8];                                              // the lower half's elements and the upper half's
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if constexpr (sizeof(T) == 4) {
            const F2* e = reinterpret_cast<const F2*>(&raw[h][0]);
#pragma unroll
            for (int k = 0; k < 4; ++k) x[4 * h + k] = e[k];
        } else {
            const unsigned y[4] = {raw[h][0].x, raw[h][0].y, raw[h][0].z, raw[h][0].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) x[4 * h + k] = f2(__uint_as_float(y[k] << 16), __uint_as_float(y[k] & 0xffff0000u));
        }
    }
    if (nw != nullptr) {
        double ss = 0.0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float a, b;
            f2_get(sizeof(T) == 2 ? f2_mul(x[k], x[k]) : x[k], a, b);      // (a bfloat16's square is exact in float32)
            ss += sizeof(T) == 2 ? (double)a : (double)a * (double)a;
            ss += sizeof(T) == 2 ? (double)b : (double)b * (double)b;
        }
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(group, ss, o);
        const F2 inv = f2(inv_rms(ss, d, p.eps));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            F2 w[4];
            kv4_weights(nw, h * half + 8 * l, p.w_f32, w);
#pragma unroll
            for (int k = 0; k < 4; ++k) x[4 * h + k] = f2_mul(f2_mul(x[4 * h + k], inv), w[k]);
        }
    }
    if (turns) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const F2 a = x[k], b = x[4 + k], c = ang[k], s = ang[4 + k];
            float ac[2], bs[2], as[2], bc[2];             // (sums one by one: packed sums of packed products are contracted)
            f2_get(f2_mul(a, c), ac[0], ac[1]);
            f2_get(f2_mul(b, s), bs[0], bs[1]);
            f2_get(f2_mul(a, s), as[0], as[1]);
            f2_get(f2_mul(b, c), bc[0], bc[1]);
            x[k] = f2(__fsub_rn(ac[0], bs[0]), __fsub_rn(ac[1], bs[1]));
            x[4 + k] = f2(__fadd_rn(as[0], bc[0]), __fadd_rn(as[1], bc[1]));
        }
    }
    if (is_q) {
        T* dst = reinterpret_cast<T*>(p.q_out) + ((size_t)token * p.n_q + head) * d + 8 * l;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int k = 0; k < N; ++k) {
                uint4 out;
                T* e = reinterpret_cast<T*>(&out);
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    float a, b;
                    f2_get(x[4 * h + k * (V / 2) + j], a, b);
                    e[2 * j] = from_f32<T>(a);
                    e[2 * j + 1] = from_f32<T>(b);
                }
                *reinterpret_cast<uint4*>(dst + h * half + k * V) = out;
            }
        return;
    }
    float lo, hi;
    f2_get(x[0], lo, hi);
    {
        const float a = lo, b = hi;
        lo = min_nan(a, b);
        hi = max_nan(a, b);
    }
#pragma unroll
    for (int k = 1; k < 8; ++k) {
        float a, b;
        f2_get(x[k], a, b);
        lo = min_nan(lo, a, b);
        hi = max_nan(hi, a, b);
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) {
        lo = min_nan(lo, __shfl_xor_sync(group, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(group, hi, o));
    }
    const Kv4Scale sc(lo, hi);
    const long long row = row_of(is_k ? head - p.n_q : head - p.n_q - p.n_kv);
    if (row < 0) return;
    unsigned* dst = reinterpret_cast<unsigned*>((is_k ? p.k : p.v) + row * (d / 2)) + l;
    const F2 x0[4] = {x[0], x[1], x[2], x[3]}, x1[4] = {x[4], x[5], x[6], x[7]};
    dst[0] = sc.codes(x0);
    dst[L] = sc.codes(x1);
    if (l == 0) p.steps[2 * row + (is_k ? 0 : 1)] = sc.bits;
}

// L lanes take every `parts`-th head of a token; LOOP: that may be several
template <typename T, int L, bool LOOP>
__global__ void __launch_bounds__(KV4_APPEND_THREADS, KV4_APPEND_BLOCKS<T, LOOP>) kv4_append_vec_kernel(const Kv4Append p) {
    const int l = threadIdx.x & (L - 1), n_heads = p.n_q + 2 * p.n_kv;
    const unsigned group = blockIdx.x * (KV4_APPEND_THREADS / L) + threadIdx.x / L;
    const unsigned high = __umulhi(group, p.magic);
    const int token = (int)((high + ((group - high) >> p.less)) >> p.shift);
    int head = (int)(group - (unsigned)token * p.parts);
    if (p.early) pdl_small();
    pdl_wait();
    if (!p.early) pdl_small();
    if (token >= p.T) return;
    const bool turns = p.table != nullptr && head < p.n_q + p.n_kv, stores = head >= p.n_q || p.parts < n_heads;
    const int pos = turns ? p.positions[token] : 0, slot = stores ? p.out_loc[token] : 0;
    const T* src = reinterpret_cast<const T*>(p.qkv) + (size_t)token * p.stride + (size_t)head * (16 * L) + 8 * l;
    uint4 raw[2][sizeof(T) / 2];
    kv4_append_ask<T, L>(src, raw);
    F2 ang[8];
    if (turns) kv4_append_angles<L>(p, pos, l, ang);
    if (!LOOP) {
        kv4_append_head<T, L>(p, raw, ang, l, token, head, [&](int kvh) { return p.row_of_slot(slot, kvh); });
        return;
    }
    const long long row0 = stores ? p.row_of_slot(slot, 0) : -1;
    auto row_of = [&](int kvh) { return row0 < 0 ? -1 : row0 + (long long)kvh * p.page_size; };
    if (p.parts == n_heads) {
        kv4_append_head<T, L>(p, raw, ang, l, token, head, row_of);
        return;
    }
    while (true) {
        uint4 next[2][sizeof(T) / 2];
        src += (size_t)p.parts * (16 * L);
        if (head + p.parts < n_heads) kv4_append_ask<T, L>(src, next);
        kv4_append_head<T, L>(p, raw, ang, l, token, head, row_of);
        head += p.parts;
        if (head >= n_heads) return;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int k = 0; k < sizeof(T) / 2; ++k) raw[h][k] = next[h][k];
    }
}

// The entry points take their arguments in one piece, 8 bytes each in the order of these structs.
struct Kv4AppendArgs {
    long long qkv, stride, positions, out_loc, qw, kw, w_f32, table, rot, max_pos, interleaved, q_out, k, v, steps, slots, page_size, n_q, n_kv, d, T, dtype, early, stream;
    double eps;
};

MSGL_API int msgl_kv4_append(const Kv4AppendArgs* x) {
    const long long stride = x->stride, slots = x->slots;
    const void *qkv = (const void*)x->qkv, *qw = (const void*)x->qw, *kw = (const void*)x->kw, *k = (const void*)x->k, *v = (const void*)x->v, *steps = (const void*)x->steps;
    const int *positions = (const int*)x->positions, *out_loc = (const int*)x->out_loc;
    const float* table = (const float*)x->table;
    void* q_out = (void*)x->q_out;
    const int w_f32 = (int)x->w_f32, rot = (int)x->rot, max_pos = (int)x->max_pos, interleaved = (int)x->interleaved, page_size = (int)x->page_size, n_q = (int)x->n_q, n_kv = (int)x->n_kv,
              d = (int)x->d, T = (int)x->T, dtype = (int)x->dtype;
    const float eps = (float)x->eps;
    cudaStream_t stream = (cudaStream_t)x->stream;
    if (T <= 0) return MSGL_OK;
    if (d < 8 || d > KV4_MAX_D || d % 8 || n_q < 0 || n_kv < 1 || page_size < 1 || rot > d || (rot & 1)) return MSGL_ERR_SIZE;
    if (dtype != MSGL_F32 && dtype != MSGL_BF16) return MSGL_ERR_DTYPE;
    if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)steps) & 15) return MSGL_ERR_ALIGN;
    Kv4Append p = {qkv, stride, positions, out_loc, qw, kw, w_f32, eps, table, rot, max_pos, interleaved, q_out, (unsigned char*)k, (unsigned char*)v, (unsigned*)steps,
                   slots, page_size, n_q, n_kv, d, T, (int)x->early, n_q + 2 * n_kv, 0u, 0, 0};
    const int n_heads = n_q + 2 * n_kv;
    const long long units = (long long)T * n_heads;
    const int item = dtype == MSGL_F32 ? 4 : 2;
    const bool whole = table == nullptr || (rot == d && !interleaved && ((uintptr_t)table & 15) == 0);
    if (whole && (d == 32 || d == 64 || d == 128 || d == 256) && (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)qw | (uintptr_t)kw) & 15) == 0 && (stride * item) % 16 == 0) {
        const int L = d / 16, per = KV4_APPEND_THREADS / L;
        if (units > 0x7fffffffLL) return MSGL_ERR_SIZE;
        const long long sms = msgl_sm_count(), at_a_time = sms * (dtype == MSGL_F32 ? KV4_APPEND_BLOCKS<float, true> : KV4_APPEND_BLOCKS<__nv_bfloat16, true>) * per;
        const bool much = units > sms * KV4_APPEND_BLOCKS<float, false> * per * KV4_APPEND_ROUNDS, loop = much || units <= at_a_time / 2;
        if (much) {          // the number of parts with the least rounds of them times heads of a part (starting a part costs 0.8 of a head's time)
            double least = 1e300;
            for (int c = n_heads; c >= 1; --c) {
                const double cost = (double)((T * (long long)c + at_a_time - 1) / at_a_time) * ((n_heads + c - 1) / c + 0.8);
                if (cost < least) { least = cost; p.parts = c; }
            }
        }
        if (p.parts > 1) {
            p.less = 1;
            while ((2ull << p.shift) < (unsigned)p.parts) ++p.shift;      // 2^(shift + 1) is the power of two from p.parts on
            p.magic = (unsigned)((((2ull << p.shift) - p.parts) << 32) / p.parts + 1);
        }
        const long long blocks = ((long long)T * p.parts + per - 1) / per;
#define KV4_VEC(TT, LL) msgl_launch_pdl(loop ? kv4_append_vec_kernel<TT, LL, true> : kv4_append_vec_kernel<TT, LL, false>, dim3((unsigned)blocks), dim3(KV4_APPEND_THREADS), 0, stream, p)
#define KV4_VEC_L(TT) do { if (L == 2) KV4_VEC(TT, 2); else if (L == 4) KV4_VEC(TT, 4); else if (L == 8) KV4_VEC(TT, 8); else KV4_VEC(TT, 16); } while (0)
        if (dtype == MSGL_F32) KV4_VEC_L(float); else KV4_VEC_L(__nv_bfloat16);
#undef KV4_VEC_L
#undef KV4_VEC
        return msgl_check_launch();
    }
    constexpr int WARPS = 4;
    const long long blocks = (units + WARPS - 1) / WARPS;
    if (blocks > 0x7fffffffLL) return MSGL_ERR_SIZE;
    const size_t smem = (size_t)WARPS * d * 4;
    if (dtype == MSGL_F32) msgl_launch_pdl(kv4_append_kernel<float>, dim3((unsigned)blocks), dim3(WARPS * 32), smem, stream, p);
    else msgl_launch_pdl(kv4_append_kernel<__nv_bfloat16>, dim3((unsigned)blocks), dim3(WARPS * 32), smem, stream, p);
    return msgl_check_launch();
}

// ---------------------------------------------------------------------------------------------------------------------------------------------
// Rows back to bfloat16 or float32.
//
// Two uses.  By pages: pages[i] of the cache becomes page i of the results, [n][kv heads][page][d].  By requests: the keys that the requests with
// at least min_q tokens see are packed into pages of KV4_RESTORED keys, request after request, and `table` names those pages as a block table does
// (the tensor-core prefill kernel then fetches whole tiles of keys; a key's place in its page is that of its position).  Keys behind a request's
// last one are zeros.  A value row that is no number, or reaches beyond them, becomes a key row that is none beside values of 0: it then shows through the scores of those who see it, where as a value it would
// meet the weights of 0 that others have for it as well.  bfloat16 results are rounded once, as a bfloat16 cache would hold them.  8,192 keys of 8 heads (42 MB) 8.8 us, 4.8 TB/s.
constexpr int KV4_RESTORED = 128;

struct Kv4Restore {
    const unsigned char* k; const unsigned char* v; const uint2* steps;
    void* k_out; void* v_out;
    const int* pages_in;             // by pages: [n]
    const int* q_start; const int* kv_len; const int* block_table; int* table;      // by requests: [B + 1], [B], [B, bt_width], [B, t_width]
    long long bt_stride;
    int B, bt_width, t_width, window, min_q, n_kv, page_size, pages, d, n;        // n: pages of results
    int word_shift, page_shift;      // of powers of two, else -1
};

// what a request needs restored: its pages of KV4_RESTORED keys from the first one that its first token sees on
__device__ __forceinline__ void kv4_span(const Kv4Restore& p, int r, int& first, int& n) {
    const int tokens = p.q_start[r + 1] - p.q_start[r], kv = min(p.kv_len[r], p.bt_width * p.page_size);
    first = n = 0;
    if (tokens < p.min_q || kv <= 0) return;
    first = (p.window > 0 ? max(p.kv_len[r] - tokens - p.window + 1, 0) : 0) / KV4_RESTORED;
    n = max(min((kv + KV4_RESTORED - 1) / KV4_RESTORED, p.t_width) - first, 0);
}

template <bool WIDE>
__device__ __forceinline__ void kv4_put(void* out, long long at, unsigned word, float step, float base) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf((float)((word >> (4 * e)) & 15u), step, base);
    if (WIDE) {
        float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + at);
        o[0] = make_float4(x[0], x[1], x[2], x[3]);
        o[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        uint4 o;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&o);
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
        *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(out) + at) = o;
    }
}

// a block: a page of results under one kv head; by requests one more along x, which writes the table
template <bool WIDE>
__global__ void __launch_bounds__(256) kv4_restore_kernel(const Kv4Restore p) {
    __shared__ int sh[2];
    const int kvh = blockIdx.y, words = p.d >> 3;
    pdl_wait();
    pdl_small();
    if ((int)blockIdx.x == p.n) {
        if (kvh > 0) return;
        int before = 0;
        for (int r = 0; r < p.B; ++r) {                   // whatever the lengths say, every entry names a page of the results
            int first, n;
            kv4_span(p, r, first, n);
            for (int i = threadIdx.x; i < p.t_width; i += 256) p.table[(long long)r * p.t_width + i] = min(max(before + i - first, 0), p.n - 1);
            before += n;
        }
        return;
    }
    const int* pages = p.pages_in;
    int from = 0, rows = p.page_size, per = p.page_size, width = 0x7fffffff;      // by pages: one page, all of its rows
    long long to = (long long)blockIdx.x;
    if (pages != nullptr) {
        pages += blockIdx.x;
    } else {
        // the request that result page blockIdx.x is of: a warp looks through the requests, 32 at a time
        if (threadIdx.x < 32) {
            int before = 0, r = -1, page = 0;
            for (int r0 = 0; r0 < p.B; r0 += 32) {
                int first = 0, n = 0;
                if (r0 + (int)threadIdx.x < p.B) kv4_span(p, r0 + threadIdx.x, first, n);
                int sum = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int u = __shfl_up_sync(0xffffffffu, sum, o);
                    if ((int)threadIdx.x >= o) sum += u;
                }
                const int at = (int)blockIdx.x - before - (sum - n);
                const unsigned hit = __ballot_sync(0xffffffffu, at >= 0 && at < n);
                if (hit) {
                    const int src = __ffs(hit) - 1;
                    page = __shfl_sync(0xffffffffu, first + at, src);
                    r = r0 + src;
                    break;
                }
                before += __shfl_sync(0xffffffffu, sum, 31);
            }
            if (threadIdx.x == 0) { sh[0] = r; sh[1] = page; }
        }
        __syncthreads();
        const int r = sh[0];
        if (r < 0) return;
        pages = p.block_table + r * p.bt_stride;
        width = p.bt_width;
        from = sh[1] * KV4_RESTORED;
        rows = min(p.kv_len[r] - from, KV4_RESTORED);
        per = KV4_RESTORED;
    }
    to = (to * p.n_kv + kvh) * per * p.d;
    // (a word of keys and one of values a thread: with four of each asked for ahead, 8,192 keys under 8 heads take 13.4 us instead of 8.7)
    for (int i = threadIdx.x; i < per * words; i += 256) {
        const int row = p.word_shift >= 0 ? i >> p.word_shift : i / words, w = i - row * words;
        const int key = from + row, at = p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size;
        const int page = row < rows && at < width ? pages[at] : -1;
        unsigned kw = 0, vw = 0;
        uint2 st = make_uint2(0u, 0u);
        if (page >= 0 && page < p.pages) {
            const long long src = ((long long)page * p.n_kv + kvh) * p.page_size + (key - at * p.page_size);
            kw = reinterpret_cast<const unsigned*>(p.k)[src * words + w];
            vw = reinterpret_cast<const unsigned*>(p.v)[src * words + w];
            st = p.steps[src];
            const float base = bf16_of(st.y >> 16);
            if (p.pages_in == nullptr && !(fabsf(base) <= FLT_MAX && fmaf(15.f, bf16_of(st.y & 0xffffu), base) < 0x1.ffp127f)) {      // (from there on bfloat16 has infinities)
                kw = vw = 0;
                st = make_uint2(0x7fc00000u, 0u);
            }
        }
        kv4_put<WIDE>(p.k_out, to + 8ll * i, kw, bf16_of(st.x & 0xffffu), bf16_of(st.x >> 16));
        kv4_put<WIDE>(p.v_out, to + 8ll * i, vw, bf16_of(st.y & 0xffffu), bf16_of(st.y >> 16));
    }
}

static int kv4_shift(int n) {
    int s = 0;
    while ((1 << s) < n) ++s;
    return (1 << s) == n ? s : -1;
}

MSGL_API int msgl_kv4_restored_page(void) { return KV4_RESTORED; }

// n: pages of results.  pages_in null: by requests.
struct Kv4RestoreArgs {
    long long k, v, steps, k_out, v_out, pages_in, n, q_start, kv_len, block_table, bt_stride, bt_width, table, t_width, B, window, min_q, n_kv, page_size, pages, d, dtype, stream;
};

MSGL_API int msgl_kv4_restore(const Kv4RestoreArgs* x) {
    const void *k = (const void*)x->k, *v = (const void*)x->v, *steps = (const void*)x->steps;
    void *k_out = (void*)x->k_out, *v_out = (void*)x->v_out;
    const int *pages_in = (const int*)x->pages_in, *q_start = (const int*)x->q_start, *kv_len = (const int*)x->kv_len, *block_table = (const int*)x->block_table;
    int* table = (int*)x->table;
    const long long bt_stride = x->bt_stride;
    const int n = (int)x->n, bt_width = (int)x->bt_width, t_width = (int)x->t_width, B = (int)x->B, window = (int)x->window, min_q = (int)x->min_q, n_kv = (int)x->n_kv,
              page_size = (int)x->page_size, pages = (int)x->pages, d = (int)x->d, dtype = (int)x->dtype;
    cudaStream_t stream = (cudaStream_t)x->stream;
    if (n <= 0) return MSGL_OK;
    if (d < 8 || d > KV4_MAX_D || d % 8 || n_kv < 1 || n_kv > 65535 || page_size < 1 || pages < 1) return MSGL_ERR_SIZE;
    if (dtype != MSGL_F32 && dtype != MSGL_BF16) return MSGL_ERR_DTYPE;
    if (pages_in != nullptr && (long long)page_size * (d >> 3) >= 1LL << 30) return MSGL_ERR_SIZE;
    if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)steps | (uintptr_t)k_out | (uintptr_t)v_out) & 15) return MSGL_ERR_ALIGN;
    if (pages_in == nullptr && (q_start == nullptr || kv_len == nullptr || block_table == nullptr || table == nullptr || B < 1 || t_width < 1)) return MSGL_ERR_SIZE;
    Kv4Restore p = {(const unsigned char*)k, (const unsigned char*)v, (const uint2*)steps, k_out, v_out, pages_in, q_start, kv_len, block_table, table, bt_stride, B, bt_width,
                    t_width, window, min_q, n_kv, page_size, pages, d, n, kv4_shift(d >> 3), kv4_shift(page_size)};
    const int blocks = pages_in == nullptr ? n + 1 : n;
    if (dtype == MSGL_F32) msgl_launch_pdl(kv4_restore_kernel<true>, dim3(blocks, n_kv), dim3(256), 0, stream, p);
    else msgl_launch_pdl(kv4_restore_kernel<false>, dim3(blocks, n_kv), dim3(256), 0, stream, p);
    return msgl_check_launch();
}

// ---------------------------------------------------------------------------------------------------------------------------------------------
// Attention of requests with few tokens, any head size in steps of 8 and either type, float32 arithmetic throughout.
//
// A block: up to 8 rows (token, query head; 2 or 4 where no request has more) of one kv head and one of `splits` equal parts of the request's keys; four warps take units of 32 keys in
// turn.  A lane owns a key for the scores (its row's words one after the other, the queries broadcast from shared memory) and words of eight
// elements for the values (where a row has 16 words or fewer, lanes stand on several keys side by side).  The warps' results meet in shared memory;
// with several splits they are left as partial results for kv4_join_kernel.  Latency decides: 4 requests of up to 1,500 keys, 16 heads on 8, float32, 17 us with the join (blocks of 8
// rows for the 2 that there are: 36).
constexpr int KV4_ANY_WARPS = 4;

struct Kv4Attn {
    const void* q; void* out;
    const unsigned char* k; const unsigned char* v; const uint2* steps;
    const int* q_start; const int* kv_len; const int* block_table;
    float* part;                     // splits > 1: [splits][T * n_q][d + 2]
    long long bt_stride, part_rows;
    int B, T, n_q, n_kv, d, page_size, pages, bt_width, window, max_q, splits, tiles_q, rows;      // tiles_q: blocks of `rows` rows a request and kv head
    float scale;
};

template <typename T, int WPL, int R>       // WPL: words of a value row a lane; R: rows of a block
__global__ void __launch_bounds__(KV4_ANY_WARPS * 32) kv4_attn_any_kernel(const Kv4Attn p) {
    extern __shared__ float any_sh[];
    constexpr int NW = KV4_ANY_WARPS;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, d = p.d, words = d >> 3, G = p.n_q / p.n_kv;
    float* qs = any_sh;                                  // [R][d]
    float* ps = qs + R * d;                              // [NW][R][32]
    float* os = ps + NW * R * 32;                        // [NW][R][d]
    float* ms = os + NW * R * d;                         // [NW][R][2]
    pdl_wait();
    pdl_small();
    const int tile = blockIdx.x % p.tiles_q, rest = blockIdx.x / p.tiles_q, kvh = rest % p.n_kv, req = rest / p.n_kv;
    const int tok0 = p.q_start != nullptr ? p.q_start[req] : req, n_tok = p.q_start != nullptr ? p.q_start[req + 1] - tok0 : 1;
    const int row0 = tile * R, n_rows = min(R, n_tok * G - row0);
    if (n_tok < 1 || n_tok > p.max_q || n_rows <= 0 || tok0 < 0 || tok0 + n_tok > p.T) return;
    const int kv = min(p.kv_len[req], p.bt_width * p.page_size), pos0 = p.kv_len[req] - n_tok;
    auto row_at = [&](int r) -> long long { return (long long)(tok0 + (row0 + r) / G) * p.n_q + kvh * G + (row0 + r) % G; };
    for (int i = tid; i < R * d; i += NW * 32) qs[i] = i / d < n_rows ? to_f32<T>(reinterpret_cast<const T*>(p.q)[row_at(i / d) * d + i % d]) : 0.f;
    __syncthreads();
    // this block's keys
    const int k_first = p.window > 0 ? max(pos0 + row0 / G - p.window + 1, 0) : 0;
    const int u0 = k_first >> 5, u1 = max((min(kv, pos0 + (row0 + n_rows - 1) / G + 1) + 31) >> 5, u0);
    const int a = u0 + (int)((long long)(u1 - u0) * blockIdx.y / p.splits), b = u0 + (int)((long long)(u1 - u0) * (blockIdx.y + 1) / p.splits);
    const float sc = p.scale * 1.4426950408889634f;
    int wp = 1;                                          // lanes that stand on one value row
    while (wp < words && wp < 32) wp <<= 1;
    const int sub = lane / wp, subs = 32 / wp, my = lane - sub * wp;
    float m[R], l[R], acc[R][8 * WPL];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY; l[r] = 0.f;
#pragma unroll
        for (int e = 0; e < 8 * WPL; ++e) acc[r][e] = 0.f;
    }
    float* pw = ps + warp * R * 32;
    for (int u = a + warp; u < b; u += NW) {
        const int key = 32 * u + lane;
        long long src = -1;
        if (key < kv) {
            const int at = key / p.page_size, page = p.block_table[req * p.bt_stride + at];
            if (page >= 0 && page < p.pages) src = ((long long)page * p.n_kv + kvh) * p.page_size + (key - at * p.page_size);
        }
        const uint2 st = src >= 0 ? p.steps[src] : make_uint2(0u, 0u);
        const float ks = bf16_of(st.x & 0xffffu), kb = bf16_of(st.x >> 16);
        const float none = (st.y & 0x7f800000u) == 0x7f800000u || (st.y & 0x7f80u) == 0x7f80u ? CUDART_NAN_F : 0.f;      // a value row that is no number: its score is none, whatever its weight
        float s[R];
#pragma unroll
        for (int r = 0; r < R; ++r) s[r] = none;
        const unsigned* k_row = reinterpret_cast<const unsigned*>(p.k) + (src >= 0 ? src : 0ll) * words;      // (a key that is not there: step and base 0)
#pragma unroll 8
        for (int w = 0; w < words; ++w) {
            const unsigned word = k_row[w];
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = fmaf((float)((word >> (4 * e)) & 15u), ks, kb);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float4 q0 = *reinterpret_cast<const float4*>(qs + r * d + 8 * w), q1 = *reinterpret_cast<const float4*>(qs + r * d + 8 * w + 4);
                s[r] = fmaf(q0.x, x[0], fmaf(q0.y, x[1], fmaf(q0.z, x[2], fmaf(q0.w, x[3], s[r]))));
                s[r] = fmaf(q1.x, x[4], fmaf(q1.y, x[5], fmaf(q1.z, x[6], fmaf(q1.w, x[7], s[r]))));
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int pos = pos0 + (row0 + r) / G;
            const bool seen = r < n_rows && key < kv && key <= pos && (p.window <= 0 || key > pos - p.window);
            const float v = seen ? s[r] * sc : -INFINITY;
            const float mn = fmaxf(m[r], warp_max(v)), mu = mn == -INFINITY ? 0.f : mn;
            const float e = seen ? exp2f(v - mu) : 0.f, f = exp2f(m[r] - mu);
            m[r] = mn;
            l[r] = fmaf(l[r], f, e);
            pw[r * 32 + lane] = e;
#pragma unroll
            for (int c = 0; c < 8 * WPL; ++c) acc[r][c] *= f;
        }
        __syncwarp();
#pragma unroll 4
        for (int j = sub; j < 32; j += subs) {
            const long long vs = __shfl_sync(0xffffffffu, src, j);
            const unsigned sy = __shfl_sync(0xffffffffu, st.y, j);
            const float step = bf16_of(sy & 0xffffu), base = bf16_of(sy >> 16);      // (0 where the key is not there)
#pragma unroll
            for (int w2 = 0; w2 < WPL; ++w2) {
                const int w = my + 32 * w2;
                const unsigned word = reinterpret_cast<const unsigned*>(p.v)[(vs >= 0 ? vs : 0ll) * words + min(w, words - 1)];
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = fmaf((float)((word >> (4 * e)) & 15u), step, base);
                const bool number = fabsf(base) <= FLT_MAX && fmaf(15.f, step, base) <= FLT_MAX;      // (a row that is no number counts only where it is seen)
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float pr = pw[r * 32 + j];
                    if (number || pr != 0.f)
#pragma unroll
                        for (int e = 0; e < 8; ++e) acc[r][8 * w2 + e] = fmaf(pr, x[e], acc[r][8 * w2 + e]);
                }
            }
        }
        __syncwarp();
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        l[r] = warp_sum(l[r]);
        for (int o = wp; o < 32; o <<= 1)
#pragma unroll
            for (int c = 0; c < 8 * WPL; ++c) acc[r][c] += __shfl_xor_sync(0xffffffffu, acc[r][c], o);
        if (sub == 0)
#pragma unroll
            for (int w2 = 0; w2 < WPL; ++w2)
                if (my + 32 * w2 < words)
#pragma unroll
                    for (int e = 0; e < 8; ++e) os[(warp * R + r) * d + 8 * (my + 32 * w2) + e] = acc[r][8 * w2 + e];
        if (lane == 0) { ms[(warp * R + r) * 2] = m[r]; ms[(warp * R + r) * 2 + 1] = l[r]; }
    }
    __syncthreads();
    for (int i = tid; i < n_rows * d; i += NW * 32) {
        const int r = i / d, c = i - r * d;
        float M = -INFINITY, L = 0.f, o = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, ms[(w * R + r) * 2]);
        const float mu = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = exp2f(ms[(w * R + r) * 2] - mu);
            L = fmaf(f, ms[(w * R + r) * 2 + 1], L);
            o = fmaf(f, os[(w * R + r) * d + c], o);
        }
        if (p.splits == 1) {
            reinterpret_cast<T*>(p.out)[row_at(r) * d + c] = from_f32<T>(L != 0.f ? o / L : 0.f);
        } else {
            float* part = p.part + (blockIdx.y * p.part_rows + row_at(r)) * (d + 2);
            part[c] = o;
            if (c == 0) { part[d] = M; part[d + 1] = L; }
        }
    }
}

// the rows of the requests taken, from their partial results: a warp 32 elements of a row
template <typename T>
__global__ void __launch_bounds__(128) kv4_join_kernel(const Kv4Attn p) {
    pdl_wait();
    pdl_small();
    const int lane = threadIdx.x & 31, G = p.n_q / p.n_kv, R = p.rows, d = p.d;
    const int tile = blockIdx.x % p.tiles_q, rest = blockIdx.x / p.tiles_q, kvh = rest % p.n_kv, req = rest / p.n_kv;
    const int tok0 = p.q_start != nullptr ? p.q_start[req] : req, n_tok = p.q_start != nullptr ? p.q_start[req + 1] - tok0 : 1;
    if (n_tok < 1 || n_tok > p.max_q || tok0 < 0 || tok0 + n_tok > p.T) return;
    for (int r = tile * R + (threadIdx.x >> 5); r < min(n_tok * G, (tile + 1) * R); r += 4) {
        const long long row = (long long)(tok0 + r / G) * p.n_q + kvh * G + r % G;
        // lane s knows the weights of splits s and s + 32
        const float* first = p.part + row * (d + 2);
        const long long next = p.part_rows * (d + 2);
        const float m0 = lane < p.splits ? first[lane * next + d] : -INFINITY, m1 = lane + 32 < p.splits ? first[(lane + 32) * next + d] : -INFINITY;
        const float l0 = lane < p.splits ? first[lane * next + d + 1] : 0.f, l1 = lane + 32 < p.splits ? first[(lane + 32) * next + d + 1] : 0.f;
        const float M = warp_max(fmaxf(m0, m1)), mu = M == -INFINITY ? 0.f : M, w0 = exp2f(m0 - mu), w1 = exp2f(m1 - mu), L = warp_sum(fmaf(w0, l0, w1 * l1));
        const int c0 = blockIdx.y * 32, c = min(c0 + lane, d - 1);
        float o = 0.f;
#pragma unroll 8
        for (int s = 0; s < p.splits; ++s) o = fmaf(__shfl_sync(0xffffffffu, s < 32 ? w0 : w1, s & 31), first[s * next + c], o);
        if (c0 + lane < d) reinterpret_cast<T*>(p.out)[row * d + c] = from_f32<T>(L != 0.f ? o / L : 0.f);
    }
}

// q_start null: request r has token r.  Requests with 1 .. max_q tokens are taken, the others' rows left alone.
struct Kv4AnyArgs {
    long long q, out, k, v, steps, q_start, kv_len, block_table, bt_stride, bt_width, part, splits, B, T, n_q, n_kv, d, page_size, pages, window, max_q, dtype, stream;
    double scale;
};

MSGL_API int msgl_kv4_attention_any(const Kv4AnyArgs* x) {
    const void *q = (const void*)x->q, *k = (const void*)x->k, *v = (const void*)x->v, *steps = (const void*)x->steps;
    void* out = (void*)x->out;
    const int *q_start = (const int*)x->q_start, *kv_len = (const int*)x->kv_len, *block_table = (const int*)x->block_table;
    float* part = (float*)x->part;
    const long long bt_stride = x->bt_stride;
    const int bt_width = (int)x->bt_width, splits = (int)x->splits, B = (int)x->B, T = (int)x->T, n_q = (int)x->n_q, n_kv = (int)x->n_kv, d = (int)x->d, page_size = (int)x->page_size,
              pages = (int)x->pages, window = (int)x->window, max_q = (int)x->max_q, dtype = (int)x->dtype;
    const float scale = (float)x->scale;
    cudaStream_t stream = (cudaStream_t)x->stream;
    if (B <= 0 || T <= 0) return MSGL_OK;
    if (d < 8 || d > KV4_MAX_D || d % 8 || n_kv < 1 || n_q < 1 || n_q % n_kv || page_size < 1 || pages < 1 || bt_width < 1 || max_q < 1 || splits < 1 || splits > 64 ||
        (long long)bt_width * page_size > 0x7fffffffLL - 64)
        return MSGL_ERR_SIZE;
    if (dtype != MSGL_F32 && dtype != MSGL_BF16) return MSGL_ERR_DTYPE;
    if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)steps) & 15) return MSGL_ERR_ALIGN;
    const long long most_rows = (long long)max_q * (n_q / n_kv);
    const int wpl = d > 256 ? 2 : 1, R = wpl == 2 || most_rows > 4 ? 8 : most_rows > 2 ? 4 : 2, tiles_q = (int)((most_rows + R - 1) / R);
    const long long grid = (long long)B * n_kv * tiles_q;
    if (grid > 0x7fffffffLL || (splits > 1 && part == nullptr)) return MSGL_ERR_SIZE;
    Kv4Attn p = {q, out, (const unsigned char*)k, (const unsigned char*)v, (const uint2*)steps, q_start, kv_len, block_table, part, bt_stride, (long long)T * n_q,
                 B, T, n_q, n_kv, d, page_size, pages, bt_width, window, max_q, splits, tiles_q, R, scale};
    auto smem_of = [](int rows, int size) { return ((size_t)rows * size * (1 + KV4_ANY_WARPS) + KV4_ANY_WARPS * rows * 34) * 4; };
    static MsglOncePerDevice attr_set;
#define KV4_ANY_EACH(DO) DO(float, 1, 2) DO(float, 1, 4) DO(float, 1, 8) DO(float, 2, 8) DO(__nv_bfloat16, 1, 2) DO(__nv_bfloat16, 1, 4) DO(__nv_bfloat16, 1, 8) DO(__nv_bfloat16, 2, 8)
    if (attr_set.due()) {
#define KV4_ANY_SET(TT, WW, RR) if (cudaFuncSetAttribute(kv4_attn_any_kernel<TT, WW, RR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_of(RR, WW * 256)) != cudaSuccess) return msgl_check_launch();
        KV4_ANY_EACH(KV4_ANY_SET)
#undef KV4_ANY_SET
        attr_set.mark();
    }
    const dim3 g((unsigned)grid, splits), b(KV4_ANY_WARPS * 32);
    const bool f32 = dtype == MSGL_F32;
#define KV4_ANY_GO(TT, WW, RR) if (f32 == (sizeof(TT) == 4) && wpl == WW && R == RR) msgl_launch_pdl(kv4_attn_any_kernel<TT, WW, RR>, g, b, smem_of(RR, d), stream, p);
    KV4_ANY_EACH(KV4_ANY_GO)
#undef KV4_ANY_GO
#undef KV4_ANY_EACH
    int rc = msgl_check_launch();
    if (rc != MSGL_OK || splits == 1) return rc;
    const dim3 gj((unsigned)grid, (d + 31) / 32);
    if (f32) msgl_launch_pdl(kv4_join_kernel<float>, gj, dim3(128), 0, stream, p);
    else msgl_launch_pdl(kv4_join_kernel<__nv_bfloat16>, gj, dim3(128), 0, stream, p);
    return msgl_check_launch();
}

#include "kv4_runs.cuh"
