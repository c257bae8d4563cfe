// pv_train.cu - log-probabilities of windows' tokens under a model's logits, the preference loss over pairs of windows
// and the clipped policy loss with a KL term, forward and backward (include/panvram_b200.h pv_logprobs ... pv_policy_grad).
//
// The mathematics, per row (a position's V logits x, its target y): with L = log2(e), a reference c and e_j = 2^(x_j L - c),
// s = sum e_j, p_j = e_j / s, log p_y = ln2 (x_y L - c) - log s, and d log p_y / d x_j = [j = y] - p_j.
// c is the maximum's product with L rounded to a whole number, plus ABOVE (2). It is the same for every numerator and for
// log p_y, so it cancels, and x_j L - c is one FMA. Where the maximum is beyond 2^29 (the product's rounding would then be too
// large; it overflows at the lowest or highest value of bf16 and fp32) the difference comes first: e_j = 2^((x_j - max) L - ABOVE).
//
// The 2^x is the hardware's approximation. Its results are short by 5.0 to 5.2e-8 on average, relative, over every octave of
// arguments below -1 (from 1.4e-7 short to 6e-8 over at single ones); between -1 and 1 the mean depends on the arguments' last
// bits (0.8 to 5e-8), and whole numbers are exact. Over a window of thousands of positions such a mean shows where single
// errors cancel. So references are whole numbers and no argument lies above -1 (the maximum's is between -2.5 and -1.5): then
// sums move from one reference to another by exact powers of two, SHORT is what a row's sum is short by, and is added back to
// its logarithm. Only logits of 0 have whole arguments. Where they are the maximum, and the sum is a whole number of their
// numerators, it holds nothing else (a fresh head): nothing is added back; else the one that is the maximum is left out.
// Measured over 65,536 positions of 5 to 5,000 words, targets drawn from the model: a log-probability's mean error is -1.8e-9
// to 4.3e-9, in every type. It costs a whole part a reference: 0 to 2.4 % of the kernels' time.
//
// The sum o over the other words is kept apart from the target's numerator e: 1 - p_y = o / (o + e) and, where e >= o,
// log p_y = -log1p(o / e), so neither loses its digits where the model is nearly sure.
// A row's statistics are in 32 bits, its log-probability and the differences taken of it in 64; sums over rows are in 64 bits
// and in a fixed order (a partial sum per tile of rows, then over the tiles), so results do not change from call to call.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include <algorithm>
#include <type_traits>

#include "panvram_b200.h"

namespace pvb { extern thread_local char g_cuda_err[256]; }

namespace {

using pvb::g_cuda_err;

constexpr float LOG2E = 1.4426950408889634f;
constexpr int SMS = 148;

// ---------------------------------------------------------------- elements
__device__ __forceinline__ float f32(float v) { return v; }
__device__ __forceinline__ float f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from32(float v);
template <> __device__ __forceinline__ float from32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// ---------------------------------------------------------------- what a row is scored against, and what follows from it
// LOGP: log-probabilities; GRAD: gradient from given derivatives; GIVEN: the same with the rows' statistics at hand too;
// POLICY: the policy loss's terms, and their gradient
enum { LOGP = 0, GRAD = 1, POLICY = 2, GIVEN = 3 };

struct Rows {
    pv_scored b;
    int64_t tpw;             // tiles (of TILE rows, or of one) per window
    int64_t stride, stride_n; int32_t stride_t;      // short rows: from a warp's tile to its next; in windows, and tiles of one
    // LOGP
    float* logp;             // or NULL
    double* part;            // a partial sum per tile (LOGP: of log-probabilities, POLICY: of loss terms), or NULL
    float4* stat;            // or NULL; GIVEN reads them: a row's maximum, reference, 1 / s and the target's 1 - p
    float* deriv;            // or NULL; POLICY: each row's derivative
    // GRAD, GIVEN
    const float* up; int64_t up_n, up_w;
    // POLICY
    pv_policy_args a;
    const double* weight;
    // GRAD, GIVEN, POLICY
    const float* scale; int32_t skip_one;
    int32_t scaled;          // GIVEN: the derivatives have the scale in them
};

// the target of row (i, t), or -1 (token and mask are loaded side by side)
__device__ __forceinline__ int target(const pv_scored& b, int64_t i, int64_t t) {
    const int64_t at = t + b.shift;
    if (at >= b.W) return -1;
    const int64_t y = b.token_bytes == 1 ? ((const uint8_t*)b.tokens)[i * b.tokens_n + at * b.tokens_w]
                                         : ((const int64_t*)b.tokens)[i * b.tokens_n + at * b.tokens_w];
    bool on = true;
    if (b.mask_bytes == 1) on = ((const uint8_t*)b.mask)[i * b.mask_n + at * b.mask_w] != 0;
    else if (b.mask_bytes == 4) on = ((const float*)b.mask)[i * b.mask_n + at * b.mask_w] != 0.f;
    return !on || y < 0 || y >= b.V || y == b.ignore ? -1 : (int)y;
}

// a row's (or a thread's part of a row's) reference
constexpr float ABOVE = 2.f;
constexpr double SHORT = 5.1e-8;
__device__ __forceinline__ bool far(float m) { return !(fabsf(m) < 536870912.f); }     // infinities too
__device__ __forceinline__ float ref_of(float m) { return (far(m) ? 0.f : rintf(m * LOG2E)) + ABOVE; }
__device__ __forceinline__ float exponent(float x, float m, float c) { return fmaf(far(m) ? x - m : x, LOG2E, -c); }
__device__ __forceinline__ float reciprocal(float v) {          // of sums of numerators: 2^-3 or more, so nothing is flushed
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void halves(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
// x becomes its numerators, two to an FMA (where the maximum is far, x less the maximum comes in)
template <int K>
__device__ __forceinline__ void less(float (&x)[K], float m) {
#pragma unroll
    for (int q = 0; q < K; q++) x[q] -= m;
}
template <int K>
__device__ __forceinline__ void numerators(float (&x)[K], float c) {
    const uint64_t l = pair(LOG2E, LOG2E), nc = pair(-c, -c);
#pragma unroll
    for (int q = 0; q < K; q += 2) {
        uint64_t v;
        asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(pair(x[q], x[q + 1])), "l"(l), "l"(nc));
        float a, b;
        halves(v, a, b);
        x[q] = ex2(a);
        x[q + 1] = ex2(b);
    }
}
template <int K>
__device__ __forceinline__ float sum_of(const float (&x)[K]) {
    uint64_t v = pair(x[0], x[1]);
#pragma unroll
    for (int q = 2; q < K; q += 2) asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(v), "l"(pair(x[q], x[q + 1])));
    float a, b;
    halves(v, a, b);
    return a + b;
}
template <int K>
__device__ __forceinline__ void times(float (&x)[K], float f) {
    const uint64_t ff = pair(f, f);
#pragma unroll
    for (int q = 0; q < K; q += 2) {
        uint64_t v;
        asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(pair(x[q], x[q + 1])), "l"(ff));
        halves(v, x[q], x[q + 1]);
    }
}

// log p of the target: x its logit, e its numerator, o the sum of the others', m the maximum (or the reference's). Where it
// does not outweigh the others, s = o + e = 2^k g with g from 0.7 to 1.4: log p = (x log2 e - c - k) ln 2 - log g - SHORT, of
// which only log g is rounded to 32 bits, as its size is small beside log p's. Where it does, o and e are short alike, and
// their quotient is not.
__device__ __forceinline__ double row_logp(float m, float o, float x, float e) {
    const bool sure = e >= o;
    const float s = o + e;
    const int b = __float_as_int(s), k = (b - 0x3F350000) >> 23;                 // 0.707 as bits
    const float l = log1pf(sure ? o * reciprocal(e) : __int_as_float(b - (k << 23)) - 1.f);
    if (m == -INFINITY || !(s < INFINITY)) return NAN;                           // nothing to normalise by, or not a number
    if (sure) return -(double)l;
    const double t = (far(m) ? ((double)x - (double)m) * 1.4426950408889634 : (double)x * (double)LOG2E) - (double)ref_of(m);
    double lost = SHORT;
    if (m == 0.f) lost = 4.f * s == rintf(4.f * s) ? 0.0 : (double)((float)SHORT * (1.f - 0.25f * reciprocal(s)));
    return (t - (double)k) * 0.6931471805599453 - (double)l - lost;
}

// exp(d) - 1 and exp(d) - d - 1, below 1 by the series of the latter, where the differences would lose their digits (at 0.25
// the second is 9 times smaller than the first); from 1 on it loses 2.4 at most.
__device__ __forceinline__ void kl_terms(float d, float& em1, float& kl) {
    if (fabsf(d) < 1.f) {
        constexpr float F[11] = {1.f / 2, 1.f / 6, 1.f / 24, 1.f / 120, 1.f / 720, 1.f / 5040, 1.f / 40320, 1.f / 362880,
                                 1.f / 3628800, 1.f / 39916800, 1.f / 479001600};      // the next is 2e-10 of the sum
        float p = F[10];
#pragma unroll
        for (int j = 9; j >= 0; j--) p = fmaf(d, p, F[j]);
        kl = d * d * p;
        em1 = d + kl;
    } else {
        em1 = expm1f(d);
        kl = em1 - d;
    }
}

// What a counted row's end reads, loaded before its logits are waited for.
struct End { float a, old, ref; };
template <int MODE>
__device__ __forceinline__ End end_args(const Rows& k, int64_t i, int64_t t) {
    End e = {0.f, 0.f, 0.f};
    if (MODE == GRAD || MODE == GIVEN) e.a = k.up[i * k.up_n + t * k.up_w];
    if (MODE == POLICY) {
        e.a = k.a.adv[i * k.a.adv_n + t * k.a.adv_w];
        e.old = k.a.old[i * k.a.old_n + t * k.a.old_w];
        if (k.a.ref) e.ref = k.a.ref[i * k.a.ref_n + t * k.a.ref_w];
    }
    return e;
}

// From a counted row's log-probability its term of the sum (before the window's weight w) and its derivative, times w and
// the upstream scale (the result).
template <int MODE>
__device__ __forceinline__ float row_end(const Rows& k, const End& e, double lp, float w, float scale, float& term) {
    if (MODE == LOGP) { term = (float)lp; return 0.f; }
    if (MODE == GRAD) { term = 0.f; return e.a * scale; }
    const float r = expf((float)(lp - (double)e.old));        // the difference in 64 bits: it is small beside its terms
    const float one = e.a == 0.f && r == INFINITY ? 0.f : r * e.a;      // a ratio that overflows by an advantage of 0 is 0, NaN stays
    const float two = fminf(fmaxf(r, 1.f - k.a.clip_low), 1.f + k.a.clip_high) * e.a;
    const bool free = !(one > two);                          // NaN stays
    float g = free ? -one : 0.f;
    term = free ? -one : -two;
    if (k.a.ref) {
        float em1, kl;
        kl_terms((float)((double)e.ref - lp), em1, kl);
        term += k.a.kl * kl;
        g -= k.a.kl * em1;
    }
    return g * w * scale;
}
template <int MODE>
__device__ __forceinline__ double weight_of(const Rows& k, int64_t i) { return MODE == POLICY ? k.weight[i] : 1.0; }

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int s = 16; s; s >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, s));
    return v;
}
template <typename F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
    for (int s = 16; s; s >>= 1) v += __shfl_xor_sync(~0u, v, s);
    return v;
}

// ---------------------------------------------------------------- 16 bytes of a row
template <typename T> struct Traits;
template <> struct Traits<float> { static constexpr uint32_t LOW = 0xFF800000u; };             // -inf, as a word of elements
template <> struct Traits<__half> { static constexpr uint32_t LOW = 0xFC00FC00u; };
template <> struct Traits<__nv_bfloat16> { static constexpr uint32_t LOW = 0xFF80FF80u; };
template <typename T> __device__ __forceinline__ T lowest() { return from32<T>(-INFINITY); }
template <typename T> constexpr int K_OF = 16 / (int)sizeof(T);

template <typename T> __device__ __forceinline__ void unpack(const uint4& r, float (&x)[K_OF<T>]);
template <> __device__ __forceinline__ void unpack<float>(const uint4& r, float (&x)[4]) {
    x[0] = __uint_as_float(r.x); x[1] = __uint_as_float(r.y); x[2] = __uint_as_float(r.z); x[3] = __uint_as_float(r.w);
}
template <> __device__ __forceinline__ void unpack<__nv_bfloat16>(const uint4& r, float (&x)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int q = 0; q < 4; q++) { x[2 * q] = __uint_as_float(w[q] << 16); x[2 * q + 1] = __uint_as_float(w[q] & 0xFFFF0000u); }
}
template <> __device__ __forceinline__ void unpack<__half>(const uint4& r, float (&x)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const float2 f = __half22float2(*(const __half2*)&w[q]);
        x[2 * q] = f.x; x[2 * q + 1] = f.y;
    }
}
template <typename T> __device__ __forceinline__ void unpack_word(uint32_t w, float& a, float& b);
template <> __device__ __forceinline__ void unpack_word<float>(uint32_t w, float& a, float& b) { a = b = __uint_as_float(w); }
template <> __device__ __forceinline__ void unpack_word<__nv_bfloat16>(uint32_t w, float& a, float& b) {
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xFFFF0000u);
}
template <> __device__ __forceinline__ void unpack_word<__half>(uint32_t w, float& a, float& b) {
    const float2 f = __half22float2(*(const __half2*)&w);
    a = f.x;
    b = f.y;
}
template <typename T> __device__ __forceinline__ uint32_t pack_word(float a, float b);
template <> __device__ __forceinline__ uint32_t pack_word<float>(float a, float) { return __float_as_uint(a); }
template <> __device__ __forceinline__ uint32_t pack_word<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *(const uint32_t*)&v;
}
template <> __device__ __forceinline__ uint32_t pack_word<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *(const uint32_t*)&v;
}
template <typename T> __device__ __forceinline__ uint4 pack(const float (&x)[K_OF<T>]);
template <> __device__ __forceinline__ uint4 pack<float>(const float (&x)[4]) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
}
template <> __device__ __forceinline__ uint4 pack<__nv_bfloat16>(const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int q = 0; q < 4; q++) { const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * q], x[2 * q + 1]); w[q] = *(const uint32_t*)&v; }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <> __device__ __forceinline__ uint4 pack<__half>(const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int q = 0; q < 4; q++) { const __half2 v = __floats2half2_rn(x[2 * q], x[2 * q + 1]); w[q] = *(const uint32_t*)&v; }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T> __device__ __forceinline__ uint32_t word_max(uint32_t a, uint32_t b);        // element by element
template <> __device__ __forceinline__ uint32_t word_max<float>(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
}
template <> __device__ __forceinline__ uint32_t word_max<__nv_bfloat16>(uint32_t a, uint32_t b) {
    const __nv_bfloat162 m = __hmax2(*(const __nv_bfloat162*)&a, *(const __nv_bfloat162*)&b);
    return *(const uint32_t*)&m;
}
template <> __device__ __forceinline__ uint32_t word_max<__half>(uint32_t a, uint32_t b) {
    const __half2 m = __hmax2(*(const __half2*)&a, *(const __half2*)&b);
    return *(const uint32_t*)&m;
}

// of all words in some pieces: packed, and widened once
template <typename T, int N>
__device__ __forceinline__ float pieces_max(const uint4 (&r)[N]) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < N; j++) {
        const uint32_t v = word_max<T>(word_max<T>(r[j].x, r[j].y), word_max<T>(r[j].z, r[j].w));
        m = j ? word_max<T>(m, v) : v;
    }
    float a, b;
    unpack_word<T>(m, a, b);
    return fmaxf(a, b);
}

// A row of V elements seen as aligned 16-byte pieces: piece v holds elements v K - off ... + K, off = how far into its
// first piece the row starts. The pieces at the row's ends are moved by element, so nothing outside the row is touched.
template <typename T>
__device__ __forceinline__ int row_off(const T* x) { return (int)(((uintptr_t)x & 15) / sizeof(T)); }
// the elements before a row's first whole piece
template <typename T>
__device__ __forceinline__ int head_of(const T* x, int V) { return min((int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T)), V); }
template <typename T>
__device__ __forceinline__ bool whole(int e0, int V) { return e0 >= 0 && e0 + K_OF<T> <= V; }
template <typename T>
__device__ __forceinline__ void store_piece(T* d, int e0, int V, bool aligned, const float (&x)[K_OF<T>]) {
    constexpr int K = K_OF<T>;
    if (aligned && whole<T>(e0, V)) { *(uint4*)(d + e0) = pack<T>(x); return; }
#pragma unroll
    for (int q = 0; q < K; q++)
        if (e0 + q >= 0 && e0 + q < V) d[e0 + q] = from32<T>(x[q]);
}
template <typename T>
__device__ __forceinline__ void store_raw(T* d, bool aligned, const uint4& v) {
    if (aligned) { *(uint4*)d = v; return; }
    const T* q = (const T*)&v;
#pragma unroll
    for (int h = 0; h < K_OF<T>; h++) d[h] = q[h];
}
// the pieces of x and d fall alike
template <typename T>
__device__ __forceinline__ bool alike(const T* x, const T* d) { return (((uintptr_t)x ^ (uintptr_t)d) & 15) == 0; }

// ---------------------------------------------------------------- asynchronous copies into shared memory
// A warp's tiles of TILE rows: first, first + stride, ... of those of all windows in turn, tpw to a window. The stride, as
// windows and tiles of one, comes with the launch, so that what follows from it alone stays out of the threads' registers.
constexpr int TILE = 32, WARPS = 8;
struct Tiles {
    int64_t r;               // the tile
    int t;                   // its place in its window
    __device__ __forceinline__ Tiles(const Rows& k) : r((int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5)), t((int)(r % k.tpw)) {}
    __device__ __forceinline__ bool live(const Rows& k) const { return r < k.b.n * k.tpw; }
    __device__ __forceinline__ bool next(const Rows& k) {    // whether the place in the window has wrapped
        r += k.stride;
        t += k.stride_t;
        if (t < (int)k.tpw) return false;
        t -= (int)k.tpw;
        return true;
    }
};
// The address of an element (window, position), in an array with strides n and w in elements of `size` bytes, that goes from
// tile to tile by additions.
__device__ __forceinline__ const char* place(const Rows& k, const Tiles& at, const void* base, int64_t n, int64_t w, int64_t size, int64_t ahead) {
    return (const char*)base + (at.r / k.tpw * n + ((int64_t)at.t * TILE + ahead) * w) * size;
}
__device__ __forceinline__ void walk(const Rows& k, const char*& p, bool wrapped, int64_t n, int64_t w, int64_t size) {
    p += (k.stride_n * n + (int64_t)k.stride_t * TILE * w) * size;
    if (wrapped) p += (n - k.tpw * TILE * w) * size;
}
// The targets of a tile's rows, a lane each (-1: not counted).
struct Targets {
    Tiles at;
    const char *tok, *mask;
    __device__ __forceinline__ Targets(const Rows& k, int lane)
        : at(k), tok(place(k, at, k.b.tokens, k.b.tokens_n, k.b.tokens_w, k.b.token_bytes, lane + (int64_t)k.b.shift)),
          mask(place(k, at, k.b.mask, k.b.mask_n, k.b.mask_w, k.b.mask_bytes, lane + (int64_t)k.b.shift)) {}
    __device__ __forceinline__ int get(const Rows& k, int lane) const {
        if (!at.live(k) || (int64_t)at.t * TILE + lane + k.b.shift >= k.b.W) return -1;
        const int64_t y = k.b.token_bytes == 1 ? *(const uint8_t*)tok : *(const int64_t*)tok;
        bool on = true;
        if (k.b.mask_bytes == 1) on = *(const uint8_t*)mask != 0;
        else if (k.b.mask_bytes == 4) on = *(const float*)mask != 0.f;
        return !on || y < 0 || y >= k.b.V || y == k.b.ignore ? -1 : (int)y;
    }
    __device__ __forceinline__ void next(const Rows& k) {
        const bool w = at.next(k);
        walk(k, tok, w, k.b.tokens_n, k.b.tokens_w, k.b.token_bytes);
        if (k.b.mask_bytes) walk(k, mask, w, k.b.mask_n, k.b.mask_w, k.b.mask_bytes);
    }
};
// What their ends read, a lane each.
template <int MODE>
struct Ends {
    const char *a, *old, *ref;
    __device__ __forceinline__ Ends(const Rows& k, const Tiles& at, int lane) : a(nullptr), old(nullptr), ref(nullptr) {
        if (MODE == GRAD) a = place(k, at, k.up, k.up_n, k.up_w, 4, lane);
        if (MODE == POLICY) {
            a = place(k, at, k.a.adv, k.a.adv_n, k.a.adv_w, 4, lane);
            old = place(k, at, k.a.old, k.a.old_n, k.a.old_w, 4, lane);
            ref = place(k, at, k.a.ref, k.a.ref_n, k.a.ref_w, 4, lane);
        }
    }
    __device__ __forceinline__ End get(const Rows& k, bool row) const {
        End e = {0.f, 0.f, 0.f};
        if (MODE == LOGP || !row) return e;
        e.a = *(const float*)a;
        if (MODE == POLICY) {
            e.old = *(const float*)old;
            if (k.a.ref) e.ref = *(const float*)ref;
        }
        return e;
    }
    __device__ __forceinline__ void next(const Rows& k, bool wrapped) {
        if (MODE == GRAD) walk(k, a, wrapped, k.up_n, k.up_w, 4);
        if (MODE == POLICY) {
            walk(k, a, wrapped, k.a.adv_n, k.a.adv_w, 4);
            walk(k, old, wrapped, k.a.old_n, k.a.old_w, 4);
            if (k.a.ref) walk(k, ref, wrapped, k.a.ref_n, k.a.ref_w, 4);
        }
    }
};

__device__ __forceinline__ uint32_t shared_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t to, const void* from) {                   // to: an address in shared memory
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// ---------------------------------------------------------------- sums over pieces
template <typename T, int U>
__device__ __forceinline__ float sum_all(const uint4 (&raw)[U], float c, float o) {       // o and the numerators' sum
    uint64_t v = pair(o, 0.f);
#pragma unroll
    for (int u = 0; u < U; u++) {
        float x[K_OF<T>];
        unpack<T>(raw[u], x);
        numerators(x, c);
#pragma unroll
        for (int q = 0; q < K_OF<T>; q += 2) asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(v), "l"(pair(x[q], x[q + 1])));
    }
    float a, b;
    halves(v, a, b);
    return a + b;
}
// the same about a maximum beyond 2^29 (or one of -inf and nothing else, with by 0)
template <typename T, int U>
__device__ __noinline__ float sum_far(const uint4* raw, int step, float by, float c, float o) {
#pragma unroll 1
    for (int u = 0; u < U; u++) {
        float x[K_OF<T>];
        unpack<T>(raw[u * step], x);
        less(x, by);
        numerators(x, c);
        o += sum_of(x);
    }
    return o;
}

// ---------------------------------------------------------------- rows of up to 256 pieces: G lanes a row, NV pieces a lane
// A warp takes tiles of 32 rows, 32 / G at a step. Its rows come through a ring of S steps of its own in shared memory: every
// lane copies its own pieces in and reads them once, into registers, where the row stays until its gradient is out. A step's
// copy goes S - 1 groups ahead of its use. The targets of a tile are loaded a tile ahead of its copies and wait with them in
// the ring; the arguments of its rows are loaded before the first of them is waited for. The target's logit is read out of
// the ring and -inf put in its place: the sum of the others and their maximum follow without a comparison an element.
//
// On a B200, 524,288 rows of 128 bf16 words: log-probabilities 35 us (3.8 TB/s), policy loss and gradient 58 us (4.6 TB/s
// read and written); 1,048,576 of 16 words 19 and 32 us. Bound by instructions: counted, a step of 8 rows of 128 words takes
// 321 of them for log-probabilities, 373 for a gradient and 577 for the policy loss (targets, addresses, shuffles, the rows'
// ends) where the words themselves, 32 a lane, take 4 each or 8 with a gradient; of 32 rows of 16 words 426, 427 and 733; of 2 of
// 401 words that start anywhere 376, 499 and 676. Issue slots are 49 to 63 % taken, the rest is their latency at 5 to 7 warps
// a scheduler. So lanes hold 32 words (64, half the lanes, lose more by the warps that no longer fit: 1,048,576 rows take
// 146 us, and 112 with 32), and 3 or 6 pieces where a quarter of 4 or 8 would be empty (131,072 rows of 1,536: 150 us with 6,
// 179 with 8). Three blocks a multiprocessor for log-probabilities (64 us, two 69), two where the numerators are kept for the
// gradient (112 us, three spill: 153). A row that starts anywhere costs half as much again (282 words of 4 bytes 180 us, 284
// aligned ones 136); loading its ends a step ahead does not help (195).
// A: rows of whole pieces, logits' and gradient's alike. Else (G 16 or more) the elements before a row's first whole piece and
// behind its last are held by a lane each, as the rows start anywhere.
template <typename T, int G, int NV, int S, int MODE, bool A>
__global__ void __launch_bounds__(WARPS * 32, (NV < 3 && A) || ((NV == 3 || NV == 4) && MODE == LOGP) ? 3 : 2) rows_group_kernel(Rows k) {
    constexpr int K = K_OF<T>, RP = 32 / G;
    static_assert(A || G >= 16, "a lane for each element at a row's ends");
    extern __shared__ uint4 rings[];                         // [WARPS][S][NV][32]
    const int lane = threadIdx.x & 31, sub = lane % G, grp = lane / G, V = (int)k.b.V;
    const float scale = MODE != LOGP && k.scale ? *k.scale : 1.f;
    if (MODE != LOGP && k.skip_one && scale == 1.f) return;
    uint4* const ring = rings + (threadIdx.x >> 5) * (S * NV * 32);
    const uint32_t ring_at = shared_at(ring + lane);
    // pieces beyond a row's end are never copied: -inf from here on
#pragma unroll
    for (int s = 0; s < S * NV; s++) ring[s * 32 + lane] = make_uint4(Traits<T>::LOW, Traits<T>::LOW, Traits<T>::LOW, Traits<T>::LOW);

    int* const ys = (int*)(rings + WARPS * S * NV * 32) + (threadIdx.x >> 5) * (S * 32);      // [WARPS][S][32]: the steps' targets

    const int64_t x_step = RP * k.b.logits_w, d_step = RP * k.b.grad_w;
    // the tile being copied, its targets, and those of the one after it
    Tiles in(k);
    const char* in_at = place(k, in, k.b.logits, k.b.logits_n, k.b.logits_w, sizeof(T), grp);
    const T* in_x = (const T*)in_at;                         // of this lane's group, a step's rows on at a time
    Targets look(k, lane);
    int in_y = look.get(k, lane), in_s = 0, in_slot = 0;
    look.next(k);
    int in_y_next = look.get(k, lane);
    const auto copy_next = [&]() {
        if (in.live(k)) {
            const int y = __shfl_sync(~0u, in_y, in_s * RP + grp);
            if (sub == 0) ys[in_slot * 32 + grp] = y;
            if (y >= 0) {
                const int head = A ? 0 : head_of(in_x, V), n = (V - head) / K;
                const uint32_t to = ring_at + in_slot * (NV * 512);
#pragma unroll
                for (int j = 0; j < NV; j++)
                    if (sub + j * G < n) copy16(to + j * 512, in_x + head + (sub + j * G) * K);
            }
            in_x += x_step;
            if (++in_s == G) {
                in_s = 0;
                in_y = in_y_next;
                walk(k, in_at, in.next(k), k.b.logits_n, k.b.logits_w, sizeof(T));
                in_x = (const T*)in_at;
                look.next(k);
                in_y_next = look.get(k, lane);
            }
        }
        if (++in_slot == S) in_slot = 0;
        copies_commit();
    };
#pragma unroll 1
    for (int s = 0; s < S; s++) copy_next();

    int slot = 0;
    Tiles p(k);
    int64_t i = p.r / k.tpw;                                 // its window
    const char* x_at = A ? nullptr : place(k, p, k.b.logits, k.b.logits_n, k.b.logits_w, sizeof(T), grp);
    const char* d_at = MODE == LOGP ? nullptr : place(k, p, k.b.grad, k.b.grad_n, k.b.grad_w, sizeof(T), grp);
    Ends<MODE> ends(k, p, lane);
    while (p.live(k)) {
        const T* x = (const T*)x_at;
        T* d = MODE != LOGP && k.b.grad ? (T*)d_at : nullptr;
        const int rows = (int)min((int64_t)TILE, k.b.W - (int64_t)p.t * TILE);
        const End end_l = ends.get(k, lane < rows);
        const double w = weight_of<MODE>(k, i);
        const float wf = (float)w;
        double sum = 0;
        // LOGP: the row of this lane's number in the tile, its maximum, others' sum, target's logit and numerator
        float my_m = 0.f, my_o = 0.f, my_x = 0.f, my_e = 0.f;
        int my_y = -1;
#pragma unroll 1
        for (int s = 0; s < G; s++) {
            copies_wait<S - 1>();
            __syncwarp();
            const int row = s * RP + grp, y = ys[slot * 32 + grp];
            const int head = A ? 0 : head_of(x, V), n = (V - head) / K, tail = head + n * K;
            int edge = -1;
            float ex = -INFINITY;
            if (!A) {
                edge = sub < head && sub < 8 ? sub : sub >= 8 && tail + sub - 8 < V ? tail + sub - 8 : -1;
                if (y >= 0 && edge >= 0) ex = f32(x[edge]);
            }
            uint4* const base = ring + slot * (NV * 32);
            uint4* const own = base + lane;
            const bool in_piece = A || (y >= head && y < tail);
            const unsigned place = in_piece ? (unsigned)(max(y, 0) - head) : 0u, piece = place / K;
            T* const at = (T*)(base + piece / G * 32 + grp * G + piece % G) + place % K;
            float xt = f32(*at);
            __syncwarp();
            const bool owner = in_piece && (int)(piece % G) == sub;
            if (owner) *at = lowest<T>();
            if (!A) {
                const float v = __shfl_sync(~0u, ex, grp * G + (y < head ? max(y, 0) : 8 + y - tail) % G);
                if (!in_piece) xt = v;
                if (edge == y) ex = -INFINITY;
            }
            uint4 raw[NV];
#pragma unroll
            for (int j = 0; j < NV; j++) {
                raw[j] = own[j * 32];
                if (!A && sub + j * G >= n) raw[j] = make_uint4(Traits<T>::LOW, Traits<T>::LOW, Traits<T>::LOW, Traits<T>::LOW);
            }
            float m = fmaxf(pieces_max<T>(raw), ex);
#pragma unroll
            for (int h = G / 2; h; h >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, h));
            m = fmaxf(m, xt);
            const float c = ref_of(m), et = ex2(exponent(xt, m, c));
            const bool any_far = __any_sync(~0u, far(m));
            float e[MODE == LOGP ? 1 : NV][K], o = 0.f;
            if constexpr (MODE == LOGP) {
                if (any_far) {
#pragma unroll 1
                    for (int j = 0; j < NV; j++)
                        if (A || sub + j * G < n) o = sum_far<T, 1>(own + j * 32, 0, far(m) ? m : 0.f, c, o);
                } else {
                    o = sum_all<T, NV>(raw, c, 0.f);
                }
            } else {
#pragma unroll
                for (int j = 0; j < NV; j++) unpack<T>(raw[j], e[j]);
                if (any_far) {
                    const float by = far(m) ? m : 0.f;
#pragma unroll
                    for (int j = 0; j < NV; j++) less(e[j], by);
                }
#pragma unroll
                for (int j = 0; j < NV; j++) {
                    numerators(e[j], c);
                    o += sum_of(e[j]);
                }
            }
            const float ee = A ? 0.f : ex2(exponent(ex, m, c));
            if (!A && edge >= 0) o += ee;
            copy_next();
            if (++slot == S) slot = 0;
#pragma unroll
            for (int h = G / 2; h; h >>= 1) o += __shfl_xor_sync(~0u, o, h);
            if constexpr (MODE == LOGP) {
                const int from = lane % RP * G;
                const float a = __shfl_sync(~0u, m, from), b = __shfl_sync(~0u, o, from), f = __shfl_sync(~0u, xt, from), g = __shfl_sync(~0u, et, from);
                const int h = __shfl_sync(~0u, y, from);
                if (lane / RP == s) { my_m = a; my_o = b; my_x = f; my_e = g; my_y = h; }
            } else {
                const End end = {__shfl_sync(~0u, end_l.a, row), MODE == POLICY ? __shfl_sync(~0u, end_l.old, row) : 0.f,
                                 MODE == POLICY ? __shfl_sync(~0u, end_l.ref, row) : 0.f};
                float g = 0.f, term = 0.f;
                if (y >= 0) {
                    g = row_end<MODE>(k, end, MODE == POLICY ? row_logp(m, o, xt, et) : 0.0, wf, scale, term);
                    if (MODE == POLICY && sub == 0) sum += (double)term;
                }
                const bool some_off = __any_sync(~0u, y < 0);
                if (d && row < rows) {
                    const bool same = A || alike(x, d);
                    const float inv = reciprocal(o + et), f = -g * inv;
#pragma unroll
                    for (int j = 0; j < NV; j++) {
                        times(e[j], f);
                        uint4 v = pack<T>(e[j]);
                        if (some_off && y < 0) v = make_uint4(0u, 0u, 0u, 0u);
                        if (sub + j * G < n) store_raw(d + head + (sub + j * G) * K, same, v);
                    }
                    if (!A && edge >= 0) d[edge] = from32<T>(y < 0 ? 0.f : edge == y ? g * (o * inv) : f * ee);
                    if (y >= 0 && owner) d[y] = from32<T>(g * (o * inv));
                }
                if (d) d += d_step;
            }
            if (!A) x += x_step;
        }
        if (MODE == LOGP) {
            const double lp = my_y >= 0 ? row_logp(my_m, my_o, my_x, my_e) : 0.0;
            sum = lp;
            if (k.logp && lane < rows) k.logp[i * k.b.W + (int64_t)p.t * TILE + lane] = (float)lp;
        }
        if (k.part) {
            sum = warp_sum(sum);
            if (lane == 0) k.part[p.r] = sum * w;
        }
        const bool wrapped = p.next(k);
        ends.next(k, wrapped);
        i += k.stride_n + wrapped;
        if (!A) walk(k, x_at, wrapped, k.b.logits_n, k.b.logits_w, sizeof(T));
        if (MODE != LOGP) walk(k, d_at, wrapped, k.b.grad_n, k.b.grad_w, sizeof(T));
    }
    copies_wait<0>();
}

// ---------------------------------------------------------------- short rows that start anywhere, one behind the other
// Here a step's rows are copied as one stretch, in the 16-byte pieces it covers whole (the elements at the stretch's two ends
// by a lane each), into an image of it in shared memory. A group of G lanes takes a row from the image in its 32-bit words,
// lane by lane; of a first or last word that it shares with its neighbour it masks the half that is not its own. The gradient
// replaces the logits in the image and leaves as the stretch came.
//
// On a B200, 1,048,576 rows of 5 bf16 words: log-probabilities 21 us, gradient 24 us, policy loss and gradient 37 us, bound by the
// instructions of a step, whatever its words: counted, 539, 597 and 820 for 32 rows (the stretch and its ends, the image, the
// targets, the rows' ends), issue slots 72, 68 and 56 % taken, the rest latency at 7 to 4 warps a scheduler. 524,288 of 101
// words 56 and 98 us, bound by instructions as the rows above, with a load and two comparisons a word more. 12 words a lane where a third of 17 would be
// empty (95 words: 47 and 84 us, with 17 55 and 103). Three blocks a multiprocessor for log-probabilities (33 words 35 us, two
// 40), and for a gradient of up to 16 numerators a lane (11 floats 26 us, two 31).
// the numerators' sum over a lane's words; FAR: about a maximum beyond 2^29 (or none, by 0)
template <typename T, bool FAR, int NW>
__device__ __forceinline__ float sum_words(const uint32_t (&raw)[NW], float by, float c) {
    constexpr int E = 4 / (int)sizeof(T);
    uint64_t v = pair(0.f, 0.f);
#pragma unroll
    for (int q = 0; q < (NW * E + 1) / 2; q++) {
        float x[2];
        if (E == 2) {
            unpack_word<T>(raw[E == 2 ? q : 0], x[0], x[1]);
        } else {
            x[0] = __uint_as_float(raw[E == 1 ? 2 * q : 0]);
            x[1] = 2 * q + 1 < NW ? __uint_as_float(raw[2 * q + 1 < NW ? 2 * q + 1 : 0]) : -INFINITY;
        }
        if (FAR) less(x, by);
        numerators(x, c);
        asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(v), "l"(pair(x[0], x[1])));
    }
    float a, b;
    halves(v, a, b);
    return a + b;
}

// NW: words a lane
template <typename T, int G, int NW, int S, int MODE>
__global__ void __launch_bounds__(WARPS * 32, MODE == LOGP || (MODE == GRAD && NW * (4 / sizeof(T)) <= 16) ? 3 : 2) rows_flat_kernel(Rows k) {
    constexpr int K = K_OF<T>, RP = 32 / G, E = 4 / (int)sizeof(T), N = (NW * E + 1) / 2 * 2;      // E: elements a word
    constexpr int SLOT = (NW * 32 * 4 + 47) / 16;            // 16-byte pieces of an image
    extern __shared__ uint4 rings[];                         // [WARPS][S][SLOT]
    const int lane = threadIdx.x & 31, sub = lane % G, grp = lane / G, V = (int)k.b.V;
    const float scale = MODE != LOGP && k.scale ? *k.scale : 1.f;
    if (MODE != LOGP && k.skip_one && scale == 1.f) return;
    uint4* const ring = rings + (threadIdx.x >> 5) * (S * SLOT);
    const uint32_t ring_at = shared_at(ring);

    int* const ys = (int*)(rings + WARPS * S * SLOT) + (threadIdx.x >> 5) * (S * 32);         // [WARPS][S][32]: the steps' targets
    const auto rows_of_tile = [&](const Tiles& p) { return (int)min((int64_t)TILE, k.b.W - (int64_t)p.t * TILE); };
    // a step's stretch: how far into its first piece it starts, its elements
    struct Stretch { int off, len; };
    const auto stretch = [&](const T* x, int s, int rows) { return Stretch{row_off(x), max(0, min(RP, rows - s * RP)) * V}; };

    Tiles in(k);
    const char* in_at = place(k, in, k.b.logits, k.b.logits_n, V, sizeof(T), 0);
    const T* in_x = (const T*)in_at;
    Targets look(k, lane);
    int in_y = look.get(k, lane), in_s = 0, in_slot = 0;
    look.next(k);
    int in_y_next = look.get(k, lane);
    const auto copy_next = [&]() {
        if (in.live(k)) {
            const int y = __shfl_sync(~0u, in_y, in_s * RP + grp);
            if (sub == 0) ys[in_slot * 32 + grp] = y;
            if (__any_sync(~0u, y >= 0)) {
                const Stretch q = stretch(in_x, in_s, rows_of_tile(in));
                const uint32_t to = ring_at + in_slot * (SLOT * 16);
                const T* const from = in_x - q.off;
                for (int p = lane + (q.off > 0); (p + 1) * K <= q.off + q.len; p += 32) copy16(to + p * 16, from + p * K);
            }
            in_x += RP * V;
            if (++in_s == G) {
                in_s = 0;
                in_y = in_y_next;
                walk(k, in_at, in.next(k), k.b.logits_n, V, sizeof(T));
                in_x = (const T*)in_at;
                look.next(k);
                in_y_next = look.get(k, lane);
            }
        }
        if (++in_slot == S) in_slot = 0;
        copies_commit();
    };
#pragma unroll 1
    for (int s = 0; s < S; s++) copy_next();

    int slot = 0;
    Tiles p(k);
    int64_t i = p.r / k.tpw;                                 // its window
    const char* x_at = place(k, p, k.b.logits, k.b.logits_n, V, sizeof(T), 0);
    const char* d_at = MODE == LOGP ? nullptr : place(k, p, k.b.grad, k.b.grad_n, V, sizeof(T), 0);
    Ends<MODE> ends(k, p, lane);
    while (p.live(k)) {
        const T* x = (const T*)x_at;
        T* d = MODE != LOGP && k.b.grad ? (T*)d_at : nullptr;
        const int rows = rows_of_tile(p);
        const End end_l = ends.get(k, lane < rows);
        const double w = weight_of<MODE>(k, i);
        const float wf = (float)w;
        double sum = 0;
        float my_m = 0.f, my_o = 0.f, my_x = 0.f, my_e = 0.f;
        int my_y = -1;
#pragma unroll 1
        for (int s = 0; s < G; s++, x += RP * V) {
            copies_wait<S - 1>();
            __syncwarp();
            const int row = s * RP + grp, y = ys[slot * 32 + grp];
            const Stretch q = stretch(x, s, rows);
            const bool any = __any_sync(~0u, y >= 0);
            uint4* const base = ring + slot * SLOT;
            T* const img = (T*)base;
            // the stretch's elements before its first whole piece and behind its last
            const int head = min((K - q.off) % K, q.len), tail = max(head, (q.off + q.len) / K * K - q.off);
            const int edge = lane < 8 ? (lane < head ? lane : -1) : lane < 16 && tail + lane - 8 < q.len ? tail + lane - 8 : -1;
            T ev = lowest<T>();
            if (any && edge >= 0) ev = x[edge];
            if (edge >= 0) img[q.off + edge] = ev;
            __syncwarp();
            // the row's words, this lane's, which of them (first: word 0; last: -1 none) another row has a part of
            const int at = q.off + grp * V, w0 = at / E, words = (at + V - 1) / E - w0 + 1, ty = at + max(y, 0);
            const int mine = (words - sub + G - 1) / G, last = E == 2 && (at + V) % 2 && (words - 1) % G == sub ? (words - 1) / G : -1;
            const bool first = E == 2 && sub == 0 && at % 2;
            uint32_t* const own = (uint32_t*)base + w0 + sub;
            float xt = 0.f;
            if (y >= 0) xt = f32(img[ty]);
            __syncwarp();
            if (y >= 0 && sub == 0) img[ty] = lowest<T>();
            __syncwarp();
            uint32_t raw[NW], most = Traits<T>::LOW;
            const int cnt = y >= 0 ? mine : 0;
#pragma unroll
            for (int j = 0; j < NW; j++) {
                raw[j] = Traits<T>::LOW;
                if (j < cnt) raw[j] = own[j * G];
                if (j == 0 && first) raw[j] = raw[j] & 0xFFFF0000u | Traits<T>::LOW & 0xFFFFu;
                if (E == 2 && j == last) raw[j] = raw[j] & 0xFFFFu | Traits<T>::LOW & 0xFFFF0000u;
                most = word_max<T>(raw[j], most);
            }
            float m, m2;
            unpack_word<T>(most, m, m2);
            m = y < 0 ? 0.f : fmaxf(fmaxf(m, m2), xt);
#pragma unroll
            for (int h = G / 2; h; h >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, h));
            const float c = ref_of(m), et = ex2(exponent(xt, m, c));
            const bool any_far = __any_sync(~0u, far(m));
            float e[MODE == LOGP ? 1 : N], o;
            if constexpr (MODE == LOGP) {
                o = any_far ? sum_words<T, true>(raw, far(m) ? m : 0.f, c) : sum_words<T, false>(raw, 0.f, c);
            } else {
                e[N - 1] = -INFINITY;
#pragma unroll
                for (int j = 0; j < NW; j++) {
                    if (E == 1) e[j] = __uint_as_float(raw[j]);
                    else unpack_word<T>(raw[j], e[2 * j < N ? 2 * j : 0], e[2 * j + 1 < N ? 2 * j + 1 : 0]);
                }
                if (any_far) less(e, far(m) ? m : 0.f);
                numerators(e, c);
                o = sum_of(e);
            }
#pragma unroll
            for (int h = G / 2; h; h >>= 1) o += __shfl_xor_sync(~0u, o, h);
            if constexpr (MODE == LOGP) {
                const int from = lane % RP * G;
                const float a = __shfl_sync(~0u, m, from), b = __shfl_sync(~0u, o, from), f = __shfl_sync(~0u, xt, from), g = __shfl_sync(~0u, et, from);
                const int h = __shfl_sync(~0u, y, from);
                if (lane / RP == s) { my_m = a; my_o = b; my_x = f; my_e = g; my_y = h; }
            } else {
                const End end = {__shfl_sync(~0u, end_l.a, row), MODE == POLICY ? __shfl_sync(~0u, end_l.old, row) : 0.f,
                                 MODE == POLICY ? __shfl_sync(~0u, end_l.ref, row) : 0.f};
                float g = 0.f, term = 0.f;
                if (y >= 0) {
                    g = row_end<MODE>(k, end, MODE == POLICY ? row_logp(m, o, xt, et) : 0.0, wf, scale, term);
                    if (MODE == POLICY && sub == 0) sum += (double)term;
                }
                if (d) {
                    // a row that is not counted: numerators of 0
                    const float inv = reciprocal(o + et), f = y < 0 ? 0.f : -g * inv;
                    times(e, f);
                    __syncwarp();
                    const int out = row < rows ? mine : 0;
#pragma unroll
                    for (int j = 0; j < NW; j++) {
                        const uint32_t z = E == 1 ? __float_as_uint(e[j]) : pack_word<T>(e[2 * j < N ? 2 * j : 0], e[2 * j + 1 < N ? 2 * j + 1 : 0]);
                        if (j < out) {
                            const bool low = !(j == 0 && first), high = E == 1 || j != last;
                            if (low && high) own[j * G] = z;
                            else if (low) *(uint16_t*)(own + j * G) = (uint16_t)z;
                            else if (high) *((uint16_t*)(own + j * G) + 1) = (uint16_t)(z >> 16);
                        }
                    }
                    __syncwarp();
                    if (y >= 0 && sub == 0) img[ty] = from32<T>(g * (o * inv));
                    __syncwarp();
                    T* const to = d - q.off;
                    for (int v = lane + (q.off > 0); (v + 1) * K <= q.off + q.len; v += 32) *(uint4*)(to + v * K) = base[v];
                    if (edge >= 0) d[edge] = img[q.off + edge];
                    d += RP * V;
                }
            }
            __syncwarp();
            copy_next();
            if (++slot == S) slot = 0;
        }
        if (MODE == LOGP) {
            const double lp = my_y >= 0 ? row_logp(my_m, my_o, my_x, my_e) : 0.0;
            sum = lp;
            if (k.logp && lane < rows) k.logp[i * k.b.W + (int64_t)p.t * TILE + lane] = (float)lp;
        }
        if (k.part) {
            sum = warp_sum(sum);
            if (lane == 0) k.part[p.r] = sum * w;
        }
        const bool wrapped = p.next(k);
        ends.next(k, wrapped);
        i += k.stride_n + wrapped;
        walk(k, x_at, wrapped, k.b.logits_n, V, sizeof(T));
        if (MODE != LOGP) walk(k, d_at, wrapped, k.b.grad_n, V, sizeof(T));
    }
    copies_wait<0>();
}

// ---------------------------------------------------------------- longer rows: a block a row
// the running maximum and sum of a thread
struct Run { float m = -INFINITY, c = 0.f, o = 0.f; };
// The reference is raised only by more than HEADROOM, so that it seldom is; it is higher by LIFT (12 > 8 log2 e) than that of
// the maximum it is made from, so that the arguments stay below -1.
constexpr float HEADROOM = 8.f, LIFT = 12.f;
__device__ __forceinline__ float run_ref(float m) { return ref_of(m) + LIFT; }
// What a sum about the maximum m with the reference c is multiplied by, to be one about M >= m with C: from reference to
// reference as they are rounded. Where only one of the two is far, the other's product with L is rounded by up to 32 and has
// to be taken as it is, too.
__device__ __forceinline__ float rescale(float m, float c, float M, float C) {
    if (!far(m) && !far(M)) return ex2(c - C);
    return ex2(far(m) && far(M) ? fmaf(m - M, LOG2E, c - C) : far(M) ? fmaf(-M, LOG2E, c) - C : fmaf(m, LOG2E, -C) + c);
}
__device__ __forceinline__ void raise(Run& r, float m) {                            // from nothing: 0 times 0
    if (__any_sync(~0u, m > r.m + HEADROOM)) {
        if (m > r.m + HEADROOM) {
            const float c = run_ref(m);
            r.o *= rescale(r.m, r.c, m, c);
            r.m = m;
            r.c = c;
        }
    }
}
__device__ __forceinline__ void warp_join(Run& r) {
    const float m = warp_max(r.m), c = run_ref(m);
    r.o = warp_sum(r.m == m ? r.o : r.o * rescale(r.m, r.c, m, c));
    r.m = m;
    r.c = c;
}
// What the warps leave for the first warp at a row's end (those of all blocks of a cluster for the first warp of each), and
// it for them: two of each in turn, so that a row's is written again only behind the barrier of the row between, which a
// first warp reaches after reading it.
template <int NW>
struct Meeting {
    float2 run[2][NW];
    float xt[2];
    float4 grad[2];          // the maximum, the reference, the factor of a numerator and the target's derivative
    // writes v to the place `at` of this and, in a cluster, of every block's Meeting
    template <int C> __device__ __forceinline__ void tell(float& at, float v) {
        if constexpr (C == 1) {
            at = v;
        } else {
#pragma unroll
            for (int c = 0; c < C; c++) put(&at, c, v);
        }
    }
    static __device__ __forceinline__ void put(float* at, int block, float v) {
        uint32_t a;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(at)), "r"(block));
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory");
    }
};
__device__ __forceinline__ void cluster_barrier() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Ends a counted row: the threads' sums join, a first warp takes them to the row's log-probability, term and derivative.
template <int MODE, int NW, int C>
__device__ __forceinline__ float4 block_end(const Rows& k, Meeting<NW * C>& at, int turn, Run& run, const End& end, double w, float scale, int64_t r,
                                            bool grad, int rank) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    warp_join(run);
    if constexpr (NW * C == 1) {
        __syncwarp();
    } else if constexpr (C == 1) {
        if (lane == 0) at.run[turn][warp] = make_float2(run.m, run.o);
        __syncthreads();
    } else {
        if (lane < C) {
            float* to = (float*)&at.run[turn][rank * NW + warp];
            at.put(to, lane, run.m);
            at.put(to + 1, lane, run.o);
        }
        cluster_barrier();
    }
    if (warp == 0) {
        const float xt = at.xt[turn];                        // the sums leave the target out
        Run all = run;
        if constexpr (NW * C > 1) {
            static_assert(NW * C <= 32, "a lane a warp");
            all = Run();
            if (lane < NW * C) {
                const float2 v = at.run[turn][lane];
                all.m = v.x;
                all.c = run_ref(v.x);
                all.o = v.y;
            }
        }
        const float m = fmaxf(NW * C > 1 ? warp_max(all.m) : all.m, xt), c = ref_of(m), e = ex2(exponent(xt, m, c));
        all.o *= all.m == -INFINITY ? 0.f : rescale(all.m, all.c, m, c);       // NaN stays
        if (NW * C > 1) all.o = warp_sum(all.o);
        all.m = m;
        float term;
        const double lp = row_logp(all.m, all.o, xt, e);
        const float g = row_end<MODE>(k, end, lp, (float)w, scale, term);
        const float inv = reciprocal(all.o + e);
        if (lane == 0) {
            if (rank == 0) {
                if (MODE == LOGP && k.logp) k.logp[r] = (float)lp;
                if (k.stat) k.stat[r] = make_float4(all.m, c, inv, all.o * inv);
                if (MODE == POLICY && k.deriv) k.deriv[r] = g;
                if (k.part) k.part[r] = MODE == LOGP ? lp : (double)term * w;
            }
            if (grad) at.grad[turn] = make_float4(all.m, c, -g * inv, g * (all.o * inv));
        }
    }
    if (!grad) return make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (NW * C == 1) __syncwarp(); else __syncthreads();
    return at.grad[turn];
}

template <typename T>
__device__ __forceinline__ void zero_row(T* d, int V, int thread, int threads) {
    constexpr int K = K_OF<T>;
    const int off = row_off(d);
    float z[K];
#pragma unroll
    for (int q = 0; q < K; q++) z[q] = 0.f;
    for (int e0 = thread * K - off; e0 < V; e0 += threads * K) store_piece(d, e0, V, true, z);
}

template <typename T>
__device__ __forceinline__ void grad_piece(const uint4& raw, T* d, int e0, int V, bool same, const float4& g) {
    float x[K_OF<T>];
    unpack<T>(raw, x);
    less(x, far(g.x) ? g.x : 0.f);
    numerators(x, g.y);
    times(x, g.z);
    store_piece(d, e0, V, same, x);
}

// Rows that fit a ring of S steps in shared memory, U pieces a thread each. Every thread copies its own pieces in
// asynchronously and reads only those, so the copies need no barrier: the ring runs ahead into the next rows while this row
// is reduced, and a step's pieces leave it when the row's gradient has been formed from them. One copy group is committed
// for every step of either pass (an empty one where nothing is copied), so at least S - 1 groups lie behind the one that a
// step needs: between a step's copy and its use lie the S - 1 steps that were copied after it, or a whole pass more.
//
// Only whole pieces go through the ring. The elements before the first and behind the last (up to K - 1 each) are held by a
// lane each of the first warp.
//
// A row's target and place take tens of instructions, and every warp needs them: a warp works them out for 32 of its block's
// rows at once, a lane each, and hands them round by shuffles.
//
// C: blocks of a cluster that share a row, each a span of its pieces; they leave each other what their warps found in
// distributed shared memory, behind one cluster barrier a row.
//
// On a B200: log-probabilities of 32,768 rows of 16,384 bf16 words 197 us (5.5 TB/s), their gradient from kept statistics 357
// us (6.0 TB/s, read and written): bound by memory. The policy loss and gradient of 16,384 rows of 65,541 words 897 us (4.8
// TB/s): two 2^x and, counted, 16 instructions a word at 24 warps a multiprocessor, which wait on each other at a row's end
// (the most frequent stall), and take 51 % of the issue slots.
// Threads a row, the fewest that hold it, since each warp pays a row's overhead (16,380 rows of 4,101 words: 68 us with
// 32 threads, 85 with 64, 102 with 128; 8,192 of 16,384: 102 us with 128, 132 with 256). 128 threads have 16 pieces each, in four
// steps of four, the others' 18 in six of three: 8,192 rows of 16,384 words take 102 us in four steps and 104 in six, but
// of 16,389 words 132 us with 256 threads, where 128 in six steps would take 107. Pieces kept in registers between the
// passes, so that copies go on during both, lost to their warps' latency (16,384 words: 523 us, and 397 us from the ring).

// warps that a multiprocessor holds with P pieces a thread in the ring, 32 at most (64 registers a thread)
template <int P> constexpr int RING_WARPS = 220 * 1024 / (P * 512) < 32 ? 220 * 1024 / (P * 512) : 32;
template <typename T, int THREADS, int U, int S, int C, int MODE>
__global__ void __launch_bounds__(THREADS, RING_WARPS<S * U> / (THREADS / 32)) rows_ring_kernel(Rows k, int steps) {
    constexpr int K = K_OF<T>, SPAN = THREADS * K, NW = THREADS / 32;       // SPAN: elements from a thread's piece to its next
    extern __shared__ uint4 ring[];                          // [S][U][THREADS]
    __shared__ Meeting<NW * C> meet;
    const float scale = MODE != LOGP && k.scale ? *k.scale : 1.f;
    if (MODE != LOGP && k.skip_one && scale == 1.f) return;
    const int tid = threadIdx.x, lane = tid & 31, V = (int)k.b.V, rank = C > 1 ? (int)blockIdx.x % C : 0;
    const int64_t W = k.b.W, rows = k.b.n * W, stride = gridDim.x / C, first_row = blockIdx.x / C;
    // of a row's whole pieces this block has span `rank`
    const int p0 = tid + rank * steps * U * THREADS;         // this thread's first piece

    // 32 rows from `first` on, a lane each: window, position, target (-1 beyond the last row)
    struct Lot { int64_t i, t; int y; };
    const auto lot_of = [&](int64_t first) {
        const int64_t r = first + lane * stride;
        Lot q = {r / W, r % W, -1};
        if (r < rows) q.y = target(k.b, q.i, q.t);
        return q;
    };

    // what is copied next: step in_j of the lowest row in in_left, the counted ones of a lot, to in_to in the ring
    constexpr uint32_t STEP = U * THREADS * 16;
    const uint32_t ring_at = shared_at(ring + tid), ring_end = ring_at + S * STEP;
    int64_t in_first = first_row, in_at = 0;                 // in_at: a lane's row in the logits
    unsigned in_left = 0;
    const T* in_x = nullptr;                                 // this thread's next piece
    int in_j = 0, in_full = 0, in_n = 0;                     // the first steps whose pieces are all in the row; the row's whole pieces
    uint32_t in_to = ring_at;
    const auto full_of = [&](int n) { return n / (U * THREADS) - rank * steps; };
    const auto find = [&]() {
        while (!in_left && in_first < rows) {
            const Lot q = lot_of(in_first);
            in_left = __ballot_sync(~0u, q.y >= 0);
            in_at = q.i * k.b.logits_n + q.t * k.b.logits_w;
            in_first += 32 * stride;
        }
        if (in_left) {
            const T* x = (const T*)k.b.logits + __shfl_sync(~0u, in_at, __ffs(in_left) - 1);
            const int head = head_of(x, V);
            in_n = (V - head) / K;
            in_full = full_of(in_n);
            in_x = x + head + (int64_t)p0 * K;
        }
    };
    find();
    const auto copy_next = [&]() {
        if (in_left) {
            if (in_j < in_full) {
#pragma unroll
                for (int u = 0; u < U; u++) copy16(in_to + u * (THREADS * 16), in_x + u * SPAN);
            } else {
                const int p = p0 + in_j * U * THREADS;
#pragma unroll
                for (int u = 0; u < U; u++)
                    if (p + u * THREADS < in_n) copy16(in_to + u * (THREADS * 16), in_x + u * SPAN);
            }
            in_x += U * SPAN;
            if (++in_j == steps) {
                in_j = 0;
                in_left &= in_left - 1;
                find();
            }
        }
        in_to += STEP;
        if (in_to == ring_end) in_to = ring_at;
        copies_commit();
    };
#pragma unroll 1
    for (int s = 0; s < S; s++) copy_next();
    if (C > 1) cluster_barrier();                            // every block of the cluster runs before one writes to another

    uint4* const own_ring = ring + tid;
    uint4* slot = own_ring;                                  // the row's first step
    int turn = 0;
    for (int64_t first = first_row; first < rows; first += 32 * stride) {
        const Lot lot = lot_of(first);
        const int64_t x_at = lot.i * k.b.logits_n + lot.t * k.b.logits_w, d_at = lot.i * k.b.grad_n + lot.t * k.b.grad_w;
        End ends = {0.f, 0.f, 0.f};
        double ws = 1.0;
        float4 stats = make_float4(0.f, 0.f, 0.f, 0.f);      // as a Meeting's grad
        if ((MODE == GIVEN || tid < 32) && lot.y >= 0) {
            ends = end_args<MODE>(k, lot.i, lot.t);
            ws = weight_of<MODE>(k, lot.i);
            if (MODE == GIVEN) {
                const float4 v = k.stat[first + lane * stride];
                const float g = k.scaled ? ends.a : ends.a * scale;
                stats = make_float4(v.x, v.y, -g * v.z, g * v.w);
            }
        }
        for (int l = 0; l < 32; l++) {
            const int64_t r = first + l * stride;
            if (r >= rows) break;
            const int y = __shfl_sync(~0u, lot.y, l);
            T* const d = MODE != LOGP && k.b.grad ? (T*)k.b.grad + __shfl_sync(~0u, d_at, l) : nullptr;
            if (y < 0) {
                if (rank == 0) {
                    if (MODE == LOGP && k.logp && tid == 0) k.logp[r] = 0.f;
                    if (k.part && tid == 0) k.part[r] = 0;
                }
                if (MODE != LOGP && d) zero_row(d, V, tid + rank * THREADS, C * THREADS);
                continue;
            }
            const T* const x = (const T*)k.b.logits + __shfl_sync(~0u, x_at, l);
            const bool grad = MODE != LOGP && d;
            const int head = head_of(x, V), n = (V - head) / K, tail = head + n * K;
            // an element at the row's ends
            int edge = -1;
            float ex = -INFINITY;
            if (tid < 32 && rank == 0) {
                edge = lane < head ? lane : lane >= 8 && tail + lane - 8 < V ? tail + lane - 8 : -1;
                if (edge >= 0) ex = f32(x[edge]);
            }
            // the target's piece, where it is this thread's: its step and its place in the ring's step
            int own_j = -1, own_u = 0;
            if (y >= head && y < tail) {
                const int q = (y - head) / K - p0;
                if (q >= 0 && q % THREADS == 0 && q < steps * U * THREADS) { own_j = q / (THREADS * U); own_u = q / THREADS % U; }
            }
            uint4* from = slot;
            const auto on = [&]() {
                from += U * THREADS;
                if (from == own_ring + S * U * THREADS) from = own_ring;
            };
            const int full = full_of(n);
            float4 g;
            if constexpr (MODE == GIVEN) {
                g = make_float4(__shfl_sync(~0u, stats.x, l), __shfl_sync(~0u, stats.y, l), __shfl_sync(~0u, stats.z, l), __shfl_sync(~0u, stats.w, l));
            } else {
                Run run;
#pragma unroll 1
                for (int j = 0; j < steps; j++) {
                    copies_wait<S - 1>();
                    if (j == own_j) {                        // the target's logit out of the ring, -inf in its place
                        T* own = (T*)(from + own_u * THREADS) + (y - head) % K;
                        meet.template tell<C>(meet.xt[turn], f32(*own));
                        *own = lowest<T>();
                    }
                    // Q pieces of this thread, the u-th on
                    const auto pieces = [&](auto Q, int u) {
                        constexpr int q = decltype(Q)::value;
                        uint4 raw[q];
#pragma unroll
                        for (int h = 0; h < q; h++) {
                            raw[h] = make_uint4(Traits<T>::LOW, Traits<T>::LOW, Traits<T>::LOW, Traits<T>::LOW);
                            if (q > 1 || p0 + (j * U + u) * THREADS < n) raw[h] = from[(u + h) * THREADS];
                        }
                        const float m = pieces_max<T>(raw);
                        bool plain = true;
                        if (__any_sync(~0u, m > run.m + HEADROOM || far(run.m))) {
                            raise(run, m);
                            plain = !__any_sync(~0u, far(run.m));
                        }
                        if (plain) {
                            run.o = sum_all<T, q>(raw, run.c, run.o);
                        } else {                             // a maximum beyond 2^29, or none yet
                            const float by = far(run.m) && run.m != -INFINITY ? run.m : 0.f;
#pragma unroll 1
                            for (int h = 0; h < q; h++)
                                if (p0 + (j * U + u + h) * THREADS < n) run.o = sum_far<T, 1>(from + (u + h) * THREADS, 0, by, run.c, run.o);
                        }
                    };
                    if (j < full) {
                        pieces(std::integral_constant<int, U>(), 0);
                    } else {                                 // one at a time, while any thread has one
#pragma unroll 1
                        for (int u = 0; u < U && p0 - tid + (j * U + u) * THREADS < n; u++) pieces(std::integral_constant<int, 1>(), u);
                    }
                    on();
                    if (grad) copies_commit(); else copy_next();
                }
                End end = {0.f, 0.f, 0.f};
                double w = 1.0;
                if (tid < 32) {
                    float v = ex;
                    if (edge == y) {
                        meet.template tell<C>(meet.xt[turn], ex);
                        v = -INFINITY;
                    }
                    raise(run, v);
                    if (!(v == -INFINITY)) run.o += ex2(exponent(v, run.m, run.c));
                    if (MODE == POLICY) {
                        end.a = __shfl_sync(~0u, ends.a, l);
                        end.old = __shfl_sync(~0u, ends.old, l);
                        end.ref = __shfl_sync(~0u, ends.ref, l);
                        w = __shfl_sync(~0u, ws, l);
                    }
                }
                g = block_end<MODE, NW, C>(k, meet, turn, run, end, w, scale, r, grad, rank);
                turn ^= 1;
                if (grad) from = slot;
            }
            if (grad) {
                const bool plain = alike(x, d) && !far(g.x);
                T* to = d + head + (int64_t)p0 * K;
#pragma unroll 1
                for (int j = 0; j < steps; j++, to += U * SPAN) {
                    if (MODE == GIVEN) copies_wait<S - 1>();
                    const auto piece = [&](int u) {
                        float v[K];
                        unpack<T>(from[u * THREADS], v);
                        numerators(v, g.y);
                        times(v, g.z);
                        *(uint4*)(to + u * SPAN) = pack<T>(v);
                    };
                    if (plain && j < full) {
#pragma unroll
                        for (int u = 0; u < U; u++) piece(u);
                    } else {
#pragma unroll 1
                        for (int u = 0; u < U; u++) {
                            const int p = p0 + (j * U + u) * THREADS;
                            if (p >= n) break;
                            if (plain) piece(u);
                            else grad_piece(from[u * THREADS], d, head + p * K, V, alike(x, d), g);
                        }
                    }
                    if (j == own_j) d[y] = from32<T>(g.w);
                    on();
                    copy_next();
                }
                if (edge >= 0) d[edge] = from32<T>(edge == y ? g.w : g.z * ex2(exponent(ex, g.x, g.y)));
            }
            slot = from;
        }
    }
    copies_wait<0>();
}

// ---------------------------------------------------------------- small kernels around the rows
__device__ double block_sum(double v) {                      // every thread of the block gets it
    __shared__ double sh[33];
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x < 32) {
        double w = threadIdx.x < (blockDim.x >> 5) ? sh[threadIdx.x] : 0.0;
        w = warp_sum(w);
        if (threadIdx.x == 0) sh[32] = w;
    }
    __syncthreads();
    return sh[32];
}

// the sums of each window's tiles: a warp a window up to SUMS_WARP tiles, else a block
constexpr int SUMS_WARP = 512;
__global__ void __launch_bounds__(1024) window_sums_kernel(const double* part, int64_t n, int64_t tpw, float* sums, double* sums64) {
    const bool warp = tpw <= SUMS_WARP;
    const int first = warp ? threadIdx.x & 31 : threadIdx.x, step = warp ? 32 : 1024;
    for (int64_t i = warp ? (int64_t)blockIdx.x * 32 + (threadIdx.x >> 5) : blockIdx.x; i < n; i += warp ? (int64_t)gridDim.x * 32 : gridDim.x) {
        double v = 0;
#pragma unroll 8
        for (int64_t j = first; j < tpw; j += step) v += part[i * tpw + j];
        v = warp ? warp_sum(v) : block_sum(v);
        if (first == 0) {
            if (sums) sums[i] = (float)v;
            if (sums64) sums64[i] = v;
        }
    }
}

// a block per FOLD of `count` partial sums
constexpr int FOLD = 4096;
__global__ void __launch_bounds__(256) fold_kernel(const double* part, int64_t count, double* out) {
    double v = 0;
#pragma unroll
    for (int u = 0; u < FOLD / 256; u++) {
        const int64_t j = (int64_t)blockIdx.x * FOLD + u * 256 + threadIdx.x;
        if (j < count) v += part[j];
    }
    v = block_sum(v);
    if (threadIdx.x == 0) out[blockIdx.x] = v;
}
// one block: the sum of `count` partial sums
__global__ void __launch_bounds__(1024) total_kernel(const double* part, int64_t count, float* out) {
    double v = 0;
#pragma unroll 8
    for (int64_t j = threadIdx.x; j < count; j += 1024) v += part[j];
    v = block_sum(v);
    if (threadIdx.x == 0) *out = (float)v;
}

// one block: the pairs' margins, loss and derivatives from the windows' sums, which lie in `tpw` parts each (summed into
// `sums` first, a warp a window, where tpw is not 1)
__global__ void __launch_bounds__(1024) pairs_kernel(const double* part, int64_t tpw, double* sums, int64_t n, const float* ref, int64_t ref_n,
                                                     float beta, float eps, float* loss, float* margins, float* coef) {
    const int64_t m = n / 2;
    if (tpw != 1) {
        for (int64_t i = threadIdx.x >> 5; i < n; i += 32) {
            double v = 0;
#pragma unroll 8
            for (int64_t j = threadIdx.x & 31; j < tpw; j += 32) v += part[i * tpw + j];
            v = warp_sum(v);
            if ((threadIdx.x & 31) == 0) sums[i] = v;
        }
        __syncthreads();
        part = sums;
    }
    double all = 0;
    for (int64_t j = threadIdx.x; j < m; j += blockDim.x) {
        const double gap = (part[j] - (double)ref[j * ref_n]) - (part[j + m] - (double)ref[(j + m) * ref_n]);
        const double h = (double)beta * gap;
        // log sigmoid(h) = min(h, 0) - log1p(exp(-|h|))
        const double l = log1p(exp(-fabs(h))), up = fmin(h, 0.0) - l, down = fmin(-h, 0.0) - l;
        all += h != h ? h : -(eps == 1.f ? 0.0 : (1.0 - eps) * up) - (eps == 0.f ? 0.0 : eps * down);   // 0 of an infinite term is 0
        if (margins) margins[j] = (float)gap;
        const double c = (double)beta / (double)m * ((double)eps - 1.0 / (1.0 + exp(h)));
        coef[j] = (float)c;
        coef[j + m] = (float)-c;
    }
    all = block_sum(all);
    if (threadIdx.x == 0) *loss = m ? (float)(all / (double)m) : 0.f;
}

// Counted positions of each window, turned into weights: up to COUNT_ONE positions by one block, a warp a window (4,072
// positions 7 us; 16,384 take it 36 us); more by a warp per (window, span of it) first (16,384 positions 3 us and 3).
constexpr int COUNT_SPAN = 256, COUNT_ONE = 4096;
// this lane's part of the counted positions [t0, t0 + COUNT_SPAN) of window i: eight tokens and masks in flight
template <typename Token, typename Mask>
__device__ __forceinline__ int count_span(const pv_scored& b, int64_t i, int64_t t0, int lane) {
    constexpr bool MASK = !std::is_void<Mask>::value;
    using M = typename std::conditional<MASK, Mask, uint8_t>::type;
    const Token* tokens = (const Token*)b.tokens + i * b.tokens_n;
    const M* mask = (const M*)b.mask + i * b.mask_n;
    Token y[8];
    M m[8];
    bool in[8];
#pragma unroll
    for (int u = 0; u < 8; u++) {
        const int64_t at = t0 + u * 32 + lane + b.shift, from = at < b.W ? at : 0;
        in[u] = at < b.W;
        y[u] = tokens[from * b.tokens_w];
        if (MASK) m[u] = mask[from * b.mask_w];
    }
    int v = 0;
#pragma unroll
    for (int u = 0; u < 8; u++) {
        const int64_t w = y[u];
        v += in[u] && w >= 0 && w < b.V && w != b.ignore && (!MASK || m[u] != (M)0);
    }
    return v;
}
__global__ void __launch_bounds__(256) count_kernel(pv_scored b, int64_t spans, int32_t* counts) {
    const int lane = threadIdx.x & 31;
    for (int64_t q = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); q < b.n * spans; q += (int64_t)gridDim.x * 8) {
        const int64_t i = q / spans, t0 = (q - i * spans) * COUNT_SPAN;
        int v;
        if (b.token_bytes == 1)
            v = b.mask_bytes == 0 ? count_span<uint8_t, void>(b, i, t0, lane) : b.mask_bytes == 1 ? count_span<uint8_t, uint8_t>(b, i, t0, lane)
                                                                                               : count_span<uint8_t, float>(b, i, t0, lane);
        else
            v = b.mask_bytes == 0 ? count_span<int64_t, void>(b, i, t0, lane) : b.mask_bytes == 1 ? count_span<int64_t, uint8_t>(b, i, t0, lane)
                                                                                               : count_span<int64_t, float>(b, i, t0, lane);
        v = (int)__reduce_add_sync(~0u, (unsigned)v);
        if (lane == 0) counts[q] = v;
    }
}
__global__ void __launch_bounds__(1024) weights_kernel(pv_scored b, const int32_t* counts, int64_t spans, int by_window, double scale,
                                                       double* weight) {
    double all = 0, some = 0;
    const int64_t n = b.n;
    const int lane = threadIdx.x & 31;
    if (counts && spans <= 32) {                             // a thread a window
#pragma unroll 4
        for (int64_t i = threadIdx.x; i < n; i += 1024) {
            int c = 0;
            for (int64_t j = 0; j < spans; j++) c += counts[i * spans + j];
            weight[i] = (double)c;
            all += (double)c;
            some += c > 0;
        }
    } else {
        for (int64_t i = threadIdx.x >> 5; i < n; i += 32) {
            int c = 0;
            if (counts) {
                for (int64_t j = lane; j < spans; j += 32) c += counts[i * spans + j];
            } else {
#pragma unroll 4
                for (int64_t t = lane; t < b.W; t += 32) c += target(b, i, t) >= 0;
            }
            c = (int)__reduce_add_sync(~0u, (unsigned)c);
            if (lane == 0) { weight[i] = (double)c; all += (double)c; some += c > 0; }
        }
    }
    all = block_sum(all);
    some = block_sum(some);
    for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
        const double c = weight[i];
        weight[i] = by_window ? (c > 0 ? scale / (c * some) : 0.0) : (all > 0 ? scale / all : 0.0);
    }
}

// ---------------------------------------------------------------- host
int fail(int code, const char* what) {
    snprintf(g_cuda_err, sizeof g_cuda_err, "%s", what);
    return code;
}
int launched() {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? PV_OK : fail(PV_ECUDA, cudaGetErrorString(e));
}

bool off(const void* p, int bytes) { return (uintptr_t)p % bytes != 0; }       // an address not aligned to its type

const char* bad_batch(const pv_scored* b) {
    if (!b) return "batch: NULL";
    // scratch, statistics and offsets are up to 32 bytes a position and 16 a window: no size below wraps round in 64 bits
    if (b->n < 0 || b->n > (1ll << 56) || b->W < 0 || b->W >= (1ll << 31) || b->V < 1 || b->V >= (1ll << 30)) return "batch: n, W or V out of range";
    if (b->shift < 0) return "batch: shift is negative";
    if (b->type < PV_T_BF16 || b->type > PV_T_FP32) return "batch: logits are bf16, fp16 or fp32";
    if (b->token_bytes != 1 && b->token_bytes != 8) return "batch: tokens are uint8 or int64";
    if (b->mask_bytes != 0 && b->mask_bytes != 1 && b->mask_bytes != 4) return "batch: the mask is uint8 or float";
    if (b->n > 0 && b->W > 0 && (!b->logits || !b->tokens || (b->mask_bytes && !b->mask))) return "batch: NULL logits, tokens or mask";
    if (b->n > 0 && b->W > (1ll << 56) / b->n) return "batch: n W is too large";
    const int size = b->type == PV_T_FP32 ? 4 : 2;
    if (off(b->logits, size) || off(b->grad, size) || off(b->tokens, b->token_bytes) || (b->mask_bytes && off(b->mask, b->mask_bytes)))
        return "batch: an address is not aligned to its type";
    return nullptr;
}

// How a batch is run, by its rows' 16-byte pieces (one more than their bytes say where a row may start inside one):
// up to 256 in registers, G lanes a row; more through a ring in shared memory. Where the policy loss is to give a gradient
// a row has to fit the ring (RING_MOST); longer ones it reads twice, the second time with their statistics at hand (131,072
// bf16 words a row, 2,048 rows: 295 us, and 342 us by clusters of four blocks that hold a row; 65,541: 1,115 us and 890).
// Rows of up to 136 words (32 bits) that do not start at 16-byte boundaries, but lie one behind the other, are copied as
// stretches (262,144 rows of 259 bf16 words: log-probabilities in 55 us that way and in 73 us with 16 lanes a row and the
// ends by themselves; longer ones fill more lanes, 131,072 rows of 1,003: 87 us with 32 lanes a row).
enum { FLAT_ROWS, SHORT_ROWS, RING_ROWS, LONG_ROWS };
constexpr int RING = 18;                                 // pieces a thread
struct Plan { int form, pieces; bool aligned; int64_t tpw, tiles, spans; };
constexpr int RING_MOST = 512 * RING;                    // two blocks of 256 threads
int size_of(int type) { return type == PV_T_FP32 ? 4 : 2; }
// every row starts at a 16-byte boundary
bool whole_pieces(const void* p, int64_t n, int64_t w, int64_t size) {
    return (((uintptr_t)p | (uint64_t)(n * size) | (uint64_t)(w * size)) & 15) == 0;
}
Plan plan_of(const pv_scored& b) {
    Plan p;
    const int64_t size = size_of(b.type), k = 16 / size;
    p.aligned = whole_pieces(b.logits, b.logits_n, b.logits_w, size);
    const int64_t pieces = (b.V + k - 1 + (p.aligned ? 0 : k - 1)) / k;
    p.pieces = (int)std::min<int64_t>(pieces, 1 << 30);
    const int64_t words = b.type == PV_T_FP32 ? b.V : b.V / 2 + 1;
    const bool whole = p.aligned && b.V % k == 0;
    const bool flat = !whole && words <= 136 && b.logits_w == b.V &&
                      (!b.grad || (b.grad_w == b.V && (((uintptr_t)b.logits ^ (uintptr_t)b.grad) & 15) == 0 && ((b.logits_n - b.grad_n) * size & 15) == 0));
    p.form = flat ? FLAT_ROWS : pieces <= 256 ? SHORT_ROWS : pieces <= RING_MOST ? RING_ROWS : LONG_ROWS;
    p.tpw = p.form <= SHORT_ROWS ? (b.W + TILE - 1) / TILE : b.W;
    p.tiles = b.n * p.tpw;
    p.spans = (b.W + COUNT_SPAN - 1) / COUNT_SPAN;
    return p;
}
// scratch: a double per tile, a double per window (and per FOLD tiles), an int per (window, span); the policy loss of long rows: their statistics
// and derivatives
struct Scratch { double *part, *win; float4* stat; float* deriv; int32_t* counts; size_t bytes; };
Scratch scratch_of(const pv_scored& b, const Plan& p, void* work) {
    Scratch s;
    char* at = (char*)work;
    s.bytes = 0;
    const auto take = [&](size_t n) { char* r = at + s.bytes; s.bytes += (n + 15) / 16 * 16; return r; };
    s.part = (double*)take((size_t)p.tiles * 8);
    s.win = (double*)take(std::max<size_t>((size_t)b.n, ((size_t)p.tiles + FOLD - 1) / FOLD) * 8);
    s.counts = (int32_t*)take((size_t)b.n * p.spans * 4);
    const size_t rows = p.form == LONG_ROWS ? (size_t)b.n * b.W : 0;
    s.stat = (float4*)take(rows * 16);
    s.deriv = (float*)take(rows * 4);
    return s;
}
// a persistent grid: as many blocks as are resident, at most one per `per_block` of the work
template <typename F>
unsigned grid_of(F* f, int threads, size_t smem, int64_t blocks) {
    int per_sm = 1;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, f, threads, smem) != cudaSuccess || per_sm < 1) per_sm = 1;
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>(blocks, (int64_t)SMS * per_sm));
}

// a kernel's dynamic shared memory, set once per thread and device
int allow_smem(const void* f, int bytes, uint64_t& set) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64 || !(set >> dev & 1)) {
        cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (dev < 64) set |= 1ull << dev;
    }
    return bytes;
}

Rows by_tiles(Rows k, unsigned grid) {
    k.stride = (int64_t)grid * WARPS;
    k.stride_n = k.stride / k.tpw;
    k.stride_t = (int32_t)(k.stride % k.tpw);
    return k;
}
template <typename T, int G, int NV, int MODE, bool A>
void group_rows(const Rows& k, cudaStream_t st) {
    constexpr int S = NV <= 4 ? 3 : 2, SMEM = WARPS * S * (NV * 512 + 128);
    const auto f = rows_group_kernel<T, G, NV, S, MODE, A>;
    static thread_local uint64_t set = 0;
    allow_smem((const void*)f, SMEM, set);
    static const unsigned most = grid_of(f, WARPS * 32, SMEM, 1 << 20);
    const unsigned grid = (unsigned)std::min<int64_t>((k.b.n * k.tpw + WARPS - 1) / WARPS, most);
    f<<<grid, WARPS * 32, SMEM, st>>>(by_tiles(k, grid));
}

template <typename T, int THREADS, int U, int S, int C, int MODE>
void ring_rows(const Rows& k, int pieces, cudaStream_t st) {
    constexpr int SMEM = S * U * THREADS * 16;
    const auto f = rows_ring_kernel<T, THREADS, U, S, C, MODE>;
    static thread_local uint64_t set = 0;
    allow_smem((const void*)f, SMEM, set);
    static const unsigned most = grid_of(f, THREADS, SMEM, 1 << 20);
    const int steps = (pieces + C * U * THREADS - 1) / (C * U * THREADS);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)std::min<int64_t>(k.b.n * k.b.W, most / C) * C);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = C > 1 ? 1 : 0;
    cudaLaunchKernelEx(&cfg, f, k, steps);
}

template <typename T, int G, int NW, int MODE>
void flat_rows(const Rows& k, cudaStream_t st) {
    constexpr int S = 3, SMEM = WARPS * S * (((NW * 32 * 4 + 47) / 16) * 16 + 128);
    const auto f = rows_flat_kernel<T, G, NW, S, MODE>;
    static thread_local uint64_t set = 0;
    allow_smem((const void*)f, SMEM, set);
    static const unsigned most = grid_of(f, WARPS * 32, SMEM, 1 << 20);
    const unsigned grid = (unsigned)std::min<int64_t>((k.b.n * k.tpw + WARPS - 1) / WARPS, most);
    f<<<grid, WARPS * 32, SMEM, st>>>(by_tiles(k, grid));
}

template <typename T, int MODE>
void short_rows(const Rows& k, const Plan& p, cudaStream_t st) {
    const bool whole = p.aligned && k.b.V % K_OF<T> == 0 && (!k.b.grad || whole_pieces(k.b.grad, k.b.grad_n, k.b.grad_w, sizeof(T)));
    if (p.form == FLAT_ROWS) {
        const int words = sizeof(T) == 4 ? (int)k.b.V : (int)k.b.V / 2 + 1;
        if (words <= 4) flat_rows<T, 1, 4, MODE>(k, st);
        else if (words <= 8) flat_rows<T, 1, 8, MODE>(k, st);
        else if (words <= 12) flat_rows<T, 1, 12, MODE>(k, st);
        else if (words <= 17) flat_rows<T, 1, 17, MODE>(k, st);
        else if (words <= 24) flat_rows<T, 2, 12, MODE>(k, st);
        else if (words <= 34) flat_rows<T, 2, 17, MODE>(k, st);
        else if (words <= 48) flat_rows<T, 4, 12, MODE>(k, st);
        else if (words <= 68) flat_rows<T, 4, 17, MODE>(k, st);
        else if (words <= 96) flat_rows<T, 8, 12, MODE>(k, st);
        else flat_rows<T, 8, 17, MODE>(k, st);
    } else if (!whole) {
        if (p.pieces <= 16) group_rows<T, 16, 1, MODE, false>(k, st);
        else if (p.pieces <= 32) group_rows<T, 16, 2, MODE, false>(k, st);
        else if (p.pieces <= 48) group_rows<T, 16, 3, MODE, false>(k, st);
        else if (p.pieces <= 64) group_rows<T, 16, 4, MODE, false>(k, st);
        else if (p.pieces <= 96) group_rows<T, 32, 3, MODE, false>(k, st);
        else if (p.pieces <= 128) group_rows<T, 32, 4, MODE, false>(k, st);
        else if (p.pieces <= 192) group_rows<T, 32, 6, MODE, false>(k, st);
        else group_rows<T, 32, 8, MODE, false>(k, st);
    } else if (p.pieces <= 1) group_rows<T, 1, 1, MODE, true>(k, st);
    else if (p.pieces <= 2) group_rows<T, 1, 2, MODE, true>(k, st);
    else if (p.pieces <= 4) group_rows<T, 1, 4, MODE, true>(k, st);
    else if (p.pieces <= 8) group_rows<T, 2, 4, MODE, true>(k, st);
    else if (p.pieces <= 12) group_rows<T, 4, 3, MODE, true>(k, st);
    else if (p.pieces <= 16) group_rows<T, 4, 4, MODE, true>(k, st);
    else if (p.pieces <= 24) group_rows<T, 8, 3, MODE, true>(k, st);
    else if (p.pieces <= 32) group_rows<T, 8, 4, MODE, true>(k, st);
    else if (p.pieces <= 48) group_rows<T, 16, 3, MODE, true>(k, st);
    else if (p.pieces <= 64) group_rows<T, 16, 4, MODE, true>(k, st);
    else if (p.pieces <= 96) group_rows<T, 32, 3, MODE, true>(k, st);
    else if (p.pieces <= 128) group_rows<T, 32, 4, MODE, true>(k, st);
    else if (p.pieces <= 192) group_rows<T, 32, 6, MODE, true>(k, st);
    else group_rows<T, 32, 8, MODE, true>(k, st);
}

template <typename T, int MODE>
void typed_rows(const Rows& k, const Plan& p, cudaStream_t st) {
    if (p.form <= SHORT_ROWS) {
        if constexpr (MODE != GIVEN) short_rows<T, MODE>(k, p, st);
    } else if (MODE == POLICY && k.b.grad) {
        if constexpr (MODE == POLICY) {
            if (p.pieces <= 32 * RING) ring_rows<T, 32, 4, 5, 1, MODE>(k, p.pieces, st);
            else if (p.pieces <= 64 * RING) ring_rows<T, 64, 3, 6, 1, MODE>(k, p.pieces, st);
            else if (p.pieces <= 128 * 16) ring_rows<T, 128, 4, 4, 1, MODE>(k, p.pieces, st);
            else if (p.pieces <= 256 * RING) ring_rows<T, 256, 3, 6, 1, MODE>(k, p.pieces, st);
            else ring_rows<T, 256, 3, 6, 2, MODE>(k, p.pieces, st);
        }
    } else if constexpr (MODE != GRAD) {
        // read once, a row need not fit the ring: a warp a row where the rows fill the GPU with 16 warps a multiprocessor
        // (16,380 rows of 4,101 words: 41 us, four warps a row 67; 8,192 of 16,384: 55 and 56), else four warps or sixteen
        const int64_t rows = k.b.n * k.b.W;
        if (rows >= SMS * 16) ring_rows<T, 32, MODE == GIVEN ? 4 : 6, MODE == GIVEN ? 3 : 2, 1, MODE>(k, p.pieces, st);
        else if (rows >= SMS * 4) ring_rows<T, 128, 4, 3, 1, MODE>(k, p.pieces, st);
        else ring_rows<T, 512, 4, 3, 1, MODE>(k, p.pieces, st);
    }
}

template <int MODE>
int launch_rows(const Rows& k, const Plan& p, cudaStream_t st) {
    if (k.b.n == 0 || k.b.W == 0) return PV_OK;
    switch (k.b.type) {
        case PV_T_BF16: typed_rows<__nv_bfloat16, MODE>(k, p, st); break;
        case PV_T_FP16: typed_rows<__half, MODE>(k, p, st); break;
        default: typed_rows<float, MODE>(k, p, st);
    }
    return launched();
}

Rows rows_of(const pv_scored& b, const Plan& p) {
    Rows k = {};
    k.b = b;
    k.tpw = p.tpw;
    return k;
}

int check_work(const Scratch& s, const void* work, size_t have) {
    if (s.bytes && (!work || have < s.bytes || ((uintptr_t)work & 15))) return fail(PV_EARG, "scratch: too small, NULL or not 16-byte aligned");
    return PV_OK;
}

int window_sums(const Plan& p, int64_t n, const double* part, float* sums, double* sums64, cudaStream_t st) {
    const int64_t blocks = p.tpw <= SUMS_WARP ? (n + 31) / 32 : n;
    window_sums_kernel<<<(unsigned)std::min<int64_t>(blocks, SMS * 2), 1024, 0, st>>>(part, n, p.tpw, sums, sums64);
    return launched();
}

bool finite(float v) { return v >= 0.f && v < INFINITY; }

int bad_policy(const pv_scored* b, const pv_policy_args* a) {
    if (!a) return fail(PV_EARG, "pv_policy: NULL arguments");
    if (!finite(a->scale)) return fail(PV_EARG, "pv_policy: scale is negative or not finite");
    if (!finite(a->clip_low) || !finite(a->clip_high)) return fail(PV_EARG, "pv_policy: clip is negative or not finite");
    if (!finite(a->kl)) return fail(PV_EARG, "pv_policy: kl is negative or not finite");
    if (off(a->old, 4) || off(a->adv, 4) || off(a->ref, 4)) return fail(PV_EARG, "pv_policy: an address is not aligned to float");
    if (a->kl != 0.f && !a->ref && b->n && b->W) return fail(PV_EARG, "pv_policy: a KL term without reference log-probabilities");
    return PV_OK;
}

int policy_rows(const pv_scored* b, const pv_policy_args* a, const Plan& p, const Scratch& s, double* part, const double* weight, const float* scale,
                       int skip_one, cudaStream_t st) {
    Rows k = rows_of(*b, p);
    k.part = part;
    k.a = *a;
    k.weight = weight;
    k.scale = scale; k.skip_one = scale && skip_one;
    if (!b->grad || p.form != LONG_ROWS) return launch_rows<POLICY>(k, p, st);
    k.b.grad = nullptr;
    k.stat = s.stat;
    k.deriv = s.deriv;
    if (const int e = launch_rows<POLICY>(k, p, st)) return e;
    Rows q = rows_of(*b, p);
    q.stat = s.stat;
    q.up = s.deriv; q.up_n = b->W; q.up_w = 1;
    q.scale = scale; q.skip_one = k.skip_one; q.scaled = 1;
    return launch_rows<GIVEN>(q, p, st);
}

}  // namespace

extern "C" {

size_t pv_score_work_bytes(const pv_scored* b) {
    if (bad_batch(b)) return 0;
    return scratch_of(*b, plan_of(*b), nullptr).bytes;
}

size_t pv_score_stat_bytes(const pv_scored* b) {
    if (bad_batch(b) || plan_of(*b).form <= SHORT_ROWS) return 0;
    return (size_t)b->n * b->W * sizeof(float4);
}

int pv_logprobs(const pv_scored* b, float* logp, float* sums, void* stat, void* work, size_t work_bytes, void* stream) {
    if (const char* why = bad_batch(b)) return fail(PV_EARG, why);
    const Plan p = plan_of(*b);
    const Scratch s = scratch_of(*b, p, work);
    if (sums && check_work(s, work, work_bytes)) return PV_EARG;
    if (off(logp, 4) || off(sums, 4) || off(stat, 16)) return fail(PV_EARG, "pv_logprobs: an address is not aligned (float, stat to 16 bytes)");
    if (b->n == 0) return PV_OK;
    Rows k = rows_of(*b, p);
    k.b.grad = nullptr;
    k.logp = logp;
    k.stat = (float4*)stat;
    k.part = sums ? s.part : nullptr;
    const cudaStream_t st = (cudaStream_t)stream;
    if (const int e = launch_rows<LOGP>(k, p, st)) return e;
    return sums ? window_sums(p, b->n, s.part, sums, nullptr, st) : PV_OK;
}

int pv_logprobs_grad(const pv_scored* b, const float* up, int64_t up_n, int64_t up_w, const void* stat, const float* scale, void* stream) {
    if (const char* why = bad_batch(b)) return fail(PV_EARG, why);
    if (b->n == 0 || b->W == 0) return PV_OK;
    if (!b->grad || !up) return fail(PV_EARG, "pv_logprobs_grad: NULL gradient");
    if (off(up, 4) || off(scale, 4)) return fail(PV_EARG, "pv_logprobs_grad: an address is not aligned to float");
    const Plan p = plan_of(*b);
    if (p.form > SHORT_ROWS && (!stat || ((uintptr_t)stat & 15))) return fail(PV_EARG, "pv_logprobs_grad: rows of this length need their statistics");
    Rows k = rows_of(*b, p);
    k.up = up; k.up_n = up_n; k.up_w = up_w;
    k.stat = (float4*)stat;
    k.scale = scale;
    return p.form <= SHORT_ROWS ? launch_rows<GRAD>(k, p, (cudaStream_t)stream) : launch_rows<GIVEN>(k, p, (cudaStream_t)stream);
}

int pv_preference(const pv_scored* b, const float* ref, int64_t ref_n, float beta, float smoothing, float* loss, float* margins, float* coef,
                  void* stat, void* work, size_t work_bytes, void* stream) {
    if (const char* why = bad_batch(b)) return fail(PV_EARG, why);
    if (b->n & 1) return fail(PV_EARG, "pv_preference: an odd number of windows");
    if (!finite(beta)) return fail(PV_EARG, "pv_preference: beta is negative or not finite");
    if (!(smoothing >= 0.f && smoothing <= 1.f)) return fail(PV_EARG, "pv_preference: smoothing is not in [0, 1]");
    if (!loss || (b->n && (!ref || !coef))) return fail(PV_EARG, "pv_preference: NULL argument");
    if (off(ref, 4) || off(loss, 4) || off(margins, 4) || off(coef, 4) || off(stat, 16))
        return fail(PV_EARG, "pv_preference: an address is not aligned (float, stat to 16 bytes)");
    const Plan p = plan_of(*b);
    const Scratch s = scratch_of(*b, p, work);
    if (check_work(s, work, work_bytes)) return PV_EARG;
    const cudaStream_t st = (cudaStream_t)stream;
    if (b->n) {
        Rows k = rows_of(*b, p);
        k.b.grad = nullptr;
        k.part = s.part;
        k.stat = (float4*)stat;
        if (const int e = launch_rows<LOGP>(k, p, st)) return e;
    }
    // up to 4,096 parts the one block adds itself (3 us; 32,768 take it 12 us), more a block a window before it (4 us and 3)
    int64_t parts = p.tpw;
    const double* from = s.part;
    if (p.tiles > 4096) {
        if (const int e = window_sums(p, b->n, s.part, nullptr, s.win, st)) return e;
        parts = 1;
        from = s.win;
    }
    pairs_kernel<<<1, 1024, 0, st>>>(from, parts, s.win, b->n, ref, ref_n, beta, smoothing, loss, margins, coef);
    return launched();
}

int pv_policy(const pv_scored* b, const pv_policy_args* a, float* loss, double* weight, void* work, size_t work_bytes, void* stream) {
    if (const char* why = bad_batch(b)) return fail(PV_EARG, why);
    if (const int e = bad_policy(b, a)) return e;
    if (!loss || (b->n && !weight) || (b->n && b->W && (!a->old || !a->adv))) return fail(PV_EARG, "pv_policy: NULL argument");
    if (off(loss, 4) || off(weight, 8)) return fail(PV_EARG, "pv_policy: an address is not aligned (loss float, weight double)");
    const Plan p = plan_of(*b);
    const Scratch s = scratch_of(*b, p, work);
    if (check_work(s, work, work_bytes)) return PV_EARG;
    const cudaStream_t st = (cudaStream_t)stream;
    if (b->n) {
        const bool one = b->n * b->W <= COUNT_ONE;
        if (!one) count_kernel<<<(unsigned)std::min<int64_t>((b->n * p.spans + 7) / 8, SMS * 8), 256, 0, st>>>(*b, p.spans, s.counts);
        weights_kernel<<<1, 1024, 0, st>>>(*b, one ? nullptr : s.counts, p.spans, a->by_window, (double)a->scale, weight);
        if (const int e = launched()) return e;
        if (const int e = policy_rows(b, a, p, s, s.part, weight, nullptr, 0, st)) return e;
    }
    // up to 16,384 parts one block adds at once (3 us), more after a block has added each FOLD of them
    if (p.tiles <= 4 * FOLD) {
        total_kernel<<<1, 1024, 0, st>>>(s.part, p.tiles, loss);
    } else {
        const int64_t folds = (p.tiles + FOLD - 1) / FOLD;
        fold_kernel<<<(unsigned)folds, 256, 0, st>>>(s.part, p.tiles, s.win);
        total_kernel<<<1, 1024, 0, st>>>(s.win, folds, loss);
    }
    return launched();
}

int pv_policy_grad(const pv_scored* b, const pv_policy_args* a, const double* weight, const float* scale, int skip_one, void* work, size_t work_bytes,
                   void* stream) {
    if (const char* why = bad_batch(b)) return fail(PV_EARG, why);
    if (const int e = bad_policy(b, a)) return e;
    if (b->n == 0 || b->W == 0) return PV_OK;
    if (!b->grad || !weight || !a->old || !a->adv) return fail(PV_EARG, "pv_policy_grad: NULL argument");
    if (off(weight, 8) || off(scale, 4)) return fail(PV_EARG, "pv_policy_grad: an address is not aligned (weight double, scale float)");
    const Plan p = plan_of(*b);
    const Scratch s = scratch_of(*b, p, work);
    if (p.form == LONG_ROWS && check_work(s, work, work_bytes)) return PV_EARG;
    return policy_rows(b, a, p, s, nullptr, weight, scale, skip_one, (cudaStream_t)stream);
}

}  // extern "C"
