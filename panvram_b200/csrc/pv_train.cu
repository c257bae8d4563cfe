// pv_train.cu - log-probabilities of windows' tokens under a model's logits, the preference loss over pairs of windows
// and the clipped policy loss with a KL term, forward and backward (include/panvram_b200.h pv_logprobs ... pv_policy_grad).
//
// The mathematics, per row (a position's V logits x, its target y): m = max x, numerators e_j = 2^((x_j - m) log2 e),
// their sum s, p_j = e_j / s, log p_y = x_y - m - log s, and d log p_y / d x_j = [j = y] - p_j.
// The difference comes before the product (not one FMA with m log2 e): logits at their type's lowest or highest value
// would overflow there. The sum o over the other words is kept apart from the target's numerator e: 1 - p_y = o / (o + e)
// and, where e >= o, log p_y = -log1p(o / e), so neither loses its digits where the model is nearly sure.
// All statistics are in 32 bits; sums over rows are in 64 bits and in a fixed order (a partial sum per tile of rows, then
// over the tiles), so results do not change from call to call.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include <algorithm>

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
enum { LOGP = 0, GRAD = 1, POLICY = 2 };

struct Rows {
    pv_scored b;
    int64_t tpw;             // tiles per window
    int32_t rows;            // rows per tile
    // LOGP
    float* logp;             // or NULL
    double* part;            // a partial sum per tile (LOGP: of log-probabilities, POLICY: of loss terms), or NULL
    // GRAD
    const float* up; int64_t up_n, up_w;
    // POLICY
    pv_policy_args a;
    const double* weight;
    // GRAD, POLICY
    const float* scale; int32_t skip_one;
};

// the target of row (i, t), or -1
__device__ __forceinline__ int target(const pv_scored& b, int64_t i, int64_t t) {
    const int64_t at = t + b.shift;
    if (at >= b.W) return -1;
    if (b.mask_bytes == 1 && ((const uint8_t*)b.mask)[i * b.mask_n + at * b.mask_w] == 0) return -1;
    if (b.mask_bytes == 4 && ((const float*)b.mask)[i * b.mask_n + at * b.mask_w] == 0.f) return -1;
    const int64_t y = b.token_bytes == 1 ? ((const uint8_t*)b.tokens)[i * b.tokens_n + at * b.tokens_w]
                                         : ((const int64_t*)b.tokens)[i * b.tokens_n + at * b.tokens_w];
    return y < 0 || y >= b.V || y == b.ignore ? -1 : (int)y;
}

__device__ __forceinline__ float numerator(float x, float m) { return ex2((x - m) * LOG2E); }

// log p of the target with logit xt: m the maximum, o the sum of the other words' numerators; *e receives the target's
__device__ __forceinline__ float row_logp(float m, float o, float xt, float* e) {
    *e = numerator(xt, m);
    if (m == -INFINITY) return NAN;                         // nothing to normalise by
    return *e >= o ? -log1pf(o / *e) : (xt - m) - logf(o + *e);
}

// exp(d) - d - 1: by its series near 0, where the difference would lose its digits
__device__ __forceinline__ float kl_term(float d, float em1) {
    if (fabsf(d) < 0.25f)
        return d * d * (0.5f + d * (1.f / 6 + d * (1.f / 24 + d * (1.f / 120 + d * (1.f / 720 + d * (1.f / 5040 + d * (1.f / 40320)))))));
    return em1 - d;
}

// One thread, per counted row: takes the log-probability, adds the row's term to `sum`, gives the row's derivative by it.
template <int MODE>
__device__ __forceinline__ float row_end(const Rows& k, int64_t i, int64_t t, float lp, float scale, double& sum) {
    if (MODE == LOGP) {
        if (k.logp) k.logp[i * k.b.W + t] = lp;
        sum += lp;
        return 0.f;
    }
    if (MODE == GRAD) return k.up[i * k.up_n + t * k.up_w] * scale;
    const float A = k.a.adv[i * k.a.adv_n + t * k.a.adv_w];
    const float r = expf(lp - k.a.old[i * k.a.old_n + t * k.a.old_w]);
    const float one = A == 0.f ? 0.f : r * A;
    const float two = fminf(fmaxf(r, 1.f - k.a.clip_low), 1.f + k.a.clip_high) * A;
    const bool free = !(one > two);                          // NaN stays
    float term = free ? -one : -two, g = free ? -one : 0.f;
    if (k.a.ref) {
        const float d = k.a.ref[i * k.a.ref_n + t * k.a.ref_w] - lp, em1 = expm1f(d);
        term += k.a.kl * kl_term(d, em1);
        g -= k.a.kl * em1;
    }
    const double w = k.weight[i];
    sum += (double)term * w;
    return g * (float)w * scale;
}

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

// ---------------------------------------------------------------- a warp per tile of rows, element by element
// Any type, stride and length: two passes over a row for its maximum and sum, a third for the gradient.
template <typename T, int MODE>
__global__ void __launch_bounds__(256) rows_any_kernel(Rows k) {
    const int lane = threadIdx.x & 31;
    const float scale = MODE != LOGP && k.scale ? *k.scale : 1.f;
    if (MODE != LOGP && k.skip_one && scale == 1.f) return;
    const int64_t tiles = k.b.n * k.tpw, step = (int64_t)gridDim.x * (blockDim.x >> 5);
    for (int64_t tile = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); tile < tiles; tile += step) {
        const int64_t i = tile / k.tpw, t0 = (tile - i * k.tpw) * k.rows, t1 = min(t0 + k.rows, k.b.W);
        double sum = 0;
        for (int64_t t = t0; t < t1; t++) {
            const T* x = (const T*)k.b.logits + i * k.b.logits_n + t * k.b.logits_w;
            T* d = k.b.grad ? (T*)k.b.grad + i * k.b.grad_n + t * k.b.grad_w : nullptr;
            const int y = target(k.b, i, t), V = (int)k.b.V;
            if (y < 0) {
                if (MODE == LOGP && k.logp && lane == 0) k.logp[i * k.b.W + t] = 0.f;
                if (MODE != LOGP && d)
                    for (int j = lane; j < V; j += 32) d[j] = from32<T>(0.f);
                continue;
            }
            float m = -INFINITY, o = 0.f;
            for (int j = lane; j < V; j += 32) m = fmaxf(m, f32(x[j]));
            m = warp_max(m);
            for (int j = lane; j < V; j += 32) o += j == y ? 0.f : numerator(f32(x[j]), m);
            o = warp_sum(o);
            float e, g = 0.f;
            const float lp = row_logp(m, o, f32(x[y]), &e);
            if (lane == 0) g = row_end<MODE>(k, i, t, lp, scale, sum);
            if (MODE == LOGP || !d) continue;
            g = __shfl_sync(~0u, g, 0);
            const float inv = 1.f / (o + e), f = -g * inv;
            for (int j = lane; j < V; j += 32) d[j] = from32<T>(j == y ? g * (o * inv) : f * numerator(f32(x[j]), m));
        }
        if (k.part && lane == 0) k.part[tile] = sum;
    }
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

// a block per window: the sum of its tiles
__global__ void __launch_bounds__(256) window_sums_kernel(const double* part, int64_t n, int64_t tpw, float* sums, double* sums64) {
    for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
        double v = 0;
        for (int64_t j = threadIdx.x; j < tpw; j += blockDim.x) v += part[i * tpw + j];
        v = block_sum(v);
        if (threadIdx.x == 0) {
            if (sums) sums[i] = (float)v;
            if (sums64) sums64[i] = v;
        }
    }
}

// one block: the sum of `count` partial sums
__global__ void __launch_bounds__(1024) total_kernel(const double* part, int64_t count, float* out) {
    double v = 0;
    for (int64_t j = threadIdx.x; j < count; j += blockDim.x) v += part[j];
    v = block_sum(v);
    if (threadIdx.x == 0) *out = (float)v;
}

// one block: the pairs' margins, loss and derivatives from the windows' sums
__global__ void __launch_bounds__(1024) pairs_kernel(const double* sums, int64_t n, const float* ref, int64_t ref_n, float beta, float eps,
                                                     float* loss, float* margins, float* coef) {
    const int64_t m = n / 2;
    double all = 0;
    for (int64_t j = threadIdx.x; j < m; j += blockDim.x) {
        const double gap = (sums[j] - (double)ref[j * ref_n]) - (sums[j + m] - (double)ref[(j + m) * ref_n]);
        const double h = (double)beta * gap;
        // log sigmoid(h) = min(h, 0) - log1p(exp(-|h|))
        const double l = log1p(exp(-fabs(h))), up = fmin(h, 0.0) - l, down = fmin(-h, 0.0) - l;
        all += h != h ? h : -(1.0 - eps) * up - (eps == 0.f ? 0.0 : eps * down);
        if (margins) margins[j] = (float)gap;
        const double c = (double)beta / (double)m * ((double)eps - 1.0 / (1.0 + exp(h)));
        coef[j] = (float)c;
        coef[j + m] = (float)-c;
    }
    all = block_sum(all);
    if (threadIdx.x == 0) *loss = m ? (float)(all / (double)m) : 0.f;
}

// counted positions of each window: a block per (window, part of it), then one block turns them into weights
constexpr int COUNT_SPAN = 16384;
__global__ void __launch_bounds__(256) count_kernel(pv_scored b, int64_t spans, int32_t* counts) {
    for (int64_t q = blockIdx.x; q < b.n * spans; q += gridDim.x) {
        const int64_t i = q / spans, t0 = (q - i * spans) * COUNT_SPAN, t1 = min(t0 + (int64_t)COUNT_SPAN, b.W);
        int v = 0;
        for (int64_t t = t0 + threadIdx.x; t < t1; t += blockDim.x) v += target(b, i, t) >= 0;
        v = (int)block_sum((double)v);
        if (threadIdx.x == 0) counts[q] = v;
    }
}
__global__ void __launch_bounds__(1024) weights_kernel(const int32_t* counts, int64_t n, int64_t spans, int by_window, double* weight) {
    double all = 0, some = 0;
    for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
        int64_t c = 0;
        for (int64_t j = 0; j < spans; j++) c += counts[i * spans + j];
        all += (double)c;
        some += c > 0;
        weight[i] = (double)c;
    }
    all = block_sum(all);
    some = block_sum(some);
    for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
        const double c = weight[i];
        weight[i] = by_window ? (c > 0 ? 1.0 / (c * some) : 0.0) : (all > 0 ? 1.0 / all : 0.0);
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

const char* bad_batch(const pv_scored* b) {
    if (!b) return "batch: NULL";
    if (b->n < 0 || b->W < 0 || b->W >= (1ll << 31) || b->V < 1 || b->V >= (1ll << 31)) return "batch: n, W or V out of range";
    if (b->shift < 0) return "batch: shift is negative";
    if (b->type < PV_T_BF16 || b->type > PV_T_FP32) return "batch: logits are bf16, fp16 or fp32";
    if (b->token_bytes != 1 && b->token_bytes != 8) return "batch: tokens are uint8 or int64";
    if (b->mask_bytes != 0 && b->mask_bytes != 1 && b->mask_bytes != 4) return "batch: the mask is uint8 or float";
    if (b->n > 0 && b->W > 0 && (!b->logits || !b->tokens || (b->mask_bytes && !b->mask))) return "batch: NULL logits, tokens or mask";
    if (b->n > 0 && b->W > (1ll << 62) / b->n) return "batch: n W is too large";
    return nullptr;
}

struct Plan { int32_t rows; int64_t tpw, tiles, spans; };
Plan plan_of(const pv_scored& b) {
    Plan p;
    p.rows = b.V >= 512 ? 1 : 16;
    p.tpw = (b.W + p.rows - 1) / p.rows;
    p.tiles = b.n * p.tpw;
    p.spans = (b.W + COUNT_SPAN - 1) / COUNT_SPAN;
    return p;
}
// scratch: a double per tile, a double per window, an int per (window, span)
struct Scratch { double *part, *win; int32_t* counts; size_t bytes; };
Scratch scratch_of(const pv_scored& b, const Plan& p, void* work) {
    Scratch s;
    const size_t a = (size_t)p.tiles * 8, w = (size_t)b.n * 8, c = ((size_t)b.n * p.spans * 4 + 15) / 16 * 16;
    s.part = (double*)work;
    s.win = (double*)((char*)work + a);
    s.counts = (int32_t*)((char*)work + a + w);
    s.bytes = a + w + c;
    return s;
}

template <int MODE>
int launch_rows(const Rows& k, cudaStream_t st) {
    const int64_t tiles = k.b.n * k.tpw;
    if (tiles == 0) return PV_OK;
    const unsigned grid = (unsigned)std::min<int64_t>((tiles + 7) / 8, SMS * 8);
    switch (k.b.type) {
        case PV_T_BF16: rows_any_kernel<__nv_bfloat16, MODE><<<grid, 256, 0, st>>>(k); break;
        case PV_T_FP16: rows_any_kernel<__half, MODE><<<grid, 256, 0, st>>>(k); break;
        default: rows_any_kernel<float, MODE><<<grid, 256, 0, st>>>(k);
    }
    return launched();
}

Rows rows_of(const pv_scored& b, const Plan& p) {
    Rows k = {};
    k.b = b;
    k.tpw = p.tpw;
    k.rows = p.rows;
    return k;
}

int check_work(const Scratch& s, const void* work, size_t have) {
    if (s.bytes && (!work || have < s.bytes || ((uintptr_t)work & 15))) return fail(PV_EARG, "scratch: too small, NULL or not 16-byte aligned");
    return PV_OK;
}

int window_sums(const Plan& p, int64_t n, const double* part, float* sums, double* sums64, cudaStream_t st) {
    window_sums_kernel<<<(unsigned)std::min<int64_t>(n, SMS * 8), 256, 0, st>>>(part, n, p.tpw, sums, sums64);
    return launched();
}

int bad_policy(const pv_scored* b, const pv_policy_args* a) {
    if (!a) return fail(PV_EARG, "pv_policy: NULL arguments");
    if (!(a->clip_low >= 0.f) || !(a->clip_high >= 0.f)) return fail(PV_EARG, "pv_policy: clip is negative");
    if (!(a->kl == 0.f) && !a->ref && b->n && b->W) return fail(PV_EARG, "pv_policy: a KL term without reference log-probabilities");
    return PV_OK;
}

}  // namespace

extern "C" {

size_t pv_score_work_bytes(const pv_scored* b) {
    if (bad_batch(b)) return 0;
    return scratch_of(*b, plan_of(*b), nullptr).bytes;
}

int pv_logprobs(const pv_scored* b, float* logp, float* sums, void* work, size_t work_bytes, void* stream) {
    if (const char* why = bad_batch(b)) return fail(PV_EARG, why);
    const Plan p = plan_of(*b);
    const Scratch s = scratch_of(*b, p, work);
    if (sums && check_work(s, work, work_bytes)) return PV_EARG;
    if (b->n == 0) return PV_OK;
    Rows k = rows_of(*b, p);
    k.b.grad = nullptr;
    k.logp = logp;
    k.part = sums ? s.part : nullptr;
    const cudaStream_t st = (cudaStream_t)stream;
    if (const int e = launch_rows<LOGP>(k, st)) return e;
    return sums ? window_sums(p, b->n, s.part, sums, nullptr, st) : PV_OK;
}

int pv_logprobs_grad(const pv_scored* b, const float* up, int64_t up_n, int64_t up_w, const float* scale, int skip_one, void* stream) {
    if (const char* why = bad_batch(b)) return fail(PV_EARG, why);
    if (b->n == 0 || b->W == 0) return PV_OK;
    if (!b->grad || !up) return fail(PV_EARG, "pv_logprobs_grad: NULL gradient");
    Rows k = rows_of(*b, plan_of(*b));
    k.up = up; k.up_n = up_n; k.up_w = up_w;
    k.scale = scale; k.skip_one = scale && skip_one;
    return launch_rows<GRAD>(k, (cudaStream_t)stream);
}

int pv_preference(const pv_scored* b, const float* ref, int64_t ref_n, float beta, float smoothing, float* loss, float* margins, float* coef,
                  void* work, size_t work_bytes, void* stream) {
    if (const char* why = bad_batch(b)) return fail(PV_EARG, why);
    if (b->n & 1) return fail(PV_EARG, "pv_preference: an odd number of windows");
    if (!loss || (b->n && (!ref || !coef))) return fail(PV_EARG, "pv_preference: NULL argument");
    const Plan p = plan_of(*b);
    const Scratch s = scratch_of(*b, p, work);
    if (check_work(s, work, work_bytes)) return PV_EARG;
    const cudaStream_t st = (cudaStream_t)stream;
    if (b->n) {
        Rows k = rows_of(*b, p);
        k.b.grad = nullptr;
        k.part = s.part;
        if (const int e = launch_rows<LOGP>(k, st)) return e;
        if (const int e = window_sums(p, b->n, s.part, nullptr, s.win, st)) return e;
    }
    pairs_kernel<<<1, 1024, 0, st>>>(s.win, b->n, ref, ref_n, beta, smoothing, loss, margins, coef);
    if (const int e = launched()) return e;
    return b->grad ? pv_logprobs_grad(b, coef, 1, 0, nullptr, 0, stream) : PV_OK;
}

int pv_policy(const pv_scored* b, const pv_policy_args* a, float* loss, double* weight, void* work, size_t work_bytes, void* stream) {
    if (const char* why = bad_batch(b)) return fail(PV_EARG, why);
    if (const int e = bad_policy(b, a)) return e;
    if (!loss || (b->n && !weight) || (b->n && b->W && (!a->old || !a->adv))) return fail(PV_EARG, "pv_policy: NULL argument");
    const Plan p = plan_of(*b);
    const Scratch s = scratch_of(*b, p, work);
    if (check_work(s, work, work_bytes)) return PV_EARG;
    const cudaStream_t st = (cudaStream_t)stream;
    if (b->n) {
        count_kernel<<<(unsigned)std::min<int64_t>(b->n * std::max<int64_t>(p.spans, 1), SMS * 8), 256, 0, st>>>(*b, p.spans, s.counts);
        weights_kernel<<<1, 1024, 0, st>>>(s.counts, b->n, p.spans, a->by_window, weight);
        if (const int e = launched()) return e;
        Rows k = rows_of(*b, p);
        k.part = s.part;
        k.a = *a;
        k.weight = weight;
        if (const int e = launch_rows<POLICY>(k, st)) return e;
    }
    total_kernel<<<1, 1024, 0, st>>>(s.part, p.tiles, loss);
    return launched();
}

int pv_policy_grad(const pv_scored* b, const pv_policy_args* a, const double* weight, const float* scale, int skip_one, void* stream) {
    if (const char* why = bad_batch(b)) return fail(PV_EARG, why);
    if (const int e = bad_policy(b, a)) return e;
    if (b->n == 0 || b->W == 0) return PV_OK;
    if (!b->grad || !weight || !a->old || !a->adv) return fail(PV_EARG, "pv_policy_grad: NULL argument");
    Rows k = rows_of(*b, plan_of(*b));
    k.a = *a;
    k.weight = weight;
    k.scale = scale; k.skip_one = scale && skip_one;
    return launch_rows<POLICY>(k, (cudaStream_t)stream);
}

}  // extern "C"
