// pv_grads.cu - the 2-norm over many tensors and their scaling by min(1, max_norm / (norm + 1e-6))
// (include/panvram_b200.h pv_grad_norm, pv_clip_grads).
//
// The tensors' addresses, counts and types travel as a kernel parameter, so a call copies no table to the device and
// can be captured. The blocks share the elements evenly, in units of UNIT, over as many tensors as a run of units spans,
// and leave one partial sum each, in 64 bits; the scaling kernel's blocks each add those partial sums in the same
// order, so no launch is spent on it and the result does not change from call to call. Squares are added eight (or four) at
// a time in 32 bits and then in 64; where such a group leaves the range of 32 bits (elements beyond about 1e18 or all below
// 1e-13) it is squared again in 64 bits, so the norm neither overflows nor underflows before it is rounded to float at the end.
//
// Bound by memory: on a B200 the norm of 8.4e8 bf16 elements in 122 tensors takes 262 us (6.4 TB/s); 8.4e7 in 146 tensors,
// clipped into float, 39 + 86 us (the second 5.9 TB/s read and written). A contiguous run a block takes 69 us there for the
// norm, rounds without the even share of the rest 37 + 108 us.
// The elements are read twice where they are scaled, as the factor needs the whole norm; the scaling begins
// with what the norm's pass read last and left in L2.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include <algorithm>
#include <vector>

#include "panvram_b200.h"

namespace pvb { extern thread_local char g_cuda_err[256]; }

namespace {

using pvb::g_cuda_err;

constexpr int UNIT = 2048, RUN = 8, THREADS = 256, SMS = 148, GRID = SMS * 8;

template <int N>
struct Table {
    uint64_t ptr[N], out[N];
    int64_t numel[N];
    uint32_t first[N + 1];           // a tensor's first unit
    uint8_t type[N], otype[N];
    int32_t count;
};
// two sizes of parameter: a launch copies all of it. 30 bytes per tensor, 32,764 bytes at most.
constexpr int SMALL = 96, LARGE = 1024;
static_assert(sizeof(Table<LARGE>) <= 32000, "a kernel's parameters");

__device__ __forceinline__ float f32(float v) { return v; }
__device__ __forceinline__ float f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from32(float v);
template <> __device__ __forceinline__ float from32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int N> struct alignas(sizeof(T) * N) Vec { T v[N]; };

template <int K>
__device__ __forceinline__ double squares(const float (&x)[K]) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < K; j++) s = fmaf(x[j], x[j], s);
    if (s > 1e-25f && s < 1e37f) return (double)s;
    double d = 0;
#pragma unroll
    for (int j = 0; j < K; j++) d = fma((double)x[j], (double)x[j], d);
    return d;
}

__device__ double block_sum(double v) {                      // every thread of the block gets it
    __shared__ double sh[33];
#pragma unroll
    for (int s = 16; s; s >>= 1) v += __shfl_xor_sync(~0u, v, s);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x < 32) {
        double w = threadIdx.x < (blockDim.x >> 5) ? sh[threadIdx.x] : 0.0;
#pragma unroll
        for (int s = 16; s; s >>= 1) w += __shfl_xor_sync(~0u, w, s);
        if (threadIdx.x == 0) sh[32] = w;
    }
    __syncthreads();
    return sh[32];
}

// the tensor that unit c lies in: the last whose first unit is not after it (empty tensors share their successor's)
template <int N>
__device__ __forceinline__ int tensor_of(const Table<N>& t, uint32_t c) {
    int lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first[mid] <= c) lo = mid; else hi = mid;
    }
    return lo;
}

// elements from `p` to its next 16-byte boundary
template <typename T>
__device__ __forceinline__ int to_boundary(const T* p) { return (int)(((16 - ((uintptr_t)p & 15)) & 15) / sizeof(T)); }

// f(tensor, first element, count) for the elements of this block: RUN units in every round over the blocks, and an even share
// of the units that are left; BACK: in reverse
template <bool BACK, int N, typename F>
__device__ __forceinline__ void spans(const Table<N>& t, F&& f) {
    const uint64_t units = t.first[t.count], round = (uint64_t)RUN * gridDim.x, rounds = units / round, done = rounds * round, left = units - done;
    const auto run = [&](uint32_t begin, uint32_t end) {
        int i = begin < end ? tensor_of(t, begin) : 0;
        while (begin < end) {
            const uint32_t first = t.first[i], to = min(end, t.first[i + 1]);
            if (to > begin) {
                const int64_t at = (int64_t)(begin - first) * UNIT;
                f(i, at, (int)min((int64_t)(to - begin) * UNIT, t.numel[i] - at));
                begin = to;
            }
            i++;
        }
    };
    const auto share = [&]() { run((uint32_t)(done + left * blockIdx.x / gridDim.x), (uint32_t)(done + left * (blockIdx.x + 1) / gridDim.x)); };
    if (BACK) share();
    for (uint64_t k = 0; k < rounds; k++) {
        const uint32_t begin = (uint32_t)((BACK ? rounds - 1 - k : k) * round + (uint64_t)RUN * blockIdx.x);
        run(begin, begin + RUN);
    }
    if (!BACK) share();
}

template <typename T>
__device__ double span_squares(const T* p, int count) {
    constexpr int K = 16 / sizeof(T);
    const int head = min(to_boundary(p), count), nv = (count - head) / K, tail = head + nv * K;
    double s = 0;
    float one[1];
    if ((int)threadIdx.x < head) { one[0] = f32(p[threadIdx.x]); s += squares(one); }
    if (tail + (int)threadIdx.x < count) { one[0] = f32(p[tail + threadIdx.x]); s += squares(one); }
    const uint4* q = (const uint4*)(p + head);
#pragma unroll 4
    for (int j = threadIdx.x; j < nv; j += THREADS) {
        const uint4 raw = q[j];
        const Vec<T, K>& v = *(const Vec<T, K>*)&raw;
        float x[K];
#pragma unroll
        for (int e = 0; e < K; e++) x[e] = f32(v.v[e]);
        s += squares(x);
    }
    return s;
}

template <int N>
__global__ void __launch_bounds__(THREADS) norm_kernel(const __grid_constant__ Table<N> t, double* part) {
    double s = 0;
    spans<false>(t, [&](int i, int64_t at, int count) {
        switch (t.type[i]) {
            case PV_T_BF16: s += span_squares((const __nv_bfloat16*)t.ptr[i] + at, count); break;
            case PV_T_FP16: s += span_squares((const __half*)t.ptr[i] + at, count); break;
            default: s += span_squares((const float*)t.ptr[i] + at, count);
        }
    });
    s = block_sum(s);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__device__ double norm_of(const double* part, int64_t parts) {
    double s = 0;
    for (int64_t j = threadIdx.x; j < parts; j += blockDim.x) s += part[j];
    return sqrt(block_sum(s));
}

__global__ void __launch_bounds__(THREADS) finish_norm_kernel(const double* part, int64_t parts, float* norm) {
    const double s = norm_of(part, parts);
    if (threadIdx.x == 0) *norm = (float)s;
}

// Sixteen bytes a store and a thread next to a thread, whatever the elements become: widened ones are loaded eight bytes a
// thread. Streaming stores, which leave the gradients in L2 for the spans to come.
template <typename T, typename O>
__device__ void scale_span(const T* p, O* o, int count, float f) {
    constexpr int K = 16 / sizeof(O);
    int head = min(to_boundary(o), count), nv = (count - head) / K;
    if (((uintptr_t)(p + head) & (sizeof(T) * K - 1)) != 0) { head = count; nv = 0; }     // the two differ in alignment: element by element
    const int tail = head + nv * K;
    for (int j = threadIdx.x; j < head; j += THREADS) o[j] = from32<O>(f32(p[j]) * f);
    for (int j = tail + threadIdx.x; j < count; j += THREADS) o[j] = from32<O>(f32(p[j]) * f);
    const auto* q = (const Vec<T, K>*)(p + head);
    uint4* w = (uint4*)(o + head);
#pragma unroll 4
    for (int j = threadIdx.x; j < nv; j += THREADS) {
        const Vec<T, K> v = q[j];
        Vec<O, K> r;
#pragma unroll
        for (int e = 0; e < K; e++) r.v[e] = from32<O>(f32(v.v[e]) * f);
        __stcs(w + j, *(const uint4*)&r);
    }
}

template <int N>
__global__ void __launch_bounds__(THREADS) clip_kernel(const __grid_constant__ Table<N> t, const double* part, int64_t parts, float max_norm,
                                                       int in_place, float* norm) {
    const double s = norm_of(part, parts), r = (double)max_norm / (s + 1e-6);
    const float f = r >= 1.0 ? 1.f : (float)r;               // NaN stays
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)s;
    if (in_place && f == 1.f) return;
    spans<true>(t, [&](int i, int64_t at, int count) {
        const bool wide = t.otype[i] == PV_T_FP32;
        switch (t.type[i]) {
            case PV_T_BF16:
                if (wide) scale_span((const __nv_bfloat16*)t.ptr[i] + at, (float*)t.out[i] + at, count, f);
                else scale_span((const __nv_bfloat16*)t.ptr[i] + at, (__nv_bfloat16*)t.out[i] + at, count, f);
                break;
            case PV_T_FP16:
                if (wide) scale_span((const __half*)t.ptr[i] + at, (float*)t.out[i] + at, count, f);
                else scale_span((const __half*)t.ptr[i] + at, (__half*)t.out[i] + at, count, f);
                break;
            default: scale_span((const float*)t.ptr[i] + at, (float*)t.out[i] + at, count, f);
        }
    });
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

int elem(uint8_t type) { return type == PV_T_FP32 ? 4 : 2; }

const char* bad_list(const pv_tensors* g) {
    if (!g || g->count < 0 || (g->count && (!g->ptr || !g->numel || !g->type))) return "tensors: NULL list";
    for (int64_t i = 0; i < g->count; i++) {
        if (g->type[i] > PV_T_FP32) return "tensors: bf16, fp16 or fp32";
        if (g->numel[i] < 0 || g->numel[i] > (1ll << 45)) return "tensors: a size is out of range";
        if (g->numel[i] && (!g->ptr[i] || g->ptr[i] % elem(g->type[i]))) return "tensors: an address is NULL or not aligned to its type";
    }
    return nullptr;
}

// a tensor that is written shares memory with another
struct Span { uint64_t a, b; bool written; };
bool overlap(const pv_tensors* g, const pv_tensors* out) {
    std::vector<Span> v;
    v.reserve((size_t)g->count * (out ? 2 : 1));
    for (int64_t i = 0; i < g->count; i++) {
        if (!g->numel[i]) continue;
        const uint64_t ga = g->ptr[i], gb = ga + (uint64_t)g->numel[i] * elem(g->type[i]);
        if (!out || (out->ptr[i] == ga && out->type[i] == g->type[i])) { v.push_back({ga, gb, true}); continue; }
        v.push_back({ga, gb, false});
        v.push_back({out->ptr[i], out->ptr[i] + (uint64_t)g->numel[i] * elem(out->type[i]), true});
    }
    std::sort(v.begin(), v.end(), [](const Span& x, const Span& y) { return x.a < y.a; });
    uint64_t end = 0, end_written = 0;
    for (const Span& s : v) {
        if (s.a < (s.written ? end : end_written)) return true;
        end = std::max(end, s.b);
        if (s.written) end_written = std::max(end_written, s.b);
    }
    return false;
}

int64_t launches_of(const pv_tensors* g) { return (g->count + LARGE - 1) / LARGE; }

template <int N>
int64_t fill(Table<N>& t, const pv_tensors* g, const pv_tensors* out, int64_t from, int64_t to) {
    uint64_t c = 0;
    t.count = (int32_t)(to - from);
    for (int64_t i = from; i < to; i++) {
        const int64_t k = i - from;
        t.ptr[k] = g->ptr[i];
        t.numel[k] = g->numel[i];
        t.type[k] = g->type[i];
        t.out[k] = out ? out->ptr[i] : g->ptr[i];
        t.otype[k] = out ? out->type[i] : g->type[i];
        t.first[k] = (uint32_t)c;
        c += (uint64_t)((g->numel[i] + UNIT - 1) / UNIT);
    }
    t.first[t.count] = (uint32_t)c;
    return c < (1ull << 32) ? (int64_t)c : -1;
}

// one launch over tensors [from, to): the norm's partial sums, or the scaling
template <int N>
int one(const pv_tensors* g, const pv_tensors* out, int64_t from, int64_t to, bool clip, double* part, int64_t* parts, float max_norm, bool in_place,
        float* norm, cudaStream_t st) {
    static thread_local Table<N> t;
    const int64_t units = fill(t, g, out, from, to);
    if (units < 0) return fail(PV_EARG, "tensors: too many elements in one list");
    const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(units, GRID));
    if (clip) {
        clip_kernel<N><<<grid, THREADS, 0, st>>>(t, part, *parts, max_norm, in_place, norm);
    } else {
        norm_kernel<N><<<grid, THREADS, 0, st>>>(t, part + *parts);
        *parts += grid;
    }
    return launched();
}

int all(const pv_tensors* g, const pv_tensors* out, bool clip, double* part, int64_t* parts, float max_norm, bool in_place, float* norm,
        cudaStream_t st) {
    for (int64_t from = 0; from < std::max<int64_t>(g->count, 1); from += LARGE) {
        const int64_t to = std::min<int64_t>(g->count, from + LARGE);
        float* nm = from == 0 ? norm : nullptr;
        const int e = to - from <= SMALL ? one<SMALL>(g, out, from, to, clip, part, parts, max_norm, in_place, nm, st)
                                         : one<LARGE>(g, out, from, to, clip, part, parts, max_norm, in_place, nm, st);
        if (e) return e;
    }
    return PV_OK;
}

int norm_parts(const pv_tensors* g, float* norm, void* work, size_t work_bytes, int64_t* parts, cudaStream_t st) {
    if (!norm || (uintptr_t)norm % 4) return fail(PV_EARG, "norm: NULL or not aligned to float");
    if (!work || work_bytes < pv_grads_work_bytes(g) || ((uintptr_t)work & 15)) return fail(PV_EARG, "scratch: too small, NULL or not 16-byte aligned");
    *parts = 0;
    return all(g, nullptr, false, (double*)work, parts, 0.f, false, nullptr, st);
}

}  // namespace

extern "C" {

size_t pv_grads_work_bytes(const pv_tensors* g) {
    if (!g || g->count < 0) return 0;
    return (size_t)std::max<int64_t>(1, launches_of(g)) * GRID * sizeof(double);
}

int pv_grad_norm(const pv_tensors* g, float* norm, void* work, size_t work_bytes, void* stream) {
    if (const char* why = bad_list(g)) return fail(PV_EARG, why);
    int64_t parts = 0;
    if (const int e = norm_parts(g, norm, work, work_bytes, &parts, (cudaStream_t)stream)) return e;
    finish_norm_kernel<<<1, THREADS, 0, (cudaStream_t)stream>>>((const double*)work, parts, norm);
    return launched();
}

int pv_clip_grads(const pv_tensors* g, const pv_tensors* out, float max_norm, float* norm, void* work, size_t work_bytes, void* stream) {
    if (const char* why = bad_list(g)) return fail(PV_EARG, why);
    if (!(max_norm >= 0.f)) return fail(PV_EARG, "max_norm: negative or NaN");
    if (out) {
        if (const char* why = bad_list(out)) return fail(PV_EARG, why);
        if (out->count != g->count) return fail(PV_EARG, "out: another number of tensors");
        for (int64_t i = 0; i < g->count; i++) {
            if (out->numel[i] != g->numel[i]) return fail(PV_EARG, "out: a tensor of another size");
            if (out->type[i] != g->type[i] && out->type[i] != PV_T_FP32) return fail(PV_EARG, "out: a tensor of neither its source's type nor float");
        }
    }
    try {
        if (overlap(g, out)) return fail(PV_EARG, "tensors: one that is written shares memory with another");
    } catch (...) {
        return fail(PV_EARG, "tensors: out of host memory");
    }
    int64_t parts = 0;
    if (const int e = norm_parts(g, norm, work, work_bytes, &parts, (cudaStream_t)stream)) return e;
    return all(g, out, true, (double*)work, &parts, max_norm, !out, norm, (cudaStream_t)stream);
}

}  // extern "C"
