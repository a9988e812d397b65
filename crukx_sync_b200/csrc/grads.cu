// Whole-model passes of a trainer over its gradients and its fp32 masters, between the backward
// pass and the encode of the update (no reference counterpart: the reference starts at the two
// weight dicts).  n tensors of any sizes per call, every tensor cut into tiles:
//
//   k_grad_sumsq   sum of squares of every gradient: one partial (double) per CTA
//   k_grad_norm    one CTA: the partials summed in a fixed order, and the square root
//   k_grad_clip    out = min(1, max_norm / (norm + 1e-6)) * grad; where there are few partials every
//                  CTA sums them itself (same order, so the same coefficient everywhere)
//   k_adamw        AdamW on fp32 masters and moments with that coefficient folded in, and the
//                  bf16 weights written beside them
//
// The tensor table travels in the kernel's parameters (up to 32 KB), so a call makes no copy, needs
// no host buffer to outlive it and can be captured into a graph.  Nothing is summed by atomics:
// the same call gives the same bits.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <exception>
#include <string>
#include <type_traits>
#include <utility>
#include <vector>

#include "../../include/crukx_b200.h"
#include "common.cuh"
#include "elements.cuh"
#include "launch.cuh"

namespace crx {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 8192;            // gradient elements per tile of the norm and the clip
constexpr int kStepTile = kThreads * 8;   // parameters per tile of the step: 8 per thread
// CTAs of one launch of the norm, at most, and so its partials.  Each takes a contiguous range of
// tiles (of 330 tensors and 2 GB: 343 us; every grid-th tile, which passes more tensors: 428).  Four times
// as many CTAs as fit the GPU at once: their ends spread, so the last wave is short (1.86 GB of bf16:
// 362 us with 8 per SM, 325 with 32 and with 64).
constexpr int kMaxGrid = 148 * 32;
// The clip and the step have one CTA per tile.  A CTA whose stores are still on their way holds
// nobody up, and the hardware deals the tiles out as SMs come free: 0.93e9 parameters took 4.37 ms
// with 16 CTAs per SM walking a range of tiles each, 4.13 with 64, 3.81 with one CTA per tile; the
// clip of 1.86 GB 0.59 and 0.54.
// Up to so many partials each CTA of the clip sums them itself (20 tensors, 0.8 MB: 9 us, 15 with a launch
// for that between; 160 MB, 4736 partials: 82 us, 78 with it).
constexpr int kClipPartials = 1024;

struct GradEntry {
    const void* g;
    void* out;
    int64_t numel;
    uint32_t tile;   // first tile of this tensor
    int32_t dtype;
};
struct StepEntry {
    const void* g;
    float* p;
    float* m;
    float* v;
    __nv_bfloat16* w;   // may be null
    int64_t numel;
    uint32_t tile;
    int16_t dtype;
    int16_t head;       // elements before the first place where every pointer is 16-byte aligned; -1: none
};
// The table is a kernel parameter, at most 32764 bytes of them.  A launch copies all of it (the norm of
// 112 tensors took 23 us of the host with a table of 960), so there are several sizes.
template <class E, int N>
struct Table {
    E e[N];
    int32_t n;
    uint32_t tiles;
};
constexpr int kSmall = 40, kMedium = 160, kGradLarge = 960, kStepLarge = 500;
static_assert(sizeof(Table<GradEntry, kGradLarge>) < 32000 && sizeof(Table<StepEntry, kStepLarge>) < 32300, "parameter space");

template <class T>
__device__ __forceinline__ int tensor_of(const T& t, uint32_t tile) {
    int lo = 0, hi = t.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.e[mid].tile <= tile) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// Sum of a double over the CTA, in a fixed order; the result is valid in every thread.
__device__ __forceinline__ double block_sum(double v, double* red) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int w = threadIdx.x >> 5;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[w] = v;
    __syncthreads();
    double t = 0;
    for (int k = 0; k < kThreads / 32; ++k) t += red[k];
    return t;
}

// Squares of N values into acc.  They are added in fp32 (N is small: N roundings at most, each 2^-24
// of the sum) unless that sum left the range in which no square that matters was lost to underflow
// and none overflowed; then the group is redone in double.  A group of zeros is not.
template <int N>
__device__ __forceinline__ void add_squares(const float* x, double& acc) {
    float s = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(x[i], x[i], s);
    if (s >= 1e-24f && s <= 1e37f) {
        acc += double(s);
        return;
    }
    float any = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) any = fmaxf(any, fabsf(x[i]));
    if (any == 0.f && s == 0.f) return;   // s: NaN would pass fmaxf
    double d = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) d = fma(double(x[i]), double(x[i]), d);
    acc += d;
}

// One tile's sum of squares.  Tile k of a tensor holds the kTile elements from head + k * kTile on;
// tile 0 also the head before its first 16-byte boundary.
template <class T>
__device__ __forceinline__ void tile_sumsq(const T* g, int64_t numel, int64_t k, double& acc) {
    constexpr int N = Vec<T>::N, U = kTile / (kThreads * N);
    const int64_t head = tmin<int64_t>(head_of<T>(g), numel);
    const int64_t base = head + k * kTile;
    const int tid = threadIdx.x;
    if (k == 0 && tid < head) {
        const float x = to_f(g[tid]);
        add_squares<1>(&x, acc);
    }
    const T* p = g + base;
    const int64_t left = numel - base;
    if (left >= kTile) {
        uint4 q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = __ldg(reinterpret_cast<const uint4*>(p) + u * kThreads + tid);
#pragma unroll
        for (int u = 0; u < U; u += 2) {
            float x[2 * N];
            Vec<T>::get(q[u], x);
            Vec<T>::get(q[u + 1], x + N);
            add_squares<2 * N>(x, acc);
        }
        return;
    }
    const int nv = left > 0 ? int(left / N) : 0;
    for (int i = tid; i < nv; i += kThreads) {
        float x[N];
        Vec<T>::get(__ldg(reinterpret_cast<const uint4*>(p) + i), x);
        add_squares<N>(x, acc);
    }
    for (int64_t i = int64_t(nv) * N + tid; i < left; i += kThreads) {
        const float x = to_f(p[i]);
        add_squares<1>(&x, acc);
    }
}

template <class Tab>
__global__ void __launch_bounds__(kThreads) k_grad_sumsq(const __grid_constant__ Tab t, double* __restrict__ partials) {
    __shared__ double red[kThreads / 32];
    const uint32_t lo = uint32_t(uint64_t(t.tiles) * blockIdx.x / gridDim.x);
    const uint32_t hi = uint32_t(uint64_t(t.tiles) * (blockIdx.x + 1) / gridDim.x);
    double acc = 0;
    int i = tensor_of(t, lo);
    for (uint32_t s = lo; s < hi; ++s) {
        while (i + 1 < t.n && t.e[i + 1].tile <= s) ++i;
        const int64_t k = s - t.e[i].tile;
        if (t.e[i].dtype == CRX_FP32) tile_sumsq(static_cast<const float*>(t.e[i].g), t.e[i].numel, k, acc);
        else if (t.e[i].dtype == CRX_BF16) tile_sumsq(static_cast<const __nv_bfloat16*>(t.e[i].g), t.e[i].numel, k, acc);
        else tile_sumsq(static_cast<const __half*>(t.e[i].g), t.e[i].numel, k, acc);
    }
    let_next_start();
    acc = block_sum(acc, red);
    if (threadIdx.x == 0) partials[blockIdx.x] = acc;
}

__device__ __forceinline__ double sum_partials(const double* __restrict__ partials, int n, double* red) {
    double v = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) v += partials[i];
    return block_sum(v, red);
}

__global__ void __launch_bounds__(kThreads) k_grad_norm(const double* __restrict__ partials, int n, float* __restrict__ norm) {
    __shared__ double red[kThreads / 32];
    after_previous();
    let_next_start();
    const double s = sum_partials(partials, n, red);
    if (threadIdx.x == 0) *norm = float(sqrt(s));
}

__device__ __forceinline__ float clip_coef(float norm, float max_norm) {
    const float c = max_norm / (norm + 1e-6f);
    return c > 1.f ? 1.f : c;   // NaN stays NaN
}

template <class T>
__device__ __forceinline__ void tile_scale(const T* g, T* out, int64_t numel, int64_t k, float c) {
    constexpr int N = Vec<T>::N, U = kTile / (kThreads * N);
    const int64_t head = tmin<int64_t>(head_of<T>(g), numel);
    const int64_t base = head + k * kTile;
    const int tid = threadIdx.x;
    if (k == 0 && tid < head) out[tid] = from_f<T>(c * to_f(g[tid]));
    const T* p = g + base;
    T* o = out + base;
    const int64_t left = numel - base;
    const bool wide = ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(o)) & 15) == 0;
    if (wide && left >= kTile) {
        uint4 q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = reinterpret_cast<const uint4*>(p)[u * kThreads + tid];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x[N];
            Vec<T>::get(q[u], x);
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] *= c;
            reinterpret_cast<uint4*>(o)[u * kThreads + tid] = Vec<T>::put(x);
        }
        return;
    }
    const int64_t n = tmin<int64_t>(left, kTile);
    const int nv = wide && n > 0 ? int(n / N) : 0;
    for (int i = tid; i < nv; i += kThreads) {
        float x[N];
        Vec<T>::get(reinterpret_cast<const uint4*>(p)[i], x);
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] *= c;
        reinterpret_cast<uint4*>(o)[i] = Vec<T>::put(x);
    }
    for (int64_t i = int64_t(nv) * N + tid; i < n; i += kThreads) o[i] = from_f<T>(c * to_f(p[i]));
}

// The tiles from the last to the first: the norm took them the other way, so the first ones here are
// what L2 still holds.
template <class Tab>
__global__ void __launch_bounds__(kThreads) k_grad_clip(const __grid_constant__ Tab t, const double* __restrict__ partials,
                                                        int n_partials, const float* __restrict__ norm_in, float max_norm,
                                                        float* __restrict__ norm_out) {
    __shared__ double red[kThreads / 32];
    after_previous();
    const float norm = n_partials ? float(sqrt(sum_partials(partials, n_partials, red))) : *norm_in;
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
    const float c = clip_coef(norm, max_norm);
    const uint32_t s = t.tiles - 1 - blockIdx.x;
    const GradEntry& e = t.e[tensor_of(t, s)];
    if (c == 1.f && e.out == e.g) return;   // in place and nothing to scale
    const int64_t k = s - e.tile;
    if (e.dtype == CRX_FP32) tile_scale(static_cast<const float*>(e.g), static_cast<float*>(e.out), e.numel, k, c);
    else if (e.dtype == CRX_BF16) tile_scale(static_cast<const __nv_bfloat16*>(e.g), static_cast<__nv_bfloat16*>(e.out), e.numel, k, c);
    else tile_scale(static_cast<const __half*>(e.g), static_cast<__half*>(e.out), e.numel, k, c);
}

struct StepHyper {
    float lr, b1, b2, a1, a2, eps, decay;   // a: 1 - b, rounded once (in fp32 1 - 0.999f is 1e-5 off)
    float bias1, bias2;             // 1 - b1^t, 1 - b2^t, unless step_p gives t
    double log_b1, log_b2;
    const float* lr_p;              // read when the kernel runs; may be null
    const int64_t* step_p;
    const float* norm;              // may be null: no clipping, no guard
    float max_norm;                 // <= 0: the norm only guards
};

// What a thread needs of the step: the clip coefficient and the rates.
struct StepRates {
    float c, b1, b2, a1, a2, decay, rate, inv_bias2, eps;
    bool skip;   // the norm is not finite: masters and moments stay as they are
};

// Root and reciprocal to 1 ulp each, values below 2^-126 taken as 0: next to an eps of kTinyEps or
// more such a root (2^-63) is nothing.  Back to back, the step of 0.93e9 parameters takes 3.80 ms with
// these, 4.14 with the ones that mind such values, 4.87 with the exactly rounded ones; their error is
// 2^-22 of an update that is itself a small part of the master.
__device__ __forceinline__ float sqrt_fast(float x) {
    float y;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr double kTinyEps = 1e-12;

// TINY: the eps is less than kTinyEps, so root and quotient are the exactly rounded ones.
template <bool TINY>
__device__ __forceinline__ void adamw_one(const StepRates& r, float g, float& p, float& m, float& v) {
    g *= r.c;
    m = fmaf(r.b1, m, r.a1 * g);
    v = fmaf(r.b2, v, r.a2 * g * g);
    const float x = v * r.inv_bias2, y = r.rate * m;
    const float up = TINY ? y / (sqrtf(x) + r.eps) : y * rcp_fast(sqrt_fast(x) + r.eps);
    p -= fmaf(r.decay, p, up);   // both terms first: p is rounded once
}

template <class T, bool TINY>
__device__ __forceinline__ void step_scalar(const StepEntry& e, const StepRates& r, int64_t i) {
    float p = e.p[i];
    if (!r.skip) {
        float m = e.m[i], v = e.v[i];
        adamw_one<TINY>(r, to_f(static_cast<const T*>(e.g)[i]), p, m, v);
        e.p[i] = p;
        e.m[i] = m;
        e.v[i] = v;
    }
    if (e.w) e.w[i] = __float2bfloat16_rn(p);
}

__device__ __forceinline__ void load8(const float* s, float* x) {
    Vec<float>::get(reinterpret_cast<const uint4*>(s)[0], x);
    Vec<float>::get(reinterpret_cast<const uint4*>(s)[1], x + 4);
}
__device__ __forceinline__ void store8(float* s, const float* x) {
    reinterpret_cast<uint4*>(s)[0] = Vec<float>::put(x);
    reinterpret_cast<uint4*>(s)[1] = Vec<float>::put(x + 4);
}
template <class T>
__device__ __forceinline__ void load8_g(const T* s, float* x) { Vec<T>::get(*reinterpret_cast<const uint4*>(s), x); }
template <>
__device__ __forceinline__ void load8_g<float>(const float* s, float* x) { load8(s, x); }

template <class T, bool TINY>
__device__ __forceinline__ void tile_step(const StepEntry& e, const StepRates& r, int64_t k) {
    const int tid = threadIdx.x;
    if (e.head < 0) {   // no common alignment
        const int64_t base = k * kStepTile, end = tmin<int64_t>(e.numel, base + kStepTile);
        for (int64_t i = base + tid; i < end; i += kThreads) step_scalar<T, TINY>(e, r, i);
        return;
    }
    if (k == 0 && tid < tmin<int64_t>(e.head, e.numel)) step_scalar<T, TINY>(e, r, tid);
    const int64_t i = e.head + k * kStepTile + tid * 8;
    if (i + 8 <= e.numel) {
        float g[8], p[8], m[8], v[8];
        load8(e.p + i, p);
        if (!r.skip) {
            load8_g(static_cast<const T*>(e.g) + i, g);
            load8(e.m + i, m);
            load8(e.v + i, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) adamw_one<TINY>(r, g[j], p[j], m[j], v[j]);
            store8(e.p + i, p);
            store8(e.m + i, m);
            store8(e.v + i, v);
        }
        if (e.w) *reinterpret_cast<uint4*>(e.w + i) = Vec<__nv_bfloat16>::put(p);
    } else {
        for (int64_t j = i; j < e.numel; ++j) step_scalar<T, TINY>(e, r, j);
    }
}

template <bool TINY, class Tab>
__global__ void __launch_bounds__(kThreads) k_adamw(const __grid_constant__ Tab t, const __grid_constant__ StepHyper h) {
    StepRates r;
    r.skip = false;
    r.c = 1.f;
    if (h.norm) {
        const float norm = *h.norm;
        r.skip = !(fabsf(norm) <= 3.402823466e38f);
        if (h.max_norm > 0.f) r.c = clip_coef(norm, h.max_norm);
    }
    const float lr = h.lr_p ? *h.lr_p : h.lr;
    float bias1 = h.bias1, bias2 = h.bias2;
    if (h.step_p) {
        const double step = double(*h.step_p);
        bias1 = float(-expm1(step * h.log_b1));
        bias2 = float(-expm1(step * h.log_b2));
    }
    r.b1 = h.b1;
    r.b2 = h.b2;
    r.a1 = h.a1;
    r.a2 = h.a2;
    r.decay = lr * h.decay;
    r.rate = lr / bias1;
    r.inv_bias2 = 1.f / bias2;
    r.eps = h.eps;
    const StepEntry& e = t.e[tensor_of(t, blockIdx.x)];
    const int64_t k = blockIdx.x - e.tile;
    if (e.dtype == CRX_FP32) tile_step<float, TINY>(e, r, k);
    else if (e.dtype == CRX_BF16) tile_step<__nv_bfloat16, TINY>(e, r, k);
    else tile_step<__half, TINY>(e, r, k);
}

// ------------------------------------------------------------------ host

int elem_size(int dtype) { return dtype == CRX_FP32 ? 4 : 2; }

int fail(char* err, size_t errlen, int status, const std::string& msg) {
    if (err && errlen) std::snprintf(err, errlen, "%s", msg.c_str());
    return status;
}

int cuda_fail(char* err, size_t errlen, const char* who, cudaError_t e) {
    return fail(err, errlen, CRX_CUDA_ERROR, std::string(who) + ": " + cudaGetErrorString(e));
}

struct Range {
    uintptr_t lo, hi;
    bool write;
    int32_t tensor;
};

// Two tensors of which at least one is written may not share memory (a race otherwise).  `r` holds
// groups of `each` ranges; those of one group mostly lie in order, so groups are merged, not sorted
// as a whole (2400 ranges: 100 us).
bool overlap(std::vector<Range>& r, size_t each, int32_t* a, int32_t* b) {
    const auto below = [](const Range& x, const Range& y) { return x.lo < y.lo; };
    for (size_t i = 0; i < r.size(); i += each)
        if (!std::is_sorted(r.begin() + i, r.begin() + std::min(r.size(), i + each), below))
            std::sort(r.begin() + i, r.begin() + std::min(r.size(), i + each), below);
    for (; each < r.size(); each *= 2)
        for (size_t i = 0; i + each < r.size(); i += 2 * each)
            if (below(r[i + each], r[i + each - 1]))
                std::inplace_merge(r.begin() + i, r.begin() + i + each, r.begin() + std::min(r.size(), i + 2 * each), below);
    const Range* any = nullptr;       // the range so far that reaches furthest
    const Range* written = nullptr;   // and the written one
    for (const Range& x : r) {
        const Range* hit = written && written->hi > x.lo ? written : x.write && any && any->hi > x.lo ? any : nullptr;
        if (hit) {
            *a = hit->tensor;
            *b = x.tensor;
            return true;
        }
        if (!any || x.hi > any->hi) any = &x;
        if (x.write && (!written || x.hi > written->hi)) written = &x;
    }
    return false;
}

int check_common(const char* who, int32_t n, const void* const* grads, const int32_t* dtypes, const int64_t* numel, char* err,
                 size_t errlen) {
    if (n < 0 || (n && (!grads || !dtypes || !numel))) return fail(err, errlen, CRX_BAD_ARGUMENT, std::string(who) + ": null pointer or negative count");
    for (int32_t i = 0; i < n; ++i) {
        if (numel[i] < 0 || numel[i] > (int64_t(1) << 40)) return fail(err, errlen, CRX_BAD_ARGUMENT, std::string(who) + ": bad element count of tensor " + std::to_string(i));
        if (dtypes[i] != CRX_BF16 && dtypes[i] != CRX_FP16 && dtypes[i] != CRX_FP32)
            return fail(err, errlen, CRX_BAD_ARGUMENT, std::string(who) + ": unknown type of tensor " + std::to_string(i));
        if (numel[i] && (!grads[i] || reinterpret_cast<uintptr_t>(grads[i]) % elem_size(dtypes[i])))
            return fail(err, errlen, CRX_BAD_ARGUMENT, std::string(who) + ": null or misaligned gradient " + std::to_string(i));
    }
    return CRX_OK;
}

uint32_t grad_tiles(const void* g, int64_t numel, int dtype) {
    const int head = dtype == CRX_FP32 ? head_of<float>(g) : head_of<__half>(g);
    const int64_t body = std::max<int64_t>(0, numel - head);
    return uint32_t(std::max<int64_t>(1, (body + kTile - 1) / kTile));
}

// Calls f(table, tables so far) for each launch's worth of the non-empty tensors.
template <class E, int N, class Fill, class Launch>
cudaError_t each_table(int32_t n, const int64_t* numel, int32_t* at, Fill fill, Launch launch) {
    Table<E, N> t;
    int32_t i = *at;
    t.n = 0;
    t.tiles = 0;
    for (; i < n && t.n < N; ++i) {
        if (numel[i] == 0) continue;
        E& e = t.e[t.n];
        e.tile = t.tiles;
        const uint32_t tiles = fill(e, i);
        if (uint64_t(t.tiles) + tiles > 0x7fffffffull) break;   // a grid's most: the rest goes into the next launch
        t.tiles += tiles;
        ++t.n;
    }
    *at = i;
    return t.n ? launch(t) : cudaSuccess;
}

template <class E, int Large, class Fill, class Launch>
cudaError_t all_tables(int32_t n, const int64_t* numel, Fill fill, Launch launch) {
    int32_t filled = 0;
    for (int32_t i = 0; i < n; ++i) filled += numel[i] != 0;
    for (int32_t at = 0; at < n;) {
        const cudaError_t e = filled <= kSmall    ? each_table<E, kSmall>(n, numel, &at, fill, launch)
                              : filled <= kMedium ? each_table<E, kMedium>(n, numel, &at, fill, launch)
                                                  : each_table<E, Large>(n, numel, &at, fill, launch);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

int64_t partials_needed(int32_t n) { return int64_t(kMaxGrid) * (1 + n / kGradLarge); }

// Every launch's partials one behind the other; *count of them.
cudaError_t launch_sumsq(int32_t n, const void* const* grads, const int32_t* dtypes, const int64_t* numel, double* partials,
                         int* count, cudaStream_t st) {
    *count = 0;
    return all_tables<GradEntry, kGradLarge>(
        n, numel,
        [&](GradEntry& e, int32_t i) {
            e.g = grads[i];
            e.out = nullptr;
            e.numel = numel[i];
            e.dtype = dtypes[i];
            return grad_tiles(grads[i], numel[i], dtypes[i]);
        },
        [&](const auto& t) {
            const int grid = int(std::min<uint32_t>(t.tiles, kMaxGrid));
            k_grad_sumsq<<<grid, kThreads, 0, st>>>(t, partials + *count);
            *count += grid;
            return cudaGetLastError();
        });
}

}  // namespace
}  // namespace crx

using namespace crx;

extern "C" {

int64_t crx_grads_workspace(int32_t n_tensors) { return n_tensors < 0 ? 0 : int64_t(sizeof(double)) * partials_needed(n_tensors); }

int crx_grad_norm(int32_t n, const void* const* grads, const int32_t* dtypes, const int64_t* numel, void* workspace,
                  int64_t workspace_bytes, float* norm, void* stream, char* err, size_t errlen) {
    try {
        if (const int s = check_common("crx_grad_norm", n, grads, dtypes, numel, err, errlen)) return s;
        if (!norm || !workspace || reinterpret_cast<uintptr_t>(workspace) % 8 || workspace_bytes < crx_grads_workspace(n))
            return fail(err, errlen, CRX_BAD_ARGUMENT, "crx_grad_norm: no room for the result or the workspace");
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        double* partials = static_cast<double*>(workspace);
        int count = 0;
        cudaError_t e = launch_sumsq(n, grads, dtypes, numel, partials, &count, st);
        if (e == cudaSuccess) {
            e = count ? launch_behind(k_grad_norm, 1, kThreads, st, static_cast<const double*>(partials), count, norm)
                      : cudaMemsetAsync(norm, 0, sizeof(float), st);
        }
        return e == cudaSuccess ? CRX_OK : cuda_fail(err, errlen, "crx_grad_norm", e);
    } catch (const std::exception& ex) {
        return fail(err, errlen, CRX_NO_MEMORY, std::string("crx_grad_norm: ") + ex.what());
    }
}

int crx_clip_grads(int32_t n, const void* const* grads, void* const* out, const int32_t* dtypes, const int64_t* numel,
                   float max_norm, const float* norm_in, void* workspace, int64_t workspace_bytes, float* norm_out, void* stream,
                   char* err, size_t errlen) {
    try {
        if (const int s = check_common("crx_clip_grads", n, grads, dtypes, numel, err, errlen)) return s;
        if (n && !out) return fail(err, errlen, CRX_BAD_ARGUMENT, "crx_clip_grads: null pointer");
        if (!(max_norm > 0.f)) return fail(err, errlen, CRX_VALUE_ERROR, "max_norm must be positive");
        if (!norm_in && (!norm_out || !workspace || reinterpret_cast<uintptr_t>(workspace) % 8 || workspace_bytes < crx_grads_workspace(n)))
            return fail(err, errlen, CRX_BAD_ARGUMENT, "crx_clip_grads: no room for the norm or the workspace");
        std::vector<Range> r;
        r.reserve(size_t(n) * 2);
        for (int32_t i = 0; i < n; ++i) {
            if (!numel[i]) continue;
            const int64_t bytes = numel[i] * elem_size(dtypes[i]);
            if (!out[i] || reinterpret_cast<uintptr_t>(out[i]) % elem_size(dtypes[i]))
                return fail(err, errlen, CRX_BAD_ARGUMENT, "crx_clip_grads: null or misaligned output " + std::to_string(i));
            const uintptr_t o = reinterpret_cast<uintptr_t>(out[i]);
            r.push_back(Range{o, o + uintptr_t(bytes), true, i});
        }
        const size_t written = std::max<size_t>(1, r.size());
        for (int32_t i = 0; i < n; ++i) {
            const uintptr_t g = reinterpret_cast<uintptr_t>(grads[i]);
            if (numel[i] && out[i] != grads[i]) r.push_back(Range{g, g + uintptr_t(numel[i]) * elem_size(dtypes[i]), false, i});
        }
        int32_t a, b;
        if (overlap(r, written, &a, &b))
            return fail(err, errlen, CRX_VALUE_ERROR, "tensors " + std::to_string(a) + " and " + std::to_string(b) + " share memory that would be written");
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        double* partials = static_cast<double*>(workspace);
        int count = 0;
        cudaError_t e = norm_in ? cudaSuccess : launch_sumsq(n, grads, dtypes, numel, partials, &count, st);
        float* write_norm = norm_out;   // by the first launch that knows it
        bool behind = norm_in == nullptr;
        if (e == cudaSuccess && count > kClipPartials) {
            e = launch_behind(k_grad_norm, 1, kThreads, st, static_cast<const double*>(partials), count, norm_out);
            norm_in = norm_out;
            write_norm = nullptr;
            count = 0;
        }
        if (e == cudaSuccess)
            e = all_tables<GradEntry, kGradLarge>(
                n, numel,
                [&](GradEntry& x, int32_t i) {
                    x.g = grads[i];
                    x.out = out[i];
                    x.numel = numel[i];
                    x.dtype = dtypes[i];
                    return grad_tiles(grads[i], numel[i], dtypes[i]);
                },
                [&](const auto& t) {
                    using Tab = std::decay_t<decltype(t)>;
                    float* const w = write_norm;
                    write_norm = nullptr;
                    if (std::exchange(behind, false))
                        return launch_behind(k_grad_clip<Tab>, t.tiles, kThreads, st, t, static_cast<const double*>(partials), count, norm_in, max_norm, w);
                    k_grad_clip<<<t.tiles, kThreads, 0, st>>>(t, partials, count, norm_in, max_norm, w);
                    return cudaGetLastError();
                });
        if (e == cudaSuccess && write_norm) {   // no elements at all
            if (norm_in) e = cudaMemcpyAsync(write_norm, norm_in, sizeof(float), cudaMemcpyDeviceToDevice, st);
            else e = cudaMemsetAsync(write_norm, 0, sizeof(float), st);
        }
        return e == cudaSuccess ? CRX_OK : cuda_fail(err, errlen, "crx_clip_grads", e);
    } catch (const std::exception& ex) {
        return fail(err, errlen, CRX_NO_MEMORY, std::string("crx_clip_grads: ") + ex.what());
    }
}

int crx_adamw_step(int32_t n, float* const* master, const void* const* grads, const int32_t* dtypes, float* const* exp_avg,
                   float* const* exp_avg_sq, void* const* weights, const int64_t* numel, const crx_adamw_args* args, void* stream,
                   char* err, size_t errlen) {
    try {
        if (const int s = check_common("crx_adamw_step", n, grads, dtypes, numel, err, errlen)) return s;
        if (!args || (n && (!master || !exp_avg || !exp_avg_sq))) return fail(err, errlen, CRX_BAD_ARGUMENT, "crx_adamw_step: null pointer");
        if (!(args->beta1 >= 0 && args->beta1 < 1 && args->beta2 >= 0 && args->beta2 < 1)) return fail(err, errlen, CRX_VALUE_ERROR, "betas must be in [0, 1)");
        // in fp32, as the kernel takes them
        if (!(float(args->eps) > 0)) return fail(err, errlen, CRX_VALUE_ERROR, "eps must be positive");
        if (!std::isfinite(float(args->weight_decay)) || (!args->lr_p && !std::isfinite(float(args->lr))))
            return fail(err, errlen, CRX_VALUE_ERROR, "lr and weight_decay must be finite");
        if (!args->step_p && args->step < 1) return fail(err, errlen, CRX_VALUE_ERROR, "step counts from 1");
        std::vector<Range> r;
        r.reserve(size_t(n) * 5);
        size_t each = 0;
        for (int kind = 0; kind < 5; ++kind) {   // masters, moments, weights, gradients
            if (kind == 3 && !weights) continue;
            const int size = kind < 3 ? 4 : 2;
            for (int32_t i = 0; i < n; ++i) {
                if (!numel[i]) continue;
                const void* q = kind == 0 ? master[i] : kind == 1 ? exp_avg[i] : kind == 2 ? exp_avg_sq[i] : kind == 3 ? weights[i] : grads[i];
                const int es = kind == 4 ? elem_size(dtypes[i]) : size;
                if (!q || reinterpret_cast<uintptr_t>(q) % es)
                    return fail(err, errlen, CRX_BAD_ARGUMENT, "crx_adamw_step: null or misaligned state or weights " + std::to_string(i));
                const uintptr_t lo = reinterpret_cast<uintptr_t>(q);
                r.push_back(Range{lo, lo + uintptr_t(numel[i]) * es, kind < 4, i});
            }
            if (kind == 0) each = std::max<size_t>(1, r.size());
        }
        int32_t a, b;
        if (overlap(r, each, &a, &b))
            return fail(err, errlen, CRX_VALUE_ERROR, "tensors " + std::to_string(a) + " and " + std::to_string(b) + " share memory that would be written");
        StepHyper h;
        h.lr = float(args->lr);
        h.b1 = float(args->beta1);
        h.b2 = float(args->beta2);
        h.a1 = float(1.0 - args->beta1);
        h.a2 = float(1.0 - args->beta2);
        h.eps = float(args->eps);
        h.decay = float(args->weight_decay);
        h.log_b1 = std::log(args->beta1);   // beta 0: -inf, and 1 - 0^t = 1
        h.log_b2 = std::log(args->beta2);
        h.bias1 = float(-std::expm1(double(args->step) * h.log_b1));
        h.bias2 = float(-std::expm1(double(args->step) * h.log_b2));
        h.lr_p = args->lr_p;
        h.step_p = args->step_p;
        h.norm = args->norm;
        h.max_norm = args->max_norm;
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        const cudaError_t e = all_tables<StepEntry, kStepLarge>(
            n, numel,
            [&](StepEntry& x, int32_t i) {
                x.g = grads[i];
                x.p = master[i];
                x.m = exp_avg[i];
                x.v = exp_avg_sq[i];
                x.w = weights ? static_cast<__nv_bfloat16*>(weights[i]) : nullptr;
                x.numel = numel[i];
                x.dtype = int16_t(dtypes[i]);
                x.head = -1;
                for (int k = 0; k < 8 && x.head < 0; ++k) {
                    const auto at = [&](const void* q, int size) { return (reinterpret_cast<uintptr_t>(q) + uintptr_t(k) * size) % 16 == 0; };
                    if (at(x.g, elem_size(dtypes[i])) && at(x.p, 4) && at(x.m, 4) && at(x.v, 4) && (!x.w || at(x.w, 2))) x.head = int16_t(k);
                }
                const int64_t body = std::max<int64_t>(0, numel[i] - std::max<int>(0, x.head));
                return uint32_t(std::max<int64_t>(1, (body + kStepTile - 1) / kStepTile));
            },
            [&](const auto& t) {
                if (args->eps < kTinyEps) k_adamw<true><<<t.tiles, kThreads, 0, st>>>(t, h);
                else k_adamw<false><<<t.tiles, kThreads, 0, st>>>(t, h);
                return cudaGetLastError();
            });
        return e == cudaSuccess ? CRX_OK : cuda_fail(err, errlen, "crx_adamw_step", e);
    } catch (const std::exception& ex) {
        return fail(err, errlen, CRX_NO_MEMORY, std::string("crx_adamw_step: ") + ex.what());
    }
}

}  // extern "C"
