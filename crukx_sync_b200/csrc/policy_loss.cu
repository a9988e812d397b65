// The clipped policy loss with a KL term over [batch, steps] tokens, from the logits, with its
// gradient to them (crx_policy_loss, crx_policy_backward; no reference counterpart).
//
// Per row of V logits, in units of log2 (c = log2(e) / temperature):
//   M = max z, R = M c, s = sum 2^(z c - R)        one pass, the maximum kept as it goes
//   logp = (z_a c - R - log2 s) ln 2
//   d loss / d z_j = u (1[j = a] - 2^(z_j c - R) / s),  u = w / D / temperature * d l / d logp
// u depends on the row's own logp alone (D is known before), so the gradient is written in the
// same visit to the row: the logits are read from HBM once and written once.
//
//   k_policy_denom   one CTA: 1 / sum of the mask (only where the caller gives no denominator)
//   k_policy_rows    a cluster of CTAs per row, rows dealt to the clusters of a persistent grid;
//                    each CTA has a slice of the row; the (M, s) of the slices meet through
//                    distributed shared memory; then the gradient, from the slice again (L2)
//   k_policy_sums    one CTA: the rows' terms summed in a fixed order, in double
//   k_policy_again   the gradient once more, scaled, from the rows' saved (u, R, s)
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <exception>
#include <string>

#include "../../include/crukx_b200.h"
#include "common.cuh"
#include "elements.cuh"

namespace crx {
namespace {

namespace cg = cooperative_groups;

constexpr int kRowThreads = 512;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kMaxCluster = 8;
constexpr float kFar = 3e38f;

// 2^x to about 2 ulp; results below 2^-126 become 0, which neither a sum of at least 1 nor a
// gradient in any of the types can tell from them.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ int64_t at(const crx_rows& r, int64_t b, int64_t t) { return b * r.stride_b + t * r.stride_t; }
__device__ __forceinline__ float value(const crx_rows& r, int64_t b, int64_t t) { return static_cast<const float*>(r.p)[at(r, b, t)]; }

__device__ __forceinline__ float weight(const crx_policy_args& a, int64_t b, int64_t t) {
    if (!a.mask.p) return 1.f;
    if (a.mask_f32) return value(a.mask, b, t);
    return static_cast<const uint8_t*>(a.mask.p)[at(a.mask, b, t)] ? 1.f : 0.f;
}

// Layout of args.rows: 1 / denominator (double, 16 bytes), a float4 per row, then the sums of the
// three terms over each cluster's rows (double).  A row's float4 is (u, R, s, 0), or (u, M, s, 1)
// for a far row (below).
__host__ __device__ __forceinline__ double* inv_denom_of(const crx_policy_args& a) { return reinterpret_cast<double*>(a.rows); }
__device__ __forceinline__ float4* saved_of(const crx_policy_args& a) { return reinterpret_cast<float4*>(a.rows) + 1; }
__host__ __device__ __forceinline__ double* partials_of(const crx_policy_args& a) {
    return reinterpret_cast<double*>(a.rows + 4 + 4 * a.batch * a.steps);
}

// The largest of N packed values (NaNs lose; they show in the sum).
template <class T> __device__ __forceinline__ float vec_max(const uint4* q, int n);
template <> __device__ __forceinline__ float vec_max<float>(const uint4* q, int n) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < n; ++i) {
        float x[4];
        Vec<float>::get(q[i], x);
        m = fmaxf(fmaxf(m, fmaxf(x[0], x[1])), fmaxf(x[2], x[3]));
    }
    return m;
}
template <class H2>
__device__ __forceinline__ H2 as2(uint32_t u) {
    H2 h;
    memcpy(&h, &u, 4);
    return h;
}
template <> __device__ __forceinline__ float vec_max<__nv_bfloat16>(const uint4* q, int n) {
    __nv_bfloat162 m = as2<__nv_bfloat162>(q[0].x);
#pragma unroll
    for (int i = 0; i < n; ++i) {
        const __nv_bfloat162 a = __hmax2(as2<__nv_bfloat162>(q[i].x), as2<__nv_bfloat162>(q[i].y));
        const __nv_bfloat162 b = __hmax2(as2<__nv_bfloat162>(q[i].z), as2<__nv_bfloat162>(q[i].w));
        m = __hmax2(m, __hmax2(a, b));
    }
    return fmaxf(__low2float(m), __high2float(m));
}
template <> __device__ __forceinline__ float vec_max<__half>(const uint4* q, int n) {
    __half2 m = as2<__half2>(q[0].x);
#pragma unroll
    for (int i = 0; i < n; ++i) {
        const __half2 a = __hmax2(as2<__half2>(q[i].x), as2<__half2>(q[i].y));
        const __half2 b = __hmax2(as2<__half2>(q[i].z), as2<__half2>(q[i].w));
        m = __hmax2(m, __hmax2(a, b));
    }
    return fmaxf(__low2float(m), __high2float(m));
}

// The running (maximum, sum of 2^(z c - R)) of one thread, R = max(M c, -kFar).  The bound keeps R
// finite where everything so far is -inf or the type's lowest value: those add 0.
struct Running {
    float m = -INFINITY, r = -kFar, s = 0.f;
    __device__ __forceinline__ void raise(float top, float c) {
        if (top > m) {
            const float r2 = fmaxf(top * c, -kFar);
            s *= exp2_fast(r - r2);
            m = top;
            r = r2;
        }
    }
    __device__ __forceinline__ void join(float m2, float s2, float c) {
        const float r2 = fmaxf(m2 * c, -kFar);
        const float big = fmaxf(r, r2);
        s = s * exp2_fast(r - big) + s2 * exp2_fast(r2 - big);
        r = big;
        m = fmaxf(m, m2);
    }
};

template <class T, int U>
__device__ __forceinline__ void add_vecs(const uint4* q, Running& run, float c) {
    run.raise(vec_max<T>(q, U), c);
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float x[Vec<T>::N];
        Vec<T>::get(q[u], x);
#pragma unroll
        for (int i = 0; i < Vec<T>::N; i += 2) {
            a += exp2_fast(fmaf(x[i], c, -run.r));
            b += exp2_fast(fmaf(x[i + 1], c, -run.r));
        }
    }
    run.s += a + b;
}

// A CTA's slice of a row: 16-byte vectors [lo, hi) of the part after the row's first 16-byte
// boundary; the first CTA also has the elements before it and the row's last ones.
struct Slice {
    int head, tail;   // elements before the boundary, and after the last whole vector (first CTA)
    int64_t body;     // element of the first whole vector
    int64_t tail_at;  // element where the tail begins
    int64_t lo, hi;
};
template <class T>
__device__ __forceinline__ Slice slice_of(const T* z, int64_t V, int rank, int C) {
    Slice s;
    const int head = int(tmin<int64_t>(head_of<T>(z), V));
    const int64_t nv = (V - head) / Vec<T>::N;
    s.lo = nv * rank / C;
    s.hi = nv * (rank + 1) / C;
    s.head = rank ? 0 : head;
    s.body = head;
    s.tail_at = head + nv * Vec<T>::N;
    s.tail = rank ? 0 : int(V - s.tail_at);
    return s;
}

struct Shared {
    float2 warp[kRowWarps];
    float2 part[2][kMaxCluster];   // (M, s) of every CTA of the cluster, double-buffered over rows
};

// (M, s) of the whole row from every thread's; the same bits in every thread of the cluster.
__device__ __forceinline__ Running row_total(Running run, Shared& sh, int parity, int rank, int C, float c) {
    for (int o = 16; o; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, run.m, o), s2 = __shfl_xor_sync(0xffffffffu, run.s, o);
        run.join(m2, s2, c);
    }
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) sh.warp[w] = make_float2(run.m, run.s);
    __syncthreads();
    Running all;
    if (C == 1) {
        for (int k = 0; k < kRowWarps; ++k) all.join(sh.warp[k].x, sh.warp[k].y, c);
        __syncthreads();   // sh.warp is written again by the next row
        return all;
    }
    cg::cluster_group cl = cg::this_cluster();
    if (w == 0) {
        for (int k = 0; k < kRowWarps; ++k) all.join(sh.warp[k].x, sh.warp[k].y, c);
        if (lane < C) *cl.map_shared_rank(&sh.part[parity][rank], lane) = make_float2(all.m, all.s);
    }
    cl.sync();
    all = Running();
    for (int k = 0; k < C; ++k) all.join(sh.part[parity][k].x, sh.part[parity][k].y, c);
    return all;
}

__device__ __forceinline__ float block_total(float v, Shared& sh) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.warp[threadIdx.x >> 5].y = v;
    __syncthreads();
    v = 0.f;
    for (int k = 0; k < kRowWarps; ++k) v += sh.warp[k].y;
    __syncthreads();
    return v;
}

// The sum of a far row: one whose largest logit M is so large in magnitude that M c does not fit
// fp32 (every logit the type's lowest value, say).  (z - M) c takes the place of z c - R, and each
// CTA of the cluster goes over the whole row.
template <class T>
__device__ __noinline__ float far_sum(const T* z, int64_t V, float M, float c, Shared& sh) {
    float s = 0.f;
    for (int64_t j = threadIdx.x; j < V; j += kRowThreads) s += exp2_fast((to_f(z[j]) - M) * c);
    return block_total(s, sh);
}

// The gradient over one CTA's slice, u 1[j = a] - k 2^(z_j c - R) with k = u / s.  u = 0 (a clipped
// token without a KL term, a token that does not count) writes zeros and reads nothing.
template <class T>
__device__ __forceinline__ void write_grad(const T* z, T* g, const Slice& sl, int64_t V, int64_t token, float u, float R, float s,
                                           float c, bool far) {
    constexpr int N = Vec<T>::N;
    const int tid = threadIdx.x;
    const float k = u == 0.f ? 0.f : u / s;
    const auto one = [&](int64_t j) {
        float x = 0.f;
        if (u != 0.f) {
            const float f = to_f(z[j]);
            x = -k * exp2_fast(far ? (f - R) * c : fmaf(f, c, -R));
            if (j == token) x += u;
        }
        g[j] = from_f<T>(x);
    };
    if (tid < sl.head) one(tid);
    if (tid < sl.tail) one(sl.tail_at + tid);
    const int64_t body = sl.body;
    const bool wide = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(g)) & 15) == 0;
    if (!wide || far) {
        for (int64_t j = body + sl.lo * N + tid; j < body + sl.hi * N; j += kRowThreads) one(j);
        return;
    }
    const uint4* zv = reinterpret_cast<const uint4*>(z + body);
    uint4* gv = reinterpret_cast<uint4*>(g + body);
    if (u == 0.f) {
        for (int64_t i = sl.lo + tid; i < sl.hi; i += kRowThreads) gv[i] = make_uint4(0, 0, 0, 0);
        return;
    }
    const int64_t token_vec = token >= body ? (token - body) / N : -1;
    const auto vec = [&](int64_t i, const uint4& q) {
        float x[N];
        Vec<T>::get(q, x);
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = -k * exp2_fast(fmaf(x[e], c, -R));
        if (i == token_vec) {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (body + i * N + e == token) x[e] += u;
        }
        gv[i] = Vec<T>::put(x);
    };
    constexpr int U = 4;
    int64_t i = sl.lo + tid;
    for (; i + (U - 1) * kRowThreads < sl.hi; i += U * kRowThreads) {
        uint4 q[U];
#pragma unroll
        for (int v = 0; v < U; ++v) q[v] = zv[i + v * kRowThreads];
#pragma unroll
        for (int v = 0; v < U; ++v) vec(i + v * kRowThreads, q[v]);
    }
    for (; i < sl.hi; i += kRowThreads) vec(i, zv[i]);
}

template <class T, bool GRAD>
__global__ void __launch_bounds__(kRowThreads) k_policy_rows(const __grid_constant__ crx_policy_args a, double inv_denom, int C) {
    __shared__ Shared sh;
    const int tid = threadIdx.x, rank = int(blockIdx.x) % C;
    const int64_t n = a.batch * a.steps, V = a.vocab, clusters = gridDim.x / C;
    const float c = float(1.4426950408889634 / double(a.temperature));
    const double inv_d = inv_denom < 0 ? *inv_denom_of(a) : inv_denom;
    double loss = 0, kl = 0, cut = 0;
    int parity = 0;
    if (C > 1) cg::this_cluster().sync();   // every CTA runs before another writes to its shared memory
    for (int64_t row = blockIdx.x / C; row < n; row += clusters) {
        const int64_t b = row / a.steps, t = row - b * a.steps;
        const float w = weight(a, b, t);
        const T* z = static_cast<const T*>(a.logits.p) + at(a.logits, b, t);
        T* g = GRAD ? static_cast<T*>(const_cast<void*>(a.grad.p)) + at(a.grad, b, t) : nullptr;
        const Slice sl = slice_of<T>(z, V, rank, C);
        if (w == 0.f) {
            if (GRAD) write_grad<T>(z, g, sl, V, -1, 0.f, 0.f, 1.f, c, false);
            if (rank == 0 && tid == 0) {
                a.logp[row] = 0.f;
                saved_of(a)[row] = make_float4(0.f, 0.f, 1.f, 0.f);
            }
            continue;
        }
        const int64_t token = a.tokens64 ? static_cast<const int64_t*>(a.tokens.p)[at(a.tokens, b, t)]
                                         : static_cast<const int32_t*>(a.tokens.p)[at(a.tokens, b, t)];
        const float za = token >= 0 && token < V ? to_f(z[token]) : NAN;
        const float A = value(a.advantages, b, t);
        const float old = a.old_logp.p ? value(a.old_logp, b, t) : 0.f;
        const float ref = a.ref_logp.p ? value(a.ref_logp, b, t) : 0.f;

        Running run;
        {
            const auto one = [&](int64_t j) {
                const float x = to_f(z[j]);
                run.raise(x, c);
                run.s += exp2_fast(fmaf(x, c, -run.r));
            };
            if (tid < sl.head) one(tid);
            if (tid < sl.tail) one(sl.tail_at + tid);
            const uint4* zv = reinterpret_cast<const uint4*>(z + sl.body);
            constexpr int U = 4;
            int64_t i = sl.lo + tid;
            for (; i + (U - 1) * kRowThreads < sl.hi; i += U * kRowThreads) {
                uint4 q[U];
#pragma unroll
                for (int v = 0; v < U; ++v) q[v] = zv[i + v * kRowThreads];
                add_vecs<T, U>(q, run, c);
            }
            for (; i < sl.hi; i += kRowThreads) {
                const uint4 q = zv[i];
                add_vecs<T, 1>(&q, run, c);
            }
        }
        run = row_total(run, sh, parity, rank, C, c);
        parity ^= 1;
        const bool far = fabsf(run.m) <= 3.402823466e38f && !(fabsf(run.m * c) < kFar);
        const float s = far ? far_sum<T>(z, V, run.m, c, sh) : run.s;
        const float R = far ? run.m : run.r;
        const float logp = ((far ? (za - R) * c : fmaf(za, c, -R)) - log2f(s)) * 0.6931471805599453f;

        const float r = a.old_logp.p ? expf(logp - old) : (logp == logp ? 1.f : logp);   // NaN logits show in the loss
        const bool clipped = (A > 0.f && r > 1.f + a.clip_high) || (A < 0.f && r < 1.f - a.clip_low);
        const float gain = A == 0.f ? 0.f : (clipped ? (A > 0.f ? 1.f + a.clip_high : 1.f - a.clip_low) : r) * A;
        float dl = clipped ? 0.f : -gain, k = 0.f;
        if (a.ref_logp.p) {
            const float x = ref - logp, e = expm1f(x);
            k = e - x;
            dl -= a.kl_coef * e;
        }
        const float u = float(double(w) * inv_d * double(dl) / double(a.temperature));
        if (rank == 0 && tid == 0) {
            a.logp[row] = logp;
            saved_of(a)[row] = make_float4(u, R, s, far ? 1.f : 0.f);
            loss += double(w) * (double(a.ref_logp.p ? a.kl_coef * k : 0.f) - double(gain));
            kl += double(w) * double(k);
            cut += clipped ? double(w) : 0.0;
        }
        if (GRAD) write_grad<T>(z, g, sl, V, token, u, R, s, c, far);
    }
    if (rank == 0 && tid == 0) {
        double* p = partials_of(a) + 3 * (blockIdx.x / C);
        p[0] = loss;
        p[1] = kl;
        p[2] = cut;
    }
}

__device__ __forceinline__ double warp_sum(double v) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__global__ void __launch_bounds__(1024) k_policy_denom(const __grid_constant__ crx_policy_args a) {
    __shared__ double red[32];
    double v = 0;
    for (int64_t i = threadIdx.x; i < a.batch * a.steps; i += 1024) {
        const int64_t b = i / a.steps;
        v += double(weight(a, b, i - b * a.steps));
    }
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x < 32) {
        v = warp_sum(red[threadIdx.x]);
        if (threadIdx.x == 0) *inv_denom_of(a) = v == 0.0 ? 0.0 : 1.0 / v;
    }
}

// Warp i sums term i.
__global__ void __launch_bounds__(96) k_policy_sums(const __grid_constant__ crx_policy_args a, double inv_denom, int clusters) {
    const int i = threadIdx.x >> 5, lane = threadIdx.x & 31;
    double v = 0;
    for (int k = lane; k < clusters; k += 32) v += partials_of(a)[3 * k + i];
    v = warp_sum(v) * (inv_denom < 0 ? *inv_denom_of(a) : inv_denom);
    if (lane == 0) *(i ? a.stats + i - 1 : a.loss) = float(v);
}

// The gradient again for a scale other than the one it was written with.  CTAs take (row, slice)
// pairs; nothing has to meet.
template <class T>
__global__ void __launch_bounds__(kRowThreads) k_policy_again(const __grid_constant__ crx_policy_args a, const float* __restrict__ scale,
                                                              int unless_one, int C) {
    const float f = *scale;
    if (unless_one && f == 1.f) return;
    const int64_t n = a.batch * a.steps;
    const float c = float(1.4426950408889634 / double(a.temperature));
    for (int64_t item = blockIdx.x; item < n * C; item += gridDim.x) {
        const int64_t row = item / C, b = row / a.steps, t = row - b * a.steps;
        const T* z = static_cast<const T*>(a.logits.p) + at(a.logits, b, t);
        T* g = static_cast<T*>(const_cast<void*>(a.grad.p)) + at(a.grad, b, t);
        const float4 saved = saved_of(a)[row];
        const int64_t token = a.tokens64 ? static_cast<const int64_t*>(a.tokens.p)[at(a.tokens, b, t)]
                                         : static_cast<const int32_t*>(a.tokens.p)[at(a.tokens, b, t)];
        const float u = saved.x == 0.f ? 0.f : saved.x * f;   // a row that does not count stays 0 whatever the scale
        write_grad<T>(z, g, slice_of<T>(z, a.vocab, int(item - row * C), C), a.vocab, token, u, saved.y, saved.z, c, saved.w != 0.f);
    }
}

// ------------------------------------------------------------------ host

int fail(char* err, size_t errlen, int status, const std::string& msg) {
    if (err && errlen) std::snprintf(err, errlen, "%s", msg.c_str());
    return status;
}

constexpr int kRowGrid = 148 * 2;   // CTAs of the persistent grid
constexpr int kMaxClusters = kRowGrid;

// CTAs per row: as many as the rows leave room for, while a slice keeps 2048 elements.
int cluster_for(int64_t n, int64_t V) {
    int C = 1;
    while (C < kMaxCluster && n * C * 2 <= kRowGrid && V >= 2048 * 2 * C) C *= 2;
    return C;
}

template <class T, bool GRAD>
cudaError_t launch_rows(const crx_policy_args& a, double inv_denom, int* clusters, cudaStream_t st) {
    const int64_t n = a.batch * a.steps;
    const int C = cluster_for(n, a.vocab);
    *clusters = int(std::min<int64_t>(n, kRowGrid / C));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(*clusters * C));
    cfg.blockDim = dim3(kRowThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(C);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = C > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, k_policy_rows<T, GRAD>, a, inv_denom, C);
}

template <class T>
cudaError_t launch_again(const crx_policy_args& a, const float* scale, int unless_one, cudaStream_t st) {
    const int64_t n = a.batch * a.steps;
    const int C = cluster_for(n, a.vocab);
    k_policy_again<T><<<unsigned(std::min<int64_t>(n * C, kRowGrid * 2)), kRowThreads, 0, st>>>(a, scale, unless_one, C);
    return cudaGetLastError();
}

int check(const char* who, const crx_policy_args* a, char* err, size_t errlen) {
    const auto bad = [&](const char* what) { return fail(err, errlen, CRX_BAD_ARGUMENT, std::string(who) + ": " + what); };
    if (!a) return bad("null arguments");
    if (a->batch < 0 || a->steps < 0 || a->vocab < 1 || a->vocab > (int64_t(1) << 31) || a->batch > (int64_t(1) << 31) || a->steps > (int64_t(1) << 31) ||
        (a->batch && a->steps > (int64_t(1) << 40) / a->batch))
        return bad("size out of range");
    if (a->dtype != CRX_BF16 && a->dtype != CRX_FP16 && a->dtype != CRX_FP32) return bad("unknown type");
    const uintptr_t es = a->dtype == CRX_FP32 ? 4 : 2;
    if (!a->loss || !a->stats || !a->rows || reinterpret_cast<uintptr_t>(a->rows) % 16) return bad("null or misaligned result or workspace");
    if (a->batch && a->steps) {
        if (!a->logits.p || !a->tokens.p || !a->advantages.p || !a->logp) return bad("null pointer");
        if (reinterpret_cast<uintptr_t>(a->logits.p) % es || reinterpret_cast<uintptr_t>(a->grad.p) % es) return bad("misaligned logits or gradient");
    }
    if (!(a->temperature > 0.f) || !(a->clip_low >= 0.f) || !(a->clip_high >= 0.f) || !(a->denom >= 0) || !std::isfinite(a->temperature))
        return fail(err, errlen, CRX_VALUE_ERROR, "temperature must be positive and finite, clip bounds and denom not negative");
    return CRX_OK;
}

}  // namespace
}  // namespace crx

using namespace crx;

extern "C" {

int64_t crx_policy_workspace(int64_t batch, int64_t steps) {
    if (batch < 0 || steps < 0) return 0;
    return 16 + 16 * batch * steps + int64_t(sizeof(double)) * 3 * kMaxClusters;
}

int crx_policy_loss(const crx_policy_args* args, void* stream, char* err, size_t errlen) {
    try {
        if (const int s = check("crx_policy_loss", args, err, errlen)) return s;
        const crx_policy_args& a = *args;
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        const int64_t n = a.batch * a.steps;
        cudaError_t e = cudaSuccess;
        if (n == 0) {
            e = cudaMemsetAsync(a.loss, 0, sizeof(float), st);
            if (e == cudaSuccess) e = cudaMemsetAsync(a.stats, 0, 2 * sizeof(float), st);
            return e == cudaSuccess ? CRX_OK : fail(err, errlen, CRX_CUDA_ERROR, std::string("crx_policy_loss: ") + cudaGetErrorString(e));
        }
        // a negative 1 / denominator: the kernels take the one that k_policy_denom wrote
        const double inv_denom = a.denom > 0 ? 1.0 / a.denom : a.mask.p ? -1.0 : 1.0 / double(n);
        if (inv_denom < 0) {
            k_policy_denom<<<1, 1024, 0, st>>>(a);
            e = cudaGetLastError();
        }
        int clusters = 0;
        const bool grad = a.grad.p != nullptr;
        if (e == cudaSuccess) {
            if (a.dtype == CRX_BF16) e = grad ? launch_rows<__nv_bfloat16, true>(a, inv_denom, &clusters, st) : launch_rows<__nv_bfloat16, false>(a, inv_denom, &clusters, st);
            else if (a.dtype == CRX_FP16) e = grad ? launch_rows<__half, true>(a, inv_denom, &clusters, st) : launch_rows<__half, false>(a, inv_denom, &clusters, st);
            else e = grad ? launch_rows<float, true>(a, inv_denom, &clusters, st) : launch_rows<float, false>(a, inv_denom, &clusters, st);
        }
        if (e == cudaSuccess) {
            k_policy_sums<<<1, 96, 0, st>>>(a, inv_denom, clusters);
            e = cudaGetLastError();
        }
        return e == cudaSuccess ? CRX_OK : fail(err, errlen, CRX_CUDA_ERROR, std::string("crx_policy_loss: ") + cudaGetErrorString(e));
    } catch (const std::exception& ex) {
        return fail(err, errlen, CRX_NO_MEMORY, std::string("crx_policy_loss: ") + ex.what());
    }
}

int crx_policy_backward(const crx_policy_args* args, const float* scale, int32_t unless_one, void* stream, char* err, size_t errlen) {
    try {
        if (const int s = check("crx_policy_backward", args, err, errlen)) return s;
        const crx_policy_args& a = *args;
        if (a.batch * a.steps == 0) return CRX_OK;
        if (!scale || !a.grad.p) return fail(err, errlen, CRX_BAD_ARGUMENT, "crx_policy_backward: null pointer");
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        const cudaError_t e = a.dtype == CRX_BF16 ? launch_again<__nv_bfloat16>(a, scale, unless_one, st)
                              : a.dtype == CRX_FP16 ? launch_again<__half>(a, scale, unless_one, st)
                                                    : launch_again<float>(a, scale, unless_one, st);
        return e == cudaSuccess ? CRX_OK : fail(err, errlen, CRX_CUDA_ERROR, std::string("crx_policy_backward: ") + cudaGetErrorString(e));
    } catch (const std::exception& ex) {
        return fail(err, errlen, CRX_NO_MEMORY, std::string("crx_policy_backward: ") + ex.what());
    }
}

}  // extern "C"
