// The clipped policy loss with a KL term over [batch, steps] tokens, from the logits, with its
// gradient to them (crx_policy_loss, crx_policy_backward; no reference counterpart).
//
// Per row of V logits, in units of log2 (c = log2(e) / temperature):
//   M = max z, R = M c, s = sum 2^(z c - R)        one pass, the maximum kept as it goes
//   logp = (z_a - M) / temperature - ln(s 2^(R - M c))      (R is M c rounded to fp32)
//   d loss / d z_j = u (1[j = a] - 2^(z_j c - R) / s),  u = w / D / temperature * d l / d logp
// u depends on the row's own logp alone (D is known before), so the gradient is written in the
// same visit to the row: the logits are read from HBM once and written once.
//
//   k_policy_plan    one CTA, where there is a mask: 1 / its sum, and the rows in the order in which
//                    they are taken: those that count, then the others (whose gradient is 0)
//   k_policy_rows    a warp, a CTA or a cluster of CTAs per row, rows dealt to a persistent grid.
//                    Every warp streams its part of the rows through a ring of its own in shared
//                    memory, filled by bulk copies that run ahead into the next rows while this one
//                    is reduced; a row that fits its ring is turned into the gradient from there
//   k_policy_sums    one CTA: the terms of the rows summed in a fixed order, in double
//   k_policy_again   the gradient once more, scaled, from the rows' saved (u, R, s)
//
// Bounds: HBM (without gradient 4096 x 152k rows, 894 MB that count, take 0.17 ms, 5.2 TB/s; with it
// 2143 MB 0.42 ms, 5.1 TB/s; a copy does 6.5).  What is left: rows that do not fit the rings come through
// L2 twice (5 % of it), the CTAs of a cluster wait for one another once a row, and the plan and the sums.
// Leaving the exponentials out changes nothing.  The second pass of a scaled loss takes 0.46 ms.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdio>
#include <exception>
#include <string>

#include "../../include/crukx_b200.h"
#include "common.cuh"
#include "elements.cuh"
#include "launch.cuh"

namespace crx {
namespace {

namespace cg = cooperative_groups;

// Sixteen warps per SM in CTAs of four, whose reductions pass under one another's streams: 4096 x 152k
// rows with their gradient take 0.42 ms, by CTAs of two warps 0.43, of sixteen 0.44; with 24 or 32 warps
// per SM and shorter rings 0.50 and 0.54.  Rings fill what shared memory there is.
constexpr int kRowThreads = 128;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kRowCtas = 4;            // per SM
constexpr int kSlots = 6;              // of a warp's ring
constexpr int kChunk = 128;            // 16-byte vectors of a slot: four per lane
constexpr int kRowGrid = 148 * kRowCtas;       // CTAs of the persistent grid
constexpr int kMaxUnits = kRowGrid * kRowWarps;
constexpr size_t kRingBytes = size_t(kRowWarps) * kSlots * kChunk * 16;
// Exponents are z c - R by one fma, exact but for its rounding, so at the maximum they are what R = M c lost
// in its own rounding: at most 2^5 for |M c| below this bound, which a sum in fp32 bears (it cancels in p and in
// logp) and beyond which 2^x soon overflows.  Larger maxima make a far row; what lies below -kFar adds nothing
// to any other.
constexpr float kFar = 0x1p30f;
constexpr int kMaxDevices = 64;

// 2^x to about 2 ulp; results below 2^-126 become 0: next to the maximum's term, 2^-32 or more, 2^-94 at most.
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

// Layout of args.rows: the plan's 1 / denominator and number of rows that count, a float4 per row,
// the sums of the three terms over each unit's rows (double), the plan's order of the rows.  A row's
// float4 is (u, R, s, 0), or (u, M, s, 1) for a far row (below).
struct Plan {
    double inv_denom;
    int64_t counted;
};
__host__ __device__ __forceinline__ Plan* plan_of(const crx_policy_args& a) { return reinterpret_cast<Plan*>(a.rows); }
__device__ __forceinline__ float4* saved_of(const crx_policy_args& a) { return reinterpret_cast<float4*>(a.rows) + 1; }
__device__ __forceinline__ double* partials_of(const crx_policy_args& a) {
    return reinterpret_cast<double*>(a.rows + 4 + 4 * a.batch * a.steps);
}
__device__ __forceinline__ int32_t* order_of(const crx_policy_args& a) { return reinterpret_cast<int32_t*>(partials_of(a) + 3 * kMaxUnits); }

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

// The running (maximum, sum of 2^(z c - R)) of one thread, R = max(M c, -kFar).  The bound lets what
// lies below it add 0 (-inf, the type's lowest value, any large negative number that rules tokens out),
// also where nothing else has come yet.
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
};

// 2^(x c + d) of both values.
__device__ __forceinline__ f32x2 exp2_pair(f32x2 x, f32x2 c, f32x2 d) {
    float a, b;
    unpack2(fma2(x, c, d), a, b);
    return pack2(exp2_fast(a), exp2_fast(b));
}

template <class T, int U>
__device__ __forceinline__ void add_vecs(const uint4* q, Running& run, float c) {
    run.raise(vec_max<T>(q, U), c);
    const f32x2 cc = pack2(c, c), d = pack2(-run.r, -run.r);
    f32x2 sum[2] = {0, 0};
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float x[Vec<T>::N];
        Vec<T>::get(q[u], x);
#pragma unroll
        for (int i = 0; i < Vec<T>::N; i += 2) sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], exp2_pair(pack2(x[i], x[i + 1]), cc, d));
    }
    float a, b;
    unpack2(add2(sum[0], sum[1]), a, b);
    run.s += a + b;
}

// A CTA's (or warp's) slice of a row: 16-byte vectors [lo, hi) of the part after the row's first
// 16-byte boundary; the first CTA also has the elements before it and the row's last ones.
struct Slice {
    int head, tail;   // elements before the boundary, and after the last whole vector (first CTA)
    int body;         // element of the first whole vector
    int tail_at;      // element where the tail begins
    int lo, hi;
};
template <class T>
__device__ __forceinline__ Slice slice_of(const T* z, int64_t V, int rank, int C) {
    Slice s;
    const int head = int(tmin<int64_t>(head_of<T>(z), V));
    const int nv = int((V - head) / Vec<T>::N);
    s.lo = int(int64_t(nv) * rank / C);
    s.hi = int(int64_t(nv) * (rank + 1) / C);
    s.head = rank ? 0 : head;
    s.body = head;
    s.tail_at = head + nv * Vec<T>::N;
    s.tail = rank ? 0 : int(V - s.tail_at);
    return s;
}

struct Shared {
    float2 warp[2][kRowWarps];     // (M, s) of every warp, double-buffered over rows
    float2 part[2][kMaxCluster];   // and of every CTA of the cluster
    uint64_t came[2];              // barriers: the cluster's parts are here
};

__device__ __forceinline__ uint32_t smem_of(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }

// CLUSTER: what the phase counted was written by other CTAs of the cluster.
template <bool CLUSTER>
__device__ __forceinline__ bool phase_done(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    if (CLUSTER)
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    else
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok;
}
// Whether the phase `parity` of the barrier completed; gives up after some seconds, which only a
// copy that never ends could bring about.
template <bool CLUSTER>
__device__ __noinline__ bool wait_longer(uint32_t bar, uint32_t parity) {
    for (int i = 0; i < (1 << 20); ++i)
        if (phase_done<CLUSTER>(bar, parity)) return true;
    return false;
}
template <bool CLUSTER = false>
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t parity) { return phase_done<CLUSTER>(bar, parity) || wait_longer<CLUSTER>(bar, parity); }

// The largest of a warp's values: as integers of the same order, one instruction for the warp.
__device__ __forceinline__ float warp_max(float x) {
    const int i = __float_as_int(x);
    const int k = __reduce_max_sync(0xffffffffu, i ^ ((i >> 31) & 0x7fffffff));
    return __int_as_float(k ^ ((k >> 31) & 0x7fffffff));
}

// (M, s) over the lanes of a warp: the maximum first, then one rescaling per lane and a sum.
__device__ __forceinline__ Running warp_total(Running run, float c) {
    const float m = warp_max(run.m);
    Running all;
    all.m = m;
    all.r = fmaxf(m * c, -kFar);
    float s = run.s * exp2_fast(fmaxf(run.m * c, -kFar) - all.r);
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    all.s = s;
    return all;
}
__device__ __forceinline__ Running lane_entry(const float2* e, int n) {
    const int lane = threadIdx.x & 31;
    Running r;
    if (lane < n) {
        const float2 v = e[lane];
        r.m = v.x;
        r.s = v.y;
    }
    return r;
}

// (M, s) of the whole row number `i` of the unit from every thread's; the same bits in every thread.
// The CTAs of a cluster send their parts into each other's shared memory, counted in by a barrier
// there: a cluster barrier would also wait for the stores of the row before.  A CTA cannot be two
// rows ahead of another, whose part of the row between it needs, so two buffers are enough.
template <bool WARP>
__device__ __forceinline__ Running row_total(Running run, Shared& sh, uint32_t i, int rank, int C, float c) {
    run = warp_total(run, c);
    if (WARP) return run;
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, half = i & 1;
    if (lane == 0) sh.warp[half][w] = make_float2(run.m, run.s);
    __syncthreads();
    if (C == 1) return warp_total(lane_entry(sh.warp[half], kRowWarps), c);
    const uint32_t came = smem_of(&sh.came[half]);
    if (w == 0) {
        run = warp_total(lane_entry(sh.warp[half], kRowWarps), c);
        if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(came), "r"(C * 8) : "memory");
        if (lane < C) {
            uint32_t to, bar;
            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_of(&sh.part[half][rank])), "r"(lane));
            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar) : "r"(came), "r"(lane));
            asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(to), "f"(run.m), "f"(run.s),
                         "r"(bar)
                         : "memory");
        }
    }
    const bool here = wait_phase<true>(came, (i >> 1) & 1);
    run = warp_total(lane_entry(sh.part[half], C), c);
    if (!here) run.s = NAN;
    return run;
}

template <bool WARP>
__device__ __forceinline__ float unit_total(float v, Shared& sh) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (WARP) return v;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.warp[0][threadIdx.x >> 5].y = v;
    __syncthreads();
    v = 0.f;
    for (int k = 0; k < kRowWarps; ++k) v += sh.warp[0][k].y;
    __syncthreads();
    return v;
}

// The sum of a far row: one whose largest logit M has |M c| >= kFar (every logit a large negative number, or
// a temperature of 1e-8).  (z - M) c, which is 0 at the maximum, takes the place of z c - R, and each CTA of
// the cluster goes over the whole row.
template <class T, bool WARP>
__device__ __noinline__ float far_sum(const T* z, int64_t V, float M, float c, Shared& sh) {
    float s = 0.f;
    for (int64_t j = WARP ? threadIdx.x & 31 : threadIdx.x; j < V; j += WARP ? 32 : kRowThreads) s += exp2_fast((to_f(z[j]) - M) * c);
    return unit_total<WARP>(s, sh);
}

// What turns a row's logits into its gradient, u 1[j = a] - k 2^(z_j c - R) with k = u / s.  u = 0 (a
// clipped token without a KL term, a token that does not count) gives zeros whatever the logits.
template <class T>
struct GradOf {
    static constexpr int N = Vec<T>::N;
    const T* z;
    T* g;
    int64_t token;
    float u, k, R, c;
    bool far, wide;   // wide: gradient rows start at the same place between 16-byte boundaries as the logits'
    int token_vec;

    __device__ __forceinline__ GradOf(const T* z, T* g, const Slice& sl, int64_t V, int64_t token_, float u, float R, float s, float c, bool far)
        : z(z), g(g), token(token_ >= 0 && token_ < V ? token_ : -1), u(u), k(u == 0.f ? 0.f : u / s), R(R), c(c), far(far) {
        wide = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(g)) & 15) == 0;
        token_vec = token >= sl.body ? int((token - sl.body) / N) : -1;
    }
    __device__ __forceinline__ void one(int64_t j, float f) const {
        float x = 0.f;
        if (u != 0.f) {
            x = -k * exp2_fast(far ? (f - R) * c : fmaf(f, c, -R));
            if (j == token) x += u;
        }
        g[j] = from_f<T>(x);
    }
    __device__ __forceinline__ void one(int64_t j) const { one(j, u == 0.f ? 0.f : to_f(z[j])); }
    // vector i of the body, its logits in q
    __device__ __forceinline__ void vec(int body, int i, const uint4& q) const {
        float x[N];
        if (u == 0.f) {
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = 0.f;
        } else {
            Vec<T>::get(q, x);
            if (far || !wide) {
#pragma unroll
                for (int e = 0; e < N; ++e) one(body + int64_t(i) * N + e, x[e]);
                return;
            }
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = -k * exp2_fast(fmaf(x[e], c, -R));
            if (i == token_vec) {
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (body + int64_t(i) * N + e == token) x[e] += u;
            }
        }
        T* o = g + body + int64_t(i) * N;
        if (wide) *reinterpret_cast<uint4*>(o) = Vec<T>::put(x);
        else
            for (int e = 0; e < N; ++e) o[e] = from_f<T>(x[e]);
    }
    __device__ __forceinline__ bool plain() const { return wide && !far && u != 0.f; }
    // the same where plain(), without the token: its lane puts that right afterwards
    __device__ __forceinline__ void vec_plain(uint4* o, const uint4& q) const {
        const f32x2 cc = pack2(c, c), d = pack2(-R, -R), kk = pack2(-k, -k);
        float x[N];
        Vec<T>::get(q, x);
#pragma unroll
        for (int e = 0; e < N; e += 2) unpack2(mul2(exp2_pair(pack2(x[e], x[e + 1]), cc, d), kk), x[e], x[e + 1]);
        *o = Vec<T>::put(x);
    }
    // a slice from global memory, by `threads` threads of which this is number `tid`
    __device__ __forceinline__ void slice(const Slice& sl, int tid, int threads) const {
        ends(sl, tid);
        const uint4* zv = reinterpret_cast<const uint4*>(z + sl.body);
        for (int i = sl.lo + tid; i < sl.hi; i += threads) vec(sl.body, i, u == 0.f ? make_uint4(0, 0, 0, 0) : zv[i]);
    }
    __device__ __forceinline__ void ends(const Slice& sl, int tid) const {
        if (tid < sl.head) one(tid);
        if (tid < sl.tail) one(sl.tail_at + tid);
    }
};

// What a row needs besides its logits.
struct RowIn {
    uint32_t row;
    int64_t at, grad_at, token;
    float w, advantage, old, ref;
};
__device__ __forceinline__ RowIn row_in(const crx_policy_args& a, uint32_t row) {
    const uint32_t b = row / uint32_t(a.steps), t = row - b * uint32_t(a.steps);
    RowIn r;
    r.row = row;
    r.at = at(a.logits, b, t);
    r.grad_at = at(a.grad, b, t);
    r.token = a.tokens64 ? static_cast<const int64_t*>(a.tokens.p)[at(a.tokens, b, t)]
                         : static_cast<const int32_t*>(a.tokens.p)[at(a.tokens, b, t)];
    r.w = weight(a, b, t);
    r.advantage = value(a.advantages, b, t);
    r.old = a.old_logp.p ? value(a.old_logp, b, t) : 0.f;
    r.ref = a.ref_logp.p ? value(a.ref_logp, b, t) : 0.f;
    return r;
}

__device__ __forceinline__ double warp_sum(double v) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The row at place i of the plan's order (of `n` places).
__device__ __forceinline__ uint32_t row_at(const int32_t* order, uint32_t i, uint32_t n) { return !order ? i : i < n ? uint32_t(order[i]) : 0; }

// A place in a warp's ring, and the phase of its barrier that says that the chunk is here.
struct Place {
    uint32_t slot = 0, phase = 0;
    __device__ __forceinline__ void next() {
        if (++slot == kSlots) {
            slot = 0;
            phase ^= 1;
        }
    }
};

// A warp's stream: the chunks of its part of every row that counts, in the plan's order (a row that
// does not fit the ring comes twice, for the gradient).
template <class T, bool GRAD, bool WARP>
struct Stream {
    const crx_policy_args& a;
    uint32_t ring, bars;       // shared addresses: kSlots chunks, kSlots barriers
    uint32_t i, step, n;       // place of the row being issued among those that count, the unit's stride, their number
    uint32_t row_after;        // the row at the place after that, loaded ahead
    const int32_t* order;
    int rank, C;
    const char* from;          // its next vector
    int left, span, again;     // vectors still to come, of how many, and whether all of them once more
    uint32_t to = 0;           // the slot that is filled next
    Place at_;                 // the first chunk that is not done with

    static constexpr int kStride = WARP ? kChunk : kChunk * kRowWarps;

    __device__ __forceinline__ Stream(const crx_policy_args& a, char* mem, uint64_t* bars_, uint32_t i, uint32_t step, uint32_t n,
                                      const int32_t* order, int rank, int C)
        : a(a), i(i), step(step), n(n), row_after(row_at(order, i, n)), order(order), rank(rank), C(C) {
        const int warp = threadIdx.x >> 5;
        ring = smem_of(mem) + uint32_t(warp) * (kSlots * kChunk * 16);
        bars = smem_of(bars_ + warp * kSlots);
        open();
        for (int k = 0; k < kSlots; ++k) issue();
    }
    // the warp's vectors of a slice, as its first one and its chunks
    static __device__ __forceinline__ int first(const Slice& sl) { return sl.lo + (WARP ? 0 : int(threadIdx.x >> 5) * kChunk); }
    static __device__ __forceinline__ int chunks(const Slice& sl) {
        const int left = sl.hi - first(sl);
        return left > 0 ? (left + kStride - 1) / kStride : 0;
    }
    // goes on to the next row that has a part for this warp
    __device__ __forceinline__ void open() {
        for (; i < n; i += step) {
            const uint32_t row = row_after, b = row / uint32_t(a.steps), t = row - b * uint32_t(a.steps);
            row_after = row_at(order, i + step, n);
            const T* z = static_cast<const T*>(a.logits.p) + at(a.logits, b, t);
            const Slice sl = slice_of<T>(z, a.vocab, rank, C);
            span = left = sl.hi - first(sl);
            if (left <= 0) continue;
            from = reinterpret_cast<const char*>(z + sl.body) + int64_t(first(sl)) * 16;
            again = GRAD && left > kSlots * kStride;
            return;
        }
    }
    // the next chunk into the slot that has come free
    __device__ __forceinline__ void issue() {
        if (i >= n) return;
        if ((threadIdx.x & 31) == 0) {
            const uint32_t bytes = uint32_t(tmin(kChunk, left)) * 16, bar = bars + to * 8;
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                             ring + to * (kChunk * 16)),
                         "l"(from), "r"(bytes), "r"(bar)
                         : "memory");
        }
        to = to + 1 == kSlots ? 0 : to + 1;
        left -= kStride;
        from += kStride * 16;
        if (left > 0) return;
        if (again) {
            again = 0;
            from -= int64_t(span - left) * 16;
            left = span;
        } else {
            i += step;
            open();
        }
    }
    // the lane's vectors of a chunk
    __device__ __forceinline__ void read(const Place& p, uint4* q) const {
        const uint32_t s = ring + p.slot * (kChunk * 16) + (threadIdx.x & 31) * 16;
#pragma unroll
        for (int v = 0; v < 4; ++v)
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(q[v].x), "=r"(q[v].y), "=r"(q[v].z), "=r"(q[v].w) : "r"(s + v * 512) : "memory");
    }
    __device__ __forceinline__ bool wait(const Place& p) const { return wait_phase(bars + p.slot * 8, p.phase); }
    __device__ __forceinline__ void release() {
        __syncwarp();   // every lane has its values
        at_.next();
        issue();
    }
};

template <class T, bool GRAD, bool WARP>
__global__ void __launch_bounds__(kRowThreads, kRowCtas) k_policy_rows(const __grid_constant__ crx_policy_args a, double inv_denom, int planned, int C) {
    extern __shared__ __align__(128) char ring[];
    __shared__ uint64_t bars[kRowWarps * kSlots];
    __shared__ Shared sh;
    const int tid = WARP ? threadIdx.x & 31 : threadIdx.x, lane = threadIdx.x & 31, threads = WARP ? 32 : kRowThreads;
    const int rank = WARP ? 0 : int(blockIdx.x) % C;
    const int64_t V = a.vocab;
    const uint32_t n = uint32_t(a.batch * a.steps);
    const uint32_t unit = WARP ? blockIdx.x * kRowWarps + (threadIdx.x >> 5) : blockIdx.x / C;
    const uint32_t units = WARP ? gridDim.x * kRowWarps : gridDim.x / C;
    if (threadIdx.x < kRowWarps * kSlots + 2)
        asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_of(threadIdx.x < kRowWarps * kSlots ? &bars[threadIdx.x] : &sh.came[threadIdx.x - kRowWarps * kSlots]))
                     : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;\nfence.proxy.async.shared::cta;" ::: "memory");
    if (!WARP && C > 1) cg::this_cluster().sync();   // every CTA runs before another writes to its shared memory
    else __syncthreads();
    after_previous();
    const float c = float(1.4426950408889634 / double(a.temperature));
    const double inv_d = inv_denom < 0 ? plan_of(a)->inv_denom : inv_denom;   // weights may sum to what fp32 has no reciprocal of
    const float inv_tau = 1.f / a.temperature;
    const int32_t* order = planned ? order_of(a) : nullptr;
    const uint32_t counted = planned ? uint32_t(plan_of(a)->counted) : n;
    double loss = 0, kl = 0, cut = 0;
    uint32_t nth = 0;   // of the unit's rows that count
    Stream<T, GRAD, WARP> in(a, ring, bars, unit, units, counted, order, rank, C);
    RowIn next;
    if (unit < n) next = row_in(a, row_at(order, unit, n));
    uint32_t row_after = row_at(order, unit + units, n);
    for (uint32_t i = unit; i < n; i += units) {
        const RowIn r = next;
        const float w = r.w;
        const uint32_t row = r.row;
        const T* z = static_cast<const T*>(a.logits.p) + r.at;
        T* g = GRAD ? static_cast<T*>(const_cast<void*>(a.grad.p)) + r.grad_at : nullptr;
        const Slice sl = slice_of<T>(z, V, rank, C);
        const float za = i < counted && r.token >= 0 && r.token < V ? to_f(z[r.token]) : NAN;
        if (i + units < n) {   // what the next row needs, and the number of the one after it: they arrive under this row
            next = row_in(a, row_after);
            row_after = row_at(order, i + 2 * units, n);
        }
        if (i >= counted) {
            if (GRAD) GradOf<T>(z, g, sl, V, -1, 0.f, 0.f, 1.f, c, false).slice(sl, tid, threads);
            if (rank == 0 && tid == 0) {
                a.logp[row] = 0.f;
                saved_of(a)[row] = make_float4(0.f, 0.f, 1.f, 0.f);
            }
            continue;
        }

        Running run;
        const auto one = [&](int j) {
            const float x = to_f(z[j]);
            run.raise(x, c);
            run.s += exp2_fast(fmaf(x, c, -run.r));
        };
        if (tid < sl.head) one(tid);
        if (tid < sl.tail) one(sl.tail_at + tid);
        const int first = in.first(sl), chunks = in.chunks(sl);
        const bool fits = chunks <= kSlots;
        bool came = true;
        Place p = in.at_;
        for (int k = 0, left = sl.hi - first; k < chunks; ++k, left -= in.kStride) {
            uint4 q[4];
            came &= in.wait(p);
            in.read(p, q);
            p.next();
            if (left < kChunk) {   // what lies behind the slice adds nothing
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    if (lane + 32 * v >= left) q[v] = Vec<T>::lowest();
            }
            add_vecs<T, 4>(q, run, c);
            if (!GRAD || !fits) in.release();
        }
        if (!came) run.s = NAN;
        run = row_total<WARP>(run, sh, nth++, rank, C, c);
        const bool far = fabsf(run.m) <= 3.402823466e38f && !(fabsf(run.m * c) < kFar);
        const float s = far ? far_sum<T, WARP>(z, V, run.m, c, sh) : run.s;
        const float R = far ? run.m : run.r;
        // the token's term from the logits themselves (halved: their difference may not fit), not through c's
        // rounding; s without what the maximum's exponent is off 0
        const float at_top = far ? s : s * exp2_fast(-fmaf(run.m, c, -R));
        const float logp = (0.5f * za - 0.5f * run.m) / (0.5f * a.temperature) - logf(at_top);

        const float A = r.advantage;
        const float ratio = a.old_logp.p ? expf(logp - r.old) : (logp == logp ? 1.f : logp);   // NaN logits show in the loss
        const bool clipped = (A > 0.f && ratio > 1.f + a.clip_high) || (A < 0.f && ratio < 1.f - a.clip_low);
        // an advantage of 0 takes any ratio, infinite ones too, but what is not a number stays one
        const float gain = A == 0.f && ratio == ratio ? 0.f : (clipped ? (A > 0.f ? 1.f + a.clip_high : 1.f - a.clip_low) : ratio) * A;
        float dl = clipped ? 0.f : -gain, k = 0.f;
        if (a.ref_logp.p) {
            const float x = r.ref - logp, e = expm1f(x);
            k = e - x;
            if (a.kl_coef != 0.f) dl -= a.kl_coef * e;   // (a k that is only reported may overflow)
        }
        const float u = float(double(w) * inv_d) * dl * inv_tau;
        if (rank == 0 && tid == 0) {
            a.logp[row] = logp;
            saved_of(a)[row] = make_float4(u, R, s, far ? 1.f : 0.f);
            loss += double(w) * double((a.kl_coef != 0.f ? a.kl_coef * k : 0.f) - gain);
            kl += double(w) * double(k);
            cut += double(clipped ? w : 0.f);
        }
        if (GRAD) {
            const GradOf<T> grad(z, g, sl, V, r.token, u, R, s, c, far);
            grad.ends(sl, tid);
            const bool plain = grad.plain();
            uint4* o = reinterpret_cast<uint4*>(g + sl.body) + first + lane;
            for (int k = 0, left = sl.hi - first; k < chunks; ++k, left -= in.kStride, o += in.kStride) {
                uint4 q[4];
                const bool here = fits || in.wait(in.at_);
                in.read(in.at_, q);
                if (!here) {   // NaN in every type
#pragma unroll
                    for (int v = 0; v < 4; ++v) q[v] = make_uint4(~0u, ~0u, ~0u, ~0u);
                }
                const int v0 = sl.hi - left + lane;
                if (plain && left >= kChunk) {
#pragma unroll
                    for (int v = 0; v < 4; ++v) grad.vec_plain(o + 32 * v, q[v]);
                    if (unsigned(grad.token_vec - v0) < 128u && ((grad.token_vec - v0) & 31) == 0) grad.one(grad.token, za);
                } else {
#pragma unroll
                    for (int v = 0; v < 4; ++v)
                        if (lane + 32 * v < left) grad.vec(sl.body, v0 + 32 * v, q[v]);
                }
                in.release();
            }
        }
    }
    let_next_start();
    if (rank == 0 && tid == 0) {
        double* p = partials_of(a) + 3 * unit;
        p[0] = loss;
        p[1] = kl;
        p[2] = cut;
    }
}

// Every warp takes a run of rows, 32 * kAtOnce at a time; the counts before it give it its places among
// the rows that count and among those that do not.
__global__ void __launch_bounds__(1024) k_policy_plan(const __grid_constant__ crx_policy_args a) {
    __shared__ double red[32];
    __shared__ uint32_t before[32];
    constexpr uint32_t kAtOnce = 8;
    const uint32_t n = uint32_t(a.batch * a.steps), steps = uint32_t(a.steps), lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const uint32_t per = (n / 32 + 32) / 32 * 32, lo = tmin(n, w * per), hi = tmin(n, lo + per);
    let_next_start();
    const auto load = [&](uint32_t i, float* x) {   // weights i + lane, i + lane + 32, ...; 0 behind the run
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; ++k) {
            const uint32_t row = i + 32 * k + lane;
            x[k] = row < hi ? weight(a, row / steps, row % steps) : 0.f;
        }
    };
    double v = 0;
    uint32_t c = 0;
    float x[kAtOnce];
    for (uint32_t i = lo; i < hi; i += 32 * kAtOnce) {
        load(i, x);
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; ++k) {
            v += double(x[k]);
            c += __popc(__ballot_sync(0xffffffffu, x[k] != 0.f));
        }
    }
    v = warp_sum(v);
    if (lane == 0) {
        red[w] = v;
        before[w] = c;
    }
    __syncthreads();
    const uint32_t mine = before[lane];
    uint32_t scan = mine;
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= uint32_t(o)) scan += y;
    }
    const uint32_t total = __shfl_sync(0xffffffffu, scan, 31);
    uint32_t in = __shfl_sync(0xffffffffu, scan - mine, w);   // rows that count before this warp's
    int32_t* order = order_of(a);
    for (uint32_t i = lo; i < hi; i += 32 * kAtOnce) {
        load(i, x);
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; ++k) {
            const uint32_t row = i + 32 * k + lane, yes = __ballot_sync(0xffffffffu, x[k] != 0.f);
            const uint32_t at_in = in + __popc(yes & lanemask_lt());
            if (row < hi) order[x[k] != 0.f ? at_in : total + row - at_in] = int32_t(row);   // (row - at_in do not count before it)
            in += __popc(yes);
        }
    }
    if (w == 0) {
        v = warp_sum(red[lane]);
        if (lane == 0) {
            plan_of(a)->inv_denom = v == 0.0 ? 0.0 : 1.0 / v;
            plan_of(a)->counted = total;
        }
    }
}

__global__ void __launch_bounds__(768) k_policy_sums(const __grid_constant__ crx_policy_args a, double inv_denom, int units) {
    __shared__ double red[24];
    const int w = threadIdx.x >> 5, i = w >> 3, lane = threadIdx.x & 31;   // eight warps per term
    double v = 0;
    after_previous();
    for (int k = threadIdx.x & 255; k < units; k += 256) v += partials_of(a)[3 * k + i];
    v = warp_sum(v);
    if (lane == 0) red[w] = v;
    __syncthreads();
    if (threadIdx.x < 3) {
        v = 0;
        for (int k = 0; k < 8; ++k) v += red[8 * threadIdx.x + k];
        v *= inv_denom < 0 ? plan_of(a)->inv_denom : inv_denom;
        *(threadIdx.x ? a.stats + threadIdx.x - 1 : a.loss) = float(v);
    }
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
        const Slice sl = slice_of<T>(z, a.vocab, int(item - row * C), C);
        GradOf<T>(z, g, sl, a.vocab, token, u, saved.y, saved.z, c, saved.w != 0.f).slice(sl, threadIdx.x, kRowThreads);
    }
}

// ------------------------------------------------------------------ host

int fail(char* err, size_t errlen, int status, const std::string& msg) {
    if (err && errlen) std::snprintf(err, errlen, "%s", msg.c_str());
    return status;
}

// A row that does not fit the rings is read a second time for its gradient, out of L2 as long as the
// rows that are being worked on at once are no more than this (of 126 MB; the gradients pass through
// it too).  4096 x 152k bf16 rows, 28% of them masked: 0.42 ms with 48 MB, 0.47 with 24 (more CTAs per
// row wait for one another), 0.52 with 96; 2048 x 152k fp32: 0.38, 0.38, 0.46.
constexpr int64_t kRowsAtOnce = int64_t(48) << 20;

// A row by one warp, where nothing waits for another warp: rows short enough, and as many of them as
// there are CTAs (2500 x 8192: 17 us against 21 by CTAs, 600 x 1024: 8 against 10); fewer rows are
// shared out (200 x 8192: 9 us against 13 by warps).
bool warp_rows(int64_t n, int64_t V, int vec) { return n >= kRowGrid && V / vec * 16 * kMaxUnits <= kRowsAtOnce; }

// CTAs per row: enough to keep the rows at once in L2 (with a gradient), and as many as the rows leave
// room for while a slice keeps a chunk per warp (64 x 152k: 15 us, with one CTA per row 37).
int cluster_for(int64_t n, int64_t V, int vec, bool grad) {
    const int64_t bytes = V / vec * 16;
    int C = 1;
    while (C < kMaxCluster && ((grad && std::min<int64_t>(n, kRowGrid / C) * bytes > kRowsAtOnce) ||
                               (n * C * 2 <= kRowGrid && bytes >= int64_t(kChunk) * 16 * 4 * C)))
        C *= 2;
    return C;
}

template <class T, bool GRAD, bool WARP>
cudaError_t launch_as(const crx_policy_args& a, double inv_denom, int C, int64_t most, int* units, cudaStream_t st) {
    const auto kernel = k_policy_rows<T, GRAD, WARP>;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kRowThreads);
    cfg.gridDim = dim3(kRowGrid / C * C);
    cfg.dynamicSmemBytes = kRingBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(C);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    // clusters that run at once: those of four and eight do not fill every GPC, and rows dealt to more
    // would wait for a second round
    static std::atomic<int> fit[kMaxDevices][4];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= kMaxDevices) return cudaErrorInvalidDevice;
    std::atomic<int>& known = fit[dev][C == 1 ? 0 : C == 2 ? 1 : C == 4 ? 2 : 3];
    int clusters = known.load(std::memory_order_relaxed);
    if (!clusters) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kRingBytes));
        if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg);
        if (e != cudaSuccess) return e;
        clusters = std::max(1, std::min(clusters, kRowGrid / C));
        known.store(clusters, std::memory_order_relaxed);
    }
    const int grid = int(std::min<int64_t>(most, clusters));
    *units = WARP ? grid * kRowWarps : grid;
    cfg.gridDim = dim3(unsigned(grid * C));
    if (a.mask.p) {   // directly behind the plan
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 2;
    }
    return cudaLaunchKernelEx(&cfg, kernel, a, inv_denom, int(a.mask.p != nullptr), C);
}

template <class T, bool GRAD>
cudaError_t launch_rows(const crx_policy_args& a, double inv_denom, int* units, cudaStream_t st) {
    const int64_t n = a.batch * a.steps;
    if (warp_rows(n, a.vocab, Vec<T>::N)) return launch_as<T, GRAD, true>(a, inv_denom, 1, (n + kRowWarps - 1) / kRowWarps, units, st);
    return launch_as<T, GRAD, false>(a, inv_denom, cluster_for(n, a.vocab, Vec<T>::N, GRAD), n, units, st);
}

template <class T>
cudaError_t launch_again(const crx_policy_args& a, const float* scale, int unless_one, cudaStream_t st) {
    const int64_t n = a.batch * a.steps;
    const int C = cluster_for(n, a.vocab, Vec<T>::N, true);
    k_policy_again<T><<<unsigned(std::min<int64_t>(n * C, kRowGrid * 2)), kRowThreads, 0, st>>>(a, scale, unless_one, C);
    return cudaGetLastError();
}

int check(const char* who, const crx_policy_args* a, char* err, size_t errlen) {
    const auto bad = [&](const char* what) { return fail(err, errlen, CRX_BAD_ARGUMENT, std::string(who) + ": " + what); };
    if (!a) return bad("null arguments");
    if (a->batch < 0 || a->steps < 0 || a->vocab < 1 || a->vocab > (int64_t(1) << 30) || a->batch > (int64_t(1) << 31) || a->steps > (int64_t(1) << 31) ||
        (a->batch && a->steps >= (int64_t(1) << 31) / a->batch))
        return bad("size out of range");
    if (a->dtype != CRX_BF16 && a->dtype != CRX_FP16 && a->dtype != CRX_FP32) return bad("unknown type");
    const uintptr_t es = a->dtype == CRX_FP32 ? 4 : 2;
    if (!a->loss || !a->stats || !a->rows || reinterpret_cast<uintptr_t>(a->rows) % 16) return bad("null or misaligned result or workspace");
    if (a->batch && a->steps) {
        if (!a->logits.p || !a->tokens.p || !a->advantages.p || !a->logp) return bad("null pointer");
        if (reinterpret_cast<uintptr_t>(a->logits.p) % es || reinterpret_cast<uintptr_t>(a->grad.p) % es) return bad("misaligned logits or gradient");
    }
    if (!(a->temperature >= 1e-30f) || !(a->clip_low >= 0.f) || !(a->clip_high >= 0.f) || !(a->denom >= 0) || !std::isfinite(a->temperature))
        return fail(err, errlen, CRX_VALUE_ERROR, "temperature must be at least 1e-30 and finite, clip bounds and denom not negative");
    return CRX_OK;
}

}  // namespace
}  // namespace crx

using namespace crx;

extern "C" {

int64_t crx_policy_workspace(int64_t batch, int64_t steps) {
    if (batch < 0 || steps < 0) return 0;
    return 16 + 20 * batch * steps + int64_t(sizeof(double)) * 3 * kMaxUnits;
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
        // a negative 1 / denominator: the kernels take the plan's
        const double inv_denom = a.denom > 0 ? 1.0 / a.denom : a.mask.p ? -1.0 : 1.0 / double(n);
        if (a.mask.p) {
            k_policy_plan<<<1, 1024, 0, st>>>(a);
            e = cudaGetLastError();
        }
        int units = 0;
        const bool grad = a.grad.p != nullptr;
        if (e == cudaSuccess) {
            if (a.dtype == CRX_BF16) e = grad ? launch_rows<__nv_bfloat16, true>(a, inv_denom, &units, st) : launch_rows<__nv_bfloat16, false>(a, inv_denom, &units, st);
            else if (a.dtype == CRX_FP16) e = grad ? launch_rows<__half, true>(a, inv_denom, &units, st) : launch_rows<__half, false>(a, inv_denom, &units, st);
            else e = grad ? launch_rows<float, true>(a, inv_denom, &units, st) : launch_rows<float, false>(a, inv_denom, &units, st);
        }
        if (e == cudaSuccess) e = launch_behind(k_policy_sums, 1, 768, st, a, inv_denom, units);
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
