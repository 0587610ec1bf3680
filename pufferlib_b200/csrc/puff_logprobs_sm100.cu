// Log-probability and entropy of chosen actions (tokens) from logits, and their gradient (sm_100a).
//
//   z = logits / temperature,  m = max z,  s = sum e^(z - m)
//   logprob = z[action] - m - log s,     entropy = log s - (1 / s) sum (z - m) e^(z - m)
//   dlogits = (dlogprob (onehot - p) - dentropy p (log p + entropy)) / temperature,   p = e^(z - m - log s)
//
// The step between the policy's logits and the ratio of pufferl.py:390-394 (the log-probability and entropy of
// pufferlib/pytorch.py sample_logits), for action heads of a few entries up to vocabularies of 10^5 and more.
//
// Memory-bound in principle, 2 to 4 bytes a logit read once forward, read and written once backward; in practice the
// exponentials and the instructions around them are close behind: five or so a 16-bit logit fit under the copy rate.  That
// is why every exponential is one ex2.approx, good to 4 half steps of fp32 where expf is good to 2: 524288 x 18 fp32 is
// 9.7e-8 off 64 bits (relative, all outputs together), fp32 arithmetic with expf 6.3e-8.
// On a B200 that copies at 6.55 TB/s: 4096 x 131072 bf16 195 us forward with entropy (5.5 TB/s), 176 without, 328
// backward (6.55); 524288 x 18 fp32 20 and 29 us; 8 x 131072 bf16 about 5 us, a cluster of eight CTAs a row.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/puff_advantage.h"
#include "puff_policy.cuh"

namespace puff {

__device__ int g_bad_action = 0;

constexpr int kLpMaxCluster = 8;

// 16 bytes from global to shared memory without a register in between
__device__ __forceinline__ void copy16_async(uint4* shared, const uint4* global)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(shared))),
                 "l"(global) : "memory");
}
__device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// bytes [shift, shift + 16) of the 32 in a, b; shift is even
__device__ __forceinline__ uint4 cut_vector(uint4 a, uint4 b, unsigned shift)
{
    uint32_t w[7] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z};
    const uint32_t last = b.w;
    if (shift & 8u) {
        w[0] = w[2], w[1] = w[3], w[2] = w[4], w[3] = w[5], w[4] = w[6], w[5] = last;
    }
    if (shift & 4u) {
        w[0] = w[1], w[1] = w[2], w[2] = w[3], w[3] = w[4], w[4] = w[5];
    }
    const unsigned bits = (shift & 2u) * 8u;
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits),
                      __funnelshift_r(w[3], w[4], bits));
}

// where row r of a tensor with rows [outer, inner] starts, in elements
struct RowMap {
    long long inner, outer_stride, inner_stride;
    bool one_run;      // a single run of rows: nothing to divide
    __device__ __forceinline__ long long at(long long r) const
    {
        if (one_run) return r * inner_stride;
        const long long o = ((r | inner) >> 32) == 0 ? static_cast<unsigned>(r) / static_cast<unsigned>(inner) : r / inner;
        return o * outer_stride + (r - o * inner) * inner_stride;
    }
};

// -inf (an illegal action) would make 0 x inf of the entropy's terms: it is raised to a value whose exponential is 0
// all the same, two packed elements at once, as long as the row's maximum is far enough above it.
template <typename T> __device__ __forceinline__ float raised_inf() { return sizeof(T) == 2 ? -60000.0f : -1e30f; }
template <> __device__ __forceinline__ float raised_inf<__nv_bfloat16>() { return -9.969209968386869e29f; }   // a bf16 value
__device__ __forceinline__ uint32_t raise2(uint32_t w, __half)
{
    const __half2 p = __hmax2_nan(*reinterpret_cast<const __half2*>(&w), __float2half2_rn(raised_inf<__half>()));
    return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t raise2(uint32_t w, __nv_bfloat16)
{
    const __nv_bfloat162 p = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&w), __float2bfloat162_rn(raised_inf<__nv_bfloat16>()));
    return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t raise2(uint32_t w, float)
{
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(__uint_as_float(w)), "f"(raised_inf<float>()));
    return __float_as_uint(y);
}
template <typename T> __device__ __forceinline__ uint4 raise_vector(const uint4& q)
{
    return make_uint4(raise2(q.x, T()), raise2(q.y, T()), raise2(q.z, T()), raise2(q.w, T()));
}
// the largest element of 16 bytes (NaN aside)
__device__ __forceinline__ float vector_max(const uint4& q, float)
{
    return fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
}
__device__ __forceinline__ float vector_max(const uint4& q, __half)
{
    const __half2* w = reinterpret_cast<const __half2*>(&q);
    const __half2 m = __hmax2(__hmax2(w[0], w[1]), __hmax2(w[2], w[3]));
    return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float vector_max(const uint4& q, __nv_bfloat16)
{
    const __nv_bfloat162* w = reinterpret_cast<const __nv_bfloat162*>(&q);
    const __nv_bfloat162 m = __hmax2(__hmax2(w[0], w[1]), __hmax2(w[2], w[3]));
    return fmaxf(__low2float(m), __high2float(m));
}

// Running softmax sums of a set of logits x, in units of log2: with t = (x - m) c, c = log2(e) / temperature,
// s = sum 2^t and u = sum t 2^t.  m is the largest x so far (-inf: none, or only -inf, which leave s and u alone).
struct SoftSums {
    float m, s, u;
};
// How t is computed.  One fused multiply-add x c - sc does it, sc being m c rounded, off by the known d = m c - sc for
// every element alike: the sums are corrected by k = 2^-d afterwards.  Where m is so large that d matters, or so low
// that the raised -inf would count, `direct`: (x - m) c, element by element.
struct SoftScale {
    float sc, d, k;
    bool direct;
};
template <typename T>
__device__ __forceinline__ SoftScale soft_scale(float m, float c)
{
    SoftScale z = {0.0f, 0.0f, 1.0f, false};
    const float top = m == -CUDART_INF_F ? 0.0f : m;
    z.sc = __fmul_rn(top, c);
    z.direct = !(fabsf(z.sc) <= 1e6f && (raised_inf<T>() - top) * c < -200.0f);
    if (!z.direct) {
        z.d = fmaf(top, c, -z.sc);
        z.k = exp2_approx(-z.d);
    }
    return z;
}

template <bool ENT>
__device__ __forceinline__ void soft_rescale(SoftSums& a, float m_new, float c)
{
    if (m_new > a.m) {
        if (a.m != -CUDART_INF_F) {
            const float t = (a.m - m_new) * c;
            const float r = exp2_approx(t);
            if (ENT) a.u = r > 0.0f ? fmaf(a.s, t, a.u) * r : 0.0f * a.u;
            a.s *= r;
        }
        a.m = m_new;
    }
}
template <bool ENT>
__device__ __forceinline__ void soft_add(SoftSums& a, float x, float c)
{
    const float t = (x - (a.m == -CUDART_INF_F ? 0.0f : a.m)) * c;
    const float e = exp2_approx(t);
    a.s += e;
    if (ENT) a.u = fmaf(e, fmaxf(t, -1e4f), a.u);   // NaN comes in through e
}
// What 16-byte vectors q[k], of which `valid` has a bit each, add to s and u under the scale z
template <typename T, bool ENT, int K>
__device__ __forceinline__ float2 soft_terms(const SoftScale& z, const uint4 (&q)[K], unsigned valid, float c)
{
    constexpr int N = Vec16<T>::N;
    float2 s = make_float2(0.0f, 0.0f), u = make_float2(0.0f, 0.0f);
    const float2 c2 = make_float2(c, c), sc2 = make_float2(-z.sc, -z.sc);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (!(valid >> k & 1u)) continue;
        float f[N];
        Vec16<T>::unpack(ENT ? raise_vector<T>(q[k]) : q[k], f);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 t = __ffma2_rn(make_float2(f[i], f[i + 1]), c2, sc2);
            const float2 e = make_float2(exp2_approx(t.x), exp2_approx(t.y));
            s = __fadd2_rn(s, e);
            if (ENT) u = __ffma2_rn(e, t, u);
        }
    }
    return make_float2(s.x + s.y, u.x + u.y);
}
// The reference m need not be the maximum: it is kept while the new terms add up to no more than 5/4 of as many ones, so
// that it lies at most 4.4 bits below the maximum (16-bit types; fp32 3.4), which write_row takes out again.  That spares
// looking for the maximum everywhere (half an instruction an element, and everything waiting for it: an exact one shared by
// the warp took 5 to 19 % longer).  Otherwise: the vectors' maximum, one rescaling, and their terms again, which rows pay
// for that climb all along: 4096 x 131072 bf16 334 us from -20 to 20, 195 without a trend.
template <typename T, bool ENT, int K>
__device__ __forceinline__ void soft_add_vectors(SoftSums& a, SoftScale& z, const uint4 (&q)[K], unsigned valid, float c)
{
    constexpr int N = Vec16<T>::N;
    float2 su = make_float2(CUDART_INF_F, 0.0f);
    if (a.m != -CUDART_INF_F && !z.direct) su = soft_terms<T, ENT, K>(z, q, valid, c);
    if (!(su.x <= 1.25f * K * N)) {
        float top = -CUDART_INF_F;
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (valid >> k & 1u) top = fmaxf(top, vector_max(q[k], T()));
        if (top > a.m) {
            soft_rescale<ENT>(a, top, c);
            z = soft_scale<T>(a.m, c);
        }
        if (z.direct) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (!(valid >> k & 1u)) continue;
                float f[N];
                Vec16<T>::unpack(q[k], f);
#pragma unroll
                for (int i = 0; i < N; ++i) soft_add<ENT>(a, f[i], c);
            }
            return;
        }
        su = soft_terms<T, ENT, K>(z, q, valid, c);
    }
    a.s = fmaf(su.x, z.k, a.s);
    if (ENT) a.u = fmaf(fmaf(-z.d, su.x, su.y), z.k, a.u);
}
__device__ __forceinline__ float warp_max(float m)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}
// sums of a team's threads over their warp: the common maximum first, then one rescaling each
template <bool ENT>
__device__ __forceinline__ void soft_warp_join(SoftSums& a, float c)
{
    soft_rescale<ENT>(a, warp_max(a.m), c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
        if (ENT) a.u += __shfl_xor_sync(0xffffffffu, a.u, o);
    }
}

// A thread's own ring of 16-byte slots in shared memory, filled by asynchronous copies and read by nobody else, so that
// no thread waits for another: kRing - 1 groups of kGroup vectors are on their way while one is used, for no registers.
// (4096 x 131072 bf16 with entropy, groups x depth at four CTAs an SM, measured while each thread had a reference of its
// own from the start: 2 x 5 192 us, 2 x 3 195, 3 x 3 186, 4 x 2 188; without entropy 176, 180, 178, 182; 2040 x 50001 fp16
// 53, 57, 55, 59.)
constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kGroup = 2, kRing = 5;
struct VectorRing {
    uint4* slots;      // [kRing][kGroup] for this thread, kLpThreads apart
    __device__ __forceinline__ uint4* at(int stage, int k) const { return slots + (stage * kGroup + k) * kLpThreads; }
    // vectors i, i + lanes, ... of a row of nvec into a stage
    __device__ __forceinline__ void request(int stage, const uint4* body, long long i, int lanes, long long nvec) const
    {
#pragma unroll
        for (int k = 0; k < kGroup; ++k)
            if (i + k * lanes < nvec) copy16_async(at(stage, k), body + i + k * lanes);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
};

// One row read by `lanes` threads (this one is number `lane`): 16-byte vectors between the row's first and last 16-byte
// boundary, single elements outside.
template <typename T, bool ENT>
__device__ __forceinline__ SoftSums row_sums(const T* row, long long vocab, int lane, int lanes, float c, const VectorRing& ring)
{
    constexpr int N = Vec16<T>::N;
    SoftSums a = {-CUDART_INF_F, 0.0f, 0.0f};
    SoftScale z = soft_scale<T>(a.m, c);
    long long head = static_cast<long long>(((16u - (reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / sizeof(T));
    if (head > vocab) head = vocab;
    const long long nvec = (vocab - head) / N;
    const uint4* body = reinterpret_cast<const uint4*>(row + head);
    // the ends: fewer than 2 N <= 32 elements, at most one each for the first warp's lanes; requested first
    const long long tail = head + nvec * N;
    const bool end = lane < head + (vocab - tail);
    const float x_end = end ? to_f32(row[lane < head ? lane : tail + (lane - head)]) : 0.0f;
    const int step = kGroup * lanes;
    long long ahead = lane;
#pragma unroll
    for (int st = 0; st < kRing - 1; ++st, ahead += step) ring.request(st, body, ahead, lanes, nvec);
    int stage = 0;
    // the first reference is the warp's, so that few lanes have to replace theirs further on, one by one (4096 x 131072 bf16
    // 195 us, 248 with a first reference of each lane's own; 100000 x 1000 84 and 92)
    if (lane - (lane & 31) < nvec) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
        float top = -CUDART_INF_F;
#pragma unroll
        for (int k = 0; k < kGroup; ++k)
            if (lane + k * lanes < nvec) top = fmaxf(top, vector_max(*ring.at(0, k), T()));
        a.m = warp_max(top);
        z = soft_scale<T>(a.m, c);
    }
    for (long long i = lane; i < nvec; i += step, ahead += step) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
        uint4 q[kGroup];
        unsigned valid = 0;
#pragma unroll
        for (int k = 0; k < kGroup; ++k)
            if (i + k * lanes < nvec) {
                q[k] = *ring.at(stage, k);
                valid |= 1u << k;
            }
        // the stage before this one is free: its vectors were in registers a round ago
        ring.request(stage == 0 ? kRing - 1 : stage - 1, body, ahead, lanes, nvec);
        soft_add_vectors<T, ENT, kGroup>(a, z, q, valid, c);
        stage = stage == kRing - 1 ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (end) {
        soft_rescale<ENT>(a, x_end, c);
        soft_add<ENT>(a, x_end, c);
    }
    return a;
}

struct LogprobOut {
    float* logprobs;
    float* entropy;
    float2* row_stats;
};
// what one thread writes for row r once its sums are known.  s = 2^n s', s' in [1, 2): where the chosen action has a good
// part of the sum, its t = (x - m) c is close to n, and so is u / s where one action has most of it.  Both are taken relative
// to n, exactly, before anything is rounded: log-probability and entropy of a confident row are small, the two values whose
// difference they would be otherwise are not.  t uses the c of the sums, whose rounding cancels.  Two legal actions up to 9
// apart in rows of 1600 to 70001: log-probability 1.6e-7 off at most, entropy 1.8e-7; 5.5e-7 and 7.3e-7 without.
template <bool ENT>
__device__ __forceinline__ void write_row(const LogprobOut& o, long long r, const SoftSums& a, float chosen, float inv_temperature)
{
    // every logit -inf: no distribution; log-probability -inf, entropy 0, no gradient
    const bool empty = a.m == -CUDART_INF_F && a.s == 0.0f;
    const int bits = __float_as_int(a.s), e = (bits >> 23 & 255) - 127;
    const bool usual = e > -127 && e < 128;       // neither subnormal nor infinite nor NaN
    const float n = usual ? static_cast<float>(e) : 0.0f;
    const float log_rest = logf(usual ? __int_as_float((bits & 0x7fffff) | 0x3f800000) : a.s);
    const float log_s = empty ? 0.0f : fmaf(n, kLn2, log_rest);
    const float t = fmaf(chosen - a.m, inv_temperature * kLog2e, -n);
    o.logprobs[r] = empty ? -CUDART_INF_F : t > -1.0f ? fmaf(t, kLn2, -log_rest) : (chosen - a.m) * inv_temperature - log_s;
    if (ENT) o.entropy[r] = empty ? 0.0f : log_rest - kLn2 * (fmaf(-n, a.s, a.u) / a.s);
    if (o.row_stats != nullptr) o.row_stats[r] = make_float2(a.m, log_s);
}
template <bool ENT>
__device__ __forceinline__ void write_padding(const LogprobOut& o, long long r, bool beyond)
{
    if (beyond) atomicExch(&g_bad_action, 1);
    o.logprobs[r] = 0.0f;
    if (ENT) o.entropy[r] = 0.0f;
    if (o.row_stats != nullptr) o.row_stats[r] = make_float2(0.0f, 0.0f);
}

// Forward, one row per warp: rows of a few KB, where a CTA would spend its time on joining (20000 x 4000 bf16: 43 us, a CTA
// a row 127).
template <typename T, bool ENT>
__global__ void __launch_bounds__(kLpThreads, 4)
puff_logprobs_warp_kernel(const T* __restrict__ logits, RowMap lmap, const long long* __restrict__ actions, RowMap amap,
                          long long rows, long long vocab, float inv_temperature, LogprobOut out)
{
    __shared__ uint4 s_ring[kRing * kGroup * kLpThreads];
    const VectorRing ring = {s_ring + threadIdx.x};
    const float c = inv_temperature * kLog2e;
    const int lane = threadIdx.x & 31;
    const long long stride = static_cast<long long>(gridDim.x) * kLpWarps;
    for (long long r = blockIdx.x * static_cast<long long>(kLpWarps) + (threadIdx.x >> 5); r < rows; r += stride) {
        const long long action = actions[amap.at(r)];
        if (action < 0 || action >= vocab) {
            if (lane == 0) write_padding<ENT>(out, r, action >= vocab);
            continue;
        }
        const T* row = logits + lmap.at(r);
        const float chosen = to_f32(row[action]);
        SoftSums a = row_sums<T, ENT>(row, vocab, lane, 32, c, ring);
        soft_warp_join<ENT>(a, c);
        if (lane == 0) write_row<ENT>(out, r, a, chosen, inv_temperature);
    }
}

// Forward, one row per CTA, or per cluster of CTAs where rows are few: each takes a share of the row's vectors and the
// first adds up what the others leave in its shared memory (8 x 131072 bf16: 22.6 us by one CTA a row, 10.2 by eight, both
// with the launch).  Rows are not kept to a grid of resident CTAs: the block scheduler places them better (190 against 231).
template <typename T, bool ENT>
__global__ void __launch_bounds__(kLpThreads, 4)
puff_logprobs_cta_kernel(const T* __restrict__ logits, RowMap lmap, const long long* __restrict__ actions, RowMap amap,
                         long long rows, long long vocab, float inv_temperature, LogprobOut out)
{
    __shared__ uint4 s_ring[kRing * kGroup * kLpThreads];
    __shared__ SoftSums s_part[kLpWarps];
    __shared__ SoftSums s_cta[kLpMaxCluster];
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    const int share = static_cast<int>(cluster.block_rank()), shares = static_cast<int>(cluster.num_blocks());
    const VectorRing ring = {s_ring + threadIdx.x};
    const float c = inv_temperature * kLog2e;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // the first CTA's shared memory may be written only once that CTA runs: all arrive here, and wait before the first write
    bool waited = shares == 1;
    if (!waited) cluster.barrier_arrive();
    for (long long r = blockIdx.x / shares; r < rows; r += gridDim.x / shares) {
        const long long action = actions[amap.at(r)];
        const bool none = action < 0 || action >= vocab;
        if (none) {
            if (share == 0 && threadIdx.x == 0) write_padding<ENT>(out, r, action >= vocab);
            continue;       // the same for every CTA of the cluster
        }
        const T* row = logits + lmap.at(r);
        const float chosen = to_f32(row[action]);
        SoftSums a = row_sums<T, ENT>(row, vocab, share * kLpThreads + threadIdx.x, shares * kLpThreads, c, ring);
        soft_warp_join<ENT>(a, c);
        if (lane == 0) s_part[warp] = a;
        __syncthreads();
        if (!waited) cluster.barrier_wait();
        waited = true;
        if (warp == 0) {
            a = lane < kLpWarps ? s_part[lane] : SoftSums{-CUDART_INF_F, 0.0f, 0.0f};
            soft_warp_join<ENT>(a, c);
            if (shares == 1) {
                if (lane == 0) write_row<ENT>(out, r, a, chosen, inv_temperature);
            } else if (lane == 0) {
                *cluster.map_shared_rank(&s_cta[share], 0) = a;
            }
        }
        if (shares > 1) {
            cluster.sync();
            if (share == 0 && warp == 0) {
                a = lane < shares ? s_cta[lane] : SoftSums{-CUDART_INF_F, 0.0f, 0.0f};
                soft_warp_join<ENT>(a, c);
                if (lane == 0) write_row<ENT>(out, r, a, chosen, inv_temperature);
            }
            if (r + gridDim.x / shares < rows) cluster.sync();   // before s_cta is written again
        } else {
            __syncthreads();
        }
    }
    if (!waited) cluster.barrier_wait();
}

// The gradient of a row's logits as p (A + B t) with t = log2 p: A = -(dlp + dh H) / temperature, B = -dh ln 2 /
// temperature.  t is one multiply-add again, x c - l with l = m c + log2 s rounded and its error d carried into A and the
// factor 2^-d of both; `direct` as in SoftScale.
struct RowGradient {
    float c, l, a, b, m, log2_s, dlp;
    bool direct;
};
template <typename T, bool ENT>
__device__ __forceinline__ RowGradient row_gradient(float m, float log_s, float h, float dlp, float dh, float inv_temperature)
{
    RowGradient g;
    g.c = inv_temperature * kLog2e;
    g.m = m;
    g.log2_s = __fmul_rn(log_s, kLog2e);
    g.dlp = dlp * inv_temperature;
    const float mc = __fmul_rn(m, g.c);      // rounded here: the errors below are of these very values
    g.l = __fadd_rn(mc, g.log2_s);
    g.direct = !(fabsf(g.l) <= 1e6f && fabsf(mc) <= 1e6f && (raised_inf<T>() - m) * g.c < -200.0f);
    float d = 0.0f;
    if (!g.direct) {
        const float back = __fsub_rn(g.l, mc);
        d = fmaf(m, g.c, -mc) + __fadd_rn(__fsub_rn(mc, __fsub_rn(g.l, back)), __fsub_rn(g.log2_s, back));
    }
    const float k = exp2_approx(-d) * inv_temperature;
    g.b = ENT ? -dh * kLn2 * k : 0.0f;
    g.a = ENT ? -fmaf(dh, fmaf(-kLn2, d, h), dlp) * k : -dlp * k;
    return g;
}
template <bool ENT>
__device__ __forceinline__ float logit_gradient(float x, const RowGradient& g)
{
    const float t = g.direct ? fmaf(x - g.m, g.c, -g.log2_s) : fmaf(x, g.c, -g.l);
    const float p = exp2_approx(t);
    return p * (ENT ? fmaf(g.b, fmaxf(t, -1e4f), g.a) : g.a);
}

// Backward of rows beyond the small kernel's: a warp takes 256 16-byte vectors of a row of dlogits (contiguous).  The
// vectors are those of the output; where the row of logits lies at another offset from a 16-byte boundary, a vector is
// cut out of the two aligned ones that hold it.  The first warp of a row also does the elements at its ends.
struct GradientRow {
    const uint4* in;
    uint4* to;
    long long head, nvec, action;
    unsigned shift;
    bool none;
};
// vectors first, first + 32, ... of the row, U of them; 4096 x 131072 bf16: eight at once 328 us, four 369; shifted ones need
// twice the registers, and eight of those spill (143 us against 94 for 2040 x 50001)
template <typename T, bool ENT, int U, bool SHIFTED>
__device__ __forceinline__ void gradient_vectors(const GradientRow& row, const RowGradient& grad, long long first)
{
    constexpr int N = Vec16<T>::N;
    const float2 a2 = make_float2(grad.a, grad.a), b2 = make_float2(grad.b, grad.b);
    const float2 c2 = make_float2(grad.c, grad.c), l2 = make_float2(-grad.l, -grad.l);
    uint4 q[U];
    if (!row.none) {
#pragma unroll
        for (int k = 0; k < U; ++k)
            if (first + 32 * k < row.nvec) q[k] = __ldg(row.in + first + 32 * k);
        if (SHIFTED) {
            uint4 next[U];
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (first + 32 * k < row.nvec) next[k] = __ldg(row.in + first + 32 * k + 1);
#pragma unroll
            for (int k = 0; k < U; ++k) q[k] = cut_vector(q[k], next[k], row.shift);
        }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
        const long long i = first + 32 * k;
        if (i >= row.nvec) break;
        float f[N];
        if (row.none) {
#pragma unroll
            for (int v = 0; v < N; ++v) f[v] = 0.0f;
        } else {
            if (grad.direct) {
                Vec16<T>::unpack(q[k], f);
#pragma unroll
                for (int v = 0; v < N; ++v) f[v] = logit_gradient<ENT>(f[v], grad);
            } else {
                Vec16<T>::unpack(ENT ? raise_vector<T>(q[k]) : q[k], f);
#pragma unroll
                for (int v = 0; v < N; v += 2) {
                    const float2 t = __ffma2_rn(make_float2(f[v], f[v + 1]), c2, l2);
                    const float2 p = make_float2(exp2_approx(t.x), exp2_approx(t.y));
                    const float2 d = __fmul2_rn(p, ENT ? __ffma2_rn(b2, t, a2) : a2);
                    f[v] = d.x;
                    f[v + 1] = d.y;
                }
            }
            const long long at = row.action - (row.head + i * N);
            if (at >= 0 && at < N) {                         // the chosen one is among these
#pragma unroll
                for (int v = 0; v < N; ++v) f[v] += at == v ? grad.dlp : 0.0f;
            }
        }
        row.to[i] = Vec16<T>::pack(f);
    }
}

constexpr int kLpUnitVecs = 8;      // vectors a lane
template <typename T, bool ENT>
__global__ void __launch_bounds__(kLpThreads, 4)
puff_logprobs_backward_kernel(const T* __restrict__ logits, RowMap lmap, const long long* __restrict__ actions,
                              RowMap amap, long long rows, long long vocab, int warps_per_row, unsigned ctas_per_row,
                              float inv_temperature, const float2* __restrict__ row_stats, const float* __restrict__ entropy,
                              const float* __restrict__ dlogprobs, const float* __restrict__ dentropy,
                              T* __restrict__ dlogits)
{
    constexpr int N = Vec16<T>::N;
    const int lane = threadIdx.x & 31;
    // 8 / warps_per_row rows a CTA, or ctas_per_row CTAs a row
    const unsigned block_row = blockIdx.x / ctas_per_row;
    const int warp = threadIdx.x >> 5;
    const long long r = static_cast<long long>(block_row) * (kLpWarps / warps_per_row) + warp / warps_per_row;
    if (r >= rows) return;
    const long long chunk = (blockIdx.x - block_row * ctas_per_row) * kLpWarps + warp % warps_per_row;
    GradientRow g;
    g.action = actions[amap.at(r)];
    const float2 st = row_stats[r];
    const float dlp = dlogprobs[r], dh = ENT ? dentropy[r] : 0.0f, h = ENT ? entropy[r] : 0.0f;
    const T* row = logits + lmap.at(r);
    T* out = dlogits + r * vocab;
    g.none = g.action < 0 || g.action >= vocab || (st.x == -CUDART_INF_F && st.y == 0.0f);
    const RowGradient grad = row_gradient<T, ENT>(st.x, st.y, h, dlp, dh, inv_temperature);
    // vectors [0, nvec) start at element `head` of the row; shift: how far behind a boundary the logits' bytes lie
    g.head = static_cast<long long>(((16u - (reinterpret_cast<uintptr_t>(out) & 15u)) & 15u) / sizeof(T));
    g.shift = static_cast<unsigned>(reinterpret_cast<uintptr_t>(row + g.head) & 15u);
    if (g.shift != 0 && g.head * static_cast<long long>(sizeof(T)) < g.shift) g.head += N;   // the aligned vector would start before the row
    g.nvec = g.shift == 0 ? (vocab - g.head) / N : ((vocab - g.head) * static_cast<long long>(sizeof(T)) + g.shift) / 16 - 1;
    if (g.nvec < 0) g.nvec = 0;
    g.in = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(row + g.head) & ~static_cast<uintptr_t>(15));
    g.to = reinterpret_cast<uint4*>(out + g.head);
    const long long first = chunk * (32 * kLpUnitVecs) + lane;
    if (g.shift == 0) {
        gradient_vectors<T, ENT, kLpUnitVecs, false>(g, grad, first);
    } else {
#pragma unroll 1
        for (int part = 0; part < 2; ++part) gradient_vectors<T, ENT, kLpUnitVecs / 2, true>(g, grad, first + part * (16 * kLpUnitVecs));
    }
    if (chunk == 0) {
        const long long tail = g.head + g.nvec * N;
        for (long long j = lane; j < g.head + (vocab - tail); j += 32) {
            const long long e = j < g.head ? j : tail + (j - g.head);
            if (e >= vocab) break;
            float d = 0.0f;
            if (!g.none) {
                d = logit_gradient<ENT>(to_f32(row[e]), grad);
                if (e == g.action) d += grad.dlp;
            }
            out[e] = from_f32<T>(d);
        }
    }
}

// Small rows, both directions.  A CTA brings 256 / G rows into shared memory by 16-byte copies of their common span,
// wherever rows begin; G threads then work on a row from there (fewer than 33 elements each), and the backward pass
// writes gradients over the logits and copies the span out.  The maximum and the sums are computed
// again in the backward pass, so that the forward pass keeps nothing of a row (reading 8 bytes of each back instead has not
// been measured).  Rows start at different banks:
// row i of the tile begins its walk i * skew elements in.  524288 x 18 fp32: 20 us forward and 29 backward, where a warp a
// row took 316 and 278; instruction issue (81 and 87 %) bounds it, DRAM stands at 40 %.
// Up to which size a row is small, against a warp a row (us, small / warp): 500000 x 256 bf16 forward 131 / 283 and backward
// 207 / 260; 200000 x 333 86 / 131 and 131 / 133; 200000 x 500 117 / 131 and 184 / 139.
constexpr int kLpSmall = 512, kLpSmallBackward = PUFF_LOGPROBS_STATS_ABOVE;      // 384
template <typename T, bool ENT, int G, bool BACKWARD>
__global__ void __launch_bounds__(kLpThreads)
puff_logprobs_small_kernel(const T* __restrict__ logits, RowMap lmap, const long long* __restrict__ actions, RowMap amap,
                           long long rows, int vocab, float inv_temperature, LogprobOut out,
                           const float* __restrict__ dlogprobs, const float* __restrict__ dentropy, T* __restrict__ dlogits)
{
    extern __shared__ uint4 s_raw[];
    constexpr int R = kLpThreads / G;
    const long long r0 = static_cast<long long>(blockIdx.x) * R;
    const int n_rows = static_cast<int>(rows - r0 < R ? rows - r0 : R);
    const int local = threadIdx.x / G, g = threadIdx.x % G;
    const bool has = local < n_rows;
    const long long action = has ? actions[amap.at(r0 + local)] : -1;
    const bool live = action >= 0 && action < vocab;
    float dlp = 0.0f, dh = 0.0f;
    if (BACKWARD && has) {
        dlp = dlogprobs[r0 + local];
        if (ENT) dh = dentropy[r0 + local];
    }
    // ---- in
    const bool one_run = lmap.inner_stride == vocab && (lmap.one_run || r0 / lmap.inner == (r0 + n_rows - 1) / lmap.inner);
    const T* src = logits + lmap.at(r0);
    const int count = n_rows * vocab;
    const unsigned out_phase = BACKWARD ? static_cast<unsigned>(reinterpret_cast<uintptr_t>(dlogits + r0 * vocab) & 15u) : 0u;
    const unsigned phase = one_run ? static_cast<unsigned>(reinterpret_cast<uintptr_t>(src) & 15u) : out_phase;
    T* tile = reinterpret_cast<T*>(reinterpret_cast<char*>(s_raw) + phase);
    constexpr int N = Vec16<T>::N;
    const int head_all = static_cast<int>(((16u - phase) & 15u) / sizeof(T));
    const int head = head_all < count ? head_all : count, body = (count - head) / N, tail = head + body * N;
    if (one_run) {
        for (int i = threadIdx.x; i < body; i += kLpThreads)
            copy16_async(reinterpret_cast<uint4*>(tile + head) + i, reinterpret_cast<const uint4*>(src + head) + i);
        if (static_cast<int>(threadIdx.x) < head + (count - tail)) {
            const int e = static_cast<int>(threadIdx.x) < head ? threadIdx.x : tail + (threadIdx.x - head);
            tile[e] = src[e];
        }
        copy_async_wait();
    } else {
        for (int i = threadIdx.x >> 5; i < n_rows; i += kLpWarps) {
            const T* row = logits + lmap.at(r0 + i);
            for (int j = threadIdx.x & 31; j < vocab; j += 32) tile[i * vocab + j] = row[j];
        }
    }
    __syncthreads();
    // ---- the sums of this thread's row, element by element from `start` on and around the end
    constexpr int kBankElems = 128 / sizeof(T);
    const int skew = G == 1 ? (sizeof(T) == 4 ? 1 - (vocab & 1) : (2 - vocab) & 3)
                            : ((G * (kBankElems / 32) - vocab) & (kBankElems - 1));
    const int start = (local * skew) % vocab;
    T* const row = tile + local * vocab;
    T* const wrapped = row - vocab;
    // (one loop with a select: as two loops, up to the end and from the beginning, lanes diverge and it takes twice as long)
    auto each = [&](auto&& f) {
        if (live)
#pragma unroll 4
            for (int j = start + g; j < start + vocab; j += G) f((j < vocab ? row : wrapped)[j]);
    };
    const float c = inv_temperature * kLog2e;
    const float chosen = live ? to_f32(row[action]) : 0.0f;
    SoftSums a = {-CUDART_INF_F, 0.0f, 0.0f};
    each([&](T& x) { a.m = fmaxf(a.m, to_f32(x)); });
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) a.m = fmaxf(a.m, __shfl_xor_sync(0xffffffffu, a.m, o));
    const SoftScale z = soft_scale<T>(a.m, c);
    if (z.direct) {
        each([&](T& x) { soft_add<ENT>(a, to_f32(x), c); });
    } else {
        float s = 0.0f, u = 0.0f;
        each([&](T& x) {
            const float t = fmaf(to_f32(x), c, -z.sc), e = exp2_approx(t);
            s += e;
            if (ENT) u = fmaf(e, fmaxf(t, -1e4f), u);
        });
        a.s = s * z.k;
        if (ENT) a.u = fmaf(-z.d, s, u) * z.k;
    }
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) {
        a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
        if (ENT) a.u += __shfl_xor_sync(0xffffffffu, a.u, o);
    }
    if (!BACKWARD) {
        if (has && g == 0) {
            if (live) write_row<ENT>(out, r0 + local, a, chosen, inv_temperature);
            else write_padding<ENT>(out, r0 + local, action >= vocab);
        }
        return;
    }
    // ---- gradients over the logits; the chosen one's is written again, with its own term
    const bool none = !live || (a.m == -CUDART_INF_F && a.s == 0.0f);
    float d_chosen = 0.0f;
    if (none) {
        if (has)
            for (int k = g; k < vocab; k += G) row[k] = from_f32<T>(0.0f);
    } else {
        const float log_s = logf(a.s);
        const float h = ENT ? log_s - kLn2 * (a.u / a.s) : 0.0f;
        const RowGradient grad = row_gradient<T, ENT>(a.m, log_s, h, dlp, dh, inv_temperature);
        if (grad.direct) {
            each([&](T& x) { x = from_f32<T>(logit_gradient<ENT>(to_f32(x), grad)); });
        } else {
            each([&](T& x) {
                const float t = fmaf(to_f32(x), grad.c, -grad.l);
                x = from_f32<T>(exp2_approx(t) * (ENT ? fmaf(grad.b, fmaxf(t, -1e4f), grad.a) : grad.a));
            });
        }
        d_chosen = logit_gradient<ENT>(chosen, grad) + grad.dlp;
    }
    __syncwarp();
    if (!none && g == 0) row[action] = from_f32<T>(d_chosen);
    __syncthreads();
    // ---- out
    T* dst = dlogits + r0 * vocab;
    if (phase == out_phase) {
        for (int i = threadIdx.x; i < body; i += kLpThreads)
            reinterpret_cast<uint4*>(dst + head)[i] = reinterpret_cast<const uint4*>(tile + head)[i];
        if (static_cast<int>(threadIdx.x) < head + (count - tail)) {
            const int e = static_cast<int>(threadIdx.x) < head ? threadIdx.x : tail + (threadIdx.x - head);
            dst[e] = tile[e];
        }
    } else {
        for (int i = threadIdx.x; i < count; i += kLpThreads) dst[i] = tile[i];
    }
}

template <typename T, bool ENT, bool BACKWARD>
static cudaError_t launch_small(const void* logits, RowMap lmap, const long long* actions, RowMap amap, long long rows,
                                long long vocab, float inv_t, LogprobOut out, const float* dlogprobs, const float* dentropy,
                                void* dlogits, cudaStream_t st)
{
    int g = 1;
    while (vocab > 32 * g) g *= 2;
    const long long tile = kLpThreads / g;
    const size_t smem = static_cast<size_t>(tile) * vocab * sizeof(T) + 32;
    if ((rows + tile - 1) / tile > 0x7fffffffLL) return cudaErrorInvalidConfiguration;   // rows that repeat with stride 0
    const int grid = static_cast<int>((rows + tile - 1) / tile);
#define PUFF_SMALL(G)                                                                                                       \
    puff_logprobs_small_kernel<T, ENT, G, BACKWARD><<<grid, kLpThreads, smem, st>>>(                                        \
        static_cast<const T*>(logits), lmap, actions, amap, rows, static_cast<int>(vocab), inv_t, out, dlogprobs, dentropy, \
        static_cast<T*>(dlogits))
    if (g == 1) PUFF_SMALL(1);
    else if (g == 2) PUFF_SMALL(2);
    else if (g == 4) PUFF_SMALL(4);
    else if (g == 8) PUFF_SMALL(8);
    else PUFF_SMALL(16);
#undef PUFF_SMALL
    return cudaGetLastError();
}

template <typename T, bool ENT>
static cudaError_t launch_logprobs(const void* logits, RowMap lmap, const long long* actions, RowMap amap, long long rows,
                                   long long vocab, float inv_t, float* logprobs, float* entropy, float* row_stats,
                                   cudaStream_t st)
{
    // (a small backward pass works the statistics out again)
    const LogprobOut out = {logprobs, entropy, vocab <= kLpSmallBackward ? nullptr : reinterpret_cast<float2*>(row_stats)};
    if (vocab <= kLpSmall)
        return launch_small<T, ENT, false>(logits, lmap, actions, amap, rows, vocab, inv_t, out, nullptr, nullptr, nullptr, st);
    const T* z = static_cast<const T*>(logits);
    const long long bytes = vocab * static_cast<long long>(sizeof(T));
    // a warp a row while rows are short and many enough to give every SM sixteen warps
    if (bytes <= 16384 && rows >= 148 * 16) {
        const long long grid = (rows + kLpWarps - 1) / kLpWarps;
        puff_logprobs_warp_kernel<T, ENT><<<static_cast<int>(grid < (1 << 30) ? grid : (1 << 30)), kLpThreads, 0, st>>>(
            z, lmap, actions, amap, rows, vocab, inv_t, out);
        return cudaGetLastError();
    }
    // otherwise a CTA, or two, four, eight while that leaves SMs idle and each thread has two vectors to read
    int shares = 1;
    while (shares < kLpMaxCluster && rows * shares < 148 * 2 && bytes >= 2LL * shares * kLpThreads * 32) shares *= 2;
    const long long grid = rows < (1 << 26) ? rows : (1 << 26);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid * shares));
    cfg.blockDim = dim3(kLpThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(shares);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, puff_logprobs_cta_kernel<T, ENT>, z, lmap, actions, amap, rows, vocab, inv_t, out);
}
template <typename T, bool ENT>
static cudaError_t launch_logprobs_backward(const void* logits, RowMap lmap, const long long* actions, RowMap amap,
                                            long long rows, long long vocab, float inv_t, const float* row_stats,
                                            const float* entropy, const float* dlogprobs, const float* dentropy,
                                            void* dlogits, cudaStream_t st)
{
    if (vocab <= kLpSmallBackward)
        return launch_small<T, ENT, true>(logits, lmap, actions, amap, rows, vocab, inv_t, LogprobOut{}, dlogprobs, dentropy,
                                          dlogits, st);
    constexpr long long per_unit = 32LL * kLpUnitVecs * Vec16<T>::N;
    const long long units = (vocab + per_unit - 1) / per_unit;
    int warps_per_row = 1;
    while (warps_per_row < kLpWarps && warps_per_row < units) warps_per_row *= 2;
    const long long ctas_per_row = (units + kLpWarps - 1) / kLpWarps, rows_per_cta = kLpWarps / warps_per_row;
    const long long grid = (rows + rows_per_cta - 1) / rows_per_cta * ctas_per_row;
    puff_logprobs_backward_kernel<T, ENT><<<static_cast<unsigned>(grid), kLpThreads, 0, st>>>(
        static_cast<const T*>(logits), lmap, actions, amap, rows, vocab, warps_per_row, static_cast<unsigned>(ctas_per_row), inv_t,
        reinterpret_cast<const float2*>(row_stats), entropy, dlogprobs, dentropy, static_cast<T*>(dlogits));
    return cudaGetLastError();
}

// bytes from the first to one past the last element of rows [outer, inner] of `width` elements
static long long rows_span(long long outer, long long inner, long long width, long long os, long long is, int size)
{
    return ((outer - 1) * os + (inner - 1) * is + width) * size;
}

// what both directions require of the logits and actions; PUFF_OK with *rows == 0 means nothing to do
static int check_logprobs(const void* logits, int dtype, const long long* actions, long long outer, long long inner,
                          long long vocab, long long los, long long lis, long long aos, long long ais,
                          float temperature, long long* rows)
{
    *rows = 0;
    const int size = dtype_bytes(dtype);
    if (size == 0) return PUFF_ERR_DTYPE;
    if (outer < 0 || inner < 0 || vocab < 0 || los < 0 || lis < 0 || aos < 0 || ais < 0) return PUFF_ERR_SHAPE;
    if (!(temperature > 0.0f) || temperature > 3.0e38f || 1.5f / temperature > 3.0e38f) return PUFF_ERR_VALUE;
    if (outer == 0 || inner == 0) return PUFF_OK;
    if (vocab == 0) return PUFF_ERR_SHAPE;
    if (inner > (1LL << 40) / outer || vocab > (1LL << 46) / (outer * inner)) return PUFF_ERR_SIZE;
    if (logits == nullptr || actions == nullptr) return PUFF_ERR_NULL;
    if (misaligned(logits, size) || misaligned(actions, 8)) return PUFF_ERR_ALIGN;
    *rows = outer * inner;
    return PUFF_OK;
}
}  // namespace puff

using namespace puff;

extern "C" int puff_policy_sm100_logprobs(const void* logits, int dtype, const long long* actions, long long outer,
                                          long long inner, long long vocab, long long logits_outer_stride,
                                          long long logits_inner_stride, long long actions_outer_stride,
                                          long long actions_inner_stride, float temperature, float* logprobs,
                                          float* entropy, float* row_stats, void* cuda_stream)
{
    long long rows;
    int rc = check_logprobs(logits, dtype, actions, outer, inner, vocab, logits_outer_stride, logits_inner_stride,
                            actions_outer_stride, actions_inner_stride, temperature, &rows);
    if (rc != PUFF_OK || rows == 0) return rc;
    if (logprobs == nullptr) return PUFF_ERR_NULL;
    if (misaligned(logprobs, 4) || misaligned(entropy, 4) || misaligned(row_stats, 8)) return PUFF_ERR_ALIGN;
    const int size = dtype_bytes(dtype);
    const long long lspan = rows_span(outer, inner, vocab, logits_outer_stride, logits_inner_stride, size);
    const long long aspan = rows_span(outer, inner, 1, actions_outer_stride, actions_inner_stride, 8);
    const float* out[3] = {logprobs, entropy, row_stats};
    const long long out_bytes[3] = {4 * rows, 4 * rows, 8 * rows};
    for (int i = 0; i < 3; ++i) {
        if (spans_overlap(out[i], out_bytes[i], logits, lspan) || spans_overlap(out[i], out_bytes[i], actions, aspan))
            return PUFF_ERR_ALIAS;
        for (int j = 0; j < i; ++j)
            if (spans_overlap(out[i], out_bytes[i], out[j], out_bytes[j])) return PUFF_ERR_ALIAS;
    }
    int sms = 0;
    rc = require_sm100(&sms);
    if (rc != PUFF_OK) return rc;
    const RowMap lmap = {inner, logits_outer_stride, logits_inner_stride, outer == 1};
    const RowMap amap = {inner, actions_outer_stride, actions_inner_stride, outer == 1};
    const float inv_t = 1.0f / temperature;
    cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
#define PUFF_RUN(T)                                                                                                        \
    (entropy != nullptr ? launch_logprobs<T, true>(logits, lmap, actions, amap, rows, vocab, inv_t, logprobs, entropy,     \
                                                   row_stats, st)                                                          \
                        : launch_logprobs<T, false>(logits, lmap, actions, amap, rows, vocab, inv_t, logprobs, entropy,    \
                                                    row_stats, st))
    const cudaError_t e = dtype == PUFF_DTYPE_F32 ? PUFF_RUN(float) : dtype == PUFF_DTYPE_F16 ? PUFF_RUN(__half) : PUFF_RUN(__nv_bfloat16);
#undef PUFF_RUN
    count_launch();
    return static_cast<int>(e);
}

extern "C" int puff_policy_sm100_logprobs_backward(const void* logits, int dtype, const long long* actions,
                                                   long long outer, long long inner, long long vocab,
                                                   long long logits_outer_stride, long long logits_inner_stride,
                                                   long long actions_outer_stride, long long actions_inner_stride,
                                                   float temperature, const float* row_stats, const float* entropy,
                                                   const float* dlogprobs, const float* dentropy, void* dlogits,
                                                   void* cuda_stream)
{
    long long rows;
    int rc = check_logprobs(logits, dtype, actions, outer, inner, vocab, logits_outer_stride, logits_inner_stride,
                            actions_outer_stride, actions_inner_stride, temperature, &rows);
    if (rc != PUFF_OK || rows == 0) return rc;
    if (row_stats == nullptr || dlogprobs == nullptr || dlogits == nullptr) return PUFF_ERR_NULL;
    if (dentropy != nullptr && entropy == nullptr) return PUFF_ERR_NULL;
    const int size = dtype_bytes(dtype);
    if (misaligned(row_stats, 8) || misaligned(entropy, 4) || misaligned(dlogprobs, 4) || misaligned(dentropy, 4) ||
        misaligned(dlogits, size))
        return PUFF_ERR_ALIGN;
    const long long span = rows * vocab * size;
    if (spans_overlap(dlogits, span, logits, rows_span(outer, inner, vocab, logits_outer_stride, logits_inner_stride, size)) ||
        spans_overlap(dlogits, span, actions, rows_span(outer, inner, 1, actions_outer_stride, actions_inner_stride, 8)) ||
        spans_overlap(dlogits, span, row_stats, 8 * rows) || spans_overlap(dlogits, span, entropy, 4 * rows) ||
        spans_overlap(dlogits, span, dlogprobs, 4 * rows) || spans_overlap(dlogits, span, dentropy, 4 * rows))
        return PUFF_ERR_ALIAS;
    int sms = 0;
    rc = require_sm100(&sms);
    if (rc != PUFF_OK) return rc;
    const RowMap lmap = {inner, logits_outer_stride, logits_inner_stride, outer == 1};
    const RowMap amap = {inner, actions_outer_stride, actions_inner_stride, outer == 1};
    const float inv_t = 1.0f / temperature;
    cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
#define PUFF_RUN(T)                                                                                                       \
    (dentropy != nullptr ? launch_logprobs_backward<T, true>(logits, lmap, actions, amap, rows, vocab, inv_t, row_stats,  \
                                                             entropy, dlogprobs, dentropy, dlogits, st)                   \
                         : launch_logprobs_backward<T, false>(logits, lmap, actions, amap, rows, vocab, inv_t, row_stats, \
                                                              entropy, dlogprobs, dentropy, dlogits, st))
    const cudaError_t e = dtype == PUFF_DTYPE_F32 ? PUFF_RUN(float) : dtype == PUFF_DTYPE_F16 ? PUFF_RUN(__half) : PUFF_RUN(__nv_bfloat16);
#undef PUFF_RUN
    count_launch();
    return static_cast<int>(e);
}

extern "C" int puff_policy_sm100_bad_action(void)
{
    int flag = 0;
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&flag, g_bad_action, sizeof(int));
    if (e == cudaSuccess && flag != 0) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_bad_action, &zero, sizeof(int));
    }
    return e == cudaSuccess ? flag : PUFF_ERR_CUDA_BASE - static_cast<int>(e);
}
