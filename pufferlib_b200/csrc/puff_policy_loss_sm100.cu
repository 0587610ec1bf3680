// Clipped policy loss with a KL term to a reference policy, forward and backward (sm_100a).
//
// Per token, with d = logprob - old_logprob, r = e^d, A the advantage and q = ref_logprob - logprob:
//     policy = max(-A r, -A clip(r, 1 - clip_low, 1 + clip_high)),    kl = e^q - 1 - q  (>= 0, 0 where q = 0)
//     loss   = mean(policy) + kl_coef mean(kl) - ent_coef mean(entropy)
//     dloss / dlogprob = w ([r not clipped against A] (-A r) - kl_coef (e^q - 1)),   dloss / dentropy = -ent_coef w
// pufferl.py:390-411 and :422 for whole minibatches (w = 1 / tokens), extended to masked tokens, a mean over
// sequences of their token means (w = 1 / (length sequences)) and the KL term.
//
// The forward pass writes the ratio and the per-token slope dloss/dlogprob / w; w needs the count of all tokens, so
// the backward pass multiplies by it.  Which side of a clip border a ratio is on is decided in 48 bits, as
// logprob - old_logprob against log(1 - clip_low) and log(1 + clip_high).
//
// Memory-bound: 13 to 29 bytes a token forward, 8 to 13 backward.  131072 x 256 masked tokens with KL and entropy: 173 us
// forward (5.6 TB/s; a copy runs at 6.55) and 80 backward; means over its sequences 196.  What was in the way: fp64 for
// differences and sums (415 us), exponentials for tokens near the old policy (284).
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/puff_advantage.h"
#include "puff_policy.cuh"

namespace puff {

constexpr int kLossThreads = 256;
constexpr int kLossWarps = kLossThreads / 32;
constexpr int kLossMaxBlocks = 148 * 4;
constexpr int kLossSums = 8;   // policy, kl, entropy, -d, e^d - 1 - d, clipped, tokens, sequences

struct LossArgs {
    const float* logprobs;
    const float* old_logprobs;
    const float* advantages;
    const float* ref_logprobs;
    const float* entropy;
    const unsigned char* mask;
    float* ratio;
    float* slope;
    float* row_scale;
    long long rows, steps;
    float clip_low_value, clip_low_rest, clip_high_value, clip_high_rest;                     // 1 - clip_low, 1 + clip_high
    float log_low, log_low_rest, log_high, log_high_rest;   // log(1 - clip_low), log(1 + clip_high), 48 bits each
    float kl_coef;
};

// e^x - 1 - x for |x| <= 1 as x^2 (1/2 + x Q(x)): the difference itself would cancel.  Q is the polynomial of degree 6
// through the Chebyshev nodes of ((e^x - 1 - x) / x^2 - 1/2) / x on [-1, 1]; the result is good to 3 half steps of fp32.
__device__ __forceinline__ float exp_excess(float x)
{
    float p = 2.799926278385101e-06f;
    p = fmaf(p, x, 2.5288434699177742e-05f);
    p = fmaf(p, x, 1.9839055312331766e-04f);
    p = fmaf(p, x, 1.3886447995901108e-03f);
    p = fmaf(p, x, 8.333336561918259e-03f);
    p = fmaf(p, x, 4.166669771075249e-02f);
    p = fmaf(p, x, 0.1666666716337204f);
    p = fmaf(p, x, 0.5f);
    return x * x * p;
}
// the rounding error of d = a - b, exactly (Knuth's two-sum).  fp32 pairs because conversions to fp64 and back bounded
// the kernel: 415 us for 131072 x 256 tokens.
__device__ __forceinline__ float difference_rest(float a, float b, float d)
{
    const float back = __fsub_rn(d, a);
    return __fsub_rn(__fsub_rn(a, __fsub_rn(d, back)), __fadd_rn(b, back));
}

struct TokenLoss {
    float policy, policy_rest, kl, excess, ratio, slope, d;
    bool clipped;
};
__device__ __forceinline__ TokenLoss token_loss(const LossArgs& p, float lp, float old, float adv, float ref)
{
    TokenLoss t;
    const float d = __fsub_rn(lp, old);
    bool above = d > p.log_high, below = d < p.log_low;
    t.d = d;
    // the usual token: no exponential, e^d = 1 + (d + (e^d - 1 - d))
    t.excess = exp_excess(d);
    const float em1 = d + t.excess;
    t.ratio = __fadd_rn(1.0f, em1);
    float ratio_rest = __fsub_rn(em1, __fsub_rn(t.ratio, 1.0f));
    if (!(fabsf(d) < 0.5f) || d == p.log_high || d == p.log_low) {
        const float rest = difference_rest(lp, old, d);
        above = above || (d == p.log_high && rest > p.log_high_rest);
        below = below || (d == p.log_low && rest < p.log_low_rest);
        const float e = expf(d);
        // beyond 80 the exponential is 0, infinite, or the rest does not matter
        t.ratio = fabsf(d) < 80.0f ? fmaf(e, rest, e) : e;
        ratio_rest = 0.0f;
        if (!(fabsf(d) < 1.0f)) t.excess = (t.ratio - 1.0f) - d;
    }
    const bool cut = (above && adv > 0.0f) || (below && adv < 0.0f);
    // the policy term as a rounded product and its error: the terms of a batch nearly cancel, their rounding does not
    const float held = cut ? (above ? p.clip_high_value : p.clip_low_value) : t.ratio;
    const float held_rest = cut ? (above ? p.clip_high_rest : p.clip_low_rest) : ratio_rest;
    t.policy = __fmul_rn(-adv, held);
    t.policy_rest = fmaf(-adv, held_rest, fmaf(-adv, held, -t.policy));
    t.slope = cut ? 0.0f : t.policy;
    t.clipped = above || below;
    t.kl = 0.0f;
    if (p.ref_logprobs != nullptr) {
        const float q = __fsub_rn(ref, lp);
        t.kl = exp_excess(q);
        float em1 = q + t.kl;
        if (!(fabsf(q) < 1.0f)) {
            const float e = expf(q);
            em1 = (fabsf(q) < 80.0f ? fmaf(e, difference_rest(ref, lp, q), e) : e) - 1.0f;
            t.kl = em1 - q;
        }
        t.slope = fmaf(-p.kl_coef, em1, t.slope);
    }
    return t;
}

// VEC adjacent values
template <int VEC> struct Pack;
template <> struct Pack<1> {
    static __device__ __forceinline__ void load(const float* p, float* f) { f[0] = __ldg(p); }
    static __device__ __forceinline__ void store(float* p, const float* f) { *p = f[0]; }
    static __device__ __forceinline__ unsigned mask(const unsigned char* p) { return __ldg(p) != 0 ? 1u : 0u; }
};
template <> struct Pack<4> {
    static __device__ __forceinline__ void load(const float* p, float* f)
    {
        const float4 v = __ldg(reinterpret_cast<const float4*>(p));
        f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
    }
    static __device__ __forceinline__ void store(float* p, const float* f) { *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]); }
    static __device__ __forceinline__ unsigned mask(const unsigned char* p)
    {
        const uchar4 v = __ldg(reinterpret_cast<const uchar4*>(p));
        return (v.x ? 1u : 0u) | (v.y ? 2u : 0u) | (v.z ? 4u : 0u) | (v.w ? 8u : 0u);
    }
};

// Sums over a thread's one or four tokens in fp32, joined in fp64: three roundings of four tokens' sum at most, where fp64
// from the tokens on was among what took 415 us.  The policy terms, which nearly cancel, carry their roundings along.
// Numbers of tokens are whole.
struct LossSums {
    float policy, policy_rest, kl, entropy, neg_d, excess;
};
// an infinite or NaN term has no rest
__device__ __forceinline__ double policy_sum(const LossSums& s)
{
    return static_cast<double>(s.policy) + (fabsf(s.policy) < CUDART_INF_F ? static_cast<double>(s.policy_rest) : 0.0);
}
struct LossTotals {
    double policy, kl, entropy, neg_d, excess;
    int clipped, tokens, rows;
};
// tokens i ... i + VEC - 1, advantages from a ...: reads, writes ratio and slope, adds to the sums
template <int VEC, bool ONE_ADVANTAGE>
__device__ __forceinline__ void add_tokens(const LossArgs& p, long long i, long long a, LossSums& sums, int& clipped, int& tokens)
{
    float lp[VEC], old[VEC], adv[VEC], ref[VEC], ent[VEC], ratio[VEC], slope[VEC];
    Pack<VEC>::load(p.logprobs + i, lp);
    Pack<VEC>::load(p.old_logprobs + i, old);
    if (ONE_ADVANTAGE) {
        adv[0] = __ldg(p.advantages + a);
#pragma unroll
        for (int v = 1; v < VEC; ++v) adv[v] = adv[0];
    } else {
        Pack<VEC>::load(p.advantages + a, adv);
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) ref[v] = ent[v] = 0.0f;
    if (p.ref_logprobs != nullptr) Pack<VEC>::load(p.ref_logprobs + i, ref);
    if (p.entropy != nullptr) Pack<VEC>::load(p.entropy + i, ent);
    const unsigned keep = p.mask != nullptr ? Pack<VEC>::mask(p.mask + i) : (1u << VEC) - 1u;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        ratio[v] = 1.0f;
        slope[v] = 0.0f;
        if (keep >> v & 1u) {
            const TokenLoss t = token_loss(p, lp[v], old[v], adv[v], ref[v]);
            ratio[v] = t.ratio;
            slope[v] = t.slope;
            const float sum = __fadd_rn(sums.policy, t.policy), back = __fsub_rn(sum, sums.policy);
            sums.policy_rest += t.policy_rest + (__fsub_rn(sums.policy, __fsub_rn(sum, back)) + __fsub_rn(t.policy, back));
            sums.policy = sum;
            sums.kl += t.kl;
            sums.entropy += ent[v];
            sums.neg_d -= t.d;
            sums.excess += t.excess;
            clipped += t.clipped ? 1 : 0;
            ++tokens;
        }
    }
    Pack<VEC>::store(p.ratio + i, ratio);
    if (p.slope != nullptr) Pack<VEC>::store(p.slope + i, slope);
}

// adds the sums of all threads of the CTA; thread 0 writes them
__device__ __forceinline__ void write_partial(const LossTotals& t, double* partial)
{
    double v[kLossSums] = {t.policy, t.kl, t.entropy, t.neg_d, t.excess, static_cast<double>(t.clipped),
                           static_cast<double>(t.tokens), static_cast<double>(t.rows)};
    __shared__ double s_part[32][kLossSums];
#pragma unroll
    for (int k = 0; k < kLossSums; ++k)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int k = 0; k < kLossSums; ++k) s_part[threadIdx.x >> 5][k] = v[k];
    __syncthreads();
    if (threadIdx.x < kLossSums) {
        double sum = 0.0;
        for (int w = 0; w < static_cast<int>(blockDim.x / 32); ++w) sum += s_part[w][threadIdx.x];
        partial[threadIdx.x * static_cast<long long>(gridDim.x) + blockIdx.x] = sum;
    }
}

// Means over tokens, an advantage each: rows do not matter.
template <int VEC>
__global__ void __launch_bounds__(kLossThreads, 4)
puff_policy_loss_kernel(LossArgs p, double* __restrict__ partial)
{
    LossTotals total = {};
    const long long units = p.rows * p.steps / VEC, stride = static_cast<long long>(gridDim.x) * kLossThreads;
    for (long long u = blockIdx.x * static_cast<long long>(kLossThreads) + threadIdx.x; u < units; u += stride) {
        LossSums sums = {};
        add_tokens<VEC, false>(p, u * VEC, u * VEC, sums, total.clipped, total.tokens);
        total.policy += policy_sum(sums);
        total.kl += sums.kl;
        total.entropy += sums.entropy;
        total.neg_d += sums.neg_d;
        total.excess += sums.excess;
    }
    write_partial(total, partial);
}

// Rows that matter: one advantage each, or SEQ, a mean each (131072 x 256 196 us, 16777216 x 1 202, 100 x 100001 144).
// TEAM threads a row, rows side by side in a warp where they are short, one a CTA (TEAM 256) where they are long and few.
// SEQ: a thread's share of the row's policy, kl and entropy sums is divided by the row's length.
template <int VEC, int TEAM, bool SEQ, bool ONE_ADVANTAGE>
__global__ void __launch_bounds__(TEAM > kLossThreads ? TEAM : kLossThreads, TEAM > kLossThreads ? 1 : 4)
puff_policy_loss_rows_kernel(LossArgs p, double* __restrict__ partial)
{
    constexpr int kThreads = TEAM > kLossThreads ? TEAM : kLossThreads;
    constexpr int kTeams = kThreads / TEAM;
    __shared__ int s_length[kThreads / 32];
    const int member = threadIdx.x % TEAM;
    LossTotals total = {};
    const long long units = p.steps / VEC, stride = static_cast<long long>(gridDim.x) * kTeams;
    const long long rounds = (p.rows + stride - 1) / stride;
    long long r = blockIdx.x * static_cast<long long>(kTeams) + threadIdx.x / TEAM;
    for (long long k = 0; k < rounds; ++k, r += stride) {      // all threads go round alike: they meet below
        double policy = 0.0, kl = 0.0, entropy = 0.0;      // of the row, for SEQ
        int length = 0;                                    // of this thread: at most steps / TEAM + VEC
        if (r < p.rows)
            for (long long u = member; u < units; u += TEAM) {
                LossSums sums = {};
                const long long i = r * p.steps + u * VEC;
                add_tokens<VEC, ONE_ADVANTAGE>(p, i, ONE_ADVANTAGE ? r : i, sums, total.clipped, length);
                policy += policy_sum(sums);
                kl += sums.kl;
                entropy += sums.entropy;
                total.neg_d += sums.neg_d;
                total.excess += sums.excess;
            }
        total.tokens += length;
        if (SEQ) {
            long long whole;
#pragma unroll
            for (int o = (TEAM < 32 ? TEAM : 32) / 2; o > 0; o >>= 1) length += __shfl_xor_sync(0xffffffffu, length, o);
            whole = length;
            if (TEAM > 32) {
                __syncthreads();
                if ((threadIdx.x & 31) == 0) s_length[threadIdx.x >> 5] = length;
                __syncthreads();
                whole = 0;
                for (int w = 0; w < kThreads / 32; ++w) whole += s_length[w];
            }
            const double scale = whole > 0 ? 1.0 / static_cast<double>(whole) : 0.0;
            policy *= scale;
            kl *= scale;
            entropy *= scale;
            if (member == 0 && r < p.rows) {
                total.rows += whole > 0 ? 1 : 0;
                if (p.row_scale != nullptr) p.row_scale[r] = static_cast<float>(scale);
            }
        }
        total.policy += policy;
        total.kl += kl;
        total.entropy += entropy;
    }
    write_partial(total, partial);
}

// The partial sums in index order -> loss, six statistics, and w (or, for sequences, w times the length)
__global__ void __launch_bounds__(256)
puff_policy_loss_final_kernel(const double* __restrict__ partial, int n_partial, int sequence, float kl_coef, float ent_coef,
                              double inv_denominator, float* __restrict__ loss, float* __restrict__ stats,
                              float* __restrict__ weight)
{
    __shared__ double s_sum[kLossSums];
    const int k = threadIdx.x >> 5, lane = threadIdx.x & 31;   // one warp per sum
    pdl_wait();
    double t = 0.0;
#pragma unroll 4
    for (int i = lane; i < n_partial; i += 32) t += partial[k * n_partial + i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (lane == 0) s_sum[k] = t;
    __syncthreads();
    if (threadIdx.x == 0) {
        const double tokens = s_sum[6];
        const double per_token = tokens > 0.0 ? 1.0 / tokens : 0.0;
        double w = inv_denominator;
        if (w == 0.0) w = sequence ? (s_sum[7] > 0.0 ? 1.0 / s_sum[7] : 0.0) : per_token;
        const double policy = s_sum[0] * w, kl = s_sum[1] * w, ent = s_sum[2] * w;
        loss[0] = static_cast<float>(policy + kl_coef * kl - ent_coef * ent);
        stats[0] = static_cast<float>(policy);
        stats[1] = static_cast<float>(kl);
        stats[2] = static_cast<float>(ent);
        stats[3] = static_cast<float>(s_sum[3] * per_token);
        stats[4] = static_cast<float>(s_sum[4] * per_token);
        stats[5] = static_cast<float>(s_sum[5] * per_token);
        if (weight != nullptr) weight[0] = static_cast<float>(w);
    }
}

// slope times weight, dloss and, for sequences, the row's scale: two or three fp32 products of factors rounded once each.
// VEC 4 with row_scale: four adjacent tokens are of one row (steps divisible by four)
template <int VEC>
__global__ void __launch_bounds__(kLossThreads)
puff_policy_loss_backward_kernel(const float* __restrict__ slope, const float* __restrict__ row_scale,
                                 const float* __restrict__ weight, const float* __restrict__ dloss,
                                 const unsigned char* __restrict__ mask, float ent_coef, float* __restrict__ dlogprobs,
                                 float* __restrict__ dentropy, long long rows, long long steps)
{
    const float w = weight[0] * dloss[0];
    const long long units = rows * steps / VEC, stride = static_cast<long long>(gridDim.x) * kLossThreads;
    for (long long u = blockIdx.x * static_cast<long long>(kLossThreads) + threadIdx.x; u < units; u += stride) {
        const long long i = u * VEC;
        float s[VEC], g[VEC], h[VEC];
        if (dlogprobs != nullptr) Pack<VEC>::load(slope + i, s);
        const unsigned keep = mask != nullptr ? Pack<VEC>::mask(mask + i) : (1u << VEC) - 1u;
        float wi = w;
        if (row_scale != nullptr)
            wi *= __ldg(row_scale + (((i | steps) >> 32) == 0 ? static_cast<unsigned>(i) / static_cast<unsigned>(steps) : i / steps));
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const bool k = keep >> v & 1u;
            g[v] = k ? s[v] * wi : 0.0f;
            h[v] = k ? -ent_coef * wi : 0.0f;
        }
        if (dlogprobs != nullptr) Pack<VEC>::store(dlogprobs + i, g);
        if (dentropy != nullptr) Pack<VEC>::store(dentropy + i, h);
    }
}

static int capped(long long blocks, int most) { return static_cast<int>(blocks < 1 ? 1 : blocks > most ? most : blocks); }

template <int VEC, int TEAM, bool SEQ>
static int launch_rows(const LossArgs& p, bool one_advantage, double* partial, cudaStream_t st)
{
    constexpr int threads = TEAM > kLossThreads ? TEAM : kLossThreads;
    const int blocks = capped((p.rows + threads / TEAM - 1) / (threads / TEAM), kLossMaxBlocks);
    if (one_advantage) puff_policy_loss_rows_kernel<VEC, TEAM, SEQ, true><<<blocks, threads, 0, st>>>(p, partial);
    else puff_policy_loss_rows_kernel<VEC, TEAM, SEQ, false><<<blocks, threads, 0, st>>>(p, partial);
    return blocks;
}
template <int VEC, bool SEQ>
static int launch_rows(const LossArgs& p, bool one_advantage, double* partial, cudaStream_t st)
{
    // as many threads a row as it has units to read, up to a warp; a CTA where a warp a row would leave SMs idle, and a
    // large one where even a CTA a row would (100 rows of 100001: 256 threads 473 us)
    const long long units = p.steps / VEC;
    if (units >= 2048 && p.rows < 148 * 2) return launch_rows<VEC, 1024, SEQ>(p, one_advantage, partial, st);
    if (units >= 256 && p.rows < 148 * kLossWarps) return launch_rows<VEC, 256, SEQ>(p, one_advantage, partial, st);
    if (units >= 32) return launch_rows<VEC, 32, SEQ>(p, one_advantage, partial, st);
    if (units >= 8) return launch_rows<VEC, 8, SEQ>(p, one_advantage, partial, st);
    if (units >= 2) return launch_rows<VEC, 2, SEQ>(p, one_advantage, partial, st);
    return launch_rows<VEC, 1, SEQ>(p, one_advantage, partial, st);
}
// the number of partial sums written
static int launch_loss(const LossArgs& p, bool sequence, bool one_advantage, bool vec, double* partial, cudaStream_t st)
{
    if (sequence) return vec ? launch_rows<4, true>(p, one_advantage, partial, st) : launch_rows<1, true>(p, one_advantage, partial, st);
    if (one_advantage && p.rows > 0) return vec ? launch_rows<4, false>(p, true, partial, st) : launch_rows<1, false>(p, true, partial, st);
    const int blocks = capped((p.rows * p.steps / (vec ? 4 : 1) + kLossThreads - 1) / kLossThreads, kLossMaxBlocks);
    if (vec) puff_policy_loss_kernel<4><<<blocks, kLossThreads, 0, st>>>(p, partial);
    else puff_policy_loss_kernel<1><<<blocks, kLossThreads, 0, st>>>(p, partial);
    return blocks;
}
}  // namespace puff

using namespace puff;

extern "C" size_t puff_policy_sm100_loss_scratch_bytes(long long rows, long long steps)
{
    if (rows <= 0 || steps <= 0) return kLossSums * sizeof(double);
    return static_cast<size_t>(kLossMaxBlocks) * kLossSums * sizeof(double);
}

extern "C" int puff_policy_sm100_loss(const float* logprobs, const float* old_logprobs, const float* advantages,
                                      int advantage_per_row, const float* ref_logprobs, const float* entropy,
                                      const unsigned char* mask, double clip_low, double clip_high, float kl_coef,
                                      float ent_coef, int reduction, double denominator, long long rows, long long steps,
                                      float* loss, float* ratio, float* stats, float* slope, float* row_scale,
                                      float* weight, void* scratch, size_t scratch_bytes, void* cuda_stream)
{
    if (rows < 0 || steps < 0) return PUFF_ERR_SHAPE;
    if (rows > 0 && steps > (1LL << 40) / rows) return PUFF_ERR_SIZE;
    if (!(clip_low >= 0.0) || !(clip_high >= 0.0) || !(denominator >= 0.0) || denominator > 1e300 ||
        (reduction != PUFF_MEAN_TOKENS && reduction != PUFF_MEAN_SEQUENCES))
        return PUFF_ERR_VALUE;
    const long long n = rows * steps;
    if (loss == nullptr || stats == nullptr) return PUFF_ERR_NULL;
    if (n > 0 && (logprobs == nullptr || old_logprobs == nullptr || advantages == nullptr || ratio == nullptr)) return PUFF_ERR_NULL;
    if (n > 0 && slope != nullptr && reduction == PUFF_MEAN_SEQUENCES && row_scale == nullptr) return PUFF_ERR_NULL;
    if (slope != nullptr && weight == nullptr) return PUFF_ERR_NULL;
    if (scratch == nullptr || misaligned(scratch, 8) || scratch_bytes < puff_policy_sm100_loss_scratch_bytes(rows, steps))
        return PUFF_ERR_WORKSPACE;
    const long long nadv = advantage_per_row ? rows : n;
    const void* in[6] = {logprobs, old_logprobs, advantages, ref_logprobs, entropy, mask};
    const long long in_bytes[6] = {4 * n, 4 * n, 4 * nadv, 4 * n, 4 * n, n};
    const void* out[7] = {loss, ratio, stats, slope, row_scale, weight, scratch};
    const long long out_bytes[7] = {4, 4 * n, 24, 4 * n, 4 * rows, 4, static_cast<long long>(scratch_bytes)};
    for (int i = 0; i < 5; ++i)
        if (misaligned(in[i], 4)) return PUFF_ERR_ALIGN;
    for (int i = 0; i < 7; ++i) {
        if (misaligned(out[i], 4)) return PUFF_ERR_ALIGN;
        for (int j = 0; j < 6; ++j)
            if (spans_overlap(out[i], out_bytes[i], in[j], in_bytes[j])) return PUFF_ERR_ALIAS;
        for (int j = 0; j < i; ++j)
            if (spans_overlap(out[i], out_bytes[i], out[j], out_bytes[j])) return PUFF_ERR_ALIAS;
    }
    int sms = 0;
    const int rc = require_sm100(&sms);
    if (rc != PUFF_OK) return rc;
    LossArgs p = {};
    p.logprobs = logprobs;
    p.old_logprobs = old_logprobs;
    p.advantages = advantages;
    p.ref_logprobs = ref_logprobs;
    p.entropy = entropy;
    p.mask = mask;
    p.ratio = ratio;
    p.slope = slope;
    p.row_scale = row_scale;
    p.rows = n > 0 ? rows : 0;
    p.steps = steps;
    p.clip_low_value = static_cast<float>(1.0 - clip_low);
    p.clip_low_rest = static_cast<float>((1.0 - clip_low) - p.clip_low_value);
    p.clip_high_value = static_cast<float>(1.0 + clip_high);
    p.clip_high_rest = clip_high < 1e30 ? static_cast<float>((1.0 + clip_high) - p.clip_high_value) : 0.0f;
    const double low = clip_low < 1.0 ? log1p(-clip_low) : -HUGE_VAL, high = log1p(clip_high);
    p.log_low = static_cast<float>(low);
    p.log_low_rest = clip_low < 1.0 ? static_cast<float>(low - p.log_low) : 0.0f;
    p.log_high = static_cast<float>(high);
    p.log_high_rest = high < HUGE_VAL ? static_cast<float>(high - p.log_high) : 0.0f;
    p.kl_coef = kl_coef;
    cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    // four tokens at a time where every array is aligned for it (and, where rows matter, so are they)
    const bool rows_matter = reduction == PUFF_MEAN_SEQUENCES || advantage_per_row;
    bool vec = (rows_matter ? steps : n) % 4 == 0 && !misaligned(mask, 4);
    for (int i = 0; i < 5; ++i) vec = vec && ((i == 2 && advantage_per_row) || !misaligned(in[i], 16));
    vec = vec && !misaligned(ratio, 16) && !misaligned(slope, 16);
    double* partial = static_cast<double*>(scratch);
    const int blocks = launch_loss(p, reduction == PUFF_MEAN_SEQUENCES, advantage_per_row != 0, vec, partial, st);
    count_launch();
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return static_cast<int>(e);
    e = launch_neighbour(puff_policy_loss_final_kernel, 1, 256, 0, st, partial, blocks,
                         reduction == PUFF_MEAN_SEQUENCES ? 1 : 0, kl_coef, ent_coef,
                         denominator > 0.0 ? 1.0 / denominator : 0.0, loss, stats, weight);
    count_launch();
    return static_cast<int>(e);
}

extern "C" int puff_policy_sm100_loss_backward(const float* slope, const float* row_scale, const float* weight,
                                               const float* dloss, const unsigned char* mask, float ent_coef,
                                               long long rows, long long steps, float* dlogprobs, float* dentropy,
                                               void* cuda_stream)
{
    if (rows < 0 || steps < 0) return PUFF_ERR_SHAPE;
    if (rows > 0 && steps > (1LL << 40) / rows) return PUFF_ERR_SIZE;
    const long long n = rows * steps;
    if (n == 0 || (dlogprobs == nullptr && dentropy == nullptr)) return PUFF_OK;
    if (slope == nullptr || weight == nullptr || dloss == nullptr) return PUFF_ERR_NULL;
    const void* in[5] = {slope, row_scale, weight, dloss, mask};
    const long long in_bytes[5] = {4 * n, 4 * rows, 4, 4, n};
    for (int i = 0; i < 4; ++i)
        if (misaligned(in[i], 4)) return PUFF_ERR_ALIGN;
    if (misaligned(dlogprobs, 4) || misaligned(dentropy, 4)) return PUFF_ERR_ALIGN;
    for (int j = 0; j < 5; ++j)
        if (spans_overlap(dlogprobs, 4 * n, in[j], in_bytes[j]) || spans_overlap(dentropy, 4 * n, in[j], in_bytes[j]))
            return PUFF_ERR_ALIAS;
    if (spans_overlap(dlogprobs, 4 * n, dentropy, 4 * n)) return PUFF_ERR_ALIAS;
    int sms = 0;
    const int rc = require_sm100(&sms);
    if (rc != PUFF_OK) return rc;
    const bool vec = (row_scale != nullptr ? steps : n) % 4 == 0 && !misaligned(mask, 4) && !misaligned(slope, 16) &&
                     !misaligned(dlogprobs, 16) && !misaligned(dentropy, 16);
    cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    const int blocks = capped((n / (vec ? 4 : 1) + kLossThreads - 1) / kLossThreads, 8 * sms);
    if (vec)
        puff_policy_loss_backward_kernel<4><<<blocks, kLossThreads, 0, st>>>(slope, row_scale, weight, dloss, mask, ent_coef,
                                                                             dlogprobs, dentropy, rows, steps);
    else
        puff_policy_loss_backward_kernel<1><<<blocks, kLossThreads, 0, st>>>(slope, row_scale, weight, dloss, mask, ent_coef,
                                                                             dlogprobs, dentropy, rows, steps);
    count_launch();
    return static_cast<int>(cudaGetLastError());
}
