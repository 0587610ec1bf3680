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
// the backward pass multiplies by it.  Which side of a clip border a ratio is on is decided in 64 bits, as
// logprob - old_logprob against log(1 - clip_low) and log(1 + clip_high).
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/puff_advantage.h"
#include "puff_policy.cuh"

namespace puff {

constexpr int kLossThreads = 256;
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
    int per_row;   // one advantage per row
    float clip_low_value, clip_high_value;
    double log_low, log_high;
    float kl_coef;
};

// e^x - 1 - x.  For |x| < 1 by its Taylor series x^2 (1/2! + x/3! + ...), the difference would cancel there;
// em1 receives e^x - 1.
__device__ __forceinline__ float exp_excess(float x, float ex, float* em1)
{
    if (fabsf(x) < 1.0f) {
        float p = 1.0f / 6227020800.0f;              // 1/13!
        p = fmaf(p, x, 1.0f / 479001600.0f);
        p = fmaf(p, x, 1.0f / 39916800.0f);
        p = fmaf(p, x, 1.0f / 3628800.0f);
        p = fmaf(p, x, 1.0f / 362880.0f);
        p = fmaf(p, x, 1.0f / 40320.0f);
        p = fmaf(p, x, 1.0f / 5040.0f);
        p = fmaf(p, x, 1.0f / 720.0f);
        p = fmaf(p, x, 1.0f / 120.0f);
        p = fmaf(p, x, 1.0f / 24.0f);
        p = fmaf(p, x, 1.0f / 6.0f);
        p = fmaf(p, x, 0.5f);
        const float k = x * x * p;
        *em1 = x + k;
        return k;
    }
    *em1 = ex - 1.0f;
    return *em1 - x;
}

// e^(a - b) with the difference's rounding carried along; *diff64 and *diff receive a - b
__device__ __forceinline__ float exp_of_difference(float a, float b, double* diff64, float* diff)
{
    const double d = static_cast<double>(a) - static_cast<double>(b);
    const float hi = static_cast<float>(d);
    const float e = expf(hi);
    *diff64 = d;
    *diff = hi;
    return fabsf(hi) < 80.0f ? fmaf(e, static_cast<float>(d - hi), e) : e;
}

struct TokenLoss {
    float policy, kl, neg_d, excess, clipped, ratio, slope;
};
__device__ __forceinline__ TokenLoss token_loss(const LossArgs& p, float lp, float old, float adv, float ref)
{
    TokenLoss t;
    double d64;
    float d, em1;
    t.ratio = exp_of_difference(lp, old, &d64, &d);
    const bool above = d64 > p.log_high, below = d64 < p.log_low;
    const bool cut = (above && adv > 0.0f) || (below && adv < 0.0f);
    t.policy = -adv * (cut ? (above ? p.clip_high_value : p.clip_low_value) : t.ratio);
    t.slope = cut ? 0.0f : t.policy;
    t.neg_d = -d;
    t.excess = exp_excess(d, t.ratio, &em1);
    t.clipped = above || below ? 1.0f : 0.0f;
    t.kl = 0.0f;
    if (p.ref_logprobs != nullptr) {
        double q64;
        float q;
        const float eq = exp_of_difference(ref, lp, &q64, &q);
        t.kl = exp_excess(q, eq, &em1);
        t.slope = fmaf(-p.kl_coef, em1, t.slope);
    }
    return t;
}

// adds the sums of all threads of the CTA; thread 0 writes them
__device__ __forceinline__ void write_partial(double (&v)[kLossSums], double* partial)
{
    __shared__ double s_part[kLossThreads / 32][kLossSums];
#pragma unroll
    for (int k = 0; k < kLossSums; ++k)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int k = 0; k < kLossSums; ++k) s_part[threadIdx.x >> 5][k] = v[k];
    __syncthreads();
    if (threadIdx.x < kLossSums) {
        double t = 0.0;
        for (int w = 0; w < kLossThreads / 32; ++w) t += s_part[w][threadIdx.x];
        partial[blockIdx.x * kLossSums + threadIdx.x] = t;
    }
}

// One warp per row.  SEQ: the row's policy, kl and entropy sums are divided by its length.
template <bool SEQ>
__global__ void __launch_bounds__(kLossThreads)
puff_policy_loss_rows_kernel(LossArgs p, double* __restrict__ partial)
{
    const int lane = threadIdx.x & 31;
    const long long stride = static_cast<long long>(gridDim.x) * (kLossThreads / 32);
    double total[kLossSums] = {};
    for (long long r = blockIdx.x * static_cast<long long>(kLossThreads / 32) + (threadIdx.x >> 5); r < p.rows; r += stride) {
        double v[kLossSums] = {};
        for (long long c = lane; c < p.steps; c += 32) {
            const long long i = r * p.steps + c;
            const bool keep = p.mask == nullptr || p.mask[i] != 0;
            float ratio = 1.0f, slope = 0.0f;
            if (keep) {
                const TokenLoss t = token_loss(p, p.logprobs[i], p.old_logprobs[i], p.advantages[p.per_row ? r : i],
                                               p.ref_logprobs != nullptr ? p.ref_logprobs[i] : 0.0f);
                ratio = t.ratio;
                slope = t.slope;
                v[0] += t.policy;
                v[1] += t.kl;
                if (p.entropy != nullptr) v[2] += p.entropy[i];
                v[3] += t.neg_d;
                v[4] += t.excess;
                v[5] += t.clipped;
                v[6] += 1.0;
            }
            p.ratio[i] = ratio;
            if (p.slope != nullptr) p.slope[i] = slope;
        }
        if (SEQ) {
            double length = v[6];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) length += __shfl_xor_sync(0xffffffffu, length, o);
            const double scale = length > 0.0 ? 1.0 / length : 0.0;
            v[0] *= scale;
            v[1] *= scale;
            v[2] *= scale;
            if (lane == 0) {
                v[7] = length > 0.0 ? 1.0 : 0.0;
                if (p.row_scale != nullptr) p.row_scale[r] = static_cast<float>(scale);
            }
        }
#pragma unroll
        for (int k = 0; k < kLossSums; ++k) total[k] += v[k];
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
    for (int i = lane; i < n_partial; i += 32) t += partial[i * kLossSums + k];
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

__global__ void __launch_bounds__(kLossThreads)
puff_policy_loss_backward_kernel(const float* __restrict__ slope, const float* __restrict__ row_scale,
                                 const float* __restrict__ weight, const float* __restrict__ dloss,
                                 const unsigned char* __restrict__ mask, float ent_coef, float* __restrict__ dlogprobs,
                                 float* __restrict__ dentropy, long long rows, long long steps)
{
    const float w = weight[0] * dloss[0];
    const long long n = rows * steps, stride = static_cast<long long>(gridDim.x) * kLossThreads;
    for (long long i = blockIdx.x * static_cast<long long>(kLossThreads) + threadIdx.x; i < n; i += stride) {
        const bool keep = mask == nullptr || mask[i] != 0;
        const float wi = row_scale != nullptr ? w * row_scale[i / steps] : w;
        if (dlogprobs != nullptr) dlogprobs[i] = keep ? slope[i] * wi : 0.0f;
        if (dentropy != nullptr) dentropy[i] = keep ? -ent_coef * wi : 0.0f;
    }
}

static int loss_blocks(long long rows, long long)
{
    long long b = (rows + kLossThreads / 32 - 1) / (kLossThreads / 32);
    return static_cast<int>(b < 1 ? 1 : b > kLossMaxBlocks ? kLossMaxBlocks : b);
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
    p.per_row = advantage_per_row != 0;
    p.clip_low_value = static_cast<float>(1.0 - clip_low);
    p.clip_high_value = static_cast<float>(1.0 + clip_high);
    p.log_low = clip_low < 1.0 ? log1p(-clip_low) : -HUGE_VAL;
    p.log_high = log1p(clip_high);
    p.kl_coef = kl_coef;
    cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    const int blocks = loss_blocks(rows, steps);
    double* partial = static_cast<double*>(scratch);
    if (reduction == PUFF_MEAN_SEQUENCES)
        puff_policy_loss_rows_kernel<true><<<blocks, kLossThreads, 0, st>>>(p, partial);
    else
        puff_policy_loss_rows_kernel<false><<<blocks, kLossThreads, 0, st>>>(p, partial);
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
    long long blocks = (n + kLossThreads - 1) / kLossThreads;
    if (blocks > 8LL * sms) blocks = 8LL * sms;
    puff_policy_loss_backward_kernel<<<static_cast<int>(blocks), kLossThreads, 0, static_cast<cudaStream_t>(cuda_stream)>>>(
        slope, row_scale, weight, dloss, mask, ent_coef, dlogprobs, dentropy, rows, steps);
    count_launch();
    return static_cast<int>(cudaGetLastError());
}
