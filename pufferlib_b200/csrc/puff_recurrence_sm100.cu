// Gated linear recurrence along the horizon, forward, backward and one step at a time (sm_100a).
//
//     f_t = sigmoid(gates_t),   a_t = f_t unless resets_t, else 0
//     h_t = a_t h_{t-1} + (1 - f_t) x_t                                                   per channel
//     lam_t = dh_t + a_{t+1} lam_{t+1},   dx_t = lam_t (1 - f_t)
//     dgate_t = lam_t f_t (1 - f_t) ([not reset_t] h_{t-1} - x_t),   dh_before = a_0 lam_0
//
// The recurrent layer of a policy over the experience buffers' [segments, horizon] rows, cut where an episode ends
// (`terminals`, pufferl.py:295) as the recurrent state of pufferl.py:112-117 is; the same first-order linear
// recurrence as the advantages, with gates for discounts.  The state is carried in fp32 whatever the tensors' type.
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/puff_advantage.h"
#include "puff_policy.cuh"

namespace puff {

constexpr int kRecTile = 16;       // steps whose inputs a warp holds in registers; also the distance of the saved states
constexpr int kRecWarps = 8;       // warps of a CTA
constexpr int kRecThreads = 32 * kRecWarps;

struct RecArgs {
    const void* gates;
    const void* inputs;
    const void* resets;      // [batch, steps] fp32 (reset_bytes 4) or one byte each (1); null: none
    const float* state;      // [batch, channels]; null: zeros
    long long batch, steps, channels;
    long long gates_batch_stride, gates_step_stride, inputs_batch_stride, inputs_step_stride;
    int reset_bytes;
};

// How the work is cut.  A warp owns 32 lanes of VEC channels and walks 16 steps at a time, all of them in registers.
// `warps` warps of a CTA take consecutive 16-step tiles of the same lanes, and `splits` ranges of `split_steps` steps
// go to different CTAs where lanes are few.  A tile (or range) maps the state before it to the state after it as
// h -> A h + B; those pairs are joined over the warps through shared memory, and over the ranges through global memory
// by a first launch that computes nothing else.
struct RecPlan {
    int warps, splits;
    long long split_steps, lane_blocks, blocks_per_row;
};

__device__ __forceinline__ bool is_reset(const RecArgs& p, long long i)
{
    if (p.reset_bytes == 4) return static_cast<const float*>(p.resets)[i] != 0.0f;
    return p.reset_bytes == 1 && static_cast<const unsigned char*>(p.resets)[i] != 0;
}

// keep = sigmoid(g) and take = 1 - keep = sigmoid(-g).  The smaller of the two is e / (1 + e) with e = e^-|g|, good to
// a few ulp however small; the larger is 1 minus it, so that the two add up to 1 and the state stays a weighted mean.
// One register holds both: the smaller one, with the sign of g.
__device__ __forceinline__ float gate_code(float g)
{
    const float e = exp2_approx(-fabsf(g) * kLog2e);
    return copysignf(__fdividef(e, 1.0f + e), g);
}
__device__ __forceinline__ void gate_pair(float code, float& keep, float& take)
{
    const float small = fabsf(code), large = 1.0f - small;
    const bool negative = __float_as_int(code) < 0;
    keep = negative ? small : large;
    take = negative ? large : small;
}
constexpr float kHold = 0.0f;      // the code of a gate that holds the state: steps past the end

// h -> A h + B over a span; A < 0: the span holds a reset, h does not matter
__device__ __forceinline__ float apply_pair(float2 ab, float h) { return ab.x < 0.0f ? ab.y : fmaf(ab.x, h, ab.y); }

// VEC adjacent elements (4 bytes, or one element of 2) in a register
template <typename T, int VEC> struct Lane;
template <> struct Lane<float, 1> {
    using Raw = float;
    static __device__ __forceinline__ void get(Raw r, float* f) { f[0] = r; }
    static __device__ __forceinline__ Raw put(const float* f) { return f[0]; }
};
template <typename T> struct Lane<T, 1> {
    using Raw = T;
    static __device__ __forceinline__ void get(Raw r, float* f) { f[0] = to_f32(r); }
    static __device__ __forceinline__ Raw put(const float* f) { return from_f32<T>(f[0]); }
};
template <> struct Lane<__half, 2> {
    using Raw = __half2;
    static __device__ __forceinline__ void get(Raw r, float* f)
    {
        const float2 p = __half22float2(r);
        f[0] = p.x;
        f[1] = p.y;
    }
    static __device__ __forceinline__ Raw put(const float* f) { return __floats2half2_rn(f[0], f[1]); }
};
template <> struct Lane<__nv_bfloat16, 2> {
    using Raw = __nv_bfloat162;
    static __device__ __forceinline__ void get(Raw r, float* f)
    {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(&r);
        f[0] = __uint_as_float(w << 16);
        f[1] = __uint_as_float(w & 0xffff0000u);
    }
    static __device__ __forceinline__ Raw put(const float* f) { return __floats2bfloat162_rn(f[0], f[1]); }
};
template <typename Raw> __device__ __forceinline__ Raw zero_raw() { return Raw(); }
template <> __device__ __forceinline__ float zero_raw<float>() { return 0.0f; }
template <> __device__ __forceinline__ __half zero_raw<__half>() { return __float2half_rn(0.0f); }
template <> __device__ __forceinline__ __nv_bfloat16 zero_raw<__nv_bfloat16>() { return __float2bfloat16_rn(0.0f); }
template <> __device__ __forceinline__ __half2 zero_raw<__half2>() { return __float2half2_rn(0.0f); }
template <> __device__ __forceinline__ __nv_bfloat162 zero_raw<__nv_bfloat162>() { return __float2bfloat162_rn(0.0f); }

// Where this thread's warp stands in the plan.  FLAT: the lanes of a warp are adjacent (batch, channel) pairs of any
// rows, for channels too few to fill a warp; otherwise they are adjacent channels of one row.
struct RecPlace {
    int group, w, lane;
    bool unit, ok;             // the group has work; this lane has a channel
    int split;
    long long b, c, index;     // index: b * channels + c
    long long t_begin, t_end;
};
template <int VEC, bool FLAT>
__device__ __forceinline__ RecPlace rec_place(const RecArgs& p, const RecPlan& plan)
{
    RecPlace q;
    const int warp = threadIdx.x >> 5;
    q.lane = threadIdx.x & 31;
    q.group = warp / plan.warps;
    q.w = warp - q.group * plan.warps;
    const long long unit = blockIdx.x * static_cast<long long>(kRecWarps / plan.warps) + q.group;
    const long long block = unit % plan.lane_blocks;
    q.split = static_cast<int>(unit / plan.lane_blocks);
    q.unit = q.split < plan.splits;
    if (FLAT) {
        q.index = block * 32 + q.lane;
        q.ok = q.index < p.batch * p.channels;
        q.b = q.ok ? q.index / p.channels : 0;
        q.c = q.ok ? q.index - q.b * p.channels : 0;
    } else {
        q.b = block / plan.blocks_per_row;
        q.c = (block - q.b * plan.blocks_per_row) * (32 * VEC) + q.lane * VEC;
        q.ok = q.c < p.channels;
        q.index = q.b * p.channels + q.c;
    }
    q.ok = q.ok && q.unit;
    q.t_begin = q.split * plan.split_steps;
    q.t_end = q.t_begin + plan.split_steps < p.steps ? q.t_begin + plan.split_steps : p.steps;
    return q;
}
// bit j: step t0 + j is a reset.  All lanes of a row share the mask; FLAT lanes have one each.
template <bool FLAT>
__device__ __forceinline__ unsigned reset_mask(const RecArgs& p, const RecPlace& q, long long t0, int n)
{
    if (p.reset_bytes == 0) return 0u;
    const long long at = q.b * p.steps + t0;
    if (!FLAT) return __ballot_sync(0xffffffffu, q.lane < n && is_reset(p, at + q.lane));
    unsigned m = 0;
    if (q.ok)
        for (int j = 0; j < n; ++j) m |= is_reset(p, at + j) ? 1u << j : 0u;
    return m;
}
template <typename Raw, int VEC>
__device__ __forceinline__ void load_tile(Raw* raw, const void* base, long long at, long long step_stride, int n, bool ok)
{
    constexpr long long size = sizeof(Raw) / VEC;
    const char* ptr = static_cast<const char*>(base) + at * size;
#pragma unroll
    for (int j = 0; j < kRecTile; ++j) {
        raw[j] = zero_raw<Raw>();
        if (ok && j < n) raw[j] = __ldg(reinterpret_cast<const Raw*>(ptr));
        ptr += step_stride * size;
    }
}
__device__ __forceinline__ void group_barrier(int group, int warps)
{
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(warps * 32) : "memory");
}

// Forward.  SUMMARY: only the pairs of the ranges.  saved (nullable): the state before steps 0, 16, 32, ... as
// [batch, ceil(steps / 16), channels].
template <typename T, int VEC, bool FLAT, bool SUMMARY>
__global__ void __launch_bounds__(kRecThreads, 2)
puff_recurrence_kernel(RecArgs p, RecPlan plan, float2* pairs, T* __restrict__ outputs, float* __restrict__ final_state,
                       float* __restrict__ saved)
{
    using L = Lane<T, VEC>;
    using Raw = typename L::Raw;
    __shared__ float2 s_pair[2][kRecWarps][VEC][32];
    if (!SUMMARY) pdl_wait();
    const RecPlace q = rec_place<VEC, FLAT>(p, plan);
    if (!q.unit) return;
    const long long lanes = p.batch * p.channels;
    const long long tiles = (p.steps + kRecTile - 1) / kRecTile;
    float carry[VEC], sum_a[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        carry[v] = !SUMMARY && q.ok && p.state != nullptr ? p.state[q.index + v] : 0.0f;
        sum_a[v] = 1.0f;
    }
    if (!SUMMARY)
        for (int r = 0; r < q.split; ++r)
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                if (q.ok) carry[v] = apply_pair(pairs[r * lanes + q.index + v], carry[v]);
    int parity = 0;
    for (long long t = q.t_begin; t < q.t_end; t += kRecTile * plan.warps, parity ^= 1) {
        const long long t0 = t + q.w * kRecTile;
        const int n = static_cast<int>(q.t_end - t0 < 0 ? 0 : q.t_end - t0 < kRecTile ? q.t_end - t0 : kRecTile);
        Raw raw_g[kRecTile], raw_x[kRecTile];
        load_tile<Raw, VEC>(raw_g, p.gates, q.b * p.gates_batch_stride + t0 * p.gates_step_stride + q.c, p.gates_step_stride, n, q.ok);
        load_tile<Raw, VEC>(raw_x, p.inputs, q.b * p.inputs_batch_stride + t0 * p.inputs_step_stride + q.c, p.inputs_step_stride, n, q.ok);
        const unsigned cut = reset_mask<FLAT>(p, q, t0, n);
        float keep[kRecTile][VEC], fresh[kRecTile][VEC];
#pragma unroll
        for (int j = 0; j < kRecTile; ++j) {
            float g[VEC], x[VEC];
            L::get(raw_g[j], g);
            L::get(raw_x[j], x);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float take;
                gate_pair(j < n ? gate_code(g[v]) : kHold, keep[j][v], take);
                fresh[j][v] = take * x[v];
            }
        }
        float h[VEC];
        if (plan.warps > 1 || SUMMARY) {
            float a[VEC], b[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                a[v] = 1.0f;
                b[v] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < kRecTile; ++j)
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    b[v] = (cut >> j) & 1u ? fresh[j][v] : fmaf(keep[j][v], b[v], fresh[j][v]);
                    a[v] *= keep[j][v];
                }
#pragma unroll
            for (int v = 0; v < VEC; ++v) s_pair[parity][threadIdx.x >> 5][v][q.lane] = make_float2(cut != 0 ? -1.0f : a[v], b[v]);
            group_barrier(q.group, plan.warps);
#pragma unroll
            for (int v = 0; v < VEC; ++v) h[v] = carry[v];
            for (int w = 0; w < plan.warps; ++w)
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const float2 ab = s_pair[parity][q.group * plan.warps + w][v][q.lane];
                    if (w == q.w) h[v] = carry[v];
                    if (SUMMARY) sum_a[v] = ab.x < 0.0f || sum_a[v] < 0.0f ? -1.0f : sum_a[v] * ab.x;
                    carry[v] = apply_pair(ab, carry[v]);
                }
        } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) h[v] = carry[v];
        }
        if (!SUMMARY) {
            if (saved != nullptr && q.ok && n > 0)
#pragma unroll
                for (int v = 0; v < VEC; ++v) saved[(q.b * tiles + t0 / kRecTile) * p.channels + q.c + v] = h[v];
            T* out = outputs + (q.b * p.steps + t0) * p.channels + q.c;
#pragma unroll
            for (int j = 0; j < kRecTile; ++j) {
#pragma unroll
                for (int v = 0; v < VEC; ++v) h[v] = (cut >> j) & 1u ? fresh[j][v] : fmaf(keep[j][v], h[v], fresh[j][v]);
                if (q.ok && j < n) *reinterpret_cast<Raw*>(out) = L::put(h);
                out += p.channels;
            }
            if (plan.warps == 1)
#pragma unroll
                for (int v = 0; v < VEC; ++v) carry[v] = h[v];
        }
    }
    if (q.ok && q.w == 0) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            if (SUMMARY) pairs[q.split * lanes + q.index + v] = make_float2(sum_a[v], carry[v]);
            else if (q.split == plan.splits - 1) final_state[q.index + v] = carry[v];
        }
    }
}

// Backward, last tile first.  The states within a tile are computed again from the saved one before it; the pairs map
// lam after a tile (dh of the next steps times their gains) to lam before it.
template <typename T, int VEC, bool FLAT, bool SUMMARY>
__global__ void __launch_bounds__(kRecThreads, 2)
puff_recurrence_backward_kernel(RecArgs p, RecPlan plan, float2* pairs, const float* __restrict__ saved,
                                const T* __restrict__ doutputs, const float* __restrict__ dfinal, T* __restrict__ dgates,
                                T* __restrict__ dinputs, float* __restrict__ dstate)
{
    using L = Lane<T, VEC>;
    using Raw = typename L::Raw;
    __shared__ float2 s_pair[2][kRecWarps][VEC][32];
    if (!SUMMARY) pdl_wait();
    const RecPlace q = rec_place<VEC, FLAT>(p, plan);
    if (!q.unit) return;
    const long long lanes = p.batch * p.channels;
    const long long tiles = (p.steps + kRecTile - 1) / kRecTile;
    float carry[VEC], sum_a[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        carry[v] = !SUMMARY && q.ok && dfinal != nullptr ? dfinal[q.index + v] : 0.0f;
        sum_a[v] = 1.0f;
    }
    if (!SUMMARY)
        for (int r = plan.splits - 1; r > q.split; --r)
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                if (q.ok) carry[v] = apply_pair(pairs[r * lanes + q.index + v], carry[v]);
    const long long span = kRecTile * plan.warps;
    int parity = 0;
    for (long long t = q.t_begin + (q.t_end - q.t_begin - 1) / span * span; t >= q.t_begin; t -= span, parity ^= 1) {
        const long long t0 = t + q.w * kRecTile;
        const int n = static_cast<int>(q.t_end - t0 < 0 ? 0 : q.t_end - t0 < kRecTile ? q.t_end - t0 : kRecTile);
        const long long at = (q.b * p.steps + t0) * p.channels + q.c;
        Raw raw_g[kRecTile], raw_x[kRecTile], raw_d[kRecTile];
        load_tile<Raw, VEC>(raw_g, p.gates, q.b * p.gates_batch_stride + t0 * p.gates_step_stride + q.c, p.gates_step_stride, n, q.ok);
        load_tile<Raw, VEC>(raw_d, doutputs, at, p.channels, n, q.ok && doutputs != nullptr);
        if (!SUMMARY)
            load_tile<Raw, VEC>(raw_x, p.inputs, q.b * p.inputs_batch_stride + t0 * p.inputs_step_stride + q.c, p.inputs_step_stride, n, q.ok);
        const unsigned cut = reset_mask<FLAT>(p, q, t0, n);
        float code[kRecTile][VEC], diff[kRecTile][VEC];   // diff: the state a step starts from, minus its input
        float h[VEC];
        if (!SUMMARY)
#pragma unroll
            for (int v = 0; v < VEC; ++v) h[v] = q.ok && n > 0 ? saved[(q.b * tiles + t0 / kRecTile) * p.channels + q.c + v] : 0.0f;
#pragma unroll
        for (int j = 0; j < kRecTile; ++j) {
            float g[VEC], x[VEC];
            L::get(raw_g[j], g);
            if (!SUMMARY) L::get(raw_x[j], x);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                code[j][v] = j < n ? gate_code(g[v]) : kHold;
                if (!SUMMARY) {
                    float keep, take;
                    gate_pair(code[j][v], keep, take);
                    const float before = (cut >> j) & 1u ? 0.0f : h[v], fresh = take * x[v];
                    diff[j][v] = before - x[v];
                    h[v] = (cut >> j) & 1u ? fresh : fmaf(keep, h[v], fresh);
                }
            }
        }
        float lam[VEC];
        if (plan.warps > 1 || SUMMARY) {
            float a[VEC], b[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                a[v] = 1.0f;
                b[v] = 0.0f;
            }
#pragma unroll
            for (int j = kRecTile - 1; j >= 0; --j) {
                float d[VEC];
                L::get(raw_d[j], d);
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    float keep, take;
                    gate_pair(code[j][v], keep, take);
                    b[v] = (cut >> j) & 1u ? 0.0f : (b[v] + d[v]) * keep;
                    a[v] *= keep;
                }
            }
#pragma unroll
            for (int v = 0; v < VEC; ++v) s_pair[parity][threadIdx.x >> 5][v][q.lane] = make_float2(cut != 0 ? -1.0f : a[v], b[v]);
            group_barrier(q.group, plan.warps);
#pragma unroll
            for (int v = 0; v < VEC; ++v) lam[v] = carry[v];
            for (int w = plan.warps - 1; w >= 0; --w)
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const float2 ab = s_pair[parity][q.group * plan.warps + w][v][q.lane];
                    if (w == q.w) lam[v] = carry[v];
                    if (SUMMARY) sum_a[v] = ab.x < 0.0f || sum_a[v] < 0.0f ? -1.0f : sum_a[v] * ab.x;
                    carry[v] = apply_pair(ab, carry[v]);
                }
        } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) lam[v] = carry[v];
        }
        if (!SUMMARY) {
            T* out_x = dinputs + at + (kRecTile - 1) * p.channels;
            T* out_g = dgates + at + (kRecTile - 1) * p.channels;
#pragma unroll
            for (int j = kRecTile - 1; j >= 0; --j) {
                float d[VEC], dx[VEC], dg[VEC];
                L::get(raw_d[j], d);
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    float keep, take;
                    gate_pair(code[j][v], keep, take);
                    lam[v] += d[v];
                    dx[v] = lam[v] * take;
                    dg[v] = dx[v] * keep * diff[j][v];
                    lam[v] = (cut >> j) & 1u ? 0.0f : lam[v] * keep;
                }
                if (q.ok && j < n) {
                    *reinterpret_cast<Raw*>(out_x) = L::put(dx);
                    *reinterpret_cast<Raw*>(out_g) = L::put(dg);
                }
                out_x -= p.channels;
                out_g -= p.channels;
            }
            if (plan.warps == 1)
#pragma unroll
                for (int v = 0; v < VEC; ++v) carry[v] = lam[v];
        }
    }
    if (q.ok && q.w == 0) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            if (SUMMARY) pairs[q.split * lanes + q.index + v] = make_float2(sum_a[v], carry[v]);
            else if (q.split == 0 && dstate != nullptr) dstate[q.index + v] = carry[v];
        }
    }
}

// One step of every row; new_state may be state.
template <typename T>
__global__ void __launch_bounds__(256)
puff_recurrence_step_kernel(const T* __restrict__ gates, const T* __restrict__ inputs, const float* state,
                            const void* resets, int reset_bytes, long long batch, long long channels,
                            long long gates_stride, long long inputs_stride, T* __restrict__ outputs, float* new_state)
{
    const long long n = batch * channels, stride = static_cast<long long>(gridDim.x) * 256;
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < n; i += stride) {
        const long long b = i / channels, c = i - b * channels;
        float keep, take;
        gate_pair(gate_code(to_f32(gates[b * gates_stride + c])), keep, take);
        const float fresh = take * to_f32(inputs[b * inputs_stride + c]);
        bool reset = false;
        if (reset_bytes == 4) reset = static_cast<const float*>(resets)[b] != 0.0f;
        else if (reset_bytes == 1) reset = static_cast<const unsigned char*>(resets)[b] != 0;
        const float h = reset ? fresh : fmaf(keep, state[i], fresh);
        new_state[i] = h;
        outputs[i] = from_f32<T>(h);
    }
}

// bytes from the first to one past the last element of a [batch, steps, channels] view
static long long view_span(long long batch, long long steps, long long channels, long long bs, long long ss, int size)
{
    return ((batch - 1) * bs + (steps - 1) * ss + channels) * size;
}

// Enough warps to keep the memory busy (about twenty on each of 148 SMs, 4 KB of loads each), first by giving tiles
// along the steps to several warps of a CTA, then to several CTAs; the second costs reading the inputs twice.
constexpr long long kRecWantWarps = 148 * 20;
constexpr int kRecMaxSplits = 64;
static RecPlan rec_plan(long long batch, long long steps, long long channels, int vec, bool flat)
{
    RecPlan plan;
    plan.blocks_per_row = (channels + 32 * vec - 1) / (32 * vec);
    plan.lane_blocks = flat ? (batch * channels + 31) / 32 : batch * plan.blocks_per_row;
    const long long tiles = (steps + kRecTile - 1) / kRecTile;
    plan.warps = 1;
    while (plan.warps < kRecWarps && plan.warps < tiles && plan.lane_blocks * plan.warps < kRecWantWarps) plan.warps *= 2;
    const long long rounds = (tiles + plan.warps - 1) / plan.warps;
    long long splits = 1;
    // a range of fewer than four rounds would spend its time on the join
    if (plan.warps == kRecWarps) splits = kRecWantWarps / (plan.lane_blocks * plan.warps);
    if (splits > rounds / 4) splits = rounds / 4;
    if (splits > kRecMaxSplits) splits = kRecMaxSplits;
    if (splits < 1) splits = 1;
    const long long per = rounds > 0 ? (rounds + splits - 1) / splits : 1;
    plan.splits = rounds > 0 ? static_cast<int>((rounds + per - 1) / per) : 1;
    plan.split_steps = per * plan.warps * kRecTile;
    return plan;
}
static int rec_grid(const RecPlan& plan)
{
    const long long groups = kRecWarps / plan.warps;
    return static_cast<int>((plan.lane_blocks * plan.splits + groups - 1) / groups);
}
// The pairs of the ranges first where there are several, then the pass itself behind it
template <typename... KArgs, typename... Args>
static cudaError_t rec_launch(void (*summary)(KArgs...), void (*kernel)(KArgs...), const RecPlan& plan, cudaStream_t st, Args... args)
{
    const int grid = rec_grid(plan);
    if (summary == nullptr) {
        kernel<<<grid, kRecThreads, 0, st>>>(static_cast<KArgs>(args)...);
        count_launch();
        return cudaGetLastError();
    }
    summary<<<grid, kRecThreads, 0, st>>>(static_cast<KArgs>(args)...);
    count_launch();
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    count_launch();
    return launch_neighbour(kernel, grid, kRecThreads, 0, st, args...);
}
// channels too few to fill half a warp's lanes: rows share warps
static bool rec_flat(long long channels, int vec) { return channels < 16 * vec; }

static int check_recurrence(const RecArgs& p, int dtype)
{
    const int size = dtype_bytes(dtype);
    if (size == 0) return PUFF_ERR_DTYPE;
    if (p.batch < 0 || p.steps < 0 || p.channels < 0 || p.gates_batch_stride < 0 || p.gates_step_stride < 0 ||
        p.inputs_batch_stride < 0 || p.inputs_step_stride < 0)
        return PUFF_ERR_SHAPE;
    if (p.resets != nullptr && p.reset_bytes != 1 && p.reset_bytes != 4) return PUFF_ERR_DTYPE;
    const long long lanes = p.batch * p.channels;
    if (p.batch > 0 && p.channels > (1LL << 36) / p.batch) return PUFF_ERR_SIZE;
    if (lanes > 0 && p.steps > (1LL << 40) / lanes) return PUFF_ERR_SIZE;
    if (misaligned(p.gates, size) || misaligned(p.inputs, size) || misaligned(p.state, 4) ||
        (p.reset_bytes == 4 && misaligned(p.resets, 4)))
        return PUFF_ERR_ALIGN;
    if (lanes > 0 && p.steps > 0 && (p.gates == nullptr || p.inputs == nullptr)) return PUFF_ERR_NULL;
    return PUFF_OK;
}
// an output [0, bytes) must not touch what the kernels read
static bool touches_inputs(const RecArgs& p, int size, const void* out, long long bytes)
{
    return spans_overlap(out, bytes, p.gates, view_span(p.batch, p.steps, p.channels, p.gates_batch_stride, p.gates_step_stride, size)) ||
           spans_overlap(out, bytes, p.inputs, view_span(p.batch, p.steps, p.channels, p.inputs_batch_stride, p.inputs_step_stride, size)) ||
           spans_overlap(out, bytes, p.resets, p.batch * p.steps * p.reset_bytes) ||
           spans_overlap(out, bytes, p.state, 4 * p.batch * p.channels);
}
}  // namespace puff

using namespace puff;

extern "C" long long puff_policy_sm100_recurrence_saved_floats(long long batch, long long steps, long long channels)
{
    if (batch <= 0 || steps <= 0 || channels <= 0) return 0;
    return batch * ((steps + kRecTile - 1) / kRecTile) * channels;
}

// one pair per range and channel, whatever the type and alignment
extern "C" size_t puff_policy_sm100_recurrence_scratch_bytes(long long batch, long long steps, long long channels)
{
    if (batch <= 0 || steps <= 0 || channels <= 0) return 0;
    const int a = rec_plan(batch, steps, channels, 1, rec_flat(channels, 1)).splits, b = rec_plan(batch, steps, channels, 2, false).splits;
    const int splits = a > b ? a : b;
    return splits > 1 ? static_cast<size_t>(splits) * batch * channels * sizeof(float2) : 0;
}

extern "C" int puff_policy_sm100_recurrence(const void* gates, const void* inputs, int dtype, const void* resets,
                                            int reset_bytes, const float* state, long long batch, long long steps,
                                            long long channels, long long gates_batch_stride,
                                            long long gates_step_stride, long long inputs_batch_stride,
                                            long long inputs_step_stride, void* outputs, float* final_state,
                                            float* saved, void* scratch, size_t scratch_bytes, void* cuda_stream)
{
    RecArgs p = {gates, inputs, resets, state, batch, steps, channels, gates_batch_stride, gates_step_stride,
                 inputs_batch_stride, inputs_step_stride, resets != nullptr ? reset_bytes : 0};
    int rc = check_recurrence(p, dtype);
    if (rc != PUFF_OK) return rc;
    const long long lanes = batch * channels, n = lanes * steps;
    if (lanes == 0) return PUFF_OK;
    if (final_state == nullptr || (n > 0 && outputs == nullptr)) return PUFF_ERR_NULL;
    const int size = dtype_bytes(dtype);
    if (misaligned(outputs, size) || misaligned(final_state, 4) || misaligned(saved, 4)) return PUFF_ERR_ALIGN;
    const long long need = static_cast<long long>(puff_policy_sm100_recurrence_scratch_bytes(batch, steps, channels));
    if (need > 0 && (scratch == nullptr || misaligned(scratch, 8) || scratch_bytes < static_cast<size_t>(need))) return PUFF_ERR_WORKSPACE;
    const long long out_bytes = n * size, saved_bytes = 4 * puff_policy_sm100_recurrence_saved_floats(batch, steps, channels);
    if (touches_inputs(p, size, outputs, out_bytes) || touches_inputs(p, size, final_state, 4 * lanes) ||
        touches_inputs(p, size, saved, saved_bytes) || spans_overlap(outputs, out_bytes, final_state, 4 * lanes) ||
        spans_overlap(outputs, out_bytes, saved, saved_bytes) || spans_overlap(final_state, 4 * lanes, saved, saved_bytes) ||
        (need > 0 && (touches_inputs(p, size, scratch, need) || spans_overlap(scratch, need, outputs, out_bytes) ||
                      spans_overlap(scratch, need, final_state, 4 * lanes) || spans_overlap(scratch, need, saved, saved_bytes))))
        return PUFF_ERR_ALIAS;
    int sms = 0;
    rc = require_sm100(&sms);
    if (rc != PUFF_OK) return rc;
    // two channels a lane where every address of the 16-bit tensors stays 4-byte aligned
    const bool pair = size == 2 && channels % 2 == 0 && gates_batch_stride % 2 == 0 && gates_step_stride % 2 == 0 &&
                      inputs_batch_stride % 2 == 0 && inputs_step_stride % 2 == 0 && !misaligned(gates, 4) &&
                      !misaligned(inputs, 4) && !misaligned(outputs, 4) && !rec_flat(channels, 2);
    const bool flat = rec_flat(channels, 1);
    const RecPlan plan = rec_plan(batch, steps, channels, pair ? 2 : 1, flat);
    float2* pairs = static_cast<float2*>(scratch);
    cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    cudaError_t e;
#define PUFF_RUN2(T, VEC, FLAT)                                                                                          \
    rec_launch(plan.splits > 1 ? puff_recurrence_kernel<T, VEC, FLAT, true> : nullptr,                                    \
               puff_recurrence_kernel<T, VEC, FLAT, false>, plan, st, p, plan, pairs, static_cast<T*>(outputs),           \
               final_state, saved)
    if (dtype == PUFF_DTYPE_F32) e = flat ? PUFF_RUN2(float, 1, true) : PUFF_RUN2(float, 1, false);
    else if (dtype == PUFF_DTYPE_F16) e = pair ? PUFF_RUN2(__half, 2, false) : flat ? PUFF_RUN2(__half, 1, true) : PUFF_RUN2(__half, 1, false);
    else e = pair ? PUFF_RUN2(__nv_bfloat16, 2, false) : flat ? PUFF_RUN2(__nv_bfloat16, 1, true) : PUFF_RUN2(__nv_bfloat16, 1, false);
#undef PUFF_RUN2
    return static_cast<int>(e);
}

extern "C" int puff_policy_sm100_recurrence_backward(const void* gates, const void* inputs, int dtype, const void* resets,
                                                     int reset_bytes, const float* saved, long long batch,
                                                     long long steps, long long channels, long long gates_batch_stride,
                                                     long long gates_step_stride, long long inputs_batch_stride,
                                                     long long inputs_step_stride, const void* doutputs,
                                                     const float* dfinal, void* dgates, void* dinputs, float* dstate,
                                                     void* scratch, size_t scratch_bytes, void* cuda_stream)
{
    RecArgs p = {gates, inputs, resets, nullptr, batch, steps, channels, gates_batch_stride, gates_step_stride,
                 inputs_batch_stride, inputs_step_stride, resets != nullptr ? reset_bytes : 0};
    int rc = check_recurrence(p, dtype);
    if (rc != PUFF_OK) return rc;
    const long long lanes = batch * channels, n = lanes * steps;
    if (lanes == 0) return PUFF_OK;
    if (n > 0 && (saved == nullptr || dgates == nullptr || dinputs == nullptr)) return PUFF_ERR_NULL;
    const int size = dtype_bytes(dtype);
    if (misaligned(saved, 4) || misaligned(doutputs, size) || misaligned(dfinal, 4) || misaligned(dgates, size) ||
        misaligned(dinputs, size) || misaligned(dstate, 4))
        return PUFF_ERR_ALIGN;
    const long long need = static_cast<long long>(puff_policy_sm100_recurrence_scratch_bytes(batch, steps, channels));
    if (need > 0 && (scratch == nullptr || misaligned(scratch, 8) || scratch_bytes < static_cast<size_t>(need))) return PUFF_ERR_WORKSPACE;
    const long long saved_bytes = 4 * puff_policy_sm100_recurrence_saved_floats(batch, steps, channels);
    const void* out[4] = {dgates, dinputs, dstate, scratch};
    const long long out_bytes[4] = {n * size, n * size, 4 * lanes, need};
    for (int i = 0; i < 4; ++i) {
        if (touches_inputs(p, size, out[i], out_bytes[i]) || spans_overlap(out[i], out_bytes[i], saved, saved_bytes) ||
            spans_overlap(out[i], out_bytes[i], doutputs, n * size) || spans_overlap(out[i], out_bytes[i], dfinal, 4 * lanes))
            return PUFF_ERR_ALIAS;
        for (int j = 0; j < i; ++j)
            if (spans_overlap(out[i], out_bytes[i], out[j], out_bytes[j])) return PUFF_ERR_ALIAS;
    }
    int sms = 0;
    rc = require_sm100(&sms);
    if (rc != PUFF_OK) return rc;
    const bool pair = size == 2 && channels % 2 == 0 && gates_batch_stride % 2 == 0 && gates_step_stride % 2 == 0 &&
                      inputs_batch_stride % 2 == 0 && inputs_step_stride % 2 == 0 && !misaligned(gates, 4) &&
                      !misaligned(inputs, 4) && !misaligned(doutputs, 4) && !misaligned(dgates, 4) &&
                      !misaligned(dinputs, 4) && !rec_flat(channels, 2);
    const bool flat = rec_flat(channels, 1);
    const RecPlan plan = rec_plan(batch, steps, channels, pair ? 2 : 1, flat);
    float2* pairs = static_cast<float2*>(scratch);
    cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    cudaError_t e;
#define PUFF_RUN2(T, VEC, FLAT)                                                                                          \
    rec_launch(plan.splits > 1 ? puff_recurrence_backward_kernel<T, VEC, FLAT, true> : nullptr,                           \
               puff_recurrence_backward_kernel<T, VEC, FLAT, false>, plan, st, p, plan, pairs, saved,                     \
               static_cast<const T*>(doutputs), dfinal, static_cast<T*>(dgates), static_cast<T*>(dinputs), dstate)
    if (dtype == PUFF_DTYPE_F32) e = flat ? PUFF_RUN2(float, 1, true) : PUFF_RUN2(float, 1, false);
    else if (dtype == PUFF_DTYPE_F16) e = pair ? PUFF_RUN2(__half, 2, false) : flat ? PUFF_RUN2(__half, 1, true) : PUFF_RUN2(__half, 1, false);
    else e = pair ? PUFF_RUN2(__nv_bfloat16, 2, false) : flat ? PUFF_RUN2(__nv_bfloat16, 1, true) : PUFF_RUN2(__nv_bfloat16, 1, false);
#undef PUFF_RUN2
    return static_cast<int>(e);
}

extern "C" int puff_policy_sm100_recurrence_step(const void* gates, const void* inputs, int dtype, const void* resets,
                                                 int reset_bytes, const float* state, long long batch,
                                                 long long channels, long long gates_stride, long long inputs_stride,
                                                 void* outputs, float* new_state, void* cuda_stream)
{
    RecArgs p = {gates, inputs, resets, nullptr, batch, 1, channels, gates_stride, channels, inputs_stride, channels,
                 resets != nullptr ? reset_bytes : 0};
    int rc = check_recurrence(p, dtype);
    if (rc != PUFF_OK) return rc;
    const long long n = batch * channels;
    if (n == 0) return PUFF_OK;
    if (state == nullptr || outputs == nullptr || new_state == nullptr) return PUFF_ERR_NULL;
    const int size = dtype_bytes(dtype);
    if (misaligned(state, 4) || misaligned(outputs, size) || misaligned(new_state, 4)) return PUFF_ERR_ALIGN;
    if (touches_inputs(p, size, outputs, n * size) || touches_inputs(p, size, new_state, 4 * n) ||
        spans_overlap(outputs, n * size, state, 4 * n) || spans_overlap(outputs, n * size, new_state, 4 * n) ||
        (new_state != state && spans_overlap(new_state, 4 * n, state, 4 * n)))
        return PUFF_ERR_ALIAS;
    int sms = 0;
    rc = require_sm100(&sms);
    if (rc != PUFF_OK) return rc;
    long long blocks = (n + 255) / 256;
    if (blocks > 8LL * sms) blocks = 8LL * sms;
    cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
#define PUFF_RUN(T)                                                                                                      \
    puff_recurrence_step_kernel<T><<<static_cast<int>(blocks), 256, 0, st>>>(static_cast<const T*>(gates),               \
        static_cast<const T*>(inputs), state, resets, p.reset_bytes, batch, channels, gates_stride, inputs_stride,       \
        static_cast<T*>(outputs), new_state)
    if (dtype == PUFF_DTYPE_F32) PUFF_RUN(float);
    else if (dtype == PUFF_DTYPE_F16) PUFF_RUN(__half);
    else PUFF_RUN(__nv_bfloat16);
#undef PUFF_RUN
    count_launch();
    return static_cast<int>(cudaGetLastError());
}
