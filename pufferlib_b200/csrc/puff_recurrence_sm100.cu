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
//
// Memory-bound: three elements moved a step forward, five backward; the arithmetic behind them, two special functions and
// some twenty instructions a step for two channels, is close to the bound, so what surrounds it (addresses, joins, waits)
// decides.  8192 x 64 x 128 bf16: 79 us forward (5.1 TB/s of 6.55) and 118 backward (5.7); fp32 128 and 209 (6.4);
// 256 x 4096 x 128 fp32 276 and 450.  One thread a channel, step after step, took 1904 us for the first pair.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/puff_advantage.h"
#include "puff_policy.cuh"

namespace puff {

constexpr int kRecTile = PUFF_RECURRENCE_SAVED_STEPS;       // 16: steps whose inputs a warp holds in registers; also the distance of the saved states
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
    unsigned wait_ns;        // how long to wait for a tile
};

// How the work is cut.  A warp owns 32 lanes of VEC channels and walks 16 steps at a time, all of them in registers.
// `warps` warps of a CTA take consecutive 16-step tiles of the same lanes, and `splits` ranges of `split_steps` steps
// go to different CTAs where lanes are few.  A tile (or range) maps the state before it to the state after it as
// h -> A h + B; those pairs are joined over the warps through shared memory, and over the ranges through global memory
// by a first launch that computes nothing else.
// Where TMA moves the tiles, a cluster of `shares` CTAs can take consecutive parts of a round instead: it joins its pairs
// through distributed shared memory and reads everything once.
struct RecPlan {
    int warps, splits, shares;
    long long split_steps, lane_blocks, blocks_per_row;
};

__device__ __forceinline__ bool is_reset(const RecArgs& p, long long i)
{
    if (p.reset_bytes == 4) return static_cast<const float*>(p.resets)[i] != 0.0f;
    return p.reset_bytes == 1 && static_cast<const unsigned char*>(p.resets)[i] != 0;
}

// keep = sigmoid(g) and take = 1 - keep = sigmoid(-g).  The smaller of the two is 1 / (1 + e^|g|), good to 8 half steps
// of fp32 (4 of ex2.approx, 2 of rcp.approx, 1 each of what surrounds them) down to 2^-126, below which it is 0; the
// larger is 1 minus it, so that the two add up to 1 and the state stays a weighted mean.  One register, the code, holds both gates: the smaller one with the sign of g.
__device__ __forceinline__ float rcp_approx(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kHold = 0.0f;      // the code of a gate that holds the state: steps past the end

// Arithmetic on the VEC channels of a lane, in packed pairs where there are two
template <int VEC>
__device__ __forceinline__ void v_fma(float (&d)[VEC], const float (&a)[VEC], const float (&b)[VEC], const float (&c)[VEC])
{
    if constexpr (VEC == 2) {
        const float2 r = __ffma2_rn(make_float2(a[0], a[1]), make_float2(b[0], b[1]), make_float2(c[0], c[1]));
        d[0] = r.x, d[1] = r.y;
    } else {
        d[0] = fmaf(a[0], b[0], c[0]);
    }
}
template <int VEC>
__device__ __forceinline__ void v_mul(float (&d)[VEC], const float (&a)[VEC], const float (&b)[VEC])
{
    if constexpr (VEC == 2) {
        const float2 r = __fmul2_rn(make_float2(a[0], a[1]), make_float2(b[0], b[1]));
        d[0] = r.x, d[1] = r.y;
    } else {
        d[0] = a[0] * b[0];
    }
}
template <int VEC>
__device__ __forceinline__ void v_add(float (&d)[VEC], const float (&a)[VEC], const float (&b)[VEC])
{
    if constexpr (VEC == 2) {
        const float2 r = __fadd2_rn(make_float2(a[0], a[1]), make_float2(b[0], b[1]));
        d[0] = r.x, d[1] = r.y;
    } else {
        d[0] = a[0] + b[0];
    }
}
// e^h, h = |g|, as 2^t (1 + r): t is h log2(e), r what t leaves out of it.  Rounded once and without r the gate is 8 half steps
// further off at 10, 63 at 85.  A bf16 value has 8 bits, so that its product with the upper 16 of log2(e) is exact, and r
// is h times the rest of it, tilted so that 1 + r stays within 0.3 half steps of e^r up to 88.  Other types: t rounded, and
// r = h - t ln 2 with ln 2 in 48 bits; there h ends at 88, where e^h is finite still and its reciprocal 0 already.
// (bf16 forward, without r, with the first form, with the second: 8192 x 64 x 128 77, 79, 80 us; 6525 x 8 x 1888 172, 176,
// 178; 4 x 8192 x 1024 70, 75, 76.)
constexpr float kLog2eUpper = 1.44268798828125f, kLog2eRest = 4.889379397354787e-06f;
constexpr float kLn2High = 0.693147182464599609375f, kLn2Low = -1.904654299957768e-09f;
template <typename T, int VEC>
__device__ __forceinline__ void gate_codes(const float (&g)[VEC], float (&code)[VEC])
{
    float t[VEC], e[VEC], r[VEC], one[VEC], d[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) one[v] = 1.0f;
    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            t[v] = fabsf(g[v]) * kLog2eUpper;
            r[v] = fabsf(g[v]) * kLog2eRest;
        }
    } else {
        float h[VEC], log2e[VEC], high[VEC], low[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            asm("min.NaN.f32 %0, %1, %2;" : "=f"(h[v]) : "f"(fabsf(g[v])), "f"(88.0f));
            log2e[v] = kLog2e;
            high[v] = -kLn2High;
            low[v] = -kLn2Low;
        }
        v_mul(t, h, log2e);
        v_fma(r, t, high, h);
        v_fma(r, t, low, r);
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) e[v] = exp2_approx(t[v]);
    v_fma(e, e, r, e);
    v_add(d, e, one);
#pragma unroll
    for (int v = 0; v < VEC; ++v) code[v] = copysignf(rcp_approx(d[v]), g[v]);
}
template <int VEC>
__device__ __forceinline__ void gate_pairs(const float (&code)[VEC], float (&keep)[VEC], float (&take)[VEC])
{
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        const float small = fabsf(code[v]), large = 1.0f - small;
        const bool negative = __float_as_int(code[v]) < 0;
        keep[v] = negative ? small : large;
        take[v] = negative ? large : small;
    }
}

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

__device__ __forceinline__ long long quotient(long long a, long long b)
{
    return ((a | b) >> 32) == 0 ? static_cast<unsigned>(a) / static_cast<unsigned>(b) : a / b;
}

// Where this thread's warp stands in the plan.  FLAT: the lanes of a warp are adjacent (batch, channel) pairs of any
// rows, for channels too few to fill a warp; otherwise they are adjacent channels of one row.
struct RecPlace {
    int group, w, lane;
    bool unit, ok;             // the group has work; this lane has a channel
    int slot;                  // this warp among those of its group, or of its cluster
    int split;
    long long b, c, index;     // index: b * channels + c
    long long t_begin, t_end;
    __device__ __forceinline__ int steps_at(long long t0) const
    {
        const long long left = t_end - t0;
        return left < 0 ? 0 : left < kRecTile ? static_cast<int>(left) : kRecTile;
    }
};
template <int VEC, bool FLAT>
__device__ __forceinline__ RecPlace rec_place(const RecArgs& p, const RecPlan& plan)
{
    RecPlace q;
    const int warp = threadIdx.x >> 5;
    q.lane = threadIdx.x & 31;
    q.group = warp / plan.warps;
    q.w = warp - q.group * plan.warps;
    const unsigned shared_by = static_cast<unsigned>(plan.shares), block_id = blockIdx.x / shared_by;
    q.slot = q.w + static_cast<int>(blockIdx.x - block_id * shared_by) * plan.warps;
    const long long unit = block_id * static_cast<long long>(kRecWarps / plan.warps) + q.group;
    q.split = plan.splits == 1 && unit < plan.lane_blocks ? 0 : static_cast<int>(quotient(unit, plan.lane_blocks));
    const long long block = unit - q.split * plan.lane_blocks;
    q.unit = q.split < plan.splits;
    if (FLAT) {
        q.index = block * 32 + q.lane;
        q.ok = q.index < p.batch * p.channels;
        q.b = q.ok ? quotient(q.index, p.channels) : 0;
        q.c = q.ok ? q.index - q.b * p.channels : 0;
    } else {
        q.b = quotient(block, plan.blocks_per_row);
        q.c = (block - q.b * plan.blocks_per_row) * (32 * VEC) + q.lane * VEC;
        q.ok = q.c < p.channels;
        q.index = q.b * p.channels + q.c;
    }
    q.ok = q.ok && q.unit;
    q.t_begin = q.split * plan.split_steps;
    q.t_end = q.t_begin + plan.split_steps < p.steps ? q.t_begin + plan.split_steps : p.steps;
    return q;
}
// The resets of a tile as a mask, bit j for step t0 + j, in two halves so that the load is a round old when its value is
// needed (asked for and used at once, it stalled every round).  All lanes of a row share the mask; FLAT lanes have one each.
template <bool FLAT>
__device__ __forceinline__ unsigned resets_ahead(const RecArgs& p, const RecPlace& q, long long t0, int n)
{
    if (p.reset_bytes == 0) return 0u;
    const long long at = q.b * p.steps + t0;
    if (!FLAT) {
        if (q.lane >= n) return 0u;
        return p.reset_bytes == 4 ? __ldg(static_cast<const unsigned*>(p.resets) + at + q.lane)
                                  : __ldg(static_cast<const unsigned char*>(p.resets) + at + q.lane);
    }
    unsigned m = 0;
    if (q.ok)
#pragma unroll 4
        for (int j = 0; j < n; ++j) m |= is_reset(p, at + j) ? 1u << j : 0u;
    return m;
}
template <bool FLAT>
__device__ __forceinline__ unsigned reset_mask(const RecArgs& p, unsigned ahead)
{
    if (FLAT || p.reset_bytes == 0) return ahead;
    // fp32: anything but +0 and -0
    return __ballot_sync(0xffffffffu, (p.reset_bytes == 4 ? ahead << 1 : ahead) != 0);
}
template <typename Raw, int VEC>
__device__ __forceinline__ void load_tile(Raw (&raw)[kRecTile], const void* base, long long at, long long step_stride, int n, bool ok)
{
    constexpr long long size = sizeof(Raw) / VEC;
    const char* ptr = static_cast<const char*>(base) + at * size;
    const long long bytes = step_stride * size;
    if (n == kRecTile) {
#pragma unroll
        for (int j = 0; j < kRecTile; ++j, ptr += bytes) {
            raw[j] = zero_raw<Raw>();
            if (ok) raw[j] = __ldg(reinterpret_cast<const Raw*>(ptr));
        }
    } else {
#pragma unroll
        for (int j = 0; j < kRecTile; ++j, ptr += bytes) {
            raw[j] = zero_raw<Raw>();
            if (ok && j < n) raw[j] = __ldg(reinterpret_cast<const Raw*>(ptr));
        }
    }
}
__device__ __forceinline__ void group_barrier(int group, int warps)
{
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(warps * 32) : "memory");
}

// ---- what a warp does with a tile in registers.  PLAIN: sixteen steps, none a reset (for any lane of the warp).
template <typename T, int VEC, bool PLAIN>
__device__ __forceinline__ void tile_gates(const typename Lane<T, VEC>::Raw& raw_g, const typename Lane<T, VEC>::Raw& raw_x, bool there, float (&keep)[VEC],
                                           float (&fresh)[VEC])
{
    using L = Lane<T, VEC>;
    float g[VEC], x[VEC], code[VEC], take[VEC];
    L::get(raw_g, g);
    L::get(raw_x, x);
    gate_codes<T>(g, code);
    if (!PLAIN && !there)
#pragma unroll
        for (int v = 0; v < VEC; ++v) code[v] = kHold;
    gate_pairs(code, keep, take);
    v_mul(fresh, take, x);
}
template <int VEC, bool PLAIN>
__device__ __forceinline__ void advance(float (&h)[VEC], const float (&keep)[VEC], const float (&fresh)[VEC], bool reset)
{
    v_fma(h, keep, h, fresh);
    if (!PLAIN && reset)
#pragma unroll
        for (int v = 0; v < VEC; ++v) h[v] = fresh[v];
}
// one pass: every step's state follows from the one before it
template <typename T, int VEC, bool PLAIN, typename Tile>
__device__ __forceinline__ void forward_stream(const Tile& raw_g, const Tile& raw_x, unsigned cut, int n, float (&h)[VEC], T* out, long long stride, bool ok)
{
    using L = Lane<T, VEC>;
#pragma unroll
    for (int j = 0; j < kRecTile; ++j, out += stride) {
        float keep[VEC], fresh[VEC];
        tile_gates<T, VEC, PLAIN>(raw_g[j], raw_x[j], j < n, keep, fresh);
        advance<VEC, PLAIN>(h, keep, fresh, (cut >> j) & 1u);
        if (ok && (PLAIN || j < n)) *reinterpret_cast<typename L::Raw*>(out) = L::put(h);
    }
}
// two passes: the tile's pair (a, b), then its states once the one before it is known
template <typename T, int VEC, bool PLAIN, typename Tile>
__device__ __forceinline__ void forward_pair(const Tile& raw_g, const Tile& raw_x, unsigned cut, int n, float (&keep)[kRecTile][VEC], float (&fresh)[kRecTile][VEC], float (&a)[VEC], float (&b)[VEC])
{
#pragma unroll
    for (int j = 0; j < kRecTile; ++j) {
        tile_gates<T, VEC, PLAIN>(raw_g[j], raw_x[j], j < n, keep[j], fresh[j]);
        if (j == 0) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                a[v] = keep[0][v];
                b[v] = fresh[0][v];
            }
        } else {
            advance<VEC, PLAIN>(b, keep[j], fresh[j], (cut >> j) & 1u);
            v_mul(a, a, keep[j]);
        }
    }
}
template <typename T, int VEC, bool PLAIN>
__device__ __forceinline__ void forward_states(const float (&keep)[kRecTile][VEC], const float (&fresh)[kRecTile][VEC], unsigned cut,
                                               int n, float (&h)[VEC], T* out, long long stride, bool ok)
{
    using L = Lane<T, VEC>;
#pragma unroll
    for (int j = 0; j < kRecTile; ++j, out += stride) {
        advance<VEC, PLAIN>(h, keep[j], fresh[j], (cut >> j) & 1u);
        if (ok && (PLAIN || j < n)) *reinterpret_cast<typename L::Raw*>(out) = L::put(h);
    }
}
// joins the pairs of a group's warps: h comes out as the value before this warp's tile (in walking order), carry as the
// one after all of them; SUMMARY keeps the product of the gains too
template <int VEC, bool SUMMARY, bool REVERSE>
__device__ __forceinline__ void join_warps(float2 (*s_pair)[VEC][32], const RecPlace& q, int warps, unsigned cut, const float (&a)[VEC],
                                           const float (&b)[VEC], float (&h)[VEC], float (&carry)[VEC], float (&sum_a)[VEC])
{
#pragma unroll
    for (int v = 0; v < VEC; ++v) s_pair[q.group * warps + q.w][v][q.lane] = make_float2(cut != 0 ? -1.0f : a[v], b[v]);
    group_barrier(q.group, warps);
#pragma unroll
    for (int v = 0; v < VEC; ++v) h[v] = carry[v];
    for (int i = 0; i < warps; ++i) {
        const int w = REVERSE ? warps - 1 - i : i;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const float2 ab = s_pair[q.group * warps + w][v][q.lane];
            if (w == q.w) h[v] = carry[v];
            if (SUMMARY) sum_a[v] = ab.x < 0.0f || sum_a[v] < 0.0f ? -1.0f : sum_a[v] * ab.x;
            carry[v] = apply_pair(ab, carry[v]);
        }
    }
}

// STREAM: one warp a group, tile after tile, the next one's loads under this one's arithmetic.  TEAM: the warps of a group
// take a tile each.  SUMMARY: as TEAM, only the pairs of the ranges.
// CLUSTER: as TEAM, by all warps of a cluster.
enum RecMode { kStream, kTeam, kSummary, kCluster };

// the pair of x, then y
__device__ __forceinline__ float2 then_pair(float2 x, float2 y)
{
    if (y.x < 0.0f) return y;
    return make_float2(x.x < 0.0f ? -1.0f : x.x * y.x, fmaf(y.x, x.y, y.y));
}
// As join_warps for a cluster whose CTAs have one group each: the warps' pairs within the CTA first, then the CTAs' through
// s_cta, into which every CTA writes its own at all the others.  s_pair is free again after the cluster's barrier, s_cta
// (written from outside) only after the next one: the caller alternates between two.
template <int VEC, bool REVERSE>
__device__ __forceinline__ void join_cluster(float2 (*s_pair)[VEC][32], float2 (*s_cta)[VEC][32], const RecPlace& q, const RecPlan& plan,
                                             unsigned cut, const float (&a)[VEC], const float (&b)[VEC], float (&h)[VEC], float (&carry)[VEC])
{
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    const int rank = static_cast<int>(cluster.block_rank());
#pragma unroll
    for (int v = 0; v < VEC; ++v) s_pair[q.w][v][q.lane] = make_float2(cut != 0 ? -1.0f : a[v], b[v]);
    __syncthreads();
    float2 before[VEC], all[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) before[v] = all[v] = make_float2(1.0f, 0.0f);
    for (int i = 0; i < kRecWarps; ++i) {
        const int w = REVERSE ? kRecWarps - 1 - i : i;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            if (w == q.w) before[v] = all[v];
            all[v] = then_pair(all[v], s_pair[w][v][q.lane]);
        }
    }
    if (q.w < plan.shares) {       // warp k tells CTA k
        float2* to = cluster.map_shared_rank(&s_cta[rank][0][q.lane], q.w);
#pragma unroll
        for (int v = 0; v < VEC; ++v) to[32 * v] = all[v];
    }
    cluster.sync();
#pragma unroll
    for (int v = 0; v < VEC; ++v) h[v] = carry[v];
    for (int i = 0; i < plan.shares; ++i) {
        const int k = REVERSE ? plan.shares - 1 - i : i;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            if (k == rank) h[v] = apply_pair(before[v], carry[v]);
            carry[v] = apply_pair(s_cta[k][v][q.lane], carry[v]);
        }
    }
}

// Forward.  saved (nullable): the state before steps 0, 16, 32, ... as [batch, ceil(steps / 16), channels].
template <typename T, int VEC, bool FLAT, RecMode MODE>
__global__ void __launch_bounds__(kRecThreads, 2)
puff_recurrence_kernel(RecArgs p, RecPlan plan, float2* pairs, T* __restrict__ outputs, float* __restrict__ final_state,
                       float* __restrict__ saved)
{
    using Raw = typename Lane<T, VEC>::Raw;
    __shared__ float2 s_pair[MODE == kStream ? 1 : 2][MODE == kStream ? 1 : kRecWarps][VEC][32];
    if (MODE != kSummary) pdl_wait();
    const RecPlace q = rec_place<VEC, FLAT>(p, plan);
    if (!q.unit) return;
    const long long lanes = p.batch * p.channels;
    const long long tiles = (p.steps + kRecTile - 1) / kRecTile;
    float carry[VEC], sum_a[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        carry[v] = MODE != kSummary && q.ok && p.state != nullptr ? p.state[q.index + v] : 0.0f;
        sum_a[v] = 1.0f;
    }
    if (MODE == kTeam)
        for (int r = 0; r < q.split; ++r)
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                if (q.ok) carry[v] = apply_pair(pairs[r * lanes + q.index + v], carry[v]);
    const long long step = kRecTile * plan.warps;
    long long t0 = q.t_begin + q.w * kRecTile;
    const long long gates_at = q.b * p.gates_batch_stride + q.c, inputs_at = q.b * p.inputs_batch_stride + q.c;
    T* out = outputs + (q.b * p.steps + t0) * p.channels + q.c;
    float* save = saved != nullptr ? saved + (q.b * tiles + t0 / kRecTile) * p.channels + q.c : nullptr;
    Raw raw_g[kRecTile], raw_x[kRecTile];
    if (MODE == kStream) {
        load_tile<Raw, VEC>(raw_g, p.gates, gates_at + t0 * p.gates_step_stride, p.gates_step_stride, q.steps_at(t0), q.ok);
        load_tile<Raw, VEC>(raw_x, p.inputs, inputs_at + t0 * p.inputs_step_stride, p.inputs_step_stride, q.steps_at(t0), q.ok);
    }
    unsigned resets = resets_ahead<FLAT>(p, q, t0, q.steps_at(t0));
    int parity = 0;
    for (long long t = q.t_begin; t < q.t_end; t += step, t0 += step, parity ^= 1) {
        const int n = q.steps_at(t0);
        const unsigned cut = reset_mask<FLAT>(p, resets);
        resets = resets_ahead<FLAT>(p, q, t0 + step, q.steps_at(t0 + step));
        const bool plain = n == kRecTile && !(FLAT ? __any_sync(0xffffffffu, cut != 0) : cut != 0);
        if (MODE == kStream) {
            Raw next_g[kRecTile], next_x[kRecTile];
            const long long t1 = t0 + step;
            load_tile<Raw, VEC>(next_g, p.gates, gates_at + t1 * p.gates_step_stride, p.gates_step_stride, q.steps_at(t1), q.ok);
            load_tile<Raw, VEC>(next_x, p.inputs, inputs_at + t1 * p.inputs_step_stride, p.inputs_step_stride, q.steps_at(t1), q.ok);
            if (save != nullptr && q.ok)
#pragma unroll
                for (int v = 0; v < VEC; ++v) save[v] = carry[v];
            if (plain) forward_stream<T, VEC, true>(raw_g, raw_x, cut, n, carry, out, p.channels, q.ok);
            else forward_stream<T, VEC, false>(raw_g, raw_x, cut, n, carry, out, p.channels, q.ok);
#pragma unroll
            for (int j = 0; j < kRecTile; ++j) {
                raw_g[j] = next_g[j];
                raw_x[j] = next_x[j];
            }
        } else {
            load_tile<Raw, VEC>(raw_g, p.gates, gates_at + t0 * p.gates_step_stride, p.gates_step_stride, n, q.ok);
            load_tile<Raw, VEC>(raw_x, p.inputs, inputs_at + t0 * p.inputs_step_stride, p.inputs_step_stride, n, q.ok);
            float keep[kRecTile][VEC], fresh[kRecTile][VEC], a[VEC], b[VEC], h[VEC];
            if (plain) forward_pair<T, VEC, true>(raw_g, raw_x, cut, n, keep, fresh, a, b);
            else forward_pair<T, VEC, false>(raw_g, raw_x, cut, n, keep, fresh, a, b);
            join_warps<VEC, MODE == kSummary, false>(s_pair[parity], q, plan.warps, cut, a, b, h, carry, sum_a);
            if (MODE == kTeam) {
                if (save != nullptr && q.ok && n > 0)
#pragma unroll
                    for (int v = 0; v < VEC; ++v) save[v] = h[v];
                if (plain) forward_states<T, VEC, true>(keep, fresh, cut, n, h, out, p.channels, q.ok);
                else forward_states<T, VEC, false>(keep, fresh, cut, n, h, out, p.channels, q.ok);
            }
        }
        out += step * p.channels;
        if (save != nullptr) save += plan.warps * p.channels;
    }
    if (q.ok && q.w == 0) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            if (MODE == kSummary) pairs[q.split * lanes + q.index + v] = make_float2(sum_a[v], carry[v]);
            else if (q.split == plan.splits - 1) final_state[q.index + v] = carry[v];
        }
    }
}

// ---- backward: lam_t = dh_t + a_{t+1} lam_{t+1}, last tile first
// the states again, as what dgate needs of them: slope = keep take (state before - input)
template <typename T, int VEC, bool PLAIN, typename Tile>
__device__ __forceinline__ void backward_states(const Tile& raw_g, const Tile& raw_x, unsigned cut, int n, float (&h)[VEC], float (&code)[kRecTile][VEC], float (&slope)[kRecTile][VEC])
{
    using L = Lane<T, VEC>;
#pragma unroll
    for (int j = 0; j < kRecTile; ++j) {
        float g[VEC], x[VEC], keep[VEC], take[VEC], fresh[VEC], minus[VEC], diff[VEC], product[VEC];
        L::get(raw_g[j], g);
        L::get(raw_x[j], x);
        gate_codes<T>(g, code[j]);
        const bool reset = !PLAIN && (cut >> j) & 1u;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            if (!PLAIN && j >= n) code[j][v] = kHold;
            if (reset) h[v] = 0.0f;
            minus[v] = -x[v];
        }
        gate_pairs(code[j], keep, take);
        v_add(diff, h, minus);
        v_mul(product, keep, take);
        v_mul(slope[j], product, diff);
        v_mul(fresh, take, x);
        advance<VEC, PLAIN>(h, keep, fresh, reset);
    }
}
// lam after the tile -> lam before it, as a pair
template <typename T, int VEC, bool PLAIN, typename Tile>
__device__ __forceinline__ void backward_pair(const float (&code)[kRecTile][VEC], const Tile& raw_d, unsigned cut, float (&a)[VEC], float (&b)[VEC])
{
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        a[v] = 1.0f;
        b[v] = 0.0f;
    }
#pragma unroll
    for (int j = kRecTile - 1; j >= 0; --j) {
        float d[VEC], keep[VEC], take[VEC];
        Lane<T, VEC>::get(raw_d[j], d);
        gate_pairs(code[j], keep, take);
        v_add(b, b, d);
        v_mul(b, b, keep);
        v_mul(a, a, keep);
        if (!PLAIN && (cut >> j) & 1u)
#pragma unroll
            for (int v = 0; v < VEC; ++v) b[v] = 0.0f;
    }
}
template <typename T, int VEC, bool PLAIN, typename Tile>
__device__ __forceinline__ void backward_gradients(const float (&code)[kRecTile][VEC], const float (&slope)[kRecTile][VEC],
                                                   const Tile& raw_d, unsigned cut, int n,
                                                   float (&lam)[VEC], T* dgates, T* dinputs, long long stride, bool ok)
{
    using L = Lane<T, VEC>;
    dgates += (kRecTile - 1) * stride;
    dinputs += (kRecTile - 1) * stride;
#pragma unroll
    for (int j = kRecTile - 1; j >= 0; --j, dgates -= stride, dinputs -= stride) {
        float d[VEC], keep[VEC], take[VEC], dx[VEC], dg[VEC];
        L::get(raw_d[j], d);
        gate_pairs(code[j], keep, take);
        v_add(lam, lam, d);
        v_mul(dx, lam, take);
        v_mul(dg, lam, slope[j]);
        if (ok && (PLAIN || j < n)) {
            *reinterpret_cast<typename L::Raw*>(dinputs) = L::put(dx);
            *reinterpret_cast<typename L::Raw*>(dgates) = L::put(dg);
        }
        v_mul(lam, lam, keep);
        if (!PLAIN && (cut >> j) & 1u)
#pragma unroll
            for (int v = 0; v < VEC; ++v) lam[v] = 0.0f;
    }
}

// The states within a tile are computed again from the saved one before it.
template <typename T, int VEC, bool FLAT, RecMode MODE>
__global__ void __launch_bounds__(kRecThreads, 2)
puff_recurrence_backward_kernel(RecArgs p, RecPlan plan, float2* pairs, const float* __restrict__ saved,
                                const T* __restrict__ doutputs, const float* __restrict__ dfinal, T* __restrict__ dgates,
                                T* __restrict__ dinputs, float* __restrict__ dstate)
{
    using L = Lane<T, VEC>;
    using Raw = typename L::Raw;
    __shared__ float2 s_pair[MODE == kStream ? 1 : 2][MODE == kStream ? 1 : kRecWarps][VEC][32];
    if (MODE != kSummary) pdl_wait();
    const RecPlace q = rec_place<VEC, FLAT>(p, plan);
    if (!q.unit) return;
    const long long lanes = p.batch * p.channels;
    const long long tiles = (p.steps + kRecTile - 1) / kRecTile;
    float carry[VEC], sum_a[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        carry[v] = MODE != kSummary && q.ok && dfinal != nullptr ? dfinal[q.index + v] : 0.0f;
        sum_a[v] = 1.0f;
    }
    if (MODE == kTeam)
        for (int r = plan.splits - 1; r > q.split; --r)
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                if (q.ok) carry[v] = apply_pair(pairs[r * lanes + q.index + v], carry[v]);
    const long long step = kRecTile * plan.warps;
    const long long gates_at = q.b * p.gates_batch_stride + q.c, inputs_at = q.b * p.inputs_batch_stride + q.c;
    const long long last = q.t_begin + quotient(q.t_end > q.t_begin ? q.t_end - q.t_begin - 1 : 0, step) * step;
    unsigned resets = resets_ahead<FLAT>(p, q, last + q.w * kRecTile, q.steps_at(last + q.w * kRecTile));
    int parity = 0;
    for (long long t = last; t >= q.t_begin; t -= step, parity ^= 1) {
        const long long t0 = t + q.w * kRecTile;
        const int n = q.steps_at(t0);
        const long long at = (q.b * p.steps + t0) * p.channels + q.c;
        Raw raw_g[kRecTile], raw_x[kRecTile], raw_d[kRecTile];
        load_tile<Raw, VEC>(raw_g, p.gates, gates_at + t0 * p.gates_step_stride, p.gates_step_stride, n, q.ok);
        if (MODE != kSummary)
            load_tile<Raw, VEC>(raw_x, p.inputs, inputs_at + t0 * p.inputs_step_stride, p.inputs_step_stride, n, q.ok);
        load_tile<Raw, VEC>(raw_d, doutputs, at, p.channels, n, q.ok && doutputs != nullptr);
        float h[VEC];
        if (MODE != kSummary)
#pragma unroll
            for (int v = 0; v < VEC; ++v) h[v] = q.ok && n > 0 ? saved[(q.b * tiles + t0 / kRecTile) * p.channels + q.c + v] : 0.0f;
        const unsigned cut = reset_mask<FLAT>(p, resets);
        resets = t > q.t_begin ? resets_ahead<FLAT>(p, q, t0 - step, q.steps_at(t0 - step)) : 0u;
        const bool plain = n == kRecTile && !(FLAT ? __any_sync(0xffffffffu, cut != 0) : cut != 0);
        float code[kRecTile][VEC], slope[kRecTile][VEC];
        if (MODE == kSummary) {
#pragma unroll
            for (int j = 0; j < kRecTile; ++j) {
                float g[VEC];
                L::get(raw_g[j], g);
                gate_codes<T>(g, code[j]);
                if (j >= n)
#pragma unroll
                    for (int v = 0; v < VEC; ++v) code[j][v] = kHold;
            }
        } else if (plain) {
            backward_states<T, VEC, true>(raw_g, raw_x, cut, n, h, code, slope);
        } else {
            backward_states<T, VEC, false>(raw_g, raw_x, cut, n, h, code, slope);
        }
        float lam[VEC];
        if (MODE != kStream) {
            float a[VEC], b[VEC];
            if (plain) backward_pair<T, VEC, true>(code, raw_d, cut, a, b);
            else backward_pair<T, VEC, false>(code, raw_d, cut, a, b);
            join_warps<VEC, MODE == kSummary, true>(s_pair[parity], q, plan.warps, cut, a, b, lam, carry, sum_a);
        }
        if (MODE != kSummary) {
            float (&l)[VEC] = MODE == kStream ? carry : lam;
            if (plain) backward_gradients<T, VEC, true>(code, slope, raw_d, cut, n, l, dgates + at, dinputs + at, p.channels, q.ok);
            else backward_gradients<T, VEC, false>(code, slope, raw_d, cut, n, l, dgates + at, dinputs + at, p.channels, q.ok);
        }
    }
    if (q.ok && q.w == 0) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            if (MODE == kSummary) pairs[q.split * lanes + q.index + v] = make_float2(sum_a[v], carry[v]);
            else if (q.split == 0 && dstate != nullptr) dstate[q.index + v] = carry[v];
        }
    }
}

}  // namespace puff

#include "puff_recurrence_tma.cuh"

namespace puff {
// One step of every row; new_state may be state.  VEC adjacent channels a thread: four where everything is aligned for it
// (16 bytes of state), which leaves the launch and one round trip to memory.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
puff_recurrence_step_kernel(const T* __restrict__ gates, const T* __restrict__ inputs, const float* state,
                            const void* __restrict__ resets, int reset_bytes, long long batch, long long channels,
                            long long gates_stride, long long inputs_stride, T* __restrict__ outputs, float* new_state)
{
    struct alignas(VEC * sizeof(T)) Group {
        T v[VEC];
    };
    struct alignas(VEC * 4) StateGroup {
        float v[VEC];
    };
    const long long groups = channels / VEC, n = batch * groups, stride = static_cast<long long>(gridDim.x) * 256;
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < n; i += stride) {
        const long long b = quotient(i, groups), c = (i - b * groups) * VEC;
        const Group gate = *reinterpret_cast<const Group*>(gates + b * gates_stride + c);
        const Group input = *reinterpret_cast<const Group*>(inputs + b * inputs_stride + c);
        const StateGroup before = *reinterpret_cast<const StateGroup*>(state + i * VEC);
        bool reset = false;
        if (reset_bytes == 4) reset = static_cast<const float*>(resets)[b] != 0.0f;
        else if (reset_bytes == 1) reset = static_cast<const unsigned char*>(resets)[b] != 0;
        Group out;
        StateGroup after;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            float g[1] = {to_f32(gate.v[v])}, code[1], keep[1], take[1];
            gate_codes<T>(g, code);
            gate_pairs(code, keep, take);
            const float fresh = take[0] * to_f32(input.v[v]);
            after.v[v] = reset ? fresh : fmaf(keep[0], before.v[v], fresh);
            out.v[v] = from_f32<T>(after.v[v]);
        }
        *reinterpret_cast<StateGroup*>(new_state + i * VEC) = after;
        *reinterpret_cast<Group*>(outputs + i * VEC) = out;
    }
}

// Up to eight steps, N of them known to the compiler: a thread takes VEC adjacent channels through all of them, every input
// asked for before the first is used.  Two channels where everything is aligned for them, one otherwise.  Against the tiles
// of sixteen, which compute steps that are not there (us, tiles / here, forward and backward): 6525 x 1 x 1888 bf16 274 / 56
// and 370 / 56, x 8 x 1888 277 / 175 and 384 / 288, x 4 x 1891 629 / 137 and 684 / 184, 700000 x 8 x 18 1141 / 193 and
// 1249 / 316.  With one kernel of eight steps and a branch at each 175 and 288 were 240 and 604; four channels a thread
// are faster forward (8 steps 164) and slower backward (326).
constexpr int kRecShort = 8;
template <typename T, int VEC> struct alignas(VEC * sizeof(T)) Adjacent {
    T v[VEC];
};
template <typename T, int VEC, int N>
__device__ __forceinline__ void load_short(Adjacent<T, VEC> (&to)[N], const T* from, long long stride)
{
#pragma unroll
    for (int j = 0; j < N; ++j, from += stride)
        to[j] = *reinterpret_cast<const Adjacent<T, VEC>*>(from);
}
template <int VEC>
__device__ __forceinline__ Adjacent<float, VEC> load_or_zero(const float* from, long long at)
{
    Adjacent<float, VEC> a = {};
    if (from != nullptr) a = *reinterpret_cast<const Adjacent<float, VEC>*>(from + at);
    return a;
}
template <int N>
__device__ __forceinline__ unsigned resets_short(const RecArgs& p, long long b)
{
    unsigned cut = 0;
    if (p.reset_bytes != 0)
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (is_reset(p, b * N + j)) cut |= 1u << j;
    return cut;
}
template <typename T, int VEC, int N>
__global__ void __launch_bounds__(256)
puff_recurrence_short_kernel(RecArgs p, T* __restrict__ outputs, float* __restrict__ final_state, float* __restrict__ saved)
{
    const long long groups = p.channels / VEC, n = p.batch * groups, stride = static_cast<long long>(gridDim.x) * 256;
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < n; i += stride) {
        const long long b = quotient(i, groups), c = (i - b * groups) * VEC;
        Adjacent<T, VEC> gate[N], input[N];
        load_short(gate, static_cast<const T*>(p.gates) + b * p.gates_batch_stride + c, p.gates_step_stride);
        load_short(input, static_cast<const T*>(p.inputs) + b * p.inputs_batch_stride + c, p.inputs_step_stride);
        Adjacent<float, VEC> h = load_or_zero<VEC>(p.state, i * VEC);
        const unsigned cut = resets_short<N>(p, b);
        if (saved != nullptr) *reinterpret_cast<Adjacent<float, VEC>*>(saved + i * VEC) = h;
        T* out = outputs + b * N * p.channels + c;
#pragma unroll
        for (int j = 0; j < N; ++j, out += p.channels) {
            Adjacent<T, VEC> o;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float g[1] = {to_f32(gate[j].v[v])}, code[1], keep[1], take[1];
                gate_codes<T>(g, code);
                gate_pairs(code, keep, take);
                const float fresh = take[0] * to_f32(input[j].v[v]);
                h.v[v] = cut >> j & 1u ? fresh : fmaf(keep[0], h.v[v], fresh);
                o.v[v] = from_f32<T>(h.v[v]);
            }
            *reinterpret_cast<Adjacent<T, VEC>*>(out) = o;
        }
        *reinterpret_cast<Adjacent<float, VEC>*>(final_state + i * VEC) = h;
    }
}
template <typename T, int VEC, int N>
__global__ void __launch_bounds__(256)
puff_recurrence_backward_short_kernel(RecArgs p, const float* __restrict__ saved, const T* __restrict__ doutputs,
                                      const float* __restrict__ dfinal, T* __restrict__ dgates, T* __restrict__ dinputs,
                                      float* __restrict__ dstate)
{
    const long long groups = p.channels / VEC, n = p.batch * groups, stride = static_cast<long long>(gridDim.x) * 256;
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < n; i += stride) {
        const long long b = quotient(i, groups), c = (i - b * groups) * VEC, at = b * N * p.channels + c;
        Adjacent<T, VEC> gate[N], input[N], dout[N];
        load_short(gate, static_cast<const T*>(p.gates) + b * p.gates_batch_stride + c, p.gates_step_stride);
        load_short(input, static_cast<const T*>(p.inputs) + b * p.inputs_batch_stride + c, p.inputs_step_stride);
        if (doutputs != nullptr) load_short(dout, doutputs + at, p.channels);
        const Adjacent<float, VEC> before = load_or_zero<VEC>(saved, i * VEC);
        Adjacent<float, VEC> lam = load_or_zero<VEC>(dfinal, i * VEC);
        const unsigned cut = resets_short<N>(p, b);
        float h[VEC], code[N][VEC], slope[N][VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) h[v] = before.v[v];
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float x = to_f32(input[j].v[v]);
                float g[1] = {to_f32(gate[j].v[v])}, cd[1], keep[1], take[1];
                gate_codes<T>(g, cd);
                gate_pairs(cd, keep, take);
                if (cut >> j & 1u) h[v] = 0.0f;
                code[j][v] = cd[0];
                slope[j][v] = keep[0] * take[0] * (h[v] - x);
                h[v] = cut >> j & 1u ? take[0] * x : fmaf(keep[0], h[v], take[0] * x);
            }
#pragma unroll
        for (int j = N - 1; j >= 0; --j) {
            Adjacent<T, VEC> dx, dg;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float cd[1] = {code[j][v]}, keep[1], take[1];
                gate_pairs(cd, keep, take);
                if (doutputs != nullptr) lam.v[v] += to_f32(dout[j].v[v]);
                dx.v[v] = from_f32<T>(lam.v[v] * take[0]);
                dg.v[v] = from_f32<T>(lam.v[v] * slope[j][v]);
                lam.v[v] = cut >> j & 1u ? 0.0f : lam.v[v] * keep[0];
            }
            *reinterpret_cast<Adjacent<T, VEC>*>(dinputs + at + j * p.channels) = dx;
            *reinterpret_cast<Adjacent<T, VEC>*>(dgates + at + j * p.channels) = dg;
        }
        if (dstate != nullptr) *reinterpret_cast<Adjacent<float, VEC>*>(dstate + i * VEC) = lam;
    }
}

// bytes from the first to one past the last element of a [batch, steps, channels] view
static long long view_span(long long batch, long long steps, long long channels, long long bs, long long ss, int size)
{
    return ((batch - 1) * bs + (steps - 1) * ss + channels) * size;
}

// Two CTAs of eight warps are resident on each of 148 SMs.  Tiles along the steps go to several warps of a CTA while a
// warp a lane block would leave more than a fifth of that idle, then ranges of steps to several CTAs, as many as one wave
// holds; the second costs reading the inputs twice.
constexpr long long kRecSlots = 148 * 2;
constexpr int kRecMaxSplits = 148;
static RecPlan rec_plan(long long batch, long long steps, long long channels, int vec, bool flat)
{
    RecPlan plan;
    plan.shares = 1;
    plan.blocks_per_row = (channels + 32 * vec - 1) / (32 * vec);
    plan.lane_blocks = flat ? (batch * channels + 31) / 32 : batch * plan.blocks_per_row;
    const long long tiles = (steps + kRecTile - 1) / kRecTile;
    plan.warps = 1;
    while (plan.warps < kRecWarps && plan.warps < tiles && plan.lane_blocks * plan.warps * 5 < kRecSlots * kRecWarps * 4) plan.warps *= 2;
    const long long rounds = (tiles + plan.warps - 1) / plan.warps;
    long long splits = 1;
    if (plan.warps == kRecWarps) splits = kRecSlots / plan.lane_blocks;
    // a range of one round would spend its time on the join
    if (splits > rounds / 2) splits = rounds / 2;
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
static cudaError_t rec_launch(void (*summary)(KArgs...), void (*kernel)(KArgs...), size_t smem, const RecPlan& plan, cudaStream_t st,
                              const Args&... args)
{
    const int grid = rec_grid(plan);
    if (smem > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (e == cudaSuccess && summary != nullptr)
            e = cudaFuncSetAttribute(summary, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (e != cudaSuccess) return e;
    }
    if (summary == nullptr) {
        kernel<<<grid, kRecThreads, smem, st>>>(static_cast<KArgs>(args)...);
        count_launch();
        return cudaGetLastError();
    }
    summary<<<grid, kRecThreads, smem, st>>>(static_cast<KArgs>(args)...);
    count_launch();
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    count_launch();
    return launch_neighbour(kernel, grid, kRecThreads, smem, st, args...);
}
// One launch of clusters of plan.shares CTAs
template <typename... KArgs, typename... Args>
static cudaError_t rec_launch_cluster(void (*kernel)(KArgs...), size_t smem, const RecPlan& plan, cudaStream_t st, const Args&... args)
{
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(plan.lane_blocks * plan.shares));
    cfg.blockDim = dim3(kRecThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(plan.shares);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    count_launch();
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}
// Turns ranges into clusters of two or four where those fill most of one wave.  Measured, ranges / clusters, us forward, bf16:
// 256 CTAs 4 x 8192 x 1024 92 / 70, 280 140 x 3000 x 64 77 / 55, 192 3 x 4000 x 1024 42 / 39, but 160 5 x 10000 x 1024 138 /
// 150, and clusters of eight, which do not all find room at once, 1 x 20000 x 2368 112 / 136.
static RecPlan with_cluster(RecPlan plan, long long steps)
{
    if (plan.splits == 1) return plan;
    const int shares = plan.lane_blocks * 4 <= kRecSlots ? 4 : 2;
    if (plan.lane_blocks * shares > kRecSlots || plan.lane_blocks * shares < 190 || steps < 2LL * shares * kRecWarps * kRecTile) return plan;
    plan.shares = shares;
    plan.splits = 1;
    plan.split_steps = steps;
    return plan;
}
// channels too few to fill half a warp's lanes: rows share warps
static bool rec_flat(long long channels, int vec) { return channels < 16 * vec; }

// do `vec` adjacent channels of the inputs stay together, and aligned, in every row?
static bool together(const RecArgs& p, int size, int vec)
{
    return p.channels % vec == 0 && p.gates_batch_stride % vec == 0 && p.gates_step_stride % vec == 0 && p.inputs_batch_stride % vec == 0 &&
           p.inputs_step_stride % vec == 0 && !misaligned(p.gates, static_cast<unsigned>(vec * size)) &&
           !misaligned(p.inputs, static_cast<unsigned>(vec * size));
}
static int short_grid(const RecArgs& p, int vec)
{
    const long long blocks = (p.batch * p.channels / vec + 255) / 256;
    return static_cast<int>(blocks < (1 << 30) ? blocks : (1 << 30));
}
// the kernel of N steps, from N = 1 on
template <typename T, int N = 1>
static cudaError_t launch_short(const RecArgs& p, void* outputs, float* final_state, float* saved, cudaStream_t st)
{
    if constexpr (N < kRecShort)
        if (p.steps > N) return launch_short<T, N + 1>(p, outputs, final_state, saved, st);
    constexpr int V = 2;
    const unsigned bytes = V * sizeof(T);
    if (together(p, sizeof(T), V) && !misaligned(outputs, bytes) && !misaligned(p.state, 4 * V) && !misaligned(final_state, 4 * V) &&
        !misaligned(saved, 4 * V))
        puff_recurrence_short_kernel<T, V, N><<<short_grid(p, V), 256, 0, st>>>(p, static_cast<T*>(outputs), final_state, saved);
    else
        puff_recurrence_short_kernel<T, 1, N><<<short_grid(p, 1), 256, 0, st>>>(p, static_cast<T*>(outputs), final_state, saved);
    count_launch();
    return cudaGetLastError();
}
template <typename T, int N = 1>
static cudaError_t launch_backward_short(const RecArgs& p, const float* saved, const void* doutputs, const float* dfinal, void* dgates,
                                         void* dinputs, float* dstate, cudaStream_t st)
{
    if constexpr (N < kRecShort)
        if (p.steps > N) return launch_backward_short<T, N + 1>(p, saved, doutputs, dfinal, dgates, dinputs, dstate, st);
    constexpr int V = 2;
    const unsigned bytes = V * sizeof(T);
    const T* d = static_cast<const T*>(doutputs);
    T *dg = static_cast<T*>(dgates), *dx = static_cast<T*>(dinputs);
    if (together(p, sizeof(T), V) && !misaligned(d, bytes) && !misaligned(dg, bytes) && !misaligned(dx, bytes) &&
        !misaligned(saved, 4 * V) && !misaligned(dfinal, 4 * V) && !misaligned(dstate, 4 * V))
        puff_recurrence_backward_short_kernel<T, V, N><<<short_grid(p, V), 256, 0, st>>>(p, saved, d, dfinal, dg, dx, dstate);
    else
        puff_recurrence_backward_short_kernel<T, 1, N><<<short_grid(p, 1), 256, 0, st>>>(p, saved, d, dfinal, dg, dx, dstate);
    count_launch();
    return cudaGetLastError();
}

static int check_recurrence(const RecArgs& p, int dtype)
{
    const int size = dtype_bytes(dtype);
    if (size == 0) return PUFF_ERR_DTYPE;
    if (p.batch < 0 || p.steps < 0 || p.channels < 0 || p.gates_batch_stride < 0 || p.gates_step_stride < 0 ||
        p.inputs_batch_stride < 0 || p.inputs_step_stride < 0)
        return PUFF_ERR_SHAPE;
    if (p.resets != nullptr && p.reset_bytes != 1 && p.reset_bytes != 4) return PUFF_ERR_DTYPE;
    if (p.batch > 0 && p.channels > (1LL << 36) / p.batch) return PUFF_ERR_SIZE;
    const long long lanes = p.batch * p.channels;
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
                 inputs_batch_stride, inputs_step_stride, resets != nullptr ? reset_bytes : 0, 0u};
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
    if (steps > 0 && steps <= kRecShort) {
        cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
        return static_cast<int>(dtype == PUFF_DTYPE_F32   ? launch_short<float>(p, outputs, final_state, saved, st)
                                : dtype == PUFF_DTYPE_F16 ? launch_short<__half>(p, outputs, final_state, saved, st)
                                                          : launch_short<__nv_bfloat16>(p, outputs, final_state, saved, st));
    }
    // two channels a lane where every address of the 16-bit tensors stays 4-byte aligned
    const bool pair = size == 2 && channels % 2 == 0 && gates_batch_stride % 2 == 0 && gates_step_stride % 2 == 0 &&
                      inputs_batch_stride % 2 == 0 && inputs_step_stride % 2 == 0 && !misaligned(gates, 4) &&
                      !misaligned(inputs, 4) && !misaligned(outputs, 4) && !rec_flat(channels, 2);
    const bool flat = rec_flat(channels, 1);
    const ViewStrides gs = {gates_batch_stride, gates_step_stride}, xs = {inputs_batch_stride, inputs_step_stride};
    const ViewStrides dense = {steps * channels, channels};
    CUtensorMap mg, mx, mo;
    const bool tma = tma_shape(p, size) && tma_view(p, gates, gs, size) && tma_view(p, inputs, xs, size) &&
                     tma_view(p, outputs, dense, size) && tma_map(&mg, p, gates, gs, dtype) && tma_map(&mx, p, inputs, xs, dtype) &&
                     tma_map(&mo, p, outputs, dense, dtype);
    RecPlan plan = rec_plan(batch, steps, channels, tma ? 4 / size : pair ? 2 : 1, flat);
    if (tma) plan = with_cluster(plan, steps);
    float2* pairs = static_cast<float2*>(scratch);
    cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    cudaError_t e;
    if (tma) {
        int* status = device_status_ptr();
        if (status == nullptr) return PUFF_ERR_DRIVER;
        p.wait_ns = tile_wait_ns();
        const size_t smem = tma_smem(2, kTmaForwardStages);
#define PUFF_RUN2(T, VEC)                                                                                                \
    (plan.shares > 1                                                                                                     \
         ? rec_launch_cluster(puff_recurrence_tma_kernel<T, VEC, kCluster>, smem, plan, st, mg, mx, mo, p, plan, pairs,   \
                              final_state, saved, status)                                                                \
         : rec_launch(plan.splits > 1 ? puff_recurrence_tma_kernel<T, VEC, kSummary> : nullptr,                           \
                      plan.warps > 1 ? puff_recurrence_tma_kernel<T, VEC, kTeam> : puff_recurrence_tma_kernel<T, VEC, kStream>, \
                      smem, plan, st, mg, mx, mo, p, plan, pairs, final_state, saved, status))
        e = dtype == PUFF_DTYPE_F32 ? PUFF_RUN2(float, 1) : dtype == PUFF_DTYPE_F16 ? PUFF_RUN2(__half, 2) : PUFF_RUN2(__nv_bfloat16, 2);
#undef PUFF_RUN2
        return static_cast<int>(e);
    }
#define PUFF_RUN2(T, VEC, FLAT)                                                                                          \
    rec_launch(plan.splits > 1 ? puff_recurrence_kernel<T, VEC, FLAT, kSummary> : nullptr,                                \
               plan.warps > 1 ? puff_recurrence_kernel<T, VEC, FLAT, kTeam> : puff_recurrence_kernel<T, VEC, FLAT, kStream>, \
               size_t{0}, plan, st, p, plan, pairs, static_cast<T*>(outputs), final_state, saved)
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
                 inputs_batch_stride, inputs_step_stride, resets != nullptr ? reset_bytes : 0, 0u};
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
    if (steps > 0 && steps <= kRecShort) {
        cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
        return static_cast<int>(
            dtype == PUFF_DTYPE_F32   ? launch_backward_short<float>(p, saved, doutputs, dfinal, dgates, dinputs, dstate, st)
            : dtype == PUFF_DTYPE_F16 ? launch_backward_short<__half>(p, saved, doutputs, dfinal, dgates, dinputs, dstate, st)
                                      : launch_backward_short<__nv_bfloat16>(p, saved, doutputs, dfinal, dgates, dinputs, dstate, st));
    }
    const bool pair = size == 2 && channels % 2 == 0 && gates_batch_stride % 2 == 0 && gates_step_stride % 2 == 0 &&
                      inputs_batch_stride % 2 == 0 && inputs_step_stride % 2 == 0 && !misaligned(gates, 4) &&
                      !misaligned(inputs, 4) && !misaligned(doutputs, 4) && !misaligned(dgates, 4) &&
                      !misaligned(dinputs, 4) && !rec_flat(channels, 2);
    const bool flat = rec_flat(channels, 1);
    const ViewStrides gs = {gates_batch_stride, gates_step_stride}, xs = {inputs_batch_stride, inputs_step_stride};
    const ViewStrides dense = {steps * channels, channels};
    CUtensorMap mg, mx, md, mdg, mdx;
    const bool tma = tma_shape(p, size) && tma_view(p, gates, gs, size) && tma_view(p, inputs, xs, size) &&
                     tma_view(p, doutputs, dense, size) && tma_view(p, dgates, dense, size) && tma_view(p, dinputs, dense, size) &&
                     tma_map(&mg, p, gates, gs, dtype) && tma_map(&mx, p, inputs, xs, dtype) && tma_map(&md, p, doutputs, dense, dtype) &&
                     tma_map(&mdg, p, dgates, dense, dtype) && tma_map(&mdx, p, dinputs, dense, dtype);
    RecPlan plan = rec_plan(batch, steps, channels, tma ? 4 / size : pair ? 2 : 1, flat);
    if (tma) plan = with_cluster(plan, steps);
    float2* pairs = static_cast<float2*>(scratch);
    cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    cudaError_t e;
    if (tma) {
        int* status = device_status_ptr();
        if (status == nullptr) return PUFF_ERR_DRIVER;
        p.wait_ns = tile_wait_ns();
        const size_t smem = tma_smem(3, kTmaBackwardStages);
#define PUFF_RUN2(T, VEC)                                                                                                \
    (plan.shares > 1                                                                                                     \
         ? rec_launch_cluster(puff_recurrence_backward_tma_kernel<T, VEC, kCluster>, smem, plan, st, mg, mx, md, mdg, mdx, \
                              p, plan, pairs, saved, dfinal, dstate, status)                                             \
         : rec_launch(plan.splits > 1 ? puff_recurrence_backward_tma_kernel<T, VEC, kSummary> : nullptr,                  \
                      plan.warps > 1 ? puff_recurrence_backward_tma_kernel<T, VEC, kTeam>                                 \
                                     : puff_recurrence_backward_tma_kernel<T, VEC, kStream>,                              \
                      smem, plan, st, mg, mx, md, mdg, mdx, p, plan, pairs, saved, dfinal, dstate, status))
        e = dtype == PUFF_DTYPE_F32 ? PUFF_RUN2(float, 1) : dtype == PUFF_DTYPE_F16 ? PUFF_RUN2(__half, 2) : PUFF_RUN2(__nv_bfloat16, 2);
#undef PUFF_RUN2
        return static_cast<int>(e);
    }
#define PUFF_RUN2(T, VEC, FLAT)                                                                                          \
    rec_launch(plan.splits > 1 ? puff_recurrence_backward_kernel<T, VEC, FLAT, kSummary> : nullptr,                       \
               plan.warps > 1 ? puff_recurrence_backward_kernel<T, VEC, FLAT, kTeam>                                      \
                              : puff_recurrence_backward_kernel<T, VEC, FLAT, kStream>,                                   \
               size_t{0}, plan, st, p, plan, pairs, saved, static_cast<const T*>(doutputs), dfinal,                       \
               static_cast<T*>(dgates), static_cast<T*>(dinputs), dstate)
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
                 resets != nullptr ? reset_bytes : 0, 0u};
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
    const bool four = channels % 4 == 0 && gates_stride % 4 == 0 && inputs_stride % 4 == 0 && !misaligned(gates, 4u * size) &&
                      !misaligned(inputs, 4u * size) && !misaligned(outputs, 4u * size) && !misaligned(state, 16) && !misaligned(new_state, 16);
    long long blocks = (n / (four ? 4 : 1) + 255) / 256;
    if (blocks > 16LL * sms) blocks = 16LL * sms;
    cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
#define PUFF_RUN2(T, VEC)                                                                                                \
    puff_recurrence_step_kernel<T, VEC><<<static_cast<int>(blocks), 256, 0, st>>>(static_cast<const T*>(gates),           \
        static_cast<const T*>(inputs), state, resets, p.reset_bytes, batch, channels, gates_stride, inputs_stride,        \
        static_cast<T*>(outputs), new_state)
    if (dtype == PUFF_DTYPE_F32) {
        if (four) PUFF_RUN2(float, 4);
        else PUFF_RUN2(float, 1);
    } else if (dtype == PUFF_DTYPE_F16) {
        if (four) PUFF_RUN2(__half, 4);
        else PUFF_RUN2(__half, 1);
    } else {
        if (four) PUFF_RUN2(__nv_bfloat16, 4);
        else PUFF_RUN2(__nv_bfloat16, 1);
    }
#undef PUFF_RUN2
    count_launch();
    return static_cast<int>(cudaGetLastError());
}
