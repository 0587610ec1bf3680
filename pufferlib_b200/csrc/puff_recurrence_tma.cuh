// The gated recurrence with its tiles moved by TMA: what every shape takes whose rows are 16-byte aligned.  A tile is 16
// steps of 32 lanes (128 bytes a step, 2 KB), fetched and written by one instruction of one lane where the plain kernels
// spend several on every step's address; results go into the shared memory their inputs came from.  Every warp runs its
// own ring, so warps meet only where a group joins its pairs.  Included by puff_recurrence_sm100.cu only.
#pragma once
#include <cuda.h>

namespace puff {

constexpr int kTmaTileBytes = kRecTile * 128;
constexpr int kTmaForwardStages = 3, kTmaBackwardStages = 2;

// every wait is bounded: 2^24 polls or kTileWaitNs
constexpr unsigned kTileWaitNs = 2000000000u;
struct TileBarrier {
    uint32_t at;
    __device__ __forceinline__ void init() const { asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(at) : "memory"); }
    __device__ __forceinline__ void expect(uint32_t bytes) const
    {
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(at), "r"(bytes) : "memory");
    }
    __device__ __forceinline__ bool passed(uint32_t parity, unsigned hint_ns) const
    {
        uint32_t ok;
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\nselp.u32 %0, 1, 0, p;\n}\n"
                     : "=r"(ok) : "r"(at), "r"(parity), "r"(hint_ns) : "memory");
        return ok != 0;
    }
    // (with no time at all it does not even look, so that a test gives up whatever has arrived)
    __device__ __forceinline__ bool wait(uint32_t parity, unsigned limit_ns) const
    {
        const unsigned hint = limit_ns < 200000u ? limit_ns : 200000u;
        if (limit_ns == 0) return false;
        if (passed(parity, hint)) return true;
        unsigned long long start, now;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(start));
        for (uint32_t polls = 0; polls < (1u << 24); ++polls) {
            if (passed(parity, hint)) return true;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
            if (now - start > limit_ns) break;
        }
        return false;
    }
};
__device__ __forceinline__ void tile_load(uint32_t to, const CUtensorMap* map, int c, int t, int b, TileBarrier bar)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(to),
                 "l"(map), "r"(c), "r"(t), "r"(b), "r"(bar.at) : "memory");
}
__device__ __forceinline__ void tile_store(const CUtensorMap* map, int c, int t, int b, uint32_t from)
{
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(c), "r"(t), "r"(b),
                 "r"(from) : "memory");
}
__device__ __forceinline__ void tile_store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void tile_store_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
// this lane's shared-memory accesses before the async copies that follow
__device__ __forceinline__ void tile_fence()
{
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
}

// every CTA of the cluster has begun: their shared memory may be written
__device__ __forceinline__ void cluster_runs()
{
    __syncwarp();
    cooperative_groups::this_cluster().sync();
}

// a lane's word of every step of a tile
template <typename Raw>
struct TmaTile {
    const uint32_t* word;
    __device__ __forceinline__ Raw operator[](int j) const { return *reinterpret_cast<const Raw*>(word + 32 * j); }
};

// shared memory of a CTA: the warps' rings, each tile 128-byte aligned, then their barriers
constexpr size_t tma_smem(int arrays, int stages) { return static_cast<size_t>(kRecWarps) * stages * (arrays * kTmaTileBytes + 8) + 128; }
template <int ARRAYS, int STAGES>
struct TileRing {
    char* tiles;       // of this warp
    uint32_t tiles_at, bars_at;
    __device__ __forceinline__ TileRing(char* smem)
    {
        const uint32_t raw = static_cast<uint32_t>(__cvta_generic_to_shared(smem)), up = (128u - (raw & 127u)) & 127u;
        const int warp = threadIdx.x >> 5;
        tiles = smem + up + warp * (STAGES * ARRAYS * kTmaTileBytes);
        tiles_at = raw + up + warp * (STAGES * ARRAYS * kTmaTileBytes);
        bars_at = raw + up + kRecWarps * (STAGES * ARRAYS * kTmaTileBytes) + warp * STAGES * 8;
    }
    __device__ __forceinline__ TileBarrier bar(int stage) const { return {bars_at + stage * 8}; }
    __device__ __forceinline__ uint32_t at(int stage, int array) const { return tiles_at + (stage * ARRAYS + array) * kTmaTileBytes; }
    __device__ __forceinline__ uint32_t* words(int stage, int array) const
    {
        return reinterpret_cast<uint32_t*>(tiles + (stage * ARRAYS + array) * kTmaTileBytes) + (threadIdx.x & 31);
    }
    __device__ __forceinline__ void init() const
    {
        if ((threadIdx.x & 31) == 0) {
            for (int s = 0; s < STAGES; ++s) bar(s).init();
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        tile_fence();
    }
    // The warp waits for its tile in `stage`.  If one of its lanes gives up, all do: the status word is set, nothing is
    // requested or waited for any more (what the kernel computes from then on counts for nothing, but the other warps of
    // its group meet it at their joins), and first what is in flight has to arrive, this tile and, if `next`, the one
    // behind it: it writes to shared memory, which must not be left before.
    __device__ __forceinline__ void wait(int stage, uint32_t phase, bool next, unsigned limit_ns, bool& given_up, int* status) const
    {
        if (given_up) return;
        const bool ok = bar(stage).wait(phase, limit_ns);
        if (__all_sync(0xffffffffu, ok)) return;
        given_up = true;
        if ((threadIdx.x & 31) == 0) atomicExch(status, PUFF_ERR_DEVICE_WAIT);
        bar(stage).wait(phase, kTileWaitNs);
        if (next) bar(stage == STAGES - 1 ? 0 : stage + 1).wait(stage == STAGES - 1 ? phase ^ 1u : phase, kTileWaitNs);
        __syncwarp();
    }
};
static unsigned tile_wait_ns()
{
    const int us = tune_value(PUFF_TUNE_TILE_WAIT_US, -1);
    return us < 0 || us > 2000000 ? kTileWaitNs : 1000u * static_cast<unsigned>(us);
}

// Forward: three stages, so that two tiles are on their way while one is worked on; the states take the inputs' place.
template <typename T, int VEC, RecMode MODE>
__global__ void __launch_bounds__(kRecThreads, 2)
puff_recurrence_tma_kernel(const __grid_constant__ CUtensorMap gates, const __grid_constant__ CUtensorMap inputs,
                           const __grid_constant__ CUtensorMap outputs, RecArgs p, RecPlan plan, float2* pairs,
                           float* __restrict__ final_state, float* __restrict__ saved, int* status)
{
    using Raw = typename Lane<T, VEC>::Raw;
    constexpr int S = kTmaForwardStages;
    extern __shared__ char s_ring[];
    __shared__ float2 s_pair[MODE == kStream || MODE == kCluster ? 1 : 2][MODE == kStream ? 1 : kRecWarps][VEC][32];
    __shared__ float2 s_cta[MODE == kCluster ? 2 : 1][MODE == kCluster ? 4 : 1][VEC][32];
    const RecPlace q = rec_place<VEC, false>(p, plan);
    const TileRing<2, S> ring(s_ring);
    ring.init();
    if (MODE != kSummary) pdl_wait();
    if (!q.unit) return;
    const long long lanes = p.batch * p.channels;
    const long long tiles = (p.steps + kRecTile - 1) / kRecTile;
    const int step = kRecTile * plan.warps * plan.shares, c0 = static_cast<int>(q.c) - q.lane * VEC, b0 = static_cast<int>(q.b);
    const int t_end = static_cast<int>(q.t_end), t_begin = static_cast<int>(q.t_begin);
    bool given_up = false;
    auto request = [&](int t, int stage) {      // the tile of this warp in the round that begins at t
        if (q.lane == 0 && t < t_end && !given_up) {
            const TileBarrier bar = ring.bar(stage);
            bar.expect(2 * kTmaTileBytes);
            tile_load(ring.at(stage, 0), &gates, c0, t + q.slot * kRecTile, b0, bar);
            tile_load(ring.at(stage, 1), &inputs, c0, t + q.slot * kRecTile, b0, bar);
        }
    };
    request(t_begin, 0);
    request(t_begin + step, 1);
    if (MODE == kCluster) cluster_runs();
    float carry[VEC], sum_a[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        carry[v] = MODE != kSummary && q.ok && p.state != nullptr ? p.state[q.index + v] : 0.0f;
        sum_a[v] = 1.0f;
    }
    long long t0 = q.t_begin + q.slot * kRecTile;
    unsigned resets = resets_ahead<false>(p, q, t0, q.steps_at(t0));
    if (MODE == kTeam)
        for (int r = 0; r < q.split; ++r)
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                if (q.ok) carry[v] = apply_pair(pairs[r * lanes + q.index + v], carry[v]);
    float* save = saved != nullptr ? saved + (q.b * tiles + t0 / kRecTile) * p.channels + q.c : nullptr;
    int stage = 0, parity = 0;
    uint32_t phase = 0;
    for (int t = t_begin; t < t_end; t += step, t0 += step, parity ^= 1) {
        const int n = q.steps_at(t0);
        const unsigned cut = reset_mask<false>(p, resets);
        const bool plain = n == kRecTile && cut == 0;
        resets = resets_ahead<false>(p, q, t0 + step, q.steps_at(t0 + step));
        ring.wait(stage, phase, t + step < t_end, p.wait_ns, given_up, status);
        uint32_t* const g_words = ring.words(stage, 0);
        uint32_t* const x_words = ring.words(stage, 1);
        const TmaTile<Raw> raw_g = {g_words}, raw_x = {x_words};
        T* const out = reinterpret_cast<T*>(x_words);
        if (MODE == kStream) {
            if (save != nullptr && q.ok)
#pragma unroll
                for (int v = 0; v < VEC; ++v) save[v] = carry[v];
            if (plain) forward_stream<T, VEC, true>(raw_g, raw_x, cut, n, carry, out, 32 * VEC, true);
            else forward_stream<T, VEC, false>(raw_g, raw_x, cut, n, carry, out, 32 * VEC, true);
        } else {
            float keep[kRecTile][VEC], fresh[kRecTile][VEC], a[VEC], b[VEC], h[VEC];
            if (plain) forward_pair<T, VEC, true>(raw_g, raw_x, cut, n, keep, fresh, a, b);
            else forward_pair<T, VEC, false>(raw_g, raw_x, cut, n, keep, fresh, a, b);
            if constexpr (MODE == kCluster) join_cluster<VEC, false>(s_pair[0], s_cta[parity], q, plan, cut, a, b, h, carry);
            else join_warps<VEC, MODE == kSummary, false>(s_pair[parity], q, plan.warps, cut, a, b, h, carry, sum_a);
            if (MODE != kSummary) {
                if (save != nullptr && q.ok && n > 0)
#pragma unroll
                    for (int v = 0; v < VEC; ++v) save[v] = h[v];
                if (plain) forward_states<T, VEC, true>(keep, fresh, cut, n, h, out, 32 * VEC, true);
                else forward_states<T, VEC, false>(keep, fresh, cut, n, h, out, 32 * VEC, true);
            }
        }
        tile_fence();
        if (MODE != kSummary && q.lane == 0) tile_store_read();      // the stage before this one has been read out
        request(t + 2 * step, stage == 0 ? S - 1 : stage - 1);
        if (MODE != kSummary && q.lane == 0 && n > 0) {
            tile_store(&outputs, c0, static_cast<int>(t0), b0, ring.at(stage, 1));
            tile_store_commit();
        }
        if (save != nullptr) save += step / kRecTile * p.channels;
        stage = stage == S - 1 ? 0 : stage + 1;
        phase ^= stage == 0 ? 1u : 0u;
    }
    if (q.ok && q.slot == 0) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            if (MODE == kSummary) pairs[q.split * lanes + q.index + v] = make_float2(sum_a[v], carry[v]);
            else if (q.split == plan.splits - 1) final_state[q.index + v] = carry[v];
        }
    }
    if (MODE != kSummary && q.lane == 0) tile_store_read();          // before the ring's memory goes
}

// Backward: two stages; dgates take the gates' place and dinputs the inputs'.  A stage is requested again once the tile
// after it has been through its first half, by when it has been read out.
template <typename T, int VEC, RecMode MODE>
__global__ void __launch_bounds__(kRecThreads, 2)
puff_recurrence_backward_tma_kernel(const __grid_constant__ CUtensorMap gates, const __grid_constant__ CUtensorMap inputs,
                                    const __grid_constant__ CUtensorMap doutputs, const __grid_constant__ CUtensorMap dgates,
                                    const __grid_constant__ CUtensorMap dinputs, RecArgs p, RecPlan plan, float2* pairs,
                                    const float* __restrict__ saved, const float* __restrict__ dfinal, float* __restrict__ dstate,
                                    int* status)
{
    using L = Lane<T, VEC>;
    using Raw = typename L::Raw;
    constexpr int S = kTmaBackwardStages, A = MODE == kSummary ? 2 : 3;      // gates, doutputs, inputs
    extern __shared__ char s_ring[];
    __shared__ float2 s_pair[MODE == kStream || MODE == kCluster ? 1 : 2][MODE == kStream ? 1 : kRecWarps][VEC][32];
    __shared__ float2 s_cta[MODE == kCluster ? 2 : 1][MODE == kCluster ? 4 : 1][VEC][32];
    const RecPlace q = rec_place<VEC, false>(p, plan);
    const TileRing<A, S> ring(s_ring);
    ring.init();
    if (MODE != kSummary) pdl_wait();
    if (!q.unit) return;
    const long long lanes = p.batch * p.channels;
    const long long tiles = (p.steps + kRecTile - 1) / kRecTile;
    const int step = kRecTile * plan.warps * plan.shares, c0 = static_cast<int>(q.c) - q.lane * VEC, b0 = static_cast<int>(q.b);
    const int t_begin = static_cast<int>(q.t_begin);
    const int first = t_begin + (static_cast<int>(q.t_end) - t_begin - 1) / step * step;
    bool given_up = false;
    auto request = [&](int t, int stage) {
        if (q.lane == 0 && t >= t_begin && !given_up) {
            const TileBarrier bar = ring.bar(stage);
            bar.expect(A * kTmaTileBytes);
            tile_load(ring.at(stage, 0), &gates, c0, t + q.slot * kRecTile, b0, bar);
            if (MODE != kSummary) tile_load(ring.at(stage, A - 1), &inputs, c0, t + q.slot * kRecTile, b0, bar);
            tile_load(ring.at(stage, 1), &doutputs, c0, t + q.slot * kRecTile, b0, bar);
        }
    };
    request(first, 0);
    request(first - step, 1);
    if (MODE == kCluster) cluster_runs();
    float carry[VEC], sum_a[VEC], h_next[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        carry[v] = MODE != kSummary && q.ok && dfinal != nullptr ? dfinal[q.index + v] : 0.0f;
        sum_a[v] = 1.0f;
    }
    auto saved_before = [&](long long at) {
#pragma unroll
        for (int v = 0; v < VEC; ++v)
            h_next[v] = MODE != kSummary && q.ok && at >= q.t_begin && at < q.t_end ? saved[(q.b * tiles + at / kRecTile) * p.channels + q.c + v] : 0.0f;
    };
    saved_before(first + q.slot * kRecTile);
    unsigned resets = resets_ahead<false>(p, q, first + q.slot * kRecTile, q.steps_at(first + q.slot * kRecTile));
    if (MODE == kTeam)
        for (int r = plan.splits - 1; r > q.split; --r)
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                if (q.ok) carry[v] = apply_pair(pairs[r * lanes + q.index + v], carry[v]);
    int stage = 0;
    uint32_t phase = 0;
    for (int t = first; t >= t_begin; t -= step) {
        const int t0 = t + q.slot * kRecTile, t1 = t0 - step;
        const int n = q.steps_at(t0);
        const unsigned cut = reset_mask<false>(p, resets);
        float h[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) h[v] = h_next[v];
        const bool plain = n == kRecTile && cut == 0;
        saved_before(t1);
        resets = t1 >= t_begin ? resets_ahead<false>(p, q, t1, q.steps_at(t1)) : 0u;
        // (the tile behind this one is requested below, but for the first round's and where nothing has to be stored first)
        ring.wait(stage, phase, t - step >= t_begin && (MODE == kSummary || t == first), p.wait_ns, given_up, status);
        const TmaTile<Raw> raw_g = {ring.words(stage, 0)}, raw_d = {ring.words(stage, 1)}, raw_x = {ring.words(stage, A - 1)};
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
        if (MODE != kSummary && t != first) {
            if (q.lane == 0) tile_store_read();
            request(t - step, stage ^ 1);
        }
        float lam[VEC];
        if (MODE != kStream) {
            float a[VEC], b[VEC];
            if (plain) backward_pair<T, VEC, true>(code, raw_d, cut, a, b);
            else backward_pair<T, VEC, false>(code, raw_d, cut, a, b);
            if constexpr (MODE == kCluster) join_cluster<VEC, true>(s_pair[0], s_cta[stage], q, plan, cut, a, b, lam, carry);
            else join_warps<VEC, MODE == kSummary, true>(s_pair[stage], q, plan.warps, cut, a, b, lam, carry, sum_a);
        }
        if (MODE != kSummary) {
            float (&l)[VEC] = MODE == kStream ? carry : lam;
            T* const dg = reinterpret_cast<T*>(ring.words(stage, 0));
            T* const dx = reinterpret_cast<T*>(ring.words(stage, A - 1));
            if (plain) backward_gradients<T, VEC, true>(code, slope, raw_d, cut, n, l, dg, dx, 32 * VEC, true);
            else backward_gradients<T, VEC, false>(code, slope, raw_d, cut, n, l, dg, dx, 32 * VEC, true);
        }
        tile_fence();
        if (MODE == kSummary) {
            request(t - 2 * step, stage);
        } else if (q.lane == 0 && n > 0) {
            tile_store(&dgates, c0, t0, b0, ring.at(stage, 0));
            tile_store(&dinputs, c0, t0, b0, ring.at(stage, A - 1));
            tile_store_commit();
        }
        stage ^= 1;
        phase ^= stage == 0 ? 1u : 0u;
    }
    if (q.ok && q.slot == 0) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            if (MODE == kSummary) pairs[q.split * lanes + q.index + v] = make_float2(sum_a[v], carry[v]);
            else if (q.split == 0 && dstate != nullptr) dstate[q.index + v] = carry[v];
        }
    }
    if (MODE != kSummary && q.lane == 0) tile_store_read();
}

// ---- host side
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// strides of a [batch, steps, channels] view in elements; those of dimensions of one entry do not matter
struct ViewStrides {
    long long batch, step;
};
static ViewStrides usual_strides(const RecArgs& p, ViewStrides s)
{
    if (p.steps == 1) s.step = p.channels;
    if (p.batch == 1) s.batch = s.step * p.steps;
    return s;
}
// whether TMA can address it: bases and strides multiples of 16 bytes, strides neither zero nor beyond 2^40 bytes
static bool tma_view(const RecArgs& p, const void* base, ViewStrides s, int size)
{
    s = usual_strides(p, s);
    return base != nullptr && !misaligned(base, 16) && s.step * size % 16 == 0 && s.batch * size % 16 == 0 && s.step > 0 && s.batch > 0 &&
           s.batch < (1LL << 40) / size && s.step < (1LL << 40) / size;
}
static bool tma_map(CUtensorMap* map, const RecArgs& p, const void* base, ViewStrides s, int dtype)
{
    const EncodeTiled encode = reinterpret_cast<EncodeTiled>(tensor_map_encoder());
    if (encode == nullptr) return false;
    s = usual_strides(p, s);
    const int size = dtype_bytes(dtype);
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(p.channels), static_cast<cuuint64_t>(p.steps), static_cast<cuuint64_t>(p.batch)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(s.step * size), static_cast<cuuint64_t>(s.batch * size)};
    const cuuint32_t box[3] = {128u / static_cast<unsigned>(size), kRecTile, 1}, ones[3] = {1, 1, 1};
    const CUtensorMapDataType type = dtype == PUFF_DTYPE_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : dtype == PUFF_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                               : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return encode(map, type, 3, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// shapes a warp's lanes fill and TMA coordinates hold
static bool tma_shape(const RecArgs& p, int size)
{
    return p.steps > 0 && p.channels * size % 16 == 0 && p.channels * size >= 64 && p.steps < (1LL << 30) && p.batch < (1LL << 31) &&
           p.channels < (1LL << 30);
}
}  // namespace puff
