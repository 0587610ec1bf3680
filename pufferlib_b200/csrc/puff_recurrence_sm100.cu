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

constexpr int kRecThreads = 128;
constexpr int kRecTile = 16;   // steps whose inputs a thread holds in registers; also the distance of the saved states

struct RecArgs {
    const void* gates;
    const void* inputs;
    const void* resets;      // [batch, steps] fp32 (reset_bytes 4) or one byte each (1); null: none
    const float* state;      // [batch, channels]; null: zeros
    long long batch, steps, channels;
    long long gates_batch_stride, gates_step_stride, inputs_batch_stride, inputs_step_stride;
    int reset_bytes;
};

__device__ __forceinline__ bool is_reset(const RecArgs& p, long long i)
{
    if (p.reset_bytes == 4) return static_cast<const float*>(p.resets)[i] != 0.0f;
    return p.reset_bytes == 1 && static_cast<const unsigned char*>(p.resets)[i] != 0;
}

// keep = sigmoid(g) and take = 1 - keep = sigmoid(-g).  The smaller of the two is e / (1 + e) with e = e^-|g|, good to
// a few ulp however small; the larger is 1 minus it, so that the two add up to 1 and the state stays a weighted mean.
__device__ __forceinline__ void gate_pair(float g, float& keep, float& take)
{
    const float e = exp2_approx(-fabsf(g) * kLog2e);
    const float small = __fdividef(e, 1.0f + e);
    const float large = 1.0f - small;
    keep = g >= 0.0f ? large : small;
    take = g >= 0.0f ? small : large;
}

// One thread per channel.  saved (nullable): the state before steps 0, 16, 32, ... as [batch, ceil(steps / 16), channels].
template <typename T>
__global__ void __launch_bounds__(kRecThreads)
puff_recurrence_kernel(RecArgs p, T* __restrict__ outputs, float* __restrict__ final_state, float* __restrict__ saved)
{
    const long long i = blockIdx.x * static_cast<long long>(kRecThreads) + threadIdx.x;
    if (i >= p.batch * p.channels) return;
    const long long b = i / p.channels, c = i - b * p.channels;
    const T* gates = static_cast<const T*>(p.gates) + b * p.gates_batch_stride + c;
    const T* inputs = static_cast<const T*>(p.inputs) + b * p.inputs_batch_stride + c;
    T* out = outputs + b * p.steps * p.channels + c;
    const long long tiles = (p.steps + kRecTile - 1) / kRecTile;
    float h = p.state != nullptr ? p.state[i] : 0.0f;
    for (long long k = 0; k < tiles; ++k) {
        if (saved != nullptr) saved[(b * tiles + k) * p.channels + c] = h;
        const long long t0 = k * kRecTile;
        const int n = static_cast<int>(p.steps - t0 < kRecTile ? p.steps - t0 : kRecTile);
        for (int j = 0; j < n; ++j) {
            const long long t = t0 + j;
            float keep, take;
            gate_pair(to_f32(gates[t * p.gates_step_stride]), keep, take);
            const float fresh = take * to_f32(inputs[t * p.inputs_step_stride]);
            h = is_reset(p, b * p.steps + t) ? fresh : fmaf(keep, h, fresh);
            out[t * p.channels] = from_f32<T>(h);
        }
    }
    final_state[i] = h;
}

template <typename T>
__global__ void __launch_bounds__(kRecThreads)
puff_recurrence_backward_kernel(RecArgs p, const float* __restrict__ saved, const T* __restrict__ doutputs,
                                const float* __restrict__ dfinal, T* __restrict__ dgates, T* __restrict__ dinputs,
                                float* __restrict__ dstate)
{
    const long long i = blockIdx.x * static_cast<long long>(kRecThreads) + threadIdx.x;
    if (i >= p.batch * p.channels) return;
    const long long b = i / p.channels, c = i - b * p.channels;
    const T* gates = static_cast<const T*>(p.gates) + b * p.gates_batch_stride + c;
    const T* inputs = static_cast<const T*>(p.inputs) + b * p.inputs_batch_stride + c;
    const long long base = b * p.steps * p.channels + c;
    const long long tiles = (p.steps + kRecTile - 1) / kRecTile;
    float lam = dfinal != nullptr ? dfinal[i] : 0.0f;
    for (long long k = tiles - 1; k >= 0; --k) {
        const long long t0 = k * kRecTile;
        const int n = static_cast<int>(p.steps - t0 < kRecTile ? p.steps - t0 : kRecTile);
        float before[kRecTile], x[kRecTile], g[kRecTile];
        unsigned cut = 0;
        float h = saved[(b * tiles + k) * p.channels + c];
#pragma unroll
        for (int j = 0; j < kRecTile; ++j) {
            x[j] = g[j] = before[j] = 0.0f;
            if (j < n) {
                const long long t = t0 + j;
                g[j] = to_f32(gates[t * p.gates_step_stride]);
                x[j] = to_f32(inputs[t * p.inputs_step_stride]);
                const bool reset = is_reset(p, b * p.steps + t);
                cut |= reset ? 1u << j : 0u;
                before[j] = reset ? 0.0f : h;
                float keep, take;
                gate_pair(g[j], keep, take);
                const float fresh = take * x[j];
                h = reset ? fresh : fmaf(keep, h, fresh);
            }
        }
#pragma unroll
        for (int j = kRecTile - 1; j >= 0; --j) {
            if (j < n) {
                const long long o = base + (t0 + j) * p.channels;
                float keep, take;
                gate_pair(g[j], keep, take);
                if (doutputs != nullptr) lam += to_f32(doutputs[o]);
                const float dx = lam * take;
                dinputs[o] = from_f32<T>(dx);
                dgates[o] = from_f32<T>(dx * keep * (before[j] - x[j]));
                lam = (cut >> j) & 1u ? 0.0f : lam * keep;
            }
        }
    }
    if (dstate != nullptr) dstate[i] = lam;
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
        gate_pair(to_f32(gates[b * gates_stride + c]), keep, take);
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

extern "C" int puff_policy_sm100_recurrence(const void* gates, const void* inputs, int dtype, const void* resets,
                                            int reset_bytes, const float* state, long long batch, long long steps,
                                            long long channels, long long gates_batch_stride,
                                            long long gates_step_stride, long long inputs_batch_stride,
                                            long long inputs_step_stride, void* outputs, float* final_state,
                                            float* saved, void* cuda_stream)
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
    const long long out_bytes = n * size, saved_bytes = 4 * puff_policy_sm100_recurrence_saved_floats(batch, steps, channels);
    if (touches_inputs(p, size, outputs, out_bytes) || touches_inputs(p, size, final_state, 4 * lanes) ||
        touches_inputs(p, size, saved, saved_bytes) || spans_overlap(outputs, out_bytes, final_state, 4 * lanes) ||
        spans_overlap(outputs, out_bytes, saved, saved_bytes) || spans_overlap(final_state, 4 * lanes, saved, saved_bytes))
        return PUFF_ERR_ALIAS;
    int sms = 0;
    rc = require_sm100(&sms);
    if (rc != PUFF_OK) return rc;
    const int grid = static_cast<int>((lanes + kRecThreads - 1) / kRecThreads);
    cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    if (dtype == PUFF_DTYPE_F32)
        puff_recurrence_kernel<float><<<grid, kRecThreads, 0, st>>>(p, static_cast<float*>(outputs), final_state, saved);
    else if (dtype == PUFF_DTYPE_F16)
        puff_recurrence_kernel<__half><<<grid, kRecThreads, 0, st>>>(p, static_cast<__half*>(outputs), final_state, saved);
    else
        puff_recurrence_kernel<__nv_bfloat16><<<grid, kRecThreads, 0, st>>>(p, static_cast<__nv_bfloat16*>(outputs), final_state, saved);
    count_launch();
    return static_cast<int>(cudaGetLastError());
}

extern "C" int puff_policy_sm100_recurrence_backward(const void* gates, const void* inputs, int dtype, const void* resets,
                                                     int reset_bytes, const float* saved, long long batch,
                                                     long long steps, long long channels, long long gates_batch_stride,
                                                     long long gates_step_stride, long long inputs_batch_stride,
                                                     long long inputs_step_stride, const void* doutputs,
                                                     const float* dfinal, void* dgates, void* dinputs, float* dstate,
                                                     void* cuda_stream)
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
    const long long saved_bytes = 4 * puff_policy_sm100_recurrence_saved_floats(batch, steps, channels);
    const void* out[3] = {dgates, dinputs, dstate};
    const long long out_bytes[3] = {n * size, n * size, 4 * lanes};
    for (int i = 0; i < 3; ++i) {
        if (touches_inputs(p, size, out[i], out_bytes[i]) || spans_overlap(out[i], out_bytes[i], saved, saved_bytes) ||
            spans_overlap(out[i], out_bytes[i], doutputs, n * size) || spans_overlap(out[i], out_bytes[i], dfinal, 4 * lanes))
            return PUFF_ERR_ALIAS;
        for (int j = 0; j < i; ++j)
            if (spans_overlap(out[i], out_bytes[i], out[j], out_bytes[j])) return PUFF_ERR_ALIAS;
    }
    int sms = 0;
    rc = require_sm100(&sms);
    if (rc != PUFF_OK) return rc;
    const int grid = static_cast<int>((lanes + kRecThreads - 1) / kRecThreads);
    cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
#define PUFF_RUN(T)                                                                                                     \
    puff_recurrence_backward_kernel<T><<<grid, kRecThreads, 0, st>>>(p, saved, static_cast<const T*>(doutputs), dfinal, \
                                                                     static_cast<T*>(dgates), static_cast<T*>(dinputs), dstate)
    if (dtype == PUFF_DTYPE_F32) PUFF_RUN(float);
    else if (dtype == PUFF_DTYPE_F16) PUFF_RUN(__half);
    else PUFF_RUN(__nv_bfloat16);
#undef PUFF_RUN
    count_launch();
    return static_cast<int>(cudaGetLastError());
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
