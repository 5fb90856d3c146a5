// A row's controls (control.hip) as device functions, for the kernels that end in logits.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "internal.h"

namespace sz {
namespace control {

enum Mode { M_INFER = 0, M_TRAIN = 1, M_VOTE = 2 };

struct RowControl {
    const float* bias;
    const uint32_t* allow;
    const uint32_t* counts;
    // z / repetition = z scale * inverse: scale is 1, or 2^+-64 for a repetition whose own reciprocal is no normal number
    float repetition, scale, inverse, presence, frequency;
};

__device__ __forceinline__ int32_t row_set(const Controls& c, uint64_t row)
{
    return c.sets == 0 ? -1 : c.set_of_row ? c.set_of_row[row] : 0;
}

__device__ __forceinline__ RowControl row_control(const Controls& c, int C, int32_t set)
{
    RowControl r{nullptr, nullptr, nullptr, 1.0f, 1.0f, 1.0f, 0.0f, 0.0f};
    if (set < 0 || (uint32_t)set >= c.sets) return r;
    if (c.bias) r.bias = c.bias + (uint64_t)set * C;
    if (c.allow) r.allow = c.allow + (uint64_t)set * ((C + 31) / 32);
    if (c.counts) {
        r.counts = c.counts + (uint64_t)set * C;
        if (c.repetition) {
            r.repetition = c.repetition[set];
            const float size = fabsf(r.repetition);
            r.scale = size < 0x1p-126f ? 0x1p64f : size > 0x1p126f ? 0x1p-64f : 1.0f;
            r.inverse = 1.0f / (r.repetition * r.scale);
        }
        if (c.presence) r.presence = c.presence[set];
        if (c.frequency) r.frequency = c.frequency[set];
    }
    return r;
}

__device__ __forceinline__ bool allowed(const RowControl& r, int c) { return !r.allow || ((r.allow[c >> 5] >> (c & 31)) & 1u); }

// a class's probability from its exponential: 0 off the list, also in a row whose sum is a NaN
__device__ __forceinline__ float probability(const RowControl& r, float e, float inv, int c)
{
    const float p = e * inv;
    return p == p || allowed(r, c) ? p : 0.0f;
}

// (the division by the repetition penalty is a product with its reciprocal: two roundings instead of one.  The division itself: 661400 x 64
// 90 us instead of 86, 1024 x 50001 177 instead of 170)
__device__ __forceinline__ float penalised(const RowControl& r, float z, uint32_t count)
{
    const float n = (float)count;
    const float seen = (z > 0.0f ? z * r.scale : z) * (z > 0.0f ? r.inverse : r.repetition) - r.presence;
    return (n > 0.0f ? seen : z) - r.frequency * n;
}

__device__ __forceinline__ float controlled(const RowControl& r, float z, int c)
{
    if (r.counts) z = penalised(r, z, r.counts[c]);
    if (r.bias) z += r.bias[c];
    return allowed(r, c) ? z : -INFINITY;
}

// e^x for x <= 0 (or NaN): 2^(x log2 e) by the hardware instruction with the rounding of the product, which would
// cost |x| 2^-24, put back to first order.  0 below -200.
__device__ __forceinline__ float exp_low(float x)
{
    const float kL = 1.44269502f, kR = 1.92596299e-8f, kLn2 = 0.693147182f;  // log2 e in two parts
    const float y = x < -200.0f ? -200.0f : x;
    const float t = y * kL;
    const float r = __builtin_fmaf(y, kR, __builtin_fmaf(y, kL, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(e, r * kLn2, e);
}

// Joins a value over LANES neighbouring lanes: within 16 by the register file's own lane exchanges (pairs, pairs of
// pairs, mirrored halves, mirrored rows: after each step all lanes of the smaller group hold the same), beyond by shuffles.
template <int CTRL>
__device__ __forceinline__ float lane_move(float v)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
template <int LANES, class F>
__device__ __forceinline__ float lanes_join(float v, F f)
{
    if (LANES > 1) v = f(v, lane_move<0xB1>(v));
    if (LANES > 2) v = f(v, lane_move<0x4E>(v));
    if (LANES > 4) v = f(v, lane_move<0x141>(v));
    if (LANES > 8) v = f(v, lane_move<0x140>(v));
    if (LANES > 16) v = f(v, __shfl_xor(v, 16));
    if (LANES > 32) v = f(v, __shfl_xor(v, 32));
    return v;
}
template <int LANES>
__device__ __forceinline__ float lanes_max(float v)
{
    return lanes_join<LANES>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v)
{
    return lanes_join<LANES>(v, [](float a, float b) { return a + b; });
}
// the last of the largest values over the lanes: (p, c) pairs, c = -1 for none
template <int LANES>
__device__ __forceinline__ void lanes_best(float& p, int& c)
{
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        const float q = __shfl_xor(p, o);
        const int b = __shfl_xor(c, o);
        if (q > p || (q == p && b > c)) { p = q; c = b; }
    }
}

// the vote of identify_speaker_list (lib.rs:1391-1402): the last maximum wins; a row without a candidate has none.
// Counts are integers: the order of the additions is of no matter.
__device__ __forceinline__ void cast_vote(const ControlRun& a, uint64_t row, int C, bool some, float p, int best)
{
    const int32_t g = a.group ? a.group[row] : 0;
    if (some && best >= 0 && p >= a.threshold && g >= 0 && (uint32_t)g < a.groups) atomicAdd(&a.votes[(uint64_t)g * C + best], 1ull);
}

struct TrainRow { int label; bool live; };
__device__ __forceinline__ TrainRow train_row(const ControlRun& a, const RowControl& rc, uint64_t i, uint64_t row, int C, bool some)
{
    TrainRow t;
    t.label = a.labels[row];
    t.live = a.row_live[i] && a.row_slot[i] >= 0 && t.label >= 0 && t.label < C && some && allowed(rc, t.label);
    return t;
}

}  // namespace control
}  // namespace sz
