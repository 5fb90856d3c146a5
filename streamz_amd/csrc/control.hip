// Controls on logits: per-request priors, candidate masks and penalties, and the softmax behind them
// (the softmax and cross-entropy of lib.rs:611-615, 887-890, 1028 when no control is set), and the votes.
//
//   z = l;  count > 0:  z = z > 0 ? z / repetition : z * repetition,  z -= presence
//   z -= frequency * count;  z += bias;  a class that is not allowed: z = -inf
//   p = exp(z - max z) / sum exp(z - max z);  a row whose every z is -inf: p = 0
//
// A class outside the mask never enters the arithmetic (its logit may be inf or NaN).
#include <algorithm>

#include "internal.h"
#include "prof.h"
#include "streamz_hip.h"

namespace sz {

namespace {

struct RowControl {
    const float* bias;
    const uint32_t* allow;
    const uint32_t* counts;
    float repetition, presence, frequency;
};

__device__ __forceinline__ RowControl row_control(const Controls& c, int C, uint64_t row)
{
    RowControl r{nullptr, nullptr, nullptr, 1.0f, 0.0f, 0.0f};
    const int32_t set = c.sets == 0 ? -1 : c.set_of_row ? c.set_of_row[row] : 0;
    if (set < 0 || (uint32_t)set >= c.sets) return r;
    if (c.bias) r.bias = c.bias + (uint64_t)set * C;
    if (c.allow) r.allow = c.allow + (uint64_t)set * ((C + 31) / 32);
    if (c.counts) {
        r.counts = c.counts + (uint64_t)set * C;
        if (c.repetition) r.repetition = c.repetition[set];
        if (c.presence) r.presence = c.presence[set];
        if (c.frequency) r.frequency = c.frequency[set];
    }
    return r;
}

__device__ __forceinline__ bool allowed(const RowControl& r, int c) { return !r.allow || ((r.allow[c >> 5] >> (c & 31)) & 1u); }

__device__ __forceinline__ float controlled(const RowControl& r, float z, int c)
{
    if (r.counts) {
        const float n = (float)r.counts[c];
        if (n > 0.0f) z = (z > 0.0f ? z / r.repetition : z * r.repetition) - r.presence;
        z -= r.frequency * n;
    }
    if (r.bias) z += r.bias[c];
    return allowed(r, c) ? z : -INFINITY;
}

__device__ __forceinline__ float wave_max(float v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// One wave per row, any number of classes.
template <bool TRAIN>
__global__ __launch_bounds__(256) void control_kernel(Controls ctl, ControlRun a)
{
    const int lane = threadIdx.x & 63;
    const int C = (int)a.classes;
    const uint64_t step = (uint64_t)gridDim.x * 4;
    for (uint64_t i = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < a.rows; i += step) {
        const uint64_t row = a.order ? a.order[i] : i;
        const RowControl rc = row_control(ctl, C, row);
        const float* in = a.in + i * a.ld_in;
        float top = -INFINITY;
        for (int c = lane; c < C; c += 64) {
            const float l = in[c];
            if (!TRAIN && a.raw) a.raw[row * a.ld_raw + c] = l;
            top = fmaxf(top, controlled(rc, l, c));
        }
        if (!TRAIN && !a.out && !a.votes) continue;
        top = wave_max(top);
        if (!TRAIN && !a.probs && !a.votes) {
            for (int c = lane; c < C; c += 64) a.out[row * a.ld_out + c] = controlled(rc, in[c], c);
            continue;
        }
        const float shift = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f;
        for (int c = lane; c < C; c += 64) sum += expf(controlled(rc, in[c], c) - shift);
        sum = wave_sum(sum);
        const bool some = !(sum <= 0.0f);  // (a NaN row stays one)
        if (!TRAIN && a.votes) {
            // the vote of identify_speaker_list (lib.rs:1391-1402): the last maximum wins; a row without a
            // candidate has none.  Counts are integers: the order of the additions is of no matter.
            const int32_t g = a.group ? a.group[row] : 0;
            int best = -1;
            float bp = -1.0f;
            for (int c = lane; c < C; c += 64) {
                const float p = expf(controlled(rc, in[c], c) - shift) / sum;
                if (p >= bp) { bp = p; best = c; }
            }
            for (int o = 32; o > 0; o >>= 1) {
                const float q = __shfl_xor(bp, o);
                const int b = __shfl_xor(best, o);
                if (q > bp || (q == bp && b > best)) { bp = q; best = b; }
            }
            if (lane == 0 && some && best >= 0 && bp >= a.threshold && g >= 0 && (uint32_t)g < a.groups)
                atomicAdd(&a.votes[(uint64_t)g * C + best], 1ull);
        } else if (!TRAIN) {
            float* out = a.out + row * a.ld_out;
            for (int c = lane; c < C; c += 64) out[c] = some ? expf(controlled(rc, in[c], c) - shift) / sum : 0.0f;
        } else {
            const int label = a.labels[row];
            const bool live = a.row_live[i] && a.row_slot[i] >= 0 && label >= 0 && label < C && allowed(rc, label) && some;
            float* out = a.out + i * a.ld_out;
            float loss = 0.0f;
            for (int c = lane; c < C; c += 64) {
                const float p = expf(controlled(rc, in[c], c) - shift) / sum;
                if (c == label) loss = -logf(fmaxf(p, 1e-12f));
                out[c] = live ? (c == label ? p - 1.0f : p) : 0.0f;
            }
            loss = wave_sum(loss);
            if (lane == 0) {
                a.loss[i] = live ? loss : 0.0f;
                a.live[i] = live ? 1 : 0;
            }
        }
    }
}

}  // namespace

int control_run(const Controls& ctl, const ControlRun& a, hipStream_t s)
{
    if (a.rows == 0 || a.classes == 0) return SZH_OK;
    ProfScope prof(a.labels ? "control_loss" : "control", s);
    const unsigned blocks = (unsigned)std::min<uint64_t>((a.rows + 3) / 4, 8192);
    if (a.labels) hipLaunchKernelGGL((control_kernel<true>), dim3(blocks), dim3(256), 0, s, ctl, a);
    else hipLaunchKernelGGL((control_kernel<false>), dim3(blocks), dim3(256), 0, s, ctl, a);
    SZ_HIP(hipGetLastError());
    return SZH_OK;
}

}  // namespace sz
