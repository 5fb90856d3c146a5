// Controls on logits: per-request priors, candidate masks and penalties, and the softmax behind them
// (the softmax and cross-entropy of lib.rs:611-615, 887-890, 1028 when no control is set), and the votes.
//
//   z = l;  count > 0:  z = z > 0 ? z / repetition : z * repetition,  z -= presence
//   z -= frequency * count;  z += bias;  a class that is not allowed: z = -inf
//   p = exp(z - max z) / sum exp(z - max z);  a row whose every z is -inf: p = 0
//
// A class outside the mask never enters the arithmetic (its logit may be inf or NaN).
//
// Bound by memory: logits, counts, biases and the result once each.  A row's controlled logits stay in registers
// between the maximum, the sum and the result, so nothing is read twice up to kRowMax classes: some lanes of a
// wave per row up to 1024 classes (control_rows_kernel), a workgroup per row beyond (control_row_kernel).
#include <algorithm>
#include <type_traits>

#include "control_kernel.h"
#include "internal.h"
#include "prof.h"
#include "streamz_hip.h"

namespace sz {

namespace {

using namespace control;

// out[c] = 0 for a lane's classes that are off the list of a row of NaNs (in a training row that does not count all are 0
// already).  Found again from the row's number: what this rare case needs takes no registers from the others.
template <int LANES>
__device__ __forceinline__ void clear_off_list(const Controls& ctl, uint64_t row, int C, int l, float* out)
{
    asm volatile("" : "+v"(row));
    const RowControl rc = row_control(ctl, C, row_set(ctl, row));
#pragma unroll 1
    for (int c = 4 * l; c < C; c += 4 * LANES)
        for (int k = c; k < min(c + 4, C); ++k)
            if (!allowed(rc, k)) out[k] = 0.0f;
}

// LANES lanes of a wave per row, Q groups of four classes per lane: class 4 (l + LANES q) + e.  A row's logits
// and the number of its set are asked for while the row before is worked on.
template <int MODE, int LANES, int Q>
__global__ __launch_bounds__(256) void control_rows_kernel(Controls ctl, ControlRun a, int vec_in, int vec_table, int vec_raw, int vec_out)
{
    constexpr int ROWS = 64 / LANES;
    const int l = threadIdx.x % LANES, C = (int)a.classes;
    const uint64_t base = ((uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * ROWS, mine = (threadIdx.x & 63) / LANES;
    const uint64_t step = (uint64_t)gridDim.x * 4 * ROWS;
    float z[Q][4], next_z[Q][4];
    uint64_t next_row = 0;
    int32_t next_set = -1;
    auto fetch = [&](uint64_t i0) {  // (lanes behind the last row take it again; they store nothing)
        const uint64_t i = i0 < a.rows ? i0 : a.rows - 1;
        next_row = a.order ? a.order[i] : i;
        const float* in = a.in + i * a.ld_in;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const int c = 4 * (l + LANES * q);
            if (vec_in && c < C) {
                const float4 v = *reinterpret_cast<const float4*>(in + c);
                next_z[q][0] = v.x; next_z[q][1] = v.y; next_z[q][2] = v.z; next_z[q][3] = v.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) next_z[q][e] = c + e < C ? in[c + e] : -INFINITY;
            }
        }
        next_set = row_set(ctl, next_row);
    };
    if (base < a.rows) fetch(base + mine);
    for (uint64_t at = base; at < a.rows; at += step) {
        const bool in_rows = at + mine < a.rows;
        const uint64_t i = in_rows ? at + mine : a.rows - 1, row = next_row;
        const RowControl rc = row_control(ctl, C, next_set);
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) z[q][e] = next_z[q][e];
        if (at + step < a.rows) fetch(at + step + mine);
        if (MODE == M_INFER && a.raw && in_rows) {
            float* raw = a.raw + row * a.ld_raw;
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                const int c = 4 * (l + LANES * q);
                if (vec_raw && c < C) *reinterpret_cast<float4*>(raw + c) = make_float4(z[q][0], z[q][1], z[q][2], z[q][3]);
                else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c + e < C) raw[c + e] = z[q][e];
                }
            }
            if (!a.out) continue;
        }
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const int c = 4 * (l + LANES * q);
            if (rc.counts) {
                uint32_t n[4] = {0, 0, 0, 0};
                if (vec_table && c < C) {
                    const uint4 v = *reinterpret_cast<const uint4*>(rc.counts + c);
                    n[0] = v.x; n[1] = v.y; n[2] = v.z; n[3] = v.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c + e < C) n[e] = rc.counts[c + e];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) z[q][e] = penalised(rc, z[q][e], n[e]);
            }
            if (rc.bias) {
                if (vec_table && c < C) {
                    const float4 v = *reinterpret_cast<const float4*>(rc.bias + c);
                    z[q][0] += v.x; z[q][1] += v.y; z[q][2] += v.z; z[q][3] += v.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c + e < C) z[q][e] += rc.bias[c + e];
                }
            }
            const uint32_t bits = c < C ? (rc.allow ? rc.allow[c >> 5] >> (c & 31) : 15u) : 0u;  // four classes lie in one word
#pragma unroll
            for (int e = 0; e < 4; ++e) z[q][e] = c + e < C && ((bits >> e) & 1u) ? z[q][e] : -INFINITY;
        }
        bool nans = false;
        if (MODE != M_INFER || a.probs) {
            float top = -INFINITY;
#pragma unroll
            for (int q = 0; q < Q; ++q) top = fmaxf(top, fmaxf(fmaxf(z[q][0], z[q][1]), fmaxf(z[q][2], z[q][3])));
            top = lanes_max<LANES>(top);
            const float shift = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f;
#pragma unroll
            for (int q = 0; q < Q; ++q) {
#pragma unroll
                for (int e = 0; e < 4; ++e) z[q][e] = exp_low(z[q][e] - shift);
                sum += (z[q][0] + z[q][1]) + (z[q][2] + z[q][3]);
            }
            sum = lanes_sum<LANES>(sum);
            const bool some = !(sum <= 0.0f);  // (a NaN row stays one)
            const float inv = some ? 1.0f / sum : 0.0f;
            nans = !(inv == inv);
#pragma unroll
            for (int q = 0; q < Q; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) z[q][e] *= inv;
            if (MODE == M_VOTE) {
                float bp = -1.0f;
                int best = -1;
#pragma unroll
                for (int q = 0; q < Q; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int c = 4 * (l + LANES * q) + e;
                        if (c < C && z[q][e] >= bp) { bp = z[q][e]; best = c; }
                    }
                lanes_best<LANES>(bp, best);
                if (l == 0 && in_rows) cast_vote(a, row, C, some, bp, best);
                continue;
            }
            if (MODE == M_TRAIN) {
                const TrainRow t = train_row(a, rc, i, row, C, some);
                float loss = 0.0f;
#pragma unroll
                for (int q = 0; q < Q; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (4 * (l + LANES * q) + e == t.label) {
                            loss = -logf(fmaxf(z[q][e], 1e-12f));
                            z[q][e] -= 1.0f;
                        }
                        if (!t.live) z[q][e] = 0.0f;
                    }
                loss = lanes_sum<LANES>(loss);
                if (l == 0 && in_rows) {
                    a.loss[i] = t.live ? loss : 0.0f;
                    a.live[i] = t.live ? 1 : 0;
                }
            }
        }
        if (!in_rows) continue;
        float* out = a.out + (MODE == M_TRAIN ? i : row) * a.ld_out;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const int c = 4 * (l + LANES * q);
            if (vec_out && c < C) *reinterpret_cast<float4*>(out + c) = make_float4(z[q][0], z[q][1], z[q][2], z[q][3]);
            else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < C) out[c + e] = z[q][e];
            }
        }
        if (nans) clear_off_list<LANES>(ctl, row, C, l, out);
    }
}

constexpr int kRowThreads = 1024, kRowMax = 50 * kRowThreads;

// joins a value of every wave
template <class F>
__device__ __forceinline__ float join_waves(float v, float* part, F f)
{
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = part[0];
#pragma unroll
    for (int w = 1; w < kRowThreads / 64; ++w) r = f(r, part[w]);
    return r;
}

// The thread's index, which the compiler takes for a new value: what it computes from it (offsets and bounds of
// every class) is not kept in registers from one use to the next.
__device__ __forceinline__ uint32_t fresh_thread()
{
    uint32_t t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

// One workgroup per row, V values per thread in registers (class t + 1024 q: whole lines whatever the row's
// alignment); V = 0: any number of classes, the row read twice more (out of the caches, mostly).
template <int MODE, int V>
__global__ __launch_bounds__(kRowThreads) void control_row_kernel(Controls ctl, ControlRun a, uint64_t first)
{
    __shared__ float part[kRowThreads / 64];
    __shared__ int part_c[kRowThreads / 64];
    const int C = (int)a.classes;
    const int n_mine = ((int)C - (int)threadIdx.x + kRowThreads - 1) / kRowThreads;
    const uint64_t i = first + blockIdx.x;
    const uint64_t row = a.order ? (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)a.order[i]) : i;
    const RowControl rc = row_control(ctl, C, __builtin_amdgcn_readfirstlane(row_set(ctl, row)));  // (addresses in scalar registers)
    const float* in = a.in + i * a.ld_in;
    float* raw = MODE == M_INFER && a.raw ? a.raw + row * a.ld_raw : nullptr;
    float* out = a.out ? a.out + (MODE == M_TRAIN ? i : row) * a.ld_out : nullptr;
    // a thread goes through its values some at a time: their loads are all in flight, and what a step needs beside
    // them does not take V registers more
    constexpr int STEP = V % 10 == 0 && V ? 10 : V < 8 ? (V ? V : 1) : 8;
    float z[V ? V : 1];
    auto each = [&](auto f) {   // f(value, class) over the thread's classes
        if (V) {
#pragma unroll
            for (int q0 = 0; q0 < V; q0 += STEP) {
                const uint32_t t = fresh_thread();
#pragma unroll
                for (int q = q0; q < q0 + STEP; ++q)
                    if (t + (uint32_t)(kRowThreads * q) < (uint32_t)C) f(z[q % (V ? V : 1)], t + (uint32_t)(kRowThreads * q));
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
#pragma unroll 4
            for (int q = 0; q < n_mine; ++q) {
                const int c = threadIdx.x + kRowThreads * q;
                float v = controlled(rc, in[c], c);
                f(v, c);
            }
        }
    };
    if (raw) {
#pragma unroll 4
        for (int c = threadIdx.x; c < C; c += kRowThreads) raw[c] = in[c];
        if (!out) return;
    }
    if (V) {
#pragma unroll
        for (int q0 = 0; q0 < V; q0 += STEP) {
            const uint32_t t = fresh_thread();
            // (tables that are not used count as zeros and ones: no branches between the loads and their use)
            uint32_t n[STEP], w[STEP];
            float h[STEP];
#pragma unroll
            for (int q = 0; q < STEP; ++q) {
                const uint32_t c = min(t + (uint32_t)(kRowThreads * (q0 + q)), (uint32_t)C - 1);
                z[(q0 + q) % (V ? V : 1)] = in[c];
                n[q] = 0; w[q] = ~0u; h[q] = 0.0f;
            }
            if (rc.counts) {
#pragma unroll
                for (int q = 0; q < STEP; ++q) n[q] = rc.counts[min(t + (uint32_t)(kRowThreads * (q0 + q)), (uint32_t)C - 1)];
            }
            if (rc.bias) {
#pragma unroll
                for (int q = 0; q < STEP; ++q) h[q] = rc.bias[min(t + (uint32_t)(kRowThreads * (q0 + q)), (uint32_t)C - 1)];
            }
            if (rc.allow) {
#pragma unroll
                for (int q = 0; q < STEP; ++q) w[q] = rc.allow[min(t + (uint32_t)(kRowThreads * (q0 + q)), (uint32_t)C - 1) >> 5];
            }
#pragma unroll
            for (int q = 0; q < STEP; ++q) {
                const float v = penalised(rc, z[(q0 + q) % (V ? V : 1)], n[q]) + h[q];
                const bool on = t + (uint32_t)(kRowThreads * (q0 + q)) < (uint32_t)C && ((w[q] >> (t & 31)) & 1u);
                z[(q0 + q) % (V ? V : 1)] = on ? v : -INFINITY;
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (MODE == M_INFER && !a.probs) {
        each([&](float& v, uint32_t c) { out[c] = v; });
        return;
    }
    float top = -INFINITY;
    each([&](float& v, uint32_t) { top = fmaxf(top, v); });
    top = join_waves(lanes_max<64>(top), part, [](float x, float y) { return fmaxf(x, y); });
    const float shift = top == -INFINITY ? 0.0f : top;
    // (up to 50 values a thread in registers are added in 32 bits; of any number of them a small one would be lost beside the sum of the others)
    std::conditional_t<V != 0, float, double> mine = 0;
    each([&](float& v, uint32_t) { v = exp_low(v - shift); mine += v; });
    float sum = (float)mine;
    sum = join_waves(lanes_sum<64>(sum), part, [](float x, float y) { return x + y; });
    const bool some = !(sum <= 0.0f);
    const float inv = some ? 1.0f / sum : 0.0f;
    // (without registers the values come again as controlled logits)
    auto prob = [&](float v) { return (V ? v : exp_low(v - shift)) * inv; };
    if (MODE == M_VOTE) {
        float bp = -1.0f;
        int best = -1;
        each([&](float& v, uint32_t c) { const float p = prob(v); if (p >= bp) { bp = p; best = (int)c; } });
        lanes_best<64>(bp, best);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) { part[threadIdx.x >> 6] = bp; part_c[threadIdx.x >> 6] = best; }
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < kRowThreads / 64; ++w)
                if (part[w] > bp || (part[w] == bp && part_c[w] > best)) { bp = part[w]; best = part_c[w]; }
            cast_vote(a, row, C, some, bp, best);
        }
        return;
    }
    const bool mend = !(inv == inv) && rc.allow;  // (the classes off the list of a row of NaNs)
    if (MODE == M_INFER) {
        each([&](float& v, uint32_t c) { out[c] = prob(v); });
        if (mend) {
            for (int c = threadIdx.x; c < C; c += kRowThreads)
                if (!allowed(rc, c)) out[c] = 0.0f;
        }
    } else {
        const TrainRow t = train_row(a, rc, i, row, C, some);
        if (threadIdx.x == 0 && !(t.label >= 0 && t.label < C)) { a.loss[i] = 0.0f; a.live[i] = 0; }
        each([&](float& v, uint32_t c) {
            const float p = prob(v);
            if ((int)c == t.label) { a.loss[i] = t.live ? -logf(fmaxf(p, 1e-12f)) : 0.0f; a.live[i] = t.live ? 1 : 0; }
            out[c] = t.live ? ((int)c == t.label ? p - 1.0f : p) : 0.0f;
        });
        if (mend && t.live) {
            for (int c = threadIdx.x; c < C; c += kRowThreads)
                if (!allowed(rc, c)) out[c] = 0.0f;
        }
    }
}

template <int MODE>
int launch(const Controls& ctl, const ControlRun& a, hipStream_t s)
{
    const uint32_t C = a.classes;
    const auto vec = [&](const void* p, uint64_t ld) { return C % 4 == 0 && ld % 4 == 0 && ((uintptr_t)p & 15) == 0 ? 1 : 0; };
    const int vi = vec(a.in, a.ld_in), vt = vec(ctl.bias, C) && vec(ctl.counts, C), vr = vec(a.raw, a.ld_raw), vo = vec(a.out, a.ld_out);
#define SZ_ROWS(LANES, Q)                                                                                                       \
    hipLaunchKernelGGL((control_rows_kernel<MODE, LANES, Q>), dim3((unsigned)std::min<uint64_t>((a.rows * (LANES) + 255) / 256, 8192)), \
                       dim3(256), 0, s, ctl, a, vi, vt, vr, vo)
    // (a launch has fewer than 2^32 threads)
#define SZ_ROW(V)                                                                                                               \
    for (uint64_t r = 0; r < a.rows; r += 1u << 20)                                                                             \
        hipLaunchKernelGGL((control_row_kernel<MODE, V>), dim3((unsigned)std::min<uint64_t>(a.rows - r, 1u << 20)), dim3(kRowThreads), 0, s, ctl, a, r)
    // (few lanes with several groups each: less of a row's work is done by every lane.  2 M rows of 16 classes: 66 us
    // on 2 lanes, 75 on 4, 108 on 1; 661400 of 64: 85 on 4, 90 on 8, 105 on 16; 150000 of 256: 82 on 32, 85 on 16, 88 on 64)
    if (C <= 4) SZ_ROWS(1, 1);
    else if (C <= 8) SZ_ROWS(2, 1);
    else if (C <= 16) SZ_ROWS(2, 2);
    else if (C <= 32) SZ_ROWS(4, 2);
    else if (C <= 64) SZ_ROWS(4, 4);
    else if (C <= 128) SZ_ROWS(16, 2);
    else if (C <= 256) SZ_ROWS(32, 2);
    else if (C <= 512) SZ_ROWS(64, 2);
    else if (C <= 1024) SZ_ROWS(64, 4);
    else if (C <= 2 * kRowThreads) SZ_ROW(2);
    else if (C <= 4 * kRowThreads) SZ_ROW(4);
    else if (C <= 8 * kRowThreads) SZ_ROW(8);
    else if (C <= 16 * kRowThreads) SZ_ROW(16);
    else if (C <= 32 * kRowThreads) SZ_ROW(32);
    else if (C <= kRowMax) SZ_ROW(50);
    else SZ_ROW(0);
#undef SZ_ROWS
#undef SZ_ROW
    SZ_HIP(hipGetLastError());
    return SZH_OK;
}

}  // namespace

int control_run(const Controls& ctl, const ControlRun& a, hipStream_t s)
{
    if (a.rows == 0 || a.classes == 0) return SZH_OK;
    ProfScope prof(a.labels ? "control_loss" : "control", s);
    return a.labels ? launch<M_TRAIN>(ctl, a, s) : a.votes ? launch<M_VOTE>(ctl, a, s) : launch<M_INFER>(ctl, a, s);
}

}  // namespace sz
