// Adapters for calls of few rows (adapt.hip): a workgroup per row for everything that only that row's adapter
// takes part in, and thin products of a few 32-row tiles for the shared hidden layer.
//
// With few rows the matrices are what is read, and nearly nothing is computed: a row's workgroup streams the small
// matrices (w1, the slot's factors, w3) straight from the caches into vector products with its activations in LDS,
// and the large one, w2, is cut over columns and k so that many compute units read a part each.
// One row of 60-512-256-16: 20.8 us for the three launches (365 as tensor operations), most of it a compute unit's first reading
// of matrices and code (about 3000 cycles for a matrix it has not seen); one launch for all three took 24 to 35 us, because a
// single compute unit then reads w2 as well.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "adapt_kernel.h"
#include "control_kernel.h"
#include "gemm_kernel.h"

namespace sz {
namespace adapt {

constexpr int kRowT = 1024, kRowWaves = kRowT / 64;
// LDS floats of the partial sums: four columns per thread
constexpr int kRowPart = 4 * kRowT;

// four values from any multiple of four bytes: one load
__device__ __forceinline__ float4 any_four(const float* p)
{
    typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
    const f32x4u v = *reinterpret_cast<const f32x4u*>(p);
    return make_float4(v[0], v[1], v[2], v[3]);
}

// out(n, sum_k x[k] W[k][n] + sum_j u[j] B[j][n]) for n < N, by the whole workgroup; x and u in LDS, W [K][N] and B [J][N]
// in memory (J may be 0).  A thread takes four neighbouring columns and every ks-th k; partial sums meet by lane
// exchanges (narrow matrices) and in LDS.  Ends with a barrier; `out` is called by one thread per column.
template <class F>
__device__ __forceinline__ void row_product(const float* x, int K, const float* __restrict__ W, const float* u, int J,
                                            const float* __restrict__ B, int N, float* part, F out)
{
    const int t = threadIdx.x;
    const bool vec = N >= 4;
    for (int n0 = 0; n0 < N; n0 += kRowPart) {
        const int cols = min(N - n0, kRowPart), groups = (cols + 3) >> 2;
        int lg = 0;
        while ((1 << lg) < groups) ++lg;  // groups of four columns, rounded up to a power of two
        const int gp = 1 << lg, slices = kRowT >> lg;
        const int c = n0 + 4 * (t & (gp - 1)), ks = t >> lg;
        const int at = vec ? min(c, N - 4) : c;  // (the last group reads the last four columns; rows may start anywhere)
        float a0 = 0.0f, a1 = 0.0f, a2 = 0.0f, a3 = 0.0f;
        auto run = [&](const float* v, int n_k, const float* __restrict__ M) {
            if (c >= N) return;
            if (vec) {
                int k = ks;
                for (; k + 7 * slices < n_k; k += 8 * slices) {
                    float4 w[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) w[i] = any_four(M + (size_t)(k + i * slices) * N + at);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float xv = v[k + i * slices];
                        a0 = __builtin_fmaf(xv, w[i].x, a0); a1 = __builtin_fmaf(xv, w[i].y, a1);
                        a2 = __builtin_fmaf(xv, w[i].z, a2); a3 = __builtin_fmaf(xv, w[i].w, a3);
                    }
                }
                // what is left of k, four pieces in flight, those behind it as zeros
                for (; k < n_k; k += 4 * slices) {
                    float4 w[4];
                    float xv[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int kk = min(k + i * slices, n_k - 1);
                        w[i] = any_four(M + (size_t)kk * N + at);
                        xv[i] = v[kk];
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool on = k + i * slices < n_k;
                        const float q = on ? xv[i] : 0.0f;   // (either may be none)
                        a0 = __builtin_fmaf(q, on ? w[i].x : 0.0f, a0); a1 = __builtin_fmaf(q, on ? w[i].y : 0.0f, a1);
                        a2 = __builtin_fmaf(q, on ? w[i].z : 0.0f, a2); a3 = __builtin_fmaf(q, on ? w[i].w : 0.0f, a3);
                    }
                }
            } else {
                const int c1 = min(c + 1, N - 1), c2 = min(c + 2, N - 1), c3 = min(c + 3, N - 1);
#pragma unroll 4
                for (int k = ks; k < n_k; k += slices) {
                    const float* m = M + (size_t)k * N;
                    const float xv = v[k];
                    a0 = __builtin_fmaf(xv, m[c], a0); a1 = __builtin_fmaf(xv, m[c1], a1);
                    a2 = __builtin_fmaf(xv, m[c2], a2); a3 = __builtin_fmaf(xv, m[c3], a3);
                }
            }
        };
        run(x, K, W);
        if (J) run(u, J, B);
        if (c - at == 1) { a0 = a1; a1 = a2; a2 = a3; }
        else if (c - at == 2) { a0 = a2; a1 = a3; }
        else if (c - at == 3) a0 = a3;
        // the k slices of a wave
        for (int o = gp; o < 64; o <<= 1) {
            a0 += __shfl_xor(a0, o); a1 += __shfl_xor(a1, o); a2 += __shfl_xor(a2, o); a3 += __shfl_xor(a3, o);
        }
        // part[slice of waves][column]: waves beside one another hold the columns' groups of 64
        const int wave = t >> 6, across = gp > 64 ? gp >> 6 : 1, per = gp < 64 ? gp : 64, rows = kRowWaves / across;
        if ((t & 63) < per) {
            float* p = part + ((size_t)(wave / across) * across * per + (wave % across) * per + (t & (per - 1))) * 4;
            *reinterpret_cast<float4*>(p) = make_float4(a0, a1, a2, a3);
        }
        __syncthreads();
        for (int n = t; n < cols; n += kRowT) {
            float s = 0.0f;
            for (int r = 0; r < rows; ++r) s += part[(size_t)r * across * per * 4 + n];
            out(n0 + n, s);
        }
        __syncthreads();
    }
}

// out(n, sum_k x[k] W[n][k] + sum_j u[j] B[n][j]) for n < N: the rows of W [N][K] and B [N][J] lie along the sum.
// Lanes of a wave share a row; ends with a barrier.
template <class F>
__device__ __forceinline__ void row_product_t(const float* x, int K, const float* __restrict__ W, const float* u, int J,
                                              const float* __restrict__ B, int N, F out)
{
    int lg = 0;
    while ((1 << lg) < K && lg < 6) ++lg;
    const int lanes = 1 << lg, per = kRowT >> lg, l = threadIdx.x & (lanes - 1);
    for (int n0 = 0; n0 < N; n0 += per) {
        const int n = n0 + (int)(threadIdx.x >> lg);
        float s = 0.0f;
        if (n < N) {
#pragma unroll 4
            for (int k = l; k < K; k += lanes) s = __builtin_fmaf(x[k], W[(size_t)n * K + k], s);
#pragma unroll 4
            for (int j = l; j < J; j += lanes) s = __builtin_fmaf(u[j], B[(size_t)n * J + j], s);
        }
        for (int o = lanes >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o);
        if (n < N && l == 0) out(n, s);
    }
    __syncthreads();
}

struct RowArgs {
    // first kernel: x -> h1, and what the slot adds to the second layer
    const float* x; uint64_t ldx;
    const float *w1, *b1;
    // second kernel: h2 -> what the slot adds to the logits, the logits and what follows them
    const float *w3, *b3;
    const float* factors; uint64_t per_slot;   // the bank, and a slot's floats
    uint64_t off_a2, off_b2, off_a3, off_b3;
    const int32_t* slot;                        // [rows]
    int slots, in, n1, n2, out, rank, ldu, ld1, ld2, ld3;
    float scale;
    float *h1, *h2, *add2, *add3, *u2, *u3;     // [rows][ld..]; u2 and u3 (training) and add3 may be null
    // backward
    float *g2, *g3, *d2, *d3;
};

__device__ __forceinline__ int row_slot_of(const RowArgs& a, uint64_t i)
{
    const int s = a.slot[i];
    return s >= 0 && s < a.slots ? s : -1;
}

// h1 = relu(x w1 + b1); u2 = scale h1 a2; add2 = u2 b2
__global__ __launch_bounds__(kRowT) void row_hidden_kernel(RowArgs a)
{
    extern __shared__ __attribute__((aligned(16))) float rl[];
    float* part = rl;
    float* h = part + kRowPart;
    float* u = h + a.n1;
    float* x = u + 64;
    const uint64_t i = blockIdx.x;
    for (int k = threadIdx.x; k < a.in; k += kRowT) x[k] = a.x[i * a.ldx + k];
    const int slot = row_slot_of(a, i);
    __syncthreads();
    row_product(x, a.in, a.w1, nullptr, 0, nullptr, a.n1, part, [&](int n, float v) {
        v = gemm::relu_max(v + a.b1[n]);
        h[n] = v;
        a.h1[i * a.ld1 + n] = v;
    });
    if (slot < 0) {
        for (int n = threadIdx.x; n < a.n2; n += kRowT) a.add2[i * a.ld2 + n] = 0.0f;
        if (a.u2) for (int j = threadIdx.x; j < a.ldu; j += kRowT) a.u2[i * a.ldu + j] = 0.0f;
        return;
    }
    const float* f = a.factors + (uint64_t)slot * a.per_slot;
    row_product(h, a.n1, f + a.off_a2, nullptr, 0, nullptr, a.rank, part, [&](int n, float v) { u[n] = a.scale * v; });
    if (a.u2) for (int j = threadIdx.x; j < a.ldu; j += kRowT) a.u2[i * a.ldu + j] = j < a.rank ? u[j] : 0.0f;
    row_product(u, a.rank, f + a.off_b2, nullptr, 0, nullptr, a.n2, part, [&](int n, float v) { a.add2[i * a.ld2 + n] = v; });
}

// a value joined over the workgroup, in every thread
template <class F>
__device__ __forceinline__ float row_join(float v, float* part, F f)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = f(v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int w = 1; w < kRowWaves; ++w) v = f(v, part[w]);
    return v;
}

// u3 = scale h2 a3, then
//   OUT_ADD    add3 = u3 b3 (the logits are a product of their own: many classes)
//   OUT_INFER  logits, controls, and what the call wants of them (c: raw, out, votes)
//   OUT_TRAIN  the loss, d3 = p - t, and back: g3 = scale d3 b3^T, d2 = (d3 w3^T + g3 a3^T)(1 - h2^2), g2 = scale d2 b2^T
enum RowOut { OUT_ADD = 0, OUT_INFER = 1, OUT_TRAIN = 2 };
template <int OUT>
__global__ __launch_bounds__(kRowT) void row_out_kernel(RowArgs a, Controls ctl, ControlRun c)
{
    extern __shared__ __attribute__((aligned(16))) float rl[];
    float* part = rl;
    float* h = part + kRowPart;
    float* u = h + a.n2;        // 64: u3, later g3
    float* z = u + 64;          // [out]
    float* d = z + a.out;       // [n2] (training)
    const uint64_t i = blockIdx.x;
    const int C = a.out;
    for (int k = threadIdx.x; k < a.n2; k += kRowT) h[k] = a.h2[i * a.ld2 + k];
    const int slot = row_slot_of(a, i);
    const float* f = a.factors + (uint64_t)(slot < 0 ? 0 : slot) * a.per_slot;
    const int J = slot < 0 ? 0 : a.rank;
    __syncthreads();
    if (J) row_product(h, a.n2, f + a.off_a3, nullptr, 0, nullptr, a.rank, part, [&](int n, float v) { u[n] = a.scale * v; });
    if (a.u3) for (int j = threadIdx.x; j < a.ldu; j += kRowT) a.u3[i * a.ldu + j] = j < J ? u[j] : 0.0f;
    if (OUT == OUT_ADD) {
        if (J) row_product(u, J, f + a.off_b3, nullptr, 0, nullptr, C, part, [&](int n, float v) { a.add3[i * a.ld3 + n] = v; });
        else for (int n = threadIdx.x; n < C; n += kRowT) a.add3[i * a.ld3 + n] = 0.0f;
        return;
    }
    const uint64_t row = c.order ? c.order[i] : i;
    const control::RowControl rc = control::row_control(ctl, C, control::row_set(ctl, row));
    float* raw = OUT == OUT_INFER && c.raw ? c.raw + row * c.ld_raw : nullptr;
    row_product(h, a.n2, a.w3, u, J, f + a.off_b3, C, part, [&](int n, float v) {
        v += a.b3[n];
        if (raw) raw[n] = v;
        z[n] = control::controlled(rc, v, n);
    });
    if (OUT == OUT_INFER && !c.out && !c.votes) return;
    float top = -INFINITY;
    for (int n = threadIdx.x; n < C; n += kRowT) top = fmaxf(top, z[n]);
    top = row_join(top, part, [](float x, float y) { return fmaxf(x, y); });
    const float shift = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    for (int n = threadIdx.x; n < C; n += kRowT) {
        const float e = control::exp_low(z[n] - shift);
        z[n] = e;
        sum += e;
    }
    sum = row_join(sum, part, [](float x, float y) { return x + y; });
    const bool some = !(sum <= 0.0f);  // (a NaN row stays one)
    const float inv = some ? 1.0f / sum : 0.0f;
    if (OUT == OUT_INFER && c.votes) {
        __syncthreads();
        if (threadIdx.x < 64) {
            float bp = -1.0f;
            int best = -1;
            for (int n = threadIdx.x; n < C; n += 64) {
                const float p = z[n] * inv;
                if (p >= bp) { bp = p; best = n; }
            }
            control::lanes_best<64>(bp, best);
            if (threadIdx.x == 0) control::cast_vote(c, row, C, some, bp, best);
        }
        return;
    }
    if (OUT == OUT_INFER) {
        for (int n = threadIdx.x; n < C; n += kRowT) c.out[row * c.ld_out + n] = control::probability(rc, z[n], inv, n);
        return;
    }
    const int label = c.labels[row];
    const bool live = c.row_live[i] && slot >= 0 && label >= 0 && label < C && some && control::allowed(rc, label);
    for (int n = threadIdx.x; n < C; n += kRowT) {
        const float p = z[n] * inv;
        const float v = live ? (n == label ? p - 1.0f : p) : 0.0f;
        if (live && n == label) c.loss[i] = -logf(fmaxf(p, 1e-12f));
        z[n] = v;
        a.d3[i * a.ld3 + n] = v;
    }
    if (inv != inv && rc.allow) {  // (the classes off the list of a row of NaNs)
        for (int n = threadIdx.x; n < C; n += kRowT)
            if (!control::allowed(rc, n)) a.d3[i * a.ld3 + n] = z[n] = 0.0f;
    }
    if (threadIdx.x == 0) {
        c.live[i] = live ? 1 : 0;
        if (!live) c.loss[i] = 0.0f;
    }
    __syncthreads();
    if (!live) {  // (uniform: nothing flows back)
        for (int j = threadIdx.x; j < a.ldu; j += kRowT) a.g3[i * a.ldu + j] = a.g2[i * a.ldu + j] = 0.0f;
        for (int n = threadIdx.x; n < a.n2; n += kRowT) a.d2[i * a.ld2 + n] = 0.0f;
        return;
    }
    row_product_t(z, C, f + a.off_b3, nullptr, 0, nullptr, a.rank, [&](int j, float v) { u[j] = a.scale * v; });
    for (int j = threadIdx.x; j < a.ldu; j += kRowT) a.g3[i * a.ldu + j] = j < a.rank ? u[j] : 0.0f;
    row_product_t(z, C, a.w3, u, a.rank, f + a.off_a3, a.n2, [&](int n, float v) {
        v *= 1.0f - h[n] * h[n];
        d[n] = v;
        a.d2[i * a.ld2 + n] = v;
    });
    row_product_t(d, a.n2, f + a.off_b2, nullptr, 0, nullptr, a.rank, [&](int j, float v) { a.g2[i * a.ldu + j] = a.scale * v; });
    for (int j = a.rank + threadIdx.x; j < a.ldu; j += kRowT) a.g2[i * a.ldu + j] = 0.0f;
}

// C = act(A W + add + bias) for few rows: a workgroup computes a 32 x 32 tile, its eight waves a part of k each
// (v_mfma_f32_32x32x2_f32, operands straight from memory), joined in LDS.  A step pairs k = e with k = 4 + e of eight.
// add: a matrix (few rows: row_hidden_kernel made it), or the rows' low-rank part as in adapt_add, the tile's slots
// dealt to the waves.
struct ThinArgs {
    const float* A; uint64_t lda;   // [M][K], 16-byte aligned rows
    const float* W;                 // [K][N]
    const float* add; uint64_t ldadd;
    const float* bias;
    float* C; uint64_t ldc;
    int M, N, K;
    const float *low, *up;          // add == nullptr
    const int32_t* row_slot;
    uint64_t up_slot;
    int ld_low, rank;
};
constexpr int kThinWaves = 8;
template <bool TANH>
__global__ __launch_bounds__(64 * kThinWaves) void thin_kernel(ThinArgs g)
{
    __shared__ __attribute__((aligned(16))) float part[kThinWaves + 1][32][32];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l31 = lane & 31, half = lane >> 5;
    const int n0 = blockIdx.x * 32, m0 = blockIdx.y * 32;
    const int blocks = (g.K + 7) / 8, per = (blocks + kThinWaves - 1) / kThinWaves;
    const int b0 = wave * per, b1 = min(blocks, b0 + per);
    const int row = min(m0 + l31, g.M - 1), col = min(n0 + l31, g.N - 1);
    const float* a = g.A + (uint64_t)row * g.lda + 4 * half;
    const float* w = g.W + (uint64_t)(4 * half) * g.N + col;
    gemm::f32x16 acc;
    if (!g.add) {
        const int mine = m0 + l31 < g.M ? g.row_slot[m0 + l31] : -1;
        uint32_t left = (uint32_t)__ballot(mine >= 0);
        if (wave == 0) {
            for (int r = half; r < 32; r += 2)
                if (!((left >> r) & 1u)) part[kThinWaves][r][l31] = 0.0f;
        }
        const int steps = g.ld_low >> 1;  // a multiple of 4; a step pairs k = st with k = st + steps
        const float* low = g.low + (uint64_t)row * g.ld_low + half * steps;
        for (int turn = 0; left; ++turn) {
            const int slot = __builtin_amdgcn_readlane(mine, __builtin_ctz(left));
            const uint32_t member = (uint32_t)__ballot(mine == slot);
            left &= ~member;
            if (turn % kThinWaves != wave) continue;
            const float* up = g.up + (uint64_t)slot * g.up_slot + col;
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[r] = 0.0f;
#pragma unroll 2
            for (int st = 0; st < steps; st += 4) {
                const float4 a4 = *reinterpret_cast<const float4*>(low + st);
                const float av[4] = {a4.x, a4.y, a4.z, a4.w};
                float bv[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int k = half * steps + st + j;
                    bv[j] = up[(uint64_t)min(k, g.rank - 1) * g.N];
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc = __builtin_amdgcn_mfma_f32_32x32x2f32(av[j], keep_if(half * steps + st + j < g.rank, bv[j]), acc, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int m = (r & 3) + 8 * (r >> 2) + 4 * half;
                if ((member >> m) & 1u) part[kThinWaves][m][l31] = acc[r];
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = 0.0f;
    const int full = min(b1, g.K / 8);   // blocks that lie inside K
    int b = b0;
    for (; b + 3 < full; b += 4) {
        float4 av[4];
        float wv[4][4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            av[q] = *reinterpret_cast<const float4*>(a + 8 * (b + q));
#pragma unroll
            for (int e = 0; e < 4; ++e) wv[q][e] = w[(uint64_t)(8 * (b + q) + e) * g.N];
        }
        __builtin_amdgcn_sched_barrier(0);  // every load is asked for before the first is waited for
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float v[4] = {av[q].x, av[q].y, av[q].z, av[q].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(v[e], wv[q][e], acc, 0, 0, 0);
        }
    }
    for (; b < b1; ++b) {
        float av[4], wv[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int k = min(8 * b + 4 * half + e, g.K - 1) - 4 * half;
            av[e] = a[k];
            wv[e] = w[(int64_t)k * g.N];
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool in = 8 * b + 4 * half + e < g.K;
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(keep_if(in, av[e]), keep_if(in, wv[e]), acc, 0, 0, 0);
        }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) part[wave][(r & 3) + 8 * (r >> 2) + 4 * half][l31] = acc[r];
    __syncthreads();
    for (int e = threadIdx.x; e < 1024; e += 64 * kThinWaves) {
        const int m = e >> 5, n = e & 31;
        if (m0 + m >= g.M || n0 + n >= g.N) continue;
        float s = 0.0f;
#pragma unroll
        for (int p = 0; p < kThinWaves; ++p) s += part[p][m][n];
        s += g.add ? g.add[(uint64_t)(m0 + m) * g.ldadd + n0 + n] : part[kThinWaves][m][n];
        s += g.bias[n0 + n];
        g.C[(uint64_t)(m0 + m) * g.ldc + n0 + n] = TANH ? gemm::fast_tanh(s) : s;
    }
}

}  // namespace adapt
}  // namespace sz
