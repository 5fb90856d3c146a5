// Kernels of the low-rank adapters (adapt.hip): grouping of a call's rows by adapter, the products with the
// rank columns, the factors' gradients and the update.  The large products are the GEMM kernels of
// gemm_kernel.h / gemm_bf16x3.h with an EPI_ADAPT_* epilogue.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "control_kernel.h"
#include "gemm_kernel.h"
#include "rng.h"

namespace sz {
namespace adapt {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// ---- grouping: the rows of a call in the order of their slots ---------------------------------
// A stable counting sort: key = slot for 0 <= slot < slots, else `slots` (rows without an adapter, last).
// One wave counts / places kGroupRows rows, 64 at a time, so that a row's rank among the rows of its key is
// the wave's running count plus the members among the lower lanes: the order, and with it every sum over
// rows, is the same on every call.
constexpr int kGroupRows = 512;

// f(row, whether it is one of the rows, its key) for the rows r0 .. r1 - 1, 64 at a time, by one wave; the slots of 512 rows are
// asked for at once
template <class F>
__device__ __forceinline__ void each_key(const int32_t* __restrict__ slot, uint32_t r0, uint32_t r1, int slots, F f)
{
    const uint32_t lane = threadIdx.x & 63;
    for (uint32_t r = r0; r < r1; r += 512) {
        int32_t s[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = slot[min(r + 64 * i + lane, r1 - 1)];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (r + 64 * i >= r1) break;
            f(r + 64 * i + lane, r + 64 * i + lane < r1, s[i] >= 0 && s[i] < slots ? s[i] : slots);
        }
    }
}

// count[key][block] of a block of rows
__global__ __launch_bounds__(64) void group_count_kernel(const int32_t* __restrict__ slot, uint32_t rows, int slots, int blocks,
                                                         uint32_t* __restrict__ count)
{
    extern __shared__ uint32_t hist[];
    for (int k = threadIdx.x; k <= slots; k += 64) hist[k] = 0;
    __syncthreads();
    const uint32_t r0 = blockIdx.x * kGroupRows, r1 = min(rows, r0 + kGroupRows);
    each_key(slot, r0, r1, slots, [&](uint32_t, bool in, int key) { if (in) atomicAdd(&hist[key], 1u); });  // (integers: any order)
    __syncthreads();
    for (int k = threadIdx.x; k <= slots; k += 64) count[(size_t)k * blocks + blockIdx.x] = hist[k];
}

__device__ __forceinline__ uint32_t wave_scan(uint32_t v)  // inclusive
{
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t u = __shfl_up(v, o);
        if ((int)(threadIdx.x & 63) >= o) v += u;
    }
    return v;
}

// count[key][0 .. blocks) becomes its exclusive prefix sums, total[key] the sum; one wave per key
__global__ __launch_bounds__(64) void group_scan_kernel(uint32_t* __restrict__ count, int blocks, uint32_t* __restrict__ total)
{
    uint32_t* c = count + (size_t)blockIdx.x * blocks;
    uint32_t run = 0;
    for (int b = 0; b < blocks; b += 64) {
        const int i = b + (int)threadIdx.x;
        const uint32_t v = i < blocks ? c[i] : 0;
        const uint32_t inc = wave_scan(v);
        if (i < blocks) c[i] = run + inc - v;
        run += __shfl(inc, 63);
    }
    if (threadIdx.x == 0) total[blockIdx.x] = run;
}

// begin[key] = first place of the key's rows, begin[slots + 1] = rows; one wave
__global__ __launch_bounds__(64) void group_begin_kernel(const uint32_t* __restrict__ total, int slots, uint32_t rows,
                                                         uint32_t* __restrict__ begin)
{
    uint32_t run = 0;
    for (int b = 0; b <= slots; b += 64) {
        const int i = b + (int)threadIdx.x;
        const uint32_t v = i <= slots ? total[i] : 0;
        const uint32_t inc = wave_scan(v);
        if (i <= slots) begin[i] = run + inc - v;
        run += __shfl(inc, 63);
    }
    if (threadIdx.x == 0) begin[slots + 1] = rows;
}

// order[place] = row, row_slot[place] = its slot or -1, for rows r0 .. r1 - 1, by one wave; next[key]: where the key's next
// row goes.  The lanes of a lane's key are found bit by bit of the key, whatever keys there are (a turn for each key
// took 50 us more at 8000 rows of 200 slots).
__device__ __forceinline__ void place_rows(const int32_t* __restrict__ slot, uint32_t r0, uint32_t r1, int slots, uint32_t* next,
                                           uint32_t* __restrict__ order, int32_t* __restrict__ row_slot)
{
    const int lane = threadIdx.x & 63, bits = 32 - __clz(slots);
    each_key(slot, r0, r1, slots, [&](uint32_t row, bool in, int key) {
        unsigned long long same = __ballot(in);
        for (int b = 0; b < bits; ++b) {
            const bool one = (key >> b) & 1;
            const unsigned long long ones = __ballot(one);
            same &= one ? ones : ~ones;
        }
        const unsigned long long before = same & ((1ull << lane) - 1);
        const uint32_t base = next[key];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_wave_barrier();  // (every lane has read next[key])
        if (in && before == 0) next[key] = base + (uint32_t)__popcll(same);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_wave_barrier();
        if (in) {
            const uint32_t place = base + (uint32_t)__popcll(before);
            order[place] = row;
            row_slot[place] = key < slots ? key : -1;
        }
    });
}
__global__ __launch_bounds__(64) void group_place_kernel(const int32_t* __restrict__ slot, uint32_t rows, int slots, int blocks,
                                                         const uint32_t* __restrict__ count, const uint32_t* __restrict__ begin,
                                                         uint32_t* __restrict__ order, int32_t* __restrict__ row_slot)
{
    extern __shared__ uint32_t next[];
    for (int k = threadIdx.x; k <= slots; k += 64) next[k] = begin[k] + count[(size_t)k * blocks + blockIdx.x];
    __syncthreads();
    const uint32_t r0 = blockIdx.x * kGroupRows;
    place_rows(slot, r0, min(rows, r0 + kGroupRows), slots, next, order, row_slot);
}

// all of it for one block of rows, in one wave
__global__ __launch_bounds__(64) void group_few_kernel(const int32_t* __restrict__ slot, uint32_t rows, int slots,
                                                       uint32_t* __restrict__ begin, uint32_t* __restrict__ order,
                                                       int32_t* __restrict__ row_slot)
{
    extern __shared__ uint32_t next[];
    for (int k = threadIdx.x; k <= slots; k += 64) next[k] = 0;
    __syncthreads();
    each_key(slot, 0, rows, slots, [&](uint32_t, bool in, int key) { if (in) atomicAdd(&next[key], 1u); });
    __syncthreads();
    uint32_t run = 0;
    for (int b = 0; b <= slots; b += 64) {
        const int i = b + (int)threadIdx.x;
        const uint32_t v = i <= slots ? next[i] : 0;
        const uint32_t inc = wave_scan(v);
        if (i <= slots) begin[i] = next[i] = run + inc - v;
        run += __shfl(inc, 63);
    }
    if (threadIdx.x == 0) begin[slots + 1] = rows;
    __syncthreads();
    place_rows(slot, 0, rows, slots, next, order, row_slot);
}

// ... and for up to kGroupWaves blocks, a wave each
constexpr int kGroupWaves = 16, kGroupMidSlots = 1000;
__global__ __launch_bounds__(64 * kGroupWaves) void group_mid_kernel(const int32_t* __restrict__ slot, uint32_t rows, int slots,
                                                                     uint32_t* __restrict__ begin, uint32_t* __restrict__ order,
                                                                     int32_t* __restrict__ row_slot)
{
    extern __shared__ uint32_t hist[];  // [kGroupWaves][slots + 1]
    __shared__ uint32_t carry[kGroupWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, keys = slots + 1;
    for (int e = threadIdx.x; e < kGroupWaves * keys; e += 64 * kGroupWaves) hist[e] = 0;
    __syncthreads();
    uint32_t* mine = hist + wave * keys;
    const uint32_t per = ((rows + kGroupWaves - 1) / kGroupWaves + 63) & ~63u;
    const uint32_t r0 = min(rows, wave * per), r1 = min(rows, r0 + per);
    each_key(slot, r0, r1, slots, [&](uint32_t, bool in, int key) { if (in) atomicAdd(&mine[key], 1u); });
    __syncthreads();
    // keys in order, the waves of a key in order: a thread per key (keys <= 64 kGroupWaves) adds its waves up
    uint32_t sum = 0;
    const int k = threadIdx.x;
    if (k < keys)
        for (int w = 0; w < kGroupWaves; ++w) { const uint32_t v = hist[w * keys + k]; hist[w * keys + k] = sum; sum += v; }
    const uint32_t inc = wave_scan(sum);
    if (lane == 63) carry[wave] = inc;
    __syncthreads();
    uint32_t base = inc - sum;
    for (int w = 0; w < wave; ++w) base += carry[w];
    if (k < keys) {
        begin[k] = base;
        for (int w = 0; w < kGroupWaves; ++w) hist[w * keys + k] += base;
    }
    if (threadIdx.x == 0) begin[slots + 1] = rows;
    __syncthreads();
    place_rows(slot, r0, r1, slots, mine, order, row_slot);
}

// ---- rows in that order -------------------------------------------------------------------------
// xs[i] = [x[order[i]] | 0 ...] with input dropout (element j of row r zeroed where uniform01(seed,
// counter0 + r, j) < dropout: the draws of szh_net_accumulate_dev), live[i] = any element left.  One wave per row.
__global__ __launch_bounds__(256) void gather_rows_kernel(const float* __restrict__ x, const uint32_t* __restrict__ order,
                                                          uint32_t rows, int in, float dropout, uint64_t seed, uint64_t counter0,
                                                          float* __restrict__ xs, int ldx, uint8_t* __restrict__ live)
{
    const uint32_t i = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= rows) return;
    const uint32_t r = order[i];
    const int lane = threadIdx.x & 63;
    bool any = false;
    for (int j = lane; j < ldx; j += 64) {
        float v = 0.0f;
        if (j < in) {
            v = x[(size_t)r * in + j];
            if (dropout > 0.0f && uniform01(seed, counter0 + r, (uint64_t)j) < dropout) v = 0.0f;
            any = any || v != 0.0f;
        }
        xs[(size_t)i * ldx + j] = v;
    }
    if (live) {
        const bool some = __any(any);
        if (lane == 0) live[i] = some ? 1 : 0;
    }
}

// ---- the first layer and its rank columns ------------------------------------------------------------
// use ? v : 0 for a loaded v.  Of a plain select the compiler may make a branch with the load in it, where it is waited for
// before the next is asked for (sixteen such loads in a row took 16 us).
__device__ __forceinline__ float keep_if(bool use, float v)
{
    asm("" : "+v"(v));
    return use ? v : 0.0f;
}
// Four neighbouring values p[at .. at + 3], those from `end` on as zeros, in two steps: what is asked for first and what is
// waited for later.  FOURS: p is 16-byte aligned, at and end in fours (a template's choice for the same reason).
template <bool FOURS>
__device__ __forceinline__ f32x4 ask_four(const float* __restrict__ p, int at, int end)
{
    if (FOURS) return *reinterpret_cast<const f32x4*>(p + min(at, end - 4));
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = p[min(at + e, end - 1)];
    return v;
}
__device__ __forceinline__ f32x4 cut_four(f32x4 v, int at, int end)
{
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = keep_if(at + e < end, v[e]);
    return v;
}

// h1 = relu(x W1 + b1) and u2 = scale h1 A2[slot] of up to 64 inputs, 512 units and rank 16 in one pass: x is read where the
// caller has it (row i is x[order[i]]), h1 is written once and not read again.  Workgroups walk along the rows, 16 at a time,
// and keep W1 in registers: a wave has 64 units, and the A2 of those for the slot it saw last (rows come sorted by
// slot).  The next rows' x is asked for while this one's is computed.  All is transposed (rows of the batch along the
// matrix instruction's columns), with unit n0 + 4 (4 (m % 4) + m / 4) + c in row m of the instruction's tile c: a result's
// register i of the four tiles is units n0 + 16 i + 4 q + 0 .. 3 of one row, a 16-byte store and the next product's operand
// as it is.  u2, a sum over all units, is joined in LDS, in the order of the waves.  Rows of another slot than the one at
// hand keep their sums: what a row gets does not depend on its neighbours.
// 66140 x 60 x 512 with rank 16: 74 us, of which the matrix instructions take 38 and writing h1 28 (the gather, the product
// and the pass over h1 that it replaces took 17, 57 and 29).  The two waves of a SIMD unit go through products, stores and
// joins nearly in step, so that these add up; a barrier at every fourth tile instead of every one lets them drift (80 -> 74),
// 32 rows at a time (82) or raised priority of one of them (80 .. 87) do not help.
constexpr int kFrontWaves = 8, kFrontIn = 64;
constexpr int kFrontGroup = 4;  // tiles from one barrier to the next
struct FrontArgs {
    const float* x;
    const uint32_t* order;   // null: x's rows are in order
    const float *w1, *b1, *a2;  // [in][n1], [n1], slot 0's [n1][rank]
    uint64_t per_slot;
    const int32_t* row_slot;
    float *h1, *u2;
    uint8_t* live;           // null, or any element of x but 0
    uint32_t rows;
    int in, ldx, n1, ld1, rank, ldu;
    float scale;
};
// FOURS: the rows of x, W1 and b1 are 16-byte aligned and in fours
template <bool FOURS>
__global__ __launch_bounds__(64 * kFrontWaves) void front_kernel(FrontArgs a)
{
    extern __shared__ __attribute__((aligned(16))) float front_lds[];  // [2 kFrontGroup][waves][16][17]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int r16 = lane & 15, q = lane >> 4;
    const uint32_t tiles = (a.rows + 15) / 16;
    const uint32_t first = (uint32_t)((uint64_t)tiles * blockIdx.x / gridDim.x), last = (uint32_t)((uint64_t)tiles * (blockIdx.x + 1) / gridDim.x);
    if (first >= last) return;
    const int n0 = 64 * wave, unit4 = n0 + 4 * (4 * (r16 & 3) + (r16 >> 2));
    f32x4 w[4][4], bias[4];  // (zeros beyond the inputs and units: relu makes 0 of those units whatever x holds)
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int k = 16 * b + 4 * q + e;
            w[b][e] = ask_four<FOURS>(a.w1 + (uint32_t)min(k, a.in - 1) * (uint32_t)a.n1, unit4, a.n1);
        }
#pragma unroll
    for (int i = 0; i < 4; ++i) bias[i] = ask_four<FOURS>(a.b1, n0 + 16 * i + 4 * q, a.n1);
    // rows of a tile, x's row for each, its slot; tiles behind the last one are the last one
    auto at = [&](uint32_t tile) { return min(16 * min(tile, last - 1) + r16, a.rows - 1); };
    auto source = [&](uint32_t tile) { return a.order ? a.order[at(tile)] : at(tile); };
    f32x4 x[4], next[4];
    uint32_t ahead = source(first + 1);
    int slot_of = a.row_slot[at(first)];
    {
        const float* p = a.x + (size_t)source(first) * a.ldx;
#pragma unroll
        for (int b = 0; b < 4; ++b) x[b] = ask_four<FOURS>(p, 16 * b + 4 * q, a.in);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) w[b][e] = cut_four(w[b][e], unit4, 16 * b + 4 * q + e < a.in ? a.n1 : 0);
    f32x4 start[4];  // the bias as the products start from it, [tile of the instruction]
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        bias[i] = cut_four(bias[i], n0 + 16 * i + 4 * q, a.n1);
#pragma unroll
        for (int c = 0; c < 4; ++c) start[c][i] = bias[i][c];
    }
    // only the last piece of x can reach beyond the inputs
    const int tail = (a.in - 1) / 16;
    auto cut_x = [&](f32x4* v) {
#pragma unroll
        for (int b = 0; b < 4; ++b)
            if (b >= tail) v[b] = cut_four(v[b], 16 * b + 4 * q, a.in);
    };
    cut_x(x);
    // where a lane's four stores of the tile at hand go, and how far on the next tile's are
    float* dst[4];
    size_t on[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = n0 + 16 * i + 4 * q;
        dst[i] = n < a.ld1 ? a.h1 + (size_t)(16 * first + r16) * a.ld1 + n : a.h1 + (size_t)(a.rows + 31) * a.ld1 + 4 * (lane & 7);
        on[i] = n < a.ld1 ? (size_t)16 * a.ld1 : 0;
    }
    // Every lane stores at every tile, those without a row into the rows behind the last one, those without a unit into
    // one of those: behind a store that may not have happened the wait for the next x would be for the store as well.
    int r_out = threadIdx.x / a.ldu, j_out = threadIdx.x % a.ldu;
    auto part_of = [&](uint32_t tile) { return reinterpret_cast<float (*)[16][17]>(front_lds) + ((tile - first) % (2 * kFrontGroup)) * waves; };
    auto join_one = [&](uint32_t tile, int r, int j) {
        const float (*part)[16][17] = part_of(tile);
        float s = 0.0f;
        if (waves == kFrontWaves) {
#pragma unroll
            for (int v = 0; v < kFrontWaves; ++v) s += part[v][j][r];
        } else {
            for (int v = 0; v < waves; ++v) s += part[v][j][r];
        }
        if (16 * tile + r < a.rows) a.u2[(size_t)(16 * tile + r) * a.ldu + j] = j < a.rank ? a.scale * s : 0.0f;
    };
    auto join = [&](uint32_t tile) {
        if ((int)threadIdx.x < 16 * a.ldu) join_one(tile, r_out, j_out);
        for (int e = threadIdx.x + blockDim.x; e < 16 * a.ldu; e += blockDim.x) join_one(tile, e / a.ldu, e % a.ldu);
    };
    int have = -1;      // the slot that f belongs to
    float f[4][4];      // A2 of unit n0 + 16 i + 4 q + c, rank column r16
    for (uint32_t tile = first; tile < last; ++tile) {
        const float* p = a.x + (size_t)ahead * a.ldx;
#pragma unroll
        for (int b = 0; b < 4; ++b) next[b] = ask_four<FOURS>(p, 16 * b + 4 * q, a.in);
        ahead = source(tile + 2);
        const int slot_next = a.row_slot[at(tile + 1)];
        const uint32_t row = 16 * tile + r16;
        const bool in = row < a.rows;
        if (a.live && wave == 0) {
            bool any = false;
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) any = any || x[b][e] != 0.0f;
            const unsigned long long some = __ballot(any);
            if (q == 0 && in) a.live[row] = ((some >> r16) & 0x0001000100010001ull) != 0;
        }
        f32x4 h[4];  // [tile of the instruction]
#pragma unroll
        for (int c = 0; c < 4; ++c) h[c] = start[c];
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int c = 0; c < 4; ++c) h[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[b][e][c], x[b][e], h[c], 0, 0, 0);
        if (tile >= first + kFrontGroup) join(tile - kFrontGroup);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f32x4 v;
#pragma unroll
            for (int c = 0; c < 4; ++c) h[c][i] = v[c] = gemm::relu_of_product(h[c][i]);
            *reinterpret_cast<f32x4*>(dst[i]) = v;
            dst[i] += on[i];
        }
        f32x4 u = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        uint32_t left = (uint32_t)__ballot(in && slot_of >= 0) & 0xffffu;
        while (left) {
            const int slot = __builtin_amdgcn_readlane(slot_of, __builtin_ctz(left));
            const bool mem = slot_of == slot;
            left &= ~(uint32_t)__ballot(mem);
            if (slot != have) {
                have = slot;
                const float* a2 = a.a2 + (size_t)slot * a.per_slot;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int c = 0; c < 4; ++c) f[i][c] = a2[(uint32_t)min(n0 + 16 * i + 4 * q + c, a.n1 - 1) * (uint32_t)a.rank + min(r16, a.rank - 1)];
                __builtin_amdgcn_sched_barrier(0);
                int unit = n0 + 4 * q, col = r16;
                asm("" : "+v"(unit), "+v"(col));  // (or thirty-two masks are kept in scalar registers all along)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int c = 0; c < 4; ++c) f[i][c] = keep_if(unit + 16 * i + c < a.n1 && col < a.rank, f[i][c]);
            }
            f32x4 v[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) v[c & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(f[i][c], h[c][i], v[c & 1], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = mem ? v[0][i] + v[1][i] : u[i];
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) x[b] = next[b];
        cut_x(x);
        slot_of = slot_next;
        // (who writes a buffer again has passed the barrier behind everyone's reads of it)
#pragma unroll
        for (int i = 0; i < 4; ++i) part_of(tile)[wave][4 * q + i][r16] = u[i];
        if ((tile - first) % kFrontGroup == kFrontGroup - 1 || tile + 1 == last) __syncthreads();
    }
    for (uint32_t tile = last - min(last - first, (uint32_t)kFrontGroup); tile < last; ++tile) join(tile);
}

// ---- products with the rank columns ----------------------------------------------------------------
// u[i][j] = scale * sum_k x[i][k] F[k][j],  F = the [K][rank] matrix of row i's slot with element (k, j) at
// k * f_k + j * f_j.  Columns from rank to ldu, and rows without a slot, are zero.  With W (the output layer of few
// classes) one pass over x gives the logits too: y = x W + bias + u B, B the slot's [rank][out] matrix.
struct LowArgs {
    const float* x;      // [rows][ldx], 16-byte aligned rows
    const float* factor; // slot 0's matrix
    uint64_t factor_slot;
    const int32_t* row_slot;
    float* u;
    uint32_t rows;
    int ldx, K, f_k, f_j, rank, ldu;
    float scale;
    int parts;           // the slots of a tile are dealt to this many workgroups (few tiles of many slots)
    // the output layer
    const float *W, *bias, *up;
    uint64_t up_slot;
    float* y;
    int out, ldy;
};

// 32 rows per workgroup on v_mfma_f32_16x16x4_f32, the K range split over its waves and joined in LDS.  A step
// pairs lane group q's k with k0 + 4 q + t, so that a lane reads 16 bytes of its row for four steps.  UNR blocks of
// 16 k are requested at once: with as many rows as there are, what a wave does is wait.  NT tiles of 16
// columns: OT of the output layer, then the rank's.  A column beyond the matrix takes another's values and is dropped.
// FOURS (OT = 0): f_k is 1 and the factor's columns are 16-byte aligned, in fours.
// Bound by memory: 66140 x 512 with rank 16 29 us (4.7 TB/s) on four waves and four blocks, 39 on eight waves; 26456 x 2048
// with rank 32 57 us on two blocks (3.8 TB/s), 70 on eight waves, 130 on four blocks (their registers leave too few waves);
// logits of 16 classes and 16 rank columns of 66140 x 256 in 27 us, 38 with the loads where the compiler puts them.
template <int NT, int OT, int WAVES, int UNR, bool FOURS>
__global__ __launch_bounds__(64 * WAVES) void low_kernel(LowArgs a)
{
    extern __shared__ __attribute__((aligned(16))) float low_lds[];
    float (*part)[32][NT * 16] = reinterpret_cast<float (*)[32][NT * 16]>(low_lds);
    constexpr int RT = NT - OT;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r16 = lane & 15, q = lane >> 4;
    const uint32_t row0 = blockIdx.x * 32;
    const uint32_t my_row = row0 + (lane & 31);
    const int mine = my_row < a.rows ? a.row_slot[my_row] : -1;
    // rows without an adapter are a group of their own (slot -1), which the output layer computes with u = 0
    uint32_t left = (uint32_t)__ballot(my_row < a.rows && (OT > 0 || mine >= 0));
    const int blocks = (a.K + 15) / 16, per = (blocks + WAVES - 1) / WAVES;
    const int b0 = wave * per, b1 = min(blocks, b0 + per), full = min(b1, a.K / 16);
    const float* x[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) x[t] = a.x + (size_t)min(row0 + 16 * t + r16, a.rows - 1) * a.ldx + 4 * q;
    if (OT == 0 && blockIdx.y == 0) {
        const uint32_t none = ~left;
        for (int e = threadIdx.x; e < 32 * a.ldu; e += 64 * WAVES) {
            const int r = e / a.ldu;
            if (row0 + r < a.rows && ((none >> r) & 1u)) a.u[(size_t)(row0 + r) * a.ldu + e % a.ldu] = 0.0f;
        }
    }
    for (int turn = 0; left; ++turn) {
        const int slot = __builtin_amdgcn_readlane(mine, __builtin_ctz(left));
        const uint32_t member = (uint32_t)__ballot(mine == slot) & left;
        left &= ~member;
        if (turn % a.parts != (int)blockIdx.y) continue;
        const float* f = a.factor + (size_t)max(slot, 0) * a.factor_slot;
        const float* col[NT];
        uint32_t step[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (n < OT) { col[n] = a.W + min(16 * n + r16, a.out - 1); step[n] = (uint32_t)a.out; }
            else { col[n] = f + (size_t)min(16 * (n - OT) + r16, a.rank - 1) * a.f_j; step[n] = (uint32_t)a.f_k; }
        }
        f32x4 acc[2][NT];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[t][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        int b = b0;
        for (; b + UNR <= full; b += UNR) {
            f32x4 xv[UNR][2];
            float w[UNR][4][NT];
#pragma unroll
            for (int i = 0; i < UNR; ++i) {
#pragma unroll
                for (int t = 0; t < 2; ++t) xv[i][t] = *reinterpret_cast<const f32x4*>(x[t] + 16 * (b + i));
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (FOURS) {
                        const f32x4 v = *reinterpret_cast<const f32x4*>(col[n] + 16 * (b + i) + 4 * q);
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[i][e][n] = v[e];
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[i][e][n] = col[n][(uint32_t)(16 * (b + i) + 4 * q + e) * step[n]];
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);  // every load is asked for before the first is waited for
#pragma unroll
            for (int i = 0; i < UNR; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int t = 0; t < 2; ++t) acc[t][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(xv[i][t][e], w[i][e][n], acc[t][n], 0, 0, 0);
        }
        for (; b < b1; ++b) {
            f32x4 xv[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) xv[t] = *reinterpret_cast<const f32x4*>(x[t] + min(16 * b, a.ldx - 4 - 4 * q));
            float w[4][NT];
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int n = 0; n < NT; ++n) w[e][n] = col[n][(uint32_t)min(16 * b + 4 * q + e, a.K - 1) * step[n]];
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool in_k = 16 * b + 4 * q + e < a.K;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float v = keep_if(in_k, w[e][n]);
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        acc[t][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(in_k ? xv[t][e] : 0.0f, v, acc[t][n], 0, 0, 0);
                }
            }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) part[wave][16 * t + 4 * q + i][16 * n + r16] = acc[t][n][i];
        __syncthreads();
        // the output layer's second product: its 2 OT tiles of 16 x 16 are dealt to the waves, their factors asked for ahead
        constexpr int TILES = (2 * OT + WAVES - 1) / WAVES;
        float up[TILES ? TILES : 1][RT * 4];
#pragma unroll
        for (int y = 0; y < TILES; ++y) {
            const float* B = a.up + (size_t)max(slot, 0) * a.up_slot + min(16 * ((wave + y * WAVES) >> 1) + r16, a.out - 1);
#pragma unroll
            for (int k = 0; k < RT * 4; ++k) up[y][k] = B[(size_t)min(4 * k + q, a.rank - 1) * a.out];
        }
        __builtin_amdgcn_sched_barrier(0);
        for (int e = threadIdx.x; e < 32 * RT * 16; e += 64 * WAVES) {
            const int r = e / (RT * 16), j = e % (RT * 16);
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) s += part[w][r][OT * 16 + j];
            s = slot >= 0 && j < a.rank ? a.scale * s : 0.0f;
            if (j < a.ldu && row0 + r < a.rows && ((member >> r) & 1u)) a.u[(size_t)(row0 + r) * a.ldu + j] = s;
            if (OT > 0) part[0][r][OT * 16 + j] = s;  // (read by this thread alone before)
        }
        if (OT > 0) {
            __syncthreads();
#pragma unroll
            for (int y = 0; y < TILES; ++y) {
                const int tile = wave + y * WAVES, yt = tile & 1, c = 16 * (tile >> 1) + r16;
                if (tile >= 2 * OT) break;
                f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < RT * 4; ++k) {
                    const float w = keep_if(slot >= 0 && 4 * k + q < a.rank, up[y][k]);
                    v = __builtin_amdgcn_mfma_f32_16x16x4f32(part[0][16 * yt + r16][OT * 16 + 4 * k + q], w, v, 0, 0, 0);
                }
                const float bias = a.bias[min(c, a.out - 1)];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = 16 * yt + 4 * q + i;
                    float s = 0.0f;
#pragma unroll
                    for (int w = 0; w < WAVES; ++w) s += part[w][r][c];
                    if (c < a.out && row0 + r < a.rows && ((member >> r) & 1u)) a.y[(size_t)(row0 + r) * a.ldy + c] = s + v[i] + bias;
                }
            }
        }
        __syncthreads();
    }
}

// ---- backward through the output layer ---------------------------------------------------------------
// g3 = scale d3 B3^T, d2 = (d3 W3^T + g3 A3^T)(1 - h2^2), g2 = scale d2 B2^T for 16 T rows per workgroup, d3 and h2 read
// and d2, g2, g3 written once.  Everything is computed transposed (rows of the batch along the matrix instruction's
// columns): a result's four registers then are four neighbouring units of one row, which is what the next product's
// operand and 16-byte loads and stores want.  The waves deal the hidden units among themselves; g2, a sum over all
// of them, is joined in LDS.  66140 x 256 x 16 with rank 16: 43 us for 140 MB (79 with the factors read value by value, 90
// and 114 on one wave with 32 and 16 rows).
struct BackArgs {
    const float *d3, *h2, *w3;        // [rows][ld3], [rows][ld2], [n2][out]
    const float *a3, *b3, *b2;        // slot 0's factors [n2][rank], [rank][out], [rank][n2]
    uint64_t per_slot;
    const int32_t* row_slot;
    float *d2, *g2, *g3;              // [rows][ld2], [rows][ldu]
    uint32_t rows;
    int n2, out, rank, ld2, ld3, ldu;
    float scale;
};
// d3(t, row, c): four classes of a row of tile t.  FOURS: the rows of W3, A3 and B2 are 16-byte aligned and in fours.
template <int RT, int WAVES, int T, bool FOURS, class D3>
__device__ __forceinline__ void back_tiles(const BackArgs& a, float (*part)[T][RT * 16][17], D3 d3)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r16 = lane & 15, q = lane >> 4;
    const uint32_t row0 = blockIdx.x * (16 * T);
    const uint32_t my_row = row0 + (lane & (16 * T - 1));
    const int mine = my_row < a.rows ? a.row_slot[my_row] : -1;
    constexpr uint32_t MASK = T == 2 ? 0xffffffffu : 0xffffu;
    uint32_t left = (uint32_t)__ballot(my_row < a.rows) & MASK;
    size_t row[T];
#pragma unroll
    for (int t = 0; t < T; ++t) row[t] = min(row0 + 16 * t + r16, a.rows - 1);
    const int tiles = (a.n2 + 15) / 16;
    const int out4 = (a.out + 3) & ~3;  // (ld3 is a multiple of 4: whole 16-byte pieces lie inside a row of d3)
    while (left) {
        const int slot = __builtin_amdgcn_readlane(mine, __builtin_ctz(left));
        const uint32_t member = (uint32_t)__ballot(mine == slot) & left;
        left &= ~member;
        if (slot < 0) {  // rows without an adapter: d3 is zero there
            for (int e = threadIdx.x; e < 16 * T * a.n2; e += 64 * WAVES)
                if ((member >> (e / a.n2)) & 1u) a.d2[(size_t)(row0 + e / a.n2) * a.ld2 + e % a.n2] = 0.0f;
            for (int e = threadIdx.x; e < 16 * T * a.ldu; e += 64 * WAVES)
                if ((member >> (e / a.ldu)) & 1u) a.g2[(size_t)(row0 + e / a.ldu) * a.ldu + e % a.ldu] = a.g3[(size_t)(row0 + e / a.ldu) * a.ldu + e % a.ldu] = 0.0f;
            continue;
        }
        const float* a3 = a.a3 + (size_t)slot * a.per_slot;
        const float* b3 = a.b3 + (size_t)slot * a.per_slot;
        const float* b2 = a.b2 + (size_t)slot * a.per_slot;
        bool mem[T];
#pragma unroll
        for (int t = 0; t < T; ++t) mem[t] = ((member >> (16 * t + r16)) & 1u) != 0;
        // g3^T: registers j = 16 n + 4 q + i of row r16 (every wave has all of it)
        f32x4 g3[T][RT], g2[T][RT];
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int n = 0; n < RT; ++n) g3[t][n] = g2[t][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int c0 = 0; c0 < out4; c0 += 16) {
            const int c = c0 + 4 * q;
            f32x4 d[T];
#pragma unroll
            for (int t = 0; t < T; ++t) d[t] = d3(t, row[t], c);
            float b[4][RT];
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int n = 0; n < RT; ++n) b[e][n] = b3[(size_t)min(16 * n + r16, a.rank - 1) * a.out + min(c + e, a.out - 1)];
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool in = c + e < a.out;
#pragma unroll
                for (int n = 0; n < RT; ++n) {
                    const float w = keep_if(in && 16 * n + r16 < a.rank, b[e][n]);
#pragma unroll
                    for (int t = 0; t < T; ++t) g3[t][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(w, in ? d[t][e] : 0.0f, g3[t][n], 0, 0, 0);
                }
            }
        }
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int n = 0; n < RT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    g3[t][n][i] *= a.scale;
                    const int j = 16 * n + 4 * q + i;
                    if (wave == 0 && mem[t] && j < a.ldu) a.g3[row[t] * a.ldu + j] = g3[t][n][i];
                }
#pragma unroll 2
        for (int tile = wave; tile < tiles; tile += WAVES) {
            const int n0 = 16 * tile, u = min(n0 + r16, a.n2 - 1);  // the unit whose weights this lane holds
            f32x4 h[T], d2[T];
#pragma unroll
            for (int t = 0; t < T; ++t) {
                h[t] = *reinterpret_cast<const f32x4*>(a.h2 + row[t] * a.ld2 + n0 + 4 * q);
                d2[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
            f32x4 wb[RT], wa[RT];
#pragma unroll
            for (int n = 0; n < RT; ++n) {
                wb[n] = ask_four<FOURS>(b2 + (size_t)min(16 * n + r16, a.rank - 1) * a.n2, n0 + 4 * q, a.n2);
                wa[n] = ask_four<FOURS>(a3 + (size_t)u * a.rank, 16 * n + 4 * q, a.rank);
            }
            for (int c0 = 0; c0 < out4; c0 += 16) {
                const int c = c0 + 4 * q;
                f32x4 d[T];
#pragma unroll
                for (int t = 0; t < T; ++t) d[t] = d3(t, row[t], c);
                f32x4 w = ask_four<FOURS>(a.w3 + (size_t)u * a.out, c, a.out);
                __builtin_amdgcn_sched_barrier(0);
                w = cut_four(w, c, a.out);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool in = c + e < a.out;
#pragma unroll
                    for (int t = 0; t < T; ++t) d2[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[e], in ? d[t][e] : 0.0f, d2[t], 0, 0, 0);
                }
            }
#pragma unroll
            for (int n = 0; n < RT; ++n) {
                wb[n] = cut_four(wb[n], n0 + 4 * q, 16 * n + r16 < a.rank ? a.n2 : 0);
                wa[n] = cut_four(wa[n], 16 * n + 4 * q, a.rank);
            }
#pragma unroll
            for (int n = 0; n < RT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int t = 0; t < T; ++t) d2[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(wa[n][e], g3[t][n][e], d2[t], 0, 0, 0);
            // Every matrix result is read before the first branch behind it: the compiler's count of wait states over several
            // ways to one place can miss the shortest (seen: a result's last register read 3 states behind, where 10 are due).
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float v = d2[t][i] * (1.0f - h[t][i] * h[t][i]);
                    asm volatile("" : "+v"(v));
                    d2[t][i] = v;
                }
#pragma unroll
            for (int t = 0; t < T; ++t) {
                // (columns between n2 and ld2 take products with zeros, or zeros: the padding of h2 and the clamped unit's
                // weights are finite or theirs alone; only whole pieces inside ld2 are stored)
                if (mem[t]) {
                    float* dst = a.d2 + row[t] * a.ld2 + n0 + 4 * q;
                    if (n0 + 4 * q + 3 < a.n2) *reinterpret_cast<f32x4*>(dst) = d2[t];
                    else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (n0 + 4 * q + i < a.n2) dst[i] = d2[t][i];
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) d2[t][i] = n0 + 4 * q + i < a.n2 ? d2[t][i] : 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int n = 0; n < RT; ++n)
#pragma unroll
                    for (int t = 0; t < T; ++t) g2[t][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(wb[n][e], d2[t][e], g2[t][n], 0, 0, 0);
        }
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int n = 0; n < RT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) part[wave][t][16 * n + 4 * q + i][r16] = g2[t][n][i];
        __syncthreads();
        for (int e = threadIdx.x; e < 16 * T * a.ldu; e += 64 * WAVES) {
            const int r = e / a.ldu, j = e % a.ldu;
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) s += part[w][r >> 4][j][r & 15];
            if ((member >> r) & 1u) a.g2[(size_t)(row0 + r) * a.ldu + j] = j < a.rank ? a.scale * s : 0.0f;
        }
        __syncthreads();
    }
}
template <int RT, int WAVES, int T, bool FOURS>
__global__ __launch_bounds__(64 * WAVES) void back_kernel(BackArgs a)
{
    __shared__ float part[WAVES][T][RT * 16][17];
    back_tiles<RT, WAVES, T, FOURS>(a, part, [&](int, size_t row, int c) { return *reinterpret_cast<const f32x4*>(a.d3 + row * a.ld3 + min(c, a.ld3 - 4)); });
}

// The output layer and back in one launch, for up to 16 rank columns and 64 classes (OT tiles of 16): u3, the logits,
// controls and softmax, the loss, d3, and what back_kernel makes of it.  A workgroup has 16 T rows; their logits and
// d3 stay in LDS, and what of h2 the second half reads is still in the cache.  66140 x 256 x 16 with rank 16: 68 us (28, 9 and
// 43 for low_kernel, the controls and back_kernel), 19 of them matrix and 26 vector instructions, which take turns on a SIMD
// unit, for 150 MB; more waves a unit do not help (71 us at five, 95 at six: registers).
struct TailArgs {
    const float* bias;
    float *u3, *d3;   // [rows][ldu], [rows][ld3]
};
template <int OT, int WAVES, int T, bool FOURS>
__global__ __launch_bounds__(64 * WAVES) void tail_kernel(BackArgs a, TailArgs o, Controls ctl, ControlRun run)
{
    constexpr int LD = 16 * OT + 4, PER = 64 * WAVES / (16 * T);  // PER lanes have a row of the softmax
    __shared__ __attribute__((aligned(16))) float sums[WAVES][T][(OT + 1) * 16][17];  // classes, then rank columns
    __shared__ __attribute__((aligned(16))) float z[16 * T][LD];                       // logits, then d3
    __shared__ float us[16 * T][17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r16 = lane & 15, q = lane >> 4;
    const uint32_t row0 = blockIdx.x * (16 * T);
    const uint32_t my_row = row0 + (lane & (16 * T - 1));
    const int mine = my_row < a.rows ? a.row_slot[my_row] : -1;
    const uint32_t adapted = (uint32_t)__ballot(mine >= 0) & (T == 2 ? 0xffffffffu : 0xffffu);
    {
        size_t row[T];
#pragma unroll
        for (int t = 0; t < T; ++t) row[t] = min(row0 + 16 * t + r16, a.rows - 1);
        // transposed as in back_tiles: register i of a lane is class 16 y + 4 q + i, or that rank column, of row r16
        f32x4 y[T][OT], u[T];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            u[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int n = 0; n < OT; ++n) y[t][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        const int tiles = (a.n2 + 15) / 16;
        for (int tile = wave; tile < tiles; tile += WAVES) {
            const int n0 = 16 * tile;
            f32x4 h[T];
            float w[4][OT], f[4];
#pragma unroll
            for (int t = 0; t < T; ++t) h[t] = *reinterpret_cast<const f32x4*>(a.h2 + row[t] * a.ld2 + n0 + 4 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int n = 0; n < OT; ++n) w[e][n] = a.w3[(size_t)min(n0 + 4 * q + e, a.n2 - 1) * a.out + min(16 * n + r16, a.out - 1)];
            auto ask = [&](int slot) {
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] = a.a3[(size_t)slot * a.per_slot + (size_t)min(n0 + 4 * q + e, a.n2 - 1) * a.rank + min(r16, a.rank - 1)];
            };
            uint32_t left = adapted;
            int slot = left ? __builtin_amdgcn_readlane(mine, __builtin_ctz(left)) : 0;
            ask(slot);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool in = n0 + 4 * q + e < a.n2;
#pragma unroll
                for (int t = 0; t < T; ++t) h[t][e] = in ? h[t][e] : 0.0f;
#pragma unroll
                for (int n = 0; n < OT; ++n) {
                    const float v = keep_if(in, w[e][n]);
#pragma unroll
                    for (int t = 0; t < T; ++t) y[t][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, h[t][e], y[t][n], 0, 0, 0);
                }
            }
            while (left) {
                left &= ~(uint32_t)__ballot(mine == slot);
                f32x4 v[T];
#pragma unroll
                for (int t = 0; t < T; ++t) v[t] = u[t];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float g = keep_if(n0 + 4 * q + e < a.n2, f[e]);
#pragma unroll
                    for (int t = 0; t < T; ++t) v[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(g, h[t][e], v[t], 0, 0, 0);
                }
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    const bool mem = __shfl(mine, 16 * t + r16) == slot;
#pragma unroll
                    for (int i = 0; i < 4; ++i) u[t][i] = mem ? v[t][i] : u[t][i];
                }
                if (left) {
                    slot = __builtin_amdgcn_readlane(mine, __builtin_ctz(left));
                    ask(slot);
                }
            }
        }
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sums[wave][t][OT * 16 + 4 * q + i][r16] = u[t][i];
#pragma unroll
                for (int n = 0; n < OT; ++n) sums[wave][t][16 * n + 4 * q + i][r16] = y[t][n][i];
            }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * T * 16; e += 64 * WAVES) {
        const int r = e >> 4, j = e & 15;
        const bool on = ((adapted >> r) & 1u) && j < a.rank;
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) s += sums[w][r >> 4][OT * 16 + j][r & 15];
        s = on ? a.scale * s : 0.0f;
        us[r][j] = s;
        if (j < a.ldu && row0 + r < a.rows) o.u3[(size_t)(row0 + r) * a.ldu + j] = s;
    }
    __syncthreads();
    const int r = threadIdx.x / PER, l = threadIdx.x % PER;
    const uint32_t i = min(row0 + r, a.rows - 1);
    const bool real = row0 + r < a.rows;
    const int slot = a.row_slot[i];
    const float* b3 = a.b3 + (size_t)max(slot, 0) * a.per_slot;
    const uint64_t row = run.order ? run.order[i] : i;
    const control::RowControl rc = control::row_control(ctl, a.out, control::row_set(ctl, row));
    float top = -INFINITY;
    for (int c = l; c < a.out; c += PER) {
        float b[16], v = 0.0f, low = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; ++j) b[j] = b3[(size_t)min(j, a.rank - 1) * a.out + c];
        const float bias = o.bias[c];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v += sums[w][r >> 4][c][r & 15];
#pragma unroll
        for (int j = 0; j < 16; ++j) low = __builtin_fmaf(us[r][j], keep_if(slot >= 0 && j < a.rank, b[j]), low);
        v = control::controlled(rc, v + low + bias, c);
        z[r][c] = v;
        top = fmaxf(top, v);
    }
    top = control::lanes_max<PER>(top);
    const float shift = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    for (int c = l; c < a.out; c += PER) {
        const float e = control::exp_low(z[r][c] - shift);
        z[r][c] = e;
        sum += e;
    }
    sum = control::lanes_sum<PER>(sum);
    const bool some = !(sum <= 0.0f);  // (a NaN row stays one)
    const float inv = some ? 1.0f / sum : 0.0f;
    const control::TrainRow tr = control::train_row(run, rc, i, row, a.out, some);
    for (int c = l; c < LD; c += PER) {
        float v = 0.0f;
        if (c < a.out && tr.live) {
            const float p = z[r][c] * inv;
            v = c == tr.label ? p - 1.0f : p;
            if (inv != inv && !control::allowed(rc, c)) v = 0.0f;
            if (real && c == tr.label) run.loss[i] = -logf(fmaxf(p, 1e-12f));
        }
        z[r][c] = v;
        if (real && c < a.out) o.d3[(size_t)i * a.ld3 + c] = v;
    }
    if (real && l == 0) {
        run.live[i] = tr.live ? 1 : 0;
        if (!tr.live) run.loss[i] = 0.0f;
    }
    __syncthreads();
    back_tiles<1, WAVES, T, FOURS>(a, reinterpret_cast<float (*)[T][16][17]>(&sums[0][0][0][0]),
                                   [&](int t, size_t, int c) { return *reinterpret_cast<const f32x4*>(&z[16 * t + r16][min(c, 16 * OT)]); });
}

// ---- factor gradients -----------------------------------------------------------------------------
// The four factors' gradients are four contractions over rows, grad[slot][m][j] = sum over the slot's rows of
// p[i][m] w[i][j], m up to a layer's width and j the rank columns; one launch does all four.  A row that does not count has
// zeros for either operand, whatever its activations are (0 x inf would be a NaN in every element of the slot).
// Rows are sorted by slot, so a chunk of rows holds the rest of one slot that begins in an earlier chunk, if of any, and slots that begin
// in it: the part of the former goes to chunk_slab[chunk][m][j], those of the latter to slot_slab[slot][m][j], which needs no table and no
// more room for the slots, however many rows there are.  factor_reduce_kernel adds a slot's chunks.
struct FactorJob {
    const float* p;        // [rows][ldp], 16-byte aligned rows
    const float* w;        // [rows][ldw], the rank columns
    float *slot_slab, *chunk_slab;
    uint64_t off;          // the factor's place in a slot's gradient: element (m, j) at off + m * g_m + j * g_j
    int ldp, M, g_m, g_j;
    int first;             // first tile of 64 columns of this job
    int first_out;         // first block of 256 elements of this job in factor_reduce_kernel
};
struct FactorArgs {
    FactorJob job[4];
    const uint32_t* begin; // [slots + 2]
    const int32_t* row_slot;
    const uint8_t* live;
    int ldw, rank, slots;
    uint32_t chunk;        // rows per chunk
};

// 64 columns of p per workgroup; its four waves take rows in turn and are joined in LDS.  A lane reads 16
// bytes of a row of p for four matrix instructions: step t's columns are 4 c + t.  G groups of four rows are asked for at
// once: 13228 rows of the wide network with rank 32 89 us by four groups, 111 by two; 66140 rows of the small one 54 us for
// 280 MB either way.
template <int NT, int G>
__global__ __launch_bounds__(256) void factor_grad_kernel(FactorArgs a)
{
    __shared__ __attribute__((aligned(16))) float part[4][64][NT * 16];
    const int which = ((int)blockIdx.x >= a.job[1].first) + ((int)blockIdx.x >= a.job[2].first) + ((int)blockIdx.x >= a.job[3].first);
    const FactorJob g = a.job[which];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c16 = lane & 15, q = lane >> 4;
    const int m0 = ((int)blockIdx.x - g.first) * 64;
    const uint32_t end = min(a.begin[a.slots], (blockIdx.y + 1) * a.chunk);
    uint32_t r = blockIdx.y * a.chunk;
    while (r < end) {
        const int slot = a.row_slot[r];
        const uint32_t stop = min(end, a.begin[slot + 1]);
        f32x4 acc[4][NT];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[t][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        // (G groups of four rows at a time: the loads of all are asked for before the first is waited for)
        for (uint32_t i = r + 4 * wave; i < stop; i += 16 * G) {
            f32x4 pv[G];
            float wv[G][NT];
            uint32_t live[G];
            const int col = m0 + 4 * c16;
#pragma unroll
            for (int g2 = 0; g2 < G; ++g2) {
                const size_t row = min(i + 16 * g2 + q, stop - 1);
                pv[g2] = *reinterpret_cast<const f32x4*>(g.p + row * g.ldp + min(col, g.ldp - 4));
                live[g2] = a.live[row];
#pragma unroll
                for (int n = 0; n < NT; ++n) wv[g2][n] = g.w[row * a.ldw + min(16 * n + c16, a.rank - 1)];
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int g2 = 0; g2 < G; ++g2) {
                const bool in = i + 16 * g2 + q < stop && live[g2] != 0;
                pv[g2] = cut_four(pv[g2], col, in ? g.M : 0);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float v = keep_if(in && 16 * n + c16 < a.rank, wv[g2][n]);
#pragma unroll
                    for (int t = 0; t < 4; ++t) acc[t][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(pv[g2][t], v, acc[t][n], 0, 0, 0);
                }
            }
        }
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) part[wave][4 * (4 * q + i) + t][16 * n + c16] = acc[t][n][i];
        __syncthreads();
        const bool begins = a.begin[slot] >= blockIdx.y * a.chunk;
        float* slab = (begins ? g.slot_slab + (size_t)slot * g.M * a.rank : g.chunk_slab + (size_t)blockIdx.y * g.M * a.rank);
        for (int e = threadIdx.x; e < 64 * a.rank; e += 256) {
            const int m = e / a.rank, j = e % a.rank;
            if (m0 + m < g.M)
                slab[(size_t)(m0 + m) * a.rank + j] = (part[0][m][j] + part[1][m][j]) + (part[2][m][j] + part[3][m][j]);
        }
        __syncthreads();
        r = stop;
    }
}

// sums[slot] += {loss, live rows} of the slot's rows (64 bits, fixed order); tail = the same as floats
__device__ __forceinline__ void slot_stats(int slot, const float* __restrict__ loss, const uint8_t* __restrict__ live,
                                           const uint32_t* __restrict__ begin, double* __restrict__ sums, float* __restrict__ tail)
{
    __shared__ double sl[256], sc[256];
    double l = 0.0, c = 0.0;
    // (eight rows a thread in flight; those behind the last as zeros)
    const uint32_t end = begin[slot + 1];
    for (uint32_t i = begin[slot] + threadIdx.x; i < end; i += 8 * 256) {
        float a[8], b[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) { const uint32_t at = min(i + 256 * k, end - 1); a[k] = loss[at]; b[k] = (float)live[at]; }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < 8; ++k) { l += (double)keep_if(i + 256 * k < end, a[k]); c += (double)keep_if(i + 256 * k < end, b[k]); }
    }
    sl[threadIdx.x] = l; sc[threadIdx.x] = c;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) { sl[threadIdx.x] += sl[threadIdx.x + o]; sc[threadIdx.x] += sc[threadIdx.x + o]; }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const double a = sums[2 * slot] + sl[0], b = sums[2 * slot + 1] + sc[0];
        sums[2 * slot] = a; sums[2 * slot + 1] = b;
        tail[2 * slot] = (float)a; tail[2 * slot + 1] = (float)b;
    }
}

// grad[slot] += the slot's chunks of the slabs (64-bit sums, in chunk order); the last workgroup of a slot adds up its rows
__global__ __launch_bounds__(256) void factor_reduce_kernel(FactorArgs a, float* __restrict__ grad, uint64_t grad_slot, const float* __restrict__ loss,
                                                            const uint8_t* __restrict__ live, double* __restrict__ sums, float* __restrict__ tail)
{
    const int slot = blockIdx.y;
    if (blockIdx.x == gridDim.x - 1) { slot_stats(slot, loss, live, a.begin, sums, tail); return; }
    const uint32_t b = a.begin[slot], e = a.begin[slot + 1];
    if (b == e) return;
    const int which = ((int)blockIdx.x >= a.job[1].first_out) + ((int)blockIdx.x >= a.job[2].first_out) + ((int)blockIdx.x >= a.job[3].first_out);
    const FactorJob g = a.job[which];
    const int i = ((int)blockIdx.x - g.first_out) * 256 + threadIdx.x;
    const int size = g.M * a.rank;
    if (i >= size) return;
    const uint32_t c0 = b / a.chunk, c1 = (e - 1) / a.chunk;
    float* out = grad + (size_t)slot * grad_slot + g.off + (size_t)(i / a.rank) * g.g_m + (size_t)(i % a.rank) * g.g_j;
    const float before = *out;
    double t = 0.0;
    for (uint32_t c = c0; c <= c1; c += 8) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float* at = c + k == c0 ? g.slot_slab + (size_t)slot * size : g.chunk_slab + (size_t)min(c + k, c1) * size;
            v[k] = at[i];
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < 8; ++k) t += (double)keep_if(c + k <= c1, v[k]);
    }
    *out = before + (float)t;
}

// params -= (lr / live) * grad for every slot with live rows (lib.rs:1047-1059, a slot at a time)
__global__ __launch_bounds__(256) void adapter_apply_kernel(float* __restrict__ params, const float* __restrict__ grad,
                                                            const float* __restrict__ tail, uint64_t per_slot, float lr)
{
    const float live = tail[2 * blockIdx.y + 1];
    if (!(live > 0.0f)) return;
    const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < per_slot) params[blockIdx.y * per_slot + i] -= grad[blockIdx.y * per_slot + i] * (lr / live);
}

// (a kernel and not a memory-set node, which must not be captured into a graph)
__global__ __launch_bounds__(256) void adapter_clear_kernel(float* __restrict__ grad, uint64_t n, double* __restrict__ sums, uint64_t n_sums)
{
    const uint64_t step = (uint64_t)gridDim.x * 256;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += step) grad[i] = 0.0f;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < n_sums; i += step) sums[i] = 0.0;
}

}  // namespace adapt
}  // namespace sz
