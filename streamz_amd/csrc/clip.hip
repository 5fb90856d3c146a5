// The norm of gradients over many tensors and their clipping.  No counterpart in the reference, whose
// training (lib.rs:1002-1060) applies every gradient as it is.
//
//   norm_G = sqrt(sum over the tensors of group G of sum g^2) / live_G,   f = norm_G > max_norm ? max_norm / norm_G : 1
//   out = f g
//
// Squares are added in 64 bits (no overflow or underflow of an f32 gradient's squares, and sums of any length
// to f32 accuracy) in an order fixed by the layout: a workgroup per piece of a tensor, then every
// workgroup of the second launch adds its group's pieces for itself.  No atomics, no flags to reset.
// Bound by memory: the gradients once from HBM, once more (out of the last-level cache where they fit) and written once.
#include <algorithm>
#include <new>
#include <vector>

#include "internal.h"
#include "prof.h"
#include "streamz_hip.h"

namespace sz {

namespace {

constexpr int kClipThreads = 256;

__device__ __forceinline__ double block_sum(double v)
{
    __shared__ double part[kClipThreads / 64];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}

// A thread's four 16-byte pieces of a round of the workgroup's 4096 values: at + 1024 j.  Pieces are cut so that
// those of a tensor are 16-byte aligned where both its addresses can be (ClipPiece::vec).
constexpr uint32_t kClipRound = 16 * kClipThreads;
constexpr uint64_t kClipMostPieces = (1ull << 32) / kClipThreads - 1;  // (a launch has fewer than 2^32 threads)

// a store that leaves the caches to the gradients still to be read again (38.8 M of them: 97 -> 80 us)
typedef float vec4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void store_past(float* p, float x, float y, float z, float w)
{
    __builtin_nontemporal_store(vec4{x, y, z, w}, reinterpret_cast<vec4*>(p));
}

__global__ __launch_bounds__(kClipThreads) void clip_squares_kernel(const ClipPiece* __restrict__ pieces, double* __restrict__ part)
{
    const ClipPiece p = pieces[blockIdx.x];
    double s0 = 0.0, s1 = 0.0, s2 = 0.0, s3 = 0.0;
    uint32_t i = 0;
    if (p.vec) {
#pragma unroll 2
        for (; i + kClipRound <= p.len; i += kClipRound) {
            float4 v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const float4*>(p.src + i + 4 * (threadIdx.x + kClipThreads * j));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s0 = __builtin_fma((double)v[j].x, (double)v[j].x, s0); s1 = __builtin_fma((double)v[j].y, (double)v[j].y, s1);
                s2 = __builtin_fma((double)v[j].z, (double)v[j].z, s2); s3 = __builtin_fma((double)v[j].w, (double)v[j].w, s3);
            }
        }
    }
#pragma unroll 4
    for (i += threadIdx.x; i < p.len; i += kClipThreads) { const double v = (double)p.src[i]; s0 = __builtin_fma(v, v, s0); }
    const double s = block_sum((s0 + s1) + (s2 + s3));
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// sums[g] of groups of very many pieces, so that the next kernel's workgroups need not add them each for itself
__global__ __launch_bounds__(kClipThreads) void clip_fold_kernel(const double* __restrict__ part, const uint32_t* __restrict__ first,
                                                                 double* __restrict__ sums)
{
    double s = 0.0;
    for (uint32_t i = first[blockIdx.x] + threadIdx.x; i < first[blockIdx.x + 1]; i += kClipThreads) s += part[i];
    s = block_sum(s);
    if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

__global__ __launch_bounds__(kClipThreads) void clip_scale_kernel(const ClipPiece* __restrict__ pieces, const double* __restrict__ part,
                                                                  const uint32_t* __restrict__ first, const double* __restrict__ sums,
                                                                  const float* __restrict__ live, uint32_t live_step, float max_norm,
                                                                  float* __restrict__ norms)
{
    const ClipPiece p = pieces[blockIdx.x];
    // the first round is on its way while the norm is put together
    float4 v[4];
    const bool round = p.vec && kClipRound <= p.len;
    if (round) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const float4*>(p.src + 4 * (threadIdx.x + kClipThreads * j));
    }
    const uint32_t b = first[p.group], e = first[p.group + 1];
    double s = 0.0;
    if (sums) s = sums[p.group];
    else {
        for (uint32_t i = b + threadIdx.x; i < e; i += kClipThreads) s += part[i];
        s = block_sum(s);
    }
    s = sqrt(s);
    if (live) {
        const double n = (double)live[(uint64_t)p.group * live_step];
        s = n > 0.0 ? s / n : 0.0;  // nothing counted: the update is nothing
    }
    if (norms && blockIdx.x == b && threadIdx.x == 0) norms[p.group] = (float)s;
    const bool clip = s > (double)max_norm;
    if (!clip && p.src == p.dst) return;
    // the factor stays in 64 bits (beside gradients near the type's end it lies below f32's normal range): one rounding a value
    const double f = clip ? (double)max_norm / s : 1.0;
    const auto scaled = [&](float x) { return clip ? (float)((double)x * f) : x; };
    uint32_t i = 0;
    if (p.vec) {
        for (; i + kClipRound <= p.len; i += kClipRound) {
            float4 o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = v[j];
            if (i + 2 * kClipRound <= p.len) {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const float4*>(p.src + i + kClipRound + 4 * (threadIdx.x + kClipThreads * j));
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                store_past(p.dst + i + 4 * (threadIdx.x + kClipThreads * j), scaled(o[j].x), scaled(o[j].y), scaled(o[j].z), scaled(o[j].w));
        }
    }
#pragma unroll 4
    for (i += threadIdx.x; i < p.len; i += kClipThreads) p.dst[i] = scaled(p.src[i]);
}

__global__ void clip_empty_kernel(const uint32_t* __restrict__ first, uint32_t groups, float* __restrict__ norms)
{
    const uint32_t g = blockIdx.x * 256 + threadIdx.x;
    if (g < groups && first[g] == first[g + 1]) norms[g] = 0.0f;
}

}  // namespace

int clip_create(const ClipTensor* tensors, uint32_t n, uint32_t groups, const float* live, uint32_t live_step, Clip** out)
{
    uint64_t total = 0;
    for (uint32_t t = 0; t < n; ++t) total += tensors[t].len;
    // pieces small enough to fill the chip, few enough that a group's partial sums are quickly added again
    const uint64_t piece = std::min<uint64_t>(std::max<uint64_t>((total / 2048 + kClipRound - 1) / kClipRound * kClipRound, kClipRound), 1u << 24);
    std::vector<uint32_t> order(n);
    for (uint32_t t = 0; t < n; ++t) order[t] = t;
    std::stable_sort(order.begin(), order.end(), [&](uint32_t a, uint32_t b) { return tensors[a].group < tensors[b].group; });
    std::vector<ClipPiece> pieces;
    std::vector<uint32_t> first(groups + 1, 0);
    uint32_t g = 0;
    for (uint32_t k = 0; k < n; ++k) {
        const ClipTensor& t = tensors[order[k]];
        while (g < t.group) first[++g] = (uint32_t)pieces.size();
        // a first piece of up to three values, if that makes both addresses behind it multiples of 16 bytes
        const uint64_t skew = ((uintptr_t)t.src & 15) / sizeof(float);
        const bool vec = ((uintptr_t)t.src & 15) == ((uintptr_t)t.dst & 15);
        if (pieces.size() + t.len / piece + 2 > kClipMostPieces) { set_error("too many tensors, or too long ones"); return SZH_EINVAL; }
        uint64_t at = 0;
        if (vec && skew && t.len > 64) {
            at = 4 - skew;
            pieces.push_back({t.src, t.dst, (uint32_t)at, t.group, 0});
        }
        for (; at < t.len; at += piece) {
            const uint32_t len = (uint32_t)std::min<uint64_t>(piece, t.len - at);
            pieces.push_back({t.src + at, t.dst + at, len, t.group, vec && (((uintptr_t)(t.src + at)) & 15) == 0 ? 1u : 0u});
        }
    }
    while (g < groups) first[++g] = (uint32_t)pieces.size();
    Clip* c = new (std::nothrow) Clip();
    if (!c) { set_error("out of host memory"); return SZH_ENOMEM; }
    c->n_pieces = (uint32_t)pieces.size();
    c->groups = groups;
    for (uint32_t k = 0; k < groups; ++k) c->fold = c->fold || first[k + 1] - first[k] > 4096;
    for (uint32_t k = 0; k < groups; ++k) c->has_empty = c->has_empty || first[k] == first[k + 1];
    c->live = live;
    c->live_step = live_step;
    hipError_t he = hipGetDevice(&c->device);
    if (he == hipSuccess) he = hipMalloc((void**)&c->d_pieces, std::max<size_t>(pieces.size(), 1) * sizeof(ClipPiece));
    if (he == hipSuccess) he = hipMalloc((void**)&c->d_part, (pieces.size() + groups) * sizeof(double));
    if (he == hipSuccess) he = hipMalloc((void**)&c->d_first, first.size() * sizeof(uint32_t));
    if (he == hipSuccess && !pieces.empty()) he = hipMemcpy(c->d_pieces, pieces.data(), pieces.size() * sizeof(ClipPiece), hipMemcpyHostToDevice);
    if (he == hipSuccess) he = hipMemcpy(c->d_first, first.data(), first.size() * sizeof(uint32_t), hipMemcpyHostToDevice);
    if (he != hipSuccess) { clip_destroy(c); return hip_fail(he, "clip tables"); }
    *out = c;
    return SZH_OK;
}

void clip_destroy(Clip* c)
{
    if (!c) return;
    if (c->d_pieces) (void)hipFree(c->d_pieces);
    if (c->d_part) (void)hipFree(c->d_part);
    if (c->d_first) (void)hipFree(c->d_first);
    delete c;
}

int net_clip(Net* n, float max_norm, float* norm_dev, hipStream_t s)
{
    if (!n->clip || n->clip_of != n->d_grad || n->clip_len != n->param_count()) {  // first call, or another class was added
        hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
        if (hipStreamIsCapturing(s, &st) == hipSuccess && st == hipStreamCaptureStatusActive) {
            set_error("the first clipping of a network allocates its tables and cannot be captured");
            return SZH_EINVAL;
        }
        clip_destroy(n->clip);
        n->clip = nullptr;
        const ClipTensor t{n->d_grad, n->d_grad, n->param_count(), 0};
        if (int rc = clip_create(&t, 1, 1, n->d_grad + n->param_count() + 1, 1, &n->clip)) return rc;
        n->clip_of = n->d_grad;
        n->clip_len = n->param_count();
    }
    return clip_run(n->clip, max_norm, norm_dev, s);
}

int clip_run(Clip* c, float max_norm, float* norms_dev, hipStream_t s)
{
    ProfScope prof("clip", s);
    if (norms_dev && c->has_empty)
        hipLaunchKernelGGL(clip_empty_kernel, dim3((c->groups + 255) / 256), dim3(256), 0, s, c->d_first, c->groups, norms_dev);
    if (c->n_pieces) {
        hipLaunchKernelGGL(clip_squares_kernel, dim3(c->n_pieces), dim3(kClipThreads), 0, s, c->d_pieces, c->d_part);
        if (c->fold)
            hipLaunchKernelGGL(clip_fold_kernel, dim3(c->groups), dim3(kClipThreads), 0, s, c->d_part, c->d_first, c->d_part + c->n_pieces);
        hipLaunchKernelGGL(clip_scale_kernel, dim3(c->n_pieces), dim3(kClipThreads), 0, s, c->d_pieces, c->d_part, c->d_first,
                           (const double*)(c->fold ? c->d_part + c->n_pieces : nullptr), c->live, c->live_step, max_norm, norms_dev);
    }
    SZ_HIP(hipGetLastError());
    return SZH_OK;
}

}  // namespace sz
