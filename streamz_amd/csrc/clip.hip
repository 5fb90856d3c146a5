// The norm of gradients over many tensors and their clipping.  No counterpart in the reference, whose
// training (lib.rs:1002-1060) applies every gradient as it is.
//
//   norm_G = sqrt(sum over the tensors of group G of sum g^2) / live_G,   f = norm_G > max_norm ? max_norm / norm_G : 1
//   out = f g
//
// Squares are added in 64 bits (no overflow or underflow of an f32 gradient's squares, and sums of any length
// to f32 accuracy) in an order fixed by the layout: a workgroup per piece of a tensor, then every
// workgroup of the second launch adds its group's pieces for itself.  No atomics, no flags to reset.
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

__global__ __launch_bounds__(kClipThreads) void clip_squares_kernel(const ClipPiece* __restrict__ pieces, double* __restrict__ part)
{
    const ClipPiece p = pieces[blockIdx.x];
    double s = 0.0;
    for (uint32_t i = threadIdx.x; i < p.len; i += kClipThreads) { const double v = (double)p.src[i]; s += v * v; }
    s = block_sum(s);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__global__ __launch_bounds__(kClipThreads) void clip_scale_kernel(const ClipPiece* __restrict__ pieces, const double* __restrict__ part,
                                                                  const uint32_t* __restrict__ first, const float* __restrict__ live,
                                                                  uint32_t live_step, float max_norm, float* __restrict__ norms)
{
    const ClipPiece p = pieces[blockIdx.x];
    const uint32_t b = first[p.group], e = first[p.group + 1];
    double s = 0.0;
    for (uint32_t i = b + threadIdx.x; i < e; i += kClipThreads) s += part[i];
    s = sqrt(block_sum(s));
    if (live) {
        const double n = (double)live[(uint64_t)p.group * live_step];
        s = n > 0.0 ? s / n : 0.0;  // nothing counted: the update is nothing
    }
    if (norms && blockIdx.x == b && threadIdx.x == 0) norms[p.group] = (float)s;
    const bool clip = s > (double)max_norm;
    if (!clip && p.src == p.dst) return;
    // the factor stays in 64 bits (beside gradients near the type's end it lies below f32's normal range): one rounding a value
    const double f = clip ? (double)max_norm / s : 1.0;
    for (uint32_t i = threadIdx.x; i < p.len; i += kClipThreads) p.dst[i] = clip ? (float)((double)p.src[i] * f) : p.src[i];
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
    const uint64_t piece = std::min<uint64_t>(std::max<uint64_t>((total / 2048 + 1023) / 1024 * 1024, 4096), 1u << 24);
    std::vector<uint32_t> order(n);
    for (uint32_t t = 0; t < n; ++t) order[t] = t;
    std::stable_sort(order.begin(), order.end(), [&](uint32_t a, uint32_t b) { return tensors[a].group < tensors[b].group; });
    std::vector<ClipPiece> pieces;
    std::vector<uint32_t> first(groups + 1, 0);
    uint32_t g = 0;
    for (uint32_t k = 0; k < n; ++k) {
        const ClipTensor& t = tensors[order[k]];
        while (g < t.group) first[++g] = (uint32_t)pieces.size();
        for (uint64_t at = 0; at < t.len; at += piece)
            pieces.push_back({t.src + at, t.dst + at, (uint32_t)std::min<uint64_t>(piece, t.len - at), t.group});
    }
    while (g < groups) first[++g] = (uint32_t)pieces.size();
    if (pieces.size() > 0x7fffffffu) { set_error("too many tensors"); return SZH_EINVAL; }
    Clip* c = new (std::nothrow) Clip();
    if (!c) { set_error("out of host memory"); return SZH_ENOMEM; }
    c->n_pieces = (uint32_t)pieces.size();
    c->groups = groups;
    for (uint32_t k = 0; k < groups; ++k) c->has_empty = c->has_empty || first[k] == first[k + 1];
    c->live = live;
    c->live_step = live_step;
    hipError_t he = hipGetDevice(&c->device);
    if (he == hipSuccess) he = hipMalloc((void**)&c->d_pieces, std::max<size_t>(pieces.size(), 1) * sizeof(ClipPiece));
    if (he == hipSuccess) he = hipMalloc((void**)&c->d_part, std::max<size_t>(pieces.size(), 1) * sizeof(double));
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
        hipLaunchKernelGGL(clip_scale_kernel, dim3(c->n_pieces), dim3(kClipThreads), 0, s, c->d_pieces, c->d_part, c->d_first, c->live,
                           c->live_step, max_norm, norms_dev);
    }
    SZ_HIP(hipGetLastError());
    return SZH_OK;
}

}  // namespace sz
