// Launches of the GEMM kernels (gemm_kernel.h, gemm_bf16x3.h) by the shape of the product, and the small kernels that
// lay weights out for them.  Included by the translation units that run products (net.hip, adapt.hip).
#pragma once
#include <algorithm>

#include "gemm_bf16x3.h"
#include "gemm_kernel.h"
#include "internal.h"
#include "prof.h"
#include "streamz_hip.h"

namespace sz {

namespace {

using namespace gemm;

inline int vec_ok(const void* p, int ld) { return (((uintptr_t)p & 15) == 0 && (ld & 3) == 0) ? 1 : 0; }

constexpr int kGemmKT = 32, kGemmDB = 0;  // K tile and LDS double-buffering of the shipped kernels
constexpr int BK = kGemmKT;

enum GemmTag { T_FWD1 = 0, T_FWD2, T_FWD3, T_DELTA2, T_DELTA1, T_DW3, T_DW2, T_DW1, T_ADAPT1, T_ADAPT2, T_ADAPT3, T_ADAPT_D2 };
const char* const kGemmTagName[] = {"fwd1", "fwd2", "fwd3", "delta2", "delta1", "dw3", "dw2", "dw1",
                                    "adapt_h1", "adapt_h2", "adapt_out", "adapt_d2"};

template <int AM, int BMd, int EPI, int TAG>
int launch_gemm(GemmArgs g, int splits, hipStream_t s)
{
    if (g.M <= 0 || g.N <= 0) return SZH_OK;
    g.a_vec = vec_ok(g.A, g.lda);
    g.b_vec = vec_ok(g.B, g.ldb);
    ProfScope prof(kGemmTagName[TAG], s);
    // 64-row tiles when 128-row tiles would leave compute units without a workgroup
    const long tiles128 = (long)((g.N + BN - 1) / BN) * ((g.M + BM - 1) / BM) * splits;
    if (g.M <= 64 && BMd == B_KROWS && g.N % (2 * BN) == 0 && (long)(g.N / (2 * BN)) * splits >= 256) {
        // one 64-row tile of rows and a k-major B: 256-column tiles (dW1)
        constexpr int BNW = BMd == B_KROWS ? 2 * BN : BN;
        dim3 grid(g.N / (2 * BN), 1, splits);
        hipLaunchKernelGGL((gemm_kernel<AM, BMd, EPI, TAG, 64, kGemmKT, kGemmDB, BNW>), grid, dim3(kGemmThreads), 0, s, g);
    } else if (g.M <= 64 || (splits == 1 && tiles128 < 256)) {
        dim3 grid((g.N + BN - 1) / BN, (g.M + 63) / 64, splits);
        hipLaunchKernelGGL((gemm_kernel<AM, BMd, EPI, TAG, 64, kGemmKT, kGemmDB>), grid, dim3(kGemmThreads), 0, s, g);
    } else {
        dim3 grid((g.N + BN - 1) / BN, (g.M + BM - 1) / BM, splits);
        hipLaunchKernelGGL((gemm_kernel<AM, BMd, EPI, TAG, 128, kGemmKT, kGemmDB>), grid, dim3(kGemmThreads), 0, s, g);
    }
    SZ_HIP(hipGetLastError());
    return SZH_OK;
}

// the same with the row tile chosen by the caller
template <int AM, int BMd, int EPI, int TAG, int TM>
int launch_gemm_rows(GemmArgs g, hipStream_t s)
{
    if (g.M <= 0 || g.N <= 0) return SZH_OK;
    g.a_vec = vec_ok(g.A, g.lda);
    g.b_vec = vec_ok(g.B, g.ldb);
    ProfScope prof(kGemmTagName[TAG], s);
    hipLaunchKernelGGL((gemm_kernel<AM, BMd, EPI, TAG, TM, kGemmKT, kGemmDB>), dim3((g.N + BN - 1) / BN, (g.M + TM - 1) / TM),
                       dim3(kGemmThreads), 0, s, g);
    SZ_HIP(hipGetLastError());
    return SZH_OK;
}

int compute_units()
{
    static int cus[64] = {};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
    if (cus[dev] == 0) {
        int v = 0;
        cus[dev] = hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && v >= 8 ? v : 256;
    }
    return cus[dev];
}

// The three large products of a training chunk on the bf16 matrix cores with every f32 operand
// split exactly into three bf16 pieces (gemm_bf16x3.h).
template <int ASRC, int BSRC, int EPI, int TAG>
int launch_gemm_x3(GemmArgs g, int splits, hipStream_t s)
{
    if (g.M <= 0 || g.N <= 0) return SZH_OK;
    if (int rc = allow_dynamic_lds((const void*)gemm_x3w_kernel<ASRC, BSRC, EPI, TAG>, XW_LDS_BYTES)) return rc;
    ProfScope prof(kGemmTagName[TAG], s);
    g.tiles_x = (g.N + XW_TN - 1) / XW_TN; g.tiles_y = (g.M + XW_TM - 1) / XW_TM; g.tiles_z = splits;
    // one workgroup per compute unit (its LDS use allows no second one), a multiple of the 8 XCDs
    const int tiles = g.tiles_x * g.tiles_y * g.tiles_z;
    const int blocks = std::min((tiles + 7) / 8 * 8, compute_units() / 8 * 8);
    hipLaunchKernelGGL((gemm_x3w_kernel<ASRC, BSRC, EPI, TAG>), dim3(blocks), dim3(XW_THREADS), XW_LDS_BYTES, s, g);
    SZ_HIP(hipGetLastError());
    return SZH_OK;
}

// The f32 products with a row-major first operand on 256 x 256 tiles walked by one workgroup per CU
// (gemm_f32w_kernel): B as [N][K].
template <int EPI, int TAG, int SRC = X3_ROWS_F32>
int launch_gemm_f32w(GemmArgs g, hipStream_t s, int splits = 1)
{
    if (g.M <= 0 || g.N <= 0) return SZH_OK;
    constexpr size_t lds = FW_LDS_BYTES + (EPI >= EPI_ADAPT_TANH ? AL_BYTES : 0);
    if (int rc = allow_dynamic_lds((const void*)gemm_f32w_kernel<SRC, SRC, EPI, TAG>, lds)) return rc;
    ProfScope prof(kGemmTagName[TAG], s);
    g.tiles_x = (g.N + XW_TN - 1) / XW_TN; g.tiles_y = (g.M + XW_TM - 1) / XW_TM; g.tiles_z = splits;
    const int tiles = g.tiles_x * g.tiles_y * g.tiles_z;
    const int blocks = std::min((tiles + 7) / 8 * 8, compute_units() / 8 * 8);
    hipLaunchKernelGGL((gemm_f32w_kernel<SRC, SRC, EPI, TAG>), dim3(blocks), dim3(XW_THREADS), lds, s, g);
    SZ_HIP(hipGetLastError());
    return SZH_OK;
}

// whether the hidden-layer forward product and its delta take that kernel: whole 256-wide tiles in both
// hidden dimensions and at least two rounds of tiles per CU (below that the 128-wide tiles, of which
// three workgroups fit a CU, are faster)
inline bool use_wide_f32(const Net* n, uint64_t rows)
{
    return n->h1 % 256 == 0 && n->h2 % 256 == 0 && (rows / 256) * (std::min(n->h1, n->h2) / 256) >= 512;
}

// whether a call of `rows` rows takes the split-bf16 kernels: opted in, whole 256-wide tiles in both
// hidden dimensions, and enough rows that 256-row tiles are not mostly padding
inline bool use_x3(const Net* n, uint64_t rows)
{
    return n->gemm_mode == SZH_GEMM_BF16X3 && n->h1 % 256 == 0 && n->h2 % 256 == 0 && rows >= 1024;
}

// ... and the output layer's products too (they run as GEMMs only beyond 64 classes)
inline bool use_x3_out(const Net* n, uint64_t rows) { return use_x3(n, rows) && n->out % 256 == 0; }

// out[c][r] = in[r][c]; 32x32 tiles through LDS
__global__ __launch_bounds__(256) void transpose_kernel(const float* __restrict__ in, int rows, int cols,
                                                        float* __restrict__ out)
{
    __shared__ float t[32][33];
    const int c0 = blockIdx.x * 32, r0 = blockIdx.y * 32;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    for (int i = ty; i < 32; i += 8)
        if (r0 + i < rows && c0 + tx < cols) t[i][tx] = in[(size_t)(r0 + i) * cols + c0 + tx];
    __syncthreads();
    for (int i = ty; i < 32; i += 8)
        if (c0 + i < cols && r0 + tx < rows) out[(size_t)(c0 + i) * rows + r0 + tx] = t[tx][i];
}

// out[c][0 .. ld) = in[0 .. rows)[c], zeros behind: the first layer's weights as the [N][K] operand of
// a product over the prepared rows' ld columns (whose columns from `rows` on hold 1, 0, 0, ...)
__global__ __launch_bounds__(256) void pad_transpose_kernel(const float* __restrict__ in, int rows, int cols, int ld,
                                                            float* __restrict__ out)
{
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= cols * ld) return;
    const int c = i / ld, k = i % ld;
    out[i] = k < rows ? in[(size_t)k * cols + c] : 0.0f;
}

}  // namespace

}  // namespace sz
