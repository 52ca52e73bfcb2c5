// Products of rows and matrices in 8-bit floating point.
#include <algorithm>

#include <cuda_fp8.h>

#include "f8.h"

namespace swlm {
namespace {

constexpr int kTileRows = 32, kTileCols = 128, kThreads = 256, kStep = 32;

__device__ __forceinline__ float code_value(unsigned char c) {
    __nv_fp8_e4m3 v;
    v.__x = c;
    return (float)v;
}

// A CTA has 128 columns of the result (a block of its scales) of 32 rows at a time, of one expert; a thread 4 rows x 4 columns.
template <bool GATED>
__global__ void __launch_bounds__(kThreads) f8_product_kernel(const swlm_f8_product a) {
    __shared__ float xs[kTileRows][kStep + 1], ws[GATED ? 2 : 1][kTileCols][kStep + 1];
    pdl_wait();
    const int expert = blockIdx.z, tid = threadIdx.x, tx = tid & 31, ty = tid >> 5, col0 = blockIdx.x * kTileCols, kb = (a.k + 127) / 128, nb = (a.n + 127) / 128;
    int from = 0, to = a.rows;
    if (a.experts) { from = min(max(a.offsets[expert], 0), a.rows); to = min(max(a.offsets[expert + 1], from), a.rows); }
    for (int row0 = from + (int)blockIdx.y * kTileRows; row0 < to; row0 += gridDim.y * kTileRows) {
        float acc[GATED ? 2 : 1][4][4] = {};
        for (int b = 0; b < kb; ++b) {
            float part[GATED ? 2 : 1][4][4] = {};
            for (int k0 = b * 128; k0 < min(b * 128 + 128, a.k); k0 += kStep) {
                for (int i = tid; i < kTileRows * kStep; i += kThreads) {
                    const int r = row0 + i / kStep, k = k0 + i % kStep;
                    xs[i / kStep][i % kStep] = r < to && k < a.k ? code_value(static_cast<const unsigned char*>(a.x.codes)[(long long)r * a.x.stride + k]) : 0.f;
                }
                for (int g = 0; g < (GATED ? 2 : 1); ++g) {
                    const swlm_f8_weight& w = g ? a.up : a.w;
                    for (int i = tid; i < kTileCols * kStep; i += kThreads) {
                        const int c = col0 + i / kStep, k = k0 + i % kStep;
                        ws[g][i / kStep][i % kStep] = c < a.n && k < a.k ? code_value(static_cast<const unsigned char*>(w.codes)[((long long)expert * a.n + c) * w.stride + k]) : 0.f;
                    }
                }
                __syncthreads();
                for (int k = 0; k < kStep; ++k)
                    for (int g = 0; g < (GATED ? 2 : 1); ++g)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int j = 0; j < 4; ++j) part[g][i][j] = fmaf(xs[ty * 4 + i][k], ws[g][tx + 32 * j][k], part[g][i][j]);
                __syncthreads();
            }
            for (int g = 0; g < (GATED ? 2 : 1); ++g) {
                const float sw = (g ? a.up : a.w).scale[((long long)expert * nb + blockIdx.x) * kb + b];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = row0 + ty * 4 + i;
                    const float s = r < to ? a.x.scale[(long long)b * a.x.scale_stride + r] * sw : 0.f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[g][i][j] = fmaf(part[g][i][j], s, acc[g][i][j]);
                }
            }
        }
        for (int i = 0; i < 4; ++i) {
            const int r = row0 + ty * 4 + i;
            float v[4];
            unsigned top = 0;
            for (int j = 0; j < 4; ++j) {
                v[j] = GATED ? f8_gated(acc[0][i][j], acc[GATED ? 1 : 0][i][j], a.act, a.alpha, a.limit) : acc[0][i][j];
                if (col0 + tx + 32 * j < a.n) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
            }
            const F8Scale s(__reduce_max_sync(0xffffffffu, top));
            if (r >= to) continue;
            for (int j = 0; j < 4; ++j) {
                const int c = col0 + tx + 32 * j;
                if (c >= a.n) continue;
                const long long at = (long long)r * a.y_stride + c;
                if (a.dtype == SWLM_F8_FP32) static_cast<float*>(a.y)[at] = v[j];
                else if (a.dtype == SWLM_F8_FP16) static_cast<__half*>(a.y)[at] = __float2half_rn(v[j]);
                else if (a.dtype == SWLM_F8_BF16) static_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16_rn(v[j]);
                else static_cast<unsigned char*>(a.y)[at] = (unsigned char)f8_codes4(v[j] * s.inverse, 0.f, 0.f, 0.f);
            }
            if (a.dtype == SWLM_F8_E4M3 && tx == 0) a.y_scale[blockIdx.x * a.y_scale_stride + r] = s.scale;
        }
    }
}

}  // namespace

int f8_product_init() { return SWLM_OK; }

int launch_f8_product(const swlm_f8_product& a, int* status, cudaStream_t s) {
    (void)status;
    if (a.rows == 0) return SWLM_OK;
    const dim3 grid(f8_blocks(a.n), std::min((a.rows + kTileRows - 1) / kTileRows, 64), std::max(a.experts, 1));
    const cudaError_t e = launch_k(a.act == SWLM_F8_PLAIN ? f8_product_kernel<false> : f8_product_kernel<true>, grid, dim3(kThreads), 0, s, a);
    return e == cudaSuccess ? SWLM_OK : cuda_fail(e, "product launch");
}

}  // namespace swlm
