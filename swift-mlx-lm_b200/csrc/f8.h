// Shared by the operators over 8-bit float weights with a scale per block of 128 x 128 and over rows sorted by expert (include/swlm.h).
#pragma once

#include <cstdint>

#include "swlm_internal.h"

namespace swlm {

constexpr int kF8Block = 128;            // columns of a row's scale, rows and columns of a matrix's
constexpr int kF8MaxRows = 1 << 30;      // row numbers stay 32-bit ones, also a tile behind the last
constexpr int kF8MaxWidth = 1 << 24;
constexpr int kExpertMax = 1024;
constexpr int kF8MaxTiles = 1 << 30;     // tiles of a product, of 16 rows x 128 columns or more: two terabytes of results have no more

// A product of few rows: rows of x per tile, CTAs of a cluster that share K, and what it takes, about (us).
struct F8FewForm { int nt, ranges; double cost; };
// How a product runs: so many columns by pairs of SMs (many rows), the others, if any, in the form of few.
struct F8ProductForm { int wide = 0; F8FewForm few{}; };
F8ProductForm f8_product_form(int rows, int n, int k, int experts, bool gated);
int f8_product_init();
int expert_rows_init();
int launch_f8_quantize(const swlm_f8_quantize& a, cudaStream_t s);
// status: a word that the device sets when a bounded wait expires
int launch_f8_product(const swlm_f8_product& a, int* status, cudaStream_t s);
int launch_expert_sort(const swlm_expert_sort& a, cudaStream_t s);
int launch_expert_sum(const swlm_expert_sum& a, cudaStream_t s);

__host__ __device__ inline int f8_blocks(int width) { return (width + kF8Block - 1) / kF8Block; }
__host__ __device__ inline int f8_size(int dtype) { return dtype == SWLM_F8_FP32 ? 4 : dtype == SWLM_F8_E4M3 ? 1 : 2; }

#ifdef __CUDACC__
// A block's scale from the bits of its largest |value|, m 2^e: the smallest power of two that is at least m 2^e / (1.75 * 2^8), so 2^(e - 8) while
// m <= 1.75, the mantissa not above 0x600000; its inverse is exact. NaN for values that are not finite.
struct F8Scale {
    float scale, inverse;
    __device__ __forceinline__ explicit F8Scale(unsigned top) {
        const int e = max((int)((top + 0x1FFFFFu) >> 23) - 8, 1);   // biased; a scale is a normal number
        const bool finite = top < 0x7F800000u;
        scale = finite ? __uint_as_float((unsigned)e << 23) : __uint_as_float(0x7FC00000u);
        inverse = finite ? __uint_as_float((unsigned)(254 - e) << 23) : scale;
    }
};
// The codes of four values that are at most 448 in size, as a word.
__device__ __forceinline__ unsigned f8_codes4(float a, float b, float c, float d) {
    unsigned word;
    asm("{\n\t.reg .b16 p, q;\n\tcvt.rn.satfinite.e4m3x2.f32 p, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 q, %4, %3;\n\tmov.b32 %0, {p, q};\n\t}"
        : "=r"(word) : "f"(a), "f"(b), "f"(c), "f"(d));
    return word;
}
#endif

}  // namespace swlm
