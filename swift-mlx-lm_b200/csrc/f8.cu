// Rows in 8-bit floating point (quantization), and what the calls over such rows check. A code is value / scale rounded once: scales are powers of two, so the
// quotient is exact, and results do not depend on the launch.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "f8.h"
#include "swlm_runtime.h"

namespace swlm {
namespace {

// ---- quantization ----------------------------------------------------------------------------------------------------------
// A lane has eight consecutive values, half a warp a block of 128 columns, and a warp kQuantBlocks of them of one row, all loaded before any is rounded.
// Neighbouring warps have neighbouring rows, whose scales lie side by side.
constexpr int kQuantThreads = 256, kQuantWarps = kQuantThreads / 32, kQuantSteps = 4, kQuantBlocks = 2 * kQuantSteps;

template <int DTYPE> struct Eight;   // eight values as they are held
template <> struct Eight<SWLM_F8_FP32> {
    float4 a, b;
    __device__ __forceinline__ void load(const void* p) { a = static_cast<const float4*>(p)[0]; b = static_cast<const float4*>(p)[1]; }
    __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ __forceinline__ void widen(float (&x)[8]) const { x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w; }
};
template <int DTYPE> struct Eight {
    uint4 v;
    __device__ __forceinline__ void load(const void* p) { v = *static_cast<const uint4*>(p); }
    __device__ __forceinline__ void zero() { v = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void widen(float (&x)[8]) const {
        const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = DTYPE == SWLM_F8_FP16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[i])) : make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
            x[2 * i] = f.x; x[2 * i + 1] = f.y;
        }
    }
};

template <int DTYPE>
__global__ void __launch_bounds__(kQuantThreads) f8_quantize_kernel(const swlm_f8_quantize a) {
    constexpr int SIZE = DTYPE == SWLM_F8_FP32 ? 4 : 2;
    pdl_wait();
    const int lane = threadIdx.x & 31, row = blockIdx.x * kQuantWarps + (threadIdx.x >> 5);
    if (row >= a.rows) return;
    const int from = a.source ? a.source[row] : row;
    if (from < 0 || from >= a.x_rows) return;
    const unsigned char* src = static_cast<const unsigned char*>(a.x) + (long long)from * a.x_stride * SIZE;
    unsigned char* dst = static_cast<unsigned char*>(a.out.codes) + (long long)row * a.out.stride;
    const int block0 = blockIdx.y * kQuantBlocks, col0 = block0 * kF8Block + lane * 8;
    Eight<DTYPE> held[kQuantSteps];
#pragma unroll
    for (int i = 0; i < kQuantSteps; ++i) {
        const int col = col0 + i * 256;
        if (col + 8 <= a.width) held[i].load(src + (long long)col * SIZE);
        else held[i].zero();
    }
#pragma unroll
    for (int i = 0; i < kQuantSteps; ++i) {
        const int col = col0 + i * 256, block = block0 + 2 * i + (lane >> 4), rest = a.width - col;
        float x[8];
        held[i].widen(x);
        if (rest > 0 && rest < 8) {   // a row's last values, whose number is no multiple of eight
            const typename std::conditional<DTYPE == SWLM_F8_FP32, float, typename std::conditional<DTYPE == SWLM_F8_FP16, __half, __nv_bfloat16>::type>::type* p =
                reinterpret_cast<decltype(p)>(src) + col;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = e < rest ? (float)p[e] : 0.f;
        }
        unsigned top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7FFFFFFFu);   // (larger numbers have larger bits, NaN the largest)
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const F8Scale s(top);
        const uint2 codes = make_uint2(f8_codes4(x[0] * s.inverse, x[1] * s.inverse, x[2] * s.inverse, x[3] * s.inverse),
                                       f8_codes4(x[4] * s.inverse, x[5] * s.inverse, x[6] * s.inverse, x[7] * s.inverse));
        if (rest >= 8) {
            *reinterpret_cast<uint2*>(dst + col) = codes;
        } else if (rest > 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < rest) dst[col + e] = (unsigned char)((e < 4 ? codes.x : codes.y) >> (8 * (e & 3)));
        }
        if ((lane & 15) == 0 && block * kF8Block < a.width) a.out.scale[(long long)block * a.out.scale_stride + row] = s.scale;
    }
}

}  // namespace

int launch_f8_quantize(const swlm_f8_quantize& a, cudaStream_t s) {
    const dim3 grid((a.rows + kQuantWarps - 1) / kQuantWarps, (f8_blocks(a.width) + kQuantBlocks - 1) / kQuantBlocks);
    void (*kernel)(swlm_f8_quantize) = a.dtype == SWLM_F8_FP32 ? f8_quantize_kernel<SWLM_F8_FP32> : a.dtype == SWLM_F8_FP16 ? f8_quantize_kernel<SWLM_F8_FP16> : f8_quantize_kernel<SWLM_F8_BF16>;
    const cudaError_t e = launch_k(kernel, grid, dim3(kQuantThreads), 0, s, a);
    return e == cudaSuccess ? SWLM_OK : cuda_fail(e, "quantize launch");
}

}  // namespace swlm

// ---- the calls ----------------------------------------------------------------------------------------------------------------

using namespace swlm;

namespace {

int refuse(const char* why) {
    set_error("f8: %s", why);
    return SWLM_ERR_INVALID;
}
bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
constexpr int64_t kMaxStride = (int64_t)1 << 36;   // so that offsets in bytes stay within 64 bits
// rows of `width` entries of `size` bytes
bool rows_ok(const void* p, int64_t stride, int64_t width, int size) { return p && aligned(p, 16) && stride >= width && stride <= kMaxStride && stride * size % 16 == 0; }
int codes_ok(const swlm_f8_rows& r, int rows, int width) {
    if (!rows_ok(r.codes, r.stride, width, 1)) return refuse("rows of codes must be 16-byte aligned, their stride a multiple of 16 and at least the width");
    if (!r.scale || !aligned(r.scale, 4) || r.scale_stride < rows || r.scale_stride > kMaxStride) return refuse("scales must be 4-byte aligned, their stride at least the rows");
    return SWLM_OK;
}
int matrix_ok(const swlm_f8_weight& w, int k) {
    if (!rows_ok(w.codes, w.stride, k, 1)) return refuse("rows of a matrix must be 16-byte aligned, their stride a multiple of 16 and at least k");
    if (!w.scale || !aligned(w.scale, 4)) return refuse("a matrix's scales must be 4-byte aligned");
    return SWLM_OK;
}
// What a product may have of rows, columns and experts. An expert has its own rows and a last tile of its own.
const char* size_refused(int rows, int n, int k, int experts) {
    if (rows < 0 || rows > kF8MaxRows || n < 1 || n > kF8MaxWidth || k < 1 || k > kF8MaxWidth) return "rows, n or k out of range";
    if (experts < 0 || experts > kExpertMax) return "experts out of range";
    if ((int64_t)std::max(experts, 1) * n > kF8MaxRows) return "too many rows of all experts' matrices";
    if (((int64_t)rows / 16 + std::max(experts, 1)) * f8_blocks(n) > kF8MaxTiles) return "too many rows, experts and columns together";
    return nullptr;
}
bool plain_type(int dtype) { return dtype == SWLM_F8_BF16 || dtype == SWLM_F8_FP16 || dtype == SWLM_F8_FP32; }

// (`code`: what the kernels left in the context's word)
int expired(int code) {
    if (!code) return SWLM_OK;
    set_error("f8: a bounded device-side wait of an earlier product expired (code %d): results since then are not valid", code);
    return SWLM_ERR_TIMEOUT;
}

cudaStream_t stream_of(swlm_ctx* ctx, void* s) { return s ? static_cast<cudaStream_t>(s) : ctx->stream; }

}  // namespace

extern "C" {

int swlm_op_f8_quantize_dev(swlm_ctx* ctx, const swlm_f8_quantize* how, void* cuda_stream) {
    if (!ctx || !how) return refuse("null argument");
    const swlm_f8_quantize& a = *how;
    if (!plain_type(a.dtype)) return refuse("unknown dtype");
    if (a.rows < 0 || a.rows > kF8MaxRows || a.x_rows < 0 || a.x_rows > kF8MaxRows || a.width < 1 || a.width > kF8MaxWidth) return refuse("rows or width out of range");
    if (!a.source && a.x_rows < a.rows) return refuse("x has too few rows");
    if (!aligned(a.source, 4)) return refuse("source must be 4-byte aligned");
    if (a.rows == 0 || a.x_rows == 0) return SWLM_OK;   // (no row of the result changes)
    if (!rows_ok(a.x, a.x_stride, a.width, f8_size(a.dtype))) return refuse("rows of x must be 16-byte aligned, their stride at least the width");
    const int rc = codes_ok(a.out, a.rows, a.width);
    if (rc) return rc;
    SWLM_CUDA(cudaSetDevice(ctx->device));
    return launch_f8_quantize(a, stream_of(ctx, cuda_stream));
}

int swlm_op_f8_product_dev(swlm_ctx* ctx, const swlm_f8_product* how, void* cuda_stream) {
    if (!ctx || !how) return refuse("null argument");
    const swlm_f8_product& a = *how;
    if (!plain_type(a.dtype) && a.dtype != SWLM_F8_E4M3) return refuse("unknown dtype");
    if (a.act < SWLM_F8_PLAIN || a.act > SWLM_F8_CLAMPED) return refuse("unknown activation");
    if (const char* why = size_refused(a.rows, a.n, a.k, a.experts)) return refuse(why);
    if (a.act == SWLM_F8_CLAMPED && (!std::isfinite(a.alpha) || !(a.limit >= 0.f))) return refuse("alpha must be finite, the limit not negative");
    if (a.rows == 0) return SWLM_OK;
    if (a.experts && (!a.offsets || !aligned(a.offsets, 4))) return refuse("experts need offsets, 4-byte aligned");
    int rc = codes_ok(a.x, a.rows, a.k);
    if (rc || (rc = matrix_ok(a.w, a.k)) || (a.act != SWLM_F8_PLAIN && (rc = matrix_ok(a.up, a.k)))) return rc;
    if (!rows_ok(a.y, a.y_stride, a.n, f8_size(a.dtype))) return refuse("rows of y must be 16-byte aligned, their stride at least n");
    if (a.dtype == SWLM_F8_E4M3 && (!a.y_scale || !aligned(a.y_scale, 4) || a.y_scale_stride < a.rows || a.y_scale_stride > kMaxStride)) return refuse("codes need scales, 4-byte aligned, their stride at least the rows");
    SWLM_CUDA(cudaSetDevice(ctx->device));
    if ((rc = expired(__atomic_load_n(ctx->f8_status, __ATOMIC_RELAXED)))) return rc;
    return launch_f8_product(a, ctx->f8_status, stream_of(ctx, cuda_stream));
}

int swlm_op_f8_product_form(int rows, int n, int k, int experts, int gated, int* form) {
    if (const char* why = size_refused(rows, n, k, experts)) return refuse(why);
    if (rows < 1 || !form) return refuse("bad argument");
    const F8ProductForm f = f8_product_form(rows, n, k, experts, gated != 0);
    form[0] = f.wide; form[1] = f.wide == n ? 0 : f.few.nt; form[2] = f.wide == n ? 0 : f.few.ranges;
    return SWLM_OK;
}

int swlm_op_f8_status(swlm_ctx* ctx) {
    if (!ctx) return refuse("null argument");
    return expired(__atomic_exchange_n(ctx->f8_status, 0, __ATOMIC_RELAXED));
}

int swlm_write_f8_status(swlm_ctx* ctx, int code) {
    if (!ctx) return refuse("null argument");
    __atomic_store_n(ctx->f8_status, code, __ATOMIC_RELAXED);
    return SWLM_OK;
}

int swlm_op_expert_sort_dev(swlm_ctx* ctx, const swlm_expert_sort* how, void* cuda_stream) {
    if (!ctx || !how) return refuse("null argument");
    const swlm_expert_sort& a = *how;
    if (a.tokens < 0 || a.top < 1 || a.experts < 1 || a.experts > kExpertMax || (int64_t)a.tokens * a.top > kF8MaxRows) return refuse("tokens, top or experts out of range");
    if (!a.offsets || (a.tokens && (!a.choice || !a.source || !a.place))) return refuse("null argument");
    if (!aligned(a.choice, 4) || !aligned(a.offsets, 4) || !aligned(a.source, 4) || !aligned(a.place, 4)) return refuse("choices, offsets, source and place must be 4-byte aligned");
    SWLM_CUDA(cudaSetDevice(ctx->device));
    return launch_expert_sort(a, stream_of(ctx, cuda_stream));
}

int swlm_op_expert_sum_dev(swlm_ctx* ctx, const swlm_expert_sum* how, void* cuda_stream) {
    if (!ctx || !how) return refuse("null argument");
    const swlm_expert_sum& a = *how;
    if (!plain_type(a.dtype) || !plain_type(a.y_dtype)) return refuse("unknown dtype");
    if (a.tokens < 0 || a.top < 1 || (int64_t)a.tokens * a.top > kF8MaxRows || a.width < 1 || a.width > kF8MaxWidth || a.y_rows < 0 || a.y_rows > kF8MaxRows)
        return refuse("tokens, top, width or rows out of range");
    if (a.tokens == 0) return SWLM_OK;
    if (!a.place || !a.weight || !aligned(a.place, 4) || !aligned(a.weight, 4)) return refuse("places and weights must be there, 4-byte aligned");
    if ((a.y_rows && !rows_ok(a.y, a.y_stride, a.width, f8_size(a.y_dtype))) || !rows_ok(a.out, a.out_stride, a.width, f8_size(a.dtype)) ||
        (a.add && !rows_ok(a.add, a.add_stride, a.width, f8_size(a.dtype)))) return refuse("rows of y, add and out must be 16-byte aligned, their strides at least the width");
    SWLM_CUDA(cudaSetDevice(ctx->device));
    return launch_expert_sum(a, stream_of(ctx, cuda_stream));
}

}  // extern "C"
