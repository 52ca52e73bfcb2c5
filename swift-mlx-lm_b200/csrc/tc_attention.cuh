// What the attention kernels on tcgen05 share: MMAs of 128 query rows, their instruction and matrix descriptors, tensor memory to registers and
// back, fences.
#pragma once

#include "swlm_internal.h"
#include "tc_device.cuh"

namespace swlm {

constexpr int kPaRows = 128, kPaKeys = 64;   // rows of a query tile, keys of a key tile

// (descriptors by their low words)
__device__ __forceinline__ void pa_mma_ss(unsigned d, unsigned a_lo, unsigned b_lo, unsigned idesc, unsigned acc) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}"
                 ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(kUmmaDescHi), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void pa_mma_ts(unsigned d, unsigned a, unsigned b_lo, unsigned idesc, unsigned acc) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 b, {%2, %3};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b_lo), "r"(kUmmaDescHi), "r"(idesc), "r"(acc) : "memory");
}
// D fp32, A and B both bf16 or both fp16, M = 128, N = n; `b_mn`: B's rows lie along K (its N index is the contiguous one)
__host__ __device__ constexpr unsigned pa_idesc(int n, bool b_mn, bool bf16) {
    return (1u << 4) | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (b_mn ? 1u << 16 : 0u) | ((unsigned)(n >> 3) << 17) | ((unsigned)(kPaRows >> 4) << 24);
}
// Descriptor (low word) of a tile whose contiguous index is N: blocks of 64 elements (128 bytes) `block` bytes apart, eight rows of K
// per 1024 bytes
__device__ __forceinline__ unsigned pa_desc_mn_lo(unsigned addr, unsigned block) { return umma_desc_lo(addr) | (block >> 4) << 16; }
#define PA_R8(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7])
#define PA_I8(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]), "r"(v[o + 7])
__device__ __forceinline__ void pa_ld32(unsigned addr, unsigned* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : PA_R8(v, 0), PA_R8(v, 8), PA_R8(v, 16), PA_R8(v, 24) : "r"(addr) : "memory");
}
__device__ __forceinline__ void pa_st32(unsigned addr, const unsigned* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(addr), PA_I8(v, 0), PA_I8(v, 8), PA_I8(v, 16), PA_I8(v, 24) : "memory");
}
__device__ __forceinline__ void pa_ld16(unsigned addr, unsigned* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];" : PA_R8(v, 0), PA_R8(v, 8) : "r"(addr) : "memory");
}
__device__ __forceinline__ void pa_st16(unsigned addr, const unsigned* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), PA_I8(v, 0), PA_I8(v, 8) : "memory");
}
__device__ __forceinline__ void pa_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pa_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pa_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pa_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pa_arrive(unsigned long long* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory"); }
__device__ __forceinline__ float pa_exp2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ unsigned pa_pack(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&v);
}
// (a, b) as bf16 pairs hi + lo
__device__ __forceinline__ void pa_split(float a, float b, unsigned& hi, unsigned& lo) {
    hi = pa_pack(a, b);
    lo = pa_pack(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xFFFF0000u));
}

}  // namespace swlm
