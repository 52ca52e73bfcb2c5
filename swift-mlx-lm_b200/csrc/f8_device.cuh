// Device code shared by the products in 8-bit floating point.
#pragma once

#include "f8.h"
#include "tc_device.cuh"

namespace swlm {
namespace f8 {

constexpr int kSms = 148;
constexpr int kCodesBytes = kF8Block * kF8Block;   // 128 rows of a block

// kind::f8f6f4: D fp32, A = B = e4m3, both K-major; 32 columns of K each
__host__ __device__ constexpr unsigned idesc(int m, int n) { return (1u << 4) | ((unsigned)(n >> 3) << 17) | ((unsigned)(m >> 4) << 24); }
// (descriptors by their low words)
template <int CG>
__device__ __forceinline__ void umma(unsigned d_tmem, unsigned a_lo, unsigned b_lo, unsigned desc, unsigned accumulate) {
    if (CG == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
            "setp.ne.b32 p, %5, 0;\n\t"
            "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %4, p;\n\t}"
            ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(kUmmaDescHi), "r"(desc), "r"(accumulate) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
            "setp.ne.b32 p, %5, 0;\n\t"
            "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
            "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a, b, %4, p;\n\t}"
            ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(kUmmaDescHi), "r"(desc), "r"(accumulate) : "memory");
}
// arrival at a barrier (of both CTAs of the pair) when the MMAs issued so far are done
template <int CG>
__device__ __forceinline__ void commit(unsigned long long* bar) {
    if (CG == 1) umma_commit(bar);
    else asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((unsigned short)3) : "memory");
}
__device__ __forceinline__ unsigned cluster_place(unsigned addr, int rank) {   // the same shared-memory place in another CTA of the cluster
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// A shared-memory address that the compiler keeps in a register: in kernels of clusters it otherwise puts it together again wherever it is used, from a special
// register that takes tens of cycles to read.
__device__ __forceinline__ unsigned held_address(const void* p) {
    unsigned r;
    asm volatile("mov.u32 %0, %1;" : "=r"(r) : "r"(smem_u32(p)));
    return r;
}
__device__ __forceinline__ void arrive(unsigned bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void arrive_cluster(unsigned bar) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }

// 16 columns of a warp's 32 lanes of tensor memory; they are there behind landed(). Both are volatile, as is the use in add_scaled: they stay in their order.
__device__ __forceinline__ void tmem_load(unsigned (&v)[16], unsigned at) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(at) : "memory");
}
__device__ __forceinline__ void landed() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Two fp32 numbers as one register pair, and acc += (a, b) * s.
__device__ __forceinline__ unsigned long long pair_of(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 of_pair(unsigned long long v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ void add_scaled(unsigned long long& acc, unsigned a, unsigned b, unsigned long long s) {
    asm volatile("{\n\t.reg .b64 x;\n\tmov.b64 x, {%1, %2};\n\tfma.rn.f32x2 %0, x, %3, %0;\n\t}" : "+l"(acc) : "r"(a), "r"(b), "l"(s));
}
__device__ __forceinline__ unsigned pack2(float a, float b, bool f16) {
    if (f16) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const unsigned*>(&h); }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&h);
}
// The gated activations (swlm_op_f8_product_dev); a NaN stays one; tanh-GELU as g / (1 + e^-2u). An exponential and a reciprocal of the special function unit, within
// three and two 2^-24 of their values, and |z| 2^-24 for each rounding of the exponential's argument (GELU's has the most, seven); no branch between values, so that they overlap.
__device__ __forceinline__ float gated(float g, float u, int act, float alpha, float limit) {
    float z = g;
    if (act == SWLM_F8_GELU) z = 1.5957691216f * (g + 0.044715f * g * g * g);
    if (act == SWLM_F8_CLAMPED) {
        g = g > limit ? limit : g;
        u = (u > limit ? limit : u < -limit ? -limit : u) + 1.0f;
        z = alpha * g;
    }
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-1.4426950408889634f * z));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return g * r * u;
}

// Work as tiles of `rows` rows x a tile of columns, those of one expert after those of the other (experts 0: one has all rows). CTAs take them in turn.
constexpr int kSweep = 8;
struct TileShape { const int* offsets; int rows, experts, tile_rows, col_tiles; };
struct Tile { int expert, row0, end, col; };   // rows row0 .. end - 1 (of which a tile has tile_rows at most), tile of columns

// An expert's rows, cut to those there are.
__device__ __forceinline__ int2 expert_rows(const TileShape& p, int e) {
    const int from = min(max(p.offsets[e], 0), p.rows);
    return make_int2(from, min(max(p.offsets[e + 1], from), p.rows));
}
// Fills first_tile [experts] with the tiles of the experts before each, by all threads of a CTA, and returns the number of tiles; `warps`: a number per warp. A
// barrier has to follow. Sums stop at what offsets that ascend come to at most, which is within kF8MaxTiles: of others, where experts share rows, later tiles are left out.
template <int THREADS>
__device__ __forceinline__ int count_tiles(const TileShape& p, int* first_tile, int* warps) {
    if (!p.experts) return (p.rows + p.tile_rows - 1) / p.tile_rows * p.col_tiles;
    constexpr int PER = (kExpertMax + THREADS - 1) / THREADS;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned most = (unsigned)(p.rows / p.tile_rows + p.experts) * p.col_tiles;
    auto add = [&](int a, int b) { return (int)min((unsigned)a + (unsigned)b, most); };
    int c[PER], sum = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int e = tid * PER + j;
        c[j] = 0;
        if (e < p.experts) {
            const int2 r = expert_rows(p, e);
            c[j] = (r.y - r.x + p.tile_rows - 1) / p.tile_rows * p.col_tiles;
        }
        sum = add(sum, c[j]);
    }
    int scan = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan = add(scan, v);
    }
    if (lane == 31) warps[warp] = scan;
    __syncthreads();
    int tiles = 0, before = __shfl_up_sync(0xffffffffu, scan, 1);
    if (lane == 0) before = 0;
    for (int w = 0; w < THREADS / 32; ++w) { before = add(before, w < warp ? warps[w] : 0); tiles = add(tiles, warps[w]); }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int e = tid * PER + j;
        if (e < p.experts) first_tile[e] = before;
        before = add(before, c[j]);
    }
    return tiles;
}
__device__ __forceinline__ Tile tile_at(const TileShape& p, const int* first_tile, int t) {
    Tile w{0, 0, p.rows, 0};
    if (p.experts) {
        int lo = 0, hi = p.experts - 1;   // the last expert whose tiles start at or before t
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (first_tile[mid] <= t) lo = mid; else hi = mid - 1;
        }
        const int2 r = expert_rows(p, lo);
        w.expert = lo; w.row0 = r.x; w.end = r.y;
        t -= first_tile[lo];
    }
    // Up to kSweep tiles of the shorter side, then those of the next place on the longer one: what CTAs at work together read is about as much of x as of the
    // matrix, and stays in L2 for longer (8192 rows x 4096 x 14336, 176 MB: 445 MB are read from memory, with all 16 tiles of columns in a sweep 526).
    const int row_tiles = (w.end - w.row0 + p.tile_rows - 1) / p.tile_rows, shorter = min(row_tiles, p.col_tiles), longer = max(row_tiles, p.col_tiles);
    const int sweep = t / (kSweep * longer), width = min(kSweep, shorter - sweep * kSweep);
    t -= sweep * kSweep * longer;
    const int a = sweep * kSweep + t % width, b = t / width;
    const bool rows_first = row_tiles <= p.col_tiles;
    w.col = rows_first ? b : a;
    const int r = rows_first ? a : b;
    w.row0 += r * p.tile_rows;
    return w;
}

// Rows of bytes as a 2-D tensor, k columns valid (beyond: zeros); box = 128 columns x box_rows, 128-byte swizzle
inline int code_map(const void* p, int64_t stride, int64_t rows, int k, int box_rows, CUtensorMap* map) {
    TensorMapEncodeFn fn = tensor_map_encode_fn();
    if (!fn) { set_error("f8: cuTensorMapEncodeTiled is not available"); return SWLM_ERR_CUDA; }
    const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)stride};
    const cuuint32_t box[2] = {(cuuint32_t)kF8Block, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) { set_error("f8: cuTensorMapEncodeTiled failed (%d)", (int)r); return SWLM_ERR_CUDA; }
    return SWLM_OK;
}

}  // namespace f8

F8FewForm f8_few_form(int rows, int n, int k, int experts, bool gated);
int f8_few_init();
int launch_f8_few(const swlm_f8_product& a, const F8FewForm& form, int* status, cudaStream_t s);
}  // namespace swlm
