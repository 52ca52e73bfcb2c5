// Products in 8-bit floating point of few rows (of few rows per expert): the weights' bytes are what counts.
//
// A CTA has 128 rows of w, the lanes of tensor memory, and NT rows of x, its columns; the blocks of K may be dealt to the CTAs of a cluster. As with many rows
// (f8_product.cu) a block's sums leave tensor memory before they are scaled and added; here the scales of the rows of x lie along a thread's
// registers. The parts then lie in shared memory, 128 columns of the result to a row of x: a warp adds the cluster's parts of a row up in the order of
// the blocks, which is a whole block of the result's scales.
#include <algorithm>

#include <cooperative_groups.h>

#include "f8_device.cuh"

namespace cg = cooperative_groups;

namespace swlm {
using namespace f8;
namespace {

constexpr int kPartPitch = 132;   // floats of a row's part (four more than its columns)

struct FewParams {
    const float *x_scale, *w_scale, *up_scale;
    long long x_scale_stride, y_stride, y_scale_stride;
    unsigned char* y;
    float* y_scale;
    const int* offsets;
    int* status;
    int rows, n, blocks, experts;   // blocks of K
    int ranges, turns;              // CTAs of a cluster; CTAs (or clusters) that take turns with the tiles of an expert's rows
    int dtype, act;
    float alpha, limit;
};

template <int NT, bool GATED> struct Few {
    static constexpr int TAKERS = NT >= 64 ? 8 : 4, WARPS = 4 + TAKERS, THREADS = WARPS * 32;
    static constexpr int MATS = GATED ? 2 : 1, COLS = MATS * NT;      // accumulators of a block
    static constexpr int BUFFERS = COLS <= 64 ? 4 : 2, TMEM = COLS * BUFFERS < 32 ? 32 : COLS * BUFFERS;
    static constexpr int STAGE = MATS * kCodesBytes + NT * kF8Block;
    static constexpr int PER_SM = NT <= 32 ? 2 : 1;
    static constexpr int STAGES = (PER_SM == 2 ? 109 * 1024 : 200 * 1024) / STAGE;
    static constexpr int SLOTS = 2 * BUFFERS;                          // blocks whose scales have room
    static constexpr int OWN = NT * MATS / (TAKERS / 4);               // accumulators of a thread: OWN / MATS columns of each matrix
    static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE + SLOTS * COLS * 4;
    static_assert(STAGES >= 3 && STAGES * STAGE >= MATS * NT * kPartPitch * 4 && TMEM <= 512 && SMEM <= 233472 / PER_SM - 2048, "room");
};

template <int NT, bool GATED>
__global__ void __launch_bounds__(Few<NT, GATED>::THREADS, Few<NT, GATED>::PER_SM)
f8_few_kernel(const FewParams p, const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap upmap) {
    using F = Few<NT, GATED>;
    constexpr int STAGES = F::STAGES, STAGE = F::STAGE, MATS = F::MATS, COLS = F::COLS, BUFFERS = F::BUFFERS, SLOTS = F::SLOTS;
    extern __shared__ __align__(1024) unsigned char few_raw[];
    unsigned char* const ring = few_raw + ((1024 - (smem_u32(few_raw) & 1023)) & 1023);   // swizzle atoms
    float* const scales = reinterpret_cast<float*>(ring + STAGES * STAGE);                // [SLOTS][MATS][NT]
    float* const parts = reinterpret_cast<float*>(ring);                                   // [MATS][NT][kPartPitch], behind the products
    __shared__ __align__(8) unsigned long long full[STAGES], empty[STAGES], sums_full[BUFFERS], sums_empty[BUFFERS];
    __shared__ unsigned tmem_base;
    __shared__ int failed_word;
    volatile int* const failed = &failed_word;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int range = (int)(blockIdx.x % p.ranges), col_tile = (int)(blockIdx.x / p.ranges), col_blocks = (p.n + kF8Block - 1) / kF8Block;
    pdl_wait();
    int expert = 0, from = 0, to = p.rows, turn = (int)blockIdx.y;
    if (p.experts) {
        expert = (int)blockIdx.y / p.turns;
        turn = (int)blockIdx.y - expert * p.turns;
        from = min(max(p.offsets[expert], 0), p.rows);
        to = min(max(p.offsets[expert + 1], from), p.rows);
    }
    if (from + turn * NT >= to) return;   // (the same for all CTAs of a cluster)
    const int block0 = (int)((long long)p.blocks * range / p.ranges), blocks = (int)((long long)p.blocks * (range + 1) / p.ranges) - block0;
    if (tid == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int i = 0; i < BUFFERS; ++i) { mbar_init(&sums_full[i], 1 + 1); mbar_init(&sums_empty[i], F::TAKERS); }
        failed_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)), "r"(F::TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = tmem_base;
    const cg::cluster_group cluster = cg::this_cluster();
    auto fail = [&](int code) { if (lane == 0) { atomicExch_system(p.status, code); *failed = 1; } __syncwarp(); };

    // (blocks so far: stages and buffers go on from one tile of rows to the next)
    int done = 0;
    for (int row0 = from + turn * NT; row0 < to; row0 += p.turns * NT) {
        if (*failed) {   // nothing more is worked on, but the cluster's barriers are kept
        } else if (warp == 0) {
            const bool el = elect_one();
            const unsigned full0 = held_address(&full[0]), empty0 = held_address(&empty[0]), at = held_address(ring);
            const int w_row = expert * p.n + col_tile * 128;
            int b = 0, s = done % STAGES;
            unsigned par = (unsigned)(~(done / STAGES) & 1);
            for (; b < blocks; ++b) {
                if (!mbar_wait_warp(empty0 + 8u * s, par)) break;
                if (el) {
                    const unsigned dst = at + s * STAGE, bar = full0 + 8u * s;
                    const int col = (block0 + b) * kF8Block;
                    mbar_expect(bar, (unsigned)STAGE);
                    tma_load_2d(dst, &wmap, col, w_row, bar);
                    if (GATED) tma_load_2d(dst + kCodesBytes, &upmap, col, w_row, bar);
                    tma_load_2d(dst + MATS * kCodesBytes, &xmap, col, row0, bar);
                }
                __syncwarp();
                if (++s == STAGES) { s = 0; par ^= 1u; }
            }
            if (b < blocks) {   // copies already requested still write shared memory
                fail(21);
                for (int i = max(done + b - STAGES, 0); i < done + b; ++i) mbar_wait_warp(full0 + 8u * (i % STAGES), (unsigned)((i / STAGES) & 1));
            }
        } else if (warp == 1) {
            constexpr unsigned desc = idesc(128, NT);
            const bool el = elect_one();
            const unsigned full0 = held_address(&full[0]), sums0 = held_address(&sums_empty[0]), at = umma_desc_lo(held_address(ring));
            int s = done % STAGES, buffer = done % BUFFERS;
            unsigned par = (unsigned)((done / STAGES) & 1), sums_par = (unsigned)(~(done / BUFFERS) & 1);
            for (int b = 0; b < blocks; ++b) {
                if (!mbar_wait_warp(sums0 + 8u * buffer, sums_par) || !mbar_wait_warp(full0 + 8u * s, par)) { fail(22); break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (el) {
                    const unsigned a = at + s * (STAGE / 16), x = a + MATS * (kCodesBytes / 16), sums = tmem + buffer * COLS;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        umma<1>(sums, a + 2 * j, x + 2 * j, desc, j > 0);
                        if (GATED) umma<1>(sums + NT, a + kCodesBytes / 16 + 2 * j, x + 2 * j, desc, j > 0);
                    }
                    commit<1>(&empty[s]);
                    commit<1>(&sums_full[buffer]);
                }
                __syncwarp();
                if (++s == STAGES) { s = 0; par ^= 1u; }
                if (++buffer == BUFFERS) { buffer = 0; sums_par ^= 1u; }
            }
        } else if (warp == 2) {
            // The factors of a block's sums: a scale of each row of x times the matrices'. A slot is free again by the time that it is written: the takers
            // have left block it - 2 BUFFERS before block it - BUFFERS was multiplied.
            constexpr int PER = (NT + 31) / 32, AHEAD = 2;
            const unsigned full0 = held_address(&sums_full[0]);
            const float* const w0 = p.w_scale + ((long long)expert * col_blocks + col_tile) * p.blocks + block0;
            const float* const u0 = GATED ? p.up_scale + ((long long)expert * col_blocks + col_tile) * p.blocks + block0 : w0;
            float x[AHEAD][PER], w[AHEAD][2];
            auto ask = [&](int u, int b) {
                if (b >= blocks) return;
                const float* src = p.x_scale + (block0 + b) * p.x_scale_stride + row0;
#pragma unroll
                for (int i = 0; i < PER; ++i) x[u][i] = lane + 32 * i < NT && row0 + lane + 32 * i < to ? src[lane + 32 * i] : 0.f;
                w[u][0] = w0[b];
                w[u][1] = u0[b];
            };
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) ask(u, u);
            bool ok = true;
            for (int b0 = 0; b0 < blocks && ok; b0 += AHEAD) {
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    const int b = b0 + u, it = done + b;
                    if (b >= blocks || !ok) break;
                    if (it >= BUFFERS) ok = mbar_wait_warp(full0 + 8u * (it % BUFFERS), (unsigned)((it / BUFFERS - 1) & 1));
                    if (!ok) { fail(23); break; }
                    float* const slot = scales + (it % SLOTS) * COLS;
#pragma unroll
                    for (int i = 0; i < PER; ++i)
                        if (lane + 32 * i < NT) {
                            slot[lane + 32 * i] = x[u][i] * w[u][0];
                            if (GATED) slot[NT + lane + 32 * i] = x[u][i] * w[u][1];
                        }
                    __syncwarp();
                    if (lane == 0) arrive(full0 + 8u * (it % BUFFERS));
                    ask(u, b + AHEAD);
                }
            }
        } else if (warp >= 4) {
            const int quarter = warp & 3, half = (warp - 4) >> 2;
            constexpr int EACH = F::OWN / MATS;      // columns of a thread of each matrix
            const unsigned full0 = held_address(&sums_full[0]), given0 = held_address(&sums_empty[0]), factors = held_address(scales) + 4u * (half * EACH);
            const unsigned at = tmem + ((unsigned)(quarter * 32) << 16) + half * EACH;
            int buffer = done % BUFFERS, slot = done % SLOTS;
            unsigned par = (unsigned)((done / BUFFERS) & 1);
            unsigned long long acc[F::OWN / 2];
#pragma unroll
            for (int i = 0; i < F::OWN / 2; ++i) acc[i] = 0;
            bool ok = true;
            for (int b = 0; b < blocks; ++b) {
                ok = mbar_wait_warp(full0 + 8u * buffer, par);
                if (!ok) { fail(24); break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned here = at + buffer * COLS, f = factors + slot * (COLS * 4);
#pragma unroll
                for (int c = 0; c < F::OWN / 16; ++c) {
                    const int m = c / (EACH / 16), j = (c % (EACH / 16)) * 16;   // matrix, first column
                    unsigned v[16];
                    tmem_load(v, here + m * NT + j);
                    unsigned long long s[8];
#pragma unroll
                    for (int i = 0; i < 8; i += 2) asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(s[i]), "=l"(s[i + 1]) : "r"(f + 4u * (m * NT + j + 2 * i)) : "memory");
                    landed();
#pragma unroll
                    for (int i = 0; i < 8; ++i) add_scaled(acc[8 * c + i], v[2 * i], v[2 * i + 1], s[i]);
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) arrive(given0 + 8u * buffer);
                if (++buffer == BUFFERS) { buffer = 0; par ^= 1u; }
                if (++slot == SLOTS) slot = 0;
            }
            if (ok) {   // all products of this CTA are done: the ring is free
                float* const mine = parts + (half * EACH) * kPartPitch + quarter * 32 + lane;
#pragma unroll
                for (int i = 0; i < F::OWN / 2; ++i) {
                    const int m = 2 * i / EACH, j = 2 * i - m * EACH;
                    const float2 v = of_pair(acc[i]);
                    mine[(m * NT + j) * kPartPitch] = v.x;
                    mine[(m * NT + j + 1) * kPartPitch] = v.y;
                }
            }
        }
        done += blocks;
        if (p.ranges > 1) cluster.sync(); else __syncthreads();
        // ---- results: a warp has a row of x, a lane four columns ----
        if (!*failed) {
            const int col = col_tile * 128 + 4 * lane, rest = p.n - col, rows = min(NT, to - row0), size = f8_size(p.dtype);
            for (int r = range * F::WARPS + warp; r < rows; r += p.ranges * F::WARPS) {
                float4 g = make_float4(0.f, 0.f, 0.f, 0.f), u = g;
                for (int c = 0; c < p.ranges; ++c) {
                    const float* part = (p.ranges > 1 ? cluster.map_shared_rank(parts, c) : parts) + r * kPartPitch + 4 * lane;
                    const float4 a = *reinterpret_cast<const float4*>(part);
                    g.x += a.x; g.y += a.y; g.z += a.z; g.w += a.w;
                    if (GATED) {
                        const float4 b = *reinterpret_cast<const float4*>(part + NT * kPartPitch);
                        u.x += b.x; u.y += b.y; u.z += b.z; u.w += b.w;
                    }
                }
                if (GATED) {
                    g.x = gated(g.x, u.x, p.act, p.alpha, p.limit); g.y = gated(g.y, u.y, p.act, p.alpha, p.limit);
                    g.z = gated(g.z, u.z, p.act, p.alpha, p.limit); g.w = gated(g.w, u.w, p.act, p.alpha, p.limit);
                }
                unsigned char* dst = p.y + ((long long)(row0 + r) * p.y_stride + col) * size;
                if (p.dtype == SWLM_F8_E4M3) {
                    unsigned top = 0;
                    if (rest > 0) top = __float_as_uint(g.x) & 0x7FFFFFFFu;
                    if (rest > 1) top = max(top, __float_as_uint(g.y) & 0x7FFFFFFFu);
                    if (rest > 2) top = max(top, __float_as_uint(g.z) & 0x7FFFFFFFu);
                    if (rest > 3) top = max(top, __float_as_uint(g.w) & 0x7FFFFFFFu);
                    const F8Scale s(__reduce_max_sync(0xffffffffu, top));
                    if (lane == 0) p.y_scale[(long long)col_tile * p.y_scale_stride + row0 + r] = s.scale;
                    const unsigned codes = f8_codes4(g.x * s.inverse, g.y * s.inverse, g.z * s.inverse, g.w * s.inverse);
                    if (rest >= 4) *reinterpret_cast<unsigned*>(dst) = codes;
                    else for (int e = 0; e < rest; ++e) dst[e] = (unsigned char)(codes >> (8 * e));
                } else if (p.dtype == SWLM_F8_FP32) {
                    const float v[4] = {g.x, g.y, g.z, g.w};
                    if (rest >= 4) *reinterpret_cast<float4*>(dst) = g;
                    else for (int e = 0; e < 3; ++e) { if (e < rest) reinterpret_cast<float*>(dst)[e] = v[e]; }
                } else {
                    const uint2 v = make_uint2(pack2(g.x, g.y, p.dtype == SWLM_F8_FP16), pack2(g.z, g.w, p.dtype == SWLM_F8_FP16));
                    if (rest >= 4) *reinterpret_cast<uint2*>(dst) = v;
                    else for (int e = 0; e < 3; ++e) { if (e < rest) reinterpret_cast<unsigned short*>(dst)[e] = (unsigned short)((e < 2 ? v.x : v.y) >> (16 * (e & 1))); }
                }
            }
        }
        // the parts have been read, here and by the cluster: the ring takes the next tile's copies (the tensor core's reads and these are ordered by the
        // barriers that the copies wait for and this one)
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        if (p.ranges > 1) cluster.sync(); else __syncthreads();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(F::TMEM) : "memory");
}

template <int NT, bool GATED>
int few_attr() {
    SWLM_CUDA(cudaFuncSetAttribute(f8_few_kernel<NT, GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Few<NT, GATED>::SMEM));
    return SWLM_OK;
}

template <int NT, bool GATED>
int few_launch(const swlm_f8_product& a, int ranges, int turns, int* status, cudaStream_t s) {
    using F = Few<NT, GATED>;
    FewParams p{};
    p.x_scale = a.x.scale; p.x_scale_stride = a.x.scale_stride; p.w_scale = a.w.scale; p.up_scale = a.up.scale;
    p.y = static_cast<unsigned char*>(a.y); p.y_stride = a.y_stride; p.y_scale = a.y_scale; p.y_scale_stride = a.y_scale_stride;
    p.offsets = a.offsets; p.status = status; p.rows = a.rows; p.n = a.n; p.blocks = f8_blocks(a.k); p.experts = a.experts;
    p.ranges = ranges; p.turns = turns; p.dtype = a.dtype; p.act = a.act; p.alpha = a.alpha; p.limit = a.limit;
    const int64_t matrix_rows = (int64_t)std::max(a.experts, 1) * a.n;
    CUtensorMap xmap, wmap, upmap;
    int rc = code_map(a.x.codes, a.x.stride, a.rows, a.k, NT, &xmap);
    if (!rc) rc = code_map(a.w.codes, a.w.stride, matrix_rows, a.k, 128, &wmap);
    upmap = wmap;
    if (!rc && GATED) rc = code_map(a.up.codes, a.up.stride, matrix_rows, a.k, 128, &upmap);
    if (rc) return rc;
    const dim3 grid((unsigned)(f8_blocks(a.n) * ranges), (unsigned)(std::max(a.experts, 1) * turns));
    const cudaError_t e = launch_clusters(f8_few_kernel<NT, GATED>, ranges, grid, dim3(F::THREADS), F::SMEM, s, p, xmap, wmap, upmap);
    return e == cudaSuccess ? SWLM_OK : cuda_fail(e, "product launch");
}

template <int NT>
int few_pick(const swlm_f8_product& a, int ranges, int turns, int* status, cudaStream_t s) {
    return a.act != SWLM_F8_PLAIN ? few_launch<NT, true>(a, ranges, turns, status, s) : few_launch<NT, false>(a, ranges, turns, status, s);
}

}  // namespace

int f8_few_init() {
    int rc;
    if ((rc = few_attr<16, false>()) || (rc = few_attr<16, true>()) || (rc = few_attr<32, false>()) || (rc = few_attr<32, true>()) || (rc = few_attr<64, false>()) ||
        (rc = few_attr<64, true>()) || (rc = few_attr<128, false>()) || (rc = few_attr<128, true>())) return rc;
    return SWLM_OK;
}

int launch_f8_few(const swlm_f8_product& a, int* status, cudaStream_t s) {
    const int experts = std::max(a.experts, 1), each = (a.rows + experts - 1) / experts;
    const int nt = each <= 16 ? 16 : each <= 32 ? 32 : each <= 64 ? 64 : 128, per_sm = nt <= 32 ? 2 : 1;
    // an expert may have more rows than the average: a few CTAs share its tiles
    const int turns = a.experts ? std::min(4, (a.rows + nt - 1) / nt) : (a.rows + nt - 1) / nt;
    const int64_t tiles = (int64_t)f8_blocks(a.n) * (a.experts ? std::min(a.experts, a.rows) : turns);
    int ranges = 1;
    while (ranges < 8 && tiles * ranges * 2 <= kSms * per_sm && f8_blocks(a.k) >= 4 * ranges) ranges *= 2;
    switch (nt) {
    case 16: return few_pick<16>(a, ranges, turns, status, s);
    case 32: return few_pick<32>(a, ranges, turns, status, s);
    case 64: return few_pick<64>(a, ranges, turns, status, s);
    default: return few_pick<128>(a, ranges, turns, status, s);
    }
}

}  // namespace swlm
