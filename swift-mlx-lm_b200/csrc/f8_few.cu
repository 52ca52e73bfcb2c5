// Products in 8-bit floating point of few rows (of few rows per expert): the weights' bytes are what counts.
//
// A tile is 128 rows of w, the lanes of tensor memory, by NT rows of x, its columns. As with many rows (f8_product.cu) a block's sums leave tensor memory before
// they are scaled and added; here the scales of the rows of x lie along a thread's registers. Where there are tiles for all SMs, CTAs take them in turn and
// copies run ahead into the next tile. Where there are few, the blocks of K are dealt to the CTAs of a cluster: their parts then lie in shared memory, 128
// columns of the result to a row of x, and a warp adds the cluster's parts of a row up in the order of the blocks.
// What bounds it: memory, and what a launch takes to start and to end. One row x 4096 x 14336 takes 14.1 us of which its 59 MB are 9 (one, two, four, eight
// CTAs along K: 35.3, 20.6, 14.1, 14.0); 41 rows x 8192 x 2048, gated, 12 to 13 of 5.2; gate and up of 64 experts, 2048 x 1024, for 256 rows 52 (268 MB: 41).
#include <algorithm>

#include <cooperative_groups.h>

#include "f8_device.cuh"

namespace cg = cooperative_groups;

namespace swlm {
using namespace f8;
namespace {

constexpr int kPartPitch = 132;   // floats of a row's part (four more than its columns)

// Clusters of 1, 2, 4 and 8 CTAs, where an SM takes one CTA and where it takes two. A cluster stays within a GPC, so that larger ones leave some SMs without a CTA.
// kAtOnce: how many run at once, by the starts and ends of the CTAs of a launch of many (fourteen of eight on a GPU whose GPCs have other SMs): a launch has no more,
// since others would start when those end. kChosenFor: tiles up to which the choice of a form deals K to clusters of that size. Fewer where an SM takes two: with 71
// and 33 for 66 and 16 one size in forty takes another form, and 80 such sizes drawn at random took 1.02 times as long (0.81 to 1.26).
constexpr int kAtOnce[2][4] = {{148, 74, 33, 15}, {296, 148, 71, 33}}, kChosenFor[2][4] = {{148, 74, 33, 14}, {296, 148, 66, 16}};
constexpr int cluster_size(int ranges) { return ranges == 1 ? 0 : ranges == 2 ? 1 : ranges == 4 ? 2 : 3; }

struct FewParams {
    const float *x_scale, *w_scale, *up_scale;
    long long x_scale_stride, y_stride, y_scale_stride;
    unsigned char* y;
    float* y_scale;
    TileShape tiles;
    int* status;
    int n, blocks, col_blocks;      // blocks of K; of n: scales of a matrix, and tiles
    int ranges;                     // CTAs of a cluster
    int dtype, act;
    float alpha, limit;
};

template <int NT, bool GATED> struct Few {
    static constexpr int TAKERS = NT >= 64 ? 8 : 4, WARPS = 4 + TAKERS, THREADS = WARPS * 32;
    static constexpr int MATS = GATED ? 2 : 1, COLS = MATS * NT;      // accumulators of a block
    static constexpr int BUFFERS = COLS <= 64 ? 4 : 2, TMEM = COLS * BUFFERS < 32 ? 32 : COLS * BUFFERS;
    static constexpr int STAGE = MATS * kCodesBytes + NT * kF8Block;
    static constexpr int PER_SM = NT <= 32 ? 2 : 1;
    static constexpr int STAGES = (PER_SM == 2 ? 104 * 1024 : 200 * 1024) / STAGE;
    static constexpr int SLOTS = 2 * BUFFERS;                          // blocks whose scales have room
    static constexpr int OWN = NT * MATS / (TAKERS / 4);               // accumulators of a thread: OWN / MATS columns of each matrix
    static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE + SLOTS * COLS * 4 + 4 * NT * 4 + kExpertMax * 4;
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
    unsigned* const tops = reinterpret_cast<unsigned*>(scales + SLOTS * COLS);            // [4][NT]
    int* const first_tile = reinterpret_cast<int*>(tops + 4 * NT);                         // [experts]
    float* const parts = reinterpret_cast<float*>(ring);                                   // [MATS][NT][kPartPitch], behind the products
    __shared__ __align__(8) unsigned long long full[STAGES], empty[STAGES], sums_full[BUFFERS], sums_empty[BUFFERS];
    __shared__ unsigned tmem_base;
    __shared__ int failed_word, warp_tiles[F::WARPS];
    volatile int* const failed = &failed_word;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int range = (int)(blockIdx.x % p.ranges), first = (int)(blockIdx.x / p.ranges), step = (int)(gridDim.x / p.ranges);
    const int block0 = (int)((long long)p.blocks * range / p.ranges), blocks = (int)((long long)p.blocks * (range + 1) / p.ranges) - block0;
    pdl_wait();
    auto load = [&](const Tile& tile, int b, int s) {   // by one thread
        const unsigned dst = smem_u32(ring) + s * STAGE, bar = smem_u32(&full[s]);
        const int col = (block0 + b) * kF8Block, w_row = tile.expert * p.n + tile.col * 128;
        mbar_expect(bar, (unsigned)STAGE);
        tma_load_2d(dst, &wmap, col, w_row, bar);
        if (GATED) tma_load_2d(dst + kCodesBytes, &upmap, col, w_row, bar);
        tma_load_2d(dst + MATS * kCodesBytes, &xmap, col, tile.row0, bar);
    };
    int early = 0;   // blocks of the first tile that are asked for before anything else is set up, where no table is needed to say which they are
    if (warp == 0) {
        if (lane == 0) {
            for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
            for (int i = 0; i < BUFFERS; ++i) { mbar_init(&sums_full[i], 1 + 1); mbar_init(&sums_empty[i], F::TAKERS); }
            failed_word = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        if (!p.tiles.experts && first < (p.tiles.rows + NT - 1) / NT * p.tiles.col_tiles) {
            early = min(STAGES, blocks);
            if (elect_one()) {
                const Tile tile = tile_at(p.tiles, first_tile, first);
                for (int b = 0; b < early; ++b) load(tile, b, b);
            }
            __syncwarp();
        }
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)), "r"(F::TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const int tiles = count_tiles<F::THREADS>(p.tiles, first_tile, warp_tiles);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = tmem_base;
    const cg::cluster_group cluster = cg::this_cluster();
    auto fail = [&](int code) { if (lane == 0) { atomicExch_system(p.status, code); *failed = 1; } __syncwarp(); };

    // A launch behind this one may set itself up (behind the allocation: it cannot get at tensor memory in between): 0.6 us of a chain of products. Not with
    // experts, where its CTAs would take places that this one's still want (routed 32 x 2048: 82.6 us, with it 85.8).
    if (!p.tiles.experts) pdl_launch_dependents();
    // Alone every warp runs through all tiles by itself; the CTAs of a cluster meet behind each. A wait that expires ends a warp's work; the cluster's barriers are kept.
    const bool alone = p.ranges == 1;
    auto meet = [&] { if (!alone) cluster.sync(); };

    if (warp == 0) {
        const bool el = elect_one();
        const unsigned full0 = held_address(&full[0]), empty0 = held_address(&empty[0]);
        int s = early % STAGES, issued = early;
        unsigned par = early == STAGES ? 0u : 1u;
        bool ok = true;
        for (int t = first; t < tiles; t += step) {
            const Tile tile = tile_at(p.tiles, first_tile, t);
            for (int b = t == first ? early : 0; b < blocks && ok; ++b) {
                if (!(ok = mbar_wait_warp(empty0 + 8u * s, par))) break;
                if (el) load(tile, b, s);
                __syncwarp();
                ++issued;
                if (++s == STAGES) { s = 0; par ^= 1u; }
            }
            meet();
            meet();
        }
        if (!ok) {   // copies already requested still write shared memory
            fail(21);
            for (int i = max(issued - STAGES, 0); i < issued; ++i) mbar_wait_warp(full0 + 8u * (i % STAGES), (unsigned)((i / STAGES) & 1));
        }
    } else if (warp == 1) {
        constexpr unsigned desc = idesc(128, NT);
        const bool el = elect_one();
        const unsigned full0 = held_address(&full[0]), sums0 = held_address(&sums_empty[0]), at = umma_desc_lo(held_address(ring));
        int s = 0, buffer = 0;
        unsigned par = 0, sums_par = 1;
        bool ok = true;
        for (int t = first; t < tiles; t += step) {
            for (int b = 0; b < blocks && ok; ++b) {
                ok = mbar_wait_warp(full0 + 8u * s, par) && mbar_wait_warp(sums0 + 8u * buffer, sums_par);
                if (!ok) { fail(22); break; }
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
            meet();
            meet();
        }
    } else if (warp == 2) {
        // The factors of a block's sums: a scale of each row of x times the matrices'. A slot is free again by the time that it is written: the takers
        // have left block it - 2 BUFFERS before block it - BUFFERS was multiplied.
        constexpr int PER = (NT + 31) / 32, AHEAD = 4;
        const unsigned full0 = held_address(&sums_full[0]);
        float* slot = scales;
        int buffer = 0, turn = 0;      // turn: how often all buffers have been used
        bool ok = true;
        for (int t = first; t < tiles; t += step) {
            const Tile tile = tile_at(p.tiles, first_tile, t);
            const long long at = ((long long)tile.expert * p.col_blocks + tile.col) * p.blocks + block0;
            float x[AHEAD][PER], w[AHEAD][2];
            auto ask = [&](int u, int b) {
                if (b >= blocks) return;
                const float* src = p.x_scale + (block0 + b) * p.x_scale_stride + tile.row0;
#pragma unroll
                for (int i = 0; i < PER; ++i) x[u][i] = lane + 32 * i < NT && tile.row0 + lane + 32 * i < tile.end ? src[lane + 32 * i] : 0.f;
                w[u][0] = p.w_scale[at + b];
                w[u][1] = GATED ? p.up_scale[at + b] : 0.f;
            };
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) ask(u, u);
            for (int b0 = 0; b0 < blocks && ok; b0 += AHEAD) {
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    const int b = b0 + u;
                    if (b >= blocks || !ok) break;
                    if (turn > 0) ok = mbar_wait_warp(full0 + 8u * buffer, (unsigned)((turn - 1) & 1));
                    if (!ok) { fail(23); break; }
#pragma unroll
                    for (int i = 0; i < PER; ++i)
                        if (lane + 32 * i < NT) {
                            slot[lane + 32 * i] = x[u][i] * w[u][0];
                            if (GATED) slot[NT + lane + 32 * i] = x[u][i] * w[u][1];
                        }
                    __syncwarp();
                    if (lane == 0) arrive(full0 + 8u * buffer);
                    ask(u, b + AHEAD);
                    if (++buffer == BUFFERS) { buffer = 0; ++turn; }
                    slot = slot == scales + (SLOTS - 1) * COLS ? scales : slot + COLS;
                }
            }
            meet();
            meet();
        }
    } else if (warp == 3) {
        for (int t = first; t < tiles; t += step) {
            meet();
            meet();
        }
    } else {
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        constexpr int EACH = F::OWN / MATS;      // columns of a thread of each matrix
        const unsigned full0 = held_address(&sums_full[0]), given0 = held_address(&sums_empty[0]), factors = held_address(scales) + 4u * (half * EACH);
        const unsigned at = tmem + ((unsigned)(quarter * 32) << 16) + half * EACH;
        const int size = f8_size(p.dtype);
        int buffer = 0;
        unsigned par = 0, slot = 0;
        bool ok = true;
        for (int t = first; t < tiles; t += step) {
            unsigned long long acc[F::OWN / 2];
#pragma unroll
            for (int i = 0; i < F::OWN / 2; ++i) acc[i] = 0;
            for (int b = 0; b < blocks && ok; ++b) {
                ok = mbar_wait_warp(full0 + 8u * buffer, par);
                if (!ok) { fail(24); break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned here = at + buffer * COLS, f = factors + slot;
#pragma unroll
                for (int c = 0; c < F::OWN / 16; ++c) {
                    const int m = c / (EACH / 16), j = (c % (EACH / 16)) * 16;   // matrix, first column
                    unsigned v[16];
                    tmem_load(v, here + m * NT + j);
                    unsigned long long s[8];
#pragma unroll
                    for (int i = 0; i < 8; i += 2) asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(s[i]), "=l"(s[i + 1]) : "r"(f + 4u * (m * NT + j + 2 * i)) : "memory");
                    landed();
                    if (c == F::OWN / 16 - 1) {   // all of them are in registers: the buffer is free
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) arrive(given0 + 8u * buffer);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) add_scaled(acc[8 * c + i], v[2 * i], v[2 * i + 1], s[i]);
                }
                if (++buffer == BUFFERS) { buffer = 0; par ^= 1u; }
                slot = slot == (SLOTS - 1) * COLS * 4 ? 0u : slot + COLS * 4;
            }
            const Tile tile = tile_at(p.tiles, first_tile, t);
            const int rows = min(NT, tile.end - tile.row0);
            if (alone) {
                // ---- results of one CTA: a lane has a column, its registers are rows of x ----
                const int col = tile.col * 128 + quarter * 32 + lane, row0 = tile.row0 + half * EACH, count = ok ? rows - half * EACH : 0;   // (a warp whose wait has expired stores nothing, but keeps the takers' barriers)
                const bool there = col < p.n;
                float value[EACH];
#pragma unroll
                for (int i = 0; i < EACH; i += 2) {
                    const float2 g = of_pair(acc[i / 2]);
                    value[i] = g.x; value[i + 1] = g.y;
                    if (GATED) {
                        const float2 u = of_pair(acc[(EACH + i) / 2]);
                        value[i] = gated(g.x, u.x, p.act, p.alpha, p.limit);
                        value[i + 1] = gated(g.y, u.y, p.act, p.alpha, p.limit);
                    }
                }
                unsigned char* dst = p.y + ((long long)row0 * p.y_stride + col) * size;
                const long long pitch = p.y_stride * size;
                if (p.dtype == SWLM_F8_E4M3) {   // the block's other columns are three other warps'
#pragma unroll
                    for (int i = 0; i < EACH; ++i) {
                        const unsigned top = __reduce_max_sync(0xffffffffu, there ? __float_as_uint(value[i]) & 0x7FFFFFFFu : 0u);
                        if (lane == 0) tops[quarter * NT + half * EACH + i] = top;
                    }
                    asm volatile("bar.sync 1, %0;" ::"n"(F::TAKERS * 32) : "memory");
#pragma unroll
                    for (int i = 0; i < EACH; ++i) {
                        const unsigned* top = tops + half * EACH + i;
                        const F8Scale s(max(max(top[0], top[NT]), max(top[2 * NT], top[3 * NT])));
                        if (i < count) {
                            if (there) dst[i * pitch] = (unsigned char)f8_codes4(value[i] * s.inverse, 0.f, 0.f, 0.f);
                            if (quarter == 0 && lane == 0) p.y_scale[(long long)tile.col * p.y_scale_stride + row0 + i] = s.scale;
                        }
                    }
                    asm volatile("bar.sync 1, %0;" ::"n"(F::TAKERS * 32) : "memory");
                } else if (p.dtype == SWLM_F8_FP32) {
#pragma unroll
                    for (int i = 0; i < EACH; ++i)
                        if (i < count && there) *reinterpret_cast<float*>(dst + i * pitch) = value[i];
                } else {
                    const bool f16 = p.dtype == SWLM_F8_FP16;
#pragma unroll
                    for (int i = 0; i < EACH; ++i)
                        if (i < count && there) *reinterpret_cast<unsigned short*>(dst + i * pitch) = (unsigned short)pack2(value[i], 0.f, f16);
                }
                continue;
            }
            // ---- results of a cluster ----
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
            meet();
            const int col = tile.col * 128 + 4 * lane, rest = p.n - col;
            for (int r = *failed ? rows : range * F::TAKERS + warp - 4; r < rows; r += p.ranges * F::TAKERS) {   // a warp has a row of x, a lane four columns
                float4 g = make_float4(0.f, 0.f, 0.f, 0.f), u = g;
                for (int c = 0; c < p.ranges; ++c) {
                    const float* part = cluster.map_shared_rank(parts, c) + r * kPartPitch + 4 * lane;
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
                unsigned char* dst = p.y + ((long long)(tile.row0 + r) * p.y_stride + col) * size;
                if (p.dtype == SWLM_F8_E4M3) {
                    unsigned top = 0;
                    if (rest > 0) top = __float_as_uint(g.x) & 0x7FFFFFFFu;
                    if (rest > 1) top = max(top, __float_as_uint(g.y) & 0x7FFFFFFFu);
                    if (rest > 2) top = max(top, __float_as_uint(g.z) & 0x7FFFFFFFu);
                    if (rest > 3) top = max(top, __float_as_uint(g.w) & 0x7FFFFFFFu);
                    const F8Scale s(__reduce_max_sync(0xffffffffu, top));
                    if (lane == 0) p.y_scale[(long long)tile.col * p.y_scale_stride + tile.row0 + r] = s.scale;
                    const unsigned codes = f8_codes4(g.x * s.inverse, g.y * s.inverse, g.z * s.inverse, g.w * s.inverse);
                    if (rest >= 4) *reinterpret_cast<unsigned*>(dst) = codes;
                    else for (int e = 0; e < rest; ++e) dst[e] = (unsigned char)(codes >> (8 * e));
                } else if (p.dtype == SWLM_F8_FP32) {
                    const float v[3] = {g.x, g.y, g.z};
                    if (rest >= 4) *reinterpret_cast<float4*>(dst) = g;
                    else {
#pragma unroll
                        for (int e = 0; e < 3; ++e) if (e < rest) reinterpret_cast<float*>(dst)[e] = v[e];
                    }
                } else {
                    const uint2 v = make_uint2(pack2(g.x, g.y, p.dtype == SWLM_F8_FP16), pack2(g.z, g.w, p.dtype == SWLM_F8_FP16));
                    if (rest >= 4) *reinterpret_cast<uint2*>(dst) = v;
                    else {
#pragma unroll
                        for (int e = 0; e < 3; ++e) if (e < rest) reinterpret_cast<unsigned short*>(dst)[e] = (unsigned short)((e < 2 ? v.x : v.y) >> (16 * (e & 1)));
                    }
                }
            }
            // the parts have been read, here and by the cluster: behind the barrier the ring takes the next tile's copies
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            meet();
        }
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
int few_launch(const swlm_f8_product& a, int ranges, int* status, cudaStream_t s) {
    using F = Few<NT, GATED>;
    FewParams p{};
    p.x_scale = a.x.scale; p.x_scale_stride = a.x.scale_stride; p.w_scale = a.w.scale; p.up_scale = a.up.scale;
    p.y = static_cast<unsigned char*>(a.y); p.y_stride = a.y_stride; p.y_scale = a.y_scale; p.y_scale_stride = a.y_scale_stride;
    p.tiles = {a.offsets, a.rows, a.experts, NT, f8_blocks(a.n)}; p.status = status; p.n = a.n; p.blocks = f8_blocks(a.k); p.col_blocks = f8_blocks(a.n);
    p.ranges = ranges; p.dtype = a.dtype; p.act = a.act; p.alpha = a.alpha; p.limit = a.limit;
    const int64_t matrix_rows = (int64_t)std::max(a.experts, 1) * a.n;
    CUtensorMap xmap, wmap, upmap;
    int rc = code_map(a.x.codes, a.x.stride, a.rows, a.k, NT, &xmap);
    if (!rc) rc = code_map(a.w.codes, a.w.stride, matrix_rows, a.k, 128, &wmap);
    upmap = wmap;
    if (!rc && GATED) rc = code_map(a.up.codes, a.up.stride, matrix_rows, a.k, 128, &upmap);
    if (rc) return rc;
    // (at most this many tiles: an expert's last one may have a single row)
    const int64_t tiles = std::min<int64_t>(((int64_t)a.rows / NT + std::max(a.experts, 1)) * p.col_blocks, kAtOnce[F::PER_SM - 1][cluster_size(ranges)]);
    const cudaError_t e = launch_clusters(f8_few_kernel<NT, GATED>, ranges, dim3((unsigned)(tiles * ranges)), dim3(F::THREADS), F::SMEM, s, p, xmap, wmap, upmap);
    return e == cudaSuccess ? SWLM_OK : cuda_fail(e, "product launch");
}

}  // namespace

int f8_few_init() {
    int rc;
    if ((rc = few_attr<16, false>()) || (rc = few_attr<16, true>()) || (rc = few_attr<32, false>()) || (rc = few_attr<64, false>()) ||
        (rc = few_attr<64, true>()) || (rc = few_attr<128, false>())) return rc;
    return SWLM_OK;
}

// A block takes a tile 0.22 to 0.36 (twice the matrices: 0.36 to 0.4), a launch's first tile starts and ends in 4.5 to 7.5, further ones in 1, the exchange of a cluster
// takes 0.5; weights come from memory at 6.2 TB/s. Gated tiles of 128 rows took three times as long as two of 64, those of 32 as long as those of 64.
F8FewForm f8_few_form(int rows, int n, int k, int experts, bool gated) {
    F8FewForm best{0, 0, 1e30};
    const int blocks = f8_blocks(k), reached = experts ? std::min(experts, rows) : 1;
    const double memory = (double)reached * n * k * (gated ? 2 : 1) / 6.2e6;
    for (int nt = 16; nt <= (gated ? 64 : 128); nt *= 2) {
        if (gated && nt == 32) continue;
        const int per_sm = nt <= 32 ? 2 : 1;
        const double alone = gated ? (nt <= 16 ? 0.36 : 0.39) : nt == 16 ? 0.22 : nt == 32 ? 0.24 : nt == 64 ? 0.27 : 0.36;
        const double ends = nt <= 32 ? 3.5 : nt == 128 ? 6.5 : gated ? 5.0 : 4.0;
        // rows of an expert end inside a tile
        const double row_tiles = experts ? rows / (double)nt + 0.5 * reached : (rows + nt - 1) / nt, tiles = std::max(row_tiles, (double)reached) * f8_blocks(n);
        for (int ranges = 1; ranges <= 8 && ranges <= blocks; ranges *= 2) {
            const double slots = ranges * kChosenFor[per_sm - 1][cluster_size(ranges)], waves = (double)(int64_t)((tiles * ranges + slots - 1) / slots);
            if (ranges > 1 && waves > 1) break;
            const double both = per_sm == 2 && tiles * ranges > kSms ? 1.5 : 1.0;   // two CTAs on an SM share it
            const double ctas = std::min(tiles * ranges, slots), step = std::max(alone * both, ctas * ((gated ? 2 : 1) * kCodesBytes + nt * kF8Block) / 10e6);   // L2 gives 10 TB/s
            const double cost = std::max(waves * ((blocks + ranges - 1) / ranges * step + 1), memory) + ends + (ranges > 1 ? 0.5 : 0.0);
            if (cost < best.cost) best = {nt, ranges, cost};
        }
    }
    return best;
}

int launch_f8_few(const swlm_f8_product& a, const F8FewForm& form, int* status, cudaStream_t s) {
    const bool gated = a.act != SWLM_F8_PLAIN;
    switch (form.nt) {
    case 16: return gated ? few_launch<16, true>(a, form.ranges, status, s) : few_launch<16, false>(a, form.ranges, status, s);
    case 32: return few_launch<32, false>(a, form.ranges, status, s);
    case 64: return gated ? few_launch<64, true>(a, form.ranges, status, s) : few_launch<64, false>(a, form.ranges, status, s);
    default: return few_launch<128, false>(a, form.ranges, status, s);
    }
}

}  // namespace swlm
