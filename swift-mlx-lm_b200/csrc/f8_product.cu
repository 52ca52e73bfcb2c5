// Products of rows and matrices in 8-bit floating point: y = sum over blocks of 128 columns of sx sw (x . w), on tcgen05.
//
// The products of a block's codes are exact and summed in fp32 in tensor memory; two scales belong to every block, so its sums leave tensor memory before the
// next block's are added: registers hold acc += (sx sw) sums, in fp32. A block is 128 bytes of a row, one swizzle row and four MMAs of K = 32.
#include <algorithm>
#include <type_traits>

#include <cooperative_groups.h>

#include "f8_device.cuh"

namespace cg = cooperative_groups;

namespace swlm {
using namespace f8;
namespace {

// ---- many rows ---------------------------------------------------------------------------------------------------------------
// Persistent pairs of CTAs that share a tile of 256 rows x 256 columns of accumulators: lanes of tensor memory are rows of x, a thread has one row and 128 of
// the columns. A warp for the copies, one for the MMAs, two for the scales, eight that take a block's sums out of one of two buffers of tensor memory while the
// next block's are multiplied into the other. GATED: the accumulators of 64 columns of w lie before those of the same 64 of `up`, so that a thread has both,
// and a tile gives 128 columns of the result.
// What bounds it: a pair's block is 64 KB from L2, which gives all SMs together some 10 TB/s: 0.47 us, 365 us for 8192 rows x 4096 x 14336 without any product
// or sum, and 400 with them (2.4 PFLOP/s). Kept up for seconds it is bound by power: 990 W, the SM clock falls from 1965 to 1240 MHz, 470 to 510 us. One CTA
// per tile of 128 rows moved half as much again and was never faster by more than a last wave's tiles.
// The takers: 16 columns at a time, so that nothing spills (439 clocks a block by themselves; with 32 columns on their way while 32 are added ptxas spills, and
// a block took 1090). Registers are dealt out anew after the start: 128 threads x 56 for the first four warps and 256 x 224 for the takers and their 128 sums,
// together the 384 x 168 of the launch.
constexpr int kWideWarps = 12, kWideThreads = kWideWarps * 32, kWideTakers = 8;
constexpr int kAccCols = 256;
constexpr int kScaleDepth = 4;      // blocks whose scales are on their way, and that have room for theirs in shared memory
constexpr int kStageRow = 80;   // results on their way out: 64 bytes of each of a warp's 32 rows (the odd pitch keeps 16-byte accesses off each other's banks)

struct WideParams {
    const float *x_scale, *w_scale, *up_scale;
    long long x_scale_stride, y_stride, y_scale_stride;
    unsigned char* y;
    float* y_scale;
    TileShape tiles;
    int* status;
    int n, blocks, col_blocks;          // blocks of K; of n: scales of a matrix
    int dtype, act;
    float alpha, limit;
};

constexpr int kStages = 6, kStage = 2 * kCodesBytes;   // a CTA's 128 rows of x, and half of the matrix's
constexpr size_t kWideSmem = 1024 + (size_t)kStages * kStage + kWideTakers * 32 * kStageRow + kScaleDepth * 128 * 8 + 2 * 128 * 4 + kExpertMax * 4;
static_assert(kWideSmem <= 232448 - 1024, "shared memory");

template <bool GATED>
__global__ void __launch_bounds__(kWideThreads, 1) f8_wide_kernel(const WideParams p, const __grid_constant__ CUtensorMap xmap,
                                                                  const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap upmap) {
    constexpr int COLS = GATED ? 128 : 256;
    extern __shared__ __align__(1024) unsigned char wide_raw[];
    unsigned char* const ring = wide_raw + ((1024 - (smem_u32(wide_raw) & 1023)) & 1023);   // swizzle atoms
    unsigned char* const staging = ring + kStages * kStage;
    float2* const scales = reinterpret_cast<float2*>(staging + kWideTakers * 32 * kStageRow);   // [kScaleDepth][128]
    unsigned* const tops = reinterpret_cast<unsigned*>(scales + kScaleDepth * 128);             // [2][128]
    int* const first_tile = reinterpret_cast<int*>(tops + 256);                                // [experts]
    __shared__ __align__(8) unsigned long long full[kStages], empty[kStages], sums_full[2], sums_empty[2];
    __shared__ unsigned tmem_base;
    __shared__ int warp_tiles[kWideWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)(blockIdx.x & 1);
    if (tid == 0) {
        for (int s = 0; s < kStages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&sums_full[i], 1 + 2); mbar_init(&sums_empty[i], 2 * kWideTakers); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)), "r"(2 * kAccCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    pdl_wait();
    const int tiles = count_tiles<kWideThreads>(p.tiles, first_tile, warp_tiles);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cg::this_cluster().sync();   // both CTAs' barriers are ready
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = tmem_base;
    const int first = (int)blockIdx.x / 2, step = (int)gridDim.x / 2;
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0) {
            // The warp runs its loop as a whole, one lane issues. Of a pair both CTAs' copies count on the barrier of the one that issues the MMAs.
            const bool el = elect_one();
            const unsigned full0 = cluster_place(smem_u32(&full[0]), 0), empty0 = held_address(&empty[0]), at = held_address(ring);
            auto load = [&](unsigned dst, const CUtensorMap* map, int col, int row, int s) { tma_load_2d_pair(dst, map, col, row, full0 + 8u * s); };
            int s = 0, issued = 0;
            unsigned par = 1;
            bool ok = true;
            for (int t = first; t < tiles && ok; t += step) {
                const Tile tile = tile_at(p.tiles, first_tile, t);
                const int x_row = tile.row0 + rank * 128, w_row = tile.expert * p.n + tile.col * COLS + rank * (COLS / 2);
                for (int b = 0; b < p.blocks; ++b) {
                    if (!mbar_wait_warp(empty0 + 8u * s, par)) { ok = false; break; }
                    if (el) {
                        const unsigned dst = at + s * kStage;
                        if (rank == 0) mbar_expect(full0 + 8u * s, 2u * kStage);
                        load(dst, &xmap, b * kF8Block, x_row, s);
                        load(dst + kCodesBytes, &wmap, b * kF8Block, w_row, s);
                        if (GATED) load(dst + kCodesBytes + kCodesBytes / 2, &upmap, b * kF8Block, w_row, s);
                    }
                    __syncwarp();
                    ++issued;
                    if (++s == kStages) { s = 0; par ^= 1u; }
                }
            }
            if (!ok) {   // copies already requested still write shared memory (in a pair's second CTA, whose barrier this is not, the limit of the wait is the time they get)
                if (el) atomicExch_system(p.status, 11);
                for (int i = max(issued - kStages, 0); i < issued; ++i) mbar_wait_warp(&full[i % kStages], (unsigned)((i / kStages) & 1));
            }
        } else if (warp == 1) {
            if (rank == 0) {
                constexpr unsigned desc = idesc(256, kAccCols);
                const bool el = elect_one();
                const unsigned full0 = held_address(&full[0]), sums0 = held_address(&sums_empty[0]), at = umma_desc_lo(held_address(ring));
                int s = 0;
                unsigned par = 0, buffer = 0, sums_par = 1;
                bool ok = true;
                for (int t = first; t < tiles && ok; t += step)
                    for (int b = 0; b < p.blocks; ++b) {
                        // (what the barriers guard is read by the tensor cores: no ordinary load has to see another CTA's stores)
                        ok = mbar_wait_warp(full0 + 8u * s, par) && mbar_wait_warp(sums0 + 8u * buffer, sums_par);
                        if (!ok) { if (el) atomicExch_system(p.status, 12); break; }
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        if (el) {
                            const unsigned a = at + s * (kStage / 16), w = a + kCodesBytes / 16, sums = tmem + buffer * kAccCols;
#pragma unroll
                            for (int j = 0; j < 4; ++j) umma<2>(sums, a + 2 * j, w + 2 * j, desc, j > 0);
                            commit<2>(&empty[s]);
                            commit<2>(&sums_full[buffer]);
                        }
                        __syncwarp();
                        if (++s == kStages) { s = 0; par ^= 1u; }
                        buffer ^= 1u;
                        sums_par ^= buffer ^ 1u;
                    }
            }
        } else {
            // Two warps for the scales, 64 rows each: what the accumulators of a row are worth, as two factors (of the two halves of the columns, or of w's
            // and up's), is in shared memory before the sums are said to be there. A slot is free again by then: the takers have left block
            // it - 4 before block it - 2 was multiplied.
            const int r0 = (warp - 2) * 64 + 2 * lane;
            const unsigned full0 = held_address(&sums_full[0]);
            float2* const mine = scales + r0;
            struct Ahead { float x[2], w[2]; } ahead[kScaleDepth];
            Tile tile{};
            int t = first, b = 0;      // the block that is asked for next
            bool any = t < tiles;
            if (any) tile = tile_at(p.tiles, first_tile, t);
            auto ask = [&](Ahead& a) {
                if (!any) return;
                const int row = tile.row0 + rank * 128 + r0, block = GATED ? tile.col : 2 * tile.col;
                const float* x = p.x_scale + b * p.x_scale_stride + row;
                const long long at = ((long long)tile.expert * p.col_blocks + block) * p.blocks + b;
                a.x[0] = row < tile.end ? *x : 0.f;
                a.x[1] = row + 1 < tile.end ? x[1] : 0.f;
                a.w[0] = p.w_scale[at];
                a.w[1] = GATED ? p.up_scale[at] : block + 1 < p.col_blocks ? p.w_scale[at + p.blocks] : 0.f;
                if (++b == p.blocks) {
                    b = 0; t += step;
                    any = t < tiles;
                    if (any) tile = tile_at(p.tiles, first_tile, t);
                }
            };
            const int total = first < tiles ? (tiles - 1 - first) / step + 1 : 0;
            const int all = total * p.blocks;
#pragma unroll
            for (int u = 0; u < kScaleDepth; ++u) ask(ahead[u]);
            bool ok = true;
            for (int it0 = 0; it0 < all && ok; it0 += kScaleDepth) {
#pragma unroll
                for (int u = 0; u < kScaleDepth; ++u) {
                    const int it = it0 + u;
                    if (it >= all || !ok) break;
                    if (it >= 2) ok = mbar_wait_warp(full0 + 8u * (u & 1), (unsigned)(((it >> 1) - 1) & 1));
                    if (!ok) { if (lane == 0) atomicExch_system(p.status, 14); break; }
                    const Ahead now = ahead[u];
                    *reinterpret_cast<float4*>(mine + u * 128) = make_float4(now.x[0] * now.w[0], now.x[0] * now.w[1], now.x[1] * now.w[0], now.x[1] * now.w[1]);
                    __syncwarp();
                    if (lane == 0) arrive(full0 + 8u * (u & 1));
                    ask(ahead[u]);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        // A warp has the 32 lanes of its quarter (warp & 3) and one half of the columns.
        const int taker = warp - 4, quarter = warp & 3, half = taker >> 2;
        const unsigned at = tmem + ((unsigned)(quarter * 32) << 16) + 128u * half;
        const unsigned full0 = held_address(&sums_full[0]), given0 = cluster_place(smem_u32(&sums_empty[0]), 0);
        const unsigned factors = held_address(scales) + 8u * (quarter * 32 + lane) + (GATED ? 0u : 4u * half);
        unsigned char* const out = staging + taker * 32 * kStageRow;
        unsigned buffer = 0, par = 0, slot = 0;
        bool ok = true;
        for (int t = first; t < tiles; t += step) {
            unsigned long long acc[64];
#pragma unroll
            for (int i = 0; i < 64; ++i) acc[i] = 0;
            for (int b = 0; b < p.blocks && ok; ++b) {
                ok = mbar_wait_warp(full0 + 8u * buffer, par);
                if (!ok) { if (lane == 0) atomicExch_system(p.status, 13); break; }   // (it stores nothing more, but keeps the takers' barriers)
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned from = at + buffer * kAccCols;
                float s_low, s_high;
                if (GATED) asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(s_low), "=f"(s_high) : "r"(factors + slot) : "memory");
                else { asm volatile("ld.shared.f32 %0, [%1];" : "=f"(s_low) : "r"(factors + slot) : "memory"); s_high = s_low; }
                const unsigned long long low = pair_of(s_low, s_low), high = pair_of(s_high, s_high);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    unsigned v[16];
                    tmem_load(v, from + 16 * c);
                    landed();
                    if (c == 7) {   // all of them are in registers: the buffer is free
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) arrive_cluster(given0 + 8u * buffer);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) add_scaled(acc[8 * c + i], v[2 * i], v[2 * i + 1], c < 4 ? low : high);
                }
                buffer ^= 1u;
                par ^= buffer ^ 1u;
                slot = (slot + 1024u) & (1024u * kScaleDepth - 1u);
            }
            const Tile done = tile_at(p.tiles, first_tile, t);
            // ---- results: value i of the thread is column col0 + i of its row ----
            constexpr int VALUES = GATED ? 64 : 128;
            float value[VALUES];
#pragma unroll
            for (int i = 0; i < VALUES; i += 2) {
                const float2 g = of_pair(acc[i / 2]);
                value[i] = g.x; value[i + 1] = g.y;
                if (GATED) {
                    const float2 u = of_pair(acc[32 + i / 2]);
                    value[i] = gated(g.x, u.x, p.act, p.alpha, p.limit);
                    value[i + 1] = gated(g.y, u.y, p.act, p.alpha, p.limit);
                }
            }
            const int row0 = done.row0 + rank * 128 + quarter * 32, col0 = done.col * COLS + half * VALUES;
            if (p.dtype == SWLM_F8_E4M3) {
                unsigned top = 0;
#pragma unroll
                for (int i = 0; i < VALUES; ++i) top = max(top, col0 + i < p.n ? __float_as_uint(value[i]) & 0x7FFFFFFFu : 0u);
                if (GATED) {   // the other half of the block's columns is another warp's
                    tops[half * 128 + quarter * 32 + lane] = top;
                    asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
                    top = max(top, tops[(half ^ 1) * 128 + quarter * 32 + lane]);
                    asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
                }
                const F8Scale s(top);
                if (ok && row0 + lane < done.end && col0 < p.n && !(GATED && half)) p.y_scale[(long long)(col0 / kF8Block) * p.y_scale_stride + row0 + lane] = s.scale;
#pragma unroll
                for (int i = 0; i < VALUES; ++i) value[i] *= s.inverse;
            }
            if (!ok) continue;
            // 64 bytes of each row at a time, by way of the staging rows: a lane then stores sixteen of every eighth row
            const int live = done.end - row0 - (lane >> 2);
            const uint4* const got = reinterpret_cast<const uint4*>(out + (lane >> 2) * kStageRow + (lane & 3) * 16);
            uint4* const put = reinterpret_cast<uint4*>(out + lane * kStageRow);
            auto send = [&](auto size, int c) {   // columns c .. of the warp's are in the staging rows
                constexpr int SIZE = decltype(size)::value, PER = 16 / SIZE;
                unsigned char* dst = p.y + ((long long)(row0 + (lane >> 2)) * p.y_stride + col0 + c) * SIZE + (lane & 3) * 16;
                const long long step8 = 8 * p.y_stride * SIZE;
                const int rest = p.n - col0 - c - (lane & 3) * PER;
                __syncwarp();
                uint4 v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = got[i * (8 * kStageRow / 16)];
                __syncwarp();
                if (rest >= PER) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (8 * i < live) *reinterpret_cast<uint4*>(dst + i * step8) = v[i];
                } else if (rest > 0) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (8 * i >= live) continue;
                        const unsigned w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
                        for (int e = 0; e < PER - 1; ++e) {
                            if (e >= rest) continue;
                            if (SIZE == 4) reinterpret_cast<unsigned*>(dst + i * step8)[e] = w[e & 3];
                            else if (SIZE == 2) reinterpret_cast<unsigned short*>(dst + i * step8)[e] = (unsigned short)(w[(e >> 1) & 3] >> (16 * (e & 1)));
                            else (dst + i * step8)[e] = (unsigned char)(w[e >> 2] >> (8 * (e & 3)));
                        }
                    }
                }
            };
            if (p.dtype == SWLM_F8_FP32) {
#pragma unroll
                for (int c = 0; c < VALUES; c += 16) {
                    if (col0 + c >= p.n) break;
#pragma unroll
                    for (int i = 0; i < 4; ++i) put[i] = make_uint4(__float_as_uint(value[c + 4 * i]), __float_as_uint(value[c + 4 * i + 1]), __float_as_uint(value[c + 4 * i + 2]), __float_as_uint(value[c + 4 * i + 3]));
                    send(std::integral_constant<int, 4>(), c);
                }
            } else if (p.dtype == SWLM_F8_E4M3) {
#pragma unroll
                for (int c = 0; c < VALUES; c += 64) {
                    if (col0 + c >= p.n) break;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float* f = value + c + 16 * i;
                        put[i] = make_uint4(f8_codes4(f[0], f[1], f[2], f[3]), f8_codes4(f[4], f[5], f[6], f[7]), f8_codes4(f[8], f[9], f[10], f[11]), f8_codes4(f[12], f[13], f[14], f[15]));
                    }
                    send(std::integral_constant<int, 1>(), c);
                }
            } else {
                const bool f16 = p.dtype == SWLM_F8_FP16;
#pragma unroll
                for (int c = 0; c < VALUES; c += 32) {
                    if (col0 + c >= p.n) break;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float* f = value + c + 8 * i;
                        put[i] = make_uint4(pack2(f[0], f[1], f16), pack2(f[2], f[3], f16), pack2(f[4], f[5], f16), pack2(f[6], f[7], f16));
                    }
                    send(std::integral_constant<int, 2>(), c);
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cg::this_cluster().sync();   // no MMA of the pair reads tensor memory or arrives at a barrier of a CTA that has left
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * kAccCols) : "memory");
    }
}

// ---- launches ----------------------------------------------------------------------------------------------------------------
template <bool GATED>
int wide_attr() {
    SWLM_CUDA(cudaFuncSetAttribute(f8_wide_kernel<GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kWideSmem));
    return SWLM_OK;
}

template <bool GATED>
int wide_launch(const swlm_f8_product& a, int* status, cudaStream_t s) {
    constexpr int COLS = GATED ? 128 : 256;
    WideParams p{};
    p.x_scale = a.x.scale; p.x_scale_stride = a.x.scale_stride; p.w_scale = a.w.scale; p.up_scale = a.up.scale;
    p.y = static_cast<unsigned char*>(a.y); p.y_stride = a.y_stride; p.y_scale = a.y_scale; p.y_scale_stride = a.y_scale_stride;
    p.tiles = {a.offsets, a.rows, a.experts, 256, (a.n + COLS - 1) / COLS}; p.status = status; p.n = a.n; p.blocks = f8_blocks(a.k);
    p.col_blocks = f8_blocks(a.n); p.dtype = a.dtype; p.act = a.act; p.alpha = a.alpha; p.limit = a.limit;
    const int64_t matrix_rows = (int64_t)std::max(a.experts, 1) * a.n;
    CUtensorMap xmap, wmap, upmap;
    int rc = code_map(a.x.codes, a.x.stride, a.rows, a.k, 128, &xmap);
    if (!rc) rc = code_map(a.w.codes, a.w.stride, matrix_rows, a.k, GATED ? 64 : 128, &wmap);
    upmap = wmap;
    if (!rc && GATED) rc = code_map(a.up.codes, a.up.stride, matrix_rows, a.k, 64, &upmap);
    if (rc) return rc;
    // (at most this many tiles: an expert's last one may have a single row)
    const int64_t tiles = std::min<int64_t>(((int64_t)a.rows / 256 + std::max(a.experts, 1)) * p.tiles.col_tiles, kSms / 2);
    const cudaError_t e = launch_clusters(f8_wide_kernel<GATED>, 2, dim3((unsigned)(2 * tiles)), dim3(kWideThreads), kWideSmem, s, p, xmap, wmap, upmap);
    return e == cudaSuccess ? SWLM_OK : cuda_fail(e, "product launch");
}

// What a product takes, about (us): a block 0.38 while the pairs are few, 0.47 with all of them reading from L2, a launch and its first tile's start and end 7.5; weights
// that are read once come from memory at 3.2 TB/s.
double wide_cost(int rows, int n, int k, int experts, bool gated) {
    const int cols = gated ? 128 : 256, reached = experts ? std::min(experts, rows) : 1;
    const double row_tiles = experts ? std::max(rows / 256.0 + 0.5 * reached, (double)reached) : (rows + 255) / 256, tiles = row_tiles * ((n + cols - 1) / cols), pairs = kSms / 2;
    auto wave = [&](double busy) { return f8_blocks(k) * (busy > pairs / 2 ? 0.47 : 0.38) + 2; };
    const double full = (double)(int64_t)(tiles / pairs), rest = tiles - full * pairs;
    // (how full an expert's tiles are is not known: their waves are not counted one by one)
    const double run = experts ? std::max(1.0, tiles / pairs) * wave(tiles) : full * wave(pairs) + (rest > 0 ? wave(rest) : 0.0);
    return std::max(run, (double)reached * n * k * (gated ? 2 : 1) / 3.2e6) + 5.5;
}

}  // namespace

int f8_product_init() {
    int rc;
    if ((rc = f8_few_init()) || (rc = wide_attr<false>()) || (rc = wide_attr<true>())) return rc;
    return SWLM_OK;
}

F8ProductForm f8_product_form(int rows, int n, int k, int experts, bool gated) {
    F8ProductForm f;
    f.few = f8_few_form(rows, n, k, experts, gated);
    const double wide = wide_cost(rows, n, k, experts, gated);
    f.wide = f.few.cost > wide ? n : 0;
    // A last wave of few tiles leaves most pairs without work: the columns that fill whole waves may go first, and the rest as a product of its own, dealt out
    // along K (777 rows x 5000 x 4100: 80 tiles on 74 pairs 35.7 us, 72 tiles and 392 columns more 34.0).
    const int cols = gated ? 128 : 256, row_tiles = (rows + 255) / 256, pairs = kSms / 2, waves = (int)((int64_t)row_tiles * ((n + cols - 1) / cols) / pairs);
    const int full = (int)std::min<int64_t>((int64_t)waves * pairs / row_tiles * cols, n);
    if (!experts && full > 0 && full < n) {
        const F8FewForm last = f8_few_form(rows, n - full, k, 0, gated);
        if (wide_cost(rows, full, k, 0, gated) + last.cost < 0.95 * std::min(f.few.cost, wide)) f = {full, last};   // (within what the model is off by, one launch)
    }
    return f;
}

int launch_f8_product(const swlm_f8_product& a, int* status, cudaStream_t s) {
    const bool gated = a.act != SWLM_F8_PLAIN;
    const F8ProductForm form = f8_product_form(a.rows, a.n, a.k, a.experts, gated);
    if (form.wide == 0) return launch_f8_few(a, form.few, status, s);
    swlm_f8_product head = a, tail = a;
    head.n = form.wide;
    const int rc = gated ? wide_launch<true>(head, status, s) : wide_launch<false>(head, status, s);
    if (rc || form.wide == a.n) return rc;
    const int64_t scales = (int64_t)(form.wide / kF8Block) * f8_blocks(a.k);
    tail.n = a.n - form.wide;
    tail.w.codes = static_cast<const unsigned char*>(a.w.codes) + form.wide * a.w.stride;
    tail.w.scale += scales;
    if (gated) {
        tail.up.codes = static_cast<const unsigned char*>(a.up.codes) + form.wide * a.up.stride;
        tail.up.scale += scales;
    }
    tail.y = static_cast<unsigned char*>(a.y) + (int64_t)form.wide * f8_size(a.dtype);
    if (a.dtype == SWLM_F8_E4M3) tail.y_scale += form.wide / kF8Block * a.y_scale_stride;
    return launch_f8_few(tail, form.few, status, s);
}

}  // namespace swlm
