// Rows sorted by expert, and back at their tokens, weighted and added up.
#include <algorithm>
#include <atomic>

#include <cooperative_groups.h>

#include "f8.h"

namespace cg = cooperative_groups;

namespace swlm {
namespace {

// ---- sort --------------------------------------------------------------------------------------------------------------------
// A stable counting sort by one cluster: every warp has a run of neighbouring pairs and counts its experts; sums over warps and, through distributed
// shared memory, over the cluster's CTAs give every warp its first row of every expert; then it numbers its pairs, 32 at a time, by those before
// them of the same expert. No number depends on the order in which warps get there.
// What bounds it is latency: a few pairs take as many warps as they need (16 tokens x 8: 32 warps 5.9 us replayed, four 3.0), many a cluster of sixteen CTAs
// (131072 pairs: eight 21 us, sixteen 13.4; rows' tokens put in order in shared memory before they are stored gained nothing).
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32, kSortUnroll = 8, kSortCtas = 16;   // at most

__global__ void __launch_bounds__(kSortThreads) expert_sort_kernel(const swlm_expert_sort a) {
    extern __shared__ int counts[];        // [warps][experts]: pairs of each warp, then each warp's next row
    __shared__ int total[kExpertMax], before[kSortWarps];
    pdl_wait();
    const cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, E = a.experts, threads = blockDim.x, warps = threads >> 5;
    const int pairs = a.tokens * a.top, runs = ctas * warps, each = (pairs + 32 * runs - 1) / (32 * runs) * 32;   // (at most 2^30 + 2^14)
    const int first = (int)min((long long)(rank * warps + warp) * each, (long long)pairs), last = min(first + each, pairs);
    int* const mine = counts + warp * E;
    for (int i = tid; i < warps * E; i += threads) counts[i] = 0;
    __syncthreads();
    int e[kSortUnroll];   // choices of the pairs in question, -1 for none; where a warp has no more than these they are read once
    auto read = [&](int i0) {
#pragma unroll
        for (int u = 0; u < kSortUnroll; ++u) {
            const int i = i0 + 32 * u + lane;
            e[u] = i < last ? a.choice[i] : -1;
            if (e[u] >= E) e[u] = -1;
        }
    };
    for (int i0 = first; i0 < last; i0 += 32 * kSortUnroll) {
        read(i0);
#pragma unroll
        for (int u = 0; u < kSortUnroll; ++u)
            if (e[u] >= 0) atomicAdd(mine + e[u], 1);
    }
    __syncthreads();
    int sum = 0;   // of expert `tid`
    if (tid < E) {
#pragma unroll
        for (int w0 = 0; w0 < kSortWarps; w0 += 16) {   // pairs of the warps before each
            if (w0 >= warps) break;
            int c[16];
#pragma unroll
            for (int w = 0; w < 16; ++w) c[w] = w0 + w < warps ? counts[(w0 + w) * E + tid] : 0;
#pragma unroll
            for (int w = 0; w < 16; ++w) {
                if (w0 + w < warps) counts[(w0 + w) * E + tid] = sum;
                sum += c[w];
            }
        }
        total[tid] = sum;
    }
    cluster.sync();
    int all = 0, others = 0;
    if (tid < E) {
#pragma unroll
        for (int c = 0; c < kSortCtas; ++c) {
            const int v = c < ctas ? *cluster.map_shared_rank(total + tid, c) : 0;
            others += c < rank ? v : 0;
            all += v;
        }
    }
    auto running = [&](int v) {   // sum over the lanes up to this one
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int w = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += w;
        }
        return v;
    };
    const int scan = running(all);   // rows of the experts up to this one, the warp's first on
    if (lane == 31) before[warp] = scan;
    __syncthreads();
    const int upto = running(lane < warps ? before[lane] : 0), rows = __shfl_sync(0xffffffffu, upto, 31);
    const int base = (warp ? __shfl_sync(0xffffffffu, upto, (warp + 31) & 31) : 0) + scan - all;
    if (tid < E) {
        if (rank == 0) {
            a.offsets[tid] = base;
            if (tid == E - 1) a.offsets[E] = rows;
        }
#pragma unroll 16
        for (int w = 0; w < warps; ++w) atomicAdd(counts + w * E + tid, base + others);   // (no thread waits for what it reads)
    }
    __syncthreads();
    for (int i = rows + rank * threads + tid; i < pairs; i += ctas * threads) a.source[i] = -1;
    for (int i0 = first; i0 < last; i0 += 32 * kSortUnroll) {
        if (each > 32 * kSortUnroll) read(i0);
#pragma unroll
        for (int u = 0; u < kSortUnroll; ++u) {
            if (i0 + 32 * u >= last) break;   // (the same for the warp)
            const int i = i0 + 32 * u + lane;
            const unsigned same = __match_any_sync(0xffffffffu, e[u]);
            const int next = e[u] >= 0 ? mine[e[u]] : 0;
            __syncwarp();
            if (e[u] >= 0 && (same >> lane) == 1u) mine[e[u]] = next + __popc(same);   // (the last of them)
            __syncwarp();
            if (i < last) {
                const int row = e[u] >= 0 ? next + __popc(same & ((1u << lane) - 1u)) : -1;
                a.place[i] = row;
                if (row >= 0) a.source[row] = i / a.top;
            }
        }
    }
    cluster.sync();   // the others have read `total`
}

// ---- sum ---------------------------------------------------------------------------------------------------------------------
// A thread has eight columns of a token and runs through the token's rows in their order; the rows' values are held as they came until they are added, so that
// 128 bytes a thread are on their way at once and four CTAs fit an SM.
constexpr int kSumThreads = 256;

template <int DTYPE> struct Values8 {   // eight values as they are held
    static constexpr int WORDS = DTYPE == SWLM_F8_FP32 ? 2 : 1, SIZE = DTYPE == SWLM_F8_FP32 ? 4 : 2;
    uint4 v[WORDS];
    __device__ __forceinline__ void load(const void* p) {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) v[i] = static_cast<const uint4*>(p)[i];
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) v[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void widen(float (&x)[8]) const {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
            const unsigned w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (DTYPE == SWLM_F8_FP32) x[4 * i + j] = __uint_as_float(w[j]);
                else {
                    const float2 f = DTYPE == SWLM_F8_FP16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[j])) : make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xFFFF0000u));
                    x[2 * j] = f.x; x[2 * j + 1] = f.y;
                }
            }
        }
    }
};
template <int DTYPE> __device__ __forceinline__ float load1(const void* p, int i) {
    if (DTYPE == SWLM_F8_FP32) return static_cast<const float*>(p)[i];
    return DTYPE == SWLM_F8_FP16 ? __half2float(static_cast<const __half*>(p)[i]) : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
template <int DTYPE> __device__ __forceinline__ void store1(void* p, int i, float v) {
    if (DTYPE == SWLM_F8_FP32) static_cast<float*>(p)[i] = v;
    else if (DTYPE == SWLM_F8_FP16) static_cast<__half*>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}
template <int DTYPE> __device__ __forceinline__ void store8(void* p, const float (&x)[8]) {
    if (DTYPE == SWLM_F8_FP32) {
        static_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        static_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        unsigned w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (DTYPE == SWLM_F8_FP16) { const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]); w[i] = *reinterpret_cast<const unsigned*>(&h); }
            else { const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]); w[i] = *reinterpret_cast<const unsigned*>(&h); }
        }
        *static_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <int Y, int OUT>
__global__ void __launch_bounds__(kSumThreads, 4) expert_sum_kernel(const swlm_expert_sum a) {
    constexpr int YSIZE = Values8<Y>::SIZE, SIZE = Values8<OUT>::SIZE, UNROLL = 8 / Values8<Y>::WORDS;
    pdl_wait();
    const unsigned chunks = (a.width + 7) / 8;
    const long long at = (long long)blockIdx.x * kSumThreads + threadIdx.x;
    const long long t = at / chunks;
    if (t >= a.tokens) return;
    const int col = (int)(at - t * chunks) * 8, rest = a.width - col;
    const int* place = a.place + t * a.top;
    const float* weight = a.weight + t * a.top;
    const unsigned char* y = static_cast<const unsigned char*>(a.y) + (long long)col * YSIZE;
    unsigned char* out = static_cast<unsigned char*>(a.out) + (t * a.out_stride + col) * SIZE;
    const unsigned char* add = a.add ? static_cast<const unsigned char*>(a.add) + (t * a.add_stride + col) * SIZE : nullptr;
    if (rest < 8) {   // a token's last columns, whose number is no multiple of eight
        for (int e = 0; e < rest; ++e) {
            float sum = 0.f;
            for (int j = 0; j < a.top; ++j)
                if (place[j] >= 0 && place[j] < a.y_rows) sum = fmaf(weight[j], load1<Y>(y + (long long)place[j] * a.y_stride * YSIZE, e), sum);
            store1<OUT>(out, e, add ? sum + load1<OUT>(add, e) : sum);
        }
        return;
    }
    Values8<OUT> base;
    if (add) base.load(add);
    float sum[8] = {};
    for (int j0 = 0; j0 < a.top; j0 += UNROLL) {
        Values8<Y> held[UNROLL];
        float w[UNROLL];
#pragma unroll
        for (int j = 0; j < UNROLL; ++j) {
            const int row = j0 + j < a.top ? place[j0 + j] : -1;
            const bool has = row >= 0 && row < a.y_rows;
            w[j] = has ? weight[j0 + j] : 0.f;
            if (has) held[j].load(y + (long long)row * a.y_stride * YSIZE);
            else held[j].zero();
        }
#pragma unroll
        for (int j = 0; j < UNROLL; ++j) {
            float x[8];
            held[j].widen(x);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] = fmaf(w[j], x[e], sum[e]);
        }
    }
    if (add) {
        float x[8];
        base.widen(x);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += x[e];
    }
    store8<OUT>(out, sum);
}

template <int Y> void (*sum_kernel(int dtype))(swlm_expert_sum) {
    return dtype == SWLM_F8_FP32 ? expert_sum_kernel<Y, SWLM_F8_FP32> : dtype == SWLM_F8_FP16 ? expert_sum_kernel<Y, SWLM_F8_FP16> : expert_sum_kernel<Y, SWLM_F8_BF16>;
}

}  // namespace

static std::atomic<int> g_sort_ctas{kSortCtas};   // most CTAs of a cluster that all devices in use take

int expert_rows_init() {
    SWLM_CUDA(cudaFuncSetAttribute(expert_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortWarps * kExpertMax * 4));
    SWLM_CUDA(cudaFuncSetAttribute(expert_sort_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    // clusters of sixteen are not promised: a device that takes none does with eight
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kSortCtas; attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(kSortCtas); cfg.blockDim = dim3(kSortThreads); cfg.dynamicSmemBytes = kSortWarps * kExpertMax * 4; cfg.attrs = attr; cfg.numAttrs = 1;
    int fit = 0;
    if (cudaOccupancyMaxActiveClusters(&fit, expert_sort_kernel, &cfg) != cudaSuccess) { cudaGetLastError(); fit = 0; }
    if (fit < 1) g_sort_ctas.store(8, std::memory_order_relaxed);
    return SWLM_OK;
}

int launch_expert_sort(const swlm_expert_sort& a, cudaStream_t s) {
    const long long pairs = (long long)a.tokens * a.top;
    int ctas = 1;
    while (ctas < g_sort_ctas.load(std::memory_order_relaxed) && pairs > (long long)ctas * 2 * kSortThreads) ctas *= 2;
    // a thread per expert, and as many warps as have pairs
    const int threads = (int)std::min<long long>(kSortThreads, std::max<long long>((a.experts + 31) / 32 * 32, (pairs + 31) / 32 * 32));
    const cudaError_t e = launch_clusters(expert_sort_kernel, ctas, dim3(ctas), dim3(threads), (size_t)threads / 32 * a.experts * 4, s, a);
    return e == cudaSuccess ? SWLM_OK : cuda_fail(e, "expert sort launch");
}

int launch_expert_sum(const swlm_expert_sum& a, cudaStream_t s) {
    const long long threads = (long long)a.tokens * ((a.width + 7) / 8), ctas = (threads + kSumThreads - 1) / kSumThreads;
    if (ctas > 0x7FFFFFFFll) { set_error("f8: too many tokens for a width of %d", a.width); return SWLM_ERR_INVALID; }
    void (*kernel)(swlm_expert_sum) = a.y_dtype == SWLM_F8_FP32 ? sum_kernel<SWLM_F8_FP32>(a.dtype) : a.y_dtype == SWLM_F8_FP16 ? sum_kernel<SWLM_F8_FP16>(a.dtype) : sum_kernel<SWLM_F8_BF16>(a.dtype);
    const cudaError_t e = launch_k(kernel, dim3((unsigned)ctas), dim3(kSumThreads), 0, s, a);
    return e == cudaSuccess ? SWLM_OK : cuda_fail(e, "expert sum launch");
}

}  // namespace swlm
