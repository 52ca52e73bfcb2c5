// Attention over a cache of 8-bit codes with one scale per block of tokens and head.
//
//   s_ij = scale * ks[j / T] * (q_i . ck_j),  p = softmax over the slots that query i attends,  out_i = sum_j p_ij vs[j / T] cv_j
//
// Codes are exact as fp16 numbers, and so are bf16 and fp16 queries after a shift of the row's exponent that brings its
// largest value to 2^12, but for values 2^-26 and less of the largest. So q . ck is an fp16 product with fp32 sums on the tensor cores, and
// a step of 16 tokens, which never crosses a block, takes its scale as one number behind it.
//
// Rows: the queries of a step times the heads of a group, 8 to a tile. A CTA has one tile (or two) and a run of slots of one (sequence,
// KV head) after the other, the same number of slots for every CTA whatever the lengths are; its four warps take steps of 32 tokens in turn,
// each over a ring of its own that cp.async fills. Scores come as S^T = K Q^T (16 tokens x 8 rows, so that a decode step's four or eight
// rows fill the tile), probabilities are transposed in registers (movmatrix) and meet the values as O^T = V^T P^T. The reference
// maximum of a row moves only when it would grow by more than 2^8. Probabilities are rounded to fp16 as p 2^7 vs / vr, vr the largest value
// scale so far: off by 2^-11 of themselves where p vs / vr >= 2^-21, below that by 2^-32 of vr. bf16 results do not show it. fp16 results, which
// have as many bits, do: unless the caller chooses, what the rounding has left follows there as a second product (2^-22 of themselves where
// p vs / vr >= 2^-10). Error against 64 bits, 41 ragged sequences of 4091 tokens in fp16: 2.7e-4 with one product, 2.1e-4 with two, of which rounding the
// result is 2.1e-4; 27.5 and 28.8 us, five tokens of six sequences over 16384 48.0 and 54.0. Partial results of a tile
// are joined by a second launch, which also adds the weights, or by the cluster of CTAs that has all of a tile's slots.
//
// What bounds it: memory, and some ten us of start, merge and the second launch. 8 x 8192 tokens, 32 / 8 heads of 128, int8: 33.5 us for 134 MB (0.61
// of the measured copy; 26 us without merge and second launch); 1 x 131072: 53.6 us (0.77). Without the products of either kind a pass takes 2 to 5 us
// less. The next launch waits for this one's end instead of being let in early: its CTAs on the SMs cost 8 of 49 us (8 x 8192 with weights).
#include <cooperative_groups.h>

#include <algorithm>
#include <climits>

#include "kv8_device.cuh"

namespace swlm {
using namespace kv8;
namespace cg = cooperative_groups;
namespace {

constexpr int kClusterCtas = 8;                 // of a cluster, at most
constexpr int kStreamBatch = 512;               // sequences whose units a CTA adds up
constexpr int kSaveRows = 64;                   // up to so many rows of a KV head the scores are kept for the weights, beyond they are worked out again

__device__ __forceinline__ unsigned smem_addr(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(unsigned dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copy4(unsigned dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait_groups() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds128(unsigned a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds64(unsigned a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void mma(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned transpose8x8(unsigned v) {
    unsigned r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <int HD> __host__ __device__ constexpr int stages() { return HD == 128 ? 2 : 3; }
template <int HD> __host__ __device__ constexpr int rows_ctas() { return HD == 128 ? 3 : 4; }   // CTAs of one tile per SM
template <int HD> __host__ __device__ constexpr int stage_bytes() { return 2 * kStep * HD + 16; }   // keys, values, (key, value) scale of either tile
template <int HD> __host__ __device__ constexpr size_t rows_smem() { return (size_t)kWarps * stages<HD>() * stage_bytes<HD>(); }

// Byte of 16-byte piece c of token r in a step's keys or values. Pieces lie so that the eight lanes of a phase meet different banks: keys are read
// with the token in the lane's upper bits (two tokens x four pieces), values with it in the lower ones (tokens 0, 2, 4, 6 x two pieces).
template <int HD> __device__ __forceinline__ int key_at(int r, int c) { return HD == 128 ? r * 128 + ((c ^ ((r & 1) << 2)) << 4) : r * 64 + (c << 4); }
template <int HD> __device__ __forceinline__ int value_at(int r, int c) {
    if (HD == 128) return r * 128 + ((c ^ (((r >> 1) & 3) << 1)) << 4);
    return (r >> 1) * 128 + (((((r & 1) << 2) | c) ^ (((r >> 1) & 3) << 1)) << 4);
}

// One lane's share of row `row` (its 16-byte pieces t, t + 4 of codes: 16 values each) as B fragments, brought to 2^12.
template <int HD>
__device__ __forceinline__ void load_query(const unsigned short* src, bool valid, bool f16, int t, unsigned (&frag)[HD / 16][2], float& down) {
    float x[HD / 4], top = 0.f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < HD / 64; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            float v[8] = {};
            if (valid) widen(*reinterpret_cast<const uint4*>(src + (t + 4 * i) * 16 + half * 8), f16, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[i * 16 + half * 8 + e] = v[e];
                top = fmaxf(top, fabsf(v[e]));
                bad = bad || v[e] != v[e];
            }
        }
    if (bad) top = INFINITY;
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    float up;
    row_shift(top, up, down);
#pragma unroll
    for (int k = 0; k < HD / 16; ++k) {
        frag[k][0] = pack_half(x[4 * k] * up, x[4 * k + 1] * up);
        frag[k][1] = pack_half(x[4 * k + 2] * up, x[4 * k + 3] * up);
    }
}

// Parts first, first + step, ... of a row's: their maxima and sums ml, pitch rows apart, and four values of each result. Eight are loaded at once.
__device__ __forceinline__ void join_parts(const float* ml, const float* po, int pitch, int dim, int parts, int first, int step, float& m, float& l, float4& o) {
    constexpr int AHEAD = 8;
    m = -INFINITY;
    l = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = first; s0 < parts; s0 += AHEAD * step) {
        float2 x[AHEAD];
        float4 v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const size_t s = min(s0 + i * step, parts - 1);
            x[i] = __ldcg(reinterpret_cast<const float2*>(ml + s * pitch * 2));
            v[i] = __ldcg(reinterpret_cast<const float4*>(po + s * pitch * dim));
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) top = fmaxf(top, x[i].x);   // (the last part may come several times)
        const float corr = m == -INFINITY ? 1.f : exp2_of(m - top);   // (no maximum so far: zeros, or NaN)
        o.x *= corr; o.y *= corr; o.z *= corr; o.w *= corr; l *= corr;
        m = top;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const float f = s0 + i * step >= parts ? 0.f : x[i].x == -INFINITY ? 1.f : exp2_of(x[i].x - m);   // (a part without slots has zeros, or NaN)
            if (f == 0.f) continue;
            l += f * x[i].y;
            o.x += f * v[i].x; o.y += f * v[i].y; o.z += f * v[i].z; o.w += f * v[i].w;
        }
    }
}

// Four values of a row's result over the CTAs of a cluster, and the row's sum.
__device__ __forceinline__ float4 join_cluster(const cg::cluster_group& cluster, int ctas, float2* ml, float* out, float& l) {
    float2 x[kClusterCtas];
    float4 v[kClusterCtas];
    float m = -INFINITY;
#pragma unroll
    for (int s = 0; s < kClusterCtas; ++s)
        if (s < ctas) {
            x[s] = *cluster.map_shared_rank(ml, s);
            v[s] = *cluster.map_shared_rank(reinterpret_cast<float4*>(out), s);
        }
#pragma unroll
    for (int s = 0; s < kClusterCtas; ++s)
        if (s < ctas) m = fmaxf(m, x[s].x);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    l = 0.f;
#pragma unroll
    for (int s = 0; s < kClusterCtas; ++s)
        if (s < ctas) {
            const float f = x[s].x == -INFINITY ? 1.f : exp2_of(x[s].x - m);   // (a part without slots has zeros, or NaN)
            l += f * x[s].y;
            o.x += f * v[s].x; o.y += f * v[s].y; o.z += f * v[s].z; o.w += f * v[s].w;
        }
    return o;
}

// TWO: probabilities meet the values as two fp16 numbers.
template <int HD, int CODE, int NT, bool SAVE, bool TWO>
__global__ void __launch_bounds__(kThreads, NT == 1 ? rows_ctas<HD>() : 2) kv8_rows_kernel(const swlm_kv8_cache c, const swlm_kv8_attend a, const RowsPlan p) {
    constexpr int KS = HD / 16, MT = HD / 16, NS = stages<HD>(), SB = stage_bytes<HD>(), TR = 8 * NT;
    extern __shared__ __align__(16) unsigned char sm[];
    __shared__ float warp_m[kWarps][TR], warp_l[kWarps][TR];
    __shared__ float2 part_ml[TR];   // of this CTA, for the others of its cluster
    __shared__ float row_m[TR], row_inv[TR];
    __shared__ int scan[kWarps + 1];
    int4* const info = reinterpret_cast<int4*>(sm + rows_smem<HD>());   // [batch + 1]: units before the sequence, its length, count, first row
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int G = a.heads / c.kv_heads, span = min(a.max_len, c.capacity);
    const bool f16 = a.dtype == SWLM_KV8_FP16;
    const int block_shift = 31 - __clz(c.block);

    // ---- this CTA's units ----
    int u = 0, u_end = 1, b = 0;
    if (p.stream) {
        int before = 0;   // units of the sequences before the ones of this turn
        for (int b0 = 0; b0 < c.batch; b0 += kThreads) {
            int mine = 0;
            Kv8Part q{};
            if (b0 + tid < c.batch) {
                q = kv8_part(b0 + tid, a.lengths, a.counts, a.starts, a.refused, a.n, a.rows);
                if (q.count) mine = sequence_units(q, span) * sequence_tiles(q, G, TR) * c.kv_heads;
            }
            int sum = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += v;
            }
            if (lane == 31) scan[warp] = sum;
            __syncthreads();
            int all = 0;
            for (int w = 0; w < kWarps; ++w) {
                if (w == warp) sum += all;
                all += scan[w];
            }
            if (b0 + tid < c.batch) info[b0 + tid] = make_int4(before + sum - mine, q.len, q.count, q.start);
            before += all;
            if (b0 + kThreads < c.batch) __syncthreads();
        }
        const int total = before;
        if (tid == 0) info[c.batch].x = total;
        __syncthreads();
        if (blockIdx.x == 0 && p.table)   // for the launch that joins the parts
            for (int i = tid; i <= c.batch; i += kThreads) p.table[i] = info[i].x;
        const Shares shares(total, (int)gridDim.x);
        if ((int)blockIdx.x >= shares.ctas) return;
        u = shares.first((int)blockIdx.x);
        u_end = shares.first((int)blockIdx.x + 1);
    } else {
        b = blockIdx.z;
    }

    // what lies where: offsets of this lane within a step's stage. Copies: piece lane + 32 i, that is row lane / (HD / 16) + i * (512 / HD)
    const int cp_r = lane / (HD / 16), cp_q = lane % (HD / 16);
    const unsigned ring = smem_addr(sm) + warp * NS * SB;

    while (u < u_end) {
        // ---- the next (sequence, KV head, tile) and the slots of it that this CTA has ----
        int h, tile, unit0, unit1;
        Kv8Part part;
        if (p.stream) {
            for (int hi = c.batch - 1; b < hi;) {   // the sequence that has unit u
                const int mid = (b + hi) >> 1;
                if (info[mid + 1].x <= u) b = mid + 1;
                else hi = mid;
            }
            const int4 q = info[b];
            part = {q.y, q.z, q.w, true};
            const int per = sequence_units(part, span), tiles = sequence_tiles(part, G, TR), rem = u - q.x, pair = rem / per;
            h = pair / tiles;
            tile = pair - h * tiles;
            unit0 = rem - pair * per;
            unit1 = min(per, unit0 + u_end - u);
            u += unit1 - unit0;
        } else {
            part = kv8_part(b, a.lengths, a.counts, a.starts, a.refused, a.n, a.rows);
            // a cluster of CTAs, or one, has all slots of a tile: equal shares of its units
            const int units = sequence_units(part, span), rank = (int)blockIdx.x % p.cluster;
            h = blockIdx.y; tile = (int)blockIdx.x / p.cluster;
            unit0 = units * rank / p.cluster;
            unit1 = units * (rank + 1) / p.cluster;
            u = u_end;
            if (tile * TR >= part.count * G) break;
        }
        const bool whole = unit0 == 0 && unit1 == sequence_units(part, span);   // this CTA has all of it
        const int rows = part.count * G, row0 = tile * TR;
        const int end = visible(part, min((row0 + TR - 1) / G, part.count - 1), span);   // of the tile's last query: it sees most
        const int from = unit0 * kUnit, to = min(unit1 * kUnit, end);
        const size_t head = (size_t)b * c.kv_heads + h;

        // ring of this warp: its step number i covers the 32 slots from `first` + i * kUnit on. Whole tiles of 16 are read: they lie within the
        // capacity, a multiple of 16; what is beyond a row's last slot is masked.
        const int first = from + warp * kStep, steps = first < to ? (to - first + kUnit - 1) / kUnit : 0;
        const unsigned char* kp = static_cast<const unsigned char*>(c.k) + (head * c.capacity + first) * HD + lane * 16;
        const unsigned char* vp = static_cast<const unsigned char*>(c.v) + (head * c.capacity + first) * HD + lane * 16;
        const float* sp = (lane & 1 ? c.v_scale : c.k_scale) + head * (c.capacity >> block_shift);
        int asked = 0;
        unsigned ask = ring;
        auto request = [&]() {
            if (asked < steps) {
                const int base = first + asked * kUnit;
                const bool both = base + 16 < to;   // (else the second tile's memory may not be there)
#pragma unroll
                for (int i = 0; i < kStep * HD / 512; ++i) {
                    if (i < 16 * HD / 512 || both) {
                        copy16(ask + key_at<HD>(cp_r + i * (512 / HD), cp_q), kp + i * 512);
                        copy16(ask + kStep * HD + value_at<HD>(cp_r + i * (512 / HD), cp_q), vp + i * 512);
                    }
                }
                if (lane < (both ? 4 : 2)) copy4(ask + 2 * kStep * HD + lane * 4, sp + ((base + (lane >> 1) * 16) >> block_shift));
                kp += kUnit * HD;
                vp += kUnit * HD;
            }
            commit();
            ++asked;
            ask = ask == ring + (NS - 1) * SB ? ring : ask + SB;
        };
#pragma unroll
        for (int i = 0; i < NS - 1; ++i) request();

        unsigned qf[NT][KS][2];
        float factor[NT][2];     // of columns 2 t and 2 t + 1 (rows of the tile): score in log2 per unit of the product
        int limit[NT][2], all_see = 0x7FFFFFFF;   // the tile's rows all attend the slots below
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = row0 + nt * 8 + g, i = min(r, rows - 1) / G;
            float down;
            load_query<HD>(static_cast<const unsigned short*>(a.q) + (int64_t)(part.start + i) * a.q_stride + (size_t)(h * G + min(r, rows - 1) - i * G) * HD, r < rows, f16, t,
                           qf[nt], down);
            down *= a.scale * kLog2e;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                factor[nt][e] = __shfl_sync(0xffffffffu, down, (2 * t + e) * 4);
                // (rows behind the last one attend what the last one does: their results are not stored)
                limit[nt][e] = visible(part, min(row0 + nt * 8 + 2 * t + e, rows - 1) / G, span);
                all_see = min(all_see, limit[nt][e]);
            }
        }
        all_see = min(all_see, __shfl_xor_sync(0xffffffffu, all_see, 1));
        all_see = min(all_see, __shfl_xor_sync(0xffffffffu, all_see, 2));
        float acc[NT][MT][4], m_ref[NT][2], top_ok[NT][2], l_run[NT][2], v_ref = kValueRef, v_inv = kValueUnit / kValueRef;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int j = 0; j < MT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[nt][j][e] = 0.f;
#pragma unroll
            for (int e = 0; e < 2; ++e) { m_ref[nt][e] = 0.f; top_ok[nt][e] = -INFINITY; l_run[nt][e] = 0.f; }
        }
        float* save = SAVE ? p.scores + (head * p.span + first + g) * p.pitch + row0 + 2 * t : nullptr;
        unsigned at = ring;
        const int k_off = key_at<HD>(g, t), v_off = kStep * HD + (HD == 128 ? value_at<HD>(2 * t, g) : value_at<HD>(2 * t, g >> 1) + (g & 1) * 8);
        for (int i = 0, base = first; i < steps; ++i, base += kUnit) {
            wait_groups<NS - 2>();
            __syncwarp();          // this step's copies of all lanes are there, and all lanes have read the step before
            request();
            // ---- scores ----
            float s[kSub][NT][4] = {};
#pragma unroll
            for (int sub = 0; sub < kSub; ++sub)
#pragma unroll
                for (int q = 0; q < HD / 64; ++q) {
                    const uint4 lo = lds128(at + (k_off ^ (q << 6)) + sub * 16 * HD), hi = lds128(at + (k_off ^ (q << 6)) + sub * 16 * HD + 8 * HD);
                    const unsigned lw[4] = {lo.x, lo.y, lo.z, lo.w}, hw[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const unsigned x = prepared<CODE>(lw[w]), y = prepared<CODE>(hw[w]);
                        const unsigned a0 = pair_of<CODE, 0>(x), a1 = pair_of<CODE, 0>(y), a2 = pair_of<CODE, 1>(x), a3 = pair_of<CODE, 1>(y);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma(s[sub][nt], a0, a1, a2, a3, qf[nt][q * 4 + w][0], qf[nt][q * 4 + w][1]);
                    }
                }
            const uint4 sc = lds128(at + 2 * kStep * HD);
            // values: this lane has HD / 8 dimensions of tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of either tile. The first tile's are on their way now
            unsigned vw[4][HD / 32];
            auto load_values = [&](int sub) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (HD == 128) {   // (rows 2 t + 1 and 8 on share the swizzle)
                        const uint4 v = lds128(at + v_off + sub * 2048 + (k & 1) * 128 + (k >> 1) * 1024);
                        vw[k][0] = v.x; vw[k][1] = v.y; vw[k][HD / 32 - 2] = v.z; vw[k][HD / 32 - 1] = v.w;
                    } else {           // (the odd token of a pair lies four pieces further on in their common line)
                        const uint2 v = lds64(at + (v_off ^ ((k & 1) << 6)) + sub * 1024 + (k >> 1) * 512);
                        vw[k][0] = v.x; vw[k][1] = v.y;
                    }
                }
            };
            load_values(0);
            float k_scale[kSub] = {__uint_as_float(sc.x), __uint_as_float(sc.z)}, v_scale[kSub] = {__uint_as_float(sc.y), __uint_as_float(sc.w)};
            const bool masked = base + kStep > all_see;
            if (masked && base + 16 >= to) k_scale[1] = v_scale[1] = 0.f;   // (of a block that may hold nothing yet)
            bool moves = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int sub = 0; sub < kSub; ++sub) {
                    const float f0 = factor[nt][0] * k_scale[sub], f1 = factor[nt][1] * k_scale[sub];
                    s[sub][nt][0] *= f0; s[sub][nt][1] *= f1; s[sub][nt][2] *= f0; s[sub][nt][3] *= f1;
                    if (masked)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (base + sub * 16 + g + 8 * (e >> 1) >= limit[nt][e & 1]) s[sub][nt][e] = -INFINITY;
                }
                moves = moves || fmaxf(fmaxf(s[0][nt][0], s[0][nt][2]), fmaxf(s[1][nt][0], s[1][nt][2])) > top_ok[nt][0] ||
                        fmaxf(fmaxf(s[0][nt][1], s[0][nt][3]), fmaxf(s[1][nt][1], s[1][nt][3])) > top_ok[nt][1];
            }
            if (SAVE) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    if (row0 + nt * 8 + 2 * t < p.pitch) {   // (the pitch is even)
#pragma unroll
                        for (int sub = 0; sub < kSub; ++sub) {
                            *reinterpret_cast<float2*>(save + nt * 8 + sub * 16 * p.pitch) = make_float2(s[sub][nt][0], s[sub][nt][1]);
                            *reinterpret_cast<float2*>(save + nt * 8 + (sub * 16 + 8) * p.pitch) = make_float2(s[sub][nt][2], s[sub][nt][3]);
                        }
                    }
                save += kUnit * p.pitch;
            }
            // ---- softmax ----
            if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = fmaxf(fmaxf(s[0][nt][e], s[0][nt][e + 2]), fmaxf(s[1][nt][e], s[1][nt][e + 2]));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        if (top > top_ok[nt][e]) {
                            const float corr = top_ok[nt][e] == -INFINITY ? 0.f : exp2_of(m_ref[nt][e] - top);
                            m_ref[nt][e] = top;
                            top_ok[nt][e] = top + kSlack;
                            l_run[nt][e] *= corr;
#pragma unroll
                            for (int j = 0; j < MT; ++j) { acc[nt][j][e] *= corr; acc[nt][j][e + 2] *= corr; }
                        }
                    }
            }
            const float v_top = fmaxf(v_scale[0], v_scale[1]);
            if (v_top > v_ref) {
                const float corr = v_ref / v_top;
                v_ref = v_top;
                v_inv = kValueUnit / v_top;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < MT; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[nt][j][e] *= corr;
            }
            unsigned pf[kSub][NT][2], pr[kSub][NT][2];   // (pr: what rounding has left of them)
#pragma unroll
            for (int sub = 0; sub < kSub; ++sub) {
                const float unit = v_scale[sub] * v_inv;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float pr = exp2_of(s[sub][nt][e] - m_ref[nt][e & 1]);
                        l_run[nt][e & 1] += pr;
                        w[e] = pr * unit;
                        if (masked && s[sub][nt][e] == -INFINITY) w[e] = 0.f;   // (a slot that the row does not attend may lie in a block that is NaN)
                    }
                    const unsigned p0 = pack_half(w[0], w[1]), p1 = pack_half(w[2], w[3]);
                    pf[sub][nt][0] = transpose8x8(p0);
                    pf[sub][nt][1] = transpose8x8(p1);
                    if (TWO) {
                        pr[sub][nt][0] = transpose8x8(pack_rest(w[0], w[1], p0));
                        pr[sub][nt][1] = transpose8x8(pack_rest(w[2], w[3], p1));
                    }
                }
            }
            // ---- values ----
#pragma unroll
            for (int sub = 0; sub < kSub; ++sub) {
                if (sub) load_values(sub);
                // what lies behind the last token may be an e4m3 NaN, which the weight 0 would not hide
                if (CODE == SWLM_KV8_E4M3 && masked)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (base + sub * 16 + 2 * t + (k & 1) + 8 * (k >> 1) >= end)
#pragma unroll
                            for (int w = 0; w < HD / 32; ++w) vw[k][w] = 0;
#pragma unroll
                for (int w = 0; w < HD / 32; ++w) {
                    const unsigned v0 = prepared<CODE>(vw[0][w]), v1 = prepared<CODE>(vw[1][w]), v2 = prepared<CODE>(vw[2][w]), v3 = prepared<CODE>(vw[3][w]);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {   // dimensions 4 w + 2 half and the next one
                        const unsigned lo = __byte_perm(v0, v1, half ? 0x7362 : 0x5140), hi = __byte_perm(v2, v3, half ? 0x7362 : 0x5140);
                        const unsigned a0 = pair_of<CODE, 0>(lo), a1 = pair_of<CODE, 1>(lo), a2 = pair_of<CODE, 0>(hi), a3 = pair_of<CODE, 1>(hi);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma(acc[nt][2 * w + half], a0, a1, a2, a3, pf[sub][nt][0], pf[sub][nt][1]);
                            if (TWO) mma(acc[nt][2 * w + half], a0, a1, a2, a3, pr[sub][nt][0], pr[sub][nt][1]);
                        }
                    }
                }
            }
            at = at == ring + (NS - 1) * SB ? ring : at + SB;
        }

        // ---- the warps' results together ----
        __syncthreads();   // every warp is done with its ring (only empty groups are outstanding)
        float* const outs = reinterpret_cast<float*>(sm);   // [warp][TR][HD]
        const float unit = v_ref * (1.f / kValueUnit);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float l = l_run[nt][e];
                l += __shfl_xor_sync(0xffffffffu, l, 4);
                l += __shfl_xor_sync(0xffffffffu, l, 8);
                l += __shfl_xor_sync(0xffffffffu, l, 16);
                if (g == 0) {
                    warp_m[warp][nt * 8 + 2 * t + e] = top_ok[nt][e] == -INFINITY ? -INFINITY : m_ref[nt][e];
                    warp_l[warp][nt * 8 + 2 * t + e] = l;
                }
            }
#pragma unroll
            for (int j = 0; j < MT; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e)   // row 2 t + e, dimensions g * HD / 8 + 2 j and the next one
                    *reinterpret_cast<float2*>(outs + (size_t)(warp * TR + nt * 8 + 2 * t + e) * HD + g * (HD / 8) + 2 * j) =
                        make_float2(acc[nt][j][e] * unit, acc[nt][j][e + 2] * unit);
        }
        __syncthreads();
        // parts of a (sequence, KV head, tile): its number plus the CTA's, which both grow along the stream
        const size_t slot = (size_t)(head * p.row_tiles + tile) + (p.stream ? blockIdx.x : 0);
        for (int item = tid; item < TR * (HD / 4); item += kThreads) {
            const int r = item / (HD / 4), d = item % (HD / 4) * 4, row = row0 + r;
            if (row >= rows) continue;
            float m = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) m = fmaxf(m, warp_m[w][r]);
            float l = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                // (a row whose scores are all NaN has no maximum and a sum that is NaN)
                const float f = warp_m[w][r] == -INFINITY ? (warp_l[w][r] == 0.f ? 0.f : 1.f) : exp2_of(warp_m[w][r] - m);
                const float4 v = *reinterpret_cast<const float4*>(outs + (size_t)(w * TR + r) * HD + d);
                l += f * warp_l[w][r];
                o.x += f * v.x; o.y += f * v.y; o.z += f * v.z; o.w += f * v.w;
            }
            if (p.cluster > 1) {
                if (d == 0) part_ml[r] = make_float2(m, l);
                *reinterpret_cast<float4*>(outs + (size_t)r * HD + d) = o;   // (the first warp's, which nobody else reads)
                continue;
            }
            if (d == 0 && (SAVE || !whole)) *reinterpret_cast<float2*>(p.part_ml + (slot * TR + r) * 2) = make_float2(m, l);
            if (!whole) {
                *reinterpret_cast<float4*>(p.part_o + (slot * TR + r) * HD + d) = o;
            } else {
                const int i = row / G;
                store_out(static_cast<unsigned short*>(a.out) + (int64_t)(part.start + i) * a.out_stride + (size_t)(h * G + row - i * G) * HD + d, o, l, f16);
            }
        }
        if (p.cluster > 1) {
            // ---- the cluster's results together ----
            const cg::cluster_group cluster = cg::this_cluster();
            const int rank = (int)cluster.block_rank();
            cluster.sync();
            for (int item = rank * kThreads + tid; item < TR * (HD / 4); item += p.cluster * kThreads) {
                const int r = item / (HD / 4), d = item % (HD / 4) * 4, row = row0 + r;
                if (row >= rows) continue;
                float l;
                const float4 o = join_cluster(cluster, p.cluster, part_ml + r, outs + (size_t)r * HD + d, l);
                const int i = row / G;
                store_out(static_cast<unsigned short*>(a.out) + (int64_t)(part.start + i) * a.out_stride + (size_t)(h * G + row - i * G) * HD + d, o, l, f16);
            }
            if (SAVE && tid < TR) {
                float m = -INFINITY, l = 0.f;
                for (int s = 0; s < p.cluster; ++s) m = fmaxf(m, cluster.map_shared_rank(part_ml, s)[tid].x);
                for (int s = 0; s < p.cluster; ++s) {
                    const float2 v = cluster.map_shared_rank(part_ml, s)[tid];
                    l += v.x == -INFINITY ? v.y : exp2_of(v.x - m) * v.y;
                }
                row_m[tid] = m == -INFINITY ? 0.f : m;
                row_inv[tid] = l == 0.f ? 0.f : 1.f / l;
            }
            cluster.barrier_arrive();
            if (SAVE) {   // this CTA's slots of all rows: there is one tile
                __syncthreads();
                float* const w = c.weight + head * c.capacity;
                for (int slot = from + tid; slot < to; slot += kThreads) {
                    const float* const sc = p.scores + (head * p.span + slot) * p.pitch;
                    float sum = 0.f;
                    for (int r = 0; r < rows; r += 2) {
                        const float2 v = *reinterpret_cast<const float2*>(sc + r);
                        if (slot < visible(part, r / G, span)) sum += exp2_of(v.x - row_m[r]) * row_inv[r];
                        if (r + 1 < rows && slot < visible(part, (r + 1) / G, span)) sum += exp2_of(v.y - row_m[r + 1]) * row_inv[r + 1];
                    }
                    w[slot] += sum;
                }
            }
            cluster.barrier_wait();   // no CTA leaves while others read its results
            break;
        }
        __syncthreads();   // the next one's copies take the results' place
    }
}

// Maximum and sum of a row over its parts, `pitch` floats apart, by a group of LANES lanes; all of them get both.
template <int LANES>
__device__ __forceinline__ void row_total(const float* ml, int pitch, int parts, int lane, float& m, float& l) {
    m = -INFINITY;
    for (int s = lane; s < parts; s += LANES) m = fmaxf(m, ml[(size_t)s * pitch]);
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    l = 0.f;
    for (int s = lane; s < parts; s += LANES) {
        const float x = ml[(size_t)s * pitch], v = ml[(size_t)s * pitch + 1];
        l += x == -INFINITY ? v : exp2_of(x - m) * v;   // (v is 0, or NaN where a part's scores are all NaN)
    }
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
}

constexpr int kJoinThreads = 256, kJoinTurns = 4, kJoinSlots = kJoinThreads * kJoinTurns;

// CTAs 0 .. join - 1 along x join the parts of the rows that have several, the others add the kept scores' weights, kJoinSlots slots each (or a half or a quarter).
template <int HD>
__global__ void __launch_bounds__(kJoinThreads) kv8_join_kernel(const swlm_kv8_cache c, const swlm_kv8_attend a, const RowsPlan p, const int join) {
    constexpr int LANES = HD / 4, PER = kJoinThreads / LANES;   // lanes of a row, rows of a CTA
    __shared__ float row_m[kSaveRows], row_inv[kSaveRows];
    __shared__ int row_limit[kSaveRows];
    __shared__ float group_m[PER], group_l[PER];
    __shared__ float4 group_o[kJoinThreads];
    pdl_wait();
    const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x, G = a.heads / c.kv_heads, TR = 8 * p.tiles;
    const Kv8Part part = kv8_part(b, a.lengths, a.counts, a.starts, a.refused, a.n, a.rows);
    const int rows = part.count * G, span = min(a.max_len, c.capacity);
    if (rows == 0) return;
    const size_t head = (size_t)b * c.kv_heads + h;
    if ((int)blockIdx.x < join) {
        // p.join_groups groups of lanes take every so many-th part of a row, the first of them puts their results together
        const int group = tid / LANES, lane = tid % LANES, d = lane * 4, sub = group % p.join_groups;
        const int row = (int)blockIdx.x * (PER / p.join_groups) + group / p.join_groups;
        const int tile = min(row, rows - 1) / TR, r = min(row, rows - 1) - tile * TR;
        const Parts parts = parts_of(p, part, b, c.batch, head, h, tile, span, G);
        const bool on = row < rows && parts.count > 1;
        float m = -INFINITY, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        if (on) join_parts(p.part_ml + (parts.slot * TR + r) * 2, p.part_o + (parts.slot * TR + r) * HD + d, TR, HD, parts.count, sub, p.join_groups, m, l, o);
        if (p.join_groups > 1) {
            if (lane == 0) { group_m[group] = m; group_l[group] = l; }
            group_o[tid] = o;
            __syncthreads();
            if (sub) return;
            float top = m;
            for (int i = 1; i < p.join_groups; ++i) top = fmaxf(top, group_m[group + i]);
            float sum = 0.f;
            float4 all = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int i = 0; i < p.join_groups; ++i) {
                const float x = group_m[group + i], f = x == -INFINITY ? 1.f : exp2_of(x - top);
                const float4 v = group_o[tid + i * LANES];
                sum += f * group_l[group + i];
                all.x += f * v.x; all.y += f * v.y; all.z += f * v.z; all.w += f * v.w;
            }
            m = top;
            l = sum;
            o = all;
        }
        if (!on) return;
        if (p.q_shift && lane == 0) p.q_shift[head * p.row_tiles * TR + row] = row_shift_of(m, l);
        const int i = row / G;
        store_out(static_cast<unsigned short*>(a.out) + (int64_t)(part.start + i) * a.out_stride + (size_t)(h * G + row - i * G) * HD + d, o, l, a.dtype == SWLM_KV8_FP16);
        return;
    }
    // the scores of this thread's slots and what they had so far are on their way while the rows' totals are worked out
    const int lanes = p.join_lanes, sub = tid & ((1 << lanes) - 1), turn = kJoinThreads >> lanes;
    const int end = visible(part, part.count - 1, span), base = ((int)blockIdx.x - join) * (kJoinSlots >> lanes), slot0 = base + (tid >> lanes);
    if (base >= end) return;
    float* const w = c.weight + head * c.capacity;
    const float* const sc = p.scores + head * p.span * p.pitch;
    float had[kJoinTurns];
    float4 x[kJoinTurns];
#pragma unroll
    for (int i = 0; i < kJoinTurns; ++i) {
        const int slot = min(slot0 + i * turn, end - 1);
        had[i] = w[slot];
        if (p.pitch == 2) {
            const float2 v = *reinterpret_cast<const float2*>(sc + (size_t)slot * 2);
            x[i] = make_float4(v.x, v.y, 0.f, 0.f);
        } else {
            x[i] = *reinterpret_cast<const float4*>(sc + (size_t)slot * p.pitch + min(4 * sub, p.pitch - 4));
        }
    }
    for (int row = tid >> 5; row < rows; row += kJoinThreads / 32) {
        const int tile = row / TR, r = row - tile * TR;
        const Parts parts = parts_of(p, part, b, c.batch, head, h, tile, span, G);
        float m, l;
        row_total<32>(p.part_ml + (parts.slot * TR + r) * 2, TR * 2, parts.count, tid & 31, m, l);
        if ((tid & 31) == 0) {
            row_m[row] = m == -INFINITY ? 0.f : m;
            row_inv[row] = l == 0.f ? 0.f : 1.f / l;
            row_limit[row] = visible(part, row / G, span);
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kJoinTurns; ++i) {
        if (base + i * turn >= end) break;
        const int slot = min(slot0 + i * turn, end - 1);
        float sum = 0.f;
        for (int row = 4 * sub; row < rows; row += 4 << lanes) {
            if (row != 4 * sub) x[i] = *reinterpret_cast<const float4*>(sc + (size_t)slot * p.pitch + row);
            const float v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (row + e < rows && slot < row_limit[row + e]) sum += exp2_of(v[e] - row_m[row + e]) * row_inv[row + e];
        }
        for (int o = 1; o < 1 << lanes; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (sub == 0 && slot0 + i * turn < end) w[slot] = had[i] + sum;
    }
}

constexpr size_t align16(size_t v) { return (v + 15) & ~(size_t)15; }

RowsPlan rows_plan(const swlm_kv8_cache& c, const swlm_kv8_attend& a, size_t* bytes) {
    RowsPlan p{};
    p.cluster = 1;
    const int span = std::min(a.max_len, c.capacity), G = a.heads / c.kv_heads;
    p.rows = a.n * G;
    p.tiles = p.rows <= 8 ? 1 : p.rows <= kSaveRows ? 2 : kPromptRows / 8;
    p.row_tiles = (p.rows + 8 * p.tiles - 1) / (8 * p.tiles);
    p.span = (span + kStep - 1) / kStep * kStep;
    const long long groups = (long long)c.batch * c.kv_heads * p.row_tiles, units = p.rows > kSaveRows ? 0 : groups * ((span + kUnit - 1) / kUnit);
    bool several;   // parts that have to be joined
    if (p.rows > kSaveRows) {
        // Runs of slots per block of rows: as many as cost least, in key tiles: rounds of one CTA per SM, each its tiles and a start and end of about two;
        // with several runs a join, and each run's results to memory and back (portions of 300 tokens over 2000: 41 us in three runs, 58 with twice as many)
        const int tiles = (span + kPromptKeys - 1) / kPromptKeys;
        int runs = 1;
        double least = 1e30;
        for (int r = 1; r <= std::min(tiles, kSms); ++r) {
            const double rounds = (double)((groups * r + kSms - 1) / kSms), cost = rounds * ((tiles + r - 1) / r + 2) + (r > 1 ? 3 + 0.016 * groups * r : 0.0);
            if (cost < least) { least = cost; runs = r; }
        }
        p.chunk = ((span + runs - 1) / runs + kPromptKeys - 1) / kPromptKeys * kPromptKeys;
        p.splits = (span + p.chunk - 1) / p.chunk;
        several = p.splits > 1;
    } else {
        // CTAs that fill the GPU once, or one per unit where there are fewer
        const int fill = kSms * (p.tiles > 1 ? 2 : c.head_dim == 128 ? rows_ctas<128>() : rows_ctas<64>());
        // A cluster joins its own results, and adds its own slots' weights, in one launch, where its CTAs have few units each and all clusters run at once. us,
        // against two launches (32 / 8 heads of 128, int8): 1 x 1000 slots 7.0 / 8.8, 4 x 1000 7.4 / 9.6, 4 x 4000 12.9 / 16.6, 16 x 1000 13.0 / 17.6,
        // 1 x 8000 (eight units a CTA) 12.6 / 12.7; with weights (and a copy of them, some 5) 1 x 2000 12.4 / 14.0, but 1 x 4000 (four) 16.5 / 13.8
        const int per = (int)std::min<long long>(units / groups, 1 << 24), deep = a.accumulate ? 2 : 4;
        while (p.cluster < kClusterCtas && p.cluster < per && 2 * p.cluster * groups <= fill) p.cluster *= 2;
        if (per > deep * p.cluster || (a.accumulate && p.row_tiles > 1)) p.cluster = 1;
        p.stream = p.cluster == 1 && c.batch <= kStreamBatch && units < (1LL << 30) && groups < 16 * fill;
        p.ctas = p.stream ? (int)std::min<long long>(fill, units) : 0;
        several = p.stream && units > groups;
    }
    const size_t places = p.splits ? (size_t)groups * p.splits : (size_t)groups + p.ctas;
    // a group of lanes takes up to eight parts at once: as many groups as a row with the most parts has such turns
    const long long most = p.splits ? p.splits : std::min<long long>(units / groups, p.ctas / groups + 2);
    p.join_groups = most > 32 ? 8 : most > 16 ? 4 : most > 8 ? 2 : 1;
    size_t at = 0;
    char* base = static_cast<char*>(a.scratch);
    auto take = [&](size_t n) { char* q = base + at; at += align16(n); return q; };
    if (several) p.part_o = reinterpret_cast<float*>(take(places * 8 * p.tiles * c.head_dim * 4));
    const bool saves = a.accumulate && p.rows <= kSaveRows;
    if (several || (saves && p.cluster == 1)) {
        p.part_ml = reinterpret_cast<float*>(take(places * 8 * p.tiles * 8));
        if (p.stream) p.table = reinterpret_cast<int*>(take(((size_t)c.batch + 1) * 4));
    }
    if (saves) {
        p.pitch = p.rows <= 2 ? 2 : (p.rows + 3) / 4 * 4;
        // Two or four lanes add the weights of a slot's rows, in as many times the CTAs, while those still run at once: each works the rows' totals out again.
        // One step of 16 tokens over 8000: 69 us with one lane, 51 with four; eight of 4 over 4000: 45 and 51
        const long long joins = (long long)c.batch * c.kv_heads * ((span + kJoinSlots - 1) / kJoinSlots);
        while (p.join_lanes < 2 && p.pitch > 4 << p.join_lanes && joins << (p.join_lanes + 1) <= 3 * kSms) ++p.join_lanes;
        p.scores = reinterpret_cast<float*>(take((size_t)c.batch * c.kv_heads * p.span * p.pitch * 4));
    } else if (a.accumulate) {
        const size_t rows = (size_t)groups * kPromptRows;
        p.q16 = reinterpret_cast<__half*>(take(rows * c.head_dim * 2));
        p.q_factor = reinterpret_cast<float*>(take(rows * 4));
        p.q_shift = reinterpret_cast<float*>(take(rows * 4));
    }
    *bytes = at;
    return p;
}

template <int HD, int CODE, int NT>
cudaError_t launch_tiles(const dim3& grid, size_t smem, const swlm_kv8_cache& c, const swlm_kv8_attend& a, const RowsPlan& p, cudaStream_t s) {
    auto launch = [&](auto kernel) { return p.cluster > 1 ? launch_clusters(kernel, p.cluster, grid, dim3(kThreads), smem, s, c, a, p) : launch_k(kernel, grid, dim3(kThreads), smem, s, c, a, p); };
    if (kv8_two_products(a)) return p.pitch ? launch(kv8_rows_kernel<HD, CODE, NT, true, true>) : launch(kv8_rows_kernel<HD, CODE, NT, false, true>);
    return p.pitch ? launch(kv8_rows_kernel<HD, CODE, NT, true, false>) : launch(kv8_rows_kernel<HD, CODE, NT, false, false>);
}

template <int HD, int CODE>
int launch_rows(const swlm_kv8_cache& c, const swlm_kv8_attend& a, const RowsPlan& p, int* status, cudaStream_t s) {
    if (p.splits) {
        const int rc = launch_kv8_prompt(c, a, p, status, s);
        if (rc) return rc;
    } else {
        const dim3 grid = p.stream ? dim3((unsigned)p.ctas) : dim3((unsigned)(p.row_tiles * p.cluster), (unsigned)c.kv_heads, (unsigned)c.batch);
        const size_t smem = rows_smem<HD>() + (p.stream ? ((size_t)c.batch + 1) * sizeof(int4) : 0);
        const cudaError_t e = p.tiles == 1 ? launch_tiles<HD, CODE, 1>(grid, smem, c, a, p, s) : launch_tiles<HD, CODE, 2>(grid, smem, c, a, p, s);
        if (e != cudaSuccess) return cuda_fail(e, "kv8 attention launch");
    }
    const int span = std::min(a.max_len, c.capacity);
    const int per = kJoinThreads / (HD / 4) / p.join_groups, join = p.part_o ? (p.rows + per - 1) / per : 0;
    const int share = kJoinSlots >> p.join_lanes, slots = p.pitch && p.cluster == 1 ? (span + share - 1) / share : 0;
    if (join + slots) {
        const cudaError_t j = launch_k(kv8_join_kernel<HD>, dim3((unsigned)(join + slots), (unsigned)c.kv_heads, (unsigned)c.batch), dim3(kJoinThreads), 0, s, c, a, p, join);
        if (j != cudaSuccess) return cuda_fail(j, "kv8 join launch");
    }
    if (p.q16) return launch_kv8_prompt_weights(c, a, p, status, s);
    return SWLM_OK;
}

template <int HD, int CODE, int NT, bool SAVE>
int init_one() {
    constexpr int smem = (int)(rows_smem<HD>() + (kStreamBatch + 1) * sizeof(int4));
    SWLM_CUDA((cudaFuncSetAttribute(kv8_rows_kernel<HD, CODE, NT, SAVE, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)));
    SWLM_CUDA((cudaFuncSetAttribute(kv8_rows_kernel<HD, CODE, NT, SAVE, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)));
    return SWLM_OK;
}
template <int HD, int CODE>
int init_rows() {
    int rc = init_one<HD, CODE, 1, false>();
    if (!rc) rc = init_one<HD, CODE, 1, true>();
    if (!rc) rc = init_one<HD, CODE, 2, false>();
    if (!rc) rc = init_one<HD, CODE, 2, true>();
    return rc;
}
// the warps' results (at most two tiles) take the rings' place
static_assert((size_t)kWarps * 16 * 128 * 4 <= rows_smem<128>() && (size_t)kWarps * 16 * 64 * 4 <= rows_smem<64>(), "results fit the rings");

}  // namespace

int kv8_attend_init() {
    int rc = init_rows<128, SWLM_KV8_INT8>();
    if (!rc) rc = init_rows<128, SWLM_KV8_E4M3>();
    if (!rc) rc = init_rows<64, SWLM_KV8_INT8>();
    if (!rc) rc = init_rows<64, SWLM_KV8_E4M3>();
    if (!rc) rc = kv8_prompt_init();
    return rc;
}

// The grid of many rows is one number: CTAs of all (sequence, KV head, block of rows, run).
bool kv8_attend_grid_fits(const swlm_kv8_cache& c, const swlm_kv8_attend& a) {
    size_t bytes;
    const RowsPlan p = rows_plan(c, a, &bytes);
    return !p.splits || (long long)c.batch * c.kv_heads * p.row_tiles * p.splits <= INT_MAX;
}

size_t kv8_attend_scratch(const swlm_kv8_cache& c, const swlm_kv8_attend& a) {
    size_t bytes;
    rows_plan(c, a, &bytes);
    return bytes;
}

int launch_kv8_attend(const swlm_kv8_cache& c, const swlm_kv8_attend& a, int* status, cudaStream_t s) {
    size_t bytes;
    const RowsPlan p = rows_plan(c, a, &bytes);
    if (c.head_dim == 128) return c.code == SWLM_KV8_INT8 ? launch_rows<128, SWLM_KV8_INT8>(c, a, p, status, s) : launch_rows<128, SWLM_KV8_E4M3>(c, a, p, status, s);
    return c.code == SWLM_KV8_INT8 ? launch_rows<64, SWLM_KV8_INT8>(c, a, p, status, s) : launch_rows<64, SWLM_KV8_E4M3>(c, a, p, status, s);
}

}  // namespace swlm
