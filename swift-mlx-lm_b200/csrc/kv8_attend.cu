// Attention over a cache of 8-bit codes with one scale per block of tokens and head.
//
//   s_ij = scale * ks[j / T] * (q_i . ck_j),  p = softmax over the slots that query i attends,  out_i = sum_j p_ij vs[j / T] cv_j
//
// Codes are exact as fp16 numbers (e4m3 ones times 2^-8), and so are bf16 and fp16 queries after a shift of the row's exponent that brings its
// largest value to 2^12, but for values 2^-26 and less of the largest. So q . ck is an fp16 product with fp32 sums on the tensor cores, and
// a step of 16 tokens, which never crosses a block, takes its scale as one number behind it.
//
// Rows: the queries of a step times the heads of a group, 8 to a tile. A CTA has one tile (or two) and a run of slots of one (sequence,
// KV head); its eight warps take steps of 16 tokens in turn, each over a ring of its own that cp.async fills. Scores come as S^T = K Q^T
// (16 tokens x 8 rows, so that a decode step's four or eight rows fill the tile), probabilities are transposed in
// registers (movmatrix) and meet the values as O^T = V^T P^T. The reference maximum of a row moves only when it would grow by more than 2^8.
// Probabilities are rounded to fp16 (2^-11 of themselves) times 2^7 vs / vr, vr the largest value scale so far: values of blocks down to 2^-24 of
// the largest scale keep that precision. Partial results of several runs are joined by a second launch, which also adds the weights.
#include <algorithm>

#include "kv8.h"

namespace swlm {
namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kStep = 16;                       // tokens of a warp's step
constexpr int kSpanStep = kWarps * kStep;       // runs of slots are multiples of it
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.f;                   // log2 of what a probability may exceed 1 by
constexpr float kValueUnit = 128.f;             // 2^7: probabilities up to 2^8 stay within fp16
constexpr int kSaveRows = 64;                   // up to so many rows of a KV head the scores are kept for the weights, beyond they are worked out again

struct RowsPlan {
    int tiles;      // 8-row tiles per CTA
    int row_tiles;  // CTAs along the rows
    int rows;       // n * group
    int chunk, splits;
    int span;       // slots that can be attended, rounded up to kStep
    int pitch;      // rows of a slot's kept scores (0: not kept)
    float* part_o;  // [batch][kv_heads][rows][splits][head_dim], not normalised
    float* part_ml; // [batch][kv_heads][rows][splits][2]: reference maximum (log2), sum
    float* scores;  // [batch][kv_heads][span][pitch], log2
};

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
__device__ __forceinline__ float lds_f32(unsigned a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ float exp2_of(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ void mma(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned transpose8x8(unsigned v) {
    unsigned r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ unsigned pack_half(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&v);
}

// Codes to fp16. int8: with the sign bit turned a byte u = c + 128 is the low byte of 1024 + u. e4m3: sign, exponent and mantissa in their places
// are the number times 2^-8, subnormal ones too (and 0x7F, which no block holds, a finite number: a stale slot's codes meet the weight 0).
template <int CODE> __device__ __forceinline__ unsigned prepared(unsigned word) { return CODE == SWLM_KV8_INT8 ? word ^ 0x80808080u : word; }
// bytes 2 * HIGH and 2 * HIGH + 1 of a prepared word
template <int CODE, int HIGH> __device__ __forceinline__ unsigned pair_of(unsigned word) {
    if (CODE == SWLM_KV8_INT8) {
        const unsigned biased = __byte_perm(word, 0x64646464u, HIGH ? 0x4342 : 0x4140);
        const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&biased), __half2half2(__ushort_as_half(0x6480)));   // 1024 + 128
        return *reinterpret_cast<const unsigned*>(&v);
    }
    const unsigned high = __byte_perm(word, 0u, HIGH ? 0x3424 : 0x1404);   // (0, byte, 0, byte)
    return (high & 0x80008000u) | ((high >> 1) & 0x3F803F80u);
}
template <int CODE> __device__ __forceinline__ constexpr float code_unit() { return CODE == SWLM_KV8_INT8 ? 1.f : 256.f; }

// Eight 16-bit values as floats.
__device__ __forceinline__ void widen(const uint4& r, bool f16, float (&x)[8]) {
    const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (f16) {
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            x[2 * i] = v.x; x[2 * i + 1] = v.y;
        } else {
            x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
}
// The power of two that brings `top`, a row's largest |value|, to 2^12 or a little more (NaN for a row that is not finite), and its inverse.
__device__ __forceinline__ void row_shift(float top, float& up, float& down) {
    const int e = (int)(__float_as_uint(top) >> 23);   // 0 for zero and subnormal ones
    const int shift = top > 0.f ? min(12 + 127 - e, 126) : 0;
    up = e == 255 ? kKv8NaN : __uint_as_float((unsigned)(127 + shift) << 23);
    down = e == 255 ? kKv8NaN : __uint_as_float((unsigned)(127 - shift) << 23);
}

// The slots that query i of a sequence attends are those below this.
__device__ __forceinline__ int visible(const Kv8Part& part, int i, int span) { return (int)min((long long)part.len + i + 1, (long long)span); }

template <int HD> __host__ __device__ constexpr int stages() { return HD == 128 ? 3 : 5; }
template <int HD> __host__ __device__ constexpr int stage_bytes() { return 2 * kStep * HD + 16; }   // keys, values, their scales
template <int HD> constexpr size_t rows_smem() { return (size_t)kWarps * stages<HD>() * stage_bytes<HD>(); }

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

template <int HD, int CODE, int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1) kv8_rows_kernel(const swlm_kv8_cache c, const swlm_kv8_attend a, const RowsPlan p) {
    constexpr int KS = HD / 16, MT = HD / 16, NS = stages<HD>(), SB = stage_bytes<HD>(), TR = 8 * NT;
    extern __shared__ __align__(16) unsigned char sm[];
    __shared__ float warp_m[kWarps][TR], warp_l[kWarps][TR];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int b = blockIdx.z, h = blockIdx.y, G = a.heads / c.kv_heads;
    const int tile = blockIdx.x / p.splits, split = blockIdx.x - tile * p.splits;
    const Kv8Part part = kv8_part(b, a.lengths, a.counts, a.starts, a.n, a.rows);
    const int rows = part.count * G, row0 = tile * TR;
    if (row0 >= rows) return;
    const int span = min(a.max_len, c.capacity);
    const int end = visible(part, min((row0 + TR - 1) / G, part.count - 1), span);   // of the tile's last query: it sees most
    const int from = split * p.chunk, to = min(from + p.chunk, end);
    if (from >= end && split > 0) return;
    const size_t head = (size_t)b * c.kv_heads + h;
    const unsigned char* keys = static_cast<const unsigned char*>(c.k) + head * c.capacity * HD;
    const unsigned char* values = static_cast<const unsigned char*>(c.v) + head * c.capacity * HD;
    const float* ks = c.k_scale + head * (c.capacity / c.block);
    const float* vs = c.v_scale + head * (c.capacity / c.block);
    const int block_shift = 31 - __clz(c.block);

    // ring of this warp: step number i covers the 16 slots from `from` + (warp + 8 i) * 16 on. Whole steps are read: they lie within the capacity,
    // a multiple of 16; what is beyond the last token is masked.
    const unsigned ring = smem_addr(sm) + warp * NS * SB;
    const int first = from + warp * kStep, steps = first < to ? (to - first + kSpanStep - 1) / kSpanStep : 0;
    auto request = [&](int i) {
        if (i < steps) {
            const unsigned dst = ring + i % NS * SB;
            const int base = first + i * kSpanStep;
            const unsigned char *k = keys + (size_t)base * HD, *v = values + (size_t)base * HD;
#pragma unroll
            for (int u = 0; u < HD / 32; ++u) {
                const int piece = lane + 32 * u, r = piece / (HD / 16), q = piece % (HD / 16);
                copy16(dst + key_at<HD>(r, q), k + piece * 16);
                copy16(dst + kStep * HD + value_at<HD>(r, q), v + piece * 16);
            }
            if (lane < 2) copy4(dst + 2 * kStep * HD + lane * 4, (lane ? vs : ks) + (base >> block_shift));
        }
        commit();
    };
#pragma unroll
    for (int i = 0; i < NS - 1; ++i) request(i);

    unsigned qf[NT][KS][2];
    float factor[NT][2];     // of columns 2 t and 2 t + 1 (rows of the tile): score in log2 per unit of the product
    int limit[NT][2];
    {
        const unsigned short* q = static_cast<const unsigned short*>(a.q);
        const bool f16 = a.dtype == SWLM_KV8_FP16;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = row0 + nt * 8 + g, i = min(r, rows - 1) / G;
            float down;
            load_query<HD>(q + (int64_t)(part.start + i) * a.q_stride + (size_t)(h * G + min(r, rows - 1) - i * G) * HD, r < rows, f16, t, qf[nt], down);
            down *= a.scale * kLog2e * code_unit<CODE>();
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                factor[nt][e] = __shfl_sync(0xffffffffu, down, (2 * t + e) * 4);
                const int rc = row0 + nt * 8 + 2 * t + e;
                limit[nt][e] = rc < rows ? visible(part, rc / G, span) : 0;
            }
        }
    }
    float acc[NT][MT][4], m_ref[NT][2], l_run[NT][2], v_ref = 0x1p-100f, v_inv = 0x1p100f * kValueUnit;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[nt][j][e] = 0.f;
        m_ref[nt][0] = m_ref[nt][1] = -INFINITY;
        l_run[nt][0] = l_run[nt][1] = 0.f;
    }
    for (int i = 0; i < steps; ++i) {
        wait_groups<NS - 2>();
        __syncwarp();          // this step's copies of all lanes are there, and all lanes have read the step before
        request(i + NS - 1);
        const unsigned at = ring + i % NS * SB;
        const int base = first + i * kSpanStep;
        // ---- scores ----
        float s[NT][4] = {};
#pragma unroll
        for (int u = 0; u < HD / 64; ++u) {
            const uint4 lo = lds128(at + key_at<HD>(g, t + 4 * u)), hi = lds128(at + key_at<HD>(g + 8, t + 4 * u));
            const unsigned lw[4] = {lo.x, lo.y, lo.z, lo.w}, hw[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const unsigned x = prepared<CODE>(lw[w]), y = prepared<CODE>(hw[w]);
                const unsigned a0 = pair_of<CODE, 0>(x), a1 = pair_of<CODE, 0>(y), a2 = pair_of<CODE, 1>(x), a3 = pair_of<CODE, 1>(y);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma(s[nt], a0, a1, a2, a3, qf[nt][u * 4 + w][0], qf[nt][u * 4 + w][1]);
            }
        }
        const float k_scale = lds_f32(at + 2 * kStep * HD), v_scale = lds_f32(at + 2 * kStep * HD + 4);
        bool moves = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int slot = base + g + 8 * (e >> 1);
                s[nt][e] = slot < limit[nt][e & 1] ? s[nt][e] * (factor[nt][e & 1] * k_scale) : -INFINITY;
                moves = moves || s[nt][e] > m_ref[nt][e & 1] + kSlack;
            }
        if (p.pitch) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int r = row0 + nt * 8 + 2 * t;
                if (r < p.pitch) {   // (the pitch is even)
                    float* dst = p.scores + (head * p.span + base + g) * p.pitch + r;
                    *reinterpret_cast<float2*>(dst) = make_float2(s[nt][0], s[nt][1]);
                    *reinterpret_cast<float2*>(dst + 8 * p.pitch) = make_float2(s[nt][2], s[nt][3]);
                }
            }
        }
        // ---- softmax ----
        if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = fmaxf(s[nt][e], s[nt][e + 2]);
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    if (top > m_ref[nt][e] + kSlack) {
                        const float corr = exp2_of(m_ref[nt][e] - top);   // 0 for a row's first slots
                        m_ref[nt][e] = top;
                        l_run[nt][e] *= corr;
#pragma unroll
                        for (int j = 0; j < MT; ++j) { acc[nt][j][e] *= corr; acc[nt][j][e + 2] *= corr; }
                    }
                }
        }
        if (v_scale > v_ref) {
            const float corr = v_ref / v_scale;
            v_ref = v_scale;
            v_inv = kValueUnit / v_scale;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < MT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[nt][j][e] *= corr;
        }
        const float unit = v_scale * v_inv;
        unsigned pf[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = s[nt][e], m = m_ref[nt][e & 1];
                const float pr = exp2_of(x - (m == -INFINITY ? 0.f : m));
                l_run[nt][e & 1] += pr;
                w[e] = x == -INFINITY ? 0.f : pr * unit;   // (a slot that the row does not attend may lie in a block that is NaN)
            }
            pf[nt][0] = transpose8x8(pack_half(w[0], w[1]));
            pf[nt][1] = transpose8x8(pack_half(w[2], w[3]));
        }
        // ---- values: this lane has HD / 8 dimensions of tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9 ----
        const unsigned va = at + kStep * HD;
        unsigned vw[4][HD / 32];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = 2 * t + (k & 1) + 8 * (k >> 1);
            if (HD == 128) {
                const uint4 v = lds128(va + value_at<HD>(r, g));
                vw[k][0] = v.x; vw[k][1] = v.y; vw[k][HD / 32 - 2] = v.z; vw[k][HD / 32 - 1] = v.w;
            } else {
                const uint2 v = lds64(va + value_at<HD>(r, g >> 1) + (g & 1) * 8);
                vw[k][0] = v.x; vw[k][1] = v.y;
            }
        }
#pragma unroll
        for (int w = 0; w < HD / 32; ++w) {
            const unsigned v0 = prepared<CODE>(vw[0][w]), v1 = prepared<CODE>(vw[1][w]), v2 = prepared<CODE>(vw[2][w]), v3 = prepared<CODE>(vw[3][w]);
#pragma unroll
            for (int half = 0; half < 2; ++half) {   // dimensions 4 w + 2 half and the next one
                const unsigned lo = __byte_perm(v0, v1, half ? 0x7362 : 0x5140), hi = __byte_perm(v2, v3, half ? 0x7362 : 0x5140);
                const unsigned a0 = pair_of<CODE, 0>(lo), a1 = pair_of<CODE, 1>(lo), a2 = pair_of<CODE, 0>(hi), a3 = pair_of<CODE, 1>(hi);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma(acc[nt][2 * w + half], a0, a1, a2, a3, pf[nt][0], pf[nt][1]);
            }
        }
    }

    // ---- the warps' results together ----
    __syncthreads();   // every warp is done with its ring
    float* const outs = reinterpret_cast<float*>(sm);   // [warp][TR][HD]
    const float unit = v_ref * (code_unit<CODE>() / kValueUnit);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float l = l_run[nt][e];
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            if (g == 0) { warp_m[warp][nt * 8 + 2 * t + e] = m_ref[nt][e]; warp_l[warp][nt * 8 + 2 * t + e] = l; }
        }
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e)   // row 2 t + e, dimensions g * HD / 8 + 2 j and the next one
                *reinterpret_cast<float2*>(outs + (size_t)(warp * TR + nt * 8 + 2 * t + e) * HD + g * (HD / 8) + 2 * j) = make_float2(acc[nt][j][e] * unit, acc[nt][j][e + 2] * unit);
    }
    __syncthreads();
    const bool f16 = a.dtype == SWLM_KV8_FP16;
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
        const size_t at = (head * p.rows + row) * p.splits + split;
        if (d == 0 && p.part_ml) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m, l);
        if (p.splits > 1) {
            *reinterpret_cast<float4*>(p.part_o + at * HD + d) = o;
        } else {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const int i = row / G;
            unsigned short* dst = static_cast<unsigned short*>(a.out) + (int64_t)(part.start + i) * a.out_stride + (size_t)(h * G + row - i * G) * HD + d;
            unsigned v[2];
            if (f16) {
                v[0] = pack_half(o.x * inv, o.y * inv); v[1] = pack_half(o.z * inv, o.w * inv);
            } else {
                const __nv_bfloat162 x = __floats2bfloat162_rn(o.x * inv, o.y * inv), y = __floats2bfloat162_rn(o.z * inv, o.w * inv);
                v[0] = *reinterpret_cast<const unsigned*>(&x); v[1] = *reinterpret_cast<const unsigned*>(&y);
            }
            *reinterpret_cast<uint2*>(dst) = make_uint2(v[0], v[1]);
        }
    }
}

// Maximum and sum of a row over the parts that it has, by a group of LANES lanes; all of them get both.
template <int LANES>
__device__ __forceinline__ void row_total(const float* ml, int parts, int lane, float& m, float& l) {
    m = -INFINITY;
    for (int s = lane; s < parts; s += LANES) m = fmaxf(m, ml[2 * s]);
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    l = 0.f;
    for (int s = lane; s < parts; s += LANES) {
        const float x = ml[2 * s], v = ml[2 * s + 1];
        l += x == -INFINITY ? v : exp2_of(x - m) * v;   // (v is 0, or NaN where a part's scores are all NaN)
    }
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
}

constexpr int kJoinThreads = 256;

// CTAs 0 .. join - 1 along x join the parts of the rows, the others add the kept scores' weights, 256 slots each.
template <int HD>
__global__ void __launch_bounds__(kJoinThreads) kv8_join_kernel(const swlm_kv8_cache c, const swlm_kv8_attend a, const RowsPlan p, const int join) {
    constexpr int LANES = HD / 4, PER = kJoinThreads / LANES;   // lanes of a row, rows of a CTA
    __shared__ float row_m[kSaveRows], row_inv[kSaveRows];
    __shared__ int row_limit[kSaveRows];
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x, G = a.heads / c.kv_heads;
    const Kv8Part part = kv8_part(b, a.lengths, a.counts, a.starts, a.n, a.rows);
    const int rows = part.count * G, span = min(a.max_len, c.capacity);
    const size_t head = (size_t)b * c.kv_heads + h;
    auto parts_of = [&](int limit) { return max(1, (limit + p.chunk - 1) / p.chunk); };   // (part 0 is always written)
    if ((int)blockIdx.x < join) {
        const int row = (int)blockIdx.x * PER + tid / LANES, lane = tid % LANES;
        const bool on = row < rows;
        const int parts = on ? parts_of(visible(part, row / G, span)) : 0;
        const size_t at = (head * p.rows + (on ? row : 0)) * p.splits;
        float m, l;
        row_total<LANES>(p.part_ml + at * 2, parts, lane, m, l);
        if (!on) return;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int s = 0; s < parts; ++s) {
            const float x = p.part_ml[(at + s) * 2];
            const float f = x == -INFINITY ? 1.f : exp2_of(x - m);   // (a part without slots has zeros)
            const float4 v = *reinterpret_cast<const float4*>(p.part_o + (at + s) * HD + lane * 4);
            o.x += f * v.x; o.y += f * v.y; o.z += f * v.z; o.w += f * v.w;
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int i = row / G;
        unsigned short* dst = static_cast<unsigned short*>(a.out) + (int64_t)(part.start + i) * a.out_stride + (size_t)(h * G + row - i * G) * HD + lane * 4;
        unsigned v[2];
        if (a.dtype == SWLM_KV8_FP16) {
            v[0] = pack_half(o.x * inv, o.y * inv); v[1] = pack_half(o.z * inv, o.w * inv);
        } else {
            const __nv_bfloat162 x = __floats2bfloat162_rn(o.x * inv, o.y * inv), y = __floats2bfloat162_rn(o.z * inv, o.w * inv);
            v[0] = *reinterpret_cast<const unsigned*>(&x); v[1] = *reinterpret_cast<const unsigned*>(&y);
        }
        *reinterpret_cast<uint2*>(dst) = make_uint2(v[0], v[1]);
        return;
    }
    if (rows == 0) return;
    const int end = visible(part, part.count - 1, span), slot = ((int)blockIdx.x - join) * kJoinThreads + tid;
    if (slot - tid >= end) return;
    for (int row = tid >> 5; row < rows; row += kJoinThreads / 32) {
        const int limit = visible(part, row / G, span);
        float m, l;
        row_total<32>(p.part_ml + (head * p.rows + row) * p.splits * 2, parts_of(limit), tid & 31, m, l);
        if ((tid & 31) == 0) {
            row_m[row] = m == -INFINITY ? 0.f : m;
            row_inv[row] = l == 0.f ? 0.f : 1.f / l;
            row_limit[row] = limit;
        }
    }
    __syncthreads();
    if (slot >= end) return;
    const float* sc = p.scores + (head * p.span + slot) * p.pitch;
    float sum = 0.f;
    for (int row = 0; row < rows; row += 2) {
        const float2 x = *reinterpret_cast<const float2*>(sc + row);
        if (slot < row_limit[row]) sum += exp2_of(x.x - row_m[row]) * row_inv[row];
        if (row + 1 < rows && slot < row_limit[row + 1]) sum += exp2_of(x.y - row_m[row + 1]) * row_inv[row + 1];
    }
    c.weight[head * c.capacity + slot] += sum;
}

// The weights of many rows: the scores are worked out again with the rows' totals known. A warp keeps the fragments of 16 tokens' keys in registers and
// walks the rows that attend them; a CTA's rows go through shared memory as fp16, 32 at a time. Nothing is added across warps.
constexpr int kAgainWarps = 4, kAgainRows = 32;
template <int HD, int CODE>
__global__ void __launch_bounds__(kAgainWarps * 32) kv8_weights_kernel(const swlm_kv8_cache c, const swlm_kv8_attend a, const RowsPlan p) {
    constexpr int KS = HD / 16, PITCH = HD + 16;   // (rows 32 bytes further on than their length: the four rows of a phase meet different banks)
    __shared__ __align__(16) __half qs[kAgainRows][PITCH];
    __shared__ float row_factor[kAgainRows], row_m[kAgainRows], row_inv[kAgainRows];
    __shared__ int row_limit[kAgainRows];
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3, G = a.heads / c.kv_heads;
    const Kv8Part part = kv8_part(b, a.lengths, a.counts, a.starts, a.n, a.rows);
    const int rows = part.count * G, span = min(a.max_len, c.capacity);
    const int end = rows ? visible(part, part.count - 1, span) : 0, cta0 = (int)blockIdx.x * kAgainWarps * kStep;
    if (cta0 >= end) return;
    const size_t head = (size_t)b * c.kv_heads + h;
    const int base = cta0 + warp * kStep;
    const bool on = base < end;
    unsigned kf[KS][4];
    float k_scale = 0.f;
    if (on) {
        const unsigned char* keys = static_cast<const unsigned char*>(c.k) + (head * c.capacity + base) * HD;
        k_scale = c.k_scale[head * (c.capacity / c.block) + base / c.block];
#pragma unroll
        for (int u = 0; u < HD / 64; ++u) {
            const uint4 lo = *reinterpret_cast<const uint4*>(keys + g * HD + (t + 4 * u) * 16), hi = *reinterpret_cast<const uint4*>(keys + (g + 8) * HD + (t + 4 * u) * 16);
            const unsigned lw[4] = {lo.x, lo.y, lo.z, lo.w}, hw[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const unsigned x = prepared<CODE>(lw[w]), y = prepared<CODE>(hw[w]);
                kf[u * 4 + w][0] = pair_of<CODE, 0>(x); kf[u * 4 + w][1] = pair_of<CODE, 0>(y);
                kf[u * 4 + w][2] = pair_of<CODE, 1>(x); kf[u * 4 + w][3] = pair_of<CODE, 1>(y);
            }
        }
    }
    float sum[2] = {0.f, 0.f};   // of tokens g and g + 8, over this lane's columns
    // the first query that attends the CTA's first slot
    const int row_from = (int)min((long long)max((long long)cta0 - part.len, 0LL) * G, (long long)rows) / 8 * 8;
    const unsigned short* q = static_cast<const unsigned short*>(a.q);
    const bool f16 = a.dtype == SWLM_KV8_FP16;
    for (int r0 = row_from; r0 < rows; r0 += kAgainRows) {
        __syncthreads();
        // four lanes per row, a quarter of it each
#pragma unroll 1
        for (int k = 0; k < kAgainRows / (kAgainWarps * 8); ++k) {
            const int r = k * kAgainWarps * 8 + warp * 8 + g, row = r0 + r, i = min(row, rows - 1) / G;
            unsigned frag[KS][2];
            float down;
            load_query<HD>(q + (int64_t)(part.start + i) * a.q_stride + (size_t)(h * G + min(row, rows - 1) - i * G) * HD, row < rows, f16, t, frag, down);
            // kept in the order of the fragments: lane t's pairs of k-step s at s * 16 + 4 t
#pragma unroll
            for (int s = 0; s < KS; ++s) *reinterpret_cast<uint2*>(&qs[r][s * 16 + 4 * t]) = make_uint2(frag[s][0], frag[s][1]);
            const int limit = row < rows ? visible(part, i, span) : 0;
            float m = -INFINITY, l = 0.f;
            if (t == 0) {
                if (row < rows) {
                    const float* ml = p.part_ml + (head * p.rows + row) * p.splits * 2;
                    const int parts = max(1, (limit + p.chunk - 1) / p.chunk);
                    for (int s = 0; s < parts; ++s) m = fmaxf(m, ml[2 * s]);
                    for (int s = 0; s < parts; ++s) l += ml[2 * s] == -INFINITY ? ml[2 * s + 1] : exp2_of(ml[2 * s] - m) * ml[2 * s + 1];
                }
                row_factor[r] = down * (a.scale * kLog2e * code_unit<CODE>());
                row_m[r] = m == -INFINITY ? 0.f : m;
                row_inv[r] = l == 0.f ? 0.f : 1.f / l;
                row_limit[r] = limit;
            }
        }
        __syncthreads();
        if (!on) continue;
        for (int rt = 0; rt < min(kAgainRows, rows - r0); rt += 8) {
            float s[4] = {};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const uint2 v = *reinterpret_cast<const uint2*>(&qs[rt + g][k * 16 + 4 * t]);
                mma(s, kf[k][0], kf[k][1], kf[k][2], kf[k][3], v.x, v.y);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = rt + 2 * t + (e & 1), slot = base + g + 8 * (e >> 1);
                if (slot < row_limit[r]) sum[e >> 1] += exp2_of(s[e] * (row_factor[r] * k_scale) - row_m[r]) * row_inv[r];
            }
        }
    }
    if (!on) return;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        float v = sum[e];
        v += __shfl_xor_sync(0xffffffffu, v, 1);
        v += __shfl_xor_sync(0xffffffffu, v, 2);
        const int slot = base + g + 8 * e;
        if (t == 0 && slot < end) c.weight[head * c.capacity + slot] += v;
    }
}

constexpr size_t align16(size_t v) { return (v + 15) & ~(size_t)15; }

RowsPlan rows_plan(const swlm_kv8_cache& c, const swlm_kv8_attend& a, size_t* bytes) {
    RowsPlan p{};
    const int span = std::min(a.max_len, c.capacity), G = a.heads / c.kv_heads;
    p.rows = a.n * G;
    p.tiles = p.rows <= 8 ? 1 : 2;
    p.row_tiles = (p.rows + 8 * p.tiles - 1) / (8 * p.tiles);
    p.span = (span + kStep - 1) / kStep * kStep;
    // runs of slots so that the CTAs fill the GPU: two per SM with one tile, one with two
    const long long ctas = (long long)c.batch * c.kv_heads * p.row_tiles;
    const int want = p.tiles == 1 ? 296 : 148;
    const int most = std::max(1, (span + kSpanStep - 1) / kSpanStep);
    const int splits = (int)std::min<long long>(std::min(most, 64), std::max<long long>(1, want / ctas));
    p.chunk = ((span + splits - 1) / splits + kSpanStep - 1) / kSpanStep * kSpanStep;
    p.splits = std::max(1, (span + p.chunk - 1) / p.chunk);
    const size_t parts = (size_t)c.batch * c.kv_heads * p.rows * p.splits;
    size_t at = 0;
    char* base = static_cast<char*>(a.scratch);
    if (p.splits > 1) { p.part_o = reinterpret_cast<float*>(base); at += align16(parts * c.head_dim * 4); }
    if (p.splits > 1 || a.accumulate) { p.part_ml = reinterpret_cast<float*>(base + at); at += align16(parts * 8); }
    if (a.accumulate && p.rows <= kSaveRows) {
        p.pitch = (p.rows + 1) / 2 * 2;
        p.scores = reinterpret_cast<float*>(base + at);
        at += align16((size_t)c.batch * c.kv_heads * p.span * p.pitch * 4);
    }
    *bytes = at;
    return p;
}

template <int HD, int CODE>
int launch_rows(const swlm_kv8_cache& c, const swlm_kv8_attend& a, const RowsPlan& p, cudaStream_t s) {
    const dim3 grid((unsigned)(p.row_tiles * p.splits), (unsigned)c.kv_heads, (unsigned)c.batch);
    const cudaError_t e = p.tiles == 1 ? launch_k(kv8_rows_kernel<HD, CODE, 1>, grid, dim3(kThreads), rows_smem<HD>(), s, c, a, p)
                                       : launch_k(kv8_rows_kernel<HD, CODE, 2>, grid, dim3(kThreads), rows_smem<HD>(), s, c, a, p);
    if (e != cudaSuccess) return cuda_fail(e, "kv8 attention launch");
    const int span = std::min(a.max_len, c.capacity);
    const int join = p.splits > 1 ? (p.rows + kJoinThreads / (HD / 4) - 1) / (kJoinThreads / (HD / 4)) : 0;
    const int slots = p.pitch ? (span + kJoinThreads - 1) / kJoinThreads : 0;
    if (join + slots) {
        const cudaError_t j = launch_k(kv8_join_kernel<HD>, dim3((unsigned)(join + slots), (unsigned)c.kv_heads, (unsigned)c.batch), dim3(kJoinThreads), 0, s, c, a, p, join);
        if (j != cudaSuccess) return cuda_fail(j, "kv8 join launch");
    }
    if (a.accumulate && !p.pitch) {
        constexpr int per = kAgainWarps * kStep;
        const cudaError_t w = launch_k(kv8_weights_kernel<HD, CODE>, dim3((unsigned)((span + per - 1) / per), (unsigned)c.kv_heads, (unsigned)c.batch), dim3(kAgainWarps * 32), 0, s, c, a, p);
        if (w != cudaSuccess) return cuda_fail(w, "kv8 weights launch");
    }
    return SWLM_OK;
}

template <int HD, int CODE>
int init_rows() {
    SWLM_CUDA(cudaFuncSetAttribute(kv8_rows_kernel<HD, CODE, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)rows_smem<HD>()));
    SWLM_CUDA(cudaFuncSetAttribute(kv8_rows_kernel<HD, CODE, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)rows_smem<HD>()));
    return SWLM_OK;
}
// the warps' results (at most two tiles) take the rings' place
static_assert((size_t)kWarps * 16 * 128 * 4 <= rows_smem<128>() && (size_t)kWarps * 16 * 64 * 4 <= rows_smem<64>(), "results fit the rings");

}  // namespace

int kv8_attend_init() {
    int rc = init_rows<128, SWLM_KV8_INT8>();
    if (!rc) rc = init_rows<128, SWLM_KV8_E4M3>();
    if (!rc) rc = init_rows<64, SWLM_KV8_INT8>();
    if (!rc) rc = init_rows<64, SWLM_KV8_E4M3>();
    return rc;
}

size_t kv8_attend_scratch(const swlm_kv8_cache& c, const swlm_kv8_attend& a) {
    size_t bytes;
    rows_plan(c, a, &bytes);
    return bytes;
}

int launch_kv8_attend(const swlm_kv8_cache& c, const swlm_kv8_attend& a, cudaStream_t s) {
    size_t bytes;
    const RowsPlan p = rows_plan(c, a, &bytes);
    if (c.head_dim == 128) return c.code == SWLM_KV8_INT8 ? launch_rows<128, SWLM_KV8_INT8>(c, a, p, s) : launch_rows<128, SWLM_KV8_E4M3>(c, a, p, s);
    return c.code == SWLM_KV8_INT8 ? launch_rows<64, SWLM_KV8_INT8>(c, a, p, s) : launch_rows<64, SWLM_KV8_E4M3>(c, a, p, s);
}

}  // namespace swlm
