// Device code shared by the kernels over an 8-bit cache.
#pragma once

#include "kv8.h"

namespace swlm {
namespace kv8 {

constexpr int kSms = 148;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.f;                   // log2 of what a probability may exceed 1 by
constexpr float kValueUnit = 128.f;             // 2^7: probabilities up to 2^8 stay within fp16
constexpr float kValueRef = 0x1p-120f;          // values' scales are taken relative to the largest so far, or to this, whose inverse times 2^7 is still finite

// The kernel of few rows:
constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kSub = 2, kStep = 16 * kSub;        // tokens of a warp's step: two tiles of 16
constexpr int kUnit = kWarps * kStep;           // slots of a step of all warps: work is dealt in these

struct RowsPlan {
    int tiles;      // 8-row tiles per CTA
    int row_tiles;  // of a KV head at most, of 8 * tiles rows each
    int rows;       // n * group
    int stream, ctas;   // CTAs over equal shares of all units (stream), or one per (sequence, KV head, tile)
    int cluster;    // CTAs of a cluster that shares the slots of one (sequence, KV head, tile) and joins its results itself (1: none)
    int splits, chunk;  // the kernel of many rows: slots of a tile in runs of `chunk` (splits 0: the kernel of few rows)
    int span;       // slots that can be attended, rounded up to kStep
    int pitch;      // rows of a slot's kept scores (0: not kept)
    int join_groups;   // groups of lanes that share a row's parts
    int join_lanes;    // lanes that share a slot's rows, as a power of two
    float* part_o;  // [places][8 * tiles][head_dim], not normalised; places: (sequence, KV head, tile) + CTA, or of many rows * splits + run
    float* part_ml; // [places][8 * tiles][2]: reference maximum (log2), sum
    float* scores;  // [batch][kv_heads][span][pitch], log2
    // many rows whose weights are added: the shifted queries as fp16 in tiles of 64 rows, [batch][kv_heads][tiles][head_dim / 64][64][64], swizzled as the
    // products read them, and per row what turns a product into log2 of a weight: times (factor times the key's scale), plus the shift
    __half* q16;
    float* q_factor;  // [batch][kv_heads][row_tiles * 256]
    float* q_shift;
    int* table;     // [batch + 1]: units before each sequence, and of all
};

__device__ __forceinline__ float exp2_of(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ unsigned pack_half(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&v);
}

// What rounding (a, b) to the fp16 pair v has left, as another pair: both together are the numbers to 2^-22 of themselves.
__device__ __forceinline__ unsigned pack_rest(float a, float b, unsigned v) {
    const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&v));
    return pack_half(a - r.x, b - r.y);
}

// Codes to fp16, exactly. int8: with the sign bit turned a byte u = c + 128 is the low byte of 1024 + u.
template <int CODE> __device__ __forceinline__ unsigned prepared(unsigned word) { return CODE == SWLM_KV8_INT8 ? word ^ 0x80808080u : word; }
// bytes 2 * HIGH and 2 * HIGH + 1 of a prepared word
template <int CODE, int HIGH> __device__ __forceinline__ unsigned pair_of(unsigned word) {
    if (CODE == SWLM_KV8_INT8) {
        const unsigned biased = __byte_perm(word, 0x64646464u, HIGH ? 0x4342 : 0x4140);
        const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&biased), __half2half2(__ushort_as_half(0x6480)));   // 1024 + 128
        return *reinterpret_cast<const unsigned*>(&v);
    }
    unsigned v;
    if (HIGH) asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(v) : "r"(word));
    else asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(v) : "r"(word));
    return v;
}

// Two fp32 operations as one instruction.
__device__ __forceinline__ unsigned long long pair_bits(const float2& v) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
    return r;
}
__device__ __forceinline__ float2 bits_pair(unsigned long long v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ float2 fma2(const float2& a, const float2& b, const float2& c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pair_bits(a)), "l"(pair_bits(b)), "l"(pair_bits(c)));
    return bits_pair(r);
}
__device__ __forceinline__ float2 add2(const float2& a, const float2& b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_bits(a)), "l"(pair_bits(b)));
    return bits_pair(r);
}
__device__ __forceinline__ float2 mul2(const float2& a, const float2& b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_bits(a)), "l"(pair_bits(b)));
    return bits_pair(r);
}

__device__ __forceinline__ float log2_of(float x) { float y; asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

// What is added to a score (log2) to make it log2 of a weight: minus the row's maximum and the logarithm of its sum. A row that attends
// nothing has no weights.
__device__ __forceinline__ float row_shift_of(float m, float l) { return l == 0.f ? -INFINITY : -((m == -INFINITY ? 0.f : m) + log2f(l)); }

// Four results of a row with sum l.
__device__ __forceinline__ void store_out(unsigned short* dst, const float4& o, float l, bool f16) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    unsigned v[2];
    if (f16) {
        v[0] = pack_half(o.x * inv, o.y * inv); v[1] = pack_half(o.z * inv, o.w * inv);
    } else {
        const __nv_bfloat162 x = __floats2bfloat162_rn(o.x * inv, o.y * inv), y = __floats2bfloat162_rn(o.z * inv, o.w * inv);
        v[0] = *reinterpret_cast<const unsigned*>(&x); v[1] = *reinterpret_cast<const unsigned*>(&y);
    }
    *reinterpret_cast<uint2*>(dst) = make_uint2(v[0], v[1]);
}

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

// Where a CTA's share of the work lies. Stream order: sequences, their KV heads, their tiles of rows, units of kUnit slots. CTA c of C takes U / C
// units, the first U % C CTAs one more, of one (sequence, KV head, tile) or of several, so that all CTAs have the same work whatever the lengths are.
struct Shares {
    int ctas, each, more;   // each CTA has a unit at least, so that the parts of one tile lie one behind the other
    __device__ __forceinline__ Shares(int units, int launched) {
        ctas = min(launched, units);
        each = ctas ? units / ctas : 0;
        more = units - each * ctas;
    }
    __device__ __forceinline__ int first(int cta) const { return cta * each + min(cta, more); }
    __device__ __forceinline__ int cta_of(int unit) const { return unit < more * (each + 1) ? unit / (each + 1) : more + (unit - more * (each + 1)) / each; }
};
__device__ __forceinline__ int sequence_units(const Kv8Part& part, int span) { return (max(visible(part, part.count - 1, span), 1) + kUnit - 1) / kUnit; }
__device__ __forceinline__ int sequence_tiles(const Kv8Part& part, int G, int TR) { return (part.count * G + TR - 1) / TR; }

// Parts of one (sequence, KV head, tile of rows): the first one's place and their number.
struct Parts { size_t slot; int count; };
__device__ __forceinline__ Parts parts_of(const RowsPlan& p, const Kv8Part& part, int b, int batch, size_t head, int h, int tile, int span, int G) {
    const size_t slot = head * p.row_tiles + tile;
    if (p.splits) {
        const int TR = 8 * p.tiles, end = visible(part, min((tile + 1) * TR - 1, part.count * G - 1) / G, span);
        return {slot * p.splits, max(1, (end + p.chunk - 1) / p.chunk)};
    }
    if (!p.stream) return {slot, 1};
    const Shares shares(p.table[batch], p.ctas);
    const int per = sequence_units(part, span), u = p.table[b] + (h * sequence_tiles(part, G, 8 * p.tiles) + tile) * per, c0 = shares.cta_of(u);
    return {slot + c0, shares.cta_of(u + per - 1) - c0 + 1};
}

// The kernel of many rows (kv8_prompt.cu): rows of a CTA, keys of a tile.
constexpr int kPromptRows = 256, kPromptKeys = 128;

}  // namespace kv8

// Whether probabilities meet the values as two fp16 numbers.
inline bool kv8_two_products(const swlm_kv8_attend& a) {
    return a.probabilities == SWLM_KV8_P_TWO || (a.probabilities == SWLM_KV8_P_BY_TYPE && a.dtype == SWLM_KV8_FP16);
}
int kv8_prompt_init();
int launch_kv8_prompt_weights(const swlm_kv8_cache& c, const swlm_kv8_attend& a, const kv8::RowsPlan& p, int* status, cudaStream_t s);
int launch_kv8_prompt(const swlm_kv8_cache& c, const swlm_kv8_attend& a, const kv8::RowsPlan& p, int* status, cudaStream_t s);
}  // namespace swlm
