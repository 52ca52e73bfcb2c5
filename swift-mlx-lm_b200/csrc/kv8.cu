// A cache of 8-bit codes with one scale per block of tokens and head: appending to it and evicting from it.
//
// append   s = max(s0, max |x| / top), c = round(x / s) with IEEE quotients, so that a code is the same whatever the launch. One CTA per
//          (block of tokens, KV head, keys or values): the new values of the block stay in registers between the search for the largest and
//          the rounding, each is read once.
// evict    select: one cluster of CTAs per (sequence, KV head) finds the `keep` largest keys by radix selection and pairs the free slots below `keep`
//          with the tokens that stay from behind. move: one CTA per (block below `keep`, KV head, keys or values) gathers what the
//          block takes, scales it anew and stores it. Only slots from `keep` on are sources of another block's slots and only slots below
//          `keep` are written, so that the blocks need no order among them, also in place; the scales of the sources, which the last block
//          may share with slots that are written, are taken along by the first kernel.
//
// What bounds them: append of 6272 tokens (8 heads of 128) 11.8 us for 39 MB, 10.1 where no scale of a block with older tokens grows: a CTA's load, search,
// barrier, quotients and stores one after the other, with 41 % of the warps and 57 to 65 % of the issue slots busy (18 instructions a value and warp
// lane, most of the quotient); of one token the launch. Eviction of 4 x 32768 tokens to 4096 (73 MB): 48 us, of which the selection, a chain of passes over shared memory and
// barriers of the cluster, takes half (with the counts of all digits read from every CTA, and a pass over ties that nobody has to tell apart, 56) and
// the move, mostly instructions, half; 1 x 4352 to 4096: 17.6 us, nearly all of it latency.
#include <cooperative_groups.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "kv8_device.cuh"
#include "swlm_runtime.h"

namespace cg = cooperative_groups;

namespace swlm {
using namespace kv8;
namespace {

constexpr float kTopInt8 = 127.f, kTopE4m3 = 448.f;

template <int CODE> __device__ __forceinline__ constexpr float kv8_top() { return CODE == SWLM_KV8_INT8 ? kTopInt8 : kTopE4m3; }

// A code is round(x / s) of the IEEE quotient. Two of Markstein's steps, q += (x - q s) / s with the rounded inverse and an exact residual, give that
// quotient from x / s's first approximation, where nothing is subnormal: five operations, two values to an instruction, no branch.

// the code of the quotient y, as a byte (|y| <= top but for the last place; the clamp is for scales that are subnormal)
template <int CODE> __device__ __forceinline__ unsigned kv8_code(float y) {
    if (CODE == SWLM_KV8_INT8) return (unsigned)__float2int_rn(fminf(fmaxf(y, -kTopInt8), kTopInt8)) & 0xFFu;
    return (unsigned)__nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
}
// A block's scale and its inverse. Scales far from 1 (whose residuals might be subnormal) go by division.
struct Divisor {
    float s, inv;
    bool ordinary;
    __device__ __forceinline__ explicit Divisor(float scale) : s(scale), inv(1.f / scale), ordinary(scale > 0x1p-60f && scale < 0x1p60f) {}
    __device__ __forceinline__ float2 quotient(const float2& x) const {
        const float2 inv2 = make_float2(inv, inv), minus = make_float2(-s, -s);
        float2 q = mul2(x, inv2);
        q = fma2(fma2(q, minus, x), inv2, q);
        return fma2(fma2(q, minus, x), inv2, q);
    }
};
// The codes of four values, as a word.
template <int CODE, bool ORDINARY> __device__ __forceinline__ unsigned kv8_codes4(const float2& x, const float2& y, const Divisor& d) {
    if (!ORDINARY)
        return kv8_code<CODE>(__fdiv_rn(x.x, d.s)) | kv8_code<CODE>(__fdiv_rn(x.y, d.s)) << 8 | kv8_code<CODE>(__fdiv_rn(y.x, d.s)) << 16 | kv8_code<CODE>(__fdiv_rn(y.y, d.s)) << 24;
    float2 p = d.quotient(x), q = d.quotient(y);
    if (CODE == SWLM_KV8_INT8) {
        // the low byte of 1.5 * 2^23 + v is v rounded to an integer, ties to even
        const float2 magic = make_float2(12582912.f, 12582912.f);
        p = add2(p, magic);
        q = add2(q, magic);
        return __byte_perm(__byte_perm(__float_as_uint(p.x), __float_as_uint(p.y), 0x0040), __byte_perm(__float_as_uint(q.x), __float_as_uint(q.y), 0x0040), 0x5410);
    }
    unsigned word;   // (the steps turn -0 into 0; its code has the sign)
    asm("{\n\t.reg .b16 p, q;\n\tcvt.rn.satfinite.e4m3x2.f32 p, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 q, %4, %3;\n\tmov.b32 %0, {p, q};\n\t}"
        : "=r"(word) : "f"(copysignf(p.x, x.x)), "f"(copysignf(p.y, x.y)), "f"(copysignf(q.x, y.x)), "f"(copysignf(q.y, y.y)));
    return word;
}
// The word's codes, held at scale `from`, at another.
template <int CODE, bool ORDINARY> __device__ __forceinline__ unsigned kv8_again(unsigned word, float from, const Divisor& d) {
    float2 x, y;
    const float2 from2 = make_float2(from, from);
    if (CODE == SWLM_KV8_INT8) {
        const unsigned u = word ^ 0x80808080u;   // c + 128, the low byte of 2^23 + u
        const float2 bias = make_float2(-8388736.f, -8388736.f);
        x = add2(make_float2(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7650)), __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7651))), bias);
        y = add2(make_float2(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7652)), __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7653))), bias);
    } else {
        const unsigned lo = pair_of<CODE, 0>(word), hi = pair_of<CODE, 1>(word);
        x = __half22float2(*reinterpret_cast<const __half2*>(&lo));
        y = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    }
    return kv8_codes4<CODE, ORDINARY>(mul2(x, from2), mul2(y, from2), d);
}

// Largest of a CTA's unsigned numbers, to all of its threads.
__device__ __forceinline__ unsigned block_max(unsigned v, unsigned* warps) {
    v = __reduce_max_sync(0xffffffffu, v);
    if (blockDim.x == 32) return v;
    if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < (int)blockDim.x / 32; ++w) v = max(v, warps[w]);
    return v;
}

// ---- append ----------------------------------------------------------------------------------------------------------------

constexpr int kAppendThreads = 256, kAppendUnits = 8;   // a unit: eight values of a token, at most 128 * 128 / 8 of them in a block
static_assert(kAppendThreads * kAppendUnits * 8 >= kKv8MaxBlock * 128, "a block fits its CTA");

template <bool F16> __device__ __forceinline__ float half_bits(unsigned bits) {
    return F16 ? __half2float(__ushort_as_half((unsigned short)bits)) : __uint_as_float(bits << 16);
}
// the two values of a word
template <bool F16> __device__ __forceinline__ float2 halves(unsigned word) {
    return F16 ? __half22float2(*reinterpret_cast<const __half2*>(&word)) : make_float2(__uint_as_float(word << 16), __uint_as_float(word & 0xFFFF0000u));
}

template <int CODE, bool F16>
__global__ void __launch_bounds__(kAppendThreads) kv8_append_kernel(const swlm_kv8_cache c, const swlm_kv8_append a) {
    __shared__ unsigned warps[kAppendThreads / 32];
    pdl_wait();
    const int b = blockIdx.z, h = blockIdx.y >> 1, which = blockIdx.y & 1, tid = threadIdx.x, T = c.block;
    const Kv8Part part = kv8_part(b, a.lengths, a.counts, a.starts, nullptr, a.n, a.rows);
    const bool ok = part.fits && part.len >= 0 && (long long)part.len + part.count <= c.capacity;
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0 && a.refused) a.refused[b] = ok ? 0 : 1;
    if (!ok) return;
    const int blk = part.len / T + (int)blockIdx.x, base = blk * T;
    const int low = max(part.len, base), high = min(part.len + part.count, base + T);   // new slots of this block
    if (low >= high) return;
    const int old = low - base;   // tokens that it has
    const unsigned short* x = static_cast<const unsigned short*>(which ? a.v : a.k);
    const int64_t stride = which ? a.v_stride : a.k_stride;
    x += part.start * stride + h * c.head_dim;
    unsigned char* codes = static_cast<unsigned char*>(which ? c.v : c.k) + ((size_t)(b * (size_t)c.kv_heads + h) * c.capacity + base) * c.head_dim;
    float* scale = (which ? c.v_scale : c.k_scale) + (size_t)(b * (size_t)c.kv_heads + h) * (c.capacity / T) + blk;
    const float s0 = old ? *scale : 0.f;

    const int per = c.head_dim == 128 ? 4 : 3, units = (high - low) << per;   // log2 of the units of a token, new units
    uint4 raw[kAppendUnits];
    unsigned top = 0;   // largest |value| as its 15 bits: the order of the numbers, infinity and NaN above all
#pragma unroll
    for (int u = 0; u < kAppendUnits; ++u) {
        const int i = tid + u * (int)blockDim.x;
        raw[u] = make_uint4(0, 0, 0, 0);
        if (i < units) {
            const int row = (i >> per) + low - part.len, d = (i & ((1 << per) - 1)) * 8;
            raw[u] = *reinterpret_cast<const uint4*>(x + row * stride + d);
        }
        const unsigned m = __vmaxu2(__vmaxu2(raw[u].x & 0x7FFF7FFFu, raw[u].y & 0x7FFF7FFFu), __vmaxu2(raw[u].z & 0x7FFF7FFFu, raw[u].w & 0x7FFF7FFFu));
        top = max(top, max(m & 0xFFFFu, m >> 16));
    }
    top = block_max(top, warps);   // (all have read the old scale when it returns, or are the only warp)
    const bool finite = top < (F16 ? 0x7C00u : 0x7F80u) && s0 == s0;
    const float s = finite ? fmaxf(s0, __fdiv_rn(half_bits<F16>(top), kv8_top<CODE>())) : kKv8NaN;
    if (blockDim.x == 32) __syncwarp();
    if (tid == 0) *scale = s;
    const bool grows = old && finite && s > s0;
    const Divisor divisor(s);
    auto store = [&](auto ordinary) {
        constexpr bool ORDINARY = decltype(ordinary)::value;
#pragma unroll
        for (int u = 0; u < kAppendUnits; ++u) {
            const int i = tid + u * (int)blockDim.x;
            if (i >= units) continue;
            const unsigned w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
            unsigned out[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) out[k] = kv8_codes4<CODE, ORDINARY>(halves<F16>(w[2 * k]), halves<F16>(w[2 * k + 1]), divisor);
            *reinterpret_cast<uint2*>(codes + (old << (per + 3)) + i * 8) = make_uint2(out[0], out[1]);
        }
        if (grows)
            for (int i = tid; i < old << per; i += blockDim.x) {
                uint2* at = reinterpret_cast<uint2*>(codes + (size_t)i * 8);
                const uint2 was = *at;
                *at = make_uint2(kv8_again<CODE, ORDINARY>(was.x, s0, divisor), kv8_again<CODE, ORDINARY>(was.y, s0, divisor));
            }
    };
    if (divisor.ordinary) store(std::true_type());
    else if (finite && s > 0.f) store(std::false_type());
    else for (int i = tid; i < units; i += blockDim.x) *reinterpret_cast<uint2*>(codes + (old << (per + 3)) + i * 8) = make_uint2(0, 0);   // zeros, or NaN by its scale
    if (which == 0)
        for (int slot = low + tid; slot < high; slot += blockDim.x) {
            const size_t at = (size_t)(b * (size_t)c.kv_heads + h) * c.capacity + slot;
            if (c.weight) c.weight[at] = 0.f;
            if (c.slot_pos) c.slot_pos[at] = (int)((unsigned)a.seen[b] + (unsigned)(slot - part.len));
        }
}

__global__ void kv8_lengths_kernel(int batch, const int32_t* in, const int32_t* counts, int n, int limit, const int32_t* refused, int32_t* out) {
    pdl_wait();
    const int b = blockIdx.x * blockDim.x + threadIdx.x;
    if (b >= batch) return;
    const long long sum = (long long)in[b] + (refused && refused[b] ? 0 : counts ? counts[b] : n);
    out[b] = refused && refused[b] ? in[b] : (int)max(min(sum, (long long)limit), (long long)INT32_MIN);
}

// ---- evict -----------------------------------------------------------------------------------------------------------------

constexpr int kSelectThreads = 512, kSelectWarps = kSelectThreads / 32, kSelectSlots = 4096;   // slots of a CTA, up to eight CTAs
constexpr int kDigitBits = 11, kDigits = 1 << kDigitBits, kGroups = kDigits / 32;
constexpr int kCachedKeys = 24 * 1024;   // keys of a CTA that stay in shared memory between the passes

// Scratch of one (sequence, KV head): where slot j < keep comes from (j itself, or ~i: the i-th of the tokens that move), the slots of the
// tokens that move and the scales of their keys and values.
struct EvictPlan {
    int* source; int* moved; float* k_scale; float* v_scale;
    __host__ __device__ EvictPlan(void* scratch, size_t head, int keep) {
        int* p = static_cast<int*>(scratch) + head * (size_t)keep * 4;
        source = p; moved = p + keep; k_scale = reinterpret_cast<float*>(p + 2 * (size_t)keep); v_scale = k_scale + keep;
    }
};

// Floats in the order of unsigned numbers, both zeros alike, NaN below all; protected tokens above all.
__device__ __forceinline__ unsigned evict_key(float w, int pos, int sink, long long recent_from) {
    if (pos < sink || pos >= recent_from) return 0xFFFFFFFFu;
    if (w != w) return 0u;
    const unsigned u = __float_as_uint(w + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One cluster per (sequence, KV head); its CTAs have equal runs of slots. The digits' counts of all of them are added up by each.
template <int CTAS, bool CACHED>
__global__ void __cluster_dims__(CTAS, 1, 1) __launch_bounds__(kSelectThreads) kv8_select_kernel(const swlm_kv8_cache c, const swlm_kv8_evict a) {
    extern __shared__ unsigned keys[];
    __shared__ __align__(16) unsigned hist[2][kDigits];   // counts of a pass, of this CTA
    __shared__ unsigned groups[2][kGroups];               // and of the 32 digits of a group
    __shared__ unsigned coarse[CTAS][kGroups], fine[CTAS][32];   // all CTAs' counts of the groups, and of the digits of the one that was found
    static_assert(kDigits == 4 * kSelectThreads && kGroups * 8 == kSelectThreads, "four digits of a thread, eight threads of a group");
    __shared__ int seg[3][kSelectWarps], counted[3];   // ties, free slots, moving tokens: of a warp, of the CTA
    pdl_wait();
    const cg::cluster_group cluster = cg::this_cluster();
    auto sync = [&]() {
        if constexpr (CTAS == 1) __syncthreads();
        else cluster.sync();
    };
    const int b = blockIdx.y, h = blockIdx.x / CTAS, rank = CTAS == 1 ? 0 : (int)cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int len = min(min(a.lengths[b], a.max_len), c.capacity), keep = a.keep;
    if (len <= keep) return;   // (the whole cluster) nothing leaves: the second kernel does not look at the plan
    const size_t head = (size_t)b * c.kv_heads + h;
    const float* weight = c.weight + head * c.capacity;
    const int32_t* pos = c.slot_pos + head * c.capacity;
    const long long recent_from = (long long)a.seen[b] - a.recent;
    // this CTA's slots: first .. last - 1
    const int share = (len + CTAS * 32 - 1) / (CTAS * 32) * 32, first = min(rank * share, len), last = min(first + share, len);
    auto key_of = [&](int i) { return evict_key(weight[i], pos[i], a.sink, recent_from); };
    for (int i = tid; i < 2 * kDigits; i += kSelectThreads) hist[0][i] = 0;
    if (CACHED) {
#pragma unroll 8
        for (int i = first + tid; i < last; i += kSelectThreads) keys[i - first] = key_of(i);
    }
    auto key = [&](int i) { return CACHED ? keys[i - first] : key_of(i); };
    __syncthreads();

    auto own_counts = [&](const unsigned* counts) {
        const uint4 v = *reinterpret_cast<const uint4*>(counts + 4 * tid);
        return v.x + v.y + v.z + v.w;
    };
    auto of_rank = [&](auto* mine, int r) { return CTAS == 1 ? mine : cluster.map_shared_rank(mine, r); };
    auto prefix_sum = [&](unsigned v) {   // of the lanes up to this one
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        return v;
    };

    // radix selection of the keep-th largest key, from the top digit down
    unsigned prefix = 0, mask = 0;
    int want = keep, pass = 0;   // how many keys are still to be found among those that share the prefix
    for (int shift = 32 - kDigitBits; ; shift = max(shift - kDigitBits, 0), ++pass) {
        unsigned* const mine = hist[pass & 1];
        for (int i = first + tid; i < last; i += kSelectThreads) {
            const unsigned k = key(i);
            if ((k & mask) == prefix) atomicAdd(&mine[(k >> shift) & (kDigits - 1)], 1u);
        }
        __syncthreads();
        unsigned sum = own_counts(mine);
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        if ((lane & 7) == 0) groups[pass & 1][tid >> 3] = sum;
        sync();   // (what the pass before counted has been read by all)
        *reinterpret_cast<uint4*>(hist[(pass + 1) & 1] + 4 * tid) = make_uint4(0, 0, 0, 0);
        // the group of digits that the wanted key is in, then the digit: 3 KB of other CTAs' counts instead of all 64 KB; every warp finds the same
        if (tid < CTAS * kGroups) coarse[tid / kGroups][tid % kGroups] = of_rank(groups[pass & 1], tid / kGroups)[tid % kGroups];
        __syncthreads();
        unsigned above;
        int group = 0, digit = 0;
        {
            unsigned hi = 0, lo = 0;   // lane l has groups 63 - 2 l and 62 - 2 l: from the top down
#pragma unroll
            for (int r = 0; r < CTAS; ++r) { hi += coarse[r][kGroups - 1 - 2 * lane]; lo += coarse[r][kGroups - 2 - 2 * lane]; }
            const unsigned upto = prefix_sum(hi + lo), before = upto - hi - lo;
            const int l = __ffs(__ballot_sync(0xffffffffu, upto >= (unsigned)want)) - 1;
            const bool first_of = before + hi >= (unsigned)want;
            group = __shfl_sync(0xffffffffu, first_of ? kGroups - 1 - 2 * lane : kGroups - 2 - 2 * lane, l);
            above = __shfl_sync(0xffffffffu, first_of ? before : before + hi, l);
        }
        if (tid < CTAS * 32) fine[tid >> 5][lane] = of_rank(mine, tid >> 5)[group * 32 + lane];
        __syncthreads();
        bool found_all;
        {
            unsigned n = 0;   // lane l has digit 31 - l of the group
#pragma unroll
            for (int r = 0; r < CTAS; ++r) n += fine[r][31 - lane];
            const unsigned upto = above + prefix_sum(n);
            const int l = __ffs(__ballot_sync(0xffffffffu, upto >= (unsigned)want)) - 1;
            digit = group * 32 + 31 - l;
            above = __shfl_sync(0xffffffffu, upto - n, l);   // keys of higher digits
            found_all = __shfl_sync(0xffffffffu, upto, l) == (unsigned)want;
        }
        const unsigned digits = (unsigned)(kDigits - 1) << shift;
        prefix = (prefix & ~digits) | (unsigned)digit << shift;   // (the last digit overlaps the one before it, with the same bits there)
        mask |= digits;
        want -= (int)above;
        if (found_all) { want = len; break; }   // all keys with this prefix stay: none of those below it has to be told from another
        if (shift == 0) break;
    }
    const unsigned limit = prefix;   // keys above it stay, and the first `want` of those equal to it

    // a run of slots per warp: ties first, then free slots below `keep` and staying ones from it on, each numbered in slot order
    const int run = (last - first + kSelectThreads - 1) / kSelectThreads * 32, from = min(first + warp * run, last), to = min(from + run, last);
    const unsigned below = (1u << lane) - 1u;
    auto before = [&](int what) {   // of seg[what]: how many there are in the runs before this warp's, of this CTA
        const unsigned v = lane < kSelectWarps ? (unsigned)seg[what][lane] : 0u, all = __reduce_add_sync(0xffffffffu, v);
        if (tid == 0) counted[what] = (int)all;
        return (int)__reduce_add_sync(0xffffffffu, lane < warp ? v : 0u);
    };
    auto of_ranks = [&](int what) { return CTAS == 1 ? 0 : (int)__reduce_add_sync(0xffffffffu, lane < rank ? (unsigned)cluster.map_shared_rank(counted, lane)[what] : 0u); };
    int tie0 = 0;
    if (want < len) {   // (the same in all CTAs)
        int ties = 0;
        for (int i = from; i < to; i += 32) ties += __popc(__ballot_sync(0xffffffffu, i + lane < to && key(min(i + lane, to - 1)) == limit));
        if (lane == 0) seg[0][warp] = ties;
        __syncthreads();
        tie0 = before(0);
        sync();
        tie0 += of_ranks(0);
    }
    auto walk = [&](auto&& each) {   // each(slot, free, moving): the lanes whose slots below `keep` are free, and whose tokens behind it stay
        int t = tie0;
#pragma unroll 4
        for (int i = from; i < to; i += 32) {
            const int slot = i + lane;
            const bool in = slot < to;
            const unsigned k = key(min(slot, to - 1));
            bool stays = k >= limit;
            if (want < len) {
                const unsigned tied = __ballot_sync(0xffffffffu, in && k == limit);
                stays = k > limit || (k == limit && t + __popc(tied & below) < want);
                t += __popc(tied);
            }
            const unsigned changes = __ballot_sync(0xffffffffu, in && stays == (slot >= keep)), kept = __ballot_sync(0xffffffffu, slot < keep);
            each(slot, changes & kept, changes & ~kept);
        }
    };
    int free0 = 0, move0 = 0;
    walk([&](int, unsigned f, unsigned m) {
        free0 += __popc(f);
        move0 += __popc(m);
    });
    if (lane == 0) {
        seg[1][warp] = free0;
        seg[2][warp] = move0;
    }
    __syncthreads();
    free0 = before(1);
    move0 = before(2);
    sync();
    free0 += of_ranks(1);
    move0 += of_ranks(2);
    if constexpr (CTAS > 1) cluster.barrier_arrive();   // (of the CTAs that may leave when all have read its counts)
    const EvictPlan plan(a.scratch, head, keep);
    const float* ks = c.k_scale + head * (c.capacity / c.block);
    const float* vs = c.v_scale + head * (c.capacity / c.block);
    walk([&](int slot, unsigned f, unsigned m) {
        if (slot < min(to, keep)) plan.source[slot] = f >> lane & 1u ? ~(free0 + __popc(f & below)) : slot;
        if (m >> lane & 1u) {
            const int i = move0 + __popc(m & below);
            plan.moved[i] = slot;
            plan.k_scale[i] = ks[slot / c.block];
            plan.v_scale[i] = vs[slot / c.block];
        }
        free0 += __popc(f);
        move0 += __popc(m);
    });
    if constexpr (CTAS > 1) cluster.barrier_wait();
}

constexpr int kMoveThreads = 256, kMoveUnits = 4;   // a unit: 16 codes
static_assert(kMoveThreads * kMoveUnits * 16 >= kKv8MaxBlock * 128, "a block fits its CTA");

// (five CTAs of 256 threads an SM, 48 registers: 71 us where 52 registers take 79, 32 heads x 12000 -> 9000 of 128 in blocks of 128, e4m3)
template <int CODE>
__global__ void __launch_bounds__(kMoveThreads, 5) kv8_move_kernel(const swlm_kv8_cache c, const swlm_kv8_cache to, const swlm_kv8_evict a, const int in_place) {
    __shared__ int source[kKv8MaxBlock];
    __shared__ float scales[kKv8MaxBlock];
    __shared__ unsigned warps[kMoveThreads / 32];
    pdl_wait();
    const int b = blockIdx.z, h = blockIdx.y >> 1, which = blockIdx.y & 1, tid = threadIdx.x, T = c.block, keep = a.keep;
    const int len = min(min(a.lengths[b], a.max_len), c.capacity);
    const int base = (int)blockIdx.x * T, n = min(min(len, keep) - base, T);   // slots of this block
    if (n <= 0) return;
    const size_t head = (size_t)b * c.kv_heads + h;
    const EvictPlan plan(a.scratch, head, keep);
    const float own = (which ? c.v_scale : c.k_scale)[head * (c.capacity / T) + blockIdx.x];
    bool takes = false;
    for (int i = tid; i < n; i += blockDim.x) {
        int src = base + i;
        float s = own;
        if (len > keep) {
            src = plan.source[base + i];
            if (src < 0) {
                const int m = ~src;
                s = which ? plan.v_scale[m] : plan.k_scale[m];
                src = plan.moved[m];
                takes = true;
            }
        }
        source[i] = src;
        scales[i] = s;
    }
    const bool changed = __syncthreads_or(takes);
    if (!changed && in_place) return;
    const unsigned char* from = static_cast<const unsigned char*>(which ? c.v : c.k) + head * c.capacity * c.head_dim;
    unsigned char* dst = static_cast<unsigned char*>(which ? to.v : to.k) + (head * to.capacity + base) * c.head_dim;
    const int per = c.head_dim == 128 ? 3 : 2, units = n << per;   // log2 of the units of a token
    uint4 raw[kMoveUnits];
    unsigned top = 0;   // largest |value|, as the bits of a float that is not negative
#pragma unroll
    for (int u = 0; u < kMoveUnits; ++u) {
        const int i = tid + u * (int)blockDim.x;
        if (i >= units) continue;
        raw[u] = *reinterpret_cast<const uint4*>(from + (size_t)source[i >> per] * c.head_dim + (i & ((1 << per) - 1)) * 16);
        if (changed) {
            const unsigned w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
            __half2 m = __half2half2(__ushort_as_half(0));   // of each pair's |code|
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned x = prepared<CODE>(w[e]), lo = pair_of<CODE, 0>(x), hi = pair_of<CODE, 1>(x);
                m = __hmax2_nan(m, __hmax2_nan(__habs2(*reinterpret_cast<const __half2*>(&lo)), __habs2(*reinterpret_cast<const __half2*>(&hi))));
            }
            const float2 both = __half22float2(m);
            top = max(top, max(__float_as_uint(fabsf(both.x * scales[i >> per])), __float_as_uint(fabsf(both.y * scales[i >> per]))));
        }
    }
    if (!changed) {
#pragma unroll
        for (int u = 0; u < kMoveUnits; ++u) {
            const int i = tid + u * (int)blockDim.x;
            if (i < units) *reinterpret_cast<uint4*>(dst + (size_t)i * 16) = raw[u];
        }
        if (tid == 0) (which ? to.v_scale : to.k_scale)[head * (to.capacity / T) + blockIdx.x] = own;
    } else {
        top = block_max(top, warps);
        const bool finite = top < 0x7F800000u;
        const float s = finite ? __fdiv_rn(__uint_as_float(top), kv8_top<CODE>()) : kKv8NaN;
        const Divisor divisor(s);
        if (tid == 0) (which ? to.v_scale : to.k_scale)[head * (to.capacity / T) + blockIdx.x] = s;
        auto store = [&](auto kind) {   // 0: zeros, or NaN by its scale
            constexpr int KIND = decltype(kind)::value;
#pragma unroll
            for (int u = 0; u < kMoveUnits; ++u) {
                const int i = tid + u * (int)blockDim.x;
                if (i >= units) continue;
                const float mine = scales[i >> per];
                const unsigned w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
                unsigned out[4] = {0, 0, 0, 0};
                if (KIND)
#pragma unroll
                    for (int e = 0; e < 4; ++e) out[e] = kv8_again<CODE, KIND == 2>(w[e], mine, divisor);
                *reinterpret_cast<uint4*>(dst + (size_t)i * 16) = make_uint4(out[0], out[1], out[2], out[3]);
            }
        };
        if (divisor.ordinary) store(std::integral_constant<int, 2>());
        else if (finite && s > 0.f) store(std::integral_constant<int, 1>());
        else store(std::integral_constant<int, 0>());
    }
    if (which == 0)
        for (int i = tid; i < n; i += blockDim.x) {
            const size_t at = head * c.capacity + source[i], put = head * to.capacity + base + i;
            const float w = c.weight[at];
            const int32_t p = c.slot_pos[at];
            to.weight[put] = w;
            to.slot_pos[put] = p;
        }
}

int after_launch(cudaError_t e, const char* what) { return e == cudaSuccess ? SWLM_OK : cuda_fail(e, what); }

}  // namespace

int launch_kv8_append(const swlm_kv8_cache& c, const swlm_kv8_append& a, cudaStream_t s) {
    // blocks that a sequence's tokens may touch: the first one may have room for a single token
    const unsigned blocks = (unsigned)((a.n + c.block - 2) / c.block + 1);
    // (a whole block in at most 8 units per thread; a single token's few values need no more than a warp, its block's older codes do)
    const int threads = std::min(kAppendThreads, std::max(32, c.block * c.head_dim / (8 * kAppendUnits)));
    const dim3 grid(blocks, 2u * (unsigned)c.kv_heads, (unsigned)c.batch);
    auto launch = [&](auto kernel) { return after_launch(launch_k(kernel, grid, dim3(threads), 0, s, c, a), "kv8 append launch"); };
    if (c.code == SWLM_KV8_INT8) return a.dtype == SWLM_KV8_FP16 ? launch(kv8_append_kernel<SWLM_KV8_INT8, true>) : launch(kv8_append_kernel<SWLM_KV8_INT8, false>);
    return a.dtype == SWLM_KV8_FP16 ? launch(kv8_append_kernel<SWLM_KV8_E4M3, true>) : launch(kv8_append_kernel<SWLM_KV8_E4M3, false>);
}

int launch_kv8_lengths(int batch, const int32_t* in, const int32_t* counts, int n, int limit, const int32_t* refused, int32_t* out, cudaStream_t s) {
    return after_launch(launch_k(kv8_lengths_kernel, dim3((unsigned)(batch + 127) / 128), dim3(128), 0, s, batch, in, counts, n, limit, refused, out), "kv8 lengths launch");
}

int kv8_init() {
    SWLM_CUDA((cudaFuncSetAttribute(kv8_select_kernel<8, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kCachedKeys * 4)));
    return kv8_attend_init();
}

size_t kv8_evict_scratch(const swlm_kv8_cache& c, const swlm_kv8_evict& a) { return (size_t)c.batch * c.kv_heads * a.keep * 16; }

int launch_kv8_evict(const swlm_kv8_cache& c, const swlm_kv8_cache& to, const swlm_kv8_evict& a, cudaStream_t s) {
    const int span = std::min(a.max_len, c.capacity);
    cudaError_t e = cudaSuccess;
    if (span > a.keep) {
        // A barrier of a cluster costs what a thousand slots do, and CTAs beside it are other heads' (us, eviction of a quarter, 1 / 2 / 4 / 8 CTAs):
        // 128 heads x 1000 slots 30.9 / 32.7 / 45.5 / 92.7, 32 x 4352 40.0 / 38.6 / 38.6 / 47.4, 8 x 12000 51 / 41 / 35 / 36, 2 x 32768 151 / 49 / 35 / 32
        const int ctas = span <= kSelectSlots ? 1 : span <= 2 * kSelectSlots ? 2 : span <= 4 * kSelectSlots ? 4 : 8;
        const dim3 grid((unsigned)c.kv_heads * ctas, (unsigned)c.batch);
        const int share = (span + ctas * 32 - 1) / (ctas * 32) * 32;   // their keys stay in shared memory, up to kCachedKeys (only eight CTAs can have more)
        auto launch = [&](auto kernel) { return launch_k(kernel, grid, dim3(kSelectThreads), share <= kCachedKeys ? (size_t)share * 4 : 0, s, c, a); };
        e = ctas == 1 ? launch(kv8_select_kernel<1, true>) : ctas == 2 ? launch(kv8_select_kernel<2, true>) : ctas == 4 ? launch(kv8_select_kernel<4, true>) :
            share <= kCachedKeys ? launch(kv8_select_kernel<8, true>) : launch(kv8_select_kernel<8, false>);
        if (e != cudaSuccess) return cuda_fail(e, "kv8 selection launch");
    } else if (c.k == to.k) {
        return SWLM_OK;   // in place, and no sequence can have more than `keep` tokens
    }
    const int threads = std::min(kMoveThreads, std::max(32, c.block * c.head_dim / (16 * kMoveUnits)));
    const dim3 grid((unsigned)((std::min(a.keep, span) + c.block - 1) / c.block), 2u * (unsigned)c.kv_heads, (unsigned)c.batch);
    const int in_place = c.k == to.k;
    return after_launch(c.code == SWLM_KV8_INT8 ? launch_k(kv8_move_kernel<SWLM_KV8_INT8>, grid, dim3(threads), 0, s, c, to, a, in_place)
                                                : launch_k(kv8_move_kernel<SWLM_KV8_E4M3>, grid, dim3(threads), 0, s, c, to, a, in_place), "kv8 move launch");
}

}  // namespace swlm

// ---- entry points: arguments are checked before anything is launched; what only the device knows is checked by the kernels -----------------

using namespace swlm;

namespace {

int refuse(const char* what) {
    set_error("kv8: %s", what);
    return SWLM_ERR_INVALID;
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

int cache_shape_ok(const swlm_kv8_cache& c) {
    if (c.batch < 1 || c.batch > kKv8MaxBatch || c.kv_heads < 1 || c.kv_heads > kKv8MaxKvHeads) return refuse("batch or KV heads out of range");
    if (c.head_dim != 64 && c.head_dim != 128) { set_error("kv8: heads of %d (64 and 128 are supported)", c.head_dim); return SWLM_ERR_UNSUPPORTED; }
    if (c.block < kKv8MinBlock || c.block > kKv8MaxBlock || (c.block & (c.block - 1))) return refuse("a block has 16, 32, 64 or 128 tokens");
    if (c.capacity < c.block || c.capacity % c.block || c.capacity > kKv8MaxLen) return refuse("the capacity is a multiple of the block, at most 2^30");
    if (c.code != SWLM_KV8_INT8 && c.code != SWLM_KV8_E4M3) return refuse("unknown code");
    return SWLM_OK;
}
int cache_ok(const swlm_kv8_cache& c) {
    const int rc = cache_shape_ok(c);
    if (rc) return rc;
    if (!c.k || !c.v || !c.k_scale || !c.v_scale) return refuse("null cache array");
    if (!aligned(c.k, 16) || !aligned(c.v, 16)) return refuse("codes must be 16-byte aligned");
    if (!aligned(c.k_scale, 4) || !aligned(c.v_scale, 4) || !aligned(c.weight, 4) || !aligned(c.slot_pos, 4)) return refuse("scales, weights and positions must be 4-byte aligned");
    return SWLM_OK;
}
int counters_ok(const int32_t* lengths, const int32_t* counts, const int32_t* starts, const int32_t* seen) {
    if (!lengths) return refuse("null lengths");
    if (!aligned(lengths, 4) || !aligned(counts, 4) || !aligned(starts, 4) || !aligned(seen, 4)) return refuse("counters must be 4-byte aligned");
    return SWLM_OK;
}
int step_ok(int dtype, int n, int rows) {
    if (dtype != SWLM_KV8_BF16 && dtype != SWLM_KV8_FP16) return refuse("unknown dtype");
    if (n < 1 || n > kKv8MaxLen / 2 || rows < 0) return refuse("tokens or rows out of range");
    return SWLM_OK;
}
bool rows_ok(const void* p, int64_t stride, int64_t width) { return aligned(p, 16) && stride >= width && stride % 8 == 0 && stride <= (int64_t)1 << 40; }

int attend_shape_ok(const swlm_kv8_cache& c, const swlm_kv8_attend& a) {
    int rc = cache_shape_ok(c);
    if (rc || (rc = step_ok(a.dtype, a.n, a.rows))) return rc;
    if (a.heads < 1 || a.heads % c.kv_heads) { set_error("kv8: %d query heads do not divide by %d KV heads", a.heads, c.kv_heads); return SWLM_ERR_INVALID; }
    if ((int64_t)a.n * (a.heads / c.kv_heads) > kKv8MaxLen) return refuse("too many query rows");
    if (a.max_len < 1 || a.max_len > kKv8MaxLen) return refuse("max_len out of range");
    if (a.probabilities != SWLM_KV8_P_BY_TYPE && a.probabilities != SWLM_KV8_P_ONE && a.probabilities != SWLM_KV8_P_TWO) return refuse("unknown form of the probabilities");
    if (!kv8_attend_grid_fits(c, a)) return refuse("too many query rows");
    return SWLM_OK;
}

struct Range { uintptr_t from, to; };
void ranges_of(const swlm_kv8_cache& c, Range* r) {
    const size_t heads = (size_t)c.batch * c.kv_heads, codes = heads * c.capacity * c.head_dim, scales = heads * (c.capacity / c.block) * 4, slots = heads * c.capacity * 4;
    const void* p[6] = {c.k, c.v, c.k_scale, c.v_scale, c.weight, c.slot_pos};
    const size_t n[6] = {codes, codes, scales, scales, slots, slots};
    for (int i = 0; i < 6; ++i) r[i] = {reinterpret_cast<uintptr_t>(p[i]), reinterpret_cast<uintptr_t>(p[i]) + n[i]};
}

int evict_shape_ok(const swlm_kv8_cache& c, const swlm_kv8_evict& a) {
    const int rc = cache_shape_ok(c);
    if (rc) return rc;
    if (a.keep < 1 || a.keep > kKv8MaxLen || a.sink < 0 || a.recent < 0 || (int64_t)a.sink + a.recent > a.keep) return refuse("keep is positive and at least sink + recent, neither of them negative");
    if (a.max_len < 1 || a.max_len > kKv8MaxLen) return refuse("max_len out of range");
    return SWLM_OK;
}

// (`code`: what the kernels left in the context's word)
int expired(int code) {
    if (!code) return SWLM_OK;
    set_error("kv8: a bounded device-side wait of an earlier attention call expired (code %d): results since then are not valid", code);
    return SWLM_ERR_TIMEOUT;
}

cudaStream_t stream_of(swlm_ctx* ctx, void* s) { return s ? static_cast<cudaStream_t>(s) : ctx->stream; }

}  // namespace

extern "C" {

int swlm_op_kv8_append_dev(swlm_ctx* ctx, const swlm_kv8_cache* cache, const swlm_kv8_append* step, void* cuda_stream) {
    if (!ctx || !cache || !step || !step->k || !step->v) return refuse("null argument");
    const swlm_kv8_cache& c = *cache;
    const swlm_kv8_append& a = *step;
    int rc = cache_ok(c);
    if (rc || (rc = step_ok(a.dtype, a.n, a.rows)) || (rc = counters_ok(a.lengths, a.counts, a.starts, a.seen))) return rc;
    if (!aligned(a.refused, 4)) return refuse("counters must be 4-byte aligned");
    if (c.slot_pos && !a.seen) return refuse("a cache with slot_pos needs seen");
    const int64_t width = (int64_t)c.kv_heads * c.head_dim;
    if (!rows_ok(a.k, a.k_stride, width) || !rows_ok(a.v, a.v_stride, width)) return refuse("k and v must be 16-byte aligned, their strides multiples of 8 and at least kv_heads * head_dim");
    SWLM_CUDA(cudaSetDevice(ctx->device));
    return launch_kv8_append(c, a, stream_of(ctx, cuda_stream));
}

size_t swlm_op_kv8_attend_scratch_bytes(const swlm_kv8_cache* cache, const swlm_kv8_attend* step) {
    if (!cache || !step || attend_shape_ok(*cache, *step)) return 0;
    return kv8_attend_scratch(*cache, *step);
}

int swlm_op_kv8_attend_dev(swlm_ctx* ctx, const swlm_kv8_cache* cache, const swlm_kv8_attend* step, void* cuda_stream) {
    if (!ctx || !cache || !step || !step->q || !step->out) return refuse("null argument");
    const swlm_kv8_cache& c = *cache;
    const swlm_kv8_attend& a = *step;
    int rc = cache_ok(c);
    if (rc || (rc = attend_shape_ok(c, a)) || (rc = counters_ok(a.lengths, a.counts, a.starts, nullptr))) return rc;
    const int64_t width = (int64_t)a.heads * c.head_dim;
    if (!rows_ok(a.q, a.q_stride, width) || !rows_ok(a.out, a.out_stride, width)) return refuse("q and out must be 16-byte aligned, their strides multiples of 8 and at least heads * head_dim");
    if (!(a.scale > 0.f) || a.scale > 1e30f) return refuse("the scale must be positive and finite");
    if (a.accumulate && !c.weight) return refuse("accumulate needs the cache's weight array");
    if (!aligned(a.refused, 4)) return refuse("counters must be 4-byte aligned");
    const size_t need = kv8_attend_scratch(c, a);
    if (need && (!a.scratch || !aligned(a.scratch, 16) || a.scratch_bytes < need)) { set_error("kv8: %zu bytes of 16-byte aligned scratch are needed", need); return SWLM_ERR_INVALID; }
    SWLM_CUDA(cudaSetDevice(ctx->device));
    if ((rc = expired(__atomic_load_n(ctx->kv8_status, __ATOMIC_RELAXED)))) return rc;
    return launch_kv8_attend(c, a, ctx->kv8_status, stream_of(ctx, cuda_stream));
}

int swlm_op_kv8_status(swlm_ctx* ctx) {
    if (!ctx) return refuse("null argument");
    return expired(__atomic_exchange_n(ctx->kv8_status, 0, __ATOMIC_RELAXED));
}

int swlm_write_kv8_status(swlm_ctx* ctx, int code) {
    if (!ctx) return refuse("null argument");
    __atomic_store_n(ctx->kv8_status, code, __ATOMIC_RELAXED);
    return SWLM_OK;
}

size_t swlm_op_kv8_evict_scratch_bytes(const swlm_kv8_cache* cache, const swlm_kv8_evict* how) {
    if (!cache || !how || evict_shape_ok(*cache, *how)) return 0;
    return kv8_evict_scratch(*cache, *how);
}

int swlm_op_kv8_evict_dev(swlm_ctx* ctx, const swlm_kv8_cache* cache, const swlm_kv8_cache* to, const swlm_kv8_evict* how, void* cuda_stream) {
    if (!ctx || !cache || !to || !how) return refuse("null argument");
    const swlm_kv8_cache &c = *cache, &d = *to;
    const swlm_kv8_evict& a = *how;
    int rc = cache_ok(c);
    if (rc || (rc = cache_ok(d)) || (rc = evict_shape_ok(c, a)) || (rc = counters_ok(a.lengths, nullptr, nullptr, a.seen))) return rc;
    if (!a.seen) return refuse("null seen");
    if (!c.weight || !c.slot_pos || !d.weight || !d.slot_pos) return refuse("eviction needs weight and slot_pos of both caches");
    if (c.batch != d.batch || c.kv_heads != d.kv_heads || c.head_dim != d.head_dim || c.block != d.block || c.code != d.code) return refuse("the two caches differ in shape or code");
    const bool same = c.k == d.k && c.v == d.v && c.k_scale == d.k_scale && c.v_scale == d.v_scale && c.weight == d.weight && c.slot_pos == d.slot_pos;
    if (same ? c.capacity != d.capacity : d.capacity < std::min(a.keep, std::min(a.max_len, c.capacity))) return refuse("the second cache has no room for the tokens that stay");
    if (!same) {
        Range x[6], y[6];
        ranges_of(c, x);
        ranges_of(d, y);
        for (const Range& i : x)
            for (const Range& j : y)
                if (i.from < j.to && j.from < i.to) return refuse("the two caches share some memory but are not the same");
    }
    const size_t need = kv8_evict_scratch(c, a);
    if (!a.scratch || !aligned(a.scratch, 16) || a.scratch_bytes < need) { set_error("kv8: %zu bytes of 16-byte aligned scratch are needed", need); return SWLM_ERR_INVALID; }
    SWLM_CUDA(cudaSetDevice(ctx->device));
    if ((rc = expired(__atomic_load_n(ctx->kv8_status, __ATOMIC_RELAXED)))) return rc;   // the weights that it would go by may not be valid
    return launch_kv8_evict(c, d, a, stream_of(ctx, cuda_stream));
}

int swlm_op_kv8_lengths_dev(swlm_ctx* ctx, int batch, const int32_t* in, const int32_t* counts, int n, int limit, const int32_t* refused,
                            int32_t* out, void* cuda_stream) {
    if (!ctx || !in || !out) return refuse("null argument");
    if (batch < 1 || batch > kKv8MaxBatch) return refuse("batch out of range");
    if (!aligned(in, 4) || !aligned(counts, 4) || !aligned(refused, 4) || !aligned(out, 4)) return refuse("counters must be 4-byte aligned");
    SWLM_CUDA(cudaSetDevice(ctx->device));
    return launch_kv8_lengths(batch, in, counts, n, limit, refused, out, stream_of(ctx, cuda_stream));
}

}  // extern "C"
