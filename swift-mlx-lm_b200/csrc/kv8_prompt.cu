// Attention of many query rows over a cache of 8-bit codes (prompt portions), on the 5th-generation tensor cores (tcgen05 / TMEM).
//
// A CTA has 256 rows in two tiles of 128, rows being the queries of a sequence times the heads of a group, and a run of its slots. Codes become fp16
// numbers on their way to shared memory, queries are shifted to fp16 (both exact, see kv8_attend.cu), so that scores are one product with fp32
// sums; a tile's scores take the factor of their block, probabilities that of the values' block over the largest so far (2^7 times, as fp16
// or as two fp16 numbers, whose products follow one another: 3 x 777 rows with weights, heads of 64, 147 us, with one 136; 2048 over 6144 361 and 276).
//
// Roles: three warps bring keys and values from the cache, convert them and store them in the swizzled layout of the products' operands (two
// slots of 128 tokens each, which both row tiles read); a warp issues the MMAs (O += P V, then S = Q K^T of the next key tile, for one row tile
// and the other in turn); eight warps do the softmax, a thread per row. Probabilities take the place of their scores in tensor memory
// and are read there as the A operand. The reference maximum of a row moves only when it would grow by more than 2^8.
//
// What bounds it (2048 tokens over 6144, 32 / 8 heads of 128: 278 us, 865 TFLOP/s, 0.53 of the measured rate): the chain of a row tile, softmax (two
// warps of a scheduler share the exponential unit, 2048 clocks a tile), product, next scores, of which the other row tile fills the gaps only
// in part; and 256 CTAs on 148 SMs. Steps to here: one row tile per CTA, two CTAs per SM 732 us; the loaders' first warp
// issuing the MMAs, paired fp32 operations 391; two row tiles that share the conversions, a warp for the MMAs 306; key tiles of 128 instead of 64
// with two score regions 297; the longest rows of all heads first 278.
#include <algorithm>
#include <type_traits>

#include "kv8_device.cuh"
#include "tc_attention.cuh"

namespace swlm {
using namespace kv8;
namespace {

constexpr int kTiles = kPromptRows / kPaRows;   // row tiles of a CTA
static_assert(kTiles == 2, "tensor memory holds two row tiles");
constexpr int kSoftmaxWarps = 4 * kTiles, kMmaWarp = kSoftmaxWarps, kLoadWarps = 3;
constexpr int kPromptThreads = (kSoftmaxWarps + 1 + kLoadWarps) * 32;   // (with 13 warps a thread would have 128 registers and not 168: 456 us, spilled)
constexpr int kSlots = 2;               // key and value tiles in shared memory
constexpr float kFoldUnit = 0x1p-20f;   // value scales down to this part of the largest go into the exponent

// Phases (a wait by parity cannot tell a phase from the one two before it), for key tile j and row tile t; all are waited for phase by phase:
//   k_full, v_full [j & 1]   by the MMA warp
//   k_free, v_free [j & 1]   by the loaders, before tile j + 2
//   s_full[t]                by the row tile's softmax warps. The scores of tile j are issued behind pv_done(j - 1), so that behind it the output may be scaled
//   p_ready[t], pv_done[t]   by the MMA warp
//   q_ready, o_done          have one phase
struct PromptBars {
    unsigned long long q_ready, o_done, k_full[kSlots], v_full[kSlots], k_free[kSlots], v_free[kSlots], s_full[kTiles], p_ready[kTiles], pv_done[kTiles];
    unsigned tmem;
    int failed;
};

template <int HD> __host__ __device__ constexpr size_t prompt_smem() { return (size_t)kPromptRows * HD * 2 + 2 * kSlots * kPromptKeys * HD * 2 + 1024; }

// GROUPS: scales of a key tile (blocks of 16, 32, 64 or 128 tokens: 8, 4, 2, 1)
// TWO: probabilities meet the values as two fp16 numbers. Of 16 probabilities the columns of their scores hold the fp16 numbers (8 columns) and what rounding has
// left (8); else the numbers alone, those of a tile in the first 64 of its 128 columns.
template <int HD, int CODE, int GROUPS, bool TWO>
__global__ void __launch_bounds__(kPromptThreads, 1) kv8_prompt_kernel(const swlm_kv8_cache c, const swlm_kv8_attend a, const RowsPlan p, int* status) {
    constexpr int HALVES = HD / 64;                        // 128-byte halves of a row
    constexpr unsigned Q_HALF = kPaRows * 128, Q_BYTES = HALVES * Q_HALF, KV_HALF = kPromptKeys * 128, KV_BYTES = HALVES * KV_HALF;
    constexpr unsigned kTmemCols = 512, O_COL = 256;       // scores / probabilities of row tile t from 128 t on, output from 256 + 128 t on
    extern __shared__ __align__(1024) unsigned char prompt_raw[];
    unsigned char* const sm = prompt_raw + ((1024 - (smem_u32(prompt_raw) & 1023)) & 1023);
    unsigned char *const q_sm = sm, *const k_sm = sm + kTiles * Q_BYTES, *const v_sm = k_sm + kSlots * KV_BYTES;
    __shared__ __align__(8) PromptBars bars;
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int G = a.heads / c.kv_heads, span = min(a.max_len, c.capacity);
    // The longest rows first, of all heads, so that the last round of CTAs is of the shortest (2048 tokens into an empty cache, 32 / 8 heads of 128: 72 us, head
    // by head 94); sequence by sequence, as only the device knows which one is long
    const int turn = (int)blockIdx.x / c.kv_heads, h = (int)blockIdx.x - turn * c.kv_heads, split = turn % p.splits;
    const int b = turn / p.splits / p.row_tiles, block = p.row_tiles - 1 - (turn / p.splits - b * p.row_tiles);
    const Kv8Part part = kv8_part(b, a.lengths, a.counts, a.starts, a.refused, a.n, a.rows);
    const int rows = part.count * G, block0 = block * kPromptRows;
    if (block0 >= rows) return;
    const int end = visible(part, min(block0 + kPromptRows - 1, rows - 1) / G, span);   // of the CTA's last query: it sees most
    const int key_lo = split * p.chunk;
    if (split > 0 && key_lo >= end) return;
    // key tiles of either row tile (its last query's); the second one has as many as the first or more, or none where it has no rows
    auto tiles_of = [&](int t) {
        const int first = block0 + t * kPaRows;
        return first < rows ? (max(min(visible(part, min(first + kPaRows - 1, rows - 1) / G, span) - key_lo, p.chunk), 0) + kPromptKeys - 1) / kPromptKeys : 0;
    };
    const int tiles0 = tiles_of(0), tiles1 = tiles_of(1), n_tiles = max(tiles0, tiles1);
    const size_t head = (size_t)b * c.kv_heads + h;
    const int block_shift = 31 - __clz(c.block);
    volatile int* const failed = &bars.failed;
    auto fail = [&](int code) { atomicExch_system(status, code); *failed = 1; };

    if (tid == 0) {
        mbar_init(&bars.q_ready, kSoftmaxWarps);
        mbar_init(&bars.o_done, 1);
        for (int i = 0; i < kSlots; ++i) {
            mbar_init(&bars.k_full[i], kLoadWarps);
            mbar_init(&bars.v_full[i], kLoadWarps);
            mbar_init(&bars.k_free[i], 1);
            mbar_init(&bars.v_free[i], 1);
        }
        for (int t = 0; t < kTiles; ++t) {
            mbar_init(&bars.s_full[t], 1);
            mbar_init(&bars.p_ready[t], 4);
            mbar_init(&bars.pv_done[t], 1);
        }
        bars.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pa_before();
    __syncthreads();
    pa_after();
    const unsigned tm = bars.tmem;

    if (warp > kMmaWarp) {
        // ---- keys and values: codes in, fp16 out ------------------------------------------------------------------------------------------------
        // A turn of a warp: 32 pieces of 16 bytes, that is ROWS tokens; its lanes are four pieces of a token's half, two tokens, (the halves,) ... The
        // eight lanes of a phase of the stores below then meet different banks. Warp w has turns w, w + 3, ...
        constexpr int ROWS = 512 / HD, TURNS = kPromptKeys / ROWS, PER = (TURNS + kLoadWarps - 1) / kLoadWarps, STEP = kLoadWarps * ROWS;
        const int w = warp - kMmaWarp - 1;
        const int piece = (lane & 3) + (HD == 128 ? (lane >> 3 & 1) * 4 : 0), key = w * ROWS + (HD == 128 ? (lane >> 4) * 2 + (lane >> 2 & 1) : lane >> 2);   // key, key + STEP, ...
        const size_t at = (head * c.capacity + key_lo + key) * HD + piece * 16;
        const unsigned char* kg = static_cast<const unsigned char*>(c.k) + at;
        const unsigned char* vg = static_cast<const unsigned char*>(c.v) + at;
        uint4 kr[PER], vr[PER];
        auto load = [&](const unsigned char* src, uint4 (&r)[PER], int j) {
            const int slot = key_lo + j * kPromptKeys + key;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                r[i] = key + i * STEP < kPromptKeys && slot + i * STEP < end ? *reinterpret_cast<const uint4*>(src + i * STEP * HD) : make_uint4(0, 0, 0, 0);   // (nothing that may be NaN)
        };
        const unsigned off = (piece >> 2) * KV_HALF + key * 128, off0 = off + (((piece * 2 & 7) ^ (key & 7)) << 4), off1 = off + (((piece * 2 & 7 | 1) ^ (key & 7)) << 4);
        auto store = [&](unsigned char* dst, const uint4 (&r)[PER]) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (key + i * STEP >= kPromptKeys) continue;
                const unsigned flip = (i * STEP & 4) << 4;   // (of the swizzle, where a step is an odd number of fours)
                const unsigned w[4] = {prepared<CODE>(r[i].x), prepared<CODE>(r[i].y), prepared<CODE>(r[i].z), prepared<CODE>(r[i].w)};
                *reinterpret_cast<uint4*>(dst + (off0 ^ flip) + i * STEP * 128) = make_uint4(pair_of<CODE, 0>(w[0]), pair_of<CODE, 1>(w[0]), pair_of<CODE, 0>(w[1]), pair_of<CODE, 1>(w[1]));
                *reinterpret_cast<uint4*>(dst + (off1 ^ flip) + i * STEP * 128) = make_uint4(pair_of<CODE, 0>(w[2]), pair_of<CODE, 1>(w[2]), pair_of<CODE, 0>(w[3]), pair_of<CODE, 1>(w[3]));
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
        };
        bool ok = true;
        if (n_tiles) { load(kg, kr, 0); load(vg, vr, 0); }
        for (int j = 0; j < n_tiles; ++j) {
            const int slot = j & 1, round = j >> 1;
            kg += kPromptKeys * HD;
            vg += kPromptKeys * HD;
            if (*failed || (round > 0 && !mbar_wait_warp(&bars.k_free[slot], (unsigned)((round - 1) & 1)))) { ok = false; break; }
            store(k_sm + slot * KV_BYTES, kr);
            if (lane == 0) pa_arrive(&bars.k_full[slot]);
            if (j + 1 < n_tiles) load(kg, kr, j + 1);
            if (round > 0 && !mbar_wait_warp(&bars.v_free[slot], (unsigned)((round - 1) & 1))) { ok = false; break; }
            store(v_sm + slot * KV_BYTES, vr);
            if (lane == 0) pa_arrive(&bars.v_full[slot]);
            if (j + 1 < n_tiles) load(vg, vr, j + 1);
        }
        if (!ok && lane == 0) fail(31);
        __syncwarp();
    } else if (warp == kMmaWarp) {
        const bool el = elect_one();
        const unsigned qd = umma_desc_lo(smem_u32(q_sm)), kd = umma_desc_lo(smem_u32(k_sm)), vd = pa_desc_mn_lo(smem_u32(v_sm), KV_HALF);
        auto scores = [&](int slot, int t) {
            if (el) {
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk)
                    pa_mma_ss(tm + t * 128u, qd + t * (Q_BYTES / 16) + (kk >> 2) * (Q_HALF / 16) + 2 * (kk & 3), kd + slot * (KV_BYTES / 16) + (kk >> 2) * (KV_HALF / 16) + 2 * (kk & 3),
                              pa_idesc(kPromptKeys, false, false), kk > 0 ? 1u : 0u);
                umma_commit(&bars.s_full[t]);
            }
            __syncwarp();
        };
        auto release = [&](unsigned long long* bar) {   // behind everything issued so far
            if (el) umma_commit(bar);
            __syncwarp();
        };
        bool ok = true;
        if (n_tiles) {
            ok = mbar_wait_warp(&bars.q_ready, 0u) && mbar_wait_warp(&bars.k_full[0], 0u);
            if (ok) {
                pa_after();
                for (int t = 0; t < kTiles; ++t)
                    if ((t ? tiles1 : tiles0) > 0) scores(0, t);
                release(&bars.k_free[0]);
            }
        }
        for (int j = 0; j < n_tiles && ok; ++j) {
            const int slot = j & 1, next = slot ^ 1;
            const unsigned phase = (unsigned)((j >> 1) & 1), next_phase = (unsigned)(((j + 1) >> 1) & 1);
            if (!mbar_wait_warp(&bars.v_full[slot], phase) || (j + 1 < n_tiles && !mbar_wait_warp(&bars.k_full[next], next_phase))) { ok = false; break; }
            for (int t = 0; t < kTiles && ok; ++t) {
                const int mine = t ? tiles1 : tiles0;
                if (j >= mine) continue;
                if (!mbar_wait_warp(&bars.p_ready[t], (unsigned)(j & 1))) { ok = false; break; }
                pa_after();
                if (el) {
#pragma unroll
                    for (int kk = 0; kk < kPromptKeys / 16; ++kk)
#pragma unroll
                        for (int rest = 0; rest < (TWO ? 2 : 1); ++rest)
                            pa_mma_ts(tm + O_COL + t * 128u, tm + t * 128u + (TWO ? 16u : 8u) * kk + 8u * rest, vd + slot * (KV_BYTES / 16) + kk * (2048 / 16), pa_idesc(HD, true, false),
                                      kk > 0 || rest > 0 || j > 0 ? 1u : 0u);
                    umma_commit(&bars.pv_done[t]);
                }
                __syncwarp();
                if (j + 1 < mine) {   // its scores take the place of the probabilities that the product reads
                    if (!mbar_wait_warp(&bars.pv_done[t], (unsigned)(j & 1))) { ok = false; break; }
                    pa_after();
                    scores(next, t);
                }
            }
            if (!ok) break;
            release(&bars.v_free[slot]);
            if (j + 1 < n_tiles) release(&bars.k_free[next]);
        }
        if (el) umma_commit(&bars.o_done);   // also behind whatever was issued before a failure
        __syncwarp();
        ok = mbar_wait_warp(&bars.o_done, 0u) && ok;   // tensor memory is not freed under MMAs in flight
        if (!ok && lane == 0) fail(32);
        __syncwarp();
    } else {
        const int t = warp >> 2, r = tid & (kPaRows - 1), row = block0 + tid, i = min(row, rows - 1) / G, tiles = t ? tiles1 : tiles0;   // r: of the row tile
        const bool row_ok = row < rows, f16 = a.dtype == SWLM_KV8_FP16;
        const int limit = visible(part, i, span);   // (rows past the last one attend what it does; they are not stored)
        float factor;
        // ---- q: this thread's row, shifted to fp16 ----------------------------------------------------------------------------------------
        {
            const unsigned short* src = static_cast<const unsigned short*>(a.q) + (int64_t)(part.start + i) * a.q_stride + (size_t)(h * G + min(row, rows - 1) - i * G) * HD;
            unsigned top = 0;   // largest |value| as its 15 bits
#pragma unroll 4
            for (int d = 0; d < HD; d += 8) {
                const uint4 v = *reinterpret_cast<const uint4*>(src + d);
                const unsigned m = __vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu), __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
                top = max(top, max(m & 0xFFFFu, m >> 16));
            }
            const bool keeps = p.q16 && split == 0;   // for the launch that adds the weights
            float up;
            row_shift(f16 ? __half2float(__ushort_as_half((unsigned short)top)) : __uint_as_float(top << 16), up, factor);
            factor *= a.scale * kLog2e;
#pragma unroll 4
            for (int d = 0; d < HD; d += 8) {
                float x[8];
                widen(*reinterpret_cast<const uint4*>(src + d), f16, x);
                uint4 v;
                v.x = pack_half(x[0] * up, x[1] * up); v.y = pack_half(x[2] * up, x[3] * up);
                v.z = pack_half(x[4] * up, x[5] * up); v.w = pack_half(x[6] * up, x[7] * up);
                const int at = r * 128 + ((((d >> 3) & 7) ^ (r & 7)) << 4);
                *reinterpret_cast<uint4*>(q_sm + t * Q_BYTES + (d >> 6) * Q_HALF + at) = v;
                if (keeps) *reinterpret_cast<uint4*>(reinterpret_cast<unsigned char*>(p.q16) + (((head * p.row_tiles + block) * (kPromptRows / 64) + (tid >> 6)) * HALVES + (d >> 6)) * 8192 + (at & 8191)) = v;
            }
            if (keeps) p.q_factor[(head * p.row_tiles + block) * kPromptRows + tid] = row_ok ? factor : 0.f;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) pa_arrive(&bars.q_ready);
        }
        // ---- softmax, a thread per row -------------------------------------------------------------------------------------------------------
        const unsigned lanes = (unsigned)((warp & 3) * 32) << 16, out_col = tm + lanes + O_COL + t * 128u;
        const float* ks = c.k_scale + head * (c.capacity >> block_shift);
        const float* vs = c.v_scale + head * (c.capacity >> block_shift);
        float m_ref = -INFINITY, l_run = 0.f, v_ref = kValueRef, v_inv = kValueUnit / kValueRef;
        constexpr int KEYS = kPromptKeys / GROUPS;            // keys of a scale
        constexpr int PARTS = KEYS < 64 ? 64 / KEYS : 1, N = 64 / PARTS;   // scales of half a tile, keys of it that share one
        float kn[GROUPS], vn[GROUPS];   // the next tile's scales; 0 behind the last token
        auto scales = [&](int j) {
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                const int slot = key_lo + j * kPromptKeys + g * KEYS;
                kn[g] = slot < end ? ks[slot >> block_shift] : 0.f;
                vn[g] = slot < end ? vs[slot >> block_shift] : 0.f;
            }
        };
        if (tiles) scales(0);
        bool ok = true;
        const unsigned region = tm + lanes + t * 128u;
        for (int j = 0; j < tiles; ++j) {
            float fk[GROUPS], vt[GROUPS];
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) { fk[g] = factor * kn[g]; vt[g] = vn[g]; }
            if (j + 1 < tiles) scales(j + 1);
            if (!mbar_wait_warp(&bars.s_full[t], (unsigned)(j & 1))) { ok = false; break; }
            pa_after();
            const int key0 = key_lo + j * kPromptKeys;
            const bool masked = !__all_sync(0xffffffffu, key0 + kPromptKeys <= limit);
            // A thread has no room for a tile's 128 scores: the halves are read for the largest one, and again for the probabilities
            float top = -INFINITY;
            unsigned v[64];
#pragma unroll
            for (int half = 1; half >= 0; --half) {
                pa_ld32(region + half * 64u, v);
                pa_ld32(region + half * 64u + 32u, v + 32);
                pa_wait_ld();
#pragma unroll
                for (int g = 0; g < PARTS; ++g) {
                    float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};   // (four chains)
                    if (masked) {
#pragma unroll
                        for (int e = 0; e < N; ++e) most[e & 3] = fmaxf(most[e & 3], key0 + half * 64 + g * N + e < limit ? __uint_as_float(v[g * N + e]) : -INFINITY);
                    } else {
#pragma unroll
                        for (int e = 0; e < N; ++e) most[e & 3] = fmaxf(most[e & 3], __uint_as_float(v[g * N + e]));
                    }
                    const float x = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
                    if (x > -INFINITY) top = fmaxf(top, x * fk[(half * 64 + g * N) / KEYS]);   // (factors are not negative: the largest score stays the largest)
                }
            }
            const bool moves = top > m_ref + kSlack;
            float v_top = vt[0];
#pragma unroll
            for (int g = 1; g < GROUPS; ++g) v_top = fmaxf(v_top, vt[g]);
            if (__any_sync(0xffffffffu, moves || v_top > v_ref)) {
                float corr = moves ? pa_exp2(m_ref - top) : 1.f;   // 0 for a row's first keys
                if (moves) { m_ref = top; l_run *= corr; }
                if (v_top > v_ref) { corr *= v_ref / v_top; v_ref = v_top; v_inv = kValueUnit / v_top; }
                if (j > 0) {   // the output so far is complete, and the next product waits for this warp
#pragma unroll 1
                    for (int d = 0; d < HD; d += 16) {
                        unsigned o[16];
                        pa_ld16(out_col + d, o);
                        pa_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                        pa_st16(out_col + d, o);
                    }
                }
            }
            const float base = m_ref == -INFINITY ? 0.f : m_ref;   // nothing attended so far: all probabilities 0
            float unit[GROUPS];
            bool folds = !masked;
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                unit[g] = vt[g] * v_inv;
                folds = folds && unit[g] >= kFoldUnit * kValueUnit;
            }
            // Probabilities of a half take the place of its own scores (TWO), or those of the first half that of its first 32 columns and those of the second that of
            // the next 32. `put`: the e-th pair of 16 scores, which all have been read when the first is written
            auto put = [&](unsigned (&out)[16], int e, float x, float y) {
                out[e] = pack_half(x, y);
                if (TWO) out[8 + e] = pack_rest(x, y, out[e]);
            };
            auto keep = [&](const unsigned (&out)[16], int at) {
#pragma unroll
                for (int e = 0; e < (TWO ? 16 : 8); ++e) v[TWO ? at + e : at / 2 + e] = out[e];
            };
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if (half) {   // (the first half is what was read last)
                    pa_ld32(region + 64u, v);
                    pa_ld32(region + 96u, v + 32);
                    pa_wait_ld();
                }
                if (folds) {
                    // the unit goes into the exponent, and out of the sum again
#pragma unroll
                    for (int g = 0; g < PARTS; ++g) {
                        const int at = (half * 64 + g * N) / KEYS;
                        const float shift = log2_of(unit[at]) - base;
                        const float2 fk2 = make_float2(fk[at], fk[at]), shift2 = make_float2(shift, shift);
                        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                        for (int e0 = 0; e0 < N; e0 += 16) {
                            unsigned out[16];
#pragma unroll
                            for (int e = 0; e < 16; e += 2) {
                                const int i = g * N + e0 + e;
                                float2 x = fma2(make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), fk2, shift2);
                                x = make_float2(pa_exp2(x.x), pa_exp2(x.y));
                                sum[e >> 1 & 1] = add2(sum[e >> 1 & 1], x);
                                put(out, e / 2, x.x, x.y);
                            }
                            keep(out, g * N + e0);
                        }
                        const float2 all = add2(sum[0], sum[1]);
                        l_run += __fdividef(all.x + all.y, unit[at]);
                    }
                } else {
#pragma unroll
                    for (int g = 0; g < PARTS; ++g) {
                        const int at = (half * 64 + g * N) / KEYS;
#pragma unroll
                        for (int e0 = 0; e0 < N; e0 += 16) {
                            unsigned out[16];
#pragma unroll
                            for (int e = 0; e < 16; e += 2) {
                                float w[2];
#pragma unroll
                                for (int k = 0; k < 2; ++k) {
                                    const int i = g * N + e0 + e + k;
                                    const bool sees = key0 + half * 64 + i < limit;   // (what a row does not attend may lie in a block that is NaN)
                                    const float x = sees ? pa_exp2(fmaf(__uint_as_float(v[i]), fk[at], -base)) : 0.f;
                                    l_run += x;
                                    w[k] = sees ? x * unit[at] : 0.f;
                                }
                                put(out, e / 2, w[0], w[1]);
                            }
                            keep(out, g * N + e0);
                        }
                    }
                }
                pa_st32(region + half * (TWO ? 64u : 32u), v);
                if (TWO) pa_st32(region + half * 64u + 32u, v + 32);
            }
            pa_wait_st();
            pa_before();
            __syncwarp();
            if (lane == 0) pa_arrive(&bars.p_ready[t]);
        }
        if (ok && (!mbar_wait_warp(&bars.o_done, 0u) || *failed)) ok = false;
        if (!ok) fail(33);
        __syncwarp();
        pa_after();
        if (ok) {
            const bool whole = end <= p.chunk;   // this CTA has all of the tile's slots
            const size_t at = ((head * p.row_tiles + block) * p.splits + split) * kPromptRows + tid;
            const float unit = v_ref * (1.f / kValueUnit);
            if (row_ok && !whole) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m_ref, l_run);
            if (p.q_shift && (whole || !row_ok)) p.q_shift[(head * p.row_tiles + block) * kPromptRows + tid] = row_ok ? row_shift_of(m_ref, l_run) : -INFINITY;
            unsigned short* dst = static_cast<unsigned short*>(a.out) + (int64_t)(part.start + i) * a.out_stride + (size_t)(h * G + min(row, rows - 1) - i * G) * HD;
#pragma unroll 1
            for (int d = 0; d < HD; d += 16) {
                unsigned o[16] = {};
                if (tiles) {
                    pa_ld16(out_col + d, o);
                    pa_wait_ld();
                }
                if (row_ok)
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const float4 x = make_float4(__uint_as_float(o[e]) * unit, __uint_as_float(o[e + 1]) * unit, __uint_as_float(o[e + 2]) * unit, __uint_as_float(o[e + 3]) * unit);
                        if (whole) store_out(dst + d + e, x, l_run, f16);
                        else *reinterpret_cast<float4*>(p.part_o + at * HD + d + e) = x;
                    }
            }
        }
    }
    pa_before();
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(kTmemCols) : "memory");
}

// The weights of many rows: weight_j += sum over rows i of exp2(s_ij + shift_i), with the rows' totals known. A CTA has 128 keys, the rows of the products
// (S^T = K Q^T: a thread per key, so that nothing is added across threads), and walks the row tiles that attend them. The
// queries of a tile, their factors and shifts come as bulk copies, SLOTS - 1 tiles ahead, while the tiles before are multiplied and summed; scores have two
// regions. Three CTAs of an SM fill each other's waits (3 x 777 rows, heads of 64, both kernels, one product of the probabilities: 136 us, with two CTAs 160; 2048
// over 6144, heads of 128: 507 and 524).
// With heads of 128 they have room for two slots only, and where there are no three CTAs per SM four are faster (2048 into an empty cache 177 us, with two slots 185).
constexpr int kWeightKeys = 128, kWeightRows = 64, kWeightSlots = 4, kWeightThreads = kWeightKeys + 32;
struct WeightBars {
    unsigned long long k_ready, o_done, q_full[kWeightSlots], s_full[2], s_free[2];
    unsigned tmem;
    int failed;
};
template <int HD, int SLOTS> __host__ __device__ constexpr size_t weights_smem() { return (size_t)kWeightKeys * HD * 2 + (size_t)SLOTS * kWeightRows * HD * 2 + 1024; }

template <int HD, int CODE, int SLOTS>
__global__ void __launch_bounds__(kWeightThreads, 3) kv8_weights_kernel(const swlm_kv8_cache c, const swlm_kv8_attend a, const RowsPlan p, int* status) {
    constexpr int HALVES = HD / 64;
    constexpr unsigned K_HALF = kWeightKeys * 128, Q_HALF = kWeightRows * 128, Q_BYTES = HALVES * Q_HALF;
    constexpr unsigned kTmemCols = 128;   // two regions of scores
    static_assert((SLOTS & (SLOTS - 1)) == 0 && SLOTS >= 2 && SLOTS <= kWeightSlots, "slots");
    extern __shared__ __align__(1024) unsigned char weights_raw[];
    unsigned char* const k_sm = weights_raw + ((1024 - (smem_u32(weights_raw) & 1023)) & 1023);
    unsigned char* const q_sm = k_sm + HALVES * K_HALF;
    __shared__ __align__(16) float rows_sm[SLOTS][2][kWeightRows];   // factors, shifts
    __shared__ __align__(8) WeightBars bars;
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int b = blockIdx.z, h = blockIdx.y, G = a.heads / c.kv_heads, span = min(a.max_len, c.capacity);
    const Kv8Part part = kv8_part(b, a.lengths, a.counts, a.starts, a.refused, a.n, a.rows);
    const int rows = part.count * G, end = rows ? visible(part, part.count - 1, span) : 0, key0 = (int)blockIdx.x * kWeightKeys;
    if (key0 >= end) return;
    const size_t head = (size_t)b * c.kv_heads + h;
    // rows from (key - length) * G on attend a key; the first tile with one that attends this CTA's first key
    const int tile0 = (int)(max((long long)key0 - part.len, 0LL) * G / kWeightRows), tiles = (rows + kWeightRows - 1) / kWeightRows - tile0;
    volatile int* const failed = &bars.failed;
    auto fail = [&](int code) { atomicExch_system(status, code); *failed = 1; };
    if (tid == 0) {
        mbar_init(&bars.k_ready, 4);
        mbar_init(&bars.o_done, 1);
        for (int i = 0; i < SLOTS; ++i) mbar_init(&bars.q_full[i], 1);
        for (int i = 0; i < 2; ++i) { mbar_init(&bars.s_full[i], 1); mbar_init(&bars.s_free[i], 4); }
        bars.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pa_before();
    __syncthreads();
    pa_after();
    const unsigned tm = bars.tmem;

    if (warp == 4) {
        // Tile t of this CTA: its copies are asked for behind s_free(t - SLOTS), its products behind s_free(t - 2), so its slot, rows and scores' region are free then
        const bool el = elect_one();
        const unsigned kd = umma_desc_lo(smem_u32(k_sm)), qd = umma_desc_lo(smem_u32(q_sm));
        const unsigned char* q = reinterpret_cast<const unsigned char*>(p.q16) + (head * p.row_tiles * (kPromptRows / kWeightRows) + tile0) * Q_BYTES;
        const float* factor = p.q_factor + head * p.row_tiles * kPromptRows + (size_t)tile0 * kWeightRows;
        const float* shift = p.q_shift + head * p.row_tiles * kPromptRows + (size_t)tile0 * kWeightRows;
        int asked = 0;
        auto ask = [&]() {
            if (el) {
                const int slot = asked & (SLOTS - 1);
                const unsigned bar = smem_u32(&bars.q_full[slot]);
                mbar_expect(bar, Q_BYTES + 2 * kWeightRows * 4);
                bulk_load(smem_u32(q_sm) + slot * Q_BYTES, q + (size_t)asked * Q_BYTES, Q_BYTES, bar);
                bulk_load(smem_u32(rows_sm[slot][0]), factor + asked * kWeightRows, kWeightRows * 4, bar);
                bulk_load(smem_u32(rows_sm[slot][1]), shift + asked * kWeightRows, kWeightRows * 4, bar);
            }
            __syncwarp();
            ++asked;
        };
        while (asked < tiles && asked < SLOTS - 1) ask();
        bool ok = mbar_wait_warp(&bars.k_ready, 0u);
        for (int t = 0; t < tiles && ok; ++t) {
            const int slot = t & (SLOTS - 1);
            if (*failed || !mbar_wait_warp(&bars.q_full[slot], (unsigned)((t / SLOTS) & 1))) { ok = false; break; }
            pa_after();
            if (el) {
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk)
                    pa_mma_ss(tm + (t & 1) * 64u, kd + (kk >> 2) * (K_HALF / 16) + 2 * (kk & 3), qd + slot * (Q_BYTES / 16) + (kk >> 2) * (Q_HALF / 16) + 2 * (kk & 3),
                              pa_idesc(kWeightRows, false, false), kk > 0 ? 1u : 0u);
                umma_commit(&bars.s_full[t & 1]);
            }
            __syncwarp();
            // what tile t - 1 had: the region of tile t + 1, the slot of tile t + SLOTS - 1
            if (t > 0 && t + 1 < tiles && !mbar_wait_warp(&bars.s_free[(t - 1) & 1], (unsigned)(((t - 1) >> 1) & 1))) { ok = false; break; }
            if (asked < tiles) ask();
        }
        if (el) umma_commit(&bars.o_done);
        __syncwarp();
        ok = mbar_wait_warp(&bars.o_done, 0u) && ok;   // tensor memory is not freed under MMAs in flight, nor shared memory left under copies
        for (int t = max(0, asked - SLOTS); t < asked; ++t) ok = mbar_wait_warp(&bars.q_full[t & (SLOTS - 1)], (unsigned)((t / SLOTS) & 1)) && ok;
        if (!ok && lane == 0) fail(34);
        __syncwarp();
    } else {
        // ---- this CTA's keys ----
        constexpr int PIECES = HD / 16, STEP = kWeightKeys / PIECES;   // (threads of a token, tokens of a turn)
        const int piece = tid % PIECES, row = tid / PIECES, chunk = piece * 2 & 7;
        const unsigned char* src = static_cast<const unsigned char*>(c.k) + (head * c.capacity + key0) * HD + piece * 16;
        const unsigned off = (piece >> 2) * K_HALF;
#pragma unroll 4
        for (int r = row; r < kWeightKeys; r += STEP) {
            const uint4 v = key0 + r < end ? *reinterpret_cast<const uint4*>(src + (size_t)r * HD) : make_uint4(0, 0, 0, 0);
            const unsigned w[4] = {prepared<CODE>(v.x), prepared<CODE>(v.y), prepared<CODE>(v.z), prepared<CODE>(v.w)};
            *reinterpret_cast<uint4*>(k_sm + off + r * 128 + ((chunk ^ (r & 7)) << 4)) = make_uint4(pair_of<CODE, 0>(w[0]), pair_of<CODE, 1>(w[0]), pair_of<CODE, 0>(w[1]), pair_of<CODE, 1>(w[1]));
            *reinterpret_cast<uint4*>(k_sm + off + r * 128 + (((chunk + 1) ^ (r & 7)) << 4)) = make_uint4(pair_of<CODE, 0>(w[2]), pair_of<CODE, 1>(w[2]), pair_of<CODE, 0>(w[3]), pair_of<CODE, 1>(w[3]));
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) pa_arrive(&bars.k_ready);
        // ---- a thread per key ----
        const int key = key0 + tid;
        const float scale = key < end ? c.k_scale[head * (c.capacity / c.block) + key / c.block] : 0.f;
        const float2 scale2 = make_float2(scale, scale);
        const long long first = ((long long)key - part.len) * G - (long long)tile0 * kWeightRows;   // the first row, from tile0 on, that attends it
        const unsigned lanes = (unsigned)(warp * 32) << 16;
        float2 sum = make_float2(0.f, 0.f);
        bool ok = true;
        for (int t = 0; t < tiles; ++t) {
            const int slot = t & (SLOTS - 1);
            if (!mbar_wait_warp(&bars.q_full[slot], (unsigned)((t / SLOTS) & 1)) || !mbar_wait_warp(&bars.s_full[t & 1], (unsigned)((t >> 1) & 1))) { ok = false; break; }
            pa_after();
            unsigned v[64];
            pa_ld32(tm + lanes + (t & 1) * 64u, v);
            pa_ld32(tm + lanes + (t & 1) * 64u + 32u, v + 32);
            pa_wait_ld();
            const bool masked = !__all_sync(0xffffffffu, first <= (long long)t * kWeightRows);
#pragma unroll
            for (int e = 0; e < kWeightRows; e += 4) {
                const float4 f = *reinterpret_cast<const float4*>(&rows_sm[slot][0][e]), m = *reinterpret_cast<const float4*>(&rows_sm[slot][1][e]);
                // (the row's factor meets the key's scale first, as in the attention: either alone may take the product out of range)
                float2 x = fma2(make_float2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), mul2(make_float2(f.x, f.y), scale2), make_float2(m.x, m.y));
                float2 y = fma2(make_float2(__uint_as_float(v[e + 2]), __uint_as_float(v[e + 3])), mul2(make_float2(f.z, f.w), scale2), make_float2(m.z, m.w));
                x = make_float2(pa_exp2(x.x), pa_exp2(x.y));
                y = make_float2(pa_exp2(y.x), pa_exp2(y.y));
                if (masked) {
                    const long long at = (long long)t * kWeightRows + e;
                    if (at < first) x.x = 0.f;
                    if (at + 1 < first) x.y = 0.f;
                    if (at + 2 < first) y.x = 0.f;
                    if (at + 3 < first) y.y = 0.f;
                }
                sum = add2(sum, add2(x, y));
            }
            pa_before();
            __syncwarp();
            if (lane == 0) pa_arrive(&bars.s_free[t & 1]);
        }
        if (!ok) fail(35);
        else if (key < end) c.weight[head * c.capacity + key] += sum.x + sum.y;
    }
    pa_before();
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(kTmemCols) : "memory");
}

template <int HD, int CODE>
int launch_prompt(const swlm_kv8_cache& c, const swlm_kv8_attend& a, const RowsPlan& p, int* status, cudaStream_t s) {
    const dim3 grid((unsigned)c.batch * c.kv_heads * p.row_tiles * p.splits);
    auto launch = [&](auto kernel) { return launch_k(kernel, grid, dim3(kPromptThreads), prompt_smem<HD>(), s, c, a, p, status); };
    auto with = [&](auto two) {
        constexpr bool TWO = decltype(two)::value;
        return c.block == 128 ? launch(kv8_prompt_kernel<HD, CODE, 1, TWO>) : c.block == 64 ? launch(kv8_prompt_kernel<HD, CODE, 2, TWO>) :
               c.block == 32 ? launch(kv8_prompt_kernel<HD, CODE, 4, TWO>) : launch(kv8_prompt_kernel<HD, CODE, 8, TWO>);
    };
    const cudaError_t e = kv8_two_products(a) ? with(std::true_type()) : with(std::false_type());
    return e == cudaSuccess ? SWLM_OK : cuda_fail(e, "kv8 prompt attention launch");
}
template <int HD, int CODE>
int launch_weights(const swlm_kv8_cache& c, const swlm_kv8_attend& a, const RowsPlan& p, int* status, cudaStream_t s) {
    const int span = std::min(a.max_len, c.capacity), tiles = (span + kWeightKeys - 1) / kWeightKeys;
    const dim3 grid((unsigned)tiles, (unsigned)c.kv_heads, (unsigned)c.batch);
    auto launch = [&](auto kernel, size_t smem) { return launch_k(kernel, grid, dim3(kWeightThreads), smem, s, c, a, p, status); };
    cudaError_t e;
    if constexpr (HD == 64) e = launch(kv8_weights_kernel<HD, CODE, 4>, weights_smem<HD, 4>());
    else if ((long long)tiles * c.kv_heads * c.batch > 2 * kSms) e = launch(kv8_weights_kernel<HD, CODE, 2>, weights_smem<HD, 2>());
    else e = launch(kv8_weights_kernel<HD, CODE, 4>, weights_smem<HD, 4>());
    return e == cudaSuccess ? SWLM_OK : cuda_fail(e, "kv8 prompt weights launch");
}
template <int HD, int CODE>
int init_prompt() {
    SWLM_CUDA((cudaFuncSetAttribute(kv8_weights_kernel<HD, CODE, 4>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)weights_smem<HD, 4>())));
    if constexpr (HD == 128) SWLM_CUDA((cudaFuncSetAttribute(kv8_weights_kernel<HD, CODE, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)weights_smem<HD, 2>())));
    auto each = [](auto kernel) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)prompt_smem<HD>()); };
    for (const cudaError_t e : {each(kv8_prompt_kernel<HD, CODE, 1, false>), each(kv8_prompt_kernel<HD, CODE, 2, false>), each(kv8_prompt_kernel<HD, CODE, 4, false>),
                                each(kv8_prompt_kernel<HD, CODE, 8, false>), each(kv8_prompt_kernel<HD, CODE, 1, true>), each(kv8_prompt_kernel<HD, CODE, 2, true>),
                                each(kv8_prompt_kernel<HD, CODE, 4, true>), each(kv8_prompt_kernel<HD, CODE, 8, true>)})
        SWLM_CUDA(e);
    return SWLM_OK;
}

}  // namespace

int kv8_prompt_init() {
    int rc = init_prompt<128, SWLM_KV8_INT8>();
    if (!rc) rc = init_prompt<128, SWLM_KV8_E4M3>();
    if (!rc) rc = init_prompt<64, SWLM_KV8_INT8>();
    if (!rc) rc = init_prompt<64, SWLM_KV8_E4M3>();
    return rc;
}

int launch_kv8_prompt_weights(const swlm_kv8_cache& c, const swlm_kv8_attend& a, const RowsPlan& p, int* status, cudaStream_t s) {
    if (c.head_dim == 128) return c.code == SWLM_KV8_INT8 ? launch_weights<128, SWLM_KV8_INT8>(c, a, p, status, s) : launch_weights<128, SWLM_KV8_E4M3>(c, a, p, status, s);
    return c.code == SWLM_KV8_INT8 ? launch_weights<64, SWLM_KV8_INT8>(c, a, p, status, s) : launch_weights<64, SWLM_KV8_E4M3>(c, a, p, status, s);
}

int launch_kv8_prompt(const swlm_kv8_cache& c, const swlm_kv8_attend& a, const RowsPlan& p, int* status, cudaStream_t s) {
    if (c.head_dim == 128) return c.code == SWLM_KV8_INT8 ? launch_prompt<128, SWLM_KV8_INT8>(c, a, p, status, s) : launch_prompt<128, SWLM_KV8_E4M3>(c, a, p, status, s);
    return c.code == SWLM_KV8_INT8 ? launch_prompt<64, SWLM_KV8_INT8>(c, a, p, status, s) : launch_prompt<64, SWLM_KV8_E4M3>(c, a, p, status, s);
}

}  // namespace swlm
