// Shared by the operators over a cache of 8-bit codes with one scale per block of tokens and head (include/swlm.h).
#pragma once

#include "swlm_internal.h"

namespace swlm {

constexpr int kKv8MinBlock = 16, kKv8MaxBlock = 128;
// Grids have one CTA layer per (sequence, KV head, keys or values): what their y and z dimensions hold
constexpr int kKv8MaxBatch = 65535, kKv8MaxKvHeads = 32767;
// Tokens of a sequence: slots are 32-bit numbers, also a chunk behind the last one
constexpr int kKv8MaxLen = 1 << 30;

int kv8_init();   // shared-memory attributes on the current device
int kv8_attend_init();
int launch_kv8_append(const swlm_kv8_cache& c, const swlm_kv8_append& a, cudaStream_t s);
int launch_kv8_evict(const swlm_kv8_cache& c, const swlm_kv8_cache& to, const swlm_kv8_evict& a, cudaStream_t s);
size_t kv8_evict_scratch(const swlm_kv8_cache& c, const swlm_kv8_evict& a);
int launch_kv8_lengths(int batch, const int32_t* in, const int32_t* counts, int n, int limit, const int32_t* refused, int32_t* out, cudaStream_t s);
// status: a word that the device sets when a bounded wait expires
int launch_kv8_attend(const swlm_kv8_cache& c, const swlm_kv8_attend& a, int* status, cudaStream_t s);
bool kv8_attend_grid_fits(const swlm_kv8_cache& c, const swlm_kv8_attend& a);
size_t kv8_attend_scratch(const swlm_kv8_cache& c, const swlm_kv8_attend& a);

#ifdef __CUDACC__
constexpr float kKv8NaN = __builtin_nanf("");

// A sequence's part in a step: where it stands and the rows of its tokens; count 0 where it has none, where what it says does not fit, or where
// `refused` (may be null) says that its tokens were not appended.
struct Kv8Part {
    int len, count, start;
    bool fits;
};
__device__ __forceinline__ Kv8Part kv8_part(int b, const int32_t* lengths, const int32_t* counts, const int32_t* starts, const int32_t* refused, int n, int rows) {
    Kv8Part p;
    p.len = lengths[b];
    p.count = counts ? counts[b] : n;
    const long long start = starts ? (long long)starts[b] : (long long)b * n;
    p.fits = p.count >= 0 && p.count <= n && (p.count == 0 || (start >= 0 && start + p.count <= rows)) && !(refused && refused[b]);
    if (!p.fits) p.count = 0;
    p.start = p.count ? (int)start : 0;
    return p;
}
#endif

}  // namespace swlm
