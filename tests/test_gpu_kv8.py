"""Operators over an 8-bit cache with one scale per block of tokens and head, against plain forms in 64 bits (tests/plain_kv8.py)."""
import ctypes as C
import math

import pytest
import torch

from plain_kv8 import TOP, Cache, attend, chosen, expected_append, half_step, numbers

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def store(pkg):
    s = pkg.WeightStore(0)
    yield s
    s.close()


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream or 1)


def starts_of(counts, gap=0):
    out, at = [], 0
    for c in counts:
        out.append(at + gap)
        at += c + gap
    return out, at + gap


def append(pkg, store, cache, k, v, lengths, counts=None, starts=None, seen=None, refused=None, n=None):
    step = pkg.Kv8Append(k=k.data_ptr(), v=v.data_ptr(), k_stride=k.stride(0), v_stride=v.stride(0), lengths=lengths.data_ptr(),
                         counts=counts.data_ptr() if counts is not None else None, starts=starts.data_ptr() if starts is not None else None,
                         seen=seen.data_ptr() if seen is not None else lengths.data_ptr(), refused=refused.data_ptr() if refused is not None else None,
                         dtype=int(k.dtype == torch.float16), n=n if n is not None else int(counts.max()), rows=k.shape[0])
    store.lib.check(store.lib.swlm_op_kv8_append_dev(store.handle, cache.described(), step, stream()))


def attend_call(pkg, store, cache, q, out, lengths, scale, counts=None, starts=None, n=None, max_len=None, accumulate=False, scratch=None):
    """The call's structure with scratch of its own (garbage in it), kept alive beside it."""
    step = pkg.Kv8Attend(q=q.data_ptr(), out=out.data_ptr(), q_stride=q.stride(0), out_stride=out.stride(0), lengths=lengths.data_ptr(),
                         counts=counts.data_ptr() if counts is not None else None, starts=starts.data_ptr() if starts is not None else None,
                         scale=scale, dtype=int(q.dtype == torch.float16), heads=q.shape[1], n=n if n is not None else int(counts.max()), rows=q.shape[0],
                         max_len=max_len or cache.k.shape[2], accumulate=int(accumulate))
    step.scratch_bytes = store.lib.swlm_op_kv8_attend_scratch_bytes(cache.described(), step)
    keep = torch.full((step.scratch_bytes + 256,), 0xFF, dtype=torch.uint8, device="cuda")   # (as floats: NaN)
    step.scratch = keep.data_ptr()
    return step, keep


def do_attend(pkg, store, cache, *args, **more):
    step, scratch = attend_call(pkg, store, cache, *args, **more)
    store.lib.check(store.lib.swlm_op_kv8_attend_dev(store.handle, cache.described(), step, stream()))
    torch.cuda.synchronize()
    assert (scratch[step.scratch_bytes:] == 0xFF).all()


def evict_call(pkg, store, cache, keep, sink, recent, lengths, seen, max_len=None):
    how = pkg.Kv8Evict(lengths=lengths.data_ptr(), seen=seen.data_ptr(), keep=keep, sink=sink, recent=recent, max_len=max_len or cache.k.shape[2])
    how.scratch_bytes = store.lib.swlm_op_kv8_evict_scratch_bytes(cache.described(), how)
    scratch = torch.full((how.scratch_bytes + 256,), 0xFF, dtype=torch.uint8, device="cuda")
    how.scratch = scratch.data_ptr()
    return how, scratch


def evict(pkg, store, cache, to, *args, **more):
    how, scratch = evict_call(pkg, store, cache, *args, **more)
    store.lib.check(store.lib.swlm_op_kv8_evict_dev(store.handle, cache.described(), to.described(), how, stream()))
    torch.cuda.synchronize()
    assert (scratch[how.scratch_bytes:] == 0xFF).all()


def same_bits(a, b):
    return torch.equal(a.reshape(-1).contiguous().view(torch.uint8), b.reshape(-1).contiguous().view(torch.uint8))


# ---- append ----------------------------------------------------------------------------------------------------------------

APPENDS = [
    # batch, kv_heads, head_dim, block, lengths, counts
    (1, 1, 64, 16, [0], [1]),
    (1, 8, 128, 64, [63], [1]),
    (3, 2, 128, 128, [5, 127, 128], [1, 1, 1]),
    (3, 3, 64, 32, [0, 31, 40], [0, 2, 70]),
    (2, 2, 128, 16, [15, 1], [34, 300]),
    (4, 1, 128, 128, [0, 100, 255, 256], [128, 129, 257, 1]),
    (2, 5, 64, 128, [77, 0], [200, 13]),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("code", [0, 1])
@pytest.mark.parametrize("batch,kv_heads,dim,block,lengths,counts", APPENDS, ids=str)
def test_append(pkg, store, batch, kv_heads, dim, block, lengths, counts, code, dtype):
    """Codes and scales are the formula's, bit for bit, and within half a step of the values in 64 bits; nothing else changes. New values outgrow
    the old scales in some blocks and not in others. Rows have gaps between heads' rows and between sequences."""
    g = torch.Generator(device="cuda").manual_seed(dim + block + code)
    cap = (max(a + c for a, c in zip(lengths, counts)) + block) // block * block
    cache = Cache(pkg, batch, kv_heads, dim, cap, block, code).fill(lengths)
    starts, rows = starts_of(counts, gap=2)
    wide = torch.randn((rows, kv_heads + 1, 2, dim), generator=g, device="cuda") * torch.exp(torch.randn((rows, 1, 1, 1), generator=g, device="cuda"))
    wide = wide.to(dtype)
    k, v = wide.view(rows, -1)[:, :kv_heads * dim], wide.view(rows, -1)[:, (kv_heads + 1) * dim:][:, :kv_heads * dim]   # one array of both
    before = cache.clone()
    seen, refused = ints(*(a + 1000 for a in lengths)), ints(*([9] * batch))
    append(pkg, store, cache, k, v, ints(*lengths), ints(*counts), ints(*starts), seen, refused, n=max(counts) + 3)
    torch.cuda.synchronize()
    assert refused.tolist() == [0] * batch
    for b, (a, c) in enumerate(zip(lengths, counts)):
        for name, x in (("k", k), ("v", v)):
            new = x[starts[b]:starts[b] + c].reshape(c, kv_heads, dim)
            codes, scales = expected_append(before, name, b, new, a)
            assert same_bits(getattr(cache, name + "_scale")[b], scales)
            assert same_bits(getattr(cache, name)[b], codes)
            each = scales.double().repeat_interleave(block, dim=1)[:, :a + c, None]
            want = torch.cat([before.values(name, b, a), new.transpose(0, 1).double()], dim=1)
            off = (numbers(codes[:, :a + c], code) * each - want).abs()
            # The code is the nearest to a y that two fp32 operations (the product with the old scale, the quotient) have made: each is off by 2^-24 of
            # its result at most, so y is by 2^-23 |y|, and the code is half a step and that from the value: next to 63.5, half + 2^-17 of a step
            assert (off <= half_step(want / each, code) * each + 2.0 ** -22 * want.abs()).all()
        weight, pos = before.weight[b].clone(), before.slot_pos[b].clone()
        weight[:, a:a + c], pos[:, a:a + c] = 0.0, torch.arange(a + 1000, a + 1000 + c, device="cuda", dtype=torch.int32)
        assert torch.equal(cache.weight[b], weight) and torch.equal(cache.slot_pos[b], pos)


@pytest.mark.parametrize("code", [0, 1])
def test_append_of_special_values(pkg, store, code):
    """A block of zeros, values whose scale is subnormal, the largest finite ones; infinity and NaN make their block NaN, and it stays so."""
    cache = Cache(pkg, 1, 1, 64, 128, 16, code)
    x = torch.zeros((96, 64), device="cuda")
    x[16:32] = 1e-38
    x[32:48] = torch.finfo(torch.bfloat16).max
    x[48:64, 3], x[70, 5], x[90, 60] = 1.0, math.inf, math.nan
    x = x.bfloat16()
    append(pkg, store, cache, x, -x, ints(0), ints(96))
    append(pkg, store, cache, torch.ones((1, 64), device="cuda").bfloat16(), torch.ones((1, 64), device="cuda").bfloat16(), ints(75), ints(1))   # behind the infinity
    torch.cuda.synchronize()
    assert cache.k_scale[0, 0].isnan().tolist()[:6] == [False] * 4 + [True] * 2 and cache.v_scale[0, 0].isnan().tolist()[:6] == [False] * 4 + [True] * 2
    got, want = cache.values("k", 0, 64)[0], x[:64].double()
    each = cache.k_scale[0, 0].double().repeat_interleave(16)[:64, None]
    # (a subnormal scale is itself off by up to half of the smallest number, 2^-150, times the largest code)
    assert ((got - want).abs() <= half_step(want / each.clamp(min=1e-300), code) * each + 2.0 ** -22 * want.abs() + TOP[code] * 2.0 ** -150).all()
    assert (got[:16] == 0).all() and (got[48:64, :3] == 0).all()
    append(pkg, store, cache, x[:1], x[:1], ints(76), ints(1))   # a NaN block takes more
    torch.cuda.synchronize()
    assert cache.k_scale[0, 0, 4].isnan()


def test_append_refuses_whole_sequences(pkg, store):
    """No room, a negative length or count, more tokens than n, rows outside the arrays: nothing of that sequence changes, the others are appended."""
    lengths, counts, starts = [60, 64, -1, 3, 3, 3, 3, 0], [4, 1, 1, -2, 5, 2, 2, 4], [0, 4, 5, 6, 6, 23, -1, 8]
    cache = Cache(pkg, 8, 2, 64, 64, 16, 0).fill(lengths)
    before = cache.clone()
    x = 100 * torch.randn((24, 128), device="cuda").half()
    refused = ints(*([5] * 8))
    append(pkg, store, cache, x, x, ints(*lengths), ints(*counts), ints(*starts), ints(*([0] * 8)), refused, n=4)
    torch.cuda.synchronize()
    assert refused.tolist() == [0, 1, 1, 1, 1, 1, 1, 0]
    for b in range(8):
        for x, y in zip(cache.arrays(), before.arrays()):
            assert same_bits(x[b], y[b]) == (b not in (0, 7))


def test_append_one_at_a_time_matches_the_formula(pkg, store):
    """A prompt's tokens one by one: every step's state follows from the one before by the formula."""
    cache = Cache(pkg, 1, 2, 64, 64, 16, 0)
    x = torch.randn((40, 2, 64), device="cuda").bfloat16() * torch.linspace(0.1, 3, 40, device="cuda")[:, None, None].bfloat16()
    for i in range(40):
        before = cache.clone()
        append(pkg, store, cache, x[i:i + 1].view(1, 128), x[i:i + 1].view(1, 128), ints(i), n=1)
        torch.cuda.synchronize()
        codes, scales = expected_append(before, "k", 0, x[i:i + 1], i)
        assert same_bits(cache.k[0], codes) and same_bits(cache.k_scale[0], scales) and same_bits(cache.v[0, :, :i + 1], codes[:, :i + 1])


# ---- attend ----------------------------------------------------------------------------------------------------------------

ATTENDS = [
    # batch, heads, kv_heads, head_dim, block, lengths before the step, counts
    (1, 1, 1, 64, 16, [0], [1]),                                  # one token in the cache
    (1, 4, 1, 128, 64, [16], [1]),
    (3, 32, 8, 128, 64, [0, 999, 300], [1, 1, 1]),
    (5, 14, 2, 64, 32, [-1, 130, 4000, 0, 127], [1, 0, 1, 1, 1]),  # seven heads of a group; a parked sequence, one without a token
    (2, 12, 1, 128, 128, [2047, 2048], [1, 1]),                   # twelve rows: two tiles
    (2, 8, 8, 64, 16, [5000, 70], [1, 1]),                        # no shared heads
    (3, 8, 2, 128, 16, [100, 0, 1500], [5, 3, 1]),                # drafted tokens
    (2, 4, 1, 64, 64, [-2, 40], [16, 9]),                         # rows that attend nothing, then some
    (1, 24, 2, 128, 32, [37], [11]),                              # 132 rows of a KV head: weights worked out again
    (2, 8, 2, 64, 128, [0, 777], [190, 77]),                      # portions of prompts
    (1, 4, 4, 128, 64, [500], [129]),
    (1, 8, 1, 128, 64, [9000], [1]),
    (1, 4, 1, 128, 16, [3000], [40]),                             # a portion whose slots are worked on in several runs
    (1, 2, 1, 64, 32, [50], [700]),                               # several blocks of rows, causal from an almost empty cache
    (2, 10, 2, 64, 64, [600, 30], [7, 13]),                       # 65 rows: one more than the scores are kept for
]


def check_attend(pkg, store, cache, batch, heads, dim, lengths, counts, dtype, accumulate, max_len=None, gap=1, q_gain=1.0, seed=3):
    starts, rows = starts_of(counts, gap)
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = (q_gain * torch.randn((rows, heads + 2, dim), generator=g, device="cuda")).to(dtype)[:, :heads]
    out = torch.full((rows, heads + 1, dim), 7.0, device="cuda").to(dtype)[:, :heads]
    before = cache.clone()
    scale, span = dim ** -0.5, min(max_len or cache.k.shape[2], cache.k.shape[2])
    do_attend(pkg, store, cache, q, out, ints(*lengths), scale, ints(*counts), ints(*starts), max_len=max_len, accumulate=accumulate, n=max(counts) + 1)
    untouched = torch.ones(rows, dtype=torch.bool, device="cuda")
    for b, (a, c) in enumerate(zip(lengths, counts)):
        at = slice(starts[b], starts[b] + c)
        untouched[at] = False
        want, tol, weight, weight_tol = attend(before, q[at], b, a, scale, span)
        assert ((out[at].double() - want).abs() <= tol).all(), (b, ((out[at].double() - want).abs() - tol).max())
        if accumulate:
            total = max(0, min(a + c, span)) if c else 0
            was = before.weight[b, :, :total].double()
            off = (cache.weight[b, :, :total].double() - was - weight[:, :total]).abs()
            assert (off <= weight_tol[:, :total] + 2.0 ** -24 * (was + weight[:, :total])).all(), b
            assert same_bits(cache.weight[b, :, total:], before.weight[b, :, total:])
    assert (out[untouched] == 7.0).all()
    for x, y in list(zip(cache.arrays(), before.arrays()))[:4] + ([] if accumulate else [(cache.weight, before.weight)]):
        assert same_bits(x, y)
    return q, out, starts


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("code,dtype", [(0, torch.bfloat16), (1, torch.float16), (1, torch.bfloat16)], ids=str)
@pytest.mark.parametrize("batch,heads,kv_heads,dim,block,lengths,counts", ATTENDS, ids=str)
def test_attend(pkg, store, batch, heads, kv_heads, dim, block, lengths, counts, code, dtype, accumulate):
    cap = (max(a + c for a, c in zip(lengths, counts)) + block) // block * block
    cache = Cache(pkg, batch, kv_heads, dim, cap, block, code).fill([max(0, a + c) for a, c in zip(lengths, counts)])
    check_attend(pkg, store, cache, batch, heads, dim, lengths, counts, dtype, accumulate)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("batch,heads,kv_heads,dim,most", [(64, 16, 8, 64, 1400), (64, 4, 4, 128, 1900), (520, 1, 1, 64, 200)], ids=str)
def test_attend_of_many_sequences(pkg, store, batch, heads, kv_heads, dim, most, accumulate):
    """Batches whose slots come in equal shares, several sequences to a CTA and sequences over several CTAs, and a batch of one CTA per head. Empty, parked
    and full sequences between others. Twice with the same scratch."""
    g = torch.Generator().manual_seed(batch + dim)
    lengths = [int(x) for x in torch.randint(0, most, (batch,), generator=g)]
    lengths[0], lengths[3], lengths[4], lengths[-1] = most, -1, 0, most
    counts = [0 if i % 17 == 5 else 1 for i in range(batch)]
    cap = (most + 64) // 64 * 64
    cache = Cache(pkg, batch, kv_heads, dim, cap, 64, 0).fill([max(0, a + c) for a, c in zip(lengths, counts)])
    starts, rows = starts_of(counts)
    q = torch.randn((rows, heads, dim), device="cuda").bfloat16()
    out, at, n, first = torch.zeros_like(q), ints(*lengths), ints(*counts), ints(*starts)
    step, scratch = attend_call(pkg, store, cache, q, out, at, dim ** -0.5, n, first, n=1, accumulate=accumulate)
    before = cache.weight.clone()
    for _ in range(2):
        out.fill_(7.0)
        cache.weight.copy_(before)
        store.lib.check(store.lib.swlm_op_kv8_attend_dev(store.handle, cache.described(), step, stream()))
        torch.cuda.synchronize()
        for b in range(0, batch, 1 if batch < 100 else 7):
            if counts[b]:
                want, tol, weight, weight_tol = attend(cache, q[starts[b]:starts[b] + 1], b, lengths[b], dim ** -0.5, cap)
                assert ((out[starts[b]:starts[b] + 1].double() - want).abs() <= tol).all(), b
                if accumulate:
                    weight += before[b].double()
                    assert ((cache.weight[b].double() - weight).abs() <= weight_tol + 2.0 ** -24 * weight.abs()).all(), b
            else:
                assert torch.equal(cache.weight[b], before[b])
    assert (scratch[step.scratch_bytes:] == 0xFF).all()


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("max_len", [130, 300, 900, 2048, 4096, None])
@pytest.mark.parametrize("batch,heads,kv_heads,dim,lengths,counts", [
    (1, 8, 8, 128, [4000], [1]),
    (4, 14, 2, 64, [1030, -1, 0, 128], [2, 1, 1, 0]),              # fourteen rows; parked, empty and without a token
    (2, 10, 2, 128, [255, 1999], [5, 3]),                          # 25 rows: two tiles
    (20, 8, 4, 64, [97 * i for i in range(20)], [1] * 20),         # two or four CTAs a cluster
], ids=str)
def test_attend_whoever_joins(pkg, store, batch, heads, kv_heads, dim, lengths, counts, max_len, accumulate):
    """The same sequences where clusters of two, four or eight CTAs have a head's slots, some of them none, and where shares of the GPU have them: which, goes by max_len."""
    cache = Cache(pkg, batch, kv_heads, dim, 16384, 64, 1).fill([max(0, a + c) for a, c in zip(lengths, counts)])
    check_attend(pkg, store, cache, batch, heads, dim, lengths, counts, torch.bfloat16, accumulate, max_len=max_len)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("code", [0, 1])
def test_weights_of_portions_by_many_ctas(pkg, store, dim, code):
    """Portions of a batch whose key tiles are more than the CTAs that run at once: one that fills the cache, from an empty cache, without tokens, of a few rows."""
    lengths, counts = [1700, 0, 900, 1300, -3], [340, 333, 0, 17, 70]
    cache = Cache(pkg, 5, 4, dim, 2048, 64, code).fill([max(0, a + c) for a, c in zip(lengths, counts)])
    check_attend(pkg, store, cache, 5, 16, dim, lengths, counts, torch.float16, True)


@pytest.mark.parametrize("counts", [[1, 1], [40, 40]], ids=str)
def test_attend_cuts_at_max_len(pkg, store, counts):
    """Slots behind max_len are not attended, whatever the lengths say (a length far beyond the capacity among them)."""
    cache = Cache(pkg, 2, 2, 64, 512, 32, 0).fill([512, 512])
    check_attend(pkg, store, cache, 2, 4, 64, [400, 2 ** 31 - 50], counts, torch.bfloat16, True, max_len=203)
    check_attend(pkg, store, cache, 2, 4, 64, [400, 2 ** 31 - 50], counts, torch.bfloat16, True)


@pytest.mark.parametrize("code", [0, 1])
@pytest.mark.parametrize("gain", [1e-30, 1e-3, 30.0, 3e4])
def test_attend_with_queries_of_any_size(pkg, store, code, gain):
    """Queries are brought to a common size by powers of two: tiny ones attend evenly, large ones to one token. bf16 has the range."""
    cache = Cache(pkg, 1, 2, 128, 512, 64, code).fill([400], key=0.05 if gain > 100 else 2.0)
    check_attend(pkg, store, cache, 1, 8, 128, [398], [2], torch.bfloat16, True, q_gain=gain)


@pytest.mark.parametrize("code", [0, 1])
def test_attend_over_value_scales_far_apart(pkg, store, code):
    """Blocks' value scales from 1e-6 to 1e3 in any order, also where the small ones carry the weight, and a block of zeros."""
    cache = Cache(pkg, 1, 1, 64, 1024, 16, code).fill([1000])
    cache.v_scale[0, 0, :63] *= torch.logspace(-6, 3, 63, device="cuda")[torch.randperm(63, generator=torch.Generator().manual_seed(1)).cuda()]
    cache.v_scale[0, 0, 5] = 0.0
    check_attend(pkg, store, cache, 1, 4, 64, [999], [1], torch.bfloat16, False)
    cache.k_scale[0, 0, :63] *= 0.01   # attention almost even
    check_attend(pkg, store, cache, 1, 4, 64, [990], [10], torch.bfloat16, False)


def test_attend_and_nan(pkg, store):
    """A NaN block makes NaN what attends it, and nothing else; so does a query that is not finite."""
    for counts in ([4], [60]):
        cache = Cache(pkg, 1, 1, 64, 256, 16, 0).fill([200])
        cache.v_scale[0, 0, 8] = math.nan   # slots 128..143
        a = 126
        q = torch.randn((counts[0], 2, 64), device="cuda").bfloat16()
        q[counts[0] - 1, 1, 7] = math.inf
        out = torch.zeros_like(q)
        do_attend(pkg, store, cache, q, out, ints(a), 0.125, n=counts[0], accumulate=True)
        assert not out[:2].isnan().any() and out[2:].isnan().all()
        assert not cache.weight[0, 0, a + counts[0]:200].isnan().any() and cache.weight[0, 0, :a + counts[0]].isnan().all()
        want, tol, _, _ = attend(cache, q[:2], 0, a, 0.125, 128)
        assert ((out[:2].double() - want).abs() <= tol).all()


def test_attend_with_tables_left_out(pkg, store):
    """No counts, no starts: n queries each, one sequence's rows behind the other's."""
    cache = Cache(pkg, 3, 2, 64, 128, 16, 1).fill([90, 100, 110])
    q = torch.randn((6, 4, 64), device="cuda").half()
    out, again = torch.zeros_like(q), torch.zeros_like(q)
    do_attend(pkg, store, cache, q, out, ints(88, 98, 108), 0.1, n=2)
    do_attend(pkg, store, cache, q, again, ints(88, 98, 108), 0.1, ints(2, 2, 2), ints(0, 2, 4), n=2)
    assert same_bits(out, again)


def test_attend_ignores_sequences_that_do_not_fit(pkg, store):
    """Counts below zero or above n, rows outside the arrays: their rows stay as they are."""
    cache = Cache(pkg, 5, 1, 64, 64, 16, 0).fill([30] * 5)
    q = torch.randn((6, 1, 64), device="cuda").half()
    out = torch.full_like(q, 7.0)
    weight = cache.weight.clone()
    do_attend(pkg, store, cache, q, out, ints(*([20] * 5)), 0.1, ints(-1, 3, 2, 2, 2), ints(0, 0, 5, -1, 2), n=2, accumulate=True)
    assert (out[[0, 1, 4, 5]] == 7.0).all() and (out[2:4] != 7.0).any(dim=-1).all()
    assert torch.equal(weight[:4], cache.weight[:4]) and not torch.equal(weight[4], cache.weight[4])


# ---- evict -----------------------------------------------------------------------------------------------------------------

def check_evicted(before, to_before, to, lengths, keep, sink, recent, seen):
    """Places, weights and positions exactly; values within half a step of a block's new scale, blocks that take nothing as they were."""
    t, code = before.block, before.code
    for b, length in enumerate(lengths):
        length = max(0, length)
        n = min(length, keep)
        for h in range(before.k.shape[1]):
            source = chosen(before, b, h, length, keep, sink, recent, seen[b])
            src = torch.tensor(source, dtype=torch.long, device="cuda")
            assert same_bits(to.weight[b, h, :n], before.weight[b, h, src]) and same_bits(to.slot_pos[b, h, :n], before.slot_pos[b, h, src])
            for name in "kv":
                codes, scales = getattr(to, name)[b, h], getattr(to, name + "_scale")[b, h]
                all_values = before.values(name, b, before.k.shape[2])[h]
                for blk in range(-(-n // t)):
                    slots = range(blk * t, min(n, blk * t + t))
                    if all(source[j] == j for j in slots):
                        assert same_bits(scales[blk], getattr(before, name + "_scale")[b, h, blk])
                        assert same_bits(codes[slots[0]:slots[-1] + 1], getattr(before, name)[b, h, slots[0]:slots[-1] + 1])
                        continue
                    want = all_values[src[slots[0]:slots[-1] + 1]]
                    s = scales[blk].double()
                    # (product and quotient in fp32: 2^-24 each of the largest value and its share)
                    assert abs(float(s) * TOP[code] / float(want.abs().max()) - 1) <= 2.0 ** -22
                    off = (numbers(codes[slots[0]:slots[-1] + 1], code) * s - want).abs()
                    assert (off <= half_step(want / s, code) * s + 2.0 ** -22 * want.abs()).all()
                    if blk * t + t > n:   # (what lies behind, in the last block)
                        assert same_bits(codes[n:blk * t + t], getattr(to_before, name)[b, h, n:blk * t + t])
        for x, y in zip(to.arrays(), to_before.arrays()):
            first = -(-n // t) if x.shape[2] != to.k.shape[2] else n
            assert same_bits(x[b, :, first:], y[b, :, first:])


EVICTS = [
    # batch, kv_heads, head_dim, block, lengths, keep, sink, recent
    (1, 1, 64, 16, [17], 16, 0, 0),
    (2, 2, 128, 64, [300, 100], 100, 4, 16),        # one of them has no more than it may keep
    (3, 3, 64, 32, [700, 0, -5], 333, 1, 0),        # an odd number kept, nothing to keep
    (1, 2, 128, 128, [4352], 4096, 4, 32),
    (2, 1, 64, 16, [1000, 999], 1, 0, 1),           # one token
    (1, 1, 64, 128, [130], 129, 60, 69),            # all that stay are protected
    (1, 8, 128, 16, [2500], 260, 4, 200),
]


@pytest.mark.parametrize("code", [0, 1])
@pytest.mark.parametrize("batch,kv_heads,dim,block,lengths,keep,sink,recent", EVICTS, ids=str)
def test_evict(pkg, store, batch, kv_heads, dim, block, lengths, keep, sink, recent, code):
    """Into another cache and in place, with the same result."""
    cap = (max(lengths) + block) // block * block
    cache = Cache(pkg, batch, kv_heads, dim, cap, block, code).fill(lengths)
    order = torch.randperm(cap, generator=torch.Generator().manual_seed(2)).int().cuda()   # slots filled out of order
    seen = [max(a, 0) + 3 for a in lengths]
    cache.slot_pos[:] = torch.where(cache.slot_pos >= 0, order[None, None] % torch.tensor([max(a, 1) for a in lengths], device="cuda")[:, None, None], cache.slot_pos)
    to = Cache(pkg, batch, kv_heads, dim, -(-keep // block) * block + block, block, code, seed=5)
    before, to_before = cache.clone(), to.clone()
    evict(pkg, store, cache, to, keep, sink, recent, ints(*lengths), ints(*seen))
    assert all(same_bits(x, y) for x, y in zip(cache.arrays(), before.arrays()))
    check_evicted(before, to_before, to, lengths, keep, sink, recent, seen)
    evict(pkg, store, cache, cache, keep, sink, recent, ints(*lengths), ints(*seen))
    check_evicted(before, before, cache, lengths, keep, sink, recent, seen)
    for b, a in enumerate(lengths):
        n = max(0, min(a, keep))
        assert all(same_bits(x[b, :, :n], y[b, :, :n]) for x, y in zip((cache.k, cache.v, cache.weight), (to.k, to.v, to.weight)))


@pytest.mark.parametrize("weights", ["equal", "zeros", "special", "steps"])
def test_evict_of_equal_and_special_weights(pkg, store, weights):
    """Of equal weights the lowest slot stays, both zeros are alike, infinities are the largest and the smallest, NaN is below them."""
    cache = Cache(pkg, 1, 2, 64, 512, 16, 0).fill([500])
    g = torch.Generator(device="cuda").manual_seed(4)
    w = cache.weight[0, :, :500]
    if weights == "equal":
        w.fill_(0.25)
    elif weights == "zeros":
        w.copy_(torch.where(torch.rand(w.shape, generator=g, device="cuda") < 0.5, 0.0, -0.0))
    elif weights == "special":
        values = torch.tensor([math.nan, math.inf, -math.inf, 1e-40, -1.0, 0.0, 3e38], device="cuda")
        w.copy_(values[torch.randint(0, 7, w.shape, generator=g, device="cuda")])
    else:
        w.copy_(torch.randint(0, 3, w.shape, generator=g, device="cuda").float())
    for keep in (77, 250, 490):
        work, before = cache.clone(), cache.clone()
        evict(pkg, store, work, work, keep, 2, 5, ints(500), ints(500))
        check_evicted(before, before, work, [500], keep, 2, 5, [500])


@pytest.mark.parametrize("n", [49152 + 700, 8 * 24576 + 700])
def test_evict_from_a_long_cache(pkg, store, n):
    """Many keys, and more than fit shared memory."""
    cache = Cache(pkg, 1, 1, 64, -(-n // 128) * 128, 128, 1).fill([n])
    to = Cache(pkg, 1, 1, 64, 2048, 128, 1)
    to_before = to.clone()
    evict(pkg, store, cache, to, 2000, 4, 64, ints(n), ints(n))
    check_evicted(cache, to_before, to, [n], 2000, 4, 64, [n])


def test_evict_of_nan_blocks(pkg, store):
    """A NaN block that stays where it is stays NaN; tokens of one that move make their new block NaN."""
    cache = Cache(pkg, 1, 1, 64, 64, 16, 0).fill([64])
    cache.weight[0, 0] = torch.arange(64, device="cuda").float()
    cache.weight[0, 0, :15] = 100.0   # tokens 47..63 take slots 15..31
    cache.k_scale[0, 0, 2:] = math.nan
    evict(pkg, store, cache, cache, 32, 0, 0, ints(64), ints(64))
    assert cache.k_scale[0, 0, :2].isnan().all() and not cache.v_scale[0, 0, :2].isnan().any()


# ---- together ------------------------------------------------------------------------------------------------------------

def test_lengths(pkg, store):
    a, c, r, out = ints(5, 0, 7, -3, 2 ** 31 - 2), ints(1, 2, 9, 0, 50), ints(0, 0, 1, 0, 0), ints(0, 0, 0, 0, 0)
    lib = store.lib

    def call(src, counts, n, limit, refused, dst):
        lib.check(lib.swlm_op_kv8_lengths_dev(store.handle, 5, src.data_ptr(), counts.data_ptr() if counts is not None else None, n, limit,
                                              refused.data_ptr() if refused is not None else None, dst.data_ptr(), stream()))
        torch.cuda.synchronize()
        return dst.tolist()

    assert call(a, c, 0, 100, r, out) == [6, 2, 7, -3, 100]
    assert call(a, c, 0, 2 ** 31 - 1, None, out) == [6, 2, 16, -3, 2 ** 31 - 1]
    assert call(a, None, 0, 4, None, a) == [4, 0, 4, -3, 4]


@pytest.mark.parametrize("code,dtype,kv_heads,heads,dim", [(0, torch.bfloat16, 2, 8, 128), (1, torch.float16, 1, 7, 64)], ids=str)
def test_a_bounded_cache_in_use(pkg, store, code, dtype, kv_heads, heads, dim):
    """Two prompts in portions, then decoded tokens, with an eviction in place whenever the longest sequence has 96 tokens: every call's result follows
    from the state before it."""
    keep, sink, recent, block, cap = 64, 4, 16, 16, 128
    cache = Cache(pkg, 2, kv_heads, dim, cap, block, code)
    lengths, seen, refused = ints(0, 0), ints(0, 0), ints(0, 0)
    lib, scale = store.lib, dim ** -0.5
    g = torch.Generator(device="cuda").manual_seed(code)

    def counters(src, counts, limit, dst):
        lib.check(lib.swlm_op_kv8_lengths_dev(store.handle, 2, src.data_ptr(), counts.data_ptr() if counts is not None else None, 0, limit,
                                              refused.data_ptr(), dst.data_ptr(), stream()))

    evictions = 0
    for step in range(60):
        counts = [30, 11] if step < 2 else [1, 1] if step % 5 else [1, 0]
        a, s = lengths.tolist(), seen.tolist()
        starts, rows = starts_of(counts)
        k, v = (torch.randn((rows, kv_heads * dim), generator=g, device="cuda").to(dtype) for _ in range(2))
        before = cache.clone()
        append(pkg, store, cache, k, v, lengths, ints(*counts), ints(*starts), seen, refused)
        torch.cuda.synchronize()
        for b, c in enumerate(counts):
            for name, x in (("k", k), ("v", v)):
                codes, scales = expected_append(before, name, b, x[starts[b]:starts[b] + c].view(c, kv_heads, dim), a[b])
                assert same_bits(getattr(cache, name)[b], codes) and same_bits(getattr(cache, name + "_scale")[b], scales)
            assert cache.slot_pos[b, 0, a[b]:a[b] + c].tolist() == list(range(s[b], s[b] + c))
        check_attend(pkg, store, cache, 2, heads, dim, a, counts, dtype, True, seed=step)
        counters(lengths, ints(*counts), cap, lengths)
        counters(seen, ints(*counts), 2 ** 31 - 1, seen)
        a, s = lengths.tolist(), seen.tolist()
        if max(a) >= 96:
            before = cache.clone()
            evict(pkg, store, cache, cache, keep, sink, recent, lengths, seen)
            check_evicted(before, before, cache, a, keep, sink, recent, s)
            counters(lengths, None, keep, lengths)
            assert lengths.tolist() == [min(x, keep) for x in a]
            evictions += 1
    assert evictions >= 1 and refused.tolist() == [0, 0]


def test_a_captured_step_replays_at_other_lengths(pkg, store):
    """Append, attention with weights, counters and an eviction into another cache as one graph: replays give what the calls do, at lengths that the
    capture has not seen, on a stream that is not the default one."""
    args = (pkg, 2, 2, 64, 640, 32, 0)
    lengths, seen, refused = ints(5, 9), ints(5, 9), ints(0, 0)
    k, v, q = (torch.randn((2, n * 64), device="cuda").bfloat16() for n in (2, 2, 8))
    out = torch.zeros((2, 8, 64), device="cuda").bfloat16()
    cache, to = Cache(*args).fill([600, 600]), Cache(pkg, 2, 2, 64, 128, 32, 0)
    step, scratch = attend_call(pkg, store, cache, q.view(2, 8, 64), out, lengths, 0.125, n=1, accumulate=True)
    how, how_scratch = evict_call(pkg, store, cache, 100, 4, 8, lengths, seen)
    lib = store.lib

    def work():
        append(pkg, store, cache, k, v, lengths, None, None, seen, refused, n=1)
        lib.check(lib.swlm_op_kv8_attend_dev(store.handle, cache.described(), step, stream()))
        for x in (lengths, seen):
            lib.check(lib.swlm_op_kv8_lengths_dev(store.handle, 2, x.data_ptr(), None, 1, 640, refused.data_ptr(), x.data_ptr(), stream()))
        lib.check(lib.swlm_op_kv8_evict_dev(store.handle, cache.described(), to.described(), how, stream()))

    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            work()
    results = []
    start = cache.clone()
    for replay in (True, False):
        for x, y in zip(cache.arrays(), start.arrays()):
            x.copy_(y)
        for x in to.arrays():
            x.zero_()
        lengths.copy_(ints(500, 77)), seen.copy_(ints(800, 77))
        torch.cuda.synchronize()
        for _ in range(3):
            graph.replay() if replay else work()
        torch.cuda.synchronize()
        results.append([x.clone() for x in cache.arrays() + to.arrays() + [out, lengths, seen]])
    assert all(same_bits(x, y) for x, y in zip(*results))
    assert lengths.tolist() == [503, 80] and refused.tolist() == [0, 0]


def test_a_cache_whose_offsets_pass_32_bits(pkg, store):
    """The last head's codes lie behind 4 GB: append, both kinds of attention and an eviction in place give what they give in a small cache."""
    heads, cap, small = 9, 1 << 23, 512
    big, little = ({"k": torch.empty((1, heads, n, 64), dtype=torch.uint8, device="cuda"), "v": torch.empty((1, heads, n, 64), dtype=torch.uint8, device="cuda"),
                    "k_scale": torch.empty((1, heads, n // 64), device="cuda"), "v_scale": torch.empty((1, heads, n // 64), device="cuda"),
                    "weight": torch.empty((1, heads, n), device="cuda"), "slot_pos": torch.empty((1, heads, n), dtype=torch.int32, device="cuda")} for n in (cap, small))
    results = []
    for arrays in (big, little):
        cache = Cache(pkg, 1, 1, 64, 64, 64, 0)
        for name, x in arrays.items():
            setattr(cache, name, x)
        g = torch.Generator(device="cuda").manual_seed(7)
        k, v = (torch.randn((300, heads * 64), generator=g, device="cuda").bfloat16() for _ in range(2))
        append(pkg, store, cache, k, v, ints(0), n=300)
        outs = []
        for n in (1, 80):
            q = torch.randn((n, heads, 64), generator=g, device="cuda").bfloat16()
            out = torch.zeros_like(q)
            do_attend(pkg, store, cache, q, out, ints(300 - n), 0.125, n=n, max_len=small, accumulate=True)
            outs.append(out)
        evict(pkg, store, cache, cache, 200, 4, 20, ints(300), ints(300), max_len=small)
        results.append(outs + [cache.k[0, :, :200].clone(), cache.v[0, :, :200].clone(), cache.k_scale[0, :, :4].clone(), cache.weight[0, :, :200].clone(), cache.slot_pos[0, :, :200].clone()])
    assert all(same_bits(x, y) for x, y in zip(*results))


def test_two_calls_at_once(pkg, store):
    """Attention over one cache on two streams, each with its own scratch and results, again and again: what the calls give one after the other."""
    cache = Cache(pkg, 2, 4, 128, 8192, 64, 0).fill([8000, 5000])
    streams = [torch.cuda.Stream() for _ in range(2)]
    calls, wants = [], []
    for i in range(2):
        q = torch.randn((2 * (1 + 4 * i), 16, 128), device="cuda").bfloat16()
        out = torch.zeros_like(q)
        step, scratch = attend_call(pkg, store, cache, q, out, ints(7000, 4000), 0.09, n=1 + 4 * i)
        keep = ints(7000, 4000)
        step.lengths = keep.data_ptr()
        store.lib.check(store.lib.swlm_op_kv8_attend_dev(store.handle, cache.described(), step, stream()))
        torch.cuda.synchronize()
        wants.append(out.clone())
        calls.append((step, out, scratch, q, keep))
    for _ in range(20):
        for (step, out, *_), s in zip(calls, streams):
            store.lib.check(store.lib.swlm_op_kv8_attend_dev(store.handle, cache.described(), step, C.c_void_p(s.cuda_stream)))
    torch.cuda.synchronize()
    assert all(same_bits(c[1], w) for c, w in zip(calls, wants))
