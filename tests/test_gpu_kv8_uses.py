"""Operators over an 8-bit cache in ways that their interface allows beside the ordinary step: the context's own stream, captured portions at other lengths, portions
on two streams at once, a step after a step after an eviction on one scratch, groups of more heads than a tile has rows."""
import ctypes as C

import pytest
import torch

from plain_kv8 import Cache
from test_gpu_kv8 import append, attend_call, check_attend, evict_call, ints, same_bits, store, stream  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,heads", [(1, 8), (40, 8)])
def test_the_contexts_own_stream(pkg, store, n, heads):  # noqa: F811
    """A null stream is the context's: the same results."""
    cache = Cache(pkg, 2, 2, 64, 512, 32, 0).fill([400, 77])
    q = torch.randn((2 * n, heads, 64), device="cuda").bfloat16()
    lengths, outs = ints(400 - n, 77 - n), []
    for where in (stream(), None):
        out = torch.zeros_like(q)
        step, scratch = attend_call(pkg, store, cache, q, out, lengths, 0.125, n=n)
        torch.cuda.synchronize()
        store.lib.check(store.lib.swlm_op_kv8_attend_dev(store.handle, cache.described(), step, where))
        torch.cuda.synchronize()
        outs.append(out)
    assert same_bits(*outs) and outs[0].abs().sum() > 0


@pytest.mark.parametrize("heads,kv_heads,counts", [(128, 1, [1, 1]), (65, 1, [1, 2]), (96, 2, [1, 1])], ids=str)
@pytest.mark.parametrize("accumulate", [False, True])
def test_groups_of_many_heads(pkg, store, heads, kv_heads, counts, accumulate):  # noqa: F811
    """One token of more heads per KV head than the kernel of few rows takes, and half of a block of rows."""
    cache = Cache(pkg, 2, kv_heads, 64, 640, 64, 1).fill([600, 10])
    check_attend(pkg, store, cache, 2, heads, 64, [600 - counts[0], 10 - counts[1]], counts, torch.float16, accumulate)


def test_max_len_beyond_the_capacity(pkg, store):  # noqa: F811
    cache = Cache(pkg, 2, 2, 64, 128, 16, 0).fill([128, 100])
    for counts in ([1, 1], [40, 30]):
        check_attend(pkg, store, cache, 2, 8, 64, [128 - counts[0], 100 - counts[1]], counts, torch.bfloat16, True, max_len=1 << 20)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_a_captured_portion_replays_at_other_lengths(pkg, store, dtype):  # noqa: F811
    """Append, attention of a portion with weights and an eviction in place, captured at one set of lengths and counts and replayed at others."""
    cache = Cache(pkg, 3, 2, 64, 1024, 32, 1)
    g = torch.Generator(device="cuda").manual_seed(8)
    k, v = (torch.randn((180, 128), generator=g, device="cuda").to(dtype) for _ in range(2))
    q = torch.randn((180, 8, 64), generator=g, device="cuda").to(dtype)
    out = torch.zeros_like(q)
    lengths, counts, starts, refused = ints(0, 10, 500), ints(60, 60, 60), ints(0, 60, 120), ints(0, 0, 0)
    step, scratch = attend_call(pkg, store, cache, q, out, lengths, 0.125, counts, starts, n=60, accumulate=True)
    step.refused = refused.data_ptr()
    after = ints(0, 0, 0)
    how, how_scratch = evict_call(pkg, store, cache, 300, 4, 32, after, after)
    lib = store.lib

    def work():
        append(pkg, store, cache, k, v, lengths, counts, starts, lengths, refused, n=60)
        lib.check(lib.swlm_op_kv8_attend_dev(store.handle, cache.described(), step, stream()))
        lib.check(lib.swlm_op_kv8_lengths_dev(store.handle, 3, lengths.data_ptr(), counts.data_ptr(), 0, 1024, refused.data_ptr(), after.data_ptr(), stream()))
        lib.check(lib.swlm_op_kv8_evict_dev(store.handle, cache.described(), cache.described(), how, stream()))

    start = cache.fill([0, 10, 500]).clone()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            work()
    results = []
    for replay in (True, False):
        for x, y in zip(cache.arrays(), start.arrays()):
            x.copy_(y)
        out.fill_(7.0)
        lengths.copy_(ints(10, 500, 1000)), counts.copy_(ints(23, 60, 60))   # (codes of the first two are garbage to the same extent; the third has no room)
        cache.k_scale.copy_(torch.where(cache.k_scale.isnan(), 0.01, cache.k_scale)), cache.v_scale.copy_(torch.where(cache.v_scale.isnan(), 0.01, cache.v_scale))
        torch.cuda.synchronize()
        graph.replay() if replay else work()
        torch.cuda.synchronize()
        results.append([x.clone() for x in cache.arrays() + [out, after, refused]])
    assert all(same_bits(x, y) for x, y in zip(*results))
    assert refused.tolist() == [0, 0, 1] and after.tolist() == [33, 560, 1000]
    assert (out[23:60] == 7.0).all() and (out[120:] == 7.0).all() and (out[:23] != 7.0).any() and (out[60:120] != 7.0).any()
    assert lib.swlm_op_kv8_status(store.handle) == 0


def test_portions_on_two_streams_at_once(pkg, store):  # noqa: F811
    """Two caches' portions with weights beside each other, again and again: what the calls give one after the other."""
    calls, wants = [], []
    for i in range(2):
        cache = Cache(pkg, 2, 4, 64 << i, 2048, 64, i).fill([1900, 1200], seed=i + 1)
        q = torch.randn((2 * 200, 16, 64 << i), device="cuda").to([torch.bfloat16, torch.float16][i])
        out, lengths = torch.zeros_like(q), ints(1700, 1000)
        step, scratch = attend_call(pkg, store, cache, q, out, lengths, 0.09, n=200, accumulate=True)
        before = cache.weight.clone()
        store.lib.check(store.lib.swlm_op_kv8_attend_dev(store.handle, cache.described(), step, stream()))
        torch.cuda.synchronize()
        wants.append((out.clone(), cache.weight.clone()))
        calls.append((cache, step, out, before, (scratch, q, lengths), torch.cuda.Stream()))
    for _ in range(10):
        for cache, step, out, before, _, s in calls:
            with torch.cuda.stream(s):
                cache.weight.copy_(before)
            store.lib.check(store.lib.swlm_op_kv8_attend_dev(store.handle, cache.described(), step, C.c_void_p(s.cuda_stream)))
    torch.cuda.synchronize()
    assert all(same_bits(c[2], w[0]) and same_bits(c[0].weight, w[1]) for c, w in zip(calls, wants))
    assert store.lib.swlm_op_kv8_status(store.handle) == 0


def test_steps_behind_one_another_share_a_scratch(pkg, store):  # noqa: F811
    """A portion with weights, a decoded token with weights and an eviction, enqueued behind one another on one stream with one scratch, no wait between."""
    cache = Cache(pkg, 1, 2, 128, 4096, 64, 0).fill([4000])
    g = torch.Generator(device="cuda").manual_seed(4)
    results = []
    qs = [torch.randn((n, 8, 128), generator=g, device="cuda").bfloat16() for n in (300, 1, 5)]
    start = cache.clone()
    most = 0
    for together in (False, True):
        for x, y in zip(cache.arrays(), start.arrays()):
            x.copy_(y)
        steps = [attend_call(pkg, store, cache, q, torch.zeros_like(q), ints(4000 - q.shape[0]), 0.09, n=q.shape[0], accumulate=True) for q in qs]
        outs = [torch.zeros_like(q) for q in qs]
        lengths = [ints(4000 - q.shape[0]) for q in qs]
        how, how_scratch = evict_call(pkg, store, cache, 1000, 4, 32, ints(4000), ints(4000))
        end = ints(4000)
        how.lengths = how.seen = end.data_ptr()
        most = max([s.scratch_bytes for s, _ in steps] + [how.scratch_bytes])
        shared = torch.full((most,), 0xFF, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        for _ in range(2):
            for (step, _), out, at in zip(steps, outs, lengths):
                step.out, step.lengths = out.data_ptr(), at.data_ptr()
                if together:
                    step.scratch = shared.data_ptr()
                store.lib.check(store.lib.swlm_op_kv8_attend_dev(store.handle, cache.described(), step, stream()))
                if not together:
                    torch.cuda.synchronize()
        if together:
            how.scratch = shared.data_ptr()
        store.lib.check(store.lib.swlm_op_kv8_evict_dev(store.handle, cache.described(), cache.described(), how, stream()))
        torch.cuda.synchronize()
        results.append([x.clone() for x in outs + cache.arrays()])
    assert all(same_bits(x, y) for x, y in zip(*results))
