"""Attention over an 8-bit cache where the step's append has refused some sequences: they are left alone, whichever kernel works on the others."""
import ctypes as C

import pytest
import torch

from plain_kv8 import Cache, attend
from test_gpu_kv8 import append, attend_call, ints, same_bits, starts_of, store, stream  # noqa: F401

pytestmark = pytest.mark.gpu

CASES = [
    # heads, kv_heads, head_dim, capacity, tokens of a sequence in the step, sequences
    (4, 2, 64, 64, 1, 4),          # a cluster's CTAs, or one, have all slots
    (16, 2, 128, 4096, 1, 6),      # shares of the GPU
    (8, 1, 128, 1024, 5, 4),       # several rows, two tiles
    (2, 2, 64, 64, 1, 520),        # a CTA per head
    (4, 2, 64, 512, 70, 4),        # portions
    (4, 1, 128, 4096, 40, 3),      # portions, slots in several runs
]


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,cap,n,batch", CASES, ids=str)
def test_attend_leaves_refused_sequences_alone(pkg, store, heads, kv_heads, dim, cap, n, batch, accumulate):  # noqa: F811
    """Every third sequence has no room for its tokens, its cache full but for one slot less than it needs; one is parked. Nothing of them changes, and no NaN of the
    slots without tokens gets anywhere; the others are as without them."""
    lengths = [cap - n + 1 if b % 3 == 1 else -1 if b == 2 else (b * 37) % (cap - n) for b in range(batch)]
    no_room = [b % 3 == 1 or b == 2 for b in range(batch)]
    cache = Cache(pkg, batch, kv_heads, dim, cap, 16, 0).fill([max(a, 0) for a in lengths])
    starts, rows = starts_of([n] * batch, gap=1)
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn((rows, kv_heads * dim), generator=g, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn((rows, heads, dim), generator=g, device="cuda").bfloat16()
    out = torch.full_like(q, 7.0)
    refused = ints(*([5] * batch))
    append(pkg, store, cache, k, v, ints(*lengths), ints(*([n] * batch)), ints(*starts), refused=refused)
    before = cache.clone()
    at, counts, first = ints(*lengths), ints(*([n] * batch)), ints(*starts)
    step, scratch = attend_call(pkg, store, cache, q, out, at, dim ** -0.5, counts, first, n=n, accumulate=accumulate)
    step.refused = refused.data_ptr()
    store.lib.check(store.lib.swlm_op_kv8_attend_dev(store.handle, cache.described(), step, stream()))
    torch.cuda.synchronize()
    assert refused.tolist() == [int(x) for x in no_room] and (scratch[step.scratch_bytes:] == 0xFF).all()
    for b in range(batch):
        if no_room[b]:
            assert (out[starts[b]:starts[b] + n] == 7.0).all(), b
            assert same_bits(cache.weight[b], before.weight[b]), b
        elif batch < 100 or b % 7 == 0:
            want, tol, weight, weight_tol = attend(before, q[starts[b]:starts[b] + n], b, lengths[b], dim ** -0.5, cap)
            assert ((out[starts[b]:starts[b] + n].double() - want).abs() <= tol).all(), b
            if accumulate:
                weight += before.weight[b].double()
                assert ((cache.weight[b].double() - weight).abs() <= weight_tol + 2.0 ** -24 * weight.abs()).all(), b
            else:
                assert same_bits(cache.weight[b], before.weight[b]), b
    assert all(same_bits(x, y) for x, y in list(zip(cache.arrays(), before.arrays()))[:4])


def test_a_captured_step_leaves_out_what_no_longer_fits(pkg, store):  # noqa: F811
    """A replayed step whose second sequence runs full: its counters, weights and rows of results stay from then on, the first one's go on."""
    cache = Cache(pkg, 2, 1, 64, 64, 16, 0).fill([20, 62])
    lengths, seen, refused = ints(20, 62), ints(20, 62), ints(0, 0)
    k, v, q = (torch.randn((2, w), device="cuda").bfloat16() for w in (64, 64, 256))
    out = torch.zeros((2, 4, 64), device="cuda").bfloat16()
    step, scratch = attend_call(pkg, store, cache, q.view(2, 4, 64), out, lengths, 0.125, n=1, accumulate=True)
    step.refused = refused.data_ptr()
    lib, side, graph = store.lib, torch.cuda.Stream(), torch.cuda.CUDAGraph()

    def work():
        append(pkg, store, cache, k, v, lengths, None, None, seen, refused, n=1)
        lib.check(lib.swlm_op_kv8_attend_dev(store.handle, cache.described(), step, stream()))
        for x, most in ((lengths, 64), (seen, 2 ** 31 - 1)):
            lib.check(lib.swlm_op_kv8_lengths_dev(store.handle, 2, x.data_ptr(), None, 1, most, refused.data_ptr(), x.data_ptr(), C.c_void_p(torch.cuda.current_stream().cuda_stream)))

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            work()
        graph.replay()
        side.synchronize()
        assert lengths.tolist() == [22, 64] and refused.tolist() == [0, 0]
        full, weight, rows = cache.clone(), cache.weight.clone(), out.clone()
        q.copy_(torch.randn_like(q))
        graph.replay()
        side.synchronize()
    assert lengths.tolist() == [23, 64] and seen.tolist() == [23, 64] and refused.tolist() == [0, 1]
    assert same_bits(out[1], rows[1]) and not same_bits(out[0], rows[0])
    assert same_bits(cache.weight[1], weight[1]) and all(same_bits(x[1], y[1]) for x, y in zip(cache.arrays(), full.arrays()))
