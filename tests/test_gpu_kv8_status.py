"""What callers of attention over an 8-bit cache learn of a wait that expired on the device. The word that a kernel would set is written by the host."""
import pytest
import torch

from plain_kv8 import Cache
from test_gpu_kv8 import append, attend_call, evict_call, ints, same_bits, stream

pytestmark = pytest.mark.gpu
OK, TIMEOUT = 0, -5


@pytest.fixture()
def own_store(pkg):
    s = pkg.WeightStore(0)   # a context of its own: the word belongs to one
    yield s
    s.close()


def test_an_expired_wait_is_reported_until_it_is_asked_for(pkg, own_store):
    store, lib = own_store, own_store.lib
    cache = Cache(pkg, 1, 2, 64, 128, 16, 0).fill([100])
    q = torch.randn((1, 4, 64), device="cuda").bfloat16()
    out, lengths = torch.full_like(q, 7.0), ints(99)
    step, scratch = attend_call(pkg, store, cache, q, out, lengths, 0.125, n=1, accumulate=True)
    how, how_scratch = evict_call(pkg, store, cache, 50, 2, 4, lengths, lengths)
    before = cache.clone()

    def attend_and_evict():
        results = (lib.swlm_op_kv8_attend_dev(store.handle, cache.described(), step, stream()),
                   lib.swlm_op_kv8_evict_dev(store.handle, cache.described(), cache.described(), how, stream()))
        torch.cuda.synchronize()
        return results

    assert lib.swlm_op_kv8_status(store.handle) == OK
    assert lib.swlm_write_kv8_status(store.handle, 33) == OK
    for _ in range(2):   # (whichever call comes first does not take the report from the others)
        assert attend_and_evict() == (TIMEOUT, TIMEOUT) and b"33" in lib.swlm_last_error()
        assert (out == 7.0).all() and all(same_bits(x, y) for x, y in zip(cache.arrays(), before.arrays()))
    with torch.cuda.stream(torch.cuda.Stream()):
        assert attend_and_evict() == (TIMEOUT, TIMEOUT)
    append(pkg, store, cache, q.view(1, 256), q.view(1, 256), ints(100), n=1)   # (an append depends on no result)
    assert lib.swlm_op_kv8_status(store.handle) == TIMEOUT and b"33" in lib.swlm_last_error()
    assert lib.swlm_op_kv8_status(store.handle) == OK
    assert attend_and_evict() == (OK, OK) and (out != 7.0).any()


def test_replays_leave_their_report_to_the_status(pkg, own_store):
    """A captured call reports nothing when it is replayed; the status does."""
    store, lib = own_store, own_store.lib
    cache = Cache(pkg, 1, 2, 64, 128, 16, 0).fill([100])
    q = torch.randn((40, 4, 64), device="cuda").bfloat16()
    out, lengths = torch.zeros_like(q), ints(60)
    step, scratch = attend_call(pkg, store, cache, q, out, lengths, 0.125, n=40)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lib.check(lib.swlm_op_kv8_attend_dev(store.handle, cache.described(), step, stream()))
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            lib.check(lib.swlm_op_kv8_attend_dev(store.handle, cache.described(), step, stream()))
        graph.replay()
        side.synchronize()
        assert lib.swlm_op_kv8_status(store.handle) == OK
        lib.swlm_write_kv8_status(store.handle, 32)
        graph.replay()
        side.synchronize()
    assert lib.swlm_op_kv8_status(store.handle) == TIMEOUT
    assert lib.swlm_op_kv8_status(store.handle) == OK
