"""What a call has copied to the device is there when it returns: steps that run next on the library's own streams, which wait for no other stream, read the new values also while
other copies keep the way to the device busy."""
import threading

import numpy as np
import pytest
import torch

import vuzunex_cases as vc

pytestmark = pytest.mark.gpu
WIDTH, ROWS, TURNS = 8192, 3, 300


@pytest.fixture(scope="module")
def store(pkg):
    s = pkg.WeightStore(0)
    yield s
    s.close()


@pytest.fixture
def busy():
    """Copies from pinned memory on another stream, one behind the other."""
    stop = threading.Event()
    host, device = torch.empty(32 << 20, dtype=torch.uint8).pin_memory(), torch.empty(32 << 20, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.Stream()

    def copies():
        with torch.cuda.stream(stream):
            while not stop.is_set():
                for _ in range(4):
                    device.copy_(host, non_blocking=True)
                stream.synchronize()

    thread = threading.Thread(target=copies)

    def start():
        thread.start()

    yield start
    stop.set()
    if thread.ident is not None:
        thread.join()
    torch.cuda.synchronize()


def norm_of(pkg, store, weight):
    P = pkg.plan
    st = P._step(P.STEP_COPY_RMSNORM, in_buf=P.BUF_HIDDEN, out_buf=P.BUF_S0, n=WIDTH, eps=1e-5, weight_bias=0.0, weight=weight)
    desc = P.BuffersDesc(hidden=WIDTH, vocab=8, max_seq=64, max_batch=ROWS, stream_dtype=P.STREAM_ALL_F32)
    return st, pkg.InferenceModel(store, [st], desc)


def turns(busy, put, look):
    """What each of two values leads to, when nothing else runs; then both in turn, many times over."""
    want = []
    for i in range(2):
        put(i)
        torch.cuda.synchronize()
        want.append(look())
    assert not np.array_equal(want[0], want[1])
    busy()
    late = 0
    for t in range(TURNS):
        put(t % 2)
        late += not np.array_equal(look(), want[t % 2])
    assert late == 0


def test_buffers(pkg, store, busy):
    rng = np.random.default_rng(1)
    store.add_dense("up.norm", vc.to_bf16_bits(1 + 0.3 * rng.standard_normal(WIDTH)))
    st, m = norm_of(pkg, store, "up.norm")
    x = [rng.standard_normal((ROWS, WIDTH)).astype(np.float32) for _ in range(2)]

    def look():
        m.run_step(st)
        return m.read_buffer_f32(pkg.plan.BUF_S0, ROWS, WIDTH)

    turns(busy, lambda i: m.write_buffer_f32(pkg.plan.BUF_HIDDEN, x[i]), look)
    m.close()


def test_weights_in_place(pkg, store, busy):
    rng, P = np.random.default_rng(2), pkg.plan
    table = [vc.to_bf16_bits(rng.standard_normal((64, WIDTH))) for _ in range(2)]
    store.add_dense("up.embed", table[0])
    st = P._step(P.STEP_EMBED, out_buf=P.BUF_HIDDEN, n=WIDTH, scale=1.0, weight="up.embed")
    m = pkg.InferenceModel(store, [st], P.BuffersDesc(hidden=WIDTH, vocab=64, max_seq=64, max_batch=ROWS, stream_dtype=P.STREAM_ALL_F32))

    def look():
        m.run_step(st, token_in=[63, 0, 62])
        return m.read_buffer_f32(P.BUF_HIDDEN, ROWS, WIDTH)

    turns(busy, lambda i: store.add_dense("up.embed", table[i]), look)
    m.close()


def test_counters_that_a_first_call_makes_are_zero_before_its_kernel(pkg):
    """They come from memory that others have filled, and are cleared while another stream keeps the SMs busy."""
    g = torch.Generator(device="cuda").manual_seed(4)
    heads, kv_heads, dim, length = 32, 8, 128, 4096
    q, k, v = (torch.randn((h, n, dim), generator=g, device="cuda").bfloat16() for h, n in ((heads, 1), (kv_heads, length), (kv_heads, length)))
    a = torch.randn((4096, 4096), device="cuda", dtype=torch.bfloat16)
    other, mine = torch.cuda.Stream(), torch.cuda.Stream()
    want = None
    for busy_first in (False, True, True, True):
        s = pkg.WeightStore(0)
        filled = torch.full((1 << 30,), 0xFF, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        del filled
        torch.cuda.empty_cache()
        out = torch.zeros((heads, dim), dtype=torch.bfloat16, device="cuda")
        scratch = torch.zeros(s.lib.swlm_op_flash_decode_scratch_bytes(1, heads, kv_heads, dim, length), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        if busy_first:
            with torch.cuda.stream(other):
                for _ in range(50):
                    a @ a
        s.lib.check(s.lib.swlm_op_flash_decode_dev(s.handle, 1, heads, kv_heads, dim, length, length, dim ** -0.5, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                                   scratch.data_ptr(), mine.cuda_stream))
        torch.cuda.synchronize()
        if want is None:
            want = out.clone()
            ref = torch.softmax((q.float().view(kv_heads, heads // kv_heads, dim) @ k.float().transpose(1, 2)) * dim ** -0.5, dim=-1) @ v.float()
            # (the result rounds to bf16, by 2^-8 of itself at most; as much again for weights of which 16 bits meet the values)
            assert (out.float() - ref.view(heads, dim)).abs().max() <= 2.0 ** -7 * ref.abs().max()
        assert torch.equal(out, want)
        s.close()
