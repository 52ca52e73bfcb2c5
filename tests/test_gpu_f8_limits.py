"""Operators over 8-bit float weights and over rows sorted by expert at the ends of their ranges: nothing to do on the device, long rows, many columns, scales far
apart, as many pairs as there may be, calls from several threads."""
import threading

import pytest
import torch

from plain_f8 import E4M3, Calls, blocks, check, expected, matrix, quantized, room, rows_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def store(pkg):
    s = pkg.WeightStore(0)
    yield s
    torch.cuda.synchronize()
    s.lib.check(s.lib.swlm_op_f8_status(s.handle))
    s.close()


@pytest.fixture(scope="module")
def calls(pkg, store):
    return Calls(pkg, store)


@pytest.fixture(autouse=True)
def memory():
    """These tests take tens of gigabytes: what one has had is free for the next, and for other programs' contexts."""
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("dtype", [torch.float32, E4M3], ids=str)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("tokens,top,n,k,experts", [(16, 4, 640, 300, 4), (2, 2, 257, 4096, 2), (10000, 2, 640, 300, 4)])
def test_no_token_chose_an_expert(calls, tokens, top, n, k, experts, gated, dtype):
    """A batch of parked tokens only: no row of codes, of a product or of their scales changes, and every token keeps what is added to it."""
    g = generator(tokens)
    rows = tokens * top
    choice = torch.full((tokens, top), -1, dtype=torch.int32, device="cuda")
    offsets, source, place = (torch.full((m,), 9, dtype=torch.int32, device="cuda") for m in (experts + 1, rows, rows))
    calls.sort(choice, offsets, source, place)
    assert (offsets == 0).all() and (source == -1).all() and (place == -1).all()
    x, w = rows_of(g, rows, k), matrix(g, n, k, experts)
    was = x[0].view(torch.uint8).clone(), x[1].clone()
    calls.quantize(torch.randn((tokens, 304), generator=g, device="cuda")[:, :k] if k < 304 else torch.randn((tokens, k), generator=g, device="cuda"), x, source)
    assert torch.equal(x[0].view(torch.uint8), was[0]) and torch.equal(x[1], was[1])
    held, scale = room(rows, n, dtype, 0x35), torch.full((blocks(n), rows), 7.0, device="cuda")
    before = held._base.view(torch.uint8).clone()
    calls.product(x, w, (held, scale) if dtype == E4M3 else held, w if gated else None, "silu" if gated else "plain", offsets)
    torch.cuda.synchronize()
    assert torch.equal(held._base.view(torch.uint8), before) and (scale == 7.0).all()
    if dtype != E4M3:
        add = room(tokens, n, torch.float32)
        add.copy_(torch.randn((tokens, n), generator=g, device="cuda"))
        out = room(tokens, n, torch.float32, 0x35)
        calls.sum(held, place.view(tokens, top), torch.full((tokens, top), float("nan"), device="cuda"), out, add)
        assert torch.equal(out, add)


@pytest.mark.parametrize("rows,n,k", [(3, 130, 1 << 22), (300, 130, 1 << 19), (2, 1 << 24, 16), (600, 1 << 19, 16)])
def test_products_of_long_rows_and_of_many_columns(calls, rows, n, k):
    g = generator(rows)
    x, w, y = rows_of(g, rows, k), matrix(g, n, k), room(rows, n, torch.float32)
    calls.product(x, w, y)
    check(y, *expected("plain", x, w))


def test_long_rows_quantized_and_added_up(calls):
    """The widest rows: 2^24 columns."""
    width = 1 << 24
    g = generator(41)
    x = torch.randn((2, width), generator=g, device="cuda").bfloat16()
    out = room(2, width, E4M3), torch.zeros((blocks(width), 2), device="cuda")
    calls.quantize(x, out, torch.tensor([1, 0], dtype=torch.int32, device="cuda"))
    for r in range(2):
        for at in (slice(0, 1 << 15), slice(width - (1 << 15), width)):
            want, scale = quantized(x[1 - r:2 - r, at].double())
            assert torch.equal(out[0][r:r + 1, at].double(), want) and torch.equal(out[1][at.start // 128:at.stop // 128, r:r + 1].double(), scale)
    assert (out[1] > 0).all()
    place, weight = torch.tensor([[1, 0], [0, -1]], dtype=torch.int32, device="cuda"), torch.tensor([[0.5, 0.25], [2.0, 1.0]], device="cuda")
    total = torch.empty((2, width), device="cuda")
    calls.sum(x, place, weight, total)
    # (products with powers of two are exact, their sum rounds once, as it does here)
    assert torch.equal(total[0], 0.5 * x[1].float() + 0.25 * x[0].float()) and torch.equal(total[1], 2.0 * x[0].float())


@pytest.mark.parametrize("gated,rows,n,k", [(False, 3, 300, 300), (True, 3, 300, 300), (False, 1100, 2600, 300)])
def test_scales_that_lie_far_apart(calls, gated, rows, n, k):
    """Scales' offsets in bytes that pass 32 bits: the bits are those of the same scales close together."""
    g = generator(42)
    far = (1 << 30) + 5
    wide = torch.randn((rows, 304), generator=g, device="cuda")[:, :k]
    near, apart = (room(rows, k, E4M3), torch.zeros((blocks(k), rows), device="cuda")), (room(rows, k, E4M3), torch.as_strided(torch.zeros(((blocks(k) - 1) * far + rows,), device="cuda"), (blocks(k), rows), (far, 1)))
    for x in (near, apart):
        calls.quantize(wide, x)
    torch.cuda.synchronize()
    assert torch.equal(near[0].view(torch.uint8), apart[0].view(torch.uint8)) and torch.equal(near[1], apart[1])
    w, up = matrix(g, n, k), matrix(g, n, k) if gated else None
    last = blocks(n) - 1
    stride = far if last < 4 else far // 8
    y = room(rows, n, E4M3), torch.zeros((blocks(n), rows), device="cuda")
    z = room(rows, n, E4M3), torch.as_strided(torch.zeros((last * stride + rows,), device="cuda"), (blocks(n), rows), (stride, 1))
    calls.product(near, w, y, up, "silu" if gated else "plain")
    calls.product(apart, w, z, up, "silu" if gated else "plain")
    torch.cuda.synchronize()
    assert torch.equal(y[0].view(torch.uint8), z[0].view(torch.uint8)) and torch.equal(y[1], z[1]) and (y[1] > 0).all()


def test_sort_of_as_many_pairs_as_there_may_be(calls):
    """2^30 pairs: a row for every choice in range, ascending by expert, and of one expert in the order of the pairs."""
    top, experts = 7, 1000
    tokens = (1 << 30) // top
    choice = torch.randint(-20, experts + 20, (tokens, top), generator=generator(43), device="cuda", dtype=torch.int32)
    offsets, source = torch.empty(experts + 1, dtype=torch.int32, device="cuda"), torch.empty(tokens * top, dtype=torch.int32, device="cuda")
    place = torch.empty((tokens, top), dtype=torch.int32, device="cuda")
    calls.sort(choice, offsets, source, place)
    flat, row = choice.view(-1), place.view(-1)
    there = (flat >= 0) & (flat < experts)
    total = int(there.sum())
    counts = torch.bincount(flat[there], minlength=experts)
    assert torch.equal(offsets[1:].long(), counts.cumsum(0)) and offsets[0] == 0 and int(offsets[-1]) == total
    assert (row[~there] == -1).all() and (source[total:] == -1).all()
    # the pair of every row, by way of its place: each row has exactly one where no two pairs have the same
    pair = torch.full((total,), -1, dtype=torch.int32, device="cuda")
    pair[row[there].long()] = torch.arange(tokens * top, dtype=torch.int32, device="cuda")[there]
    assert (pair >= 0).all()
    assert torch.equal(source[:total], pair // top)
    expert = flat[pair.long()]
    assert ((expert[1:] > expert[:-1]) | ((expert[1:] == expert[:-1]) & (pair[1:] > pair[:-1]))).all()


def test_calls_from_several_threads(calls, pkg, store):
    """Threads with streams of their own and one context: the bits are those of the calls alone."""
    sizes = [(5, 700, 900, "plain"), (300, 640, 1024, "silu"), (1100, 2600, 300, "plain"), (1, 4096, 700, "clamped")]
    data, want = [], []
    for i, (rows, n, k, act) in enumerate(sizes):
        g = generator(50 + i)
        data.append((rows_of(g, rows, k), matrix(g, n, k), matrix(g, n, k) if act != "plain" else None, act))
        y = room(rows, n, torch.bfloat16)
        calls.product(data[-1][0], data[-1][1], y, *data[-1][2:])
        want.append(y.clone())
    rooms = [[room(rows, n, torch.bfloat16) for _ in range(30)] for rows, n, _, _ in sizes]
    streams = [torch.cuda.Stream() for _ in sizes]
    torch.cuda.synchronize()
    errors = []

    def work(i):
        try:
            mine = Calls(pkg, store, streams[i].cuda_stream)
            for y in rooms[i]:
                mine.product(data[i][0], data[i][1], y, *data[i][2:])
        except Exception as e:   # (an assertion in a thread would go unseen)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sizes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for got, expect in zip(rooms, want):
        for y in got:
            assert torch.equal(y, expect)
