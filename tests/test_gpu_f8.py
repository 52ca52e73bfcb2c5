"""Operators over 8-bit float weights with a scale per block of 128 x 128 and over rows sorted by expert, against plain forms in 64 bits
(tests/plain_f8.py)."""
import math

import pytest
import torch

from plain_f8 import E4M3, Calls, blocks, check, check_codes, expected, matrix, quantized, room, row_values, rows_of, sort

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


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


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def code_room(rows, width, fill=0x35):
    scale = torch.full((blocks(width), rows + 5), 7.0, device="cuda")
    return room(rows, width, E4M3, fill), scale[:, :rows]


def around(view):
    """All of the memory that a view of rows lies in, as bytes."""
    return view._base.reshape(-1).view(torch.uint8) if view._base is not None else view.reshape(-1).view(torch.uint8)


def same_but(view, before, allowed):
    """Memory is as it was outside of `allowed`, a selection of the view's entries."""
    kept = view._base.clone()
    other = torch.as_strided(kept, view.shape, view.stride(), view.storage_offset())
    was = torch.as_strided(before, view.shape, view.stride(), view.storage_offset())
    other.view(torch.uint8 if other.element_size() == 1 else other.dtype)[allowed] = was.view(torch.uint8 if was.element_size() == 1 else was.dtype)[allowed]
    return torch.equal(kept.view(torch.uint8), before.view(torch.uint8))


# ---- quantize --------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 128), (3, 7), (8, 129), (9, 255), (17, 1024), (2, 1025), (5, 2056), (40, 333)])
def test_quantize(calls, rows, width, dtype):
    """Codes and scales are the definition's, bit for bit, over values of many sizes, with gaps behind rows that stay as they are."""
    g = generator(rows * width)
    x = room(rows, width, dtype)
    x.copy_(torch.randn((rows, width), generator=g, device="cuda") * torch.exp(2 * torch.randn((rows, 1), generator=g, device="cuda")))
    out = code_room(rows, width)
    before = out[0]._base.clone(), out[1]._base.clone()
    calls.quantize(x, out)
    want, scale = quantized(x.double())
    assert torch.equal(out[0].double(), want) and torch.equal(out[1].double(), scale)
    assert same_but(out[0], before[0], ...) and same_but(out[1], before[1], ...)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_quantize_at_the_scales_borders(calls, dtype):
    """Largest values at, below and above 448 times a power of two, zeros, the smallest and the largest numbers; ties of codes go to even."""
    info = torch.finfo(dtype)
    x = torch.zeros((12, 128), device="cuda", dtype=dtype)
    x[0, 5], x[1, 6], x[2, 7] = 448.0, 448.0 * (1 + info.eps), 448.0 * (1 - info.eps / 2)
    x[3, 0], x[4, 1], x[5, 2], x[6, 3] = 1.75 / 64, -1.75 / 64, info.max, -info.max
    x[7, 100], x[8, 3], x[9] = info.smallest_normal, info.smallest_normal * info.eps, 0.0   # (the second is the smallest subnormal number)
    x[10] = torch.arange(128, device="cuda") / 8 + 1.0 / 16   # between codes
    x[10, 0] = 448.0
    x[11] = torch.arange(128, device="cuda") * 2.0 ** -10
    x[11, 0] = 300.0
    out = code_room(12, 128)
    calls.quantize(x, out)
    want, scale = quantized(x.double())
    assert torch.equal(out[0].double(), want) and torch.equal(out[1].double(), scale)
    assert out[1][0, 9] == 2.0 ** -126 and (out[0][9].float() == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_quantize_of_values_that_are_not_finite(calls, dtype):
    """They make their row's block NaN, and nothing else."""
    x = torch.randn((4, 300), generator=generator(3), device="cuda").to(dtype)
    x = torch.nn.functional.pad(x, (0, 4))[:, :300]
    x[0, 3], x[1, 200], x[2, 299] = math.inf, -math.inf, math.nan
    out = code_room(4, 300)
    calls.quantize(x, out)
    want, scale = quantized(x.double())
    assert torch.equal(out[0].double().nan_to_num(1e9), want.nan_to_num(1e9)) and torch.equal(out[1].double().nan_to_num(-1.0), scale.nan_to_num(-1.0))
    assert out[1].isnan().sum() == 3


def test_quantize_of_gathered_rows(calls):
    """Rows in any order, the same one several times; places without a row stay as they are."""
    x = torch.randn((5, 264), generator=generator(4), device="cuda").bfloat16()
    source = [4, 0, 4, -1, 2, 5, 1 << 30, 0, -(1 << 31)]
    out = code_room(len(source), 264)
    before = out[0].view(torch.uint8).clone(), out[1].clone()
    calls.quantize(x, out, ints(*source))
    want, scale = quantized(x.double())
    for r, s in enumerate(source):
        if 0 <= s < 5:
            assert torch.equal(out[0][r].double(), want[s]) and torch.equal(out[1][:, r].double(), scale[:, s])
        else:
            assert torch.equal(out[0].view(torch.uint8)[r], before[0][r]) and torch.equal(out[1][:, r], before[1][:, r])


# ---- product ---------------------------------------------------------------------------------------------------------------

SHAPES = [(1, 1, 1), (1, 128, 128), (1, 4096, 700), (2, 129, 130), (3, 8, 1000), (7, 100, 17), (16, 256, 384), (17, 200, 129), (33, 1000, 64), (64, 128, 2049),
          (65, 127, 256), (100, 384, 512), (128, 130, 300), (129, 513, 257), (300, 640, 1024), (513, 264, 100)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,n,k", SHAPES)
def test_product(calls, rows, n, k, dtype):
    g = generator(rows + n + k)
    x, w, y = rows_of(g, rows, k), matrix(g, n, k), room(rows, n, dtype, 0x35)
    before = y._base.clone()
    calls.product(x, w, y)
    check(y, *expected("plain", x, w))
    assert same_but(y, before, ...)


@pytest.mark.parametrize("act", ["silu", "gelu", "clamped"])
@pytest.mark.parametrize("rows,n,k", SHAPES)
def test_gated_product(calls, rows, n, k, act):
    g = generator(rows + n + k + 1)
    x, w, up, y = rows_of(g, rows, k), matrix(g, n, k), matrix(g, n, k), room(rows, n, torch.float32, 0x35)
    before = y._base.clone()
    calls.product(x, w, y, up, act)
    check(y, *expected(act, x, w, up))
    assert same_but(y, before, ...)


@pytest.mark.parametrize("act", ["plain", "silu", "gelu", "clamped"])
@pytest.mark.parametrize("rows,n,k", SHAPES)
def test_product_into_codes(calls, rows, n, k, act):
    g = generator(rows + n + k + 2)
    x, w, up, y = rows_of(g, rows, k), matrix(g, n, k), matrix(g, n, k), code_room(rows, n)
    before = y[0]._base.clone(), y[1]._base.clone()
    calls.product(x, w, y, up if act != "plain" else None, act)
    check_codes(*y, *expected(act, x, w, up))
    assert same_but(y[0], before[0], ...) and same_but(y[1], before[1], ...)


@pytest.mark.parametrize("rows,n,k", [(5, 200, 384), (200, 200, 384)])
def test_product_keeps_what_is_not_a_number_in_its_place(calls, rows, n, k):
    """A NaN code or scale of a row makes that row's results NaN, one of a matrix its column's or its block's, and no other."""
    g = generator(7)
    x, w = rows_of(g, rows, k), matrix(g, n, k)
    want, off = expected("plain", x, w)
    bad = torch.zeros((rows, n), dtype=torch.bool, device="cuda")
    x[0].view(torch.uint8)[1, 200] = 0x7F
    x[1][2, 3] = math.nan
    w[0].view(torch.uint8)[0, 50, 130] = 0xFF
    w[1][0, 1, 0] = math.nan
    bad[1], bad[3], bad[:, 50], bad[:, 128:] = True, True, True, True
    y = room(rows, n, torch.float32)
    calls.product(x, w, y)
    assert torch.equal(y.isnan(), bad)
    check(torch.where(bad, 0.0, y), torch.where(bad, 0.0, want), off)


@pytest.mark.parametrize("rows", [1, 200])
def test_product_over_scales_of_many_sizes(calls, rows):
    """Blocks' scales from 2^-40 to 2^40, rows of zeros, matrices of zeros."""
    g = generator(8)
    x, w = rows_of(g, rows, 512), matrix(g, 256, 512)
    x[1].copy_(torch.exp2(torch.randint(-40, 41, x[1].shape, generator=g, device="cuda").float()))
    w[1].copy_(torch.exp2(torch.randint(-40, 41, w[1].shape, generator=g, device="cuda").float()) * 1.1)
    x[0].view(torch.uint8)[0, :300] = 0
    w[0].view(torch.uint8)[0, 9] = 0x80   # minus zeros
    y = room(rows, 256, torch.float32)
    calls.product(x, w, y)
    check(y, *expected("plain", x, w))
    assert (y[:, 9] == 0).all()


OFFSETS = [[0, 1], [0, 0, 1], [0, 3, 3, 3, 10], [0, 200, 201, 201, 330], [0, 0, 0, 129], [0, 64, 128, 257], [5, 40, 300], [0] * 40 + [7], list(range(65))]


@pytest.mark.parametrize("act,dtype", [("plain", torch.bfloat16), ("silu", torch.float32), ("clamped", E4M3)])
@pytest.mark.parametrize("offsets", OFFSETS, ids=str)
def test_product_of_experts(calls, offsets, act, dtype):
    """Every expert's rows meet its own matrix; experts without rows, rows before the first and behind the last expert's, which stay as they are."""
    experts, rows, n, k = len(offsets) - 1, offsets[-1] + 4, 200, 272
    g = generator(sum(offsets) + experts)
    x, w, up = rows_of(g, rows, k), matrix(g, n, k, experts), matrix(g, n, k, experts)
    y = code_room(rows, n) if dtype == E4M3 else room(rows, n, dtype, 0x35)
    held = y[0] if dtype == E4M3 else y
    before = held._base.clone()
    calls.product(x, w, y, up if act != "plain" else None, act, ints(*offsets))
    for e in range(experts):
        at = slice(offsets[e], offsets[e + 1])
        part = x[0][at], x[1][:, at]
        if offsets[e] < offsets[e + 1]:
            want = expected(act, part, w, up, e)
            if dtype == E4M3:
                check_codes(y[0][at], y[1][:, at], *want)
            else:
                check(y[at], *want)
    assert same_but(held, before, slice(offsets[0], offsets[-1]))


@pytest.mark.parametrize("offsets,reach", [([0, 5, 100], [(0, 5), (5, 20)]), ([-7, 5, 5], [(0, 5), (5, 5)]), ([0, 1 << 30, 1 << 30], [(0, 20), (20, 20)]),
                                           ([-(1 << 31), -3, (1 << 31) - 1], [(0, 0), (0, 20)])])
def test_product_cuts_offsets_to_its_rows(calls, offsets, reach):
    g = generator(11)
    x, w, y = rows_of(g, 20, 130), matrix(g, 130, 130, 2), room(20, 130, torch.float32)
    calls.product(x, w, y, offsets=ints(*offsets))
    for e, (a, b) in enumerate(reach):
        if a < b:
            check(y[a:b], *expected("plain", (x[0][a:b], x[1][:, a:b]), w, e=e))


# ---- sort, sum -------------------------------------------------------------------------------------------------------------

def do_sort(calls, choice, experts):
    n = choice.numel()
    offsets, source, place = (torch.full((m + 2,), -77, dtype=torch.int32, device="cuda") for m in (experts + 1, n, n))
    calls.sort(choice, offsets[1:experts + 2], source[1:n + 1], place[1:n + 1])
    for x in (offsets, source, place):
        assert x[0] == -77
    assert offsets[-1] == -77 and source[-1] == -77 and place[-1] == -77
    return offsets[1:-1], source[1:n + 1], place[1:n + 1].view(choice.shape)


@pytest.mark.parametrize("tokens,top,experts", [(1, 1, 1), (1, 8, 64), (5, 3, 7), (16, 8, 64), (100, 2, 1000), (257, 8, 32), (333, 7, 1024), (1024, 4, 33), (4097, 8, 256),
                                                (20000, 8, 512), (40000, 5, 1024), (3, 40, 100)])
def test_sort(calls, tokens, top, experts):
    """Choices out of range on either side, some experts without tokens, a token with the same choice twice."""
    g = generator(tokens + top)
    choice = (torch.randn((tokens, top), generator=g, device="cuda") * experts / 3).to(torch.int32) + experts // 8
    choice[-1, -1] = -(1 << 31)
    choice[0, 0] = (1 << 31) - 1 if tokens > 1 else 0
    got = do_sort(calls, choice, experts)
    for a, b in zip(got, sort(choice, experts)):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("value", [-1, 0, 4, 5])
@pytest.mark.parametrize("tokens", [0, 1, 33, 5000])
def test_sort_of_equal_choices(calls, tokens, value):
    choice = torch.full((tokens, 4), value, dtype=torch.int32, device="cuda")
    room_for = choice if tokens else torch.zeros((1, 4), dtype=torch.int32, device="cuda")[:0]
    if tokens:
        for a, b in zip(do_sort(calls, choice, 5), sort(choice, 5)):
            assert torch.equal(a.cpu(), b)
    else:
        offsets, other = torch.full((6,), 9, dtype=torch.int32, device="cuda"), ints(9)
        call = calls.pkg.ExpertSort(choice=other.data_ptr(), offsets=offsets.data_ptr(), source=other.data_ptr(), place=other.data_ptr(), tokens=0, top=4, experts=5)
        calls.lib.check(calls.lib.swlm_op_expert_sort_dev(calls.handle, call, calls.stream))
        assert (offsets == 0).all() and other.item() == 9 and room_for.numel() == 0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("y_dtype", TYPES, ids=str)
@pytest.mark.parametrize("tokens,top,width", [(1, 1, 1), (3, 2, 7), (5, 8, 264), (20, 9, 100), (7, 17, 33), (300, 3, 1032)])
def test_sum(calls, tokens, top, width, y_dtype, dtype):
    """Rows taken several times and not at all, places without a row (whose weight is NaN), with and without something to add to, in place too."""
    g = generator(tokens * top + width)
    rows = tokens * top
    y = room(rows, width, y_dtype)
    y.copy_(torch.randn((rows, width), generator=g, device="cuda"))
    place = torch.randint(-rows // 4 - 1, rows + rows // 4 + 1, (tokens, top), generator=g, device="cuda", dtype=torch.int32)
    weight = torch.randn((tokens, top), generator=g, device="cuda")
    there = (place >= 0) & (place < rows)
    weight[~there] = math.nan
    base = torch.randn((tokens, width), generator=g, device="cuda").to(dtype)
    picked = y.double()[place.clamp(0, rows - 1).reshape(-1).long()].view(tokens, top, width) * torch.where(there, weight, 0.0).double()[..., None]
    for add in (False, True):
        out = room(tokens, width, dtype, 0x35)
        if add:
            out.copy_(base)
        before = out._base.clone()
        calls.sum(y, place, weight, out, out if add else None)
        want = picked.sum(dim=1) + (base.double() if add else 0.0)
        # every addend rounds the sum once, by 2^-24 of what it has come to
        check(out, want, (picked.abs().sum(dim=1) + base.double().abs()) * (top + 1) * 2.0 ** -24)
        assert same_but(out, before, ...)


# ---- all of them -----------------------------------------------------------------------------------------------------------

def routed_rooms(tokens, width, ff, experts, top):
    n = tokens * top
    return {"offsets": torch.zeros(experts + 1, dtype=torch.int32, device="cuda"), "source": torch.zeros(n, dtype=torch.int32, device="cuda"),
            "place": torch.zeros((tokens, top), dtype=torch.int32, device="cuda"), "rows": code_room(n, width), "mid": code_room(n, ff), "y": room(n, width, torch.bfloat16),
            "out": room(tokens, width, torch.bfloat16)}


def routed(calls, x, choice, share, w, up, down, act, r):
    calls.sort(choice, r["offsets"], r["source"], r["place"])
    calls.quantize(x, r["rows"], r["source"])
    calls.product(r["rows"], w, r["mid"], up, act, r["offsets"])
    calls.product(r["mid"], down, r["y"], offsets=r["offsets"])
    calls.sum(r["y"], r["place"], share, r["out"])


@pytest.mark.parametrize("tokens,width,ff,experts,top,act", [(1, 256, 128, 4, 2, "silu"), (19, 384, 200, 8, 3, "clamped"), (150, 264, 136, 3, 2, "gelu"), (70, 512, 256, 64, 8, "silu")])
def test_routed_feed_forward(calls, tokens, width, ff, experts, top, act):
    """Each operator on what the one before it has left: its result is the plain form's of that, so that roundings of one do not blur the next."""
    g = generator(tokens)
    x = torch.randn((tokens, width), generator=g, device="cuda").bfloat16()
    choice = torch.rand((tokens, experts), generator=g, device="cuda").topk(top).indices.int()
    choice[torch.rand((tokens, top), generator=g, device="cuda") < 0.1] = -1
    share = torch.rand((tokens, top), generator=g, device="cuda")
    w, up, down = matrix(g, ff, width, experts), matrix(g, ff, width, experts), matrix(g, width, ff, experts)
    r = routed_rooms(tokens, width, ff, experts, top)
    routed(calls, x, choice, share, w, up, down, act, r)
    offsets, source, place = sort(choice, experts)
    assert torch.equal(r["offsets"].cpu(), offsets) and torch.equal(r["source"].cpu(), source) and torch.equal(r["place"].cpu(), place)
    total = int(offsets[-1])
    want, scale = quantized(x.double()[source[:total].long().cuda()])
    assert torch.equal(r["rows"][0][:total].double(), want) and torch.equal(r["rows"][1][:, :total].double(), scale)
    for e in range(experts):
        at = slice(int(offsets[e]), int(offsets[e + 1]))
        if at.start < at.stop:
            check_codes(r["mid"][0][at], r["mid"][1][:, at], *expected(act, (r["rows"][0][at], r["rows"][1][:, at]), w, up, e))
            check(r["y"][at], *expected("plain", (r["mid"][0][at], r["mid"][1][:, at]), down, e=e))
    there = r["place"] >= 0
    picked = r["y"].double()[r["place"].clamp(min=0).long()] * torch.where(there, share, 0.0).double()[..., None]
    check(r["out"], picked.sum(dim=1), picked.abs().sum(dim=1) * top * 2.0 ** -24)


def test_routed_feed_forward_in_a_graph(calls, store, pkg):
    """Captured once and replayed over other tokens and choices: the same bits as the calls alone; and on a stream of its own beside another."""
    tokens, width, ff, experts, top = 33, 256, 192, 6, 2
    g = generator(77)
    w, up, down = matrix(g, ff, width, experts), matrix(g, ff, width, experts), matrix(g, width, ff, experts)
    sets = []
    for _ in range(3):
        choice = torch.rand((tokens, experts), generator=g, device="cuda").topk(top).indices.int()
        sets.append((torch.randn((tokens, width), generator=g, device="cuda").bfloat16(), choice, torch.rand((tokens, top), generator=g, device="cuda")))
    want = []
    for x, choice, share in sets:
        r = routed_rooms(tokens, width, ff, experts, top)
        routed(calls, x, choice, share, w, up, down, "silu", r)
        want.append(r["out"].clone())
    x, choice, share = (t.clone() for t in sets[0])
    r = routed_rooms(tokens, width, ff, experts, top)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        routed(calls, x, choice, share, w, up, down, "silu", r)
    for (a, b, c), expect in zip(sets, want):
        x.copy_(a), choice.copy_(b), share.copy_(c)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(r["out"], expect)
    streams = [torch.cuda.Stream() for _ in range(2)]
    rooms = [routed_rooms(tokens, width, ff, experts, top) for _ in streams]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                routed(Calls(pkg, store, s.cuda_stream), *sets[i], w, up, down, "silu", rooms[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(rooms[i]["out"], want[i])


def test_the_contexts_own_stream(calls, pkg, store):
    x = torch.randn((4, 256), generator=generator(5), device="cuda").bfloat16()
    out = code_room(4, 256)
    torch.cuda.synchronize()
    own = Calls(pkg, store, 0)
    own.quantize(x, out)
    store.lib.check(store.lib.swlm_op_f8_status(store.handle))
    torch.cuda.synchronize()
    assert torch.equal(out[0].double(), quantized(x.double())[0])


def test_status(calls, store):
    """An expired wait is reported by the next product, which does nothing, until it has been asked for."""
    g = generator(6)
    x, w, y = rows_of(g, 4, 128), matrix(g, 128, 128), room(4, 128, torch.float32, 0x35)
    before = y.clone()
    lib = store.lib
    lib.check(lib.swlm_write_f8_status(store.handle, 3))
    call = calls.product_call(x, w, y)
    assert lib.swlm_op_f8_product_dev(store.handle, call, calls.stream) == -5
    torch.cuda.synchronize()
    assert torch.equal(y.view(torch.int32), before.view(torch.int32))
    assert lib.swlm_op_f8_status(store.handle) == -5 and lib.swlm_op_f8_status(store.handle) == 0
    calls.product(x, w, y)
    check(y, *expected("plain", x, w))


def test_rows_are_values(calls):
    """Quantized rows stand for the values to half a step of a code."""
    x = torch.randn((6, 500), generator=generator(9), device="cuda")
    out = code_room(6, 500)
    wide = room(6, 500, torch.float32)
    wide.copy_(x)
    calls.quantize(wide, out)
    each = out[1].double().t().repeat_interleave(128, dim=1)[:, :500]
    assert ((row_values(out) - x.double()).abs() <= torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * each)).all()
