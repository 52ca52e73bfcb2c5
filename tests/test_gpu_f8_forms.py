"""Every form that a product over 8-bit float weights takes, by sizes that mean it, against 64 bits (tests/plain_f8.py); runs of them at once, again and
in graphs."""
import ctypes as C

import pytest
import torch

from plain_f8 import E4M3, Calls, blocks, check, check_codes, expected, matrix, room, rows_of

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


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def code_room(rows, width):
    return room(rows, width, E4M3, 0x35), torch.full((blocks(width), rows), 7.0, device="cuda")


def form_of(lib, rows, n, k, experts, gated):
    f = (C.c_int * 3)()
    lib.check(lib.swlm_op_f8_product_form(rows, n, k, experts, gated, f))
    return ("few" if f[0] == 0 else "wide" if f[0] == n else "both", f[1], f[2])


# what each size is there for: the form of the other columns than those that pairs of SMs take
FORMS = [
    (False, 1, 5000, 700, "few", 16, 2), (False, 1, 1, 700, "few", 16, 4), (False, 3, 130, 1030, "few", 16, 8), (False, 513, 264, 100, "few", 16, 1),
    (False, 2100, 1, 17, "few", 32, 1), (False, 1500, 1, 700, "few", 32, 2), (False, 513, 1, 700, "few", 32, 4), (False, 300, 1, 1030, "few", 32, 8),
    (False, 777, 5000, 17, "few", 64, 1), (False, 2900, 1, 2049, "few", 64, 2), (False, 1500, 1, 2049, "few", 64, 4), (False, 513, 1, 2600, "few", 64, 8),
    (False, 2100, 4100, 17, "few", 128, 1), (False, 70, 9300, 4100, "few", 128, 2), (False, 1100, 2100, 17, "wide", 0, 0), (False, 1100, 2600, 300, "wide", 0, 0),
    (False, 2900, 2800, 700, "wide", 0, 0), (False, 777, 5000, 2600, "both", 64, 2), (False, 2100, 2100, 2049, "both", 64, 4),
    (True, 2, 2957, 290, "few", 16, 1), (True, 600, 1, 700, "few", 16, 2), (True, 1, 1, 700, "few", 16, 4), (True, 5, 130, 1030, "few", 16, 8), (True, 2900, 129, 17, "few", 64, 1),
    (True, 2900, 1, 700, "few", 64, 2), (True, 1500, 1, 1030, "few", 64, 4), (True, 600, 1, 2049, "few", 64, 8), (True, 2900, 392, 17, "wide", 0, 0),
    (True, 1000, 1500, 260, "wide", 0, 0), (True, 2900, 1500, 700, "wide", 0, 0), (True, 300, 5000, 4100, "both", 64, 4),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, E4M3], ids=str)
@pytest.mark.parametrize("gated,rows,n,k,kind,tile,ctas", FORMS)
def test_forms(calls, gated, rows, n, k, kind, tile, ctas, dtype):
    assert form_of(calls.lib, rows, n, k, 0, gated) == (kind, tile, ctas)
    g = generator(rows + n + k)
    x, w, up = rows_of(g, rows, k), matrix(g, n, k), matrix(g, n, k) if gated else None
    act = ("silu", "gelu", "clamped")[rows % 3] if gated else "plain"
    y = code_room(rows, n) if dtype == E4M3 else room(rows, n, dtype, 0x35)
    held = y[0] if dtype == E4M3 else y
    before = held._base.view(torch.uint8).clone()
    calls.product(x, w, y, up, act)
    want = expected(act, x, w, up)
    if dtype == E4M3:
        check_codes(*y, *want)
    else:
        check(y, *want)
    # what lies behind the rows' columns is as it was
    now, size = held._base.view(torch.uint8), held.element_size()
    assert torch.equal(now[:, n * size:], before[:, n * size:])


def spread(rows, experts, seed):
    """Offsets of experts of very unequal shares, some without rows."""
    share = torch.rand(experts, generator=torch.Generator().manual_seed(seed)) ** 4
    share[:: 3] = 0.0
    share[-1] = 0.1
    ends = (share.cumsum(0) / share.sum() * rows).int()
    ends[-1] = rows
    return torch.cat([torch.zeros(1, dtype=torch.int32), ends]).cuda()


EXPERTS = [(False, 3000, 700, 150, 5, "few"), (True, 3000, 700, 150, 5, "wide"), (False, 6000, 300, 260, 40, "wide"), (True, 200, 1100, 300, 64, "few"), (False, 200, 1100, 300, 64, "few"),
           (False, 1000, 640, 520, 33, "few"), (False, 500, 640, 520, 33, "few"), (True, 400, 640, 520, 33, "few"), (False, 5, 260, 1100, 9, "few"), (True, 1, 130, 2100, 300, "few"), (False, 2000, 130, 130, 1024, "few")]


@pytest.mark.parametrize("dtype", [torch.float16, E4M3], ids=str)
@pytest.mark.parametrize("gated,rows,n,k,experts,kind", EXPERTS)
def test_forms_of_experts(calls, gated, rows, n, k, experts, kind, dtype):
    assert form_of(calls.lib, rows, n, k, experts, gated)[0] == kind
    g = generator(rows + n + k + experts)
    x, w, up = rows_of(g, rows, k), matrix(g, n, k, experts), matrix(g, n, k, experts) if gated else None
    # (scales whose products stay within fp16)
    y = code_room(rows, n) if dtype == E4M3 else room(rows, n, dtype, 0x35)
    w[1].mul_(2.0 ** -4)
    offsets = spread(rows, experts, rows)
    act = "clamped" if gated else "plain"
    calls.product(x, w, y, up, act, offsets)
    ends = offsets.tolist()
    assert max(b - a for a, b in zip(ends, ends[1:])) >= 1.5 * rows / experts   # they are far from equal
    for e in range(experts):
        at = slice(ends[e], ends[e + 1])
        if at.start < at.stop:
            want = expected(act, (x[0][at], x[1][:, at]), w, up, e)
            if dtype == E4M3:
                check_codes(y[0][at], y[1][:, at], *want)
            else:
                check(y[at], *want)


SOME = [(False, 1100, 2600, 300), (True, 1000, 1500, 260), (False, 777, 5000, 2600), (False, 513, 1, 2600), (False, 2100, 4100, 17), (True, 600, 1, 2049), (False, 1, 5000, 700)]


def prepared(calls, seed=0):
    out = []
    for i, (gated, rows, n, k) in enumerate(SOME):
        g = generator(100 * seed + i)
        out.append((rows_of(g, rows, k), matrix(g, n, k), room(rows, n, torch.bfloat16), matrix(g, n, k) if gated else None, "silu" if gated else "plain"))
    return out


def test_the_same_bits_again_and_on_streams_at_once(calls, pkg, store):
    """All forms alone, then on three streams at once several times over."""
    sets = prepared(calls)
    for s in sets:
        calls.product(*s)
    torch.cuda.synchronize()
    want = [s[2].clone() for s in sets]
    streams = [torch.cuda.Stream() for _ in range(3)]
    rooms = [[torch.zeros_like(s[2]._base)[:, :s[2].shape[1]] for s in sets] for _ in streams]
    torch.cuda.synchronize()
    for turn in range(4):
        for i, st in enumerate(streams):
            on = Calls(pkg, store, st.cuda_stream)
            for j in range(len(sets)):
                at = (i + j + turn) % len(sets)
                x, w, _, up, act = sets[at]
                on.product(x, w, rooms[i][at], up, act)
    torch.cuda.synchronize()
    for r in rooms:
        for got, expect in zip(r, want):
            assert torch.equal(got, expect)


def test_graphs_of_all_forms(calls):
    sets, others = prepared(calls), prepared(calls, 1)
    for s in others:
        calls.product(*s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for s in sets:
            calls.product(*s)
    for s, o in zip(sets, others):   # other values in the captured arrays
        for a, b in ((s[0], o[0]), (s[1], o[1]), (s[3], o[3])):
            if a is not None:
                a[0].view(torch.uint8).copy_(b[0].view(torch.uint8)), a[1].copy_(b[1])
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for s, o in zip(sets, others):
        assert torch.equal(s[2], o[2])


def test_nothing_to_do(calls, pkg):
    """No rows, no tokens: nothing is looked at, and a sort's offsets are zero."""
    lib, h = calls.lib, calls.handle
    lib.check(lib.swlm_op_f8_quantize_dev(h, pkg.F8Quantize(rows=0, width=8, x_rows=0), calls.stream))
    lib.check(lib.swlm_op_f8_product_dev(h, pkg.F8Product(rows=0, n=8, k=8), calls.stream))
    lib.check(lib.swlm_op_expert_sum_dev(h, pkg.ExpertSum(tokens=0, top=2, width=8), calls.stream))
    offsets = torch.full((5,), 3, dtype=torch.int32, device="cuda")
    lib.check(lib.swlm_op_expert_sort_dev(h, pkg.ExpertSort(offsets=offsets.data_ptr(), tokens=0, top=2, experts=4), calls.stream))
    # no row of y: every token keeps what is added to it
    place, weight = torch.full((3, 2), -1, dtype=torch.int32, device="cuda"), torch.ones((3, 2), device="cuda")
    add, out = torch.randn((3, 8), device="cuda"), torch.zeros((3, 8), device="cuda")
    call = pkg.ExpertSum(place=place.data_ptr(), weight=weight.data_ptr(), add=add.data_ptr(), add_stride=8, out=out.data_ptr(), out_stride=8, tokens=3, top=2, width=8, y_rows=0,
                         y_dtype=2, dtype=2)
    lib.check(lib.swlm_op_expert_sum_dev(h, call, calls.stream))
    torch.cuda.synchronize()
    assert (offsets == 0).all() and torch.equal(out, add)


def far(compact, stride):
    """The same rows, each `stride` entries behind the one before it."""
    out = torch.zeros((compact.shape[0] * stride,), dtype=torch.uint8 if compact.element_size() == 1 else compact.dtype, device="cuda")
    view = torch.as_strided(out.view(compact.dtype), compact.shape, (stride, 1))
    (view.view(torch.uint8) if compact.element_size() == 1 else view).copy_(compact.view(torch.uint8) if compact.element_size() == 1 else compact)
    return view


def test_rows_that_lie_far_apart(calls):
    """Offsets in bytes that pass 32 bits, in rows, experts' matrices and results: the bits are those of the same rows close together."""
    rows, n, k, experts, stride, w_stride = 3, 130, 200, 3, 5 << 28, 12 << 20
    g = generator(5)
    x = torch.randn((rows, k), generator=g, device="cuda").bfloat16()
    near, apart = code_room(rows, k), code_room(rows, k)
    calls.quantize(x, near)
    wide = far(x, stride)
    calls.quantize(wide, apart)
    torch.cuda.synchronize()
    assert torch.equal(near[0].view(torch.uint8), apart[0].view(torch.uint8)) and torch.equal(near[1], apart[1])
    del wide
    w = matrix(g, n, k, experts)
    w_far = torch.as_strided(torch.zeros((experts * n * w_stride,), dtype=torch.uint8, device="cuda").view(E4M3), (experts, n, k), (n * w_stride, w_stride, 1))
    w_far.view(torch.uint8).copy_(w[0].view(torch.uint8))
    offsets = torch.tensor([0, 1, 1, rows], dtype=torch.int32, device="cuda")
    y, y_far = room(rows, n, torch.bfloat16), far(room(rows, n, torch.bfloat16), stride)
    calls.product(near, w, y, offsets=offsets)
    calls.product((far(near[0], 2 * stride), near[1]), (w_far, w[1]), y_far, offsets=offsets)
    torch.cuda.synchronize()
    assert torch.equal(y, y_far)
    out = room(rows, n, torch.bfloat16)
    calls.sum(y_far, torch.arange(rows, dtype=torch.int32, device="cuda").view(rows, 1), torch.ones((rows, 1), device="cuda"), out)
    torch.cuda.synchronize()
    assert torch.equal(out, y)


@pytest.mark.parametrize("dtype", [torch.float32, E4M3], ids=str)
def test_many_rows_that_lie_far_apart(calls, dtype):
    """The same where pairs of SMs take a product."""
    rows, n, k, stride = 1100, 2600, 300, 5 << 20
    assert form_of(calls.lib, rows, n, k, 0, False)[0] == "wide"
    g = generator(6)
    x, w = rows_of(g, rows, k), matrix(g, n, k)
    y = code_room(rows, n) if dtype == E4M3 else room(rows, n, dtype)
    held = y[0] if dtype == E4M3 else y
    y_far = far(held, stride)
    scale = torch.zeros_like(y[1]) if dtype == E4M3 else None
    calls.product(x, w, y)
    calls.product((far(x[0], stride), x[1]), w, (y_far, scale) if dtype == E4M3 else y_far)
    torch.cuda.synchronize()
    same = torch.equal(held.view(torch.uint8), y_far.view(torch.uint8)) if dtype == E4M3 else torch.equal(held, y_far)
    assert same and (dtype != E4M3 or torch.equal(scale, y[1]))


@pytest.mark.parametrize("gated,rows,n,k,kind", [(False, 1100, 2600, 300, "wide"), (True, 1000, 1500, 260, "wide"), (False, 777, 5000, 2600, "both"), (False, 513, 1, 2600, "few"),
                                                 (True, 5, 130, 1030, "few"), (True, 2900, 129, 17, "few")])
def test_what_is_not_a_number_stays_in_its_place(calls, gated, rows, n, k, kind):
    """A NaN among a row's codes, and one in a row's scale, make that row's codes and scales NaN and leave the others' bits as they are; so do NaN rows of
    other experts that share a tile with them."""
    assert form_of(calls.lib, rows, n, k, 0, gated)[0] == kind
    g = generator(rows + 9)
    x, pair = rows_of(g, rows, k), [matrix(g, n, k, 2), matrix(g, n, k, 2) if gated else None]
    w, up = ((m[0][:1], m[1][:1]) if m is not None else None for m in pair)
    act = "silu" if gated else "plain"
    want, got = code_room(rows, n), code_room(rows, n)
    calls.product(x, w, want, up, act)
    bad = sorted({rows // 3, rows - 1})
    x[0].view(torch.uint8)[bad[0], k - 1] = 0xFF
    x[1][blocks(k) - 1, bad[-1]] = float("nan")
    calls.product(x, w, got, up, act)
    torch.cuda.synchronize()
    fine = torch.ones(rows, dtype=torch.bool, device="cuda")
    fine[bad] = False
    assert torch.equal(got[0].view(torch.uint8)[fine], want[0].view(torch.uint8)[fine]) and torch.equal(got[1][:, fine], want[1][:, fine])
    assert got[0][~fine].float().isnan().all() and got[1][:, ~fine].isnan().all()
    if rows > 2:   # one expert has the rows before the first bad one, another those from it on
        cut = torch.tensor([0, bad[0], rows], dtype=torch.int32, device="cuda")
        y = room(rows, n, torch.float32)
        calls.product(x, pair[0], y, pair[1], act, cut)
        torch.cuda.synchronize()
        assert y[:bad[0]].isfinite().all() and y[bad].isnan().all()
