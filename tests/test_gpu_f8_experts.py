"""Products over 8-bit float weights with experts: every form, with several tiles for a cluster and within the experts' rows; many experts of many
rows, offsets that are none; against 64 bits (tests/plain_f8.py)."""
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


def device_ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def form_of(lib, rows, n, k, experts, gated):
    """Rows of a tile and CTAs that share it."""
    f = (C.c_int * 3)()
    lib.check(lib.swlm_op_f8_product_form(rows, n, k, experts, gated, f))
    return (256, 2) if f[0] == n else (f[1], f[2])


def all_but_the_ends(rows, experts, equal):
    """Offsets from row 3 to the third last: nearly equal shares and every fourth expert without any, or an expert that has all but a row of each other."""
    live = rows - 6
    if equal:
        share = torch.tensor([0.0 if e % 4 == 1 else 1.0 + 0.1 * (e % 3) for e in range(experts)], dtype=torch.float64)
        ends = (share.cumsum(0) / share.sum() * live).round().int().tolist()
    else:
        ends = [e + 1 if e < experts // 2 else e + 1 + live - experts for e in range(experts)]
    return [3] + [3 + end for end in ends]


# rows of a tile and CTAs that share it; those CTAs' clusters are fewer than the tiles where one expert has nearly all rows
FORMS = [
    (False, 95, 521, 108, 62, 16, 1), (False, 428, 132, 3309, 54, 16, 2), (False, 405, 101, 808, 58, 16, 4), (False, 711, 400, 100, 56, 32, 1), (False, 189, 1541, 1167, 11, 32, 2),
    (False, 771, 101, 809, 56, 32, 4), (False, 5781, 101, 385, 66, 64, 1), (False, 1648, 101, 1537, 56, 64, 2), (False, 400, 1024, 4096, 6, 64, 2), (False, 1181, 101, 2090, 24, 64, 4),
    (False, 4150, 131, 551, 47, 128, 1), (False, 3506, 101, 4508, 52, 128, 2), (False, 4585, 391, 110, 22, 256, 2), (True, 3873, 101, 103, 63, 16, 1), (True, 337, 413, 3765, 32, 16, 2),
    (True, 738, 101, 385, 40, 16, 4), (True, 5428, 101, 110, 69, 64, 1), (True, 2297, 101, 642, 55, 64, 2), (True, 400, 1024, 4096, 6, 64, 2), (True, 512, 512, 2048, 16, 64, 2),
    (True, 959, 101, 1335, 30, 64, 4), (True, 6000, 101, 4065, 66, 256, 2),
]
# the same where there are always clusters enough
FEWER = [(False, 9, 101, 981, 3, 16, 8), (False, 142, 101, 956, 15, 32, 8), (False, 335, 101, 2625, 13, 64, 8), (True, 9, 101, 1017, 3, 16, 8), (True, 197, 101, 4691, 11, 64, 8),
         (True, 3363, 129, 130, 47, 256, 2)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, E4M3], ids=str)
@pytest.mark.parametrize("equal", [True, False])
@pytest.mark.parametrize("gated,rows,n,k,experts,tile,ctas", FORMS + FEWER)
def test_forms_with_experts(calls, gated, rows, n, k, experts, tile, ctas, equal, dtype):
    """Every expert's rows are right, the same bits again and again; the rows of none, their scales and what lies behind the columns stay as they are."""
    assert form_of(calls.lib, rows, n, k, experts, gated) == (tile, ctas)
    offsets = all_but_the_ends(rows, experts, equal)
    if not equal and (gated, rows, n, k, experts, tile, ctas) in FORMS:
        columns = n if tile < 256 else (n + 1) // 2 if not gated else n   # (pairs of SMs have twice the columns in a tile, unless it is two matrices')
        assert sum((b - a + tile - 1) // tile for a, b in zip(offsets, offsets[1:])) * blocks(columns) > 148 * (2 if tile <= 32 else 1) // ctas
    g = generator(rows + n + k + experts)
    x, w, up = rows_of(g, rows, k), matrix(g, n, k, experts), matrix(g, n, k, experts) if gated else None
    act = ("silu", "gelu", "clamped")[rows % 3] if gated else "plain"
    scale = torch.full((blocks(n), rows + 5), 7.0, device="cuda")
    held = room(rows, n, dtype, 0x35)
    y = (held, scale[:, :rows]) if dtype == E4M3 else held
    before = held._base.view(torch.uint8).clone()
    at = device_ints(offsets)
    calls.product(x, w, y, up, act, at)
    torch.cuda.synchronize()
    for e in range(experts):
        here = slice(offsets[e], offsets[e + 1])
        if here.start < here.stop:
            want = expected(act, (x[0][here], x[1][:, here]), w, up, e)
            if dtype == E4M3:
                check_codes(held[here], scale[:, here], *want)
            else:
                check(held[here], *want)
    first, end, bytes_of = offsets[0], offsets[-1], n * held.element_size()
    now, was = held._base.view(torch.uint8), scale.clone()
    assert end == rows - 3 and torch.equal(now[:first], before[:first]) and torch.equal(now[end:], before[end:]) and torch.equal(now[:, bytes_of:], before[:, bytes_of:])
    assert (scale[:, :first] == 7.0).all() and (scale[:, end:] == 7.0).all()
    once = now.clone()
    for _ in range(3):
        now[first:end, :bytes_of] = 0x35
        scale[:, first:end] = 7.0
        calls.product(x, w, y, up, act, at)
        torch.cuda.synchronize()
        assert torch.equal(now, once) and torch.equal(scale, was)


@pytest.mark.parametrize("gated", [False, True])
def test_many_experts_of_many_rows(calls, gated):
    """65536 tokens of 8 choices among 1024 experts: some have no row, some thousands."""
    rows, n, k, experts = 65536 * 8, 8192, 16, 1024
    g = generator(31)
    x, w, up = rows_of(g, rows, k), matrix(g, n, k, experts), matrix(g, n, k, experts) if gated else None
    share = torch.rand(experts, generator=torch.Generator().manual_seed(31)) ** 3
    share[::5] = 0.0
    ends = (share.double().cumsum(0) / share.double().sum() * rows).round().int().tolist()
    offsets = [0] + ends[:-1] + [rows]
    y = torch.full((rows, n), 0x35, dtype=torch.uint8, device="cuda").view(E4M3), torch.full((blocks(n), rows), -1.0, device="cuda")
    act = "silu" if gated else "plain"
    calls.product(x, w, y, up, act, device_ints(offsets))
    assert (y[1] > 0).all()   # every row has been there
    for e in [e for e in range(experts) if offsets[e] < offsets[e + 1]][::60] + [experts - 1]:
        at = slice(offsets[e], offsets[e + 1])
        check_codes(y[0][at], y[1][:, at], *expected(act, (x[0][at], x[1][:, at]), w, up, e))


def test_offsets_that_do_not_ascend(calls):
    """Experts that claim the same rows: a row's results are some such expert's, and nothing but those rows is written."""
    rows, n, k, claims = 204, 130, 130, 20
    g = generator(32)
    x, w, y = rows_of(g, rows, k), matrix(g, n, k, 2 * claims), room(rows, n, torch.float32, 0x35)
    before = y._base.clone()
    calls.product(x, w, y, offsets=device_ints([0, 200] * claims + [0]))   # every second expert has rows 0 .. 199, the others none
    torch.cuda.synchronize()
    found = torch.zeros((200, n), dtype=torch.bool, device="cuda")
    for e in range(0, 2 * claims, 2):
        want, off = expected("plain", (x[0][:200], x[1][:, :200]), w, e=e)
        found |= (y[:200].double() - want).abs() <= off + 2.0 ** -24 * (want.abs() + off)
    assert found.all()
    assert torch.equal(y._base[200:], before[200:]) and torch.equal(y._base[:, n:], before[:, n:])
