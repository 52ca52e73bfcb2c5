"""Products over 8-bit float weights with experts: many experts of many rows, offsets that are none, against 64 bits (tests/plain_f8.py)."""
import pytest
import torch

from plain_f8 import E4M3, Calls, blocks, check_codes, expected, matrix, room, rows_of

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
