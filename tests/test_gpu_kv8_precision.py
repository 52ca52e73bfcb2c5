"""How exact attention over an 8-bit cache is where results are fp16: what rounding probabilities to fp16 costs must not show in them."""
import pytest
import torch

from plain_kv8 import HALF, TOP, Cache, attend, numbers
from test_gpu_kv8 import attend_call, do_attend, ints, same_bits, store, stream  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("code", [0, 1])
@pytest.mark.parametrize("heads,dim,n,before", [
    (4, 64, 1, 11), (4, 128, 1, 30), (16, 64, 1, 9), (8, 128, 3, 5),     # one row tile and two
    (4, 64, 40, 1), (4, 128, 70, 0),                                      # portions
    (4, 128, 1, 300), (4, 64, 40, 700),                                    # parts joined by a cluster and by a launch of their own
], ids=str)
def test_fp16_results_are_rounded_once(pkg, store, heads, dim, n, before, code, block):  # noqa: F811
    """Values whose products with the probabilities nearly cancel: a probability that is off by 2^-12 of itself would show in most results."""
    total = before + n
    cache = Cache(pkg, 1, 1, dim, 1024, block, code).fill([total], key=0.2)
    q = torch.randn((n, heads, dim), generator=torch.Generator(device="cuda").manual_seed(6), device="cuda").half()
    out = torch.zeros_like(q)
    scale = dim ** -0.5
    do_attend(pkg, store, cache, q, out, ints(before), scale, n=n)
    qd, k, v = q.double(), cache.values("k", 0, total)[0], cache.values("v", 0, total)[0]
    each = cache.v_scale[0, 0].double().repeat_interleave(block)[:total]
    assert (numbers(cache.v[0, 0, :total], code).abs() <= TOP[code]).all()
    hidden = torch.arange(total, device="cuda")[None, :] > before + torch.arange(n, device="cuda")[:, None]
    p = torch.softmax((torch.einsum("nhd,td->hnt", qd, k) * scale).masked_fill(hidden, -torch.inf), dim=-1)
    want, size = (torch.einsum("hnt,td->nhd", p, x) for x in (v, v.abs()))
    # A score's error: sums of 16 products in fp32, 2^-22 of the magnitudes met so far, dim / 16 times, and four such steps around the exponential; twice
    # in a probability, its own and its sum's; the sum itself 2^-24 for each of its additions (a row's slots go to four warps or more, or one thread)
    reach = (torch.einsum("nhd,td->hnt", qd.abs(), k.abs()) * scale).amax(dim=-1).T[:, :, None]
    prob = 2 * (dim / 16 + 4) * 2.0 ** -22 * (reach + 1) + (total + 32) * 2.0 ** -24
    # Probabilities times 2^7 and the value's scale over the largest, as the sum of two fp16 numbers: 2^-22 of themselves, or 2^-25 where the second one is
    # subnormal; products with the codes are added to fp32 sums, 16 at a time
    tol = (prob + 2.0 ** -22 + (total / 16 + 32) * 2.0 ** -22) * size + total * 2.0 ** -25 * each.max() * TOP[code] / 128
    tol = tol + (want.abs() + tol) * HALF[torch.float16] + 2.0 ** -25
    assert ((out.double() - want).abs() <= tol).all(), ((out.double() - want).abs() / tol).max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("n,length", [(1, 900), (5, 300), (40, 700)])
def test_a_caller_chooses_how_probabilities_meet_values(pkg, store, n, length, dtype):  # noqa: F811
    """By type is two for fp16 and one for bf16, bit for bit; either is within the bounds of one number, and the other differs from it in fp16."""
    cache = Cache(pkg, 1, 2, 128, 1024, 32, 0).fill([length])
    q = torch.randn((n, 8, 128), generator=torch.Generator(device="cuda").manual_seed(9), device="cuda").to(dtype)
    outs, lengths = [], ints(length - n)
    want, tol, _, _ = attend(cache, q, 0, length - n, 0.09, 1024)
    for how in (pkg.KV8_P_BY_TYPE, pkg.KV8_P_ONE, pkg.KV8_P_TWO):
        out = torch.zeros_like(q)
        step, scratch = attend_call(pkg, store, cache, q, out, lengths, 0.09, n=n)
        step.probabilities = how
        store.lib.check(store.lib.swlm_op_kv8_attend_dev(store.handle, cache.described(), step, stream()))
        torch.cuda.synchronize()
        assert ((out.double() - want).abs() <= tol).all(), how
        outs.append(out)
    assert same_bits(outs[0], outs[2 if dtype == torch.float16 else 1])
    if dtype == torch.float16:
        assert not same_bits(outs[1], outs[2])
        assert (outs[2].double() - want).norm() < (outs[1].double() - want).norm()
