"""Attention over an 8-bit cache whose keys or values are far from 1."""
import pytest
import torch

from plain_kv8 import Cache, attend
from test_gpu_kv8 import check_attend, do_attend, ints, store  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("key,query", [(2.0 ** 114, 2.0 ** -113), (2.0 ** -119, 2.0 ** 120)], ids=["large keys", "small keys"])
def test_weights_where_keys_and_queries_are_far_apart(pkg, store, n, key, query):  # noqa: F811
    """Scores are ordinary numbers although a product of the shifted query and a key's code, times the key's scale alone, is not."""
    cache = Cache(pkg, 1, 2, 64, 512, 32, 0).fill([400], key=key)
    check_attend(pkg, store, cache, 1, 8, 64, [400 - n], [n], torch.bfloat16, True, q_gain=query)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("code", [0, 1])
@pytest.mark.parametrize("n", [1, 4, 60])
def test_values_of_any_size_keep_their_precision(pkg, store, n, code, dim):  # noqa: F811
    """All value scales times a power of two: every result times it, bit for bit, but for what is subnormal."""
    cache = Cache(pkg, 1, 2, dim, 1024, 32, code).fill([900])
    q = torch.randn((n, 8, dim), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").bfloat16()
    outs = []
    for power in (0, -100, -112, 100):
        work = cache.clone()
        work.v_scale *= 2.0 ** power
        out = torch.zeros_like(q)
        do_attend(pkg, store, work, q, out, ints(900 - n), dim ** -0.5, n=n)
        outs.append(out.double() * 2.0 ** -power)
        # Results below 2^-126 are multiples of 2^-133: off by 2^-134 at most, and the first cache's by half a step of a number below 2^-126, 2^-135.
        bound = torch.full_like(outs[0], 2.0 ** -133 * 2.0 ** -power)
        # Scales below 2^-120, the smallest that probabilities are taken relative to, make other products of probability and scale, which are rounded
        # otherwise: each result is within its own bound of the same number (a code of e4m3 stands for up to 448, its smallest scales here are 2^-121)
        if (work.v_scale[:, :, :29] < 2.0 ** -120).any():
            bound += 2 * attend(cache, q, 0, 900 - n, dim ** -0.5, 1024)[1]
        assert ((outs[-1] - outs[0]).abs() <= bound).all(), power
