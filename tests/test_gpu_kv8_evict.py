"""Eviction from an 8-bit cache by clusters of one, two, four and eight CTAs: which, goes by the slots that a sequence may have."""
import math

import pytest
import torch

from plain_kv8 import Cache
from test_gpu_kv8 import check_evicted, evict, ints, same_bits, store  # noqa: F401

pytestmark = pytest.mark.gpu


def weigh(cache, lengths, kind):
    """Weights of all tokens: `special` ones have every kind of tie and order; slots filled out of order."""
    g = torch.Generator(device="cuda").manual_seed(11)
    for b, n in enumerate(lengths):
        w = cache.weight[b, :, :max(n, 0)]
        if kind == "equal":
            w.fill_(0.5)
        elif kind == "steps":
            w.copy_(torch.randint(0, 3, w.shape, generator=g, device="cuda").float())
        elif kind == "special":
            values = torch.tensor([math.nan, math.inf, -math.inf, 1e-40, -1.0, 0.0, -0.0, 3e38], device="cuda")
            w.copy_(values[torch.randint(0, 8, w.shape, generator=g, device="cuda")])
        cache.slot_pos[b, :, :max(n, 0)] = torch.stack([torch.randperm(max(n, 0), generator=g, device="cuda") for _ in range(w.shape[0])]).int()
    return cache


@pytest.mark.parametrize("kind", ["ordinary", "equal", "steps", "special"])
@pytest.mark.parametrize("span", [4096, 4097, 8192, 8193, 12000, 16384, 16385])
def test_evict_of_ragged_sequences_by_clusters(pkg, store, span, kind):  # noqa: F811
    """A sequence that fills the span beside one that has a few tokens more than may stay (most CTAs of its cluster without a slot), one that has fewer (its
    cluster leaves at once) and one that has none. Into another cache and in place, with the same result."""
    keep, sink, recent, block = 1500, 4, 40, 128
    lengths = [span, keep + 7, 900, 0]
    cap = -(-span // block) * block
    cache = weigh(Cache(pkg, 4, 3, 64, cap, block, span % 2).fill(lengths), lengths, kind)
    to = Cache(pkg, 4, 3, 64, -(-keep // block) * block, block, span % 2, seed=5)
    before, to_before = cache.clone(), to.clone()
    args = (keep, sink, recent, ints(*lengths), ints(*lengths))
    evict(pkg, store, cache, to, *args, max_len=span)
    assert all(same_bits(x, y) for x, y in zip(cache.arrays(), before.arrays()))
    check_evicted(before, to_before, to, lengths, keep, sink, recent, lengths)
    evict(pkg, store, cache, cache, *args, max_len=span)
    check_evicted(before, before, cache, lengths, keep, sink, recent, lengths)


@pytest.mark.parametrize("span,keep", [(12000, 9000), (16384, 16000), (8193, 8192), (16385, 8200)])
def test_evict_of_ties_that_lie_in_several_ctas(pkg, store, span, keep):  # noqa: F811
    """Equal weights of which the lowest slots stay, and those that stay end within a later CTA's slots."""
    block = 128
    cap = -(-span // block) * block
    cache = weigh(Cache(pkg, 1, 2, 64, cap, block, 0).fill([span]), [span], "steps")
    before = cache.clone()
    evict(pkg, store, cache, cache, keep, 3, 100, ints(span), ints(span))
    check_evicted(before, before, cache, [span], keep, 3, 100, [span])
