"""Attention over an 8-bit cache whose keys or values are far from 1."""
import pytest
import torch

from plain_kv8 import Cache
from test_gpu_kv8 import check_attend, store  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("key,query", [(2.0 ** 114, 2.0 ** -113), (2.0 ** -119, 2.0 ** 120)], ids=["large keys", "small keys"])
def test_weights_where_keys_and_queries_are_far_apart(pkg, store, n, key, query):  # noqa: F811
    """Scores are ordinary numbers although a product of the shifted query and a key's code, times the key's scale alone, is not."""
    cache = Cache(pkg, 1, 2, 64, 512, 32, 0).fill([400], key=key)
    check_attend(pkg, store, cache, 1, 8, 64, [400 - n], [n], torch.bfloat16, True, q_gain=query)
