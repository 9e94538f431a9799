"""Attention over 8-bit caches whose value vectors have unlike scales, on the GPU against the definition in 64 bits."""
import pytest
import torch

import attention_reference as R
from test_attention_gpu import cache_of, normal

pytestmark = pytest.mark.gpu

EIGHT_BIT = ("int8", "e4m3", "e5m2")


def leaning(queries, keys, dim, heads=2, at=None):
    """Queries and keys [1, n, heads, dim]: queries lie near one direction, key `at` in it, with about a fifth of a row's weight
    over 4000 keys (exp(0.86 dim / sqrt(dim)) of them for heads of 64)."""
    q = 1.0 + 0.2 * normal(101, 1, queries, heads, dim)
    k = 0.3 * normal(102, 1, keys, heads, dim)
    if at is not None:
        k[:, at] = 0.86 * (64 / dim) ** 0.5
    return q.half(), k.half()


@pytest.mark.parametrize("dtype", EIGHT_BIT)
@pytest.mark.parametrize("queries,dim", [(1, 64), (20, 64), (9, 80), (150, 64), (150, 80)])
@pytest.mark.parametrize("size", [1.0, 0.1, 0.01])
@pytest.mark.parametrize("at,every", [(5, 4000), (5, 40), (2000, 40)])
def test_zero_value_vectors(gpu, dtype, queries, dim, size, at, every):
    """A vector of zeros is written with the scale 1, thousands of times that of its neighbours. It adds nothing to the result, and
    takes nothing from the precision of theirs."""
    pkg, context, ops = gpu
    q, k = leaning(queries, 4000, dim, at=at)
    v = (size * normal(103, 1, 4000, 2, dim)).half()
    v[:, 1::every] = 0.0
    cache, exact = cache_of(pkg, k, v, dtype)
    assert (cache.v_scales[0, :, 1::every] == 1.0).all()
    for parts in ((cache, None), (None, cache)):
        y = ops.shared_prefix_attention(q, *parts)
        context.check()
        want, bound = R.attention(q, exact, None)
        assert R.off(y, want, bound) <= 1.0


@pytest.mark.parametrize("dtype", EIGHT_BIT)
@pytest.mark.parametrize("queries", [1, 150])
def test_zeros_alone(gpu, dtype, queries):
    """Only zero vectors, negative zeros among them, and then others behind whole tiles of them."""
    pkg, context, ops = gpu
    q, k = leaning(queries, 700, 64)
    v = torch.zeros_like(k)
    v[:, 1::2] = -0.0
    cache, _ = cache_of(pkg, k, v, dtype)
    y = ops.shared_prefix_attention(q, cache)
    context.check()
    assert (y == 0).all()
    v[:, 500:] = (0.01 * normal(104, 1, 200, 2, 64)).half()
    cache, exact = cache_of(pkg, k, v, dtype)
    y = ops.shared_prefix_attention(q, cache)
    context.check()
    want, bound = R.attention(q, exact, None)
    assert R.off(y, want, bound) <= 1.0
