"""Attention gives the same bits from call to call where tiles end inside a part and hold values that are not finite."""
import math

import pytest
import torch

import attention_reference as R
from test_attention_gpu import cache_of, int32, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "e5m2"])
@pytest.mark.parametrize("queries,dim", [(20, 64), (150, 64), (150, 80)])
@pytest.mark.parametrize("inside", [False, True])
def test_the_same_bits_behind_lengths(gpu, dtype, queries, dim, inside):
    """Causal, lengths that are no multiple of the MMA's 16 keys, and NaN behind them; `inside`: one in front of them too."""
    pkg, context, ops = gpu
    batch, keys = 3, queries + 45
    q, k, v = normal(131, batch, queries, 4, dim), normal(132, batch, keys, 2, dim), normal(133, batch, keys, 2, dim)
    lengths = [keys - 3, keys - 17, queries + 1]
    for b, n in enumerate(lengths):
        v[b, n:] = math.nan
    if inside:
        v[:, queries - 2, 1, 5] = math.nan
    cache, exact = cache_of(pkg, k, v, dtype)
    call = lambda: ops.shared_prefix_attention(q, cache, own_lengths=int32(lengths), causal=True)
    first = call()
    for _ in range(50):
        assert torch.equal(first.view(torch.int16), call().view(torch.int16))
    context.check()
    want, bound = R.attention(q, exact, None, lengths, None, True)
    assert torch.isfinite(want).all() != inside
    assert R.off(first, want, bound) <= 1.0
    assert torch.isfinite(first[torch.isfinite(want)]).all()
