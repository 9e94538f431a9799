"""Attention scores so large that their neighbours in 32 bits are 8 apart, on the GPU."""
import math

import pytest
import torch

from test_attention_gpu import normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("queries", [1, 20, 150])
@pytest.mark.parametrize("step", [8, 16, -8])
def test_scores_a_last_bit_apart(gpu, queries, step):
    """Scores of 1.25 * 2^26 + `step` (j // 64) in units of log2, each exact in 32 bits: from one 64 keys to the next a weight changes by
    2^step. A weight is rounded to a half in the products and not in the sum (2^-11 of sum p |v|, or half of a half's least step
    where the row's largest is at least 2^6), the result is rounded to a half (2^-11, or half its least step), and 2^x, sums of
    320 products and the quotient are a few last bits of 32 off."""
    pkg, context, ops = gpu
    keys, dim = 320, 64
    scale = math.log(2.0)                                 # times log2(e) is 1 in 32 bits
    places = torch.arange(keys, device="cuda") // 64
    q = torch.zeros((1, queries, 1, dim), device="cuda").half()
    q[..., 0], q[..., 1] = 4096.0, 1.0
    k = torch.zeros((1, keys, 1, dim), device="cuda").half()
    k[0, :, 0, 0] = 20480.0
    k[0, :, 0, 1] = (step * places).half()
    v = normal(111, 1, keys, 1, dim)
    y = ops.shared_prefix_attention(q, pkg.KVCache(k, v), scale=scale)
    context.check()
    p = torch.exp2((step * places).double())
    p = p / p.sum()
    want, share = p @ v[0, :, 0].double(), p @ v[0, :, 0].double().abs()
    bound = 2 ** -11 * want.abs() + 2 ** -25 + (2 ** -11 + 2 ** -14) * share + keys * 2 ** -31 * v.double().abs().max()
    assert ((y[0, :, 0].double() - want).abs() <= bound).all()
