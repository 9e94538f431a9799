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


def rescaled(pkg, cache, exact, factors):
    """The same cache with the value scales of tokens (slot, token) multiplied; what it stands for in 64 bits."""
    scales, values = cache.v_scales.clone(), exact[1].clone()
    for (slot, token), factor in factors.items():
        scales[slot, :, token] *= factor
        values[slot, token] *= factor
    return pkg.KVCache(cache.k, cache.v, cache.type, cache.k_scales, scales), (exact[0], values)


@pytest.mark.parametrize("dtype", EIGHT_BIT)
@pytest.mark.parametrize("queries,dim", [(5, 64), (33, 64), (12, 80), (150, 64), (150, 128)])
@pytest.mark.parametrize("factor", [2.0 ** 30, -2.0 ** 30, 2.0 ** 120])
def test_hidden_value_scales(gpu, dtype, queries, dim, factor):
    """Tokens that the causal mask hides from the earlier queries take no part in theirs, however large their value scale is."""
    pkg, context, ops = gpu
    batch, keys = 2, queries + 40
    q = normal(121, batch, queries, 4, dim)
    cache, exact = cache_of(pkg, normal(122, batch, keys, 2, dim), normal(123, batch, keys, 2, dim), dtype)
    late = 3                                              # the last tokens, which the last queries see
    odd, _ = rescaled(pkg, cache, exact, {(b, keys - 1 - i): factor for b in range(batch) for i in range(late)})
    y = ops.shared_prefix_attention(q, odd, causal=True)[:, :-late]
    same = ops.shared_prefix_attention(q, cache, causal=True)[:, :-late]
    context.check()
    want, bound = R.attention(q, exact, None, causal=True)
    assert R.off(y, want[:, :-late], bound[:, :-late]) <= 1.0
    assert R.off(same, want[:, :-late], bound[:, :-late]) <= 1.0


@pytest.mark.parametrize("dtype", EIGHT_BIT)
@pytest.mark.parametrize("queries", [1, 20, 150])
@pytest.mark.parametrize("first", [True, False])
def test_a_large_scale_of_no_weight(gpu, dtype, queries, first):
    """A key whose weight is nothing (e^-45) and whose value scale is 2^20 times the others': its own share of the result is below
    2^-26, and it takes nothing from the precision of theirs. The bound is that of the cache without it."""
    pkg, context, ops = gpu
    dim, keys, at = 64, 300, 0 if first else 299
    q, k = leaning(queries, keys, dim, at=7)
    k[:, at] = -5.0                                       # 64 * -5 / 8 and more
    v = (0.01 * normal(124, 1, keys, 2, dim)).half()
    cache, exact = cache_of(pkg, k, v, dtype)
    odd, _ = rescaled(pkg, cache, exact, {(0, at): 2.0 ** 20})
    rest = slice(1, None) if first else slice(0, -1)
    want, bound = R.attention(q, tuple(x[:, rest] for x in exact), None)
    # the key's own share: its weight is below e^(-30 - 3), its values below 0.05 * 2^20
    scores = torch.einsum("bqhd,bkhd->bhqk", q.double(), exact[0]) / 8.0
    share = torch.softmax(scores, -1)[..., at].amax() * 0.1 * 2.0 ** 20
    assert share <= 2.0 ** -26
    for parts in ((odd, None), (None, odd)):
        y = ops.shared_prefix_attention(q, *parts)
        context.check()
        assert R.off(y, want, bound + share) <= 1.0


@pytest.mark.parametrize("dtype", EIGHT_BIT)
@pytest.mark.parametrize("queries", [1, 20, 150])
@pytest.mark.parametrize("height", [0.86, 3.0, 20.0])
def test_a_zero_vector_takes_the_weight(gpu, dtype, queries, height):
    """A key with a fifth of the weight, nearly all of it or all but 2^-200 holds a vector of zeros."""
    pkg, context, ops = gpu
    q, k = leaning(queries, 4000, 64, at=70)
    k[:, 70] = height
    v = (0.1 * normal(125, 1, 4000, 2, 64)).half()
    v[:, 70] = 0.0
    cache, exact = cache_of(pkg, k, v, dtype)
    y = ops.shared_prefix_attention(q, cache)
    context.check()
    want, bound = R.attention(q, exact, None)
    assert R.off(y, want, bound) <= 1.0


@pytest.mark.parametrize("dtype", EIGHT_BIT)
@pytest.mark.parametrize("queries,keys", [(1, 700), (150, 700), (150, 6000), (20, 6000)])
def test_huge_scores_and_small_values(gpu, dtype, queries, keys):
    """Scores of 10^8, thousands apart, over values whose scales are far from 1: the largest takes all the weight, wherever it
    stands. The weight is rounded to a half for the product and not in the sum (2^-11), the result is rounded to a half (2^-11, or half
    its least step), and 2^x and the quotient are a few last bits of 32 off."""
    pkg, context, ops = gpu
    dim = 64
    q = torch.full((1, queries, 1, dim), 4096.0, device="cuda").half()
    generator = torch.Generator(device="cuda")
    generator.manual_seed(126)
    for sign in (1.0, -1.0):
        for size in (0.01, 100.0):
            k = (2048.0 + 2.0 * (torch.randperm(keys, generator=generator, device="cuda") % 1000)) * sign
            at = int(k.argmax())
            k[at] = (k[at] + 4.0)                         # one key stands out, by 10^5
            k = k[None, :, None, None].expand(1, keys, 1, dim).half().contiguous()
            cache, exact = cache_of(pkg, k, (size * normal(127, 1, keys, 1, dim)).half(), dtype)
            if int(exact[0][0, :, 0, 0].argmax()) != at:
                continue                                  # the cache's type does not tell it from the next
            top = exact[0][0, :, 0, 0].topk(2)[0]
            if float(top[0] - top[1]) * 4096.0 * 8.0 < 1e4:
                continue
            y = ops.shared_prefix_attention(q, cache)
            context.check()
            want = exact[1][:, at:at + 1].expand(1, queries, 1, dim)
            assert ((y.double() - want).abs() <= (2 ** -10 + 2 ** -20) * want.abs() + 2 ** -25).all()


@pytest.mark.parametrize("dtype", EIGHT_BIT)
@pytest.mark.parametrize("queries", [1, 20, 150])
@pytest.mark.parametrize("scale", [2.0 ** 90, 2.0 ** 110, 2.0 ** 127])
def test_the_largest_scales(gpu, dtype, queries, scale):
    """A value scale near the top of 32 bits on a key that has weight: its values of 1 and more are infinite in FP16, its zeros are not there."""
    pkg, context, ops = gpu
    q, k = leaning(queries, 200, 64, at=3)
    v = normal(128, 1, 200, 2, 64)
    v[:, 3, :, :32] = 2.0
    v[:, 3, :, 32:] = 0.0
    cache, exact = cache_of(pkg, k, v, dtype)
    scales = cache.v_scales.clone()
    scales[:, :, 3] = scale
    odd = pkg.KVCache(cache.k, cache.v, cache.type, cache.k_scales, scales)
    y = ops.shared_prefix_attention(q, odd)
    context.check()
    assert torch.isinf(y[..., :32]).all() and (y[..., :32] > 0).all()
    assert torch.isfinite(y[..., 32:]).all()
