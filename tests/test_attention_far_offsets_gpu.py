"""The kv cache and attention where a slot, a token or a head lies more than 2^32 bytes from the first."""
import pytest
import torch

import attention_reference as R
from test_attention_gpu import normal, scalar_type

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "int8", "e5m2"])
@pytest.mark.parametrize("axis", ["slot", "token", "head"])
def test_far_apart(gpu, dtype, axis):
    pkg, context, ops = gpu
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    width = 2 if dtype == "f16" else 1
    slots, tokens, heads, dim = 2, 70, 2, 64
    strides = [tokens * heads * dim, heads * dim, dim]
    far = {"slot": 0, "token": 1, "head": 2}[axis]
    strides[far] = ((1 << 32) + (1 << 20)) // width // ((slots, tokens, heads)[far] - 1) // 16 * 16
    if axis == "token":
        strides[0] = heads * dim                          # slots lie within a token's room
    if axis == "head":
        strides[0], strides[1] = tokens * dim, dim
    reach = dim + sum(s * (n - 1) for s, n in zip(strides, (slots, tokens, heads)))
    assert (reach - dim) * width > 1 << 32
    element = {"f16": torch.float16, "int8": torch.int8, "e5m2": torch.float8_e5m2}[dtype]
    k, v = (torch.empty(reach, dtype=element, device="cuda").as_strided((slots, tokens, heads, dim), (*strides, 1)) for _ in "kv")
    scales = (None, None) if dtype == "f16" else tuple(torch.ones((slots, heads, tokens), device="cuda") for _ in "kv")
    cache = pkg.KVCache(k, v, scalar_type(pkg, dtype), *scales)
    key, value = normal(161, slots, tokens, heads, dim), normal(162, slots, tokens, heads, dim)
    ops.kv_cache_write(cache, key, value)
    back = ops.kv_cache_read(cache, tokens)
    exact = [R.values_of(*R.quantise(x, dtype)) for x in (key, value)]
    for got, want in zip(back, exact):
        assert torch.equal(got, want.half())
    for queries in (1, 20, 150):
        q = normal(163, slots, queries, 4, dim)
        want, bound = R.attention(q, exact, None)
        for parts in ((cache, None), (None, cache)):
            y = ops.shared_prefix_attention(q, *parts)
            context.check()
            assert R.off(y, want, bound) <= 1.0
