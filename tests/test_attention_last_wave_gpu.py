"""Attention of more row tiles than the GPU has places for at a time: the tiles of the last wave are a pass of their own, whose keys
are split and whose shares are joined, while the others are written directly."""
import contextlib

import pytest
import torch

import attention_reference as R
from test_attention_gpu import NoFront, cache_of, int32, normal

pytestmark = pytest.mark.gpu

QUERIES = 200                                             # two tiles of 128 rows of a head


def heads_for(dtype, dim, more):
    """Heads of each of two entries so that there are `more` tiles more than places, and the places."""
    per_sm = 2 if dim > 64 else 4 if dtype == "f16" else 3
    places = per_sm * torch.cuda.get_device_properties(0).multi_processor_count
    assert (places + more) % 4 == 0
    return (places + more) // 4, places


@contextlib.contextmanager
def counted_scratch(pkg, context):
    """Operators that go through Python, and the bytes of scratch that their calls ask for."""
    ops, asked = pkg.Ops(context, poison_outputs=True), []
    ops._front = NoFront()
    original = context.scratch

    def scratch(size):
        asked.append(size)
        return original(size)

    context.scratch = scratch
    try:
        yield ops, asked
    finally:
        del context.scratch


@pytest.mark.parametrize("dtype,dim", [("f16", 64), ("f16", 128), ("int8", 64), ("e4m3", 80), ("e5m2", 64)])
@pytest.mark.parametrize("form", ["plain", "causal", "prefix"])
@pytest.mark.parametrize("more", [4, 40])
def test_last_wave(gpu, dtype, dim, form, more):
    pkg, context, ops = gpu
    heads, places = heads_for(dtype, dim, more)
    q = normal(141, 2, QUERIES, heads, dim)
    own, exact_own = cache_of(pkg, normal(142, 2, 1100, heads, dim), normal(143, 2, 1100, heads, dim), dtype)
    prefix, exact_prefix = (None, None) if form != "prefix" else cache_of(pkg, normal(144, 2, 530, heads, dim), normal(145, 2, 530, heads, dim), dtype)
    # rows without a key, a last tile of one key, and all
    lengths = {"plain": None, "causal": [1025, 133], "prefix": [1100, 0]}[form]
    arguments = dict(own_lengths=None if lengths is None else int32(lengths), causal=form == "causal")
    with counted_scratch(pkg, context) as (counting, asked):
        y = counting.shared_prefix_attention(q, own, prefix, **arguments)
    share = more * 128 * (dim + 2) * 4                    # of the last wave's tiles alone
    assert len(asked) == 1 and asked[0] % share == 0 and asked[0] // share >= 2
    assert torch.equal(y, ops.shared_prefix_attention(q, own, prefix, **arguments))
    context.check()
    want, bound = R.attention(q, exact_own, exact_prefix, lengths, None, form == "causal")
    assert R.off(y, want, bound) <= 1.0
    if form == "causal":
        assert (y[1, :QUERIES - 133] == 0).all()


@pytest.mark.parametrize("dtype,dim", [("f16", 64), ("int8", 80)])
def test_few_tiles_are_all_split(gpu, dtype, dim):
    """Less than a wave: one pass, all of it split."""
    pkg, context, ops = gpu
    q = normal(151, 2, QUERIES, 3, dim)
    own, exact = cache_of(pkg, normal(152, 2, 1100, 3, dim), normal(153, 2, 1100, 3, dim), dtype)
    with counted_scratch(pkg, context) as (counting, asked):
        y = counting.shared_prefix_attention(q, own, own_lengths=int32([1100, 65]), causal=True)
    context.check()
    share = 12 * 128 * (dim + 2) * 4
    assert len(asked) == 1 and asked[0] % share == 0 and asked[0] // share >= 2
    want, bound = R.attention(q, exact, None, [1100, 65], None, True)
    assert R.off(y, want, bound) <= 1.0
