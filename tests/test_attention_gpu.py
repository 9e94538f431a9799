"""The kv cache and shared-prefix attention on the GPU against the definitions in 64 bits."""
import math

import pytest
import torch

import attention_reference as R

pytestmark = pytest.mark.gpu


def scalar_type(pkg, dtype):
    return {"f16": pkg.ScalarType.Float16, "int8": pkg.ScalarType.Int8, "e4m3": pkg.ScalarType.Float8E4M3,
            "e5m2": pkg.ScalarType.Float8E5M2}[dtype]


def normal(seed, *shape, spread=0.3):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    x = torch.randn(shape, generator=generator, device="cuda")
    return (x * torch.exp(spread * torch.randn(shape[:-1] + (1,), generator=generator, device="cuda"))).half()


def cache_of(pkg, k, v, dtype):
    """(KVCache, (k, v) as 64-bit values) holding FP16 tokens [slots, tokens, heads, dim]."""
    (kq, ks), (vq, vs) = R.quantise(k, dtype), R.quantise(v, dtype)
    turned = [None if s is None else s.transpose(1, 2).contiguous() for s in (ks, vs)]
    return pkg.KVCache(kq, vq, scalar_type(pkg, dtype), *turned), (R.values_of(kq, ks), R.values_of(vq, vs))


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---- the cache ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("rows,tokens,heads,dim", [(1, 1, 1, 16), (2, 77, 10, 64), (3, 33, 5, 80), (2, 130, 3, 128), (5, 1, 20, 64), (1, 9, 7, 48)])
def test_write_and_read(gpu, dtype, rows, tokens, heads, dim):
    pkg, context, ops = gpu
    k, v = normal(1, rows, tokens, heads, dim, spread=2.0), normal(2, rows, tokens, heads, dim)
    k[0, 0, 0] = 0.0                                      # a vector of zeros has the scale 1
    cache = ops.kv_cache(rows, tokens + 3, heads, dim, scalar_type(pkg, dtype))
    ops.kv_cache_write(cache, k, v, positions=2)
    got = ops.kv_cache_read(cache, tokens, positions=2)
    context.check()
    for x, elements, scales, back in ((k, cache.k, cache.k_scales, got[0]), (v, cache.v, cache.v_scales, got[1])):
        q, s = R.quantise(x, dtype)
        assert torch.equal(elements[:, 2:2 + tokens].float(), q.float())
        if s is not None:
            assert torch.equal(scales[:, :, 2:2 + tokens], s.transpose(1, 2))
            assert torch.equal(scales[:, :, :2], torch.ones_like(scales[:, :, :2]))
        assert torch.equal(elements[:, :2].float(), torch.zeros_like(elements[:, :2].float()))
        assert torch.equal(elements[:, 2 + tokens:].float(), torch.zeros_like(elements[:, 2 + tokens:].float()))
        assert torch.equal(back, R.values_of(q, s).clamp(-65504, 65504).half())


@pytest.mark.parametrize("dtype", R.TYPES)
def test_every_half(gpu, dtype):
    """All finite halves, sixteen to a vector in the order of their bits and in an order that mixes their sizes."""
    pkg, context, ops = gpu
    bits = torch.arange(65536, dtype=torch.int32, device="cuda").to(torch.int16).view(torch.float16)
    x = bits[torch.isfinite(bits)]
    generator = torch.Generator(device="cuda")
    generator.manual_seed(3)
    k = x.view(1, -1, 1, 16)
    v = x[torch.randperm(x.numel(), generator=generator, device="cuda")].view(1, -1, 1, 16)
    cache = ops.kv_cache(1, k.shape[1], 1, 16, scalar_type(pkg, dtype))
    ops.kv_cache_write(cache, k, v)
    back = ops.kv_cache_read(cache, k.shape[1])
    context.check()
    for source, elements, scales, read in ((k, cache.k, cache.k_scales, back[0]), (v, cache.v, cache.v_scales, back[1])):
        q, s = R.quantise(source, dtype)
        assert torch.equal(elements.float(), q.float())
        assert s is None or torch.equal(scales, s.transpose(1, 2))
        assert torch.equal(read, R.values_of(q, s).clamp(-65504, 65504).half())


def test_ties_go_to_even(gpu):
    """INT8: a maximum of 127 makes the scale 1, and halves of odd multiples are ties."""
    pkg, context, ops = gpu
    x = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5, 3.5, 62.5, 63.5, -126.5, 0.25, 0.75, 1e-7, -1e-7], device="cuda").half()
    cache = ops.kv_cache(1, 1, 1, 16, pkg.ScalarType.Int8)
    ops.kv_cache_write(cache, x.view(1, 1, 1, 16), x.view(1, 1, 1, 16))
    context.check()
    assert cache.k.flatten().tolist() == [127, 0, 2, 2, 0, -2, -2, 126, 4, 62, 64, -126, 0, 1, 0, 0]


@pytest.mark.parametrize("dtype", R.TYPES)
def test_infinities_and_nan(gpu, dtype):
    """The scale is of the finite values; infinities saturate; a NaN is 0 in INT8 and stays NaN elsewhere."""
    pkg, context, ops = gpu
    x = normal(4, 1, 3, 1, 16)
    x[0, 0, 0, 3], x[0, 0, 0, 5], x[0, 1, 0, 2], x[0, 2, 0, :] = math.inf, -math.inf, math.nan, math.inf
    cache = ops.kv_cache(1, 3, 1, 16, scalar_type(pkg, dtype))
    ops.kv_cache_write(cache, x, x)
    back = ops.kv_cache_read(cache, 3)[0]
    context.check()
    if dtype == "f16":
        assert torch.equal(back.view(torch.int16), x.view(torch.int16))
        return
    clean = x.clone()
    finite_max = torch.where(torch.isfinite(x), x.abs(), 0).amax(-1)
    largest = {"int8": 127.0, "e4m3": 448.0, "e5m2": 57344.0}[dtype]
    scale = cache.k_scales.transpose(1, 2).double()
    assert torch.equal(scale, R.quantise(torch.where(torch.isfinite(clean), clean, 0), dtype)[1].double())
    assert float(finite_max[0, 2, 0]) == 0.0 and float(scale[0, 2, 0]) == 1.0
    want = R.values_of(*R.quantise(torch.where(torch.isfinite(clean), clean, 0), dtype))
    want[x == math.inf] = (largest * scale[..., None]).expand(x.shape)[x == math.inf]
    want[x == -math.inf] = -(largest * scale[..., None]).expand(x.shape)[x == -math.inf]
    nan = torch.isnan(x)
    assert torch.equal(back[~nan], want.half()[~nan])
    assert (back[nan] == 0).all() if dtype == "int8" else torch.isnan(back[nan]).all()


@pytest.mark.parametrize("dtype", ["f16", "int8"])
def test_positions_and_counts(gpu, dtype):
    """Rows at places of their own, some of which lie outside the slot: those tokens are not written and read as zeros."""
    pkg, context, ops = gpu
    rows, tokens, heads, dim, capacity = 5, 4, 3, 32, 10
    k, v = normal(5, rows, tokens, heads, dim), normal(6, rows, tokens, heads, dim)
    positions, counts = [0, 8, -2, 3, 2 ** 31 - 1], [4, 4, 4, 2, 4]
    cache = ops.kv_cache(rows + 2, capacity, heads, dim, scalar_type(pkg, dtype))
    before = cache.k.float().clone()
    ops.kv_cache_write(cache, k, v, positions=int32(positions), counts=int32(counts), first_slot=1)
    back = ops.kv_cache_read(cache, tokens, positions=int32(positions), counts=int32(counts), rows=rows, first_slot=1)
    context.check()
    q, s = R.quantise(k, dtype)
    want_cache, want_back = before, torch.zeros_like(k)
    for r in range(rows):
        for t in range(min(tokens, counts[r])):
            if 0 <= positions[r] + t < capacity:
                want_cache[1 + r, positions[r] + t] = q[r, t].float()
                want_back[r, t] = R.values_of(q, s)[r, t].half()
    assert torch.equal(cache.k.float(), want_cache)
    assert torch.equal(back[0], want_back)


@pytest.mark.parametrize("dtype", R.TYPES)
def test_strided_tokens_and_cache(gpu, dtype):
    """Tokens inside a wider tensor, heads first or tokens first, into a cache of either order."""
    pkg, context, ops = gpu
    rows, tokens, heads, dim = 2, 21, 4, 32
    wide = normal(7, rows, heads, tokens, 2 * dim + 16)
    k, v = wide[..., :dim].transpose(1, 2), wide[..., dim:2 * dim].transpose(1, 2)
    q = R.quantise(k, dtype)[0]
    storage = [torch.zeros((rows, tokens, heads, dim), dtype=q.dtype, device="cuda") for _ in "kv"]
    scales = [None, None] if dtype == "f16" else [torch.ones((rows, heads, tokens), device="cuda") for _ in "kv"]
    cache = pkg.KVCache(*storage, scalar_type(pkg, dtype), *scales)
    ops.kv_cache_write(cache, k, v)
    back = ops.kv_cache_read(cache, tokens)
    context.check()
    for x, elements, read in ((k, storage[0], back[0]), (v, storage[1], back[1])):
        q, s = R.quantise(x, dtype)
        assert torch.equal(elements.float(), q.float())
        assert torch.equal(read, R.values_of(q, s).half())


# ---- attention ---------------------------------------------------------------------------------------------
def check(gpu, batch, queries, q_heads, kv_heads, dim, dtype, prefixes=0, prefix=0, own=0, own_dtype=None, own_lengths=None,
          prefix_lengths=None, causal=False, scale=None, seed=11, factor=1.0):
    pkg, context, ops = gpu
    q = normal(seed, batch, queries, q_heads, dim) * factor
    parts, exact = [None, None], [None, None]
    for i, (slots, tokens, kind) in enumerate(((batch, own, own_dtype or dtype), (prefixes, prefix, dtype))):
        if slots and tokens:
            parts[i], exact[i] = cache_of(pkg, normal(seed + 1 + i, slots, tokens, kv_heads, dim), normal(seed + 3 + i, slots, tokens, kv_heads, dim), kind)
    y = ops.shared_prefix_attention(q, parts[0], parts[1], own_lengths=None if own_lengths is None else int32(own_lengths),
                                    prefix_lengths=None if prefix_lengths is None else int32(prefix_lengths), causal=causal, scale=scale)
    context.check()
    want, bound = R.attention(q, exact[0], exact[1], own_lengths, prefix_lengths, causal, scale)
    assert R.off(y, want, bound) <= 1.0


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("queries,heads,kv_heads,dim", [(1, 1, 1, 16), (1, 5, 5, 64), (3, 8, 2, 128), (17, 4, 4, 80), (40, 6, 2, 48), (130, 2, 2, 64)])
@pytest.mark.parametrize("keys", [1, 15, 77, 300])
def test_own_keys_only(gpu, dtype, queries, heads, kv_heads, dim, keys):
    check(gpu, 2, queries, heads, kv_heads, dim, dtype, own=keys)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("batch,prefixes,queries,heads,kv_heads,dim", [
    (4, 1, 1, 4, 4, 64), (6, 2, 1, 8, 2, 128), (6, 3, 5, 4, 2, 80), (4, 2, 64, 2, 2, 64), (2, 2, 1, 4, 1, 64), (40, 1, 1, 4, 2, 64), (4, 2, 150, 2, 1, 128)])
@pytest.mark.parametrize("prefix,own", [(77, 0), (200, 33), (1000, 1)])
def test_prefix_and_own_keys(gpu, dtype, batch, prefixes, queries, heads, kv_heads, dim, prefix, own):
    check(gpu, batch, queries, heads, kv_heads, dim, dtype, prefixes, prefix, own)


@pytest.mark.parametrize("queries,repeat", [(1, 1), (1, 8), (4, 1), (150, 2)])
def test_long_keys_are_split(gpu, queries, repeat):
    check(gpu, 3, queries, 2 * repeat, 2, 64, "f16", 1, 9001, 700, own_lengths=[700, 4, 399])


@pytest.mark.parametrize("dtype", ["f16", "int8"])
@pytest.mark.parametrize("queries,dim", [(1, 64), (2, 64), (37, 64), (37, 128), (200, 64), (200, 128)])
def test_lengths_that_leave_rows_empty(gpu, dtype, queries, dim):
    """Lengths of zero, one, more than the capacity and below zero; entries whose both parts are empty give zeros."""
    check(gpu, 6, queries, 4, 2, dim, dtype, 3, 50, 70, prefix_lengths=[0, 1, 99], own_lengths=[0, 70, 1, 0, 200, -5])
    check(gpu, 6, queries, 4, 2, dim, dtype, own=70, own_lengths=[0, 70, 1, 33, 200, -5])


@pytest.mark.parametrize("dtype", ["f16", "e4m3"])
@pytest.mark.parametrize("queries,own,lengths", [(5, 5, None), (5, 40, [40, 3, 5, 0]), (33, 33, [33, 12, 1, 32]), (150, 300, [300, 100, 150, 17]), (129, 129, None)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 64), (6, 2, 80)])
@pytest.mark.parametrize("prefixes", [0, 2])
def test_causal(gpu, dtype, queries, own, lengths, heads, kv_heads, dim, prefixes):
    check(gpu, 4, queries, heads, kv_heads, dim, dtype, prefixes, 60 if prefixes else 0, own, own_lengths=lengths, causal=True)


@pytest.mark.parametrize("prefix_type,own_type", [("int8", "f16"), ("f16", "e5m2"), ("e4m3", "int8")])
@pytest.mark.parametrize("queries", [1, 70])
def test_parts_of_unlike_types(gpu, prefix_type, own_type, queries):
    check(gpu, 4, queries, 4, 2, 64, prefix_type, 2, 90, 40, own_dtype=own_type, own_lengths=[40, 1, 0, 39])
    check(gpu, 2, queries, 4, 2, 64, prefix_type, 2, 90, 40, own_dtype=own_type)


@pytest.mark.parametrize("queries", [1, 150])
@pytest.mark.parametrize("dtype", ["f16", "int8"])
def test_large_scores(gpu, queries, dtype):
    """Scores of some hundreds, of both signs, and a scale of its own: one key takes nearly all the weight."""
    check(gpu, 2, queries, 4, 4, 64, dtype, 1, 500, 100, factor=20.0)
    check(gpu, 2, queries, 4, 4, 64, dtype, 1, 500, 100, scale=0.0)
    check(gpu, 2, queries, 4, 4, 64, dtype, 1, 500, 100, scale=-0.7)


@pytest.mark.parametrize("queries", [1, 150])
def test_rising_scores_and_value_scales(gpu, queries):
    """Scores that grow from key to key, so that the running maximum moves all the time, and values whose scales span 2^20."""
    pkg, context, ops = gpu
    keys, dim = 700, 64
    q = torch.ones((1, queries, 1, dim), device="cuda").half()
    k = torch.linspace(-3.0, 3.0, keys, device="cuda")[None, :, None, None].expand(1, keys, 1, dim).half().contiguous()
    v = normal(21, 1, keys, 1, dim) * torch.exp2(torch.randint(-14, 6, (1, keys, 1, 1), device="cuda").float()).half()
    for source in (k, k.flip(1)):
        for dtype in R.TYPES:
            cache, exact = cache_of(pkg, source.contiguous(), v, dtype)
            y = ops.shared_prefix_attention(q, cache)
            context.check()
            want, bound = R.attention(q, exact, None)
            assert R.off(y, want, bound) <= 1.0


@pytest.mark.parametrize("queries,keys", [(1, 700), (150, 700), (150, 6000), (1, 6000), (40, 6000)])
def test_huge_scores(gpu, queries, keys):
    """Scores of 10^8, whose neighbours differ by thousands: the largest takes all the weight, wherever it stands. The weight,
    2^x with x up to the reference's last bit, is rounded to a half for the product and not in the sum (2^-11), the result is
    rounded to a half (2^-11, or half its least step), and 2^x and the quotient are a few last bits of 32 off."""
    pkg, context, ops = gpu
    dim = 64
    q = torch.full((1, queries, 1, dim), 4096.0, device="cuda").half()
    v = normal(22, 1, keys, 1, dim)
    generator = torch.Generator(device="cuda")
    generator.manual_seed(23)
    for sign in (1.0, -1.0):
        k = (2048.0 + 2.0 * (torch.randperm(keys, generator=generator, device="cuda") % 1000)) * sign
        at = int(k.argmax())
        k[at] = (k[at] + 4.0)                             # one key stands out, by 10^5
        k = k[None, :, None, None].expand(1, keys, 1, dim).half().contiguous()
        y = ops.shared_prefix_attention(q, pkg.KVCache(k, v))
        context.check()
        want = v[:, at:at + 1].expand(1, queries, 1, dim).double()
        assert ((y.double() - want).abs() <= (2 ** -10 + 2 ** -20) * want.abs() + 2 ** -25).all()


@pytest.mark.parametrize("queries", [1, 3, 20, 150])
@pytest.mark.parametrize("dim", [64, 80])
def test_hidden_places_hold_anything(gpu, queries, dim):
    """NaN and infinities behind lengths and behind the causal mask take no part; those that a row sees do."""
    pkg, context, ops = gpu
    batch, keys = 3, queries + 40
    q, k, v = normal(31, batch, queries, 4, dim), normal(32, batch, keys, 2, dim), normal(33, batch, keys, 2, dim)
    lengths = [keys, keys - 17, queries]
    for b, n in enumerate(lengths):
        k[b, n:], v[b, n:] = math.nan, math.inf
    pk, pv = normal(34, 1, 100, 2, dim), normal(35, 1, 100, 2, dim)
    pk[:, 90:], pv[:, 90:] = math.inf, math.nan
    exact = lambda *x: tuple(t.double() for t in x)
    prefix, own = pkg.KVCache(pk, pv), pkg.KVCache(k, v)
    for causal in (False, True):
        y = ops.shared_prefix_attention(q, own, prefix, own_lengths=int32(lengths), prefix_lengths=int32([90]), causal=causal)
        context.check()
        want, bound = R.attention(q, exact(k, v), exact(pk, pv), lengths, [90], causal)
        assert torch.isfinite(want).all()
        assert R.off(y, want, bound) <= 1.0
    if queries > 2:
        # tokens that only the last queries see
        at = queries // 2
        v[0, lengths[0] - queries + at, 0, 3] = math.inf
        v[1, lengths[1] - queries + at, 1, 5] = math.nan
        k[2, lengths[2] - queries + at, 0, 1] = math.nan
        y = ops.shared_prefix_attention(q, own, prefix, own_lengths=int32(lengths), prefix_lengths=int32([90]), causal=True)
        context.check()
        kh, vh = k.clone(), v.clone()
        want, bound = R.attention(q, exact(torch.where(torch.isnan(kh), 0, kh), vh), exact(pk, pv), lengths, [90], True)
        want[2, at:, :2] = math.nan                       # a NaN score makes the whole row NaN
        assert torch.isfinite(want[:, :at]).all()
        assert R.off(y[:, :at], want[:, :at], bound[:, :at]) <= 1.0
        assert not torch.isfinite(y[0, at:, 0:2, 3].float()).any() and not torch.isfinite(y[1, at:, 2:4, 5].float()).any()
        assert torch.isnan(y[2, at:, :2]).all()
        whole = torch.isfinite(want)
        assert torch.isfinite(y.float()[whole]).all()


@pytest.mark.parametrize("queries", [1, 33, 150])
def test_layouts(gpu, queries):
    """Heads first or tokens first, queries inside a wider tensor, an output of another order, the output in the queries' place."""
    pkg, context, ops = gpu
    batch, heads, kv_heads, dim, keys = 4, 6, 3, 64, 90
    wide = normal(41, batch, heads, queries, dim + 24)
    q = wide[..., 8:8 + dim].transpose(1, 2)
    k, v = normal(42, batch, kv_heads, keys, dim).transpose(1, 2), normal(43, batch, kv_heads, keys, dim).transpose(1, 2)
    pk, pv = normal(44, 2, 130, kv_heads * dim), normal(45, 2, 130, kv_heads * dim)
    prefix = pkg.KVCache.of(pk, pv, kv_heads)
    want, bound = R.attention(q, (k.double(), v.double()), (prefix.k.double(), prefix.v.double()))
    out = torch.full((batch, queries, heads, 2 * dim), math.nan, device="cuda").half()
    y = ops.shared_prefix_attention(q, pkg.KVCache(k, v), prefix, out=out[..., dim:])
    context.check()
    assert R.off(y, want, bound) <= 1.0 and torch.isnan(out[..., :dim]).all()
    y = ops.shared_prefix_attention(q, pkg.KVCache(k, v), prefix, out=q)
    context.check()
    assert y is q and R.off(q, want, bound) <= 1.0
    assert torch.equal(wide[..., :8], normal(41, batch, heads, queries, dim + 24)[..., :8])
    # one prefix seen through a stride of zero is the same as a prefix of its own for each entry
    expanded = pkg.KVCache(prefix.k[:1].expand(4, -1, -1, -1), prefix.v[:1].expand(4, -1, -1, -1))
    for n in (7, 90):
        a = ops.shared_prefix_attention(k[:, :n].contiguous(), expanded)
        b = ops.shared_prefix_attention(k[:, :n].contiguous(), None, pkg.KVCache(prefix.k[:1], prefix.v[:1]))
        context.check()
        want, bound = R.attention(k[:, :n], None, (prefix.k[:1].double(), prefix.v[:1].double()))
        assert R.off(a, want, bound) <= 1.0 and R.off(b, want, bound) <= 1.0


def test_empty_calls(gpu):
    pkg, context, ops = gpu
    cache = ops.kv_cache(2, 5, 2, 64)
    assert ops.shared_prefix_attention(torch.empty((2, 0, 4, 64), device="cuda").half(), cache).shape == (2, 0, 4, 64)
    assert ops.shared_prefix_attention(torch.empty((0, 3, 4, 64), device="cuda").half(), None, cache).shape == (0, 3, 4, 64)
    nothing = ops.kv_cache(2, 0, 2, 64)
    y = ops.shared_prefix_attention(normal(1, 2, 3, 4, 64), nothing)
    context.check()
    assert (y == 0).all()
    ops.kv_cache_write(cache, torch.empty((2, 0, 2, 64), device="cuda").half(), torch.empty((2, 0, 2, 64), device="cuda").half())
    assert ops.kv_cache_read(cache, 0)[0].shape == (2, 0, 2, 64)
    context.check()


def test_offsets_past_32_bits(gpu):
    """A cache whose last tokens lie more than 2^32 elements from its first."""
    pkg, context, ops = gpu
    free = torch.cuda.mem_get_info()[0]
    if free < 24 << 30:
        pytest.skip("needs 24 GB")
    heads, dim, capacity = 8, 128, (2 ** 32) // (8 * 128) + 600
    storage = [torch.empty((1, heads, capacity, dim), dtype=torch.int8, device="cuda") for _ in "kv"]
    scales = [torch.ones((1, heads, capacity), device="cuda") for _ in "kv"]
    cache = pkg.KVCache(storage[0].transpose(1, 2), storage[1].transpose(1, 2), pkg.ScalarType.Int8, *scales)
    k, v = normal(51, 1, 500, heads, dim), normal(52, 1, 500, heads, dim)
    start = capacity - 500
    ops.kv_cache_write(cache, k, v, positions=start)
    back = ops.kv_cache_read(cache, 500, positions=start)
    (kq, ks), (vq, vs) = R.quantise(k, "int8"), R.quantise(v, "int8")
    tail = pkg.KVCache(cache.k[:, start:], cache.v[:, start:], pkg.ScalarType.Int8, scales[0][:, :, start:].contiguous(), scales[1][:, :, start:].contiguous())
    q = normal(53, 1, 2, heads, dim)
    y = ops.shared_prefix_attention(q, tail)
    context.check()
    assert torch.equal(back[0], R.values_of(kq, ks).half()) and torch.equal(back[1], R.values_of(vq, vs).half())
    want, bound = R.attention(q, (R.values_of(kq, ks), R.values_of(vq, vs)), None)
    assert R.off(y, want, bound) <= 1.0


class NoFront:
    """Answers None to everything: the Python path runs."""

    def __getattr__(self, name):
        return lambda *arguments: None


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("queries", [1, 50])
def test_front_and_python_path_agree(gpu, dtype, queries):
    pkg, context, ops = gpu
    slow = pkg.Ops(context, poison_outputs=True)
    slow._front = NoFront()
    k, v, q = normal(95, 3, 40, 2, 64), normal(96, 3, 40, 2, 64), normal(97, 6, queries, 4, 64)
    own, _ = cache_of(pkg, normal(98, 6, 30, 2, 64), normal(99, 6, 30, 2, 64), dtype)
    results = []
    for o in (ops, slow):
        cache = o.kv_cache(4, 64, 2, 64, scalar_type(pkg, dtype))
        assert o.kv_cache_write(cache, k, v, positions=int32([0, 5, 40]), counts=int32([40, 3, 40]), first_slot=1) is None
        prefix = pkg.KVCache(cache.k[1:], cache.v[1:], cache.type, *(None if s is None else s[1:] for s in (cache.k_scales, cache.v_scales)))
        out = [cache.k.float(), cache.v.float(), *o.kv_cache_read(cache, 20, positions=3), *o.kv_cache_read(cache, 9, int32([1, 60]), int32([9, 2]), 2, 1)]
        given = torch.empty_like(q)
        out += [o.shared_prefix_attention(q, own, prefix, own_lengths=int32([30, 0, 1, 7, 30, 2]), prefix_lengths=int32([64, 8, 0]), causal=True),
                o.shared_prefix_attention(q, None, prefix, scale=0.3), o.shared_prefix_attention(q, own, scale=1, out=given)]
        assert out[-1] is given
        results.append(out)
    context.check()
    for fast, plain in zip(*results):
        assert fast.shape == plain.shape and fast.dtype == plain.dtype and torch.equal(fast, plain)
    with pytest.raises(pkg.CudaError, match="slot per batch entry"):       # found by the library behind the front
        ops.shared_prefix_attention(q[:4], own)
    with pytest.raises(pkg.CudaError, match="behind the capacity"):
        ops.kv_cache_read(own, 31)
    with pytest.raises(pkg.CudaError, match="more rows than slots"):
        ops.kv_cache_write(own, normal(1, 7, 3, 2, 64), normal(2, 7, 3, 2, 64))


# ---- a run of them, streams and graphs ---------------------------------------------------------------------
@pytest.mark.parametrize("dtype", R.TYPES)
def test_prompt_then_tokens(gpu, dtype):
    """A prompt written once, then for each step one token of every sequence appended and attended to, eagerly and in a graph whose
    positions move on the device: the same bits, and those of the definition."""
    pkg, context, ops = gpu
    batch, heads, kv_heads, dim, prompt, steps = 6, 8, 4, 64, 100, 5
    pk, pv = normal(61, 2, prompt, kv_heads, dim), normal(62, 2, prompt, kv_heads, dim)
    k, v, q = normal(63, batch, steps, kv_heads, dim), normal(64, batch, steps, kv_heads, dim), normal(65, batch, steps, heads, dim)
    prefix = ops.kv_cache(2, prompt, kv_heads, dim, scalar_type(pkg, dtype))
    ops.kv_cache_write(prefix, pk, pv)
    exact = R.values_of(*R.quantise(pk, dtype)), R.values_of(*R.quantise(pv, dtype))
    exact_own = R.values_of(*R.quantise(k, dtype)), R.values_of(*R.quantise(v, dtype))

    def fresh():
        return ops.kv_cache(batch, 64, kv_heads, dim, scalar_type(pkg, dtype)), int32([0] * batch), int32([1] * batch)

    own, positions, lengths = fresh()
    eager = []
    for step in range(steps):
        ops.kv_cache_write(own, k[:, step:step + 1], v[:, step:step + 1], positions=positions)
        eager.append(ops.shared_prefix_attention(q[:, step:step + 1], own, prefix, own_lengths=lengths, causal=True))
        positions += 1
        lengths += 1
    context.check()
    for step in range(steps):
        n = [step + 1] * batch
        want, bound = R.attention(q[:, step:step + 1], tuple(x[:, :step + 1] for x in exact_own), exact, n, None, True)
        assert R.off(eager[step], want, bound) <= 1.0

    own, positions, lengths = fresh()
    k_in, v_in, q_in = k[:, :1].contiguous(), v[:, :1].contiguous(), q[:, :1].contiguous()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        context.set_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.kv_cache_write(own, k_in, v_in, positions=positions)
            y = ops.shared_prefix_attention(q_in, own, prefix, own_lengths=lengths, causal=True)
            positions += 1
            lengths += 1
        for step in range(steps):
            k_in.copy_(k[:, step:step + 1]), v_in.copy_(v[:, step:step + 1]), q_in.copy_(q[:, step:step + 1])
            graph.replay()
            assert torch.equal(y, eager[step])
        stream.synchronize()
    context.set_stream(torch.cuda.current_stream())


def test_two_graphs_on_two_streams(gpu):
    """Split calls of one context captured on two streams and replayed at the same time share no scratch."""
    pkg, context, ops = gpu
    cache, _ = cache_of(pkg, normal(71, 1, 8000, 4, 64), normal(72, 1, 8000, 4, 64), "f16")
    queries = [normal(73 + i, 8, 1, 8, 64) for i in range(2)]
    want = [ops.shared_prefix_attention(q, None, cache) for q in queries]
    context.check()
    streams, graphs, out = [torch.cuda.Stream() for _ in "ab"], [], []
    torch.cuda.synchronize()
    for stream, q in zip(streams, queries):
        graph = torch.cuda.CUDAGraph()
        context.set_stream(stream)
        with torch.cuda.graph(graph, stream=stream):
            out.append(ops.shared_prefix_attention(q, None, cache))
        graphs.append(graph)
    context.set_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    for _ in range(20):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_results_do_not_change_from_call_to_call(gpu):
    pkg, context, ops = gpu
    prefix, _ = cache_of(pkg, normal(81, 1, 5000, 4, 64), normal(82, 1, 5000, 4, 64), "int8")
    own, _ = cache_of(pkg, normal(83, 6, 50, 4, 64), normal(84, 6, 50, 4, 64), "int8")
    q = normal(85, 6, 2, 8, 64)
    first = ops.shared_prefix_attention(q, own, prefix)
    for _ in range(5):
        assert torch.equal(first, ops.shared_prefix_attention(q, own, prefix))
    context.check()


def test_scratch_of_another_stream(gpu):
    """The context's stream is not the current one: the call's scratch is not handed out while its kernels run."""
    pkg, context, ops = gpu
    cache, exact = cache_of(pkg, normal(91, 1, 20000, 4, 64), normal(92, 1, 20000, 4, 64), "f16")
    q = normal(93, 8, 1, 8, 64)
    want = ops.shared_prefix_attention(q, None, cache)
    context.check()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    context.set_stream(stream)
    outs = []
    for _ in range(10):
        outs.append(ops.shared_prefix_attention(q, None, cache))
        torch.empty(1 << 20, dtype=torch.float32, device="cuda").fill_(math.nan)       # whoever gets memory next writes over it
    stream.synchronize()
    context.set_stream(torch.cuda.current_stream())
    assert all(torch.equal(y, want) for y in outs)
