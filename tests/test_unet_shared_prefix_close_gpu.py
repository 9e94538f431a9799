"""The UNet loop's attention over a shared text context against the definition over the very same cache, so that what the cache's
type rounds is no part of the difference, and a context that is wrong is seen."""
import importlib

import pytest
import torch

import attention_reference as R
from test_unet_shared_prefix import MINIATURE, inputs

harness = importlib.import_module("sdxl-end2end_b200.unet_harness")

pytestmark = pytest.mark.gpu

# Both sides round attention's result to FP16 and are the same otherwise. On the CPU, two such predictions of this network (the
# library's attention and the definition's) are 0.0022 of the largest value apart; a context of zeros changes it by 0.30,
# prompts that are swapped by 0.41. Three times the first is the limit, ten times the limit what a wrong context has to show.
TOLERANCE = 6.6e-3


class Defined(harness.UNetHarness):
    """Attention by its definition in 64 bits, over the caches that the operators have written."""

    @staticmethod
    def _by_definition(query, heads, own, prefix):
        parts = [None if c is None else tuple(R.values_of(x, None if s is None else s.transpose(1, 2)) for x, s in ((c.k, c.k_scales), (c.v, c.v_scales)))
                 for c in (own, prefix)]
        return R.attention(query.unflatten(2, (heads, -1)), *parts)[0].half().flatten(2)

    def _self_attention(self, query, key, value, heads):
        return self._by_definition(query, heads, harness.KVCache.of(key, value, heads), None)

    def _cross_attention(self, query, block, heads):
        return self._by_definition(query, heads, None, self._kv_caches[block])


def forward(kind, ops, data, kv_cache):
    latents, context, pooled, time_ids = (x.cuda() for x in data)
    unet = kind(ops, MINIATURE, precision="f16", seed=3, attention="shared_prefix", kv_cache=kv_cache)
    unet.prepare_conditioning(context)
    out = unet.forward(latents, 801.0, pooled, time_ids)
    unet.close()
    return out


@pytest.mark.parametrize("kv_cache", ["f16", "int8", "e4m3", "e5m2"])
def test_close_to_the_definition(gpu, kv_cache):
    package, context, ops = gpu
    latents, text, pooled, time_ids = inputs(6, 2)
    want = forward(Defined, ops, (latents, text, pooled, time_ids), kv_cache)
    got = forward(harness.UNetHarness, ops, (latents, text, pooled, time_ids), kv_cache)
    context.check()
    assert torch.isfinite(got).all()
    largest = float(want.abs().max())
    assert float((got - want).abs().max()) <= TOLERANCE * largest
    for wrong in (text.flip(0), torch.zeros_like(text)):
        other = forward(harness.UNetHarness, ops, (latents, wrong, pooled, time_ids), kv_cache)
        assert float((other - want).abs().max()) >= 10 * TOLERANCE * largest


@pytest.mark.parametrize("kv_cache", ["int8", "e4m3", "e5m2"])
def test_a_context_padded_with_zeros(gpu, kv_cache):
    """Tokens of zeros at the end of a prompt: their values are vectors of zeros (to_v has no bias)."""
    package, context, ops = gpu
    latents, text, pooled, time_ids = inputs(6, 2)
    text = 0.02 * text
    text[0, 20:], text[1, 50:] = 0.0, 0.0
    want = forward(Defined, ops, (latents, text, pooled, time_ids), kv_cache)
    got = forward(harness.UNetHarness, ops, (latents, text, pooled, time_ids), kv_cache)
    context.check()
    assert float((got - want).abs().max()) <= TOLERANCE * float(want.abs().max())
