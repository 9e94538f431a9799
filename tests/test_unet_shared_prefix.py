"""The UNet loop with the package's attention: images that share a prompt, and the context's keys and values in 8 bits."""
import importlib

import numpy as np
import pytest
import torch

import attention_reference as R
from fake_ops import FakeOps

harness = importlib.import_module("sdxl-end2end_b200.unet_harness")
pkg = importlib.import_module("sdxl-end2end_b200")

MINIATURE = harness.UNetConfig(channels=(64, 128, 256), heads=(1, 2, 4), transformer_depth=(1, 1, 2),
                               cross_attention_dim=96, time_embed_dim=128, addition_time_embed_dim=8,
                               addition_input_dim=80, layers_per_block=2, norm_groups=32)
NAMES = {pkg.ScalarType.Int8: "int8", pkg.ScalarType.Float8E4M3: "e4m3", pkg.ScalarType.Float8E5M2: "e5m2", pkg.ScalarType.Float16: "f16"}


class FakeAttention(FakeOps):
    """The stand-in with the cache and attention by their definitions."""

    def kv_cache(self, slots, capacity, heads, dim, type):
        element = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2, "f16": torch.float16}[NAMES[type]]
        scales = [None, None] if NAMES[type] == "f16" else [torch.ones((slots, heads, capacity)) for _ in "kv"]
        return pkg.KVCache(*(torch.zeros((slots, capacity, heads, dim)).to(element) for _ in "kv"), type, *scales)

    def kv_cache_write(self, cache, key, value):
        for x, elements, scales in ((key, cache.k, cache.k_scales), (value, cache.v, cache.v_scales)):
            q, s = R.quantise(x, NAMES[cache.type])
            elements.copy_(q)
            scales.copy_(s.transpose(1, 2))

    def shared_prefix_attention(self, query, own=None, prefix=None):
        self.log.append(("attention", own is not None, prefix is not None))
        parts = [None if part is None else tuple(R.values_of(x, None if s is None else s.transpose(1, 2)) for x, s in
                                                 ((part.k, part.k_scales), (part.v, part.v_scales))) for part in (own, prefix)]
        return R.attention(query, *parts)[0].half()


def inputs(batch, prompts, size=16, seed=5):
    rng = np.random.default_rng(seed)
    half = lambda *shape: torch.from_numpy(rng.standard_normal(shape, dtype=np.float32)).half()
    latents, context, pooled = half(batch, 4, size, size), half(prompts, 77, MINIATURE.cross_attention_dim), half(batch, MINIATURE.pooled_dim)
    return latents, context, pooled, torch.tensor([[128, 128, 0, 0, 128, 128]] * batch).half()


def forward(ops, data, device, each=False, **options):
    latents, context, pooled, time_ids = (x.to(device) for x in data)
    unet = harness.UNetHarness(ops, MINIATURE, precision="f16", device=torch.device(device) if device == "cpu" else None, seed=3,
                               parameters=None, **options)
    if each:
        context = context.repeat_interleave(latents.shape[0] // context.shape[0], 0)
    for _ in range(2):                                    # the second time into the caches that are there
        unet.prepare_conditioning(context)
    out = unet.forward(latents, 801.0, pooled, time_ids)
    unet.close()
    return out


def test_wiring_and_refusals():
    """Through the stand-in: the same prediction as with the library's attention on a context repeated for every image."""
    ops = FakeAttention()
    data = inputs(4, 2)
    want = forward(FakeOps(), data, "cpu", each=True)
    got = forward(ops, data, "cpu", attention="shared_prefix")
    assert float((got - want).abs().max()) <= 1e-2 * float(want.abs().max())
    calls = [entry for entry in ops.log if entry[0] == "attention"]
    assert calls.count(("attention", True, False)) == calls.count(("attention", False, True)) == len(calls) // 2 > 0
    eight = forward(FakeAttention(), data, "cpu", attention="shared_prefix", kv_cache="int8")
    assert 0 < float((eight - want).abs().max()) <= 5e-2 * float(want.abs().max())
    with pytest.raises(pkg.CudaError, match="batch mismatch"):
        forward(FakeOps(), data, "cpu")
    with pytest.raises(pkg.CudaError, match="batch mismatch"):
        forward(FakeAttention(), (data[0], data[1].repeat(2, 1, 1)[:3], *data[2:]), "cpu", attention="shared_prefix")
    for options in ({"attention": "other"}, {"kv_cache": "int8"}, {"attention": "shared_prefix", "kv_cache": "int4"}):
        with pytest.raises(pkg.CudaError, match="unknown attention"):
            harness.UNetHarness(FakeOps(), MINIATURE, precision="f16", device=torch.device("cpu"), **options)


@pytest.mark.gpu
@pytest.mark.parametrize("kv_cache,tolerance", [("f16", 2e-2), ("int8", 5e-2), ("e4m3", 2e-1), ("e5m2", 3e-1)])
def test_shared_prompts(gpu, kv_cache, tolerance):
    """Two prompts for six images against the library's attention on the context repeated for every image. FP16 differs by the
    roundings of the weights; the 8-bit caches add those of keys and values (half a step: 2^-8 of a vector's largest value,
    2^-4 or 2^-3 of each value), which the attention over 77 tokens averages out in part."""
    package, context, ops = gpu
    data = inputs(6, 2)
    want = forward(ops, data, "cuda", each=True)
    got = forward(ops, data, "cuda", attention="shared_prefix", kv_cache=kv_cache)
    context.check()
    assert torch.isfinite(got).all()
    assert float((got - want).abs().max()) <= tolerance * float(want.abs().max())


@pytest.mark.gpu
def test_denoising_loop(gpu):
    """Three captured steps give the bits of eager ones, with the prompt's keys and values in INT8."""
    package, context, ops = gpu
    results = []
    for use_graph in (False, True):
        unet = harness.UNetHarness(ops, MINIATURE, precision="e4m3", seed=3, attention="shared_prefix", kv_cache="int8")
        loop = harness.EulerDenoiser(unet, 4, height=128, width=128, steps=3, use_graph=use_graph)
        latents, embeds, pooled, time_ids = (x.cuda() for x in inputs(8, 2, seed=9))
        loop.set_conditioning(embeds, pooled, time_ids)
        loop.set_latents(latents[:4])
        results.append(loop.run().clone())
        context.check()
        unet.close()
    assert torch.isfinite(results[0]).all() and torch.equal(results[0], results[1])
