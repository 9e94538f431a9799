"""The UNet loop's shared-prefix attention where two levels have the same width and unlike heads."""
import dataclasses
import importlib

import pytest
import torch

from fake_ops import FakeOps
from test_unet_shared_prefix import MINIATURE, FakeAttention, inputs

harness = importlib.import_module("sdxl-end2end_b200.unet_harness")


@pytest.mark.parametrize("heads", [(1, 2, 4), (1, 4, 2)])
@pytest.mark.parametrize("kv_cache", ["f16", "int8"])
def test_levels_of_equal_width(heads, kv_cache):
    """The same prediction as with the library's attention, up to the cache's roundings."""
    config = dataclasses.replace(MINIATURE, channels=(64, 128, 128), heads=heads)
    latents, context, pooled, time_ids = inputs(2, 2)
    out = []
    for ops, options in ((FakeOps(), {}), (FakeAttention(), {"attention": "shared_prefix", "kv_cache": kv_cache})):
        unet = harness.UNetHarness(ops, config, precision="f16", device=torch.device("cpu"), seed=3, **options)
        unet.prepare_conditioning(context)
        out.append(unet.forward(latents, 801.0, pooled, time_ids))
    assert float((out[0] - out[1]).abs().max()) <= (1e-2 if kv_cache == "f16" else 2e-2) * float(out[0].abs().max())
    for block, cache in unet._kv_caches.items():
        level = {"mid_block": 2}.get(block.split(".")[0])
        if level is None:
            level = int(block.split(".")[1]) if block.startswith("down") else 2 - int(block.split(".")[1])
        assert cache.heads == heads[level]
