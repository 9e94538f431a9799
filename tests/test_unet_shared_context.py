"""The UNet loop with the package's attention over the text context and PyTorch's over the image tokens."""
import importlib

import pytest
import torch

from fake_ops import FakeOps
from test_unet_shared_prefix import FakeAttention, forward, inputs
from test_unet_shared_prefix_close_gpu import TOLERANCE

pkg = importlib.import_module("sdxl-end2end_b200")


@pytest.mark.parametrize("kv_cache,tolerance", [("f16", 1e-2), ("int8", 1e-2)])
def test_context_alone(kv_cache, tolerance):
    """Only the text context goes through the operator, whose prefix it is; rows serve several images. The INT8 cache is off by half a
    step of a vector's largest value (2^-8), 0.003 of the largest prediction in this network."""
    data = inputs(4, 2)
    want = forward(FakeOps(), data, "cpu", each=True)
    ops = FakeAttention()
    got = forward(ops, data, "cpu", attention="shared_context", kv_cache=kv_cache)
    assert float((got - want).abs().max()) <= tolerance * float(want.abs().max())
    calls = [entry for entry in ops.log if entry[0] == "attention"]
    assert len(calls) > 0 and set(calls) == {("attention", False, True)}
    with pytest.raises(pkg.CudaError, match="batch mismatch"):
        forward(FakeAttention(), (data[0], data[1].repeat(2, 1, 1)[:3], *data[2:]), "cpu", attention="shared_context")


@pytest.mark.gpu
def test_context_alone_on_the_gpu(gpu):
    """Against shared_prefix, which differs in the image tokens' attention alone: both sides round its result to FP16."""
    package, context, ops = gpu
    data = inputs(6, 2)
    for kv_cache in ("f16", "int8"):
        want = forward(ops, data, "cuda", attention="shared_prefix", kv_cache=kv_cache)
        got = forward(ops, data, "cuda", attention="shared_context", kv_cache=kv_cache)
        context.check()
        assert torch.isfinite(got).all()
        assert float((got - want).abs().max()) <= TOLERANCE * float(want.abs().max())
