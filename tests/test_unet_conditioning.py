"""A denoising loop whose text context changes between generations."""
import importlib

import pytest
import torch

from fake_ops import FakeOps
from test_unet_shared_prefix import MINIATURE, FakeAttention, inputs

harness = importlib.import_module("sdxl-end2end_b200.unet_harness")
pkg = importlib.import_module("sdxl-end2end_b200")


def context_of(rows, tokens, seed):
    generator = torch.Generator().manual_seed(seed)
    return torch.randn((rows, tokens, MINIATURE.cross_attention_dim), generator=generator).half()


class Recorded:
    """Stands in for a captured graph: a replay reads the memory of its capture."""

    def __init__(self, unet):
        self.read = [t.data_ptr() for t in (unet._kv_source, *unet._kv.values())]
        self.kept = [unet._kv_source, *unet._kv.values()]
        self.replays = 0

    def replay(self):
        self.replays += 1


def recording_loop(ops, images, **options):
    unet = harness.UNetHarness(ops, MINIATURE, precision="f16", device=torch.device("cpu"), seed=3, **options)
    loop = harness.EulerDenoiser(unet, images, height=128, width=128, steps=3, use_graph=True)
    captures = []

    def capture():
        loop._step_body()                                 # what a capture warms up with
        loop._graph = Recorded(unet)
        captures.append(loop._graph)

    loop._capture = capture
    return unet, loop, captures


@pytest.mark.parametrize("shared", [True, False])
def test_a_graph_is_captured_again_when_its_memory_goes(shared):
    ops = FakeAttention() if shared else FakeOps()
    unet, loop, captures = recording_loop(ops, 4, **({"attention": "shared_prefix", "kv_cache": "int8"} if shared else {}))
    latents, _, pooled, time_ids = inputs(8, 8)
    shapes = [(4, 77), (4, 77), (8, 77), (4, 77), (4, 154)] if shared else [(8, 77), (8, 77), (8, 154)]
    wanted = []
    for i, (rows, tokens) in enumerate(shapes):
        loop.set_conditioning(context_of(rows, tokens, i), pooled, time_ids)
        loop.set_latents(latents[:4])
        for _ in range(2):
            loop.step()
            assert captures[-1].read == [t.data_ptr() for t in (unet._kv_source, *unet._kv.values())]
        wanted.append(len(captures))
    assert wanted == ([1, 1, 2, 3, 4] if shared else [1, 1, 2])
    assert sum(graph.replays for graph in captures) == 2 * len(shapes)


def test_a_loop_of_another_batch_on_the_same_unet():
    """The time embedding's plan is of one batch: another loop's batch replaces it."""
    unet, loop, captures = recording_loop(FakeAttention(), 2, attention="shared_prefix")
    latents, _, pooled, time_ids = inputs(4, 4)
    loop.set_conditioning(context_of(2, 77, 1), pooled, time_ids)
    loop.set_latents(latents[:2])
    loop.step()
    unet.forward(latents[:2], 801.0, pooled[:2], time_ids[:2])
    loop.step()
    assert len(captures) == 2
    loop.step()
    assert len(captures) == 2


@pytest.mark.parametrize("images,shared,rows", [(4, True, 1), (3, True, 3), (4, True, 6), (6, True, 8), (6, True, 3), (4, True, 0), (4, True, 16),
                                                (4, False, 4), (4, False, 2), (4, False, 9)])
def test_rows_that_serve_no_prompt_pair(images, shared, rows):
    """An odd number of rows has one for both the unconditional and the conditional half; others do not divide the batch. What was
    set before stays."""
    unet, loop, captures = recording_loop(FakeAttention(), images, **({"attention": "shared_prefix"} if shared else {}))
    _, _, pooled, time_ids = inputs(2 * images, 1)
    loop.set_conditioning(context_of(2 * images, 77, 1), pooled, time_ids)
    source, kept = unet._kv_source, unet._kv_source.clone()
    with pytest.raises(pkg.CudaError, match="batch mismatch"):
        loop.set_conditioning(context_of(rows, 77, 2), pooled, time_ids)
    assert unet._kv_source is source and torch.equal(source, kept)
    assert unet.generation == 1


@pytest.mark.gpu
@pytest.mark.parametrize("options", [{}, {"attention": "shared_prefix"}, {"attention": "shared_prefix", "kv_cache": "int8"}])
def test_captured_loop_follows_the_context(gpu, options):
    """Contexts of other shapes and texts, captured and eager: the same bits."""
    package, context, ops = gpu
    results = {}
    for use_graph in (False, True):
        unet = harness.UNetHarness(ops, MINIATURE, precision="e4m3", seed=3, **options)
        loop = harness.EulerDenoiser(unet, 4, height=128, width=128, steps=2, use_graph=use_graph)
        latents, _, pooled, time_ids = (x.cuda() for x in inputs(8, 8, seed=9))
        out = []
        shapes = [(4, 77), (8, 77), (2, 77), (4, 154), (4, 77), (4, 77)] if options else [(8, 77), (8, 154), (8, 77)]
        for i, (rows, tokens) in enumerate(shapes):
            loop.set_conditioning(context_of(rows, tokens, i).cuda(), pooled, time_ids)
            loop.set_latents(latents[:4])
            out.append(loop.run().clone())
            torch.full((1 << 24,), float("nan"), device="cuda")          # whoever gets memory next writes over it
        results[use_graph] = out
        context.check()
        unet.close()
    for eager, captured in zip(results[False], results[True]):
        assert torch.isfinite(eager).all() and torch.equal(eager, captured)
    for one, other in zip(results[False], results[False][1:]):
        assert not torch.equal(one, other)
