"""Layouts that the cache's copies and attention would write over themselves are refused, those that only look like it are not.
Without a GPU."""
import itertools
import os
import subprocess

import pytest


@pytest.fixture(scope="module")
def answers(pkg, tmp_path_factory):
    """A program that reads lines `dim e0 e1 e2 s0 s1 s2` and prints what write, read and attention say of something written
    with these extents and strides: 1 where it is refused for overlapping, else 0. Its context has no device and no workspace."""
    pkg.build()
    folder = tmp_path_factory.mktemp("overlap")
    source = folder / "overlap.cpp"
    source.write_text(r'''
#include "context.cuh"
#include <cstdio>
#include <cstring>
int main() {
    unsigned long long dim, e[3], s[3];
    while (std::scanf("%llu %llu %llu %llu %llu %llu %llu", &dim, e, e + 1, e + 2, s, s + 1, s + 2) == 7) {
        sdxlq_context ctx;
        const auto refused = [&](int status) { return status == SDXLQ_ERR_INVALID_ARGUMENT && std::strstr(ctx.last_error.c_str(), "overlap") != nullptr; };
        void* const somewhere = reinterpret_cast<void*>(0x10000);
        sdxlq_kv_cache cache{};
        cache.k = cache.v = somewhere; cache.slots = e[0]; cache.capacity = e[1]; cache.heads = e[2]; cache.head_dim = dim; cache.dtype = SDXLQ_FP16;
        cache.slot_stride = s[0]; cache.token_stride = s[1]; cache.head_stride = s[2];
        sdxlq_kv_tokens tokens{};
        tokens.k = tokens.v = somewhere; tokens.rows = e[0]; tokens.tokens = e[1];
        tokens.row_stride = 1ull << 36; tokens.token_stride = 1ull << 24; tokens.head_stride = dim;
        const int write = refused(sdxlq_kv_cache_write(&ctx, &cache, &tokens));
        tokens.row_stride = s[0]; tokens.token_stride = s[1]; tokens.head_stride = s[2];
        cache.slot_stride = 1ull << 36; cache.token_stride = 1ull << 24; cache.head_stride = dim;
        const int read = refused(sdxlq_kv_cache_read(&ctx, &cache, &tokens));
        sdxlq_attention_desc d{};
        d.q = d.y = somewhere; d.batch = e[0]; d.q_tokens = e[1]; d.q_heads = e[2]; d.head_dim = dim; d.scale = 1.0f;
        d.y_batch_stride = s[0]; d.y_token_stride = s[1]; d.y_head_stride = s[2];
        d.own = cache; d.own.heads = 1;
        const int attention = refused(sdxlq_shared_prefix_attention(&ctx, &d));
        std::printf("%d %d %d\n", write, read, attention);
    }
}
''')
    package = os.path.dirname(pkg.library_path())
    subprocess.run(["g++", "-std=c++20", "-I", pkg.api._build.CSRC, "-I", "/usr/local/cuda/include", str(source), "-L", package, "-lsdxlq",
                    "-L/usr/local/cuda/lib64", "-lcudart", f"-Wl,-rpath,{package}", "-o", str(folder / "overlap")], check=True)

    def ask(layouts):
        # no device is visible: a layout that is not refused must end before a launch
        text = "".join(" ".join(str(n) for n in (dim, *extents, *strides)) + "\n" for dim, extents, strides in layouts)
        run = subprocess.run([str(folder / "overlap")], input=text, capture_output=True, text=True, check=True, env={**os.environ, "CUDA_VISIBLE_DEVICES": ""})
        return [tuple(int(n) for n in line.split()) for line in run.stdout.splitlines()]

    return ask


def writes_itself(dim, extents, strides):
    """By every offset."""
    seen = set()
    for at in itertools.product(*(range(n) for n in extents)):
        first = sum(i * s for i, s in zip(at, strides))
        for offset in range(first, first + dim, 8):
            if offset in seen:
                return True
            seen.add(offset)
    return False


REFUSED = [(64, (2, 5, 4), (64, 64, 64)), (64, (2, 5, 4), (64 * 20, 64, 64)), (64, (2, 5, 4), (64 * 19, 256, 64)),
           (64, (2, 5, 4), (1280, 192, 64)), (128, (3, 1, 2), (128, 0, 128)), (16, (4, 4, 4), (64, 16, 56)), (64, (2, 5, 4), (0, 256, 64)),
           (64, (2, 2 ** 31 - 1, 4), (2 ** 40, 2 ** 40, 64))]
ALLOWED = [(64, (2, 5, 4), (64, 512, 128)), (64, (2, 5, 4), (64 * 20, 256, 64)), (64, (2, 5, 4), (64 * 20, 64, 64 * 5)), (64, (2, 5, 4), (256, 512, 64)),
           (64, (2, 5, 4), (2560, 512, 128)), (128, (1, 3, 1), (0, 128, 0)), (64, (1, 1, 1), (0, 0, 0)), (16, (3, 2, 5), (16, 240, 48)),
           (64, (1, 2 ** 31 - 1, 4), (0, 2 ** 40, 64))]


def test_layouts(answers):
    refused, allowed = answers(REFUSED), answers(ALLOWED)
    assert refused == [(1, 1, 1)] * (len(REFUSED) - 1) + [(1, 1, 0)]        # the last is too many rows for attention
    assert allowed == [(0, 0, 0)] * len(ALLOWED)
    for dim, extents, strides in REFUSED[:-1]:
        assert writes_itself(dim, extents, strides)
    for dim, extents, strides in ALLOWED[:-1]:
        assert not writes_itself(dim, extents, strides)


def test_every_small_layout(answers):
    """Whatever writes itself is refused; what a tensor's dimensions in any order, some of them sliced, give is not."""
    strides = [8, 16, 24, 32, 48, 64, 96, 128]
    layouts = [(16, extents, s) for extents in ((2, 2, 2), (2, 3, 2), (1, 3, 4)) for s in itertools.product(strides, repeat=3)]
    for (dim, extents, s), said in zip(layouts, answers(layouts)):
        assert said in ((0, 0, 0), (1, 1, 1))
        if writes_itself(dim, extents, s):
            assert said == (1, 1, 1), (extents, s)
    nested = []
    for order in itertools.permutations(range(3)):
        for gaps in itertools.product((0, 8), repeat=3):
            stride, reach, extents = [0, 0, 0], 16, (2, 3, 4)
            for axis, gap in zip(order, gaps):
                stride[axis] = reach + gap
                reach = stride[axis] * extents[axis]
            nested.append((16, extents, tuple(stride)))
    assert answers(nested) == [(0, 0, 0)] * len(nested)
