"""What the attention operators refuse, and the layout of their structures, without a GPU."""
import ctypes
import math
import os
import subprocess

import pytest
import torch

import attention_reference as R
from conftest import ROOT


@pytest.fixture(scope="module")
def api(pkg):
    pkg.build()
    return pkg.api


def test_structures_match_the_c_layout(api, tmp_path):
    structures = {"sdxlq_kv_cache": api._CKvCache, "sdxlq_kv_tokens": api._CKvTokens, "sdxlq_attention_desc": api._CAttentionDesc}
    lines = "".join(f'  printf("%zu ", sizeof({name}));\n' + "".join(f'  printf("%zu ", offsetof({name}, {field}));\n' for field, _ in s._fields_)
                    for name, s in structures.items())
    source = tmp_path / "layout.c"
    source.write_text('#include "sdxlq.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void) {\n' + lines + "  return 0;\n}\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(source), "-o", str(tmp_path / "layout")], check=True)
    printed = [int(v) for v in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()]
    expected = []
    for s in structures.values():
        expected += [ctypes.sizeof(s)] + [getattr(s, field).offset for field, _ in s._fields_]
    assert printed == expected


@pytest.fixture(scope="module")
def refusals(api, tmp_path_factory):
    """A program that gives the C entry points descriptors with one thing wrong, in a context that has no device: what is
    refused is refused before any call to CUDA. Prints name, status and message."""
    folder = tmp_path_factory.mktemp("refusals")
    source = folder / "refusals.cpp"
    source.write_text(r'''
#include "context.cuh"
#include <cmath>
#include <cstdio>
#include <functional>
static sdxlq_kv_cache cache(uint64_t slots, int32_t dtype) {
    sdxlq_kv_cache c{};
    c.k = reinterpret_cast<void*>(0x10000);
    c.v = reinterpret_cast<void*>(0x20000);
    c.k_scales = c.v_scales = dtype == SDXLQ_FP16 ? nullptr : reinterpret_cast<float*>(0x30000);
    c.slots = slots; c.capacity = 50; c.heads = 4; c.head_dim = 64;
    c.slot_stride = 50 * 256; c.token_stride = 256; c.head_stride = 64; c.dtype = dtype;
    return c;
}
int main() {
    sdxlq_context ctx;
    const auto copy = [&](const char* name, std::function<void(sdxlq_kv_cache&, sdxlq_kv_tokens&)> change) {
        for (int read = 0; read < 2; ++read) {
            sdxlq_kv_cache c = cache(3, SDXLQ_INT8);
            sdxlq_kv_tokens t{};
            t.k = reinterpret_cast<void*>(0x40000); t.v = reinterpret_cast<void*>(0x50000);
            t.rows = 3; t.tokens = 5; t.row_stride = 5 * 256; t.token_stride = 256; t.head_stride = 64;
            change(c, t);
            ctx.last_error = "";
            const int status = read ? sdxlq_kv_cache_read(&ctx, &c, &t) : sdxlq_kv_cache_write(&ctx, &c, &t);
            std::printf("%s|%d|%s\n", name, status, ctx.last_error.c_str());
        }
    };
    using C = sdxlq_kv_cache&; using T = sdxlq_kv_tokens&;
    copy("no tokens", [](C, T t) { t.tokens = 0; });
    copy("no rows", [](C, T t) { t.rows = 0; });
    copy("type", [](C c, T) { c.dtype = SDXLQ_FP32; });
    copy("null values", [](C c, T) { c.v = nullptr; });
    copy("no scales", [](C c, T) { c.v_scales = nullptr; });
    copy("no heads", [](C c, T) { c.heads = 0; });
    copy("head size 8", [](C c, T) { c.head_dim = 8; });
    copy("head size 144", [](C c, T) { c.head_dim = 144; });
    copy("head size 20 f16", [](C c, T) { c.dtype = SDXLQ_FP16; c.head_dim = 20; });
    copy("stride", [](C c, T) { c.token_stride = 264; });
    copy("huge stride", [](C c, T) { c.slot_stride = uint64_t(1) << 50; });
    copy("one place for all slots", [](C c, T t) { c.slot_stride = 0; t.row_stride = 0; });
    copy("one place for all tokens", [](C c, T t) { c.token_stride = 0; t.token_stride = 32; });
    copy("one place for all heads", [](C c, T t) { c.head_stride = 48; t.head_stride = 0; });
    copy("alignment", [](C c, T) { c.k = reinterpret_cast<void*>(0x10008); });
    copy("null tokens", [](C, T t) { t.v = nullptr; });
    copy("token stride", [](C, T t) { t.token_stride = 252; });
    copy("token alignment", [](C, T t) { t.k = reinterpret_cast<void*>(0x40002); });
    copy("rows", [](C, T t) { t.first_slot = 1; });
    copy("first slot", [](C, T t) { t.first_slot = ~0ull; });
    copy("start", [](C, T t) { t.start = 46; });
    copy("huge capacity", [](C c, T) { c.capacity = uint64_t(1) << 32; });
    const auto attend = [&](const char* name, std::function<void(sdxlq_attention_desc&)> change) {
        sdxlq_attention_desc d{};
        d.q = reinterpret_cast<void*>(0x60000); d.y = reinterpret_cast<void*>(0x70000);
        d.batch = 4; d.q_tokens = 3; d.q_heads = 8; d.head_dim = 64;
        d.q_batch_stride = d.y_batch_stride = 3 * 512; d.q_token_stride = d.y_token_stride = 512; d.q_head_stride = d.y_head_stride = 64;
        d.prefix = cache(2, SDXLQ_INT8); d.own = cache(4, SDXLQ_FP16); d.scale = 0.125f;
        change(d);
        ctx.last_error = "";
        const int status = sdxlq_shared_prefix_attention(&ctx, &d);
        std::printf("%s|%d|%s|%zu\n", name, status, ctx.last_error.c_str(), sdxlq_shared_prefix_attention_scratch(&ctx, &d));
    };
    using D = sdxlq_attention_desc&;
    attend("empty batch", [](D d) { d.batch = 0; });
    attend("no queries", [](D d) { d.q_tokens = 0; });
    attend("null query", [](D d) { d.q = nullptr; });
    attend("null output", [](D d) { d.y = nullptr; });
    attend("no query heads", [](D d) { d.q_heads = 0; });
    attend("query size", [](D d) { d.head_dim = 36; });
    attend("wide query", [](D d) { d.head_dim = 136; });
    attend("query alignment", [](D d) { d.q = reinterpret_cast<void*>(0x60002); });
    attend("output stride", [](D d) { d.y_token_stride = 508; });
    attend("one output for all entries", [](D d) { d.y_batch_stride = 0; });
    attend("one output for all heads", [](D d) { d.y_head_stride = 0; });
    attend("many rows", [](D d) { d.q_tokens = 1u << 30; });
    attend("scale", [](D d) { d.scale = NAN; });
    attend("no keys", [](D d) { d.prefix.slots = 0; d.own.slots = 0; });
    attend("head mismatch", [](D d) { d.own.head_dim = 32; });
    attend("head multiple", [](D d) { d.q_heads = 6; });
    attend("parts differ", [](D d) { d.own.heads = 2; });
    attend("own slots", [](D d) { d.own.slots = 2; });
    attend("prefix slots", [](D d) { d.prefix.slots = 3; });
    attend("own type", [](D d) { d.own.dtype = SDXLQ_INT32; });
    attend("prefix scales", [](D d) { d.prefix.k_scales = nullptr; });
    attend("small scratch", [](D d) { d.scratch = reinterpret_cast<void*>(0x80000); d.scratch_bytes = 64; });
    attend("scratch alignment", [](D d) { d.scratch = reinterpret_cast<void*>(0x80008); d.scratch_bytes = 1 << 30; });
    attend("no workspace", [](D) {});
    std::printf("null context|%d||\n", sdxlq_shared_prefix_attention(nullptr, nullptr));
    std::printf("null descriptor|%d|%s|\n", sdxlq_shared_prefix_attention(&ctx, nullptr), ctx.last_error.c_str());
    std::printf("null cache|%d|%s|\n", sdxlq_kv_cache_write(&ctx, nullptr, nullptr), ctx.last_error.c_str());
}
''')
    package = os.path.dirname(api.library_path())
    subprocess.run(["g++", "-std=c++20", "-I", api._build.CSRC, "-I", "/usr/local/cuda/include", str(source), "-L", package, "-lsdxlq",
                    "-L/usr/local/cuda/lib64", "-lcudart", f"-Wl,-rpath,{package}", "-o", str(folder / "refusals")], check=True)
    lines = subprocess.run([str(folder / "refusals")], capture_output=True, text=True, check=True).stdout.splitlines()
    found = {}
    for line in lines:
        name, status, message = line.split("|")[:3]
        found.setdefault(name, []).append((int(status), message))
    return found


INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 5


@pytest.mark.parametrize("name,status,words", [
    ("no tokens", 0, ""), ("no rows", 0, ""), ("type", INVALID, "expects FP16, INT8 or FP8"), ("null values", INVALID, "null keys or values"),
    ("no scales", INVALID, "needs scales"), ("no heads", INVALID, "no heads"), ("head size 8", UNSUPPORTED, "multiple of 8 for FP16"),
    ("head size 144", UNSUPPORTED, "at most 128"), ("head size 20 f16", UNSUPPORTED, "multiple of 8"), ("stride", UNSUPPORTED, "16 bytes"),
    ("huge stride", UNSUPPORTED, "16 bytes"), ("alignment", UNSUPPORTED, "16 bytes"), ("null tokens", INVALID, "null tokens"),
    ("token stride", UNSUPPORTED, "tokens and their strides"), ("token alignment", UNSUPPORTED, "tokens and their strides"),
    ("rows", INVALID, "more rows than slots"), ("first slot", INVALID, "more rows than slots"), ("start", INVALID, "behind the capacity"),
    ("huge capacity", UNSUPPORTED, "too large"), ("one place for all slots", INVALID, "overlaps"),
    ("one place for all tokens", INVALID, "overlaps"), ("one place for all heads", INVALID, "overlaps"),
    ("one output for all entries", INVALID, "overlap"), ("one output for all heads", INVALID, "overlap"),
    ("empty batch", 0, ""), ("no queries", 0, ""), ("null query", INVALID, "null query"), ("null output", INVALID, "null query or output"),
    ("no query heads", INVALID, "no heads"), ("query size", UNSUPPORTED, "multiple of 8"), ("wide query", UNSUPPORTED, "at most 128"),
    ("query alignment", UNSUPPORTED, "16 bytes"), ("output stride", UNSUPPORTED, "16 bytes"), ("many rows", UNSUPPORTED, "too large"),
    ("scale", INVALID, "finite"), ("no keys", INVALID, "neither"), ("head mismatch", INVALID, "differ in head size"),
    ("head multiple", INVALID, "multiple of key heads"), ("parts differ", INVALID, "differ in heads"), ("own slots", INVALID, "slot per batch entry"),
    ("prefix slots", INVALID, "multiple of the prefixes"), ("own type", INVALID, "expects FP16"), ("prefix scales", INVALID, "needs scales"),
    ("small scratch", WORKSPACE, "scratch"), ("scratch alignment", WORKSPACE, "scratch"), ("no workspace", WORKSPACE, "scratch"),
    ("null context", INVALID, ""), ("null descriptor", INVALID, "null descriptor"), ("null cache", INVALID, "null descriptor")])
def test_refused(refusals, name, status, words):
    assert refusals[name]
    for got, message in refusals[name]:
        assert got == status, message
        assert words in message


# ---- the Python mirror ---------------------------------------------------------------------------------------
def f16(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def test_cache_objects_check_their_tensors(pkg):
    int8, scales = torch.zeros((2, 5, 3, 32), dtype=torch.int8), torch.ones((2, 3, 5))
    pkg.KVCache(int8, int8, pkg.ScalarType.Int8, scales, scales)
    cache = pkg.KVCache.of(f16(2, 5, 96), f16(2, 5, 96), 3)
    assert (cache.slots, cache.capacity, cache.heads, cache.head_dim) == (2, 5, 3, 32)
    for wrong in (lambda: pkg.KVCache(f16(2, 5, 3, 32), f16(2, 5, 3, 32), pkg.ScalarType.Int8, scales, scales),
                  lambda: pkg.KVCache(f16(2, 5, 3, 32), f16(2, 5, 3, 16)),
                  lambda: pkg.KVCache(f16(2, 5, 96), f16(2, 5, 96)),
                  lambda: pkg.KVCache(f16(2, 5, 32, 3).transpose(2, 3), f16(2, 5, 32, 3).transpose(2, 3)),
                  lambda: pkg.KVCache(f16(2, 5, 3, 32), f16(2, 3, 5, 32).transpose(1, 2)),
                  lambda: pkg.KVCache(f16(2, 5, 3, 32), f16(2, 5, 3, 32), pkg.ScalarType.Float16, scales, scales),
                  lambda: pkg.KVCache(int8, int8, pkg.ScalarType.Int8),
                  lambda: pkg.KVCache(int8, int8, pkg.ScalarType.Int8, scales, scales.transpose(1, 2)),
                  lambda: pkg.KVCache(int8, int8, pkg.ScalarType.Int8, scales.double(), scales),
                  lambda: pkg.KVCache(int8, int8, pkg.ScalarType.Float32, scales, scales),
                  lambda: pkg.KVCache.of(f16(2, 5, 96), f16(2, 5, 96), 5),
                  lambda: pkg.KVCache.of(f16(2, 5, 3, 32), f16(2, 5, 3, 32), 3)):
        with pytest.raises(pkg.CudaError):
            wrong()


class NoContext:
    """Stands in for a context: nothing here may reach the library."""
    device = address = stream_address = 0
    _lib = None
    _front = None


def test_operators_check_their_arguments(pkg):
    ops = pkg.Ops(NoContext())
    cache = pkg.KVCache(f16(2, 5, 3, 32), f16(2, 5, 3, 32))
    k = f16(2, 1, 3, 32)
    q = f16(2, 1, 6, 32)
    int32 = lambda *values: torch.tensor(values, dtype=torch.int32)
    for wrong, words in (
            (lambda: ops.kv_cache_write(cache, k.float(), k.float()), "FP16"),
            (lambda: ops.kv_cache_write(cache, k, f16(2, 2, 3, 32)), "FP16"),
            (lambda: ops.kv_cache_write(cache, f16(2, 1, 4, 32), f16(2, 1, 4, 32)), "cache's heads"),
            (lambda: ops.kv_cache_write(cache, k, k, positions=torch.zeros(2)), "INT32"),
            (lambda: ops.kv_cache_write(cache, k, k, positions=int32(0)), "2 elements"),
            (lambda: ops.kv_cache_write(cache, k, k, counts=int32(1, 1, 1)), "2 elements"),
            (lambda: ops.kv_cache_write(cache, k, k, positions=-1), "in front"),
            (lambda: ops.kv_cache_write(cache, k, k, first_slot=-1), "in front"),
            (lambda: ops.kv_cache_write(cache, k, k), "context's device"),
            (lambda: ops.kv_cache_read(cache, -1), "negative"),
            (lambda: ops.kv_cache_read(cache, 1, first_slot=3), "negative"),
            (lambda: ops.kv_cache_read(cache, 1), "context's device"),
            (lambda: ops.kv_cache(1, 1, 1, 64, pkg.ScalarType.Float32), "expects"),
            (lambda: ops.shared_prefix_attention(q.float(), cache), "FP16 queries"),
            (lambda: ops.shared_prefix_attention(f16(2, 6, 32), cache), "FP16 queries"),
            (lambda: ops.shared_prefix_attention(f16(2, 1, 32, 6).transpose(2, 3), cache), "elements together"),
            (lambda: ops.shared_prefix_attention(q, cache, out=f16(2, 1, 6, 16)), "output"),
            (lambda: ops.shared_prefix_attention(q, cache, out=f16(1, 1, 6, 32).expand(2, -1, -1, -1)), "output"),
            (lambda: ops.shared_prefix_attention(q, cache, prefix_lengths=int32(1)), "without the part"),
            (lambda: ops.shared_prefix_attention(q, cache, own_lengths=int32(1)), "2 elements"),
            (lambda: ops.shared_prefix_attention(q, cache, own_lengths=torch.zeros(2, dtype=torch.int64)), "INT32"),
            (lambda: ops.shared_prefix_attention(q, cache, pkg.KVCache(f16(0, 5, 3, 32), f16(0, 5, 3, 32))), "no slots"),
            (lambda: ops.shared_prefix_attention(q, cache), "context's device")):
        with pytest.raises(pkg.CudaError, match=words):
            wrong()


def test_the_reference_itself():
    """The definition against a sum written out, and a planted mistake of one key that the bound must see."""
    torch.manual_seed(1)
    q, k, v = torch.randn(2, 3, 4, 16), torch.randn(2, 7, 2, 16).double(), torch.randn(2, 7, 2, 16).double()
    pk, pv = torch.randn(1, 5, 2, 16).double(), torch.randn(1, 5, 2, 16).double()
    y, bound = R.attention(q, (k, v), (pk, pv), [7, 2], None, True)
    for b, i, h in ((0, 2, 3), (0, 0, 1), (1, 0, 0), (1, 1, 2)):
        n = [7, 2][b]
        seen = list(range(max(0, min(n, n - 3 + i + 1))))
        keys = [pk[0, j, h // 2] for j in range(5)] + [k[b, j, h // 2] for j in seen]
        vals = [pv[0, j, h // 2] for j in range(5)] + [v[b, j, h // 2] for j in seen]
        w = [math.exp(float(q[b, i, h].double() @ key) / 4.0) for key in keys]
        want = sum(x * val for x, val in zip(w, vals)) / sum(w)
        assert torch.allclose(y[b, i, h], want, rtol=1e-12, atol=1e-12)
    assert R.off(y.half(), y, bound) <= 1.0
    planted, _ = R.attention(q, (k, v), (pk[:, :4], pv[:, :4]), [7, 2], None, True)
    assert R.off(planted.half(), y, bound) > 1.0


@pytest.mark.parametrize("dtype", R.TYPES)
def test_the_reference_quantiser(dtype):
    torch.manual_seed(2)
    x = (torch.randn(50, 32) * torch.exp(2 * torch.randn(50, 1))).half()
    x[3] = 0
    q, s = R.quantise(x, dtype)
    back = R.values_of(q, s)
    half_step = {"f16": 0.0, "int8": None, "e4m3": 2 ** -4, "e5m2": 2 ** -3}[dtype]
    if dtype == "int8":
        assert ((back - x.double()).abs() <= s.double()[:, None] / 2 * (1 + 1e-9)).all()
    else:
        least = 0.0 if s is None else s.double()[:, None] * 2.0 ** {"e4m3": -10, "e5m2": -17}[dtype]
        assert ((back - x.double()).abs() <= (half_step * x.double().abs()).maximum(torch.as_tensor(least))).all()
