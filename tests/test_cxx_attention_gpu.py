"""The kv cache and attention through the C++20 host side (sdxl-end2end_b200/cpp/sdxlq_ops.hpp): the same bits as through
the Python one, which runs the same kernels."""
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PACKAGE = os.path.join(ROOT, "sdxl-end2end_b200")


def build_driver(directory) -> str:
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    binary = os.path.join(directory, "attention_driver")
    result = subprocess.run([shutil.which("g++") or "g++", "-std=c++20", "-Wall", "-Wextra", "-O1", "-I", os.path.join(ROOT, "include"),
                             "-I", os.path.join(PACKAGE, "cpp"), "-I", os.path.join(cuda, "include"),
                             os.path.join(ROOT, "tests", "cpp", "attention_driver.cpp"), "-o", binary, "-L", PACKAGE, "-lsdxlq",
                             "-L", os.path.join(cuda, "lib64"), "-lcudart", f"-Wl,-rpath,{PACKAGE}", f"-Wl,-rpath,{os.path.join(cuda, 'lib64')}"],
                            capture_output=True, text=True)
    assert result.returncode == 0, result.stderr
    return binary


def test_the_driver_compiles(tmp_path, pkg):
    pkg.load_library()
    build_driver(str(tmp_path))


@pytest.mark.gpu
@pytest.mark.parametrize("prompts,images,keys,tokens,heads,dim,dtype", [(2, 4, 77, 100, 5, 64, "Int8"), (1, 3, 130, 1, 4, 32, "Float8E4M3"),
                                                                        (2, 2, 33, 7, 2, 128, "Float16")])
def test_same_bits_as_the_python_operators(tmp_path, pkg, prompts, images, keys, tokens, heads, dim, dtype):
    pkg.load_library()
    kind = getattr(pkg.ScalarType, dtype)
    generator = torch.Generator().manual_seed(keys)
    k, v = (torch.randn(prompts, keys, heads, dim, generator=generator).half() for _ in "kv")
    q = torch.randn(images, tokens, heads, dim, generator=generator).half()
    case, result = str(tmp_path / "case.bin"), str(tmp_path / "result.bin")
    with open(case, "wb") as handle:
        handle.write(np.array([prompts, images, keys, tokens, heads, dim, int(kind)], np.uint64).tobytes())
        for tensor in (k, v, q):
            handle.write(tensor.numpy().tobytes())
    run = subprocess.run([build_driver(str(tmp_path)), case, result], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr + run.stdout
    raw = torch.from_numpy(np.fromfile(result, np.float16))

    context = pkg.Context(0)
    ops = pkg.Ops(context)
    cache = ops.kv_cache(prompts, keys, heads, dim, kind)
    ops.kv_cache_write(cache, k.cuda(), v.cuda())
    held = ops.kv_cache_read(cache, keys)
    want = [*held, ops.shared_prefix_attention(q.cuda(), None, cache)]
    context.check()
    at = 0
    for tensor in want:
        assert torch.equal(raw[at:at + tensor.numel()].view(torch.int16), tensor.cpu().flatten().view(torch.int16))
        at += tensor.numel()
    assert at == raw.numel()
    context.close()
