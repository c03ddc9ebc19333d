"""Scratch whose zeroing fails is not kept: the next call would take its arrivals for zero.  tl_zeroed on a fake device, and that the scratch with arrivals in it comes from there."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "torchlette_b200", "csrc")
CUDA = os.path.dirname(os.path.dirname(os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")))


def test_zeroed_scratch(tmp_path):
    exe = str(tmp_path / "zeroed")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-O1", "-I", CSRC, "-I", os.path.join(CUDA, "include"), os.path.join(ROOT, "tests", "pool_stub", "stub_zeroed.cpp"),
                    "-o", exe], check=True)
    subprocess.run([exe], check=True)


@pytest.mark.parametrize("source,name", [("tl_paged_attention.cu", "paged_scratch"), ("tl_api.cu", "zscratch"), ("tl_qgemv_stream.cu", "stream_scratch")])
def test_only_zeroed_scratch_is_kept(source, name):
    text = open(os.path.join(CSRC, source)).read()
    assert f"tl_zeroed(ctx->pool, &ctx->{name}," in text and not re.search(rf"\b{name} = (?!nullptr)|device_malloc\(&ctx->{name}\b", text)
