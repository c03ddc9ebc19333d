"""Scratch whose zeroing fails is not kept: the next call would take its arrivals for zero.  tl_zeroed on a fake device, and that attention's scratch comes from it."""
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "torchlette_b200", "csrc")
CUDA = os.path.dirname(os.path.dirname(os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")))


def test_zeroed_scratch(tmp_path):
    exe = str(tmp_path / "zeroed")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-O1", "-I", CSRC, "-I", os.path.join(CUDA, "include"), os.path.join(ROOT, "tests", "pool_stub", "stub_zeroed.cpp"),
                    "-o", exe], check=True)
    subprocess.run([exe], check=True)


def test_attention_keeps_only_zeroed_scratch():
    text = open(os.path.join(CSRC, "tl_paged_attention.cu")).read()
    assert re.findall(r"tl_zeroed\(ctx->pool, &ctx->paged_scratch\b", text) and not re.search(r"paged_scratch = |device_malloc\(&ctx->paged_scratch", text)
