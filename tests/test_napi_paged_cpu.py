"""The paged cache's calls and sampling as JavaScript makes them: the addon against a fake N-API (tests/napi_stub/stub_paged.c), and the checks that stand in front of it
in TypeScript, which nothing here can run and which are looked at as text."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHIM = os.path.join(ROOT, "torchlette_b200", "csrc", "napi", "tl_napi.c")
STUB = os.path.join(ROOT, "tests", "napi_stub", "stub_paged.c")
TS = os.path.join(ROOT, "torchlette_b200", "ts", "index.ts")


def test_the_addon_refuses_what_its_buffers_do_not_hold(tmp_path):
    exe = str(tmp_path / "stub_paged")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Wextra", "-Werror", "-O1", "-no-pie", "-I", os.path.join(ROOT, "include"), SHIM, STUB,
                    "-Wl,--unresolved-symbols=ignore-all", "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip().endswith("ALL OK"), r.stdout + r.stderr


def _function(name):
    text = open(TS).read()
    at = text.index(f"export function {name}(")
    return text[at:text.index("\n}\n", at)]


@pytest.mark.parametrize("name,tensors", [("pagedAppend", ["positions", "tokenSeq", "q", "k", "v", "out", "qNorm", "kNorm", "cos", "sin"]),
                                          ("pagedAttention", ["positions", "tokenSeq", "q", "out", "slopes"]),
                                          ("sample", ["logits", "uniforms", "temperature", "topK", "topP", "minP", "out"])])
def test_typescript_looks_at_every_tensor(name, tensors):
    """Each tensor whose buffer is handed over is named in a check before the addon is called; what is new has the cache's type, not q's."""
    body = _function(name)
    call = body.index("addon." + name)
    checked = "".join(re.findall(r"(?:fits|refuseUnless|tokensOf)\([^;]*;", body[:call]))
    for t in tensors:
        assert re.search(rf"\b{t}\b", checked), t
    assert "q.dtype" not in re.sub(r"(?:fits|refuseUnless)\([^;]*;", "", body)


@pytest.mark.parametrize("name", ["pagedAppend", "pagedAttention", "sample"])
def test_typescript_needs_no_allocation(name):
    """A capture takes no allocations: each call writes where it is told to."""
    body = _function(name)
    assert "config.out ?? empty(" in body and body.count("empty(") == 1
