"""A CTA may touch another one's shared memory only once that one runs: in every kernel that a cluster is launched for, a wait of the whole cluster stands before the
first access of another CTA's shared memory.  What a missing wait does depends on when the CTAs start, so the sources are looked at."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torchlette_b200", "csrc")
REMOTE = re.compile(r"map_shared_rank\(|ld_cluster_f32\(|mapa_u32\(|\.tell\(|\.send\(|\.narrow<|template narrow|cluster_sum\(|totals\(")
WAIT = re.compile(r"cluster\.sync\(\)|cluster_sync_all\(\)|barrier\.cluster\.wait")


def _body(text, signature):
    """The function whose declaration holds `signature`, comments taken out."""
    at = text.index("{", text.index(")", text.index(signature)))
    depth, end = 0, at
    while True:
        depth += {"{": 1, "}": -1}.get(text[end], 0)
        end += 1
        if depth == 0:
            return re.sub(r"//[^\n]*", "", text[at:end])


@pytest.mark.parametrize("source,signature", [("tl_sample.cu", "sample_kernel(SampleArgs"), ("tl_attention.cu", "void decode_merge("),
                                              ("tl_matmul_tc.cu", "dense_tc_kernel(")])
def test_the_cluster_runs_before_its_shared_memory_is_touched(source, signature):
    text = open(os.path.join(CSRC, source)).read()
    body = _body(text, signature)
    first = REMOTE.search(body)
    assert first, "no access of another CTA's shared memory"
    assert WAIT.search(body[:first.start()]), f"{first.group()} comes before any wait of the cluster"
    arrive, wait = body.find("barrier.cluster.arrive"), body.find("barrier.cluster.wait")
    assert (arrive < 0) == (wait < 0) and arrive <= wait
