"""A token that is not there has no rows either: both append kernels return before they read one.  (A read past the caller's rows may go unseen on a GPU, so the
source is looked at; tests/test_gpu_paged_absent.py has the results.)"""
import os
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torchlette_b200", "csrc", "tl_paged_append.cu")


@pytest.mark.parametrize("kernel,read", [("append_kernel(AppendArgs p)", r"ld_f32\("), ("append_vec_kernel(const __grid_constant__ AppendArgs p)", r"\.load\(from")])
def test_positions_are_looked_at_before_rows_are_read(kernel, read):
    text = re.sub(r"//[^\n]*", "", open(SOURCE).read())
    body = text[text.index(kernel):]
    first = re.search(read, body).start()
    left = re.search(r"if \(!(is_there|place)\([^;]*\)\) (return|continue);", body)
    assert left and left.start() < first
