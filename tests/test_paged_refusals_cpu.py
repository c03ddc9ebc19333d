"""More of what the backend refuses, or passes on as it is meant, in the paged cache's calls."""
import ctypes as C

import pytest

from test_paged_cpu import ATTEND, AT, _cache, _paged, _t, be, ctx, stub  # noqa: F401
from torchlette_b200 import backend as tb
from torchlette_b200 import binding as B


def test_transposed_tables_are_refused(be):  # noqa: F811
    cache, pos, q, k, v = _paged(be), _t(be, [3], "i32"), _t(be, [3, 4, 64]), _t(be, [3, 2, 64]), _t(be, [3, 2, 64])
    good, turned = _t(be, [50, 32], "f32"), be.ops.transpose(_t(be, [32, 50], "f32"))
    assert turned.shape == good.shape
    for cos, sin in ((turned, good), (good, turned)):
        with pytest.raises(tb.TlError, match="cos and sin"):
            be.ops.pagedAppend(cache, pos, q, k, v, cos, sin)
    assert not [c for c in be.calls if c[0] != "tl_alloc"]


@pytest.mark.parametrize("shape", [[9, 0, 16, 64], [9, 2, 0, 64], [9, 2, 16, 0]])
def test_a_cache_without_heads_slots_or_dimensions_is_refused(be, shape):  # noqa: F811
    with pytest.raises(tb.TlError, match="createPagedCache"):
        tb.PagedCache(be, _t(be, shape), _t(be, shape), _t(be, [3, 4], "i32"))
    tb.PagedCache(be, _t(be, [0, 2, 16, 64]), _t(be, [0, 2, 16, 64]), _t(be, [0, 0], "i32"))  # one without pages yet is not


def test_a_window_past_32_bits_is_none_and_a_negative_one_is_refused(be):  # noqa: F811
    cache, pos, q = _paged(be), _t(be, [3], "i32"), _t(be, [3, 4, 64])
    for window, told in ((0, 0), (7, 7), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31, 2 ** 31 - 1), (2 ** 32, 2 ** 31 - 1), (2 ** 32 + 5, 2 ** 31 - 1)):
        be.ops.pagedAttention(cache, pos, q, 0.1, window=window)
        assert be.calls[-1][0] == "tl_paged_attention" and be.calls[-1][-2] == told
    calls = len(be.calls)
    for window in (-1, -2 ** 32, -2 ** 32 + 3):
        with pytest.raises(tb.TlError, match="window"):
            be.ops.pagedAttention(cache, pos, q, 0.1, window=window)
    assert len(be.calls) == calls


def test_attention_over_its_own_queries_is_refused(ctx):  # noqa: F811
    lib = B.load()
    assert ATTEND["q"] == ATTEND["out"]
    assert lib.tl_paged_attention(ctx, C.byref(_cache()), *ATTEND.values()) == B.TL_ERR_INVALID_ARG
    assert b"overlaps" in lib.tl_last_error(ctx)
