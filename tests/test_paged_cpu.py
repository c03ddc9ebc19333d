"""The paged cache's calls and sampling without a GPU: what they refuse, by the C ABI on a context made for it (tests/ctx_stub) and by the
backend's own checks; which indexes of the device become addresses; and the arguments that the backend hands over."""
import ctypes as C
import itertools
import os
import subprocess

import pytest

from torchlette_b200 import backend as tb
from torchlette_b200 import binding as B

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = os.path.dirname(os.path.dirname(os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")))


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("ctx") / "stub_ctx.so")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "torchlette_b200", "csrc"), "-I",
                    os.path.join(CUDA, "include"), os.path.join(ROOT, "tests", "ctx_stub", "stub_ctx.cpp"), "-o", so], check=True)
    lib = C.CDLL(so)
    lib.stub_ctx.restype = C.c_void_p
    lib.stub_bad_token.argtypes = [C.c_int, C.c_longlong, C.c_int, C.c_int, C.c_int, C.c_longlong]
    lib.stub_bad_page.argtypes = [C.c_int, C.c_longlong]
    lib.stub_page_at.argtypes = [C.c_int] * 5
    lib.stub_page_at.restype = C.c_longlong
    shares = [C.c_longlong, C.c_int, C.c_int, C.c_longlong]
    for name, kinds, result in (("share_ctas", shares, C.c_int), ("share_begin", shares + [C.c_int], C.c_longlong), ("share_owner", shares + [C.c_longlong], C.c_int),
                                ("divide_wrong", [C.c_int, C.c_int], C.c_longlong)):
        f = getattr(lib, "stub_" + name)
        f.argtypes, f.restype = kinds, result
    return lib


@pytest.fixture(scope="module")
def ctx(stub):
    return stub.stub_ctx()


AT = 1 << 20  # an address that no refused call touches


def _cache(**more):
    fields = dict(k_pages=AT, v_pages=AT, page_table=AT, n_pages=8, page_size=16, n_kv_heads=2, head_dim=64, dtype=B.TL_F16, n_seqs=3, max_pages=4)
    return B.PagedCache(**{**fields, **more})


APPEND = dict(positions=AT, token_seq=None, tokens=3, q=AT, q_ts=256, q_hs=64, heads=4, q_out=2 * AT, o_ts=256, o_hs=64, k=AT, k_ts=128, k_hs=64, v=AT,
              v_ts=128, v_hs=64, q_weight=None, k_weight=None, weight_dtype=0, eps=1e-6, cos=AT, sin=AT, rows=100)


@pytest.mark.parametrize("cache,args,status,text", [
    (dict(page_size=0), {}, B.TL_ERR_INVALID_ARG, b"bad shape"),
    (dict(n_kv_heads=0), {}, B.TL_ERR_INVALID_ARG, b"bad shape"),
    (dict(max_pages=-1), {}, B.TL_ERR_INVALID_ARG, b"bad shape"),
    (dict(dtype=7), {}, B.TL_ERR_INVALID_ARG, b"dtype"),
    (dict(head_dim=65), {}, B.TL_ERR_INVALID_ARG, b"head_dim"),
    (dict(head_dim=1026), {}, B.TL_ERR_INVALID_ARG, b"head_dim"),
    (dict(k_pages=None), {}, B.TL_ERR_INVALID_ARG, b"null pointer"),
    (dict(page_table=None), {}, B.TL_ERR_INVALID_ARG, b"null pointer"),
    (dict(max_pages=1 << 28), {}, B.TL_ERR_UNSUPPORTED, b"2^31"),
    (dict(page_size=1 << 26, max_pages=1), {}, B.TL_ERR_UNSUPPORTED, b"2^31"),
    ({}, dict(tokens=4), B.TL_ERR_INVALID_ARG, b"token_seq"),
    ({}, dict(tokens=-1), B.TL_ERR_INVALID_ARG, b"bad shape"),
    ({}, dict(positions=None), B.TL_ERR_INVALID_ARG, b"null pointer"),
    ({}, dict(k=None), B.TL_ERR_INVALID_ARG, b"null k or v"),
    ({}, dict(q=None), B.TL_ERR_INVALID_ARG, b"only one of q and q_out"),
    ({}, dict(q_out=None), B.TL_ERR_INVALID_ARG, b"only one of q and q_out"),
    ({}, dict(q_out=AT, o_ts=300), B.TL_ERR_INVALID_ARG, b"in place"),
    ({}, dict(heads=0), B.TL_ERR_INVALID_ARG, b"n_heads"),
    ({}, dict(sin=None), B.TL_ERR_INVALID_ARG, b"both tables"),
    ({}, dict(rows=-1), B.TL_ERR_INVALID_ARG, b"both tables"),
    ({}, dict(q_weight=AT, weight_dtype=9), B.TL_ERR_INVALID_ARG, b"weight dtype"),
    ({}, dict(v_ts=-64), B.TL_ERR_INVALID_ARG, b"negative stride"),
])
def test_append_refuses(ctx, cache, args, status, text):
    lib = B.load()
    assert lib.tl_paged_append(ctx, C.byref(_cache(**cache)), *{**APPEND, **args}.values()) == status
    assert text in lib.tl_last_error(ctx), lib.tl_last_error(ctx)


ATTEND = dict(positions=AT, token_seq=None, tokens=3, q=AT, q_ts=256, q_hs=64, heads=4, out=AT, scale=0.1, softcap=0.0, window=0, slopes=None)


@pytest.mark.parametrize("cache,args,status,text", [
    (dict(head_dim=0), {}, B.TL_ERR_INVALID_ARG, b"bad shape"),
    (dict(head_dim=60), {}, B.TL_ERR_UNSUPPORTED, b"head_dim"),
    (dict(head_dim=264), {}, B.TL_ERR_UNSUPPORTED, b"head_dim"),
    (dict(k_pages=AT + 8), {}, B.TL_ERR_INVALID_ARG, b"16 bytes"),
    (dict(n_kv_heads=3), {}, B.TL_ERR_INVALID_ARG, b"heads"),
    ({}, dict(heads=0), B.TL_ERR_INVALID_ARG, b"heads"),
    ({}, dict(tokens=5), B.TL_ERR_INVALID_ARG, b"token_seq"),
    ({}, dict(q=None), B.TL_ERR_INVALID_ARG, b"null pointer"),
    ({}, dict(out=None), B.TL_ERR_INVALID_ARG, b"null pointer"),
    ({}, dict(q=AT + 4), B.TL_ERR_INVALID_ARG, b"16 bytes"),
    ({}, dict(out=AT + 2), B.TL_ERR_INVALID_ARG, b"16 bytes"),
    ({}, dict(q_ts=260), B.TL_ERR_INVALID_ARG, b"16 bytes"),
    ({}, dict(q_hs=-64), B.TL_ERR_INVALID_ARG, b"16 bytes"),
    ({}, dict(scale=float("nan")), B.TL_ERR_INVALID_ARG, b"finite"),
    ({}, dict(softcap=-1.0), B.TL_ERR_INVALID_ARG, b"softcap"),
    ({}, dict(softcap=float("inf")), B.TL_ERR_INVALID_ARG, b"finite"),
    ({}, dict(softcap=1e-40), B.TL_ERR_INVALID_ARG, b"1e-30"),
    ({}, dict(window=-3), B.TL_ERR_INVALID_ARG, b"window"),
])
def test_attention_refuses(ctx, cache, args, status, text):
    lib = B.load()
    assert lib.tl_paged_attention(ctx, C.byref(_cache(**cache)), *{**ATTEND, **args}.values()) == status
    assert text in lib.tl_last_error(ctx), lib.tl_last_error(ctx)


SAMPLE = dict(logits=AT, dtype=B.TL_F32, rows=2, vocab=1000, stride=1000, temperature=None, top_k=None, top_p=None, min_p=None, uniforms=AT, out=AT)


@pytest.mark.parametrize("args,status,text", [
    (dict(dtype=5), B.TL_ERR_INVALID_ARG, b"dtype"), (dict(vocab=0), B.TL_ERR_INVALID_ARG, b"bad shape"),
    (dict(rows=-1), B.TL_ERR_INVALID_ARG, b"bad shape"), (dict(stride=999), B.TL_ERR_INVALID_ARG, b"bad shape"),
    (dict(vocab=(1 << 24) + 1, stride=1 << 25), B.TL_ERR_UNSUPPORTED, b"2^24"), (dict(logits=None), B.TL_ERR_INVALID_ARG, b"null pointer"),
    (dict(out=None), B.TL_ERR_INVALID_ARG, b"null pointer"),
])
def test_sample_refuses(ctx, args, status, text):
    lib = B.load()
    assert lib.tl_sample(ctx, *{**SAMPLE, **args}.values()) == status
    assert text in lib.tl_last_error(ctx), lib.tl_last_error(ctx)


def test_nothing_to_do_is_no_error_and_a_null_context_is(ctx):
    lib = B.load()
    empty = _cache(k_pages=None, v_pages=None, page_table=None, n_pages=0, n_seqs=0, max_pages=0)
    assert lib.tl_paged_append(ctx, C.byref(empty), *{**APPEND, "tokens": 0, "positions": None, "k": None}.values()) == B.TL_OK
    assert lib.tl_paged_attention(ctx, C.byref(empty), *{**ATTEND, "tokens": 0, "positions": None, "q": None}.values()) == B.TL_OK
    assert lib.tl_sample(ctx, *{**SAMPLE, "rows": 0, "logits": None}.values()) == B.TL_OK
    assert lib.tl_paged_append(ctx, None, *APPEND.values()) == B.TL_ERR_INVALID_ARG
    assert lib.tl_paged_append(None, C.byref(empty), *APPEND.values()) == B.TL_ERR_INVALID_ARG
    assert lib.tl_paged_attention(None, C.byref(empty), *ATTEND.values()) == B.TL_ERR_INVALID_ARG
    assert lib.tl_sample(None, *SAMPLE.values()) == B.TL_ERR_INVALID_ARG


def test_only_indexes_in_range_become_addresses(stub):
    """Every (position, sequence, page) that passes lies inside the table and the pages, and every one that lies there passes."""
    n_seqs, max_pages, page_size, n_pages, heads, dim = 3, 4, 5, 6, 2, 8
    big = 2 ** 31 - 1
    for pos, seq, rows in itertools.product([0, 4, 5, 19, 20, 21, big], [-(2 ** 31), -1, 0, 2, 3, big], [-1, 0, 4, 19, 20, 21]):
        want = 2 if not 0 <= seq < n_seqs else 1 if pos >= max_pages * page_size or (rows >= 0 and pos >= rows) else 0
        assert stub.stub_bad_token(pos, seq, n_seqs, max_pages, page_size, rows) == want
    for page in (-(2 ** 31), -1, 0, 5, 6, big):
        assert bool(stub.stub_bad_page(page, n_pages)) == (not 0 <= page < n_pages)
    size = n_pages * heads * page_size * dim
    for page, slot in itertools.product(range(n_pages), range(page_size)):
        at = stub.stub_page_at(page, slot, heads, page_size, dim)
        assert at == ((page * heads) * page_size + slot) * dim and 0 <= at and at + ((heads - 1) * page_size + 1) * dim <= size
    # offsets past 2^31
    assert stub.stub_page_at(big, 15, 8, 16, 128) == (big * 8 * 16 + 15) * 128


def test_every_unit_has_one_owner(stub):
    """The shares cover the units without gaps, each is long enough to hold a tile, and the owner of a unit is the CTA whose share holds it."""
    lead = stub.stub_lead()
    for units, most, least, parts in itertools.product([lead + 1, lead + 2, 37, 295, 296, 297, 1000, 40_001], [1, 2, 148, 296], [1, 24], [1, 8, 300, 5000]):
        args = units, most, least, parts
        ctas = stub.stub_share_ctas(*args)
        assert 1 <= ctas <= most and ctas * (lead + 1) <= units and (ctas >= min(units // least, most) or ctas == units // (lead + 1))
        begins = [stub.stub_share_begin(*args, c) for c in range(ctas + 1)]
        assert begins[0] == 0 and begins[-1] == units and all(b - a >= lead + 1 for a, b in zip(begins, begins[1:]))
        assert max(b - a for a, b in zip(begins, begins[1:])) - min(b - a for a, b in zip(begins, begins[1:])) <= 1
        for c in range(ctas):
            assert stub.stub_share_owner(*args, begins[c]) == c and stub.stub_share_owner(*args, begins[c + 1] - 1) == c
    big = (1 << 40) + 12345, 296, 24, 1  # units of a call at the limits
    for c in range(296):
        assert stub.stub_share_owner(*big, stub.stub_share_begin(*big, c)) == c == stub.stub_share_owner(*big, stub.stub_share_begin(*big, c + 1) - 1)
    assert [stub.stub_tiles(a, b, 16) for a, b in ((0, 0), (5, 5), (0, 1), (0, 16), (0, 17), (3, 19), (15, 17), (16, 17), (2 ** 31 - 20, 2 ** 31 - 17), (2 ** 31 - 20, 2 ** 31 - 1))] == [
        0, 0, 1, 1, 2, 2, 2, 1, 1, 2]


@pytest.mark.parametrize("tiles,most", [([1, 7, 300, 2, 2, 90], 37), ([5000], 296), ([33] * 50, 296), ([1000, 1, 1, 999], 296), ([1] * 700, 296), ([3, 1] * 20, 148),
                                        ([1], 296), ([1, 1], 296), ([2000] + [1] * 100, 148)])
def test_parts_meet_in_slots_of_their_own(stub, tiles, most):
    """The shares walked on the host as the kernel walks them: every tile is taken once, the CTAs that have tiles of a part are those between the owners of its first and
    last, each leaves what it made of a part in a slot that no other part uses, and no two groups of thirteen count their arrivals in one place."""
    lead = stub.stub_lead()
    starts_at = list(itertools.accumulate([0] + [lead + n for n in tiles]))
    args = starts_at[-1], most, 24, len(tiles)
    ctas, taken, slots, places = stub.stub_share_ctas(*args), [0] * len(tiles), set(), set()
    for cta in range(ctas):
        begin, end = (stub.stub_share_begin(*args, x) for x in (cta, cta + 1))
        has = 0
        for part, n in enumerate(tiles):
            tile0 = starts_at[part] + lead
            u, stop = max(0, begin - tile0), min(n, end - tile0)
            if u >= stop:
                continue
            has += stop - u
            assert taken[part] == u
            taken[part] = stop
            first, last = (stub.stub_share_owner(*args, x) for x in (tile0, tile0 + n - 1))
            assert first <= cta <= last and (cta == first) == (u == 0) and (cta == last) == (stop == n)
            if (u, stop) != (0, n):
                slot = 2 * cta + (u == 0)
                assert slot not in slots
                slots.add(slot)
                if (cta - first) % 13 == 0:
                    place = 2 * cta + (cta == first)
                    assert place not in places and place < 2 * most
                    places.add(place)
        assert has > 0
    assert taken == tiles


@pytest.mark.parametrize("d", [1, 2, 3, 5, 7, 16, 24, 48, 100, 255, 256, 257, 641, 65_535, 65_537, 1_000_003, 2 ** 30, 2 ** 30 + 1, 2 ** 31 - 1])
def test_division_by_the_page_size(stub, d):
    assert stub.stub_divide_wrong(d, 5000) == -1


# ---- the backend's own checks, and what it hands over ----------------------------------------------------------------------


class _Backend:
    """A backend whose calls are written down."""

    def __init__(self):
        self._handle, self.calls = 8, []
        self.ops = tb.CudaOps(self)
        outer = self

        class Calls:
            def __getattr__(self, name):
                return lambda *a: outer.calls.append((name,) + a) or (4096 if name == "tl_alloc" else None)
        self._calls = Calls()


@pytest.fixture
def be():
    return _Backend()


def _t(be, shape, dtype="f16", at=1 << 16, **more):
    return tb.CudaTensor(be, shape, dtype, at, 0, ownsBuffer=False, **more)


def _paged(be, dtype="f16", g=2, d=64):
    return tb.PagedCache(be, _t(be, [9, g, 16, d], dtype, 100), _t(be, [9, g, 16, d], dtype, 200), _t(be, [3, 4], "i32", 300))


def test_a_cache_of_the_wrong_tensors_is_refused(be):
    pages, table = _t(be, [9, 2, 16, 64]), _t(be, [3, 4], "i32")
    for bad in ((_t(be, [9, 2, 16]), pages, table), (pages, _t(be, [9, 2, 16, 32]), table), (pages, _t(be, [9, 2, 16, 64], "f32"), table),
                (_t(be, [9, 2, 16, 64], "u32"), _t(be, [9, 2, 16, 64], "u32"), table), (pages, pages, _t(be, [3, 4], "f32")),
                (pages, pages, _t(be, [12], "i32")), (_t(be, [9, 2, 16, 64], transposed=True), pages, table)):
        with pytest.raises(tb.TlError):
            tb.PagedCache(be, *bad)


def test_the_descriptor_follows_the_tensors(be):
    cache = _paged(be)
    d = B.PagedCache.from_buffer_copy(cache.descriptor())
    assert (d.k_pages, d.v_pages, d.page_table, d.n_pages, d.page_size, d.n_kv_heads, d.head_dim, d.dtype, d.n_seqs, d.max_pages) == (
        100, 200, 300, 9, 16, 2, 64, B.TL_F16, 3, 4)
    cache.pageTable.buffer = 400  # another table for the next step
    assert B.PagedCache.from_buffer_copy(cache.descriptor()).page_table == 400


def _named(call):
    names = ["name", "ctx", "cache", "positions", "token_seq", "tokens", "q", "q_ts", "q_hs", "heads", "q_out", "o_ts", "o_hs", "k", "k_ts", "k_hs", "v", "v_ts",
             "v_hs", "q_weight", "k_weight", "weight_dtype", "eps", "cos", "sin", "rows"]
    assert len(call) == len(names)
    return dict(zip(names, call))


def test_append_hands_over_strides(be):
    cache, pos = _paged(be), _t(be, [3], "i32", 500)
    cos, sin, w = _t(be, [50, 32], "f32", 600), _t(be, [50, 32], "f32", 700), _t(be, [64], "f32", 800)
    q, k, v = _t(be, [3, 4, 64], at=1000), _t(be, [3, 128], at=2000), _t(be, [3, 2, 64], at=3000)
    out = be.ops.pagedAppend(cache, pos, q, k, v, cos, sin, qNorm=w, eps=1e-5)
    a = _named(be.calls[-1])
    assert out.shape == [3, 4, 64] and a["q_out"] == 4096 and (a["q"], a["k"], a["v"], a["cos"], a["sin"], a["rows"]) == (1000, 2000, 3000, 600, 700, 50)
    assert (a["q_ts"], a["q_hs"], a["o_ts"], a["o_hs"], a["k_ts"], a["k_hs"], a["v_ts"], a["v_hs"], a["heads"]) == (256, 64, 256, 64, 128, 64, 128, 64, 4)
    assert (a["q_weight"], a["k_weight"], a["weight_dtype"], a["eps"], a["token_seq"]) == (800, None, 0, 1e-5, None)
    # one product's rows
    a = be.ops.pagedAppend(cache, pos, _t(be, [3, 8 * 64], at=1000), None, None, out=_t(be, [3, 256], at=5000)) and _named(be.calls[-1])
    assert (a["q"], a["k"], a["v"], a["heads"], a["q_out"]) == (1000, 1000 + 256 * 2, 1000 + 384 * 2, 4, 5000)
    assert (a["q_ts"], a["k_ts"], a["v_ts"], a["q_hs"], a["k_hs"], a["v_hs"], a["o_ts"], a["o_hs"]) == (512, 512, 512, 64, 64, 64, 256, 64)
    # heads first, in place
    q = _t(be, [4, 3, 64], at=1000)
    assert be.ops.pagedAppend(cache, pos, q, _t(be, [2, 3, 64]), _t(be, [2, 3, 64]), headsFirst=True, out=q) is q
    a = _named(be.calls[-1])
    assert (a["q_ts"], a["q_hs"], a["o_ts"], a["o_hs"], a["k_ts"], a["k_hs"]) == (64, 192, 64, 192, 64, 192) and a["q_out"] == a["q"]
    # k and v alone
    assert be.ops.pagedAppend(cache, pos, None, k, v) is None
    a = _named(be.calls[-1])
    assert (a["q"], a["q_out"], a["heads"], a["cos"], a["rows"]) == (None, None, 0, None, 0)


def test_the_backend_refuses_what_does_not_fit(be):
    cache, pos = _paged(be), _t(be, [3], "i32")
    q, k, v, cos = _t(be, [3, 4, 64]), _t(be, [3, 2, 64]), _t(be, [3, 2, 64]), _t(be, [50, 32], "f32")
    out_of = [((cache, _t(be, [3], "f32"), q, k, v), {}), ((cache, pos, q, k, None), {}), ((cache, pos, q, None, None), {}),
              ((cache, pos, _t(be, [2, 4, 64]), k, v), {}), ((cache, pos, _t(be, [3, 4, 64], "f32"), k, v), {}), ((cache, pos, q, _t(be, [3, 3, 64]), v), {}),
              ((cache, pos, q, k, v, cos), {}), ((cache, pos, q, k, v, cos, _t(be, [50, 64], "f32")), {}),
              ((cache, pos, q, k, v, _t(be, [50, 32]), _t(be, [50, 32])), {}), ((cache, pos, q, k, v), dict(qNorm=_t(be, [32], "f32"))),
              ((cache, pos, q, k, v), dict(qNorm=_t(be, [64], "f32"), kNorm=_t(be, [64], "f16"))), ((cache, pos, q, k, v), dict(tokenSeq=_t(be, [2], "i32"))),
              ((cache, pos, q, k, v), dict(out=_t(be, [3, 3, 64]))), ((cache, pos, None, k, v), dict(out=q)),
              ((cache, pos, _t(be, [3, 4 * 64]), None, None), dict(headsFirst=True)), ((cache, pos, _t(be, [3, 4 * 64]), None, None), {}),
              ((cache, pos, None, None, None), {})]
    for args, more in out_of:
        with pytest.raises(tb.TlError):
            be.ops.pagedAppend(*args, **more)
    for args, more in [((cache, pos, _t(be, [3, 4, 32]), 0.1), {}), ((cache, pos, _t(be, [3, 4, 64], "bf16"), 0.1), {}),
                       ((cache, pos, q, 0.1), dict(slopes=_t(be, [3], "f32"))), ((cache, pos, q, 0.1), dict(slopes=_t(be, [4]))),
                       ((cache, pos, q, 0.1), dict(out=_t(be, [3, 128]))), ((cache, _t(be, [3, 1], "i32"), q, 0.1), {})]:
        with pytest.raises(tb.TlError):
            be.ops.pagedAttention(*args, **more)
    logits, u = _t(be, [2, 100], "f32"), _t(be, [2], "f32")
    for args, more in [((logits, _t(be, [3], "f32")), {}), ((logits, u), dict(topK=u)), ((logits, u), dict(topP=_t(be, [1], "f32"))),
                       ((_t(be, [2, 100], "u32"), u), {}), ((logits, u), dict(out=u)), ((_t(be, [2, 100], "f32", transposed=True), u), {})]:
        with pytest.raises(tb.TlError):
            be.ops.sample(*args, **more)
    assert not [c for c in be.calls if c[0] != "tl_alloc"]


def test_attention_and_sample_hand_over(be):
    cache, pos = _paged(be), _t(be, [3], "i32", 500)
    y = be.ops.pagedAttention(cache, pos, _t(be, [3, 256], at=1000), 0.25, softcap=30.0, window=7, slopes=_t(be, [4], "f32", 900), tokenSeq=_t(be, [3], "i32", 950))
    assert y.shape == [3, 256] and be.calls[-1] == ("tl_paged_attention", 8, cache.descriptor(), 500, 950, 3, 1000, 256, 64, 4, 4096, 0.25, 30.0, 7, 900)
    y = be.ops.sample(_t(be, [1, 2, 100], "bf16", 1000), _t(be, [2], "f32", 20), topK=_t(be, [2], "i32", 30), minP=_t(be, [2], "f32", 40))
    assert y.shape == [2] and y.dtype == "i32" and be.calls[-1] == ("tl_sample", 8, 1000, B.TL_BF16, 2, 100, 100, None, 30, None, 40, 20, 4096)
