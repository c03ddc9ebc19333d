"""Infinite and NaN values that a token sees, in paged attention: what the definition makes of them, wherever they lie in a split sequence, in about the time of a
finite call."""
import ctypes as C

import pytest
import torch

from test_gpu_paged import OPTIONS, Cache, assert_close, attention_ref, normal, run_attention, wrap
from test_gpu_paged_scores import reference
from torchlette_b200 import binding as B

pytestmark = pytest.mark.gpu
INF = float("inf")


def compare(got, ref, slack, dtype):
    for kind in (torch.isnan, torch.isposinf, torch.isneginf):
        wrong = kind(got) != kind(ref)
        assert not wrong.any(), f"{kind.__name__}: {int(kind(got).sum())} for {int(kind(ref).sum())}, first at {wrong.nonzero()[0].tolist()}"
    fine = ref.isfinite()
    assert_close(got[fine], ref[fine], slack[fine], dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 2, 128, 16), (24, 1, 64, 5), (3, 3, 80, 16), (9, 1, 256, 16), (2, 1, 8, 16)])
def test_values_anywhere(backend, dtype, heads, kv_heads, dim, page):
    """Short sequences, ones of a few tiles and ones over many CTAs: an infinity, both of them in one dimension, a NaN, a whole row of infinities."""
    gen = torch.Generator(device="cuda").manual_seed(dim + page)
    lengths = [1, 7, 40, 90, 3000, 260, 33, 2500, 64, 700, 17]
    c = Cache(backend, gen, lengths, kv_heads, dim, page, dtype)
    for i, n in enumerate(lengths):
        c.fill(gen, i, n, dtype)
        rows, slots = c.rows(i, n)
        put = lambda at, d, x: c.v.__setitem__((rows[at], i % kv_heads, slots[at], d), x)  # noqa: E731
        put(n // 2, 1, INF)
        put(n - 1, 2, -INF)
        if i in (2, 4, 5, 9):
            put(0, 3, INF)
            put(n // 3 + 1, 3, -INF)
            put(n // 5, 5, float("nan"))
        if i in (6, 7):
            put(n // 4, slice(None), -INF)
    q = normal(gen, (len(lengths), heads, dim), dtype)
    pos = torch.tensor(lengths, dtype=torch.int32, device="cuda") - 1
    got = run_attention(backend, c, q, pos, None, dim ** -0.5)
    compare(got, *reference(c, q, lengths, dim ** -0.5), dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_values_behind_small_and_no_probabilities(backend, dtype):
    """An infinite value of a key with e^-60 of the largest probability counts; one whose score is -infinity is zero times infinity."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    lengths = [100, 1000]
    c = Cache(backend, gen, lengths, 1, 64, 16, dtype)
    q = torch.zeros(2, 1, 64, device="cuda", dtype=c.k.dtype)
    q[:, 0, 0] = 8.0
    for i, n in enumerate(lengths):
        c.fill(gen, i, n, dtype)
        rows, slots = c.rows(i, n)
        c.k[rows, 0, slots, 0] = 0.0
        c.k[rows[50], 0, slots[50], 0] = -60.0
        c.v[rows[50], 0, slots[50], 4] = INF
        c.k[rows[60], 0, slots[60], 0] = -INF
        c.v[rows[60], 0, slots[60], 5] = INF
    pos = torch.tensor(lengths, dtype=torch.int32, device="cuda") - 1
    got = run_attention(backend, c, q, pos, None, 0.125)
    ref, slack = reference(c, q, lengths, 0.125)
    assert ref[:, 0, 4].isposinf().all() and ref[:, 0, 5].isnan().all()
    compare(got, ref, slack, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("page", [16, 7])
@pytest.mark.parametrize("options", OPTIONS[1:], ids="+".join)
def test_values_under_options(backend, dtype, page, options):
    """Windows that see an infinity or no longer do, caps and biases, several tokens of a sequence."""
    gen, options = torch.Generator(device="cuda").manual_seed(page), dict(options)
    lengths = [400, 1200, 20]
    c = Cache(backend, gen, lengths, 2, 128, page, dtype)
    for i, n in enumerate(lengths):
        c.fill(gen, i, n, dtype)
        rows, slots = c.rows(i, n)
        c.v[rows[n - 10], i % 2, slots[n - 10], 100] = INF
        c.v[rows[n - 16], i % 2, slots[n - 16], 100] = -INF
        c.v[rows[n // 2], 0, slots[n // 2], 31] = -INF
    tokens = [(0, 399), (1, 1199), (2, 19), (0, 388), (0, 395), (1, 615), (1, -1), (2, 3), (1, 300)]
    seq, pos = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in zip(*tokens))
    q = normal(gen, (len(tokens), 12, 128), dtype)
    if "slopes" in options:
        options["slopes"] = torch.rand(12, generator=gen, device="cuda") / 20
    got = run_attention(backend, c, q, pos, seq, 0.09, **options)
    ref, slack = attention_ref(c, q, pos, seq.tolist(), 0.09, dtype=dtype, **options)
    assert ref.isinf().any() or options == {"window": 1}
    compare(got, ref, slack, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_a_call_with_infinities_takes_no_longer_than_a_few(backend, dtype):
    """One infinity and one NaN in each of 6 x 4 000 keys: one pass more over the values, not two over the keys for every 32 dimensions of every row."""
    be = backend
    gen = torch.Generator(device="cuda").manual_seed(3)
    lengths = [4000] * 6
    c = Cache(be, gen, lengths, 2, 128, 16, dtype)
    for i, n in enumerate(lengths):
        c.fill(gen, i, n, dtype)
    q = normal(gen, (6, 8, 128), dtype)
    pos = torch.tensor(lengths, dtype=torch.int32, device="cuda") - 1
    out = torch.empty(6, 1024, device="cuda", dtype=q.dtype)

    def took():
        times, stream = [], C.c_void_p()
        B.check(be._ctx, be._lib.tl_ctx_stream(be._ctx, C.byref(stream)))
        with torch.cuda.stream(torch.cuda.ExternalStream(stream.value)):
            for _ in range(4):
                ends = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
                ends[0].record()
                be.ops.pagedAttention(c.cache, wrap(be, pos), wrap(be, q), 0.09, out=wrap(be, out))
                ends[1].record()
                be.sync()
                times.append(ends[0].elapsed_time(ends[1]))
        return min(times)

    torch.cuda.synchronize()
    plain = took()
    for i, n in enumerate(lengths):
        rows, slots = c.rows(i, n)
        c.v[rows[n // 2], 0, slots[n // 2], 70] = INF
        c.v[rows[n // 3], 1, slots[n // 3], 9] = float("nan")
    torch.cuda.synchronize()
    odd = took()
    compare(out.view(6, 8, 128), *reference(c, q, lengths, 0.09), dtype)
    assert odd < 1.0, f"{odd:.2f} ms against {plain:.3f} for finite values"
