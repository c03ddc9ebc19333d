"""Appending to a paged cache and attention over it, against the same in 64 bits; what must stay untouched does, bit for bit.

Tolerances.  A stored value is off by half a step of its type at most (2^-11 of it in f16, 2^-8 in bf16, 2^-24 in f32, and 2^-25 below f16's normal numbers)
on top of what f32 arithmetic leaves:
  append     y = a c - b s with a = x w / sqrt(mean(x^2) + eps).  A sum of D squares by lanes of at least D / 32 in a chain: relative error of the mean at most
             (D / 32 + 7) 2^-24, half of that of its root, and about a dozen roundings after it: (D / 64 + 16) 2^-24 (|a c| + |b s|).
  attention  a score x is off by dx = c 2^-24 scale sum|q k| with c the roundings of one dot product (f32: D / 32 + 8; on the tensor cores 4 for each 16 products,
             whose sum keeps at least 22 bits of the largest), tanh and the bias by a few of their own; exp of a difference d by (2 + |d|) 2^-23, and
             the two sums over n keys by n 2^-24: relative to sum(p |v|) the output is off by 2 dx + (2 + max|d|) 2^-22 + 2 n 2^-24.  A probability in
             two or three 16-bit terms keeps 22 bits: 2^-22 more."""
import numpy as np
import pytest
import torch

from torchlette_b200 import backend as tb
from torchlette_b200 import binding as B

pytestmark = pytest.mark.gpu

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i32": torch.int32}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"f32": 2.0 ** -140, "f16": 2.0 ** -25, "bf16": 2.0 ** -130}
JUNK = 1 << 30  # in a page table: not a page


def wrap(be, t, dtype=None):
    names = {v: k for k, v in TORCH.items()}
    return tb.CudaTensor(be, list(t.shape), dtype or names[t.dtype], t.data_ptr(), t.numel() * t.element_size(), ownsBuffer=False)


def normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(TORCH[dtype])


class Cache:
    """Pages in random order for sequences with `room` positions each, full of NaN; the table holds junk behind a sequence's last page."""

    def __init__(self, be, gen, room, kv_heads, dim, page, dtype, spare=2):
        self.page, self.kv_heads, self.dim = page, kv_heads, dim
        counts = [-(-n // page) for n in room]
        pages = sum(counts) + spare
        order = torch.randperm(pages, generator=gen, device="cuda").tolist()
        self.table = torch.full((len(room), max(counts + [1]) + 1), JUNK, dtype=torch.int32)
        for i, c in enumerate(counts):
            for j in range(c):
                self.table[i, j] = order.pop()
        self.table = self.table.cuda()
        self.k = torch.full((pages, kv_heads, page, dim), float("nan"), device="cuda", dtype=TORCH[dtype])
        self.v = self.k.clone()
        self.tensors = [wrap(be, t) for t in (self.k, self.v, self.table)]
        self.cache = be.createPagedCache(*self.tensors)

    def rows(self, seq, n):
        """Pages and slots of a sequence's first n positions."""
        at = torch.arange(n, device="cuda")
        return self.table[seq, at // self.page].long(), at % self.page

    def fill(self, gen, seq, n, dtype, scale=1.0):
        page, slot = self.rows(seq, n)
        self.k[page, :, slot] = normal(gen, (n, self.kv_heads, self.dim), dtype, scale)
        self.v[page, :, slot] = normal(gen, (n, self.kv_heads, self.dim), dtype)


def assert_close(got, ref, slack, dtype):
    got, ref = got.double(), ref.double()
    off = (got - ref).abs()
    allowed = HALF_STEP[dtype] * (ref.abs() + slack) + slack + LEAST[dtype]
    bad = ~(off <= allowed)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, the worst {float((off / allowed)[bad].nan_to_num(nan=1e9).max()):.3g} times what is allowed"


# ---------------------------------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------------------------------

def turned(x, weight, eps, cos, sin):
    """[T, heads, D] in 64 bits, and |a c| + |b s|."""
    x = x.double()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    if cos is None:
        return x, x.abs()
    a, b = x.chunk(2, -1)
    c, s = cos.double()[:, None], sin.double()[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], -1), torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], -1)


# new tokens: (sequence, position); a negative position is a token that is not there
STEP = [(0, 0), (1, 15), (2, 16), (3, -1), (4, 31), (5, 40)]
PROMPTS = [(2, p) for p in range(3, 40)] + [(0, p) for p in range(17)] + [(1, -5)] + [(4, 6)]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 2, 128, 16), (7, 1, 64, 16), (3, 3, 80, 5), (2, 1, 256, 1), (8, 4, 32, 64), (5, 5, 6, 7), (2, 2, 1024, 3),
                                                     (4, 2, 16, 16), (4, 1, 112, 16)])
@pytest.mark.parametrize("form", ["step", "fused", "prompts", "heads_first", "in_place", "plain", "k_and_v"])
def test_append(backend, dtype, heads, kv_heads, dim, page, form):
    be, eps = backend, 1e-5
    gen = torch.Generator(device="cuda").manual_seed(heads * 1000 + dim + page)
    tokens = STEP if form in ("step", "fused") else PROMPTS
    t = len(tokens)
    c = Cache(be, gen, [41] * 6, kv_heads, dim, page, dtype)
    pos = torch.tensor([p for _, p in tokens], dtype=torch.int32, device="cuda")
    seq = torch.tensor([s for s, _ in tokens], dtype=torch.int32, device="cuda")
    qkv = normal(gen, (t, heads + 2 * kv_heads, dim), dtype, 2.0)
    q, k, v = (x.contiguous() for x in qkv.split([heads, kv_heads, kv_heads], 1))
    angle = torch.arange(41, device="cuda")[:, None] / 1e4 ** (torch.arange(dim // 2, device="cuda") / (dim // 2))
    cos, sin = angle.cos().contiguous(), angle.sin().contiguous()
    weights = [1 + normal(gen, (dim,), "f32", 0.3) for _ in range(2)]
    if dtype == "bf16":
        weights = [w.bfloat16() for w in weights]
    more = {} if form == "plain" else {"qNorm": wrap(be, weights[0]), "kNorm": wrap(be, weights[1]), "eps": eps}
    if form == "plain":
        weights, cos, sin = [None, None], None, None
    if form == "k_and_v":
        weights[0] = None
        del more["qNorm"]
    rope = (wrap(be, cos), wrap(be, sin)) if cos is not None else (None, None)
    if form not in ("step", "fused"):
        more["tokenSeq"] = wrap(be, seq)
    out = torch.full((t, heads, dim), 7.0, device="cuda", dtype=TORCH[dtype])
    before = c.k.clone()
    order = (lambda x: x.transpose(0, 1).contiguous()) if form == "heads_first" else lambda x: x
    held = [order(x) for x in (q, k, v)]
    if form == "heads_first":
        out = order(out)
        more["headsFirst"] = True
    if form == "in_place":
        out = held[0]
        q = q.clone()
    args = [wrap(be, x) for x in held]
    if form == "fused":
        args = [wrap(be, qkv.view(t, -1)), None, None]
    if form == "k_and_v":
        args[0] = None
    else:
        more["out"] = wrap(be, out)
    torch.cuda.synchronize()
    result = be.ops.pagedAppend(c.cache, wrap(be, pos), *args, *rope, **more)
    be.sync()
    assert (result is None) == (form == "k_and_v")
    here = pos >= 0
    at = pos.clamp(min=0).long()
    slack = (dim / 64 + 16) * 2.0 ** -24
    turn = lambda x, w: turned(x, w, eps, cos[at] if cos is not None else None, sin[at] if sin is not None else None)  # noqa: E731
    if form != "k_and_v":
        y, mag = turn(q, weights[0])
        got = order(out) if form == "heads_first" else out
        assert_close(got[here], y[here], slack * mag[here], dtype)
        kept = q if form == "in_place" else torch.full_like(q, 7.0)
        assert torch.equal(got[~here], kept[~here]), "a token that is not there was written"
    y, mag = turn(k, weights[1])
    page_at, slot = c.table[seq.long(), at // page].long(), at % page
    assert_close(c.k[page_at, :, slot][here], y[here], slack * mag[here], dtype)
    assert torch.equal(c.v[page_at, :, slot][here], v[here])
    for pages in (c.k, c.v):  # all else is as it was
        pages[page_at[here], :, slot[here]] = float("nan")
        assert torch.equal(pages.view(torch.int16 if dtype != "f32" else torch.int32), before.view(torch.int16 if dtype != "f32" else torch.int32))


def test_append_to_a_contiguous_cache_serves_decode_attention(backend):
    """[B, kvH, capacity, D] as pages of `capacity`: three steps against decodeAttention over the same tensors."""
    be, b, g, cap, d, h = backend, 3, 2, 20, 64, 4
    gen = torch.Generator(device="cuda").manual_seed(5)
    k, v = torch.zeros(b, g, cap, d, device="cuda", dtype=torch.float16), torch.zeros(b, g, cap, d, device="cuda", dtype=torch.float16)
    table = torch.arange(b, dtype=torch.int32, device="cuda")[:, None].contiguous()
    kt, vt = wrap(be, k), wrap(be, v)
    cache = be.createPagedCache(kt, vt, wrap(be, table))
    for step in range(3):
        q, kn, vn = (normal(gen, (b, n, d), "f16") for n in (h, g, g))
        pos = torch.full((b,), step, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        qr = be.ops.pagedAppend(cache, wrap(be, pos), wrap(be, q), wrap(be, kn), wrap(be, vn))
        one = be.ops.decodeAttention(be.ops.reshape(qr, [b, h, 1, d]), kt, vt, step + 1, 0.125)
        two = be.ops.pagedAttention(cache, wrap(be, pos), qr, 0.125)
        be.sync()
        assert torch.equal(k[:, :, step], kn) and torch.equal(v[:, :, step], vn)
        np.testing.assert_allclose(np.float64(be.ops.read(two)), np.float64(be.ops.read(one)).reshape(b, h * d), rtol=2 * 2.0 ** -11 + 1e-4, atol=1e-4)
        for t in (qr, one, two):
            t.destroy()


# ---------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------

def attention_ref(c, q, pos, seq, scale, softcap=0.0, window=0, slopes=None, dtype="f16"):
    """[T, H, D] in 64 bits and what may be off."""
    t, h, d = q.shape
    rep = h // c.kv_heads
    out, slack = torch.zeros(t, h, d, dtype=torch.float64, device="cuda"), torch.zeros(t, h, 1, dtype=torch.float64, device="cuda")
    slack = slack.expand(t, h, d).clone()
    for i in range(t):
        p = int(pos[i])
        if p < 0:
            continue
        lo = max(0, p + 1 - window) if window else 0
        page, slot = c.rows(int(seq[i]), p + 1)
        k, v = (x[page, :, slot][lo:].double().repeat_interleave(rep, 1) for x in (c.k, c.v))  # [n, H, D]
        qd = q[i].double()
        x = torch.einsum("hd,jhd->hj", qd, k) * scale
        mag = torch.einsum("hd,jhd->hj", qd.abs(), k.abs()).amax(1, keepdim=True) * abs(scale)
        roundings = d / 32 + 8 if dtype == "f32" else d / 16 * 4
        dx = roundings * 2.0 ** -24 * mag
        if softcap:
            x = softcap * torch.tanh(x / softcap)
            dx = dx + 8 * 2.0 ** -24 * softcap
        if slopes is not None:
            bias = slopes.double()[:, None] * (torch.arange(lo, p + 1, device="cuda") - p)
            dx = dx + 4 * 2.0 ** -24 * (bias.abs().amax(1, keepdim=True) + x.abs().amax(1, keepdim=True))
            x = x + bias
        top = x.amax(1, keepdim=True)
        w = torch.exp(x - top)
        w = w / w.sum(1, keepdim=True)
        # keys whose probability is below 2^-30 of the largest carry nothing
        spread = (top - x).clamp(max=21.0).amax(1, keepdim=True)
        out[i] = torch.einsum("hj,jhd->hd", w, v)
        rel = 2 * dx + (2 + spread) * 2.0 ** -22 + 2 * (p + 1 - lo) * 2.0 ** -24 + 2.0 ** -22
        slack[i] = rel * torch.einsum("hj,jhd->hd", w, v.abs())
    return out, slack


def run_attention(be, c, q, pos, seq, scale, **more):
    t, h, d = q.shape
    out = torch.full((t + 2, h * d), 9.0, device="cuda", dtype=q.dtype)
    slopes = more.pop("slopes", None)
    if slopes is not None:
        more["slopes"] = wrap(be, slopes)
    if seq is not None:
        more["tokenSeq"] = wrap(be, seq)
    torch.cuda.synchronize()
    be.ops.pagedAttention(c.cache, wrap(be, pos), wrap(be, q), scale, out=wrap(be, out[1:-1]), **more)
    be.sync()
    assert (out[0] == 9.0).all() and (out[-1] == 9.0).all()
    return out[1:-1].view(t, h, d)


OPTIONS = [{}, {"window": 1}, {"window": 19}, {"softcap": 5.0}, {"slopes": True}, {"softcap": 3.0, "window": 33, "slopes": True}]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 2, 128, 16), (4, 4, 64, 16), (9, 3, 80, 5), (24, 1, 128, 64), (2, 1, 256, 1), (16, 8, 128, 48), (3, 1, 8, 16),
                                                     (40, 2, 64, 16), (5, 1, 192, 24), (20, 1, 256, 16)])
@pytest.mark.parametrize("options", OPTIONS, ids=lambda o: "+".join(o) or "plain")
def test_attention(backend, dtype, heads, kv_heads, dim, page, options):
    be, options = backend, dict(options)
    gen = torch.Generator(device="cuda").manual_seed(dim + heads)
    lengths = [1, 2, 15, 16, 17, 31, 0, 63, 64, 65, 200, 333, 0, 1000]
    c = Cache(be, gen, lengths, kv_heads, dim, page, dtype)
    for i, n in enumerate(lengths):
        c.fill(gen, i, n, dtype)
    q = normal(gen, (len(lengths), heads, dim), dtype)
    pos = torch.tensor(lengths, dtype=torch.int32, device="cuda") - 1
    if "slopes" in options:
        options["slopes"] = torch.rand(heads, generator=gen, device="cuda")
    scale = 1.3 / dim ** 0.5
    got = run_attention(be, c, q, pos, None, scale, **options)
    ref, slack = attention_ref(c, q, pos, range(len(lengths)), scale, dtype=dtype, **options)
    assert_close(got, ref, slack, dtype)
    assert (got[pos < 0] == 0).all()
    assert torch.equal(got, run_attention(be, c, q, pos, None, scale, **options)), "two runs differ"


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attention_of_several_tokens_of_a_sequence(backend, dtype):
    """A prompt's last tokens and other sequences' in one call, in any order."""
    be = backend
    gen = torch.Generator(device="cuda").manual_seed(11)
    c = Cache(be, gen, [100, 7, 300], 2, 64, 16, dtype)
    for i, n in enumerate([100, 7, 300]):
        c.fill(gen, i, n, dtype)
    tokens = [(2, 299), (0, 0), (2, 298), (1, 6), (2, 10), (0, 99), (0, -1), (2, 299), (0, 98)]
    seq, pos = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in zip(*tokens))
    q = normal(gen, (len(tokens), 6, 64), dtype)
    q[7] = q[0]
    got = run_attention(be, c, q, pos, seq, 0.125)
    ref, slack = attention_ref(c, q, pos, seq.tolist(), 0.125, dtype=dtype)
    assert_close(got, ref, slack, dtype)


@pytest.mark.parametrize("dtype,dim,heads,kv_heads,page,lengths", [
    ("bf16", 128, 16, 2, 64, [20_011]), ("f16", 128, 8, 1, 16, [70_001]), ("f16", 64, 32, 8, 16, [4000, 1, 3900, 17, 0, 2500, 4001, 33]),
    ("bf16", 128, 4, 4, 128, [1 + (i * 37) % 150 for i in range(300)]), ("f32", 128, 8, 2, 16, [9000, 5]), ("f16", 256, 8, 4, 16, [3000, 2999, 64])])
def test_attention_long_and_many(backend, dtype, dim, heads, kv_heads, page, lengths):
    be = backend
    gen = torch.Generator(device="cuda").manual_seed(dim + len(lengths))
    c = Cache(be, gen, lengths, kv_heads, dim, page, dtype)
    for i, n in enumerate(lengths):
        c.fill(gen, i, n, dtype, 2.0)  # some probabilities stand out
    q = normal(gen, (len(lengths), heads, dim), dtype)
    pos = torch.tensor(lengths, dtype=torch.int32, device="cuda") - 1
    got = run_attention(be, c, q, pos, None, dim ** -0.5)
    ref, slack = attention_ref(c, q, pos, range(len(lengths)), dim ** -0.5, dtype=dtype)
    assert_close(got, ref, slack, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_attention_infinite_and_nan_values(backend, dtype):
    """NaN lies in every slot that no token sees (Cache); here visible values are infinite, and one sequence's NaN stays its own."""
    be = backend
    gen = torch.Generator(device="cuda").manual_seed(3)
    lengths = [40, 50, 60]
    c = Cache(be, gen, lengths, 1, 64, 16, dtype)
    for i, n in enumerate(lengths):
        c.fill(gen, i, n, dtype)
    page, slot = c.rows(0, 40)
    c.v[page[5], 0, slot[5], 3] = float("inf")
    c.v[page[9], 0, slot[9], 7] = -float("inf")
    page, slot = c.rows(1, 50)
    c.v[page[8], 0, slot[8], 2] = float("nan")
    q = normal(gen, (3, 2, 64), dtype)
    pos = torch.tensor(lengths, dtype=torch.int32, device="cuda") - 1
    got = run_attention(be, c, q, pos, None, 0.125)
    ref, slack = attention_ref(c, q, pos, range(3), 0.125, dtype=dtype)
    assert (got[0, :, 3] == float("inf")).all() and (got[0, :, 7] == -float("inf")).all() and got[1, :, 2].isnan().all()
    fine = ref.isfinite()
    assert torch.equal(got.isfinite(), fine)
    assert_close(got[fine], ref[fine], slack[fine], dtype)


def test_attention_reads_strided_queries(backend):
    be = backend
    gen = torch.Generator(device="cuda").manual_seed(4)
    c = Cache(be, gen, [30, 77], 2, 64, 16, "bf16")
    for i, n in enumerate([30, 77]):
        c.fill(gen, i, n, "bf16")
    rows = normal(gen, (2, 4 + 2 * 2, 64), "bf16")  # of a fused product
    q = rows[:, :4]
    pos = torch.tensor([29, 76], dtype=torch.int32, device="cuda")
    out = torch.empty(2, 4, 64, device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    B.check(be._ctx, be._lib.tl_paged_attention(be._ctx, B.PagedCache.from_buffer_copy(c.cache.descriptor()), pos.data_ptr(), None, 2, rows.data_ptr(), 8 * 64, 64, 4,
                                                out.data_ptr(), 0.125, 0.0, 0, None))
    be.sync()
    ref, slack = attention_ref(c, q, pos, [0, 1], 0.125, dtype="bf16")
    assert_close(out, ref, slack, "bf16")


@pytest.mark.parametrize("page", [16, 5])
def test_indexes_out_of_range_are_skipped_and_reported(page):
    """Positions, sequences and pages that are not there: no memory is touched, the other tokens are right, the next sync says so, once."""
    be = tb.CudaBackend(0)  # its error count is its own
    try:
        _out_of_range(be, page)
    finally:
        be.destroy()


def _out_of_range(be, page_size):
    gen = torch.Generator(device="cuda").manual_seed(6)
    c = Cache(be, gen, [40, 40, 40, 40], 2, 64, page_size, "f16")
    for i in range(4):
        c.fill(gen, i, 40, "f16")
    room = c.table.shape[1] * page_size
    q, k, v = (normal(gen, (4, n, 64), "f16") for n in (4, 2, 2))
    cos = torch.ones(60, 32, device="cuda")
    errors = be.getGpuUncapturedErrorCount()
    for pos, seq, word in (([39, room, 5, 39], [0, 1, 2, 3], "position"), ([39, 2 ** 31 - 1, 5, 39], [0, 1, 2, 3], "position"),
                           ([39, 5, 5, 39], [0, 4, 2, 3], "sequence"), ([39, 5, 5, 39], [0, -1, 2, 3], "sequence"),
                           ([39, room - 1, 5, 39], [0, 1, 2, 3], "page")):  # the last page of the table is junk
        p, s = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (pos, seq))
        before = c.k.clone(), c.v.clone()
        out = torch.full((4, 4, 64), 7.0, device="cuda", dtype=torch.float16)
        torch.cuda.synchronize()
        be.ops.pagedAppend(c.cache, wrap(be, p), wrap(be, q), wrap(be, k), wrap(be, v), wrap(be, cos), wrap(be, cos), tokenSeq=wrap(be, s), out=wrap(be, out))
        with pytest.raises(tb.TlError, match=word) as e:
            be.sync()
        assert e.value.status == B.TL_ERR_INVALID_ARG
        be.sync()
        for i in (0, 2, 3):
            page, slot = c.rows(i, 40)
            assert torch.equal(c.v[page[pos[i]], :, slot[pos[i]]], v[i])
            for now, then in zip((c.k, c.v), before):
                now[page[pos[i]], :, slot[pos[i]]] = then[page[pos[i]], :, slot[pos[i]]]
        for now, then in zip((c.k, c.v), before):
            assert torch.equal(now.view(torch.int16), then.view(torch.int16))
        if word != "page":
            assert (out[1] == 7.0).all()
        y = torch.full((4, 256), 7.0, device="cuda", dtype=torch.float16)
        torch.cuda.synchronize()
        be.ops.pagedAttention(c.cache, wrap(be, p), wrap(be, q), 0.125, tokenSeq=wrap(be, s), out=wrap(be, y))
        with pytest.raises(tb.TlError, match=word):
            be.sync()
        be.sync()
        keep = [0, 2, 3]
        ref, slack = attention_ref(c, q[keep], p[keep], [seq[i] for i in keep], 0.125)
        assert_close(y.view(4, 4, 64)[keep], ref, slack, "f16")
        if word != "page":
            assert (y[1] == 0).all()
    assert be.getGpuUncapturedErrorCount() == errors + 10


def test_a_page_of_the_past_that_is_not_there(backend_of_its_own):
    """Its keys do not count, the others do: the same as attention over them alone."""
    be = backend_of_its_own
    gen = torch.Generator(device="cuda").manual_seed(9)
    for page_size, dtype in ((16, "bf16"), (7, "bf16"), (8, "f32")):
        c = Cache(be, gen, [100], 2, 64, page_size, dtype)
        c.fill(gen, 0, 100, dtype)
        q, pos = normal(gen, (1, 4, 64), dtype), torch.tensor([99], dtype=torch.int32, device="cuda")
        c.table[0, 2] = JUNK
        out = torch.empty(1, 256, device="cuda", dtype=TORCH[dtype])
        torch.cuda.synchronize()
        be.ops.pagedAttention(c.cache, wrap(be, pos), wrap(be, q), 0.125, out=wrap(be, out))
        with pytest.raises(tb.TlError, match="page"):
            be.sync()
        at = torch.cat([torch.arange(2 * page_size), torch.arange(3 * page_size, 100)]).cuda()
        k, v = (x[c.table[0, at // page_size].long(), :, at % page_size].double().repeat_interleave(2, 1) for x in (c.k, c.v))
        w = torch.softmax(torch.einsum("hd,jhd->hj", q[0].double(), k) * 0.125, 1)
        ref = torch.einsum("hj,jhd->hd", w, v)
        assert_close(out.view(4, 64), ref, torch.full_like(ref, 2e-4), dtype)
        c.table[:] = JUNK  # none is there
        torch.cuda.synchronize()
        be.ops.pagedAttention(c.cache, wrap(be, pos), wrap(be, q), 0.125, out=wrap(be, out))
        with pytest.raises(tb.TlError, match="page"):
            be.sync()
        assert (out == 0).all()


@pytest.fixture
def backend_of_its_own():
    be = tb.CudaBackend(0)  # its error count and scratch are its own
    yield be
    be.destroy()


def test_a_first_call_in_a_capture_is_refused(backend_of_its_own):
    be = backend_of_its_own
    gen = torch.Generator(device="cuda").manual_seed(10)
    c = Cache(be, gen, [20], 1, 64, 16, "f16")
    c.fill(gen, 0, 20, "f16")
    q, pos, out = normal(gen, (1, 2, 64), "f16"), torch.tensor([19], dtype=torch.int32, device="cuda"), torch.zeros(1, 128, device="cuda", dtype=torch.float16)
    torch.cuda.synchronize()
    call = lambda: be.ops.pagedAttention(c.cache, wrap(be, pos), wrap(be, q), 0.125, out=wrap(be, out))  # noqa: E731
    be.beginCapture()
    with pytest.raises(tb.TlError, match="before capturing") as e:
        call()
    assert e.value.status == B.TL_ERR_UNSUPPORTED
    be.destroyGraph(be.endCapture())
    call()
    be.sync()
    be.beginCapture()
    call()
    graph = be.endCapture()
    out.zero_()
    torch.cuda.synchronize()
    be.replay(graph)
    be.sync()
    ref, slack = attention_ref(c, q, pos, [0], 0.125)
    assert_close(out.view(1, 2, 64), ref, slack, "f16")
    be.destroyGraph(graph)


@pytest.mark.parametrize("page", [16, 6])
def test_a_cache_past_32_bits(backend, page):
    """Pages behind the 2^31st element, and the 2^32nd byte: append there and attention over it."""
    be, g, d = backend, 8, 128
    gen = torch.Generator(device="cuda").manual_seed(12)
    pages = 2 ** 31 // (g * page * d) + 40
    k, v = (torch.empty(pages, g, page, d, device="cuda", dtype=torch.float16) for _ in range(2))
    n = 5 * page + 3
    table = torch.arange(pages - 1, pages - 7, -1, dtype=torch.int32, device="cuda")[None].contiguous()
    tensors = [wrap(be, k), wrap(be, v), wrap(be, table)]
    cache = be.createPagedCache(*tensors)
    kn, vn, q = normal(gen, (n, g, d), "f16"), normal(gen, (n, g, d), "f16"), normal(gen, (1, 16, d), "f16")
    pos, seq = torch.arange(n, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    be.ops.pagedAppend(cache, wrap(be, pos), None, wrap(be, kn), wrap(be, vn), tokenSeq=wrap(be, seq))
    out = be.ops.pagedAttention(cache, wrap(be, pos[-1:]), wrap(be, q), 0.09)
    be.sync()
    at = torch.arange(n, device="cuda")
    assert torch.equal(k[table[0, at // page].long(), :, at % page], kn) and torch.equal(v[table[0, at // page].long(), :, at % page], vn)
    w = torch.softmax(torch.einsum("hd,jhd->hj", q[0].double(), kn.double().repeat_interleave(2, 1)) * 0.09, 1)
    ref = torch.einsum("hj,jhd->hd", w, vn.double().repeat_interleave(2, 1))
    got = torch.from_numpy(np.float64(be.ops.read(out))).cuda().view(16, d)
    assert_close(got, ref, torch.full_like(ref, 1e-4), "f16")
    out.destroy()


def test_a_captured_step_replays_with_new_positions(backend):
    """append and attention in one graph: positions, tokens and the page table change between replays."""
    be = backend
    gen = torch.Generator(device="cuda").manual_seed(8)
    c = Cache(be, gen, [90, 90, 90], 2, 128, 16, "bf16")
    q, k, v = (torch.zeros(3, n, 128, device="cuda", dtype=torch.bfloat16) for n in (4, 2, 2))
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    qo, out = torch.zeros_like(q), torch.zeros(3, 512, device="cuda", dtype=torch.bfloat16)

    def step():
        be.ops.pagedAppend(c.cache, wrap(be, pos), wrap(be, q), wrap(be, k), wrap(be, v), out=wrap(be, qo))
        be.ops.pagedAttention(c.cache, wrap(be, pos), wrap(be, qo), 0.1, out=wrap(be, out))

    torch.cuda.synchronize()
    step()
    be.sync()
    graphs = []
    for _ in range(2):  # two graphs of the same call, replayed in turn
        be.beginCapture()
        step()
        graphs.append(be.endCapture())
    for n in range(40):
        for x in (q, k, v):
            x.copy_(normal(gen, x.shape, "bf16"))
        pos.copy_(torch.tensor([n, n if n < 20 else -1, 2 * n], dtype=torch.int32))
        if n == 30:  # the sequences change places
            c.table.copy_(c.table[[2, 1, 0]].clone())
            break
        if n and 2 * n > 1:
            page, slot = c.rows(2, 2 * n)
            c.k[page[2 * n - 1], :, slot[2 * n - 1]] = c.v[page[2 * n - 1], :, slot[2 * n - 1]] = normal(gen, (2, 128), "bf16")
        torch.cuda.synchronize()
        be.replay(graphs[n % 2])
        be.sync()
        ref, slack = attention_ref(c, q, pos, range(3), 0.1, dtype="bf16")
        assert_close(out.view(3, 4, 128), ref, slack, "bf16")
    pos.copy_(torch.tensor([59, -1, 30], dtype=torch.int32))
    torch.cuda.synchronize()
    be.replay(graphs[0])
    be.sync()
    ref, slack = attention_ref(c, q, pos, range(3), 0.1, dtype="bf16")
    assert_close(out.view(3, 4, 128), ref, slack, "bf16")
    for g in graphs:
        be.destroyGraph(g)
