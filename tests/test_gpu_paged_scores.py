"""Paged attention's scores at the ends of their range: soft caps of any size, scores that are no numbers or infinite.

Tolerance with a cap, over what tests/test_gpu_paged.py derives for plain scores (dx for a dot product, then 2 dx + (2 + spread) 2^-22 + 2 n 2^-24 + 2^-22 of
sum p |v|).  c tanh(x / c) has two forms in 16-bit types.  Near zero, x times an even polynomial of x / c: two roundings of x / c, which reach the polynomial
through a term of at most .02, one of the polynomial, one of the product: below 4 x 2^-24 |x|.  From |x / c| = 1/4 on, c (1 - 2 / (1 + t)) with t = e^(2x / c):
t is off by 2^-22 and by 2 |x / c| 2^-23 of itself, which reaches 2 / (1 + t) times 2 t / (1 + t)^2 <= 1/2 (times |x / c| never above .45): .95 x 2^-23; the quotient is off by 2 ulp of
itself, the last sum by half a step: below 4 x 2^-23 c in all, and c is at most |c tanh(x / c)| / .244: 33 x 2^-24 of the capped score.  f32's tanh: 2 ulp,
its argument's rounding, a product: 4 x 2^-24."""
import pytest
import torch

from test_gpu_paged import Cache, assert_close, normal, run_attention

pytestmark = pytest.mark.gpu


def reference(c, q, lengths, scale, softcap=0.0):
    """[T, H, D] in 64 bits and what may be off."""
    t, h, d = q.shape
    out, slack = (torch.zeros(t, h, d, dtype=torch.float64, device="cuda") for _ in range(2))
    for i, n in enumerate(lengths):
        page, slot = c.rows(i, n)
        k, v = (x[page, :, slot].double().repeat_interleave(h // c.kv_heads, 1) for x in (c.k, c.v))
        x = torch.einsum("hd,jhd->hj", q[i].double(), k) * scale
        mag = torch.einsum("hd,jhd->hj", q[i].double().abs(), k.abs().nan_to_num(0, 0, 0)).amax(1, keepdim=True) * abs(scale)  # of finite scores
        dx = (d / 32 + 8 if q.dtype == torch.float32 else d / 16 * 4) * 2.0 ** -24 * mag
        if softcap:
            x = softcap * torch.tanh(x / softcap)
            dx = dx + 33 * 2.0 ** -24 * x.abs().amax(1, keepdim=True)
        w = torch.softmax(x, 1)
        spread = (x.amax(1, keepdim=True) - x).clamp(max=21.0).amax(1, keepdim=True)
        out[i] = torch.einsum("hj,jhd->hd", w, v)
        slack[i] = (2 * dx + (2 + spread) * 2.0 ** -22 + 2 * n * 2.0 ** -24 + 2.0 ** -22) * torch.einsum("hj,jhd->hd", w, v.abs())
    return out, slack


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 2, 128, 16), (16, 1, 64, 16), (2, 1, 256, 5)])
@pytest.mark.parametrize("softcap", [1e-3, 1.0, 20.0, 50.0, 1e3, 1e4, 1e6, 1e9, 1e30, 3e38])
def test_caps_of_any_size(backend, dtype, heads, kv_heads, dim, page, softcap):
    gen = torch.Generator(device="cuda").manual_seed(dim)
    lengths = [500, 33, 1]
    c = Cache(backend, gen, lengths, kv_heads, dim, page, dtype)
    for i, n in enumerate(lengths):
        c.fill(gen, i, n, dtype)
    q, scale = normal(gen, (3, heads, dim), dtype, 4.0), dim ** -0.5  # scores of about +-4, some beyond 12
    pos = torch.tensor(lengths, dtype=torch.int32, device="cuda") - 1
    got = run_attention(backend, c, q, pos, None, scale, softcap=softcap)
    ref, slack = reference(c, q, lengths, scale, softcap)
    assert_close(got, ref, slack, dtype)


def finite_or_nan(got, ref, slack, dtype):
    assert torch.equal(got.isnan(), ref.isnan()), f"NaN in {int(got.isnan().sum())} places for {int(ref.isnan().sum())}"
    fine = ref.isfinite()
    assert_close(got[fine], ref[fine], slack[fine], dtype)


LENGTHS = [1, 17, 33, 65, 16, 49, 300, 2001, 1, 4000]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 2, 128, 16), (24, 1, 64, 5), (6, 2, 256, 16)])
@pytest.mark.parametrize("what", ["query", "newest key", "first key", "every seventh key", "infinite key", "plus infinity", "one key"])
def test_scores_that_are_no_numbers(backend, dtype, heads, kv_heads, dim, page, what):
    """NaN where a visible score is NaN, +infinity, or all of them are -infinity, wherever the key lies among the tiles, warps and CTAs; the other rows as ever."""
    gen = torch.Generator(device="cuda").manual_seed(heads + len(what))
    c = Cache(backend, gen, LENGTHS, kv_heads, dim, page, dtype)
    q = normal(gen, (len(LENGTHS), heads, dim), dtype)
    q[:, 0, 0] = q[:, 0, 0].abs() + 0.5
    q[:, -1, 0] = -q[:, -1, 0].abs() - 0.5
    inf, nan = float("inf"), float("nan")
    for i, n in enumerate(LENGTHS):
        c.fill(gen, i, n, dtype)
        rows, slots = c.rows(i, n)
        if what == "query" and i != 4:
            q[i, i % heads, 3] = nan
        elif what == "newest key":
            c.k[rows[-1], i % kv_heads, slots[-1], 5] = nan
        elif what == "first key":
            c.k[rows[0], 0, slots[0], 5] = nan
        elif what == "every seventh key" and i % 2:
            c.k[rows[3::7], 0, slots[3::7], 0] = nan
        elif what == "infinite key":  # the first head of the KV head 0 sees -infinity everywhere, others +infinity
            c.k[rows, 0, slots, 0] = -inf
        elif what == "plus infinity":
            c.k[rows[n // 2], kv_heads - 1, slots[n // 2], 0] = inf
        elif what == "one key":  # -infinity for the first head, all other scores finite
            c.k[rows[n // 3], 0, slots[n // 3], 0] = -inf
    pos = torch.tensor(LENGTHS, dtype=torch.int32, device="cuda") - 1
    got = run_attention(backend, c, q, pos, None, dim ** -0.5)
    finite_or_nan(got, *reference(c, q, LENGTHS, dim ** -0.5), dtype)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_a_row_that_sees_nothing_is_zeros_beside_nan(backend, dtype):
    gen = torch.Generator(device="cuda").manual_seed(1)
    c = Cache(backend, gen, [40, 40], 1, 64, 16, dtype)
    for i in range(2):
        c.fill(gen, i, 40, dtype)
    q = normal(gen, (2, 2, 64), dtype)
    q[:, 0, 0] = float("nan")
    got = run_attention(backend, c, q, torch.tensor([39, -1], dtype=torch.int32, device="cuda"), None, 0.125)
    assert got[0, 0].isnan().all() and got[0, 1].isfinite().all() and (got[1] == 0).all()
