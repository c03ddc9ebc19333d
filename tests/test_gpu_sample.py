"""Sampling against the definition in 64 bits, token for token: filters alone and together, ties, masked rows, values that are no numbers,
random numbers at the ends of their range."""
import numpy as np
import pytest

from torchlette_b200 import backend as tb  # noqa: F401
from torchlette_b200 import binding as B

pytestmark = pytest.mark.gpu


def reference(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """One row by the definition; x f64 (of the stored values)."""
    x = np.where(np.isnan(x), -np.inf, x)
    if x.max() == -np.inf:
        return -1
    if u is None or not t > 0:
        return int(np.argmax(x))
    with np.errstate(all="ignore"):
        w = np.where(x == x.max(), 1.0, np.exp(np.where(x == -np.inf, -np.inf, (x - x.max()) / t)))
    order = np.lexsort((np.arange(len(x)), -x))
    if k > 0:
        order = order[:k]
    if p < 1:
        mass = np.cumsum(w[order])
        order = order[:int((mass < max(p, 0) * mass[-1]).sum()) + 1]
    if m > 0:
        order = order[w[order] >= min(m, 1.0)]
    order = np.sort(order)
    mass = np.cumsum(w[order])
    u = 0.0 if not u > 0 else min(u, 1.0)
    return int(order[min(int((mass <= u * mass[-1]).sum()), np.flatnonzero(w[order])[-1])])


def stored(x, dtype):
    """(what is uploaded, its values in f64)"""
    if dtype == "f32":
        x = x.astype(np.float32)
        return x, x.astype(np.float64)
    if dtype == "f16":
        with np.errstate(over="ignore"):
            x = x.astype(np.float16)
        return x, x.astype(np.float64)
    b = np.ascontiguousarray(x.astype(np.float32)).view(np.uint32)
    nan = np.isnan(x)
    b = np.where(nan, 0x7fc00000, b + 0x7fff + ((b >> 16) & 1)).astype(np.uint32) >> 16
    return b.astype(np.uint16), (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def sample(be, bits, dtype, u=None, **params):
    up = lambda a, d: None if a is None else be.ops.tensorFromArray(np.asarray(a), [len(a)], d)  # noqa: E731
    held = [be.ops.tensorFromArray(bits, list(bits.shape), dtype), up(u, "f32")]
    kinds = {"temperature": "f32", "topK": "i32", "topP": "f32", "minP": "f32"}
    more = {n: up(a, kinds[n]) for n, a in params.items()}
    y = be.ops.sample(held[0], held[1], **more)
    got = be.ops.read(y).tolist()
    for t in held + list(more.values()) + [y]:
        if t is not None:
            t.destroy()
    return got


def check(be, x, dtype, u, t=None, k=None, p=None, m=None):
    bits, values = stored(x, dtype)
    rows = len(x)
    f = lambda a, off: [off] * rows if a is None else [float(np.float32(v)) for v in a]  # noqa: E731
    params = {n: a for n, a in (("temperature", t), ("topK", k), ("topP", p), ("minP", m)) if a is not None}
    got = sample(be, bits, dtype, u, **params)
    us = [None] * rows if u is None else f(u, 0)
    want = [reference(values[i], us[i], f(t, 1.0)[i], 0 if k is None else int(k[i]), f(p, 1.0)[i], f(m, 0.0)[i]) for i in range(rows)]
    assert got == want


FILTERS = {"none": (0, 1.0, 0.0), "top_k": (50, 1.0, 0.0), "top_k_one": (1, 1.0, 0.0), "top_k_wide": (3000, 1.0, 0.0), "top_p": (0, 0.9, 0.0),
           "top_p_low": (0, 0.1, 0.0), "min_p": (0, 1.0, 0.05), "k_and_p": (40, 0.8, 0.0), "all": (200, 0.95, 0.02), "p_and_min": (0, 0.99, 0.001)}


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4097, 32_000, 151_936])
@pytest.mark.parametrize("name", FILTERS)
def test_filters(backend, dtype, vocab, name):
    rng = np.random.default_rng(vocab + len(name))
    rows = 5 if vocab > 100_000 else 9
    k, p, m = FILTERS[name]
    x = rng.standard_normal((rows, vocab)) * rng.uniform(0.3, 4.0, (rows, 1))
    u, t = rng.uniform(size=rows).astype(np.float32), rng.uniform(0.5, 1.5, rows)
    check(backend, x, dtype, u, t, [k] * rows if k else None, [p] * rows if p < 1 else None, [m] * rows if m else None)


def test_rows_with_parameters_of_their_own(backend):
    rng = np.random.default_rng(1)
    rows, vocab = 24, 5000
    x = rng.standard_normal((rows, vocab)) * 2
    t = np.where(np.arange(rows) % 5 == 3, 0.0, rng.uniform(0.3, 2, rows))
    check(backend, x, "f32", rng.uniform(size=rows), t, rng.choice([0, -3, 1, 7, 100, 4999, 5000, 6000], rows), rng.choice([0.0, 0.3, 0.9, 1.0, 2.0, -1.0], rows),
          rng.choice([0.0, -1.0, 0.1, 1.0, 3.0], rows))


@pytest.mark.parametrize("k,p", [(0, 0.5), (0, 0.9), (3, 1.0), (700, 0.5), (1500, 1.0), (0, 1.0), (999, 0.999)])
def test_ties_go_to_the_lowest_index(backend, k, p):
    """All equal, two values, and few values: the borders fall between equal logits."""
    rng = np.random.default_rng(2)
    for x in (np.zeros((4, 2000)), rng.integers(0, 2, (4, 2000)) * 1.0, rng.integers(-3, 3, (4, 9001)) * 0.5, np.where(rng.uniform(size=(4, 2000)) < 0.5, -0.0, 0.0)):
        u = np.array([0.0, 0.25, 0.7, 1 - 2.0 ** -24])
        for dtype in ("f32", "bf16"):
            check(backend, x, dtype, u, None, [k] * 4 if k else None, [p] * 4 if p < 1 else None)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_masked_rows_and_values_that_are_no_numbers(backend, dtype):
    rng = np.random.default_rng(3)
    low = {"f32": -3.4028234663852886e38, "f16": -65504.0, "bf16": -3.3895313892515355e38}[dtype]
    x = rng.standard_normal((12, 3001)) * 2
    x[0] = -np.inf                      # nothing is left
    x[1] = np.nan
    x[2, 1:] = -np.inf                  # one is left
    x[3, :3000] = -np.inf
    x[4] = low                          # all at the type's lowest value
    x[5, 5:] = low
    x[6, ::3] = np.nan
    x[7, [10, 20, 2000]] = np.inf       # infinities share the mass
    x[8, 100] = np.inf
    x[8, 7] = np.nan
    x[9, rng.uniform(size=3001) < 0.9] = -np.inf
    x[10] = -np.inf
    x[10, 77] = low
    u = rng.uniform(size=12)
    for t, k, p, m in ((None, None, None, None), ([0.7] * 12, [5] * 12, [0.9] * 12, None), (None, None, [0.5] * 12, [0.1] * 12), (None, [2000] * 12, None, None),
                       ([0.0] * 12, [5] * 12, None, None), (None, None, [0.0] * 12, None)):
        check(backend, x, dtype, u, t, k, p, m)
    check(backend, x, dtype, None)


def test_random_numbers_and_temperatures_at_the_ends(backend):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((10, 777)) * 3
    u = np.array([0.0, -0.0, 2.0 ** -149, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, np.nan, np.inf, 0.5], dtype=np.float32)
    for k, p in ((None, None), ([9] * 10, None), (None, [0.8] * 10)):
        check(backend, x, "f32", u, None, k, p)
    for t in (1e-30, 2.0 ** -149, 1e-3, 1e6, 3e38, np.inf):
        check(backend, x, "f32", rng.uniform(size=10), [t] * 10, [20] * 10)
        check(backend, x, "f32", rng.uniform(size=10), [t] * 10, None, [0.6] * 10)
        check(backend, x, "f32", rng.uniform(size=10), [t] * 10)
    for t in (0.0, -1.0, np.nan):
        check(backend, x, "f32", rng.uniform(size=10), [t] * 10, [20] * 10)
    check(backend, x, "f32", rng.uniform(size=10), None, None, [np.nan] * 10, [np.nan] * 10)


def test_wide_spread_and_close_values(backend):
    """Values over all magnitudes (the borders need every bit of the keys) and values one step apart."""
    rng = np.random.default_rng(5)
    x = np.stack([np.exp(rng.uniform(-80, 80, 6000)) * rng.choice([-1, 1], 6000), np.float32(1) + rng.integers(0, 50, 6000) * 2.0 ** -23,
                  rng.integers(-9, 9, 6000) * 2.0 ** -149, rng.standard_normal(6000) * 1e-3])
    for t in ([1.0] * 4, [1e30, 2.0 ** -20, 2.0 ** -140, 1e-4]):
        for k, p in (([100] * 4, None), (None, [0.9] * 4), ([2500] * 4, [0.4] * 4), (None, None)):
            check(backend, x, "f32", rng.uniform(size=4), t, k, p)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_rows_apart_and_not_aligned(backend, dtype):
    """Strides through the C ABI: rows further apart than a vocabulary, an odd vocabulary, a start off any alignment but the type's."""
    be = backend
    rng = np.random.default_rng(6)
    bits, values = stored(rng.standard_normal((3, 1501)) * 2, dtype)
    u = rng.uniform(size=3).astype(np.float32)
    t, ut, out = be.ops.tensorFromArray(bits, [3, 1501], dtype), be.ops.tensorFromArray(u, [3], "f32"), be.ops.empty([3], "i32")
    kt = be.ops.tensorFromArray(np.array([30] * 3), [3], "i32")
    for start, vocab in ((1, 1500), (3, 800), (0, 1501), (8, 16)):
        be._calls.tl_sample(be._handle, t.buffer + start * bits.itemsize, B.DTYPE_ID[dtype], 3, vocab, 1501, None, kt.buffer, None, None, ut.buffer, out.buffer)
        assert be.ops.read(out).tolist() == [reference(values[i, start:start + vocab], float(u[i]), 1.0, 30) for i in range(3)]
    for x in (t, ut, out, kt):
        x.destroy()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_vocabulary_of_millions(backend, dtype):
    """One row over more than a cluster keeps the masses of, with and without filters."""
    rng = np.random.default_rng(8)
    x = rng.standard_normal((1, 5_000_001)) * 2
    for k, p, m in ((None, None, None), ([100], [0.9], None), (None, [0.7], None), ([5000], None, None), (None, None, [0.01])):
        check(backend, x, dtype, rng.uniform(size=1), [0.9], k, p, m)


def test_many_rows_again_and_in_a_graph(backend):
    be = backend
    rng = np.random.default_rng(7)
    bits, values = stored(rng.standard_normal((130, 20_000)) * 2, "f16")
    u, t, k, p = rng.uniform(size=130).astype(np.float32), rng.uniform(0.5, 1, 130), [64] * 130, [0.9] * 130
    want = [reference(values[i], float(u[i]), float(np.float32(t[i])), 64, float(np.float32(0.9))) for i in range(130)]
    assert sample(be, bits, "f16", u, temperature=t, topK=k, topP=p) == want
    held = [be.ops.tensorFromArray(np.asarray(a), s, d) for a, s, d in ((bits, [130, 20_000], "f16"), (u, [130], "f32"), (t, [130], "f32"), (k, [130], "i32"), (p, [130], "f32"))]
    out = be.ops.empty([130], "i32")
    be.sync()
    be.beginCapture()
    be.ops.sample(held[0], held[1], temperature=held[2], topK=held[3], topP=held[4], out=out)
    graph = be.endCapture()
    be.replay(graph)
    assert be.ops.read(out).tolist() == want
    u2 = rng.uniform(size=130).astype(np.float32)
    be._upload(held[1].buffer, u2)
    be.replay(graph)
    assert be.ops.read(out).tolist() == [reference(values[i], float(u2[i]), float(np.float32(t[i])), 64, float(np.float32(0.9))) for i in range(130)]
    be.destroyGraph(graph)
    for x in held + [out]:
        x.destroy()
