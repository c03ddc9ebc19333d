"""Rows whose cluster's last CTAs have the least to read: the smallest vocabularies of every cluster size, many calls behind one another."""
import numpy as np
import pytest

from test_gpu_sample import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("vocab", [4097, 8193, 16385, 32769])
def test_short_slices(backend, vocab, dtype):
    gen = np.random.default_rng(vocab)
    for _ in range(3):
        x, u = gen.standard_normal((4, vocab)) * 3, gen.random(4)
        x[0, -1] = 30.0  # the last CTA has the row's largest
        check(backend, x, dtype, u, k=[1, 50, 50, 192])
        check(backend, x, dtype, u, p=[.9, .9, .5, .99])
        check(backend, x, dtype, None)


def test_calls_behind_one_another(backend):
    be, gen = backend, np.random.default_rng(1)
    x = gen.standard_normal((3, 4097)).astype(np.float32)
    logits, out = be.ops.tensorFromArray(x, [3, 4097], "f32"), [be.ops.empty([3], "i32") for _ in range(200)]
    for y in out:
        be.ops.sample(logits, out=y)
    want = x.argmax(1).tolist()
    assert all(be.ops.read(y).tolist() == want for y in out)
    for t in [logits] + out:
        t.destroy()
