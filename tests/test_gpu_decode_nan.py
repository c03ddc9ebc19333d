"""Decode attention over keys that are NaN: the rows that see them are NaN, also where such a key is the only one of its tile, warp or CTA."""
import pytest
import torch

from test_gpu_paged import normal, wrap

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (16, 1, 128), (2, 2, 128)])
@pytest.mark.parametrize("n", [1, 17, 33, 49, 65, 129, 1025, 4001])
@pytest.mark.parametrize("masked", [False, True])
def test_nan_keys(backend, dtype, heads, kv_heads, dim, n, masked):
    be = backend
    gen = torch.Generator(device="cuda").manual_seed(n)
    q, k, v = normal(gen, (3, heads, 1, dim), dtype), normal(gen, (3, kv_heads, n + 4, dim), dtype), normal(gen, (3, kv_heads, n + 4, dim), dtype)
    k[1, 0, n - 1, 3] = float("nan")  # the newest one
    k[2, kv_heads - 1, :min(16, n), 0] = float("nan")  # a whole tile
    more = {}
    mask = torch.zeros(n, device="cuda")
    if masked:
        mask[n // 2:max(n // 2, n - 1)] = -float("inf")  # half of the keys, the newest not among them
        more["mask"] = wrap(be, mask)
    torch.cuda.synchronize()
    y = be.ops.decodeAttention(wrap(be, q), wrap(be, k), wrap(be, v), n, dim ** -0.5, **more)
    got = torch.from_numpy(be.ops.read(y)).cuda()  # bf16: its bits
    got = (got.view(torch.bfloat16) if dtype == "bf16" else got).double().reshape(3, heads * dim)
    y.destroy()
    rep = heads // kv_heads
    kd, vd = (x[:, :, :n].double().repeat_interleave(rep, 1) for x in (k, v))
    w = torch.softmax(torch.einsum("bhd,bhjd->bhj", q[:, :, 0].double(), kd) * dim ** -0.5 + mask.double(), -1)
    ref = torch.einsum("bhj,bhjd->bhd", w, vd).reshape(3, heads * dim)
    assert torch.equal(got.isnan(), ref.isnan())
    fine = ref.isfinite()
    half = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}[dtype]
    # one rounding, and scores off by 2^-24 of sums of |q k| below 4 sqrt(dim), keys added up in chains of n
    assert ((got - ref).abs()[fine] <= half * ref.abs()[fine] + (2 * dim + n) * 2.0 ** -23).all()
