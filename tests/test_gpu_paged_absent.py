"""Appending a padded batch whose rows end with the tokens that are there."""
import ctypes as C

import pytest
import torch

from test_gpu_paged import TORCH, Cache, normal
from torchlette_b200 import backend as tb
from torchlette_b200 import binding as B

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [128, 6])  # whole vectors, and the general kernel
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("absent", ["negative", "sequence", "position"])
def test_tokens_that_are_not_there_need_no_rows(dim, dtype, absent):
    be = tb.CudaBackend(0)  # its error count is its own
    try:
        gen = torch.Generator(device="cuda").manual_seed(dim)
        c = Cache(be, gen, [20, 20], 2, dim, 16, dtype)
        there, tokens = 2, 40
        pos = torch.full((tokens,), {"negative": -1, "sequence": 3, "position": 2 ** 30}[absent], dtype=torch.int32, device="cuda")
        seq = torch.full((tokens,), 7 if absent == "sequence" else 0, dtype=torch.int32, device="cuda")
        pos[:there], seq[:there] = torch.tensor([4, 17], device="cuda"), torch.tensor([1, 0], device="cuda")
        # two rows of q, k and v, and room behind them that belongs to nobody
        q, k, v = (normal(gen, (tokens, n, dim), dtype) for n in (4, 2, 2))
        before = [c.k.clone(), c.v.clone()]
        out = torch.full_like(q, 7.0)
        torch.cuda.synchronize()
        B.check(be._ctx, be._lib.tl_paged_append(be._ctx, C.byref(B.PagedCache.from_buffer_copy(c.cache.descriptor())), pos.data_ptr(), seq.data_ptr(), tokens,
                                                 q.data_ptr(), 4 * dim, dim, 4, out.data_ptr(), 4 * dim, dim, k.data_ptr(), 2 * dim, dim, v.data_ptr(), 2 * dim, dim,
                                                 None, None, 0, 1e-6, None, None, 0))
        if absent == "negative":
            be.sync()
        else:
            with pytest.raises(tb.TlError, match=absent):
                be.sync()
        assert torch.equal(out[:there], q[:there]) and (out[there:] == 7.0).all()
        for pages, then, rows in zip((c.k, c.v), before, (k, v)):
            for t in range(there):
                page, slot = c.rows(int(seq[t]), 18)
                p = int(pos[t])
                assert torch.equal(pages[page[p], :, slot[p]], rows[t])
                pages[page[p], :, slot[p]] = float("nan")
            bits = torch.int32 if TORCH[dtype] == torch.float32 else torch.int16
            assert torch.equal(pages.view(bits), then.view(bits))
    finally:
        be.destroy()
