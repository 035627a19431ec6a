"""The paged operators and sampling with every buffer given by its device address, as
tensors of another library are: results as with buffers, and the same refusals."""
import numpy as np
import pytest

import strict_amd
import test_gpu_paged as paged
from strict_amd import PagedKV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,lengths", [([1, 1], [300, 40]), ([30, 2], [90, 200])])
def test_attention(ctx, new, lengths):
    c = paged.Case(ctx, 1, "bf16", new, lengths, 4, 2, 64, 16)
    q, want = paged.run_attention(c)
    kv = c.upload()
    by_address = PagedKV(*(b.ptr for b in c.buffers), batch=c.batch, max_pages=c.max_pages, num_pages=c.num_pages,
                         page_size=16, kv_heads=2, head_dim=64, dtype="bf16")
    dq, out = ctx.upload(q), ctx.upload(paged.to16(np.full(q.shape, 0.5), "bf16"))
    work = ctx.alloc(ctx.attn_paged_workspace(kv, c.tokens, 4, max(new)))
    ctx.attn_paged(by_address, dq.ptr, out.ptr, c.tokens, 4, max(new), float(np.float32(0.125)), work.ptr)
    ctx.sync()
    assert (out.to_host() == want).all()
    for workspace, text in ((None, "workspace is NULL"), (work.ptr + 16, "not inside an allocation"), (work.ptr + 8, "workspace")):
        with pytest.raises(strict_amd.StrictHipError) as e:
            ctx.attn_paged(by_address, dq.ptr, out.ptr, c.tokens, 4, max(new), 0.125, workspace)
        assert text in e.value.message
    for b in (dq, out, work):
        b.free()
    c.free()


@pytest.mark.parametrize("n", [1000, 5000])
def test_sampling(ctx, n):
    rng = np.random.default_rng(n)
    x, u = rng.normal(0, 2, (3, n)).astype(np.float32), rng.random(3).astype(np.float32)
    bufs = [ctx.upload(a) for a in (x, np.full(3, 0.8, np.float32), np.full(3, 20, np.int32), np.full(3, 0.9, np.float32),
                                    np.zeros(3, np.float32), u, np.full(3, -7, np.int32))]
    work = ctx.alloc(ctx.sample_workspace(3, n))
    got = []
    for args in ((*bufs, work), (*(b.ptr for b in bufs), work.ptr)):
        bufs[6].copy_from_host(np.full(3, -7, np.int32))
        ctx.sample(args[0], 3, n, *args[1:])
        ctx.sync()
        got.append(bufs[6].to_host())
    assert (got[0] == got[1]).all() and (got[0] >= 0).all()
    with pytest.raises(strict_amd.StrictHipError) as e:
        ctx.sample(bufs[0], 3, n, *bufs[1:], None)
    assert "workspace is NULL" in e.value.message
    for b in (*bufs, work):
        b.free()
