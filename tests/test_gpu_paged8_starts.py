"""Attention over pages of 8-bit values with starts out of order: a sequence's rows are its
own and are written, however many rows the sequences have together."""
import numpy as np
import pytest

import test_gpu_paged as paged
from strict_amd import PagedKV8
from test_gpu_paged import from16, to16
from test_gpu_paged8 import Case8

pytestmark = pytest.mark.gpu


def attended(c, starts, new):
    """The rows of a call over the case's cache with other starts, NaN where none is written."""
    kv = c.upload()
    index = c.ctx.upload(np.asarray(starts, np.int32))
    kv = PagedKV8(*c.buffers[:3], index, **c.sizes())
    q = to16(np.random.default_rng(1).normal(0, 1.5, (c.tokens, c.heads, c.d)), c.dtype)
    dq, out = c.ctx.upload(q), c.ctx.upload(to16(np.full(q.shape, np.nan), c.dtype))
    work = c.ctx.alloc(c.ctx.attn_paged_workspace(kv, c.tokens, c.heads, max(new)))
    c.ctx.attn_paged(kv, dq, out, c.tokens, c.heads, max(new), float(np.float32(c.d ** -0.5)), work)
    c.ctx.sync()
    got = from16(out.to_host(), c.dtype)
    for b in (index, dq, out, work):
        b.free()
    c.free()
    return from16(q, c.dtype), got


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("extra", [1, 300])  # (with 300 pages more tiles are cut)
@pytest.mark.parametrize("again", [1, 3, 70])
@pytest.mark.parametrize("heads,kv_heads", [(4, 1), (32, 2)])
def test_rows_of_several_sequences(ctx, dtype, extra, again, heads, kv_heads):
    # sequence 0 has rows 0 .. 299; of the others every second has rows 200 .. 299 again, with as
    # many positions and the same pages, so that whichever writes them writes the same
    n, back = 300, 100
    c = Case8(ctx, again, dtype, [n] + [0] * (2 * again), [n + 40] * (2 * again + 1), heads, kv_heads, 64, 16,
              rows_behind=0, extra_entries=extra)
    c.table[:] = c.table[0]
    starts = np.array([0, n] + [n - back, n] * again, np.int32)
    assert len(starts) == c.batch + 1 and c.tokens == n
    q, got = attended(c, starts, [n])
    c.new = [n] + [0] * (2 * again)
    c.starts = np.array([0] + [n] * (2 * again + 1), np.int32)
    ref, tol = paged.attention_oracle(c, q, 0, 0, float(np.float32(64 ** -0.5)))
    assert not np.isnan(got).any(), f"{np.isnan(got).any((1, 2)).sum()} rows are not written"
    assert (np.abs(got - ref) <= tol).all()
