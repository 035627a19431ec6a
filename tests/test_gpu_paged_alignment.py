"""Calls of the paged operators and of sampling whose 32-bit arrays do not lie at multiples of 4 bytes are
refused: loads at places that a wave shares would read the integers at the multiple before."""
import numpy as np
import pytest

import strict_amd
import test_gpu_paged as paged
from strict_amd import PagedKV, PagedKV8
from test_gpu_paged8 import Case8

pytestmark = pytest.mark.gpu


def refused(call, text):
    with pytest.raises(strict_amd.StrictHipError) as e:
        call()
    assert e.value.status == strict_amd.SH_ERR_INVALID_ARGUMENT and text in e.value.message, e.value.message


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("bits", [8, 16])
def test_index(ctx, bits, off):
    c = (Case8 if bits == 8 else paged.Case)(ctx, off, "f16", [1, 2], [20, 9], 4, 2, 64, 16)
    kv = c.upload()
    pools = len(c.buffers) - 3
    nbytes = c.tokens * 4 * 64 * 2
    q, out, k, v = (ctx.alloc(nbytes) for _ in range(4))
    qkv, gain = ctx.alloc(c.tokens * 8 * 64 * 2), ctx.upload(np.ones(64, np.float32))
    work = ctx.alloc(ctx.attn_paged_workspace(kv, c.tokens, 4, 2))
    calls = [lambda kv: ctx.attn_paged(kv, q, out, c.tokens, 4, 2, 1.0, work),
             lambda kv: ctx.qk_norm_rope_paged(kv, qkv, gain, gain, q, c.tokens, 4, 1e-6, 1e4)]
    if bits == 8:
        calls.append(lambda kv: ctx.paged_read(kv, k, v, c.tokens))
    for i in range(pools, len(c.buffers)):
        area = ctx.alloc(c.buffers[i].nbytes + 16)
        buffers = list(c.buffers)
        buffers[i] = area.ptr + off
        shifted = (PagedKV8 if bits == 8 else PagedKV)(*buffers, batch=c.batch, max_pages=c.max_pages, num_pages=c.num_pages,
                                                       page_size=c.page, kv_heads=2, head_dim=64)
        for call in calls:
            refused(lambda: call(shifted), "4-byte aligned")
        area.free()
    for b in (q, out, k, v, qkv, gain, work):
        b.free()
    c.free()


@pytest.mark.parametrize("off", [1, 2, 3])
def test_page_numbers(ctx, off):
    pool, numbers, area = ctx.alloc(5 * 32), ctx.upload(np.zeros(3, np.int32)), ctx.alloc(32)
    for src, dst in ((area.ptr + off, numbers), (numbers, area.ptr + off)):
        refused(lambda: ctx.pages_copy(pool, 1, 5, 32, src, dst, 3), "4-byte aligned")
    for b in (pool, numbers, area):
        b.free()


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("n", [50, 5000])
def test_sampling_parameters(ctx, off, n):
    rows = 3
    x, index, area = ctx.upload(np.zeros((rows, n), np.float32)), ctx.alloc(4 * rows), ctx.alloc(64)
    own = {name: ctx.upload(np.zeros(rows, np.float32)) for name in ("temperature", "top_k", "top_p", "min_p", "u")}
    work = ctx.alloc(ctx.sample_workspace(rows, n))
    for name in own:
        b = {**own, name: area.ptr + off}
        refused(lambda: ctx.sample(x, rows, n, b["temperature"], b["top_k"], b["top_p"], b["min_p"], b["u"], index, work),
                "4-byte aligned")
    ctx.sample(x, rows, n, None, None, None, None, own["u"], index, work)
    ctx.sync()
    assert (index.to_host(np.int32, (rows,)) == 0).all()
    for b in (x, index, area, work, *own.values()):
        b.free()
