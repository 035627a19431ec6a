"""q of the head norms with RoPE into pages of 8-bit values is that into 16-bit ones, bit for
bit, at positions whose angles are as large as calls take."""
import numpy as np
import pytest

from strict_amd import PagedKV, PagedKV8
from test_gpu_paged import to16

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("theta", [2.0, 1e4, 1e6, 3e38])
@pytest.mark.parametrize("length", [700, 40000, 1 << 28])
def test_same_q(ctx, dtype, d, theta, length):
    # (no position has a page: nothing is stored)
    page, heads, tokens = 65536, 8, 600
    max_pages = -(-length // page)
    rng = np.random.default_rng(length % 1000 + d)
    index = [ctx.upload(np.asarray(a, np.int32)) for a in (np.full((1, max_pages), -1), [length], [0, tokens])]
    qkv = ctx.upload(to16(rng.normal(0, 1, (tokens, heads + 2, d)), dtype))
    gain = ctx.upload(rng.normal(1, 0.2, d).astype(np.float32))
    sizes = dict(batch=1, max_pages=max_pages, num_pages=1, page_size=page, kv_heads=1, head_dim=d, dtype=dtype)
    pools = [ctx.alloc(page * d * 2) for _ in range(2)]
    pages = ctx.alloc(PagedKV8.page_bytes(1, page, d))
    got = []
    for kv in (PagedKV(*pools, *index, **sizes), PagedKV8(pages, *index, **sizes)):
        q = ctx.upload(np.zeros((tokens, heads, d), np.int16))
        ctx.qk_norm_rope_paged(kv, qkv, gain, gain, q, tokens, heads, 1e-6, theta)
        ctx.sync()
        got.append(q.to_host())
        q.free()
    for b in (*index, qkv, gain, *pools, pages):
        b.free()
    assert (got[0] == got[1]).all(), f"{(got[0] != got[1]).sum()} of {got[0].size} differ"
