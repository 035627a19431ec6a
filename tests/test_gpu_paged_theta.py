"""RoPE of the paged cache at the largest angles, and beyond them."""
import numpy as np
import pytest

import strict_amd
import test_gpu_paged as paged

pytestmark = pytest.mark.gpu


def rope(ctx, theta, length, page=16, max_pages=None, d=128):
    """q of one token at position length - 1 whose page alone is there."""
    c = paged.Case(ctx, 4, "f16", [1], [1], 2, 1, d, page, rows_behind=0)
    need = -(-length // page)
    max_pages = need if max_pages is None else max_pages
    table = np.full((1, max_pages), -1, np.int32)
    table[0, need - 1] = 0
    x = c.rng.normal(0, 1.7, (1, 4, d))
    bufs = [ctx.upload(a) for a in (c.k, c.v, table, np.array([length], np.int32), np.array([0, 1], np.int32),
                                    paged.to16(x, "f16"), np.ones(d, np.float32), np.zeros((1, 2, d), np.int16))]
    kv = strict_amd.PagedKV(*bufs[:5], batch=1, max_pages=max_pages, num_pages=c.num_pages, page_size=page, kv_heads=1,
                            head_dim=d, dtype="f16")
    try:
        ctx.qk_norm_rope_paged(kv, bufs[5], bufs[6], bufs[6], bufs[7], 1, 2, 1e-6, theta)
        ctx.sync()
        got = paged.from16(bufs[7].to_host(), "f16")
    finally:
        for b in bufs:
            b.free()
    ref, size = paged.norm_rope_oracle(paged.from16(paged.to16(x, "f16"), "f16")[:, :2], np.ones(d),
                                       np.array([length - 1.0]), float(np.float32(1e-6)), theta)
    assert (np.abs(got - ref) <= paged.U["f16"] * np.abs(ref) + 32 * paged.F * size + 2.0 ** -25).all()


@pytest.mark.parametrize("theta,length", [(1.0, 1 << 28), (1e6, 1 << 28), (0.5, 1 << 20), (2.0 ** -7, 4_000_000), (2.0 ** -20, 600)])
def test_largest_angles(ctx, theta, length):
    rope(ctx, theta, length, page=65536 if length > 1 << 26 else 16)


@pytest.mark.parametrize("theta,length", [(2.0 ** -7, 6_000_000), (1e-8, 100_003), (1e-38, 17)])
def test_angles_past_what_fp64_resolves_are_refused(ctx, theta, length):
    with pytest.raises(strict_amd.StrictHipError) as e:
        rope(ctx, float(np.float32(theta)), length)
    assert e.value.status == strict_amd.SH_ERR_INVALID_ARGUMENT and "theta" in e.value.message
