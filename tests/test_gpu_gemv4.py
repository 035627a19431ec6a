"""4-bit weights: their quantisation and layout byte by byte, and the products against 64
bits (numpy), each within what fp32 sums and the result's rounding add up to."""
import numpy as np
import pytest

import strict_amd
from test_gpu_paged import F, U, from16, to16

pytestmark = pytest.mark.gpu

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])


def quantised(w):
    """Codes and scale bytes of rows of groups of 32 by the header's rule."""
    n, k = w.shape
    g = w.astype(np.float64).reshape(n, k // 32, 32)
    whole = np.isfinite(g).all(-1)
    g = np.where(whole[..., None], g, 0.0)
    most = np.abs(g).max(-1)
    e = np.maximum(np.ceil(np.log2(np.maximum(most, 1e-300) / 6)), -127).astype(int)
    e += most > 6 * 2.0 ** e
    e -= (e > -127) & (most <= 6 * 2.0 ** (e - 1))
    z = np.abs(g) / 2.0 ** e[..., None]
    middle = (E2M1[1:8] + E2M1[:7]) / 2
    low = np.searchsorted(middle, z)
    low = low + ((low < 7) & (z == middle[np.minimum(low, 6)]) & (low % 2 == 1))
    code = np.where(whole[..., None], low + 8 * np.signbit(w.reshape(g.shape)), 0).reshape(n, k)
    return code.astype(np.uint8), np.where(whole, e + 127, 255).astype(np.uint8)


def packed(code):
    return code[:, 0::2] | (code[:, 1::2] << 4)


def values(code, scale):
    n, k = code.shape
    s = np.where(scale == 255, np.nan, 2.0 ** (scale.astype(int) - 127))
    return (E2M1[code].reshape(n, k // 32, 32) * s[..., None]).reshape(n, k)


@pytest.mark.parametrize("n,k", [(1, 32), (7, 96), (33, 1024)])
def test_quantize(ctx, n, k):
    rng = np.random.default_rng(n + k)
    w = rng.normal(0, 1, (n, k)) * np.repeat(2.0 ** rng.integers(-140, 120, (n, k // 32)), 32, 1)
    if n > 7:
        near = np.concatenate([E2M1, (E2M1[1:8] + E2M1[:7]) / 2, 6 * (1 + 2.0 ** -23) * np.ones(1), 6 * (1 - 2.0 ** -24) * np.ones(1)])
        w[1] = rng.choice(near, k) * np.repeat(2.0 ** rng.integers(-126, 125, k // 32), 32)
        w[2, :32] = 0
        w[3, 5], w[4, 40], w[5, 70] = np.nan, np.inf, -np.inf
        w[6] = np.float32(3.4028235e38)
        w[8] = np.float32(1e-45)
        w[9, ::2] = -0.0
    w = w.astype(np.float32)
    dw, q, s = ctx.upload(w), ctx.empty((n, k // 2), np.uint8), ctx.empty((n, k // 32), np.uint8)
    ctx.quantize_e2m1(dw, q, s, n, k)
    ctx.sync()
    code, scale = quantised(w)
    assert (s.to_host() == scale).all()
    assert (q.to_host() == packed(code)).all()
    for b in (dw, q, s):
        b.free()


def run(ctx, code, scale, x, dtype, out, ldx=None, ldy=None):
    n, k = code.shape
    batch = len(x)
    ldx, ldy = ldx or k, ldy or n
    rows = np.full((batch, ldx), np.nan)
    rows[:, :k] = x
    bufs = [ctx.upload(packed(code)), ctx.upload(scale), ctx.alloc(ctx.e2m1_tiles_bytes(n, k)),
            ctx.upload(to16(rows.reshape(-1)[:(batch - 1) * ldx + k], dtype))]
    ctx.memset(bufs[2], 0xff)
    fill = np.full((batch, ldy), 0.5, np.float32)
    y = ctx.upload(fill if out == "f32" else to16(fill, dtype))
    ctx.pack_e2m1_tiles(bufs[0], bufs[1], bufs[2], n, k)
    ctx.gemv_w4a16(bufs[3], bufs[2], y, batch, k, n, dtype=dtype, out=out, ldx=ldx, ldy=ldy)
    ctx.sync()
    got = y.to_host()
    got = got.astype(np.float64) if out == "f32" else from16(got, dtype)
    for b in bufs + [y]:
        b.free()
    assert (got[:, n:] == 0.5).all(), "between the rows"
    return got[:, :n]


def check(got, code, scale, x, dtype, out):
    w = values(code, scale)
    with np.errstate(invalid="ignore", over="ignore"):
        ref = x @ w.T
        # k products, each exact, added in some order, with a rounding at each sum and each
        # group's scaling; below fp32's normal range steps of 2^-149 each
        tol = (code.shape[1] + 40) * F * (np.abs(x) @ np.abs(w).T) + code.shape[1] * 2.0 ** -149
        if out != "f32":
            tol += U[dtype] * np.abs(ref) + (2.0 ** -25 if dtype == "f16" else 2.0 ** -134)
        most = {"f32": 3.4028236e38, "f16": 65520.0, "bf16": 3.3961775e38}["f32" if out == "f32" else dtype]
        ref = np.where(np.abs(ref) >= most, np.sign(ref) * np.inf, ref)
        good = (got == ref) | (np.isnan(got) & np.isnan(ref)) | (np.abs(got - ref) <= tol)
        # where the sizes of the products add up beyond fp32's largest, 2^128 - 2^104, so may some
        # of the sums, which are infinite then, of either sign, and NaN together
        good |= (np.abs(x) @ np.abs(w).T >= 2.0 ** 128 - 2.0 ** 104) & ~np.isfinite(got)
    at = np.argwhere(~good)
    assert good.all(), (len(at), at[:5], got[tuple(at[0])], ref[tuple(at[0])], tol[tuple(at[0])])


def random_weights(rng, n, k, around=-7, spread=3):
    code = rng.integers(0, 16, (n, k)).astype(np.uint8)
    return code, (127 + around + rng.integers(-spread, spread + 1, (n, k // 32))).astype(np.uint8)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("out", ["f32", "16"])
@pytest.mark.parametrize("n,k", [(1, 32), (15, 64), (16, 128), (17, 160), (33, 992), (100, 4128), (1030, 1024)])
@pytest.mark.parametrize("batch", [1, 2, 4, 5, 8, 9, 16, 17, 33, 48, 49, 64])
def test_products(ctx, dtype, out, n, k, batch):
    rng = np.random.default_rng(n + k + batch)
    out = "f32" if out == "f32" else dtype
    code, scale = random_weights(rng, n, k)
    x = from16(to16(rng.normal(0, 1, (batch, k)), dtype), dtype)
    check(run(ctx, code, scale, x, dtype, out), code, scale, x, dtype, out)


@pytest.mark.parametrize("n,k,batch", [(151_936 // 8, 1024, 1), (40_000, 96, 3), (16, 65_536, 2), (3000, 8160, 37), (40_000, 96, 9),
                                       (20_001, 1184, 40), (40_000, 160, 48), (40_000, 160, 64), (40_000, 96, 20), (70_000, 544, 6)])
def test_products_of_large_matrices(ctx, n, k, batch):
    rng = np.random.default_rng(n)
    code, scale = random_weights(rng, n, k)
    x = from16(to16(rng.normal(0, 1, (batch, k)), "bf16"), "bf16")
    check(run(ctx, code, scale, x, "bf16", "f32"), code, scale, x, "bf16", "f32")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("batch", [1, 7, 40])
def test_strides(ctx, dtype, batch):
    # NaN between the rows of x, values that stay between those of y
    rng = np.random.default_rng(batch)
    code, scale = random_weights(rng, 70, 224)
    x = from16(to16(rng.normal(0, 1, (batch, 224)), dtype), dtype)
    check(run(ctx, code, scale, x, dtype, "f32", ldx=248, ldy=75), code, scale, x, dtype, "f32")
    check(run(ctx, code, scale, x, dtype, dtype, ldx=232, ldy=71), code, scale, x, dtype, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("batch", [1, 20])
def test_scales_of_any_size(ctx, dtype, batch):
    # beyond the 16-bit types' ranges, at fp32's ends, NaN; groups of zeros under any of them
    rng = np.random.default_rng(batch)
    n, k = 96, 480
    code, scale = random_weights(rng, n, k)
    g = code.reshape(n, -1, 32)
    scale[0:16, 3] = rng.integers(80, 110, 16)
    scale[16:32] = rng.integers(135, 160, (16, k // 32))
    scale[33, 7] = 255
    scale[34, 0], code[34] = 255, 0
    scale[48:64], scale[50] = rng.integers(0, 6, (16, k // 32)), 0
    scale[64:70], scale[70] = 0, 254
    code[70] = 0
    code[70, 5] = 1  # (one product: the sum of several may pass through infinity)
    g[64:70, 1::2] = 8
    scale[65, 1::2], scale[66, 1::2] = 254, 0
    x = rng.normal(0, 1, (batch, k))
    if dtype == "bf16":
        x[0] *= 2.0 ** 100
    x = from16(to16(x, dtype), dtype)
    check(run(ctx, code, scale, x, dtype, "f32"), code, scale, x, dtype, "f32")


def test_large_activations_by_small_weights(ctx):
    # products with weights of another size would leave fp32's range
    rng = np.random.default_rng(5)
    code, scale = random_weights(rng, 32, 256, around=-100, spread=20)
    x = from16(to16(rng.normal(0, 1, (3, 256)) * 2.0 ** 125, "bf16"), "bf16")
    check(run(ctx, code, scale, x, "bf16", "f32"), code, scale, x, "bf16", "f32")


@pytest.mark.parametrize("dtype,size", [("f16", 2.0 ** -17), ("f16", 2.0 ** -22), ("bf16", 2.0 ** -122), ("bf16", 2.0 ** -130)])
def test_activations_below_the_normal_range(ctx, dtype, size):
    rng = np.random.default_rng(8)
    code, scale = random_weights(rng, 32, 256, around=3)
    x = from16(to16(rng.normal(0, 1, (3, 256)) * size, dtype), dtype)
    check(run(ctx, code, scale, x, dtype, "f32"), code, scale, x, dtype, "f32")


def test_activations_that_are_not_finite(ctx):
    rng = np.random.default_rng(6)
    code, scale = random_weights(rng, 40, 96)
    code[code % 8 == 0] = 3  # (0 times infinity apart: row 5)
    code[5, 10] = 0
    x = rng.normal(0, 1, (6, 96))
    x[1, 10], x[2, 95], x[4, 3] = np.inf, np.nan, -np.inf
    x = from16(to16(x, "f16"), "f16")
    check(run(ctx, code, scale, x, "f16", "f32"), code, scale, x, "f16", "f32")


def test_quantised_then_multiplied(ctx):
    # as a program does: fp32 weights to products, against the weights themselves
    rng = np.random.default_rng(7)
    n, k = 50, 320
    w = rng.normal(0, 0.02, (n, k)).astype(np.float32)
    x = to16(rng.normal(0, 1, (2, k)), "f16")
    dw, q, s, t = ctx.upload(w), ctx.alloc(n * k // 2), ctx.alloc(n * k // 32), ctx.alloc(ctx.e2m1_tiles_bytes(n, k))
    dx, y = ctx.upload(x), ctx.empty((2, n), np.float32)
    ctx.quantize_e2m1(dw, q, s, n, k)
    ctx.pack_e2m1_tiles(q, s, t, n, k)
    ctx.gemv_w4a16(dx, t, y, 2, k, n)
    ctx.sync()
    xf = from16(x, "f16")
    code, scale = quantised(w)
    check(y.to_host().astype(np.float64), code, scale, xf, "f16", "f32")
    # a value of its group of size up to 6 2^e is off by 2^e at most (between 4 and 6)
    off = np.repeat(2.0 ** (scale.astype(int) - 127), 32, 1)
    assert (np.abs(y.to_host() - xf @ w.T) <= np.abs(xf) @ off.T * 1.001).all()
    for b in (dw, q, s, t, dx, y):
        b.free()


def refused(call, text):
    with pytest.raises(strict_amd.StrictHipError) as e:
        call()
    assert e.value.status == strict_amd.SH_ERR_INVALID_ARGUMENT and text in e.value.message, e.value.message


def test_refusals(ctx):
    n, k, batch = 40, 96, 3
    w, q, s = ctx.alloc(n * k * 4), ctx.alloc(n * k // 2), ctx.alloc(n * k // 32)
    size = ctx.e2m1_tiles_bytes(n, k)
    t, x, y = ctx.alloc(size), ctx.alloc(batch * k * 2), ctx.alloc(batch * n * 4)
    off = lambda b, by=8: b.view(by, b.nbytes - by)  # noqa: E731
    for bad, text in ((0, "K"), (-32, "K"), (48, "K"), ((1 << 24) + 32, "K")):
        refused(lambda: ctx.quantize_e2m1(w, q, s, n, bad), text)
        refused(lambda: ctx.e2m1_tiles_bytes(n, bad), text)
        refused(lambda: ctx.pack_e2m1_tiles(q, s, t, n, bad), text)
        refused(lambda: ctx.gemv_w4a16(x, t, y, batch, bad, n), text)
    for bad in (-1, (1 << 28) + 1):
        refused(lambda: ctx.quantize_e2m1(w, q, s, bad, k), "N")
        refused(lambda: ctx.gemv_w4a16(x, t, y, batch, k, bad, ldy=1 << 30), "N")
    for bad in (0, -1, 65):
        refused(lambda: ctx.gemv_w4a16(x, t, y, bad, k, n), "batch")
    refused(lambda: ctx.gemv_w4a16(x, t, y, batch, k, n, ldx=k - 8), "ldx")
    refused(lambda: ctx.gemv_w4a16(x, t, y, batch, k, n, ldx=k + 4), "ldx")
    refused(lambda: ctx.gemv_w4a16(x, t, y, batch, k, n, ldy=n - 1), "ldy")
    refused(lambda: ctx.quantize_e2m1(off(w), q, s, n - 1, k), "16-byte")
    refused(lambda: ctx.quantize_e2m1(w, off(q), s, n - 1, k), "16-byte")
    refused(lambda: ctx.pack_e2m1_tiles(off(q, 2), s, t, n - 1, k), "4-byte")
    refused(lambda: ctx.pack_e2m1_tiles(q, s, off(t), 16, k), "16-byte")
    refused(lambda: ctx.gemv_w4a16(off(x), t, y, batch - 1, k, n), "16-byte")
    refused(lambda: ctx.gemv_w4a16(x, off(t), y, batch, k, 16), "16-byte")
    refused(lambda: ctx.gemv_w4a16(x, t, off(y, 2), batch - 1, k, n), "aligned")
    refused(lambda: ctx.gemv_w4a16(x, t, off(y, 1), batch - 1, k, n, out="f16"), "aligned")
    # extents
    refused(lambda: ctx.quantize_e2m1(w, q, s, n + 1, k), "W")
    refused(lambda: ctx.pack_e2m1_tiles(q, s, t, n + 16, k), "q")
    refused(lambda: ctx.gemv_w4a16(x, t, y, batch + 1, k, n), "x")
    refused(lambda: ctx.gemv_w4a16(x, t, y, batch, k, n + 16), "w_tiled")
    refused(lambda: ctx.gemv_w4a16(x, t, y, batch, k, n, ldy=n + 1), "y")
    refused(lambda: ctx.gemv_w4a16(x, None, y, batch, k, n), "w_tiled")
    # over one another
    refused(lambda: ctx.quantize_e2m1(w, w.view(256, n * k // 2), s, n, k), "overlap")
    refused(lambda: ctx.quantize_e2m1(w, q, q.view(16, n * k // 32), n, k), "overlap")
    area = ctx.alloc(size + n * k)
    refused(lambda: ctx.pack_e2m1_tiles(area.view(size - 16, n * k // 2), s, area, n, k), "overlaps")
    refused(lambda: ctx.pack_e2m1_tiles(q, area.view(size - 4, n * k // 32), area, n, k), "overlaps")
    refused(lambda: ctx.gemv_w4a16(x, t, x, 1, k, n), "overlaps")
    refused(lambda: ctx.gemv_w4a16(x, area, area.view(0, batch * n * 4), batch, k, n), "overlaps")
    with pytest.raises(ValueError):
        ctx.gemv_w4a16(x, t, y, batch, k, n, dtype="f32")
    with pytest.raises(ValueError):
        ctx.gemv_w4a16(x, t, y, batch, k, n, dtype="f16", out="bf16")
    ctx.quantize_e2m1(None, None, None, 0, k)  # nothing to do
    ctx.pack_e2m1_tiles(None, None, None, 0, k)
    ctx.gemv_w4a16(None, None, None, 1, k, 0)
    for b in (w, q, s, t, x, y, area):
        b.free()
