"""sh_sample_f32 against its definition in 64 bits (numpy).

The token has to be the same. Where a border (u times the sum, top-p's limit)
lies within 1e-9 of the sum of a cumulated weight, both its sides are right: the
kernel's weights are rounded to 2^-43 of the largest (2^20 of them: 2^-23 at
most, but of errors that are as often up as down, so below 2^-33 of a sum that is
at least 1) and fp64 sums in another order differ by less.
"""
import numpy as np
import pytest

import strict_amd

pytestmark = pytest.mark.gpu

NEAR = 1e-9


def oracle(x, t, k, p, least, u):
    """The set of tokens that are right for one row."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return {-1}
    order = np.argsort(-x, kind="stable")
    if not t > 0 or k == 1:
        return {int(order[0])}
    with np.errstate(invalid="ignore", over="ignore"):
        y = np.where(x == top, 0.0, (top - x) / np.float64(t))
    w = np.where(np.isfinite(y), np.exp(-np.where(np.isfinite(y), y, 0)), 0.0)
    kept = order[:k] if 0 < k < len(x) else order
    kept = kept[w[kept] > 0]
    choices = [len(kept)]
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(w[kept])[:-1]]) / w[kept].sum()
        n = max(1, int((before < p).sum()))
        choices = {n} | {i for i in (n - 1, n, n + 1) if 1 <= i <= len(kept) and abs(before[min(i, len(kept) - 1)] - p) < NEAR}
    right = set()
    least = min(float(least), 1.0) if least > 0 else 0.0
    u = min(float(u), 1.0) if u > 0 else 0.0
    for n in choices:
        some = np.sort(kept[:n][w[kept[:n]] >= least])
        c = np.cumsum(w[some])
        c /= c[-1]
        for target in {max(u - NEAR, 0.0) if u < 1 else u, u, u + NEAR if u > 0 else 0.0}:
            right.add(int(some[min(int(np.searchsorted(c, target, side="right")), len(some) - 1)]))
    return right


def sample(ctx, x, t, k, p, least, u, ld=None, n=None):
    rows, n = len(u), x.shape[1] if n is None else n
    f32 = lambda v: None if v is None else ctx.upload(np.asarray(v, np.float32))  # noqa: E731
    bufs = [ctx.upload(x), f32(t), None if k is None else ctx.upload(np.asarray(k, np.int32)), f32(p), f32(least), f32(u)]
    index = ctx.upload(np.full(rows + 1, -77, np.int32))
    work = ctx.alloc(ctx.sample_workspace(rows, n))
    ctx.memset(work, 0xa5)
    got = []
    for _ in range(2):  # the second on a used work buffer
        ctx.sample(bufs[0], rows, n, *bufs[1:], index, work, ld)
        ctx.sync()
        got.append(index.to_host())
    assert (got[0] == got[1]).all() and got[0][rows] == -77
    for b in bufs + [index, work]:
        if b is not None:
            b.free()
    return got[0][:rows]


def check(ctx, x, t, k, p, least, u, ld=None, n=None):
    got = sample(ctx, x, t, k, p, least, u, ld, n)
    one = lambda v, r, d: d if v is None else np.asarray(v, np.float32)[r]  # noqa: E731
    for r in range(len(u)):
        row = x[r] if n is None else x[r, :n]
        right = oracle(row, one(t, r, 1.0), 0 if k is None else int(k[r]), one(p, r, 1.0), one(least, r, 0.0),
                       np.float32(u[r]))
        assert int(got[r]) in right, (r, int(got[r]), right, one(t, r, 1.0), None if k is None else k[r],
                                      one(p, r, 1.0), one(least, r, 0.0), u[r])


SIZES = [1, 2, 3, 63, 64, 257, 2047, 2048, 2049, 5000, 50257, 151936]


@pytest.mark.parametrize("n", SIZES)
@pytest.mark.parametrize("ties", [False, True])
def test_parameters(ctx, n, ties):
    rng = np.random.default_rng(n)
    rows = 48 if n < 50000 else 24
    x = rng.normal(0, 2.5, (rows, n)).astype(np.float32)
    likely = rng.integers(0, n, (rows, 30))
    for r in range(rows):
        x[r, likely[r]] += rng.uniform(0, 12, 30).astype(np.float32)
    if ties:
        x = (np.round(x * 8) / 8).astype(np.float32)
    check(ctx, x, rng.choice([0.0, 0.2, 0.7, 1.0, 1.5, 5.0], rows), rng.choice([0, -1, 1, 2, 20, 50, 1000, 4000, n, n + 5], rows),
          rng.choice([1.0, 0.99, 0.95, 0.5, 0.1, 0.0, 1.5], rows), rng.choice([0.0, 0.01, 0.1, 1.0, 2.0, -1.0], rows),
          rng.random(rows).astype(np.float32))


@pytest.mark.parametrize("n", [40, 3000, 151936])
def test_defaults_and_row_stride(ctx, n):
    rng = np.random.default_rng(n + 1)
    x = rng.normal(0, 3, (7, n + 5)).astype(np.float32)
    x[:, n:] = 1000  # (not of the row)
    u = rng.random(7).astype(np.float32)
    check(ctx, x, None, None, None, None, u, ld=n + 5, n=n)
    check(ctx, x, None, np.full(7, 9), None, None, u, ld=n + 5, n=n)
    check(ctx, x, None, None, np.full(7, 0.6), None, u, ld=n + 5, n=n)
    check(ctx, x, None, None, None, np.full(7, 0.3), u, ld=n + 5, n=n)


@pytest.mark.parametrize("n", [30, 2500, 60000])
def test_uniform_numbers_at_their_ends(ctx, n):
    rng = np.random.default_rng(n + 2)
    x = rng.normal(0, 1, (8, n)).astype(np.float32)
    x[:, [0, 1, n - 1]] = -np.inf
    u = np.array([0.0, 1.0, 1 - 2.0 ** -24, 2.0 ** -149, -3.0, 7.0, np.nan, 0.5], np.float32)
    got = sample(ctx, x, None, None, None, None, u)
    assert got[0] == got[3] == got[4] == got[6] == 2 and got[1] == got[5] == n - 2
    check(ctx, x[[2, 7]], None, None, None, None, u[[2, 7]])


@pytest.mark.parametrize("n", [10, 2100, 70000])
def test_masked_infinite_and_missing_values(ctx, n):
    rng = np.random.default_rng(n + 3)
    x = rng.normal(0, 2, (9, n)).astype(np.float32)
    lowest = np.finfo(np.float32).min
    x[0, :] = -np.inf
    x[1, :] = np.nan
    x[2, :] = lowest  # (a row of the type's lowest: all alike)
    x[3, :] = lowest
    x[3, n // 2] = -3
    x[4, rng.integers(0, n, n // 3)] = np.nan
    x[5, [n - 1, n // 2]] = np.inf
    x[6, :] = -np.inf
    x[6, n - 2] = lowest
    x[7, ::2] = -np.inf
    x[7, 1::2] = np.float32(3e38)
    x[8, :] = 0.0
    x[8, ::3] = -0.0
    rows = 9
    u = rng.random(rows).astype(np.float32)
    for t in (0.0, 1e-30, 1.0, 1e30, np.inf, np.nan):
        for k, p in ((None, None), (np.full(rows, 7), None), (None, np.full(rows, 0.7)), (np.full(rows, 7), np.full(rows, 0.7))):
            check(ctx, x, np.full(rows, t), k, p, None, u)
    got = sample(ctx, x, None, None, None, None, u)
    assert got[0] == got[1] == -1 and got[5] in (n - 1, n // 2) and got[6] == n - 2 and got[3] == n // 2


@pytest.mark.parametrize("n", [2300, 40000, 200001])
def test_more_equal_values_than_the_list_holds(ctx, n):
    # all alike, and a few values of many tokens each
    rng = np.random.default_rng(n + 4)
    x = np.concatenate([np.zeros((6, n)), rng.integers(0, 3, (6, n)) * 0.5]).astype(np.float32)
    rows = 12
    u = rng.random(rows).astype(np.float32)
    k = np.tile([0, 2200, 5, 0, n - 3, 2100], 2)
    p = np.tile([0.5, 1.0, 1.0, 0.999, 0.9, 0.3], 2)
    check(ctx, x, np.ones(rows), k, p, np.tile([0, 0.5], 6), u)


def test_flat_rows_by_digits(ctx):
    # high temperature: the selection ends among close values, past what the list holds
    rng = np.random.default_rng(8)
    x = rng.normal(0, 2.5, (8, 151936)).astype(np.float32)
    check(ctx, x, np.full(8, 40.0), [3000, 50000, 0, 0, 100000, 2049, 5000, 0], [0.9, 0.5, 0.5, 0.99, 1.0, 0.3, 1.0, 0.01],
          [0, 0, 0.8, 0, 0.9, 0, 0, 0], rng.random(8).astype(np.float32))


def test_largest_row(ctx):
    rng = np.random.default_rng(9)
    n = 1 << 20
    x = rng.normal(0, 1, (3, n)).astype(np.float32)
    x[1] = 0
    check(ctx, x, np.ones(3), [0, 0, n - 1], [1.0, 0.5, 0.9], [0, 0, 0], np.array([0.999, 0.7, 0.2], np.float32))


@pytest.mark.parametrize("rows", [1, 300, 2000])
def test_many_rows(ctx, rows):
    rng = np.random.default_rng(rows)
    x = rng.normal(0, 2, (rows, 2500)).astype(np.float32)
    check(ctx, x, rng.choice([0.0, 0.8], rows), rng.choice([0, 10], rows), rng.choice([1.0, 0.9], rows), None,
          rng.random(rows).astype(np.float32))


def test_frequencies(ctx):
    # u over a fine grid hits each token as often as its probability says
    x = np.log(np.array([[1, 2, 3, 4]], np.float32)).repeat(1000, 0)
    got = sample(ctx, x, None, None, None, None, (np.arange(1000) + 0.5) / 1000)
    assert np.bincount(got, minlength=4).tolist() == [100, 200, 300, 400]


def test_refusals(ctx):
    x, row = ctx.upload(np.zeros((2, 3000), np.float32)), ctx.upload(np.zeros(2, np.float32))
    index = ctx.upload(np.zeros(2, np.int32))
    work = ctx.alloc(ctx.sample_workspace(2, 3000))

    def refused(text, x=x, rows=2, n=3000, t=row, k=row, p=row, least=row, u=row, index=index, work=work, ld=None):
        with pytest.raises(strict_amd.StrictHipError) as e:
            ctx.sample(x, rows, n, t, k, p, least, u, index, work, ld)
        assert e.value.status == strict_amd.SH_ERR_INVALID_ARGUMENT and text in e.value.message, e.value.message

    refused("n must be", n=0)
    refused("n must be", n=(1 << 20) + 1)
    refused("rows", rows=-1)
    refused("ld", ld=2999)
    refused("x", ld=3001)
    refused("x is NULL", x=None)
    refused("u is NULL", u=None)
    refused("index is NULL", index=None)
    short = row.view(0, 4)
    for name in ("t", "k", "p", "least", "u", "index"):
        host = ctx.alloc(4)
        refused("not inside", **{name: host})
        host.free()
    refused("work buffer", work=work.view(0, work.nbytes - 16))
    refused("aligned", work=ctx.alloc(work.nbytes + 8).view(8, work.nbytes))
    ctx.sample(x, 0, 3000, None, None, None, None, None, None, work)
    assert short.nbytes == 4
    for b in (x, row, index, work):
        b.free()
