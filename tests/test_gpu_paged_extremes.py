"""Attention over pages where fp32 runs out: scores far beyond the exponent's range,
values whose sums do. What the rows are is known, or as in test_gpu_paged.py."""
import numpy as np
import pytest

import test_gpu_paged as paged

pytestmark = pytest.mark.gpu


def pointed(seed, ctx, dtype, new, lengths, at, size=1.0):
    """A case whose query rows all point where position `at` of each sequence's k does:
    its product with them is 250 size^2 or more, of the others no more than a third of that."""
    c = paged.Case(ctx, seed, dtype, new, lengths, 4, 2, 128, 16)
    way = c.rng.choice([-1.0, 1.0], 128)
    k = paged.from16(c.k, dtype)
    for b, p in enumerate(at):
        k[c.table[b, p // 16], :, p % 16] = 2 * way
    c.k[:] = paged.to16(k * size, dtype)
    q = way * (1 + np.abs(c.rng.normal(0, 0.2, (c.tokens, 4, 128)))) * size
    return c, paged.to16(q, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new,lengths,at", [([1, 1], [600, 40], [123, 39]), ([40, 3], [600, 90], [7, 80]),
                                            ([1], [9000], [4321])])
@pytest.mark.parametrize("log2", [14, 16, 18, 20, 21, 22, 26, 30, 36, 60, 119, 126])
def test_one_score_far_above_the_others(ctx, dtype, new, lengths, at, log2):
    # (by 100 times the scale and more: the others have no weight)
    c, q = pointed(log2, ctx, dtype, new, lengths, at)
    _, got = paged.run_attention(c, q=q, scale=float(np.float32(c.rng.uniform(1, 2) * 2.0 ** log2)))
    for b, p in enumerate(at):
        v = c.v[c.table[b, p // 16], :, p % 16].repeat(2, 0)
        assert (got[c.starts[b]:c.starts[b] + new[b]] == v).all(), b


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new,lengths,at", [([1, 1], [600, 40], [123, 39]), ([40, 3], [600, 90], [7, 80])])
@pytest.mark.parametrize("log2", [16, 30, 119, 126])
def test_the_least_of_large_negative_scores(ctx, dtype, new, lengths, at, log2):
    # (products with the scale below fp32's range among them)
    c, q = pointed(log2, ctx, dtype, new, lengths, at)
    way = np.sign(paged.from16(q, dtype)[0, 0])
    k = np.broadcast_to(-2 * way, c.k.shape).copy()
    for b, p in enumerate(at):
        k[c.table[b, p // 16], :, p % 16] = -way
    c.k[:] = paged.to16(k, dtype)
    _, got = paged.run_attention(c, q=q, scale=float(np.float32(c.rng.uniform(1, 2) * 2.0 ** log2)))
    for b, p in enumerate(at):
        v = c.v[c.table[b, p // 16], :, p % 16].repeat(2, 0)
        assert (got[c.starts[b]:c.starts[b] + new[b]] == v).all(), b


@pytest.mark.parametrize("new,lengths,at", [([1], [700], [123]), ([40], [700], [600])])
@pytest.mark.parametrize("dtype,size", [("f16", 2.0 ** 10), ("f16", 2.0 ** 13), ("bf16", 2.0 ** 18), ("bf16", 2.0 ** 55)])
def test_large_queries_and_keys(ctx, dtype, size, new, lengths, at):
    c, q = pointed(int(np.log2(size)), ctx, dtype, new, lengths, at, size)
    _, got = paged.run_attention(c, q=q)
    v = c.v[c.table[0, at[0] // 16], :, at[0] % 16].repeat(2, 0)
    assert (got[c.starts[0]:c.starts[0] + new[0]] == v).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new,lengths", [([1, 1], [600, 5]), ([40, 3], [600, 90]), ([1], [20000])])
@pytest.mark.parametrize("log2", [-40, 0, 8, 12, 13, 14, 15, 16, 19, 20, 21, 22, 26, 40, 100, 118, 126])
def test_equal_scores_far_from_zero(ctx, dtype, new, lengths, log2):
    # about 300 times the scale, and less that: means of the values
    for sign in (1, -1):
        c, q = pointed(log2 + 50, ctx, dtype, new, lengths, [0] * len(new))
        way = np.sign(paged.from16(q, dtype)[0, 0])
        c.k[:] = paged.to16(np.broadcast_to(sign * 2 * way, c.k.shape), dtype)
        _, got = paged.run_attention(c, q=q, scale=float(np.float32(c.rng.uniform(1, 2) * 2.0 ** log2)))
        c.k[:] = 0
        ref, tol = paged.attention_oracle(c, paged.from16(q, dtype), 0, 0, 1.0)
        n = sum(new)
        assert (np.abs(paged.from16(got, dtype) - ref)[:n] <= tol[:n]).all(), sign


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new,lengths", [([1], [600]), ([40], [600])])
@pytest.mark.parametrize("base", [-2.0 ** 23, -2.0 ** 19, 2.0 ** 12, 2.0 ** 19, 2.0 ** 22, 2.0 ** 23])
def test_close_scores_far_from_zero(ctx, dtype, new, lengths, base):
    # whole numbers base + 0 .. 9, exact in fp32: the weights are those of 0 .. 9
    c = paged.Case(ctx, 5, dtype, new, lengths, 4, 2, 64, 16)
    some = c.rng.integers(0, 10, c.k.shape[:3])
    k = np.zeros(c.k.shape)
    k[..., 0], k[..., 1] = some, 64
    c.k[:] = paged.to16(k, dtype)
    q = np.zeros((c.tokens, 4, 64))
    q[..., 0], q[..., 1] = 1, base / 64
    ones = np.zeros((c.tokens, 4, 64))
    ones[..., 0] = 1
    if abs(base) / 64 > 60000:  # (fp16)
        k[..., 1:9], q[..., 1:9] = 64, base / 512
        c.k[:] = paged.to16(k, dtype)
    _, got = paged.run_attention(c, q=paged.to16(q, dtype), scale=1.0)
    c.k[:] = paged.to16(np.where(np.arange(64) == 0, k, 0), dtype)
    ref, tol = paged.attention_oracle(c, ones, 0, 0, 1.0)
    out = paged.from16(got, dtype)
    n = sum(new)
    assert (np.abs(out - ref)[:n] <= tol[:n]).all()


@pytest.mark.parametrize("new,lengths", [([1, 1], [600, 40]), ([40, 9], [600, 300]), ([1], [20000])])
@pytest.mark.parametrize("top", [2.0 ** 110, 2.0 ** 122, 2.0 ** 125])
def test_values_whose_sums_leave_the_range(ctx, new, lengths, top):
    c = paged.Case(ctx, 7, "bf16", new, lengths, 4, 2, 128, 16)
    c.v[:] = paged.to16(np.clip(paged.from16(c.v, "bf16"), -7, 7) * top, "bf16")
    paged.check_attention(c)
    c.v[:] = paged.to16(np.full(c.v.shape, 2.0 ** 127), "bf16")
    _, got = paged.run_attention(c)
    n = sum(new)
    assert (got[:n] == paged.to16([2.0 ** 127], "bf16")).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new,lengths", [([1], [600]), ([1, 1, 1], [1000, 77, 3]), ([40, 9], [600, 300])])
@pytest.mark.parametrize("d", [64, 128])
def test_values_that_are_all_alike(ctx, dtype, new, lengths, d):
    # a mean of one value is that value, whatever the weights are rounded to: sums of at most
    # 1,000 of them, in fp32 off by less than 2,016 2^-24 = 2^-13, are rounded back to it. One
    # position's score is above all others', which are one another's: their roundings do not
    # average out.
    c = paged.Case(ctx, 6, dtype, new, lengths, 16, 2, d, 16)
    value = paged.to16(c.rng.uniform(1, 2, (2, 1, d)) * c.rng.choice([-1, 1], (2, 1, d)), dtype)
    c.v[:] = value
    k = np.zeros(c.k.shape)
    for b in range(c.batch):
        k[c.table[b, 0], :, 0, 0] = 1
    c.k[:] = paged.to16(k, dtype)
    q = np.zeros((c.tokens, 16, d))
    q[..., 0] = c.rng.uniform(0, 3, (c.tokens, 16))
    _, got = paged.run_attention(c, q=paged.to16(q, dtype), scale=1.0)
    n = sum(new)
    assert (got[:n] == value[:, 0].repeat(8, 0)).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new,lengths", [([1], [20000]), ([40], [20000])])
@pytest.mark.parametrize("above", [4.0, 10.0, 16.0])
def test_many_small_weights(ctx, dtype, new, lengths, above):
    # one position far above the others, whose weights (in fp16 below the normal range) carry the values
    c = paged.Case(ctx, 8, dtype, new, lengths, 4, 2, 64, 16)
    k, v = np.zeros(c.k.shape), np.ones(c.v.shape)
    at = c.table[0, 9000 // 16], 9000 % 16
    k[at[0], :, at[1], 0] = above
    v[at[0], :, at[1]] = 0
    c.k[:], c.v[:] = paged.to16(k, dtype), paged.to16(v, dtype)
    q = np.zeros((c.tokens, 4, 64))
    q[..., 0] = 1
    paged.check_attention(c, q=paged.to16(q, dtype), scale=1.0)
