"""Attention over pages of 8-bit values where fp32 runs out, and where some rows of a tile
are not numbers: tiles that are cut, that are not, and those of two halves. The rows are
known, or those of test_gpu_paged.py's oracle."""
import numpy as np
import pytest

import test_gpu_paged as paged
from test_gpu_paged import from16, to16
from test_gpu_paged8 import Case8

pytestmark = pytest.mark.gpu

# Chunks: tables of up to 1,152 positions and few tiles (two halves), with 130 sequences more
# that have no tokens (a workgroup of one half a tile), with 300 pages more (cut). Single tokens: the
# latter two.
CHUNKS, TOKENS = ["halves", "whole", "cut"], ["whole", "cut"]


def case(seed, ctx, dtype, variant, new, lengths, heads=4, d=128):
    more = 130 if variant == "whole" else 0
    return Case8(ctx, seed, dtype, list(new) + [0] * more, list(lengths) + [0] * more, heads, 2, d, 16,
                 extra_entries=300 if variant == "cut" else 1)


def variants(*cases):
    """(variant, *case) of each case, whose first entry is its new tokens."""
    return [(v, *c) for c in cases for v in (CHUNKS if max(c[0]) > 8 else TOKENS)]


def put(c, k=None, v=None):
    """Other values, also after a call."""
    c.sent = None
    if k is not None:
        c.k = to16(np.broadcast_to(k, c.kb.shape), c.dtype)
    if v is not None:
        c.v = to16(np.broadcast_to(v, c.vb.shape), c.dtype)


def check_rows(c, got, at, new):
    for b, p in enumerate(at):
        v = c.v[c.table[b, p // 16], :, p % 16].repeat(2, 0)
        assert (got[c.starts[b]:c.starts[b] + new[b]] == v).all(), b


def pointed(seed, ctx, dtype, variant, new, lengths, at, size=1.0):
    """A case whose query rows all point where position `at` of each sequence's k does:
    its product with them is 250 size^2 or more, of the others no more than a third of that."""
    c = case(seed, ctx, dtype, variant, new, lengths)
    way = c.rng.choice([-1.0, 1.0], 128)
    k = from16(c.k, dtype)
    for b, p in enumerate(at):
        k[c.table[b, p // 16], :, p % 16] = 2 * way
    put(c, k * size)
    q = way * (1 + np.abs(c.rng.normal(0, 0.2, (c.tokens, 4, 128)))) * size
    return c, to16(q, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("variant,new,lengths,at", variants(([1, 1], [600, 40], [123, 39]), ([40, 3], [600, 90], [7, 80]),
                                                            ([40, 3], [600, 90], [403, 80])))
@pytest.mark.parametrize("log2", [14, 21, 30, 60, 126])
def test_one_score_far_above_the_others(ctx, dtype, variant, new, lengths, at, log2):
    # (by 100 times the scale and more: the others have no weight)
    c, q = pointed(log2, ctx, dtype, variant, new, lengths, at)
    _, got = paged.run_attention(c, q=q, scale=float(np.float32(c.rng.uniform(1, 2) * 2.0 ** log2)))
    check_rows(c, got, at, new)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("variant,new,lengths,at", variants(([1, 1], [600, 40], [123, 39]), ([40, 3], [600, 90], [7, 80]),
                                                            ([40, 3], [600, 90], [403, 80])))
@pytest.mark.parametrize("log2", [16, 30, 126])
def test_the_least_of_large_negative_scores(ctx, dtype, variant, new, lengths, at, log2):
    # (products with the scale below fp32's range among them)
    c, q = pointed(log2, ctx, dtype, variant, new, lengths, at)
    way = np.sign(from16(q, dtype)[0, 0])
    k = np.broadcast_to(-2 * way, c.kb.shape).copy()
    for b, p in enumerate(at):
        k[c.table[b, p // 16], :, p % 16] = -way
    put(c, k)
    _, got = paged.run_attention(c, q=q, scale=float(np.float32(c.rng.uniform(1, 2) * 2.0 ** log2)))
    check_rows(c, got, at, new)


@pytest.mark.parametrize("variant,new,lengths,at", variants(([1], [700], [123]), ([40], [700], [600])))
@pytest.mark.parametrize("dtype,size", [("f16", 2.0 ** 13), ("bf16", 2.0 ** 18), ("bf16", 2.0 ** 55)])
def test_large_queries_and_keys(ctx, dtype, size, variant, new, lengths, at):
    c, q = pointed(int(np.log2(size)), ctx, dtype, variant, new, lengths, at, size)
    _, got = paged.run_attention(c, q=q)
    check_rows(c, got, at, new)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("variant,new,lengths", variants(([1, 1], [600, 5]), ([40, 3], [600, 90])))
@pytest.mark.parametrize("log2", [0, 13, 16, 22, 40, 126])
def test_equal_scores_far_from_zero(ctx, dtype, variant, new, lengths, log2):
    # about 300 times the scale, and less that: means of the values
    for sign in (1, -1):
        c, q = pointed(log2 + 50, ctx, dtype, variant, new, lengths, [0] * len(new))
        way = np.sign(from16(q, dtype)[0, 0])
        put(c, sign * 2 * way)
        _, got = paged.run_attention(c, q=q, scale=float(np.float32(c.rng.uniform(1, 2) * 2.0 ** log2)))
        put(c, 0.0)
        ref, tol = paged.attention_oracle(c, from16(q, dtype), 0, 0, 1.0)
        n = sum(new)
        assert (np.abs(from16(got, dtype) - ref)[:n] <= tol[:n]).all(), sign


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("variant,new,lengths", variants(([1], [600]), ([40], [600])))
@pytest.mark.parametrize("base", [-2.0 ** 23, -2.0 ** 19, 2.0 ** 12, 2.0 ** 22, 2.0 ** 23])
def test_close_scores_far_from_zero(ctx, dtype, variant, new, lengths, base):
    # whole numbers base + 0 .. 9, exact in fp32 (0 .. 9 and 64 in a row of E4M3 too): the
    # weights are those of 0 .. 9
    c = case(5, ctx, dtype, variant, new, lengths, d=64)
    k, q, ones = np.zeros(c.kb.shape), np.zeros((c.tokens, 4, 64)), np.zeros((c.tokens, 4, 64))
    k[..., 0], k[..., 1] = c.rng.integers(0, 10, c.kb.shape[:3]), 64
    q[..., 0], q[..., 1] = 1, base / 64
    ones[..., 0] = 1
    if abs(base) / 64 > 60000:  # (fp16)
        k[..., 1:9], q[..., 1:9] = 64, base / 512
    put(c, k)
    assert (from16(c.k, dtype) == k).all()
    _, got = paged.run_attention(c, q=to16(q, dtype), scale=1.0)
    put(c, np.where(np.arange(64) == 0, k, 0))
    ref, tol = paged.attention_oracle(c, ones, 0, 0, 1.0)
    n = sum(new)
    assert (np.abs(from16(got, dtype) - ref)[:n] <= tol[:n]).all()


@pytest.mark.parametrize("variant,new,lengths", variants(([1, 1], [600, 40]), ([40, 9], [600, 300])))
@pytest.mark.parametrize("top", [2.0 ** 110, 2.0 ** 125])
def test_values_whose_sums_leave_the_range(ctx, variant, new, lengths, top):
    c = case(7, ctx, "bf16", variant, new, lengths)
    put(c, v=np.clip(from16(c.v, "bf16"), -7, 7) * top)
    paged.check_attention(c)
    put(c, v=2.0 ** 127)
    _, got = paged.run_attention(c)
    assert (got[:sum(new)] == to16([2.0 ** 127], "bf16")).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("variant,new,lengths", variants(([1, 1, 1], [1000, 77, 3]), ([40, 9], [600, 300])))
@pytest.mark.parametrize("d", [64, 128])
def test_values_that_are_all_alike(ctx, dtype, variant, new, lengths, d):
    # a mean of one value is that value, whatever the weights are rounded to: sums of at most
    # 1,000 of them, in fp32 off by less than 2,016 2^-24 = 2^-13, are rounded back to it. One
    # position's score is above all others', which are one another's.
    c = case(6, ctx, dtype, variant, new, lengths, 16, d)
    put(c, v=c.rng.uniform(1, 2, (2, 1, d)) * c.rng.choice([-1, 1], (2, 1, d)))
    k = np.zeros(c.kb.shape)
    for b in range(len(new)):
        k[c.table[b, 0], :, 0, 0] = 1
    put(c, k)
    q = np.zeros((c.tokens, 16, d))
    q[..., 0] = c.rng.uniform(0, 3, (c.tokens, 16))
    _, got = paged.run_attention(c, q=to16(q, dtype), scale=1.0)
    assert (got[:sum(new)] == c.v[0, :, 0].repeat(8, 0)).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("variant,new,lengths", variants(([1], [1000]), ([40], [1000]), ([1], [20000]), ([40], [20000])))
@pytest.mark.parametrize("above", [4.0, 10.0, 16.0])
def test_many_small_weights(ctx, dtype, variant, new, lengths, above):
    # one position far above the others, whose weights (in fp16 below the normal range) carry the values
    c = case(8, ctx, dtype, variant, new, lengths, d=64)
    k, v = np.zeros(c.kb.shape), np.ones(c.vb.shape)
    p = lengths[0] * 9 // 20
    k[c.table[0, p // 16], :, p % 16, 0] = above
    v[c.table[0, p // 16], :, p % 16] = 0
    put(c, k, v)
    q = np.zeros((c.tokens, 4, 64))
    q[..., 0] = 1
    paged.check_attention(c, q=to16(q, dtype), scale=1.0)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("variant", CHUNKS)
@pytest.mark.parametrize("heads,d", [(4, 128), (32, 64)])
@pytest.mark.parametrize("at", [100, 400, 580])
@pytest.mark.parametrize("which", ["k", "v"])
def test_not_a_number_in_either_half(ctx, dtype, variant, heads, d, at, which):
    # of KV head 0 alone: all rows of its heads see positions 100 (of the first half of a tile's
    # units) and 400 (of the second), those of tokens 20 to 39 position 580; the others' rows are
    # those of the oracle
    c = case(at + heads, ctx, dtype, variant, [40], [600], heads, d)
    page = c.table[0, at // 16]
    if which == "k":
        c.kb[page, 0, at % 16, d // 2] = 127
    else:
        c.vs[page, 0, at % 16] = 255
    paged.check_attention(c)
    paged.check_attention(c, window=70, sinks=120)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("variant,new,lengths", variants(([1, 1, 1], [1000, 77, 3]), ([40, 9], [600, 300])))
def test_the_same_bits_each_time(ctx, dtype, variant, new, lengths):
    c = case(9, ctx, dtype, variant, new, lengths)
    q, first = paged.run_attention(c)
    for _ in range(3):
        assert (paged.run_attention(c, q=q)[1] == first).all()
