"""The operators over a KV cache in pages against their formulas in 64 bits
(numpy), each value within what the roundings of its computation add up to.

u: half a step of the 16-bit type (fp16 2^-11, bf16 2^-8 relative to the value);
f = 2^-24, the same of fp32.
"""
import numpy as np
import pytest
import torch

import strict_amd
from strict_amd import PagedKV

pytestmark = pytest.mark.gpu

U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
F = 2.0 ** -24
TORCH = {"f16": torch.float16, "bf16": torch.bfloat16}


def to16(x, dtype):
    """The values as 16-bit patterns."""
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(TORCH[dtype]).view(torch.int16).numpy()


def from16(bits, dtype):
    return torch.from_numpy(np.ascontiguousarray(bits)).view(TORCH[dtype]).double().numpy()


class Case:
    """A batch over pages in shuffled order, `spare` pages that are no sequence's."""

    def __init__(self, ctx, seed, dtype, new, lengths, heads, kv_heads, d, page, first_row=0, rows_behind=1,
                 spare=2, extra_entries=1, scale=1.0):
        rng = self.rng = np.random.default_rng(seed)
        self.ctx, self.dtype = ctx, dtype
        self.new, self.lengths = list(new), list(lengths)
        self.heads, self.kv_heads, self.d, self.page = heads, kv_heads, d, page
        self.batch = len(self.new)
        need = [-(-max(l, 0) // page) for l in self.lengths]
        self.num_pages = sum(need) + spare
        order = rng.permutation(self.num_pages).astype(np.int32)
        self.max_pages = max(need + [1]) + extra_entries
        self.table = np.full((self.batch, self.max_pages), -1, np.int32)
        at = 0
        for b, k in enumerate(need):
            self.table[b, :k] = order[at:at + k]
            at += k
        self.starts = np.concatenate([[first_row], first_row + np.cumsum(self.new)]).astype(np.int32)
        self.tokens = int(self.starts[-1]) + rows_behind
        shape = (self.num_pages, kv_heads, page, d)
        self.k = to16(rng.normal(0, scale, shape), dtype)
        self.v = to16(rng.normal(0, 1, shape), dtype)

    def upload(self):
        self.buffers = [self.ctx.upload(a) for a in (self.k, self.v, self.table,
                                                     np.array(self.lengths, np.int32), self.starts)]
        self.kv = PagedKV(*self.buffers, batch=self.batch, max_pages=self.max_pages, num_pages=self.num_pages,
                          page_size=self.page, kv_heads=self.kv_heads, head_dim=self.d, dtype=self.dtype)
        return self.kv

    def free(self):
        for b in self.buffers:
            b.free()

    def gathered(self, bits, b, kv_head):
        """k or v of sequence b's positions (garbage where the table has no page), and whether there is one."""
        length = max(self.lengths[b], 0)
        pos = np.arange(length)
        entry = self.table[b, pos // self.page]
        there = (entry >= 0) & (entry < self.num_pages)
        rows = bits[np.where(there, entry, 0), kv_head, pos % self.page]
        return from16(rows, self.dtype), there


def attention_oracle(c, q, window, sinks, scale):
    """The rows of the sequences in 64 bits and how far a value may be off; NaN in unseen places has no effect."""
    ref, tol = np.zeros(q.shape), np.zeros(q.shape)
    u, group = U[c.dtype], c.heads // c.kv_heads
    for b in range(c.batch):
        length = max(c.lengths[b], 0)
        for kvh in range(c.kv_heads):
            k, there = c.gathered(c.k, b, kvh)
            v, _ = c.gathered(c.v, b, kvh)
            for i in range(c.new[b]):
                row, pos = c.starts[b] + i, c.lengths[b] - c.new[b] + i
                p = np.arange(length)
                seen = (p <= pos) & there
                if window:
                    seen &= (p > pos - window) | (p < sinks)
                if not seen.any():
                    continue
                ks, vs = k[seen], v[seen]
                for h in range(kvh * group, (kvh + 1) * group):
                    with np.errstate(invalid="ignore", over="ignore"):
                        s = scale * (ks @ q[row, h])
                        w = np.exp(s - s.max())
                        w /= w.sum()
                        some = w > 0
                        ref[row, h] = w[some] @ vs[some] if not np.isnan(w).any() else np.nan
                        # a score: d products and sums, the scale; its weight: that, 2^x, its rounding to 16 bits
                        # (below fp16's 2^-14, at 2^7 times the weight, by up to 2^-25: 2^-32 of it); the sums: a rounding and a rescaling per position; the output's
                        a = w[some] @ np.abs(vs[some])
                        ds = scale * (np.abs(ks[some]) @ np.abs(q[row, h])).max(initial=0.0) * (c.d + 4) * F
                        n = len(s)
                        tol[row, h] = (u * np.abs(ref[row, h]) + u * a * (1 + u) + a * (2 * ds + (2 * n + 16) * F)
                                       + n * 2.0 ** -32 * np.abs(vs).max() + 2.0 ** -25)
    return ref, tol


def run_attention(c, window=0, sinks=0, scale=None, max_new=None, q=None, fill=0.5):
    scale = c.d ** -0.5 if scale is None else scale
    q = to16(c.rng.normal(0, 1.5, (c.tokens, c.heads, c.d)), c.dtype) if q is None else q
    kv = c.upload()
    out = c.ctx.upload(to16(np.full(q.shape, fill), c.dtype))
    dq = c.ctx.upload(q)
    max_new = max(c.new + [0]) if max_new is None else max_new
    work = c.ctx.alloc(c.ctx.attn_paged_workspace(kv, c.tokens, c.heads, max_new))
    c.ctx.memset(work, 0xff)  # (stale parts would be NaN)
    c.ctx.attn_paged(kv, dq, out, c.tokens, c.heads, max_new, float(np.float32(scale)), work, window, sinks)
    c.ctx.sync()
    got = out.to_host()
    for x in (out, dq, work):
        x.free()
    c.free()
    return q, got


def check_attention(c, window=0, sinks=0, scale=None, max_new=None, q=None):
    q, got = run_attention(c, window, sinks, scale, max_new, q)
    scale = float(np.float32(c.d ** -0.5 if scale is None else scale))
    ref, tol = attention_oracle(c, from16(q, c.dtype), window, sinks, scale)
    out = from16(got, c.dtype)
    mine = np.zeros(len(out), bool)
    for b in range(c.batch):
        mine[c.starts[b]:c.starts[b] + c.new[b]] = True
    assert (out[~mine] == 0.5).all(), "rows of no sequence were written"
    same = (out == ref) | (np.isnan(out) & np.isnan(ref))
    with np.errstate(invalid="ignore"):
        bad = mine[:, None, None] & ~same & ~(np.abs(out - ref) <= tol)
    at = np.argwhere(bad)
    assert not bad.any(), (len(at), at[:5], out[tuple(at[0])], ref[tuple(at[0])], tol[tuple(at[0])])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", [(16, 8, 128), (12, 12, 64), (5, 1, 128), (48, 3, 64)])
@pytest.mark.parametrize("lengths,page", [([1], 16), ([777, 1, 64, 65, 0, 300], 16), ([2100, 128, 127], 64)])
def test_decode(ctx, dtype, heads, kv_heads, d, lengths, page):
    new = [1 if l else 0 for l in lengths]
    check_attention(Case(ctx, len(lengths) * heads + d, dtype, new, lengths, heads, kv_heads, d, page))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d,page", [(16, 8, 128, 16), (4, 4, 64, 32), (6, 2, 128, 64), (7, 1, 64, 128)])
@pytest.mark.parametrize("new,lengths", [([130], [130]), ([33, 0, 1, 200], [500, 40, 1, 201]), ([5, 64, 17], [5, 64, 900])])
def test_chunks(ctx, dtype, heads, kv_heads, d, page, new, lengths):
    check_attention(Case(ctx, sum(new) + d, dtype, new, lengths, heads, kv_heads, d, page, first_row=2))


@pytest.mark.parametrize("heads,kv_heads,d,new", [(8, 4, 128, [1, 3, 1]), (6, 2, 64, [150, 20, 1])])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 4), (64, 64), (100, 130), (5000, 4)])
def test_window_and_sinks(ctx, heads, kv_heads, d, new, window, sinks):
    check_attention(Case(ctx, window + sinks, "bf16", new, [700, 333, 1], heads, kv_heads, d, 16),
                    window=window, sinks=sinks)


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [40, 9, 2, 30]])
def test_rows_that_see_nothing_and_bad_pages(ctx, new):
    # table entries that are no page, at the start, inside and at the end; fewer positions than new tokens
    c = Case(ctx, 5, "f16", new, [200, 90, 20, 120], 4, 2, 64, 16)
    c.table[0, 0] = -1
    c.table[0, 3] = c.num_pages
    c.table[0, 4] = np.iinfo(np.int32).min
    c.table[0, 12] = np.iinfo(np.int32).max
    c.table[1, :] = -7
    c.lengths[2] = min(2, new[2] - 1) if new[2] > 1 else 0
    c.table[3, 1:7] = 1 << 30
    check_attention(c)
    check_attention(c, window=20, sinks=3)


@pytest.mark.parametrize("new", [[1, 1], [70, 3]])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("dtype,bad", [("f16", np.nan), ("bf16", np.inf), ("bf16", -np.inf)])
def test_unseen_places_hold_anything(ctx, dtype, bad, new, window):
    # what no row sees: behind the last position in its page, spare pages, before the window
    c = Case(ctx, 9, dtype, new, [150, 71], 4, 2, 128, 32, scale=1.0)
    keep = np.zeros((c.num_pages, c.page), bool)
    for b in range(c.batch):
        p = np.arange(c.lengths[b])
        if window:
            p = p[p > c.lengths[b] - c.new[b] - window]
        keep[c.table[b, p // c.page], p % c.page] = True
    for bits in (c.k, c.v):
        x = from16(bits, dtype).astype(np.float32)
        x[~keep[:, None, :, None] & np.ones(x.shape, bool)] = bad
        bits[:] = to16(x, dtype)
    check_attention(c, window=window)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_later_tokens_of_a_chunk_hold_anything(ctx, dtype):
    # token 20's k and v are not finite: tokens before it must not notice, those from it on do
    c = Case(ctx, 11, dtype, [40, 5], [90, 50], 4, 2, 64, 16)
    page, at = c.table[0, 70 // 16], 70 % 16
    for bits, bad in ((c.k, np.inf), (c.v, np.nan)):
        x = from16(bits, dtype).astype(np.float32)
        x[page, :, at, :3] = bad
        bits[:] = to16(x, dtype)
    q, got = run_attention(c)
    ref, tol = attention_oracle(c, from16(q, dtype), 0, 0, 64 ** -0.5)
    out = from16(got, dtype)
    before, others = slice(0, 20), slice(40, 45)
    for rows in (before, others):
        assert (np.abs(out[rows] - ref[rows]) <= tol[rows]).all()


def test_scores_of_minus_infinity_have_no_weight(ctx):
    c = Case(ctx, 12, "f16", [1, 20], [100, 80], 2, 1, 64, 16)
    q = to16(np.abs(c.rng.normal(0, 1, (c.tokens, 2, 64))) + 0.1, "f16")
    x = from16(c.k, "f16").astype(np.float32)
    for b, p in ((0, 3), (0, 99), (1, 10)):
        x[c.table[b, p // 16], 0, p % 16, 5] = -np.inf
    c.k[:] = to16(x, "f16")
    check_attention(c, q=q)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new", [[1], [40]])
def test_large_scores(ctx, dtype, new):
    # a few weights carry the row; scores far beyond exp's range
    check_attention(Case(ctx, 13, dtype, new, [600], 4, 2, 128, 16, scale=30.0), scale=1.0)


def test_more_new_tokens_than_announced(ctx):
    check_attention(Case(ctx, 14, "bf16", [100, 3], [300, 50], 4, 2, 64, 16), max_new=1)


@pytest.mark.parametrize("batch", [300, 700])
def test_many_sequences(ctx, batch):
    rng = np.random.default_rng(batch)
    lengths = [int(l) for l in rng.integers(0, 60, batch)]
    new = [min(l, int(rng.integers(0, 4))) for l in lengths]
    check_attention(Case(ctx, batch, "f16", new, lengths, 2, 1, 64, 16))


def test_one_long_sequence_among_short_ones(ctx):
    check_attention(Case(ctx, 15, "bf16", [1] * 9, [30000] + [5] * 8, 8, 1, 128, 64))


@pytest.mark.parametrize("group", [17, 128])
def test_many_query_heads(ctx, group):
    check_attention(Case(ctx, 16, "f16", [3, 1], [120, 300], group, 1, 64, 16))


def test_pool_past_2_to_32_values(ctx):
    # the sequence's pages are the pool's last ones, 9 GiB in
    d, kv_heads, page, num = 128, 8, 64, 70000
    nbytes = num * kv_heads * page * d * 2
    small = Case(ctx, 17, "f16", [1, 20], [200, 100], 8, 8, d, page)
    k, v = ctx.alloc(nbytes), ctx.alloc(nbytes)
    per = kv_heads * page * d * 2
    first = num - small.num_pages
    try:
        k.view(first * per, small.num_pages * per).copy_from_host(small.k)
        v.view(first * per, small.num_pages * per).copy_from_host(small.v)
        table = np.where(small.table >= 0, small.table + first, -1).astype(np.int32)
        bufs = [ctx.upload(a) for a in (table, np.array(small.lengths, np.int32), small.starts)]
        kv = PagedKV(k, v, *bufs, batch=2, max_pages=small.max_pages, num_pages=num, page_size=page,
                     kv_heads=kv_heads, head_dim=d, dtype="f16")
        q = to16(small.rng.normal(0, 1.5, (small.tokens, 8, d)), "f16")
        dq, out = ctx.upload(q), ctx.upload(to16(np.full(q.shape, 0.5), "f16"))
        work = ctx.alloc(ctx.attn_paged_workspace(kv, small.tokens, 8, 20))
        scale = float(np.float32(d ** -0.5))
        ctx.attn_paged(kv, dq, out, small.tokens, 8, 20, scale, work)
        ctx.sync()
        ref, tol = attention_oracle(small, from16(q, "f16"), 0, 0, scale)
        got = from16(out.to_host(), "f16")
        assert (np.abs(got - ref)[:21] <= tol[:21]).all()
        # and the append there
        qkv = ctx.upload(to16(small.rng.normal(0, 1, (small.tokens, 24, d)), "f16"))
        gain = ctx.upload(np.ones(d, np.float32))
        ctx.qk_norm_rope_paged(kv, qkv, gain, gain, dq, small.tokens, 8, 1e-6, 1e4)
        ctx.sync()
        back = v.view(first * per, small.num_pages * per, np.int16, small.v.shape).to_host()
        vs = qkv.to_host()[:, 16:]
        for b in range(2):
            for i in range(small.new[b]):
                p = small.lengths[b] - small.new[b] + i
                assert (back[small.table[b, p // page], :, p % page] == vs[small.starts[b] + i]).all()
        for x in bufs + [dq, out, work, qkv, gain]:
            x.free()
    finally:
        k.free()
        v.free()


# ---- head norms, RoPE and the pages --------------------------------------------------

def norm_rope_oracle(x, gain, pos, eps, theta):
    d = x.shape[-1]
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gain
    angle = pos[:, None, None] * theta ** (-2.0 * np.arange(d // 2) / d)
    c, s = np.cos(angle), np.sin(angle)
    a, b = y[..., :d // 2], y[..., d // 2:]
    size = np.sqrt(a * a + b * b)
    return np.concatenate([a * c - b * s, b * c + a * s], -1), np.concatenate([size, size], -1)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d,pad", [(16, 8, 128, 0), (12, 12, 64, 8), (1, 1, 64, 0), (71, 1, 128, 24)])
@pytest.mark.parametrize("new,lengths,page", [([1], [1], 16), ([3, 0, 1], [100003, 5, 40], 64), ([17, 66], [20, 70], 32)])
def test_norm_rope(ctx, dtype, heads, kv_heads, d, pad, new, lengths, page):
    c = Case(ctx, heads + d + sum(new), dtype, new, lengths, heads, kv_heads, d, page, first_row=1, rows_behind=2)
    all_heads = heads + 2 * kv_heads
    ld = all_heads * d + pad
    qkv = to16(c.rng.normal(0, 1.7, (c.tokens, ld)), dtype)
    qkv[0, :d] = 0  # (of no sequence)
    qkv[1, :d] = 0  # a head of zeros
    gains = [(1 + c.rng.normal(0, 0.3, d)).astype(np.float32) for _ in range(2)]
    eps, theta = float(np.float32(1e-6)), 1e6
    kv = c.upload()
    bufs = [ctx.upload(a) for a in (qkv, *gains, to16(np.full((c.tokens, heads, d), 0.5), dtype))]
    ctx.qk_norm_rope_paged(kv, *bufs, c.tokens, heads, eps, theta, ld)
    ctx.sync()
    q, k, v = (b.to_host() for b in (bufs[3], c.buffers[0], c.buffers[1]))
    x = from16(qkv[:, :all_heads * d], dtype).reshape(c.tokens, all_heads, d)
    want_k, want_v = c.k.copy(), c.v.copy()
    checked = np.zeros((c.num_pages, page), bool)
    u = U[dtype]
    got_q = from16(q, dtype)
    mine = np.zeros(c.tokens, bool)
    for b in range(c.batch):
        rows = np.arange(c.starts[b], c.starts[b] + new[b])
        mine[rows] = True
        pos = lengths[b] - new[b] + np.arange(new[b])
        # the mean of squares, its root and quotient, three products, the factors, the rotation: below 32 fp32
        # roundings of the pair's size (d / 16 + 4 of the sum's count half)
        for part, gain, got in ((x[rows, :heads], gains[0], got_q[rows]),
                                (x[rows, heads:heads + kv_heads], gains[1],
                                 from16(k, dtype)[c.table[b, pos // page], :, pos % page])):
            ref, size = norm_rope_oracle(part, gain.astype(np.float64), pos.astype(np.float64), eps, theta)
            assert (np.abs(got - ref) <= u * np.abs(ref) + 32 * F * size + 2.0 ** -25).all()
        want_v[c.table[b, pos // page], :, pos % page] = qkv[rows, (heads + kv_heads) * d:all_heads * d].reshape(-1, kv_heads, d)
        checked[c.table[b, pos // page], pos % page] = True
    assert (v == want_v).all()
    assert (k.transpose(0, 2, 1, 3)[~checked] == want_k.transpose(0, 2, 1, 3)[~checked]).all(), "another position changed"
    assert (got_q[~mine] == 0.5).all()
    for b in bufs:
        b.free()
    c.free()


def test_norm_rope_bad_pages_and_short_lengths(ctx):
    # no page, or before position 0: nothing stored, the rest as it should be
    c = Case(ctx, 3, "f16", [4, 6, 2], [40, 30, 20], 2, 1, 64, 16)
    c.table[0, :] = -1
    c.table[1, 1] = c.num_pages + 3
    c.lengths[2] = 1
    qkv = to16(c.rng.normal(0, 1, (c.tokens, 4, 64)), "f16")
    kv = c.upload()
    bufs = [ctx.upload(a) for a in (qkv, np.ones(64, np.float32), np.ones(64, np.float32), qkv[:, :2])]
    ctx.qk_norm_rope_paged(kv, *bufs, c.tokens, 2, 1e-6, 1e4)
    ctx.sync()
    want = c.v.copy()
    want[c.table[2, 0], 0, 0] = qkv[c.starts[2] + 1, 3]
    assert (c.buffers[1].to_host() == want).all()
    for b in bufs:
        b.free()
    c.free()


@pytest.mark.parametrize("batch", [63, 64, 200, 5000])
def test_norm_rope_finds_every_row(ctx, batch):
    rng = np.random.default_rng(batch)
    new = [int(n) for n in rng.integers(0, 3, batch)]
    c = Case(ctx, batch, "bf16", new, [n + int(rng.integers(0, 20)) for n in new], 1, 1, 64, 16)
    qkv = to16(rng.normal(0, 1, (c.tokens, 3, 64)), "bf16")
    kv = c.upload()
    bufs = [ctx.upload(a) for a in (qkv, np.ones(64, np.float32), np.ones(64, np.float32), qkv[:, :1])]
    ctx.qk_norm_rope_paged(kv, *bufs, c.tokens, 1, 1e-6, 1e4)
    ctx.sync()
    want = c.v.copy()
    for b in range(batch):
        for i in range(new[b]):
            p = c.lengths[b] - new[b] + i
            want[c.table[b, p // 16], 0, p % 16] = qkv[c.starts[b] + i, 2]
    assert (c.buffers[1].to_host() == want).all()
    for b in bufs:
        b.free()
    c.free()


# ---- page copies -------------------------------------------------------------------------

@pytest.mark.parametrize("planes,num_pages,page_bytes,gap,count", [(1, 4, 16, 0, 2), (24, 33, 24576, 0, 7),
                                                                 (5, 20, 16400, 48, 9), (56, 12, 32768, 64, 0)])
def test_pages_copy(ctx, planes, num_pages, page_bytes, gap, count):
    rng = np.random.default_rng(planes)
    stride = num_pages * page_bytes + gap
    host = rng.integers(0, 256, planes * stride, dtype=np.uint8)
    order = rng.permutation(num_pages).astype(np.int32)
    src, dst = order[:count].copy(), order[count:2 * count].copy()
    if count > 6:
        src[1] = src[0]  # a page may go to several
        src[2], dst[3] = -1, num_pages  # skipped
        src[4] = dst[4]  # onto itself
    pool, s, d = ctx.upload(host), ctx.upload(np.append(src, 0).astype(np.int32)), ctx.upload(np.append(dst, 0).astype(np.int32))
    ctx.pages_copy(pool, planes, num_pages, page_bytes, s, d, count, stride)
    ctx.sync()
    want = host.copy()
    for p in range(planes):
        plane = want[p * stride:p * stride + num_pages * page_bytes].reshape(num_pages, page_bytes)
        for a, b in zip(src, dst):
            if 0 <= a < num_pages and 0 <= b < num_pages:
                plane[b] = plane[a]
    assert (pool.to_host() == want).all()
    for x in (pool, s, d):
        x.free()


# ---- refusals -------------------------------------------------------------------------

def test_refusals(ctx):
    c = Case(ctx, 1, "f16", [2], [20], 4, 2, 64, 16)
    kv = c.upload()
    rows = ctx.upload(np.zeros((c.tokens, 8, 64), np.int16))
    q, out = ctx.upload(np.zeros((c.tokens, 4, 64), np.int16)), ctx.upload(np.zeros((c.tokens, 4, 64), np.int16))
    gain = ctx.upload(np.ones(64, np.float32))
    work = ctx.alloc(ctx.attn_paged_workspace(kv, c.tokens, 4, 2))

    def view(**kw):
        names = dict(batch=1, max_pages=c.max_pages, num_pages=c.num_pages, page_size=16, kv_heads=2, head_dim=64)
        buffers = [kw.pop(n, b) for n, b in zip(("k", "v", "table", "lengths", "starts"), c.buffers)]
        return PagedKV(*buffers, **{**names, **kw})

    def refused(call, text, status=strict_amd.SH_ERR_INVALID_ARGUMENT):
        with pytest.raises(strict_amd.StrictHipError) as e:
            call()
        assert e.value.status == status and text in e.value.message, e.value.message

    def attn(kv=kv, q=q, out=out, tokens=c.tokens, heads=4, max_new=2, scale=1.0, work=work, window=0, sinks=0):
        return lambda: ctx.attn_paged(kv, q, out, tokens, heads, max_new, scale, work, window, sinks)

    def rope(kv=kv, rows=rows, gain=gain, q=q, tokens=c.tokens, heads=4, eps=1e-6, theta=1e4, ld=None):
        return lambda: ctx.qk_norm_rope_paged(kv, rows, gain, gain, q, tokens, heads, eps, theta, ld)

    for make in (attn, rope):
        refused(make(kv=view(page_size=24)), "page_size")
        refused(make(kv=view(num_pages=c.num_pages + 1)), "k pages")
        refused(make(kv=view(max_pages=c.max_pages + 999)), "page_table")
        refused(make(kv=view(batch=2)), "page_table")
        refused(make(kv=view(head_dim=96)), "head_dim", 7)
        refused(make(kv=view(starts=None)), "starts is NULL")
        refused(make(kv=view(v=c.buffers[1].ptr + 2)), "v pages")
        refused(make(kv=view(k=c.buffers[0].ptr + 2, num_pages=c.num_pages - 1)), "aligned")
        refused(make(heads=5), "heads")
        refused(make(tokens=-1), "tokens")
        refused(make(tokens=c.tokens + 1), "not inside")
        refused(make(q=None), "q is NULL")
        make(tokens=0, q=None)()
    refused(attn(scale=0.0), "scale")
    refused(attn(scale=float("nan")), "scale")
    refused(attn(scale=float("inf")), "scale")
    refused(attn(window=-1), "window")
    refused(attn(sinks=-1), "sinks")
    refused(attn(max_new=-1), "max_new")
    refused(attn(out=q), "overlaps")
    refused(attn(work=work.view(0, work.nbytes - 16)), "work buffer")
    big = ctx.alloc(work.nbytes + 16)
    refused(attn(work=big.view(8, work.nbytes)), "aligned")
    refused(rope(eps=-1.0), "eps")
    refused(rope(theta=0.0), "theta")
    refused(rope(theta=float("inf")), "theta")
    refused(rope(ld=8 * 64 - 8), "ld")
    refused(rope(ld=8 * 64 + 4), "ld")
    refused(rope(q=rows), "overlaps")
    refused(lambda: ctx.pages_copy(work, 1, 4, 24, gain, gain, 1), "page_bytes")
    refused(lambda: ctx.pages_copy(gain, 1, 64, 16, gain, gain, 1), "pool")
    refused(lambda: ctx.pages_copy(big.ptr + 8, 1, 4, 16, gain, gain, 1), "aligned")
    refused(lambda: ctx.pages_copy(work, 2, 4, 16, gain, gain, 1, plane_stride=32), "plane_stride")
    for x in (rows, q, out, gain, work, big):
        x.free()
    c.free()
