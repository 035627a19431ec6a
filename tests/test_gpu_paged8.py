"""The operators over a KV cache in pages of 8-bit values against their formulas in 64
bits (numpy): what is stored byte by byte, attention as in test_gpu_paged.py, whose
oracle and tolerances these are with k and v as the bytes and scales say."""
import numpy as np
import pytest

import strict_amd
import test_gpu_paged as paged
from strict_amd import PagedKV8
from test_gpu_paged import F, U, from16, to16

pytestmark = pytest.mark.gpu

E4M3 = np.array([(b & 7) * 2.0 ** -9 if b < 8 else (8 + (b & 7)) * 2.0 ** ((b >> 3) - 10) for b in range(127)])
VALUES = np.concatenate([E4M3, [np.nan], -E4M3, [np.nan]])
LARGEST = {"f16": 1.875 * 2.0 ** 15, "bf16": 1.875 * 2.0 ** 127}


def quantised(y, dtype):
    """Rows of 64-bit values as bytes and scales by the header's rule, and how far each
    value lies from where the next byte would begin, relative to its row's largest."""
    y = np.where(np.isinf(y), np.nan, np.clip(y, -LARGEST[dtype], LARGEST[dtype]))
    most = np.nan_to_num(np.abs(y)).max(-1)
    e = np.maximum(np.ceil(np.log2(np.maximum(most, 1e-300) / 448)), -127).astype(int)
    e += most > 448 * 2.0 ** e
    e -= (e > -127) & (most <= 448 * 2.0 ** (e - 1))
    z = np.abs(y) / 2.0 ** e[..., None]
    middle = (E4M3[1:] + E4M3[:-1]) / 2
    low = np.searchsorted(middle, z)  # (NaN: 126)
    margin = np.minimum(np.abs(z - middle[np.minimum(low, 125)]), np.abs(z - middle[np.maximum(low - 1, 0)])) * 2.0 ** e[..., None]
    low = low + ((low < 126) & (z == middle[np.minimum(low, 125)]) & (low % 2 == 1))
    byte = np.where(np.isnan(y), 127, low) + 128 * np.signbit(y)
    return byte.astype(np.uint8), (e + 127).astype(np.uint8), margin / np.maximum(most, 1e-300)[..., None]


def values(byte, scale):
    return VALUES[byte] * np.where(scale == 255, np.nan, 2.0 ** (scale.astype(int) - 127))[..., None]


class Case8(paged.Case):
    """A Case of 8-bit pages: kb, vb bytes [pages, kv_heads, page, d], ks, vs their scales.
    k and v: their values as 16-bit patterns, as the operators read them (from an upload
    on, those that it sent); set, quantised."""

    sent = None

    def _get(self, which):
        if self.sent:
            return self.sent[which]
        with np.errstate(over="ignore"):
            return to16(values(getattr(self, which + "b"), getattr(self, which + "s")), self.dtype)

    def _set(self, which, bits):
        b, s, _ = quantised(from16(bits, self.dtype), self.dtype)
        setattr(self, which + "b", b)
        setattr(self, which + "s", s)

    k = property(lambda self: self._get("k"), lambda self, bits: self._set("k", bits))
    v = property(lambda self: self._get("v"), lambda self, bits: self._set("v", bits))

    def bytes(self):
        return np.concatenate([a.reshape(self.num_pages, -1) for a in (self.kb, self.vb, self.ks, self.vs)], 1)

    def split(self, pages):
        """kb, vb, ks, vs of pages that came back."""
        n, rows = self.kv_heads * self.page * self.d, self.kv_heads * self.page
        shape = (self.num_pages, self.kv_heads, self.page, self.d)
        return (pages[:, :n].reshape(shape), pages[:, n:2 * n].reshape(shape),
                pages[:, 2 * n:2 * n + rows].reshape(shape[:3]), pages[:, 2 * n + rows:].reshape(shape[:3]))

    def sizes(self):
        return dict(batch=self.batch, max_pages=self.max_pages, num_pages=self.num_pages, page_size=self.page,
                    kv_heads=self.kv_heads, head_dim=self.d, dtype=self.dtype)

    def upload(self):
        self.sent = None
        self.sent = {"k": self.k, "v": self.v}
        self.buffers = [self.ctx.upload(a) for a in (self.bytes(), self.table, np.array(self.lengths, np.int32), self.starts)]
        assert self.buffers[0].nbytes == self.num_pages * PagedKV8.page_bytes(self.kv_heads, self.page, self.d)
        self.kv = PagedKV8(*self.buffers, **self.sizes())
        return self.kv


# ---- what is stored --------------------------------------------------------------------

def store(c, qkv, gains, heads, eps=float(np.float32(1e-6)), theta=1e6, ld=None):
    """The pages and q after a call."""
    kv = c.upload()
    bufs = [c.ctx.upload(a) for a in (qkv, *gains, to16(np.full((c.tokens, heads, c.d), 0.5), c.dtype))]
    c.ctx.qk_norm_rope_paged(kv, *bufs, c.tokens, heads, eps, theta, ld)
    c.ctx.sync()
    pages, q = c.split(c.buffers[0].to_host().reshape(c.num_pages, -1)), bufs[3].to_host()
    for b in bufs:
        b.free()
    c.free()
    return pages, q


def check_rows(got, ref, exact_input):
    """Bytes and scales of rows against those of the 64-bit rows `ref` (and their type):
    equal, but for computed values within 2^-36 of their row's size of a border."""
    byte, scale, margin = quantised(*ref)
    same = (got[0] == byte) | (np.isnan(VALUES[got[0]]) & np.isnan(VALUES[byte]))
    if exact_input:
        assert (got[1] == scale).all() and same.all()
        return
    # (a row's largest value on the border between two scales: values then as near)
    edge = got[1] != scale
    finite = np.nan_to_num(np.abs(ref[0])).max(-1)
    power = finite / 448 / 2.0 ** np.round(np.log2(np.maximum(finite, 1e-300) / 448))
    assert (~edge | (np.abs(power - 1) < 2.0 ** -36)).all()
    assert (same | (margin < 2.0 ** -36) | edge[..., None]).all()
    assert edge.sum() <= edge.size // 100 and (~same).sum() <= same.size // 100


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d,pad", [(16, 8, 128, 0), (12, 12, 64, 8), (1, 1, 64, 0), (71, 1, 128, 24)])
@pytest.mark.parametrize("new,lengths,page", [([1], [1], 16), ([3, 0, 1], [7003, 5, 40], 64), ([17, 66], [20, 70], 32)])
def test_store(ctx, dtype, heads, kv_heads, d, pad, new, lengths, page):
    c = Case8(ctx, heads + d + sum(new), dtype, new, lengths, heads, kv_heads, d, page, first_row=1, rows_behind=2)
    all_heads = heads + 2 * kv_heads
    ld = all_heads * d + pad
    # rows far apart in size; some of zeros
    qkv = c.rng.normal(0, 1.7, (c.tokens, ld)) * np.repeat(2.0 ** c.rng.integers(-9, 6, (c.tokens, ld // 8)), 8, 1)
    qkv[:, heads * d:] *= (c.rng.random((c.tokens, 1)) < 0.9)
    qkv = to16(qkv, dtype)
    gains = [(1 + c.rng.normal(0, 0.3, d)).astype(np.float32) for _ in range(2)]
    eps = float(np.float32(1e-6))
    before = c.kb.copy(), c.vb.copy(), c.ks.copy(), c.vs.copy()
    pages, q = store(c, qkv, gains, heads, eps, 1e6, ld)
    x = from16(qkv[:, :all_heads * d], dtype).reshape(c.tokens, all_heads, d)
    got_q, mine, written = from16(q, dtype), np.zeros(c.tokens, bool), np.zeros((c.num_pages, page), bool)
    for b in range(c.batch):
        rows = np.arange(c.starts[b], c.starts[b] + new[b])
        mine[rows] = True
        pos = lengths[b] - new[b] + np.arange(new[b])
        at = c.table[b, pos // page], slice(None), pos % page
        ref, size = paged.norm_rope_oracle(x[rows, :heads], gains[0].astype(np.float64), pos.astype(np.float64), eps, 1e6)
        assert (np.abs(got_q[rows] - ref) <= U[dtype] * np.abs(ref) + 32 * F * size + 2.0 ** -25).all()
        ref, _ = paged.norm_rope_oracle(x[rows, heads:heads + kv_heads], gains[1].astype(np.float64), pos.astype(np.float64), eps, 1e6)
        check_rows((pages[0][at], pages[2][at]), (ref, dtype), False)
        check_rows((pages[1][at], pages[3][at]), (x[rows, heads + kv_heads:], dtype), True)
        written[at[0], at[2]] = True
    assert (got_q[~mine] == 0.5).all()
    for now, then in zip(pages, before):
        assert (now.swapaxes(1, 2)[~written] == then.swapaxes(1, 2)[~written]).all(), "another position changed"


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_store_rounds_and_saturates(ctx, dtype):
    # v rows of one value and its neighbours: every step of the format, half-way places, the
    # largest and smallest of the type, values that are not finite
    c = Case8(ctx, 1, dtype, [300], [300], 1, 1, 64, 16)
    top = 2.0 ** 15 if dtype == "f16" else 2.0 ** 127
    v = c.rng.normal(0, 1, (c.tokens, 64))
    middle = (E4M3[1:] + E4M3[:-1]) / 2
    near = np.concatenate([E4M3, middle, -E4M3, -middle, middle * (1 + 2.0 ** -7), middle * (1 - 2.0 ** -7)])
    for r in range(100):
        v[r] = c.rng.choice(near, 64) * 2.0 ** (r % 12 - 6)
        v[r, r % 64] = 448 * 2.0 ** (r % 12 - 6)  # the scale's own border
    for r in range(100, 164):
        v[r] *= top * c.rng.choice([2.0 ** -1, 0.24, 0.3])
    v = np.clip(v, -1.99 * top, 1.99 * top)
    v[164:180] *= 2.0 ** (-14 if dtype == "f16" else -130)
    v[164:180, 1:] *= 2.0 ** -8
    v[180, 3], v[181, 0], v[181, 63], v[182, :] = np.nan, np.inf, -np.inf, np.nan
    v[183] = 0
    v[184] = -0.0
    v[185, 5], v[186, 6] = 1.99 * top, -1.9 * top
    qkv = to16(np.stack([np.ones_like(v), np.ones_like(v), v], 1), dtype)
    pages, _ = store(c, qkv, [np.ones(64, np.float32)] * 2, 1)
    pos = np.arange(300)
    at = c.table[0, pos // 16], 0, pos % 16
    check_rows((pages[1][at], pages[3][at]), (from16(qkv[:300, 2], dtype), dtype), True)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_store_large_small_and_broken_keys(ctx, dtype):
    c = Case8(ctx, 2, dtype, [60], [60], 1, 1, 128, 16)
    x = c.rng.normal(0, 1, (c.tokens, 3, 128))
    x[3, 1] = 0          # 0 / sqrt(eps)
    x[4, 1, 7] = np.nan  # a row of NaN
    x[5, 1, 7] = np.inf  # x / infinity: 0, and one of NaN
    gain = np.ones(128, np.float32)
    gain[:8] = 1e6 if dtype == "f16" else 3e38  # beyond what either type holds
    gain[64:72] = 0
    qkv = to16(x, dtype)
    pages, _ = store(c, qkv, [np.ones(128, np.float32), gain], 1)
    pos = np.arange(60)
    at = c.table[0, pos // 16], 0, pos % 16
    with np.errstate(invalid="ignore"):
        ref, _ = paged.norm_rope_oracle(from16(qkv[:60, 1], dtype)[:, None], gain.astype(np.float64), pos.astype(np.float64),
                                        float(np.float32(1e-6)), 1e6)
    keep = pos != 5  # (of an infinity, NaN in one pair and 0 times what the angle says elsewhere)
    check_rows((pages[0][at][keep], pages[2][at][keep]), (ref[keep, 0], dtype), False)


def test_store_bad_pages_and_short_lengths(ctx):
    # no page, or before position 0: nothing stored, the rest as it should be
    c = Case8(ctx, 3, "f16", [4, 6, 2], [40, 30, 20], 2, 1, 64, 16)
    c.table[0, :] = -1
    c.table[1, 1] = c.num_pages + 3
    c.lengths[2] = 1
    qkv = to16(c.rng.normal(0, 1, (c.tokens, 4, 64)), "f16")
    before = c.vb.copy()
    pages, _ = store(c, qkv, [np.ones(64, np.float32)] * 2, 2)
    before[c.table[2, 0], 0, 0] = quantised(from16(qkv[c.starts[2] + 1, 3], "f16")[None], "f16")[0][0]
    assert (pages[1] == before).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kv_heads,d,page", [(8, 128, 16), (1, 64, 16), (12, 64, 128), (33, 128, 32)])
def test_read_back(ctx, dtype, kv_heads, d, page):
    # any bytes and scales, rows of no sequence and positions without a page left as they are
    c = Case8(ctx, kv_heads, dtype, [5, 0, 40, 3], [5, 20, 333, 2], kv_heads, kv_heads, d, page, first_row=1)
    for a in (c.kb, c.vb):
        a[:] = c.rng.integers(0, 256, a.shape)
    for a in (c.ks, c.vs):
        a[:] = c.rng.integers(100, 150, a.shape)
        a[c.rng.random(a.shape) < 0.1] = c.rng.choice([0, 1, 2, 80, 240, 254, 255])
    c.table[2, 330 // page] = -1
    kv = c.upload()
    fill = to16(np.full((c.tokens, kv_heads, d), 0.5), dtype)
    out = [ctx.upload(fill) for _ in range(2)]
    ctx.paged_read(kv, *out, c.tokens)
    ctx.sync()
    for got, bits in zip((b.to_host() for b in out), (c.k, c.v)):
        want = fill.copy()
        for b in range(c.batch):
            for i in range(c.new[b]):
                p = c.lengths[b] - c.new[b] + i
                if p >= 0 and c.table[b, p // page] >= 0:
                    want[c.starts[b] + i] = bits[c.table[b, p // page], :, p % page]
        nan = np.isnan(from16(want, dtype))
        assert (np.isnan(from16(got, dtype)) == nan).all() and (got == want)[~nan].all()
    for b in out:
        b.free()
    c.free()


# ---- attention ------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", [(16, 8, 128), (12, 12, 64), (5, 1, 128), (48, 3, 64)])
@pytest.mark.parametrize("lengths,page", [([1], 16), ([777, 1, 64, 65, 0, 300, 129], 16), ([2100, 128, 127], 64)])
def test_decode(ctx, dtype, heads, kv_heads, d, lengths, page):
    new = [1 if l else 0 for l in lengths]
    paged.check_attention(Case8(ctx, len(lengths) * heads + d, dtype, new, lengths, heads, kv_heads, d, page))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d,page", [(16, 8, 128, 16), (4, 4, 64, 32), (6, 2, 128, 64), (7, 1, 64, 128)])
@pytest.mark.parametrize("new,lengths", [([130], [130]), ([33, 0, 1, 200], [500, 40, 1, 201]), ([5, 64, 17], [5, 64, 900])])
def test_chunks(ctx, dtype, heads, kv_heads, d, page, new, lengths):
    paged.check_attention(Case8(ctx, sum(new) + d, dtype, new, lengths, heads, kv_heads, d, page, first_row=2))


@pytest.mark.parametrize("heads,kv_heads,d,new", [(8, 4, 128, [1, 3, 1]), (6, 2, 64, [150, 20, 1])])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 4), (64, 64), (100, 130), (5000, 4)])
def test_window_and_sinks(ctx, heads, kv_heads, d, new, window, sinks):
    paged.check_attention(Case8(ctx, window + sinks, "bf16", new, [700, 333, 1], heads, kv_heads, d, 16),
                          window=window, sinks=sinks)


@pytest.mark.parametrize("heads,kv_heads,d", [(8, 4, 128), (6, 2, 64)])
@pytest.mark.parametrize("window,sinks", [(500, 12), (500, 13), (1000, 24), (1024, 300)])
def test_long_windows_and_sinks(ctx, heads, kv_heads, d, window, sinks):
    paged.check_attention(Case8(ctx, window + sinks, "f16", [1, 2, 1, 0, 1], [3000, 1030, 600, 5, 1], heads, kv_heads, d, 16),
                          window=window, sinks=sinks)


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [40, 9, 2, 30]])
def test_rows_that_see_nothing_and_bad_pages(ctx, new):
    c = Case8(ctx, 5, "f16", new, [200, 90, 20, 120], 4, 2, 64, 16)
    c.table[0, 0] = -1
    c.table[0, 3] = c.num_pages
    c.table[0, 4] = np.iinfo(np.int32).min
    c.table[0, 12] = np.iinfo(np.int32).max
    c.table[1, :] = -7
    c.lengths[2] = min(2, new[2] - 1) if new[2] > 1 else 0
    c.table[3, 1:7] = 1 << 30
    paged.check_attention(c)
    paged.check_attention(c, window=20, sinks=3)


@pytest.mark.parametrize("new", [[1, 1], [70, 3]])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("dtype,byte,scale", [("f16", 127, 130), ("bf16", 255, 10), ("f16", 56, 255), ("bf16", 0, 255), ("f16", 126, 254)])
def test_unseen_places_hold_anything(ctx, dtype, byte, scale, new, window):
    # what no row sees: behind the last position in its page, spare pages, before the window
    c = Case8(ctx, 9, dtype, new, [150, 71], 4, 2, 128, 32, scale=1.0)
    keep = np.zeros((c.num_pages, c.page), bool)
    for b in range(c.batch):
        p = np.arange(c.lengths[b])
        if window:
            p = p[p > c.lengths[b] - c.new[b] - window]
        keep[c.table[b, p // c.page], p % c.page] = True
    for a, s in ((c.kb, c.ks), (c.vb, c.vs)):
        a.swapaxes(1, 2)[~keep] = byte
        s.swapaxes(1, 2)[~keep] = scale
    paged.check_attention(c, window=window)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_later_tokens_of_a_chunk_hold_anything(ctx, dtype):
    # token 20's k and v are NaN: tokens before it must not notice, those from it on do
    c = Case8(ctx, 11, dtype, [40, 5], [90, 50], 4, 2, 64, 16)
    page, at = c.table[0, 70 // 16], 70 % 16
    c.kb[page, :, at, :3] = 127
    c.vs[page, :, at] = 255
    q, got = paged.run_attention(c)
    ref, tol = paged.attention_oracle(c, from16(q, dtype), 0, 0, 64 ** -0.5)
    out = from16(got, dtype)
    for rows in (slice(0, 20), slice(40, 45)):
        assert (np.abs(out[rows] - ref[rows]) <= tol[rows]).all()
    assert np.isnan(out[20:40]).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new", [[1], [40]])
@pytest.mark.parametrize("log2", [0, 5, 30, 60])
def test_rows_of_very_different_size(ctx, dtype, new, log2):
    # scales over the type's whole range; a few weights carry the row
    c = Case8(ctx, 13, dtype, new, [600], 4, 2, 128, 16)
    span = min(log2, 6 if dtype == "f16" else log2)
    for s in (c.ks, c.vs):
        s[:] = (s + c.rng.integers(-span, span + 1, s.shape)).astype(np.uint8)
    paged.check_attention(c, scale=2.0 ** -span)


def test_pages_of_a_wider_type(ctx):
    # bf16's scales read by fp16: keys that are infinite there, of queries of either sign
    c = Case8(ctx, 14, "f16", [1, 20], [100, 80], 2, 1, 64, 16)
    q = to16(np.abs(c.rng.normal(0, 1, (c.tokens, 2, 64))) + 0.1, "f16")
    for b, p in ((0, 3), (0, 99), (1, 10)):
        c.kb[c.table[b, p // 16], 0, p % 16] = 0x80  # -0, and one of minus infinity
        c.kb[c.table[b, p // 16], 0, p % 16, 5] = 0xfe
        c.ks[c.table[b, p // 16], 0, p % 16] = 200
    paged.check_attention(c, q=q)


def test_more_new_tokens_than_announced(ctx):
    paged.check_attention(Case8(ctx, 14, "bf16", [100, 3], [300, 50], 4, 2, 64, 16), max_new=1)


@pytest.mark.parametrize("batch", [300, 700])
def test_many_sequences(ctx, batch):
    rng = np.random.default_rng(batch)
    lengths = [int(l) for l in rng.integers(0, 60, batch)]
    new = [min(l, int(rng.integers(0, 4))) for l in lengths]
    paged.check_attention(Case8(ctx, batch, "f16", new, lengths, 2, 1, 64, 16))


def test_one_long_sequence_among_short_ones(ctx):
    paged.check_attention(Case8(ctx, 15, "bf16", [1] * 9, [30000] + [5] * 8, 8, 1, 128, 64))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", [(8, 8, 128), (12, 12, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 5)])
def test_tiles_for_every_cu(ctx, dtype, heads, kv_heads, d, window, sinks):
    rng = np.random.default_rng(heads)
    new = [int(n) for n in rng.integers(1, 140, 12)] + [18] * 22
    lengths = [n + int(rng.integers(0, 520 - n)) for n in new]
    paged.check_attention(Case8(ctx, d, dtype, new, lengths, heads, kv_heads, d, 32), window=window, sinks=sinks)


@pytest.mark.parametrize("batch", [63, 64, 65, 4095, 4096, 4097])
def test_batches_of_chunks(ctx, batch):
    # (those of more than 4,096 sequences are cut)
    rng = np.random.default_rng(batch)
    lengths = [int(l) for l in rng.integers(0, 6, batch)]
    new = [min(l, int(rng.integers(0, 4))) for l in lengths]
    lengths[0], new[0], lengths[-1], new[-1] = 40, 37, 70, 66
    paged.check_attention(Case8(ctx, batch, "f16", new, lengths, 4, 1, 64, 16), max_new=66)


# Tables of 300 pages more than are used: sequences that could be long, whose tiles are cut.
WIDE = dict(page=16, extra_entries=300)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", [(16, 8, 128), (12, 12, 64), (15, 1, 128), (4, 4, 64)])
@pytest.mark.parametrize("new,lengths", [([1] * 7, [777, 1, 64, 65, 128, 300, 2129]), ([130], [130]), ([33, 0, 1, 200], [500, 40, 1, 201]),
                                         ([5, 64, 17, 128], [5, 64, 900, 2500])])
def test_wide_tables(ctx, dtype, heads, kv_heads, d, new, lengths):
    paged.check_attention(Case8(ctx, sum(new) + d, dtype, new, lengths, heads, kv_heads, d, first_row=2, **WIDE))


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [40, 9, 2, 30]])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3), (5000, 5)])
def test_bad_pages_in_wide_tables(ctx, new, window, sinks):
    c = Case8(ctx, 5, "bf16", new, [200, 90, 20, 120], 4, 2, 128, **WIDE)
    c.table[0, [0, 3, 4]] = -1, c.num_pages, np.iinfo(np.int32).min
    c.table[1, :] = -7
    c.lengths[2] = min(2, new[2] - 1) if new[2] > 1 else 0
    c.table[3, 1:7] = 1 << 30
    paged.check_attention(c, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new", [[1, 1], [40, 5]])
@pytest.mark.parametrize("extra", [1, 300])
@pytest.mark.parametrize("d", [64, 128])
def test_not_numbers_that_rows_see(ctx, dtype, new, extra, d):
    # the last token's k and v are NaN: tokens before it and other sequences must not notice
    c = Case8(ctx, 11, dtype, new, [90, 50], 4, 2, d, 16, extra_entries=extra)
    page, at = c.table[0, 89 // 16], 89 % 16
    c.kb[page, :, at, :3] = 127
    c.vs[page, :, at] = 255
    q, got = paged.run_attention(c)
    ref, tol = paged.attention_oracle(c, from16(q, dtype), 0, 0, d ** -0.5)
    out, last = from16(got, dtype), new[0] - 1
    for rows in (slice(0, last), slice(new[0], sum(new))):
        assert (np.abs(out[rows] - ref[rows]) <= tol[rows]).all()
    assert np.isnan(out[last]).all()


@pytest.mark.parametrize("lengths,new,max_new", [([300, 50, 700], [100, 3, 1], 1), ([300, 50, 700], [100, 3, 300], 33)])
@pytest.mark.parametrize("extra", [1, 300])
def test_more_tokens_than_announced(ctx, lengths, new, max_new, extra):
    paged.check_attention(Case8(ctx, 14, "f16", new, lengths, 6, 2, 128, 16, extra_entries=extra), max_new=max_new)


@pytest.mark.parametrize("batch,lengths,most", [(70, (0, 60), 40), (700, (0, 60), 30), (200, (100, 500), 3)])
@pytest.mark.parametrize("extra", [1, 300])
def test_many_ragged_chunks(ctx, batch, lengths, most, extra):
    rng = np.random.default_rng(batch)
    lengths = [int(l) for l in rng.integers(*lengths, batch)]
    new = [min(l, int(rng.integers(0, most + 1))) for l in lengths]
    new[batch // 2], lengths[batch // 2] = 300, 310  # one prompt among them
    paged.check_attention(Case8(ctx, batch, "bf16", new, lengths, 4, 1, 64, 16, first_row=5, extra_entries=extra))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", [(16, 8, 128), (12, 12, 64), (15, 1, 128), (8, 4, 64)])
@pytest.mark.parametrize("positions,new", [(256, [1] * 9), (512, [1, 0, 1, 1]), (512, [8, 3, 1, 15, 0, 2]), (528, [1, 2, 1]), (1024, [1, 1]),
                                           (1152, [1, 40]), (1168, [40, 1]), (2304, [1, 3])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
def test_short_caches(ctx, dtype, heads, kv_heads, d, positions, new, window, sinks):
    # tables of up to 1,152 positions (16-row tiles at head_dim 64: 2,304), and longer ones
    rng = np.random.default_rng(positions + heads)
    lengths = [int(rng.integers(max(n, 1), positions - 15)) for n in new]
    lengths[0] = positions - 16  # (a Case's tables have a page more)
    c = Case8(ctx, positions + d, dtype, new, lengths, heads, kv_heads, d, 16)
    assert c.max_pages * c.page == positions
    paged.check_attention(c, window=window, sinks=sinks)
    if new[0] > 1:  # more tokens than positions: the first ones see nothing
        c.lengths[0], c.lengths[1] = 5, 0
        paged.check_attention(c, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
def test_not_numbers_and_large_scores_in_short_caches(ctx, dtype, d):
    # 700 tiles for at most 512 workgroups: those that share one with a NaN stay right
    lengths = [3 + 17 * i % 180 for i in range(350)]
    c = Case8(ctx, d, dtype, [1] * 350, lengths, 4, 2, d, 16)
    assert c.max_pages * c.page <= 256
    page, at = c.table[17, 0], 2
    c.kb[page, 0, at, 3] = 127
    page, at = c.table[40, 0], 1
    c.vs[page, 1, at] = 255
    q, got = paged.run_attention(c)
    ref, tol = paged.attention_oracle(c, from16(q, dtype), 0, 0, d ** -0.5)
    out, sound = from16(got, dtype)[:350], np.ones((350, 4), bool)
    sound[17, :2] = sound[40, 2:] = False
    assert np.isnan(out[~sound]).all()
    assert (np.abs(out - ref[:350]) <= tol[:350])[sound].all()
    large = Case8(ctx, d + 1, dtype, [1, 2, 1], [100, 60, 2], 4, 2, d, 16, scale=1.0)
    paged.check_attention(large, scale=300.0)


@pytest.mark.parametrize("group", [17, 128])
def test_many_query_heads(ctx, group):
    paged.check_attention(Case8(ctx, 16, "f16", [3, 1], [120, 300], group, 1, 64, 16))


def test_pool_past_2_to_32_bytes(ctx):
    # the sequence's pages are the pool's last ones, 5 GiB in
    d, kv_heads, page, num = 128, 8, 64, 42000
    small = Case8(ctx, 17, "f16", [1, 20], [200, 100], 8, 8, d, page)
    per = PagedKV8.page_bytes(kv_heads, page, d)
    pool, first = ctx.alloc(num * per), num - small.num_pages
    try:
        part = pool.view(first * per, small.num_pages * per)
        part.copy_from_host(small.bytes())
        table = np.where(small.table >= 0, small.table + first, -1).astype(np.int32)
        bufs = [ctx.upload(a) for a in (table, np.array(small.lengths, np.int32), small.starts)]
        kv = PagedKV8(pool, *bufs, **{**small.sizes(), "num_pages": num})
        q = to16(small.rng.normal(0, 1.5, (small.tokens, 8, d)), "f16")
        dq, out = ctx.upload(q), ctx.upload(to16(np.full(q.shape, 0.5), "f16"))
        scale = float(np.float32(d ** -0.5))
        for max_new, rows in ((20, 21), (1, 21)):
            work = ctx.alloc(ctx.attn_paged_workspace(kv, small.tokens, 8, max_new))
            ctx.attn_paged(kv, dq, out, small.tokens, 8, max_new, scale, work)
            ctx.sync()
            ref, tol = paged.attention_oracle(small, from16(q, "f16"), 0, 0, scale)
            assert (np.abs(from16(out.to_host(), "f16") - ref)[:rows] <= tol[:rows]).all()
            work.free()
        # and the append there
        qkv = ctx.upload(to16(small.rng.normal(0, 1, (small.tokens, 24, d)), "f16"))
        gain = ctx.upload(np.ones(d, np.float32))
        back = [ctx.alloc(small.tokens * 8 * d * 2) for _ in range(2)]
        ctx.qk_norm_rope_paged(kv, qkv, gain, gain, dq, small.tokens, 8, 1e-6, 1e4)
        ctx.paged_read(kv, *back, small.tokens)
        ctx.sync()
        v = from16(qkv.to_host().reshape(small.tokens, 24, d)[:21, 16:], "f16")
        b, s, _ = quantised(v, "f16")
        assert (from16(back[1].to_host(np.int16, (small.tokens, 8, d))[:21], "f16") == values(b, s)).all()
        for x in bufs + [dq, out, qkv, gain] + back:
            x.free()
    finally:
        pool.free()


# ---- refusals ------------------------------------------------------------------------------------

def refused(call, text, status=strict_amd.SH_ERR_INVALID_ARGUMENT):
    with pytest.raises(strict_amd.StrictHipError) as e:
        call()
    assert e.value.status == status and text in e.value.message, e.value.message


def test_refusals(ctx):
    c = Case8(ctx, 20, "f16", [1], [20], 4, 2, 64, 16)
    kv = c.upload()
    tokens, nbytes, pool = c.tokens, c.tokens * 4 * 64 * 2, c.buffers[0].nbytes
    q, out, k, v = (ctx.alloc(nbytes) for _ in range(4))
    qkv, gain = ctx.alloc(tokens * 8 * 64 * 2), ctx.upload(np.ones(64, np.float32))
    need = ctx.attn_paged_workspace(kv, tokens, 4, 1)
    work = ctx.alloc(need)
    small = ctx.alloc(need - 16)
    attend = lambda kv=kv, q=q, out=out, work=work, n=tokens, scale=1.0, **more: ctx.attn_paged(kv, q, out, n, 4, 1, scale, work, **more)  # noqa: E731
    append = lambda kv=kv, qkv=qkv, q=q, g=gain, n=tokens, **more: ctx.qk_norm_rope_paged(kv, qkv, g, gain, q, n, 4, 1e-6, 1e4, **more)  # noqa: E731
    read = lambda kv=kv, k=k, v=v, n=tokens: ctx.paged_read(kv, k, v, n)  # noqa: E731
    # sizes
    for name, value, text in (("batch", -1, "batch"), ("page_size", 24, "page_size"), ("num_pages", 0, "num_pages"),
                              ("max_pages", 1 << 28, "max_pages"), ("kv_heads", 0, "kv_heads")):
        bad = PagedKV8(*c.buffers, **{**c.sizes(), name: value})
        for call in (attend, append, read):
            refused(lambda: call(kv=bad), text)
    wide = PagedKV8(*c.buffers, **{**c.sizes(), "head_dim": 96})
    for call in (attend, append, read):
        refused(lambda: call(kv=wide), "head_dim", strict_amd._lib.SH_ERR_UNSUPPORTED)
        refused(lambda: call(n=-1), "tokens")
    huge = PagedKV8(*c.buffers, **{**c.sizes(), "num_pages": 1 << 30, "page_size": 65536, "kv_heads": 1024, "max_pages": 1, "head_dim": 128})
    refused(lambda: ctx.attn_paged_workspace(huge, 1, 1024, 1), "num_pages")
    refused(lambda: read(kv=huge), "num_pages")
    more = PagedKV8(*c.buffers, **{**c.sizes(), "num_pages": c.num_pages + 1})  # a page that is not there
    for call in (attend, append, read):
        refused(lambda: call(kv=more), "pages")
    refused(lambda: attend(work=small), "work buffer has")
    refused(lambda: attend(scale=0.0), "scale")
    refused(lambda: attend(window=-1), "window")
    refused(lambda: append(ld=8 * 64 - 8), "ld")
    refused(lambda: append(ld=8 * 64 + 4), "ld")
    # alignment
    off = lambda b: b.view(8, b.nbytes - 8)  # noqa: E731
    shifted = PagedKV8(c.buffers[0].ptr + 8, *c.buffers[1:], **{**c.sizes(), "num_pages": c.num_pages - 1})
    for call in (attend, append, read):
        refused(lambda: call(kv=shifted), "16-byte")
    refused(lambda: attend(q=off(q), n=tokens - 1), "16-byte")
    refused(lambda: attend(out=off(out), n=tokens - 1), "16-byte")
    refused(lambda: append(qkv=off(qkv), n=tokens - 1), "16-byte")
    refused(lambda: read(k=off(k), n=tokens - 1), "16-byte")
    # tensors over one another, the cache or the index
    inside = c.buffers[0]
    refused(lambda: attend(out=q), "overlaps")
    refused(lambda: attend(work=inside.view(0, min(need, pool)) if need <= pool else work, out=inside.view(0, nbytes)), "overlaps")
    refused(lambda: append(q=qkv.view(0, nbytes)), "overlaps")
    refused(lambda: append(q=inside.view(0, nbytes)), "overlaps")
    refused(lambda: append(qkv=inside.view(0, min(pool, qkv.nbytes))), "overlaps")
    refused(lambda: append(g=inside.view(0, 256)), "overlaps")
    refused(lambda: read(k=v), "overlaps")
    refused(lambda: read(k=inside.view(pool - nbytes // 16 * 16 if pool % 16 == 0 else 0, nbytes // 2)), "overlaps")
    area = ctx.alloc(need + nbytes + pool + 512)
    for i in (1, 2, 3):
        def indexed(at):
            b = list(c.buffers)
            b[i] = area.view(at, b[i].nbytes)
            return PagedKV8(*b, **c.sizes())
        for at in (256 + 4 - c.buffers[i].nbytes, 256 + nbytes - 4):
            refused(lambda: attend(kv=indexed(at), out=area.view(256, nbytes)), "page table")
            refused(lambda: append(kv=indexed(at), q=area.view(256, nbytes)), "page table")
        for at in (256 + 4 - c.buffers[i].nbytes, 256 + nbytes // 2 - 4):
            refused(lambda: read(kv=indexed(at), v=area.view(256, nbytes // 2)), "page table")
        for at in (256 + 4 - c.buffers[i].nbytes, 256 + need - 4):
            refused(lambda: attend(kv=indexed(at), work=area.view(256, need)), "work buffer overlaps")
    # null pointers
    refused(lambda: read(k=None), "k")
    refused(lambda: attend(q=None), "q")
    # nothing to do
    attend(n=0)
    append(n=0)
    read(n=0)
    for b in (q, out, k, v, qkv, gain, work, small, area):
        b.free()
    c.free()
