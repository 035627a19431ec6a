"""A decoder layer's step in few bits as a server runs it: 4-bit linears, head norms with
RoPE into pages of 8-bit values, attention over them, the LM head, rules on its logits and
the draw; with forks and moves in the pool, captured into graphs, in contexts at once. Each
operator is checked against 64 bits on what the one before it gave."""
import ctypes
import threading

import numpy as np
import pytest

import strict_amd
import test_gpu_gemv4 as gemv4
import test_gpu_paged as paged
import test_gpu_paged8 as paged8
import test_gpu_sample as sampling
from strict_amd import PagedKV8
from strict_amd.paged import PagedCache
from test_gpu_logits import Rules
from test_gpu_paged import F, U, from16, to16
from test_gpu_paged_serving import EPS, LONG, THETA, Captured, same

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return ctypes.CDLL("libamdhip64.so")


class Linear:
    def __init__(self, ctx, rng, n, k):
        self.code, self.scale = gemv4.random_weights(rng, n, k, around=-6, spread=1)
        self.n, self.k = n, k
        q, s = ctx.upload(gemv4.packed(self.code)), ctx.upload(self.scale)
        self.tiled = ctx.alloc(ctx.e2m1_tiles_bytes(n, k))
        ctx.pack_e2m1_tiles(q, s, self.tiled, n, k)
        ctx.sync()
        q.free()
        s.free()

    def check(self, got, x, dtype, out):
        gemv4.check(got, self.code, self.scale, x, dtype, out)


class Model:
    """One layer and a head over a cache of 8-bit pages; `most` tokens a step."""

    def __init__(self, ctx, seed, dtype, heads, kv_heads, d, vocab, most, **cache):
        rng = self.rng = np.random.default_rng(seed)
        self.ctx, self.dtype, self.heads, self.kv_heads, self.d, self.vocab = ctx, dtype, heads, kv_heads, d, vocab
        self.hidden, self.all_heads = heads * d, heads + 2 * kv_heads
        self.linears = [Linear(ctx, rng, n, k) for n, k in ((self.all_heads * d, self.hidden), (self.hidden, self.hidden), (vocab, self.hidden))]
        self.cache = PagedCache(ctx, 1, kv_heads, d, dtype=dtype, bits=8, **cache)
        ctx.memset(self.cache.pool, 0xff)  # NaN wherever nothing was written
        self.kv = self.cache.kv[0]
        self.gains = [(1 + rng.normal(0, 0.3, d)).astype(np.float32) for _ in range(2)]
        self.gain_bufs = [ctx.upload(g) for g in self.gains]
        empty = lambda *shape, t=np.int16: ctx.empty(shape, t)  # noqa: E731
        self.b = dict(x=empty(most, self.hidden), qkv=empty(most, self.all_heads, d), q=empty(most, heads, d),
                      out=empty(most, heads, d), o=empty(most, self.hidden), logits=empty(most, vocab, t=np.float32),
                      index=empty(most, t=np.int32), k=empty(most, kv_heads, d), v=empty(most, kv_heads, d))
        self.u = rng.random(most).astype(np.float32)
        self.b["u"] = ctx.upload(self.u)
        self.rules = Rules(vocab, tokens=rng.integers(0, vocab, (most, 30)).astype(np.int32), lengths=rng.integers(0, 31, most).astype(np.int32),
                           repetition=np.full(most, 1.3, np.float32), presence=np.full(most, 0.5, np.float32),
                           masks=rng.integers(0, 1 << 32, (1, (vocab + 31) // 32), dtype=np.uint32),
                           mask_of=rng.integers(-1, 1, most).astype(np.int32))
        self.rule_bufs = self.rules.upload(ctx)
        self.work = ctx.alloc(max(ctx.attn_paged_workspace(self.kv, most, heads, most), ctx.sample_workspace(most, vocab)))
        self.said = [[[], []] for _ in range(cache["rows"])]

    def inputs(self, seed, tokens):
        x = to16(np.random.default_rng(seed).normal(0, 1, (tokens, self.hidden)), self.dtype)
        self.b["x"].copy_from_host(x)
        return x

    def run(self, tokens, max_new):
        ctx, b, d, t = self.ctx, self.b, self.d, self.dtype
        qkv, o, head = self.linears
        ctx.gemv_w4a16(b["x"], qkv.tiled, b["qkv"], tokens, qkv.k, qkv.n, dtype=t, out=t)
        ctx.qk_norm_rope_paged(self.kv, b["qkv"], *self.gain_bufs, b["q"], tokens, self.heads, EPS, THETA)
        ctx.attn_paged(self.kv, b["q"], b["out"], tokens, self.heads, max_new, float(np.float32(d ** -0.5)), self.work)
        ctx.gemv_w4a16(b["out"], o.tiled, b["o"], tokens, o.k, o.n, dtype=t, out=t)
        ctx.gemv_w4a16(b["o"], head.tiled, b["logits"], tokens, head.k, head.n, dtype=t)
        self.adjust(tokens)
        ctx.sample(b["logits"], tokens, self.vocab, None, None, None, None, b["u"], b["index"], self.work)
        ctx.paged_read(self.kv, b["k"], b["v"], tokens)

    def adjust(self, tokens):
        self.ctx.adjust_logits(self.b["logits"], self.b["logits"], tokens, self.vocab, self.rule_bufs)

    def host(self, name, tokens):
        return self.b[name].to_host()[:tokens]

    def results(self, tokens):
        self.ctx.sync()
        return [self.host(n, tokens).copy() for n in ("qkv", "q", "out", "o", "logits", "index", "k", "v")]

    def step(self, new):
        tokens, table, dtype = self.cache.step(new), self.cache.table, self.dtype
        x = self.inputs(int(self.rng.integers(1 << 30)), tokens)
        self.run(tokens, max(new.values()))
        self.ctx.sync()
        qkv, o, head = self.linears
        val = lambda n: from16(self.host(n, tokens), dtype)  # noqa: E731
        rows = val("qkv")
        qkv.check(rows.reshape(tokens, -1), from16(x, dtype), dtype, dtype)
        got_q, out, at = val("q"), val("out"), 0
        for row in sorted(r for r, n in new.items() if n):
            n, length = new[row], table.lengths[row]
            pos, mine = np.arange(length - n, length), slice(at, at + n)
            ref, size = paged.norm_rope_oracle(rows[mine, :self.heads], self.gains[0].astype(np.float64), pos.astype(np.float64), EPS, THETA)
            assert (np.abs(got_q[mine] - ref) <= U[dtype] * np.abs(ref) + 32 * F * size + 2.0 ** -25).all()
            k, _ = paged.norm_rope_oracle(rows[mine, self.heads:self.heads + self.kv_heads], self.gains[1].astype(np.float64), pos.astype(np.float64), EPS, THETA)
            byte, scale, margin = paged8.quantised(k, dtype)
            stored = val("k")[mine]
            assert ((stored == paged8.values(byte, scale)) | (margin < 2.0 ** -36)).all()
            byte, scale, _ = paged8.quantised(rows[mine, self.heads + self.kv_heads:], dtype)
            assert (val("v")[mine] == paged8.values(byte, scale)).all()
            ks, vs = self.said[row]
            ks.extend(self.host("k", tokens)[mine])
            vs.extend(self.host("v", tokens)[mine])
            assert len(ks) == length
            ref, tol = paged.attention_oracle(History(self, row, n), got_q[mine], 0, 0, float(np.float32(self.d ** -0.5)))
            assert (np.abs(out[mine] - ref) <= tol).all(), row
            at += n
        o.check(val("o"), out.reshape(tokens, -1), dtype, dtype)
        # the head before and after the rules, and the draw
        adjusted, index = self.host("logits", tokens), self.host("index", tokens)
        self.ctx.gemv_w4a16(self.b["o"], head.tiled, self.b["logits"], tokens, head.k, head.n, dtype=dtype)
        self.ctx.sync()
        plain = self.host("logits", tokens)
        head.check(plain.astype(np.float64), val("o"), dtype, "f32")
        a = {name: v if name == "masks" else v[:tokens] for name, v in self.rules.arrays.items()}
        assert np.array_equal(Rules(self.vocab, **a).oracle(plain), adjusted)
        for r in range(tokens):
            sampling.check(self.ctx, adjusted[r:r + 1], None, None, None, None, self.u[r:r + 1])
        assert np.array_equal(index, sampling.sample(self.ctx, adjusted, None, None, None, None, self.u[:tokens]))

    def fork(self, row, to):
        self.cache.fork(row, to)
        self.said[to] = [list(x) for x in self.said[row]]

    def free(self, row):
        self.cache.free(row)
        self.said[row] = [[], []]

    def dispose(self):
        self.cache.dispose()
        for b in [*self.b.values(), *self.gain_bufs, self.work, *(l.tiled for l in self.linears)]:
            b.free()
        self.rules.free()


class History:
    """A sequence as attention_oracle takes one: its tokens in one page."""

    def __init__(self, model, row, n):
        ks, vs = model.said[row]
        self.dtype, self.heads, self.kv_heads, self.d = model.dtype, model.heads, model.kv_heads, model.d
        self.batch, self.new, self.lengths, self.starts = 1, [n], [len(ks)], [0]
        self.k, self.v = (np.array(x).swapaxes(0, 1) for x in (ks, vs))

    def gathered(self, bits, b, kv_head):
        return from16(bits[kv_head], self.dtype), np.ones(bits.shape[1], bool)


@pytest.mark.parametrize("dtype,heads,kv_heads,d,page", [("f16", 8, 2, 64, 16), ("bf16", 4, 4, 128, 32)])
def test_a_server(ctx, dtype, heads, kv_heads, d, page):
    # prompts, decode, a fork whose rows part, an end, a compaction, a late prompt
    m = Model(ctx, 1, dtype, heads, kv_heads, d, 1003, 60, rows=4, max_pages=300 // page, num_pages=500 // page, page_size=page)
    m.step({0: 40, 2: 13})
    m.step({0: 1, 2: 1, 3: 50})
    m.fork(0, 1)
    for _ in range(2):
        m.step({0: 1, 1: 1, 2: 1, 3: 1})
    assert m.cache.table.pages[0][-1] != m.cache.table.pages[1][-1]
    m.free(0)
    m.free(2)
    m.step({1: 1, 3: 1})
    before = m.cache.table.array()
    assert m.cache.compact() > 0 and (before != m.cache.table.array()).any()
    m.step({1: 2, 0: 47, 3: 1})
    m.dispose()


@pytest.mark.parametrize("max_pages", [20, 300])  # (tiles of the second are cut)
def test_captured_steps(hip, max_pages):
    # replays with other values, eager steps of another model in between, two graphs of one work buffer
    with strict_amd.Context(0) as ctx:
        make = lambda seed, new: (Model(ctx, seed, "f16", 4, 2, 64, 700, 40, rows=3, max_pages=max_pages, num_pages=70, page_size=16), new)  # noqa: E731
        models = [make(3, {0: 1, 1: 1, 2: 1}), make(4, {0: 30, 2: 5})]
        for m, new in models:
            m.cache.step({0: 20, 1: 13, 2: 7})
            m.inputs(1, 40)
            m.run(40, 20)
            m.tokens = m.cache.step(new)
        models[1][0].work.free()
        models[1][0].work = models[0][0].work
        eager = []
        for m, new in models:
            got = []
            for i in range(3):
                m.inputs(10 + i, m.tokens)
                m.run(m.tokens, max(new.values()))
                got.append(m.results(m.tokens))
            eager.append(got)
        graphs = [Captured(hip, ctx, type("", (), {"run": lambda self, m=m, new=new: m.run(m.tokens, max(new.values()))})()) for m, new in models]
        for i in (0, 1, 2, 1, 0):
            for m, _ in models:
                m.inputs(10 + i, m.tokens)
                for name in ("q", "out", "o", "logits", "index", "k", "v"):
                    ctx.memset(m.b[name], 0xff)
            for g in (graphs, graphs[::-1])[i % 2]:
                g.launch()
            for (m, _), want in zip(models, eager):
                assert same(m.results(m.tokens), want[i]), i
            m, new = models[i % 2]
            m.inputs(10, m.tokens)
            m.run(m.tokens, max(new.values()))  # (eager between the replays)
        for g in graphs:
            g.destroy()
        models[1][0].work = ctx.alloc(16)
        for m, _ in models:
            m.dispose()


def test_contexts_at_once():
    # a thread and a stream each: as alone
    def work(i, results):
        with strict_amd.Context(0) as ctx:
            m = Model(ctx, 20 + i, "bf16", 4, 1, 128, 900 + i, 30, rows=2, max_pages=9, num_pages=20, page_size=32)
            got = []
            for j, new in enumerate(({0: 25}, {0: 1, 1: 20 + i}, {0: 1, 1: 1})):
                tokens = m.cache.step(new)
                m.inputs(j, tokens)
                m.run(tokens, max(new.values()))
                got.append(m.results(tokens))
            m.dispose()
            results[i] = got
    alone, together = {}, {}
    for i in range(3):
        work(i, alone)
    threads = [threading.Thread(target=work, args=(i, together)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(3):
        assert all(same(a, b) for a, b in zip(alone[i], together[i])), i


def test_pages_of_other_sizes_are_refused_by_the_cache(ctx):
    with pytest.raises(ValueError):
        PagedCache(ctx, 1, 2, 64, rows=1, max_pages=2, num_pages=4, bits=4)
    with pytest.raises(strict_amd.StrictHipError):
        PagedCache(ctx, 1, 2, 96, rows=1, max_pages=2, num_pages=4, bits=8)


# ---- chunks announced as long, and what the device may hold ---------------------------------

@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d,page", [(16, 8, 128, 16), (4, 4, 64, 32), (6, 2, 128, 64), (7, 1, 64, 128), (128, 1, 64, 16)])
@pytest.mark.parametrize("new,lengths", [([1], [1]), ([300, 0, 2], [300, 9, 900]), ([33, 140, 257, 20], [100, 1500, 257, 3000])])
def test_long_chunks(ctx, dtype, heads, kv_heads, d, page, new, lengths):
    if heads == 128 and sum(new) > 400:
        new, lengths = [33, 20], [100, 700]
    paged.check_attention(paged8.Case8(ctx, sum(new) + d, dtype, new, lengths, heads, kv_heads, d, page, first_row=2), max_new=LONG)


@pytest.mark.parametrize("heads,kv_heads,d", [(8, 4, 128), (6, 2, 64)])
@pytest.mark.parametrize("window,sinks", [(1, 1), (7, 4), (100, 130)])
def test_long_chunks_with_windows_and_bad_pages(ctx, heads, kv_heads, d, window, sinks):
    c = paged8.Case8(ctx, window + sinks, "bf16", [350, 20, 1], [900, 333, 1], heads, kv_heads, d, 16)
    paged.check_attention(c, window=window, sinks=sinks, max_new=LONG)
    c.table[0, 0], c.table[0, 3], c.table[0, 42], c.table[1, 5:9] = -1, c.num_pages, 1 << 30, -7
    paged.check_attention(c, window=window, sinks=sinks, max_new=LONG)
    paged.check_attention(c, max_new=LONG)


@pytest.mark.parametrize("extra", [1, 300])
@pytest.mark.parametrize("new", [[1, 1, 1], [40, 200, 9], [3] * 130, [40] * 70])
def test_starts_and_lengths_that_are_not_theirs(ctx, new, extra):
    # whatever the device holds there, only rows of the results and pages of the cache are written
    n = len(new)
    c = paged8.Case8(ctx, 31, "f16", new, [300] * n, 4, 2, 64, 16, rows_behind=3, extra_entries=extra)
    c.upload()
    nbytes, pool = c.tokens * 4 * 64 * 2, c.buffers[0].nbytes
    guarded, pages = ctx.alloc(3 * nbytes), ctx.alloc(pool + 2048)
    kv = PagedKV8(pages.view(1024, pool), *c.buffers[1:], **c.sizes())
    out, k, v = guarded.view(nbytes, nbytes), guarded.view(nbytes, nbytes // 2), guarded.view(nbytes + nbytes // 2, nbytes // 2)
    dq = ctx.upload(to16(c.rng.normal(0, 1, (c.tokens, 4, 64)), "f16"))
    qkv = ctx.upload(to16(c.rng.normal(0, 1, (c.tokens, 8, 64)), "f16"))
    gain = ctx.upload(np.ones(64, np.float32))
    work = ctx.alloc(ctx.attn_paged_workspace(kv, c.tokens, 4, max(new)))
    rng = np.random.default_rng(32)
    ends = np.array([0, 1, -1, c.tokens, c.tokens + 1, 7, np.iinfo(np.int32).max, np.iinfo(np.int32).min], np.int64)
    for _ in range(20):
        c.buffers[2].copy_from_host(rng.choice(np.append(ends, 300), n).astype(np.int32))
        c.buffers[3].copy_from_host(rng.choice(ends, n + 1).astype(np.int32))
        ctx.memset(guarded, 0x5a)
        ctx.memset(pages, 0x5a)
        pages.view(1024, pool).copy_from_host(c.bytes())
        ctx.attn_paged(kv, dq, out, c.tokens, 4, max(new), 0.125, work, int(rng.choice([0, 50])), 4)
        ctx.paged_read(kv, k, v, c.tokens)
        ctx.sync()
        assert (pages.to_host()[1024:1024 + pool] == c.bytes().reshape(-1)).all()
        ctx.qk_norm_rope_paged(kv, qkv, gain, gain, out, c.tokens, 4, EPS, THETA)
        ctx.sync()
        host, around = guarded.to_host(), pages.to_host()
        assert (host[:nbytes] == 0x5a).all() and (host[2 * nbytes:] == 0x5a).all()
        assert (around[:1024] == 0x5a).all() and (around[1024 + pool:] == 0x5a).all()
    for b in (guarded, pages, dq, qkv, gain, work):
        b.free()
    c.free()
