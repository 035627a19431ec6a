"""The operators over a KV cache in pages as a server uses them together: sequences
that start, fork, end and move in the pool, steps captured into a graph, two
contexts at once. Values are checked against the formulas in 64 bits (as in
test_gpu_paged.py, whose tolerances these are)."""
import ctypes
import threading

import numpy as np
import pytest

import strict_amd
import test_gpu_paged as paged
import test_gpu_sample as sampling
from strict_amd.paged import OutOfPages, PagedCache

pytestmark = pytest.mark.gpu

THREAD_LOCAL = 1  # hipStreamCaptureModeThreadLocal
EPS, THETA = float(np.float32(1e-6)), 1e4


@pytest.fixture(scope="module")
def hip():
    return ctypes.CDLL("libamdhip64.so")


class Server:
    """A cache of `layers` layers with what each sequence's tokens were: k as the
    device stored it (checked when it was written), v as it was given."""

    def __init__(self, ctx, seed, dtype, layers, heads, kv_heads, d, vocab, **cache):
        self.rng, self.ctx, self.dtype, self.vocab = np.random.default_rng(seed), ctx, dtype, vocab
        self.heads, self.kv_heads, self.d = heads, kv_heads, d
        self.cache = PagedCache(ctx, layers, kv_heads, d, dtype=dtype, **cache)
        ctx.memset(self.cache.pool, 0xff)  # NaN wherever nothing was written
        self.said = [[([], []) for _ in range(layers)] for _ in range(cache["rows"])]  # [row][layer]
        self.gains = [(1 + self.rng.normal(0, 0.3, d)).astype(np.float32) for _ in range(2)]
        self.gain_bufs = [ctx.upload(g) for g in self.gains]

    def plane(self, layer, which):
        t = self.cache.table
        shape = (t.num_pages, self.kv_heads, t.page_size, self.d)
        nbytes = t.num_pages * self.cache.page_bytes
        return self.cache.pool.view((2 * layer + which) * nbytes, nbytes, np.int16, shape).to_host()

    def fork(self, row, to):
        self.cache.fork(row, to)
        self.said[to] = [(list(k), list(v)) for k, v in self.said[row]]

    def free(self, row):
        self.cache.free(row)
        self.said[row] = [([], []) for _ in self.said[row]]

    def step(self, new, window=0, sinks=0):
        """A step of all layers, each operator checked; returns the sampled tokens."""
        ctx, rng, d = self.ctx, self.rng, self.d
        tokens, all_heads = self.cache.step(new), self.heads + 2 * self.kv_heads
        table, rows = self.cache.table, sorted(r for r, n in new.items() if n)
        max_new = max(new.values())
        q = ctx.alloc(tokens * self.heads * d * 2).view(0, tokens * self.heads * d * 2, np.int16, (tokens, self.heads, d))
        out = ctx.upload(paged.to16(np.full((tokens, self.heads, d), 0.5), self.dtype))
        work = ctx.alloc(ctx.attn_paged_workspace(self.cache.kv[0], tokens, self.heads, max_new))
        scale = float(np.float32(d ** -0.5))
        for layer, kv in enumerate(self.cache.kv):
            bits = paged.to16(rng.normal(0, 1.5, (tokens, all_heads, d)), self.dtype)
            qkv = ctx.upload(bits)
            ctx.qk_norm_rope_paged(kv, qkv, *self.gain_bufs, q, tokens, self.heads, EPS, THETA)
            ctx.attn_paged(kv, q, out, tokens, self.heads, max_new, scale, work, window, sinks)
            ctx.sync()
            kd, vd = self.plane(layer, 0), self.plane(layer, 1)
            x, got_q, got = paged.from16(bits, self.dtype), paged.from16(q.to_host(), self.dtype), paged.from16(out.to_host(), self.dtype)
            u, at = paged.U[self.dtype], 0
            for row in rows:
                n, length = new[row], table.lengths[row]
                pos = np.arange(length - n, length)
                page, slot = np.array(table.pages[row])[pos // table.page_size], pos % table.page_size
                mine = slice(at, at + n)
                for part, gain, stored in ((x[mine, :self.heads], self.gains[0], got_q[mine]),
                                           (x[mine, self.heads:self.heads + self.kv_heads], self.gains[1],
                                            paged.from16(kd[page, :, slot], self.dtype))):
                    ref, size = paged.norm_rope_oracle(part, gain.astype(np.float64), pos.astype(np.float64), EPS, THETA)
                    assert (np.abs(stored - ref) <= u * np.abs(ref) + 32 * paged.F * size + 2.0 ** -25).all()
                ks, vs = self.said[row][layer]
                ks.extend(kd[page, :, slot])
                vs.extend(bits[mine, self.heads + self.kv_heads:])
                assert len(ks) == length
                # the whole sequence is where the table says, as it was written
                pos = np.arange(length)
                page, slot = np.array(table.pages[row])[pos // table.page_size], pos % table.page_size
                assert (kd[page, :, slot] == np.array(ks)).all() and (vd[page, :, slot] == np.array(vs)).all()
                seq = History(self, row, layer, n)
                ref, tol = paged.attention_oracle(seq, got_q[mine], window, sinks, scale)
                assert (np.abs(got[mine] - ref) <= tol).all(), (row, layer)
                at += n
            qkv.free()
        logits = rng.normal(0, 2.5, (tokens, self.vocab)).astype(np.float32)
        u = rng.random(tokens).astype(np.float32)
        t, k, p = (np.resize(v, tokens) for v in (np.float32([0.7, 0.0, 1.3]), np.int32([50, 0, 0]), np.float32([1, 0.9, 0.8])))
        sampling.check(ctx, logits, t, k, p, None, u)
        for b in (q, out, work):
            b.free()

    def dispose(self):
        self.cache.dispose()
        for b in self.gain_bufs:
            b.free()


class History:
    """A sequence as attention_oracle takes one: its tokens in one page."""

    def __init__(self, server, row, layer, n):
        ks, vs = server.said[row][layer]
        self.dtype, self.heads, self.kv_heads, self.d = server.dtype, server.heads, server.kv_heads, server.d
        self.batch, self.new, self.lengths, self.starts = 1, [n], [len(ks)], [0]
        self.k, self.v = (np.array(x).swapaxes(0, 1) for x in (ks, vs))

    def gathered(self, bits, b, kv_head):
        return paged.from16(bits[kv_head], self.dtype), np.ones(bits.shape[1], bool)


@pytest.mark.parametrize("dtype,heads,kv_heads,d,page", [("f16", 8, 2, 64, 16), ("bf16", 4, 4, 128, 32)])
def test_a_server(ctx, dtype, heads, kv_heads, d, page):
    # prompts, decode, a fork whose rows part, an end, a compaction, a late prompt
    s = Server(ctx, 1, dtype, 2, heads, kv_heads, d, 2500, rows=4, max_pages=300 // page, num_pages=700 // page,
               page_size=page)
    s.step({0: 100, 2: 37})
    s.step({0: 1, 2: 1, 3: 150})
    s.fork(0, 1)
    for _ in range(3):
        s.step({0: 1, 1: 1, 2: 1, 3: 1})
    assert s.cache.table.pages[0][-1] != s.cache.table.pages[1][-1]
    s.free(0)
    s.free(2)
    s.step({1: 1, 3: 1})
    before = s.cache.table.array()
    assert s.cache.compact() > 0 and (before != s.cache.table.array()).any()
    s.step({1: 1, 3: 1})
    s.step({1: 2, 0: 130, 3: 1}, window=40, sinks=4)
    with pytest.raises(OutOfPages):
        s.cache.step({2: 301})
    s.step({0: 1, 1: 1, 3: 1}, window=40, sinks=4)
    s.dispose()


def test_rows_that_share_a_page_in_the_middle(ctx):
    # forks of a fork that part at once: one copy each but for the last holder
    s = Server(ctx, 2, "f16", 1, 2, 1, 64, 300, rows=4, max_pages=8, num_pages=20, page_size=16)
    s.step({0: 21})
    for to in (1, 2, 3):
        s.fork(to - 1, to)
    s.step({0: 1, 1: 3, 2: 16, 3: 1})
    s.step({0: 1, 1: 1, 2: 1, 3: 1})
    s.dispose()


class Step:
    """One step's operators on buffers that stay: head norms and pages, attention,
    a page copy, and a token from the attention's values as logits."""

    def __init__(self, ctx, seed, new, lengths, heads=4, kv_heads=2, d=64, page=16, work=None):
        self.ctx = ctx
        self.c = c = paged.Case(ctx, seed, "f16", new, lengths, heads, kv_heads, d, page, rows_behind=0, spare=2, extra_entries=4)
        # (every entry a page of its own, so that lengths may grow)
        c.num_pages = c.batch * c.max_pages + 2
        order = c.rng.permutation(c.num_pages - 2).astype(np.int32)
        c.table = order.reshape(c.batch, c.max_pages)
        shape = (c.num_pages, kv_heads, page, d)
        c.k, c.v = (paged.to16(c.rng.normal(0, 1, shape), "f16") for _ in range(2))
        self.kv = c.upload()
        self.max_new = max(new)
        self.vocab = heads * d * c.tokens // 2
        self.bufs = dict(
            qkv=ctx.empty((c.tokens, heads + 2 * kv_heads, d), np.int16), q=ctx.empty((c.tokens, heads, d), np.int16),
            out=ctx.empty((c.tokens, heads, d), np.int16), gain=ctx.upload(np.ones(d, np.float32)),
            src=ctx.upload(np.array([order[0]], np.int32)), dst=ctx.upload(np.array([c.num_pages - 1], np.int32)),
            k=ctx.upload(np.array([40, 0], np.int32)), p=ctx.upload(np.array([1, 0.9], np.float32)),
            u=ctx.upload(np.array([0.3, 0.6], np.float32)), index=ctx.empty(2, np.int32),
            logits=ctx.empty((2, 5000), np.float32))
        need = max(ctx.attn_paged_workspace(self.kv, c.tokens, heads, self.max_new), ctx.sample_workspace(2, 5000))
        self.mine = work is None
        self.work = ctx.alloc(need) if work is None else work
        assert self.work.nbytes >= need

    def inputs(self, seed, more):
        """New tokens' values and lengths, as the next step has them."""
        rng, c, b = np.random.default_rng(seed), self.c, self.bufs
        b["qkv"].copy_from_host(paged.to16(rng.normal(0, 1.5, b["qkv"].shape), "f16"))
        b["logits"].copy_from_host(rng.normal(0, 2, (2, 5000)).astype(np.float32))
        c.buffers[0].copy_from_host(c.k)
        c.buffers[1].copy_from_host(c.v)
        c.buffers[3].copy_from_host(np.array([min(l + more, c.max_pages * c.page) for l in c.lengths], np.int32))

    def run(self):
        ctx, c, b = self.ctx, self.c, self.bufs
        ctx.qk_norm_rope_paged(self.kv, b["qkv"], b["gain"], b["gain"], b["q"], c.tokens, c.heads, EPS, THETA)
        ctx.attn_paged(self.kv, b["q"], b["out"], c.tokens, c.heads, self.max_new, 0.125, self.work, 90, 4)
        ctx.pages_copy(c.buffers[0], 1, c.num_pages, c.kv_heads * c.page * c.d * 2, b["src"], b["dst"], 1)
        ctx.sample(b["logits"], 2, 5000, None, b["k"], b["p"], None, b["u"], b["index"], self.work)

    def results(self):
        self.ctx.sync()
        return [x.to_host().copy() for x in (self.bufs["q"], self.bufs["out"], self.bufs["index"], *self.c.buffers[:2])]

    def clear(self):
        self.ctx.memset(self.bufs["out"], 0xff)
        self.ctx.memset(self.bufs["index"], 0xff)

    def free(self):
        for b in self.bufs.values():
            b.free()
        self.c.free()
        if self.mine:
            self.work.free()


def same(a, b):
    return all(np.array_equal(x, y) for x, y in zip(a, b))


class Captured:
    def __init__(self, hip, ctx, step):
        self.hip, self.ctx = hip, ctx
        stream, graph, self.run = ctypes.c_void_p(ctx.stream()), ctypes.c_void_p(), ctypes.c_void_p()
        assert hip.hipStreamBeginCapture(stream, THREAD_LOCAL) == 0
        try:
            step.run()
        finally:
            ended = hip.hipStreamEndCapture(stream, ctypes.byref(graph))
        assert ended == 0
        assert hip.hipGraphInstantiate(ctypes.byref(self.run), graph, None, None, ctypes.c_size_t(0)) == 0
        assert hip.hipGraphDestroy(graph) == 0

    def launch(self):
        assert self.hip.hipGraphLaunch(self.run, ctypes.c_void_p(self.ctx.stream())) == 0

    def destroy(self):
        assert self.hip.hipGraphExecDestroy(self.run) == 0


@pytest.mark.parametrize("new,lengths", [([1, 1, 1], [300, 40, 17]), ([30, 1, 90], [400, 40, 90])])
def test_captured_steps(hip, new, lengths):
    # replays with other values and lengths, with eager steps in between, repeat the eager results
    with strict_amd.Context(0) as ctx:
        step, other = Step(ctx, 3, new, lengths), Step(ctx, 4, [1, 9], [100, 9])
        other.inputs(0, 0)
        other.run()
        first = other.results()
        graph = Captured(hip, ctx, step)
        for i in range(5):
            step.inputs(i, 7 * i)
            step.run()
            eager = step.results()
            step.inputs(i, 7 * i)
            step.clear()
            if i % 2:
                other.inputs(0, 0)
                other.run()  # (nothing waits between)
            graph.launch()
            assert same(step.results(), eager), i
            assert same(other.results(), first), i
        graph.destroy()
        step.free()
        other.free()


def test_two_graphs_of_one_work_buffer(hip):
    # in turn on one stream
    with strict_amd.Context(0) as ctx:
        work = ctx.alloc(64 << 20)
        steps = [Step(ctx, 5, [1, 1], [500, 90], work=work), Step(ctx, 6, [140, 3], [300, 60], work=work)]
        want, graphs = [], []
        for s in steps:
            s.inputs(1, 0)
            s.run()
            want.append(s.results())
            graphs.append(Captured(hip, ctx, s))
        for _ in range(3):
            for s in steps:
                s.inputs(1, 0)
                s.clear()
            for g in graphs + graphs[::-1]:
                g.launch()
            for s, w in zip(steps, want):
                assert same(s.results(), w)
        for g in graphs:
            g.destroy()
        for s in steps:
            s.free()
        work.free()


def test_contexts_at_once():
    # a thread and a stream each, buffers of its own: as alone
    def work(i, results):
        with strict_amd.Context(0) as ctx:
            step = Step(ctx, 10 + i, [1, 60 + i, 5], [900, 61 + i, 400])
            got = []
            for j in range(6):
                step.inputs(j, j)
                step.run()
                got.append(step.results())
            step.free()
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


def test_a_page_in_several_tables_and_twice_in_one(ctx):
    # what is only read may be shared in any way
    c = paged.Case(ctx, 21, "bf16", [1, 1, 40], [100, 100, 140], 4, 2, 64, 16)
    c.table[1, :6] = c.table[0, :6]
    c.table[2, 1:4] = c.table[2, 0]
    paged.check_attention(c)


@pytest.mark.parametrize("new", [[1, 1], [40, 7]])
@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (1, 2 ** 31 - 1)])
def test_largest_windows_and_sinks(ctx, new, window, sinks):
    # rows before position 0 among them
    c = paged.Case(ctx, 22, "f16", new, [200, 7], 4, 2, 64, 16)
    c.lengths[1] = min(5, new[1])
    paged.check_attention(c, window=window, sinks=sinks)


def refused(call, text):
    with pytest.raises(strict_amd.StrictHipError) as e:
        call()
    assert e.value.status == strict_amd.SH_ERR_INVALID_ARGUMENT and text in e.value.message, e.value.message


def test_tensors_that_overlap(ctx):
    c = paged.Case(ctx, 23, "f16", [1], [20], 4, 2, 64, 16)
    kv = c.upload()
    need = ctx.attn_paged_workspace(kv, c.tokens, 4, 1)
    nbytes = c.tokens * 4 * 64 * 2
    big = ctx.alloc(need + 4 * nbytes)
    work, inside, behind = big.view(0, need), big.view(need - 16, nbytes), big.view(need + nbytes, nbytes)
    attn = lambda q, out, work, scale=1.0, kv=kv: (  # noqa: E731
        lambda: ctx.attn_paged(kv, q, out, c.tokens, 4, 1, scale, work))
    refused(attn(inside, behind, work), "work buffer overlaps")
    refused(attn(behind, inside, work), "work buffer overlaps")
    refused(attn(behind, c.buffers[0], work), "out overlaps the cache")
    refused(attn(behind, c.buffers[1], work), "out overlaps the cache")
    pool = ctx.alloc(need + c.buffers[0].nbytes)
    low = strict_amd.PagedKV(pool, *c.buffers[1:], batch=1, max_pages=c.max_pages, num_pages=c.num_pages, page_size=16,
                             kv_heads=2, head_dim=64, dtype="f16")
    refused(attn(behind, big.view(need + 2 * nbytes, nbytes), pool, kv=low), "work buffer overlaps")
    refused(attn(behind, big.view(need + 2 * nbytes, nbytes), work, 3e38), "scale")
    gain = ctx.upload(np.ones(64, np.float32))
    qkv = ctx.alloc(c.tokens * 8 * 64 * 2)
    same = strict_amd.PagedKV(c.buffers[0], c.buffers[0], *c.buffers[2:], batch=1, max_pages=c.max_pages,
                              num_pages=c.num_pages, page_size=16, kv_heads=2, head_dim=64, dtype="f16")
    rope = lambda kv, qkv, q: (lambda: ctx.qk_norm_rope_paged(kv, qkv, gain, gain, q, c.tokens, 4, 1e-6, 1e4))  # noqa: E731
    refused(rope(same, qkv, behind), "k and v pages overlap")
    refused(rope(kv, qkv, c.buffers[1]), "cache overlaps")
    refused(rope(kv, c.buffers[0], behind), "cache overlaps")
    for b in (big, pool, gain, qkv):
        b.free()
    c.free()
    need = ctx.sample_workspace(2, 4000)
    big = ctx.alloc(need + 64000)
    small = ctx.upload(np.zeros(2, np.float32))
    index = ctx.empty(2, np.int32)
    refused(lambda: ctx.sample(big.view(need - 64, 32000), 2, 4000, None, None, None, None, small, index, big.view(0, need)),
            "work buffer overlaps x")
    for b in (big, small, index):
        b.free()


# ---- chunks announced as long ----------------------------------------------------------

LONG = 100000


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d,page", [(16, 8, 128, 16), (4, 4, 64, 32), (6, 2, 128, 64), (7, 1, 64, 128), (128, 1, 64, 16)])
@pytest.mark.parametrize("new,lengths", [([1], [1]), ([300, 0, 2], [300, 9, 900]), ([33, 140, 257, 20], [100, 1500, 257, 3000])])
def test_long_chunks(ctx, dtype, heads, kv_heads, d, page, new, lengths):
    if heads == 128 and sum(new) > 400:
        new, lengths = [33, 20], [100, 700]
    paged.check_attention(paged.Case(ctx, sum(new) + d, dtype, new, lengths, heads, kv_heads, d, page, first_row=2), max_new=LONG)


@pytest.mark.parametrize("heads,kv_heads,d", [(8, 4, 128), (6, 2, 64)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 4), (64, 64), (100, 130), (5000, 4)])
def test_long_chunks_with_windows(ctx, heads, kv_heads, d, window, sinks):
    c = paged.Case(ctx, window + sinks, "bf16", [350, 20, 1], [900, 333, 1], heads, kv_heads, d, 16)
    paged.check_attention(c, window=window, sinks=sinks, max_new=LONG)


def test_long_chunks_with_bad_pages(ctx):
    new = [300, 9, 2, 30]
    c = paged.Case(ctx, 5, "f16", new, [900, 90, 20, 120], 4, 2, 64, 16)
    c.table[0, 0] = -1
    c.table[0, 3] = c.num_pages
    c.table[0, 4] = np.iinfo(np.int32).min
    c.table[0, 42] = np.iinfo(np.int32).max
    c.table[1, :] = -7
    c.lengths[2] = 1
    c.table[3, 1:7] = 1 << 30
    paged.check_attention(c, max_new=LONG)
    paged.check_attention(c, window=20, sinks=3, max_new=LONG)


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("dtype,bad", [("f16", np.nan), ("bf16", np.inf)])
def test_long_chunks_leave_unseen_places(ctx, dtype, bad, window):
    c = paged.Case(ctx, 9, dtype, [270, 3], [350, 71], 4, 2, 128, 32)
    keep = np.zeros((c.num_pages, c.page), bool)
    for b in range(c.batch):
        p = np.arange(c.lengths[b])
        if window:
            p = p[p > c.lengths[b] - c.new[b] - window]
        keep[c.table[b, p // c.page], p % c.page] = True
    for bits in (c.k, c.v):
        x = paged.from16(bits, dtype).astype(np.float32)
        x[~keep[:, None, :, None] & np.ones(x.shape, bool)] = bad
        bits[:] = paged.to16(x, dtype)
    paged.check_attention(c, window=window, max_new=LONG)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_long_chunks_with_later_tokens_that_are_not_finite(ctx, dtype):
    c = paged.Case(ctx, 11, dtype, [280, 5], [300, 50], 4, 2, 64, 16)
    page, at = c.table[0, 200 // 16], 200 % 16
    for bits, bad in ((c.k, np.inf), (c.v, np.nan)):
        x = paged.from16(bits, dtype).astype(np.float32)
        x[page, :, at, :3] = bad
        bits[:] = paged.to16(x, dtype)
    q, got = paged.run_attention(c, max_new=LONG)
    ref, tol = paged.attention_oracle(c, paged.from16(q, dtype), 0, 0, 64 ** -0.5)
    out = paged.from16(got, dtype)
    for rows in (slice(0, 180), slice(280, 285)):
        assert (np.abs(out[rows] - ref[rows]) <= tol[rows]).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_long_chunks_with_large_scores(ctx, dtype):
    paged.check_attention(paged.Case(ctx, 13, dtype, [260], [600], 4, 2, 128, 16, scale=30.0), scale=1.0, max_new=LONG)
    paged.check_attention(paged.Case(ctx, 14, dtype, [40], [9000], 4, 2, 64, 16), max_new=LONG)


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 200, 9]])
def test_starts_and_lengths_that_are_not_theirs(ctx, new):
    # whatever the device holds there, only rows of out and pages of the cache are written
    c = paged.Case(ctx, 31, "f16", new, [300, 300, 300], 4, 2, 64, 16, rows_behind=3)
    kv = c.upload()
    nbytes = c.tokens * 4 * 64 * 2
    guarded = ctx.alloc(3 * nbytes)
    out = guarded.view(nbytes, nbytes)
    dq = ctx.upload(paged.to16(c.rng.normal(0, 1, (c.tokens, 4, 64)), "f16"))
    qkv = ctx.upload(paged.to16(c.rng.normal(0, 1, (c.tokens, 8, 64)), "f16"))
    gain = ctx.upload(np.ones(64, np.float32))
    work = ctx.alloc(ctx.attn_paged_workspace(kv, c.tokens, 4, max(new)))
    rng = np.random.default_rng(32)
    ends = np.array([0, 1, -1, c.tokens, c.tokens + 1, 7, np.iinfo(np.int32).max, np.iinfo(np.int32).min], np.int64)
    for _ in range(30):
        c.buffers[3].copy_from_host(rng.choice(np.append(ends, 300), 3).astype(np.int32))
        c.buffers[4].copy_from_host(rng.choice(ends, 4).astype(np.int32))
        ctx.memset(guarded, 0x5a)
        ctx.attn_paged(kv, dq, out, c.tokens, 4, max(new), 0.125, work, int(rng.choice([0, 50])), 4)
        ctx.sync()
        host = guarded.to_host()
        assert (host[:nbytes] == 0x5a).all() and (host[2 * nbytes:] == 0x5a).all()
        assert (c.buffers[0].to_host() == c.k).all() and (c.buffers[1].to_host() == c.v).all()
        ctx.qk_norm_rope_paged(kv, qkv, gain, gain, out, c.tokens, 4, EPS, THETA)
        ctx.sync()
        host = guarded.to_host()
        assert (host[:nbytes] == 0x5a).all() and (host[2 * nbytes:] == 0x5a).all()
        for b, bits in zip(c.buffers[:2], (c.k, c.v)):
            b.copy_from_host(bits)
    for b in (guarded, dq, qkv, gain, work):
        b.free()
    c.free()
