"""Calls of the paged operators and of sampling that are refused before anything is
launched: sizes whose products leave 64 bits, tensors over one another."""
import numpy as np
import pytest

import strict_amd
import test_gpu_paged as paged
from strict_amd import PagedKV

pytestmark = pytest.mark.gpu


def refused(call, text):
    with pytest.raises(strict_amd.StrictHipError) as e:
        call()
    assert e.value.status == strict_amd.SH_ERR_INVALID_ARGUMENT and text in e.value.message, e.value.message


@pytest.mark.parametrize("num_pages", [1 << 30, (1 << 30) + 1, (1 << 28) + 1])
def test_pools_past_64_bits(ctx, num_pages):
    # (their sizes come round to nothing, to one page of 16 GiB and to little more than 2^62)
    c = paged.Case(ctx, 1, "f16", [1], [20], 1, 1, 128, 16)
    c.upload()
    kv = PagedKV(*c.buffers, batch=1, max_pages=1, num_pages=num_pages, page_size=65536, kv_heads=1024, head_dim=128)
    rows = ctx.upload(np.zeros((3 * 1024, 128), np.int16))
    q, out = (ctx.upload(np.zeros((1024, 128), np.int16)) for _ in range(2))
    gain = ctx.upload(np.ones(128, np.float32))
    work = ctx.alloc(1 << 20)
    refused(lambda: ctx.attn_paged_workspace(kv, 1, 1024, 1), "num_pages")
    refused(lambda: ctx.attn_paged(kv, q, out, 1, 1024, 1, 1.0, work), "num_pages")
    refused(lambda: ctx.qk_norm_rope_paged(kv, rows, gain, gain, q, 1, 1024, 1e-6, 1e4), "num_pages")
    for b in (rows, q, out, gain, work):
        b.free()
    c.free()


def test_attention_over_its_own_index(ctx):
    # out or the work buffer over the page table, the lengths or the starts: at their first and last bytes
    c = paged.Case(ctx, 2, "f16", [1], [20], 4, 2, 64, 16)
    c.upload()
    need = ctx.attn_paged_workspace(c.kv, c.tokens, 4, 1)
    nbytes = c.tokens * 4 * 64 * 2
    q, out = ctx.alloc(nbytes), ctx.alloc(nbytes)
    for which, text, size in (("out", "page table, lengths or starts", nbytes), ("work", "work buffer overlaps", need)):
        area = ctx.alloc(size + 64)
        for i in (2, 3, 4):
            index = c.buffers[i]
            for at in (0, 16 + size - 4):  # the index before the written range's start, and at its end
                buffers = list(c.buffers)
                buffers[i] = area.view(at, index.nbytes) if at else area.view(16 - index.nbytes + 4, index.nbytes)
                kv = PagedKV(*buffers, batch=1, max_pages=c.max_pages, num_pages=c.num_pages, page_size=16, kv_heads=2,
                             head_dim=64)
                over = area.view(16, size)
                args = (kv, q, over if which == "out" else out, c.tokens, 4, 1, 1.0)
                work = ctx.alloc(need) if which == "out" else over
                refused(lambda: ctx.attn_paged(*args, work), text)
                if which == "out":
                    work.free()
        area.free()
    q.free()
    out.free()
    c.free()


def test_head_norms_over_their_own_index(ctx):
    # q or a pool over the page table, the lengths, the starts or a gain
    c = paged.Case(ctx, 3, "f16", [1], [20], 4, 2, 64, 16)
    c.upload()
    nbytes, pool = c.tokens * 4 * 64 * 2, c.buffers[0].nbytes
    q, qkv, gain = ctx.alloc(nbytes), ctx.alloc(c.tokens * 8 * 64 * 2), ctx.upload(np.ones(64, np.float32))
    for which, size in (("q", nbytes), ("k", pool), ("v", pool)):
        area = ctx.alloc(size + 512)
        over = area.view(256, size)
        for i in (2, 3, 4, "q_gain", "k_gain"):
            index_bytes = c.buffers[i].nbytes if isinstance(i, int) else 256
            for at in (256 - index_bytes + 4, 256 + size - 4):
                index = area.view(at, index_bytes)
                buffers = [b if j != i else index for j, b in enumerate(c.buffers)]
                if which in "kv":
                    buffers["kv".index(which)] = over
                gains = [index if i == name else gain for name in ("q_gain", "k_gain")]
                kv = PagedKV(*buffers, batch=1, max_pages=c.max_pages, num_pages=c.num_pages, page_size=16, kv_heads=2,
                             head_dim=64)
                refused(lambda: ctx.qk_norm_rope_paged(kv, qkv, *gains, over if which == "q" else q, c.tokens, 4, 1e-6, 1e4),
                        "overlaps the page table, lengths, starts or gains")
        area.free()
    for b in (q, qkv, gain):
        b.free()
    c.free()


def test_page_numbers_in_the_pool(ctx):
    planes, num, page_bytes, count = 2, 5, 32, 3
    extent = planes * num * page_bytes
    area = ctx.alloc(extent + 256)
    other = ctx.upload(np.zeros(count, np.int32))
    pool = area.view(128, extent)
    for at in (128 - 4 * count + 4, 128 + extent - 4):
        inside = area.view(at, 4 * count)
        for src, dst in ((inside, other), (other, inside)):
            refused(lambda: ctx.pages_copy(pool, planes, num, page_bytes, src, dst, count), "in the pools")
    ctx.memset(area, 0xff)  # (page numbers that are none)
    for at in (128 - 4 * count, 128 + extent):
        ctx.pages_copy(pool, planes, num, page_bytes, area.view(at, 4 * count), area.view(at, 4 * count), count)
    ctx.sync()
    area.free()
    other.free()


def test_sampling_over_its_own_parameters(ctx):
    # the work buffer over index, u or a parameter, index over these or over x
    rows, n = 3, 3000
    need = ctx.sample_workspace(rows, n)
    names = ["x", "temperature", "top_k", "top_p", "min_p", "u", "index"]
    own = {name: ctx.upload(np.zeros(rows, np.float32)) for name in names[1:]}
    own["x"] = ctx.upload(np.zeros((rows, n), np.float32))
    work, area = ctx.alloc(need), ctx.alloc(need + 256)

    def call(n=n, work=work, **other):
        b = {**own, **other}
        ctx.sample(b["x"], rows, n, b["temperature"], b["top_k"], b["top_p"], b["min_p"], b["u"], b["index"], work)

    for name in names[1:]:
        for at in (128 - 4 * rows + 4, 128 + need - 4):
            refused(lambda: call(work=area.view(128, need), **{name: area.view(at, 4 * rows)}), "work buffer overlaps index")
    # index over another, of rows short and long
    for short in (n, 100):
        for name in names[1:6]:
            for at in (-4 * rows + 4, 4 * rows - 4):
                refused(lambda: call(short, index=area.view(128 + at, 4 * rows), **{name: area.view(128, 4 * rows)}),
                        "index overlaps x")
        for at in (-4 * rows + 4, 4 * rows * short - 4):
            refused(lambda: call(short, index=area.view(128 + at, 4 * rows), x=area.view(128, 4 * rows * short)),
                    "index overlaps x")
    # what is only read may be shared
    call(temperature=own["u"], top_p=own["u"], min_p=own["u"])
    ctx.sync()
    for b in [work, area, *own.values()]:
        b.free()


def test_logits_past_their_allocation(ctx):
    x, u, index = ctx.upload(np.zeros((2, 3000), np.float32)), ctx.upload(np.zeros(2, np.float32)), ctx.empty(2, np.int32)
    work = ctx.alloc(ctx.sample_workspace(2, 3000))
    refused(lambda: ctx.sample(x, 2, 3000, None, None, None, None, u, index, work, 3001), "x (")
    refused(lambda: ctx.sample(x, 2, 3000, None, None, None, None, u, index, work, 3001), "is not inside an allocation")
    for b in (x, u, index, work):
        b.free()


@pytest.mark.parametrize("planes", [1, 3])
def test_more_pages_than_a_launch_has_workgroups(ctx, planes):
    # 2^24 and more pairs, small pages: all but a few skipped
    num, page_bytes = (1 << 24) + 100, 16
    count = num - 5
    src = np.full(count, -1, np.int32)
    dst = np.full(count, num, np.int32)
    some = np.array([0, 1, 70000, (1 << 24) - 2, (1 << 24) - 1, 1 << 24, count - 1])
    src[some], dst[some] = np.arange(len(some)), num - 1 - np.arange(len(some))
    pool, s, d = ctx.alloc(planes * num * page_bytes), ctx.upload(src), ctx.upload(dst)
    ctx.memset(pool, 0)
    first = np.arange(planes * len(some) * 2, dtype=np.int64).reshape(planes, -1) + 1
    last = [pool.view((p * num + num - len(some)) * page_bytes, len(some) * page_bytes, np.int64) for p in range(planes)]
    for p in range(planes):
        pool.view(p * num * page_bytes, len(some) * page_bytes).copy_from_host(first[p])
    ctx.pages_copy(pool, planes, num, page_bytes, s, d, count)
    ctx.sync()
    for p in range(planes):
        assert (last[p].to_host().reshape(-1, 2)[::-1] == first[p].reshape(-1, 2)).all()
    for b in (pool, s, d):
        b.free()
