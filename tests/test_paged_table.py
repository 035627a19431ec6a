"""The page table's promise that nothing changes when a method raises, and the cache's
that it keeps nothing on the device when it cannot be made (CPU)."""
import numpy as np
import pytest

from strict_amd.paged import PageTable


def state(t):
    return [list(p) for p in t.pages], list(t.lengths), list(t.holders), sorted(t._free)


@pytest.mark.parametrize("n", [1.0, 2.5, float("nan"), "3", None, np.float64(4)])
def test_numbers_of_tokens_that_are_none(n):
    # (also of a row whose shared last page the call would have parted from the other's)
    t = PageTable(3, 8, 20, 4)
    t.extend({0: 6})
    t.fork(0, 1)
    before = state(t)
    for new in ({0: n}, {0: 1, 1: n}, {2: n}):
        with pytest.raises(TypeError):
            t.extend(new)
        assert state(t) == before


def test_numbers_of_other_whole_types():
    t = PageTable(2, 8, 20, 4)
    t.extend({np.int64(0): np.int32(5), 1: np.uint8(3)})
    assert t.lengths == [5, 3] and all(type(n) is int for n in t.lengths)


class Buffer:
    def __init__(self, ctx, nbytes):
        self.ctx, self.nbytes, self.ptr = ctx, nbytes, 1 << 20
        ctx.held.append(self)

    def view(self, offset, nbytes):
        return self

    def copy_from_host(self, a):
        self.ctx.sent.append(np.array(a))

    def free(self):
        self.ctx.held.remove(self)


class Host:
    """What PagedCache asks of a context, without a device."""

    def __init__(self, allocations=99):
        self.held, self.sent, self.left = [], [], allocations

    def alloc(self, nbytes):
        if self.left == 0:
            raise MemoryError
        self.left -= 1
        return Buffer(self, nbytes)

    def empty(self, shape, dtype):
        return self.alloc(int(np.prod(shape)) * 4)

    def pages_copy(self, *args):
        pass


@pytest.fixture
def cache(monkeypatch):
    """PagedCache on a Host."""
    import strict_amd.paged as module
    monkeypatch.setattr(module, "PagedKV", lambda *a, **k: (a, k))
    return module.PagedCache


def test_steps_count_in_any_whole_type(cache):
    ctx = Host()
    c = cache(ctx, 1, 1, 64, rows=2, max_pages=64, num_pages=200, page_size=16)
    ctx.sent.clear()
    assert c.step({0: np.uint8(200), 1: np.uint8(100)}) == 300
    assert ctx.sent[-1].tolist() == [0, 200, 300] and ctx.sent[-2].tolist() == [200, 100]


@pytest.mark.parametrize("allocations", range(5))
def test_a_cache_that_finds_no_memory_keeps_none(cache, allocations):
    ctx = Host(allocations)
    with pytest.raises(MemoryError):
        cache(ctx, 2, 1, 64, rows=2, max_pages=4, num_pages=8, page_size=16)
    assert ctx.held == []


def test_a_cache_of_no_type_keeps_no_memory():
    from strict_amd.paged import PagedCache
    ctx = Host()
    with pytest.raises(ValueError):
        PagedCache(ctx, 2, 1, 64, rows=2, max_pages=4, num_pages=8, page_size=16, dtype="f32")
    assert ctx.held == []


def test_a_cache_gives_back_what_it_took(cache):
    ctx = Host()
    with cache(ctx, 2, 1, 64, rows=2, max_pages=4, num_pages=8, page_size=16):
        assert len(ctx.held) == 5
    assert ctx.held == []
