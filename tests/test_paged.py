"""CPU checks of the paged cache: the division of an attention call and the
argument checks (tests/cpp/paged_check.cpp), and the host's page bookkeeping
against a model that keeps every row's tokens apart."""
import subprocess
from pathlib import Path

import numpy as np
import pytest

from strict_amd.paged import OutOfPages, PageTable

ROOT = Path(__file__).resolve().parent.parent


def test_division_of_work_and_refusals(tmp_path):
    exe = tmp_path / "paged_check"
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-I", str(ROOT / "include"), "-I",
                    str(ROOT / "strict_amd" / "csrc"), str(ROOT / "tests" / "cpp" / "paged_check.cpp"),
                    "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "failures=0" in r.stdout


class _Pool:
    """Pages of token numbers, as the device would hold them."""

    def __init__(self, table):
        self.table, self.data = table, np.full((table.num_pages, table.page_size), -1)

    def copy(self, pairs):
        assert len({d for _, d in pairs}) == len(pairs)
        assert not {s for s, _ in pairs} & {d for _, d in pairs}
        before = self.data.copy()
        for s, d in pairs:
            self.data[d] = before[s]

    def append(self, row, tokens):
        t = self.table
        for i, token in enumerate(tokens):
            p = t.lengths[row] - len(tokens) + i
            self.data[t.pages[row][p // t.page_size], p % t.page_size] = token

    def read(self, row):
        t = self.table
        return [self.data[t.pages[row][p // t.page_size], p % t.page_size] for p in range(t.lengths[row])]


def _consistent(t):
    count = [0] * t.num_pages
    for row, pages in enumerate(t.pages):
        assert len(set(pages)) == len(pages) == -(-t.lengths[row] // t.page_size)
        for p in pages:
            count[p] += 1
    assert count == t.holders
    assert sorted(t._free) == [p for p in range(t.num_pages) if count[p] == 0]


@pytest.mark.parametrize("seed", range(12))
def test_rows_keep_their_tokens(seed):
    rng = np.random.default_rng(seed)
    rows, page = 6, int(rng.integers(1, 6))
    t = PageTable(rows, 9, int(rng.integers(12, 40)), page)
    pool, tokens, next_token = _Pool(t), [[] for _ in range(rows)], 0
    refused = 0
    for _ in range(300):
        what = rng.random()
        row, to = (int(r) for r in rng.integers(0, rows, 2))
        if what < 0.55:
            new = {int(r): int(rng.integers(0, 2 * page + 2)) for r in rng.permutation(rows)[:rng.integers(1, 4)]}
            state = ([list(p) for p in t.pages], list(t.lengths), list(t.holders), sorted(t._free))
            try:
                pool.copy(t.extend(new))
            except OutOfPages:
                refused += 1
                assert state == ([list(p) for p in t.pages], list(t.lengths), list(t.holders), sorted(t._free))
                continue
            for r, n in new.items():
                fresh = list(range(next_token, next_token + n))
                next_token += n
                pool.append(r, fresh)
                tokens[r] += fresh
        elif what < 0.75:
            if tokens[to]:
                with pytest.raises(ValueError):
                    t.fork(row, to)
            else:
                t.fork(row, to)
                tokens[to] = list(tokens[row])
        elif what < 0.9:
            t.free(row)
            tokens[row] = []
        else:
            pool.copy(t.compact())
            assert t._free == list(range(t.num_pages - t.free_pages, t.num_pages))
        _consistent(t)
        for r in range(rows):
            assert pool.read(r) == tokens[r]
    assert refused > 0 or t.num_pages > 20


def test_refusals():
    t = PageTable(2, 3, 4, 4)
    with pytest.raises(OutOfPages):
        t.extend({0: 13})  # four pages, a table of three
    with pytest.raises(OutOfPages):
        t.extend({0: 12, 1: 8})  # five pages of four
    with pytest.raises(ValueError):
        t.extend({0: -1})
    t.extend({0: 12})
    assert t.free_pages == 1 and t.array().tolist() == [[0, 1, 2], [-1, -1, -1]]
    t.fork(0, 1)
    assert t.free_pages == 1
    with pytest.raises(ValueError):
        PageTable(1, 0, 1, 1)


def test_shared_last_page_is_copied_once_per_row_but_the_last():
    t = PageTable(3, 4, 8, 4)
    t.extend({0: 6})
    t.fork(0, 1)
    t.fork(0, 2)
    copies = t.extend({0: 1, 1: 1, 2: 1})
    assert copies == [(1, 2), (1, 3)]  # the third keeps the page
    assert [p[0] for p in t.pages] == [0, 0, 0] and [p[1] for p in t.pages] == [2, 3, 1]


def test_full_last_page_stays_shared():
    t = PageTable(2, 4, 8, 4)
    t.extend({0: 8})
    t.fork(0, 1)
    assert t.extend({0: 1, 1: 1}) == []
    assert t.pages == [[0, 1, 2], [0, 1, 3]]


@pytest.mark.parametrize("row", [-1, 2])
def test_rows_that_are_not_there(row):
    t = PageTable(2, 4, 8, 4)
    t.extend({0: 5, 1: 5})
    before = t.array()
    for call in (lambda: t.extend({0: 1, row: 1}), lambda: t.free(row), lambda: t.fork(0, row), lambda: t.fork(row, 1)):
        with pytest.raises(IndexError):
            call()
    assert (t.array() == before).all() and t.lengths == [5, 5]
