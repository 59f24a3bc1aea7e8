"""The page pool called from several threads, and at sizes at which a list that is
searched would show."""
import time

import pytest

from huggingfaceeacp_amd import gemma_q8 as G


def forked(pool, count):
    """`count` forks of one sequence that each write: their copies are recorded."""
    first = pool.open()
    pool.extend(first, 1)
    forks = [pool.fork(first) for _ in range(count)]
    for s in forks:
        pool.extend(s, 1)
    return forks


class Between:
    """The library, with something done to the pool after the copies are counted."""

    def __init__(self, inner, what):
        self.inner, self.what = inner, what

    def __getattr__(self, name):
        if name == "gq8_page_pool_copy_count":
            def count(handle):
                n = self.inner.gq8_page_pool_copy_count(handle)
                if self.what:
                    what, self.what = self.what, None
                    what()
                return n
            return count
        return getattr(self.inner, name)


def test_copies_dropped_by_another_thread_are_not_returned(monkeypatch):
    pool = G.PagePool(8, 4, 6, 2)
    forks = forked(pool, 3)
    library = Between(G.library(), lambda: pool.close(forks[1]))
    monkeypatch.setattr(G, "library", lambda: library)
    pairs = pool.take_copies()
    assert pairs.tolist() == [[0, 1], [0, 3]]
    assert pool.take_copies().shape == (0, 2)


def test_copies_added_by_another_thread_are_returned(monkeypatch):
    pool = G.PagePool(8, 4, 6, 2)
    forks = forked(pool, 2)

    def more():
        pool.extend(pool.fork(forks[0]), 1)

    library = Between(G.library(), more)
    monkeypatch.setattr(G, "library", lambda: library)
    assert pool.take_copies().tolist() == [[0, 1], [0, 2], [0, 3]]


def test_a_large_compaction_and_the_end_of_what_it_moved():
    """200,000 recorded copies: each is found without a search through the others
    (with one, both calls take many seconds)."""
    n = 200_000
    pool = G.PagePool(2 * n, 1, 2, n)
    a, b = pool.open(), pool.open()
    pool.extend(a, n)
    pool.extend(b, n)
    pool.close(a)
    before = time.process_time()
    assert pool.compact() == n
    table, rows = pool.tables([b])
    assert rows[0] == n and sorted(table[0]) == list(range(n))
    pool.truncate(b, n // 2)
    pairs = pool.take_copies()
    assert len(pairs) == n // 2
    assert set(pairs[:, 1].tolist()) == set(table[0, :n // 2].tolist())
    pool.extend(b, n // 2)
    pool.close(b)
    assert pool.free_pages == 2 * n
    assert time.process_time() - before < 2.0


@pytest.mark.parametrize("pages", [1, 63, 64, 65, 4096, 4097, 300_000])
def test_the_lowest_free_page_is_given_out(pages):
    pool = G.PagePool(pages, 1, 3, pages)
    a = pool.open()
    pool.extend(a, pages)
    assert pool.tables([a])[0][0].tolist() == list(range(pages)) and pool.free_pages == 0
    b = pool.open()
    with pytest.raises(G.Gq8Error) as info:
        pool.extend(b, 1)
    assert info.value.status == G.ERR_CAPACITY
    kept = pages // 2
    pool.truncate(a, kept)
    assert pool.free_pages == pages - kept
    pool.extend(b, 1)
    assert pool.tables([b])[0][0, 0] == kept
    pool.close(a)
    pool.extend(b, min(2, pages - 1))
    wanted = [kept] + [p for p in range(pages) if p != kept][:min(2, pages - 1)]
    assert pool.tables([b])[0][0, :len(wanted)].tolist() == wanted
    pool.close(b)
    assert pool.free_pages == pages


def test_a_page_that_a_copy_reads_moves_in_a_compaction():
    """Both copies read its old number, which is given out once they are taken."""
    pool = G.PagePool(6, 4, 6, 2)
    first = [pool.open(), pool.open()]
    for s in first:
        pool.extend(s, 4)
    b = pool.open()
    pool.extend(b, 2)
    c = pool.fork(b)
    pool.extend(c, 1)  # its copy reads b's page
    assert pool.tables([b, c])[0][:, 0].tolist() == [2, 3]
    for s in first:
        pool.close(s)
    assert pool.compact() == 2
    assert pool.tables([b, c])[0][:, 0].tolist() == [1, 0]
    assert pool.free_pages == 3  # not page 2
    assert sorted(pool.take_copies().tolist()) == [[2, 0], [2, 1]]
    assert pool.free_pages == 4


def test_tables_are_of_a_size_that_the_operators_take():
    """A sequence's rows are at most 2^30 for every operator."""
    assert G.PagePool(4, 1 << 20, 1, 1 << 10).table_width == 1 << 10
    for width in ((1 << 10) + 1, 1 << 11):
        with pytest.raises(G.Gq8Error) as info:
            G.PagePool(4, 1 << 20, 1, width)
        assert info.value.status == G.ERR_SHAPE
