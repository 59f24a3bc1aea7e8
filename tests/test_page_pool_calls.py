"""The page pool called from several threads, and at sizes at which a list that is
searched would show."""
import numpy as np
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
