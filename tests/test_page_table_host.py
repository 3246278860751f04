"""PageTable's bookkeeping without a GPU: sequences that gave positions back hold pages to spare, which serve
nobody else."""

from __future__ import annotations

import numpy as np
import pytest

from lucid_amd.nn.generation import PageTable


def _table(seqs=3, pages=8, page=4):
    """A table whose uploads are kept instead: ``sent`` is what the device would hold."""
    t = PageTable.__new__(PageTable)
    t.seqs, t.pages, t.page = seqs, pages, page
    t._table, t._lengths = np.zeros((seqs, pages), np.int32), np.zeros((seqs,), np.int32)
    t._held, t._free = [0] * seqs, list(range(pages - 1, -1, -1))
    t.sent = {"table": t._table.copy(), "lengths": t._lengths.copy()}

    def upload(table, stream):
        if table:
            t.sent["table"] = t._table.copy()
        t.sent["lengths"] = t._lengths.copy()

    t._upload = upload
    return t


def _check(t):
    """The device's rows are the host's, and every page has one owner."""
    owned = [int(p) for s in range(t.seqs) for p in t._table[s, :t._held[s]]]
    assert sorted(owned + t._free) == list(range(t.pages))
    for s in range(t.seqs):
        assert t._held[s] * t.page >= t._lengths[s]
        assert (t.sent["table"][s, :t._held[s]] == t._table[s, :t._held[s]]).all()
    assert (t.sent["lengths"] == t._lengths).all()


def test_pages_taken_beside_spare_ones_reach_the_device():
    t = _table()
    t.grow([9, 0, 0])
    t.shrink([8, 0, 0])  # one position, three pages
    t.grow([0, 5, 0])    # two pages: as many as the first sequence has to spare
    _check(t)
    t.grow([0, 0, 1])    # one: fewer than that
    _check(t)


def test_spare_pages_do_not_count_as_free():
    """Refused before anything changes, where the free pages alone do not suffice."""
    t = _table()
    t.grow([20, 0, 0])
    t.shrink([19, 0, 0])  # five pages with one sequence, three free
    held, free, lengths = list(t._held), list(t._free), t._lengths.copy()
    with pytest.raises(MemoryError, match="4 pages needed, 3 free"):
        t.grow([0, 13, 0])
    with pytest.raises(MemoryError, match="4 pages needed, 3 free"):
        t.grow([0, 8, 5])
    assert t._held == held and t._free == free and (t._lengths == lengths).all()
    t.grow([19, 12, 0])  # its own pages serve the sequence again
    assert not t._free
    _check(t)


def test_any_order_of_calls():
    rng = np.random.default_rng(0)
    t = _table(seqs=4, pages=20)
    for _ in range(3000):
        call = rng.integers(0, 3)
        if call == 0:
            counts = rng.integers(0, 9, 4) * (rng.random(4) < 0.5)
            needed = sum(max(0, -(-int(n) // 4) - h) for n, h in zip(t._lengths + counts, t._held))
            if needed > len(t._free):
                with pytest.raises(MemoryError):
                    t.grow(counts)
            else:
                t.grow(counts)
        elif call == 1:
            t.shrink(rng.integers(0, t._lengths + 1))
        else:
            t.release(int(rng.integers(0, 4)))
        _check(t)
