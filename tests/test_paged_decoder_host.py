"""What PagedDecoder refuses and restores, without a GPU: its page table keeps the host's side only."""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest

from lucid_amd.nn.generation import PageTable
from lucid_amd.paged_decoder import PagedDecoder


def _decoder(seqs=3, pages=12, page=4, vocab=50, positions=32):
    table = PageTable.__new__(PageTable)
    table.seqs, table.pages, table.page = seqs, pages, page
    table._table = np.zeros((seqs, pages), np.int32)
    table._lengths = np.zeros((seqs,), np.int32)
    table._held, table._free = [0] * seqs, list(range(pages - 1, -1, -1))
    table._upload = lambda *a: None
    pd = PagedDecoder.__new__(PagedDecoder)
    pd.table, pd.vocab, pd.positions = table, vocab, positions
    pd.qdec = SimpleNamespace(head=lambda h: h)
    return pd


@pytest.mark.parametrize("key", [-1, -3, 3, 70])
def test_sequence_keys_outside_the_table_are_refused(key):
    """A negative key would sort first and take the last row: its tokens would land in another sequence."""
    pd = _decoder()
    with pytest.raises(ValueError, match="sequence"):
        pd.prefill({key: np.array([1, 2]), 0: np.array([3])})
    assert (pd.table.host_lengths() == 0).all()
    pd.table.grow([2, 2, 2])
    with pytest.raises(ValueError, match="sequence"):
        pd.step({key: 5, 0: 1})
    assert (pd.table.host_lengths() == 2).all()


def test_generate_gives_its_sequences_back_when_a_step_fails(monkeypatch):
    """Pages used up on the way: the next call finds the sequences free, and those of others untouched."""
    pd = _decoder()
    pd.table.grow([0, 0, 3])  # somebody else's
    monkeypatch.setattr(pd, "prefill", lambda prompts: pd.table.grow([len(prompts[0]), len(prompts[1]), 0]))
    monkeypatch.setattr(pd, "_choose", lambda logits, n, top: (np.zeros(n, np.int32),) * 3, raising=False)

    def step(tokens):
        raise MemoryError("no pages")

    monkeypatch.setattr(pd, "step", step)
    with pytest.raises(MemoryError):
        pd.generate([np.array([1, 2, 3]), np.array([4])], 3)
    assert pd.table.host_lengths().tolist() == [0, 0, 3]
    assert len(pd.table._free) == pd.table.pages - 1


def test_a_failed_prefill_leaves_the_table_as_it_was(monkeypatch):
    pd = _decoder()
    pd.table.grow([0, 5, 0])

    def hidden(*a):
        raise MemoryError("no memory")

    monkeypatch.setattr(pd, "_hidden", hidden)
    monkeypatch.setattr("lucid_amd.paged_decoder._ints", lambda a: a)
    with pytest.raises(MemoryError):
        pd.prefill({0: np.array([1, 2]), 2: np.array([3])})
    assert pd.table.host_lengths().tolist() == [0, 5, 0]
    assert len(pd.table._free) == pd.table.pages - 2


def test_a_failed_step_takes_its_positions_back(monkeypatch):
    pd = _decoder()
    pd.table.grow([4, 3, 2])

    def hidden(*a):
        raise MemoryError("no memory")

    monkeypatch.setattr(pd, "_hidden", hidden)
    monkeypatch.setattr("lucid_amd.paged_decoder._ints", lambda a: a)
    with pytest.raises(MemoryError):
        pd.step({0: 1, 1: 2, 2: 3})
    assert pd.table.host_lengths().tolist() == [4, 3, 2]
    pd.table.grow([1, 0, 0])  # the page it took serves the next try
    assert len(pd.table._free) == pd.table.pages - 4
    for counts in ([6, 0, 0], [-1, 0, 0], [1, 1]):
        with pytest.raises(ValueError):
            pd.table.shrink(counts)
    assert pd.table.host_lengths().tolist() == [5, 3, 2]


@pytest.mark.parametrize("token", [-1, 50, 1 << 31])
def test_step_refuses_tokens_outside_the_vocabulary(token):
    """The embedding would give a row of NaN, which every later step of that sequence would attend."""
    pd = _decoder()
    pd.table.grow([2, 2, 2])
    with pytest.raises(ValueError, match="vocabulary"):
        pd.step({1: token, 2: 3})
    with pytest.raises(ValueError, match="vocabulary"):
        pd.prefill({0: np.array([token])})
    with pytest.raises(ValueError, match="vocabulary"):
        pd.score([[token, 2]])
    assert (pd.table.host_lengths() == 2).all()


@pytest.mark.parametrize("s", [-1, 3])
def test_release_refuses_sequences_outside_the_table(s):
    """A negative number would end the last sequence."""
    pd = _decoder()
    pd.table.grow([2, 2, 2])
    with pytest.raises(ValueError, match="sequence"):
        pd.table.release(s)
    assert (pd.table.host_lengths() == 2).all() and len(pd.table._free) == pd.table.pages - 3
