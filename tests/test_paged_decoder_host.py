"""What PagedDecoder refuses and restores, without a GPU: its page table keeps the host's side only."""

from __future__ import annotations

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
