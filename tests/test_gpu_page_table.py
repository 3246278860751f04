"""The page table on the device after sequences gave positions back."""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_a_sequence_grows_beside_one_with_pages_to_spare(gpu):
    """Rejected drafts leave pages with their sequence; the pages that another one takes reach the device, and the step
    attends its own rows."""
    import lucid_amd as L
    from lucid_amd.nn.generation import PagedKVCache, PageTable

    rng = np.random.default_rng(0)
    table = PageTable(2, 8, 4)
    cache = PagedKVCache(table, 1, 64)
    rows = {}

    def append(s, n):
        counts = [0, 0]
        counts[s] = n
        table.grow(counts)
        kv = rng.standard_normal((2, n, 1, 64)).astype(np.float16)
        starts = L.tensor(np.cumsum([0] + counts).astype(np.int32), device="gpu")
        cache.append(L.tensor(kv[0], device="gpu"), L.tensor(kv[1], device="gpu"), starts)
        rows[s] = kv if s not in rows else np.concatenate([rows[s][:, :table.host_lengths()[s] - n], kv], 1)

    append(0, 9)
    table.shrink([7, 0])
    append(1, 7)
    append(0, 3)
    assert np.array_equal(table.table.numpy()[1, :2], table._table[1, :2])
    q = L.tensor(rng.standard_normal((2, 1, 64)).astype(np.float16), device="gpu")
    got = cache.attend(q, out_dtype=L.float32).numpy()
    for s in range(2):
        k, v = (a[:, 0].astype(np.float64) for a in rows[s])
        w = np.exp(k @ q.numpy()[s, 0].astype(np.float64) / 8)
        # float32 sums of 16-bit rows: weights of 22 bits, some hundred operations of 2^-24
        assert np.allclose(got[s, 0], w @ v / w.sum(), rtol=0, atol=1e-5), s
