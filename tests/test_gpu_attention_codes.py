"""Pages of codes whose scale is not finite: the row reads as NaN, and nothing outside the pages is read."""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _dev(a):
    import lucid_amd as L

    return L.tensor(np.ascontiguousarray(a), device="gpu")


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("n", [70, 1500])
def test_int8_row_with_an_infinity(gpu, dtype, n):
    """One value row of sequence 0 holds an infinity: that sequence is NaN, the other one finite."""
    import lucid_amd as L
    import lucid_amd.nn.functional as F
    from lucid_amd.nn.generation import PagedKVCache, PageTable

    rng = np.random.default_rng(n)
    pages = -(-n // 16)
    pt = PageTable(2, 2 * pages, 16)
    cache = PagedKVCache(pt, 1, 64, np.int8)
    pt.grow([n, n])
    k, v = (rng.standard_normal((2 * n, 1, 64)).astype(np.float32) for _ in range(2))
    v[n // 2, 0, 5] = np.inf
    cache.append(_dev(k), _dev(v), _dev(np.array([0, n, 2 * n], np.int32)))
    q = rng.standard_normal((2, 3, 64)).astype(np.float32)
    q = _dev(L.bf16_from_f32(q) if dtype == "bfloat16" else q.astype(np.float16))
    for out in (L.float32, q.dtype):
        got = cache.attend(q, out_dtype=out).numpy()
        got = L.bf16_to_f32(got) if out == L.bfloat16 else got
        assert np.isnan(got[0]).all() and np.isfinite(got[1]).all()
