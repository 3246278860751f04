"""Attention over 4-bit pages of whole tiles and of others: pages and rows that are not to be had, sizes far from one for
every type of output (the bound of test_gpu_paged4_range.py)."""

from __future__ import annotations

import numpy as np
import pytest

from _decode import dev, i32, rounded, types, values
from test_gpu_paged4 import TYPES, Cache4
from test_gpu_paged4_range import _check, _store

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [200, 2500])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("page,hd", [(16, 128), (64, 64), (64, 128), (128, 64), (128, 128), (192, 96), (64, 256)])
def test_bad_pages_and_rows_that_are_not_finite(gpu, n, dtype, page, hd):
    """A page outside the pool (the first, one between, the last) or a table that is too short: NaN for that sequence.  A
    group of NaN reaches its own key head.  Positions past the length never do, though they lie in a page that is used."""
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng([n, page, hd])
    cache = Cache4(rng, [n] * 8, 2, page, hd)
    used = -(-n // page)
    page_no, slot = cache.p.at(3, n // 2)
    cache.meta["k"][page_no, 1, slot, :, -1] = np.nan
    page_no, slot = cache.p.at(4, n - 1)
    cache.meta["v"][page_no, 0, slot] = np.nan
    cache.p.table[0, 0], cache.p.table[1, used // 2], cache.p.table[2, used - 1] = -1, cache.p.pages, 2 ** 31 - 1
    q, qh = rounded(rng.standard_normal((8, 4, hd)), dtype)
    t = cache.tensors()
    for out in (dtype, "float32"):
        got = values(F.paged_attention(dev(qh), max_length=n, out_dtype=types()[out], **t))
        assert np.isnan(got[:3]).all()
        assert np.isnan(got[3, 2:]).all() and np.isnan(got[4, :2]).all()
        assert np.isfinite(got[3, :2]).all() and np.isfinite(got[4, 2:]).all() and np.isfinite(got[5:]).all()
        _check(cache, q, got, 2, hd ** -0.5, out, 2.0 ** -22, 16, skip=5)
    t["lengths"] = i32([n] * 6 + [t["table"].shape[1] * page + 1, 0])
    got = values(F.paged_attention(dev(qh), max_length=n, **t))
    assert np.isnan(got[6]).all() and np.isfinite(got[5]).all() and (got[7] == 0).all()


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("size", [1e-20, 1e20])
@pytest.mark.parametrize("page", [16, 64])
def test_sizes_far_from_one(gpu, dtype, out, size, page):
    """Keys of any size, and values where the output's type has room for them."""
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(4)
    cache = Cache4(rng, [90, 1400], 1, page, 64, size=size)
    if out == "float16":
        for b, length in enumerate(cache.lens):
            _, vs, vb = cache.rows[b]["v"]
            vs *= 2.0 ** -np.round(np.log2(size))
            vb *= 2.0 ** -np.round(np.log2(size))
            _store(cache, b, np.arange(length))
    q, qh = rounded(rng.standard_normal((2, 2, 64)), dtype)
    scale = 0.125 / size
    got = values(F.paged_attention(dev(qh), max_length=1400, scale=scale, out_dtype=types()[out], **cache.tensors()))
    _check(cache, q, got, 2, scale, out, 2.0 ** -22, 16)


@pytest.mark.parametrize("page", [3, 100, 320, 5000])
@pytest.mark.parametrize("lens", [[90, 256, 640], [4000, 1, 999]])
@pytest.mark.parametrize("hd,dtype", [(64, "float16"), (128, "bfloat16"), (160, "float16")])
def test_pages_of_any_length(gpu, page, lens, hd, dtype):
    """Pages that end inside a tile, that hold several tiles, that hold whole sequences."""
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng([page, hd])
    cache = Cache4(rng, lens, 1, page, hd)
    q, qh = rounded(rng.standard_normal((3, 2, hd)), dtype)
    for out in (dtype, "float32"):
        got = values(F.paged_attention(dev(qh), max_length=max(lens), out_dtype=types()[out], **cache.tensors()))
        _check(cache, q, got, 2, hd ** -0.5, out, 2.0 ** -22, 16)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_queries_at_any_address(gpu, dtype):
    """Rows of queries that 16-byte reads do not fit."""
    import lucid_amd as L
    from lucid_amd import _C

    rng = np.random.default_rng(1)
    cache = Cache4(rng, [90, 1500], 2, 16, 64)
    ld = 4 * 64 + 3
    x, host = rounded(rng.standard_normal((2, ld)), dtype)
    t, rows, out = cache.tensors(), dev(host), L.empty((2, 4, 64), L.float32, "gpu")
    size = _C.lib().lq_paged_attention_workspace_size(2, 4, 2, 64, 1500)
    ws = L.empty((size,), np.uint8, "gpu")
    _C.call("lq_paged_attention", rows.data_ptr(), _C.F16 if dtype == "float16" else _C.BF16, ld, 2, 4, 2, 64,
            t["k_pages"].data_ptr(), t["v_pages"].data_ptr(), _C.U4, t["k_scale"].data_ptr(), t["v_scale"].data_ptr(),
            cache.p.pages, 16, t["table"].data_ptr(), t["table"].shape[1], t["lengths"].data_ptr(), 1500, 0.125,
            out.data_ptr(), _C.F32, ws.data_ptr(), size, None)
    _check(cache, x[:, :256].reshape(2, 4, 64), out.numpy(), 2, 0.125, "float32", 2.0 ** -22, 16)
