"""Values at the ends of bfloat16's range: a weighted mean lies within its values, however large their sum is.

With equal scores all weights are equal and their size cancels; the sum of n equal products is off by n u
at most (u = 2^-24) and the quotient by a few u more, so the mean is the value itself within (n + 8) u and
the output's rounding."""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LARGEST = 3.3895313892515355e38  # bfloat16's


def _dev(a):
    import lucid_amd as L

    return L.tensor(np.ascontiguousarray(a), device="gpu")


def _bf16(a):
    import lucid_amd as L

    return L.bf16_from_f32(np.asarray(a, np.float32))


def _values(t):
    import lucid_amd as L

    a = t.numpy()
    return (L.bf16_to_f32(a) if t.dtype == L.bfloat16 else a).astype(np.float64)


def _check(got, want, n, eps):
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= ((n + 8) * U + eps) * np.abs(want)).all()


@pytest.mark.parametrize("size", [LARGEST, 1.0, 1e-25])
@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("hd", [64, 128, 72])
def test_prompts(gpu, size, out, hd):
    import lucid_amd as L
    import lucid_amd.nn.functional as F
    from lucid_amd import _C

    eps = U if out == "float32" else 2.0 ** -8
    dt = getattr(L, out)
    sign = np.where(np.arange(hd) % 3 == 0, -1.0, 1.0)
    value = L.bf16_to_f32(_bf16(size)).astype(np.float64)
    for lens, h, path in (([300, 2], 2, "prompt tile 64"), ([300] + [3] * 60, 32, "prompt tile 128")):
        n = sum(lens)
        q, k = _bf16(np.ones((n, h, hd))), _bf16(np.ones((n, 1, hd)))
        v = _bf16(np.broadcast_to(sign * size, (n, 1, hd)))
        st = _dev(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
        got = _values(F.prompt_attention(_dev(q), _dev(k), _dev(v), st, out_dtype=dt))
        assert _C.last_path() == path
        _check(got, sign * value, 300, eps)


@pytest.mark.parametrize("size", [LARGEST, 1.0, 1e-25])
@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("hd", [64, 128, 72])
@pytest.mark.parametrize("n,bound", [(3, 3), (700, 700), (3000, 3000)])
def test_pages(gpu, size, out, hd, n, bound):
    import lucid_amd as L
    import lucid_amd.nn.functional as F

    eps = U if out == "float32" else 2.0 ** -8
    pages = -(-n // 16)
    sign = np.where(np.arange(hd) % 3 == 0, -1.0, 1.0)
    q, k = _bf16(np.ones((1, 4, hd))), _bf16(np.ones((pages, 2, 16, hd)))
    v = _bf16(np.broadcast_to(sign * size, (pages, 2, 16, hd)))
    value = L.bf16_to_f32(_bf16(size)).astype(np.float64)
    table, lens = _dev(np.arange(pages, dtype=np.int32)[None]), _dev(np.array([n], np.int32))
    got = _values(F.paged_attention(_dev(q), _dev(k), _dev(v), table, lens, bound, out_dtype=getattr(L, out)))
    _check(got, sign * value, n, eps)
    # int8 rows: the scale carries the size
    codes = np.broadcast_to((127 * sign).astype(np.int8), (pages, 2, 16, hd))
    sv = np.full((pages, 2, 16), size / 127, np.float32)
    sk = np.full((pages, 2, 16), 1 / 127, np.float32)
    got = _values(F.paged_attention(_dev(q), _dev(np.full((pages, 2, 16, hd), 127, np.int8)), _dev(codes), table, lens,
                                    bound, k_scale=_dev(sk), v_scale=_dev(sv), out_dtype=getattr(L, out)))
    _check(got, sign * 127 * sv[0, 0, 0].astype(np.float64), n, eps)


def test_rows_no_vector_fits(gpu):
    import lucid_amd as L
    from lucid_amd import _C

    n, hd = 70, 40
    ld = hd + 3
    one = np.zeros((n, ld))
    one[:, :hd] = 1
    q, v = _dev(_bf16(one)), _dev(_bf16(one * LARGEST))
    out, st = _dev(np.zeros((n, 1, hd), np.float32)), _dev(np.array([0, 30, n], np.int32))
    _C.call("lq_prompt_attention", q.data_ptr(), ld, q.data_ptr(), ld, v.data_ptr(), ld, _C.BF16, st.data_ptr(),
            st.data_ptr(), 2, n, n, 1, 1, hd, 1, hd ** -0.5, out.data_ptr(), _C.F32, None)
    assert _C.last_path() == "prompt rows"
    value = L.bf16_to_f32(_bf16(LARGEST)).astype(np.float64)
    _check(out.numpy().astype(np.float64), np.full((n, 1, hd), value), n, U)


@pytest.mark.parametrize("hd", [64, 128, 72])
@pytest.mark.parametrize("n", [70, 1500])
def test_infinite_values_in_pages(gpu, hd, n):
    """An infinity among bfloat16 values gives an infinity in its dim (NaN where both signs meet), and nothing
    elsewhere, whether a weight enters as two terms or three."""
    import lucid_amd as L
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(n + hd)
    pages = -(-n // 16)
    k, v = (rng.standard_normal((pages, 1, 16, hd)) for _ in range(2))
    v[1, 0, 3, 5], v[2, 0, 1, 6], v[3, 0, 0, 6], v[0, 0, 2, 9] = np.inf, np.inf, -np.inf, -np.inf
    q = _dev(_bf16(rng.standard_normal((1, 3, hd))))
    table, lens = _dev(np.arange(pages, dtype=np.int32)[None]), _dev(np.array([n], np.int32))
    for dt in (L.float32, L.bfloat16):
        got = _values(F.paged_attention(q, _dev(_bf16(k)), _dev(_bf16(v)), table, lens, n, out_dtype=dt))[0]
        assert (got[:, 5] == np.inf).all() and np.isnan(got[:, 6]).all() and (got[:, 9] == -np.inf).all()
        assert np.isfinite(np.delete(got, [5, 6, 9], 1)).all()


@pytest.mark.parametrize("hd", [64, 128, 72])
@pytest.mark.parametrize("h", [2, 32])
def test_infinite_values_in_prompts(gpu, hd, h):
    """Queries before an infinity are finite, those from it on have it in its dim alone."""
    import lucid_amd as L
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(hd)
    lens = [200] + [3] * 60
    n = sum(lens)
    q, k, v = (rng.standard_normal((n, m, hd)) for m in (h, 1, 1))
    v[90, 0, 7] = -np.inf
    st = _dev(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
    for dt in (L.float32, L.bfloat16):
        got = _values(F.prompt_attention(_dev(_bf16(q)), _dev(_bf16(k)), _dev(_bf16(v)), st, out_dtype=dt))
        assert (got[90:200, :, 7] == -np.inf).all()
        got[90:200, :, 7] = 0
        assert np.isfinite(got).all()
