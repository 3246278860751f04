"""Root-mean-square norm on the GPU.  The sum is bit-exact (one rounding of x + res).  With u = 2^-24: a thread
adds at most 64 squares in four runs and the tree adds 12 roundings, so the sum of squares is within 28 u (wide rows:
D / 1024 + 16); mean, eps, root and quotient 4 u more, the root halving what came before; two products: 40 u (+ D /
2048) relative in all, then the output's rounding.  A code is off by half a step and 127 (4 u) more."""

from __future__ import annotations

import numpy as np
import pytest

from _decode import HALF, U, close, dev, rounded, types, values

pytestmark = pytest.mark.gpu


def _inputs(rng, rows, dim, dtype, residual, weight):
    strong = np.where(rng.random(dim) < 0.1, 30.0, 1.0)
    x = rounded(rng.standard_normal((rows, dim)) * strong * rng.choice([1e-3, 1, 50], (rows, 1)), dtype)
    res = rounded(rng.standard_normal((rows, dim)), dtype) if residual else (None, None)
    g = rounded(1 + 0.3 * rng.standard_normal(dim), weight) if weight else (None, None)
    return x, res, g


def _norm(h, g, eps):
    h = h.astype(np.float64)
    y = h / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    return y * g.astype(np.float64) if g is not None else y


def _tensors(*hosts):
    return [dev(h) if h is not None else None for h in hosts]


SHAPES = [(1, 1), (3, 7), (5, 8), (2, 367), (9, 512), (4, 513), (3, 1000), (6, 1024), (2, 2048), (3, 2056), (2, 4096),
          (5, 5120), (2, 8192), (1, 8200), (2, 16384), (1, 16383), (2, 16385), (1, 40000)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,dim", SHAPES)
@pytest.mark.parametrize("residual,weight", [(True, "same"), (False, None), (True, "float32")])
def test_norm_and_codes(gpu, dtype, rows, dim, residual, weight):
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng([rows, dim, residual])
    (x, xh), (res, rh), (g, gh) = _inputs(rng, rows, dim, dtype, residual, dtype if weight == "same" else weight)
    h = rounded(x + res, dtype)[0] if residual else x
    want = _norm(h, g, 1e-5)
    rel = (40 + dim / 2048) * U
    xt, rt, gt = _tensors(xh, rh, gh)
    for out in (dtype, "float32"):
        got = F.rms_norm(xt, gt, residual=rt, out_dtype=types()[out])
        if residual:
            got, total = got
            assert np.array_equal(values(total), h)
        tiny = {"float16": 2.0 ** -25}.get(out, 1e-38)
        close(values(got).astype(np.float64), want, (rel + HALF[out] * (out != "float32")) * np.abs(want) + tiny, out)
    codes, scales, *total = F.rms_norm_quantize(xt, gt, residual=rt)
    if residual:
        assert np.array_equal(values(total[0]), h)
    codes, scales = codes.numpy().astype(np.float64), scales.numpy().astype(np.float64)[:, None]
    top = np.abs(want).max(1, keepdims=True)
    close(scales, top / 127, (rel + 2 * U) * top / 127, "scales")
    assert np.abs(codes).max() <= 127 and (np.abs(codes).max(1) == 127).all()
    close(codes * scales, want, scales * (0.5 + 127 * 4 * U) + (rel + 2 * U) * np.abs(want), "codes")


@pytest.mark.parametrize("dim", [512, 2000, 2001, 20000])
def test_sum_in_place_strides_and_no_sum(gpu, dim):
    """Rows inside wider ones, the sum in the residual's or x's own place or not at all: the bits of the plain call."""
    import lucid_amd.nn.functional as F
    from lucid_amd import _C

    rng = np.random.default_rng(dim)
    rows, ld = 5, dim + 24
    x, res = (rng.standard_normal((rows, ld)).astype(np.float32) for _ in range(2))
    g = dev(rng.standard_normal(dim).astype(np.float32))
    want, total = (t.numpy() for t in F.rms_norm(dev(x[:, :dim]), g, residual=dev(res[:, :dim])))
    wc, ws, _ = (t.numpy() for t in F.rms_norm_quantize(dev(x[:, :dim]), g, residual=dev(res[:, :dim])))
    for place in ("x", "res", None):
        for quantize in (False, True):
            xt, rt = dev(x), dev(res)
            st = {"x": xt, "res": rt, None: None}[place]
            sp = st.data_ptr() if st is not None else None
            y = dev(np.full((rows, ld), 9, np.int8 if quantize else np.float32))
            scales = dev(np.zeros(rows, np.float32))
            common = (xt.data_ptr(), _C.F32, ld, rt.data_ptr(), ld, sp, ld, g.data_ptr(), _C.F32, 1e-5, rows, dim)
            if quantize:
                _C.call("lq_rms_norm_quantize", *common, y.data_ptr(), ld, scales.data_ptr(), None)
                assert np.array_equal(y.numpy()[:, :dim], wc) and np.array_equal(scales.numpy(), ws)
            else:
                _C.call("lq_rms_norm", *common, y.data_ptr(), _C.F32, ld, None)
                assert np.array_equal(y.numpy()[:, :dim], want)
            assert (y.numpy()[:, dim:] == 9).all()
            for name, t, host in (("x", xt, x), ("res", rt, res)):
                back = t.numpy()
                assert np.array_equal(back[:, :dim], total if place == name else host[:, :dim])
                assert np.array_equal(back[:, dim:], host[:, dim:])


@pytest.mark.parametrize("dim", [64, 1100, 4096, 8192 + 3, 20000])
def test_rows_at_the_ends_of_the_range(gpu, dim):
    """Squares that overflow or vanish in float32, zeros, an infinity, NaN."""
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(dim)
    x = rng.uniform(0.5, 1, (7, dim)).astype(np.float32) * rng.choice([-1, 1], (7, dim)).astype(np.float32)
    x[0] *= np.float32(3e38)
    x[1] *= np.float32(1e25)
    x[2] *= np.float32(1e-30)
    x[3] = 0
    x[4, dim // 2] = np.inf
    x[5, dim // 3] = np.nan
    for eps in (1e-5, 1e-37):
        want = _norm(x, None, np.float64(np.float32(eps)))
        got = F.rms_norm(dev(x), eps=eps).numpy().astype(np.float64)
        fine = [0, 1, 2, 3, 6]
        close(got[fine], want[fine], (60 + dim / 2048) * U * np.abs(want[fine]) + 1e-38, f"eps {eps}")
        assert np.isnan(got[4, dim // 2]) and np.isnan(got[5]).all()
        codes, scales = (t.numpy() for t in F.rms_norm_quantize(dev(x), eps=eps))
        assert not np.isfinite(scales[[4, 5]]).any()
        assert scales[3] == 0 and (codes[3] == 0).all()
        back = codes[fine].astype(np.float64) * scales[fine, None]
        top = np.abs(want[fine]).max(1, keepdims=True)
        close(back, want[fine], top / 127 * 0.51 + 1e-38, "codes")


def test_half_sums_overflow_to_infinity(gpu):
    """x + res past float16's range is an infinity, as a float16 addition gives it."""
    import lucid_amd.nn.functional as F

    x = np.full((1, 64), 60000, np.float16)
    y, total = F.rms_norm(dev(x), residual=dev(x))
    assert np.isinf(values(total)).all() and np.isnan(values(y)).all()


def test_many_rows(gpu):
    """More rows than one dimension of a launch takes, four to a workgroup."""
    import lucid_amd.nn.functional as F

    rows = (1 << 22) * 4 + 5
    x = np.tile(np.array([[3.0, -4.0]], np.float16), (rows, 1))
    x[-1] = [1, 0]
    codes, scales = (t.numpy() for t in F.rms_norm_quantize(dev(x), eps=1e-9))
    assert (codes[:-1] == [95, -127]).all() and (codes[-1] == [127, 0]).all()
    close(scales[:-1].astype(np.float64), 4 / np.sqrt(12.5) / 127, 45 * U * scales[0], "scales")


def test_rows_feed_the_int8_product(gpu):
    """Codes and scales as the activations of lq_gemm_w8a8: exact sums of codes times both scales."""
    import lucid_amd.nn.functional as F
    from lucid_amd import _C
    from lucid_amd.quantization._gemm import WeightCache, gemm_w8a8

    rng = np.random.default_rng(5)
    for rows in (1, 7, 200):
        x = rng.standard_normal((rows, 512)).astype(np.float32)
        w = rng.integers(-127, 128, (96, 512)).astype(np.int8)
        sw = rng.uniform(0.001, 0.01, 96).astype(np.float32)
        codes, scales = F.rms_norm_quantize(dev(x))
        y = gemm_w8a8(codes, _C.I8, scales, None, WeightCache(dev(w), dev(sw), None), None, _C.OUT_F32).numpy()
        acc = codes.numpy().astype(np.int64) @ w.T.astype(np.int64)
        s = scales.numpy()[:, None] * sw[None]
        assert np.array_equal(y, acc.astype(np.float32) * s)
