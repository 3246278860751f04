"""Attention over 4-bit pages whose rows differ far in size, against float64.

The bound is that of test_gpu_paged4.py but for what fp16 drops of a weight times its value's scale: half its least
step is 2^-35 of the largest such product that a query meets, whatever the scales of the rows that it ignores (that
file allows 2^-31 of the largest weight times the largest scale, wherever they are)."""

from __future__ import annotations

import numpy as np
import pytest

from _decode import HALF, U, close, dev, rounded, types, values, values4
from test_gpu_paged4 import TYPES, Cache4

pytestmark = pytest.mark.gpu


def _check(cache, q, got, group, scale, out, w_eps=None, offset=None, skip=0):
    if w_eps is None:
        w_eps, offset = (2.0 ** -22, 16) if out == "float32" else (2.0 ** -11, 256)
    for b, n in list(enumerate(cache.lens))[skip:]:
        for h in range(q.shape[1]):
            (kc, ks, kb), (vc, vs, vb) = (tuple(a[:, h // group] for a in cache.rows[b][c]) for c in "kv")
            x = q[b, h].astype(np.float64)
            s = values4(kc, ks, kb) @ x * scale
            w = np.exp(s - s.max())
            w /= w.sum()
            want = w @ values4(vc, vs, vb)
            vs, vb = (np.abs(a[:, 0]).astype(np.float64) for a in (vs, vb))
            K = scale * 1.4427 * (((2 * offset + 15) * np.abs(ks).astype(np.float64) + np.abs(kb))
                                  @ np.abs(x).reshape(-1, 32).sum(1)).max()
            rel = 2 * ((cache.hd + 16) * U * K + 16 * U) + 2 * w_eps + (n + 64) * U
            size = rel * (w @ (31 * vs + vb)) + n * 2.0 ** -35 * (w * vs).max() * 31
            bound = size * (1 + HALF[out]) + HALF[out] * np.abs(want) + (2.0 ** -25 if out == "float16" else 1e-38)
            close(got[b, h].astype(np.float64), want, bound, f"sequence {b}, head {h}")


def _run(cache, rng, h, dtype, out, scale, positive=False):
    import lucid_amd.nn.functional as F

    q = rng.standard_normal((len(cache.lens), h, cache.hd))
    q, qh = rounded(np.abs(q) + 0.3 if positive else q, dtype)
    got = values(F.paged_attention(dev(qh), max_length=max(cache.lens), scale=scale, out_dtype=types()[out], **cache.tensors()))
    return q, got


def _store(cache, b, pos):
    """The rows of sequence b at positions pos, as they are in ``rows``, into the pages."""
    page_no, slot = cache.p.at(b, pos)
    for c in "kv":
        codes, scale, bias = cache.rows[b][c]
        cache.codes[c][page_no, :, slot], cache.meta[c][page_no, :, slot] = codes[pos], np.stack([scale, bias], -2)[pos]


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("n", [90, 3000])
@pytest.mark.parametrize("k", [12, 24, 40, 100])
def test_a_row_that_attention_ignores(gpu, dtype, out, page, n, k):
    """Values of 2^k times the others' scale where the score lies some 60 below them: at 2^100 such a row still counts."""
    rng = np.random.default_rng([n, k, page])
    cache = Cache4(rng, [n, 70], 2, page, 64)
    for b, length in enumerate(cache.lens):
        pos = np.array([0, length // 2, length - 1])
        (kc, ks, kb), (vc, vs, vb) = (cache.rows[b][c] for c in "kv")
        kc[pos], ks[pos], kb[pos] = 0, 0, -8
        vs[pos], vb[pos] = vs[pos] * 2.0 ** k, vb[pos] * 2.0 ** k
        _store(cache, b, pos)
    q, got = _run(cache, rng, 4, dtype, out, 0.125, positive=True)
    _check(cache, q, got, 2, 0.125, out)


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("order", ["rising", "falling", "any"])
@pytest.mark.parametrize("n,hd,spread", [(200, 32, 1.0), (700, 64, 8.0), (2600, 128, 1.0), (2600, 96, 8.0)])
def test_scales_from_tiny_to_large(gpu, dtype, out, order, n, hd, spread):
    """Rows of scales over 58 powers of two beside scores that rule some of them out: what the sums are relative to moves
    through the whole sequence."""
    rng = np.random.default_rng([n, hd, len(order)])
    cache = Cache4(rng, [n, 33], 1, 16, hd)
    for b, length in enumerate(cache.lens):
        e = rng.uniform(-50, 8, length)
        e = np.floor({"rising": np.sort(e), "falling": -np.sort(-e), "any": e}[order])[:, None, None]
        _, vs, vb = cache.rows[b]["v"]
        vs *= 2.0 ** e
        vb *= 2.0 ** e
        _store(cache, b, np.arange(length))
    q, got = _run(cache, rng, 3, dtype, out, spread * hd ** -0.5)
    _check(cache, q, got, 3, spread * hd ** -0.5, out)


@pytest.mark.parametrize("dtype,out", [("float16", "float32"), ("bfloat16", "bfloat16"), ("bfloat16", "float32")])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("n,power,offset", [(640, 120, 1.0), (20000, 120, -1.0), (640, 120, 0.0), (4096, 125, 0.0),
                                            (20000, -90, 1.0), (640, -90, 0.0)])
def test_values_near_the_ends_of_the_range(gpu, dtype, out, page, n, power, offset):
    """Many values of 1e36, or some of the type's largest, have finite sums; of 1e-27 they keep their bits."""
    rng = np.random.default_rng([n, power + 100])
    cache = Cache4(rng, [n, 20], 1, page, 64, offset=offset)
    for b, length in enumerate(cache.lens):
        _, vs, vb = cache.rows[b]["v"]
        vs *= 2.0 ** power
        vb *= 2.0 ** power
        _store(cache, b, np.arange(length))
    q, got = _run(cache, rng, 2, dtype, out, 0.125)
    _check(cache, q, got, 2, 0.125, out)


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("lens,h,hkv,hd,page", [([3, 9, 700, 900], 32, 8, 128, 64), ([4000, 70], 8, 8, 64, 16),
                                                ([1300, 5000], 12, 3, 96, 32), ([80, 2000], 4, 2, 256, 64)])
def test_sixteen_bit_outputs_are_rounded_once(gpu, dtype, out, lens, h, hkv, hd, page):
    """Weights of 22 bits and codes with 16 added for every output type.  Over all outputs of a call the 2-norm of the
    error is what rounding the exact ones gives, 5% more (some thousand roundings, whose mean square varies by 1 or 2%), and
    8.4e-6 of the outputs': the float32 outputs' 4e-6 (test_gpu_paged4.py) with terms of 31 scales where those have 15."""
    rng = np.random.default_rng([hd, page])
    cache = Cache4(rng, lens, hkv, page, hd)
    group = h // hkv
    q, got = _run(cache, rng, h, dtype, out, hd ** -0.5)
    _check(cache, q, got, group, hd ** -0.5, out, 2.0 ** -22, 16)
    want = np.array([[cache.attend(b, j, q[b, j], group, hd ** -0.5, 0, 0, 0)[0] for j in range(h)] for b in range(len(lens))])
    norm = np.linalg.norm
    alone = norm(rounded(want, out)[0] - want)
    assert norm(got - want) <= 1.05 * alone + 8.4e-6 * norm(want)


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("n,hd,spread", [(300, 64, 40.0), (3000, 128, 40.0), (2000, 192, 8.0)])
def test_scores_far_apart(gpu, dtype, out, n, hd, spread):
    """Attention that a few keys rule, whose scores are large beside what decides between them."""
    rng = np.random.default_rng([n, hd])
    cache = Cache4(rng, [n, 100], 1, 64, hd, offset=0.5)
    q, got = _run(cache, rng, 4, dtype, out, spread * hd ** -0.5)
    _check(cache, q, got, 4, spread * hd ** -0.5, out, 2.0 ** -22, 16)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("n,hd", [(300, 64), (300, 128), (3000, 64), (3000, 128)])
def test_float32_outputs_keep_the_bits_of_the_weights(gpu, dtype, n, hd):
    """The weights that count have exponents near 0, whose rounding is 2^-25 of a weight and not 2^-20: what is left are
    some ten roundings to a score of a few units (2^-22 each), alike in the 2-norm: 2^-22 root(10), and as much for the
    sums: 1.1e-6 at most where all meet."""
    rng = np.random.default_rng(n + hd)
    cache = Cache4(rng, [n], 2, 64, hd)
    q, got = _run(cache, rng, 8, dtype, "float32", hd ** -0.5)
    want = np.array([cache.attend(0, j, q[0, j], 4, hd ** -0.5, 0, 0, 0)[0] for j in range(8)])
    assert np.linalg.norm(got[0] - want) <= 1.1e-6 * np.linalg.norm(want)


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("n,hd,page", [(200, 64, 16), (2500, 128, 64), (90, 256, 128)])
def test_queries_of_very_different_dims(gpu, dtype, out, n, hd, page):
    """Groups of dims whose queries are far smaller than the others' and whose keys are far larger: each counts as much
    as the others (fp16 queries as far as that type goes)."""
    rng = np.random.default_rng([n, hd])
    cache = Cache4(rng, [n, 70], 1, page, hd, offset=0.3)
    groups = hd // 32
    powers = np.array([0.0, 44.0, -20.0, 60.0, 7.0, -70.0, 30.0, 1.0])[:groups] if dtype == "bfloat16" else \
        np.array([0.0, 10.0, -3.0, 12.0, 2.0, 5.0, 9.0, 1.0])[:groups]
    for b, length in enumerate(cache.lens):
        _, ks, kb = cache.rows[b]["k"]
        ks *= 2.0 ** powers
        kb *= 2.0 ** powers
        _store(cache, b, np.arange(length))
    import lucid_amd.nn.functional as F

    q, qh = rounded(rng.standard_normal((2, 3, hd)) * np.repeat(2.0 ** -powers, 32), dtype)
    got = values(F.paged_attention(dev(qh), max_length=n, out_dtype=types()[out], **cache.tensors()))
    _check(cache, q, got, 3, hd ** -0.5, out, 2.0 ** -22, 16)


@pytest.mark.parametrize("out", ["bfloat16", "float32"])
@pytest.mark.parametrize("size", [1e-37, 1e-30, 1e30, 1e38])
@pytest.mark.parametrize("n", [70, 1500])
def test_queries_of_any_size(gpu, out, size, n):
    """bfloat16 queries at the ends of the range, a row of zeros among them, keys of the inverse size."""
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(n)
    cache = Cache4(rng, [n, 70], 1, 16, 64)
    power = -np.round(np.log2(size))
    for b, length in enumerate(cache.lens):
        _, ks, kb = cache.rows[b]["k"]
        ks *= 2.0 ** power
        kb *= 2.0 ** power
        _store(cache, b, np.arange(length))
    x = rng.uniform(-1, 1, (2, 3, 64)) * 2.0 ** -power
    x[1, 1] = 0
    q, qh = rounded(x, "bfloat16")
    got = values(F.paged_attention(dev(qh), max_length=n, out_dtype=types()[out], **cache.tensors()))
    _check(cache, q, got, 3, 0.125, out, 2.0 ** -22, 16)


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("scale", [1e-45, 1e-38, 1e-12])
def test_tiny_scales(gpu, dtype, out, scale):
    """A scale so small that all positions weigh the same, with queries of zeros and of ordinary size."""
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(3)
    cache = Cache4(rng, [90, 1100], 1, 16, 64)
    x = rng.standard_normal((2, 3, 64))
    x[:, 1] = 0
    q, qh = rounded(x, dtype)
    got = values(F.paged_attention(dev(qh), max_length=1100, scale=scale, out_dtype=types()[out], **cache.tensors()))
    _check(cache, q, got, 3, scale, out, 2.0 ** -22, 16)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("n,hd,page", [(640, 64, 16), (3000, 128, 64)])
@pytest.mark.parametrize("power", [-114, -60, 0, 60, 100])
def test_values_of_any_size_keep_their_bits(gpu, dtype, n, hd, page, power):
    """The 2-norm of a float32 output's error is the same part of the output, however small or large the values: the 4e-6
    of test_gpu_paged4.py."""
    rng = np.random.default_rng([n, hd])
    cache = Cache4(rng, [n], 2, page, hd)
    _, vs, vb = cache.rows[0]["v"]
    vs *= 2.0 ** power
    vb *= 2.0 ** power
    _store(cache, 0, np.arange(n))
    q, got = _run(cache, rng, 4, dtype, "float32", hd ** -0.5)
    want = np.array([cache.attend(0, j, q[0, j], 2, hd ** -0.5, 0, 0, 0)[0] for j in range(4)])
    assert np.linalg.norm(got[0] - want) <= 4e-6 * np.linalg.norm(want)


@pytest.mark.parametrize("dtype,out", [("float16", "float32"), ("bfloat16", "bfloat16"), ("bfloat16", "float32")])
@pytest.mark.parametrize("n", [200, 3000, 9000])
@pytest.mark.parametrize("first", [0, 150, 2900])
def test_large_values_from_some_position_on(gpu, dtype, out, n, first):
    """Values of 2^100 after ones of 2^60, their scores as much lower, so that both count."""
    if first >= n:
        first = n - 20
    rng = np.random.default_rng([n, first])
    cache = Cache4(rng, [n, 40], 1, 64, 64)
    (kc, ks, kb), (vc, vs, vb) = (cache.rows[0][c] for c in "kv")
    vs *= 2.0 ** 60
    vb *= 2.0 ** 60
    pos = np.arange(first, n, 7)
    kc[pos], ks[pos], kb[pos] = 0, 0, -3.5  # some 28 below the others
    vs[pos] *= 2.0 ** 40
    vb[pos] *= 2.0 ** 40
    _store(cache, 0, np.arange(n))
    q, got = _run(cache, rng, 2, dtype, out, 0.125, positive=True)
    _check(cache, q, got, 2, 0.125, out, 2.0 ** -22, 16)
