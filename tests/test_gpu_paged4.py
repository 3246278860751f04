"""Attention over 4-bit pages against float64.

Bound, from the roundings alone (u = 2^-24).  Codes enter a score as c + 16 or c + 256 for a 16-bit output, as c - 7.5 else, and
what that adds is taken off again: with K = scale * log2(e) * sum_d |q_d| ((2 * 256 + 15, or 2 * 16 + 15) |scale| +
|bias|), the largest magnitudes that meet in a score, its error is at most (hd + 16) u K; a weight is off by twice that
times ln 2, and by the exponential's few u.  It enters the product with its value's scale in fp16: one term (half a step
is 2^-11) for a 16-bit output, two (2^-22) for float32, and not below fp16's smallest step, half of which is 2^-31 of the
largest weight times the largest scale; n keys add (n + 64) u.  Values meet as weight * (31 scale + |bias|).  The output is rounded once.

That bound is of the worst case, some thousand times what independent roundings add up to: over all outputs of a call the
2-norm of the error is also held to 4e-6 of the outputs' for float32 (codes enter as c - 7.5 there: some hundred
operations of u on terms up to 4 times the result, root(300) * 4 u = 4e-6 where all meet, measured 2e-7), and to half
a step for 16 bits (an output's rounding is 0.29 steps in the mean, a weight's as much for fp16)."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from _decode import HALF, Pages, U, close, dev, i32, pack4, quantize4, rounded, types, values, values4

pytestmark = pytest.mark.gpu


class Cache4:
    """A 4-bit cache of random rows; unused slots hold codes 15 with scales and biases of NaN."""

    def __init__(self, rng, lens, hkv, page, hd, size=1.0, offset=0.0, stride=None):
        self.p = Pages(rng, lens, page, stride=stride)
        shape = (self.p.pages, hkv, page)
        self.codes = {c: np.full((*shape, hd), 15, np.uint8) for c in "kv"}
        self.meta = {c: np.full((*shape, 2, n), np.nan, np.float32) for c, n in (("k", hd // 32), ("v", 1))}
        self.rows = []
        strong = np.where(rng.random((hkv, hd)) < 0.06, 4.0, 1.0)
        for b, n in enumerate(lens):
            row = {}
            for c, step in (("k", 32), ("v", hd)):
                x = rng.standard_normal((max(n, 0), hkv, hd)) * size + offset
                q = quantize4((x * strong if c == "k" else x).astype(np.float32), step)
                row[c] = q
                if n > 0:
                    page_no, slot = self.p.at(b, np.arange(n))
                    self.codes[c][page_no, :, slot] = q[0]
                    self.meta[c][page_no, :, slot] = np.stack(q[1:], -2)
            self.rows.append(row)
        self.lens, self.hkv, self.hd = lens, hkv, hd

    def tensors(self):
        return dict(k_pages=dev(pack4(self.codes["k"])), v_pages=dev(pack4(self.codes["v"])),
                    k_scale=dev(rounded(self.meta["k"], "bfloat16")[1]), v_scale=dev(rounded(self.meta["v"], "bfloat16")[1]),
                    table=i32(self.p.table), lengths=i32(self.lens))

    def attend(self, b, h, q, group, scale, w_eps, out_eps, offset):
        """(output, bound) of query head h of sequence b."""
        n, hk, hd = self.lens[b], h // group, self.hd
        if n <= 0:
            return np.zeros(hd), np.zeros(hd)
        (kc, ks, kb), (vc, vs, vb) = (tuple(a[:, hk] for a in self.rows[b][c]) for c in "kv")
        q = q.astype(np.float64)
        s = values4(kc, ks, kb) @ q * scale
        w = np.exp(s - s.max())
        w /= w.sum()
        out = w @ values4(vc, vs, vb)
        Q = np.abs(q).reshape(-1, 32).sum(1)
        K = scale * 1.4427 * (((2 * offset + 15) * np.abs(ks).astype(np.float64) + np.abs(kb)) @ Q).max()
        rel = 2 * ((hd + 16) * U * K + 16 * U) + 2 * w_eps + (n + 64) * U
        size = w @ (31 * np.abs(vs[:, 0]).astype(np.float64) + np.abs(vb[:, 0]))
        tiny = 2.0 ** -25 if out_eps == HALF["float16"] else 1e-38
        size = rel * size + n * 2.0 ** -31 * w.max() * 31 * np.abs(vs).max()
        return out, size * (1 + out_eps) + out_eps * np.abs(out) + tiny


def _check(cache, q, got, group, scale, dtype, out):
    wants = np.array([[cache.attend(b, h, q[b, h], group, scale, 0, HALF[out], 16)[0] for h in range(q.shape[1])]
                      for b in range(q.shape[0])])
    assert np.linalg.norm(got - wants) <= (4e-6 if out == "float32" else HALF[out]) * np.linalg.norm(wants)
    w_eps, offset = (2.0 ** -22, 16) if out == "float32" else (2.0 ** -11, 256)
    for b in range(q.shape[0]):
        for h in range(q.shape[1]):
            want, bound = cache.attend(b, h, q[b, h], group, scale, w_eps, HALF[out], offset)
            close(got[b, h].astype(np.float64), want, bound, f"sequence {b}, head {h}")


TYPES = [("float16", "float32"), ("float16", "float16"), ("bfloat16", "bfloat16"), ("bfloat16", "float32")]
CASES = [  # lens, heads, kv heads, hd, page
    ([1], 1, 1, 64, 16),
    ([5, 0, 63, 64, 65, -2], 4, 2, 64, 16),
    ([300, 31, 640], 8, 8, 64, 16),
    ([129, 1000], 8, 2, 128, 64),
    ([77, 256, 257], 34, 2, 32, 8),      # 17 query heads to a key head
    ([200, 90], 6, 2, 96, 1),
    ([333], 4, 4, 160, 128),
    ([100, 513], 3, 1, 192, 16),
    ([64, 255], 4, 2, 224, 32),
    ([700], 16, 1, 256, 16),
]


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("lens,h,hkv,hd,page", CASES)
def test_short_sequences(gpu, dtype, out, lens, h, hkv, hd, page):
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng([hd, page, h])
    cache = Cache4(rng, lens, hkv, page, hd, offset=0.7)
    q, qh = rounded(rng.standard_normal((len(lens), h, hd)), dtype)
    got = values(F.paged_attention(dev(qh), max_length=max(lens), out_dtype=types()[out], **cache.tensors()))
    _check(cache, q, got, h // hkv, hd ** -0.5, dtype, out)


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("lens,h,hkv,hd,page,bound", [
    ([5000, 3, 0, 1800], 4, 2, 64, 16, 5000),
    ([9000, 1025], 8, 2, 128, 64, 9000),
    ([2500, 2500, 1], 20, 1, 96, 128, 4000),
    ([1500, 40], 2, 2, 256, 64, 1100),        # a length past the bound
    ([70] * 40 + [3000], 2, 1, 128, 16, 3000),
    ([4097, 1300], 3, 1, 192, 32, 4097),
])
def test_long_sequences(gpu, dtype, out, lens, h, hkv, hd, page, bound):
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng([hd, page, bound])
    cache = Cache4(rng, lens, hkv, page, hd)
    q, qh = rounded(rng.standard_normal((len(lens), h, hd)) * 2, dtype)
    got = values(F.paged_attention(dev(qh), max_length=bound, out_dtype=types()[out], **cache.tensors()))
    _check(cache, q, got, h // hkv, hd ** -0.5, dtype, out)


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("size", [1e-20, 1e20])
def test_sizes_far_from_one(gpu, dtype, out, size):
    """Scales and biases have bfloat16's range, whatever the queries' type."""
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(3)
    cache = Cache4(rng, [90, 1400], 1, 16, 64, size=size)
    q, qh = rounded(rng.standard_normal((2, 2, 64)), dtype)
    scale = 0.125 / size
    got = values(F.paged_attention(dev(qh), max_length=1400, scale=scale, out_dtype=types()["float32"], **cache.tensors()))
    _check(cache, q, got, 2, scale, dtype, "float32")


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("bound", [200, 2000])
def test_scales_of_either_sign(gpu, dtype, out, bound):
    """Pages that a caller filled: code * scale + bias holds for a negative scale too."""
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(bound)
    cache = Cache4(rng, [bound, 70], 2, 16, 64)
    for b, n in enumerate(cache.lens):
        page_no, slot = cache.p.at(b, np.arange(n))
        for c in "kv":
            _, scale, bias = cache.rows[b][c]
            turned = rng.random(scale.shape) < (0.5 if b else 1.0)
            bias[turned] += rounded(15 * scale[turned], "bfloat16")[0]
            bias[:] = rounded(bias, "bfloat16")[0]
            scale[turned] *= -1
            cache.meta[c][page_no, :, slot] = np.stack([scale, bias], -2)
    q, qh = rounded(rng.standard_normal((2, 4, 64)), dtype)
    got = values(F.paged_attention(dev(qh), max_length=bound, out_dtype=types()[out], **cache.tensors()))
    _check(cache, q, got, 2, 0.125, dtype, out)


@pytest.mark.parametrize("n,bound", [(100, 100), (3000, 3000)])
def test_one_key_rules(gpu, n, bound):
    """A score far above the others, rising late: the sums follow the maximum."""
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(n)
    cache = Cache4(rng, [n], 1, 16, 64)
    q, qh = rounded(np.full((1, 2, 64), 3.0), "float16")
    for c, step, x in (("k", 32, 5.0), ("v", 64, -2.5)):
        row = quantize4(np.full((1, 64), x, np.float32) + rng.standard_normal((1, 64)).astype(np.float32), step)
        page_no, slot = cache.p.at(0, n - 2)
        cache.codes[c][page_no, 0, slot], cache.meta[c][page_no, 0, slot] = row[0], np.stack(row[1:], -2)
        for a, r in zip(cache.rows[0][c], row):
            a[n - 2, 0] = r[0]
    got = values(F.paged_attention(dev(qh), max_length=bound, out_dtype=types()["float32"], **cache.tensors()))
    _check(cache, q, got, 2, 0.125, "float16", "float32")


@pytest.mark.parametrize("n", [70, 2000])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_bad_pages_and_rows_that_are_not_finite(gpu, n, dtype):
    """A page outside the pool or a table that is too short: NaN for that sequence; a group of NaN reaches its own
    key head; positions past the length never do."""
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(n)
    cache = Cache4(rng, [n] * 5, 2, 16, 64)
    page_no, slot = cache.p.at(2, n // 2)
    cache.meta["k"][page_no, 1, slot, :, 1] = np.nan
    page_no, slot = cache.p.at(3, n - 1)
    cache.meta["v"][page_no, 0, slot] = np.nan
    cache.p.table[0, 1], cache.p.table[1, 2] = -1, cache.p.pages
    q, qh = rounded(rng.standard_normal((5, 4, 64)), dtype)
    t = cache.tensors()
    for out in (dtype, "float32"):
        got = values(F.paged_attention(dev(qh), max_length=n, out_dtype=types()[out], **t))
        assert np.isnan(got[:2]).all()
        assert np.isnan(got[2, 2:]).all() and np.isnan(got[3, :2]).all()
        assert np.isfinite(got[2, :2]).all() and np.isfinite(got[3, 2:]).all() and np.isfinite(got[4]).all()
    t["lengths"] = i32([t["table"].shape[1] * 16 + 1] + [n] * 4)
    got = values(F.paged_attention(dev(qh), max_length=n, **t))
    assert np.isnan(got[0]).all() and np.isfinite(got[4]).all()


def test_rows_of_wider_queries_and_other_streams(gpu):
    """The first heads of a fused projection's rows, from a created stream and from a replayed graph."""
    import lucid_amd.nn.functional as F
    from lucid_amd import _C
    from lucid_amd.graphs import CapturedForward

    rng = np.random.default_rng(8)
    for lens in ([40, 300], [2000, 1100]):
        cache = Cache4(rng, lens, 2, 16, 64)
        q, qh = rounded(rng.standard_normal((2, 8, 64)), "float16")
        t = cache.tensors()
        want = values(F.paged_attention(dev(qh[:, :4]), max_length=max(lens), **t))
        qd = dev(qh)
        got = values(F.paged_attention(qd, max_length=max(lens), heads=4, **t))
        assert np.array_equal(got, want)
        st = ctypes.c_void_p()
        _C.call("lq_stream_create", ctypes.byref(st))
        _C.synchronize()
        out = F.paged_attention(qd, max_length=max(lens), heads=4, stream=st, **t)
        _C.call("lq_stream_synchronize", st)
        assert np.array_equal(values(out), want)
        del out
        _C.call("lq_stream_destroy", st)
        cap = CapturedForward(lambda x: F.paged_attention(x, max_length=max(lens), heads=4, **t), qd)
        for _ in range(3):
            _, qh = rounded(rng.standard_normal((2, 8, 64)), "float16")
            cap.load(qh)
            got = values(cap())
            assert np.array_equal(got, values(F.paged_attention(dev(qh), max_length=max(lens), heads=4, **t)))


def test_results_repeat(gpu):
    """The same bits from call to call, also where a sequence is joined from many parts."""
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(4)
    cache = Cache4(rng, [30000, 700], 1, 64, 128)
    _, qh = rounded(rng.standard_normal((2, 4, 128)), "bfloat16")
    t, q = cache.tensors(), dev(qh)
    want = values(F.paged_attention(q, max_length=30000, **t))
    for _ in range(3):
        assert np.array_equal(values(F.paged_attention(q, max_length=30000, **t)), want)


def test_pool_past_32_bits(gpu):
    """Rows whose byte offsets pass 2^32: the same result as from a small pool."""
    import lucid_amd as L
    import lucid_amd.nn.functional as F
    from lucid_amd import _C

    rng = np.random.default_rng(6)
    n, page, hd = 200, 64, 128
    small = Cache4(rng, [n], 1, page, hd)
    t = small.tensors()
    _, qh = rounded(rng.standard_normal((1, 2, hd)), "float16")
    want = values(F.paged_attention(dev(qh), max_length=n, **t))
    pages = (1 << 32) // (page * hd // 2) + 9  # the last pages' codes begin past 2^32 bytes
    big = dict(k_pages=L.empty((pages, 1, page, hd // 2), np.uint8, "gpu"), v_pages=L.empty((pages, 1, page, hd // 2), np.uint8, "gpu"),
               k_scale=L.empty((pages, 1, page, 2, 4), L.bfloat16, "gpu"), v_scale=L.empty((pages, 1, page, 2, 1), L.bfloat16, "gpu"))
    table = np.array([[pages - 1, pages - 5, 3, pages - 8]], np.int32)
    for name, a in big.items():
        item = t[name].numel() // small.p.pages * np.dtype(t[name].dtype).itemsize
        for j in range(4):
            _C.call("lq_memcpy_d2d", a.data_ptr() + int(table[0, j]) * item,
                    t[name].data_ptr() + int(small.p.table[0, j]) * item, item, None)
    got = values(F.paged_attention(dev(qh), table=i32(table), lengths=i32([n]), max_length=n, **big))
    assert np.array_equal(got, want)
