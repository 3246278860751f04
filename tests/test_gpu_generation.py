"""Serving ops on the GPU against plain float64 restatements: the paged append (bit-exact), single
token attention over pages, attention over packed prompts, token log probabilities and their
gradient (against the formula and against differences).

Bounds, from the roundings alone.  u = 2^-24 (half a step of float32), eps = half a step of the
16-bit type.  Attention: a score is a float32 sum of hd products, scaled into log2 units, so its
error is at most (hd + 8) u S with S = scale * log2(e) * sum_d |q_d k_d| (+ the rounding of a
stored maximum); a weight's relative error is that times ln 2 twice (the weight and the sum), plus
the exponential's few u, plus eps once or twice where the weights enter the products in 16 bits
(16-bit outputs) or 2^-16 where they enter as two terms; sums over n keys add n u.  The output is
rounded once more (by half of the type's smallest step below its normal range).  Log probabilities: e^d has the relative error (2 |d| + 8) u, a sum of n terms
n / 64 u more per lane and level."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def _types():
    import lucid_amd as L

    return {"float32": L.float32, "float16": L.float16, "bfloat16": L.bfloat16, "int8": L.int8}


def _round(a, dtype):
    """(values as float64, host array in the storage type) of float32 ``a`` rounded to ``dtype``."""
    import lucid_amd as L

    a = np.asarray(a, np.float32)
    if dtype == "bfloat16":
        bits = L.bf16_from_f32(a)
        return L.bf16_to_f32(bits).astype(np.float64), bits
    h = a.astype(np.float16 if dtype == "float16" else np.float32)
    return h.astype(np.float64), h


def _values(t):
    import lucid_amd as L

    a = t.numpy()
    return L.bf16_to_f32(a).astype(np.float64) if t.dtype == L.bfloat16 else a.astype(np.float64)


def _dev(a):
    import lucid_amd as L

    return L.tensor(np.ascontiguousarray(a), device="gpu")


def _i32(a):
    return _dev(np.asarray(a, np.int32))


def _attend(q, k, v, scale, weight_eps, out_eps):
    """(output, bound) of one query head q [hd] over keys k / v [n, hd] in float64."""
    n, hd = k.shape
    if n == 0:
        return np.zeros(hd), np.zeros(hd)
    s = (k @ q) * scale
    w = np.exp(s - s.max())
    w /= w.sum()
    out = w @ v
    S = scale * 1.4427 * (np.abs(k) @ np.abs(q)).max()
    rel = 2 * ((hd + 8) * U * S + 16 * U) + 2 * weight_eps + (n + 64) * U
    tiny = 2.0 ** -25 if out_eps == HALF["float16"] else 1e-38  # half of the type's smallest step
    return out, rel * (w @ np.abs(v)) * (1 + out_eps) + out_eps * np.abs(out) + tiny


def _check(got, want, bound, what=""):
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} outside the bound, worst "
                           f"{np.nanmax(np.abs(got - want) / bound):.3g} times, NaN {np.isnan(got).sum()}")


def _weight_eps(dtype, out):
    return 2.0 ** -16 if out == "float32" else HALF[dtype]


# ------------------------------------------------------------------------------ append


class Pool:
    """A host page pool with a shuffled table; unused slots hold NaN (or code 77 with a NaN scale)."""

    def __init__(self, rng, lens, hkv, page, hd, cache, spare=3, stride=None):
        self.lens, self.page = list(lens), page
        used = [-(-max(n, 0) // page) for n in lens]
        self.pages = sum(used) + spare
        ids = rng.permutation(self.pages)[:sum(used)]
        width = max(used + [1]) if stride is None else stride
        self.table = rng.integers(-5, self.pages + 5, (len(lens), width)).astype(np.int32)  # unused entries: anything
        at = 0
        for b, u in enumerate(used):
            self.table[b, :u] = ids[at:at + u]
            at += u
        shape = (self.pages, hkv, page, hd)
        self.cache = cache
        self.k, self.v = np.full(shape, np.nan, np.float32), np.full(shape, np.nan, np.float32)

    def slot(self, b, p):
        return self.table[b, p // self.page], p % self.page


def _source(rng, tokens, hkv, hd, src):
    return _round(rng.standard_normal((tokens, 2, hkv, hd)) * rng.choice([0.1, 1, 30], (tokens, 1, 1, 1)), src)


@pytest.mark.parametrize("src", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("cache", ["float16", "bfloat16", "int8"])
@pytest.mark.parametrize("lens,new,hkv,hd,page", [
    ([5, 1, 40, 17], [5, 1, 7, 0], 2, 64, 16),
    ([3, 0, 8], [1, 1, 1], 1, 40, 8),        # a step, one sequence of length 0
    ([9, 30], [9, 2], 3, 7, 5),              # rows no vector fits
    ([300], [300], 8, 128, 64),
    ([20, 70], [4, 3], 2, 256, 1),
])
def test_append_is_exact(gpu, src, cache, lens, new, hkv, hd, page):
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng([len(src), len(cache), hd, page])
    T = _types()
    pool = Pool(rng, lens, hkv, page, hd, cache)
    step = all(n == 1 for n in new)
    tokens = sum(new)
    x, host = _source(rng, tokens, hkv, hd, src)
    if cache == "int8":
        x[0, 0, 0] = 0  # a row of zeros
        host[0, 0, 0] = _round(np.zeros(hd), src)[1]
    shape = (pool.pages, hkv, page, hd)
    fill = np.full(shape, 77, np.int8) if cache == "int8" else _round(np.full(shape, 77.0), cache)[1]
    k, v = _dev(fill), _dev(fill)
    scales = {}
    if cache == "int8":
        scales = {n: _dev(np.full(shape[:3], 0.5, np.float32)) for n in ("k_scale", "v_scale")}
    starts = None if step else _i32(np.concatenate([[0], np.cumsum(new)]))
    F.paged_kv_append(_dev(host[:, 0]), _dev(host[:, 1]), k, v, _i32(pool.table), _i32(lens), starts, **scales)
    assert k.dtype == T[cache]
    want_k, want_v = fill.copy(), fill.copy()
    want_s = [np.full(shape[:3], 0.5, np.float32) for _ in range(2)]
    t = 0
    for b, (n, m) in enumerate(zip(lens, new)):
        for i in range(m):
            p = n - m + i
            if p >= 0:
                pg, sl = pool.slot(b, p)
                for j, dst in enumerate((want_k, want_v)):
                    row = x[t, j].astype(np.float32)
                    if cache == "int8":
                        top = np.abs(row).max(-1)
                        with np.errstate(divide="ignore", invalid="ignore"):
                            inv = np.float32(127) / top
                            codes = np.clip(np.rint(row * inv[:, None]), -127, 127)
                        dst[pg, :, sl] = np.where(top[:, None] > 0, codes, 0).astype(np.int8)
                        want_s[j][pg, :, sl] = top / np.float32(127)
                    else:
                        dst[pg, :, sl] = _round(row, cache)[1]
            t += 1
    np.testing.assert_array_equal(k.numpy(), want_k)
    np.testing.assert_array_equal(v.numpy(), want_v)
    if cache == "int8":
        np.testing.assert_array_equal(scales["k_scale"].numpy(), want_s[0])
        np.testing.assert_array_equal(scales["v_scale"].numpy(), want_s[1])


def test_append_leaves_out_what_has_no_place(gpu):
    """Page numbers outside the pool, positions past the table, tokens before the first start:
    nothing of them is written, the rest is."""
    import lucid_amd.nn.functional as F

    hkv, hd, page = 1, 8, 4
    table = np.array([[0, 99], [-1, 1], [2, 3]], np.int32)
    lens = np.array([6, 6, 11], np.int32)  # the third sequence has 3 positions past its two pages
    starts = np.array([1, 7, 13, 24], np.int32)  # token 0 belongs to no sequence
    x = np.arange(24 * hd, dtype=np.float32).reshape(24, hkv, hd) / 64
    k, v = (_dev(np.full((4, hkv, page, hd), -1, np.float16)) for _ in range(2))
    F.paged_kv_append(_dev(x), _dev(-x), k, v, _i32(table), _i32(lens), _i32(starts))
    want = np.full((4, hkv, page, hd), -1, np.float32)
    want[0, 0] = x[1:5, 0]          # positions 0 .. 3 of sequence 0; 4, 5 have a bad page
    want[1, 0, :2] = x[11:13, 0]    # positions 4, 5 of sequence 1; 0 .. 3 have a bad page
    want[2, 0], want[3, 0] = x[13:17, 0], x[17:21, 0]
    np.testing.assert_array_equal(k.numpy().astype(np.float32), want.astype(np.float16).astype(np.float32))
    np.testing.assert_array_equal(v.numpy().astype(np.float32),
                                  np.where(want == -1, -1, -want).astype(np.float16).astype(np.float32))


def test_append_int8_of_rows_that_are_not_finite(gpu):
    import lucid_amd.nn.functional as F

    x = np.ones((3, 1, 16), np.float32)
    x[0, 0, 3], x[1, 0, 5], x[2] = np.nan, np.inf, 1e-38
    k, v = (_dev(np.zeros((3, 1, 1, 16), np.int8)) for _ in range(2))
    s, s2 = (_dev(np.zeros((3, 1, 1), np.float32)) for _ in range(2))
    F.paged_kv_append(_dev(x), _dev(x), k, v, _i32([[0], [1], [2]]), _i32([1, 1, 1]), None, s, s2)
    with np.errstate(invalid="ignore"):
        back = k.numpy().astype(np.float32) * s.numpy()[..., None]
    assert np.isnan(s.numpy()[0]) and np.isnan(back[0]).all()
    assert np.isinf(s.numpy()[1]) and not np.isfinite(back[1]).any()
    assert s.numpy()[2] == 0 and (k.numpy()[2] == 0).all()


# ------------------------------------------------------------------------------ paged attention


def _paged(rng, lens, h, hkv, hd, page, dtype, cache, out, max_length=None, stride=None, scale=None, poison=True):
    import lucid_amd.nn.functional as F

    B = len(lens)
    pool = Pool(rng, lens, hkv, page, hd, cache, stride=stride)
    shape = (pool.pages, hkv, page, hd)
    kv, host = {}, {}
    scales = {}
    strong = 1 + 3 * (rng.random((hkv, 1, hd)) < 1 / 16)
    for name, wide in (("k", strong), ("v", 1.0)):
        x = rng.standard_normal(shape) * wide
        if cache == "int8":
            top = np.abs(x).max(-1)
            codes = np.rint(x * (127 / top)[..., None]).astype(np.int8)
            sc = (top / 127 * rng.choice([1e-6, 1.0], shape[:3] if name == "v" else (1, 1, 1))).astype(np.float32)
            kv[name], host[name] = codes * sc[..., None].astype(np.float64), codes
            scales[name + "_scale"] = sc
        else:
            kv[name], host[name] = _round(x, cache)
    # slots no sequence holds: infinities and NaN must not reach an output
    if poison:
        free = np.ones(shape[0] * page, bool).reshape(shape[0], page)
        for b, n in enumerate(lens):
            for p in range(max(n, 0)):
                free[pool.slot(b, p)] = False
        pg, sl = np.nonzero(free)
        if cache == "int8":
            for sc in scales.values():
                sc[pg, :, sl] = np.nan
        else:
            bad = _round(np.array([np.nan, np.inf]), cache)[1]
            host["k"][pg, :, sl], host["v"][pg, :, sl] = bad[0], bad[1]
            host["v"][pg[::2], :, sl[::2]] = bad[0]
    q, qh = _round(rng.standard_normal((B, h, hd)), dtype)
    T = _types()
    got = F.paged_attention(_dev(qh), _dev(host["k"]), _dev(host["v"]), _i32(pool.table), _i32(lens),
                            max(max(lens), 0) if max_length is None else max_length, scale,
                            out_dtype=T[out], **{n: _dev(s) for n, s in scales.items()})
    assert got.dtype == T[out]
    got = _values(got)
    weps, oeps = _weight_eps(dtype, out), U if out == "float32" else HALF[out]
    for b, n in enumerate(lens):
        at = [pool.slot(b, p) for p in range(max(n, 0))]
        pg, sl = [a[0] for a in at], [a[1] for a in at]
        for j in range(h):
            hk = j // (h // hkv)
            kk, vv = (kv[c][pg, hk, sl] if n > 0 else np.zeros((0, hd)) for c in ("k", "v"))
            want, bound = _attend(q[b, j], kk, vv, hd ** -0.5 if scale is None else scale, weps, oeps)
            _check(got[b, j], want, bound, f"sequence {b} of {n}, head {j}")


@pytest.mark.parametrize("dtype,cache,out", [("float16", "float16", "float32"), ("float16", "float16", "float16"),
                                             ("bfloat16", "bfloat16", "bfloat16"), ("bfloat16", "bfloat16", "float32"),
                                             ("float16", "int8", "float16"), ("bfloat16", "int8", "float32")])
@pytest.mark.parametrize("lens,h,hkv,hd,page", [
    ([1], 1, 1, 64, 16),
    ([0, 1, 2, 31, 32, 33, -3], 4, 2, 64, 8),
    ([63, 64, 65, 127, 129], 8, 1, 128, 64),
    ([300, 5], 6, 2, 40, 7),           # a page that is no power of two, a head dim of few chunks
    ([200, 17], 17, 1, 72, 16),        # more queries per key head than one tile of 16
    ([100], 3, 3, 256, 32),
    ([40, 90], 32, 2, 248, 128),
    ([77], 5, 5, 8, 1),
    ([50, 60], 40, 1, 96, 256),
])
def test_paged_attention(gpu, dtype, cache, out, lens, h, hkv, hd, page):
    _paged(np.random.default_rng(len(lens) * 1000 + hd + h), lens, h, hkv, hd, page, dtype, cache, out)


@pytest.mark.parametrize("cache", ["float16", "int8"])
@pytest.mark.parametrize("lens,h,hkv,hd,page", [([4097, 1, 1300], 4, 2, 64, 16), ([2049], 8, 1, 128, 128),
                                                ([9000, 8191], 2, 1, 128, 64)])
def test_paged_attention_split_over_the_positions(gpu, cache, lens, h, hkv, hd, page):
    for out in ("float32", "float16"):
        _paged(np.random.default_rng(hd + len(lens)), lens, h, hkv, hd, page, "float16", cache, out)


@pytest.mark.parametrize("max_length", [0, 1, 700, 5000])
def test_paged_attention_attends_lengths_past_the_bound(gpu, max_length):
    """max_length only plans the split."""
    _paged(np.random.default_rng(max_length), [3000, 0, 12, 1500], 4, 2, 64, 16, "float16", "float16", "float32",
           max_length=max_length)


def test_paged_attention_many_sequences_and_a_wide_table(gpu):
    rng = np.random.default_rng(4)
    _paged(rng, [int(n) for n in rng.integers(0, 60, 300)], 2, 1, 64, 16, "bfloat16", "bfloat16", "bfloat16", stride=9)


@pytest.mark.parametrize("scale", [1e-3, 2.0])
def test_paged_attention_scale(gpu, scale):
    _paged(np.random.default_rng(8), [70, 300], 4, 2, 64, 16, "float16", "float16", "float32", scale=scale)


def test_paged_attention_of_pages_outside_the_pool_is_nan(gpu):
    """A page number outside the pool, or a length past the table, gives NaN for that sequence
    and touches no other."""
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(1)
    k, v = (_dev(rng.standard_normal((4, 2, 8, 64)).astype(np.float16)) for _ in range(2))
    q = _dev(rng.standard_normal((4, 4, 64)).astype(np.float16))
    table, lens = [[0, 1], [2, 4], [-1, 3], [3, 0]], [16, 9, 12, 17]
    got = F.paged_attention(q, k, v, _i32(table), _i32(lens), 17).numpy()
    assert np.isfinite(got[0]).all()
    assert np.isnan(got[1]).all() and np.isnan(got[2]).all() and np.isnan(got[3]).all()
    lens[1], lens[3] = 8, 16  # the bad entries are not reached
    got = F.paged_attention(q, k, v, _i32(table), _i32(lens), 16).numpy()
    assert np.isfinite(got[[0, 1, 3]]).all()


def test_paged_attention_keeps_infinite_scores_like_the_formula(gpu):
    """A key whose score is -inf has weight 0; a NaN within the length reaches its own head only."""
    import lucid_amd.nn.functional as F

    k = np.ones((1, 2, 8, 64), np.float16)
    v = np.random.default_rng(2).standard_normal((1, 2, 8, 64)).astype(np.float16)
    k[0, 0, 3] = -np.inf
    k[0, 1, 2, 5] = np.nan
    q = np.ones((1, 2, 64), np.float16)
    got = F.paged_attention(_dev(q), _dev(k), _dev(v), _i32([[0]]), _i32([8]), 8, out_dtype=np.float32).numpy()
    want = v[0, 0, [0, 1, 2, 4, 5, 6, 7]].astype(np.float64).mean(0)
    np.testing.assert_allclose(got[0, 0], want, atol=1e-4)
    assert np.isnan(got[0, 1]).all()


@pytest.mark.parametrize("cache,hd", [("float16", 64), ("float16", 128), ("int8", 128), ("float16", 40), ("int8", 64),
                                      ("float16", 192)])
@pytest.mark.parametrize("seqs,longest,h,hkv", [(150, 1400, 2, 1), (40, 3000, 4, 4), (3, 1100, 20, 1), (200, 1025, 1, 1)])
def test_paged_attention_shared_positions(gpu, cache, hd, seqs, longest, h, hkv):
    """Lengths of every kind on one line of work: more sequences than a workgroup has threads, parts
    that begin and end inside sequences, empty ones between, two tiles of query heads."""
    from lucid_amd import _C

    rng = np.random.default_rng(seqs + hd)
    lens = [int(n) for n in np.exp(rng.uniform(0, np.log(longest), seqs))]
    lens[seqs // 2], lens[-1], lens[0] = longest, 0, 0
    lens[1:seqs // 3:7] = [0] * len(lens[1:seqs // 3:7])
    _paged(rng, lens, h, hkv, hd, 16, "float16", cache, "float32")
    assert _C.last_path() == "paged shared"


def test_paged_attention_paths(gpu):
    from lucid_amd import _C

    for hd in (64, 128):
        _paged(np.random.default_rng(1), [40, 1000], 2, 1, hd, 16, "float16", "float16", "float16")
        assert _C.last_path() == "paged whole few"
        _paged(np.random.default_rng(2), [int(n) for n in np.random.default_rng(2).integers(0, 90, 140)], 4, 2, hd, 16,
               "bfloat16", "bfloat16", "bfloat16")
        assert _C.last_path() == "paged whole"


def test_paged_cache_past_32_bits(gpu):
    """A pool of more than 2^32 bytes and 2^31 values: the last pages hold what was appended and are
    attended."""
    import lucid_amd as L
    import lucid_amd.nn.functional as F

    hkv, page, hd = 8, 64, 64
    pages = (1 << 31) // (hkv * page * hd) + 40
    k, v = (L.empty((pages, hkv, page, hd), L.float16, "gpu") for _ in range(2))
    assert k.nbytes > 1 << 32
    rng = np.random.default_rng(0)
    table = np.array([[pages - 1, 3, pages - 2]], np.int32)
    x = rng.standard_normal((150, 2, hkv, hd)).astype(np.float16)
    F.paged_kv_append(_dev(x[:, 0]), _dev(x[:, 1]), k, v, _i32(table), _i32([150]), _i32([0, 150]))
    q = rng.standard_normal((1, hkv, hd)).astype(np.float16)
    for bound in (150, 2000):
        got = F.paged_attention(_dev(q), k, v, _i32(table), _i32([150]), bound, out_dtype=L.float32).numpy()
        for j in range(hkv):
            want, b = _attend(q[0, j].astype(np.float64), x[:, 0, j].astype(np.float64), x[:, 1, j].astype(np.float64),
                              hd ** -0.5, 2.0 ** -16, U)
            _check(got[0, j], want, b, f"head {j}")


@pytest.mark.parametrize("hd", [64, 128, 72])
@pytest.mark.parametrize("n", [70, 1500])
def test_paged_attention_of_infinite_values(gpu, hd, n):
    """An infinity among the values gives an infinity in its dim (NaN where both signs meet) and
    nothing elsewhere."""
    import lucid_amd as L
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(n + hd)
    pages = -(-n // 16)
    k, v = (rng.standard_normal((pages, 1, 16, hd)).astype(np.float16) for _ in range(2))
    v[1, 0, 3, 5], v[2, 0, 1, 6], v[3, 0, 0, 6], v[0, 0, 2, 9] = np.inf, np.inf, -np.inf, -np.inf
    q = rng.standard_normal((1, 3, hd)).astype(np.float16)
    table = np.arange(pages, dtype=np.int32)[None]
    for dt in (L.float32, L.float16):
        got = _values(F.paged_attention(_dev(q), _dev(k), _dev(v), _i32(table), _i32([n]), n, out_dtype=dt))[0]
        assert (got[:, 5] == np.inf).all() and np.isnan(got[:, 6]).all() and (got[:, 9] == -np.inf).all()
        assert np.isfinite(np.delete(got, [5, 6, 9], 1)).all()


# ------------------------------------------------------------------------------ prompts


def _prompt(rng, nq, nk, h, hkv, hd, dtype, out, causal=True, fused=False, mutate=None, scale=None):
    import lucid_amd as L
    import lucid_amd.nn.functional as F

    T = _types()
    tq, tk = sum(nq), sum(nk)
    qs, ks = np.concatenate([[0], np.cumsum(nq)]), np.concatenate([[0], np.cumsum(nk)])
    q, qh = _round(rng.standard_normal((tq, h, hd)), dtype)
    k, kh = _round(rng.standard_normal((tk, hkv, hd)) * (1 + 3 * (rng.random((hkv, hd)) < 1 / 16)), dtype)
    v, vh = _round(rng.standard_normal((tk, hkv, hd)), dtype)
    if mutate:
        mutate(k, kh, v, vh)
    if fused:
        qkv = _dev(np.concatenate([qh, kh, vh], 1))
        got = F.prompt_attention_qkv(qkv, h, hkv, _i32(qs), causal, scale, T[out])
    else:
        got = F.prompt_attention(_dev(qh), _dev(kh), _dev(vh), _i32(qs), _i32(ks), causal, scale, T[out])
    assert got.dtype == T[out]
    got = _values(got)
    weps, oeps = _weight_eps(dtype, out), U if out == "float32" else HALF[out]
    sc = hd ** -0.5 if scale is None else scale
    for s in range(len(nq)):
        for j in range(h):
            hk = j // (h // hkv)
            kk, vv = k[ks[s]:ks[s + 1], hk], v[ks[s]:ks[s + 1], hk]
            rows = sorted(set(range(min(nq[s], 3))) | set(range(max(nq[s] - 3, 0), nq[s])) |
                          set(int(i) for i in rng.integers(0, max(nq[s], 1), 12) if nq[s]))
            for i in rows:
                n = max(min(nk[s] - nq[s] + i + 1, nk[s]), 0) if causal else nk[s]
                want, bound = _attend(q[qs[s] + i, j], kk[:n], vv[:n], sc, weps, oeps)
                _check(got[qs[s] + i, j], want, bound, f"sequence {s}, query {i} of {nq[s]}, head {j}, {n} keys")


@pytest.mark.parametrize("dtype,out", [("float16", "float32"), ("float16", "float16"), ("bfloat16", "bfloat16"),
                                       ("bfloat16", "float32")])
@pytest.mark.parametrize("lens,h,hkv,hd", [
    ([1], 1, 1, 64),
    ([1, 2, 31, 32, 33, 63, 64, 65], 4, 2, 64),
    ([127, 0, 128, 129, 1], 4, 1, 128),
    ([257, 300], 2, 2, 40),
    ([200, 7], 6, 2, 256),
    ([150], 5, 5, 72),
    ([90, 1, 130], 8, 1, 200),
    ([50], 3, 1, 8),
    ([700], 2, 1, 96),
])
def test_prompt_attention(gpu, dtype, out, lens, h, hkv, hd):
    for fused in (False, True):
        _prompt(np.random.default_rng(sum(lens) + hd), lens, lens, h, hkv, hd, dtype, out, fused=fused)


@pytest.mark.parametrize("nq,nk,causal", [
    ([5, 100, 1, 64], [69, 300, 500, 64], True),   # what follows a cached prefix
    ([40, 3], [10, 0], True),                      # queries that see no key
    ([70, 1, 33, 6], [129, 200, 1, 0], False),
    ([0, 12], [50, 12], True),
])
def test_prompt_attention_of_other_keys(gpu, nq, nk, causal):
    for dtype, out, hd in (("float16", "float32", 64), ("bfloat16", "bfloat16", 128)):
        _prompt(np.random.default_rng(sum(nk)), nq, nk, 4, 2, hd, dtype, out, causal)


def test_prompt_attention_long(gpu):
    _prompt(np.random.default_rng(3), [2500, 1100], [2500, 1100], 2, 1, 128, "bfloat16", "bfloat16")
    _prompt(np.random.default_rng(4), [2100], [4200], 2, 1, 64, "float16", "float32")


def test_prompt_attention_many_sequences(gpu):
    rng = np.random.default_rng(5)
    lens = [int(n) for n in rng.integers(0, 9, 333)]
    _prompt(rng, lens, lens, 2, 1, 64, "float16", "float16")


@pytest.mark.parametrize("hd", [64, 128, 40])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_prompt_attention_keys_not_seen_never_reach_a_query(gpu, hd, dtype):
    """Infinities and NaN in later keys and values: every query before them is untouched."""
    import lucid_amd as L
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(hd)
    n, h, hkv = 150, 4, 2
    q, qh = _round(rng.standard_normal((n, h, hd)), dtype)
    k, kh = _round(rng.standard_normal((n, hkv, hd)), dtype)
    v, vh = _round(rng.standard_normal((n, hkv, hd)), dtype)
    bad = _round(np.array([np.nan, np.inf, -np.inf]), dtype)[1]
    clean = F.prompt_attention(_dev(qh), _dev(kh), _dev(vh), _i32([0, n]), out_dtype=L.float32).numpy()
    for first in (1, 31, 37, 64, 100, 149):
        kb, vb = kh.copy(), vh.copy()
        kb[first, :, :3], vb[first, 0, 1], vb[first, 1, 5] = bad, bad[1], bad[0]
        got = F.prompt_attention(_dev(qh), _dev(kb), _dev(vb), _i32([0, n]), out_dtype=L.float32).numpy()
        weps = 2.0 ** -15
        assert np.isfinite(got[:first]).all(), first
        assert np.abs(got[:first] - clean[:first]).max() <= 8 * weps * np.abs(v).max()
        assert not np.isfinite(got[first]).all()


@pytest.mark.parametrize("dtype,out", [("float16", "float32"), ("bfloat16", "bfloat16")])
@pytest.mark.parametrize("hd", [64, 128, 40, 192, 256])
def test_prompt_attention_many_workgroups(gpu, dtype, out, hd):
    """The kernel of 128 queries a workgroup, over 64 sequences at most and over more."""
    from lucid_amd import _C

    rng = np.random.default_rng(hd)
    lens = [300, 1, 0, 129, 128, 127, 64, 65, 200] + [int(n) for n in rng.integers(0, 40, 27)]
    _prompt(rng, lens, lens, 32, 4, hd, dtype, out, fused=True)
    assert _C.last_path() == "prompt tile 128"
    more = [int(n) for n in rng.integers(0, 20, 90)] + [260]
    _prompt(rng, more, [n + 30 for n in more], 16, 8, hd, dtype, out)
    assert _C.last_path() == "prompt tile 128"
    _prompt(rng, lens[:9], lens[:9], 2, 1, hd, dtype, out)
    assert _C.last_path() == "prompt tile 64"


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prompt_attention_keys_not_seen_many_workgroups(gpu, hd):
    import lucid_amd as L
    import lucid_amd.nn.functional as F
    from lucid_amd import _C

    rng = np.random.default_rng(hd)
    lens, h = [150] + [3] * 60, 32
    total = sum(lens)
    st = _i32(np.concatenate([[0], np.cumsum(lens)]))
    q, k, v = (rng.standard_normal((total, n, hd)).astype(np.float16) for n in (h, 2, 2))
    clean = F.prompt_attention(_dev(q), _dev(k), _dev(v), st, out_dtype=L.float32).numpy()
    assert _C.last_path() == "prompt tile 128"
    for first in (5, 70, 149):
        vb = v.copy()
        vb[first, 0, 1], vb[first, 1, 2] = np.inf, np.nan
        got = F.prompt_attention(_dev(q), _dev(k), _dev(vb), st, out_dtype=L.float32).numpy()
        ok = np.r_[0:first, 150:total]
        assert np.abs(got[ok] - clean[ok]).max() <= 8 * 2.0 ** -15 * np.abs(v).max()
        assert np.isinf(got[first:150, :h // 2, 1]).all() and np.isnan(got[first:150, h // 2:, 2]).all()
        # the dims beside them are untouched
        assert np.isfinite(np.delete(got, [1, 2], 2)).all()


def test_prompt_attention_of_rows_no_vector_fits(gpu):
    """Rows an odd number of elements apart, and a base that is not 16-byte aligned."""
    from lucid_amd import _C

    rng = np.random.default_rng(2)
    n, h, hd = 70, 2, 40
    for ld, shift in ((h * hd + 3, 0), (h * hd + 8, 1)):
        buf = rng.standard_normal((3, n * ld + 8)).astype(np.float16)
        d = [_dev(b) for b in buf]
        x = [b[shift:shift + n * ld].reshape(n, ld)[:, :h * hd].reshape(n, h, hd).astype(np.float64) for b in buf]
        out, st = _dev(np.zeros((n, h, hd), np.float32)), _i32([0, 30, 70])
        _C.call("lq_prompt_attention", d[0].data_ptr() + 2 * shift, ld, d[1].data_ptr() + 2 * shift, ld,
                d[2].data_ptr() + 2 * shift, ld, _C.F16, st.data_ptr(), st.data_ptr(), 2, n, n, h, h, hd, 1, hd ** -0.5,
                out.data_ptr(), _C.F32, None)
        assert _C.last_path() == "prompt rows"
        got = out.numpy()
        for t in range(n):
            a = 0 if t < 30 else 30
            for j in range(h):
                want, bound = _attend(x[0][t, j], x[1][a:t + 1, j], x[2][a:t + 1, j], hd ** -0.5, 2.0 ** -16, U)
                _check(got[t, j], want, bound, f"row {t}")


def test_prompt_attention_rows_of_no_sequence_are_left(gpu):
    from lucid_amd import _C
    import lucid_amd as L

    rng = np.random.default_rng(0)
    x = _dev(rng.standard_normal((20, 1, 64)).astype(np.float16))
    out = _dev(np.full((20, 1, 64), 5, np.float32))
    st = _i32([3, 9, 9, 15])
    _C.call("lq_prompt_attention", x.data_ptr(), 64, x.data_ptr(), 64, x.data_ptr(), 64, _C.F16, st.data_ptr(),
            st.data_ptr(), 3, 20, 20, 1, 1, 64, 1, 0.125, out.data_ptr(), _C.F32, None)
    got = out.numpy()
    assert (got[:3] == 5).all() and (got[15:] == 5).all() and (got[3:15] != 5).any(axis=(1, 2)).all()
    # starts past the totals: nothing outside is read or written
    st = _i32([0, 4, 50])
    _C.call("lq_prompt_attention", x.data_ptr(), 64, x.data_ptr(), 64, x.data_ptr(), 64, _C.F16, st.data_ptr(),
            st.data_ptr(), 2, 18, 18, 1, 1, 64, 1, 0.125, out.data_ptr(), _C.F32, None)
    assert (out.numpy()[18:] == 5).all() and np.isfinite(out.numpy()).all()


# ------------------------------------------------------------------------------ log probabilities


def _logits(rng, rows, vocab, dtype, masked=False):
    x = rng.standard_normal((rows, vocab)) * 2.5
    x[np.arange(rows), rng.integers(0, vocab, rows)] += 9
    if masked:
        gone = rng.random((rows, vocab)) < 0.7
        gone[:, vocab // 2] = False
        x[gone] = -np.inf
    return _round(x, dtype)


def _order(x, top):
    """Columns of the best values: larger first, NaN above everything, lower index on ties."""
    key = np.where(np.isnan(x), np.inf, x)
    rank = np.lexsort((np.broadcast_to(np.arange(x.shape[1]), x.shape), -key, ~np.isnan(x)), axis=1)
    return rank[:, :top]


def _logprob_want(x, t, top):
    rows, vocab = x.shape
    with np.errstate(all="ignore"):
        m = x.max(1, keepdims=True)
        base = np.where(np.isinf(m) & (m < 0), 0, m)
        e = np.exp(x - base)
        S = e.sum(1)
        lse = base[:, 0] + np.log(S)
        p = e / S[:, None]
        d = np.where(p > 0, x - lse[:, None], 0)
        ent = np.where(S == 0, 0, -(p * d).sum(1))
        spread = (p * np.abs(d)).sum(1)
        ok = (t >= 0) & (t < vocab)
        lp = np.where(ok, x[np.arange(rows), np.clip(t, 0, vocab - 1)] - lse, 0)
        ids = _order(x, top)
        tlp = np.take_along_axis(x, ids, 1) - lse[:, None]
    # e^d is off by (2 |d| + 8) u, the sums by (n / 64 + 32) u
    rel = (2 * (spread + np.abs(ent) + 30) + vocab / 64 + 64) * U
    return lp, ent, lse, tlp, ids, rel


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,vocab,top,masked", [
    (1, 1, 1, False), (1, 1, 0, False), (3, 2, 2, False), (5, 31, 7, True), (4, 64, 64, False), (7, 257, 5, True),
    (3, 1000, 20, False), (9, 1023, 1, True), (2, 4099, 32, True), (8, 32000, 5, False), (3, 50257, 8, True),
    (2, 100003, 64, False), (300, 130, 3, False), (1, 200000, 8, True),
])
def test_token_logprobs(gpu, dtype, rows, vocab, top, masked):
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(rows * 7 + vocab)
    x, xh = _logits(rng, rows, vocab, dtype, masked)
    t = rng.integers(0, vocab, rows).astype(np.int32)
    t[rows // 2:: 3] = -100
    t[1::4] = vocab
    lp, ent, lse, tlp, tid = (a.numpy() for a in F.token_logprobs(_dev(xh), _i32(t), top))
    wlp, went, wlse, wtlp, wids, rel = _logprob_want(x, t, top)
    np.testing.assert_array_equal(tid, wids)
    _check(lse, wlse, rel + 2 * U * np.abs(wlse), "lse")
    _check(ent, went, rel * (2 + np.abs(went)) + 4 * U * np.abs(went), "entropy")
    fin = np.isfinite(wlp)
    np.testing.assert_array_equal(lp[~fin], wlp[~fin])
    _check(lp[fin], wlp[fin], (rel + 2 * U * np.abs(wlse) + U * np.abs(wlp))[fin], "logprobs")
    fin = np.isfinite(wtlp)
    np.testing.assert_array_equal(tlp[~fin], wtlp[~fin])
    bound = np.broadcast_to((rel + 2 * U * np.abs(wlse))[:, None], wtlp.shape)
    _check(tlp[fin], wtlp[fin], bound[fin] + U * np.abs(wtlp[fin]), "alternatives")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [5, 777, 40000])
def test_token_logprobs_ties_and_rows_that_are_not_ordinary(gpu, dtype, vocab):
    """Equal values everywhere (ties to the lowest index), signed zeros, the type's lowest value,
    a row that allows nothing, rows with NaN and +inf."""
    import lucid_amd.nn.functional as F

    top = min(vocab, 9)
    x = np.zeros((9, vocab), np.float32)
    x[1, ::2] = -0.0
    x[2] = -np.inf
    x[3] = -np.inf
    x[3, vocab - 2] = 1.5
    x[4] = np.finfo(np.float32).min if dtype == "float32" else -3.3895314e38  # bfloat16's lowest
    x[5, 3], x[5, vocab - 1] = np.nan, np.nan
    x[6, 2] = np.inf
    x[7] = np.linspace(-4, 4, vocab).astype(np.float32).round(1)
    x[8] = -x[4]
    v, xh = _round(x, dtype)
    t = np.full(9, vocab - 2, np.int32)
    lp, ent, lse, tlp, tid = (a.numpy() for a in F.token_logprobs(_dev(xh), _i32(t), top))
    np.testing.assert_array_equal(tid, _order(v, top))
    tol = (vocab / 64 + 64) * U
    for r in (0, 1):
        assert abs(lse[r] - np.log(vocab)) <= tol * 2 and abs(ent[r] - np.log(vocab)) <= tol * 15
    assert lse[2] == -np.inf and ent[2] == 0 and lp[2] == -np.inf and (tlp[2] == -np.inf).all()
    assert lse[3] == 1.5 and ent[3] == 0 and lp[3] == 0 and (tlp[3, 1:] == -np.inf).all() and tlp[3, 0] == 0
    assert np.isfinite(lse[4]) and abs(ent[4] - np.log(vocab)) <= tol * 15
    assert np.isnan(lse[5]) and np.isnan(lp[5]) and np.isnan(ent[5])
    assert np.isnan(lp[6])
    assert np.isfinite(lse[8]) and abs(ent[8] - np.log(vocab)) <= tol * 15


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("top", [2, 64])
def test_token_logprobs_best_in_few_threads(gpu, dtype, top):
    """All large values within the chunks of eight neighbouring threads: more than are collected at
    once, with and without ties."""
    import lucid_amd.nn.functional as F

    n = 4 if dtype == "float32" else 8
    vocab = 200000
    rng = np.random.default_rng(top)
    chunk = np.arange(vocab) // n % 512
    x = rng.standard_normal((2, vocab)).astype(np.float32)
    large = chunk < 8
    x[0, large] = 50 + rng.permutation(large.sum()) / 8
    x[1, large] = 50
    v, xh = _round(x, dtype)
    lp, ent, lse, tlp, tid = (a.numpy() for a in F.token_logprobs(_dev(xh), _i32([0, 1]), top))
    np.testing.assert_array_equal(tid, _order(v, top))
    want = _logprob_want(v, np.array([0, 1]), top)
    _check(lse, want[2], want[5] + 2 * U * np.abs(want[2]), "lse")


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("rows,vocab,top", [(1, 200003, 64), (3, 70001, 5), (128, 140000, 1), (5, 150001, 0)])
def test_token_logprobs_rows_in_parts(gpu, dtype, rows, vocab, top):
    """Rows shared by several workgroups: odd part boundaries, rows whose allowed tokens lie in one
    part, ties across parts, NaN and a row that allows nothing."""
    import lucid_amd.nn.functional as F
    from lucid_amd import _C

    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((rows, vocab)).astype(np.float32) * 2
    if rows > 2:
        x[0, :-40] = -np.inf       # fewer allowed than alternatives, all at the end
        x[1, ::1000] = 30          # ties in every part
        x[2] = -np.inf
    if rows > 4:
        x[3, vocab // 2] = np.nan
    v, xh = _round(x, dtype)
    t = rng.integers(vocab - 30, vocab, rows).astype(np.int32)
    lp, ent, lse, tlp, tid = (a.numpy() for a in F.token_logprobs(_dev(xh), _i32(t), top))
    assert _C.last_path() == "logprobs parts"
    keep = np.arange(min(rows, 6))
    wlp, went, wlse, wtlp, wids, rel = _logprob_want(v[keep], t[keep], top)
    np.testing.assert_array_equal(tid[keep], wids)
    some = ~np.isneginf(wlse)  # a row that allows nothing is looked at below
    for got, want, bound in ((lse, wlse, rel + 2 * U * np.abs(wlse)), (lp, wlp, rel + 3 * U * np.abs(wlse)),
                             (ent, went, rel * (2 + np.abs(went)) + 4 * U * np.abs(went))):
        fin = np.isfinite(want)
        _check(got[keep][fin & some], want[fin & some], bound[fin & some])
        np.testing.assert_array_equal(np.isnan(got[keep][~fin & some]), np.isnan(want[~fin & some]))
    if rows > 2:
        assert lse[2] == -np.inf and ent[2] == 0 and lp[2] == -np.inf


def test_token_logprobs_one_by_one(gpu):
    """Many rows (one workgroup each) with more candidates above the cut than are collected."""
    import lucid_amd.nn.functional as F
    from lucid_amd import _C

    rows, vocab, top = 130, 200000, 7
    rng = np.random.default_rng(8)
    large = np.arange(vocab) // 8 % 512 < 8
    x = np.zeros((rows, vocab), np.float32)
    x[0, large] = 50 + rng.permutation(large.sum()) % 256 / 4
    x[129, large] = 50
    v, xh = _round(x, "bfloat16")
    _, _, _, tlp, tid = (a.numpy() for a in F.token_logprobs(_dev(xh), _i32(np.zeros(rows)), top))
    assert _C.last_path() == "logprobs rows"
    for r in (0, 1, 129):
        np.testing.assert_array_equal(tid[r], _order(v[r:r + 1], top)[0])


def test_token_logprobs_strided_rows_and_optional_outputs(gpu):
    from lucid_amd import _C

    rng = np.random.default_rng(3)
    rows, vocab = 5, 333
    for dtype, code in (("float32", _C.F32), ("float16", _C.F16), ("bfloat16", _C.BF16)):
        for ld in (333, 334, 340, 701):
            x, xh = _round(rng.standard_normal((rows, ld)) * 3, dtype)
            dx, lse = _dev(xh), _dev(np.zeros(rows, np.float32))
            size = _C.lib().lq_token_logprobs_workspace_size(rows, vocab, 0)
            ws = _dev(np.zeros(max(size, 16), np.uint8))
            _C.call("lq_token_logprobs", dx.data_ptr(), code, ld, rows, vocab, None, 0, None, None, lse.data_ptr(), None,
                    None, ws.data_ptr(), size, None)
            want = _logprob_want(x[:, :vocab], np.zeros(rows, np.int32), 0)
            _check(lse.numpy(), want[2], want[5] + 2 * U * np.abs(want[2]), "lse")


def _grad_want(x, t, lse, ent, g, ge):
    with np.errstate(all="ignore"):
        lp = x - lse[:, None]
        p = np.where(np.isneginf(lse)[:, None], 0, np.exp(lp))
        ok = (t >= 0) & (t < x.shape[1])
        gg = np.where(ok, g, 0)[:, None]
        hot = np.zeros_like(x)
        hot[np.arange(len(t))[ok], t[ok]] = 1
        hot[np.isneginf(lse)] = 0
        inner = np.where(p > 0, lp + ent[:, None], 0)
        want = gg * (hot - p) - ge[:, None] * p * inner
        size = np.abs(gg) * (hot + p) + np.abs(ge)[:, None] * p * (np.where(p > 0, np.abs(lp), 0) + np.abs(ent)[:, None])
        rel = (3 * np.where(p > 0, np.abs(lp), 0) + 16) * U
    return want, size * rel


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,vocab,masked", [(1, 1, False), (3, 2, False), (5, 31, True), (7, 257, True),
                                               (64, 1000, False), (2, 32000, False), (3, 50257, True), (700, 65, True)])
@pytest.mark.parametrize("entropy", [False, True])
def test_token_logprobs_backward(gpu, dtype, rows, vocab, masked, entropy):
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(rows + vocab)
    x, xh = _logits(rng, rows, vocab, dtype, masked)
    if rows > 4:
        x[4], xh[4] = -np.inf, _round(np.full(vocab, -np.inf), dtype)[1]
    t = rng.integers(0, vocab, rows).astype(np.int32)
    t[1::3] = -100
    t[2::5] = vocab
    dx, dt = _dev(xh), _i32(t)
    _, ent, lse, _, _ = F.token_logprobs(dx, dt)
    g, ge = rng.standard_normal(rows).astype(np.float32), (rng.standard_normal(rows) * 0.3).astype(np.float32)
    got = F.token_logprobs_backward(dx, dt, lse, _dev(g), ent if entropy else None, _dev(ge) if entropy else None)
    assert got.dtype == _types()[dtype]
    want, err = _grad_want(x, t, lse.numpy().astype(np.float64), ent.numpy().astype(np.float64), g.astype(np.float64),
                           ge.astype(np.float64) * entropy)
    eps, tiny = (U, 1e-38) if dtype == "float32" else (HALF[dtype], 2.0 ** -25 if dtype == "float16" else 1e-38)
    _check(_values(got), want, err + eps * (np.abs(want) + err) + tiny, "grad")


def test_token_logprobs_backward_against_differences(gpu):
    """The gradient against central differences of the float64 forward."""
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(11)
    rows, vocab = 4, 23
    x, xh = _logits(rng, rows, vocab, "float32")
    x[1, 5] = xh[1, 5] = -np.inf
    t = np.array([3, 7, -100, 22], np.int32)
    g, ge = rng.standard_normal(rows), rng.standard_normal(rows)
    dx, dt = _dev(xh), _i32(t)
    _, ent, lse, _, _ = F.token_logprobs(dx, dt)
    got = F.token_logprobs_backward(dx, dt, lse, _dev(g.astype(np.float32)), ent, _dev(ge.astype(np.float32))).numpy()

    def loss(y):
        lp, e = _logprob_want(y, t, 0)[:2]
        return g * lp + ge * e

    h = 1e-5
    for j in range(vocab):
        up, dn = x.copy(), x.copy()
        up[:, j] += h
        dn[:, j] -= h
        with np.errstate(invalid="ignore"):
            diff = (loss(up) - loss(dn)) / (2 * h)
        # h^2 of the third derivative (below 10) and the differences' own rounding, beside float32's
        assert np.abs(got[:, j] - diff).max() <= 1e-9 + 2e-15 * 50 / h + 64 * U * 10


def test_token_logprobs_backward_strided_and_in_place(gpu):
    from lucid_amd import _C
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(9)
    rows, vocab = 6, 1001
    for dtype, code in (("float32", _C.F32), ("bfloat16", _C.BF16)):
        _, xh = _logits(rng, rows, vocab, dtype)
        t, g = _i32(rng.integers(0, vocab, rows)), _dev(rng.standard_normal(rows).astype(np.float32))
        _, ent, lse, _, _ = F.token_logprobs(_dev(xh), t)
        want = F.token_logprobs_backward(_dev(xh), t, lse, g, ent, g).numpy()
        for ldx, ldg in ((1001, 1003), (1010, 1001), (1024, 1024)):
            wide = np.zeros((rows, ldx), xh.dtype)
            wide[:, :vocab] = xh
            dx = _dev(wide)
            out = _dev(np.zeros((rows, ldg), xh.dtype))
            for dst, ld in ((out, ldg), (dx, ldx)):  # beside, then in place
                _C.call("lq_token_logprobs_backward", dx.data_ptr(), code, ldx, rows, vocab, t.data_ptr(),
                        lse.data_ptr(), ent.data_ptr(), g.data_ptr(), g.data_ptr(), dst.data_ptr(), ld, None)
                got = dst.numpy()
                np.testing.assert_array_equal(got[:, :vocab], want)
                assert (got[:, vocab:] == np.zeros((), xh.dtype)).all()


# ------------------------------------------------------------------------------ together


def test_cache_classes_and_graph_replay(gpu):
    """PageTable / PagedKVCache through appends, growth and release; the step's launches captured
    in a graph and replayed after the table grew, against the eager results each time."""
    import lucid_amd as L
    from lucid_amd import _C
    from lucid_amd.bench_configs import Graph
    from lucid_amd.nn.generation import PagedKVCache, PageTable

    rng = np.random.default_rng(6)
    B, h, hkv, hd = 3, 4, 2, 64
    pt = PageTable(B, 12, 8, 40)
    cache = PagedKVCache(pt, hkv, hd, L.float16)
    dense = [np.zeros((0, 2, hkv, hd), np.float32) for _ in range(B)]

    def feed(counts):
        pt.grow(counts)
        x = rng.standard_normal((sum(counts), 2, hkv, hd)).astype(np.float16)
        cache.append(_dev(x[:, 0]), _dev(x[:, 1]), _i32(np.concatenate([[0], np.cumsum(counts)])))
        at = 0
        for b, n in enumerate(counts):
            dense[b] = np.concatenate([dense[b], x[at:at + n]])
            at += n

    def check(q, got):
        for b in range(B):
            for j in range(h):
                want, bound = _attend(q[b, j].astype(np.float64), dense[b][:, 0, j // 2].astype(np.float64),
                                      dense[b][:, 1, j // 2].astype(np.float64), hd ** -0.5, 2.0 ** -16, U)
                _check(got[b, j], want, bound, f"{b} {j}")

    feed([9, 1, 0])
    q = rng.standard_normal((B, h, hd)).astype(np.float16)
    check(q, cache.attend(_dev(q), out_dtype=L.float32).numpy())
    # one step captured: append of one token per sequence, then attention
    kq, kk, kv = (_dev(np.zeros((B, n, hd), np.float16)) for n in (h, hkv, hkv))
    out = _dev(np.zeros((B, h, hd), np.float32))
    size = _C.lib().lq_paged_attention_workspace_size(B, h, hkv, hd, 40)
    ws = _dev(np.zeros(max(size, 16), np.uint8))
    stream = ctypes.c_void_p()
    _C.call("lq_stream_create", ctypes.byref(stream))

    def step(st):
        cache.append(kk, kv, stream=st)
        _C.call("lq_paged_attention", kq.data_ptr(), _C.F16, h * hd, B, h, hkv, hd, cache.k.data_ptr(),
                cache.v.data_ptr(), _C.F16, None, None, pt.pages, pt.page, pt.table.data_ptr(), pt.table.shape[1],
                pt.lengths.data_ptr(), 40, hd ** -0.5, out.data_ptr(), _C.F32, ws.data_ptr(), size, st)

    _C.synchronize()
    graph = Graph(step, stream)
    for it in range(12):
        pt.grow([1, 1, 1])
        x = rng.standard_normal((3, B, h, hd)).astype(np.float16)
        for dst, a in ((kq, x[0]), (kk, x[1, :, :hkv]), (kv, x[2, :, :hkv])):
            a = np.ascontiguousarray(a)
            _C.call("lq_memcpy_h2d", dst.data_ptr(), a.ctypes.data, a.nbytes, None)
        graph.launch()
        _C.call("lq_stream_synchronize", stream)
        for b in range(B):
            dense[b] = np.concatenate([dense[b], np.stack([x[1, b, :hkv], x[2, b, :hkv]])[None].astype(np.float32)])
        check(x[0], out.numpy())
        np.testing.assert_array_equal(cache.attend(kq, out_dtype=L.float32, max_length=40).numpy(), out.numpy())
    with pytest.raises(MemoryError):
        pt.grow([19, 18, 18])  # 40 positions at most each, 12 pages in all
    with pytest.raises(ValueError):
        pt.grow([100, 0, 0])
    before = pt.host_lengths()
    pt.release(0)
    dense[0] = dense[0][:0]
    assert pt.host_lengths()[0] == 0 and (pt.host_lengths()[1:] == before[1:]).all()
    feed([30, 0, 1])  # the released pages serve again
    q = rng.standard_normal((B, h, hd)).astype(np.float16)
    check(q, cache.attend(_dev(q), out_dtype=L.float32).numpy())
    del graph
    _C.call("lq_stream_destroy", stream)


def test_ops_replayed_from_a_graph(gpu):
    """Prompt attention, log probabilities and their gradient recorded once and replayed with new
    inputs, eager work of the same ops and synchronizations between the replays."""
    import lucid_amd as L
    import lucid_amd.nn.functional as F
    from lucid_amd.graphs import CapturedForward

    rng = np.random.default_rng(31)
    st, t = _i32([0, 50, 130]), _i32([3, -100, 7, 500])
    g = _dev(rng.standard_normal(4).astype(np.float32))

    def fn(qkv, x):
        lp, ent, lse, top, ids = F.token_logprobs(x, t, 6)
        return (F.prompt_attention_qkv(qkv, 4, 2, st, out_dtype=L.float32), lp, ent, lse, top, ids,
                F.token_logprobs_backward(x, t, lse, g, ent, g))

    make = lambda: (rng.standard_normal((130, 8, 64)).astype(np.float16),  # noqa: E731
                    (rng.standard_normal((4, 3001)) * 3).astype(np.float32))
    a, b = make()
    qkv, x = _dev(a), _dev(b)
    cap = CapturedForward(fn, qkv, x)
    for _ in range(4):
        a, b = make()
        cap.load(a, b)
        got = [y.numpy() for y in cap()]
        want = [y.numpy() for y in fn(_dev(a), _dev(b))]
        L.synchronize()
        for y, z in zip(got, want):
            np.testing.assert_array_equal(y, z)


def test_ops_on_a_stream_of_their_own(gpu):
    """Every op on a created stream gives the bits of the default stream."""
    from lucid_amd import _C
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(12)
    stream = ctypes.c_void_p()
    _C.call("lq_stream_create", ctypes.byref(stream))
    qkv = _dev(rng.standard_normal((100, 8, 64)).astype(np.float16))
    st = _i32([0, 60, 100])
    x, t = _dev(rng.standard_normal((4, 999)).astype(np.float32)), _i32([1, 2, 3, 4])
    g = _dev(np.ones(4, np.float32))
    k, v = (_dev(rng.standard_normal((8, 2, 16, 64)).astype(np.float16)) for _ in range(2))
    q = _dev(rng.standard_normal((2, 4, 64)).astype(np.float16))
    table, lens = _i32([[0, 1, 2, 3], [4, 5, 6, 7]]), _i32([64, 50])
    _C.synchronize()
    got = []
    for s in (None, stream):
        a = F.prompt_attention_qkv(qkv, 4, 2, st, stream=s)
        b = F.paged_attention(q, k, v, table, lens, 64, stream=s)
        c = F.token_logprobs(x, t, 5, stream=s)
        d = F.token_logprobs_backward(x, t, c[2], g, c[1], g, stream=s)
        _C.call("lq_stream_synchronize", s)
        got.append([y.numpy() for y in (a, b, *c, d)])
    for y, z in zip(*got):
        np.testing.assert_array_equal(y, z)
    _C.call("lq_stream_destroy", stream)
