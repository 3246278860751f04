"""Rotation and append on the GPU, bit for bit: float32 products and sums operation by operation, one rounding to
each place; the rows of int8 and 4-bit pages by their documented rules of the rotated float32 values."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from _decode import Pages, dev, i32, pack4, quantize4, rotate, rounded, types, values

pytestmark = pytest.mark.gpu


def _same(got, want):
    """Equal values, NaN and NaN alike."""
    return np.array_equal(got, want, equal_nan=True)


class Cache:
    """Pages filled with a mark, on the device and as the append should leave them."""

    def __init__(self, pages, hkv, hd, kind):
        shape = (pages.pages, hkv, pages.page, hd)
        self.kind, self.hd = kind, hd
        if kind == "uint4":
            self.want = {c: np.full((*shape[:3], hd // 2), 0x77, np.uint8) for c in "kv"}
            self.meta = {c: np.full((*shape[:3], 2, n), 7, np.float32) for c, n in (("k", hd // 32), ("v", 1))}
        elif kind == "int8":
            self.want = {c: np.full(shape, 77, np.int8) for c in "kv"}
            self.meta = {c: np.full(shape[:3], 7, np.float32) for c in "kv"}
        else:
            self.want, self.meta = {c: np.full(shape, 77, np.float32) for c in "kv"}, {}
        self.dev = {c: dev(rounded(a, kind)[1] if kind in ("float16", "bfloat16") else a) for c, a in self.want.items()}
        self.scale = {c: dev(rounded(a, "bfloat16")[1] if kind == "uint4" else a) for c, a in self.meta.items()}

    def put(self, c, page, slot, row):
        """Rows [heads, hd] of float32 values at one place."""
        if self.kind == "uint4":
            codes, scale, bias = quantize4(row, 32 if c == "k" else self.hd)
            self.want[c][page, :, slot] = pack4(codes)
            self.meta[c][page, :, slot] = np.stack([scale, bias], -2)
        elif self.kind == "int8":
            top = np.abs(row).max(-1)
            with np.errstate(divide="ignore"):
                inv = np.float32(127) / top
            self.want[c][page, :, slot] = np.where(top[:, None] > 0, np.rint(row * np.where(top > 0, inv, 0)[:, None]), 0)
            self.meta[c][page, :, slot] = top / np.float32(127)
        else:
            self.want[c][page, :, slot] = rounded(row, self.kind)[0]

    def check(self):
        for c, t in self.dev.items():
            assert _same(values(t) if self.kind in ("float16", "bfloat16") else t.numpy(), self.want[c]), c
        for c, t in self.scale.items():
            assert _same(values(t), self.meta[c]), c

    def args(self):
        return dict(k_pages=self.dev["k"], v_pages=self.dev["v"], k_scale=self.scale.get("k"), v_scale=self.scale.get("v"))


def _positions(lens, new):
    seq = np.repeat(np.arange(len(lens)), new)
    pos = np.concatenate([np.arange(n - m, n) for n, m in zip(lens, new)] + [np.zeros(0, int)]).astype(int)
    return seq, pos


CASES = [  # lens, new, heads, kv heads, hd, rot, page
    ([5, 1, 40, 17], [5, 1, 7, 0], 4, 2, 64, 64, 16),
    ([3, 0, 8], [1, 1, 1], 3, 1, 96, 96, 8),     # a step, one sequence of length 0
    ([300], [300], 32, 8, 128, 128, 64),
    ([20, 70], [4, 3], 6, 2, 256, 64, 1),        # part of the dims
    ([9, 30, 2], [9, 2, 2], 5, 5, 32, 32, 5),
    ([33, 8], [33, 8], 2, 1, 128, 0, 16),        # no dims
    ([12], [12], 3, 3, 64, 22, 4),               # partners that no vector fits
]


@pytest.mark.parametrize("kind", ["float16", "bfloat16", "int8", "uint4"])
@pytest.mark.parametrize("src", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("lens,new,h,hkv,hd,rot,page", CASES)
def test_rotated_append(gpu, kind, src, interleaved, lens, new, h, hkv, hd, rot, page):
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng([hd, rot, page, len(src), len(kind)])
    out = kind if kind in ("float16", "bfloat16") else rng.choice(["float16", "bfloat16"])
    tokens = sum(new)
    x, host = rounded(rng.standard_normal((tokens, h + 2 * hkv, hd)) * rng.choice([0.1, 1, 30], (tokens, 1, 1)), src)
    angles = rng.standard_normal((max(lens), rot)).astype(np.float32) if rot else np.zeros((max(lens), 0), np.float32)
    pages = Pages(rng, lens, page)
    seq, pos = _positions(lens, new)
    y = rotate(x[:, :h + hkv], pos, angles, interleaved) if rot else x[:, :h + hkv]
    if rot == 0:
        angles_dev = dev(np.zeros((max(lens), 0), np.float32))
    else:
        angles_dev = dev(angles)
    step = all(n == 1 for n in new)
    starts = None if step else i32(np.cumsum([0] + new))
    cache = Cache(pages, hkv, hd, kind)
    for t in range(tokens):
        if pos[t] < 0:
            continue
        page_no, slot = pages.at(seq[t], pos[t])
        cache.put("k", page_no, slot, y[t, h:])
        cache.put("v", page_no, slot, x[t, h + hkv:])
    q, k = F.paged_kv_append_rotary(dev(host[:, :h]), dev(host[:, h:h + hkv]), dev(host[:, h + hkv:]), angles_dev,
                                    table=i32(pages.table), lengths=i32(lens), starts=starts, interleaved=interleaved,
                                    q_dtype=types()[out], **cache.args())
    cache.check()
    want = rounded(y, out)[0]
    assert _same(values(q), want[:, :h]) and _same(values(k), want[:, h:])
    if src == out:  # a fused projection's rows, in place
        fused, again = dev(host), Cache(pages, hkv, hd, kind)
        F.paged_kv_append_rotary_qkv(fused, h, angles_dev, table=i32(pages.table), lengths=i32(lens), starts=starts,
                                     interleaved=interleaved, **again.args())
        back = values(fused)
        assert _same(back[:, :h + hkv], want) and _same(back[:, h + hkv:], x[:, h + hkv:])
        again.want, again.meta = cache.want, cache.meta
        again.check()
        fused = dev(host)
        if rot:
            F.rotary_qkv(fused, h, hkv, angles_dev, i32(lens), starts, interleaved)
            assert _same(values(fused)[:, :h + hkv], want)


@pytest.mark.parametrize("src", ["float32", "bfloat16"])
@pytest.mark.parametrize("hd", [32, 64, 96, 128, 160, 256])
def test_plain_append_to_four_bits(gpu, src, hd):
    """lq_paged_kv_append: 4-bit rows of values as they come, among them equal ones, far ones, tiny ones."""
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(hd)
    lens, hkv, page = [37, 9], 3, 8
    x = rng.standard_normal((46, 2, hkv, hd)) * rng.choice([1e-3, 1, 100], (46, 1, 1, 1))
    x[0], x[1], x[2] = 0, 1.001, -3.0
    x[3] += 1000
    x[4] *= 1e-36
    x[5] = rng.standard_normal((2, hkv, hd)) * 1e-42 if src == "float32" else 0
    x[6, :, :, ::2] = 1e37
    x[7] = np.where(np.arange(hd) % 2, 1, -1) * 3e38  # a width that passes float32
    x[8, 0, 0, 5], x[9, 1, 1, 7], x[10, 0, 2, hd - 1] = np.nan, np.inf, -np.inf
    with np.errstate(over="ignore"):
        x, host = rounded(x, src)
    pages = Pages(rng, lens, page)
    cache = Cache(pages, hkv, hd, "uint4")
    seq, pos = _positions(lens, lens)
    for t in range(46):
        for i, c in enumerate("kv"):
            cache.put(c, *pages.at(seq[t], pos[t]), x[t, i])
    F.paged_kv_append(dev(host[:, 0]), dev(host[:, 1]), table=i32(pages.table), lengths=i32(lens),
                      starts=i32([0, 37, 46]), **cache.args())
    cache.check()


@pytest.mark.parametrize("hd,rot", [(64, 64), (64, 20)])
def test_tokens_without_a_place(gpu, hd, rot):
    """Positions outside the angles: NaN rows, nothing appended.  Bad pages and tables that are too short: rotated, not
    appended.  Rows of no sequence: as they were."""
    import lucid_amd.nn.functional as F
    from lucid_amd import _C

    rng = np.random.default_rng(rot)
    lens, new, page = [6, 12, 3, 0], [3, 4, 2, 1], 4
    angles = rng.standard_normal((10, rot)).astype(np.float32)  # positions 10 and 11 of sequence 1 have none
    pages = Pages(rng, lens, page, stride=3)
    pages.table[2, 0] = pages.pages  # sequence 2's page lies outside the pool
    pages.table[0, 1] = -1           # positions 4 and 5 of sequence 0
    tokens = 14                      # two rows before the first start, two past the last
    starts = np.cumsum([2] + new)
    x, host = rounded(rng.standard_normal((tokens, 4, hd)), "float16")
    cache = Cache(pages, 1, hd, "float16")
    fused = dev(host)
    F.paged_kv_append_rotary_qkv(fused, 2, dev(angles), table=i32(pages.table), lengths=i32(lens), starts=i32(starts),
                                 **cache.args())
    seq, pos = _positions(lens, new)
    pos[-1] = -1
    y = rotate(x[2:12, :3], pos, angles, False)
    for t in range(10):
        if 0 <= pos[t] < 10 and seq[t] != 2 and not (seq[t] == 0 and pos[t] >= 4):
            cache.put("k", *pages.at(seq[t], pos[t]), y[t, 2:])
            cache.put("v", *pages.at(seq[t], pos[t]), x[2 + t, 3:])
    cache.check()
    back = values(fused)
    want = x.copy()
    want[2:12, :3] = rounded(y, "float16")[0]
    assert _same(back, want)


@pytest.mark.parametrize("kind", ["bfloat16", "uint4"])
def test_unaligned_rows(gpu, kind):
    """Rows and tables of angles that 16-byte accesses do not fit: the bits of the aligned call."""
    import lucid_amd as L
    from lucid_amd import _C

    rng = np.random.default_rng(1)
    lens, h, hkv, hd, rot, page = [9, 4], 3, 2, 64, 32, 4
    ld = (h + 2 * hkv) * hd + 3
    x, host = rounded(rng.standard_normal((13, ld)), "bfloat16")
    angles = rng.standard_normal((9, rot)).astype(np.float32)
    pages = Pages(rng, lens, page)
    seq, pos = _positions(lens, lens)
    heads = x[:, :ld - 3].reshape(13, -1, hd)
    y = rotate(heads[:, :h + hkv], pos, angles, True)
    cache = Cache(pages, hkv, hd, kind)
    for t in range(13):
        cache.put("k", *pages.at(seq[t], pos[t]), y[t, h:])
        cache.put("v", *pages.at(seq[t], pos[t]), heads[t, h + hkv:])
    src, ang = dev(host), dev(np.concatenate([[0], angles.ravel()]).astype(np.float32))
    qo = L.empty((13, h * hd + 1), L.bfloat16, "gpu")
    p = src.data_ptr()
    a, table, lengths, starts = cache.args(), i32(pages.table), i32(lens), i32([0, 9, 13])
    _C.call("lq_paged_kv_append_rotary", p, ld, p + 2 * h * hd, p + 2 * (h + hkv) * hd, ld, _C.BF16, 13, starts.data_ptr(),
            2, h, hkv, hd, ang.data_ptr() + 4, 9, rot, 1, table.data_ptr(), table.shape[1], lengths.data_ptr(),
            qo.data_ptr(), h * hd + 1, None, 0, _C.BF16, a["k_pages"].data_ptr(), a["v_pages"].data_ptr(),
            _C.U4 if kind == "uint4" else _C.BF16, a["k_scale"].data_ptr() if a["k_scale"] is not None else None,
            a["v_scale"].data_ptr() if a["v_scale"] is not None else None, pages.pages, page, None)
    assert _C.last_path() == "rotary single"
    cache.check()
    assert _same(values(qo)[:, :h * hd].reshape(13, h, hd), rounded(y[:, :h], "bfloat16")[0])


def test_angles(gpu):
    import lucid_amd.nn.functional as F

    a = F.rotary_angles(70000, 64, 500000.0, 4.0).numpy()
    p, i = np.array([0, 1, 69999])[:, None], np.arange(32)[None]
    w = p / 4.0 * 500000.0 ** (-2.0 * i / 64)
    assert np.array_equal(a[[0, 1, 69999]], np.concatenate([np.cos(w), np.sin(w)], 1).astype(np.float32))


def test_on_a_stream_and_from_a_graph(gpu):
    """The same rows and pages from a created stream, and from a graph replayed with new contents."""
    import lucid_amd as L
    import lucid_amd.nn.functional as F
    from lucid_amd import _C
    from lucid_amd.graphs import CapturedForward

    rng = np.random.default_rng(2)
    lens, h, hkv, hd = [17, 5, 64], 4, 2, 64
    pages = Pages(rng, lens, 16)
    table, lengths, angles = i32(pages.table), i32(lens), F.rotary_angles(64, hd)

    def host():
        return rng.standard_normal((3, h + 2 * hkv, hd)).astype(np.float32)

    def call(x, cache, stream=None):
        q, k = F.paged_kv_append_rotary(x[0], x[1], x[2], angles, table=table, lengths=lengths, stream=stream, **cache.args())
        return q

    def parts(x):
        return [dev(x[:, :h]), dev(x[:, h:h + hkv]), dev(x[:, h + hkv:])]

    first, second = Cache(pages, hkv, hd, "uint4"), Cache(pages, hkv, hd, "uint4")
    x = host()
    want = call(parts(x), first).numpy()
    st = ctypes.c_void_p()
    _C.call("lq_stream_create", ctypes.byref(st))
    t = parts(x)
    _C.synchronize()
    q = call(t, second, st)
    _C.call("lq_stream_synchronize", st)
    assert np.array_equal(q.numpy(), want) and np.array_equal(first.dev["k"].numpy(), second.dev["k"].numpy())
    _C.call("lq_stream_destroy", st)
    third, held = Cache(pages, hkv, hd, "uint4"), parts(x)
    cap = CapturedForward(lambda *a: call(a, third), *held)
    for _ in range(3):
        x = host()
        cap.load(x[:, :h], x[:, h:h + hkv], x[:, h + hkv:])
        got = cap().numpy()
        eager = Cache(pages, hkv, hd, "uint4")
        assert np.array_equal(got, call(parts(x), eager).numpy())
        for c in "kv":
            assert np.array_equal(third.dev[c].numpy(), eager.dev[c].numpy())
            assert np.array_equal(values(third.scale[c]), values(eager.scale[c]), equal_nan=True)
