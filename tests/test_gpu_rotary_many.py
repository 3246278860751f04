"""Rotation and append of prompts long enough for the kernel that takes four rows a lane, bit for bit against the numpy
restatement: rows of queries, keys and values in one wave, partners exchanged between lanes and loaded, heads that leave lanes
and whole rounds without a row."""

from __future__ import annotations

import numpy as np
import pytest

from _decode import Pages, dev, i32, rotate, rounded, types, values
from test_gpu_rotary import Cache, _positions, _same

pytestmark = pytest.mark.gpu

CASES = [  # lens, new, heads, kv heads, hd, rot, page
    ([700, 900, 0, 3], [600, 897, 1, 2], 32, 8, 128, 128, 64),  # 16 rows of 48 a wave
    ([1500, 200], [1500, 150], 28, 7, 96, 96, 16),              # six lanes between partners: loaded; lanes past the row
    ([1700], [1650], 33, 5, 64, 64, 8),                         # 43 rows, 32 a wave: the last round in part
    ([500, 2600], [400, 2500], 16, 4, 256, 64, 32),             # part of the dims, 8 rows a wave
    ([1200, 1300], [1200, 1300], 20, 4, 256, 96, 128),          # part of the dims, partners loaded
    ([2200], [2200], 24, 4, 32, 32, 5),                         # lanes past the row of 32
    ([1600], [1600], 32, 8, 128, 0, 16),                        # no dims
]


@pytest.mark.parametrize("kind", ["float16", "bfloat16", "int8", "uint4"])
@pytest.mark.parametrize("src", ["float32", "bfloat16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("lens,new,h,hkv,hd,rot,page", CASES)
def test_rotated_append(gpu, kind, src, interleaved, lens, new, h, hkv, hd, rot, page):
    import lucid_amd.nn.functional as F
    from lucid_amd import _C

    rng = np.random.default_rng([hd, rot, page, len(src), len(kind)])
    out = "float16" if kind == "float16" else "bfloat16"
    tokens = sum(new)
    assert tokens * (h + 2 * hkv) >= 65536 and h + 2 * hkv > 4  # the case is what it is meant to be
    x, host = rounded(rng.standard_normal((tokens, h + 2 * hkv, hd)) * rng.choice([0.1, 1, 30], (tokens, 1, 1)), src)
    angles = rng.standard_normal((max(lens), rot)).astype(np.float32)
    pages = Pages(rng, lens, page)
    seq, pos = _positions(lens, new)
    y = rotate(x[:, :h + hkv], pos, angles, interleaved) if rot else x[:, :h + hkv]
    cache = Cache(pages, hkv, hd, kind)
    for t in np.nonzero(pos >= 0)[0]:
        place = pages.at(seq[t], pos[t])
        cache.put("k", *place, y[t, h:])
        cache.put("v", *place, x[t, h + hkv:])
    given = dict(table=i32(pages.table), lengths=i32(lens), starts=i32(np.cumsum([0] + new)), interleaved=interleaved)
    q, k = F.paged_kv_append_rotary(dev(host[:, :h]), dev(host[:, h:h + hkv]), dev(host[:, h + hkv:]), dev(angles),
                                    q_dtype=types()[out], **given, **cache.args())
    assert _C.last_path() == "rotary four rows"
    cache.check()
    want = rounded(y, out)[0]
    assert _same(values(q), want[:, :h]) and _same(values(k), want[:, h:])
    if src == out:  # a fused projection's rows, in place
        fused, again = dev(host), Cache(pages, hkv, hd, kind)
        F.paged_kv_append_rotary_qkv(fused, h, dev(angles), **given, **again.args())
        assert _C.last_path() == "rotary four rows"
        back = values(fused)
        assert _same(back[:, :h + hkv], want) and _same(back[:, h + hkv:], x[:, h + hkv:])
        again.want, again.meta = cache.want, cache.meta
        again.check()
        if rot:
            fused = dev(host)
            F.rotary_qkv(fused, h, hkv, dev(angles), given["lengths"], given["starts"], interleaved)
            assert _C.last_path() == "rotary four rows"
            back = values(fused)
            assert _same(back[:, :h + hkv], want) and _same(back[:, h + hkv:], x[:, h + hkv:])


@pytest.mark.parametrize("src", ["float32", "bfloat16"])
@pytest.mark.parametrize("hd,hkv", [(64, 40), (96, 18), (128, 20), (256, 9)])
def test_plain_append_to_four_bits(gpu, src, hd, hkv):
    import lucid_amd.nn.functional as F
    from lucid_amd import _C

    rng = np.random.default_rng(hd)
    lens = [1500, 400]
    x, host = rounded(rng.standard_normal((4000 if hkv < 10 else 1900, 2, hkv, hd)), src)
    lens = [len(x) - 400, 400]
    assert len(x) * 2 * hkv >= 65536
    pages = Pages(rng, lens, 16)
    cache = Cache(pages, hkv, hd, "uint4")
    seq, pos = _positions(lens, lens)
    for t in range(len(x)):
        for i, c in enumerate("kv"):
            cache.put(c, *pages.at(seq[t], pos[t]), x[t, i])
    F.paged_kv_append(dev(host[:, 0]), dev(host[:, 1]), table=i32(pages.table), lengths=i32(lens),
                      starts=i32([0, lens[0], len(x)]), **cache.args())
    assert _C.last_path() == "rotary four rows"
    cache.check()


def test_tokens_without_a_place(gpu):
    """Positions past the angles, bad pages, rows of no sequence, among many that have a place; rows and pages beside them
    stay as they were."""
    import lucid_amd.nn.functional as F
    from lucid_amd import _C

    rng = np.random.default_rng(0)
    lens, new, h, hkv, hd, page = [900, 800, 5], [850, 700, 5], 30, 8, 64, 16
    angles = rng.standard_normal((890, hd)).astype(np.float32)  # the last ten positions of sequence 0 have none
    pages = Pages(rng, lens, page)
    pages.table[1, 20], pages.table[1, 21] = pages.pages, -7
    tokens, first = sum(new) + 9, 4
    x, host = rounded(rng.standard_normal((tokens, h + 2 * hkv, hd)), "bfloat16")
    seq, pos = _positions(lens, new)
    y = rotate(x[first:first + sum(new), :h + hkv], pos, angles, False)
    cache = Cache(pages, hkv, hd, "int8")
    for t in range(sum(new)):
        if pos[t] < 890 and not (seq[t] == 1 and pos[t] // page in (20, 21)):
            cache.put("k", *pages.at(seq[t], pos[t]), y[t, h:])
            cache.put("v", *pages.at(seq[t], pos[t]), x[first + t, h + hkv:])
    fused = dev(host)
    F.paged_kv_append_rotary_qkv(fused, h, dev(angles), table=i32(pages.table), lengths=i32(lens),
                                 starts=i32(first + np.cumsum([0] + new)), **cache.args())
    assert _C.last_path() == "rotary four rows"
    cache.check()
    want = x.copy()
    want[first:first + sum(new), :h + hkv] = rounded(y, "bfloat16")[0]
    assert _same(values(fused), want)
