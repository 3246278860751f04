"""How the positions of many sequences are shared among workgroups, over every kind of cache.

With queries of zero every weight is the same power of two, and values are integers from -8 to 7: all sums are exact, and an
output is the mean of its sequence's values to within the division (a reciprocal and a product: 3 half steps of
float32).  A position that is lost, counted twice or given to another sequence shows."""

from __future__ import annotations

import numpy as np
import pytest

from _decode import Pages, U, close, dev, i32, pack4, rounded, types, values

pytestmark = pytest.mark.gpu


def _lens(rng, seqs, longest):
    lens = rng.integers(0, 300, seqs)
    lens[rng.random(seqs) < 0.2] = 0
    lens[rng.integers(seqs)] = 1
    lens[rng.integers(seqs)] = longest
    return [int(n) for n in lens]


@pytest.mark.parametrize("cache", ["float16", "bfloat16", "int8", "uint4"])
@pytest.mark.parametrize("seqs,longest,heads,kv_heads", [
    (1, 9001, 2, 1),
    (2, 5000, 4, 4),
    (63, 3000, 2, 2),
    (64, 12000, 2, 1),
    (65, 3000, 2, 2),
    (300, 2500, 1, 1),
    (1100, 4000, 20, 1),
])
def test_every_position_once(gpu, cache, seqs, longest, heads, kv_heads):
    import lucid_amd.nn.functional as F

    hd, page = 64, 16
    rng = np.random.default_rng([seqs, heads])
    lens = _lens(rng, seqs, longest)
    p = Pages(rng, lens, page)
    shape = (p.pages, kv_heads, page)
    codes = rng.integers(0, 16, (*shape, hd))
    if cache == "uint4":
        meta = lambda n: dev(rounded(np.broadcast_to(np.float32([[1], [-8]]), (*shape, 2, n)).copy(), "bfloat16")[1])
        kw = dict(k_pages=dev(pack4(codes.astype(np.uint8))), v_pages=dev(pack4(codes.astype(np.uint8))),
                  k_scale=meta(hd // 32), v_scale=meta(1))
    elif cache == "int8":
        one = np.ones(shape, np.float32)
        kw = dict(k_pages=dev((codes - 8).astype(np.int8)), v_pages=dev((codes - 8).astype(np.int8)),
                  k_scale=dev(one), v_scale=dev(one))
    else:
        rows = rounded(codes - 8.0, cache)[1]
        kw = dict(k_pages=dev(rows), v_pages=dev(rows))
    dtype = cache if cache == "bfloat16" else "float16"
    q = dev(rounded(np.zeros((seqs, heads, hd)), dtype)[1])
    got = values(F.paged_attention(q, table=i32(p.table), lengths=i32(lens), max_length=longest,
                                   out_dtype=types()["float32"], **kw))
    want = np.zeros((seqs, heads, hd))
    for b, n in enumerate(lens):
        if n > 0:
            at, slot = p.at(b, np.arange(n))
            want[b] = np.repeat((codes[at, :, slot] - 8).mean(0), heads // kv_heads, 0)
    close(got.astype(np.float64), want, 3 * U * np.abs(want), f"{seqs} sequences")
