"""How exact the attention kernels' outputs are as a whole, by the 2-norm of their error against float64.

A worst-case bound of one output grows with the head dim and the keys and hides a lost term of the weights;
the norm over many outputs does not, since roundings are independent.  u = 2^-24.  For queries and keys of
unit variance a score stays below 8 in log2 units, where float32 rounds it to 4 u at most; its sum of
products, its exponential and the sum of the weights add as much again, so a float32 output is off by
less than 16 u = 2^-20 as a whole.  Weights of 16 significant bits would leave 2^-18 or more.

A 16-bit output is rounded once; where the weights keep more bits than it does, the error is that of the
rounding alone (a tenth more allowed)."""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F32_BOUND = 2.0 ** -20


def _round(a, dtype):
    import lucid_amd as L

    a = np.asarray(a, np.float32)
    if dtype == "bfloat16":
        bits = L.bf16_from_f32(a)
        return L.bf16_to_f32(bits).astype(np.float64), bits
    h = a.astype(dtype)
    return h.astype(np.float64), h


def _dev(a):
    import lucid_amd as L

    return L.tensor(np.ascontiguousarray(a), device="gpu")


def _types():
    import lucid_amd as L

    return {"float32": L.float32, "float16": L.float16, "bfloat16": L.bfloat16}


def _values(t):
    import lucid_amd as L

    a = t.numpy()
    return L.bf16_to_f32(a).astype(np.float64) if t.dtype == L.bfloat16 else a.astype(np.float64)


def _off(got, want):
    return np.linalg.norm(got - want) / np.linalg.norm(want)


def _attend(q, k, v):
    """q [h, hd] over k / v [n, hkv, hd] in float64."""
    h, hkv = q.shape[0], k.shape[1]
    out = np.empty_like(q)
    for j in range(h):
        s = k[:, j // (h // hkv)] @ q[j] * q.shape[1] ** -0.5
        w = np.exp(s - s.max())
        out[j] = w @ v[:, j // (h // hkv)] / w.sum()
    return out


@pytest.mark.parametrize("dtype,cache", [("float16", "float16"), ("bfloat16", "bfloat16"), ("float16", "int8"),
                                         ("bfloat16", "int8")])
@pytest.mark.parametrize("hd", [64, 72, 128, 256])
@pytest.mark.parametrize("n,bound", [(40, 40), (700, 700), (700, 5000)])
def test_paged_attention(gpu, dtype, cache, hd, n, bound):
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(hd + n)
    h, hkv, page = 16, 2, 16
    pages = -(-n // page)
    scales, kv = {}, {}
    for name in ("k", "v"):
        x = rng.standard_normal((pages, hkv, page, hd))
        if cache == "int8":
            top = np.abs(x).max(-1)
            codes, sc = np.rint(x * (127 / top)[..., None]).astype(np.int8), (top / 127).astype(np.float32)
            kv[name] = codes * sc[..., None].astype(np.float64), codes
            scales[name + "_scale"] = _dev(sc)
        else:
            kv[name] = _round(x, cache)
    q, qh = _round(rng.standard_normal((1, h, hd)), dtype)
    k, v = (kv[c][0].transpose(0, 2, 1, 3).reshape(-1, hkv, hd)[:n] for c in ("k", "v"))
    want = _attend(q[0], k, v)
    for out in ("float32", dtype):
        got = _values(F.paged_attention(_dev(qh), _dev(kv["k"][1]), _dev(kv["v"][1]),
                                        _dev(np.arange(pages, dtype=np.int32)[None]), _dev(np.array([n], np.int32)), bound,
                                        out_dtype=_types()[out], **scales))[0]
        allowed = F32_BOUND if out == "float32" else 1.1 * _off(_round(want, dtype)[0], want)
        assert _off(got, want) <= allowed, (out, _off(got, want), allowed)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("hd", [64, 72, 128, 192, 256])
@pytest.mark.parametrize("heads,many", [(4, False), (64, True)])
def test_prompt_attention_float32(gpu, dtype, hd, heads, many):
    """Both kernels: 64 queries a workgroup and 128."""
    import lucid_amd as L
    import lucid_amd.nn.functional as F
    from lucid_amd import _C

    rng = np.random.default_rng(hd)
    lens = [200, 3, 90] if not many else [200, 3, 90] + [130] * 14
    total, starts = sum(lens), np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    q, qh = _round(rng.standard_normal((total, heads, hd)), dtype)
    k, kh = _round(rng.standard_normal((total, 2, hd)), dtype)
    v, vh = _round(rng.standard_normal((total, 2, hd)), dtype)
    got = F.prompt_attention(_dev(qh), _dev(kh), _dev(vh), _dev(starts), out_dtype=L.float32).numpy().astype(np.float64)
    assert _C.last_path() == ("prompt tile 128" if many else "prompt tile 64")
    rows = [0, 1, 63, 64, 130, 199, 201, 202, 203, 250, 292]
    for t in rows:
        a = starts[np.searchsorted(starts, t, side="right") - 1]
        want = _attend(q[t], k[a:t + 1], v[a:t + 1])
        assert _off(got[t], want) <= F32_BOUND, (t, _off(got[t], want))
