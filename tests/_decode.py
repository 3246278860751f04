"""Plain restatements of the decode step's operators, for their tests: numpy, float32 operation by operation where
the result is compared bit for bit, float64 where it is compared within a bound."""

from __future__ import annotations

import numpy as np

U = 2.0 ** -24  # half a step of float32
HALF = {"float32": U, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def types():
    import lucid_amd as L

    return {"float32": L.float32, "float16": L.float16, "bfloat16": L.bfloat16, "int8": L.int8}


def rounded(a, dtype):
    """(values as float32, host array in the storage type) of float32 ``a`` rounded to ``dtype``."""
    import lucid_amd as L

    a = np.asarray(a, np.float32)
    if dtype == "bfloat16":
        bits = L.bf16_from_f32(a)
        return L.bf16_to_f32(bits), bits
    with np.errstate(over="ignore"):
        h = a.astype(np.float16 if dtype == "float16" else np.float32)
    return h.astype(np.float32), h


def values(t):
    """A device tensor's values, float32."""
    import lucid_amd as L

    a = t.numpy()
    return L.bf16_to_f32(a) if t.dtype == L.bfloat16 else a.astype(np.float32)


def dev(a):
    import lucid_amd as L

    return L.tensor(np.ascontiguousarray(a), device="gpu")


def i32(a):
    return dev(np.asarray(a, np.int32))


def bf16_toward(x, up):
    """float32 values as the bfloat16 at or above (below) them, as float32."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    away = (x >= 0) if up else (x < 0)
    return ((u + np.where(away, 0xffff, 0).astype(np.uint64)) & np.uint64(0xffff0000)).astype(np.uint32).view(np.float32)


def quantize4(x, step):
    """(codes [..., hd], scale [..., hd / step], bias) of float32 rows, by the documented rule in float32."""
    x = np.asarray(x, np.float32)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // step, step)
    with np.errstate(all="ignore"):
        bias = bf16_toward(g.min(-1), False)
        scale = bf16_toward((g.max(-1) - bias) * (np.float32(1) / np.float32(15)), True)
        inv = np.float32(1) / scale
        none = ~(inv < np.inf)
        scale, inv = np.where(none, 0, scale).astype(np.float32), np.where(none, 0, inv).astype(np.float32)
        codes = np.rint((g - bias[..., None]) * inv[..., None]).clip(0, 15)
        bad = ~np.isfinite(g).all(-1) | ~(g.max(-1) - bias < np.inf)
    scale[bad] = bias[bad] = np.nan
    codes[bad] = 0
    return codes.reshape(x.shape).astype(np.uint8), scale, bias


def pack4(codes):
    return codes[..., 0::2] | codes[..., 1::2] << 4


def unpack4(packed):
    return np.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1], -1)


def values4(codes, scale, bias):
    """What codes stand for, float64."""
    g = codes.astype(np.float64).reshape(*scale.shape, codes.shape[-1] // scale.shape[-1])
    return (g * scale[..., None].astype(np.float64) + bias[..., None].astype(np.float64)).reshape(codes.shape)


def rotate(x, pos, angles, interleaved):
    """Float32 rows [tokens, heads, hd] turned by their positions' angles, operation by operation; NaN without."""
    rot = angles.shape[1]
    half = rot // 2
    ok = (pos >= 0) & (pos < angles.shape[0])
    a = angles[np.where(ok, pos, 0)][:, None]
    c, s = a[..., :half], a[..., half:]
    y = x.copy()
    p, q = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, half), slice(half, rot))
    u, w = x[..., p], x[..., q]
    y[..., p], y[..., q] = u * c - w * s, w * c + u * s
    y[~ok] = np.nan
    return y


def close(got, want, bound, what=""):
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} outside the bound, worst "
                           f"{np.nanmax(np.abs(got - want) / bound):.3g} times, NaN {np.isnan(got).sum()}")


class Pages:
    """A shuffled page table; entries past a sequence's pages hold anything."""

    def __init__(self, rng, lens, page, spare=3, stride=None):
        used = [-(-max(n, 0) // page) for n in lens]
        self.lens, self.page, self.pages = list(lens), page, sum(used) + spare
        ids = rng.permutation(self.pages)[:sum(used)]
        self.table = rng.integers(-5, self.pages + 5, (len(lens), max(used + [1]) if stride is None else stride))
        self.table = self.table.astype(np.int32)
        at = 0
        for b, u in enumerate(used):
            self.table[b, :u] = ids[at:at + u]
            at += u

    def at(self, b, pos):
        """(page numbers, slots) of positions of sequence b."""
        return self.table[b, np.asarray(pos) // self.page], np.asarray(pos) % self.page
