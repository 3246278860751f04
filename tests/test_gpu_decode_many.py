"""Norm, rotation, 4-bit append and verification of more rows than one dimension of a launch takes workgroups: rows repeat
with a period of 7, and every row must have what a call of seven rows gives it."""

from __future__ import annotations

import numpy as np
import pytest

from _decode import dev, i32

pytestmark = pytest.mark.gpu
MANY = (1 << 22) + 3


@pytest.fixture(autouse=True)
def _memory_goes_back():
    yield
    from lucid_amd import _C

    if _C._lib is not None and _C.device_count():
        _C.call("lq_empty_cache")


def _repeat(a, n):
    return a[np.arange(n) % 7]


def _same(got, few):
    got, few = (np.ascontiguousarray(a).view(np.uint8).reshape(len(a), -1) for a in (got, few))
    assert all((got[i::7] == few[i]).all() for i in range(7))


@pytest.mark.parametrize("dim,rows", [(2, 4 * MANY), (8, 4 * MANY), (1026, MANY)])
def test_norm(gpu, dim, rows):
    import lucid_amd.nn.functional as F

    x = np.random.default_rng(dim).standard_normal((7, dim)).astype(np.float16)
    few, many = (F.rms_norm_quantize(dev(_repeat(x, n))) for n in (7, rows))
    for f, m in zip(few, many):
        _same(m.numpy(), f.numpy())


def test_rotation_and_append(gpu):
    import lucid_amd.nn.functional as F
    import lucid_amd as L

    rng = np.random.default_rng(1)
    qkv, angles = rng.standard_normal((7, 3, 32)).astype(np.float16), F.rotary_angles(8, 32)
    out = []
    for n in (7, MANY):
        t, lengths = dev(_repeat(qkv, n)), i32(1 + np.arange(n) % 7)
        F.rotary_qkv(t, 1, 1, angles, lengths)
        pages, meta = (L.empty((n, 1, 1, 16), np.uint8, "gpu") for _ in "kv"), L.bfloat16
        k, v = pages
        ks, vs = L.empty((n, 1, 1, 2, 1), meta, "gpu"), L.empty((n, 1, 1, 2, 1), meta, "gpu")
        F.paged_kv_append_qkv(t, 1, k, v, i32(np.arange(n)[:, None]), i32(np.ones(n)), k_scale=ks, v_scale=vs)
        out.append([a.numpy() for a in (t, k, v, ks, vs)])
    for few, many in zip(*out):
        _same(many, few)


@pytest.mark.parametrize("vocab", [3, 4097])
def test_verification(gpu, vocab):
    import lucid_amd.nn.functional as F

    n = MANY if vocab == 3 else (1 << 21) + 3  # two workgroups to a sequence of 4097
    rng = np.random.default_rng(2)
    x, u = rng.standard_normal((7, vocab)).astype(np.float16), rng.random(7).astype(np.float32)
    out = []
    for m in (7, n):
        logits = dev(_repeat(x, m))
        _, _, lse, _, _ = F.token_logprobs(logits, i32(np.zeros(m)))
        out.append([a.numpy() for a in F.verify_drafts(logits, lse, i32(np.zeros(m)), i32(np.arange(m + 1)),
                                                       dev(np.zeros(m, np.float32)), dev(_repeat(u, m)))])
        del logits
    for few, many in zip(*out):
        _same(many, few)
