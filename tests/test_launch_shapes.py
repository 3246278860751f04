"""Calls of more workgroups than one dimension of a launch takes (2^32 work items): the shapes on the host, the
serving ops on the GPU at the first sizes past it."""

from __future__ import annotations

import os
import shutil
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_every_workgroup_has_a_place(tmp_path):
    exe = tmp_path / "launch_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", os.path.join(ROOT, "lucid_amd", "csrc"),
                    os.path.join(ROOT, "tests", "native", "launch_check.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stderr
    assert out.stdout.strip() == "ok"


def _dev(a):
    import lucid_amd as L

    return L.tensor(np.ascontiguousarray(a), device="gpu")


@pytest.fixture(autouse=True)
def _memory_goes_back():
    yield
    from lucid_amd import _C

    if _C._lib is not None and _C.device_count():
        _C.call("lq_empty_cache")


@pytest.mark.gpu
def test_log_probabilities_of_many_rows(gpu):
    import lucid_amd.nn.functional as F

    rows = (1 << 26) + 3  # 64 threads to a row
    x = np.zeros((rows, 2), np.float16)
    x[:, 1] = np.arange(rows) % 7
    lp, _, lse, _, ids = F.token_logprobs(_dev(x), _dev(np.zeros(rows, np.int32)), 1)
    want = np.log1p(np.exp(np.arange(7.0)))
    at = np.arange(rows) % 7
    # values to 6, sums of two exponentials: a few roundings of float32
    assert (np.abs(lse.numpy() - want[at].astype(np.float32)) <= 40 * 2.0 ** -24).all()
    assert (np.abs(lp.numpy() + want[at].astype(np.float32)) <= 40 * 2.0 ** -24).all()
    assert (ids.numpy()[:, 0] == (at > 0)).all()


@pytest.mark.gpu
def test_gradient_of_many_rows_of_unlike_strides(gpu):
    from lucid_amd import _C

    rows = (1 << 24) + 5
    x = np.zeros((rows, 3), np.float16)
    x[:, 1], x[:, 2] = np.arange(rows) % 5, -np.inf
    lse = np.log1p(np.exp(np.arange(5.0))).astype(np.float32)[np.arange(rows) % 5]
    dx, t, dl, g = (_dev(a) for a in (x, np.zeros(rows, np.int32), lse, np.ones(rows, np.float32)))
    out = _dev(np.zeros((rows, 4), np.float16))
    _C.call("lq_token_logprobs_backward", dx.data_ptr(), _C.F16, 3, rows, 3, t.data_ptr(), dl.data_ptr(), None,
            g.data_ptr(), None, out.data_ptr(), 4, None)
    got = out.numpy()
    p = 1 / (1 + np.exp(np.arange(5.0)))
    want = np.stack([1 - p, p - 1, 0 * p, 0 * p], 1)[np.arange(rows) % 5]
    assert (np.abs(got - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -20).all()


@pytest.mark.gpu
@pytest.mark.parametrize("cache,tokens,hd", [("int8", (1 << 24) + 9, 8), ("float16", (1 << 24) + 9, 3),
                                             ("int8", (1 << 26) + 1, 1), ("float16", (1 << 26) + 5, 8)])
def test_append_of_many_tokens(gpu, cache, tokens, hd):
    import lucid_amd as L
    import lucid_amd.nn.functional as F

    page = 1 << 20
    pages = -(-tokens // page)
    x = (np.arange(tokens * hd, dtype=np.int32) % 113 + 1).astype(np.float16).reshape(tokens, 1, hd)
    k, v = (L.empty((pages, 1, page, hd), np.dtype(cache), "gpu") for _ in range(2))
    scales = {}
    if cache == "int8":
        scales = {n: L.empty((pages, 1, page), L.float32, "gpu") for n in ("k_scale", "v_scale")}
    src = _dev(x)
    F.paged_kv_append(src, src, k, v, _dev(np.arange(pages, dtype=np.int32)[None]), _dev(np.array([tokens], np.int32)),
                      _dev(np.array([0, tokens], np.int32)), **scales)
    for name, t in (("k", k), ("v", v)):
        got = t.numpy().reshape(-1, hd)[:tokens]
        if cache == "int8":
            top = x.astype(np.float32).reshape(tokens, hd).max(1)
            scale = scales[name + "_scale"].numpy().reshape(-1)[:tokens]
            np.testing.assert_array_equal(scale, top / np.float32(127))
            inv = np.float32(127) / top
            np.testing.assert_array_equal(got, np.rint(x[:, 0].astype(np.float32) * inv[:, None]).astype(np.int8))
        else:
            np.testing.assert_array_equal(got, x[:, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["float16", "int8"])
def test_paged_attention_of_many_heads(gpu, cache):
    """One position each: the output is the value, bit for bit."""
    import lucid_amd as L
    import lucid_amd.nn.functional as F

    B, heads, hd = 1025, 32768, 8
    values = (np.arange(heads * hd).reshape(1, heads, 1, hd) % 127).astype(cache)
    one = {n: _dev(np.ones((1, heads, 1), np.float32)) for n in ("k_scale", "v_scale")} if cache == "int8" else {}
    kv = _dev(values)
    q = _dev(np.zeros((B, heads, hd), np.float16))
    lens = np.ones(B, np.int32)
    lens[-2] = 0
    out = F.paged_attention(q, kv, kv, _dev(np.zeros((B, 1), np.int32)), _dev(lens), 1, **one)
    got = out.numpy()
    assert got.dtype == L.float16 and (got[-2] == 0).all()
    got[-2] = values[0, :, 0]
    assert (got == values[0, :, 0].astype(np.float16)).all()


@pytest.mark.gpu
def test_prompt_attention_of_many_heads(gpu):
    import lucid_amd.nn.functional as F

    seqs, heads, hd = 513, 32768, 8
    v = (np.arange(seqs * hd).reshape(seqs, 1, hd) % 127).astype(np.float16)
    got = F.prompt_attention(_dev(np.zeros((seqs, heads, hd), np.float16)), _dev(v), _dev(v),
                             _dev(np.arange(seqs + 1, dtype=np.int32))).numpy()
    assert (got == v).all()
