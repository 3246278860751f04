"""Serving ops without a GPU: the places of tokens and positions, the entry points' refusals (all
before any HIP call), the Python layer's argument checks."""

from __future__ import annotations

import os
import shutil
import subprocess

import numpy as np
import pytest

from lucid_amd import _C
import lucid_amd.nn.functional as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 4096  # a non-NULL pointer that no refused call reads


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_places_of_tokens_and_positions(tmp_path):
    exe = tmp_path / "place_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", os.path.join(ROOT, "lucid_amd", "csrc"),
                    os.path.join(ROOT, "tests", "native", "place_check.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stderr
    assert out.stdout.strip() == "ok"


APPEND = dict(k=P, v=P, src=_C.F32, ld=128, tokens=4, starts=P, seqs=2, hkv=2, hd=64, table=P, stride=3, lengths=P,
              kp=P, vp=P, cache=_C.F16, ks=None, vs=None, pages=8, page=16, stream=None)
PAGED = dict(q=P, type=_C.F16, ldq=256, B=2, H=4, hkv=2, hd=64, k=P, v=P, cache=_C.F16, ks=None, vs=None, pages=8,
             page=16, table=P, stride=3, lengths=P, longest=48, scale=0.125, out=P, out_type=_C.F32, ws=P, size=1 << 40,
             stream=None)
PROMPT = dict(q=P, ldq=256, k=P, ldk=128, v=P, ldv=128, type=_C.F16, qs=P, ks=P, seqs=2, tq=9, tk=9, H=4, hkv=2, hd=64,
              causal=1, scale=0.125, out=P, out_type=_C.F16, stream=None)
LOGP = dict(x=P, type=_C.F32, ld=100, rows=3, vocab=100, targets=P, top=5, lp=P, ent=P, lse=P, tlp=P, tid=P, ws=P,
            size=1 << 40, stream=None)
GRAD = dict(x=P, type=_C.F32, ld=100, rows=3, vocab=100, targets=P, lse=P, ent=P, g=P, ge=P, grad=2 * P, ldg=100,
            stream=None)

REFUSALS = [
    ("lq_paged_kv_append", APPEND, change) for change in (
        dict(src=_C.I8), dict(cache=_C.F32), dict(cache=_C.I8), dict(cache=_C.I8, ks=P), dict(ld=127), dict(tokens=-1),
        dict(seqs=-1), dict(hkv=0), dict(hd=0), dict(page=0), dict(pages=-1), dict(stride=-1), dict(k=None),
        dict(v=None), dict(table=None), dict(lengths=None), dict(kp=None), dict(vp=None), dict(starts=None),
        dict(tokens=1 << 31), dict(pages=1 << 31))
] + [
    ("lq_paged_attention", PAGED, change) for change in (
        dict(type=_C.F32), dict(cache=_C.BF16), dict(cache=_C.I8), dict(out_type=_C.BF16), dict(B=-1), dict(H=3),
        dict(hkv=0), dict(hd=60), dict(hd=264, ldq=4096), dict(hd=0), dict(ldq=255), dict(page=0), dict(pages=-1),
        dict(stride=-1), dict(longest=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
        dict(scale=float("inf")), dict(q=None), dict(k=None), dict(v=None), dict(table=None), dict(lengths=None),
        dict(out=None))
] + [
    ("lq_prompt_attention", PROMPT, change) for change in (
        dict(type=_C.F32), dict(out_type=_C.BF16), dict(seqs=-1), dict(tq=-1), dict(tk=-1), dict(H=3), dict(hkv=0),
        dict(hd=60), dict(hd=0), dict(hd=264, ldq=4096, ldk=4096, ldv=4096), dict(ldq=255), dict(ldk=127),
        dict(ldv=127), dict(scale=0.0), dict(scale=float("nan")), dict(q=None), dict(k=None), dict(v=None),
        dict(qs=None), dict(ks=None), dict(out=None), dict(tq=1 << 31))
] + [
    ("lq_token_logprobs", LOGP, change) for change in (
        dict(type=_C.I8), dict(rows=-1), dict(vocab=0), dict(ld=99), dict(top=-1), dict(top=65), dict(top=101, vocab=100),
        dict(x=None), dict(targets=None), dict(tlp=None), dict(tid=None), dict(vocab=3, top=4))
] + [
    ("lq_token_logprobs_backward", GRAD, change) for change in (
        dict(type=_C.I8), dict(rows=-1), dict(vocab=0), dict(ld=99), dict(ldg=99), dict(x=None), dict(targets=None),
        dict(lse=None), dict(g=None), dict(grad=None), dict(ent=None), dict(grad=P, ldg=101))
]


@pytest.mark.parametrize("name,args,change", REFUSALS, ids=lambda v: str(v) if isinstance(v, dict) and len(v) < 6 else
                         v if isinstance(v, str) else "")
def test_bad_arguments_are_refused_before_any_launch(name, args, change):
    assert set(change) <= set(args)
    with pytest.raises(_C.LucidError, match=name):
        _C.call(name, *{**args, **change}.values())


@pytest.mark.parametrize("name,args,change", [
    ("lq_paged_kv_append", APPEND, dict(tokens=0, k=None, v=None)),
    ("lq_paged_kv_append", APPEND, dict(seqs=0, starts=None, tokens=0)),
    ("lq_paged_kv_append", APPEND, dict(pages=0, kp=None, vp=None)),
    ("lq_paged_attention", PAGED, dict(B=0, q=None, out=None)),
    ("lq_prompt_attention", PROMPT, dict(seqs=0)),
    ("lq_prompt_attention", PROMPT, dict(tq=0, q=None, out=None)),
    ("lq_token_logprobs", LOGP, dict(rows=0, x=None)),
    ("lq_token_logprobs_backward", GRAD, dict(rows=0, x=None)),
])
def test_empty_calls_succeed_without_a_launch(name, args, change):
    _C.call(name, *{**args, **change}.values())


def test_cpu_tensors_are_refused():
    import lucid_amd as L

    x = L.tensor(np.zeros((2, 10), np.float32))
    t = L.tensor(np.zeros(2, np.int32))
    with pytest.raises(L.LucidError, match="GPU tensors"):
        F.token_logprobs(x, t)
    q = L.tensor(np.zeros((2, 2, 64), np.float16))
    with pytest.raises(L.LucidError, match="GPU tensors"):
        F.prompt_attention(q, q, q, t)
