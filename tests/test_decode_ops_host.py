"""The decode step's operators without a GPU: what the entry points refuse before any launch, calls that have nothing
to do, the Python layer's checks."""

from __future__ import annotations

import numpy as np
import pytest

from _decode import bf16_toward, quantize4
from lucid_amd import _C
import lucid_amd.nn.functional as F

P = 4096  # a non-NULL pointer that no refused call reads
NAN, INF = float("nan"), float("inf")

RMS = dict(x=P, type=_C.F16, ldx=64, res=2 * P, ldres=64, sum=P, ldsum=64, gamma=P, gtype=_C.F32, eps=1e-5, rows=3, D=64,
           y=3 * P, ytype=_C.F32, ldy=64, stream=None)
RMSQ = dict(x=P, type=_C.BF16, ldx=64, res=2 * P, ldres=64, sum=5 * P, ldsum=70, gamma=None, gtype=0, eps=1e-5, rows=3,
            D=64, codes=3 * P, ldc=64, scales=4 * P, stream=None)
ROTARY = dict(q=P, ldq=384, k=2 * P, v=3 * P, ldkv=384, src=_C.F16, tokens=4, starts=P, seqs=2, H=2, Hkv=2, hd=64,
              angles=P, positions=9, rot=64, interleaved=0, table=P, stride=3, lengths=P, qo=P, ldqo=384, ko=2 * P,
              ldko=384, qtype=_C.F16, kp=5 * P, vp=6 * P, cache=_C.F16, ks=None, vs=None, pages=8, page=16, stream=None)
PAGED4 = dict(q=P, type=_C.F16, ldq=256, B=2, H=4, hkv=2, hd=64, k=P, v=P, cache=_C.U4, ks=P, vs=P, pages=8,
              page=16, table=P, stride=3, lengths=P, longest=48, scale=0.125, out=P, out_type=_C.F32, ws=P, size=1 << 40,
              stream=None)
APPEND4 = dict(k=P, v=P, src=_C.F32, ld=128, tokens=4, starts=P, seqs=2, hkv=2, hd=64, table=P, stride=3, lengths=P,
               kp=P, vp=P, cache=_C.U4, ks=P, vs=P, pages=8, page=16, stream=None)
VERIFY = dict(x=P, type=_C.F32, ld=100, lse=P, d=P, ldd=100, dlse=P, drafts=P, starts=P, seqs=2, rows=7, vocab=100, au=P,
              su=P, tokens=P, accepted=P, ws=P, size=1 << 40, stream=None)

REFUSALS = [
    ("lq_rms_norm", RMS, c) for c in (
        dict(type=_C.I8), dict(ytype=_C.I8), dict(gtype=_C.I8), dict(rows=-1), dict(D=0), dict(D=-1), dict(ldx=63),
        dict(ldres=63), dict(ldsum=63), dict(ldy=63), dict(eps=0.0), dict(eps=-1.0), dict(eps=NAN), dict(eps=INF),
        dict(x=None), dict(y=None), dict(sum=P, ldx=80), dict(sum=2 * P, ldsum=80), dict(y=P), dict(y=2 * P),
        dict(sum=3 * P))
] + [
    ("lq_rms_norm_quantize", RMSQ, c) for c in (
        dict(type=_C.I8), dict(gamma=P, gtype=_C.U4), dict(ldc=63), dict(codes=None), dict(scales=None), dict(eps=0.0),
        dict(codes=P), dict(D=1 << 31, ldx=1 << 32, ldc=1 << 32, ldres=1 << 32, ldsum=1 << 32))
] + [
    ("lq_paged_kv_append_rotary", ROTARY, c) for c in (
        dict(src=_C.I8), dict(qtype=_C.F32), dict(cache=_C.BF16), dict(cache=_C.F32), dict(cache=_C.I8),
        dict(cache=_C.U4, ks=P), dict(tokens=-1), dict(seqs=-1), dict(H=-1), dict(Hkv=0), dict(hd=0), dict(ldq=127),
        dict(ldkv=127), dict(ldqo=127), dict(ldko=127), dict(rot=63), dict(rot=66), dict(rot=-2), dict(positions=-1),
        dict(page=0), dict(pages=-1), dict(stride=-1), dict(q=None), dict(k=None), dict(v=None), dict(angles=None),
        dict(table=None), dict(lengths=None), dict(qo=None), dict(kp=None), dict(vp=None), dict(starts=None),
        dict(src=_C.F32), dict(ldqo=400), dict(ldko=400), dict(ko=3 * P), dict(tokens=1 << 31), dict(pages=1 << 31),
        dict(hd=264, ldq=4096, ldkv=4096, ldqo=4096, ldko=4096), dict(cache=_C.U4, hd=48, rot=48, ks=P, vs=P),
        dict(cache=_C.U4, ks=P, vs=P, kp=P + 2))
] + [
    ("lq_paged_attention", PAGED4, c) for c in (
        dict(ks=None), dict(vs=None), dict(hd=48), dict(hd=288, ldq=4096), dict(type=_C.F32), dict(k=P + 8),
        dict(ks=P + 4), dict(vs=P + 2), dict(out_type=_C.BF16), dict(scale=0.0), dict(longest=5000, size=100))
] + [
    ("lq_paged_kv_append", APPEND4, c) for c in (
        dict(ks=None), dict(vs=None), dict(hd=40), dict(hd=288, ld=4096), dict(src=_C.I8), dict(ld=127), dict(k=None),
        dict(kp=None), dict(starts=None))
] + [
    ("lq_verify_drafts", VERIFY, c) for c in (
        dict(type=_C.I8), dict(seqs=-1), dict(rows=-1), dict(vocab=0), dict(vocab=1 << 31, ld=1 << 32, ldd=1 << 32),
        dict(ld=99), dict(ldd=99), dict(x=None), dict(lse=None), dict(d=None), dict(dlse=None), dict(drafts=None),
        dict(starts=None), dict(au=None), dict(su=None), dict(tokens=None), dict(accepted=None), dict(ws=None),
        dict(ws=P + 8), dict(size=8))
]


@pytest.mark.parametrize("name,args,change", REFUSALS, ids=lambda v: str(v) if isinstance(v, dict) and len(v) < 6 else
                         v if isinstance(v, str) else "")
def test_bad_arguments_are_refused_before_any_launch(name, args, change):
    assert set(change) <= set(args)
    with pytest.raises(_C.LucidError, match=name):
        _C.call(name, *{**args, **change}.values())


@pytest.mark.parametrize("name,args,change", [
    ("lq_rms_norm", RMS, dict(rows=0, x=None, y=None)),
    ("lq_rms_norm_quantize", RMSQ, dict(rows=0, x=None, codes=None)),
    ("lq_paged_kv_append_rotary", ROTARY, dict(tokens=0, q=None, k=None)),
    ("lq_paged_kv_append_rotary", ROTARY, dict(seqs=0, starts=None, tokens=0)),
    ("lq_paged_kv_append_rotary", ROTARY, dict(pages=0, kp=None, vp=None, H=0, ko=None, ldko=0)),
    ("lq_paged_kv_append", APPEND4, dict(tokens=0, k=None)),
    ("lq_paged_kv_append", APPEND4, dict(pages=0, kp=None, vp=None)),
    ("lq_paged_attention", PAGED4, dict(B=0, q=None, out=None)),
    ("lq_verify_drafts", VERIFY, dict(seqs=0, starts=None)),
])
def test_empty_calls_succeed_without_a_launch(name, args, change):
    _C.call(name, *{**args, **change}.values())


def test_workspace_sizes():
    lib = _C.lib()
    assert lib.lq_verify_drafts_workspace_size(0, 100) == 0 and lib.lq_verify_drafts_workspace_size(3, 0) == 0
    assert lib.lq_verify_drafts_workspace_size(3, 1) > 0


def test_cpu_tensors_are_refused():
    import lucid_amd as L

    x = L.tensor(np.zeros((2, 64), np.float32))
    i = L.tensor(np.zeros(2, np.int32))
    u = L.tensor(np.zeros(2, np.float32))
    q = L.tensor(np.zeros((2, 3, 64), np.float16))
    for call in (lambda: F.rms_norm(x), lambda: F.rms_norm_quantize(x), lambda: F.verify_drafts(x, u, i, i, u, u),
                 lambda: F.rotary_qkv(q, 1, 1, x, i),
                 lambda: F.paged_kv_append_rotary(q, q, q, x, q, q, i, i),
                 lambda: F.paged_kv_append_rotary_qkv(q, 1, x, q, q, i, i)):
        with pytest.raises(L.LucidError, match="GPU tensors"):
            call()


@pytest.mark.parametrize("args", [(0, 64), (4, 0), (4, 3), (4, 64, 0.0), (4, 64, 10000.0, -1.0)])
def test_angles_of_bad_sizes(args):
    with pytest.raises(ValueError, match="rotary_angles"):
        F.rotary_angles(*args)


def test_cache_types():
    from lucid_amd.nn.generation import PagedKVCache

    for dt in (np.float32, np.uint8, np.int32):
        with pytest.raises(TypeError, match="PagedKVCache"):
            PagedKVCache(None, 1, 64, dt)
    for hd in (48, 0, -32):
        with pytest.raises(ValueError, match="multiples of 32"):
            PagedKVCache(None, 1, hd, "uint4")


def test_four_bit_rule_covers_its_group():
    """Every value lies within half a scale, and 2^-7 of it, of what its code stands for."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((4000, 32)) * rng.choice([1e-20, 1, 1e20], (4000, 1))
         + rng.choice([0, 5, -300], (4000, 1))).astype(np.float32)
    codes, scale, bias = quantize4(x, 32)
    back = codes * scale.astype(np.float64) + bias
    assert (np.abs(back - x) <= scale * (0.5 + 2.0 ** -7) + np.abs(x) * 2.0 ** -23).all()
    assert (bias[:, 0] <= x.min(1)).all() and (bf16_toward(bias, True) == bias).all()
