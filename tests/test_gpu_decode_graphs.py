"""A decode step's operators in one chain: eager, on a created stream, and from two captured graphs that are replayed in turn
with eager work between."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from _decode import dev, i32

pytestmark = pytest.mark.gpu
H, HKV, HD, VOCAB = 4, 2, 64, 9001


class Step:
    """Sequences that take one token each: norm, rotated append, attention, verification of what was drafted."""

    def __init__(self, lens, page, seed):
        import lucid_amd.nn.functional as F
        from lucid_amd.nn.generation import PagedKVCache, PageTable

        self.lens, self.longest, seqs = lens, max(lens), len(lens)
        rng = np.random.default_rng(seed)
        each = [-(-n // page) for n in lens]
        table = PageTable(seqs, sum(each), page, self.longest)
        table.grow(np.array(lens))
        self.cache = PagedKVCache(table, HKV, HD, "uint4")
        self.angles = F.rotary_angles(self.longest, HD)
        # what the earlier tokens left, the last one's place with them
        rows = dev(rng.standard_normal((sum(lens), H + 2 * HKV, HD)).astype(np.float16))
        self.cache.append_rotary_qkv(rows, H, self.angles, i32(np.cumsum([0] + lens)))
        self.starts, self.drafts = i32(2 * np.arange(seqs + 1)), i32(rng.integers(0, VOCAB, 2 * seqs))
        self.seqs = seqs

    def inputs(self, rng):
        n = self.seqs
        return [rng.standard_normal((n, H * HD)).astype(np.float32), rng.standard_normal((n, H * HD)).astype(np.float32),
                rng.standard_normal((n, H + 2 * HKV, HD)).astype(np.float16),
                (3 * rng.standard_normal((2 * n, VOCAB))).astype(np.float16), rng.random(2 * n).astype(np.float32),
                rng.random(n).astype(np.float32)]

    def __call__(self, x, res, qkv, logits, accept, sample, stream=None):
        import lucid_amd as L
        import lucid_amd.nn.functional as F

        codes, scales, total = F.rms_norm_quantize(x, residual=res, stream=stream)
        y, _ = F.rms_norm(x, residual=res, out_dtype=L.bfloat16, stream=stream)
        q, k, v = qkv
        q, _ = self.cache.append_rotary(q, k, v, self.angles, stream=stream)
        out = self.cache.attend(q, out_dtype=L.float32, max_length=self.longest, stream=stream)
        _, _, lse, _, _ = F.token_logprobs(logits, self.drafts, stream=stream)
        tokens, kept = F.verify_drafts(logits, lse, self.drafts, self.starts, accept, sample, stream=stream)
        return codes, scales, total, y, out, tokens, kept

    def host(self, args):
        """Inputs as the call takes them: the projection in three tensors."""
        x, res, qkv, *rest = args
        return [x, res, qkv[:, :H], qkv[:, H:H + HKV], qkv[:, H + HKV:], *rest]

    def run(self, x, res, q, k, v, *rest, stream=None):
        return self(x, res, (q, k, v), *rest, stream=stream)

    def eager(self, args, stream=None):
        from lucid_amd import _C

        held = [dev(a) for a in self.host(args)]
        if stream is not None:
            _C.synchronize()
        out = self.run(*held, stream=stream)
        if stream is not None:
            _C.call("lq_stream_synchronize", stream)
        got = [t.numpy() for t in out]
        del out
        return got


def _same(a, b):
    for x, y in zip(a, b):
        assert np.array_equal(np.ascontiguousarray(x).view(np.uint8), np.ascontiguousarray(y).view(np.uint8))


def test_on_a_created_stream(gpu):
    from lucid_amd import _C

    rng = np.random.default_rng(0)
    for lens, page in (([40, 300, 1], 16), ([2000, 70], 64)):
        step = Step(lens, page, 1)
        args = step.inputs(rng)
        want = step.eager(args)
        st = ctypes.c_void_p()
        _C.call("lq_stream_create", ctypes.byref(st))
        _same(step.eager(args, st), want)
        _C.call("lq_stream_destroy", st)


def test_two_graphs_in_turn(gpu):
    from lucid_amd.graphs import CapturedForward

    rng = np.random.default_rng(3)
    steps = [Step([2000, 70], 64, 1), Step([1500, 1, 1300], 16, 2)]
    caps = []
    for s in steps:
        held = [dev(a) for a in s.host(s.inputs(rng))]
        caps.append(CapturedForward(s.run, *held))
    for _ in range(3):
        for s, cap in zip(steps, caps):
            args = s.inputs(rng)
            want = s.eager(args)
            s.eager(s.inputs(rng))  # other contents in the workspace and the cache
            cap.load(*s.host(args))
            _same([t.numpy() for t in cap()], want)
