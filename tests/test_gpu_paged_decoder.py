"""The decoder served from pages: against the dense-cache decoder on prompts of one length, with
sequences of different lengths that come and go, its scores against log-softmax on the host, its
gradient against the formula."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def served():
    import lucid_amd.backends as backends
    from lucid_amd.bench_configs import decoder
    from lucid_amd.quantization import quantize_dynamic

    old = backends.quantized.engine
    backends.quantized.engine = "reference"
    try:
        dec, glue = decoder(np.random.default_rng(21))
        qdec = quantize_dynamic(dec)
    finally:
        backends.quantized.engine = old
    return qdec, glue


def _cos(a, b):
    a, b = a.astype(np.float64), b.astype(np.float64)
    return ((a * b).sum(-1) / (np.linalg.norm(a, axis=-1) * np.linalg.norm(b, axis=-1))).min()


def test_same_lengths_agree_with_the_dense_cache(gpu, served):
    """The same codes, products and norms; only the attention kernels differ, in the last bits of
    float32, so that few activation codes move (cosine of the logits)."""
    from lucid_amd import _C
    from lucid_amd.bench_configs import Int8Decoder
    from lucid_amd.paged_decoder import PagedDecoder

    qdec, glue = served
    B, T, steps = 4, 48, 5
    prompt = np.random.default_rng(3).integers(0, glue["tok"].shape[0], (B, T))
    rt = Int8Decoder(qdec, glue, batch=B, max_prompt=T, max_positions=T + steps)
    st = ctypes.c_void_p()
    _C.call("lq_stream_create", ctypes.byref(st))
    rt.set_prompt(prompt)
    rt.prefill(st)
    _C.call("lq_stream_synchronize", st)
    pd = PagedDecoder(qdec, glue, seqs=B, pages=B * 4)
    logits = pd.prefill(dict(enumerate(prompt)))
    assert _cos(logits.numpy(), rt.logits.numpy()) > 0.999
    for _ in range(steps):
        tok = rt.next.numpy()
        rt.decode(st)
        _C.call("lq_stream_synchronize", st)
        logits = pd.step(dict(enumerate(tok.tolist())))
        assert _cos(logits.numpy(), rt.logits.numpy()) > 0.995
    _C.call("lq_stream_destroy", st)


@pytest.mark.parametrize("cache", ["float16", "int8"])
def test_sequences_come_and_go(gpu, served, cache):
    """Continuations do not depend on which pages a sequence got or who else held the pool: the
    same requests, served again after others came and went, give the same tokens."""
    from lucid_amd.paged_decoder import PagedDecoder

    qdec, glue = served
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, glue["tok"].shape[0], n) for n in (40, 1, 17, 90)]
    pd = PagedDecoder(qdec, glue, seqs=4, pages=16, cache_dtype=np.dtype(cache))
    first, scores, others = pd.generate(prompts, 6)
    assert np.isfinite(scores).all() and (scores <= 0).all()
    np.testing.assert_array_equal(others[:, :, 0], first)  # greedy: the best alternative is the token
    logits = pd.prefill({2: prompts[0], 0: prompts[1]})  # two of four
    assert logits.shape == (2, pd.vocab)
    one = pd.step({2: 5})
    assert one.shape == (1, pd.vocab) and np.isfinite(one.numpy()).all()
    assert pd.table.host_lengths().tolist() == [1, 0, 41, 0]
    pd.table.release(2)
    pd.table.release(0)
    again, scores2, _ = pd.generate(prompts, 6)
    np.testing.assert_array_equal(first, again)
    np.testing.assert_array_equal(scores, scores2)
    with pytest.raises(MemoryError):
        pd.prefill({0: rng.integers(0, 10, 200), 1: rng.integers(0, 10, 200)})
    with pytest.raises(ValueError):
        pd.step({0: 1})


def test_scores_and_gradient(gpu, served):
    from lucid_amd.paged_decoder import PagedDecoder

    qdec, glue = served
    rng = np.random.default_rng(9)
    prompts = [rng.integers(0, glue["tok"].shape[0], n) for n in (20, 3, 1)]
    pd = PagedDecoder(qdec, glue, seqs=1, pages=1)
    logits, targets = pd._score_rows(prompts)
    x, t = logits.numpy().astype(np.float64), targets.numpy()
    lse = np.log(np.exp(x - x.max(1, keepdims=True)).sum(1)) + x.max(1)
    ok = t >= 0
    want = np.where(ok, x[np.arange(24), np.maximum(t, 0)] - lse, 0)
    lp, ent, got_lse, _, _ = pd.score(prompts)
    assert (np.abs(lp.numpy() - want) < 1e-4).all() and (np.abs(got_lse.numpy() - lse) < 1e-5).all()
    assert [i for i in range(24) if not ok[i]] == [19, 22, 23]
    w = rng.standard_normal(24).astype(np.float32)
    value, grad, bias = pd.tune(prompts, w, 0.05)
    p = np.exp(x - lse[:, None])
    H = lse - (p * x).sum(1)
    hot = np.zeros_like(x)
    hot[np.arange(24)[ok], t[ok]] = 1
    g = (w * ok)[:, None] * (hot - p) - 0.05 * p * (x - lse[:, None] + H[:, None])
    assert abs(value - ((w * want).sum() + 0.05 * H.sum())) < 1e-3
    assert np.abs(grad.numpy() - g).max() < 1e-5 and np.abs(bias - g.sum(0)).max() < 1e-4
