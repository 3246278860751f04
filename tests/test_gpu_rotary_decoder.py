"""The decode step's operators run together: a decoder with root-mean-square norms, rotated keys and 4-bit pages,
whose drafts are verified; and the drafts of the decoder with positions added."""

from __future__ import annotations

import numpy as np
import pytest

from _decode import dev

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


def _make(served, cls, cache, seqs=3, pages=60):
    from lucid_amd.paged_decoder import PagedDecoder, RotaryDecoder

    qdec, glue = served
    if cls == "rotary":
        return RotaryDecoder(qdec, glue["tok"], seqs, pages, cache_dtype=cache, positions=600)
    return PagedDecoder(qdec, glue, seqs, pages, cache_dtype=cache)


@pytest.mark.parametrize("cls", ["rotary", "added"])
@pytest.mark.parametrize("cache,least", [("float16", 0.999), ("int8", 0.995), ("uint4", 0.97)])
def test_steps_agree_with_scoring(gpu, served, cls, cache, least):
    """A prompt, then steps over the pages: the logits of scoring the whole in one pass, whose attention reads the
    values before they were rounded to pages (4 bits are off by a few hundredths)."""
    pd = _make(served, cls, cache)
    rng = np.random.default_rng(3)
    toks = [rng.integers(0, pd.vocab, n) for n in (33, 9, 70)]
    cut = 5
    logits = [pd.prefill({s: t[:-cut] for s, t in enumerate(toks)}).numpy()]
    for i in range(cut, 1, -1):
        logits.append(pd.step({s: int(t[-i]) for s, t in enumerate(toks)}).numpy())
    whole, _ = pd._score_rows([t[:-1] for t in toks])
    whole, at = whole.numpy(), np.cumsum([len(t) - 1 for t in toks])
    for i, got in enumerate(logits):
        assert _cos(got, whole[at - cut + i]) > least


@pytest.mark.parametrize("cls", ["rotary", "added"])
def test_drafts_run_as_steps_do(gpu, served, cls):
    """Several tokens in one pass leave what single steps leave: drafts that are kept for certain (random number 0) and
    the sequences after them, against a decoder that steps."""
    rng = np.random.default_rng(4)
    a, b = _make(served, cls, "uint4"), _make(served, cls, "uint4")
    prompts = {s: rng.integers(0, a.vocab, n) for s, n in enumerate((20, 3, 41))}
    for pd in (a, b):
        pd.prefill(prompts)
    more = {0: [5, 17, 300, 9], 2: [7]}
    accept = np.zeros(5, np.float32)
    got = a.speculate(more, accept, np.array([0.3, 0.6], np.float32))
    assert got[0][:3].tolist() == [17, 300, 9] and len(got[0]) == 4 and len(got[2]) == 1
    assert a.table.host_lengths().tolist() == [24, 3, 42]
    for tok in more[0][:-1]:
        b.step({0: tok})
    b.step({0: more[0][-1], 2: 7})
    assert b.table.host_lengths().tolist() == [24, 3, 42]
    nxt = {0: 11, 1: 12, 2: 13}
    assert _cos(a.step(nxt).numpy(), b.step(nxt).numpy()) > 0.99


def test_refused_drafts_leave_the_sequence(gpu, served):
    """A draft outside the distribution's reach is dropped with what follows; the sequence goes on as if it had
    never been there, and the new token is the one its logits give."""
    rng = np.random.default_rng(5)
    a, b = _make(served, "rotary", "float16"), _make(served, "rotary", "float16")
    prompt = {1: rng.integers(0, a.vocab, 30)}
    for pd in (a, b):
        pd.prefill(prompt)
    logits = b.step({1: 8}).numpy()[0].astype(np.float64)
    worst = int(logits.argmin())
    got = a.speculate({1: [8, worst, 3]}, np.full(3, 1 - 2.0 ** -24, np.float32), np.array([0.5], np.float32))
    assert a.table.host_lengths().tolist() == [0, 31, 0] and len(got[1]) == 1 and got[1][0] != worst
    p = np.exp(logits - logits.max())
    p[worst] = 0
    share = np.cumsum(p) / p.sum()
    assert abs(share[got[1][0]] - 0.5) < 0.01  # the token at the middle of the distribution
    assert _cos(a.step({1: 4}).numpy(), b.step({1: 4}).numpy()) > 0.999


def test_a_draft_model_with_the_same_distribution(gpu, served):
    """Drafts proposed with the target's own probabilities are kept at any random number below 1."""
    import lucid_amd.nn.functional as F
    from lucid_amd._tensor import tensor

    rng = np.random.default_rng(6)
    pd = _make(served, "rotary", "uint4")
    pd.prefill({0: rng.integers(0, pd.vocab, 12)})
    toks = [4, 99, 1000]
    table, _ = pd.table.rows([0])
    first = pd.speculate({0: toks}, np.zeros(3, np.float32), np.array([0.1], np.float32))
    assert len(first[0]) == 3
    pd.table.shrink(np.array([3, 0, 0]))
    # the same pass, its own logits given as the draft's
    seen = []
    head = pd.qdec.head

    class Head:
        def __call__(self, h):
            seen.append(head(h))
            return seen[-1]

    class Layers:
        layers, head = pd.qdec.layers, Head()

    pd.qdec = Layers()
    pd.speculate({0: toks}, np.zeros(3, np.float32), np.array([0.1], np.float32))
    pd.table.shrink(np.array([3, 0, 0]))
    drafts = tensor(np.array([99, 1000, -100], np.int32), device="gpu")
    lse = F.token_logprobs(seen[0], drafts)[2]
    got = pd.speculate({0: toks}, np.full(3, 1 - 2.0 ** -24, np.float32), np.array([0.1], np.float32), seen[0], lse)
    assert got[0][:2].tolist() == [99, 1000]


def test_generation_over_four_bits_repeats(gpu, served):
    """Continuations do not depend on the pages a sequence got."""
    pd = _make(served, "rotary", "uint4")
    rng = np.random.default_rng(7)
    prompts = [rng.integers(0, pd.vocab, n) for n in (17, 40)]
    first = pd.generate(prompts, 6)
    pd.prefill({2: rng.integers(0, pd.vocab, 50)})
    second = pd.generate(prompts, 6)
    for x, y in zip(first, second):
        assert np.array_equal(x, y)


def test_calls_that_draft_nothing_or_are_refused(gpu, served):
    """No sequences, a token without drafts, and refusals that leave the sequences as they were."""
    a, b = _make(served, "rotary", "float16"), _make(served, "rotary", "float16")
    prompt = {0: np.arange(5, 25)}
    for pd in (a, b):
        pd.prefill(prompt)
    assert a.speculate({}, [], []) == {}
    logits = b.step({0: 8}).numpy()[0].astype(np.float64)
    got = a.speculate({0: [8]}, np.zeros(1, np.float32), np.array([0.25], np.float32))
    share = np.cumsum(np.exp(logits - logits.max()))
    assert len(got[0]) == 1 and abs(share[got[0][0]] / share[-1] - 0.25) < 0.01
    before = a.table.host_lengths().tolist()
    zeros = np.zeros(2, np.float32)
    for tokens, accept, sample in (({0: [1, 2]}, zeros[:1], zeros[:1]), ({0: [1, 2]}, zeros, zeros),
                                   ({0: [1, a.vocab]}, zeros, zeros[:1]), ({0: []}, [], zeros[:1]),
                                   ({1: [1, 2]}, zeros, zeros[:1]), ({7: [1, 2]}, zeros, zeros[:1]),
                                   ({0: np.ones(a.positions, np.int64)}, np.zeros(a.positions), zeros[:1])):
        with pytest.raises((ValueError, IndexError)):
            a.speculate(tokens, accept, sample)
        assert a.table.host_lengths().tolist() == before
    assert _cos(a.step({0: 4}).numpy(), b.step({0: 4}).numpy()) > 0.999
