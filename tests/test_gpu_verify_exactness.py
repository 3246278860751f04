"""The exponentials behind the verification of drafts, and what its launches write.

Three tokens of weights e^c, e^a and e^b, drawn at 1/2: the first one exactly where e^c > e^a + e^b.  c is the float32
next to log(e^a + e^b), so that the two sides differ by some 2^-25 of them in the mean and by less than 2^-40 in some of many
draws: tokens compare exponentials that closely."""

from __future__ import annotations

import numpy as np
import pytest

from _decode import dev, i32

pytestmark = pytest.mark.gpu


def _draw(x, lse):
    """The token that each row of x [rows, vocab] gives at 1/2."""
    import lucid_amd.nn.functional as F

    rows = len(x)
    tokens, _ = F.verify_drafts(dev(x), dev(lse), i32(np.full(rows, -100)), i32(np.arange(rows + 1)),
                                dev(np.zeros(rows, np.float32)), dev(np.full(rows, 0.5, np.float32)))
    return tokens.numpy()


@pytest.mark.parametrize("span,lse", [(0.01, 0.0), (1.0, 0.0), (30.0, 0.0), (20.0, 17.25)])
def test_exponentials_of_64_bits(gpu, span, lse):
    """Every draw whose sides differ by more than 2^-48.6 of them is decided as by 64-bit mantissas.  In units of 2^-53 of
    its value an exponential is off by 2 for its table (a library function within one step), 1 for its last sum, 0.4 for
    the series' next term and less for the rest, 6 at most; three of them and the two sums by 20 units, 2^-48.6."""
    rng = np.random.default_rng(int(span * 100))
    n = 1 << 21
    a, b = rng.uniform(-span, span, (2, n)).astype(np.float32)
    b = a + (b - a) / 8  # neither rules the sum
    wide = np.longdouble
    assert np.finfo(wide).nmant >= 63
    both = np.exp(a.astype(wide)) + np.exp(b.astype(wide))
    c = np.log(both).astype(np.float32)
    gap = np.exp(c.astype(wide)) / both - 1
    close = np.argsort(np.abs(gap))[:4096]
    x = np.stack([c, a, b], 1)[close]
    known = np.abs(gap[close]) > wide(2.0) ** -48.6
    assert known.sum() > 3500 and (np.abs(gap[close]) < 2.0 ** -32).all()
    got = _draw(x, np.full(len(x), lse, np.float32))
    assert np.array_equal((got == 0)[known], (gap[close] > 0)[known])
    assert (got >= 0).all() and (got < 3).all()


def test_exponentials_of_equal_logits(gpu):
    """Two equal weights and a third one of e^-40 of them: at 1/2 the second token, however far the logits lie from 0."""
    a = np.concatenate([np.linspace(-600, 600, 2001), [0, -700]]).astype(np.float32)
    x = np.stack([a, a, a - 40], 1)
    assert (_draw(x, np.zeros(len(x), np.float32)) == 1).all()
    assert (_draw(x[:, [0, 1]], np.zeros(len(x), np.float32)) == 1).all()  # the sum up to the first is not above half of all


@pytest.mark.parametrize("sure", [False, True])
@pytest.mark.parametrize("starts", [[2, 5, 5, 8], [0, 4, 10, 25], [-3, 2, 11, 12], [7, 3, 9, 9], [9, 6, 2, 0], [10, 10, 10, 10],
                                    [2 ** 31 - 1, -2 ** 31, 5, 10]])
def test_nothing_is_written_beside_the_results(gpu, sure, starts):
    """Results and workspace inside larger buffers of marks, whatever the starts hold."""
    from lucid_amd import _C

    rng = np.random.default_rng(3)
    rows, vocab, mark = 10, 1500, 0x5a
    x, d = rng.standard_normal((2, rows, vocab)).astype(np.float32)
    held = [dev(x), dev(np.log(np.exp(x.astype(np.float64)).sum(1)).astype(np.float32)), dev(d),
            dev(np.log(np.exp(d.astype(np.float64)).sum(1)).astype(np.float32)), i32(rng.integers(0, vocab, rows)),
            dev(rng.random(rows).astype(np.float32)), dev(rng.random(3).astype(np.float32)), i32(starts)]
    p = [t.data_ptr() for t in held]
    size = _C.lib().lq_verify_drafts_workspace_size(3, vocab)
    places, buffers = [], []
    for nbytes in (4 * rows, 4 * 3, size):
        buffers.append(dev(np.full(nbytes + 512, mark, np.uint8)))
        places.append(buffers[-1].data_ptr() + 256)
    _C.call("lq_verify_drafts", p[0], _C.F32, vocab, p[1], None if sure else p[2], vocab, None if sure else p[3], p[4], p[7],
            3, rows, vocab, p[5], p[6], places[0], places[1], places[2], size, None)
    for b, nbytes in zip(buffers, (4 * rows, 4 * 3, size)):
        got = b.numpy()
        assert (got[:256] == mark).all() and (got[256 + nbytes:] == mark).all()
    tokens, kept = buffers[0].numpy()[256:256 + 4 * rows].view(np.int32), buffers[1].numpy()[256:268].view(np.int32)
    untouched = int(np.full(4, mark, np.uint8).view(np.int32)[0])
    lo, hi = np.clip(starts[:-1], 0, rows), np.clip(starts[1:], 0, rows)
    inside = np.zeros(rows, bool)
    for s, (a, b) in enumerate(zip(lo, hi)):
        inside[a:b] = True
        assert 0 <= kept[s] <= max(b - a - 1, 0)
    assert (tokens[~inside] == untouched).all()
    assert ((tokens[inside] >= -1) & (tokens[inside] < vocab)).all()
