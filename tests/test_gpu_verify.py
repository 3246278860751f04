"""Verification of drafted tokens against a float64 restatement.  Tokens and counts are whole numbers and equal:
exponentials and sums are 64-bit on both sides, and a border within their error (some 2^-50) of a random number of 24
bits does not occur in these inputs."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from _decode import dev, i32, rounded

pytestmark = pytest.mark.gpu


def _lse(x):
    x = x.astype(np.float64)
    with np.errstate(all="ignore"):
        m = x.max(1)
        return (m + np.log(np.exp(x - m[:, None]).sum(1))).astype(np.float32)


def _want(x, lse, drafts, starts, au, su, d=None, dlse=None):
    tokens, accepted = np.full(len(x), 12345, np.int32), np.zeros(len(starts) - 1, np.int32)
    prob = lambda a, l, r: np.exp(a[r].astype(np.float64) - np.float64(l[r]))  # noqa: E731
    with np.errstate(all="ignore"):
        for s, (lo, hi) in enumerate(zip(starts[:-1], starts[1:])):
            if hi <= lo:
                continue
            tokens[lo:hi] = -1
            r, t = lo, -1
            while r < hi - 1:
                t = drafts[r]
                if not 0 <= t < x.shape[1]:
                    break
                q = prob(d, dlse, r)[t] if d is not None else 1.0
                if not np.float64(au[r]) * q < prob(x, lse, r)[t]:
                    break
                tokens[r] = t
                r += 1
            accepted[s] = r - lo
            p = prob(x, lse, r)
            w = p
            if r < hi - 1:
                if d is not None:
                    w = p - prob(d, dlse, r)
                    w = np.where(w > 0, w, 0)
                else:
                    w = p.copy()
                    if 0 <= t < len(p):
                        w[t] = 0
                if not w.sum() > 0:
                    w = p
            upto = np.cumsum(w)
            if upto[-1] > 0 and np.isfinite(upto[-1]):
                over = np.nonzero((upto > np.float64(su[s]) * upto[-1]) & (w > 0))[0]
                tokens[r] = over[0] if len(over) else np.nonzero(w > 0)[0][-1]
    return tokens, accepted


def _case(rng, each, vocab, dtype, sure, banned=0.0):
    rows = sum(each)
    x = rng.standard_normal((rows, vocab)) * 2
    x[np.arange(rows), rng.integers(0, vocab, rows)] += 6
    d = x + rng.standard_normal((rows, vocab))
    if banned:
        x[rng.random((rows, vocab)) < banned] = -np.inf
        x[np.arange(rows), rng.integers(0, vocab, rows)] = 1.0
    x, xh = rounded(x, dtype)
    d, dh = rounded(d, dtype)
    p = np.exp(d.astype(np.float64) - _lse(d)[:, None])
    drafts = np.array([rng.choice(vocab, p=row / row.sum()) if rng.random() < 0.7 else int(a)
                       for row, a in zip(p, x.argmax(1))], np.int32)
    u = lambda n: (rng.integers(0, 1 << 24, n) / (1 << 24)).astype(np.float32)  # noqa: E731
    return dict(x=x, lse=_lse(x), drafts=drafts, starts=np.cumsum([0] + each), au=u(rows), su=u(len(each)),
                d=None if sure else d, dlse=None if sure else _lse(d)), xh, dh


def _run(c, xh, dh, stream=None):
    import lucid_amd.nn.functional as F

    return F.verify_drafts(dev(xh), dev(c["lse"]), i32(c["drafts"]), i32(c["starts"]), dev(c["au"]), dev(c["su"]),
                           dev(dh) if c["d"] is not None else None, dev(c["dlse"]) if c["d"] is not None else None, stream)


def _check(c, xh, dh):
    tokens, accepted = (t.numpy() for t in _run(c, xh, dh))
    want, kept = _want(**c)
    mine = want != 12345
    assert np.array_equal(accepted, kept)
    assert np.array_equal(tokens[mine], want[mine])
    return kept


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("sure", [False, True])
@pytest.mark.parametrize("each,vocab", [
    ([1], 1), ([2], 1), ([3, 1, 5], 7), ([5, 0, 1, 4, 2], 257), ([9] * 20, 1000), ([4, 4], 4096), ([3, 6], 4097),
    ([5] * 8, 32000), ([2, 8, 1], 50001), ([70, 140, 3], 64), ([1] * 300, 33),
])
def test_against_float64(gpu, dtype, sure, each, vocab):
    rng = np.random.default_rng([vocab, len(each), sure])
    _check(*_case(rng, each, vocab, dtype, sure))


def test_kept_runs_of_every_length(gpu):
    """Drafts that are certain to be kept, up to one that is not: past 64 drafts too."""
    rng = np.random.default_rng(1)
    each = [n + 1 for n in (0, 1, 2, 63, 64, 65, 127, 128, 129, 200)]
    c, xh, dh = _case(rng, each, 40, "float32", True)
    c["drafts"] = c["x"].argmax(1).astype(np.int32)
    c["au"][:] = 0
    assert np.array_equal(_check(c, xh, dh), np.array(each) - 1)
    for s, n in enumerate(each):
        if n > 1:
            c["drafts"][c["starts"][s] + (n - 1) * 2 // 3] = [-1, 40][s % 2]
    assert np.array_equal(_check(c, xh, dh), [(n - 1) * 2 // 3 for n in each])


@pytest.mark.parametrize("sure", [False, True])
@pytest.mark.parametrize("vocab", [50, 9000])
def test_forbidden_tokens_and_borders(gpu, sure, vocab):
    """Tokens of probability 0 are never drawn, at random numbers 0 and just below 1 either."""
    rng = np.random.default_rng(vocab)
    c, xh, dh = _case(rng, [4] * 30, vocab, "float32", sure, banned=0.9)
    c["su"][:10], c["su"][10:20] = 0, 1 - 2.0 ** -24
    c["au"][::3], c["au"][1::3] = 0, 1 - 2.0 ** -24
    kept = _check(c, xh, dh)
    tokens = _run(c, xh, dh)[0].numpy()
    new = c["starts"][:-1] + kept
    assert np.isfinite(c["x"][new, tokens[new]]).all()


def test_rows_without_a_token_and_equal_distributions(gpu):
    """No allowed token or NaN: -1.  A draft's distribution that covers the target's: the target's own weights."""
    rng = np.random.default_rng(2)
    for sure in (False, True):
        c, xh, dh = _case(rng, [3] * 6, 300, "float32", sure)
        c["x"][0:3], c["x"][3, 7], c["x"][6:9] = -np.inf, np.nan, -np.inf
        c["x"][6:9, 5] = 2.0
        c["drafts"][6:9] = 5  # the only token: kept at any random number below 1, or nothing else is left
        c["lse"] = _lse(c["x"])
        if not sure:
            c["d"][9:12], c["dlse"][9:12] = c["x"][9:12], c["lse"][9:12] - np.float32(1e-3)  # q > p everywhere
            c["au"][9:12] = 1 - 2.0 ** -24
        tokens, accepted = (t.numpy() for t in _run(c, c["x"], c["d"]))
        want, kept = _want(**c)
        assert np.array_equal(tokens, want) and np.array_equal(accepted, kept)
        assert tokens[0] == -1 and tokens[3] == -1 and (tokens[6:9][:kept[2] + 1] == 5).all()


def test_rows_of_no_sequence_and_wild_starts(gpu):
    """Rows before the first start and past the last are as they were; starts past the rows take what there is."""
    import lucid_amd as L
    import lucid_amd.nn.functional as F
    from lucid_amd import _C

    rng = np.random.default_rng(3)
    c, xh, dh = _case(rng, [3, 4, 3], 500, "float32", False)
    for starts in ([2, 5, 5, 8], [0, 4, 10, 25], [-3, 2, 11, 12], [7, 3, 9, 9]):
        out, acc = dev(np.full(10, 12345, np.int32)), dev(np.zeros(3, np.int32))
        size = _C.lib().lq_verify_drafts_workspace_size(3, 500)
        ws, held = L.empty((size,), np.uint8, "gpu"), [dev(a) for a in (xh, c["lse"], dh, c["dlse"], c["drafts"], c["au"], c["su"])]
        st = i32(starts)
        p = [t.data_ptr() for t in held]
        _C.call("lq_verify_drafts", p[0], _C.F32, 500, p[1], p[2], 500, p[3], p[4], st.data_ptr(), 3, 10, 500, p[5], p[6],
                out.data_ptr(), acc.data_ptr(), ws.data_ptr(), size, None)
        if sorted(starts) != starts:
            continue  # nothing outside the arrays is touched: that is all that is promised
        clipped = np.clip(starts, 0, 10)
        want, kept = _want(**{**c, "starts": clipped})
        assert np.array_equal(out.numpy(), want) and np.array_equal(acc.numpy(), kept)


def test_wide_rows_and_strides(gpu):
    """Rows inside wider ones, of two different strides."""
    import lucid_amd as L
    from lucid_amd import _C

    rng = np.random.default_rng(4)
    each, vocab = [3, 5], 6001
    c, xh, dh = _case(rng, each, vocab, "bfloat16", False)
    pad = lambda a, n: dev(np.concatenate([a, np.zeros((len(a), n), a.dtype)], 1))  # noqa: E731
    held = [pad(xh, 7), pad(dh, 130)] + [dev(a) for a in (c["lse"], c["dlse"], c["drafts"], c["au"], c["su"])]
    p = [t.data_ptr() for t in held]
    out, acc, st = dev(np.zeros(8, np.int32)), dev(np.zeros(2, np.int32)), i32(c["starts"])
    size = _C.lib().lq_verify_drafts_workspace_size(2, vocab)
    ws = L.empty((size,), np.uint8, "gpu")
    _C.call("lq_verify_drafts", p[0], _C.BF16, vocab + 7, p[2], p[1], vocab + 130, p[3], p[4], st.data_ptr(), 2, 8, vocab,
            p[5], p[6], out.data_ptr(), acc.data_ptr(), ws.data_ptr(), size, None)
    want, kept = _want(**c)
    assert np.array_equal(out.numpy(), want) and np.array_equal(acc.numpy(), kept)


def test_on_a_stream_and_from_a_graph(gpu):
    import lucid_amd.nn.functional as F
    from lucid_amd import _C
    from lucid_amd.graphs import CapturedForward

    rng = np.random.default_rng(5)
    c, xh, dh = _case(rng, [4, 2, 6], 9001, "float16", False)
    want, kept = _want(**c)
    st = ctypes.c_void_p()
    _C.call("lq_stream_create", ctypes.byref(st))
    held = [dev(xh), dev(c["lse"]), i32(c["drafts"]), i32(c["starts"]), dev(c["au"]), dev(c["su"]), dev(dh), dev(c["dlse"])]
    _C.synchronize()
    tokens, accepted = F.verify_drafts(*held, st)
    _C.call("lq_stream_synchronize", st)
    assert np.array_equal(tokens.numpy(), want) and np.array_equal(accepted.numpy(), kept)
    del tokens, accepted
    _C.call("lq_stream_destroy", st)
    cap = CapturedForward(lambda *a: F.verify_drafts(*a), *held)
    for _ in range(3):
        c, xh, dh = _case(rng, [4, 2, 6], 9001, "float16", False)
        cap.load(xh, c["lse"], c["drafts"], c["starts"], c["au"], c["su"], dh, c["dlse"])
        tokens, accepted = cap()
        want, kept = _want(**c)
        assert np.array_equal(tokens.numpy(), want) and np.array_equal(accepted.numpy(), kept)


def test_tokens_follow_the_target(gpu):
    """Over all random numbers of a grid, the first token of a sequence has the target's share exactly where the
    draft was certain: p(draft) of the acceptances, the rest by their weights (counts within the grid's step)."""
    n, vocab = 4096, 8
    x = np.log(np.array([0.05, 0.3, 0.1, 0.15, 0.2, 0.02, 0.08, 0.1])).astype(np.float32)
    grid = ((np.arange(n) + 0.5) / n).astype(np.float32)
    xs = np.repeat(x[None], 2 * n, 0)
    c = dict(x=xs, lse=_lse(xs), drafts=np.full(2 * n, 1, np.int32), starts=np.arange(0, 2 * n + 1, 2), au=np.repeat(grid, 2),
             su=np.random.default_rng(0).permutation(grid), d=None, dlse=None)
    tokens, accepted = (t.numpy() for t in _run(c, xs, None))
    assert abs(int((accepted == 1).sum()) - round(0.3 * n)) <= 1
    rejected = tokens[::2][accepted == 0]
    assert (rejected != 1).all() and set(rejected) <= set(range(vocab))
