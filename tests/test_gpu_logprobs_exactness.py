"""The entropy and the log sum of rows that one token rules, as a trained model's are, by the root mean square
of their error over many rows.

u = 2^-24.  Where the largest term of S = sum e^d is 1, S and the logarithm are rounded at that size: some 14
additions over the workgroup's threads and one for each group of a thread's elements, half a u at most and
0.3 u on average each, independent of each other: below 4 u for rows of up to 200000.  The exponentials'
error is relative to terms that are small here.  log S - (sum e^d d) / S is then off by less than 8 u on
average, whatever the entropy; the log sum by that and the rounding of its own size."""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _dev(a):
    import lucid_amd as L

    return L.tensor(np.ascontiguousarray(a), device="gpu")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,vocab", [(160, 100003), (160, 32000), (160, 1000), (64, 200000)])
@pytest.mark.parametrize("lead", [2, 6, 10])
def test_rows_that_one_token_rules(gpu, dtype, rows, vocab, lead):
    import lucid_amd as L
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(vocab + lead)
    x = rng.standard_normal((rows, vocab)) * 2.5
    x[np.arange(rows), rng.integers(0, vocab, rows)] = x.max(1) + lead + 2 * rng.random(rows)
    x = x.astype(np.float32)
    if dtype == "bfloat16":
        bits = L.bf16_from_f32(x)
        x, xh = L.bf16_to_f32(bits), bits
    else:
        xh = x
    x = x.astype(np.float64)
    m = x.max(1, keepdims=True)
    e = np.exp(x - m)
    S = e.sum(1)
    want_lse = m[:, 0] + np.log(S)
    p = e / S[:, None]
    want = -(p * np.log(np.maximum(p, 1e-300))).sum(1)
    _, ent, lse, _, _ = (a.numpy().astype(np.float64) for a in F.token_logprobs(_dev(xh), _dev(np.zeros(rows, np.int32))))
    assert np.sqrt(np.mean((ent - want) ** 2)) <= 8 * U * max(1.0, want.max())
    assert np.sqrt(np.mean((lse - want_lse) ** 2)) <= 8 * U + U * np.abs(want_lse).max()
