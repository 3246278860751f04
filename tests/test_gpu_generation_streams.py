"""Serving ops on a stream of their own, with work pending elsewhere."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

N = 4096


def _dev(a):
    import lucid_amd as L

    return L.tensor(np.ascontiguousarray(a), device="gpu")


def _i32(a):
    return _dev(np.asarray(a, np.int32))


@pytest.fixture
def stream(gpu):
    from lucid_amd import _C

    st = ctypes.c_void_p()
    _C.call("lq_stream_create", ctypes.byref(st))
    yield st
    _C.call("lq_stream_synchronize", st)
    _C.call("lq_stream_destroy", st)


def test_a_result_on_a_stream_leaves_the_default_streams_pending_reads_alone(gpu, stream):
    """x is dropped with products that read it still queued on the default stream; a result of x's size
    made on another stream at that moment is not put where x was."""
    from lucid_amd import _C
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(0)
    a, b = (rng.integers(-127, 128, (N, N)).astype(np.int8) for _ in range(2))
    tokens, h, hd = 1024, 64, 128  # fp16 rows of x's size
    assert tokens * h * hd * 2 == a.nbytes
    q, k = (_dev(rng.standard_normal((tokens, n, hd)).astype(np.float16)) for n in (h, 1))
    starts = _i32([0, 5, tokens])
    want = F.prompt_attention(q, k, k, starts).numpy()
    gpu.synchronize()
    _C.call("lq_empty_cache")
    B, out = _dev(b), gpu.empty((N, N), np.int32, "gpu")
    x = _dev(a)
    gpu.synchronize()
    at = x.data_ptr()
    for _ in range(100):
        _C.call("lq_gemm_w8a8", x.data_ptr(), N, B.data_ptr(), N, out.data_ptr(), N, N, N, N, None, 0, None, 0, None,
                None, None, None, None, None, 0, 0, _C.OUT_I32, 0, None, 0, None)
    del x
    y = F.prompt_attention(q, k, k, starts, stream=stream)
    assert y.data_ptr() != at
    _C.call("lq_stream_synchronize", stream)
    np.testing.assert_array_equal(y.numpy(), want)
    rows = rng.choice(N, 16, replace=False)
    np.testing.assert_array_equal(out.numpy()[rows], a[rows].astype(np.int64) @ b.astype(np.int64).T)


@pytest.mark.parametrize("longest", [900, 3000])
def test_the_table_grows_behind_queued_attention(gpu, stream, longest):
    """Steps queued one after the other without waiting: append, attend, grow, append, attend.  Every step's
    attention is that of the lengths it was queued with."""
    from lucid_amd import _C
    from lucid_amd.nn.generation import PagedKVCache, PageTable

    rng = np.random.default_rng(longest)
    B, h, hkv, hd, steps = 24, 4, 2, 64, 6
    first = [longest] + [int(n) for n in rng.integers(1, longest, B - 1)]
    bound = longest + steps
    kv = [[_dev(rng.standard_normal((sum(n), hkv, hd)).astype(np.float16)) for _ in range(2)]
          for n in [first] + [[1] * B] * steps]
    q = [_dev(rng.standard_normal((B, h, hd)).astype(np.float16)) for _ in range(steps)]
    starts = _i32(np.concatenate([[0], np.cumsum(first)]))
    one = _i32(np.arange(B + 1))

    def serve(st, wait):
        pt = PageTable(B, B * (bound // 16 + 1), 16)
        cache = PagedKVCache(pt, hkv, hd)
        _C.synchronize()
        pt.grow(first, st)
        cache.append(*kv[0], starts, stream=st)
        outs = []
        for i in range(steps):
            pt.grow([1] * B, st)
            cache.append(*kv[i + 1], one, stream=st)
            outs.append(cache.attend(q[i], max_length=bound, stream=st))
            if wait:
                _C.synchronize()
        pt.release(0, st)
        pt.grow([40] + [0] * (B - 1), st)  # the released pages' next owner
        cache.append(*kv[0], _i32([0, 40] + [40] * (B - 1)), stream=st)
        _C.synchronize()
        return [o.numpy() for o in outs]

    for got, want in zip(serve(stream, False), serve(None, True)):
        np.testing.assert_array_equal(got, want)


def test_calls_of_two_launches_on_a_stream_of_their_own(gpu, stream):
    """Long sequences and long rows: the workspace is the call's own there, and the bits are the default
    stream's, with eager calls of other sizes between."""
    from lucid_amd import _C
    import lucid_amd.nn.functional as F

    rng = np.random.default_rng(4)
    lens = [5000, 1, 0, 2300]
    pages = 470
    table = np.zeros((4, 320), np.int32)
    ids, at = rng.permutation(pages), 0
    for b, n in enumerate(lens):
        table[b, :-(-n // 16)] = ids[at:at + -(-n // 16)]
        at += -(-n // 16)
    k, v = (_dev(rng.standard_normal((pages, 2, 16, 64)).astype(np.float16)) for _ in range(2))
    codes = _dev(rng.integers(-127, 128, (pages, 2, 16, 64)).astype(np.int8))
    scale = _dev((rng.random((pages, 2, 16)) / 100 + 1e-3).astype(np.float32))
    q, dt, dl = _dev(rng.standard_normal((4, 8, 64)).astype(np.float16)), _i32(table), _i32(lens)
    x = _dev((rng.standard_normal((5, 150001)) * 3).astype(np.float32))
    t = _i32([3, -100, 7, 150000, 0])
    _C.synchronize()

    def ops(s):
        out = [F.paged_attention(q, k, v, dt, dl, 5000, stream=s)]
        assert _C.last_path() == "paged shared"
        out.append(F.paged_attention(q, codes, codes, dt, dl, 5000, k_scale=scale, v_scale=scale, stream=s))
        assert _C.last_path() == "paged shared"
        out += F.token_logprobs(x, t, 7, stream=s)
        assert _C.last_path() == "logprobs parts"
        return out

    want = [y.numpy() for y in ops(None)]
    queued = []
    for _ in range(3):
        queued.append(ops(stream))
        F.token_logprobs(x, t, 64)  # the thread's own workspace, meanwhile
    _C.call("lq_stream_synchronize", stream)
    for got in queued:
        for y, z in zip(got, want):
            np.testing.assert_array_equal(y.numpy(), z)


def test_calls_of_two_launches_replayed_from_a_graph(gpu):
    """Recorded once, replayed after the lengths, the table and the logits changed, with eager calls that use
    the thread's own workspace and synchronizations between."""
    import lucid_amd as L
    from lucid_amd import _C
    import lucid_amd.nn.functional as F
    from lucid_amd.graphs import CapturedForward

    rng = np.random.default_rng(5)
    pages = 700
    k, v = (_dev(rng.standard_normal((pages, 1, 16, 128)).astype(np.float16)) for _ in range(2))
    t = _i32([3, -100, 7])
    paths = []

    def fn(q, table, lens, x):
        a = F.paged_attention(q, k, v, table, lens, 4000, out_dtype=L.float32)
        paths.append(_C.last_path())
        b = F.token_logprobs(x, t, 6)
        paths.append(_C.last_path())
        return (a, *b)

    def make():
        lens = np.array([4000, *rng.integers(0, 4000, 1), rng.integers(1, 40)], np.int32)
        return (rng.standard_normal((3, 4, 128)).astype(np.float16), rng.integers(0, pages, (3, 250)).astype(np.int32),
                rng.permutation(lens), (rng.standard_normal((3, 90001)) * 3).astype(np.float32))

    cap = CapturedForward(fn, *(_dev(a) for a in make()))
    assert set(paths[::2]) == {"paged shared"} and set(paths[1::2]) == {"logprobs parts"}
    for _ in range(6):
        arrays = make()
        cap.load(*arrays)
        got = [y.numpy() for y in cap()]
        want = [y.numpy() for y in fn(*(_dev(a) for a in arrays))]
        L.synchronize()
        for y, z in zip(got, want):
            np.testing.assert_array_equal(y, z)
