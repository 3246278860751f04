"""On which stream the serving ops' memory is allocated, uploaded and used, without a GPU: the library is
replaced by one that hands out addresses as the caching allocator does and writes down every call."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from lucid_amd import _C
import lucid_amd as L
import lucid_amd.nn.functional as F
import lucid_amd.nn.generation as G

S = ctypes.c_void_p(0x5000)  # a created stream


class Library:
    """Nothing that was queued ever ends: a freed block serves the stream it was freed on and no other, and
    with a use recorded on another stream it serves nobody."""

    def __init__(self):
        self.next, self.live, self.free, self.calls, self.made = 1 << 20, {}, [], [], []

    def lq_malloc(self, out, size):
        return self.lq_malloc_async(out, size, None)

    def lq_malloc_async(self, out, size, stream):
        size = -(-int(size) // 512) * 512
        key = getattr(stream, "value", stream)
        for i, (ptr, n, on, uses) in enumerate(self.free):
            if n == size and on == key and not uses - {on}:
                del self.free[i]
                break
        else:
            ptr, self.next = self.next, self.next + size
        self.live[ptr] = (size, set())
        out._obj.value = ptr
        self.made.append((ptr, key))
        return 0

    def lq_free(self, ptr):
        size, uses = self.live.pop(ptr)
        self.free.append((ptr, size, None, uses))
        return 0

    def lq_record_stream(self, ptr, stream):
        self.live[ptr][1].add(stream.value)
        return 0

    def lq_paged_attention_workspace_size(self, *a):
        return 4096

    def lq_token_logprobs_workspace_size(self, *a):
        return 8192

    def call(self, name, *args):
        self.calls.append((name, args))


@pytest.fixture
def lib(monkeypatch):
    fake = Library()
    monkeypatch.setattr(_C, "lib", lambda: fake)
    monkeypatch.setattr(_C, "call", fake.call)
    monkeypatch.setattr(_C, "_lib", fake)
    monkeypatch.setattr(G.workspace, "_local", type("Local", (), {})())
    yield fake


def _t(shape, dtype=np.float16):
    return L.empty(shape, dtype, "gpu")


def _ops(stream):
    """Every op that allocates, on operands of its own; what each returned."""
    qkv, starts = _t((40, 8, 64)), _t((3,), np.int32)
    yield "prompt", lambda: F.prompt_attention_qkv(qkv, 4, 2, starts, stream=stream)
    q, k, table, lens = _t((2, 4, 64)), _t((8, 2, 16, 64)), _t((2, 4), np.int32), _t((2,), np.int32)
    yield "paged", lambda: F.paged_attention(q, k, k, table, lens, 5000, stream=stream)
    x, t, f = _t((4, 99), np.float32), _t((4,), np.int32), _t((4,), np.float32)
    yield "logprobs", lambda: F.token_logprobs(x, t, 5, stream=stream)
    yield "backward", lambda: F.token_logprobs_backward(x, t, f, f, f, f, stream=stream)


@pytest.mark.parametrize("op", ["prompt", "paged", "logprobs", "backward"])
def test_results_and_workspace_of_a_created_stream_are_allocated_for_it(lib, op):
    """A block freed on the default stream, with work queued there that still reads it, never becomes the
    result or the workspace of a call on another stream."""
    run = dict(_ops(S))[op]
    run()
    sizes = [n for n, _ in lib.live.values()] + [n for _, n, _, _ in lib.free]
    pending = [_t((n,), np.uint8) for n in sizes for _ in range(3)]  # blocks of every size the call asks for
    freed = {p.data_ptr() for p in pending}
    del pending
    lib.made.clear()
    out = run()
    assert lib.made and all(on == S.value for _, on in lib.made)
    assert not freed & {ptr for ptr, _ in lib.made}
    # and what the call made is not handed out again before the stream's work is done
    for t in out if isinstance(out, tuple) else (out,):
        assert S.value in lib.live[t.data_ptr()][1]
    assert all(ptr in lib.live or any(ptr == p and S.value in uses for p, _, _, uses in lib.free)
               for ptr, _ in lib.made)


@pytest.mark.parametrize("op", ["prompt", "paged", "logprobs", "backward"])
@pytest.mark.parametrize("null", [None, ctypes.c_void_p(), 0])
def test_calls_on_the_default_stream_reuse_its_memory(lib, op, null):
    run = dict(_ops(null))[op]
    run()
    lib.made.clear()
    first = run()
    assert all(on is None for _, on in lib.made)
    ptr = (first[0] if isinstance(first, tuple) else first).data_ptr()
    del first
    again = run()
    assert ptr in {t.data_ptr() for t in (again if isinstance(again, tuple) else (again,))}
    assert all(args[-1] is None for name, args in lib.calls if name.startswith("lq_token") or "attention" in name)


def test_values_behind_codes_are_there_before_another_stream_reads_them(lib):
    """Logits held as codes are dequantized on the default stream; a call elsewhere waits for it."""
    from lucid_amd._tensor import QuantSource, Tensor

    q = QuantSource(_t((4, 99), np.int8), _C.I8, _t((), np.float32), _t((), np.float32), -128, 127)
    x = Tensor._code_backed(q, (4, 99))
    F.token_logprobs(x, _t((4,), np.int32), stream=S)
    names = [name for name, _ in lib.calls]
    at = names.index("lq_dequantize_per_tensor")
    assert lib.calls[at + 1] == ("lq_stream_synchronize", (None,))
    assert "lq_token_logprobs" in names[at + 2:]


def test_the_table_changes_on_the_stream_that_reads_it(lib):
    """grow and release change the device's table and lengths behind the kernels that are queued there."""
    pt = G.PageTable(3, 8, 4)
    lib.calls.clear()
    for stream in (S, None):
        pt.grow([5, 0, 1], stream)
        pt.release(0, stream)
        uploads = [args for name, args in lib.calls if name == "lq_memcpy_h2d"]
        assert [args[0] for args in uploads] == [t.data_ptr() for t in (pt.table, pt.lengths, pt.lengths)]
        assert all(args[-1] is stream for args in uploads)
        lib.calls.clear()
    for t in pt.rows([2, 1], S):
        assert S.value in lib.live[t.data_ptr()][1]
    assert len(lib.calls) == 2 and all(args[-1] is S for _, args in lib.calls)
