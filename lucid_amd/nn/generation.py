"""Serving ops of a decoder: a paged key-value cache, the attention that reads it, attention over
packed prompts, and the log probabilities of tokens with their gradient.

The functions are part of ``lucid_amd.nn.functional``; :class:`PagedKVCache` keeps the pages, the
page table and the lengths of one layer's cache, :class:`PageTable` shares a table between the
layers of a model.  No counterpart in the reference, whose decode attends a dense cache
(lucid/nn/functional/attention.py, ``scaled_dot_product_attention``).  Everything runs on the
default stream (``stream=None``) or on a stream of ``lq_stream_create``.  Results and workspace are
allocated for the stream of the call; that the operands are ready there is the caller's to order,
and an operand that may be dropped before that stream's work is done is marked with
``Tensor.record_stream`` by the caller.  A call is captured into a graph through
``lucid_amd.graphs.CapturedForward``, which keeps what the call allocates.
"""

from __future__ import annotations

import ctypes

import numpy as np

from lucid_amd import _C
from lucid_amd._tensor import FLOAT_TYPE_CODE, Tensor, bfloat16, empty, float16, float32, tensor
from lucid_amd.quantization._device import require_gpu, workspace


def _sig() -> None:
    P, I64, I, F, SZ = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_size_t
    _C.register_signatures({
        "lq_paged_kv_append": (I, [P, P, I, I64, I64, P, I64, I64, I64, P, I64, P, P, P, I, P, P, I64, I64, P]),
        "lq_paged_attention_workspace_size": (SZ, [I64, I64, I64, I64, I64]),
        "lq_paged_attention": (I, [P, I, I64, I64, I64, I64, I64, P, P, I, P, P, I64, I64, P, I64, P, I64, F, P, I, P,
                                   SZ, P]),
        "lq_prompt_attention": (I, [P, I64, P, I64, P, I64, I, P, P, I64, I64, I64, I64, I64, I64, I, F, P, I, P]),
        "lq_token_logprobs_workspace_size": (SZ, [I64, I64, I64]),
        "lq_token_logprobs": (I, [P, I, I64, I64, I64, P, I64, P, P, P, P, P, P, SZ, P]),
        "lq_token_logprobs_backward": (I, [P, I, I64, I64, I64, P, P, P, P, P, P, I64, P]),
    })


_sig()

_CACHE_TYPE = {float16: _C.F16, bfloat16: _C.BF16, np.dtype(np.int8): _C.I8}


def _need(x, op: str, name: str, ndim: int, dtypes) -> np.dtype:
    """``x`` as a device tensor of ``ndim`` axes and one of ``dtypes``."""
    require_gpu(x, op)
    if x.ndim != ndim:
        raise ValueError(f"{op}: {name} must have {ndim} axes, got shape {tuple(x.shape)}")
    if x.dtype not in dtypes:
        raise TypeError(f"{op}: {name} is {x.dtype}; expected one of {', '.join(str(d) for d in dtypes)}")
    return x.dtype


def _ints(x, op: str, name: str, n: int | None = None) -> Tensor:
    _need(x, op, name, 1, (np.dtype(np.int32),))
    if n is not None and x.shape[0] != n:
        raise ValueError(f"{op}: {name} must hold {n} numbers, got {x.shape[0]}")
    return x


def _pages(op, k_pages, v_pages, k_scale, v_scale, table, lengths):
    """(pages, kv heads, page, head dim) of a cache's tensors, checked against each other."""
    dt = _need(k_pages, op, "k_pages", 4, tuple(_CACHE_TYPE))
    _need(v_pages, op, "v_pages", 4, (dt,))
    if tuple(v_pages.shape) != tuple(k_pages.shape):
        raise ValueError(f"{op}: k_pages {tuple(k_pages.shape)} and v_pages {tuple(v_pages.shape)} differ")
    if dt == np.int8:
        for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
            if s is None:
                raise ValueError(f"{op}: an int8 cache needs {name}")
            _need(s, op, name, 3, (float32,))
            if tuple(s.shape) != tuple(k_pages.shape[:3]):
                raise ValueError(f"{op}: {name} must have shape {tuple(k_pages.shape[:3])}, got {tuple(s.shape)}")
    _need(table, op, "table", 2, (np.dtype(np.int32),))
    _ints(lengths, op, "lengths", table.shape[0])
    return tuple(int(n) for n in k_pages.shape)


def _stream(stream, *operands):
    """``stream``, the default one as None.  An operand behind codes gets its values on the default
    stream; another stream's work waits for them."""
    if not getattr(stream, "value", stream):
        return None
    behind = [t for t in operands if t is not None and t.is_code_backed and t._buf is None]
    for t in behind:
        t.data_ptr()
    if behind:
        _C.call("lq_stream_synchronize", None)
    return stream


def _scratch(nbytes: int, stream):
    """(address, holder) of workspace for one call: the thread's own on the default stream; on
    another stream memory of its own, allocated for that stream."""
    if nbytes == 0:
        return None, None
    if stream is None:
        return workspace.get(nbytes), None
    t = empty((nbytes,), np.uint8, "gpu", stream)
    return t.data_ptr(), t


def _opt(t) -> int | None:
    return t.data_ptr() if t is not None else None


def paged_kv_append(k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor,
                    starts: Tensor | None = None, k_scale: Tensor | None = None, v_scale: Tensor | None = None,
                    stream=None) -> None:
    """New tokens' keys and values ``[tokens, kv_heads, head_dim]`` into the pages of their
    sequences, whose ``lengths`` count the new tokens already.  ``starts`` [seqs + 1] packs
    several tokens per sequence; without it every sequence has one.  See ``lq_paged_kv_append``."""
    op = "paged_kv_append"
    pages, hkv, page, hd = _pages(op, k_pages, v_pages, k_scale, v_scale, table, lengths)
    dt = _need(k, op, "k", 3, tuple(FLOAT_TYPE_CODE))
    _need(v, op, "v", 3, (dt,))
    if tuple(k.shape) != tuple(v.shape) or tuple(k.shape[1:]) != (hkv, hd):
        raise ValueError(f"{op}: k {tuple(k.shape)} and v {tuple(v.shape)} must be [tokens, {hkv}, {hd}]")
    seqs, tokens = int(table.shape[0]), int(k.shape[0])
    if starts is not None:
        _ints(starts, op, "starts", seqs + 1)
    elif tokens != seqs:
        raise ValueError(f"{op}: {tokens} tokens for {seqs} sequences need starts")
    stream = _stream(stream, k, v, k_scale, v_scale)
    _C.call("lq_paged_kv_append", k.data_ptr(), v.data_ptr(), FLOAT_TYPE_CODE[dt], hkv * hd, tokens, _opt(starts), seqs,
            hkv, hd, table.data_ptr(), table.shape[1], lengths.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
            _CACHE_TYPE[k_pages.dtype], _opt(k_scale), _opt(v_scale), pages, page, stream)


def paged_kv_append_qkv(qkv: Tensor, heads: int, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor,
                        starts: Tensor | None = None, k_scale: Tensor | None = None, v_scale: Tensor | None = None,
                        stream=None) -> None:
    """:func:`paged_kv_append` of a fused projection's rows ``[tokens, heads + 2 kv_heads,
    head_dim]`` (queries, keys, values), read in place."""
    op = "paged_kv_append_qkv"
    pages, hkv, page, hd = _pages(op, k_pages, v_pages, k_scale, v_scale, table, lengths)
    dt = _need(qkv, op, "qkv", 3, tuple(FLOAT_TYPE_CODE))
    if heads < 1 or tuple(qkv.shape[1:]) != (heads + 2 * hkv, hd):
        raise ValueError(f"{op}: qkv {tuple(qkv.shape)} for {heads} heads and {hkv} key heads of {hd}")
    seqs, tokens = int(table.shape[0]), int(qkv.shape[0])
    if starts is not None:
        _ints(starts, op, "starts", seqs + 1)
    elif tokens != seqs:
        raise ValueError(f"{op}: {tokens} tokens for {seqs} sequences need starts")
    stream = _stream(stream, qkv, k_scale, v_scale)
    k = qkv.data_ptr() + heads * hd * dt.itemsize
    _C.call("lq_paged_kv_append", k, k + hkv * hd * dt.itemsize, FLOAT_TYPE_CODE[dt], (heads + 2 * hkv) * hd, tokens,
            _opt(starts), seqs, hkv, hd, table.data_ptr(), table.shape[1], lengths.data_ptr(), k_pages.data_ptr(),
            v_pages.data_ptr(), _CACHE_TYPE[k_pages.dtype], _opt(k_scale), _opt(v_scale), pages, page, stream)


def _out_type(out_dtype, dt, op: str) -> np.dtype:
    out = np.dtype(out_dtype) if out_dtype is not None else dt
    if out not in (dt, float32):
        raise TypeError(f"{op}: out_dtype must be {dt} or float32, got {out}")
    return out


def _scale(scale, hd: int, op: str) -> float:
    s = hd ** -0.5 if scale is None else float(scale)
    if not 0.0 < s < float("inf"):
        raise ValueError(f"{op}: scale must be positive and finite, got {scale}")
    return s


def paged_attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, max_length: int,
                    scale: float | None = None, k_scale: Tensor | None = None, v_scale: Tensor | None = None,
                    out_dtype=None, stream=None, heads: int | None = None) -> Tensor:
    """Attention of one new token per sequence, ``q`` [seqs, heads, head_dim], over its pages;
    ``max_length`` is the host's bound of ``lengths``.  With ``heads`` the queries are the first
    heads of wider rows (a fused projection's).  See ``lq_paged_attention``."""
    op = "paged_attention"
    pages, hkv, page, hd = _pages(op, k_pages, v_pages, k_scale, v_scale, table, lengths)
    dt = _need(q, op, "q", 3, (float16, bfloat16))
    B, ldq = int(q.shape[0]), int(q.shape[1]) * hd
    h = int(q.shape[1]) if heads is None else heads
    if not 0 < h <= q.shape[1]:
        raise ValueError(f"{op}: {h} heads of q {tuple(q.shape)}")
    if q.shape[2] != hd or B != table.shape[0] or h % hkv:
        raise ValueError(f"{op}: q {tuple(q.shape)} does not fit {table.shape[0]} sequences, {hkv} key heads of {hd}")
    if k_pages.dtype not in (dt, np.dtype(np.int8)):
        raise TypeError(f"{op}: a cache of {k_pages.dtype} for queries of {dt}")
    stream = _stream(stream, k_scale, v_scale)
    out = empty((B, h, hd), _out_type(out_dtype, dt, op), "gpu", stream)
    size = _C.lib().lq_paged_attention_workspace_size(B, h, hkv, hd, max_length)
    ws, _held = _scratch(size, stream)
    _C.call("lq_paged_attention", q.data_ptr(), FLOAT_TYPE_CODE[dt], ldq, B, h, hkv, hd, k_pages.data_ptr(),
            v_pages.data_ptr(), _CACHE_TYPE[k_pages.dtype], _opt(k_scale), _opt(v_scale), pages, page, table.data_ptr(),
            table.shape[1], lengths.data_ptr(), max_length, _scale(scale, hd, op), out.data_ptr(),
            FLOAT_TYPE_CODE[out.dtype], ws, size, stream)
    return out


def prompt_attention(q: Tensor, k: Tensor, v: Tensor, q_starts: Tensor, k_starts: Tensor | None = None,
                     causal: bool = True, scale: float | None = None, out_dtype=None, stream=None) -> Tensor:
    """Attention over packed sequences: ``q`` [tokens, heads, head_dim], ``k`` / ``v`` [tokens,
    kv_heads, head_dim], ``q_starts`` / ``k_starts`` [seqs + 1] (the same for both unless given).
    Rows of the result that belong to no sequence (before the first start, past the last) are not
    written and hold whatever the memory held.  See ``lq_prompt_attention``."""
    op = "prompt_attention"
    dt = _need(q, op, "q", 3, (float16, bfloat16))
    _need(k, op, "k", 3, (dt,))
    _need(v, op, "v", 3, (dt,))
    total, h, hd = (int(n) for n in q.shape)
    if tuple(k.shape) != tuple(v.shape) or k.shape[2] != hd or not k.shape[1] or h % k.shape[1]:
        raise ValueError(f"{op}: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit")
    hkv = int(k.shape[1])
    return _prompt(op, q.data_ptr(), h * hd, k.data_ptr(), hkv * hd, v.data_ptr(), hkv * hd, dt, q_starts, k_starts,
                   total, int(k.shape[0]), h, hkv, hd, causal, scale, out_dtype, stream)


def prompt_attention_qkv(qkv: Tensor, heads: int, kv_heads: int, starts: Tensor, causal: bool = True,
                         scale: float | None = None, out_dtype=None, stream=None) -> Tensor:
    """:func:`prompt_attention` of a fused projection's rows ``[tokens, heads + 2 kv_heads,
    head_dim]``, read in place.  Rows of no sequence are not written."""
    op = "prompt_attention_qkv"
    dt = _need(qkv, op, "qkv", 3, (float16, bfloat16))
    if kv_heads < 1 or heads < 1 or heads % kv_heads or qkv.shape[1] != heads + 2 * kv_heads:
        raise ValueError(f"{op}: qkv {tuple(qkv.shape)} for {heads} heads and {kv_heads} key heads")
    total, hd = int(qkv.shape[0]), int(qkv.shape[2])
    ld, q = (heads + 2 * kv_heads) * hd, qkv.data_ptr()
    k = q + 2 * heads * hd
    return _prompt(op, q, ld, k, ld, k + 2 * kv_heads * hd, ld, dt, starts, None, total, total, heads, kv_heads, hd,
                   causal, scale, out_dtype, stream)


def _prompt(op, q, ldq, k, ldk, v, ldv, dt, q_starts, k_starts, total_q, total_k, h, hkv, hd, causal, scale, out_dtype,
            stream) -> Tensor:
    _ints(q_starts, op, "q_starts")
    k_starts = q_starts if k_starts is None else _ints(k_starts, op, "k_starts", q_starts.shape[0])
    if q_starts.shape[0] < 1:
        raise ValueError(f"{op}: starts hold one number more than there are sequences")
    stream = _stream(stream)
    out = empty((total_q, h, hd), _out_type(out_dtype, dt, op), "gpu", stream)
    _C.call("lq_prompt_attention", q, ldq, k, ldk, v, ldv, FLOAT_TYPE_CODE[dt], q_starts.data_ptr(), k_starts.data_ptr(),
            int(q_starts.shape[0]) - 1, total_q, total_k, h, hkv, hd, 1 if causal else 0, _scale(scale, hd, op),
            out.data_ptr(), FLOAT_TYPE_CODE[out.dtype], stream)
    return out


def token_logprobs(logits: Tensor, targets: Tensor, top: int = 0, stream=None):
    """``(logprobs, entropy, lse, top_logprobs, top_ids)`` of ``targets`` [rows] under ``logits``
    [rows, vocab]; the last two are ``[rows, top]``.  See ``lq_token_logprobs``."""
    op = "token_logprobs"
    dt = _need(logits, op, "logits", 2, tuple(FLOAT_TYPE_CODE))
    rows, vocab = int(logits.shape[0]), int(logits.shape[1])
    _ints(targets, op, "targets", rows)
    if not 0 <= top <= min(vocab, 64):
        raise ValueError(f"{op}: top must be within [0, {min(vocab, 64)}], got {top}")
    stream = _stream(stream, logits)
    lp, ent, lse = (empty((rows,), float32, "gpu", stream) for _ in range(3))
    top_lp, top_ids = empty((rows, top), float32, "gpu", stream), empty((rows, top), np.int32, "gpu", stream)
    size = _C.lib().lq_token_logprobs_workspace_size(rows, vocab, top)
    ws, _held = _scratch(size, stream)
    _C.call("lq_token_logprobs", logits.data_ptr(), FLOAT_TYPE_CODE[dt], vocab, rows, vocab, targets.data_ptr(), top,
            lp.data_ptr(), ent.data_ptr(), lse.data_ptr(), top_lp.data_ptr(), top_ids.data_ptr(), ws, size,
            stream)
    return lp, ent, lse, top_lp, top_ids


def token_logprobs_backward(logits: Tensor, targets: Tensor, lse: Tensor, g_logprobs: Tensor,
                            entropy: Tensor | None = None, g_entropy: Tensor | None = None, stream=None) -> Tensor:
    """The gradient in ``logits`` of ``sum(g_logprobs * logprobs)``, plus ``sum(g_entropy *
    entropy)`` where ``g_entropy`` and the forward's ``entropy`` are given, of the logits' type.
    See ``lq_token_logprobs_backward``."""
    op = "token_logprobs_backward"
    dt = _need(logits, op, "logits", 2, tuple(FLOAT_TYPE_CODE))
    rows, vocab = int(logits.shape[0]), int(logits.shape[1])
    _ints(targets, op, "targets", rows)
    if g_entropy is not None and entropy is None:
        raise ValueError(f"{op}: g_entropy needs the forward's entropy")
    for name, t in (("lse", lse), ("g_logprobs", g_logprobs), ("entropy", entropy), ("g_entropy", g_entropy)):
        if t is not None:
            _need(t, op, name, 1, (float32,))
            if t.shape[0] != rows:
                raise ValueError(f"{op}: {name} must hold {rows} numbers, got {t.shape[0]}")
    stream = _stream(stream, logits, lse, g_logprobs, entropy, g_entropy)
    grad = empty((rows, vocab), dt, "gpu", stream)
    _C.call("lq_token_logprobs_backward", logits.data_ptr(), FLOAT_TYPE_CODE[dt], vocab, rows, vocab,
            targets.data_ptr(), lse.data_ptr(), _opt(entropy) if g_entropy is not None else None,
            g_logprobs.data_ptr(), _opt(g_entropy), grad.data_ptr(), vocab, stream)
    return grad


# --------------------------------------------------------------------------- the cache


class PageTable:
    """Which pages each of ``seqs`` sequences holds, shared by the caches of a model's layers.

    ``table`` [seqs, per_seq] and ``lengths`` [seqs] are device int32 tensors that keep their
    address, so captured graphs read the current state; the host keeps the free pages.

    Everything that reads or writes the caches of a table runs on one stream, and ``grow`` and
    ``release`` are given that stream: they change the table and the lengths in place behind what is
    queued there, and a released page's next owner writes it behind the last reader."""

    def __init__(self, seqs: int, pages: int, page: int = 64, max_length: int | None = None) -> None:
        if seqs < 1 or pages < 1 or page < 1:
            raise ValueError(f"PageTable: {seqs} sequences, {pages} pages of {page}")
        self.seqs, self.pages, self.page = seqs, pages, page
        per = pages if max_length is None else -(-max_length // page)
        self._table = np.zeros((seqs, per), np.int32)
        self._lengths = np.zeros((seqs,), np.int32)
        self._held = [0] * seqs
        self._free = list(range(pages - 1, -1, -1))
        self.table = tensor(self._table, device="gpu")
        self.lengths = tensor(self._lengths, device="gpu")

    @property
    def max_length(self) -> int:
        """The longest sequence now."""
        return int(self._lengths.max())

    def host_lengths(self) -> np.ndarray:
        return self._lengths.copy()

    def rows(self, seqs, stream=None) -> tuple[Tensor, Tensor]:
        """Copies of some sequences' table rows and lengths, for work on ``stream``."""
        stream, copies = _stream(stream), []
        for a in (np.ascontiguousarray(self._table[seqs]), np.ascontiguousarray(self._lengths[seqs])):
            copies.append(empty(a.shape, a.dtype, "gpu", stream))
            _C.call("lq_memcpy_h2d", copies[-1].data_ptr(), a.ctypes.data, a.nbytes, stream)
        return copies[0], copies[1]

    def grow(self, counts, stream=None) -> None:
        """``counts[s]`` more positions for every sequence: takes pages as needed and uploads the
        table and the lengths, on ``stream``.  Nothing changes when the free pages do not suffice."""
        counts = np.asarray(counts, np.int64)
        if counts.shape != (self.seqs,) or (counts < 0).any():
            raise ValueError(f"PageTable.grow: {self.seqs} counts of 0 or more expected")
        new = self._lengths + counts
        need = [-(-int(n) // self.page) for n in new]
        if max(need) > self._table.shape[1]:
            raise ValueError(f"PageTable.grow: a sequence of {int(new.max())} positions needs {max(need)} pages, its "
                             f"row holds {self._table.shape[1]}")
        more = sum(n - h for n, h in zip(need, self._held))
        if more > len(self._free):
            raise MemoryError(f"PageTable.grow: {more} pages needed, {len(self._free)} free")
        for s, n in enumerate(need):
            while self._held[s] < n:
                self._table[s, self._held[s]] = self._free.pop()
                self._held[s] += 1
        self._lengths = new.astype(np.int32)
        self._upload(more > 0, stream)

    def shrink(self, counts, stream=None) -> None:
        """``counts[s]`` positions fewer at every sequence's end; its pages stay with it."""
        new = self._lengths - np.asarray(counts, np.int64)
        if new.shape != (self.seqs,) or (new < 0).any() or (new > self._lengths).any():
            raise ValueError(f"PageTable.shrink: {self.seqs} counts of 0 to the lengths expected")
        self._lengths = new.astype(np.int32)
        self._upload(False, stream)

    def release(self, s: int, stream=None) -> None:
        """Sequence ``s`` ends: its pages are free again and its length is 0, on ``stream``."""
        if not 0 <= s < self.seqs:
            raise ValueError(f"PageTable.release: sequence {s} of {self.seqs}")
        self._free.extend(int(p) for p in self._table[s, :self._held[s]][::-1])
        self._held[s] = 0
        self._lengths[s] = 0
        self._upload(False, stream)

    def _upload(self, table: bool, stream) -> None:
        stream = _stream(stream)
        if table:
            _C.call("lq_memcpy_h2d", self.table.data_ptr(), self._table.ctypes.data, self._table.nbytes, stream)
        _C.call("lq_memcpy_h2d", self.lengths.data_ptr(), self._lengths.ctypes.data, self._lengths.nbytes, stream)


class PagedKVCache:
    """One layer's pages over a :class:`PageTable`: ``append`` what the projection made, then
    ``attend`` with the step's queries, on the stream that the table is grown on.  ``dtype`` float16, bfloat16 or int8 (codes with one
    scale per row)."""

    def __init__(self, table: PageTable, kv_heads: int, head_dim: int, dtype=float16) -> None:
        dt = np.dtype(dtype)
        if dt not in _CACHE_TYPE:
            raise TypeError(f"PagedKVCache: dtype must be float16, bfloat16 or int8, got {dt}")
        self.pages, shape = table, (table.pages, kv_heads, table.page, head_dim)
        self.k, self.v = empty(shape, dt, "gpu"), empty(shape, dt, "gpu")
        self.k_scale = self.v_scale = None
        if dt == np.int8:
            self.k_scale, self.v_scale = empty(shape[:3], float32, "gpu"), empty(shape[:3], float32, "gpu")

    def append(self, k: Tensor, v: Tensor, starts: Tensor | None = None, stream=None) -> None:
        paged_kv_append(k, v, self.k, self.v, self.pages.table, self.pages.lengths, starts, self.k_scale, self.v_scale,
                        stream)

    def append_qkv(self, qkv: Tensor, heads: int, starts: Tensor | None = None, stream=None) -> None:
        paged_kv_append_qkv(qkv, heads, self.k, self.v, self.pages.table, self.pages.lengths, starts, self.k_scale,
                            self.v_scale, stream)

    def attend(self, q: Tensor, scale: float | None = None, out_dtype=None, max_length: int | None = None,
               stream=None, heads: int | None = None) -> Tensor:
        return paged_attention(q, self.k, self.v, self.pages.table, self.pages.lengths,
                               self.pages.max_length if max_length is None else max_length, scale, self.k_scale,
                               self.v_scale, out_dtype, stream, heads)
