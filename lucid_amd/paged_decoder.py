"""A decoder that serves sequences of different lengths from a paged key-value cache.

:class:`PagedDecoder` runs the dynamically quantized decoder of
:func:`lucid_amd.bench_configs.decoder` (6 layers, d 512, 8 heads, FFN 2048, vocab 32000)
through its modules: prompts of any lengths enter packed (``F.prompt_attention_qkv``), their
keys and values go to pages (``F.paged_kv_append_qkv``), every step attends them
(``F.paged_attention``), ended sequences give their pages back, and ``F.token_logprobs`` gives
the tokens' scores and alternatives.  :meth:`PagedDecoder.tune` is the training direction: the
gradient of weighted token scores and entropies in the head's logits
(``F.token_logprobs_backward``) and in its bias.

``python3 -m lucid_amd.paged_decoder [steps]`` serves eight prompts and prints what it took.
"""

from __future__ import annotations

import numpy as np

import lucid_amd.nn.functional as F
from lucid_amd import _C
from lucid_amd._tensor import Tensor, empty, float16, float32, tensor
from lucid_amd.bench_configs import D_MODEL, HEADS
from lucid_amd.nn.generation import PagedKVCache, PageTable


def _ints(a) -> Tensor:
    return tensor(np.ascontiguousarray(a, np.int32), device="gpu")


class PagedDecoder:
    """``qdec`` (``quantize_dynamic`` of the decoder) and its embeddings ``glue``, serving up to
    ``seqs`` sequences at a time from ``pages`` pages of ``page`` positions per layer;
    ``cache_dtype`` float16 or int8.  One stream: everything runs on the default one."""

    def __init__(self, qdec, glue: dict, seqs: int, pages: int, page: int = 16, cache_dtype=float16) -> None:
        self.qdec = qdec
        self.tok, self.pos = (tensor(np.ascontiguousarray(glue[n]), device="gpu") for n in ("tok", "pos"))
        self.vocab, self.positions = glue["tok"].shape[0], glue["pos"].shape[0]
        self.head_dim = D_MODEL // HEADS
        self.table = PageTable(seqs, pages, page, self.positions)
        self.cache = [PagedKVCache(self.table, HEADS, self.head_dim, cache_dtype) for _ in qdec.layers]

    # ------------------------------------------------------------------ the layers

    def _norm(self, x: Tensor, res: Tensor | None = None) -> Tensor:
        """The layer norm of ``x``, to which ``res`` is added first (in place)."""
        y, rows = empty(x.shape, float32, "gpu"), int(x.shape[0])
        if res is None:
            _C.call("lq_layer_norm_f32", x.data_ptr(), D_MODEL, y.data_ptr(), D_MODEL, rows, D_MODEL, None, None,
                    np.float32(1e-5), None)
        else:
            _C.call("lq_add_layer_norm_f32", x.data_ptr(), D_MODEL, res.data_ptr(), D_MODEL, y.data_ptr(), D_MODEL,
                    rows, D_MODEL, None, None, np.float32(1e-5), None)
        return y

    def _hidden(self, ids: np.ndarray, positions: np.ndarray, attend) -> Tensor:
        """The last norm's rows for packed tokens; ``attend(layer, qkv)`` is the attention of
        fp16 rows ``[tokens, 3 heads, head_dim]``, float32 out."""
        rows = len(ids)
        x, p = F.embedding(_ints(ids), self.tok), F.embedding(_ints(positions), self.pos)
        _C.call("lq_add_f32", x.data_ptr(), p.data_ptr(), x.data_ptr(), rows * D_MODEL, None)
        res = None
        for i, layer in enumerate(self.qdec.layers):
            qkv = layer.qkv(self._norm(x, res)).to(dtype=float16).reshape(rows, 3 * HEADS, self.head_dim)
            res = layer.out(attend(i, qkv).reshape(rows, D_MODEL))
            up = layer.up(self._norm(x, res))
            _C.call("lq_gelu_tanh_f32", up.data_ptr(), up.data_ptr(), up.numel(), None)
            res = layer.down(up)
        return self._norm(x, res)

    @staticmethod
    def _rows(x: Tensor, rows: np.ndarray) -> Tensor:
        """Some rows of a [rows, D] tensor."""
        return F.embedding(_ints(rows), x)

    def _check(self, prompts) -> list[np.ndarray]:
        out = [np.asarray(p, np.int64).ravel() for p in prompts]
        for p in out:
            self._known(p, "prompt")
            if len(p) > self.positions:
                raise ValueError(f"a prompt of {len(p)} tokens, {self.positions} positions")
        return [p.astype(np.int32) for p in out]

    def _known(self, ids: np.ndarray, what: str) -> None:
        if len(ids) and (ids.min() < 0 or ids.max() >= self.vocab):
            raise ValueError(f"{what} token ids out of the vocabulary")

    def _sequences(self, keys) -> list[int]:
        seqs = sorted(keys)
        if seqs and (seqs[0] < 0 or seqs[-1] >= self.table.seqs):
            raise ValueError(f"sequences {seqs}: this decoder serves 0 .. {self.table.seqs - 1}")
        return seqs

    # ------------------------------------------------------------------ serving

    def prefill(self, prompts: dict[int, np.ndarray]) -> Tensor:
        """Prompts into the empty sequences they are keyed by; the logits ``[len(prompts),
        vocab]`` after each, in the order of the sequences."""
        seqs = self._sequences(prompts)
        toks = dict(zip(seqs, self._check([prompts[s] for s in seqs])))
        held = self.table.host_lengths()
        for s in seqs:
            if held[s] or not len(toks[s]):
                raise ValueError(f"sequence {s} holds {held[s]} positions; its prompt has {len(toks[s])} tokens")
        counts = np.zeros(self.table.seqs, np.int64)
        for s in seqs:
            counts[s] = len(toks[s])
        self.table.grow(counts)
        ends = np.cumsum(counts)
        starts = _ints(np.concatenate([[0], ends]))

        def attend(i, qkv):
            self.cache[i].append_qkv(qkv, HEADS, starts)
            return F.prompt_attention_qkv(qkv, HEADS, HEADS, starts, out_dtype=float32)

        try:
            h = self._hidden(np.concatenate([toks[s] for s in seqs]),
                             np.concatenate([np.arange(len(toks[s])) for s in seqs]), attend)
            return self.qdec.head(self._rows(h, ends[seqs] - 1))
        except BaseException:  # their positions hold nothing
            for s in seqs:
                self.table.release(s)
            raise

    def step(self, tokens: dict[int, int]) -> Tensor:
        """One token more for some of the sequences; the logits ``[len(tokens), vocab]``, in the
        order of the sequences."""
        seqs = self._sequences(tokens)
        held = self.table.host_lengths()
        if any(held[s] == 0 or held[s] >= self.positions for s in seqs):
            raise ValueError("a step needs sequences that hold something and have a position left")
        ids = np.array([tokens[s] for s in seqs], np.int64)
        self._known(ids, "step")
        counts = np.zeros(self.table.seqs, np.int64)
        counts[seqs] = 1
        self.table.grow(counts)
        starts = _ints(np.concatenate([[0], np.cumsum(counts)]))
        whole = len(seqs) == self.table.seqs

        def attend(i, qkv):
            cache = self.cache[i]
            cache.append_qkv(qkv, HEADS, starts)
            if whole:
                return cache.attend(qkv, out_dtype=float32, heads=HEADS)
            return F.paged_attention(qkv, cache.k, cache.v, table, lengths, self.table.max_length, None, cache.k_scale,
                                     cache.v_scale, float32, None, HEADS)

        try:
            if not whole:  # the stepping sequences' rows of the table
                table, lengths = self.table.rows(seqs)
            return self.qdec.head(self._hidden(ids, held[seqs], attend))
        except BaseException:  # the last positions hold nothing
            self.table.shrink(counts)
            raise

    def generate(self, prompts: list, steps: int, top: int = 5):
        """Greedy continuations of up to ``seqs`` prompts: tokens ``[len(prompts), steps]``, their
        log probabilities, and the alternatives' ids ``[len(prompts), steps, top]``."""
        n = len(prompts)
        logits = self.prefill(dict(enumerate(prompts)))
        out, scores, others = [], [], []
        try:
            for k in range(steps):
                for kept, new in zip((out, scores, others), self._choose(logits, n, top)):
                    kept.append(new)
                if k + 1 < steps:
                    logits = self.step(dict(enumerate(out[-1].tolist())))
        finally:
            for s in range(n):
                self.table.release(s)
        return np.stack(out, 1), np.stack(scores, 1), np.stack(others, 1)

    def _choose(self, logits: Tensor, n: int, top: int):
        """The most likely tokens after ``n`` sequences, their log probabilities, the alternatives' ids."""
        best = empty((n,), np.int32, "gpu")
        _C.call("lq_argmax_f32", logits.data_ptr(), n, self.vocab, best.data_ptr(), None)
        lp, _, _, _, ids = F.token_logprobs(logits, best, top)
        return best.numpy(), lp.numpy(), ids.numpy()

    # ------------------------------------------------------------------ scoring and tuning

    def _score_rows(self, prompts):
        toks = self._check(prompts)
        starts = _ints(np.cumsum([0] + [len(t) for t in toks]))
        h = self._hidden(np.concatenate(toks), np.concatenate([np.arange(len(t)) for t in toks]),
                         lambda i, qkv: F.prompt_attention_qkv(qkv, HEADS, HEADS, starts, out_dtype=float32))
        # a row predicts the token after it; the last row of a prompt predicts none
        targets = np.concatenate([np.append(t[1:], -100) if len(t) else t for t in toks])
        return self.qdec.head(h), _ints(targets)

    def score(self, prompts: list, top: int = 0):
        """``F.token_logprobs`` of every prompt's tokens under those before them, packed (the last
        row of a prompt has no target: log probability 0)."""
        logits, targets = self._score_rows(prompts)
        return F.token_logprobs(logits, targets, top)

    def tune(self, prompts: list, weights: np.ndarray, entropy_weight: float = 0.0):
        """The objective ``sum(weights * logprobs) + entropy_weight * sum(entropy)`` over the
        packed rows of ``prompts``, its gradient in the logits (device) and in the head's bias
        (host)."""
        logits, targets = self._score_rows(prompts)
        rows = int(logits.shape[0])
        weights = np.ascontiguousarray(weights, np.float32).reshape(rows)
        lp, ent, lse, _, _ = F.token_logprobs(logits, targets)
        g, ge = (tensor(a, device="gpu") for a in (weights, np.full(rows, entropy_weight, np.float32)))
        grad = F.token_logprobs_backward(logits, targets, lse, g, ent, ge)
        value = float((weights * lp.numpy()).sum(dtype=np.float64) + entropy_weight * ent.numpy().sum(dtype=np.float64))
        return value, grad, grad.numpy().sum(0, dtype=np.float64)


def _main(argv: list[str]) -> None:
    import time

    import lucid_amd.backends as backends
    from lucid_amd.bench_configs import VOCAB, decoder
    from lucid_amd.quantization import quantize_dynamic

    steps = int(argv[0]) if argv else 32
    backends.quantized.engine = "reference"  # the per-channel int8 layers
    rng = np.random.default_rng(7)
    dec, glue = decoder(rng)
    rt = PagedDecoder(quantize_dynamic(dec), glue, seqs=8, pages=8 * 40)
    prompts = [rng.integers(0, VOCAB, n) for n in (512, 300, 1, 77, 160, 31, 16, 450)]
    rt.generate(prompts, 2)
    t0 = time.perf_counter()
    toks, scores, _ = rt.generate(prompts, steps)
    dt = time.perf_counter() - t0
    rows = sum(map(len, prompts))
    print(f"{len(prompts)} prompts of {rows} tokens and {toks.size} generated tokens: {dt * 1e3:.1f} ms; "
          f"mean log probability {scores.mean():.3f}")
    value, _, bias = rt.tune(prompts, np.ones(rows) / rows, 0.01 / rows)
    print(f"objective {value:.4f}, largest bias gradient {np.abs(bias).max():.3e}")


if __name__ == "__main__":
    import sys

    _main(sys.argv[1:])
