"""Operators that serve ragged sequences from a paged key-value cache, as cases that can be timed and compared.

* ``append``: the keys and values of new tokens into the pages of their sequences;
* ``paged``: attention of one new token per sequence over its pages;
* ``prompt``: causal attention over packed prompts of different lengths, with grouped heads;
* ``logprobs``: log probabilities of given tokens, entropy and the best alternatives;
* ``logprobs_backward``: the gradient of the last in the logits.

``run()`` computes them from their formulas with elementary torch operations where ``own`` is false and
calls the C ABI of ``include/lq_api.h`` where it is true.  ``exact()`` is the definition in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPE = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
CODE = {"float32": 6, "float16": 5, "bfloat16": 10, "int8": 1}  # element types of include/lq_api.h
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2, "int8": 1}


def listed():
    return [
        # one decode step of the framework's own decoder: 8 sequences, 8 heads of 64, a float32 projection
        {"name": "append_step_b8", "kind": "append", "seqs": 8, "longest": 640, "step": True, "kv_heads": 8,
         "head_dim": 64, "page": 16, "source": "float32", "cache": "float16", "mix": 1},
        # prompts of a serving batch as they arrive: 1 to 4096 tokens, some after a cached prefix
        {"name": "append_prompts_16", "kind": "append", "seqs": 16, "longest": 4096, "step": False, "kv_heads": 8,
         "head_dim": 128, "page": 64, "source": "bfloat16", "cache": "bfloat16", "mix": 2},
        # the attention of the decoder's step: positions up to 640, float32 out for the dynamic input step
        {"name": "paged_step_b8", "kind": "paged", "seqs": 8, "longest": 640, "heads": 8, "kv_heads": 8,
         "head_dim": 64, "page": 16, "dtype": "float16", "cache": "float16", "out": "float32", "mix": 3},
        # a full serving batch, grouped heads, ragged lengths
        {"name": "paged_ragged_b64", "kind": "paged", "seqs": 64, "longest": 8191, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 64, "dtype": "bfloat16", "cache": "bfloat16", "out": "bfloat16", "mix": 4},
        # two long documents on an int8 cache: few rows, a long axis
        {"name": "paged_long_int8_b2", "kind": "paged", "seqs": 2, "longest": 131071, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 128, "dtype": "float16", "cache": "int8", "out": "float16", "mix": 5},
        # the decoder's prefill: 8 prompts of at most 512 tokens, q / k / v in one projection, float32 out
        {"name": "prompt_b8_512", "kind": "prompt", "seqs": 8, "longest": 512, "heads": 8, "kv_heads": 8,
         "head_dim": 64, "dtype": "float16", "out": "float32", "fused": True, "mix": 6},
        # a serving batch of ragged prompts with grouped heads
        {"name": "prompt_ragged_b12", "kind": "prompt", "seqs": 12, "longest": 4000, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "dtype": "bfloat16", "out": "bfloat16", "fused": True, "mix": 7},
        # one long prompt
        {"name": "prompt_long_b1", "kind": "prompt", "seqs": 1, "longest": 12288, "heads": 32, "kv_heads": 4,
         "head_dim": 128, "dtype": "bfloat16", "out": "bfloat16", "fused": False, "mix": 8},
        # the decoder's step: its logits, the sampled tokens' scores and five alternatives
        {"name": "logprobs_step_b8", "kind": "logprobs", "rows": 8, "vocab": 32000, "dtype": "float32", "top": 5,
         "masked": False},
        # scoring prompts under a vocabulary of odd length, part of it masked out
        {"name": "logprobs_score_4096", "kind": "logprobs", "rows": 4096, "vocab": 100003, "dtype": "bfloat16",
         "top": 8, "masked": True},
        # a small tuning batch: the gradient of the tokens' log probabilities alone
        {"name": "backward_b64", "kind": "logprobs_backward", "rows": 64, "vocab": 32000, "dtype": "float32",
         "entropy": False},
        # a large tuning batch with an entropy term
        {"name": "backward_8192", "kind": "logprobs_backward", "rows": 8192, "vocab": 32000, "dtype": "bfloat16",
         "entropy": True},
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], even in its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("append", "paged", "paged", "prompt", "prompt", "logprobs", "logprobs_backward"))
    mix, dtype = rng.randrange(1 << 20), rng.choice(("float16", "bfloat16"))
    kv = rng.choice((1, 2, 4, 8, rng.randint(1, 8)))
    hd = rng.choice((64, 64, 128, 128, 128, 8 * rng.randint(4, 32)))
    page = 1 << rng.randint(3, 8)
    if kind == "append":
        step = rng.random() < 0.5
        return {"kind": kind, "seqs": _log(rng, 1, 256) if step else rng.randint(1, 16),
                "longest": _log(rng, 8, 4096), "step": step, "kv_heads": kv, "head_dim": min(hd, 128), "page": page,
                "source": rng.choice(("float32", dtype)), "cache": dtype, "mix": mix}
    if kind == "paged":
        seqs = _log(rng, 1, 128)
        group = rng.choice((1, 2, 4, 8, rng.randint(1, 16)))
        longest = _log(rng, 1, min(131072, 64 * 8192 * 8 * 128 // (seqs * kv * hd)))
        return {"kind": kind, "seqs": seqs, "longest": longest, "heads": kv * group, "kv_heads": kv, "head_dim": hd,
                "page": page, "dtype": dtype, "cache": rng.choice((dtype, dtype, "int8")),
                "out": rng.choice((dtype, dtype, "float32")), "mix": mix}
    if kind == "prompt":
        group = rng.choice((1, 2, 4, 8, rng.randint(1, 8)))
        seqs = _log(rng, 1, 64)
        longest = _log(rng, 1, min(8192, int(math.sqrt((1 << 31) / (seqs * kv * group)))))
        return {"kind": kind, "seqs": seqs, "longest": longest, "heads": kv * group, "kv_heads": kv, "head_dim": hd,
                "dtype": dtype, "out": rng.choice((dtype, dtype, "float32")), "fused": rng.random() < 0.5, "mix": mix}
    rows = _log(rng, 1, 4096)
    vocab = _log(rng, 128, min(200000, 262144 * 1024 // rows))
    if kind == "logprobs":
        return {"kind": kind, "rows": rows, "vocab": vocab, "dtype": rng.choice(("float32", dtype)),
                "top": rng.choice((0, 1, 5, rng.randint(1, 32))), "masked": rng.random() < 0.5}
    return {"kind": kind, "rows": rows, "vocab": vocab, "dtype": rng.choice(("float32", dtype)),
            "entropy": rng.random() < 0.5}


# ------------------------------------------------------------------------------ inputs


def _lengths(case):
    """The sequences' lengths: the longest first, one of a single token, the rest spread between."""
    rng, n = random.Random(case["mix"]), case["longest"]
    lens = [_log(rng, max(1, n // 32), n) for _ in range(case["seqs"])]
    lens[0] = n
    if len(lens) > 2:
        lens[2] = 1
    return lens


def _new(case, lens):
    """How many of each sequence's positions are new: one in a step, else all or what follows a prefix."""
    if case["step"]:
        return [1] * len(lens)
    return [n if i % 3 else max(1, n - n // 4) for i, n in enumerate(lens)]


def _pages(lens, page):
    return [-(-n // page) for n in lens]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind = case["kind"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    def starts(values):
        return ints([sum(values[:i]) for i in range(len(values) + 1)])

    if kind in ("append", "paged"):
        lens, hkv, hd, ps = _lengths(case), case["kv_heads"], case["head_dim"], case["page"]
        used = _pages(lens, ps)
        pool = sum(used) + 4
        ids = torch.randperm(pool, generator=g, device="cuda")[:sum(used)].to(torch.int32)
        table = torch.zeros((len(lens), max(used)), dtype=torch.int32, device="cuda")
        at = torch.arange(max(used), device="cuda")[None, :] < ints(used)[:, None]
        table[at] = ids
        s = {"case": case, "table": table, "lengths": ints(lens), "pool": pool}
        shape = (pool, hkv, ps, hd)
        if kind == "append":
            new = _new(case, lens)
            s["starts"] = starts(new)
            # one projection's rows: keys, then values
            s["kv"] = normal(sum(new), 2, hkv, hd).to(DTYPE[case["source"]])
            s["k"] = torch.zeros(shape, dtype=DTYPE[case["cache"]], device="cuda")
            s["v"] = torch.zeros(shape, dtype=DTYPE[case["cache"]], device="cuda")
            return s
        # keys with a few strong channels, as projections have them
        strong = 1.0 + 3.0 * (torch.rand((hkv, 1, hd), generator=g, device="cuda") < 1 / 32)
        if case["cache"] == "int8":
            for name, wide in (("k", strong), ("v", 1.0)):
                x = normal(*shape) * wide
                top = x.abs().amax(-1)
                s[name] = (x * (127 / top)[..., None]).round().to(torch.int8)
                s[name + "_scale"] = top / 127
        else:
            s["k"] = (normal(*shape) * strong).to(DTYPE[case["cache"]])
            s["v"] = normal(*shape).to(DTYPE[case["cache"]])
        s["q"] = normal(len(lens), case["heads"], hd).to(DTYPE[case["dtype"]])
        s["out"] = torch.empty((len(lens), case["heads"], hd), dtype=DTYPE[case["out"]], device="cuda")
        return s
    if kind == "prompt":
        lens, h, hkv, hd = _lengths(case), case["heads"], case["kv_heads"], case["head_dim"]
        total = sum(lens)
        strong = 1.0 + 3.0 * (torch.rand((hkv, hd), generator=g, device="cuda") < 1 / 32)
        q, k, v = normal(total, h, hd), normal(total, hkv, hd) * strong, normal(total, hkv, hd)
        if case["fused"]:  # one projection's rows: queries, keys, values
            qkv = torch.cat([q, k, v], 1).to(DTYPE[case["dtype"]])
            q, k, v = qkv[:, :h], qkv[:, h:h + hkv], qkv[:, h + hkv:]
        else:
            q, k, v = (t.to(DTYPE[case["dtype"]]) for t in (q, k, v))
        out = torch.empty((total, h, hd), dtype=DTYPE[case["out"]], device="cuda")
        return {"case": case, "q": q, "k": k, "v": v, "starts": starts(lens), "out": out}
    rows, vocab = case["rows"], case["vocab"]
    # logits of a model that has learned something: a few likely tokens over a broad rest
    x = normal(rows, vocab).mul_(2.5)
    likely = torch.randint(0, vocab, (rows, 4), generator=g, device="cuda")
    x.scatter_add_(1, likely, 8 + 4 * torch.rand((rows, 4), generator=g, device="cuda"))
    if case.get("masked"):  # half of the rows allow one token in four, as a grammar does
        banned = torch.rand((rows, vocab), generator=g, device="cuda") < 0.75
        banned[::2] = False
        banned.scatter_(1, likely, False)
        x.masked_fill_(banned, -math.inf)
    x = x.to(DTYPE[case["dtype"]])
    targets = likely[:, 0].to(torch.int32)
    targets[5::7] = -100  # prompt tokens carry no loss
    s = {"case": case, "logits": x, "targets": targets}
    f32 = dict(dtype=torch.float32, device="cuda")
    if kind == "logprobs":
        top = case["top"]
        s.update(logprobs=torch.empty(rows, **f32), entropy=torch.empty(rows, **f32), lse=torch.empty(rows, **f32),
                 top_logprobs=torch.empty((rows, top), **f32),
                 top_ids=torch.empty((rows, top), dtype=torch.int32, device="cuda"))
        return s
    parts = [_row_sums(rows_of.double()) for rows_of in x.split(256)]
    s.update(lse=torch.cat([p[0] for p in parts]).float(), entropy=torch.cat([p[1] for p in parts]).float(),
             g_logprobs=normal(rows), g_entropy=normal(rows) * 0.1, grad=torch.empty_like(x))
    return s


def _row_sums(x):
    """(lse, entropy) of logit rows, as the forward pass left them."""
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(1)
    return m[:, 0] + total.log(), total.log() - (e * (x - m)).sum(1) / total


# ------------------------------------------------------------------------------ one pass


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        return _run_own(s, case, kind)
    if kind == "append":
        return _append(s, case)
    if kind == "paged":
        return _paged(s, case)
    if kind == "prompt":
        return _prompt(s, case)
    if kind == "logprobs":
        return _logprobs(s, case)
    return _logprobs_backward(s, case)


def _token_places(starts, total):
    """The sequence of each packed token and its place there."""
    t = torch.arange(total, device=starts.device, dtype=torch.int32)
    seq = torch.searchsorted(starts, t, right=True) - 1
    return seq, t - starts[seq]


def _append(s, case):
    starts, kv, ps = s["starts"], s["kv"], case["page"]
    seq, i = _token_places(starts, kv.shape[0])
    pos = s["lengths"][seq] - (starts[seq + 1] - starts[seq]) + i
    page, slot = s["table"][seq, pos // ps].long(), (pos % ps).long()
    s["k"][page, :, slot] = kv[:, 0].to(s["k"].dtype)
    s["v"][page, :, slot] = kv[:, 1].to(s["v"].dtype)
    return s["k"], s["v"]


def _softmax(scores, seen):
    """Weights over the last axis of the scores that are seen; a row that sees nothing has none."""
    scores = scores.masked_fill(~seen, -math.inf)
    m = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(m == -math.inf, torch.zeros_like(m), m))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-37)


def _paged(s, case):
    B, h, hd = s["q"].shape
    hkv, ps = case["kv_heads"], case["page"]

    def rows(name):  # a sequence's pages in order, [B, hkv, positions, hd] in 32 bits
        x = s[name][s["table"].long()].float()
        if case["cache"] == "int8":
            x = x * s[name + "_scale"][s["table"].long()][..., None]
        return x.transpose(1, 2).reshape(B, hkv, -1, hd)

    q = s["q"].float().reshape(B, hkv, h // hkv, hd)
    k = rows("k").transpose(2, 3).contiguous()
    seen = torch.arange(k.shape[3], device=q.device) < s["lengths"][:, None, None, None]
    w = _softmax(torch.matmul(q, k) * (hd ** -0.5), seen)
    return torch.matmul(w, rows("v")).reshape(B, h, hd).to(DTYPE[case["out"]])


def _prompt(s, case):
    q, k, v, starts = s["q"], s["k"], s["v"], s["starts"]
    total, h, hd = q.shape
    hkv, n, B = k.shape[1], case["longest"], case["seqs"]
    seq, i = _token_places(starts, total)
    at = (starts[:-1, None] + torch.arange(n, device=q.device, dtype=torch.int32)).clamp_max(total - 1).long()
    # padded to the longest: [B, hkv, group, n, hd] against [B, hkv, 1, n, hd]
    qp = q[at].float().reshape(B, n, hkv, h // hkv, hd).permute(0, 2, 3, 1, 4).reshape(B, hkv, -1, hd)
    kp = k[at].float().permute(0, 2, 3, 1).contiguous()
    vp = v[at].float().permute(0, 2, 1, 3).contiguous()
    scores = (torch.matmul(qp, kp) * (hd ** -0.5)).reshape(B, hkv, h // hkv, n, n)
    place = torch.arange(n, device=q.device)
    w = _softmax(scores, place[None, :] <= place[:, None]).reshape(B, hkv, -1, n)
    out = torch.matmul(w, vp).reshape(B, h, n, hd)
    return out[seq, :, i.long()].to(DTYPE[case["out"]])


def _logprobs(s, case):
    x, t, top = s["logits"].float(), s["targets"].long(), case["top"]
    m = x.amax(1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    total = e.sum(1)
    log_total = torch.log(total)
    lse = m[:, 0] + log_total
    entropy = log_total - torch.where(e > 0, e * d, torch.zeros_like(e)).sum(1) / total
    given = (t >= 0) & (t < x.shape[1])
    picked = x.gather(1, t.clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    logprobs = torch.where(given, picked - lse, torch.zeros_like(lse))
    # ordered by value, then by the lower index: whole numbers that say both
    bits = (x + 0.0).view(torch.int32)
    order = ((bits ^ ((bits >> 31) & 0x7fffffff)).long() << 32) - torch.arange(x.shape[1], device=x.device)
    ids = order.topk(top, 1).indices
    return logprobs, entropy, lse, x.gather(1, ids) - lse[:, None], ids.to(torch.int32)


def _logprobs_backward(s, case):
    x, t = s["logits"].float(), s["targets"].long()
    logp = x - s["lse"][:, None]
    p = torch.exp(logp)
    given = (t >= 0) & (t < x.shape[1])
    g = torch.where(given, s["g_logprobs"], torch.zeros_like(s["g_logprobs"]))
    grad = -g[:, None] * p
    if case["entropy"]:
        inner = torch.where(p > 0, p * (logp + s["entropy"][:, None]), torch.zeros_like(p))
        grad = grad - s["g_entropy"][:, None] * inner
    rows = torch.arange(x.shape[0], device=x.device)
    grad[rows, t.clamp(0, x.shape[1] - 1)] += g
    return grad.to(s["logits"].dtype)


def _run_own(s, case, kind):
    """The framework's calls, on memory that the program holds."""
    if own:
        from lucid_amd import _C
        import lucid_amd.nn.functional  # noqa: F401  (declares the entry points)

        lib = _C.lib()

        def ptr(t):
            return None if t is None else t.data_ptr()

        def scratch(size):
            return torch.empty((max(size, 16),), dtype=torch.uint8, device="cuda")

        if kind == "append":
            kv, hkv, hd = s["kv"], case["kv_heads"], case["head_dim"]
            tokens = kv.shape[0]
            _C.call("lq_paged_kv_append", ptr(kv), ptr(kv[:, 1]), CODE[case["source"]], 2 * hkv * hd, tokens,
                    None if case["step"] else ptr(s["starts"]), case["seqs"], hkv, hd, ptr(s["table"]),
                    s["table"].shape[1], ptr(s["lengths"]), ptr(s["k"]), ptr(s["v"]), CODE[case["cache"]], None, None,
                    s["pool"], case["page"], None)
            return s["k"], s["v"]
        if kind == "paged":
            B, h, hd = s["q"].shape
            hkv = case["kv_heads"]
            size = lib.lq_paged_attention_workspace_size(B, h, hkv, hd, case["longest"])
            ws = scratch(size)
            _C.call("lq_paged_attention", ptr(s["q"]), CODE[case["dtype"]], h * hd, B, h, hkv, hd, ptr(s["k"]),
                    ptr(s["v"]), CODE[case["cache"]], ptr(s.get("k_scale")), ptr(s.get("v_scale")), s["pool"],
                    case["page"], ptr(s["table"]), s["table"].shape[1], ptr(s["lengths"]), case["longest"], hd ** -0.5,
                    ptr(s["out"]), CODE[case["out"]], ptr(ws), size, None)
            return s["out"]
        if kind == "prompt":
            q, k, v, starts = s["q"], s["k"], s["v"], s["starts"]
            total, h, hd = q.shape
            _C.call("lq_prompt_attention", ptr(q), q.stride(0), ptr(k), k.stride(0), ptr(v), v.stride(0),
                    CODE[case["dtype"]], ptr(starts), ptr(starts), case["seqs"], total, total, h, k.shape[1], hd, 1,
                    hd ** -0.5, ptr(s["out"]), CODE[case["out"]], None)
            return s["out"]
        x = s["logits"]
        rows, vocab = x.shape
        if kind == "logprobs":
            size = lib.lq_token_logprobs_workspace_size(rows, vocab, case["top"])
            ws = scratch(size)
            _C.call("lq_token_logprobs", ptr(x), CODE[case["dtype"]], vocab, rows, vocab, ptr(s["targets"]),
                    case["top"], ptr(s["logprobs"]), ptr(s["entropy"]), ptr(s["lse"]), ptr(s["top_logprobs"]),
                    ptr(s["top_ids"]), ptr(ws), size, None)
            return s["logprobs"], s["entropy"], s["lse"], s["top_logprobs"], s["top_ids"]
        _C.call("lq_token_logprobs_backward", ptr(x), CODE[case["dtype"]], vocab, rows, vocab, ptr(s["targets"]),
                ptr(s["lse"]), ptr(s["entropy"]) if case["entropy"] else None, ptr(s["g_logprobs"]),
                ptr(s["g_entropy"]) if case["entropy"] else None, ptr(s["grad"]), vocab, None)
        return s["grad"]


# ------------------------------------------------------------------------------ work, exact


def work(case):
    kind = case["kind"]
    if kind == "append":
        lens = _lengths(case)
        values = 2 * sum(_new(case, lens)) * case["kv_heads"] * case["head_dim"]
        return {"bytes": values * (SIZE[case["source"]] + SIZE[case["cache"]]) + 4 * sum(_pages(lens, case["page"])),
                "flops": values}
    if kind == "paged":
        lens, hd = _lengths(case), case["head_dim"]
        row = hd * SIZE[case["cache"]] + (4 if case["cache"] == "int8" else 0)
        ends = len(lens) * case["heads"] * hd * (SIZE[case["dtype"]] + SIZE[case["out"]])
        return {"bytes": 2 * sum(lens) * case["kv_heads"] * row + ends + 4 * sum(_pages(lens, case["page"])),
                "flops": 4 * sum(lens) * case["heads"] * hd}
    if kind == "prompt":
        lens, hd = _lengths(case), case["head_dim"]
        row = hd * (SIZE[case["dtype"]] * (case["heads"] + 2 * case["kv_heads"]) + SIZE[case["out"]] * case["heads"])
        return {"bytes": sum(lens) * row, "flops": 4 * case["heads"] * hd * sum(n * (n + 1) // 2 for n in lens)}
    rows, vocab = case["rows"], case["vocab"]
    if kind == "logprobs":
        return {"bytes": rows * vocab * SIZE[case["dtype"]] + rows * (16 + 8 * case["top"]), "flops": 5 * rows * vocab}
    return {"bytes": 2 * rows * vocab * SIZE[case["dtype"]] + 20 * rows, "flops": 5 * rows * vocab}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "append":  # a rounding of its inputs, no computed values
        return None
    if kind == "paged":
        return _exact_paged(s, case)
    if kind == "prompt":
        return _exact_prompt(s, case)
    if kind == "logprobs":
        return _exact_logprobs(s, case)
    out = []
    for r in range(0, case["rows"], 512):
        cut = slice(r, r + 512)
        x, t = s["logits"][cut].double(), s["targets"][cut].long()
        logp = torch.log_softmax(x, 1)
        p = logp.exp()
        hot = torch.zeros_like(x)
        ok = (t >= 0).double()
        hot.scatter_(1, t.clamp_min(0)[:, None], ok[:, None])
        grad = s["g_logprobs"][cut].double()[:, None] * (hot - p * ok[:, None])
        if case["entropy"]:
            plogp = torch.nan_to_num(p * logp, nan=0.0)
            grad -= s["g_entropy"][cut].double()[:, None] * (plogp - p * plogp.sum(1, keepdim=True))
        out.append(grad)
    return torch.cat(out)


def _exact_paged(s, case):
    h, hkv, hd, ps = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    out = torch.zeros((case["seqs"], h, hd), dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        t = torch.arange(n, device="cuda")
        page, slot = s["table"][b, t // ps].long(), t % ps
        k, v = s["k"][page, :, slot].double(), s["v"][page, :, slot].double()
        if case["cache"] == "int8":
            k = k * s["k_scale"][page, :, slot].double()[..., None]
            v = v * s["v_scale"][page, :, slot].double()[..., None]
        for j in range(hkv):
            rows = slice(j * (h // hkv), (j + 1) * (h // hkv))
            w = torch.softmax(s["q"][b, rows].double() @ k[:, j].t() / math.sqrt(hd), 1)
            out[b, rows] = w @ v[:, j]
    return out


def _exact_prompt(s, case):
    h, hkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    out = torch.zeros((s["q"].shape[0], h, hd), dtype=torch.float64, device="cuda")
    first = 0
    for n in _lengths(case):
        for j in range(h):
            k = s["k"][first:first + n, j // (h // hkv)].double()
            v = s["v"][first:first + n, j // (h // hkv)].double()
            for i in range(0, n, 4096):
                e = min(n, i + 4096)
                a = s["q"][first + i:first + e, j].double() @ k[:e].t() / math.sqrt(hd)
                late = torch.arange(e, device="cuda")[None, :] > torch.arange(i, e, device="cuda")[:, None]
                out[first + i:first + e, j] = torch.softmax(a.masked_fill_(late, -math.inf), 1) @ v[:e]
        first += n
    return out


def _exact_logprobs(s, case):
    out = []
    for r in range(0, case["rows"], 512):
        x, t = s["logits"][r:r + 512].double(), s["targets"][r:r + 512].long()
        lse = torch.logsumexp(x, 1)
        logp = x - lse[:, None]
        picked = logp.gather(1, t.clamp_min(0)[:, None])[:, 0]
        entropy = -torch.nan_to_num(logp.exp() * logp, nan=0.0).sum(1)
        best, ids = torch.sort(logp, dim=1, descending=True, stable=True)
        out.append((torch.where(t >= 0, picked, torch.zeros_like(picked)), entropy, lse, best[:, :case["top"]],
                    ids[:, :case["top"]].to(torch.int32)))
    return tuple(torch.cat(c) for c in zip(*out))
