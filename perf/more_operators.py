"""Operators of a rotary decoder's serving step, as cases that can be timed and compared.

* ``norm``: root-mean-square norm of rows, with the residual's addition, out as 8-bit codes with a scale
  per row or as floats;
* ``rotate``: queries and keys rotated by their positions, keys and values appended to a paged cache;
* ``paged4``: attention of one new token per sequence over pages that hold 4 bits a value;
* ``step4``: the two as a decode step runs them: rotation and append to 4 bits, then attention;
* ``verify``: drafted tokens accepted or replaced under the target's distribution.

``run()`` computes them from their formulas with elementary torch operations where ``own`` is false and
calls the C ABI of ``include/lq_api.h`` where it is true.  ``exact()`` is the definition in 64 bits.

The 4-bit cache: keys share a scale and a bias between 32 dims, values between all dims of a row; both are
bfloat16, a value is ``code * scale + bias``; codes lie two to a byte, the even dim in the low half.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPE = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
CODE = {"float32": 6, "float16": 5, "bfloat16": 10, "uint4": 11}  # element types of include/lq_api.h
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}
GROUP = 32  # dims of a key that share a scale and a bias


def listed():
    return [
        # one decode step of the framework's own decoder: 8 rows of 512 in float32
        {"name": "norm_step_b8", "kind": "norm", "rows": 8, "dim": 512, "dtype": "float32", "gamma": "float32",
         "residual": True, "out": "int8"},
        # the norm after the last layer, whose rows go to a product in 16 bits
        {"name": "norm_last_777", "kind": "norm", "rows": 777, "dim": 5120, "dtype": "float16", "gamma": "float16",
         "residual": True, "out": "float16"},
        # packed prompts, an odd number of rows
        {"name": "norm_prompts_4097", "kind": "norm", "rows": 4097, "dim": 4096, "dtype": "bfloat16",
         "gamma": "bfloat16", "residual": True, "out": "int8"},
        # a long batch of wide rows
        {"name": "norm_wide_16384", "kind": "norm", "rows": 16384, "dim": 8192, "dtype": "bfloat16",
         "gamma": "bfloat16", "residual": True, "out": "int8"},
        # a decode step of the framework's own decoder: 8 heads of 64 from a float32 projection
        {"name": "rotate_step_b8", "kind": "rotate", "seqs": 8, "longest": 640, "step": True, "heads": 8, "kv_heads": 8,
         "head_dim": 64, "rot": 64, "interleaved": False, "page": 16, "source": "float32", "cache": "float16", "mix": 1},
        # prompts of a serving batch, grouped heads, some after a cached prefix
        {"name": "rotate_prompts_16", "kind": "rotate", "seqs": 16, "longest": 4096, "step": False, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "rot": 128, "interleaved": False, "page": 64, "source": "bfloat16",
         "cache": "bfloat16", "mix": 2},
        # the decoder's step over 4-bit pages: positions up to 640, float32 out for the dynamic input step
        {"name": "paged4_step_b8", "kind": "paged4", "seqs": 8, "longest": 640, "heads": 8, "kv_heads": 8,
         "head_dim": 64, "page": 16, "dtype": "float16", "out": "float32", "mix": 3},
        # a full serving batch, grouped heads, ragged lengths
        {"name": "paged4_ragged_b64", "kind": "paged4", "seqs": 64, "longest": 8191, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 64, "dtype": "bfloat16", "out": "bfloat16", "mix": 4},
        # two long documents: few rows, a long axis
        {"name": "paged4_long_b2", "kind": "paged4", "seqs": 2, "longest": 131071, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 128, "dtype": "float16", "out": "float16", "mix": 5},
        # a decode step: rotation, append to 4 bits, attention over them
        {"name": "step4_b32", "kind": "step4", "seqs": 32, "longest": 2047, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "rot": 128, "interleaved": False, "page": 64, "dtype": "bfloat16", "out": "bfloat16",
         "mix": 6},
        # drafts that were looked up in the prompt, so that each was certain: four to a sequence
        {"name": "verify_sure_b8", "kind": "verify", "seqs": 8, "drafts": 4, "vocab": 32000, "dtype": "float32",
         "sure": True, "mix": 7},
        # up to seven drafts of a small model, with its distributions, a vocabulary of odd length
        {"name": "verify_b64", "kind": "verify", "seqs": 64, "drafts": 7, "vocab": 100003, "dtype": "bfloat16",
         "sure": False, "mix": 8},
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], even in its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("norm", "norm", "rotate", "rotate", "paged4", "paged4", "paged4", "step4", "verify", "verify"))
    mix, dtype = rng.randrange(1 << 20), rng.choice(("float16", "bfloat16"))
    if kind == "norm":
        dim = rng.choice((_log(rng, 64, 16384), 8 * _log(rng, 8, 2048)))
        wide = rng.choice((dtype, dtype, "float32"))
        return {"kind": kind, "rows": _log(rng, 1, min(65536, (1 << 26) // dim)), "dim": dim, "dtype": wide,
                "gamma": rng.choice((wide, "float32")), "residual": rng.random() < 0.75,
                "out": rng.choice(("int8", "int8", wide))}
    if kind == "verify":
        seqs = _log(rng, 1, 128)
        k = rng.randint(1, 12)
        return {"kind": kind, "seqs": seqs, "drafts": k, "vocab": _log(rng, 128, min(200000, (1 << 25) // (seqs * k))),
                "dtype": rng.choice((dtype, "float32")), "sure": rng.random() < 0.4, "mix": mix}
    kv = rng.choice((1, 2, 4, 8, rng.randint(1, 8)))
    group = rng.choice((1, 2, 4, 8, rng.randint(1, 16)))
    page = 1 << rng.randint(3, 8)
    if kind == "rotate":
        step = rng.random() < 0.5
        hd = rng.choice((64, 128, 128, 8 * rng.randint(4, 32)))
        rot = rng.choice((hd, hd, 2 * rng.randint(1, hd // 2)))
        return {"kind": kind, "seqs": _log(rng, 1, 256) if step else rng.randint(1, 16),
                "longest": _log(rng, 8, min(4096, (1 << 25) // (kv * group * hd))), "step": step, "heads": kv * group,
                "kv_heads": kv, "head_dim": hd, "rot": rot, "interleaved": rng.random() < 0.3, "page": page,
                "source": rng.choice(("float32", dtype)), "cache": dtype, "mix": mix}
    hd = rng.choice((64, 64, 128, 128, 128, 32 * rng.randint(1, 8)))
    seqs = _log(rng, 1, 128)
    longest = _log(rng, 1, min(131072, 64 * 8192 * 8 * 128 // (seqs * kv * hd)))
    case = {"kind": kind, "seqs": seqs, "longest": longest, "heads": kv * group, "kv_heads": kv, "head_dim": hd,
            "page": page, "dtype": dtype, "out": rng.choice((dtype, dtype, "float32")) if kind == "paged4" else dtype,
            "mix": mix}
    if kind == "step4":
        case.update(rot=rng.choice((hd, hd // 2)), interleaved=rng.random() < 0.3)
    return case


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
    if case.get("step", True):
        return [1] * len(lens)
    return [n if i % 3 else max(1, n - n // 4) for i, n in enumerate(lens)]


def _drafts(case):
    """How many tokens were drafted for each sequence."""
    rng = random.Random(case["mix"])
    return [case["drafts"]] + [rng.randint(0, case["drafts"]) for _ in range(case["seqs"] - 1)]


def _pages(lens, page):
    return [-(-n // page) for n in lens]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind = case["kind"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    def starts(values):
        return ints([sum(values[:i]) for i in range(len(values) + 1)])

    if kind == "norm":
        rows, dim, dt = case["rows"], case["dim"], DTYPE[case["dtype"]]
        # a residual stream: some channels far stronger than the rest, rows of different size
        strong = 1.0 + 20.0 * (uniform(dim) < 1 / 128)
        s = {"case": case, "x": (normal(rows, dim) * strong * (0.5 + uniform(rows, 1))).to(dt),
             "res": normal(rows, dim).to(dt) if case["residual"] else None,
             "gamma": (1.0 + 0.2 * normal(dim)).to(DTYPE[case["gamma"]]), "eps": 1e-5}
        s["sum"] = torch.empty_like(s["x"]) if case["residual"] else None
        if case["out"] == "int8":
            s.update(codes=torch.empty((rows, dim), dtype=torch.int8, device="cuda"),
                     scales=torch.empty(rows, dtype=torch.float32, device="cuda"))
        else:
            s["y"] = torch.empty((rows, dim), dtype=DTYPE[case["out"]], device="cuda")
        return s
    if kind == "verify":
        n, vocab, dt = _drafts(case), case["vocab"], DTYPE[case["dtype"]]
        rows = sum(n) + len(n)
        # a target that has learned something: a few likely tokens over a broad rest; a draft model near it
        x = normal(rows, vocab).mul_(2.0)
        x.scatter_add_(1, torch.randint(0, vocab, (rows, 4), generator=g, device="cuda"), 8 + 4 * uniform(rows, 4))
        d = x + 0.7 * normal(rows, vocab)
        # what the draft model drew (the largest of its perturbed logits), or looked up: likely tokens
        drafts = (d - torch.log(-torch.log(uniform(rows, vocab).clamp(1e-20, 1 - 1e-7)))).argmax(1).to(torch.int32)
        s = {"case": case, "logits": x.to(dt), "starts": starts([k + 1 for k in n]), "drafts": drafts,
             "accept_u": uniform(rows), "sample_u": uniform(len(n))}
        s["drafts"][s["starts"][1:].long() - 1] = -100  # a sequence's last row has no draft
        s["draft_logits"] = None if case["sure"] else d.to(dt)

        def lse(t):
            return torch.cat([torch.logsumexp(part.double(), 1) for part in t.split(64)]).float()

        s["lse"], s["draft_lse"] = lse(s["logits"]), None if case["sure"] else lse(s["draft_logits"])
        s.update(tokens=torch.empty(rows, dtype=torch.int32, device="cuda"),
                 accepted=torch.empty(len(n), dtype=torch.int32, device="cuda"))
        return s
    lens, hkv, h, hd, ps = _lengths(case), case["kv_heads"], case["heads"], case["head_dim"], case["page"]
    used = _pages(lens, ps)
    pool = sum(used) + 4
    ids = torch.randperm(pool, generator=g, device="cuda")[:sum(used)].to(torch.int32)
    table = torch.zeros((len(lens), max(used)), dtype=torch.int32, device="cuda")
    table[torch.arange(max(used), device="cuda")[None, :] < ints(used)[:, None]] = ids
    s = {"case": case, "table": table, "lengths": ints(lens), "pool": pool}
    shape = (pool, hkv, ps, hd)
    if kind != "paged4":
        new, rot = _new(case, lens), case["rot"]
        s["starts"] = starts(new)
        # one projection's rows: queries, keys, values
        s["qkv"] = normal(sum(new), h + 2 * hkv, hd).to(DTYPE[case["source" if kind == "rotate" else "dtype"]])
        # cosines, then sines, of every position's angles
        rate = 10000.0 ** (-2.0 * torch.arange(rot // 2, device="cuda", dtype=torch.float64) / rot)
        angle = torch.arange(case["longest"] + 1, device="cuda", dtype=torch.float64)[:, None] * rate
        s["angles"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        s["q"] = torch.empty((sum(new), h, hd), dtype=DTYPE[case["cache" if kind == "rotate" else "dtype"]], device="cuda")
    if kind == "rotate":
        s["k"] = torch.zeros(shape, dtype=DTYPE[case["cache"]], device="cuda")
        s["v"] = torch.zeros(shape, dtype=DTYPE[case["cache"]], device="cuda")
        return s
    # keys with a few strong channels and an offset, as projections have them
    strong = 1.0 + 3.0 * (uniform(hkv, 1, hd) < 1 / 32)
    offset = normal(hkv, 1, hd) * (uniform(hkv, 1, hd) < 1 / 8)
    for name, step in (("k", GROUP), ("v", hd)):
        parts = []
        for lo in range(0, pool, 256):
            x = normal(min(256, pool - lo), *shape[1:])
            parts.append(_quantize4((x * strong + offset) if name == "k" else x, step))
        s[name], s[name + "_scale"] = (torch.cat(p) for p in zip(*parts))
    if kind == "paged4":
        s["q"] = normal(len(lens), h, hd).to(DTYPE[case["dtype"]])
    s["out"] = torch.empty((len(lens), h, hd), dtype=DTYPE[case["out"]], device="cuda")
    return s


# ------------------------------------------------------------------------------ 4 bits


def _bf16_toward(x, up):
    """float32 values as the next bfloat16 at or above (below) them."""
    bits = x.contiguous().view(torch.int32)
    away = (bits >= 0) if up else (bits < 0)  # the magnitude grows
    return ((bits + torch.where(away, 0xffff, 0).to(torch.int32)) & -65536).view(torch.float32)


def _quantize4(x, step):
    """Rows of 4-bit codes, two to a byte, and [scales, biases] of every ``step`` dims, for x [..., hd]."""
    g = x.unflatten(-1, (-1, step))
    low, high = g.amin(-1).float(), g.amax(-1)
    bias = _bf16_toward(low, False)
    scale = _bf16_toward(((high - bias) / 15).float(), True)
    inv = torch.where(scale > 0, 1 / scale, torch.zeros_like(scale))
    codes = ((g - bias[..., None]) * inv[..., None]).round().clamp(0, 15).flatten(-2).to(torch.uint8)
    return codes[..., 0::2] | codes[..., 1::2] << 4, torch.cat([scale, bias], -1).to(torch.bfloat16)


def _values4(codes, scale, wide):
    """What 4-bit rows stand for, in ``wide``."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(wide)
    factor, bias = scale.to(wide).chunk(2, -1)
    return (c.unflatten(-1, (factor.shape[-1], -1)) * factor[..., None] + bias[..., None]).flatten(-2)


# ------------------------------------------------------------------------------ one pass


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        return _run_own(s, case, kind)
    if kind == "norm":
        return _norm(s, case)
    if kind == "rotate":
        q, k = _rotated(s, case, torch.float32)
        _append(s, case, k)
        return q.to(s["q"].dtype), s["k"], s["v"]
    if kind == "step4":
        q, k = _rotated(s, case, torch.float32)
        _append4(s, case, k)
        q = q.to(s["q"].dtype)
        return q, _paged4(s, case, q)
    if kind == "paged4":
        return _paged4(s, case, s["q"])
    return _verify(s, case)


def _norm(s, case):
    h = s["x"].float()
    if case["residual"]:
        h = (h + s["res"].float()).to(s["x"].dtype).float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + s["eps"]) * s["gamma"].float()
    total = h.to(s["x"].dtype) if case["residual"] else None
    if case["out"] != "int8":
        return [y.to(DTYPE[case["out"]]), total] if case["residual"] else [y.to(DTYPE[case["out"]])]
    top = y.abs().amax(1, keepdim=True)
    codes, scales = (y * (127 / top)).round(), top / 127
    out = [(codes * scales).to(torch.bfloat16), scales[:, 0]]  # 8 bits: a sixteen-bit type has room for them
    return out + [total] if case["residual"] else out


def _places(s, case):
    """(sequence, position) of each packed token."""
    starts, lengths = s["starts"], s["lengths"]
    t = torch.arange(s["qkv"].shape[0], device=starts.device, dtype=torch.int32)
    seq = torch.searchsorted(starts, t, right=True) - 1
    return seq, lengths[seq] - (starts[seq + 1] - starts[seq]) + t - starts[seq]


def _rotated(s, case, wide):
    """The tokens' rotated queries and keys."""
    h, hkv, rot = case["heads"], case["kv_heads"], case["rot"]
    x = s["qkv"][:, :h + hkv].to(wide)
    cos, sin = s["angles"][_places(s, case)[1].long()].to(wide)[:, None].chunk(2, -1)
    if case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    x = torch.cat([turned, x[..., rot:]], -1)
    return x[:, :h], x[:, h:]


def _append(s, case, k):
    seq, pos = _places(s, case)
    page, slot = s["table"][seq, pos // case["page"]].long(), (pos % case["page"]).long()
    s["k"][page, :, slot] = k.to(s["k"].dtype)
    s["v"][page, :, slot] = s["qkv"][:, case["heads"] + case["kv_heads"]:].to(s["v"].dtype)


def _append4(s, case, k):
    seq, pos = _places(s, case)
    page, slot = s["table"][seq, pos // case["page"]].long(), (pos % case["page"]).long()
    v = s["qkv"][:, case["heads"] + case["kv_heads"]:].float()
    for name, x, step in (("k", k, GROUP), ("v", v, case["head_dim"])):
        s[name][page, :, slot], s[name + "_scale"][page, :, slot] = _quantize4(x, step)


def _paged4(s, case, q):
    B, h, hd = q.shape
    hkv, ps = case["kv_heads"], case["page"]

    def rows(name):  # a sequence's pages in order, [B, hkv, positions, hd] in 32 bits
        at = s["table"].long()
        x = _values4(s[name][at], s[name + "_scale"][at], torch.float32)
        return x.transpose(1, 2).reshape(B, hkv, -1, hd)

    q = q.float().reshape(B, hkv, h // hkv, hd)
    k = rows("k").transpose(2, 3).contiguous()
    seen = torch.arange(k.shape[3], device=q.device) < s["lengths"][:, None, None, None]
    scores = (torch.matmul(q, k) * (hd ** -0.5)).masked_fill(~seen, -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    w = e / e.sum(-1, keepdim=True)
    return torch.matmul(w, rows("v")).reshape(B, h, hd).to(DTYPE[case["out"]])


def _verify(s, case):
    """In 64 bits: the tokens are whole numbers that a border decides."""
    x, starts, drafts, k = s["logits"], s["starts"].long(), s["drafts"].long(), case["drafts"]
    vocab, rows = x.shape[1], torch.arange(x.shape[0], device=x.device)
    token = drafts.clamp(0, vocab - 1)
    p = torch.exp(x[rows, token].double() - s["lse"].double())
    q = torch.ones_like(p)
    if not case["sure"]:
        q = torch.exp(s["draft_logits"][rows, token].double() - s["draft_lse"].double())
    ok = (drafts >= 0) & (drafts < vocab) & (s["accept_u"].double() * q < p)
    # a sequence's drafts side by side; those before the first that fails are accepted
    place = starts[:-1, None] + torch.arange(k + 1, device=x.device)
    has = place < starts[1:, None] - 1
    at = place.clamp_max(x.shape[0] - 1)
    accepted = (ok[at] & has).int().cumprod(1).sum(1)
    row = starts[:-1] + accepted
    rejected = row < starts[1:] - 1
    target = torch.exp(x[row].double() - s["lse"][row].double()[:, None])
    if case["sure"]:
        rest = target.scatter(1, token[row][:, None], 0.0)
    else:
        rest = (target - torch.exp(s["draft_logits"][row].double() - s["draft_lse"][row].double()[:, None])).clamp_min(0)
    rest = torch.where((rejected & (rest.sum(1) > 0))[:, None], rest, target)
    upto = rest.cumsum(1)
    new = (upto <= s["sample_u"].double()[:, None] * upto[:, -1:]).sum(1).clamp_max(vocab - 1)
    tokens = torch.full_like(s["drafts"], -1)
    kept = has & (torch.arange(k + 1, device=x.device) < accepted[:, None])
    tokens[at[kept]] = s["drafts"][at[kept]]
    tokens[row] = new.to(torch.int32)
    return tokens, accepted.to(torch.int32)


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

        if kind == "norm":
            rows, dim = s["x"].shape
            given = (ptr(s["x"]), CODE[case["dtype"]], dim, ptr(s["res"]), dim, ptr(s["sum"]), dim, ptr(s["gamma"]),
                     CODE[case["gamma"]], s["eps"], rows, dim)
            if case["out"] == "int8":
                _C.call("lq_rms_norm_quantize", *given, ptr(s["codes"]), dim, ptr(s["scales"]), None)
                values = torch.empty((rows, dim), dtype=torch.bfloat16, device="cuda")
                torch.mul(s["codes"], s["scales"][:, None], out=values)  # the values that the codes stand for
                out = [values, s["scales"]]
            else:
                _C.call("lq_rms_norm", *given, ptr(s["y"]), CODE[case["out"]], dim, None)
                out = [s["y"]]
            return out + [s["sum"]] if case["residual"] else out
        if kind == "verify":
            rows, vocab = s["logits"].shape
            size = lib.lq_verify_drafts_workspace_size(case["seqs"], vocab)
            ws = scratch(size)
            _C.call("lq_verify_drafts", ptr(s["logits"]), CODE[case["dtype"]], vocab, ptr(s["lse"]),
                    ptr(s["draft_logits"]), vocab, ptr(s["draft_lse"]), ptr(s["drafts"]), ptr(s["starts"]),
                    case["seqs"], rows, vocab, ptr(s["accept_u"]), ptr(s["sample_u"]), ptr(s["tokens"]),
                    ptr(s["accepted"]), ptr(ws), size, None)
            return s["tokens"], s["accepted"]
        h, hkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
        if kind != "paged4":
            qkv, ld = s["qkv"], (h + 2 * hkv) * hd
            cache, source = (case["cache"], case["source"]) if kind == "rotate" else ("uint4", case["dtype"])
            out_type = CODE[case["cache" if kind == "rotate" else "dtype"]]
            _C.call("lq_paged_kv_append_rotary", ptr(qkv), ld, ptr(qkv[:, h]), ptr(qkv[:, h + hkv]), ld, CODE[source],
                    qkv.shape[0], None if case.get("step", True) else ptr(s["starts"]), case["seqs"], h, hkv, hd,
                    ptr(s["angles"]), s["angles"].shape[0], case["rot"], int(case["interleaved"]), ptr(s["table"]),
                    s["table"].shape[1], ptr(s["lengths"]), ptr(s["q"]), h * hd, None, 0, out_type, ptr(s["k"]),
                    ptr(s["v"]), CODE[cache], ptr(s.get("k_scale")), ptr(s.get("v_scale")), s["pool"], case["page"],
                    None)
            if kind == "rotate":
                return s["q"], s["k"], s["v"]
        size = lib.lq_paged_attention_workspace_size(case["seqs"], h, hkv, hd, case["longest"])
        ws = scratch(size)
        _C.call("lq_paged_attention", ptr(s["q"]), CODE[case["dtype"]], h * hd, case["seqs"], h, hkv, hd, ptr(s["k"]),
                ptr(s["v"]), CODE["uint4"], ptr(s["k_scale"]), ptr(s["v_scale"]), s["pool"], case["page"],
                ptr(s["table"]), s["table"].shape[1], ptr(s["lengths"]), case["longest"], hd ** -0.5, ptr(s["out"]),
                CODE[case["out"]], ptr(ws), size, None)
        return (s["q"], s["out"]) if kind == "step4" else s["out"]


# ------------------------------------------------------------------------------ work, exact


def work(case):
    kind = case["kind"]
    if kind == "norm":
        n, e = case["rows"] * case["dim"], SIZE[case["dtype"]]
        read = n * e * (2 if case["residual"] else 1) + case["dim"] * SIZE[case["gamma"]]
        wrote = n * (e if case["residual"] else 0) + (n + 4 * case["rows"] if case["out"] == "int8" else n * e)
        return {"bytes": read + wrote, "flops": 6 * n}
    if kind == "verify":  # a row of the target to a sequence, and the draft's where one was rejected: taken as all
        rows = case["seqs"] * (1 if case["sure"] else 2)
        return {"bytes": rows * case["vocab"] * SIZE[case["dtype"]] + 16 * sum(_drafts(case)) + 20 * case["seqs"],
                "flops": 12 * rows * case["vocab"]}
    lens, h, hkv, hd = _lengths(case), case["heads"], case["kv_heads"], case["head_dim"]
    row4 = hd + 4 * (hd // GROUP) + 4  # a key and a value of 4 bits with their scales and biases
    moved, flops = 4 * sum(_pages(lens, case["page"])), 0
    if kind != "paged4":
        new = sum(_new(case, lens))
        source, out = (case["source"], case["cache"]) if kind == "rotate" else (case["dtype"], case["dtype"])
        moved += new * ((h + 2 * hkv) * hd * SIZE[source] + h * hd * SIZE[out] + 4 * case["rot"])
        moved += new * hkv * (2 * hd * SIZE[out] if kind == "rotate" else row4)
        flops += 3 * new * (h + hkv) * case["rot"]
    if kind != "rotate":
        moved += sum(lens) * hkv * row4 + case["seqs"] * h * hd * (SIZE[case["dtype"]] + SIZE[case["out"]])
        flops += 4 * sum(lens) * h * hd
    return {"bytes": moved, "flops": flops}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "verify":  # whole numbers alone
        return None
    if kind == "norm":
        parts = [_exact_norm(s, case, slice(r, r + 2048)) for r in range(0, case["rows"], 2048)]
        return [torch.cat(p) for p in zip(*parts)]
    if kind == "paged4":
        return _exact_paged4(s, case, s["q"].double())
    # the rotation as complex numbers
    h, hkv, rot, ps = case["heads"], case["kv_heads"], case["rot"], case["page"]
    new, lens = _new(case, _lengths(case)), _lengths(case)
    pos = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, new)]).cuda()
    seq = torch.cat([torch.full((m,), i) for i, m in enumerate(new)]).cuda()
    x = s["qkv"][:, :h + hkv].double()
    turn = torch.complex(s["angles"][pos, :rot // 2].double(), s["angles"][pos, rot // 2:].double())[:, None]
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (slice(rot // 2), slice(rot // 2, rot))
    z = torch.complex(x[..., first], x[..., second]) * turn
    x[..., first], x[..., second] = z.real, z.imag
    page, slot = s["table"][seq, pos // ps].long(), pos % ps
    if kind == "rotate":
        k = torch.zeros(s["k"].shape, dtype=torch.float64, device="cuda")
        k[page, :, slot] = x[:, h:]
        return x[:, :h], k, None  # the values are roundings of their inputs
    for name, t, step in (("k", x[:, h:], GROUP), ("v", s["qkv"][:, h + hkv:].double(), case["head_dim"])):
        groups = t.unflatten(-1, (-1, step))
        low, high = groups.amin(-1), groups.amax(-1)
        bias = low.to(torch.bfloat16)  # the nearest one, or its neighbour below
        bias = torch.where(bias.double() > low, torch.nextafter(bias, torch.full_like(bias, -math.inf)), bias)
        width = (high - bias.double()) / 15
        scale = width.to(torch.bfloat16)
        scale = torch.where(scale.double() < width, torch.nextafter(scale, torch.full_like(scale, math.inf)), scale)
        codes = ((groups - bias.double()[..., None]) / scale.double()[..., None]).nan_to_num(0.0).round().clamp(0, 15)
        codes = codes.flatten(-2).to(torch.uint8)
        s[name][page, :, slot] = codes[..., 0::2] + 16 * codes[..., 1::2]
        s[name + "_scale"][page, :, slot] = torch.cat([scale, bias], -1)
    return x[:, :h], _exact_paged4(s, case, x[:, :h].to(s["q"].dtype).double())


def _exact_norm(s, case, cut):
    h = s["x"][cut].double()
    if case["residual"]:  # the norm is of the sum as it is stored
        total = h + s["res"][cut].double()
        h = total.to(s["x"].dtype).double()
    y = h / torch.sqrt(h.square().mean(1, keepdim=True) + s["eps"]) * s["gamma"].double()
    if case["out"] != "int8":
        return (y, total) if case["residual"] else (y,)
    scale = y.abs().amax(1, keepdim=True) / 127
    out = ((y / scale).round() * scale, scale[:, 0])
    return out + (total,) if case["residual"] else out


def _exact_paged4(s, case, q):
    h, hkv, ps = case["heads"], case["kv_heads"], case["page"]
    out = torch.zeros((case["seqs"], h, case["head_dim"]), dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        t = torch.arange(n, device="cuda")
        page, slot = s["table"][b, t // ps].long(), t % ps
        k, v = (_values4(s[c][page, :, slot], s[c + "_scale"][page, :, slot], torch.float64) for c in ("k", "v"))
        for j in range(hkv):
            rows = slice(j * (h // hkv), (j + 1) * (h // hkv))
            w = torch.softmax(q[b, rows] @ k[:, j].t() / math.sqrt(case["head_dim"]), 1)
            out[b, rows] = w @ v[:, j]
    return out
