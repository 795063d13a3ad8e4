"""Operators of a language model's decoder layer as tile programs, as measurable cases.

Three operators of ``xtile_amd.kernels``: the root-mean-square norm with the
residual's addition and rows in 8 bits (``rms_norm``), products with 4-bit
weights (``matmul_q4``) and attention with caps, distance biases and masks
(``masked_attention``).  A case is one of them at one size.  ``run`` computes it
from elementary torch operations, or, where ``own`` is true, launches the
program that ``prepare`` planned, over buffers that the caller keeps.
``listed`` holds fixed cases from the smallest calls to the largest, ``draw``
gives more of the same ranges.
"""

from __future__ import annotations

import math

import torch

own = False

_TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}
_EPS = 1e-6


def listed():
    return [
        # One token between two layers: what counts is the launch and the time
        # of one row.
        _norm("norm_token", 1, 4096, "bf16"),
        # A prompt's activations on their way into an 8-bit product: far
        # beyond the caches.
        _norm("norm_prompt_i8", 8192, 4096, "bf16", quantize=True),
        # A row length that is no power of two, in 32 bits, without a residual.
        _norm("norm_f32_rows", 5000, 1000, "f32", residual=False),
        # One token through a square layer.
        _q4("q4_token", 1, 4096, 4096, "f16", 128, out="f16"),
        # One token through the wide layer of a feed-forward block, small groups.
        _q4("q4_token_wide", 1, 11008, 4096, "bf16", 32, out="f32"),
        # A batch of decoding sequences back from the wide layer, activations
        # in 8 bits with a scale for each row.
        _q4("q4_batch_i8", 16, 4096, 11008, "i8", 128, out="f32"),
        # A few dozen tokens through a layer that no tile divides.
        _q4("q4_ragged", 37, 1000, 1056, "bf16", 32, out="bf16"),
        # A prompt, scores capped, four query heads to a key head.
        _attention("attend_prompt_cap", 1, 8, 4, 4096, 4096, 128, "bf16", cap=30.0, causal=True),
        # Documents packed into one long row of tokens, each blind to the others.
        _attention("attend_documents", 1, 16, 1, 8192, 8192, 64, "f16", causal=True, docs=11),
        # Short sequences with a prefix that every token sees, token-major as
        # the projections write them.
        _attention("attend_prefix_short", 4, 4, 2, 577, 577, 96, "bf16", causal=True, prefix=True, token_major=True),
        # A batch of sequences of different lengths, one new token each, with
        # a bias that falls with distance.
        _attention("attend_token_batch", 32, 8, 4, 1, 8192, 128, "bf16", causal=True, slopes=True, lengths=True),
        # One sequence with a very long cache, one new token.
        _attention("attend_token_long", 1, 8, 8, 1, 131072, 128, "f16", cap=50.0, causal=True, lengths=True),
    ]


def _norm(name, rows, cols, dtype, residual=True, quantize=False):
    return {"name": name, "kind": "norm", "rows": rows, "cols": cols, "dtype": dtype, "residual": residual,
            "quantize": quantize}


def _q4(name, m, n, k, dtype, group, out):
    return {"name": name, "kind": "q4", "m": m, "n": n, "k": k, "dtype": dtype, "group": group, "out": out}


def _attention(name, batch, kv_heads, group, nq, nk, d, dtype, cap=0.0, causal=False, window=0, slopes=False,
               lengths=False, prefix=False, docs=0, token_major=False):
    return {"name": name, "kind": "attention", "batch": batch, "kv_heads": kv_heads, "group": group, "nq": nq,
            "nk": nk, "d": d, "dtype": dtype, "cap": cap, "causal": causal, "window": window, "slopes": slopes,
            "lengths": lengths, "prefix": prefix, "docs": docs, "token_major": token_major}


# -- more cases of the same ranges --------------------------------------------


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_norm(rng):
    return _norm("", _log(rng, 1, 8192), _log(rng, 64, 8192), rng.choice(["f32", "f16", "bf16"]),
                 residual=rng.random() < 0.6, quantize=rng.random() < 0.5)


def _draw_q4(rng):
    group = rng.choice([32, 64, 128, 256])
    dtype = rng.choice(["f16", "bf16", "i8"])
    return _q4("", _log(rng, 1, 64), _log(rng, 64, 11008), group * _log(rng, max(1, 256 // group), 11008 // group),
               dtype, group, out="f32" if dtype == "i8" else rng.choice(["f32", dtype]))


def _draw_attention(rng):
    tokens = rng.random() < 0.5  # new tokens against a cache, or a whole prompt
    d = rng.choice([32, 64, 96, 128, 128, 160, 256])
    dtype = rng.choice(["f16", "bf16"])
    cap = rng.choice([0.0, 0.0, 30.0, 50.0])
    if tokens:
        return _attention("", _log(rng, 1, 32), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 8]),
                          _log(rng, 1, 16), _log(rng, 64, 131072), d, dtype, cap=cap, causal=True,
                          slopes=rng.random() < 0.4, lengths=True, window=rng.choice([0, 0, 0, 1000]),
                          token_major=rng.random() < 0.3)
    n = _log(rng, 16, 4096)
    kind = rng.choice(["causal", "documents", "prefix", "window", "full"])
    return _attention("", _log(rng, 1, 8), rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 4]), n, n, d, dtype,
                      cap=cap, causal=kind != "full", window=_log(rng, 1, 1024) if kind == "window" else 0,
                      slopes=rng.random() < 0.3, prefix=kind == "prefix",
                      docs=rng.randint(2, 12) if kind == "documents" else 0, token_major=rng.random() < 0.4)


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    # No drawn case costs more than the largest listed one, nor holds more
    # scores than its plain form does.
    most = max(_cost(c) for c in listed())
    while True:
        c = rng.choice([_draw_norm, _draw_q4, _draw_attention, _draw_attention])(rng)
        small = c["kind"] != "attention" or c["batch"] * c["kv_heads"] * c["group"] * c["nq"] * c["nk"] <= 1 << 30
        if small and _cost(c) <= most:
            del c["name"]
            return c


# -- what a pass cannot do without --------------------------------------------


def _lengths(case):
    """The keys that each sequence holds: all of them, or cut by up to a half."""
    b, nq, nk = case["batch"], case["nq"], case["nk"]
    if not case["lengths"]:
        return [nk] * b
    return [max(min(nq, nk), nk - (i * nk) // (2 * b)) for i in range(b)]


def _prefix(case):
    return [case["nk"] // 8 + (13 * i) % 29 for i in range(case["batch"])]


def _visible(case):
    """Pairs of a query and a key that it sees, over the batch, for one head."""
    nq, docs = case["nq"], case["docs"]
    total = 0
    prefixes = _prefix(case) if case["prefix"] else [0] * case["batch"]
    for length, pre in zip(_lengths(case), prefixes):
        start = length - nq if case["lengths"] else 0
        pre = min(pre, length)
        if docs:  # equal pieces, each its own triangle
            ends = [-(-(i + 1) * nq // docs) for i in range(docs)]
            sizes = [b - a for a, b in zip([0] + ends, ends)]
            total += sum(s * (s + 1) // 2 if case["causal"] else s * s for s in sizes)
            continue
        for i in range(nq):
            p = start + i
            hi = min(p + 1, length) if case["causal"] else length
            lo = max(0, min(hi, p - case["window"] + 1)) if case["window"] else 0
            total += max(0, hi - lo) + max(0, min(pre, lo)) + max(0, pre - max(hi, 0))
    return total


def work(case):
    if case["kind"] == "norm":
        n, esize = case["rows"] * case["cols"], _SIZE[case["dtype"]]
        moved = n * esize * (3 if case["residual"] else 1) + case["cols"] * esize
        moved += n + case["rows"] * 4 if case["quantize"] else n * esize
        return {"bytes": moved, "flops": 6 * n}
    if case["kind"] == "q4":
        m, n, k = case["m"], case["n"], case["k"]
        moved = n * k // 2 + n * (k // case["group"]) * 2 + m * k * _SIZE[case["dtype"]] + m * n * _SIZE[case["out"]]
        moved += 4 * m if case["dtype"] == "i8" else 0
        return {"bytes": moved, "flops": 2 * m * n * k}
    heads = case["kv_heads"] * case["group"]
    seen = _lengths(case)
    if case["window"] and case["lengths"]:
        seen = [min(s, case["window"] + case["nq"] - 1) for s in seen]
    moved = 2 * case["batch"] * heads * case["nq"] * case["d"] * 2 + 2 * case["kv_heads"] * sum(seen) * case["d"] * 2
    return {"bytes": moved, "flops": 4 * case["d"] * heads * _visible(case)}


# -- inputs ---------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _prepare_norm(case, g):
    rows, cols, t = case["rows"], case["cols"], _TORCH[case["dtype"]]
    x = torch.randn(rows, cols, generator=g, device="cuda").to(t)
    r = (3 * torch.randn(rows, cols, generator=g, device="cuda")).to(t) if case["residual"] else None
    gamma = (1 + 0.2 * torch.randn(1, cols, generator=g, device="cuda")).to(t)
    return {"x": x, "r": r, "gamma": gamma}


def _prepare_q4(case, g):
    m, n, k, group = case["m"], case["n"], case["k"], case["group"]
    w = torch.randint(-8, 8, (n, k), generator=g, device="cuda", dtype=torch.int8)
    scales = (0.002 + 0.01 * torch.rand(n, k // group, generator=g, device="cuda")).half()
    s = {"w": w, "scales": scales, "row_scale": None}
    if case["dtype"] == "i8":
        s["x"] = torch.randint(-127, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
        s["row_scale"] = 0.01 + 0.04 * torch.rand(m, 1, generator=g, device="cuda")
    else:
        s["x"] = torch.randn(m, k, generator=g, device="cuda").to(_TORCH[case["dtype"]])
    return s


def _prepare_attention(case, g):
    b, hk, gr, nq, nk, d = (case[k] for k in ("batch", "kv_heads", "group", "nq", "nk", "d"))
    t = _TORCH[case["dtype"]]
    q_shape, k_shape = (b, hk * gr, nq, d), (b, hk, nk, d)
    if case["token_major"]:
        q_shape, k_shape = (b, nq, hk * gr * d), (b, nk, hk * d)
    s = {"q": (2 * torch.randn(q_shape, generator=g, device="cuda")).to(t),
         "k": torch.randn(k_shape, generator=g, device="cuda").to(t),
         "v": torch.randn(k_shape, generator=g, device="cuda").to(t)}
    i32 = {"dtype": torch.int32, "device": "cuda"}
    s["slopes"] = s["start"] = s["length"] = s["prefix"] = s["docs"] = None
    if case["slopes"]:
        h = hk * gr
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, h + 1, device="cuda", dtype=torch.float32) / h).view(hk, gr)
    if case["lengths"]:
        s["length"] = torch.tensor(_lengths(case), **i32).view(b, 1)
        s["start"] = s["length"] - nq
    if case["prefix"]:
        s["prefix"] = torch.tensor(_prefix(case), **i32).view(b, 1)
    if case["docs"]:
        s["docs"] = ((torch.arange(nk, device="cuda") * case["docs"]) // nk).to(torch.int32).expand(b, nk).contiguous()
    return s


_PREPARE = {"norm": _prepare_norm, "q4": _prepare_q4, "attention": _prepare_attention}


def prepare(case, seed):
    state = _PREPARE[case["kind"]](case, _generator(seed))
    state["case"] = dict(case)
    if own:
        _PLAN[case["kind"]](case, state)
    return state


# -- the framework's programs ---------------------------------------------------


def _dsl(name):
    import xtile_amd as xt

    return {"f32": xt.float32, "f16": xt.float16, "bf16": xt.bfloat16, "i8": xt.int8}[name]


def _plan_norm(case, s):
    import xtile_amd as xt
    from xtile_amd import kernels as K

    s["program"] = xt.compile(K.rms_norm(case["rows"], case["cols"], _dsl(case["dtype"]), residual=case["residual"],
                                         quantize=case["quantize"], eps=_EPS))
    s["sum"] = torch.empty_like(s["x"]) if case["residual"] else None
    if case["quantize"]:
        s["rows8"] = torch.empty(s["x"].shape, dtype=torch.int8, device="cuda")
        s["scale"] = torch.empty(case["rows"], 1, device="cuda")
        s["y"] = torch.empty(s["x"].shape, dtype=torch.bfloat16, device="cuda")
    else:
        s["y"] = torch.empty_like(s["x"])
    ins = [s["x"], s["r"]] if case["residual"] else [s["x"]]
    outs = [s["sum"]] if case["residual"] else []
    outs += [s["rows8"], s["scale"]] if case["quantize"] else [s["y"]]
    s["buffers"] = [*ins, s["gamma"], *outs]


def _plan_q4(case, s):
    import xtile_amd as xt
    from xtile_amd import kernels as K

    s["program"] = xt.compile(K.matmul_q4(case["m"], case["n"], case["k"], group=case["group"],
                                          dtype=_dsl(case["dtype"]), scales=xt.float16, out=_dsl(case["out"]),
                                          row_scale=case["dtype"] == "i8"))
    s["y"] = torch.empty(case["m"], case["n"], dtype=_TORCH[case["out"]], device="cuda")
    s["w"] = xt.pack_q4(s["w"])
    s["buffers"] = [s["x"], s["w"], s["scales"], *([] if s["row_scale"] is None else [s["row_scale"]]), s["y"]]


def _plan_attention(case, s):
    import xtile_amd as xt
    from xtile_amd import kernels as K

    s["program"] = xt.compile(K.masked_attention(
        case["batch"], case["kv_heads"], case["group"], case["nq"], case["nk"], case["d"], dtype=_dsl(case["dtype"]),
        cap=case["cap"] or None, causal=case["causal"], window=case["window"] or None, slopes=case["slopes"],
        start=case["lengths"], length=case["lengths"], prefix=case["prefix"], docs=bool(case["docs"]),
        token_major=case["token_major"]))
    s["y"] = torch.empty_like(s["q"])
    extra = [s[k] for k in ("slopes", "start", "length", "prefix", "docs", "docs") if s[k] is not None]
    s["buffers"] = [s["q"], s["k"], s["v"], *extra, s["y"]]


_PLAN = {"norm": _plan_norm, "q4": _plan_q4, "attention": _plan_attention}


def _run_own(case, s):
    import xtile_amd as xt

    xt.launch(s["program"], *s["buffers"])
    if case["kind"] != "norm":
        return [s["y"]]
    if case["quantize"]:  # the values that the 8-bit rows stand for
        torch.mul(s["rows8"], s["scale"], out=s["y"])
    return [s["y"]] if s["sum"] is None else [s["sum"], s["y"]]


# -- the plain forms ------------------------------------------------------------


def _plain_norm(case, s):
    h = s["x"].float()
    if case["residual"]:
        h = h + s["r"].float()
    y = h * torch.rsqrt((h * h).mean(dim=1, keepdim=True) + _EPS) * s["gamma"].float()
    if case["quantize"]:
        scale = y.abs().amax(dim=1, keepdim=True) / 127
        q = torch.where(scale > 0, y / scale, torch.zeros_like(y)).round().clamp(-127, 127)
        y = (q * scale).bfloat16()
    else:
        y = y.to(s["x"].dtype)
    return [h.to(s["x"].dtype), y] if case["residual"] else [y]


def _plain_q4(case, s):
    n, k, group = case["n"], case["k"], case["group"]
    w = (s["w"].float().view(n, k // group, group) * s["scales"].float()[:, :, None]).view(n, k)
    y = s["x"].float() @ w.t()
    if s["row_scale"] is not None:
        y = y * s["row_scale"]
    return [y.to(_TORCH[case["out"]])]


def _heads_first(case, x, heads, n):
    """[batch, kv_heads, heads / kv_heads * n, d] in 32 bits."""
    b, hk, d = case["batch"], case["kv_heads"], case["d"]
    x = x.float()
    if case["token_major"]:
        x = x.view(b, n, heads, d).transpose(1, 2)
    return x.reshape(b, hk, heads // hk * n, d)


def _plain_attention(case, s):
    b, hk, gr, nq, nk, d = (case[k] for k in ("batch", "kv_heads", "group", "nq", "nk", "d"))
    q = _heads_first(case, s["q"], hk * gr, nq)
    k = _heads_first(case, s["k"], hk, nk)
    v = _heads_first(case, s["v"], hk, nk)
    x = (q @ k.transpose(2, 3)).mul_(1 / math.sqrt(d)).view(b, hk, gr, nq, nk)
    if case["cap"]:
        x = x.div_(case["cap"]).tanh_().mul_(case["cap"])
    j = torch.arange(nk, device="cuda").view(1, 1, nk)
    p = torch.arange(nq, device="cuda").view(1, nq, 1)
    if s["start"] is not None:
        p = p + s["start"].view(b, 1, 1)
    if case["slopes"]:
        x = x.sub_(s["slopes"].view(1, hk, gr, 1, 1) * (p - j).abs().float()[:, None, None])
    seen = torch.ones(1, nq, nk, dtype=torch.bool, device="cuda")
    if case["causal"]:
        seen = seen & (j <= p)
    if case["window"]:
        seen = seen & (p - j < case["window"])
    if case["prefix"]:
        seen = seen | (j < s["prefix"].view(b, 1, 1))
    if s["length"] is not None:
        seen = seen & (j < s["length"].view(b, 1, 1))
    if case["docs"]:
        seen = seen & (s["docs"][:, :nq, None] == s["docs"][:, None, :])
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(dim=-1, keepdim=True)
    x = x.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = x.sum(dim=-1, keepdim=True)
    y = (x.view(b, hk, gr * nq, nk) @ v).view(b, hk, gr, nq, d)
    y = torch.where(total > 0, y / total, torch.zeros_like(y)).to(s["q"].dtype).view(b, hk * gr, nq, d)
    if case["token_major"]:
        y = y.transpose(1, 2).reshape(b, nq, hk * gr * d)
    return [y]


_PLAIN = {"norm": _plain_norm, "q4": _plain_q4, "attention": _plain_attention}


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    return _PLAIN[case["kind"]](case, state)


# -- the definitions in 64 bits -------------------------------------------------


def _exact_norm(case, s):
    x = s["x"].to(torch.float64)
    total = x if s["r"] is None else x.add(s["r"].to(torch.float64))
    root = total.pow(2).sum(1).div(case["cols"]).add(_EPS).sqrt()
    y = total / root[:, None] * s["gamma"].to(torch.float64)
    if case["quantize"]:
        step = y.abs().max(1).values[:, None] / 127.0
        y = torch.round(y / step) * step
    return [y] if s["r"] is None else [total, y]


def _exact_q4(case, s):
    m, n, group = case["m"], case["n"], case["group"]
    y = torch.zeros(m, n, dtype=torch.float64, device="cuda")
    for i in range(case["k"] // group):
        at = slice(i * group, (i + 1) * group)
        part = s["x"][:, at].to(torch.float64) @ s["w"][:, at].to(torch.float64).t()
        y += part * s["scales"][:, i].to(torch.float64)
    if s["row_scale"] is not None:
        y *= s["row_scale"].to(torch.float64)
    return [y]


def _exact_attention(case, s):
    b, hk, gr, nq, nk, d = (case[k] for k in ("batch", "kv_heads", "group", "nq", "nk", "d"))
    major = case["token_major"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    keys = torch.arange(nk, device="cuda")
    for i in range(b):
        first = int(s["start"][i, 0]) if s["start"] is not None else 0
        at = torch.arange(first, first + nq, device="cuda")[:, None]
        blind = torch.zeros(nq, nk, dtype=torch.bool, device="cuda")
        if case["causal"]:
            blind |= keys > at
        if case["window"]:
            blind |= keys <= at - case["window"]
        if s["prefix"] is not None:
            blind[:, : int(s["prefix"][i, 0])] = False
        if s["length"] is not None:
            blind[:, int(s["length"][i, 0]):] = True
        if s["docs"] is not None:
            blind |= s["docs"][i, :nq].unsqueeze(1).ne(s["docs"][i])
        for h in range(hk * gr):
            c = h // gr
            if major:
                q, k, v = (s[n][i, :, e * d:(e + 1) * d].double() for n, e in (("q", h), ("k", c), ("v", c)))
            else:
                q, k, v = s["q"][i, h].double(), s["k"][i, c].double(), s["v"][i, c].double()
            x = torch.mm(q, k.t()) / math.sqrt(d)
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if s["slopes"] is not None:
                x = x - s["slopes"][c, h % gr].double() * torch.abs(at - keys)
            x[blind] = -math.inf
            y = torch.nan_to_num(torch.softmax(x, dim=1), nan=0.0) @ v
            if major:
                out[i, :, h * d:(h + 1) * d] = y
            else:
                out[i, h] = y
    return [out]


def exact(case, seed):
    state = _PREPARE[case["kind"]](case, _generator(seed))
    return {"norm": _exact_norm, "q4": _exact_q4, "attention": _exact_attention}[case["kind"]](case, state)
