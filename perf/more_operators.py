"""Operators that a language model answers with, as measurable cases.

Four operators of ``xtile_amd.kernels``: rows in microscaled 4-bit floating point
and back (``quantize_mx4``, ``dequantize_mx4``), products of such rows
(``matmul_mx4``), attention of a tree of drafted tokens to a cache
(``masked_attention`` with ``parents``) and the choice of a token from its logits
(``sample``).  A case is one of them at one size.  ``run`` computes it from
elementary torch operations, or, where ``own`` is true, launches the program that
``prepare`` planned, over buffers that the caller keeps.  ``listed`` holds fixed
cases from the smallest calls to the largest, ``draw`` gives more of the same
ranges.
"""

from __future__ import annotations

import math

import torch

own = False

_TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # One token's activations on their way into a 4-bit product.
        _rows("mx4_rows_token", 1, 4096, "bf16"),
        # A prompt's activations, far beyond the caches; the rounded values are
        # kept too, as training through the rounding does.
        _rows("mx4_rows_prompt", 8192, 4096, "bf16"),
        # A layer's weights back in 16 bits, for a path that has no 4-bit product.
        _rows("mx4_values_layer", 11008, 4096, "f16", back=True),
        # One token through a square layer.
        _product("mx4_token", 1, 4096, 4096, "bf16"),
        # A batch of decoding sequences through the wide layer of a feed-forward
        # block.
        _product("mx4_batch", 16, 11008, 4096, "f32"),
        # A few dozen tokens through a layer that no tile divides.
        _product("mx4_ragged", 37, 1000, 1056, "bf16"),
        # A prompt through the wide layer.
        _product("mx4_prompt", 4096, 11008, 4096, "bf16"),
        # A small tree of drafted tokens of one sequence.
        _tree("tree_small", 1, 8, 4, 16, 4096, 128, "bf16"),
        # A batch of sequences of different lengths, each with its own tree.
        _tree("tree_batch", 16, 8, 4, 32, 8192, 128, "bf16"),
        # A full tree at the end of a very long cache, scores capped.
        _tree("tree_long", 1, 8, 8, 64, 131072, 128, "f16", cap=50.0),
        # The next token of one sequence, from its most probable ones.
        _sample("sample_token", 1, 32768, "f32", top_k=50, top_p=0.9),
        # The next tokens of a batch, over a large vocabulary.
        _sample("sample_batch", 64, 131072, "f32", top_p=0.95, min_p=0.001),
    ]


def _rows(name, rows, cols, dtype, back=False):
    return {"name": name, "kind": "rows", "rows": rows, "cols": cols, "dtype": dtype, "back": back}


def _product(name, m, n, k, out):
    return {"name": name, "kind": "product", "m": m, "n": n, "k": k, "out": out}


def _tree(name, batch, kv_heads, group, nq, nk, d, dtype, cap=0.0, window=0, slopes=False, token_major=False):
    return {"name": name, "kind": "tree", "batch": batch, "kv_heads": kv_heads, "group": group, "nq": nq, "nk": nk,
            "d": d, "dtype": dtype, "cap": cap, "window": window, "slopes": slopes, "token_major": token_major}


def _sample(name, rows, vocab, dtype, top_k=0, top_p=0.0, min_p=0.0, temperature=True):
    return {"name": name, "kind": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "temperature": temperature,
            "top_k": top_k, "top_p": top_p, "min_p": min_p}


# -- more cases of the same ranges --------------------------------------------


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_rows(rng):
    return _rows("", _log(rng, 1, 11008), 32 * _log(rng, 2, 256), rng.choice(["f32", "f16", "bf16"]),
                 back=rng.random() < 0.3)


def _draw_product(rng):
    return _product("", _log(rng, 1, 4096), _log(rng, 64, 11008), 32 * _log(rng, 8, 344),
                    rng.choice(["f32", "f16", "bf16"]))


def _draw_tree(rng):
    nq = _log(rng, 1, 64)
    return _tree("", _log(rng, 1, 32), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 8]), nq,
                 _log(rng, max(64, nq), 131072), rng.choice([32, 64, 96, 128, 128, 160, 256]),
                 rng.choice(["f16", "bf16"]), cap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                 window=rng.choice([0, 0, 0, 1000]), slopes=rng.random() < 0.3, token_major=rng.random() < 0.3)


def _draw_sample(rng):
    return _sample("", _log(rng, 1, 256), _log(rng, 512, 200000), rng.choice(["f32", "f32", "f16", "bf16"]),
                   top_k=rng.choice([0, 0, _log(rng, 1, 2000)]), top_p=rng.choice([0.0, round(rng.uniform(0.05, 0.99), 3)]),
                   min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.2), 4)]), temperature=rng.random() < 0.7)


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 500)


def draw(rng):
    # No drawn case costs more than the largest listed one, nor holds more
    # scores than its plain form does.
    most = max(_cost(c) for c in listed())
    while True:
        c = rng.choice([_draw_rows, _draw_product, _draw_product, _draw_tree, _draw_tree, _draw_sample])(rng)
        small = c["kind"] != "tree" or c["batch"] * c["kv_heads"] * c["group"] * c["nq"] * c["nk"] <= 1 << 30
        if small and _cost(c) <= most:
            del c["name"]
            return c


# -- what a pass cannot do without --------------------------------------------


def _starts(case):
    """The tokens that each sequence's cache holds before its drafted ones."""
    b, room = case["batch"], case["nk"] - case["nq"]
    return [room - (i * room) // (2 * b) for i in range(b)]


def work(case):
    if case["kind"] == "rows":
        n, esize = case["rows"] * case["cols"], _SIZE[case["dtype"]]
        packed = n // 2 + n // 32
        # quantised: x, the packed rows, their scales and the values; back: packed, scales, values
        return {"bytes": n * esize + packed if case["back"] else 2 * n * esize + packed, "flops": 4 * n}
    if case["kind"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * (k // 2 + k // 32) + m * n * _SIZE[case["out"]], "flops": 2 * m * n * k}
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * _SIZE[case["dtype"]] + case["rows"] * 24, "flops": 8 * n}
    heads, d = case["kv_heads"] * case["group"], case["d"]
    seen = [s + case["nq"] for s in _starts(case)]
    if case["window"]:
        seen = [min(s, case["window"] + case["nq"] - 1) for s in seen]
    moved = 2 * case["batch"] * heads * case["nq"] * d * 2 + 2 * case["kv_heads"] * sum(seen) * d * 2
    moved += case["batch"] * case["nq"] * 4
    # a drafted token sees the cache; what it sees of the tree is little beside that
    return {"bytes": moved, "flops": 4 * d * heads * case["nq"] * sum(seen)}


# -- inputs ---------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _power(e):
    """2 ** e in 64 bits, of integers of a double's normal range."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _mx4(x):
    """(nibbles [R, C] uint8, exponent bytes [R, C / 32] uint8) of a float tensor, in 64 bits."""
    rows, cols = x.shape
    b = x.double().view(rows, cols // 32, 32)
    top = b.abs().amax(dim=2)
    byte = (torch.frexp(top).exponent - 1 - 2 + 127).clamp_(min=0)
    byte = torch.where(top == 0, torch.zeros_like(byte), byte)
    y = b * _power(127 - byte)[:, :, None]
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0).to(a.dtype))
    a = ((a / step).round() * step).clamp_(max=6.0)
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = code | (torch.signbit(y).to(torch.uint8) << 3)
    return code.view(rows, cols), byte.to(torch.uint8)


def _packed(code, byte):
    """As the programs hold them: two nibbles a byte, the first the lower one, in int8."""
    return (code[:, 0::2] | (code[:, 1::2] << 4)).view(torch.int8), byte.view(torch.int8)


def _prepare_rows(case, g):
    rows, cols = case["rows"], case["cols"]
    # a few columns are much larger than the rest, as in a model's activations
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x *= torch.exp(torch.randn(1, cols, generator=g, device="cuda"))
    x = x.to(_TORCH[case["dtype"]])
    if not case["back"]:
        return {"x": x}
    q, s = _packed(*_mx4(x))
    return {"q": q, "s": s}


def _prepare_product(case, g):
    m, n, k = case["m"], case["n"], case["k"]
    s = {}
    s["x"], s["xs"] = _packed(*_mx4(torch.randn(m, k, generator=g, device="cuda")))
    s["w"], s["ws"] = _packed(*_mx4(0.02 * torch.randn(n, k, generator=g, device="cuda")))
    return s


def _prepare_tree(case, g):
    b, hk, gr, nq, nk, d = (case[k] for k in ("batch", "kv_heads", "group", "nq", "nk", "d"))
    t = _TORCH[case["dtype"]]
    q_shape, k_shape = (b, hk * gr, nq, d), (b, hk, nk, d)
    if case["token_major"]:
        q_shape, k_shape = (b, nq, hk * gr * d), (b, nk, hk * d)
    s = {"q": (2 * torch.randn(q_shape, generator=g, device="cuda")).to(t),
         "k": torch.randn(k_shape, generator=g, device="cuda").to(t),
         "v": torch.randn(k_shape, generator=g, device="cuda").to(t)}
    h = hk * gr
    s["slopes"] = None
    if case["slopes"]:
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, h + 1, device="cuda", dtype=torch.float32) / h).view(hk, gr)
    s["start"] = torch.tensor(_starts(case), dtype=torch.int32, device="cuda").view(b, 1)
    s["length"] = s["start"] + nq
    # a token continues one of the eight before it, or the sequence itself
    back = (8 * torch.rand(b, nq, generator=g, device="cuda")).to(torch.int32)
    node = torch.arange(nq, device="cuda", dtype=torch.int32)
    s["parents"] = (node - 1 - back).clamp(min=-1).contiguous()
    return s


def _prepare_sample(case, g):
    rows, vocab = case["rows"], case["vocab"]
    # a model's logits: most far below the few that it means
    x = 2.5 * torch.randn(rows, vocab, generator=g, device="cuda")
    x += 4 * (torch.rand(rows, vocab, generator=g, device="cuda") < 20 / vocab)
    s = {"x": x.to(_TORCH[case["dtype"]]), "u": torch.rand(rows, 1, generator=g, device="cuda")}
    ones = torch.ones(rows, 1, device="cuda")
    s["temperature"] = 0.6 + 0.6 * torch.rand(rows, 1, generator=g, device="cuda") if case["temperature"] else None
    s["top_k"] = (ones * case["top_k"]).to(torch.int32) if case["top_k"] else None
    s["top_p"] = ones * case["top_p"] if case["top_p"] else None
    s["min_p"] = ones * case["min_p"] if case["min_p"] else None
    return s


_PREPARE = {"rows": _prepare_rows, "product": _prepare_product, "tree": _prepare_tree, "sample": _prepare_sample}


def prepare(case, seed):
    state = _PREPARE[case["kind"]](case, _generator(seed))
    state["case"] = dict(case)
    if own:
        _PLAN[case["kind"]](case, state)
    return state


# -- the framework's programs ---------------------------------------------------


def _dsl(name):
    import xtile_amd as xt

    return {"f32": xt.float32, "f16": xt.float16, "bf16": xt.bfloat16}[name]


def _plan_rows(case, s):
    import xtile_amd as xt
    from xtile_amd import kernels as K

    rows, cols = case["rows"], case["cols"]
    s["y"] = torch.empty(rows, cols, dtype=_TORCH[case["dtype"]], device="cuda")
    if case["back"]:
        s["program"] = xt.compile(K.dequantize_mx4(rows, cols, _dsl(case["dtype"])))
        s["buffers"] = [s["q"], s["s"], s["y"]]
        return
    s["program"] = xt.compile(K.quantize_mx4(rows, cols, _dsl(case["dtype"]), values=True))
    s["q"] = torch.empty(rows, cols // 2, dtype=torch.int8, device="cuda")
    s["s"] = torch.empty(rows, cols // 32, dtype=torch.int8, device="cuda")
    s["buffers"] = [s["x"], s["q"], s["s"], s["y"]]


def _plan_product(case, s):
    import xtile_amd as xt
    from xtile_amd import kernels as K

    s["program"] = xt.compile(K.matmul_mx4(case["m"], case["n"], case["k"], out=_dsl(case["out"])))
    s["y"] = torch.empty(case["m"], case["n"], dtype=_TORCH[case["out"]], device="cuda")
    s["buffers"] = [s["x"], s["xs"], s["w"], s["ws"], s["y"]]


def _plan_tree(case, s):
    import xtile_amd as xt
    from xtile_amd import kernels as K

    s["program"] = xt.compile(K.masked_attention(
        case["batch"], case["kv_heads"], case["group"], case["nq"], case["nk"], case["d"], dtype=_dsl(case["dtype"]),
        cap=case["cap"] or None, window=case["window"] or None, slopes=case["slopes"], start=True, length=True,
        parents=True, token_major=case["token_major"]))
    s["y"] = torch.empty_like(s["q"])
    extra = [s[k] for k in ("slopes", "start", "length", "parents") if s[k] is not None]
    s["buffers"] = [s["q"], s["k"], s["v"], *extra, s["y"]]


def _plan_sample(case, s):
    import xtile_amd as xt
    from xtile_amd import kernels as K

    names = [k for k in ("temperature", "top_k", "top_p", "min_p") if s[k] is not None]
    s["program"] = xt.compile(K.sample(case["rows"], case["vocab"], _dsl(case["dtype"]), **{k: True for k in names}))
    s["y"] = torch.empty(case["rows"], 1, dtype=torch.int32, device="cuda")
    s["buffers"] = [s["x"], s["u"], *[s[k] for k in names], s["y"]]


_PLAN = {"rows": _plan_rows, "product": _plan_product, "tree": _plan_tree, "sample": _plan_sample}


def _run_own(case, s):
    import xtile_amd as xt

    xt.launch(s["program"], *s["buffers"])
    if case["kind"] == "rows" and not case["back"]:
        return [s["y"], s["s"]]
    return [s["y"]]


# -- the plain forms ------------------------------------------------------------


def _values(q, s):
    """The values of packed rows and their scales, in 32 bits."""
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=q.device)
    u = q.view(torch.uint8)
    rows, half = u.shape
    v = torch.stack((table[(u & 15).int()], table[(u >> 4).int()]), dim=2).view(rows, s.shape[1], 2 * half // s.shape[1])
    exponent = s.view(torch.uint8).int()
    scale = (exponent << 23).view(torch.float32).masked_fill_(exponent == 0, 2.0**-127)
    return (v * scale[:, :, None]).view(rows, 2 * half)


def _plain_rows(case, s):
    if case["back"]:
        return [_values(s["q"], s["s"]).to(_TORCH[case["dtype"]])]
    q, scale = _packed(*_mx4(s["x"]))
    return [_values(q, scale).to(s["x"].dtype), scale]


def _plain_product(case, s):
    y = _values(s["x"], s["xs"]) @ _values(s["w"], s["ws"]).t()
    return [y.to(_TORCH[case["out"]])]


def _heads_first(case, x, heads, n):
    """[batch, kv_heads, heads / kv_heads * n, d] in 32 bits."""
    b, hk, d = case["batch"], case["kv_heads"], case["d"]
    x = x.float()
    if case["token_major"]:
        x = x.view(b, n, heads, d).transpose(1, 2)
    return x.reshape(b, hk, heads // hk * n, d)


def _ancestors(parents):
    """[batch, nq, nq]: whether a token is another's ancestor, or itself."""
    b, nq = parents.shape
    own_ = torch.eye(nq, dtype=torch.bool, device=parents.device).expand(b, nq, nq)
    step = (parents[:, :, None] == torch.arange(nq, device=parents.device)).float()
    reach = own_
    for _ in range(max(1, (nq - 1).bit_length())):  # paths of up to twice the length
        reach = reach | ((step @ reach.float()) > 0)
        step = ((step @ step) > 0).float()
    return reach


def _plain_tree(case, s):
    b, hk, gr, nq, nk, d = (case[k] for k in ("batch", "kv_heads", "group", "nq", "nk", "d"))
    q = _heads_first(case, s["q"], hk * gr, nq)
    k = _heads_first(case, s["k"], hk, nk)
    v = _heads_first(case, s["v"], hk, nk)
    x = (q @ k.transpose(2, 3)).mul_(1 / math.sqrt(d)).view(b, hk, gr, nq, nk)
    if case["cap"]:
        x = x.div_(case["cap"]).tanh_().mul_(case["cap"])
    start = s["start"].long()
    reach = _ancestors(s["parents"])
    depth = reach.sum(dim=2) - 1
    # the position of a key: its place in the cache, or its depth in the tree behind it
    node = torch.arange(nk, device="cuda") - start
    in_tree = (node >= 0) & (node < nq)
    at = node.clamp(0, nq - 1)
    k_pos = torch.where(in_tree, start + depth.gather(1, at), start + node)
    away = (start + depth)[:, :, None] - k_pos[:, None, :]
    seen = torch.where(in_tree[:, None, :], reach.gather(2, at[:, None, :].expand(b, nq, nk)), (node < 0)[:, None, :])
    if case["window"]:
        seen = seen & (away < case["window"])
    seen = seen & (torch.arange(nk, device="cuda") < s["length"])[:, None, :]
    if case["slopes"]:
        x = x.sub_(s["slopes"].view(1, hk, gr, 1, 1) * away.abs().float()[:, None, None])
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(dim=-1, keepdim=True)
    x = x.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = x.sum(dim=-1, keepdim=True)
    y = (x.view(b, hk, gr * nq, nk) @ v).view(b, hk, gr, nq, d)
    y = torch.where(total > 0, y / total, torch.zeros_like(y)).to(s["q"].dtype).view(b, hk * gr, nq, d)
    if case["token_major"]:
        y = y.transpose(1, 2).reshape(b, nq, hk * gr * d)
    return [y]


def _plain_sample(case, s):
    vocab = case["vocab"]
    z, order = s["x"].sort(dim=1, descending=True, stable=True)  # equal ones: the lowest index first
    z = z.double()
    z = z - z[:, :1]
    if s["temperature"] is not None:
        z = z / s["temperature"].double()
    w = z.exp()
    rank = torch.arange(vocab, device="cuda")
    kept = torch.ones_like(w, dtype=torch.bool)
    if s["top_k"] is not None:
        kept &= rank < s["top_k"]
    total = (w * kept).cumsum(dim=1)
    if s["top_p"] is not None:
        kept &= total - w < s["top_p"].double() * total[:, -1:]  # what comes before it has not reached p
    if s["min_p"] is not None:
        kept &= w >= s["min_p"].double()
    total = (w * kept).cumsum(dim=1)
    at = (total > s["u"].double() * total[:, -1:]).int().argmax(dim=1, keepdim=True)
    return [order.gather(1, at).int()]


_PLAIN = {"rows": _plain_rows, "product": _plain_product, "tree": _plain_tree, "sample": _plain_sample}


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    return _PLAIN[case["kind"]](case, state)


# -- the definitions in 64 bits -------------------------------------------------


def _exact_values(q, s):
    """The values of packed rows, bit by bit."""
    out = torch.zeros(q.shape[0], 2 * q.shape[1], dtype=torch.float64, device=q.device)
    scale = torch.exp2((s.long() & 255).double() - 127).repeat_interleave(2 * q.shape[1] // s.shape[1], dim=1)
    bits = q.long() & 255
    for i in range(2):
        n = (bits >> (4 * i)) & 15
        exponent, mantissa = (n >> 1) & 3, (n & 1).double()
        size = torch.where(exponent > 0, torch.exp2(exponent.double() - 1) * (1 + mantissa / 2), mantissa / 2)
        out[:, i::2] = torch.where(n > 7, -size, size)
    return out * scale


def _exact_rows(case, s):
    if case["back"]:
        return [_exact_values(s["q"], s["s"])]
    x = s["x"].double()
    rows, cols = x.shape
    blocks = x.reshape(rows * cols // 32, 32)
    peak = blocks.abs().max(dim=1).values
    exponent = torch.where(peak > 0, torch.floor(torch.log2(peak)) - 2, -127.0).clamp(min=-127)
    unit = torch.exp2(exponent)[:, None]
    size = blocks.abs() / unit
    # the nearest of the eight magnitudes; halfway between two the one whose last bit is 0
    nearest = torch.zeros_like(size)
    for i in range(1, 8):
        half = (_E2M1[i - 1] + _E2M1[i]) / 2
        over = size > half if i % 2 else size >= half
        nearest = torch.where(over, _E2M1[i], nearest)
    y = torch.where(blocks < 0, -nearest, nearest) * unit
    return [y.view(rows, cols), (exponent + 127).to(torch.uint8).view(torch.int8).view(rows, cols // 32)]


def _exact_product(case, s):
    x = _exact_values(s["x"], s["xs"])
    y = torch.empty(case["m"], case["n"], dtype=torch.float64, device="cuda")
    for n in range(0, case["n"], 2048):
        y[:, n:n + 2048] = torch.mm(x, _exact_values(s["w"][n:n + 2048], s["ws"][n:n + 2048]).t())
    return [y]


def _exact_tree(case, s):
    b, hk, gr, nq, nk, d = (case[k] for k in ("batch", "kv_heads", "group", "nq", "nk", "d"))
    major = case["token_major"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i in range(b):
        first, length, parents = int(s["start"][i, 0]), int(s["length"][i, 0]), s["parents"][i].tolist()
        place = torch.arange(nk, dtype=torch.float64)
        blind = torch.ones(nq, nk, dtype=torch.bool)
        blind[:, :first] = False
        depth = [0] * nq
        for t in range(nq):  # up the tree, one token at a time
            up = t
            while up >= 0:
                blind[t, first + up] = False
                if up != t:
                    depth[t] += 1
                up = parents[up]
            place[first + t] = first + depth[t]
        blind[:, length:] = True
        far = torch.tensor([first + x for x in depth], dtype=torch.float64)[:, None] - place
        if case["window"]:
            blind |= far >= case["window"]
        blind, far = blind.cuda(), far.abs().cuda()
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
                x = x - s["slopes"][c, h % gr].double() * far
            x[blind] = -math.inf
            y = torch.nan_to_num(torch.softmax(x, dim=1), nan=0.0) @ v
            if major:
                out[i, :, h * d:(h + 1) * d] = y
            else:
                out[i, h] = y
    return [out]


def _exact_sample(case, s):
    tokens = []
    for r in range(case["rows"]):
        x = s["x"][r].double()
        t = float(s["temperature"][r, 0]) if s["temperature"] is not None else 1.0
        # by value, then by index: a sort by index is kept by a stable one by value
        order = torch.argsort(-x, stable=True)
        if s["top_k"] is not None:
            order = order[: int(s["top_k"][r, 0])]
        p = torch.softmax(x[order] / t, dim=0)
        before = torch.cat((torch.zeros(1, dtype=torch.float64, device="cuda"), torch.cumsum(p, 0)[:-1]))
        n = len(order)
        if s["top_p"] is not None:
            n = min(n, int((before < float(s["top_p"][r, 0])).sum()))
        if s["min_p"] is not None:
            n = min(n, int((p >= float(s["min_p"][r, 0]) * p[0]).sum()))
        cdf = torch.cumsum(p[:n], 0)
        tokens.append(order[(cdf <= float(s["u"][r, 0]) * cdf[-1]).sum().clamp(max=n - 1)])
    return [torch.stack(tokens).int().view(-1, 1)]


def exact(case, seed):
    state = _PREPARE[case["kind"]](case, _generator(seed))
    return {"rows": _exact_rows, "product": _exact_product, "tree": _exact_tree, "sample": _exact_sample}[
        case["kind"]](case, state)
