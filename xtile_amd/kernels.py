"""Example tile programs: the reference's kernels/*.py, written with this DSL.

Each builder returns a parsed Module for one configuration.  They reproduce
the reference programs (kernels/add.py:6-30, kernels/softmax.py:10-36,
kernels/matmul.py:6-38, kernels/conv2d.py:10-59) with
the tile sizes of the five benchmark configurations:

  C1 add      fp32 1024x1024, 32x64 tiles, grid (32, 16, 1)
  C2 softmax  fp32 8192x4096, one 1x4096 row per Block, grid (8192, 1, 1)
  C3 matmul   f16 4096^3 -> f32, 128x128 Block tiles (full K), B shared along axis 0
  C4 conv2d   f16 NHWC 32x56x56x64, 3x3x64x64 filter, stride 1, pad 1 -> f32
  C5 matmul   bf16 4096x11008x4096 -> f32, 256x128 tiles, grid (86, 16, 1),
              A shared along axis 0 (`shared = 1`)

Beside them: `layernorm`, `column_softmax`, `bias_add` and `attention`, and the
operators of a language model's layer: `rms_norm`, `matmul_q4`, `quantize_mx4`,
`dequantize_mx4`, `matmul_mx4`, `masked_attention` and `sample`.
"""

from __future__ import annotations

from . import (
    Array,
    add as tile_add,
    astype,
    attend,
    bfloat16,
    bid,
    cdiv,
    convert,
    dequantize_mx4 as tile_dequantize_mx4,
    exp,
    float16,
    float32,
    int8,
    int32,
    kernel,
    load,
    load_conv2d,
    matmul,
    matmul_mx4 as tile_matmul_mx4,
    matmul_q4 as tile_matmul_q4,
    max as tile_max,
    mul as tile_mul,
    mx4_scale,
    quantize,
    quantize_mx4 as tile_quantize_mx4,
    reciprocal,
    rms_norm as tile_rms_norm,
    row_scale as tile_row_scale,
    rsqrt,
    reshape,
    sample as tile_sample,
    store,
    sub as tile_sub,
    sum as tile_sum,
    transpose,
)


# -- add ---------------------------------------------------------------------


@kernel
def add_kernel(lhs, rhs, out, tile_h, tile_w):
    b0 = bid(0)
    b1 = bid(1)
    a = load(lhs, index=(b0, b1), shape=(tile_h, tile_w))
    b = load(rhs, index=(b0, b1), shape=(tile_h, tile_w))
    store(out, index=(b0, b1), tile=a + b)


def add(rows: int, cols: int, tile_h: int = 32, tile_w: int = 64):
    arr = Array(shape=(rows, cols), dtype=float32)
    grid = (cdiv(rows, tile_h), cdiv(cols, tile_w), 1)
    return convert(add_kernel, args=(arr, arr, arr, tile_h, tile_w), grid=grid, double_buffering=True)


@kernel
def add_rows_kernel(lhs, rhs, out, trow, col):
    """The reference's kernels/add.py program: full-width row tiles."""
    bid_x = bid(0)
    a = load(lhs, index=(bid_x, 0), shape=(trow, col))
    b = load(rhs, index=(bid_x, 0), shape=(trow, col))
    store(out, index=(bid_x, 0), tile=a + b)


def add_rows(rows: int, cols: int, trow: int = 64):
    arr = Array(shape=(rows, cols), dtype=float32)
    return convert(
        add_rows_kernel,
        args=(arr, arr, arr, trow, cols),
        grid=(cdiv(rows, trow), 1, 1),
        double_buffering=True,
    )


# -- softmax -----------------------------------------------------------------


@kernel
def softmax_kernel(inp, out, trow, col):
    bid_x = bid(0)
    x = load(inp, index=(bid_x, 0), shape=(trow, col))
    x = x - tile_max(x, axis=-1)
    x = exp(x)
    r = tile_sum(x, axis=-1)
    x = x / r
    store(out, index=(bid_x, 0), tile=x)


def softmax(rows: int, cols: int, trow: int = 1):
    arr = Array(shape=(rows, cols), dtype=float32)
    return convert(
        softmax_kernel,
        args=(arr, arr, trow, cols),
        grid=(cdiv(rows, trow), 1, 1),
        double_buffering=True,
    )


# -- matmul ------------------------------------------------------------------


@kernel
def matmul_kernel(lhs, rhs, res, tm, tn, tk):
    """A row panel per bid(0), B column panel per bid(1) shared along axis 0."""
    bid_m = bid(0)
    bid_n = bid(1)
    a = load(lhs, index=(bid_m, 0), shape=(tm, tk))
    b = load(rhs, index=(0, bid_n), shape=(tk, tn), shared=1)
    store(res, index=(bid_m, bid_n), tile=matmul(a, b))


@kernel
def matmul_nm_kernel(lhs, rhs, res, tm, tn, tk):
    """Grid (N/tn, M/tm): bid(0) walks N, so the A panel is `shared = 1`."""
    bid_n = bid(0)
    bid_m = bid(1)
    a = load(lhs, index=(bid_m, 0), shape=(tm, tk), shared=1)
    b = load(rhs, index=(0, bid_n), shape=(tk, tn))
    store(res, index=(bid_m, bid_n), tile=matmul(a, b))


def matmul_f16(m: int, n: int, k: int, tm: int = 128, tn: int = 128):
    a = Array(shape=(m, k), dtype=float16)
    b = Array(shape=(k, n), dtype=float16)
    c = Array(shape=(m, n), dtype=float32)
    return convert(
        matmul_kernel,
        args=(a, b, c, tm, tn, k),
        grid=(cdiv(m, tm), cdiv(n, tn), 1),
        double_buffering=True,
    )


def matmul_bf16(m: int, n: int, k: int, tm: int = 256, tn: int = 128):
    a = Array(shape=(m, k), dtype=bfloat16)
    b = Array(shape=(k, n), dtype=bfloat16)
    c = Array(shape=(m, n), dtype=float32)
    return convert(
        matmul_nm_kernel,
        args=(a, b, c, tm, tn, k),
        grid=(cdiv(n, tn), cdiv(m, tm), 1),
        double_buffering=True,
    )


@kernel
def matmul_i8_kernel(lhs, rhs, res, scale, bias, tm, tn, tk):
    """kernels/matmul.py:6-19: i8 x i8 -> f32, then * scale + bias per column
    and astype(int8); B, scale and bias are shared along axis 0."""
    bid_x = bid(0)
    bid_y = bid(1)
    lhs_tile = load(lhs, index=(bid_x, 0), shape=(tm, tk))
    rhs_tile = load(rhs, index=(0, bid_y), shape=(tk, tn), shared=1)
    s_tile = load(scale, index=(0, bid_y), shape=(1, tn), shared=1)
    b_tile = load(bias, index=(0, bid_y), shape=(1, tn), shared=1)
    t = matmul(lhs_tile, rhs_tile)
    t = t * s_tile + b_tile
    t = astype(t, dtype=int8)
    store(res, index=(bid_x, bid_y), tile=t)


def matmul_i8(m: int, n: int, k: int, tm: int = 64, tn: int = 64):
    """The reference's matmul program (kernels/matmul.py:22-38, 64 x 64 tiles)."""
    a = Array(shape=(m, k), dtype=int8)
    b = Array(shape=(k, n), dtype=int8)
    c = Array(shape=(m, n), dtype=int8)
    s = Array(shape=(1, n), dtype=float32)
    bias = Array(shape=(1, n), dtype=float32)
    return convert(
        matmul_i8_kernel,
        args=(a, b, c, s, bias, tm, tn, k),
        grid=(cdiv(m, tm), cdiv(n, tn), 1),
        double_buffering=True,
    )


# -- conv2d ------------------------------------------------------------------


@kernel
def conv2d_kernel(inp, filt, out, tile_h, tile_w, cin, cout, kh, kw, pt, pl, pb, pr, sh, sw, dh, dw):
    bid_n = bid(0)
    bid_h = bid(1)
    bid_w = bid(2)
    zero = 0
    f = load(filt, index=(zero, zero, zero, zero), shape=(kh, kw, cin, cout), shared=2)
    t = load_conv2d(
        inp,
        f,
        index=(bid_n, bid_h, bid_w, zero),
        shape=(1, tile_h, tile_w, cout),
        group=1,
        pad=(pt, pl, pb, pr),
        stride=(sh, sw),
        dilation=(dh, dw),
    )
    store(out, index=(bid_n, bid_h, bid_w, zero), tile=t)


def conv2d(n, h, w, cin, cout, kh=3, kw=3, tile_h=4, tile_w=56, dtype=float16, pad=None, stride=(1, 1),
           dilation=(1, 1)):
    """NHWC conv; `pad` is (top, left, bottom, right), by default "same" for odd
    filters as in kernels/conv2d.py:29.  The output is (n, oh, ow, cout)."""
    if pad is None:
        pad = (kh // 2, kw // 2, kh // 2, kw // 2)
    oh = (h + pad[0] + pad[2] - dilation[0] * (kh - 1) - 1) // stride[0] + 1
    ow = (w + pad[1] + pad[3] - dilation[1] * (kw - 1) - 1) // stride[1] + 1
    if oh <= 0 or ow <= 0 or oh % tile_h or ow % tile_w:
        raise ValueError("tile_h / tile_w must divide the output height / width")
    inp = Array(shape=(n, h, w, cin), dtype=dtype)
    filt = Array(shape=(kh, kw, cin, cout), dtype=dtype)
    out = Array(shape=(n, oh, ow, cout), dtype=float32)
    return convert(
        conv2d_kernel,
        args=(inp, filt, out, tile_h, tile_w, cin, cout, kh, kw, *pad, *stride, *dilation),
        grid=(n, oh // tile_h, ow // tile_w),
        double_buffering=True,
    )


# -- programs for the tile interpreter ----------------------------------------


@kernel
def layernorm_kernel(inp, gamma, beta, inv_n, eps, out, trow, col):
    """Row layernorm, the xt form of the reference's layernorm program
    (test/nova/to_x1.mlir:82-128: reduce, broadcast subtract, square, reduce,
    scale by 1/C plus epsilon, rsqrt, scale by gamma, add beta).  The DSL has
    no scalar operands, so 1/C and epsilon are (1, 1) tiles."""
    row = bid(0)
    x = load(inp, index=(row, 0), shape=(trow, col))
    g = load(gamma, index=(0, 0), shape=(1, col), shared=1)
    b = load(beta, index=(0, 0), shape=(1, col), shared=1)
    n = load(inv_n, index=(0, 0), shape=(1, 1), shared=1)
    e = load(eps, index=(0, 0), shape=(1, 1), shared=1)
    mean = tile_mul(tile_sum(x, axis=1), n)
    xc = tile_sub(x, mean)
    var = tile_mul(tile_sum(tile_mul(xc, xc), axis=1), n)
    r = rsqrt(tile_add(var, e))
    y = tile_add(tile_mul(tile_mul(xc, r), g), b)
    store(out, index=(row, 0), tile=y)


def layernorm(rows: int, cols: int, trow: int = 64):
    if rows % trow:
        raise ValueError("trow must divide rows")
    a = Array(shape=(rows, cols), dtype=float32)
    v = Array(shape=(1, cols), dtype=float32)
    s = Array(shape=(1, 1), dtype=float32)
    return convert(layernorm_kernel, args=(a, v, v, s, s, a, trow, cols), grid=(rows // trow, 1, 1),
                   double_buffering=True)


@kernel
def column_softmax_kernel(inp, out, row, tcol):
    """Softmax down the columns of a (row, tcol) tile: reductions over axis 0."""
    c = bid(0)
    x = load(inp, index=(0, c), shape=(row, tcol))
    m = tile_max(x, axis=0)
    ex = exp(tile_sub(x, m))
    y = tile_mul(ex, reciprocal(tile_sum(ex, axis=0)))
    store(out, index=(0, c), tile=y)


def column_softmax(rows: int, cols: int, tcol: int = 32):
    if cols % tcol:
        raise ValueError("tcol must divide cols")
    a = Array(shape=(rows, cols), dtype=float32)
    return convert(column_softmax_kernel, args=(a, a, rows, tcol), grid=(cols // tcol, 1, 1))


@kernel
def bias_add_kernel(inp, bias, out, trow, tcol):
    """x + bias with a (1, tcol) bias row broadcast over the tile's rows."""
    r = bid(0)
    c = bid(1)
    x = load(inp, index=(r, c), shape=(trow, tcol))
    b = load(bias, index=(0, c), shape=(1, tcol), shared=1)
    store(out, index=(r, c), tile=tile_add(x, b))


def bias_add(rows: int, cols: int, trow: int = 32, tcol: int = 64):
    a = Array(shape=(rows, cols), dtype=float32)
    v = Array(shape=(1, cols), dtype=float32)
    return convert(bias_add_kernel, args=(a, v, a, trow, tcol), grid=(rows // trow, cols // tcol, 1))


@kernel
def attention_kernel(q, k, v, o, tq, d, nk):
    """softmax(Q K^T) V for one query tile of one head: Q, V and the result
    are [heads, rows, d], K is [heads, nk, d].  The head's K and V tiles are
    shared by its query tiles (`shared = 1`); K^T comes from the DSL's rank-3
    transpose (xtile/dsl.py:426-438); P V multiplies the f32 probabilities by
    an f32 V, since matmul operands share a dtype (xtile/dsl.py:369-374)."""
    i = bid(0)
    h = bid(1)
    qt = reshape(load(q, index=(h, i, 0), shape=(1, tq, d)), shape=(tq, d))
    kt = load(k, index=(h, 0, 0), shape=(1, nk, d), shared=1)
    vt = reshape(load(v, index=(h, 0, 0), shape=(1, nk, d), shared=1), shape=(nk, d))
    ktt = reshape(transpose(kt), shape=(d, nk))
    s = matmul(qt, ktt)
    p = exp(tile_sub(s, tile_max(s, axis=1)))
    p = tile_mul(p, reciprocal(tile_sum(p, axis=1)))
    store(o, index=(h, i, 0), tile=reshape(matmul(p, vt), shape=(1, tq, d)))


def attention(heads: int, nq: int, nk: int, d: int, tq: int = 64, qk=float16):
    """Grid (nq / tq, heads, 1).  `qk` is the element type of Q and K (f16,
    bf16 or f32: their product is f32); V and the result are f32."""
    if nq % tq:
        raise ValueError("tq must divide nq")
    qa = Array(shape=(heads, nq, d), dtype=qk)
    ka = Array(shape=(heads, nk, d), dtype=qk)
    va = Array(shape=(heads, nk, d), dtype=float32)
    oa = Array(shape=(heads, nq, d), dtype=float32)
    return convert(attention_kernel, args=(qa, ka, va, oa, tq, d, nk), grid=(nq // tq, heads, 1))


# -- operators of a language model's layer -------------------------------------


def rms_norm(rows: int, cols: int, dtype=bfloat16, *, residual: bool = True, quantize: bool = False, eps: float = 1e-6,
             gamma=None, trow: int = 1):
    """Root-mean-square norm of rows, after the residual's addition, to rows of the
    input's type or to int8 rows with a float32 scale each.

    Buffers: x, [the residual], gamma (1, cols) of dtype `gamma` (default: `dtype`),
    [the sum], then y, or the int8 rows and their (rows, 1) scales.  The sum is
    held in 32 bits for the norm and rounded where it is stored; it may be stored
    over x or the residual (pass one tensor twice)."""
    if rows % trow:
        raise ValueError("trow must divide rows")
    x = Array(shape=(rows, cols), dtype=dtype)
    g = Array(shape=(1, cols), dtype=gamma or dtype)
    rows8, scales = Array(shape=(rows, cols), dtype=int8), Array(shape=(rows, 1), dtype=float32)
    to_rows8 = quantize
    ins = 2 if residual else 1

    def body(args):
        r = bid(0)
        h = load(args[0], index=(r, 0), shape=(trow, cols))
        if residual:
            h = tile_add(h, load(args[1], index=(r, 0), shape=(trow, cols)))
            store(args[3], index=(r, 0), tile=h)
        y = tile_rms_norm(h, load(args[ins], index=(0, 0), shape=(1, cols), shared=1), eps=eps)
        if to_rows8:
            s = tile_row_scale(y)
            store(args[-2], index=(r, 0), tile=_quantize(y, s))
            store(args[-1], index=(r, 0), tile=s)
        else:
            store(args[-1], index=(r, 0), tile=y)

    arrays = [x] * ins + [g] + ([x] if residual else []) + ([rows8, scales] if quantize else [x])
    return convert(_named("rms_norm_kernel", body, len(arrays)), args=tuple(arrays), grid=(rows // trow, 1, 1))


def matmul_q4(m: int, n: int, k: int, *, group: int = 128, dtype=bfloat16, scales=float16, out=float32,
              row_scale: bool = False):
    """x (m, k) against n rows of k 4-bit weights with a scale for each `group` of a row.

    Buffers: x of `dtype` (float16, bfloat16 or int8), the weights (n, k / 2) int8
    from `pack_q4`, their scales (n, k / group), [row scales (m, 1) float32], y (m, n)."""
    if group < 1 or k % group:
        raise ValueError("group must divide k")
    arrays = [Array(shape=(m, k), dtype=dtype), Array(shape=(n, k // 2), dtype=int8),
              Array(shape=(n, k // group), dtype=scales)]
    if row_scale:
        arrays.append(Array(shape=(m, 1), dtype=float32))

    def body(args):
        tiles = [load(a, index=(0, 0), shape=t.shape) for a, t in zip(args, arrays)]
        y = tile_matmul_q4(*tiles[:3], row_scale=tiles[3] if row_scale else None, dtype=out)
        store(args[-1], index=(0, 0), tile=y)

    args = (*arrays, Array(shape=(m, n), dtype=out))
    return convert(_named("matmul_q4_kernel", body, len(args)), args=args, grid=(1, 1, 1))


def quantize_mx4(rows: int, cols: int, dtype=bfloat16, *, values: bool = False):
    """Rows in microscaled 4-bit floating point: blocks of 32 values with a scale each.

    Buffers: x (rows, cols), the rows (rows, cols / 2) int8, their scales (rows,
    cols / 32) int8 and, with `values`, what they stand for (rows, cols) of `dtype`."""
    arrays = [Array(shape=(rows, cols), dtype=dtype), *_mx4_arrays(rows, cols)]
    if values:
        arrays.append(arrays[0])

    def body(args):
        x = load(args[0], index=(0, 0), shape=(rows, cols))
        s = mx4_scale(x)
        q = tile_quantize_mx4(x, s)
        store(args[1], index=(0, 0), tile=q)
        store(args[2], index=(0, 0), tile=s)
        if values:
            store(args[3], index=(0, 0), tile=tile_dequantize_mx4(q, s, dtype=dtype))

    return convert(_named("quantize_mx4_kernel", body, len(arrays)), args=tuple(arrays), grid=(1, 1, 1))


def dequantize_mx4(rows: int, cols: int, dtype=bfloat16):
    """The values of such rows.  Buffers: the rows (rows, cols / 2) int8, their scales
    (rows, cols / 32) int8, y (rows, cols) of `dtype`."""
    arrays = [*_mx4_arrays(rows, cols), Array(shape=(rows, cols), dtype=dtype)]

    def body(args):
        q, s = (load(a, index=(0, 0), shape=t.shape) for a, t in zip(args, arrays[:2]))
        store(args[2], index=(0, 0), tile=tile_dequantize_mx4(q, s, dtype=dtype))

    return convert(_named("dequantize_mx4_kernel", body, 3), args=tuple(arrays), grid=(1, 1, 1))


def matmul_mx4(m: int, n: int, k: int, *, out=float32):
    """x (m, k) against n rows of k weights, both in microscaled 4-bit floating point.

    Buffers: the rows of x (m, k / 2) int8 and their scales (m, k / 32) int8, the
    weights (n, k / 2) and theirs (n, k / 32), y (m, n) of `out`."""
    arrays = [*_mx4_arrays(m, k), *_mx4_arrays(n, k)]

    def body(args):
        tiles = [load(a, index=(0, 0), shape=t.shape) for a, t in zip(args, arrays)]
        store(args[4], index=(0, 0), tile=tile_matmul_mx4(*tiles, dtype=out))

    args = (*arrays, Array(shape=(m, n), dtype=out))
    return convert(_named("matmul_mx4_kernel", body, len(args)), args=args, grid=(1, 1, 1))


def sample(rows: int, vocab: int, dtype=float32, *, temperature: bool = False, top_k: bool = False,
           top_p: bool = False, min_p: bool = False, trow: int | None = None):
    """One token of each row of logits; `xtile_amd.sample` states which.

    Buffers: logits (rows, vocab), uniform (rows, 1) float32, those of temperature
    (float32), top_k (int32), top_p and min_p (float32) that are asked for, (rows, 1)
    each, then the tokens (rows, 1) int32.  `trow` rows a Block (default: all)."""
    trow = rows if trow is None else trow
    if trow < 1 or rows % trow:
        raise ValueError("trow must divide rows")
    one = Array(shape=(rows, 1), dtype=float32)
    asked = {"temperature": (temperature, one), "top_k": (top_k, Array(shape=(rows, 1), dtype=int32)),
             "top_p": (top_p, one), "min_p": (min_p, one)}
    extras = {name: array for name, (wanted, array) in asked.items() if wanted}

    def body(args):
        r = bid(0)
        x = load(args[0], index=(r, 0), shape=(trow, vocab))
        u, *rest = (load(a, index=(r, 0), shape=(trow, 1)) for a in args[1:-1])
        store(args[-1], index=(r, 0), tile=tile_sample(x, u, **dict(zip(extras, rest))))

    args = (Array(shape=(rows, vocab), dtype=dtype), one, *extras.values(), Array(shape=(rows, 1), dtype=int32))
    return convert(_named("sample_kernel", body, len(args)), args=args, grid=(rows // trow, 1, 1))


def masked_attention(batch: int, kv_heads: int, group: int, nq: int, nk: int, d: int, *, dtype=bfloat16, scale=None,
                     cap=None, causal: bool = False, window=None, slopes: bool = False, start: bool = False,
                     length: bool = False, prefix: bool = False, docs: bool = False, parents: bool = False,
                     token_major: bool = False):
    """Attention of `group` query heads to each key head, one Block a key head.

    Buffers: q and the result [batch, kv_heads * group, nq, d], k and v [batch,
    kv_heads, nk, d], or, `token_major`, [batch, nq, kv_heads * group * d] and
    [batch, nk, kv_heads * d]; between v and the result, where asked for: slopes
    (kv_heads, group) float32; start, length, prefix (batch, 1) int32; the documents
    of the queries (batch, nq) and of the keys (batch, nk) int32; the parents of
    drafted tokens (batch, nq) int32, at most 64 of them.  Their meaning is `attend`'s.
    `scale` defaults to d ** -0.5."""
    if min(batch, kv_heads, group, nq, nk, d) < 1:
        raise ValueError("masked_attention sizes must be positive")
    heads = kv_heads * group
    q_shape = (batch, nq, heads * d) if token_major else (batch, heads, nq, d)
    k_shape = (batch, nk, kv_heads * d) if token_major else (batch, kv_heads, nk, d)
    per_batch = Array(shape=(batch, 1), dtype=int32)
    named = {"slopes": (slopes, Array(shape=(kv_heads, group), dtype=float32)), "start": (start, per_batch),
             "length": (length, per_batch), "prefix": (prefix, per_batch),
             "q_docs": (docs, Array(shape=(batch, nq), dtype=int32)),
             "k_docs": (docs, Array(shape=(batch, nk), dtype=int32)),
             "parents": (parents, Array(shape=(batch, nq), dtype=int32))}
    extras = {name: array for name, (wanted, array) in named.items() if wanted}
    scale = d**-0.5 if scale is None else scale

    def body(args):
        h, b = bid(0), bid(1)
        if token_major:
            q = reshape(load(args[0], index=(b, 0, h), shape=(1, nq, group * d)), shape=(nq, group * d))
            k, v = (reshape(load(a, index=(b, 0, h), shape=(1, nk, d)), shape=(nk, d)) for a in args[1:3])
        else:
            q = reshape(load(args[0], index=(b, h, 0, 0), shape=(1, group, nq, d)), shape=(group, nq, d))
            k, v = (reshape(load(a, index=(b, h, 0, 0), shape=(1, 1, nk, d)), shape=(nk, d)) for a in args[1:3])
        tiles = {}
        for (name, array), arg in zip(extras.items(), args[3:]):
            index, shape = ((h, 0), (1, group)) if name == "slopes" else ((b, 0), (1, array.shape[1]))
            tiles[name] = load(arg, index=index, shape=shape)
        o = attend(q, k, v, scale=scale, cap=cap, causal=causal, window=window, **tiles)
        if token_major:
            store(args[-1], index=(b, 0, h), tile=reshape(o, shape=(1, nq, group * d)))
        else:
            store(args[-1], index=(b, h, 0, 0), tile=reshape(o, shape=(1, group, nq, d)))

    qa, ka = Array(shape=q_shape, dtype=dtype), Array(shape=k_shape, dtype=dtype)
    args = (qa, ka, ka, *extras.values(), qa)
    return convert(_named("masked_attention_kernel", body, len(args)), args=args, grid=(kv_heads, batch, 1))


_quantize = quantize


def _mx4_arrays(rows: int, cols: int):
    """Packed rows and their scales."""
    if cols % 32:
        raise ValueError("rows in microscaled 4-bit floating point are whole blocks of 32")
    return Array(shape=(rows, cols // 2), dtype=int8), Array(shape=(rows, cols // 32), dtype=int8)


def _named(name: str, body, count: int):
    """A kernel of `count` positional arguments, for builders whose arrays depend on their options."""
    import inspect

    def fn(*args):
        body(args)

    fn.__name__ = name
    params = [inspect.Parameter(f"arg{i}", inspect.Parameter.POSITIONAL_OR_KEYWORD) for i in range(count)]
    fn.__signature__ = inspect.Signature(params)
    return kernel(fn)


CONFIGS = {
    "c1_add": lambda: add(1024, 1024, 32, 64),
    "c2_softmax": lambda: softmax(8192, 4096, 1),
    "c3_matmul_f16": lambda: matmul_f16(4096, 4096, 4096, 128, 128),
    "c4_conv2d_f16": lambda: conv2d(32, 56, 56, 64, 64, 3, 3, 4, 56),
    "c5_matmul_bf16": lambda: matmul_bf16(4096, 11008, 4096, 256, 128),
    "c6_matmul_i8": lambda: matmul_i8(4096, 4096, 4096, 64, 64),
}
