"""Microscaled 4-bit rows, products of them, drafted trees and sampling in 64 bits, on the CPU."""

from __future__ import annotations

import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize_mx4(x):
    """(codes [R, C] uint8, bytes [R, C / 32] uint8) of a float64 array [R, C]."""
    rows, cols = x.shape
    b = x.reshape(rows, cols // 32, 32)
    odd = ~np.isfinite(b).all(axis=2)
    b = np.where(odd[:, :, None], 0.0, b)
    top = np.abs(b).max(axis=2)
    exponent = np.frexp(top)[1] - 1 - 2  # top = m 2**e, 1/2 <= m < 1
    byte = np.where(top > 0, np.maximum(exponent, -127) + 127, 0)
    y = np.ldexp(b, (127 - byte)[:, :, None])
    size = np.abs(y)
    code = np.zeros(size.shape, dtype=np.uint8)
    for i in range(1, 8):  # nearest; halfway to the even code
        half = (E2M1[i - 1] + E2M1[i]) / 2
        code = np.where(size > half if i % 2 else size >= half, i, code)
    code = (code | (np.signbit(y).astype(np.uint8) << 3)).astype(np.uint8)
    code = np.where(odd[:, :, None], 0, code)
    return code.reshape(rows, cols).astype(np.uint8), np.where(odd, 255, byte).astype(np.uint8)


def pack(code):
    return (code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8)


def unpack(packed):
    out = np.empty((packed.shape[0], 2 * packed.shape[1]), dtype=np.uint8)
    out[:, 0::2], out[:, 1::2] = packed & 15, packed >> 4
    return out


def values(code, byte):
    """What codes and their bytes stand for."""
    v = np.where(code > 7, -E2M1[code & 7], E2M1[code & 7])
    scale = np.where(byte == 255, np.nan, np.ldexp(1.0, byte.astype(np.int64) - 127))
    return v * np.repeat(scale, 32, axis=1)


def matmul_mx4(x, w):
    """(y, how far a kernel may be off it) of the float64 values x [M, K] and w [N, K].

    A block's 32 products are multiples of 1/4 below 2**13 of them, exact in 32 bits; the
    K / 32 blocks and eight parts meet in sums in 32 bits, each off by at most 2**-23 of
    the magnitudes' sum (truncated or rounded), and what is below the normal numbers may
    be lost."""
    y = x @ w.T
    size = np.abs(x) @ np.abs(w).T
    return y, (x.shape[1] // 32 + 8) * 2.0**-23 * size + 2.0**-126 * (x.shape[1] // 32 + 8)


def sample(x, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """The token of one row: x float64 [V], the rest numbers (None: absent)."""
    x = np.where(np.isnan(x), -np.inf, x) + 0.0
    top = x.max()
    if top == -np.inf:
        return -1
    t = 1.0 if temperature is None else float(temperature)
    order = np.argsort(-x, kind="stable")
    z = x[order]
    if t > 0 and top != np.inf:
        with np.errstate(invalid="ignore"):
            w = np.where(z == top, 1.0, np.where(z == -np.inf, 0.0, np.exp((z - top) / t)))
    else:
        w = (z == top).astype(np.float64)
    n = len(z)
    if top_k is not None and 0 < top_k < n:
        n = int(top_k)
    if top_p is not None and top_p < 1:
        before = np.concatenate(([0.0], np.cumsum(w[:n])[:-1]))
        n = max(1, int((before < float(top_p) * w[:n].sum()).sum()))
    if min_p is not None and min_p > 0:
        n = min(n, int((w >= min(float(min_p), 1.0)).sum()))
    cdf = np.cumsum(w[:n])
    u = float(u) if u > 0 else 0.0
    at = int((cdf <= u * cdf[-1]).sum()) if u < 1 else n
    if at >= n:  # the last one with a weight
        at = int(np.nonzero(w[:n])[0][-1])
    return int(order[at])


def ancestors(parents):
    """[nq, nq]: whether drafted token u is t's ancestor or t itself, up the tree one by one."""
    n = len(parents)
    out = np.zeros((n, n), dtype=bool)
    for t in range(n):
        up = t
        while True:
            out[t, up] = True
            if not 0 <= parents[up] < up:
                break
            up = parents[up]
    return out


def tree_seen(parents, start, length, nk, window=None):
    """([nq, nk] what each drafted token sees, [nq, nk] how far each key is)."""
    reach = ancestors(parents)
    depth = reach.sum(axis=1) - 1
    j = np.arange(nk, dtype=np.int64)
    u = j - start
    drafted = (u >= 0) & (u < len(parents))
    at = np.clip(u, 0, len(parents) - 1)
    position = np.where(drafted, start + depth[at], j)
    away = (start + depth)[:, None] - position[None, :]
    seen = np.where(drafted[None, :], reach[:, at], (u < 0)[None, :]) & (j < length)[None, :]
    if window is not None:
        seen &= away < window
    return seen, np.abs(away)


def attend_seen(q, k, v, scale, sees, distance, cap=None, slopes=None):
    """q [b, hk * g, nq, d], k and v [b, hk, nk, d], sees and distance [b, nq, nk] tensors;
    (result, how far a kernel may be off it), as operators_ref.attend has it."""
    import math

    import torch

    from .operators_ref import half_step

    b, h, nq, d = q.shape
    hk, nk = k.shape[1:3]
    g = h // hk
    sees, distance = sees[:, None], distance[:, None].double()
    kk, vv = (t.double().repeat_interleave(g, dim=1) for t in (k, v))
    hidden = ~sees.any(dim=2, keepdim=True).transpose(2, 3)
    kk, vv = kk.masked_fill(hidden, 0.0), vv.masked_fill(hidden, 0.0)
    qd = q.double()
    s = (qd @ kk.transpose(2, 3).contiguous()) * scale
    size = ((qd.abs() @ kk.abs().transpose(2, 3).contiguous()) * scale).masked_fill(~sees, 0)
    off = (d + 8) * 2.0**-24 * size
    if cap is not None:
        s = cap * torch.tanh(s / cap)
        off = off + 8 * 2.0**-24 * cap
    if slopes is not None:
        bias = slopes.double().reshape(1, h, 1, 1) * distance
        s = s - bias
        off = off + 8 * 2.0**-24 * bias.masked_fill(~sees, 0)
    s = s.masked_fill(~sees, -math.inf)
    off = off + 8 * 2.0**-24 * s.abs().masked_fill(~sees, 0).nan_to_num(0, 0, 0)
    top = s.amax(dim=3, keepdim=True)
    p = (s - top.masked_fill(top == -math.inf, 0.0)).exp()
    total = p.sum(dim=3, keepdim=True)
    p = torch.where(total == 0, torch.zeros_like(p), p / total)
    # NaN among the values is NaN in the rows that see it, and nothing in others (0 NaN is NaN)
    bad = torch.isnan(vv)
    vv = vv.masked_fill(bad, 0.0)
    y = p.masked_fill(~sees, 0.0) @ vv
    y = y.masked_fill(sees.double().expand(b, h, nq, nk) @ bad.double() > 0, math.nan)
    u = half_step(q)
    size = p @ vv.abs()
    far = (u + 2 * off.amax(dim=3, keepdim=True) + (nk + 64) * 2.0**-24) * size + u * y.abs()
    if q.dtype == torch.float16:
        far = far + 2.0**-25 * (sees.double() @ vv.abs()) + 2.0**-25
    return y, far * (1 + 2.0**-10) + 1e-30
