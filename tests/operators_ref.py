"""The operators of a language model's layer in 64 bits, and how far their kernels may be off."""

from __future__ import annotations

import math

HALF = {"float32": 2.0**-24, "float16": 2.0**-11, "bfloat16": 2.0**-8}  # half a step, relative


def half_step(t) -> float:
    return HALF[str(t.dtype).replace("torch.", "")]


def rms_norm(x, r, gamma, eps):
    """(h, y) in 64 bits."""
    h = x.double() if r is None else x.double() + r.double()
    return h, h / (h.square().mean(dim=1, keepdim=True) + eps).sqrt() * gamma.double()


def matmul_q4(x, w, scales, row_scale=None):
    """w: the unpacked weights (N, K)."""
    group = w.shape[1] // scales.shape[1]
    y = x.double() @ (w.double() * scales.double().repeat_interleave(group, dim=1)).t()
    return y if row_scale is None else y * row_scale.double()


def visible(b, nq, nk, device, causal=False, window=None, start=None, length=None, prefix=None, q_docs=None,
            k_docs=None):
    """(batch, nq, nk) truth values."""
    import torch

    def per_batch(t):
        return t.long().view(b, 1, 1)

    j = torch.arange(nk, device=device).view(1, 1, nk)
    p = torch.arange(nq, device=device).view(1, nq, 1).expand(b, nq, 1)
    if start is not None:
        p = p + per_batch(start)
    band = torch.ones(b, nq, nk, dtype=torch.bool, device=device)
    if causal:
        band &= j <= p
    if window is not None:
        band &= p - j < window
    if prefix is not None:
        band |= j < per_batch(prefix)
    if length is not None:
        band &= j < per_batch(length)
    if q_docs is not None:
        band &= q_docs.view(b, nq, 1) == k_docs.view(b, 1, nk)
    return band, (p - j).abs()


def attend(q, k, v, scale, cap=None, slopes=None, **masks):
    """q [b, hk * g, nq, d], k and v [b, hk, nk, d]; (result, how far a kernel may be off it).

    A weight is rounded to the inputs' type (half a step u of itself; float16
    weights below its normal range by 2^-25), the result by another u.  A score is
    a float32 sum of D products, off by (D + 8) 2^-24 of the products' magnitudes,
    plus 8 2^-24 of the cap or the bias; e^score is off by that much relatively, as
    are the total and the sum (n + 64 roundings more)."""
    import torch

    b, h, nq, d = q.shape
    hk, nk = k.shape[1:3]
    g = h // hk
    sees, distance = visible(b, nq, nk, q.device, **masks)
    sees, distance = sees[:, None], distance[:, None].double()
    kk, vv = (t.double().repeat_interleave(g, dim=1) for t in (k, v))
    hidden = ~sees.any(dim=2, keepdim=True).transpose(2, 3)  # keys that no row sees: whatever they hold
    kk, vv = kk.masked_fill(hidden, 0.0), vv.masked_fill(hidden, 0.0)
    qd = q.double()
    s = (qd @ kk.transpose(2, 3)) * scale
    size = ((qd.abs() @ kk.abs().transpose(2, 3)) * scale).masked_fill(~sees, 0).nan_to_num(0, 0, 0)
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
    y = p.masked_fill(~sees, 0.0) @ vv
    u = half_step(q)
    size = p @ vv.abs()
    far = (u + 2 * off.amax(dim=3, keepdim=True) + (nk + 64) * 2.0**-24) * size + u * y.abs()
    if q.dtype == torch.float16:
        far = far + 2.0**-25 * (sees.double() @ vv.abs()) + 2.0**-25
    return y, far * (1 + 2.0**-10) + 1e-30


def assert_within(got, want, far, what=""):
    import torch

    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN at other places"
    odd = ~fine & ~torch.isnan(want)
    assert torch.equal(got[odd], want[odd]), f"{what}: infinities differ"
    worst = ((got - want).abs() / far)[fine]
    assert worst.numel() == 0 or float(worst.max()) <= 1, f"{what}: {float(worst.max()):.3g} times what it may be off"
