"""Calls of rms_norm, matmul_q4 and attend at the edges of what they take, against 64 bits."""

from __future__ import annotations

import math

import pytest

import xtile_amd as xt
from tests import operators_ref as ref
from xtile_amd import kernels as K

pytestmark = pytest.mark.gpu


def rand(shape, dtype, cuda, seed, scale=1.0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device=cuda)).to(dtype)


def say(*what):
    print("[gpu]", *what, flush=True)


# -- attend ------------------------------------------------------------------------


def attend_rows(q, k, v, sees, scale, slopes=None, start=0):
    """One head, row by row over the keys it sees alone, in 64 bits: (result, sum of
    the weighted magnitudes).  sees: (rows, keys)."""
    import torch

    out, size = [], []
    j = torch.arange(k.shape[0], device=k.device)
    for t in range(q.shape[0]):
        at = sees[t]
        s = (k[at].double() @ q[t].double()) * scale
        if slopes is not None:
            s = s - slopes * (start + t - j[at]).abs().double()
        p = torch.softmax(s, dim=0)
        out.append(p @ v[at].double())
        size.append(p @ v[at].double().abs())
    return torch.stack(out), torch.stack(size)


@pytest.mark.parametrize("n,docs", [(2, 1), (150, 75)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_attend_split_with_infinities_where_a_row_sees_nothing(cuda, dtype, n, docs):
    """Two documents, an infinity among the second's values.  The first's rows see nothing
    in the splits that hold it, and scores near -200 in the others."""
    import torch

    t, nk = getattr(torch, dtype), 3000
    p = K.masked_attention(1, 1, 1, n, nk, 64, dtype=getattr(xt, dtype), docs=True)
    say(xt.plan(p)["kernel"])
    assert "splits=" in xt.plan(p)["kernel"]
    q = (5 + 0.1 * rand((n, 64), torch.float32, cuda, 1)).to(t)
    k = (-5 + 0.1 * rand((nk, 64), torch.float32, cuda, 2)).to(t)
    v = rand((nk, 64), t, cuda, 3)
    qd = torch.full((1, n), 2, dtype=torch.int32, device=cuda)
    qd[0, :docs] = 1
    kd = torch.full((1, nk), 2, dtype=torch.int32, device=cuda)
    kd[0, :1500] = 1
    v[2000, 5] = math.inf
    o = torch.full_like(q, 7)
    xt.launch(p, q.view(1, 1, n, 64), k.view(1, 1, nk, 64), v.view(1, 1, nk, 64), qd, kd, o.view(1, 1, n, 64))
    want, size = attend_rows(q, k, v, qd[0][:, None] == kd[0], 0.125)
    # a score is a sum of 64 products of about 25, 200 in all: off by (64 + 16) 2^-24 of it
    far = (ref.half_step(q) + 2 * 80 * 2.0**-24 * 210 + (nk + 64) * 2.0**-24) * size + ref.half_step(q) * want.abs()
    far = far + (2.0**-25 * nk if dtype == "float16" else 0)
    ref.assert_within(o[:docs], want[:docs], far[:docs])
    ref.assert_within(o[docs:], want[docs:], far[docs:].nan_to_num(1.0, posinf=1.0))


@pytest.mark.parametrize("n", [3, 70])
def test_attend_split_with_infinities_far_from_the_rows_keys(cuda, n):
    """The same by a distance bias: what the first document's rows see lies far away."""
    import torch

    nk, start = 3000, 2900
    p = K.masked_attention(1, 1, 1, n, nk, 64, slopes=True, start=True, docs=True)
    assert "splits=" in xt.plan(p)["kernel"]
    q, k, v = (rand(s, torch.bfloat16, cuda, i) for i, s in enumerate([(n, 64), (nk, 64), (nk, 64)]))
    qd = torch.full((1, n), 2, dtype=torch.int32, device=cuda)
    qd[0, : n // 2] = 1
    kd = torch.full((1, nk), 2, dtype=torch.int32, device=cuda)
    kd[0, :1000] = 1
    v[1700, 9] = math.nan
    slopes = torch.full((1, 1), 0.25, device=cuda)
    o = torch.full_like(q, 7)
    xt.launch(p, q.view(1, 1, n, 64), k.view(1, 1, nk, 64), v.view(1, 1, nk, 64), slopes,
              torch.tensor([[start]], dtype=torch.int32, device=cuda), qd, kd, o.view(1, 1, n, 64))
    want, size = attend_rows(q, k, v, qd[0][:, None] == kd[0], 0.125, 0.25, start)
    # biases to 750, in which a score is off by 8 2^-24 of them, products by 80 2^-24 of some 10
    far = (2.0**-8 + 2 * (8 * 750 + 80 * 10) * 2.0**-24 + (nk + 64) * 2.0**-24) * size + 2.0**-8 * want.abs()
    ref.assert_within(o[: n // 2], want[: n // 2], far[: n // 2])
    assert bool(torch.isnan(o[n // 2 :, 9]).all()) and bool(torch.isfinite(o[n // 2 :, 10]).all())


def capped(cuda, n, nk, d, cap, dtype, spread=1.0, seed=1, edit=None, length=None):
    """(result, what it should be, how far it may be off)"""
    import torch

    t, scale = getattr(torch, dtype), d**-0.5
    p = K.masked_attention(1, 1, 1, n, nk, d, dtype=getattr(xt, dtype), cap=cap, causal=False, length=length is not None)
    say(xt.plan(p)["kernel"], cap)
    q, k, v = (rand((s, d), t, cuda, seed + i, c) for i, (s, c) in enumerate([(n, spread), (nk, spread), (nk, 1.0)]))
    if edit:
        edit(q, k, v)
    o = torch.full_like(q, 7)
    le = [] if length is None else [torch.tensor([[length]], dtype=torch.int32, device=cuda)]
    xt.launch(p, q.view(1, 1, n, d), k.view(1, 1, nk, d), v.view(1, 1, nk, d), *le, o.view(1, 1, n, d))
    k, v = k[:length], v[:length]
    qd, kd, vd = q.double(), k.double(), v.double()
    s = qd @ kd.t() * scale
    # the product's sum, then: up to cap / 2 a polynomial off by 6.2e-7 of the score, beyond
    # it cap (1 - 2 / (e^2z + 1)), whose exponent, exponential, sum and reciprocal leave at
    # most 16 2^-24 of its own size; two products by constants more.  Caps to 256 take the
    # latter for all of a tile: 8 2^-24 of the cap
    off = (d + 8) * 2.0**-24 * (qd.abs() @ kd.abs().t() * scale) + 24 * 2.0**-24 * s.abs()
    off = off + (8 * 2.0**-24 * cap if cap <= 256 else 0)
    x = cap * torch.tanh(s / cap)
    off = torch.minimum(off, torch.full_like(off, 2 * cap))
    w = torch.softmax(x, dim=1)
    want, size = w @ vd, w @ vd.abs()
    u = ref.half_step(q)
    far = (u + 2 * off.amax(dim=1, keepdim=True) + (nk + 64) * 2.0**-24) * size + u * want.abs()
    if dtype == "float16":
        far = far + 2.0**-25 * vd.abs().sum(0) + 2.0**-25
    return o, want, far


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("n,nk,d", [(1, 300, 128), (90, 300, 128), (90, 150, 128), (40, 300, 256), (3, 90, 32)])
@pytest.mark.parametrize("cap", [260.0, 884.0, 1e4, 1e5, 1e6, 1e9, 1e30, 3e38])
def test_attend_large_caps(cuda, cap, n, nk, d, dtype):
    """Towards no cap at all."""
    o, want, far = capped(cuda, n, nk, d, cap, dtype, 1.5)
    ref.assert_within(o, want, far)


@pytest.mark.parametrize("n", [1, 90])
@pytest.mark.parametrize("cap", [1e-38, 1e-30, 1e-6, 1e-3, 0.05])
def test_attend_small_caps(cuda, cap, n):
    """Towards equal scores."""
    o, want, far = capped(cuda, n, 300, 64, cap, "bfloat16")
    ref.assert_within(o, want, far)


@pytest.mark.parametrize("n", [1, 90])
@pytest.mark.parametrize("cap", [0.5, 5.0, 50.0, 257.0, 1e4])
def test_attend_caps_of_scores_small_and_large(cuda, cap, n):
    """Scores on both sides of half the cap in one tile, then also keys that are not
    finite where no row sees them."""
    import torch

    def edit(q, k, v):
        k[::3] *= 30
        k[1::3] *= 0.05

    o, want, far = capped(cuda, n, 300, 64, cap, "bfloat16", edit=edit)
    ref.assert_within(o, want, far)

    def odd(q, k, v):
        edit(q, k, v)
        k[251:] = math.nan
        v[251:] = math.inf

    o2, want, far = capped(cuda, n, 300, 64, cap, "bfloat16", edit=odd, length=251)
    ref.assert_within(o2, want, far)


@pytest.mark.parametrize("nk,split", [(131072, True), (3000, False)])
def test_attend_float16_weights_far_below_the_largest(cuda, nk, split):
    """One key holds nearly all of the weight, the others some 2^-25.5 each."""
    import torch

    d = 64
    p = K.masked_attention(1, 1, 1, 1, nk, d, dtype=xt.float16)
    q, k = torch.zeros(1, 1, 1, d, device=cuda).half(), torch.zeros(1, 1, nk, d, device=cuda).half()
    v = torch.ones(1, 1, nk, d, device=cuda).half()
    q[0, 0, 0, 0], k[0, 0, 7, 0] = 1.0, 25.5 * math.log(2) * 8  # the scale is 1 / 8
    v[0, 0, 7] = 0
    k[0, 0, 100:200, 0], v[0, 0, 100:200, 3] = 30.0, -2.0
    o = torch.zeros_like(q)
    bufs = [t.data_ptr() for t in (q, k, v, o)], [2 * t.numel() for t in (q, k, v, o)]
    if split:
        xt.launch(p, q, k, v, o)
    else:
        xt._native.launch(p, None, *bufs, torch.cuda.current_stream().cuda_stream)
    w = torch.softmax(k[0, 0].double() @ q[0, 0, 0].double() / 8, 0)
    want = w @ v[0, 0].double()
    # a weight of the largest's 2^-25.5 is held as one of 2^-18.5: steps of 2^-24
    far = (2.0**-11 + 200 * 2.0**-24) * (w @ v[0, 0].double().abs()) + nk * 2.0**-32 * 1.0 + 2.0**-11 * want.abs() + 2.0**-25
    say(float(want[0]), float(o[0, 0, 0, 0]))
    assert float(far.max()) < 0.08 * float(want.max())
    ref.assert_within(o[0, 0, 0], want, far)


@pytest.mark.parametrize("n", [1, 40, 64])
def test_attend_infinite_values_of_small_weight(cuda, n):
    """A weight that the values' type does not hold is not zero: its infinity counts."""
    import torch

    q, k, v = (torch.zeros(1, 1, s, 64, device=cuda).half() for s in (n, 64, 64))
    q[..., 0] = 1
    k[0, 0, 3, 0] = 40 * math.log(2) * 8
    v[0, 0, 50, 6], v[0, 0, 51, 7] = math.inf, -math.inf
    p = K.masked_attention(1, 1, 1, n, 64, 64, dtype=xt.float16)
    o = torch.zeros_like(q)
    xt.launch(p, q, k, v, o)
    assert bool((o[..., 6] == math.inf).all()) and bool((o[..., 7] == -math.inf).all())
    assert bool((o[..., :6] == 0).all()) and bool((o[..., 8:] == 0).all())


@pytest.mark.parametrize("n", [1, 64])
def test_attend_values_near_the_largest(cuda, n):
    """The sums hold them: weights above one, between two rescalings, do not overflow."""
    import torch

    q, k, v = (torch.zeros(1, 1, s, 64, device=cuda).bfloat16() for s in (n, 1024, 1024))
    q[..., 0] = 1
    k[0, 0, 1000, 0] = 38.0  # a score of 4.75: 2^6.85 times the others' weight
    v[0, 0, 1000, 2], v[0, 0, :, 4] = 3e38, 1.0
    p = K.masked_attention(1, 1, 1, n, 1024, 64)
    o = torch.zeros_like(q)
    xt.launch(p, q, k, v, o)
    w = math.exp(38.0 / 8) / (math.exp(38.0 / 8) + 1023)
    want = w * float(v[0, 0, 1000, 2])
    assert bool(((o[..., 2].double() - want).abs() <= want * (2 * 2.0**-8 + 1200 * 2.0**-24)).all())
    assert bool((o[..., 4] == 1).all())


@pytest.mark.parametrize("n,nk", [(1, 100), (3, 100), (70, 100), (2, 2000)])
@pytest.mark.parametrize("start,window", [(2**31 - 1, 2**31 - 1), (2**31 - 50, 2**31 - 30), (2**30, 2**30 - 20),
                                          (2**30 - 1, 2**30 + 50), (2**31 - 1, 5), (2**30 - 60, 2**30), (-(2**31), 7),
                                          (-(2**30) - 5, 2**31 - 1), (97, 2**31 - 1)])
@pytest.mark.parametrize("causal", [False, True])
def test_attend_windows_at_far_positions(cuda, causal, start, window, n, nk):
    """Positions of 31 bits and windows as large, of which a row sees none, some or all keys."""
    import torch

    p = K.masked_attention(1, 1, 1, n, nk, 64, causal=causal, window=window, start=True)
    q, k, v = (rand((1, 1, s, 64), torch.bfloat16, cuda, i) for i, s in enumerate((n, nk, nk)))
    st = torch.tensor([[start]], dtype=torch.int32, device=cuda)
    o = torch.full_like(q, 7)
    xt.launch(p, q, k, v, st, o)
    want, far = ref.attend(q, k, v, 0.125, causal=causal, window=window, start=st)
    ref.assert_within(o, want, far)


# -- matmul_q4 -----------------------------------------------------------------------


@pytest.mark.parametrize("what", ["weights", "scales"])
def test_matmul_q4_of_rows_whose_pitch_passes_a_tiles_31_bits(cuda, what):
    """32 rows of weights, or of their scales, 2 GiB apart from the first to the last."""
    import torch

    m, n, k = 12288, 32, 64
    wp, sp = (70_000_000, 2) if what == "weights" else (32, 36_000_000)
    p16 = xt.float16

    @xt.kernel
    def part(x, w, s, y):
        t = xt.matmul_q4(xt.load(x, index=(0, 0), shape=(m, k)), xt.load(w, index=(0, 0), shape=(n, k // 2)),
                         xt.load(s, index=(0, 0), shape=(n, 2)))
        xt.store(y, index=(0, 0), tile=t)

    p = xt.convert(part, args=(xt.Array((m, k), p16), xt.Array((n, wp), xt.int8), xt.Array((n, sp), p16),
                               xt.Array((m, n), xt.float32)), grid=(1, 1, 1))
    say(xt.plan(p)["kernel"])
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randint(-3, 4, (m, k), generator=g, device=cuda).half()
    w = torch.randint(-8, 8, (n, k), generator=g, device=cuda, dtype=torch.int8)
    s = torch.exp2(-torch.randint(0, 5, (n, 2), generator=g, device=cuda).float()).half()
    bw = torch.zeros(n, wp, dtype=torch.int8, device=cuda)
    bs = torch.zeros(n, sp, dtype=torch.float16, device=cuda)
    bw[:, : k // 2], bs[:, :2] = xt.pack_q4(w), s
    y = torch.full((m, n), 7.0, device=cuda)
    xt.launch(p, x, bw, bs, y)
    assert torch.equal(y.double(), ref.matmul_q4(x, w, s))


# -- rms_norm ------------------------------------------------------------------------


@pytest.mark.parametrize("cols", [1, 4, 7])
def test_rms_norm_of_many_short_rows(cuda, cols):
    """More than 2^22 rows of fewer than eight values."""
    import torch

    rows = (1 << 22) + 37
    m = K.rms_norm(rows, cols, xt.float32, residual=False)
    say(xt.plan(m)["kernel"])
    x, g = rand((rows, cols), torch.float32, cuda, 1), rand((1, cols), torch.float32, cuda, 2)
    y = torch.full_like(x, 7)
    xt.launch(m, x, g, y)
    _, want = ref.rms_norm(x, None, g, 1e-6)
    ref.assert_within(y, want, want.abs() * 40 * 2.0**-24 + 1e-37)


@pytest.mark.parametrize("over", ["x", "r"])
def test_rms_norm_scales_of_one_column_over_an_input(cuda, over):
    """Rows of one value, whose scales have the input's shape and type."""
    import torch

    m = K.rms_norm(37, 1, xt.float32, quantize=True)
    x, r, g = rand((37, 1), torch.float32, cuda, 1), rand((37, 1), torch.float32, cuda, 2), torch.full((1, 1), 3.0, device=cuda)
    want_h, want = ref.rms_norm(x, r, g, 1e-6)
    h, q, s = torch.zeros_like(x), torch.zeros(37, 1, dtype=torch.int8, device=cuda), {"x": x, "r": r}[over]
    xt.launch(m, x, r, g, h, q, s)
    assert torch.equal(h, want_h.float()) and torch.equal(q, 127 * torch.sign(want_h).to(torch.int8))
    ref.assert_within(s, want.abs() / 127, want.abs() / 127 * 40 * 2.0**-24)


@pytest.mark.parametrize("rows,cols", [(4096, 4096), (2, 100000)])
def test_rms_norm_rows_in_8_bits_are_quotients_to_the_nearest(cuda, rows, cols):
    """Of the values and the scale in 32 bits, as float32 division rounds them."""
    import torch

    x, g = rand((rows, cols), torch.float32, cuda, 1), rand((1, cols), torch.float32, cuda, 2)
    y, s = torch.zeros_like(x), torch.zeros(rows, 1, device=cuda)
    q = torch.zeros(rows, cols, dtype=torch.int8, device=cuda)
    xt.launch(K.rms_norm(rows, cols, xt.float32, residual=False), x, g, y)
    xt.launch(K.rms_norm(rows, cols, xt.float32, residual=False, quantize=True), x, g, q, s)
    want = torch.round(y / s).clamp(-127, 127)
    assert int((q.float() != want).sum()) == 0


@pytest.mark.parametrize("cols", [5, 64, 2000, 40000])
def test_rms_norm_rows_in_8_bits_of_products_below_the_normal_numbers(cuda, cols):
    """Values and gamma so small that the largest of their products has a bit or two: the
    integers keep their sign and stay within 127."""
    import torch

    x, g = 1e-19 * rand((9, cols), torch.float32, cuda, 1), torch.full((1, cols), 1.5e-26, device=cuda)
    q, s = torch.full((9, cols), 99, dtype=torch.int8, device=cuda), torch.zeros(9, 1, device=cuda)
    xt.launch(K.rms_norm(9, cols, xt.float32, residual=False, quantize=True, eps=1e-38), x, g, q, s)
    assert int(q.min()) >= -127 and bool((q.float() * x >= 0).all())
    _, want = ref.rms_norm(x, None, g, 1e-38)
    # the squares, too, are near the smallest normal number: 2^-8 of a quotient at most
    assert bool(((q.double() - (want / s.double()).clamp(-127, 127)).abs() <= 0.5 + 2.0**-1).all())


# -- launches ------------------------------------------------------------------------


def test_a_launch_looks_its_program_up_once(cuda):
    """One call into the library, which asks for a workspace only where the program has one."""
    import ctypes

    import torch

    xt.launch(K.add(64, 64), *(torch.zeros(64, 64, device=cuda) for _ in range(3)))  # the native call is loaded
    module, lib = xt._launch_native.__self__, xt._native.lib
    alloc_t = ctypes.CFUNCTYPE(ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t)
    run_t = ctypes.CFUNCTYPE(ctypes.c_int, *([ctypes.c_void_p, ctypes.c_char_p, ctypes.c_void_p, ctypes.c_int]
                                             + [ctypes.c_void_p] * 4))
    own = ctypes.cast(lib.xt_gpu_run_buffers_alloc, ctypes.c_void_p).value
    calls, asked = [], []

    def run(m, func, bufs, n, alloc, context, stream, err):
        @alloc_t
        def counted(c, size):
            asked.append(size)
            return alloc_t(alloc)(c, size)

        calls.append(func)
        return run_t(own)(m, func, bufs, n, ctypes.cast(counted, ctypes.c_void_p), context, stream, err)

    counting, release = run_t(run), ctypes.cast(lib.xt_free, ctypes.c_void_p).value
    module.bind(ctypes.cast(counting, ctypes.c_void_p).value, release, xt._native.NativeModule)
    try:
        a, c = torch.ones(64, 64, device=cuda), torch.zeros(64, 64, device=cuda)
        xt.launch(K.add(64, 64), a, a, c)
        assert len(calls) == 1 and not asked and bool((c == 2).all())
        p = K.masked_attention(1, 2, 4, 1, 5000, 64)
        q, k, v = (rand(s, torch.bfloat16, cuda, i) for i, s in enumerate([(1, 8, 1, 64), (1, 2, 5000, 64), (1, 2, 5000, 64)]))
        o = torch.zeros_like(q)
        xt.launch(p, q, k, v, o)
        assert len(calls) == 2 and asked == [xt.workspace(p)]
    finally:
        module.bind(own, release, xt._native.NativeModule)
    o2 = torch.zeros_like(q)
    xt.launch(p, q, k, v, o2)
    assert torch.equal(o, o2) and len(calls) == 2
