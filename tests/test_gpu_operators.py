"""rms_norm, matmul_q4 and attend programs on the GPU against 64 bits."""

from __future__ import annotations

import math

import pytest

import xtile_amd as xt
from tests import operators_ref as ref
from xtile_amd import kernels as K

pytestmark = pytest.mark.gpu

DSL = {"f32": xt.float32, "f16": xt.float16, "bf16": xt.bfloat16, "i8": xt.int8}


def torch_dtype(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}[name]


def rand(shape, name, cuda, seed, scale=1.0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device=cuda)).to(torch_dtype(name))


def say(*what):
    print("[gpu]", *what, flush=True)


# -- rms_norm ------------------------------------------------------------------


def norm_case(cuda, rows, cols, dtype, residual, quantize, trow=1, gamma=None, seed=1, edit=None, over=None):
    """Launches one and checks every result; over: which input the sum is stored over."""
    import torch

    m = K.rms_norm(rows, cols, DSL[dtype], residual=residual, quantize=quantize, trow=trow,
                   gamma=DSL[gamma] if gamma else None)
    say("rms_norm", xt.plan(m)["kernel"])
    x = rand((rows, cols), dtype, cuda, seed)
    r = rand((rows, cols), dtype, cuda, seed + 1, 3.0) if residual else None
    g = rand((1, cols), gamma or dtype, cuda, seed + 2)
    if edit:
        edit(x, r, g)
    want_h, want = ref.rms_norm(x, r, g, 1e-6)
    h = {"x": x, "r": r}[over] if over else torch.full_like(x, 7)
    y = torch.full_like(x, 7)
    q, s = torch.full((rows, cols), 99, dtype=torch.int8, device=cuda), torch.full((rows, 1), 7.0, device=cuda)
    xt.launch(m, *([x, r] if residual else [x]), g, *([h] if residual else []), *([q, s] if quantize else [y]))
    torch.cuda.synchronize()
    u = ref.half_step(x)
    if residual:  # the sum in 32 bits, then to the type
        ref.assert_within(h, want_h, want_h.abs() * (u + 2.0**-24) * (1 + 2.0**-7) + 1e-37, "sum")
    # h one rounding, the sum of squares a tree of at most 8 + 8 + 6 + 16 additions
    # of which the root halves the error, the root, the division and two products
    f32 = 40 * 2.0**-24
    if not quantize:
        far = want.abs() * (u + f32) + (2.0**-25 if dtype == "f16" else 1e-37)
        ref.assert_within(y, want, far, "y")
        return y
    want_s = want.abs().amax(dim=1, keepdim=True) / 127
    ref.assert_within(s, want_s, want_s.abs() * f32 + 1e-44, "scale")
    nan = torch.isnan(want_s) | torch.isinf(want_s)
    off = (q.double() * want_s - want).abs() / want_s.clamp(min=1e-300)
    off = off.masked_fill(nan | (want_s == 0), 0.0)
    assert float(off.max()) <= 0.5 + 127 * 2 * f32, float(off.max())
    assert bool((q[(want_s == 0).expand_as(q)] == 0).all())
    assert int(q.min()) >= -127
    return q


@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 7), (5, 64), (37, 1000), (2, 1025), (130, 2049), (3, 8192),
                                       (2, 8193), (2, 32768), (3, 40001)])
def test_rms_norm(cuda, rows, cols, dtype, residual, quantize):
    norm_case(cuda, rows, cols, dtype, residual, quantize)


def test_rms_norm_blocks_of_rows_and_another_gamma(cuda):
    norm_case(cuda, 24, 520, "bf16", True, True, trow=6, gamma="f32")
    norm_case(cuda, 24, 3000, "f16", False, False, trow=4, gamma="bf16")


@pytest.mark.parametrize("over", ["x", "r"])
@pytest.mark.parametrize("cols", [100, 5000, 50000])
def test_rms_norm_stores_the_sum_over_an_input(cuda, cols, over):
    norm_case(cuda, 9, cols, "bf16", True, False, over=over)
    norm_case(cuda, 9, cols, "f32", True, True, over=over)


@pytest.mark.parametrize("cols", [100, 5000, 50000])
def test_rms_norm_rows_of_zeros_tiny_and_not_finite(cuda, cols):
    def edit(x, r, g):
        x[0] = 0
        x[1] = 1e-30
        x[2, 5] = math.inf
        x[3, 6] = math.nan
        x[4] = 3e-39

    norm_case(cuda, 6, cols, "f32", False, False, edit=edit)
    norm_case(cuda, 6, cols, "f32", False, True, edit=edit)


def test_rms_norm_unaligned(cuda):
    import torch

    m = K.rms_norm(5, 333, xt.bfloat16, residual=False)
    buf = rand((5 * 333 + 1,), "bf16", cuda, 3)
    x, g = buf[1:].view(5, 333), rand((1, 333), "bf16", cuda, 4)
    y = torch.zeros(5 * 333 + 3, dtype=torch.bfloat16, device=cuda)
    xt.launch(m, x, g, y[1:-2].view(5, 333))
    _, want = ref.rms_norm(x, None, g, 1e-6)
    ref.assert_within(y[1:-2].view(5, 333), want, want.abs() * (2.0**-8 + 40 * 2.0**-24) + 1e-37)
    assert y[0] == 0 and bool((y[-2:] == 0).all())


@pytest.mark.parametrize("over", [None, "x", "r"])
@pytest.mark.parametrize("cols", [8, 9, 15, 511, 513, 1023, 2047, 4099, 8191, 9001])
def test_rms_norm_rows_that_eight_does_not_divide(cuda, cols, over):
    """A row's last vector begins inside its neighbour: it counts once, also in place."""
    norm_case(cuda, 7, cols, "bf16", True, over == "x", over=over)
    norm_case(cuda, 7, cols, "f32", True, over != "x", over=over, gamma="f16")


def test_rms_norm_refuses_results_over_what_it_reads_elsewhere(cuda):
    import torch

    m = K.rms_norm(4, 64, xt.float32)
    buf = torch.zeros(8 * 64 + 64, device=cuda)
    x, shifted, g = buf[: 4 * 64].view(4, 64), buf[64 : 5 * 64].view(4, 64), torch.ones(1, 64, device=cuda)
    y = torch.zeros(4, 64, device=cuda)
    with pytest.raises(ValueError, match="meets buffer"):
        xt.launch(m, x, y, g, torch.zeros_like(x), shifted)
    with pytest.raises(ValueError, match="both stored"):
        xt.launch(m, x, torch.zeros_like(x), g, y, y)


# -- matmul_q4 -------------------------------------------------------------------


def q4_inputs(cuda, m, n, k, group, dtype, scales, seed=1, exact=False):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randint(-8, 8, (n, k), generator=g, device=cuda, dtype=torch.int8)
    if exact:  # every product and sum a whole number of 2^-6 below 2^24 of them
        s = torch.exp2(-torch.randint(0, 7, (n, k // group), generator=g, device=cuda).float())
        x = torch.randint(-3, 4, (m, k), generator=g, device=cuda)
    else:
        s = 0.001 + 0.01 * torch.rand(n, k // group, generator=g, device=cuda)
        x = torch.randint(-127, 128, (m, k), generator=g, device=cuda) if dtype == "i8" else torch.randn(
            m, k, generator=g, device=cuda)
    rs = 0.01 + torch.rand(m, 1, generator=g, device=cuda)
    return x.to(torch_dtype(dtype)), w, s.to(torch_dtype(scales)), rs


Q4_SIZES = [(1, 1, 32, 32), (1, 64, 4096, 128), (3, 70, 96, 32), (16, 33, 1056, 32), (17, 129, 320, 64), (33, 16, 192, 192),
            (64, 48, 512, 256), (70, 100, 480, 96), (2, 31, 1280, 640), (130, 17, 2048, 128), (1, 40, 160, 160)]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("m,n,k,group", Q4_SIZES)
def test_matmul_q4_exact(cuda, m, n, k, group, dtype):
    """Whole numbers: every rounding is exact, so the result is."""
    import torch

    p = K.matmul_q4(m, n, k, group=group, dtype=DSL[dtype], scales=xt.float32)
    say(xt.plan(p)["kernel"])
    x, w, s, _ = q4_inputs(cuda, m, n, k, group, dtype, "f32", exact=True)
    y = torch.full((m, n), 7.0, device=cuda)
    xt.launch(p, x, xt.pack_q4(w), s, y)
    assert torch.equal(y.double(), ref.matmul_q4(x, w, s))


@pytest.mark.parametrize("scales", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dtype,out", [("f16", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("i8", "f32"), ("i8", "bf16")])
@pytest.mark.parametrize("m,n,k,group", [(1, 300, 4096, 128), (16, 100, 1056, 32), (50, 65, 704, 64)])
def test_matmul_q4(cuda, m, n, k, group, dtype, out, scales):
    """In 32 bits a chunk of 128 sums values of at most 31 and 24 times |x|, at most
    136 roundings of 2^-24 each; the chunks and the waves add k / 128 + 16."""
    import torch

    p = K.matmul_q4(m, n, k, group=group, dtype=DSL[dtype], scales=DSL[scales], out=DSL[out], row_scale=dtype == "i8")
    x, w, s, rs = q4_inputs(cuda, m, n, k, group, dtype, scales)
    y = torch.full((m, n), 7.0, device=cuda, dtype=torch_dtype(out))
    xt.launch(p, x, xt.pack_q4(w), s, *([rs] if dtype == "i8" else []), y)
    want = ref.matmul_q4(x, w, s, rs if dtype == "i8" else None)
    size = ref.matmul_q4(x.double().abs(), torch.ones_like(w), s, rs if dtype == "i8" else None)
    # integers are exact within a chunk
    chunk = 0 if dtype == "i8" else 136 * (31 + 24)
    far = 2.0**-24 * (chunk + 8 * (k / 128 + 20)) * size + ref.half_step(y) * want.abs() + 2.0**-25
    ref.assert_within(y, want, far)
    # the roundings of a sum do not all go one way: by their root mean square
    err = float((y.double() - want).norm() / want.norm())
    assert err <= ref.half_step(y) + 4e-6, err


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("m,n,k,group", [(24, 4100, 224, 32), (50, 4090, 416, 32), (33, 4096, 384, 128), (130, 2060, 320, 64),
                                         (5, 300, 32 * 131, 32), (9, 65, 96 * 41, 96)])
def test_matmul_q4_exact_where_tiles_fill_the_card(cuda, m, n, k, group, dtype):
    """Two and four tiles of rows to a workgroup, and rings that go round."""
    test_matmul_q4_exact(cuda, m, n, k, group, dtype)


@pytest.mark.parametrize("dtype", ["f16", "i8"])
@pytest.mark.parametrize("scales", ["f32", "f16"])
@pytest.mark.parametrize("m", [1, 12, 40])
def test_matmul_q4_of_pitched_rows(cuda, m, scales, dtype):
    """Rows apart by more than they hold: by whole 16 bytes, and by an odd number, with
    scales that begin at an odd element; what lies behind a row is NaN or never read."""
    import torch

    n, k, group = (4099, 160, 32) if m == 40 else (45, 160, 32)
    x, w, s, _ = q4_inputs(cuda, m, n, k, group, dtype, scales, exact=True)
    want, packed, el = ref.matmul_q4(x, w, s), xt.pack_q4(w), DSL[dtype]
    for xp, wp in ((k + 32, k // 2 + 16), (k + 1, k // 2 + 3)):
        sp = k // group + 2
        xa, wa = xt.Array((m, xp), el), xt.Array((n, wp), xt.int8)
        sa, ya = xt.Array((n, sp), DSL[scales]), xt.Array((m, n), xt.float32)

        @xt.kernel
        def parts(x, w, s, y):
            t = xt.matmul_q4(xt.load(x, index=(0, 0), shape=(m, k)), xt.load(w, index=(0, 0), shape=(n, k // 2)),
                             xt.load(s, index=(0, 0), shape=(n, k // group)))
            xt.store(y, index=(0, 0), tile=t)

        p = xt.convert(parts, args=(xa, wa, sa, ya), grid=(1, 1, 1))
        bx = torch.full((m, xp), 99 if dtype == "i8" else math.nan, device=cuda).to(x.dtype)
        bw = torch.full((n, wp), -1, dtype=torch.int8, device=cuda)
        bs = torch.full((n * sp + 1,), math.nan, dtype=s.dtype, device=cuda)[1:].view(n, sp)
        bx[:, :k], bw[:, : k // 2], bs[:, : k // group] = x, packed, s
        y = torch.full((m, n), 7.0, device=cuda)
        say(xt.plan(p)["kernel"], m, scales, dtype, xp, wp)
        xt.launch(p, bx, bw, bs, y)
        assert torch.equal(y.double(), want)


def test_matmul_q4_refuses_rows_two_gigabytes_apart(cuda):
    import torch

    @xt.kernel
    def part(x, w, s, y):
        t = xt.matmul_q4(xt.load(x, index=(0, 0), shape=(2, 32)), xt.load(w, index=(0, 0), shape=(16, 16)),
                         xt.load(s, index=(0, 0), shape=(16, 1)))
        xt.store(y, index=(0, 0), tile=t)

    x = torch.empty(2, 1 << 30, dtype=torch.float16, device=cuda)
    w, s = torch.zeros(16, 16, dtype=torch.int8, device=cuda), torch.ones(16, 1, device=cuda)
    p = xt.convert(part, args=(xt.Array(tuple(x.shape), xt.float16), xt.Array((16, 16), xt.int8),
                               xt.Array((16, 1), xt.float32), xt.Array((2, 16), xt.float32)), grid=(1, 1, 1))
    with pytest.raises(ValueError, match="2.31 bytes"):
        xt.launch(p, x, w, s, torch.zeros(2, 16, device=cuda))


def test_matmul_q4_of_parts_of_arrays(cuda):
    """Blocks over columns of the result, and row pitches of larger arrays."""
    import torch

    xa, wa = xt.Array((5, 512), xt.float16), xt.Array((96, 256), xt.int8)
    sa, ya = xt.Array((96, 8), xt.float16), xt.Array((5, 96), xt.float32)

    @xt.kernel
    def part(x, w, s, y):
        i = xt.bid(0)
        t = xt.matmul_q4(xt.load(x, index=(0, 1), shape=(5, 256)), xt.load(w, index=(i, 1), shape=(32, 128)),
                         xt.load(s, index=(i, 1), shape=(32, 4)))
        xt.store(y, index=(0, i), tile=t)

    p = xt.convert(part, args=(xa, wa, sa, ya), grid=(3, 1, 1))
    x, w, s, _ = q4_inputs(cuda, 5, 96, 512, 64, "f16", "f16", exact=True)
    y = torch.zeros(5, 96, device=cuda)
    xt.launch(p, x, xt.pack_q4(w), s, y)
    assert torch.equal(y.double(), ref.matmul_q4(x[:, 256:], w[:, 256:], s[:, 4:]))


def test_matmul_q4_unaligned_and_not_finite(cuda):
    import torch

    p = K.matmul_q4(3, 20, 128, group=32, dtype=xt.bfloat16, scales=xt.float16)
    x, w, s, _ = q4_inputs(cuda, 3, 20, 128, 32, "bf16", "f16", exact=True)
    packed = xt.pack_q4(w)
    bx = torch.zeros(3 * 128 + 1, dtype=torch.bfloat16, device=cuda)[1:].view(3, 128)
    bw = torch.zeros(20 * 64 + 3, dtype=torch.int8, device=cuda)[3:].view(20, 64)
    bs = torch.zeros(20 * 4 + 1, dtype=torch.float16, device=cuda)[1:].view(20, 4)
    bx.copy_(x), bw.copy_(packed), bs.copy_(s)
    y = torch.zeros(3, 20, device=cuda)
    xt.launch(p, bx, bw, bs, y)
    assert torch.equal(y.double(), ref.matmul_q4(x, w, s))
    bx[1, 3] = math.nan
    xt.launch(p, bx, bw, bs, y)
    assert bool(torch.isnan(y[1]).all()) and torch.equal(y[[0, 2]].double(), ref.matmul_q4(x, w, s)[[0, 2]])


@pytest.mark.parametrize("m", [3, 20])
def test_matmul_q4_large_and_infinite_values(cuda, m):
    """Up to 2^115 a row's sums are held; an infinity makes its row NaN."""
    import torch

    p = K.matmul_q4(m, 33, 256, group=128, dtype=xt.bfloat16, scales=xt.float32, out=xt.float32)
    x, w, s, _ = q4_inputs(cuda, m, 33, 256, 128, "bf16", "f32", exact=True)
    s *= 2.0**-20
    x[1] *= 2.0**113
    y = torch.full((m, 33), 7.0, device=cuda)
    xt.launch(p, x, xt.pack_q4(w), s, y)
    assert torch.equal(y.double(), ref.matmul_q4(x, w, s))
    x[2, 250] = math.inf
    xt.launch(p, x, xt.pack_q4(w), s, y)
    assert bool(torch.isnan(y[2]).all())
    y[2], x[2] = 0, 0
    assert torch.equal(y.double(), ref.matmul_q4(x, w, s))


def test_matmul_q4_refuses_a_result_over_an_operand(cuda):
    import torch

    p = K.matmul_q4(32, 32, 64, group=32, dtype=xt.float16, scales=xt.float32, out=xt.float32)
    buf = torch.zeros(4096, device=cuda)
    x, w, s = buf.view(torch.float16)[:2048].view(32, 64), torch.zeros(32, 32, dtype=torch.int8, device=cuda), torch.ones(
        32, 2, device=cuda)
    with pytest.raises(ValueError, match="meets buffer 0"):
        xt.launch(p, x, w, s, buf[512 : 512 + 1024].view(32, 32))


# -- attend ------------------------------------------------------------------------


def attend_case(cuda, b, hk, g, nq, nk, d, dtype="bf16", cap=None, causal=False, window=None, slopes=False, start=None,
                length=None, prefix=None, docs=None, token_major=False, scale=None, qscale=2.0, seed=1, edit=None,
                misaligned=False, over_q=False):
    """Launches one and checks it; start, length, prefix: a number per sequence;
    docs: (of the queries, of the keys), lists per sequence."""
    import torch

    p = K.masked_attention(b, hk, g, nq, nk, d, dtype=DSL[dtype], cap=cap, causal=causal, window=window, slopes=slopes,
                           start=start is not None, length=length is not None, prefix=prefix is not None,
                           docs=docs is not None, token_major=token_major, scale=scale)
    say(xt.plan(p)["kernel"], "workspace", xt.workspace(p), dict(start=start, length=length, prefix=prefix))
    scale = d**-0.5 if scale is None else scale
    q = rand((b, hk * g, nq, d), dtype, cuda, seed, qscale)
    k, v = rand((b, hk, nk, d), dtype, cuda, seed + 1), rand((b, hk, nk, d), dtype, cuda, seed + 2)
    if edit:
        edit(q, k, v)
    sl = torch.exp2(-torch.arange(1, hk * g + 1, device=cuda).float() * 8 / (hk * g)).view(hk, g) if slopes else None

    def ints(values, shape):
        return None if values is None else torch.tensor(values, dtype=torch.int32, device=cuda).view(shape)

    st, le, pr = (ints(t, (b, 1)) for t in (start, length, prefix))
    qd, kd = (None, None) if docs is None else (ints(docs[0], (b, nq)), ints(docs[1], (b, nk)))
    want, far = ref.attend(q, k, v, scale, cap=cap, slopes=sl, causal=causal, window=window, start=st, length=le,
                           prefix=pr, q_docs=qd, k_docs=kd)

    def lay(t):
        if token_major:
            t = t.transpose(1, 2).reshape(b, t.shape[2], -1)
        if misaligned:
            moved = torch.zeros(t.numel() + 1, dtype=t.dtype, device=cuda)[1:].view(t.shape)
            moved.copy_(t)
            return moved
        return t.contiguous()

    lq, lk, lv = lay(q), lay(k), lay(v)
    o = lq if over_q else torch.full((lq.numel() + 16,), 7.0, dtype=lq.dtype, device=cuda)[: lq.numel()].view(lq.shape)
    extras = [t for t in (sl, st, le, pr, qd, kd) if t is not None]
    xt.launch(p, lq, lk, lv, *extras, o)
    torch.cuda.synchronize()
    got = o.view(b, nq, hk * g, d).transpose(1, 2) if token_major else o
    ref.assert_within(got, want, far, xt.plan(p)["kernel"])
    return got


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
def test_attend_heads_of_every_width(cuda, d, dtype):
    attend_case(cuda, 1, 2, 2, 150, 200, d, dtype)                        # many rows
    attend_case(cuda, 2, 1, 4, 3, 700, d, dtype, causal=True, start=[600, 697], length=[603, 700])  # few, split
    attend_case(cuda, 1, 2, 3, 5, 77, d, dtype, token_major=True, cap=20.0)


@pytest.mark.parametrize("nq,nk", [(1, 1), (1, 31), (1, 32), (1, 33), (2, 64), (7, 65), (31, 127), (32, 128), (33, 129),
                                   (64, 64), (65, 63), (127, 191), (128, 256), (129, 257), (300, 500)])
@pytest.mark.parametrize("causal", [False, True])
def test_attend_lengths(cuda, nq, nk, causal):
    attend_case(cuda, 1, 2, 1, nq, nk, 64, "f16", causal=causal)
    attend_case(cuda, 2, 1, 3, nq, nk, 128, "bf16", causal=causal, start=[nk - nq, -1], length=[nk, max(nk - 3, 0)])


@pytest.mark.parametrize("nq", [1, 5, 40, 200])
@pytest.mark.parametrize("what", ["cap", "slopes", "window", "prefix", "docs", "all"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attend_masks_and_biases(cuda, what, nq, dtype):
    import random

    r, b, nk = random.Random(nq), 2, 290
    every = what == "all"
    start = [40, 250]
    docs = None
    if what == "docs" or every:
        kd = [sorted(r.randint(-2, 3) for _ in range(nk)), [r.randint(-2, 3) for _ in range(nk)]]
        docs = ([[kd[i][min(start[i] + t, nk - 1)] for t in range(nq)] for i in range(b)], kd)
    attend_case(cuda, b, 2, 2, nq, nk, 64, dtype, cap=5.0 if what == "cap" or every else None, causal=what != "cap",
                slopes=what == "slopes" or every, window=33 if what == "window" or every else None, start=start,
                length=[nk, 277], prefix=[70, 0] if what == "prefix" or every else None, docs=docs)


@pytest.mark.parametrize("nq", [1, 8, 200])
def test_attend_rows_that_see_nothing(cuda, nq):
    import torch

    y = attend_case(cuda, 3, 1, 2, nq, 600, 64, causal=True, start=[-nq // 2, -nq - 5, 3], length=[600, 600, 0])
    assert bool((y[1:] == 0).all())
    y = attend_case(cuda, 1, 1, 2, nq, 600, 64, docs=([[9] * nq], [[1] * 600]))
    assert bool((y == 0).all())
    y = attend_case(cuda, 1, 1, 1, nq, 70, 64, causal=True, window=5, start=[100])
    assert bool((y == 0).all()) and not torch.isnan(y).any()


@pytest.mark.parametrize("n,d", [(1, 64), (20, 96), (300, 128)])
def test_attend_one_tensor_for_queries_keys_and_values(cuda, n, d):
    import torch

    x = rand((2, 1, n, d), "bf16", cuda, 5)
    p = K.masked_attention(2, 1, 1, n, n, d, causal=True)
    o = torch.zeros_like(x)
    xt.launch(p, x, x, x, o)
    want, far = ref.attend(x, x, x, 1 / math.sqrt(d), causal=True)
    ref.assert_within(o, want, far)
    with pytest.raises(ValueError, match="meets buffer"):
        xt.launch(p, x, x, x, x)


def test_rms_norm_of_a_tensor_added_to_itself(cuda):
    import torch

    m = K.rms_norm(6, 1003, xt.float32)
    x, g = rand((6, 1003), "f32", cuda, 1), rand((1, 1003), "f32", cuda, 2)
    want_h, want = ref.rms_norm(x, x, g, 1e-6)
    y = torch.zeros_like(x)
    xt.launch(m, x, x, g, x, y)  # the sum over both
    assert torch.equal(x.double(), want_h)
    ref.assert_within(y, want, want.abs() * 40 * 2.0**-24 + 1e-37)


@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("nk", [193, 257, 321, 640])
def test_attend_rows_whose_keys_two_groups_of_waves_share(cuda, nk, d):
    """An odd number of tiles, groups without a visible tile, and rows without a key."""
    attend_case(cuda, 1, 2, 1, 150, nk, d, "bf16")
    attend_case(cuda, 3, 1, 2, 90, nk, d, "f16", causal=True, start=[nk - 90, -20, 40], length=[nk, nk - 1, 30],
                slopes=True)
    docs = [[t // 70 for t in range(nk)]] * 2
    attend_case(cuda, 2, 1, 1, nk, nk, d, "bf16", causal=True, docs=(docs, docs), prefix=[3, 200], over_q=True)


@pytest.mark.parametrize("n", [200, 500])
def test_attend_infinite_values_where_two_groups_of_waves_share_keys(cuda, n):
    """Values of both groups' tiles that earlier rows do not see."""
    import torch

    q, k, v = (rand((1, 1, n, 64), "f16", cuda, s) for s in (1, 2, 3))
    v[0, 0, 40, 3], v[0, 0, 90, 4], v[0, 0, 130, 5], v[0, 0, n - 1, 6] = math.inf, -math.inf, math.nan, math.nan
    p = K.masked_attention(1, 1, 1, n, n, 64, dtype=xt.float16, causal=True)
    o = torch.zeros_like(q)
    xt.launch(p, q, k, v, o)
    o = o[0, 0].float()
    assert bool(torch.isfinite(o[:40]).all()) and bool((o[40:, 3] == math.inf).all())
    assert bool(torch.isfinite(o[:90, 4]).all()) and bool((o[90:, 4] == -math.inf).all())
    assert bool(torch.isfinite(o[:130, 5]).all()) and bool(torch.isnan(o[130:, 5]).all())
    assert bool(torch.isfinite(o[:-1, 6]).all()) and bool(torch.isnan(o[-1, 6])) and bool(torch.isfinite(o[:, 7:]).all())


@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("nq,g", [(1, 1), (3, 4), (70, 1)])
def test_attend_windows_split_by_themselves(cuda, d, nq, g):
    """A window's keys alone are split, wherever in the cache it lies, or before it."""
    attend_case(cuda, 4, 1, g, nq, 4100, d, "bf16", causal=True, window=1100, start=[4100 - nq, 30, 2000, -5000],
                length=[4100, 4000, 1999, 4100])
    attend_case(cuda, 3, 2, g, nq, 2100, d, "f16", causal=True, window=300, slopes=True, start=[2090, 0, 1111])


def test_attend_extreme_positions(cuda):
    big = 2**31 - 1
    attend_case(cuda, 2, 1, 1, 3, 100, 64, causal=True, start=[big, -big - 1], length=[big, 100], prefix=[big, -big])
    attend_case(cuda, 1, 1, 1, 3, 100, 64, causal=True, window=2**31 - 1, start=[97], length=[-5])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("nq,g", [(1, 1), (4, 2), (100, 2)])
def test_attend_hidden_values_have_no_effect(cuda, dtype, nq, g):
    """NaN, infinities and the type's lowest value in hidden keys and values: past a
    length, past the diagonal, in another document."""
    import torch

    nk = 300

    def edit(q, k, v):
        low = torch.finfo(v.dtype).min
        for t, at in ((k, 251), (v, 251)):
            t[:, :, at:] = math.nan
            t[:, :, at + 3] = math.inf
            t[:, :, at + 4] = low

    attend_case(cuda, 1, 2, g, nq, nk, 64, dtype, length=[251], edit=edit)
    start = 180

    def edit2(q, k, v):  # seen by no row of this launch, in the diagonal's tile
        k[:, :, start + nq :] = math.nan
        v[:, :, start + nq] = -math.inf
        v[:, :, start + nq + 1 :] = math.nan

    attend_case(cuda, 1, 2, g, nq, nk, 64, dtype, causal=True, start=[start], edit=edit2)
    kd = [1] * 50 + [2] * 250

    def edit3(q, k, v):
        v[:, :, :50] = math.nan
        k[:, :, 20:40] = math.inf

    attend_case(cuda, 1, 2, g, nq, nk, 64, dtype, docs=([[2] * nq], [kd]), edit=edit3)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attend_infinite_values_reach_the_rows_that_see_them(cuda, dtype):
    """A causal launch: rows before the key are finite, rows behind it are not."""
    import torch

    q, k, v = (rand((1, 1, 100, 64), dtype, cuda, s) for s in (1, 2, 3))
    v[0, 0, 40, 3], v[0, 0, 41, 3], v[0, 0, 50, 4], v[0, 0, 60, 5] = math.inf, 1.0, -math.inf, math.nan
    v[0, 0, 70, 4] = math.inf
    p = K.masked_attention(1, 1, 1, 100, 100, 64, dtype=DSL[dtype], causal=True)
    o = torch.zeros_like(q)
    xt.launch(p, q, k, v, o)
    o = o[0, 0].float()
    assert bool(torch.isfinite(o[:40]).all()) and bool((o[40:, 3] == math.inf).all())
    assert bool(torch.isfinite(o[:50, 4]).all()) and bool((o[50:70, 4] == -math.inf).all()) and bool(
        torch.isnan(o[70:, 4]).all())
    assert bool(torch.isfinite(o[:60, 5]).all()) and bool(torch.isnan(o[60:, 5]).all())
    assert bool(torch.isfinite(o[:, 6:]).all())


def test_attend_large_scores_and_scales(cuda):
    attend_case(cuda, 1, 1, 1, 40, 300, 64, "bf16", qscale=60.0)
    attend_case(cuda, 1, 1, 1, 40, 300, 64, "f16", qscale=60.0, cap=30.0)
    attend_case(cuda, 1, 1, 1, 2, 300, 64, "f16", scale=1e-8)


@pytest.mark.parametrize("nq", [2, 60])
def test_attend_unaligned_rows_go_through_registers(cuda, nq):
    attend_case(cuda, 1, 2, 2, nq, 200, 96, "bf16", causal=True, start=[100], misaligned=True)
    attend_case(cuda, 2, 2, 2, nq, 190, 64, "f16", length=[190, 33], misaligned=True, token_major=True)


@pytest.mark.parametrize("nq,nk", [(1, 4000), (90, 200)])
def test_attend_result_over_the_queries(cuda, nq, nk):
    attend_case(cuda, 1, 2, 2, nq, nk, 64, "bf16", over_q=True)


def test_attend_split_rows_with_shared_keys(cuda):
    """More than 32 rows of one key head over many keys: 128-row tiles, split."""
    attend_case(cuda, 1, 1, 4, 20, 3000, 128, "bf16", causal=True, start=[2900], length=[2930])
    attend_case(cuda, 1, 2, 1, 150, 2500, 64, "f16", docs=([[5] * 150], [[4] * 900 + [5] * 1600]))


def test_attend_one_tile_a_block_of_rows(cuda):
    """Blocks of query rows, each with a start of its own, keys shared."""
    import torch

    q = rand((1, 96, 64), "bf16", cuda, 1)
    k, v = rand((1, 96, 64), "bf16", cuda, 2), rand((1, 96, 64), "bf16", cuda, 3)

    @xt.kernel
    def tiles(q, k, v, starts, o):
        i = xt.bid(0)
        qt = xt.load(q, index=(0, i, 0), shape=(1, 32, 64))
        kt = xt.reshape(xt.load(k, index=(0, 0, 0), shape=(1, 96, 64), shared=1), shape=(96, 64))
        vt = xt.reshape(xt.load(v, index=(0, 0, 0), shape=(1, 96, 64), shared=1), shape=(96, 64))
        s = xt.load(starts, index=(i, 0), shape=(1, 1))
        xt.store(o, index=(0, i, 0), tile=xt.attend(qt, kt, vt, scale=0.125, causal=True, start=s))

    a = xt.Array((1, 96, 64), xt.bfloat16)
    p = xt.convert(tiles, args=(a, a, a, xt.Array((3, 1), xt.int32), a), grid=(3, 1, 1))
    o = torch.zeros_like(q)
    xt.launch(p, q, k, v, torch.tensor([[0], [32], [64]], dtype=torch.int32, device=cuda), o)
    want, far = ref.attend(q[None], k[None], v[None], 0.125, causal=True)
    ref.assert_within(o[None], want, far)


def test_attend_refuses_a_result_over_its_keys(cuda):
    import torch

    p = K.masked_attention(1, 1, 1, 64, 64, 64)
    q, k, v = (torch.zeros(1, 1, 64, 64, dtype=torch.bfloat16, device=cuda) for _ in range(3))
    for o in (k, v):
        with pytest.raises(ValueError, match="meets buffer"):
            xt.launch(p, q, k, v, o)
    both = torch.zeros(65 * 64, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(ValueError, match="meets buffer 0"):
        xt.launch(p, both[: 64 * 64].view(1, 1, 64, 64), k, v, both[64:].view(1, 1, 64, 64))


def test_attend_offsets_past_32_bits(cuda):
    """Keys of more than 4 GiB: the last ones, against the same on their own."""
    import torch

    nk, d, w = (1 << 25) + 100, 64, 90
    k = torch.zeros(1, 1, nk, d, dtype=torch.bfloat16, device=cuda)
    v = torch.zeros_like(k)
    q = rand((1, 1, 2, d), "bf16", cuda, 1)
    k[:, :, -200:], v[:, :, -200:] = rand((1, 1, 200, d), "bf16", cuda, 2), rand((1, 1, 200, d), "bf16", cuda, 3)
    p = K.masked_attention(1, 1, 1, 2, nk, d, causal=True, window=w, start=True)
    say(xt.plan(p)["kernel"])
    o = torch.zeros_like(q)
    xt.launch(p, q, k, v, torch.tensor([[nk - 2]], dtype=torch.int32, device=cuda), o)
    at = torch.tensor([[198]], device=cuda)
    want, far = ref.attend(q, k[:, :, -200:], v[:, :, -200:], d**-0.5, causal=True, window=w, start=at)
    ref.assert_within(o, want, far)


# -- launches ------------------------------------------------------------------------


def decode_program(cuda, seed):
    import torch

    p = K.masked_attention(1, 2, 4, 1, 5000, 64, causal=True, start=True, length=True)
    assert xt.workspace(p) > 0
    q, k, v = (rand(s, "bf16", cuda, seed + i) for i, s in enumerate([(1, 8, 1, 64), (1, 2, 5000, 64), (1, 2, 5000, 64)]))
    st = torch.tensor([[4321]], dtype=torch.int32, device=cuda)
    return p, q, k, v, st, st + 1


def test_split_launches_on_streams_and_in_graphs(cuda):
    """Two graphs of split launches, replayed with eager work between, and launches on
    a side stream by handle: each has a workspace of its own."""
    import torch

    progs = [decode_program(cuda, 10 * i) for i in range(3)]
    want = []
    for p, q, *rest in progs:
        o = torch.zeros_like(q)
        xt.launch(p, q, *rest, o)
        want.append(o)
    torch.cuda.synchronize()
    graphs = []
    for p, q, *rest in progs[:2]:
        o = torch.zeros_like(q)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            xt.launch(p, q, *rest, o)
        graphs.append((g, o))
    side = torch.cuda.Stream()
    for _ in range(4):
        for g, o in graphs:
            o.zero_()
        side.wait_stream(torch.cuda.current_stream())
        p, q, *rest = progs[2]
        o2 = torch.zeros_like(q)
        side.wait_stream(torch.cuda.current_stream())
        xt.launch(p, q, *rest, o2, stream=side)
        for g, _ in graphs:
            g.replay()
        scratch = torch.full((1 << 20,), 3.0, device=cuda).sum()  # eager work that takes freed memory
        torch.cuda.synchronize()
        assert float(scratch) == 3.0 * (1 << 20)
        for (g, o), w in zip(graphs, want):
            assert torch.equal(o, w)
        assert torch.equal(o2, want[2])


def test_split_launch_without_a_workspace(cuda):
    """The C entry that takes none: the keys are not split; and too small a one is refused."""
    import torch

    p, q, k, v, st, le = decode_program(cuda, 3)
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    xt.launch(p, q, k, v, st, le, a)
    bufs = [q, k, v, st, le, b]
    ptrs, sizes = [t.data_ptr() for t in bufs], [t.numel() * t.element_size() for t in bufs]
    stream = torch.cuda.current_stream().cuda_stream
    xt._native.launch(p, None, ptrs, sizes, stream)
    want, far = ref.attend(q, k, v, 0.125, causal=True, start=st, length=le)
    ref.assert_within(a, want, far)
    ref.assert_within(b, want, far)
    work = torch.zeros(xt.workspace(p), dtype=torch.uint8, device=cuda)
    with pytest.raises(ValueError, match="works in"):
        xt._native.launch(p, None, ptrs, sizes, stream, work.data_ptr(), work.numel() - 1)
    with pytest.raises(ValueError, match="works in"):
        xt._native.launch(p, None, ptrs, sizes, stream, work.data_ptr() + 1, work.numel())


def test_results_are_the_same_run_to_run(cuda):
    import torch

    p, q, k, v, st, le = decode_program(cuda, 5)
    n = K.matmul_q4(4, 200, 4096, group=64)
    x, w, s, _ = q4_inputs(cuda, 4, 200, 4096, 64, "bf16", "f16")
    w = xt.pack_q4(w)
    got = []
    for _ in range(3):
        o, y = torch.zeros_like(q), torch.zeros(4, 200, device=cuda)
        xt.launch(p, q, k, v, st, le, o)
        xt.launch(n, x, w, s, y)
        got.append((o, y))
    assert all(torch.equal(o, got[0][0]) and torch.equal(y, got[0][1]) for o, y in got)


@pytest.mark.parametrize("tokens", [1, 45])
def test_a_layer_of_them(cuda, tokens):
    """Norm to 8-bit rows, 4-bit projections, attention with a distance bias over a
    cache, the projection back and the next norm, against the same in 64 bits on
    the kernels' own intermediate values."""
    import torch

    width, hk, g, d, cache = 256, 2, 2, 64, 300
    start = 200
    x, r = rand((tokens, width), "bf16", cuda, 1), rand((tokens, width), "bf16", cuda, 2)
    gamma = rand((1, width), "bf16", cuda, 3)
    h = torch.zeros_like(x)
    q8, s8 = torch.zeros(tokens, width, dtype=torch.int8, device=cuda), torch.zeros(tokens, 1, device=cuda)
    xt.launch(K.rms_norm(tokens, width, quantize=True), x, r, gamma, h, q8, s8)
    want_h, want_y = ref.rms_norm(x, r, gamma, 1e-6)
    rows = q8.double() * s8.double()
    assert float(((rows - want_y).abs() / s8).max()) <= 0.501

    def project(inp, n, k, seed, **kw):
        _, w, s, _ = q4_inputs(cuda, 1, n, k, 64, "bf16", "f16", seed=seed)
        y = torch.zeros(tokens, n, dtype=torch.bfloat16, device=cuda)
        rs = kw.pop("rs", None)
        p = K.matmul_q4(tokens, n, k, group=64, out=xt.bfloat16, row_scale=rs is not None, **kw)
        xt.launch(p, inp, xt.pack_q4(w), s, *([rs] if rs is not None else []), y)
        want = ref.matmul_q4(inp, w, s, rs)
        assert float((y.double() - want).norm() / want.norm()) <= 2.0**-8 + 4e-6
        return y

    q = project(q8, hk * g * d, width, 4, dtype=xt.int8, rs=s8)
    k = torch.zeros(1, cache, hk * d, dtype=torch.bfloat16, device=cuda)
    v = torch.zeros_like(k)
    k[:, :start], v[:, :start] = rand((1, start, hk * d), "bf16", cuda, 5), rand((1, start, hk * d), "bf16", cuda, 6)
    k[0, start : start + tokens] = project(q8, hk * d, width, 7, dtype=xt.int8, rs=s8)
    v[0, start : start + tokens] = project(q8, hk * d, width, 8, dtype=xt.int8, rs=s8)
    slopes = torch.tensor([[0.5, 0.25], [0.125, 0.0625]], device=cuda)
    st = torch.tensor([[start]], dtype=torch.int32, device=cuda)
    a = torch.zeros(1, tokens, hk * g * d, dtype=torch.bfloat16, device=cuda)
    p = K.masked_attention(1, hk, g, tokens, cache, d, causal=True, slopes=True, start=True, length=True, token_major=True)
    xt.launch(p, q.view(1, tokens, -1), k, v, slopes, st, st + tokens, a)

    def heads(t, n):
        return t.view(1, -1, n, d).transpose(1, 2)

    want, far = ref.attend(heads(q, hk * g), heads(k, hk), heads(v, hk), d**-0.5, slopes=slopes, causal=True, start=st,
                           length=st + tokens)
    ref.assert_within(heads(a, hk * g), want, far)
    o = project(a.view(tokens, -1), width, hk * g * d, 9)
    y = torch.zeros_like(x)
    xt.launch(K.rms_norm(tokens, width), o, h, gamma, h, y)  # the sum over the residual
    _, want = ref.rms_norm(o, want_h.bfloat16(), gamma, 1e-6)
    ref.assert_within(y, want, want.abs() * (2.0**-8 + 40 * 2.0**-24) + 1e-37)
