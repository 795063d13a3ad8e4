"""Microscaled 4-bit rows and products of them on the GPU, against the definition in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest

import xtile_amd as xt
from xtile_amd import kernels as K

from . import answers_ref as ref
from .gpu_util import kernels_of
from .operators_ref import HALF

pytestmark = pytest.mark.gpu

DTYPES = {"f32": xt.float32, "f16": xt.float16, "bf16": xt.bfloat16}


def torch_dtype(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def from_bits(bits, dtype):
    """A CPU tensor of a type from its bits."""
    import torch

    if dtype == "f32":
        return torch.from_numpy(bits.astype(np.uint32).view(np.int32).copy()).view(torch.float32)
    return torch.from_numpy(bits.astype(np.uint16).view(np.int16).copy()).view(torch_dtype(dtype))


def int8(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).view(torch.int8).cuda()


def uint8(t):
    import torch

    return t.cpu().view(torch.uint8).numpy()


def run_quantize(x, dtype):
    """(codes, bytes, values) of a CPU tensor."""
    import torch

    rows, cols = x.shape
    print(f"[gpu] quantize_mx4 {dtype} {rows} x {cols}", flush=True)
    q = torch.full((rows, cols // 2), 77, dtype=torch.int8, device="cuda")
    s = torch.full((rows, cols // 32), 77, dtype=torch.int8, device="cuda")
    y = torch.full((rows, cols), 7.0, dtype=x.dtype, device="cuda")
    xt.launch(K.quantize_mx4(rows, cols, DTYPES[dtype], values=True), x.cuda(), q, s, y)
    return ref.unpack(uint8(q)), uint8(s), y.cpu().double().numpy()


def check_quantize(x, dtype):
    code, byte, y = run_quantize(x, dtype)
    want_code, want_byte = ref.quantize_mx4(x.double().numpy())
    assert np.array_equal(byte, want_byte)
    assert np.array_equal(code, want_code)
    assert np.array_equal(y, ref.values(want_code, want_byte), equal_nan=True)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("order", ["rising", "mixed"])
def test_every_value_of_16_bits(dtype, order):
    bits = np.arange(65536)
    if order == "mixed":
        # finite values of all sizes side by side, so that most of a block is far below its largest
        bits = bits[np.isfinite(from_bits(bits, dtype).double().numpy())]
        bits = np.random.default_rng(1).permutation(bits)[: 63488 // 32 * 32]
    check_quantize(from_bits(bits, dtype).view(-1, 32 if order == "mixed" else 64), dtype)


def test_values_of_32_bits():
    """Bits at random; then, of every exponent, all sixteenths of a block's largest magnitude
    (each tie among them) and the numbers next to them."""
    rng = np.random.default_rng(2)
    check_quantize(from_bits(rng.integers(0, 1 << 32, 1 << 18), "f32").view(-1, 128), "f32")
    rows = []
    for field in range(255):
        top = (field << 23) | int(rng.integers(0, 1 << 23))
        unit = np.ldexp(1.0, max(field, 1) - 127)
        block = np.concatenate(([0.0], np.arange(1, 32) / 16 * unit))
        bits = block.astype(np.float32).view(np.uint32).astype(np.int64)
        bits = bits + rng.integers(-1, 2, 32) * (bits > 0)
        bits |= rng.integers(0, 2, 32) << 31
        bits[0] = top
        rows.append(bits)
    check_quantize(from_bits(np.array(rows), "f32"), "f32")


@pytest.mark.parametrize("dtype,rows,cols", [("f32", 1, 32), ("bf16", 1, 4096), ("f16", 7, 96), ("bf16", 513, 1056),
                                             ("f32", 129, 160), ("f16", 33, 8192)])
def test_sizes(dtype, rows, cols):
    import torch

    g = torch.Generator().manual_seed(rows + cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(3 * torch.randn(rows, 1, generator=g))).to(torch_dtype(dtype))
    x[:, -32:] = 0.0
    x[0, 0] = -0.0
    check_quantize(x, dtype)


def pitched_rows_program(dtype, rows, cols, wide, trow, at):
    """Rows of `cols` from column tile `at` of wider arrays, `trow` a Block."""

    @xt.kernel
    def rows_kernel(x, q, s, y):
        b = xt.bid(0)
        t = xt.load(x, index=(b, at), shape=(trow, cols))
        scale = xt.mx4_scale(t)
        packed = xt.quantize_mx4(t, scale)
        xt.store(q, index=(b, at), tile=packed)
        xt.store(s, index=(b, at), tile=scale)
        xt.store(y, index=(b, at), tile=xt.dequantize_mx4(packed, scale, dtype=DTYPES[dtype]))

    x = xt.Array(shape=(rows, wide), dtype=DTYPES[dtype])
    q = xt.Array(shape=(rows, wide // 2), dtype=xt.int8)
    s = xt.Array(shape=(rows, wide // 32), dtype=xt.int8)
    return xt.convert(rows_kernel, args=(x, q, s, x), grid=(rows // trow, 1, 1))


@pytest.mark.parametrize("dtype,skip", [("bf16", 1), ("f32", 3), ("f16", 0)])
def test_blocks_pitches_and_alignment(dtype, skip):
    """Tiles of wider arrays, from any element on; what lies beside them stays."""
    import torch

    rows, cols, wide, at = 12, 96, 480, 2
    g = torch.Generator().manual_seed(5)
    x = torch.randn(rows, wide, generator=g).to(torch_dtype(dtype))

    def placed(shape, dtype, fill):
        n = shape[0] * shape[1]
        return torch.full((n + skip + 5,), fill, dtype=dtype, device="cuda")[skip:skip + n].view(shape)

    dx, y = placed(x.shape, x.dtype, 0), placed(x.shape, x.dtype, 9)
    q, s = placed((rows, wide // 2), torch.int8, 77), placed((rows, wide // 32), torch.int8, 77)
    dx.copy_(x)
    xt.launch(pitched_rows_program(dtype, rows, cols, wide, 3, at), dx, q, s, y)
    lo, hi = at * cols, (at + 1) * cols
    code, byte = ref.quantize_mx4(x[:, lo:hi].double().numpy())
    assert np.array_equal(uint8(q[:, lo // 2:hi // 2]), ref.pack(code))
    assert np.array_equal(uint8(s[:, lo // 32:hi // 32]), byte)
    assert np.array_equal(y[:, lo:hi].cpu().double().numpy(), ref.values(code, byte))
    for t, fill, a, b in ((q, 77, lo // 2, hi // 2), (s, 77, lo // 32, hi // 32), (y, 9, lo, hi)):
        assert bool((t[:, :a] == fill).all()) and bool((t[:, b:] == fill).all())


def test_values_over_their_input():
    """The values may take x's place, of one argument or two of the same tensor."""
    import torch

    x = torch.randn(40, 256).bfloat16()
    code, byte = ref.quantize_mx4(x.double().numpy())
    q = torch.empty(40, 128, dtype=torch.int8, device="cuda")
    s = torch.empty(40, 8, dtype=torch.int8, device="cuda")
    one = x.cuda()
    xt.launch(K.quantize_mx4(40, 256, values=True), one, q, s, one)
    assert np.array_equal(one.cpu().double().numpy(), ref.values(code, byte))
    assert np.array_equal(uint8(q), ref.pack(code))

    @xt.kernel
    def round_kernel(buf):
        t = xt.load(buf, index=(0, 0), shape=(40, 256))
        scale = xt.mx4_scale(t)
        xt.store(buf, index=(0, 0), tile=xt.dequantize_mx4(xt.quantize_mx4(t, scale), scale, dtype=xt.bfloat16))

    one = x.cuda()
    xt.launch(xt.convert(round_kernel, args=(xt.Array(shape=(40, 256), dtype=xt.bfloat16),), grid=(1, 1, 1)), one)
    assert np.array_equal(one.cpu().double().numpy(), ref.values(code, byte))


@pytest.mark.parametrize("dtype,rows,cols", [("f32", 9, 512), ("f16", 1, 32), ("bf16", 300, 96)])
def test_dequantize(dtype, rows, cols):
    """Every code with every scale, rounded once to the type (what passes it: infinite)."""
    import torch

    rng = np.random.default_rng(rows)
    code = rng.integers(0, 16, (rows, cols)).astype(np.uint8)
    byte = rng.integers(0, 256, (rows, cols // 32)).astype(np.uint8)
    byte.reshape(-1)[:4] = [0, 255, 254, 1][: byte.size]
    y = torch.empty(rows, cols, dtype=torch_dtype(dtype), device="cuda")
    xt.launch(K.dequantize_mx4(rows, cols, DTYPES[dtype]), int8(ref.pack(code)), int8(byte), y)
    want = torch.from_numpy(ref.values(code, byte)).float().to(y.dtype)  # 32 bits hold every value
    assert torch.equal(torch.isnan(y.cpu()), torch.isnan(want))
    fine = ~torch.isnan(want)
    assert torch.equal(y.cpu()[fine], want[fine])


# -- products -------------------------------------------------------------------


def random_rows(rng, rows, k, lo=110, hi=130):
    code = rng.integers(0, 16, (rows, k)).astype(np.uint8)
    byte = rng.integers(lo, hi, (rows, k // 32)).astype(np.uint8)
    return code, byte


def run_product(x, w, out):
    import torch

    m, n, k = x[0].shape[0], w[0].shape[0], x[0].shape[1]
    print(f"[gpu] matmul_mx4 {m} x {n} x {k} -> {out}", flush=True)
    y = torch.full((m, n), 3.0, dtype=torch_dtype(out), device="cuda")
    xt.launch(K.matmul_mx4(m, n, k, out=DTYPES[out]), int8(ref.pack(x[0])), int8(x[1]), int8(ref.pack(w[0])), int8(w[1]), y)
    return y.cpu().double().numpy()


def check_product(got, x, w, out):
    want, far = ref.matmul_mx4(ref.values(*x), ref.values(*w))
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    u = {"f32": HALF["float32"], "f16": HALF["float16"], "bf16": HALF["bfloat16"]}[out]
    far = far + u * np.abs(want) + (2.0**-25 if out == "f16" else 0.0)
    worst = (np.abs(got - want) / far)[~nan]
    assert worst.size == 0 or worst.max() <= 1, worst.max()


@pytest.mark.parametrize("m,n,k,out", [
    (1, 1, 32, "f32"), (1, 16, 256, "f32"), (1, 100, 4096, "bf16"), (3, 17, 64, "f16"), (8, 33, 96, "f32"), (9, 64, 288, "f32"),
    (16, 257, 1056, "bf16"), (17, 100, 512, "f32"), (31, 15, 224, "f32"), (33, 129, 1056, "bf16"), (64, 64, 8192, "f32"),
    (65, 1000, 320, "f16"), (100, 300, 2080, "f32"), (128, 128, 256, "f32"), (129, 257, 544, "bf16"), (256, 512, 1024, "f32"),
    (300, 700, 4128, "f32"), (513, 1025, 288, "bf16"), (1000, 2000, 1056, "f32"),
])
def test_products(m, n, k, out):
    rng = np.random.default_rng(m * n + k)
    x, w = random_rows(rng, m, k, 122, 130), random_rows(rng, n, k, 122, 130)
    check_product(run_product(x, w, out), x, w, out)


def product_buffers(x, w, out="f32"):
    import torch

    m, n = x[0].shape[0], w[0].shape[0]
    return [int8(ref.pack(x[0])), int8(x[1]), int8(ref.pack(w[0])), int8(w[1]),
            torch.full((m, n), 3.0, dtype=torch_dtype(out), device="cuda")]


# Sizes of which each kernel takes some; none is a multiple of a tile, nor K of a stage.
KERNELS = [(3, 100, 1056, "few_kernel<8, 8>"), (5, 9000, 1056, "few_kernel<8, 4>"), (15, 100, 4128, "few_kernel<16, 8>"),
           (12, 9000, 1056, "few_kernel<16, 4>"), (63, 4090, 2080, "mid_kernel<1, 1, 8>"), (125, 4090, 1056, "mid_kernel<1, 2, 4>"),
           (250, 4090, 1056, "mid_kernel<2, 2, 4>"), (1001, 4090, 544, "many_kernel<128, 128, 4, 3, 0>"),
           (1500, 4090, 1056, "many_kernel<128, 128, 4, 2, 0>"), (4090, 4000, 288, "many_kernel<256, 256, 8, 2, 0>"),
           # rows of scales that begin at whole words
           (1001, 4090, 640, "many_kernel<128, 128, 4, 3, 1>"), (1500, 4090, 1152, "many_kernel<128, 128, 4, 2, 1>"),
           (4090, 4000, 384, "many_kernel<256, 256, 8, 2, 1>")]


@pytest.mark.parametrize("m,n,k,kernel", KERNELS)
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_every_kernel(m, n, k, kernel, out):
    rng = np.random.default_rng(k)
    x, w = random_rows(rng, m, k, 122, 130), random_rows(rng, n, k, 122, 130)
    bufs = product_buffers(x, w, out)
    program = K.matmul_mx4(m, n, k, out=DTYPES[out])
    print(f"[gpu] matmul_mx4 {m} x {n} x {k} -> {out}: {kernel}", flush=True)
    assert kernels_of(program, bufs) == ["matmul_mx4_" + kernel]
    check_product(bufs[4].cpu().double().numpy(), x, w, out)


@pytest.mark.parametrize("k", [32, 64, 96, 128, 224, 256, 288, 384, 480, 512, 544, 640, 768, 800, 896, 1024, 1056, 1152, 1280,
                               1312, 1408, 2176, 2304])
@pytest.mark.parametrize("m,n", [(1000, 4090), (1500, 4090), (4090, 4000)])
def test_large_tiles_of_every_depth(m, n, k):
    """From fewer stages than buffers to more, with and without a part of one; scales of 255 in
    the last row and column."""
    rng = np.random.default_rng(k)
    x, w = random_rows(rng, m, k, 122, 130), random_rows(rng, n, k, 122, 130)
    x[1][-1, -1] = w[1][-1, 0] = 255
    check_product(run_product(x, w, "f32"), x, w, "f32")


@pytest.mark.parametrize("m,n,k", [(5, 40, 512), (40, 60, 288), (300, 290, 544)])
def test_scales_of_all_sizes(m, n, k):
    """Blocks whose scales are far apart, down to 0; and rows and columns with one of 255."""
    rng = np.random.default_rng(k)
    x, w = random_rows(rng, m, k, 0, 180), random_rows(rng, n, k, 80, 190)
    x[1][0] = 0
    x[1][2, -1] = 255
    x[0][2] = 0  # zeros do not hide it
    w[1][7, 0] = 255
    got = run_product(x, w, "f32")
    check_product(got, x, w, "f32")
    assert np.isnan(got[2]).all() and np.isnan(got[:, 7]).all() and not np.isnan(np.delete(got, 7, 1)[[0, 1, 3, 4]]).any()


def test_one_hot():
    """Each code and place by itself: which value of x meets which of w."""
    k, n = 512, 64
    rng = np.random.default_rng(0)
    w = random_rows(rng, n, k, 120, 134)
    for first in range(0, k, 128):
        code = np.zeros((128, k), dtype=np.uint8)
        code[np.arange(128), first + np.arange(128)] = 2  # 1.0
        x = code, np.full((128, k // 32), 127, dtype=np.uint8)
        assert np.array_equal(run_product(x, w, "f32"), ref.values(*w).T[first:first + 128])


def pitched_product_program(m, n, k, tm, tn, wide, at, out):
    """Columns from tile `at` of wider arrays, a Block for each tm x tn of the result."""

    @xt.kernel
    def product_kernel(x, xs, w, ws, y):
        i, j = xt.bid(0), xt.bid(1)
        a = xt.load(x, index=(i, at), shape=(tm, k // 2))
        s = xt.load(xs, index=(i, at), shape=(tm, k // 32))
        b = xt.load(w, index=(j, at), shape=(tn, k // 2))
        r = xt.load(ws, index=(j, at), shape=(tn, k // 32))
        xt.store(y, index=(i, j), tile=xt.matmul_mx4(a, s, b, r, dtype=DTYPES[out]))

    def rows(r, c):
        return xt.Array(shape=(r, c), dtype=xt.int8)

    args = (rows(m, wide // 2), rows(m, wide // 32), rows(n, wide // 2), rows(n, wide // 32),
            xt.Array(shape=(m, n), dtype=DTYPES[out]))
    return xt.convert(product_kernel, args=args, grid=(m // tm, n // tn, 1))


@pytest.mark.parametrize("skip", [0, 1, 6])
@pytest.mark.parametrize("m,n,k,tm,tn", [(6, 96, 96, 3, 48), (40, 64, 160, 20, 64), (512, 384, 288, 256, 192),
                                           (2048, 3840, 640, 1024, 1920), (4096, 4096, 384, 2048, 2048)])
def test_product_blocks_pitches_and_alignment(m, n, k, tm, tn, skip):
    """Tiles of wider arrays at any byte; what lies beside them, scales of 255, has no effect."""
    import torch

    wide, at = 3 * k, 1
    rng = np.random.default_rng(skip + k)

    def placed(a):
        t = torch.full((a.size + skip + 7,), -1, dtype=torch.int8, device="cuda")[skip:skip + a.size].view(a.shape)
        t.copy_(torch.from_numpy(a.view(np.int8)))
        return t

    def wider(rows):
        code, byte = rng.integers(0, 16, (rows, wide)).astype(np.uint8), np.full((rows, wide // 32), 255, dtype=np.uint8)
        byte[:, at * k // 32:(at + 1) * k // 32] = rng.integers(120, 134, (rows, k // 32))
        part = code[:, at * k:(at + 1) * k], byte[:, at * k // 32:(at + 1) * k // 32]
        return part, placed(ref.pack(code)), placed(byte)

    x, dx, dxs = wider(m)
    w, dw, dws = wider(n)
    y = torch.full((m, n), 3.0, device="cuda")
    print(f"[gpu] matmul_mx4 {m} x {n} x {k} in tiles, skip {skip}", flush=True)
    xt.launch(pitched_product_program(m, n, k, tm, tn, wide, at, "f32"), dx, dxs, dw, dws, y)
    check_product(y.cpu().double().numpy(), x, w, "f32")


def test_product_by_itself():
    """One tensor as both operands."""
    import torch

    rng = np.random.default_rng(9)
    x = random_rows(rng, 50, 256, 122, 130)
    q, s, y = int8(ref.pack(x[0])), int8(x[1]), torch.empty(50, 50, device="cuda")
    xt.launch(K.matmul_mx4(50, 50, 256), q, s, q, s, y)
    check_product(y.cpu().double().numpy(), x, x, "f32")


def test_quantized_rows_through_a_product():
    """As a layer runs: activations rounded, then the product, twice on two streams."""
    import torch

    m, n, k = 24, 160, 1056
    g = torch.Generator().manual_seed(3)
    x, w = torch.randn(m, k, generator=g).bfloat16(), (0.05 * torch.randn(n, k, generator=g)).bfloat16()
    wc = ref.quantize_mx4(w.double().numpy())
    xc = ref.quantize_mx4(x.double().numpy())
    dw, dws = int8(ref.pack(wc[0])), int8(wc[1])
    rows, product = K.quantize_mx4(m, k), K.matmul_mx4(m, n, k, out=xt.bfloat16)
    results = []
    for stream in (torch.cuda.Stream(), torch.cuda.Stream()):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            dx = x.cuda()
            q = torch.empty(m, k // 2, dtype=torch.int8, device="cuda")
            s = torch.empty(m, k // 32, dtype=torch.int8, device="cuda")
            y = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
            xt.launch(rows, dx, q, s)
            xt.launch(product, q, s, dw, dws, y)
            results.append((stream, y))
    for stream, y in results:
        stream.synchronize()
        check_product(y.cpu().double().numpy(), xc, wc, "bf16")


def test_graph_replays():
    import torch

    m, n, k = 5, 96, 512
    rows, product = K.quantize_mx4(m, k), K.matmul_mx4(m, n, k)
    rng = np.random.default_rng(4)
    w = random_rows(rng, n, k, 122, 130)
    dw, dws = int8(ref.pack(w[0])), int8(w[1])
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    q = torch.empty(m, k // 2, dtype=torch.int8, device="cuda")
    s = torch.empty(m, k // 32, dtype=torch.int8, device="cuda")
    y = torch.empty(m, n, device="cuda")

    def step():
        xt.launch(rows, x, q, s)
        xt.launch(product, q, s, dw, dws, y)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(3):
        new = torch.randn(m, k, generator=torch.Generator().manual_seed(seed)).bfloat16()
        x.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        check_product(y.cpu().double().numpy(), ref.quantize_mx4(new.double().numpy()), w, "f32")
