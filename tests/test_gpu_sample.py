"""Sampling on the GPU against its definition in 64 bits: the same tokens."""

from __future__ import annotations

import numpy as np
import pytest

import xtile_amd as xt
from xtile_amd import kernels as K

from . import answers_ref as ref

pytestmark = pytest.mark.gpu

DTYPES = {"f32": xt.float32, "f16": xt.float16, "bf16": xt.bfloat16}


def torch_dtype(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def column(v, rows, dtype):
    """A (rows, 1) tensor of a number, or of one for each row."""
    import torch

    return torch.tensor(v, dtype=dtype).expand(rows).reshape(rows, 1).contiguous().cuda()


def run(x, u, dtype, without_workspace=False, trow=None, **params):
    """Tokens of a CPU tensor of logits; params: numbers or lists of one a row."""
    import torch

    rows, vocab = x.shape
    asked = {k: v for k, v in params.items() if v is not None}
    m = K.sample(rows, vocab, DTYPES[dtype], trow=trow, **{k: True for k in asked})
    print(f"[gpu] {xt.plan(m)['kernel']}", flush=True)
    y = torch.full((rows, 1), -7, dtype=torch.int32, device="cuda")
    bufs = [x.cuda(), column(u, rows, torch.float32)]
    for name in ("temperature", "top_k", "top_p", "min_p"):
        if name in asked:
            bufs.append(column(asked[name], rows, torch.int32 if name == "top_k" else torch.float32))
    bufs.append(y)
    if without_workspace:
        from xtile_amd import _xtile

        _xtile.launch(m, None, [t.data_ptr() for t in bufs], [t.numel() * t.element_size() for t in bufs],
                      torch.cuda.current_stream().cuda_stream)
    else:
        xt.launch(m, *bufs)
    return y.view(-1).tolist()


def want(x, u, **params):
    rows = x.shape[0]

    def of(v, r, kind=np.float32):
        return None if v is None else kind(v[r] if isinstance(v, (list, tuple)) else v)

    return [ref.sample(x[r].double().numpy(), of(u, r),
                       **{k: of(v, r, np.int32 if k == "top_k" else np.float32) for k, v in params.items()})
            for r in range(rows)]


def check(x, u, dtype="f32", **params):
    w = want(x, u, **params)
    assert run(x, u, dtype, **params) == w
    assert run(x, u, dtype, without_workspace=True, **params) == w


def logits(rows, vocab, dtype, seed, spread=2.5):
    import torch

    g = torch.Generator().manual_seed(seed)
    return (spread * torch.randn(rows, vocab, generator=g)).to(torch_dtype(dtype))


def uniforms(rows, seed):
    return np.random.default_rng(seed).random(rows).astype(np.float32).tolist()


OPTIONS = [{}, {"temperature": 0.7}, {"top_k": 40}, {"top_p": 0.9}, {"min_p": 0.05},
           {"temperature": 1.3, "top_k": 1000, "top_p": 0.97, "min_p": 0.001}]


@pytest.mark.parametrize("options", OPTIONS, ids=lambda o: "-".join(o) or "none")
@pytest.mark.parametrize("rows,vocab,dtype", [(1, 32768, "f32"), (9, 50001, "bf16"), (5, 1000, "f16"), (3, 131072, "f32"),
                                              (70, 4097, "f32")])
def test_sizes(rows, vocab, dtype, options):
    check(logits(rows, vocab, dtype, vocab), uniforms(rows, vocab), dtype, **options)


@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 8, 31, 63, 65, 255, 2047, 2048, 2049])
def test_short_rows(vocab):
    rows = 12
    x = logits(rows, vocab, "f32", vocab)
    check(x, uniforms(rows, vocab))
    check(x, uniforms(rows, vocab), top_p=0.5, top_k=[1, 2, 3, vocab, vocab + 1, 0, -1, 5, vocab - 1, 9, 100, 1])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("options", [{}, {"top_k": 3000}, {"top_p": 0.3}, {"top_k": 20000, "top_p": 0.6}, {"min_p": 0.3}],
                         ids=lambda o: "-".join(o) or "none")
def test_many_equal_logits(dtype, options):
    """Halves, so that thousands are equal: by index."""
    x = (logits(6, 30000, "f32", 3, 1.0) * 2).round().div(2).to(torch_dtype(dtype))
    check(x, uniforms(6, 8), dtype, **options)


@pytest.mark.parametrize("vocab", [6, 2048, 2049, 5000, 70000])
def test_rows_of_one_value(vocab):
    """Weights are all 1: the token is the one that u, and the cuts, count out."""
    import torch

    x = torch.full((5, vocab), -3.25)
    u = [0.0, 0.5, 0.25, 0.999, 0.7]
    assert run(x, u, "f32") == [int(np.floor(np.float64(np.float32(v)) * vocab)) for v in u]
    check(x, u)
    check(x, u, top_k=[1, 2, 5, 3000, vocab], top_p=[0.5, 0.1, 1.0, 0.0, 0.75])
    check(x, u, temperature=[0.0, 1e-30, 1e30, float("inf"), 2.0])


def long_rows(rows, vocab, kind):
    """Rows dealt to several workgroups: of halves, of two values, and with most in one bin."""
    import torch

    x = logits(rows, vocab, "f32", vocab, 1.0)
    if kind == "halves":
        return (x * 2).round() / 2
    if kind == "two":
        return torch.where(x > 1.5, 1.0, -1.0)
    x = x * 1e-4
    x[:, 7] = 9.0
    return x


@pytest.mark.parametrize("options", [{}, {"top_k": [3000, 50, 60000, 1]}, {"top_p": 0.3}, {"top_k": 20000, "top_p": 0.6},
                                     {"min_p": [0.3, 0.0, 1.0, 1e-9]}, {"top_k": 256, "top_p": 0.9, "min_p": 0.01},
                                     {"temperature": [0.0, 100.0, 0.01, 1.0], "top_p": 0.99}],
                         ids=lambda o: "-".join(o) or "none")
@pytest.mark.parametrize("kind", ["halves", "two", "narrow"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sliced_rows(dtype, kind, options):
    """Runs that fit a list, ones that do not, and rows of nothing between them."""
    rows, vocab = 4, 66001
    assert xt.workspace(K.sample(rows, vocab, DTYPES[dtype], **{k: True for k in options}))
    x = long_rows(rows, vocab, kind).to(torch_dtype(dtype))
    check(x, uniforms(rows, 11), dtype, **options)
    x[2] = -float("inf")
    x[1, ::3] = float("nan")
    check(x, uniforms(rows, 12), dtype, **options)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("vocab", [8192, 8193, 8199, 20001, 32760, 32767, 32768, 32769])
def test_rows_kept_in_registers(dtype, vocab):
    """Around the sizes of 16-bit rows that are read once, with equal logits and NaN among them."""
    x = logits(7, vocab, dtype, vocab)
    x[2, ::2] = float("nan")
    x[3, :] = float("-inf")
    x[4, 1:] = x[4, 0]
    for options in ({}, {"top_k": [50, 1, 300, 5, vocab - 1, 0, 9000]}, {"top_p": 0.7, "min_p": 0.01}):
        check(x, uniforms(7, vocab), dtype, **options)


def test_odd_logits():
    """Infinities, NaN and zeros of both signs."""
    import torch

    inf, nan = float("inf"), float("nan")
    rows = [[-inf] * 9, [nan] * 9, [nan, -inf, 1.0, nan, 0.0, -inf, 1.0, 1.0, nan], [inf, 0.0, inf, -inf, nan, inf, 1.0, 2.0, 3.0],
            [0.0, -0.0, 0.0, -0.0, -1.0, -inf, 0.0, -0.0, 0.0], [-inf] * 8 + [-1e38], [3e38, -3e38, 3e38, 0, 0, 0, 0, 0, 0],
            [1e-45, -1e-45, 0.0, 1e-45, 0, 0, 0, 0, 0]]
    x = torch.tensor(rows)
    for u in (0.0, 0.3, 0.6, 0.999):
        for options in ({}, {"temperature": 0.5}, {"temperature": 0.0}, {"temperature": inf}, {"top_k": 4}, {"top_p": 0.5},
                        {"min_p": 0.9}, {"top_k": 2, "top_p": 0.2, "min_p": 1.0}):
            check(x, u, **options)
    assert run(x, 0.3, "f32")[:2] == [-1, -1]


def test_odd_parameters():
    """Each parameter past its range, and NaN."""
    inf, nan = float("inf"), float("nan")
    x = logits(8, 700, "f32", 1)
    check(x, [0.0, -1.0, 1.0, 2.0, nan, inf, -inf, float(np.nextafter(np.float32(1), np.float32(0)))])
    check(x, uniforms(8, 2), temperature=[0.0, -1.0, nan, inf, 1e-45, 3e38, -inf, 1e-3])
    check(x, uniforms(8, 3), top_p=[0.0, -1.0, 1.0, 2.0, nan, inf, -inf, 1e-30])
    check(x, uniforms(8, 4), min_p=[0.0, -1.0, 1.0, 2.0, nan, inf, -inf, 1e-30])
    check(x, uniforms(8, 5), top_k=[0, -1, 1, 700, 701, 2**31 - 1, -2**31, 699])


@pytest.mark.parametrize("dtype,vocab", [("f32", 70000), ("bf16", 70000), ("bf16", 20000)])
def test_odd_parameters_of_long_rows(dtype, vocab):
    """The same of rows dealt to slices, and of ones kept in registers."""
    inf, nan = float("inf"), float("nan")
    x = logits(8, vocab, dtype, 1)
    assert (xt.workspace(K.sample(8, vocab, DTYPES[dtype])) > 0) == (vocab == 70000)
    u = [0.0, -1.0, 1.0, 2.0, nan, inf, -inf, float(np.nextafter(np.float32(1), np.float32(0)))]
    for options in ({}, {"top_k": 40}, {"top_k": 9000}, {"top_p": 0.5}, {"min_p": 0.01}, {"top_k": 9000, "top_p": 0.9, "min_p": 0.001}):
        check(x, u, dtype, **options)
    check(x, uniforms(8, 2), dtype, temperature=[0.0, -1.0, nan, inf, 1e-45, 3e38, -inf, 1e-3])
    check(x, uniforms(8, 3), dtype, top_p=[0.0, -1.0, 1.0, 2.0, nan, inf, -inf, 1e-30])
    check(x, uniforms(8, 4), dtype, min_p=[0.0, -1.0, 1.0, 2.0, nan, inf, -inf, 1e-30])
    check(x, uniforms(8, 5), dtype, top_k=[0, -1, 1, vocab, vocab + 1, 2**31 - 1, -2**31, vocab - 1])


@pytest.mark.parametrize("vocab", [9, 700, 3000, 40000, 70000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_only_the_largest_with_cuts(vocab, dtype):
    """Temperatures that leave the largest logits alone, and infinities, under every cut."""
    x = logits(6, vocab, dtype, vocab)
    x[1, [vocab // 3, vocab - 1]] = 50.0
    x[2, [0, vocab // 2]] = float("inf")
    x[3, :] = float("inf")
    x[4, :] = -2.0
    x[5, 1:] = float("-inf")
    heat = [0.0, 0.0, 1.0, 2.0, -1.0, 0.5]
    for options in ({"top_k": 50}, {"top_k": 1000, "min_p": 0.5}, {"top_p": 0.5}, {"top_k": 3, "top_p": 0.5, "min_p": 1.0}):
        for seed in (1, 2):
            check(x, uniforms(6, seed), dtype, temperature=heat, **options)


def test_every_token_can_be_drawn():
    """u at and next to each border of a few exact weights."""
    import torch

    x = torch.zeros(1, 8)
    for i in range(8):
        for u, token in ((i / 8, i), (float(np.nextafter(np.float32((i + 1) / 8), np.float32(0))), i)):
            assert run(x, u, "f32") == [token]


@pytest.mark.parametrize("skip", [0, 1, 3])
@pytest.mark.parametrize("dtype,vocab", [("f32", 3001), ("bf16", 3001), ("bf16", 9001), ("f32", 40001)], ids=str)
def test_blocks_pitches_and_alignment(dtype, vocab, skip):
    """Rows of a wider array from any element on, parameters in a column of theirs; what lies
    beside the tokens stays."""
    import torch

    rows, wide, trow = 8, 3 * vocab, 2

    @xt.kernel
    def sample_kernel(x, u, p, y):
        b = xt.bid(0)
        t = xt.load(x, index=(b, 1), shape=(trow, vocab))
        xt.store(y, index=(b, 2), tile=xt.sample(t, xt.load(u, index=(b, 1), shape=(trow, 1)),
                                                 top_p=xt.load(p, index=(b, 0), shape=(trow, 1))))

    m = xt.convert(sample_kernel, args=(xt.Array(shape=(rows, wide), dtype=DTYPES[dtype]),
                                        xt.Array(shape=(rows, 3), dtype=xt.float32),
                                        xt.Array(shape=(rows, 2), dtype=xt.float32),
                                        xt.Array(shape=(rows, 4), dtype=xt.int32)), grid=(rows // trow, 1, 1))
    x = logits(rows, wide, dtype, 6)
    flat = torch.zeros(rows * wide + 8, dtype=x.dtype, device="cuda")
    dx = flat[skip:skip + rows * wide].view(rows, wide)
    dx.copy_(x)
    u, p = torch.rand(rows, 3), torch.full((rows, 2), 0.8)
    y = torch.full((rows, 4), -7, dtype=torch.int32, device="cuda")
    xt.launch(m, dx, u.cuda(), p.cuda(), y)
    part = x[:, vocab:2 * vocab]
    w = [ref.sample(part[r].double().numpy(), float(u[r, 1]), top_p=float(p[r, 0])) for r in range(rows)]
    assert y[:, 2].tolist() == w
    assert bool((y[:, [0, 1, 3]] == -7).all())


def test_streams_and_graphs():
    """Two programs at once, and one captured and replayed."""
    import torch

    rows, vocab = 4, 40000
    m = K.sample(rows, vocab, top_p=True)
    p = torch.full((rows, 1), 0.9, device="cuda")
    x, u = logits(rows, vocab, "f32", 1), torch.tensor(uniforms(rows, 1)).view(rows, 1)
    jobs = []
    for i in range(2):
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            dx, du = (x + i).roll(i, 1).cuda(), u.cuda()
            y = torch.empty(rows, 1, dtype=torch.int32, device="cuda")
            for _ in range(3):
                xt.launch(m, dx, du, p, y)
            jobs.append((stream, dx, y))
    for stream, dx, y in jobs:
        stream.synchronize()
        assert y.view(-1).tolist() == want(dx.cpu(), u.view(-1).tolist(), top_p=0.9)
    dx, du = x.cuda(), u.cuda()
    y = torch.empty(rows, 1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        xt.launch(m, dx, du, p, y)
    for seed in range(3):
        new, nu = logits(rows, vocab, "f32", 10 + seed), torch.tensor(uniforms(rows, seed)).view(rows, 1)
        dx.copy_(new)
        du.copy_(nu)
        graph.replay()
        torch.cuda.synchronize()
        assert y.view(-1).tolist() == want(new, nu.view(-1).tolist(), top_p=0.9)


@pytest.mark.parametrize("rows,vocab", [(7, 70000), (3, 700)], ids=["sliced", "alone"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("end", ["hidden", "far"])
def test_top_k_past_the_last_weight(rows, vocab, dtype, end):
    """Top-k reaches into tokens without a weight, in the bin of the last one that it takes; with
    uniforms of every kind and the other cuts."""
    inf, nan = float("inf"), float("nan")
    assert bool(xt.workspace(K.sample(rows, vocab, DTYPES[dtype], top_k=True))) == (vocab > 10000)
    x = logits(rows, vocab, dtype, vocab, 1.0)
    few = vocab // 70
    x[:, ::70] = -inf if end == "hidden" else -2000.0  # whose weight is 0 in 64 bits too
    below = float(np.nextafter(np.float32(1), np.float32(0)))
    u = [1.0, 2.0, inf, nan, below, 0.0, 0.5][:rows]
    for k in (vocab - few // 2, vocab - 1, vocab - few, vocab - few + 1):
        for options in ({}, {"top_p": 0.9}, {"min_p": 0.001}, {"top_p": below, "min_p": 1e-30}):
            check(x, u, dtype, top_k=k, **options)
            check(x, u[::-1], dtype, top_k=k, **options)


@pytest.mark.parametrize("vocab,shift", [(9, 50), (2048, 50), (2049, 49), (1 << 17, 44), ((1 << 17) + 1, 43), (1 << 22, 39)])
def test_units_of_weights(vocab, shift):
    """A tail of one unit each, rounded up from 2**-0.99 of one, counts; of 2**-1.01 nothing does."""
    import torch

    below = float(np.nextafter(np.float32(1), np.float32(0)))
    for octaves, unit in ((shift + 0.99, 1), (shift + 1.01, 0)):
        x = torch.full((4, vocab), -octaves * np.log(2.0))
        x[:, 0] = 0.0
        u = [1.0, below, 0.5, 0.0]
        total = 2**shift + unit * (vocab - 1)
        # token t > 0 ends at 2**shift + t units; the first that exceeds u of them all, in whole numbers
        past = [total - 1 if v >= 1 else int(v * 2**24) * total // 2**24 for v in u]
        tokens = [max(0, p + 1 - 2**shift) for p in past]
        assert run(x, u, "f32") == tokens
        assert run(x, u, "f32", without_workspace=True) == tokens


def time_of(program, bufs):
    """Microseconds of a launch, from replays of a graph of ten."""
    import torch

    xt.launch(program, *bufs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(10):
            xt.launch(program, *bufs)
    times = []
    for _ in range(7):
        first, last = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        first.record()
        graph.replay()
        last.record()
        torch.cuda.synchronize()
        times.append(first.elapsed_time(last) * 100)
    return sorted(times)[3]


def weightless_rows(rows, vocab, dtype, kind):
    """Rows of which few tokens have a weight: (logits, temperature)."""
    x = logits(rows, vocab, dtype, vocab)
    if kind == "masked":
        x[:, 30:] = -float("inf")
    return x, {"masked": 1.0, "greedy": 0.0, "cold": 0.02}[kind]


@pytest.mark.parametrize("kind", ["masked", "greedy", "cold"])
@pytest.mark.parametrize("rows,vocab,dtype", [(2, 131072, "f32"), (3, 20000, "bf16")])
def test_top_k_of_more_than_have_a_weight(rows, vocab, dtype, kind):
    """The same tokens as without top-k, in little more time: the kernel need not tell tokens
    without a weight apart."""
    x, heat = weightless_rows(rows, vocab, dtype, kind)
    u = uniforms(rows, 3)
    for options in ({}, {"top_p": 0.9, "min_p": 0.01}):
        for k in (50, 256, 257, 1000):
            check(x, u, dtype, temperature=heat, top_k=k, **options)
            assert run(x, u, dtype, temperature=heat, top_k=k, **options) == run(x, u, dtype, temperature=heat, **options)


@pytest.mark.parametrize("k", [50, 1000])
@pytest.mark.parametrize("kind", ["masked", "greedy", "cold"])
@pytest.mark.parametrize("rows,vocab,dtype", [(2, 131072, "f32"), (3, 20000, "bf16")])
def test_time_of_top_k_of_more_than_have_a_weight(rows, vocab, dtype, kind, k):
    """Less than four times that without top-k."""
    import torch

    x, heat = weightless_rows(rows, vocab, dtype, kind)
    y = torch.empty(rows, 1, dtype=torch.int32, device="cuda")
    bufs = [x.cuda(), column(uniforms(rows, 3), rows, torch.float32), column(heat, rows, torch.float32)]
    without = time_of(K.sample(rows, vocab, DTYPES[dtype], temperature=True), [*bufs, y])
    with_it = time_of(K.sample(rows, vocab, DTYPES[dtype], temperature=True, top_k=True), [*bufs, column(k, rows, torch.int32), y])
    assert with_it < 4 * without, (with_it, without)


@pytest.mark.parametrize("vocab", [9, 66001])
def test_distances_past_the_range(vocab):
    """Logits farther apart than float's largest, whose weights are not 0 at the temperatures above
    it: 2^-3 for the farthest at 3.3e38.  At 1e36 those of the third token on are below 2^-400,
    which moves no sum: a uniform of 1, held just below it, gives the last one before them."""
    x = logits(4, vocab, "f32", vocab).abs().neg() * 1e37
    x[:, 0], x[:, 1], x[:, 2:4] = 3.3e38, 3.2e38, -3.3e38
    if vocab > 9:
        x[:, 5000:] = -float("inf")
    below = np.nextafter(1.0, 0.0)
    for heat in (3.3e38, 1e38, 1e36):
        for k in (2, 4, 9, 200, 1000):
            for options in ({}, {"top_p": 0.9}, {"min_p": 0.2}):
                asked = {"temperature": heat, "top_k": min(k, vocab), **options}
                for u in ([0.0, 0.5, 0.9, 1.0], [0.3, 0.99, 0.75, 0.125]):
                    w = [ref.sample(x[r].double().numpy(), min(np.float64(np.float32(u[r])), below),
                                    **{n: np.float32(v) if n != "top_k" else v for n, v in asked.items()}) for r in range(4)]
                    assert run(x, u, "f32", **asked) == w
                    assert run(x, u, "f32", without_workspace=True, **asked) == w
