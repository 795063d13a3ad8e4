"""Microscaled products, attention of drafted trees and sampling together on the GPU, as a decode
step of drafted tokens runs them; and buffers past 32 bits."""

from __future__ import annotations

import numpy as np
import pytest

import xtile_amd as xt
from xtile_amd import kernels as K

from . import answers_ref as ref
from . import operators_ref

pytestmark = pytest.mark.gpu

WIDTH, KV_HEADS, GROUP, D, TOKENS, CACHE, VOCAB = 256, 2, 3, 64, 12, 5000, 70001
HEADS = KV_HEADS * GROUP


def rand(shape, seed, dtype="bfloat16"):
    import torch

    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(getattr(torch, dtype)).cuda()


def int8(shape):
    import torch

    return torch.zeros(*shape, dtype=torch.int8, device="cuda")


def of_mx4(q, s):
    """The float64 values of rows on the GPU."""
    import torch

    q, s = (t.cpu().view(torch.uint8).numpy() for t in (q, s))
    return ref.values(ref.unpack(q), s)


class Linear:
    """A weight matrix in microscaled 4-bit rows and the buffers of a product with it."""

    def __init__(self, n, k, seed, out="bfloat16"):
        import torch

        self.w, self.ws = int8((n, k // 2)), int8((n, k // 32))
        xt.launch(K.quantize_mx4(n, k), rand((n, k), seed) / k**0.5, self.w, self.ws)
        self.x, self.xs = int8((TOKENS, k // 2)), int8((TOKENS, k // 32))
        self.y = torch.zeros(TOKENS, n, dtype=getattr(torch, out), device="cuda")
        self.rows = xt.compile(K.quantize_mx4(TOKENS, k))
        self.product = xt.compile(K.matmul_mx4(TOKENS, n, k, out=getattr(xt, out)))

    def __call__(self, x):
        self.given = x
        xt.launch(self.rows, x, self.x, self.xs)
        xt.launch(self.product, self.x, self.xs, self.w, self.ws, self.y)
        return self.y

    def check(self):
        code, byte = ref.quantize_mx4(self.given.cpu().double().numpy())
        x = of_mx4(self.x, self.xs)
        assert np.array_equal(x, ref.values(code, byte))
        want, far = ref.matmul_mx4(x, of_mx4(self.w, self.ws))
        got = self.y.cpu().double().numpy()
        far = far + operators_ref.half_step(self.y) * (np.abs(want) + far)
        assert bool((np.abs(got - want) <= far).all())


class Step:
    """Norm, three 4-bit products, attention of the tree, the product back, the next norm, the
    logits and a token each; all buffers kept."""

    def __init__(self, seed):
        import torch

        self.x = rand((TOKENS, WIDTH), seed)
        self.gamma = rand((1, WIDTH), seed + 1)
        self.h, self.n1, self.n2 = (torch.zeros_like(self.x) for _ in range(3))
        self.to_q, self.to_k, self.to_v = (Linear(n * D, WIDTH, seed + 2 + i) for i, n in enumerate((HEADS, KV_HEADS, KV_HEADS)))
        self.back = Linear(WIDTH, HEADS * D, seed + 5)
        self.to_logits = Linear(VOCAB, WIDTH, seed + 6, "float32")
        self.k, self.v = rand((1, CACHE, KV_HEADS * D), seed + 7), rand((1, CACHE, KV_HEADS * D), seed + 8)
        self.start = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
        self.length = torch.zeros_like(self.start)
        self.parents = torch.zeros(1, TOKENS, dtype=torch.int32, device="cuda")
        self.a = torch.zeros(1, TOKENS, HEADS * D, dtype=torch.bfloat16, device="cuda")
        self.u = torch.zeros(TOKENS, 1, device="cuda")
        self.top_p = torch.full((TOKENS, 1), 0.9, device="cuda")
        self.heat = torch.full((TOKENS, 1), 0.3, device="cuda")
        self.tokens = torch.full((TOKENS, 1), -7, dtype=torch.int32, device="cuda")
        self.norm = xt.compile(K.rms_norm(TOKENS, WIDTH, residual=False))
        self.add_norm = xt.compile(K.rms_norm(TOKENS, WIDTH))
        self.attend = xt.compile(K.masked_attention(1, KV_HEADS, GROUP, TOKENS, CACHE, D, start=True, length=True, parents=True,
                                                    token_major=True))
        self.sample = xt.compile(K.sample(TOKENS, VOCAB, temperature=True, top_p=True))
        assert xt.workspace(self.attend) and xt.workspace(self.sample)

    def set(self, seed):
        """Other drafted tokens, behind as many as the seed says."""
        import torch

        rng = np.random.default_rng(seed)
        self.x.copy_(rand((TOKENS, WIDTH), 100 + seed))
        self.start.fill_(4000 + seed)
        self.length.fill_(4000 + seed + TOKENS)
        tree = [int(max(-1, t - 1 - rng.integers(0, 4))) for t in range(TOKENS)]
        self.parents.copy_(torch.tensor([tree], dtype=torch.int32))
        self.u.copy_(torch.from_numpy(rng.random((TOKENS, 1)).astype(np.float32)))
        self.at = torch.arange(4000 + seed, 4000 + seed + TOKENS, device="cuda")
        return tree

    def run(self, at):
        xt.launch(self.norm, self.x, self.gamma, self.n1)
        q, k, v = self.to_q(self.n1), self.to_k(self.n1), self.to_v(self.n1)
        self.k[0].index_copy_(0, at, k)
        self.v[0].index_copy_(0, at, v)
        xt.launch(self.attend, q.view(1, TOKENS, -1), self.k, self.v, self.start, self.length, self.parents, self.a)
        o = self.back(self.a.view(TOKENS, -1))
        xt.launch(self.add_norm, o, self.x, self.gamma, self.h, self.n2)
        xt.launch(self.sample, self.to_logits(self.n2), self.u, self.heat, self.top_p, self.tokens)

    def check(self, tree):
        """Each result against 64 bits of what it was made from."""
        import torch

        for linear in (self.to_q, self.to_k, self.to_v, self.back, self.to_logits):
            linear.check()

        def heads(t, n):
            return t.view(1, -1, n, D).transpose(1, 2).cpu()

        start = int(self.start)
        sees, distance = (torch.from_numpy(m)[None] for m in ref.tree_seen(tree, start, start + TOKENS, CACHE))
        want, far = ref.attend_seen(heads(self.to_q.y, HEADS), heads(self.k, KV_HEADS), heads(self.v, KV_HEADS), D**-0.5, sees,
                                    distance, None, None)
        operators_ref.assert_within(heads(self.a, HEADS), want, far)
        logits = self.to_logits.y.cpu().double().numpy()
        want = [ref.sample(logits[t], np.float32(self.u[t, 0].item()), temperature=np.float32(0.3), top_p=np.float32(0.9))
                for t in range(TOKENS)]
        assert self.tokens.view(-1).tolist() == want


def test_a_step_of_drafted_tokens():
    step = Step(1)
    for seed in (0, 1):
        tree = step.set(seed)
        step.run(step.at)
        step.check(tree)


def test_two_captured_steps():
    """Each with its own workspaces, replayed together with other work between, on two streams."""
    import torch

    steps = [Step(1), Step(20)]
    at = [s.set(0) and s.at.clone() for s in steps]
    for s, a in zip(steps, at):
        s.run(a)
    torch.cuda.synchronize()
    graphs = []
    for s, a in zip(steps, at):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.run(a)
        graphs.append(g)
    side = torch.cuda.Stream()
    for seed in (3, 4, 5):
        trees = []
        for s, a in zip(steps, at):
            trees.append(s.set(seed))
            a.copy_(s.at)
        scratch = torch.full((1 << 22,), 3.0, device="cuda")  # takes what was freed
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        assert bool((scratch == 3.0).all())
        for s, a, tree in zip(steps, at, trees):
            s.check(tree)
            got = s.tokens.clone()
            s.run(a)
            assert torch.equal(s.tokens, got)


@pytest.mark.parametrize("nq,g", [(5, 3), (9, 5), (40, 4)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_trees_over_keys_of_any_alignment(nq, g, d):
    """Caches that begin two bytes past a multiple of 16."""
    import torch

    nk, start = 700, 600
    parents = [int(max(-1, t - 1 - t % 3)) for t in range(nq)]
    q = rand((1, g, nq, d), 1)
    flat = [rand((nk * d + 8,), 2 + i) for i in range(2)]
    k, v = (f[1 : 1 + nk * d].view(1, 1, nk, d) for f in flat)
    at = torch.tensor([[start]], dtype=torch.int32, device="cuda")
    o = torch.zeros_like(q)
    p = K.masked_attention(1, 1, g, nq, nk, d, start=True, length=True, parents=True)
    print(f"[gpu] {xt.plan(p)['kernel']}", flush=True)
    xt.launch(p, q, k, v, at, at + nq, torch.tensor([parents], dtype=torch.int32, device="cuda"), o)
    sees, distance = (torch.from_numpy(m)[None] for m in ref.tree_seen(parents, start, start + nq, nk))
    want, far = ref.attend_seen(q.cpu(), k.cpu(), v.cpu(), d**-0.5, sees, distance, None, None)
    operators_ref.assert_within(o.cpu(), want, far)


# -- offsets past 32 bits -------------------------------------------------------------------


def test_rows_past_32_bits():
    """The last rows of more than 4 GiB, against the same on their own; and back."""
    import torch

    rows, cols, last = (1 << 16) + 1000, 1 << 15, 8
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-last:] = rand((last, cols), 1)
    q, s = int8((rows, cols // 2)), int8((rows, cols // 32))
    xt.launch(K.quantize_mx4(rows, cols), x, q, s)
    code, byte = ref.quantize_mx4(x[-last:].cpu().double().numpy())
    assert np.array_equal(of_mx4(q[-last:], s[-last:]), ref.values(code, byte))
    assert not bool(q[:-last].any())
    x.fill_(7.0)
    xt.launch(K.dequantize_mx4(rows, cols), q, s, x)
    assert np.array_equal(x[-last:].cpu().double().numpy(), ref.values(code, byte))
    assert not bool(x[:-last].any())


@pytest.mark.parametrize("m,n", [(1, (1 << 20) + 200), (40, (1 << 20) + 200), ((1 << 20) + 200, 130)])
def test_products_past_32_bits(m, n):
    """Rows of more than 4 GiB: the last ones' products."""
    import torch

    k, last = 1 << 13, 40
    rng = np.random.default_rng(1)

    def rows(count):
        q, s = int8((count, k // 2)), torch.full((count, k // 32), 120, dtype=torch.int8, device="cuda")
        few = min(count, last)
        q[-few:] = torch.from_numpy(rng.integers(-128, 128, (few, k // 2)).astype(np.int8)).cuda()
        return q, s

    x, xs = rows(m)
    w, ws = rows(n)
    y = torch.full((m, n), 7.0, dtype=torch.float32, device="cuda")
    p = K.matmul_mx4(m, n, k)
    print(f"[gpu] {xt.plan(p)['kernel']} {m} x {n}", flush=True)
    xt.launch(p, x, xs, w, ws, y)
    want, far = ref.matmul_mx4(of_mx4(x[-last:], xs[-last:]), of_mx4(w[-last:], ws[-last:]))
    assert bool((np.abs(y[-last:, -last:].cpu().double().numpy() - want) <= far).all())
    assert not bool(y[:-last].any()) and not bool(y[:, :-last].any())


def test_a_product_with_a_result_past_32_bits():
    import torch

    m, n, k, last = 70000, 16400, 64, 24
    rng = np.random.default_rng(2)
    x, w = (torch.from_numpy(rng.integers(-128, 128, (r, k // 2)).astype(np.int8)).cuda() for r in (m, n))
    xs, ws = (torch.from_numpy(rng.integers(100, 128, (r, k // 32)).astype(np.int8)).cuda() for r in (m, n))
    y = torch.full((m, n), 7.0, dtype=torch.float32, device="cuda")
    p = K.matmul_mx4(m, n, k)
    print(f"[gpu] {xt.plan(p)['kernel']}", flush=True)
    xt.launch(p, x, xs, w, ws, y)
    for at in (slice(0, last), slice(m // 2, m // 2 + last), slice(m - last, m)):
        for to in (slice(0, last), slice(n - last, n)):
            want, far = ref.matmul_mx4(of_mx4(x[at], xs[at]), of_mx4(w[to], ws[to]))
            assert bool((np.abs(y[at, to].cpu().double().numpy() - want) <= far).all())


def test_a_product_of_more_small_tiles_than_one_launch_has():
    """Larger tiles take it: weights beside 16-byte places, which the largest do not take."""
    import torch

    n, k, last = 1 << 28, 32, 40
    rng = np.random.default_rng(3)
    w = int8((n * k // 2 + 16,))[1 : 1 + n * k // 2].view(n, k // 2)
    ws = torch.full((n, 1), 127, dtype=torch.int8, device="cuda")
    w[-last:] = torch.from_numpy(rng.integers(-128, 128, (last, k // 2)).astype(np.int8)).cuda()
    x, xs = torch.from_numpy(rng.integers(-128, 128, (1, k // 2)).astype(np.int8)).cuda(), ws[:1].clone()
    y = torch.full((1, n), 7.0, dtype=torch.bfloat16, device="cuda")
    print("[gpu] matmul_mx4 1 x 2^28 x 32", flush=True)
    xt.launch(K.matmul_mx4(1, n, k, out=xt.bfloat16), x, xs, w, ws, y)
    want, far = ref.matmul_mx4(of_mx4(x, xs), of_mx4(w[-last:], ws[-last:]))
    assert bool((np.abs(y[:, -last:].cpu().double().numpy() - want) <= far + 2.0**-8 * np.abs(want)).all())
    assert not bool(y[:, :-last].any())


@pytest.mark.parametrize("nq,g", [(2, 1), (8, 5), (40, 4)])
def test_trees_at_the_end_of_keys_past_32_bits(nq, g):
    """Keys of more than 4 GiB: the last ones, against the same on their own."""
    import torch

    nk, d, window = (1 << 25) + 100, 64, 90
    k = torch.zeros(1, 1, nk, d, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    q = rand((1, g, nq, d), 1)
    k[:, :, -300:], v[:, :, -300:] = rand((1, 1, 300, d), 2), rand((1, 1, 300, d), 3)
    tree = [int(max(-1, t - 1 - t % 2)) for t in range(nq)]
    o = torch.zeros_like(q)
    p = K.masked_attention(1, 1, g, nq, nk, d, window=window, start=True, parents=True)
    print(f"[gpu] {xt.plan(p)['kernel']}", flush=True)
    xt.launch(p, q, k, v, torch.tensor([[nk - nq]], dtype=torch.int32, device="cuda"),
              torch.tensor([tree], dtype=torch.int32, device="cuda"), o)
    sees, distance = (torch.from_numpy(m)[None] for m in ref.tree_seen(tree, 300 - nq, 300, 300, window))
    want, far = ref.attend_seen(q.cpu(), k[:, :, -300:].cpu(), v[:, :, -300:].cpu(), d**-0.5, sees, distance, None, None)
    operators_ref.assert_within(o.cpu(), want, far)


def test_logits_past_32_bits():
    """The last row of more than 4 GiB of logits."""
    import torch

    rows, vocab = 1100, 1 << 20
    x = torch.full((rows, vocab), -1.0, device="cuda")
    x[-1] = rand((vocab,), 1, "float32")
    u = torch.full((rows, 1), 0.625, device="cuda")
    top_k = torch.full((rows, 1), 1000, dtype=torch.int32, device="cuda")
    y = torch.full((rows, 1), -7, dtype=torch.int32, device="cuda")
    xt.launch(K.sample(rows, vocab, top_k=True), x, u, top_k, y)
    assert y[:-1].view(-1).tolist() == [625] * (rows - 1)
    assert int(y[-1]) == ref.sample(x[-1].cpu().double().numpy(), np.float32(0.625), top_k=np.int32(1000))
