"""Attention of a tree of drafted tokens on the GPU, against the definition in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest

import xtile_amd as xt
from xtile_amd import kernels as K

from . import answers_ref as ref
from .operators_ref import assert_within

pytestmark = pytest.mark.gpu


def random_parents(rng, nq, reach=8):
    return [int(max(-1, t - 1 - rng.integers(0, reach))) for t in range(nq)]


def run(batch, hk, g, nq, nk, d, parents, start=None, length=None, dtype="bf16", cap=None, window=None, slopes=False,
        token_major=False, seed=0, spoil=None, without_workspace=False, scale=None):
    """parents, start, length: of each sequence.  spoil(k, v): changes the cache before the launch."""
    import torch

    t = torch.bfloat16 if dtype == "bf16" else torch.float16
    gen = torch.Generator().manual_seed(seed)
    h = hk * g
    q = (2 * torch.randn(batch, h, nq, d, generator=gen)).to(t)
    k, v = (torch.randn(batch, hk, nk, d, generator=gen).to(t) for _ in range(2))
    if spoil:
        spoil(k, v)
    sl = torch.exp2(-8.0 * torch.arange(1, h + 1) / h).view(hk, g) if slopes else None
    m = K.masked_attention(batch, hk, g, nq, nk, d, dtype=xt.bfloat16 if dtype == "bf16" else xt.float16, cap=cap,
                           window=window, slopes=slopes, start=start is not None, length=length is not None,
                           parents=True, token_major=token_major, scale=scale)
    print(f"[gpu] {xt.plan(m)['kernel']}", flush=True)

    def laid_out(x):
        return (x.transpose(1, 2).reshape(x.shape[0], x.shape[2], -1) if token_major else x).contiguous().cuda()

    def ints(x):
        return torch.tensor(x, dtype=torch.int32).view(batch, -1).cuda()

    bufs = [laid_out(q), laid_out(k), laid_out(v)]
    if slopes:
        bufs.append(sl.cuda())
    bufs += [ints(x) for x in (start, length, parents) if x is not None]
    o = torch.full_like(bufs[0], 7.0)
    bufs.append(o)
    if without_workspace:
        from xtile_amd import _xtile

        _xtile.launch(m, None, [b.data_ptr() for b in bufs], [b.numel() * b.element_size() for b in bufs],
                      torch.cuda.current_stream().cuda_stream)
    else:
        xt.launch(m, *bufs)
    got = o.cpu()
    if token_major:
        got = got.view(batch, nq, h, d).transpose(1, 2)
    seen = [ref.tree_seen(parents[i], start[i] if start else 0, min(length[i], nk) if length else nk, nk, window)
            for i in range(batch)]
    sees, distance = (torch.from_numpy(np.stack([s[e] for s in seen])) for e in (0, 1))
    want, far = ref.attend_seen(q, k, v, d**-0.5 if scale is None else scale, sees, distance, cap, sl)
    assert_within(got, want, far, xt.plan(m)["kernel"])
    return got, sees


@pytest.mark.parametrize("nq", [1, 2, 5, 16, 31, 33, 63, 64])
@pytest.mark.parametrize("g,nk", [(1, 200), (4, 700)])
def test_tokens(nq, g, nk):
    rng = np.random.default_rng(nq)
    parents = [random_parents(rng, nq), random_parents(rng, nq, 2)]
    run(2, 2, g, nq, nk, 64, parents, start=[nk - nq, nk // 3], length=[nk, nk // 3 + nq])


@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("nq,g", [(7, 4), (24, 8)])
def test_heads(d, dtype, nq, g):
    rng = np.random.default_rng(d)
    run(1, 2, g, nq, 333, d, [random_parents(rng, nq)], start=[300], length=[300 + nq], dtype=dtype)


SHAPES = {"chain": [t - 1 for t in range(40)], "star": [-1] * 40, "of one": [0 if t else -1 for t in range(40)],
          "binary": [(t - 1) // 2 if t else -1 for t in range(40)],
          # parents that are none: the token itself, one behind it, far away
          "odd": [t if t % 5 == 0 else t + 3 if t % 5 == 1 else -7 if t % 5 == 2 else 2**31 - 1 if t % 5 == 3 else t - 2
                  for t in range(40)]}


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("options", [{}, {"window": 5}, {"window": 1}, {"slopes": True}, {"window": 70, "slopes": True, "cap": 30.0},
                                     {"cap": 3000.0}],
                         ids=lambda o: "-".join(o) or "none")
@pytest.mark.parametrize("g", [1, 5])
def test_shapes(shape, options, g):
    run(1, 2, g, 40, 300, 64, [SHAPES[shape]], start=[230], length=[270], **options)
    run(1, 2, g, 3, 300, 64, [SHAPES[shape][:3]], start=[129], length=[132], **options)


def test_a_chain_is_a_causal_row():
    """Tokens that follow each other see what causal ones do.  The two take keys in other orders:
    each is within `far` of the formula, so they are within twice that of each other."""
    import torch

    nq, nk, start = 20, 500, 411
    got, _ = run(1, 2, 3, nq, nk, 128, [[t - 1 for t in range(nq)]], start=[start], length=[start + nq], window=100)
    gen = torch.Generator().manual_seed(0)
    q = (2 * torch.randn(1, 6, nq, 128, generator=gen)).bfloat16().cuda()
    k, v = (torch.randn(1, 2, nk, 128, generator=gen).bfloat16().cuda() for _ in range(2))
    o = torch.empty_like(q)
    at = torch.tensor([[start]], dtype=torch.int32, device="cuda")
    xt.launch(K.masked_attention(1, 2, 3, nq, nk, 128, causal=True, window=100, start=True, length=True), q, k, v, at,
              at + nq, o)
    sees, distance = (torch.from_numpy(x)[None] for x in ref.tree_seen([t - 1 for t in range(nq)], start, start + nq, nk, 100))
    want, far = ref.attend_seen(q.cpu(), k.cpu(), v.cpu(), 128**-0.5, sees, distance, None, None)
    assert_within(o.cpu(), want, far)
    assert bool(((got.double() - o.cpu().double()).abs() <= 2 * far).all())


@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("nq,g,nk,start", [(11, 3, 64, 50), (64, 1, 65, 0), (7, 5, 1000, 700), (16, 4, 577, 561)])
def test_33_to_64_rows(d, nq, g, nk, start):
    """Tiles in turn, of which the last is part of one, in the wave's half of them or not."""
    rng = np.random.default_rng(d + nk)
    parents = [random_parents(rng, nq), random_parents(rng, nq, 2)]
    run(2, 1, g, nq, nk, d, parents, start=[start, 3], length=[start + nq, nk], dtype="f16" if d % 64 else "bf16")
    run(2, 1, g, nq, nk, d, parents, start=[start, 31], length=[start + nq, 31 + nq], window=40, token_major=True)


@pytest.mark.parametrize("start,length", [
    (0, 64), (0, 10), (0, 0), (5, 5), (64, 64), (100, 50), (-3, 9), (-64, 64), (-100, 100), (90, 100), (99, 100), (100, 100),
    (2**31 - 1, 100), (-2**31, 100), (2**30, 2**31 - 1), (30, -5), (30, 2**31 - 1)])
@pytest.mark.parametrize("window", [None, 3, 2**31 - 1])
def test_places(start, length, window):
    """Trees that begin before the cache, reach past it or past the length, or lie far from it."""
    rng = np.random.default_rng(1)
    for g in (1, 4):
        got, sees = run(1, 1, g, 12, 100, 64, [random_parents(rng, 12, 3)], start=[start], length=[length], window=window)
        blind = ~sees.any(dim=2)[0]
        assert bool((got[0][:, blind] == 0).all())


def test_without_start_and_length():
    rng = np.random.default_rng(2)
    run(2, 2, 2, 9, 40, 64, [random_parents(rng, 9), random_parents(rng, 9)])
    run(2, 2, 2, 9, 40, 64, [random_parents(rng, 9), random_parents(rng, 9)], start=[20, 3])


@pytest.mark.parametrize("batch,hk,g,nq,nk,d,options", [
    (1, 8, 8, 64, 20000, 128, {"cap": 50.0, "dtype": "f16"}), (1, 2, 4, 7, 30000, 64, {"slopes": True}),
    (3, 4, 4, 32, 5000, 128, {}), (1, 1, 1, 13, 9000, 256, {"window": 1000}), (2, 1, 8, 64, 4000, 96, {"token_major": True})])
def test_split_caches(batch, hk, g, nq, nk, d, options):
    """Long caches, with the workspace and without."""
    rng = np.random.default_rng(nk)
    parents = [random_parents(rng, nq) for _ in range(batch)]
    start = [nk - nq - i * nk // 5 for i in range(batch)]
    for without in (False, True):
        run(batch, hk, g, nq, nk, d, parents, start=start, length=[s + nq for s in start], without_workspace=without, **options)


@pytest.mark.parametrize("nq,g", [(4, 2), (40, 4)])
def test_hidden_keys_and_values_of_any_kind(nq, g):
    """Infinities and NaN in what no token sees, and in drafted tokens that only some see."""
    import torch

    start, nk = 150, 260
    parents = [[-1 if t < 2 else t - 2 for t in range(nq)]]  # two chains

    def spoil(k, v):
        k[:, :, start + nq:] = float("nan")
        v[:, :, start + nq:] = float("inf")
        v[:, :, start + 1] = float("nan")  # of the second chain

    got, _ = run(1, 2, g, nq, nk, 64, parents, start=[start], length=[nk], spoil=spoil)
    nan = torch.isnan(got)
    assert bool(nan[:, :, 1::2].all()) and not bool(nan[:, :, 0::2].any())


def test_result_over_its_query():
    import torch

    nq, nk = 10, 128
    rng = np.random.default_rng(3)
    parents = random_parents(rng, nq)
    gen = torch.Generator().manual_seed(1)
    q = torch.randn(1, 2, nq, 64, generator=gen).bfloat16().cuda()
    k, v = (torch.randn(1, 1, nk, 64, generator=gen).bfloat16().cuda() for _ in range(2))
    at = torch.tensor([[100]], dtype=torch.int32, device="cuda")
    pa = torch.tensor([parents], dtype=torch.int32, device="cuda")
    m = K.masked_attention(1, 1, 2, nq, nk, 64, start=True, parents=True)
    o = torch.empty_like(q)
    xt.launch(m, q, k, v, at, pa, o)
    xt.launch(m, q, k, v, at, pa, q)
    assert torch.equal(q, o)
    with pytest.raises(ValueError, match="meets buffer 4"):
        over = torch.empty(q.numel() // 2, dtype=torch.int32, device="cuda")
        xt.launch(m, q, k, v, at, over[:nq].view(1, nq), over.view(torch.bfloat16).view(q.shape))


def test_graph_replays():
    """A captured launch takes the tree that its buffers hold at each replay."""
    import torch

    nq, nk, start = 16, 6000, 5000
    gen = torch.Generator().manual_seed(1)
    q = torch.randn(1, 8, nq, 128, generator=gen).bfloat16().cuda()
    k, v = (torch.randn(1, 2, nk, 128, generator=gen).bfloat16().cuda() for _ in range(2))
    at = torch.tensor([[start]], dtype=torch.int32, device="cuda")
    pa = torch.full((1, nq), -1, dtype=torch.int32, device="cuda")
    m = K.masked_attention(1, 2, 4, nq, nk, 128, start=True, parents=True)
    o, eager = torch.empty_like(q), torch.empty_like(q)
    xt.launch(m, q, k, v, at, pa, o)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        xt.launch(m, q, k, v, at, pa, o)
    seen = []
    for seed in range(3):
        pa.copy_(torch.tensor([random_parents(np.random.default_rng(seed), nq)], dtype=torch.int32))
        at.fill_(start + seed)
        graph.replay()
        torch.cuda.synchronize()
        xt.launch(m, q, k, v, at, pa, eager)
        assert torch.equal(o, eager)
        seen.append(o.clone())
    assert not torch.equal(seen[0], seen[1])
