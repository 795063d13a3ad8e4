"""Calls of rms_norm, matmul_q4 and attend at the edges of what they take, as far as no GPU is needed."""

from __future__ import annotations

import pytest

import xtile_amd as xt
from xtile_amd import _xtile
from xtile_amd import kernels as K


def launch_at(m, *addresses):
    """Enqueues `m` over buffers at addresses that are none of any memory: for calls
    that are refused before anything is launched."""
    args = xt.signature(m)["args"]
    sizes = []
    for a in args:
        n = {"f32": 4, "i32": 4, "f16": 2, "bf16": 2, "i8": 1}[a["dtype"]]
        for e in a["shape"]:
            n *= e
        sizes.append(n)
    _xtile.launch(m, None, list(addresses), sizes, 0)


def apart(n):
    return [(i + 1) << 44 for i in range(n)]


@pytest.mark.parametrize("rows,cols", [(1 << 26, 4), (1 << 26, 1), ((1 << 26) - 1, 8), ((1 << 26) - 3, 1000), (1 << 24, 1025),
                                       (1 << 22, 8193), (1 << 22, 40001)])
def test_rms_norm_refuses_rows_beyond_one_launch(rows, cols):
    """2^32 work-items or more, counted as they are launched: 64, 256 or 1024 threads a
    row, rows of 8 to 1024 values four to a workgroup."""
    m = K.rms_norm(rows, cols, xt.float32, residual=False)
    with pytest.raises(ValueError, match="exceed one launch"):
        launch_at(m, *apart(3))


def traced(body, *arrays, grid=(1, 1, 1)):
    return xt.convert(K._named("traced", lambda a: body(*a), len(arrays)), args=arrays, grid=grid)


@pytest.mark.parametrize("grid", [(2, 1, 1), (1, 2, 1), (1, 1, 2)])
def test_results_over_inputs_that_several_blocks_read_are_refused(grid):
    """Every Block has the same tile: one would read what another has stored."""
    x, g = xt.Array((4, 64), xt.float32), xt.Array((1, 64), xt.float32)

    def norm(x, g, y):
        xt.store(y, index=(0, 0), tile=xt.rms_norm(xt.load(x, index=(0, 0), shape=(4, 64)), xt.load(g, index=(0, 0), shape=(1, 64))))

    m = traced(norm, x, g, x, grid=grid)
    a, b, _ = apart(3)
    with pytest.raises(ValueError, match="meets buffer 0"):
        launch_at(m, a, b, a)
    h = xt.Array((4, 64), xt.float16)

    def attention(q, k, v, o):
        xt.store(o, index=(0, 0), tile=xt.attend(*(xt.load(t, index=(0, 0), shape=(4, 64)) for t in (q, k, v)), scale=1.0))

    m = traced(attention, h, h, h, h, grid=grid)
    a, b, c, _ = apart(4)
    with pytest.raises(ValueError, match="meets buffer 0"):
        launch_at(m, a, b, c, a)


@pytest.mark.parametrize("which", ["q", "k", "v", "o"])
def test_attend_refuses_rows_whose_elements_lie_apart(which):
    """A tile of one of three interleaved arrays, reshaped to rows."""
    rows, apart3 = xt.Array((40, 64), xt.float16), xt.Array((40, 64, 3), xt.float16)

    def body(q, k, v, o):
        def tile(name, a):
            if name != which:
                return xt.load(a, index=(0, 0), shape=(40, 64))
            return xt.reshape(xt.load(a, index=(0, 0, 1), shape=(40, 64, 1)), shape=(40, 64))

        y = xt.attend(tile("q", q), tile("k", k), tile("v", v), scale=1.0)
        if which == "o":
            xt.store(o, index=(0, 0, 1), tile=xt.reshape(y, shape=(40, 64, 1)))
        else:
            xt.store(o, index=(0, 0), tile=y)

    m = traced(body, *(apart3 if name == which else rows for name in "qkvo"))
    with pytest.raises(NotImplementedError, match="side by side"):
        xt.plan(m)


def test_attend_takes_rows_of_an_array_whose_last_dim_is_one():
    def body(q, k, v, o):
        q, k, v = (xt.reshape(xt.load(t, index=(0, 0, 0), shape=(40, 64, 1)), shape=(40, 64)) for t in (q, k, v))
        xt.store(o, index=(0, 0, 0), tile=xt.reshape(xt.attend(q, k, v, scale=1.0), shape=(40, 64, 1)))

    a = xt.Array((40, 64, 1), xt.float16)
    assert "attend f16 heads=1 rows=40 keys=40 d=64" in xt.plan(traced(body, a, a, a, a))["kernel"]
