"""rms_norm, row_scale, quantize, matmul_q4 and attend: text, passes, refusals, plans, weights' layout."""

from __future__ import annotations

import re

import pytest

import xtile_amd as xt
from xtile_amd import kernels as K

PROGRAMS = {
    "norm": lambda: K.rms_norm(6, 100, trow=2),
    "norm_rows8": lambda: K.rms_norm(6, 100, xt.float32, residual=False, quantize=True, eps=0.0, gamma=xt.float16),
    "q4": lambda: K.matmul_q4(3, 70, 96, group=32, out=xt.bfloat16),
    "q4_i8": lambda: K.matmul_q4(3, 70, 96, group=48 * 2, dtype=xt.int8, scales=xt.float32, row_scale=True),
    "attend": lambda: K.masked_attention(2, 3, 2, 5, 77, 64),
    "attend_all": lambda: K.masked_attention(2, 3, 2, 5, 77, 64, dtype=xt.float16, scale=0.1, cap=30.0, causal=True,
                                             window=9, slopes=True, start=True, length=True, prefix=True, docs=True,
                                             token_major=True),
}


@pytest.mark.parametrize("name", PROGRAMS)
def test_text_goes_round(name):
    """The printer writes what the tracer wrote; canonicalize keeps it."""
    m = PROGRAMS[name]()
    text, plan, sig = str(m), xt.plan(m), xt.signature(m)
    again = xt.parse(text)
    xt.canonicalize(again)
    printed = str(again)
    assert xt.plan(again) == plan and xt.signature(again) == sig
    ops = re.findall(r"= (xt\.(?:rms_norm|row_scale|quantize|matmul_q4|attend))\(.*?\)( \{.*?\})? : (.*)", text)
    assert ops and re.findall(r"= (xt\.(?:rms_norm|row_scale|quantize|matmul_q4|attend))\(.*?\)( \{.*?\})? : (.*)",
                              printed) == ops
    assert str(xt.parse(printed)) == printed


def test_serialize_unrolls_them():
    m = xt.xt_serialize(K.rms_norm(3, 64, quantize=True))
    assert str(m).count("xt.rms_norm") == 3 and str(m).count("xt.quantize") == 3


@pytest.mark.parametrize("name,kernel", [
    ("norm", "rms_norm bf16->bf16 residual tile=2x100 grid=(3,1,1)"),
    ("norm_rows8", "rms_norm f32->i8 tile=1x100 grid=(6,1,1)"),
    ("q4", "matmul_q4 bf16->bf16 tile=3x70 k=96 group=32 grid=(1,1,1)"),
    ("q4_i8", "matmul_q4 i8->f32 tile=3x70 k=96 group=96 grid=(1,1,1)"),
    ("attend", "attend bf16 heads=2 rows=5 keys=77 d=64 grid=(3,2,1)"),
    ("attend_all", "attend f16 heads=2 rows=5 keys=77 d=64 cap causal window=9 slopes start length prefix docs "
                   "grid=(3,2,1)"),
])
def test_plans(name, kernel):
    assert xt.plan(PROGRAMS[name]())["kernel"] == kernel


def test_work_of_plans():
    p = xt.plan(K.rms_norm(8, 64, quantize=True))
    assert p["bytes"] == 8 * 64 * (2 + 2 + 2 + 1) + 8 * 4 + 64 * 2
    p = xt.plan(K.matmul_q4(3, 70, 96, group=32))
    assert p["bytes"] == 3 * 96 * 2 + 70 * 48 + 70 * 3 * 2 + 3 * 70 * 4 and p["flops"] == 2 * 3 * 70 * 96
    p = xt.plan(K.masked_attention(2, 3, 2, 5, 77, 64))
    assert p["flops"] == 4 * 64 * 2 * 3 * 2 * 5 * 77
    assert p["bytes"] == 2 * 64 * 2 * 3 * (2 * 2 * 5 + 2 * 77)
    p = xt.plan(K.masked_attention(1, 1, 1, 5, 5, 64, causal=True))
    assert p["flops"] == 4 * 64 * 15


def test_buffers_below_element_alignment_are_refused():
    """Before anything is launched: the addresses are not those of any memory."""
    from xtile_amd import _xtile

    m = K.matmul_q4(1, 64, 64, group=32, dtype=xt.float16, scales=xt.float32)
    sizes = [128, 64 * 32, 64 * 2 * 4, 64 * 4]
    for k, at in ((0, 4097), (2, 4098), (3, 4098)):
        ptrs = [4096] * 4
        ptrs[k] = at
        with pytest.raises(ValueError, match=f"buffer {k} is not aligned"):
            _xtile.launch(m, None, ptrs, sizes, 0)


def test_workspace():
    """Few rows over many keys work in one; the C ABI says how large."""
    assert xt.workspace(K.masked_attention(1, 8, 4, 4096, 4096, 128)) == 0
    assert xt.workspace(K.matmul_q4(1, 64, 64, group=32)) == 0
    assert xt.workspace(K.add(64, 64)) == 0
    m = K.masked_attention(1, 2, 4, 1, 5000, 64, causal=True)
    splits = int(re.search(r"splits=(\d+)", xt.plan(m)["kernel"])[1])
    assert splits > 1 and xt.workspace(m) == 2 * 4 * splits * (64 + 2) * 4
    with pytest.raises(TypeError):
        xt.workspace(object())


def test_pack_q4():
    import torch

    w = torch.randint(-8, 8, (5, 3, 64), dtype=torch.int8)
    p = xt.pack_q4(w)
    assert p.shape == (5, 3, 32) and p.dtype == torch.int8 and torch.equal(xt.unpack_q4(p), w)
    one = xt.pack_q4(torch.arange(-8, 0).view(1, 8))  # weights k - 8, so nibbles k: 0 2 | 4 6 | 1 3 | 5 7
    assert one.view(torch.uint8).tolist() == [[0x20, 0x64, 0x31, 0x75]]
    for bad, error in ((torch.zeros(4, 12, dtype=torch.int8), ValueError), (torch.zeros(8), TypeError),
                       (torch.full((8,), 8), ValueError), (torch.full((8,), -9), ValueError), ([1] * 8, TypeError)):
        with pytest.raises(error):
            xt.pack_q4(bad)
    for bad, error in ((torch.zeros(4, dtype=torch.int32), TypeError), (torch.zeros(6, dtype=torch.int8), ValueError)):
        with pytest.raises(error):
            xt.unpack_q4(bad)
    assert xt.pack_q4(torch.zeros(0, 8, dtype=torch.int8)).shape == (0, 4)


def trace(body, *arrays):
    return xt.convert(K._named("traced", lambda a: body(*a), len(arrays)), args=arrays, grid=(1, 1, 1))


def tile(a):
    return xt.load(a, index=(0,) * a.array.ndim, shape=a.array.shape)


F, H, B, I8, I32 = xt.float32, xt.float16, xt.bfloat16, xt.int8, xt.int32


@pytest.mark.parametrize("error,text,body,arrays", [
    (ValueError, "rank-2", lambda x, g: xt.rms_norm(tile(x), tile(g)), [((2, 3, 4), F), ((1, 4), F)]),
    (ValueError, "gamma", lambda x, g: xt.rms_norm(tile(x), tile(g)), [((2, 4), F), ((1, 5), F)]),
    (TypeError, "requires", lambda x, g: xt.rms_norm(tile(x), tile(g)), [((2, 4), I8), ((1, 4), F)]),
    (TypeError, "result", lambda x, g: xt.rms_norm(tile(x), tile(g), dtype=I8), [((2, 4), F), ((1, 4), F)]),
    (ValueError, "eps", lambda x, g: xt.rms_norm(tile(x), tile(g), eps=-1.0), [((2, 4), F), ((1, 4), F)]),
    (ValueError, "eps", lambda x, g: xt.rms_norm(tile(x), tile(g), eps=float("nan")), [((2, 4), F), ((1, 4), F)]),
    (TypeError, "eps", lambda x, g: xt.rms_norm(tile(x), tile(g), eps="1"), [((2, 4), F), ((1, 4), F)]),
    (TypeError, "tensor", lambda x, g: xt.rms_norm(x, tile(g)), [((2, 4), F), ((1, 4), F)]),
    (TypeError, "requires", lambda x: xt.row_scale(tile(x)), [((2, 4), I8)]),
    (ValueError, "scale", lambda x, s: xt.quantize(tile(x), tile(s)), [((2, 4), F), ((1, 4), F)]),
    (TypeError, "float32 scale", lambda x, s: xt.quantize(tile(x), tile(s)), [((2, 4), F), ((2, 1), H)]),
    (ValueError, "two weights a byte", lambda x, w, s: xt.matmul_q4(tile(x), tile(w), tile(s)),
     [((2, 64), H), ((4, 64), I8), ((4, 1), H)]),
    (ValueError, "multiple of 32", lambda x, w, s: xt.matmul_q4(tile(x), tile(w), tile(s)),
     [((2, 64), H), ((4, 32), I8), ((4, 4), H)]),
    (ValueError, "scales", lambda x, w, s: xt.matmul_q4(tile(x), tile(w), tile(s)),
     [((2, 64), H), ((4, 32), I8), ((5, 2), H)]),
    (TypeError, "requires", lambda x, w, s: xt.matmul_q4(tile(x), tile(w), tile(s)),
     [((2, 64), F), ((4, 32), I8), ((4, 2), H)]),
    (TypeError, "result", lambda x, w, s: xt.matmul_q4(tile(x), tile(w), tile(s), dtype=I8),
     [((2, 64), H), ((4, 32), I8), ((4, 2), H)]),
    (ValueError, "row scale", lambda x, w, s, r: xt.matmul_q4(tile(x), tile(w), tile(s), row_scale=tile(r)),
     [((2, 64), I8), ((4, 32), I8), ((4, 2), H), ((1, 2), F)]),
    (TypeError, "one dtype", lambda q, k: xt.attend(tile(q), tile(k), tile(k), scale=1.0), [((2, 64), F), ((5, 64), F)]),
    (ValueError, "one shape", lambda q, k, v: xt.attend(tile(q), tile(k), tile(v), scale=1.0),
     [((2, 64), H), ((5, 64), H), ((6, 64), H)]),
    (ValueError, "query", lambda q, k: xt.attend(tile(q), tile(k), tile(k), scale=1.0), [((2, 65), H), ((5, 64), H)]),
    (ValueError, "scale", lambda q, k: xt.attend(tile(q), tile(k), tile(k), scale=0.0), [((2, 64), H), ((5, 64), H)]),
    (ValueError, "cap", lambda q, k: xt.attend(tile(q), tile(k), tile(k), scale=1.0, cap=float("inf")),
     [((2, 64), H), ((5, 64), H)]),
    (ValueError, "window", lambda q, k: xt.attend(tile(q), tile(k), tile(k), scale=1.0, window=0),
     [((2, 64), H), ((5, 64), H)]),
    (TypeError, "window", lambda q, k: xt.attend(tile(q), tile(k), tile(k), scale=1.0, window=1.5),
     [((2, 64), H), ((5, 64), H)]),
    (TypeError, "causal", lambda q, k: xt.attend(tile(q), tile(k), tile(k), scale=1.0, causal=1),
     [((2, 64), H), ((5, 64), H)]),
    (ValueError, "together", lambda q, k, d: xt.attend(tile(q), tile(k), tile(k), scale=1.0, q_docs=tile(d)),
     [((2, 64), H), ((5, 64), H), ((1, 2), I32)]),
    (ValueError, "length of shape", lambda q, k, n: xt.attend(tile(q), tile(k), tile(k), scale=1.0, length=tile(n)),
     [((2, 64), H), ((5, 64), H), ((2, 1), I32)]),
    (ValueError, "start of shape", lambda q, k, n: xt.attend(tile(q), tile(k), tile(k), scale=1.0, start=tile(n)),
     [((2, 64), H), ((5, 64), H), ((1, 1), F)]),
    (ValueError, "slopes of shape", lambda q, k, n: xt.attend(tile(q), tile(k), tile(k), scale=1.0, slopes=tile(n)),
     [((2, 128), H), ((5, 64), H), ((1, 1), F)]),
])
def test_tracer_refusals(error, text, body, arrays):
    with pytest.raises(error, match=text):
        trace(body, *(xt.Array(*a) for a in arrays))


BASE = {name: str(make()) for name, make in PROGRAMS.items()}


@pytest.mark.parametrize("name,old,new,text", [
    ("norm", "eps = 1.000000e-06 : f32", "eps = 1 : i64", "eps attribute must be"),
    ("norm", "eps = 1.000000e-06 : f32", "eps = -1.0 : f32", "eps attribute must be"),
    ("norm", "{eps = 1.000000e-06 : f32} ", "", "requires attribute 'eps'"),
    ("attend", "scale = 1.250000e-01 : f32", "scale = 0.0 : f32", "scale attribute must be"),
    ("attend", "extras = array<i32: 0, 0, 0, 0, 0, 0>", "extras = array<i32: 0, 0, 0>", "exactly 6"),
    ("attend", "extras = array<i32: 0, 0, 0, 0, 0, 0>", "extras = array<i32: 0, 1, 0, 0, 0, 0>", "operand count"),
    ("attend", "extras = array<i32: 0, 0, 0, 0, 0, 0>", "extras = array<i32: 0, 2, 0, 0, 0, 0>", "0 or 1"),
    ("attend_all", "window = 9 : i64", "window = 0 : i64", "window attribute"),
    ("attend_all", "window = 9 : i64", "window = 4294967296 : i64", "window attribute"),
    ("attend_all", "causal = true", "causal = 1 : i64", "causal attribute"),
    ("attend_all", "cap = 3.000000e+01 : f32", "cap = 1.0e+60 : f32", "cap attribute"),
])
def test_verifier_refusals(name, old, new, text):
    assert old in BASE[name]
    with pytest.raises(ValueError, match=text):
        xt.parse(BASE[name].replace(old, new))


@pytest.mark.parametrize("op,attrs,ins,out,text", [
    ("rms_norm", "{eps = 1.0e-6 : f32} ", ["2x4xf32", "1x4xf32"], "2x5xf32", "shapes to match"),
    ("rms_norm", "{eps = 1.0e-6 : f32} ", ["2x4xf32", "2x4xf32"], "2x4xf32", "gamma"),
    ("rms_norm", "{eps = 1.0e-6 : f32} ", ["2x4xi8", "1x4xf32"], "2x4xf32", "element types"),
    ("rms_norm", "{eps = 1.0e-6 : f32} ", ["2x4x1xf32", "1x4xf32"], "2x4x1xf32", "rank-2"),
    ("row_scale", "", ["2x4xf32"], "2x1xf16", "f32 result with one value a row"),
    ("row_scale", "", ["2x4xi8"], "2x1xf32", "operand"),
    ("quantize", "", ["2x4xf32", "1x4xf32"], "2x4xi8", "scale with one value a row"),
    ("quantize", "", ["2x4xf32", "2x1xf32"], "2x4xf32", "i8 result"),
    ("quantize", "", ["2x4xi8", "2x1xf32"], "2x4xi8", "operand"),
    ("matmul_q4", "", ["2x64xf16", "4x32xi8", "4x2xf16"], "2x5xf32", "result shape must match"),
    ("matmul_q4", "", ["2x64xf16", "4x32xi8", "4x2xf16"], "2x4xi8", "scales and result"),
    ("matmul_q4", "", ["2x64xf32", "4x32xi8", "4x2xf16"], "2x4xf32", "requires an i8"),
    ("matmul_q4", "", ["2x64xf16", "4x64xi8", "4x2xf16"], "2x4xf32", "two weights a byte"),
    ("matmul_q4", "", ["2x64xf16", "4x32xi8", "4x4xf16"], "2x4xf32", "multiple of 32"),
    ("matmul_q4", "", ["2x64xf16", "4x32xi8", "4x2xf16", "1x2xf32"], "2x4xf32", "row scale"),
    ("attend", "{scale = 1.0 : f32, extras = array<i32: 0, 0, 0, 0, 0, 0>} ", ["2x64xf32", "5x64xf32", "5x64xf32"],
     "2x64xf32", "f16 or bf16"),
    ("attend", "{scale = 1.0 : f32, extras = array<i32: 0, 0, 0, 0, 0, 0>} ", ["2x64xf16", "5x64xf16", "6x64xf16"],
     "2x64xf16", "one shape"),
    ("attend", "{scale = 1.0 : f32, extras = array<i32: 0, 0, 0, 0, 0, 0>} ", ["2x64xf16", "5x64xf16", "5x64xf16"],
     "2x64xf32", "to match"),
    ("attend", "{scale = 1.0 : f32, extras = array<i32: 0, 0, 0, 0, 0, 0>} ", ["2x65xf16", "5x64xf16", "5x64xf16"],
     "2x65xf16", "query tensor"),
    ("attend", "{scale = 1.0 : f32, extras = array<i32: 0, 0, 0, 0, 1, 0>} ",
     ["2x64xf16", "5x64xf16", "5x64xf16", "1x2xi32"], "2x64xf16", "together"),
    ("attend", "{scale = 1.0 : f32, extras = array<i32: 0, 1, 0, 0, 0, 0>} ",
     ["2x64xf16", "5x64xf16", "5x64xf16", "1x1xf32"], "2x64xf16", "start must be"),
    ("attend", "{extras = array<i32: 0, 0, 0, 0, 0, 0>} ", ["2x64xf16", "5x64xf16", "5x64xf16"], "2x64xf16",
     "requires attribute 'scale'"),
    ("attend", "{scale = 1.0 : f32} ", ["2x64xf16", "5x64xf16", "5x64xf16"], "2x64xf16", "requires attribute 'extras'"),
])
def test_verifier_refuses_types(op, attrs, ins, out, text):
    params = ", ".join(f"%a{i}: tensor<{t}>" for i, t in enumerate(ins))
    types = ", ".join(f"tensor<{t}>" for t in ins)
    names = ", ".join(f"%a{i}" for i in range(len(ins)))
    with pytest.raises(ValueError, match=text):
        xt.parse(f"func.func @f({params}) {{\n  %r = xt.{op}({names}) {attrs}: {types} -> tensor<{out}>\n"
                 "  func.return\n}")


def store(t, a):
    xt.store(a, index=(0,) * a.array.ndim, tile=t)


def fused_norm(x, g, y):
    store(xt.rms_norm(xt.exp(tile(x)), tile(g)), y)


def scale_alone(x, s):
    store(xt.row_scale(tile(x)), s)


def norm_twice(x, g, y):
    store(xt.rms_norm(xt.rms_norm(tile(x), tile(g)), tile(g)), y)


def both_in_one(x, r, g, y):
    h = xt.add(tile(x), tile(r))
    store(h, y)
    store(xt.rms_norm(h, tile(g)), y)


def over_gamma(x, g):
    store(xt.rms_norm(tile(x), tile(g)), g)


def q4_then(x, w, s, y):
    store(xt.exp(xt.matmul_q4(tile(x), tile(w), tile(s))), y)


def attend_of(x, k, y):
    store(xt.attend(xt.exp(tile(x)), tile(k), tile(k), scale=1.0), y)


def attend_plain(x, k, y):
    store(xt.attend(tile(x), tile(k), tile(k), scale=1.0), y)


def attend_over_keys(x, k):
    store(xt.attend(tile(x), tile(k), tile(k), scale=1.0), k)


@pytest.mark.parametrize("text,body,arrays", [
    ("rms_norm programs must be", fused_norm, [((2, 4), F), ((1, 4), F), ((2, 4), F)]),
    ("run on the result of an rms_norm", scale_alone, [((2, 4), F), ((2, 1), F)]),
    ("rms_norm programs must be", norm_twice, [((2, 4), F), ((1, 4), F), ((2, 4), F)]),
    ("is stored twice", both_in_one, [((2, 4), F), ((2, 4), F), ((1, 4), F), ((2, 4), F)]),
    ("is also an operand", over_gamma, [((1, 4), F), ((1, 4), F)]),
    ("matmul_q4 programs must be", q4_then, [((2, 64), H), ((4, 32), I8), ((4, 2), H), ((2, 4), F)]),
    ("loaded tiles", attend_of, [((2, 64), H), ((5, 64), H), ((2, 64), H)]),
    ("32 to 256 columns", attend_plain, [((2, 48), H), ((5, 48), H), ((2, 48), H)]),
    ("32 to 256 columns", attend_plain, [((2, 288), H), ((5, 288), H), ((2, 288), H)]),
    ("is also an operand", attend_over_keys, [((5, 64), H), ((5, 64), H)]),
])
def test_planner_refusals(text, body, arrays):
    m = trace(body, *(xt.Array(*a) for a in arrays))
    with pytest.raises(NotImplementedError, match=text):
        xt.plan(m)


def test_rows_in_an_order_that_no_stride_gives_are_refused():
    """(rows, heads) swapped by a reshape: not evenly spaced."""

    def body(q, k, o):
        qt = xt.reshape(xt.load(q, index=(0, 0, 0), shape=(4, 3, 64)), shape=(3, 4, 64))
        xt.store(o, index=(0, 0, 0), tile=xt.attend(qt, tile(k), tile(k), scale=1.0))

    a = [xt.Array((8, 5, 64), H), xt.Array((5, 64), H), xt.Array((3, 4, 64), H)]
    with pytest.raises(NotImplementedError, match="evenly spaced"):
        xt.plan(trace(body, *a))


def test_builder_refusals():
    with pytest.raises(ValueError, match="trow"):
        K.rms_norm(5, 64, trow=2)
    with pytest.raises(ValueError, match="group"):
        K.matmul_q4(1, 64, 96, group=64)
    with pytest.raises(ValueError, match="positive"):
        K.masked_attention(1, 1, 1, 0, 5, 64)


@pytest.mark.parametrize("name", PROGRAMS)
def test_launch_refuses_what_is_not_on_a_gpu(name):
    import torch

    m = PROGRAMS[name]()
    dtypes = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8, "i32": torch.int32}
    bufs = [torch.zeros(a["shape"], dtype=dtypes[a["dtype"]]) for a in xt.signature(m)["args"]]
    with pytest.raises(ValueError, match="not on a GPU"):
        xt.launch(m, *bufs)
    with pytest.raises(ValueError, match="buffers"):
        xt.launch(m, *bufs[1:])


def test_both_bindings_agree():
    compiled = pytest.importorskip("xtile_amd._compiled").load()
    for name, text in BASE.items():
        wrapped = "module {\n" + text + "\n}"
        c, m = compiled.parse(wrapped), xt.parse(text)
        assert compiled.plan(c)[0] == xt.plan(m)["kernel"] and compiled.workspace(c) == xt.workspace(m)
