"""mx4_scale, quantize_mx4, dequantize_mx4, matmul_mx4, attend with parents and sample: text, passes, refusals, plans."""

from __future__ import annotations

import re

import numpy as np
import pytest

import xtile_amd as xt
from xtile_amd import kernels as K

from . import answers_ref as ref

PROGRAMS = {
    "rows": lambda: K.quantize_mx4(6, 96),
    "rows_values": lambda: K.quantize_mx4(6, 96, xt.float16, values=True),
    "values": lambda: K.dequantize_mx4(6, 96, xt.float32),
    "product": lambda: K.matmul_mx4(3, 70, 96, out=xt.bfloat16),
    "sample": lambda: K.sample(4, 100),
    "sample_all": lambda: K.sample(4, 100, xt.bfloat16, temperature=True, top_k=True, top_p=True, min_p=True, trow=2),
    "tree": lambda: K.masked_attention(2, 3, 2, 5, 77, 64, parents=True),
    "tree_all": lambda: K.masked_attention(2, 3, 2, 5, 77, 64, dtype=xt.float16, cap=30.0, window=9, slopes=True, start=True,
                                           length=True, parents=True, token_major=True),
}
OPS = r"= (xt\.(?:mx4_scale|quantize_mx4|dequantize_mx4|matmul_mx4|sample|attend))\(.*?\)( \{.*?\})? : (.*)"


@pytest.mark.parametrize("name", PROGRAMS)
def test_text_goes_round(name):
    """The printer writes what the tracer wrote; canonicalize keeps it."""
    m = PROGRAMS[name]()
    text, plan, sig = str(m), xt.plan(m), xt.signature(m)
    again = xt.parse(text)
    xt.canonicalize(again)
    printed = str(again)
    assert xt.plan(again) == plan and xt.signature(again) == sig
    ops = re.findall(OPS, text)
    assert ops and re.findall(OPS, printed) == ops
    assert str(xt.parse(printed)) == printed


def test_serialize_unrolls_them():
    assert str(xt.xt_serialize(K.sample(6, 64, trow=2))).count("xt.sample") == 3


@pytest.mark.parametrize("name,kernel", [
    ("rows", "quantize_mx4 bf16 rows scales tile=6x96 grid=(1,1,1)"),
    ("rows_values", "quantize_mx4 f16 rows scales values tile=6x96 grid=(1,1,1)"),
    ("values", "dequantize_mx4 f32 tile=6x96 grid=(1,1,1)"),
    ("product", "matmul_mx4 bf16 tile=3x70 k=96 grid=(1,1,1)"),
    ("sample", "sample f32 tile=4x100 grid=(1,1,1)"),
    ("sample_all", "sample bf16 tile=2x100 temperature top_k top_p min_p grid=(2,1,1)"),
    ("tree", "attend bf16 heads=2 rows=5 keys=77 d=64 parents grid=(3,2,1)"),
    ("tree_all", "attend f16 heads=2 rows=5 keys=77 d=64 cap window=9 slopes start length parents grid=(3,2,1)"),
])
def test_plans(name, kernel):
    assert xt.plan(PROGRAMS[name]())["kernel"] == kernel


def test_programs_without_parents_keep_their_text():
    assert "extras = array<i32: 0, 0, 0, 0, 0, 0>}" in str(K.masked_attention(1, 1, 1, 1, 8, 64)).replace(", scale", "}")


def test_work_of_plans():
    assert xt.plan(K.quantize_mx4(8, 64))["bytes"] == 8 * 64 * 2 + 8 * 32 + 8 * 2
    assert xt.plan(K.quantize_mx4(8, 64, values=True))["bytes"] == 2 * 8 * 64 * 2 + 8 * 32 + 8 * 2
    assert xt.plan(K.dequantize_mx4(8, 64, xt.float32))["bytes"] == 8 * 64 * 4 + 8 * 32 + 8 * 2
    p = xt.plan(K.matmul_mx4(3, 70, 96))
    assert p["bytes"] == 73 * (48 + 3) + 3 * 70 * 4 and p["flops"] == 2 * 3 * 70 * 96
    assert xt.plan(K.sample(4, 100, top_p=True))["bytes"] == 4 * 100 * 4 + 3 * 4 * 4
    p = xt.plan(K.masked_attention(2, 3, 2, 5, 77, 64, parents=True))
    assert p["bytes"] == 2 * 64 * 2 * 3 * (2 * 2 * 5 + 2 * 77) + 2 * 5 * 4
    assert p["flops"] == 4 * 64 * 2 * 3 * 2 * 5 * 77


def splits_of(kv_heads, nk, d=128):
    kernel = xt.plan(K.masked_attention(1, kv_heads, 4, 16, nk, d, start=True, length=True, parents=True))["kernel"]
    return int(kernel.split("splits=")[1].split()[0]) if "splits=" in kernel else 1


@pytest.mark.parametrize("kv_heads,nk,splits", [
    (1, 300, 1), (8, 512, 4), (8, 1024, 8), (8, 3000, 23), (4, 4096, 32), (1, 8192, 64),  # two tiles of keys each
    (8, 4096, 16), (4, 8192, 32), (8, 8192, 32), (12, 4096, 16), (16, 2048, 8)])          # four
def test_splits_of_trees(kv_heads, nk, splits):
    """Few tiles over short caches have small parts, until the workgroups are many."""
    assert splits_of(kv_heads, nk) == splits


def test_slices_of_sampled_rows():
    def slices(*a, **kw):
        return xt.workspace(K.sample(*a, **kw)) // 123248

    assert [slices(r, v) for r, v in ((1, 32767), (1, 32768), (32, 32768), (33, 32768), (128, 131072), (129, 2**20))] == [0, 1, 32, 0, 128, 0]
    assert [slices(r, v, top_k=True) for r, v in ((1, 65535), (1, 65536), (32, 131072), (33, 131072))] == [0, 1, 32, 0]
    assert "slices=4" in xt.plan(K.sample(128, 131072))["kernel"]
    assert "slices" not in xt.plan(K.sample(1, 1000))["kernel"]


def test_buffers_below_element_alignment_are_refused():
    """Before anything is launched: the addresses are not those of any memory."""
    from xtile_amd import _xtile

    m = K.sample(1, 64, top_k=True)
    for k, at in ((0, 4098), (1, 4097), (2, 4098), (3, 4099)):
        ptrs = [4096] * 4
        ptrs[k] = at
        with pytest.raises(ValueError, match=f"buffer {k} is not aligned"):
            _xtile.launch(m, None, ptrs, [256, 4, 4, 4], 0)


def test_buffers_that_meet_are_refused():
    """Results over operands or each other, before anything is launched."""
    from xtile_amd import _xtile

    a = 1 << 20
    for m, ptrs, sizes, text in (
            (K.quantize_mx4(2, 64), [a, a + 64, a + 4096], [256, 64, 4], "buffer 1 is stored and meets buffer 0"),
            (K.quantize_mx4(2, 64), [a, a + 4096, a + 4100], [256, 64, 4], "both stored and meet"),
            (K.quantize_mx4(2, 64, values=True), [a, a + 4096, a + 8192, a + 16], [256, 64, 4, 256], "buffer 3 is stored and meets"),
            (K.dequantize_mx4(2, 64), [a, a + 4096, a], [64, 4, 256], "buffer 2 is stored and meets buffer 0"),
            (K.matmul_mx4(2, 2, 64), [a, a + 4096, a + 8192, a + 12288, a + 4096], [64, 4, 64, 4, 16],
             "buffer 4 is stored and meets buffer 1"),
            (K.sample(2, 64, min_p=True), [a, a + 4096, a + 8192, a + 4096], [512, 8, 8, 8], "buffer 3 is stored and meets buffer 1")):
        with pytest.raises(ValueError, match=text):
            _xtile.launch(m, None, ptrs, sizes, 0)


def trace(body, *arrays):
    return xt.convert(K._named("traced", lambda a: body(*a), len(arrays)), args=arrays, grid=(1, 1, 1))


def tile(a):
    return xt.load(a, index=(0,) * a.array.ndim, shape=a.array.shape)


F, H, B, I8, I32 = xt.float32, xt.float16, xt.bfloat16, xt.int8, xt.int32


@pytest.mark.parametrize("error,text,body,arrays", [
    (ValueError, "rank-2", lambda x: xt.mx4_scale(tile(x)), [((2, 32, 1), F)]),
    (ValueError, "whole blocks", lambda x: xt.mx4_scale(tile(x)), [((2, 48), F)]),
    (TypeError, "requires", lambda x: xt.mx4_scale(tile(x)), [((2, 32), I8)]),
    (TypeError, "tensor", lambda x: xt.mx4_scale(x), [((2, 32), F)]),
    (ValueError, "mx4_scale", lambda x, s: xt.quantize_mx4(tile(x), tile(s)), [((2, 64), F), ((2, 1), I8)]),
    (ValueError, "mx4_scale", lambda x, s: xt.quantize_mx4(tile(x), tile(s)), [((2, 64), F), ((2, 2), F)]),
    (TypeError, "requires", lambda x, s: xt.quantize_mx4(tile(x), tile(s)), [((2, 64), I32), ((2, 2), I8)]),
    (ValueError, "scales", lambda q, s: xt.dequantize_mx4(tile(q), tile(s)), [((2, 32), I8), ((2, 1), I8)]),
    (ValueError, "rows with", lambda q, s: xt.dequantize_mx4(tile(q), tile(s)), [((2, 24), I8), ((2, 1), I8)]),
    (TypeError, "int8", lambda q, s: xt.dequantize_mx4(tile(q), tile(s)), [((2, 32), I8), ((2, 2), F)]),
    (TypeError, "result", lambda q, s: xt.dequantize_mx4(tile(q), tile(s), dtype=I8), [((2, 32), I8), ((2, 2), I8)]),
    (ValueError, "one length", lambda q, s, w, r: xt.matmul_mx4(tile(q), tile(s), tile(w), tile(r)),
     [((2, 32), I8), ((2, 2), I8), ((5, 16), I8), ((5, 1), I8)]),
    (ValueError, "scales", lambda q, s, w, r: xt.matmul_mx4(tile(q), tile(s), tile(w), tile(r)),
     [((2, 32), I8), ((2, 2), I8), ((5, 32), I8), ((4, 2), I8)]),
    (TypeError, "result", lambda q, s: xt.matmul_mx4(tile(q), tile(s), tile(q), tile(s), dtype=I32),
     [((2, 32), I8), ((2, 2), I8)]),
    (ValueError, "rank-2", lambda x, u: xt.sample(tile(x), tile(u)), [((2, 5, 1), F), ((2, 1), F)]),
    (TypeError, "logits", lambda x, u: xt.sample(tile(x), tile(u)), [((2, 5), I8), ((2, 1), F)]),
    (ValueError, "uniform of shape", lambda x, u: xt.sample(tile(x), tile(u)), [((2, 5), F), ((1, 2), F)]),
    (ValueError, "uniform of shape", lambda x, u: xt.sample(tile(x), tile(u)), [((2, 5), F), ((2, 1), H)]),
    (ValueError, "top_k of shape", lambda x, u: xt.sample(tile(x), tile(u), top_k=tile(u)), [((2, 5), F), ((2, 1), F)]),
    (ValueError, "min_p of shape", lambda x, u, k: xt.sample(tile(x), tile(u), min_p=tile(k)),
     [((2, 5), F), ((2, 1), F), ((2, 1), I32)]),
    (TypeError, "tensor", lambda x, u: xt.sample(tile(x), 0.5), [((2, 5), F), ((2, 1), F)]),
    (ValueError, "parents of shape", lambda q, k, p: xt.attend(tile(q), tile(k), tile(k), scale=1.0, parents=tile(p)),
     [((2, 64), H), ((5, 64), H), ((1, 5), I32)]),
    (ValueError, "parents of shape", lambda q, k, p: xt.attend(tile(q), tile(k), tile(k), scale=1.0, parents=tile(p)),
     [((2, 64), H), ((5, 64), H), ((1, 2), F)]),
    (ValueError, "without causal", lambda q, k, p: xt.attend(tile(q), tile(k), tile(k), scale=1.0, causal=True, parents=tile(p)),
     [((2, 64), H), ((5, 64), H), ((1, 2), I32)]),
    (ValueError, "without causal", lambda q, k, p, n: xt.attend(tile(q), tile(k), tile(k), scale=1.0, prefix=tile(n), parents=tile(p)),
     [((2, 64), H), ((5, 64), H), ((1, 2), I32), ((1, 1), I32)]),
    (ValueError, "without causal", lambda q, k, p, n: xt.attend(tile(q), tile(k), tile(k), scale=1.0, q_docs=tile(p), k_docs=tile(n),
                                                               parents=tile(p)),
     [((2, 64), H), ((5, 64), H), ((1, 2), I32), ((1, 5), I32)]),
])
def test_tracer_refusals(error, text, body, arrays):
    with pytest.raises(error, match=text):
        trace(body, *(xt.Array(*a) for a in arrays))


@pytest.mark.parametrize("name", ["mx4_scale", "sample"])
def test_only_while_tracing(name):
    with pytest.raises(RuntimeError, match="converting"):
        getattr(xt, name)(*([None] * (2 if name == "sample" else 1)))


BASE = {name: str(make()) for name, make in PROGRAMS.items()}


@pytest.mark.parametrize("name,old,new,text", [
    ("sample", "extras = array<i32: 0, 0, 0, 0>", "extras = array<i32: 0, 0, 0>", "exactly 4"),
    ("sample", "extras = array<i32: 0, 0, 0, 0>", "extras = array<i32: 1, 0, 0, 0>", "operand count"),
    ("sample", "extras = array<i32: 0, 0, 0, 0>", "extras = array<i32: 0, 2, 0, 0>", "0 or 1"),
    ("sample", "{extras = array<i32: 0, 0, 0, 0>} ", "", "requires attribute 'extras'"),
    ("tree", "extras = array<i32: 0, 0, 0, 0, 0, 0, 1>", "extras = array<i32: 0, 0, 0, 0, 0, 0, 0>", "operand count"),
    ("tree", "extras = array<i32: 0, 0, 0, 0, 0, 0, 1>", "extras = array<i32: 0, 0, 0, 0, 0, 0, 0, 1>", "7 with parents"),
    ("tree", "extras = array<i32: 0, 0, 0, 0, 0, 0, 1>", "extras = array<i32: 0, 0, 1, 0, 0, 0, 0>", "length must be"),
    ("tree", "extras = array<i32: 0, 0, 0, 0, 0, 0, 1>", "causal = true, extras = array<i32: 0, 0, 0, 0, 0, 0, 1>", "without causal"),
])
def test_verifier_refusals(name, old, new, text):
    assert old in BASE[name]
    with pytest.raises(ValueError, match=text):
        xt.parse(BASE[name].replace(old, new))


@pytest.mark.parametrize("op,attrs,ins,out,text", [
    ("mx4_scale", "", ["2x64xi8"], "2x2xi8", "operand"),
    ("mx4_scale", "", ["2x40xf32"], "2x1xi8", "whole blocks"),
    ("mx4_scale", "", ["2x64xf32"], "2x2xf32", "one scale a block"),
    ("mx4_scale", "", ["2x64xf32"], "2x3xi8", "one scale a block"),
    ("mx4_scale", "", ["2x64x1xf32"], "2x2xi8", "rank-2"),
    ("quantize_mx4", "", ["2x64xf32", "2x1xi8"], "2x32xi8", "scale a block"),
    ("quantize_mx4", "", ["2x64xf32", "2x2xi8"], "2x64xi8", "two values a byte"),
    ("quantize_mx4", "", ["2x64xf32", "2x2xi8"], "2x32xi32", "two values a byte"),
    ("dequantize_mx4", "", ["2x32xi8", "2x1xi8"], "2x64xf32", "scales"),
    ("dequantize_mx4", "", ["2x32xf32", "2x2xi8"], "2x64xf32", "i8 rows"),
    ("dequantize_mx4", "", ["2x32xi8", "2x2xi8"], "2x64xi8", "result"),
    ("dequantize_mx4", "", ["2x32xi8", "2x2xi8"], "2x32xf32", "two values for each byte"),
    ("matmul_mx4", "", ["2x32xi8", "2x2xi8", "4x16xi8", "4x1xi8"], "2x4xf32", "one length"),
    ("matmul_mx4", "", ["2x32xi8", "2x2xi8", "4x32xi8", "4x1xi8"], "2x4xf32", "scales"),
    ("matmul_mx4", "", ["2x32xi8", "2x2xi8", "4x32xi8", "4x2xi8"], "4x2xf32", "result shape must match"),
    ("matmul_mx4", "", ["2x32xi8", "2x2xi8", "4x32xi8", "4x2xi8"], "2x4xi32", "result"),
    ("sample", "{extras = array<i32: 0, 0, 0, 0>} ", ["2x32xi8", "2x1xf32"], "2x1xi32", "logits"),
    ("sample", "{extras = array<i32: 0, 0, 0, 0>} ", ["2x32xf32", "1x2xf32"], "2x1xi32", "uniform must be"),
    ("sample", "{extras = array<i32: 0, 1, 0, 0>} ", ["2x32xf32", "2x1xf32", "2x1xf32"], "2x1xi32", "top_k must be"),
    ("sample", "{extras = array<i32: 0, 0, 0, 0>} ", ["2x32xf32", "2x1xf32"], "2x1xf32", "one token a row"),
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


def scaled_by_another(x, z, q):
    store(xt.quantize_mx4(tile(x), xt.mx4_scale(tile(z))), q)


def scaled_by_a_loaded(x, s, q):
    store(xt.quantize_mx4(tile(x), tile(s)), q)


def scale_of_a_sum(x, s):
    t = tile(x)
    store(xt.mx4_scale(xt.add(t, t)), s)


def rows_over_scales(x, q, z):
    t = tile(x)
    s = xt.mx4_scale(t)
    store(xt.quantize_mx4(t, s), q)
    store(s, z)
    store(s, z)


def values_of_twice(q, s, y, z):
    store(xt.dequantize_mx4(tile(q), tile(s)), y)
    store(xt.dequantize_mx4(tile(q), tile(s)), z)


def product_then(x, s, y):
    store(xt.exp(xt.matmul_mx4(tile(x), tile(s), tile(x), tile(s))), y)


def product_over(x, s, z):
    store(xt.matmul_mx4(tile(x), tile(s), tile(z), tile(s), dtype=F), z)


def sample_of_exp(x, u, y):
    store(xt.sample(xt.exp(tile(x)), tile(u)), y)


def sample_plain(x, u, y):
    store(xt.sample(tile(x), tile(u)), y)


def tree_plain(q, k, p, y):
    store(xt.attend(tile(q), tile(k), tile(k), scale=1.0, parents=tile(p)), y)


@pytest.mark.parametrize("text,body,arrays", [
    ("must be the stores of mx4_scale", scaled_by_another, [((2, 64), F), ((2, 64), F), ((2, 32), I8)]),
    ("must be the stores of mx4_scale", scaled_by_a_loaded, [((2, 64), F), ((2, 2), I8), ((2, 32), I8)]),
    ("must be the stores of mx4_scale", scale_of_a_sum, [((2, 64), F), ((2, 2), I8)]),
    ("must be the stores of mx4_scale", rows_over_scales, [((2, 64), F), ((2, 32), I8), ((2, 2), I8)]),
    ("must be the stores of mx4_scale", values_of_twice, [((2, 32), I8), ((2, 2), I8), ((2, 64), F), ((2, 64), F)]),
    ("matmul_mx4 programs must be", product_then, [((2, 32), I8), ((2, 2), I8), ((2, 2), F)]),
    ("sample programs must be", sample_of_exp, [((2, 32), F), ((2, 1), F), ((2, 1), I32)]),
    ("at most 2\\^22 logits", sample_plain, [((1, 2**22 + 1), F), ((1, 1), F), ((1, 1), I32)]),
    ("fewer than 2\\^22 rows", sample_plain, [((2**22, 8), F), ((2**22, 1), F), ((2**22, 1), I32)]),
    ("at most 64 drafted tokens", tree_plain, [((65, 64), H), ((80, 64), H), ((1, 65), I32), ((65, 64), H)]),
])
def test_planner_refusals(text, body, arrays):
    m = trace(body, *(xt.Array(*a) for a in arrays))
    with pytest.raises(NotImplementedError, match=text):
        xt.plan(m)


def test_parts_of_the_rows_program():
    """Any of its results alone."""

    def scale_only(x, s):
        store(xt.mx4_scale(tile(x)), s)

    def rows_only(x, q):
        t = tile(x)
        store(xt.quantize_mx4(t, xt.mx4_scale(t)), q)

    def values_only(x, y):
        t = tile(x)
        s = xt.mx4_scale(t)
        store(xt.dequantize_mx4(xt.quantize_mx4(t, s), s, dtype=B), y)

    for body, arrays, kernel in ((scale_only, [((2, 64), F), ((2, 2), I8)], "quantize_mx4 f32 scales tile=2x64"),
                                 (rows_only, [((2, 64), F), ((2, 32), I8)], "quantize_mx4 f32 rows tile=2x64"),
                                 (values_only, [((2, 64), B), ((2, 64), B)], "quantize_mx4 bf16 values tile=2x64")):
        assert xt.plan(trace(body, *(xt.Array(*a) for a in arrays)))["kernel"].startswith(kernel)


def test_values_of_another_type_than_their_input():
    """The values' type is that of the store, and it need not be the input's."""

    def body(x, y):
        t = tile(x)
        s = xt.mx4_scale(t)
        store(xt.dequantize_mx4(xt.quantize_mx4(t, s), s, dtype=F), y)

    with pytest.raises(NotImplementedError, match="of the operand's type"):
        xt.plan(trace(body, xt.Array((2, 64), B), xt.Array((2, 64), F)))


def test_builder_refusals():
    for make in (lambda: K.quantize_mx4(2, 48), lambda: K.dequantize_mx4(2, 16), lambda: K.matmul_mx4(2, 2, 33)):
        with pytest.raises(ValueError, match="blocks of 32"):
            make()
    with pytest.raises(ValueError, match="trow"):
        K.sample(5, 64, trow=2)


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
    for text in BASE.values():
        c, m = compiled.parse("module {\n" + text + "\n}"), xt.parse(text)
        assert compiled.plan(c)[0] == xt.plan(m)["kernel"] and compiled.workspace(c) == xt.workspace(m)


# -- the oracle itself ------------------------------------------------------------


def test_the_oracle_of_rows():
    x = np.array([[6.0, 5.0, 4.9, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, -0.3, -0.0, 7.0] + [0.0] * 20])
    code, byte = ref.quantize_mx4(x)
    assert byte.tolist() == [[127]]
    assert code[0, :12].tolist() == [7, 6, 6, 6, 4, 4, 2, 2, 0, 9, 8, 7]
    assert ref.values(code, byte)[0, :12].tolist() == [6, 4, 4, 4, 2, 2, 1, 1, 0, -0.5, 0, 6]
    assert np.array_equal(ref.unpack(ref.pack(code)), code)
    for top, want in ((2.0**-130, 0), (2.0**127, 252), (np.inf, 255), (np.nan, 255), (1.0, 125), (0.0, 0)):
        block = np.zeros((1, 32))
        block[0, 3] = top
        assert ref.quantize_mx4(block)[1].tolist() == [[want]]


def test_the_oracle_of_sampling():
    x = np.log(np.array([0.1, 0.4, 0.3, 0.2]))
    assert [ref.sample(x, u) for u in (0.0, 0.39, 0.41, 0.69, 0.71, 0.89, 0.91, 0.999)] == [1, 1, 2, 2, 3, 3, 0, 0]
    assert [ref.sample(x, 0.99, top_k=k) for k in (1, 2, 3, 4, 0, -1)] == [1, 2, 3, 0, 0, 0]
    assert [ref.sample(x, 0.99, top_p=p) for p in (0.0, 0.3, 0.5, 0.75, 0.95, 1.0)] == [1, 1, 2, 3, 0, 0]
    assert [ref.sample(x, 0.99, min_p=p) for p in (0.9, 0.7, 0.45, 0.2)] == [1, 2, 3, 0]
    assert ref.sample(np.zeros(4), 0.5) == 2 and ref.sample(np.full(3, -np.inf), 0.5) == -1


def test_the_oracle_of_trees():
    seen, away = ref.tree_seen([-1, 0, 0, 1, 7], 3, 8, 9)
    assert seen.astype(int).tolist() == [[1, 1, 1, 1, 0, 0, 0, 0, 0], [1, 1, 1, 1, 1, 0, 0, 0, 0], [1, 1, 1, 1, 0, 1, 0, 0, 0],
                                         [1, 1, 1, 1, 1, 0, 1, 0, 0], [1, 1, 1, 0, 0, 0, 0, 1, 0]]
    assert away[3, :8].tolist() == [5, 4, 3, 2, 1, 1, 0, 2]
    assert ref.tree_seen([-1, 0], 3, 5, 5, window=2)[0].astype(int).tolist() == [[0, 0, 1, 1, 0], [0, 0, 0, 1, 1]]
