"""Tracing DSL: records one Block's tile program and emits `xt` dialect text.

The user-facing API mirrors the reference tracer (`xtile/dsl.py`): the same
function names, keyword arguments, validation rules and error types, and the
same textual `func.func` output, so that existing kernels and golden text keep
working.  The emitted text is consumed by the native `xt` parser of this
package (`xtile_amd/csrc/ir.cpp`).

Reference behaviour followed here (file:line into the reference tree):
  * dtypes `float32`/`int8`                       xtile/dsl.py:14-15
  * Array validation                              xtile/dsl.py:19-33
  * int kernel args become compile-time constants xtile/dsl.py:181-192
  * SSA naming stems and `%zero`/`%cN` constants  xtile/dsl.py:699-732
  * load / load_conv2d / store validation         xtile/dsl.py:225-313,469-488
  * binary broadcast rule (rhs dims 1), result = lhs shape   xtile/dsl.py:658-679,754-759
  * reductions keep the reduced dim at 1          xtile/dsl.py:622-644
  * `a / b` is `a * reciprocal(b)`                xtile/dsl.py:354-357
  * text format                                   xtile/dsl.py:490-620

Extension (not in the reference, documented as such): `float16` and
`bfloat16` dtypes.  Narrow-float `matmul` and `load_conv2d` produce a float32
result, mirroring the reference's int8 -> float32 rule (xtile/dsl.py:369-370).
Also an extension: `int32` arrays (positions, lengths, documents), and the
operators of a language model's layer, each one op over whole tiles:
`rms_norm`, `row_scale` and `quantize` (rows in 8 bits), `matmul_q4` (4-bit
weights), `mx4_scale`, `quantize_mx4`, `dequantize_mx4` and `matmul_mx4`
(microscaled 4-bit floating point), `attend` (masked attention) and `sample`
(a token from its logits).
"""

from __future__ import annotations

import inspect
import math
from dataclasses import dataclass
from typing import Callable, Sequence


# ---------------------------------------------------------------------------
# dtypes and arrays
# ---------------------------------------------------------------------------


@dataclass(frozen=True)
class DType:
    name: str
    mlir_name: str


float32 = DType(name="float32", mlir_name="f32")
int8 = DType(name="int8", mlir_name="i8")
# Extension dtypes (MFMA input types on gfx950).
float16 = DType(name="float16", mlir_name="f16")
bfloat16 = DType(name="bfloat16", mlir_name="bf16")
# Extension dtype of what `attend` takes beside its tiles: positions, lengths, documents.
int32 = DType(name="int32", mlir_name="i32")

_NARROW_FLOATS = (float16, bfloat16)
_FLOATS = (float32, *_NARROW_FLOATS)


def _all_positive_ints(values: object) -> bool:
    return (
        isinstance(values, tuple)
        and len(values) > 0
        and all(isinstance(v, int) and v > 0 for v in values)
    )


@dataclass(frozen=True)
class Array:
    """A global-memory array argument: static shape plus element type."""

    shape: tuple[int, ...]
    dtype: DType

    def __post_init__(self) -> None:
        if not isinstance(self.shape, tuple) or not self.shape:
            raise TypeError("shape must be a non-empty tuple of integers")
        if not _all_positive_ints(self.shape):
            raise TypeError("shape must contain positive integers")
        if not isinstance(self.dtype, DType):
            raise TypeError("dtype must be an xtile dtype")

    @property
    def ndim(self) -> int:
        return len(self.shape)


def _memref_type(array: Array) -> str:
    return "memref<" + "x".join(map(str, array.shape)) + "x" + array.dtype.mlir_name + ">"


def _tensor_type(shape: Sequence[int], dtype: DType) -> str:
    return "tensor<" + "x".join(map(str, shape)) + "x" + dtype.mlir_name + ">"


# ---------------------------------------------------------------------------
# traced values
# ---------------------------------------------------------------------------


class KernelFunction:
    """A Python function marked with `@xt.kernel`."""

    def __init__(self, fn: Callable[..., object]) -> None:
        self.fn = fn
        self.__name__ = fn.__name__
        self.__doc__ = fn.__doc__
        self.__wrapped__ = fn


@dataclass(frozen=True)
class KernelArg:
    index: int
    python_name: str
    array: Array


@dataclass(frozen=True)
class ScalarArg:
    index: int
    python_name: str
    value: int


@dataclass(frozen=True)
class BlockId:
    dim: int


@dataclass(frozen=True)
class ConstantIndex:
    value: int


@dataclass(frozen=True)
class TensorValue:
    ssa_name: str
    shape: tuple[int, ...]
    dtype: DType

    def __sub__(self, other: object) -> "TensorValue":
        return sub(self, other)

    def __mul__(self, other: object) -> "TensorValue":
        return mul(self, other)

    def __add__(self, other: object) -> "TensorValue":
        return add(self, other)

    def __truediv__(self, other: object) -> "TensorValue":
        return truediv(self, other)


Coord = "BlockId | ConstantIndex"


# Each recorded operation renders its own line of `xt` text.  The renderer
# needs the final argument names, which are only known once tracing ends
# (they depend on how often each array is loaded and stored).


@dataclass(frozen=True)
class _Load:
    result: TensorValue
    array: KernelArg
    index: tuple
    shared: int | None

    def render(self, names: dict[int, str]) -> str:
        attr = f" {{shared = {self.shared} : i64}}" if self.shared in (1, 2) else ""
        coords = _coords_text(self.index)
        types = ", ".join([_memref_type(self.array.array)] + ["i32"] * len(self.index))
        return (
            f"{self.result.ssa_name} = xt.load(%{names[self.array.index]}, {coords}){attr}"
            f" : ({types}) -> {_tensor_type(self.result.shape, self.result.dtype)}"
        )


@dataclass(frozen=True)
class _LoadConv2D:
    result: TensorValue
    array: KernelArg
    filter: TensorValue
    index: tuple
    group: int
    pad: tuple[int, int, int, int]
    stride: tuple[int, int]
    dilation: tuple[int, int]

    def render(self, names: dict[int, str]) -> str:
        def arr(values: Sequence[int]) -> str:
            return "array<i64: " + ", ".join(map(str, values)) + ">"

        attrs = (
            f"{{dilation = {arr(self.dilation)}, group = {self.group} : i64, "
            f"pad = {arr(self.pad)}, stride = {arr(self.stride)}}}"
        )
        types = ", ".join(
            [
                _memref_type(self.array.array),
                _tensor_type(self.filter.shape, self.filter.dtype),
            ]
            + ["i32"] * len(self.index)
        )
        return (
            f"{self.result.ssa_name} = xt.load_conv2d(%{names[self.array.index]}, "
            f"{self.filter.ssa_name}, {_coords_text(self.index)}) {attrs} : ({types}) -> "
            f"{_tensor_type(self.result.shape, self.result.dtype)}"
        )


@dataclass(frozen=True)
class _Store:
    array: KernelArg
    index: tuple
    tile: TensorValue

    def render(self, names: dict[int, str]) -> str:
        types = ", ".join(
            [_tensor_type(self.tile.shape, self.tile.dtype), _memref_type(self.array.array)]
            + ["i32"] * len(self.index)
        )
        return (
            f"xt.store({self.tile.ssa_name}, %{names[self.array.index]}, "
            f"{_coords_text(self.index)}) : ({types}) -> ()"
        )


@dataclass(frozen=True)
class _Compute:
    """Any tensor -> tensor op: `%r = xt.op(%a[, %b[, %c]]) [{axis}] : types -> type`."""

    op_name: str
    result: TensorValue
    operands: tuple[TensorValue, ...]
    axis: int | None = None

    def render(self, names: dict[int, str]) -> str:
        attr = f" {{axis = {self.axis} : i64}}" if self.axis is not None else ""
        operand_names = ", ".join(v.ssa_name for v in self.operands)
        operand_types = ", ".join(_tensor_type(v.shape, v.dtype) for v in self.operands)
        return (
            f"{self.result.ssa_name} = {self.op_name}({operand_names}){attr} : "
            f"{operand_types} -> {_tensor_type(self.result.shape, self.result.dtype)}"
        )


@dataclass(frozen=True)
class _Operator:
    """A tensor -> tensor op with attributes of its own (`attrs`: names and their text)."""

    op_name: str
    result: TensorValue
    operands: tuple[TensorValue, ...]
    attrs: tuple[tuple[str, str], ...] = ()

    def render(self, names: dict[int, str]) -> str:
        attr = " {" + ", ".join(f"{k} = {v}" for k, v in sorted(self.attrs)) + "}" if self.attrs else ""
        operand_names = ", ".join(v.ssa_name for v in self.operands)
        operand_types = ", ".join(_tensor_type(v.shape, v.dtype) for v in self.operands)
        return (
            f"{self.result.ssa_name} = {self.op_name}({operand_names}){attr} : "
            f"{operand_types} -> {_tensor_type(self.result.shape, self.result.dtype)}"
        )


def _float_text(value: float) -> str:
    """An f32 attribute's text, as the printer of the native IR writes it."""
    text = f"{value:.6e}"
    if float(text) != value:
        text = f"{value:.17g}"
        if not any(c in text for c in ".en"):
            text += ".0"
    return text + " : f32"


def _coords_text(index: tuple) -> str:
    parts = []
    for item in index:
        if isinstance(item, BlockId):
            parts.append(f"%bid#{item.dim}")
        else:
            parts.append("%zero" if item.value == 0 else f"%c{item.value}")
    return ", ".join(parts)


# ---------------------------------------------------------------------------
# tracer
# ---------------------------------------------------------------------------


class TraceContext:
    """Symbolic execution of one Block of a kernel."""

    def __init__(
        self,
        kernel: KernelFunction,
        args: tuple,
        grid: tuple[int, int, int],
        double_buffering: bool,
    ) -> None:
        if not (isinstance(grid, tuple) and len(grid) == 3 and _all_positive_ints(grid)):
            raise ValueError("grid must be a 3-tuple of positive integers")
        params = list(inspect.signature(kernel.fn).parameters.values())
        if len(params) != len(args):
            raise ValueError("convert args must match the kernel signature")

        self.kernel_name = kernel.fn.__name__
        self.grid = grid
        self.double_buffering = double_buffering
        kernel_args: list[KernelArg | ScalarArg] = []
        for position, (param, value) in enumerate(zip(params, args)):
            if isinstance(value, Array):
                kernel_args.append(KernelArg(position, param.name, value))
            elif isinstance(value, int):
                kernel_args.append(ScalarArg(position, param.name, value))
            else:
                raise TypeError("convert args must be xt.Array values or integers")
        self.kernel_args = tuple(kernel_args)
        self.ops: list = []
        self.used_block_ids = False
        self.load_counts = [0] * len(kernel_args)
        self.store_counts = [0] * len(kernel_args)
        self._stem_counts: dict[str, int] = {}
        self._constants: dict[int, str] = {}

    # -- helpers ------------------------------------------------------------

    def trace_arguments(self) -> tuple:
        return tuple(a if isinstance(a, KernelArg) else a.value for a in self.kernel_args)

    def _fresh(self, stem: str) -> str:
        n = self._stem_counts.get(stem, 0) + 1
        self._stem_counts[stem] = n
        return f"%{stem}" if n == 1 else f"%{stem}{n}"

    def _value(self, stem: str, shape: tuple[int, ...], dtype: DType) -> TensorValue:
        return TensorValue(self._fresh(stem), tuple(shape), dtype)

    @staticmethod
    def _need_arg(array: object) -> None:
        if not isinstance(array, KernelArg):
            raise TypeError("xtile load/store expect kernel arguments")

    @staticmethod
    def _need_tensor(value: object) -> None:
        if not isinstance(value, TensorValue):
            raise TypeError("xtile operation expects a tensor value")

    @staticmethod
    def _need_shape(shape: object) -> None:
        if not _all_positive_ints(shape):
            raise TypeError("shape must be a tuple of positive integers")

    def _coords(self, index: object) -> tuple:
        if not isinstance(index, tuple) or not index:
            raise TypeError("index must be a non-empty tuple of values")
        out = []
        for item in index:
            if isinstance(item, BlockId):
                out.append(item)
            elif isinstance(item, int):
                if item not in self._constants:
                    self._constants[item] = "%zero" if item == 0 else self._fresh(f"c{item}")
                out.append(ConstantIndex(item))
            else:
                raise TypeError("index values must be xt.bid(...) results or integers")
        return tuple(out)

    @staticmethod
    def _int_tuple(name: str, value: object, length: int, positive: bool = False) -> None:
        if not isinstance(value, tuple) or len(value) != length:
            raise TypeError(f"{name} must be a tuple of {length} integers")
        for item in value:
            if not isinstance(item, int):
                raise TypeError(f"{name} must be a tuple of {length} integers")
            if positive and item <= 0:
                raise ValueError(f"{name} values must be positive")
            if not positive and item < 0:
                raise ValueError(f"{name} values must be non-negative")

    # -- block ids, loads and stores -----------------------------------------

    def bid(self, dim: int) -> BlockId:
        if dim not in (0, 1, 2):
            raise ValueError("xt.bid only supports dimensions 0, 1, and 2")
        self.used_block_ids = True
        return BlockId(dim)

    def load(self, array, index, shape, shared=None) -> TensorValue:
        self._need_arg(array)
        coords = self._coords(index)
        self._need_shape(shape)
        if shared is not None and shared not in (0, 1, 2):
            raise ValueError("shared must be 0, 1, 2, or None")
        rank = array.array.ndim
        if rank != len(shape):
            raise ValueError("xt.load requires shape rank to match the source array rank")
        if len(coords) != len(shape):
            raise ValueError("xt.load requires index rank to match the source array rank")
        result = self._value("x", shape, array.array.dtype)
        self.ops.append(_Load(result, array, coords, shared))
        self.load_counts[array.index] += 1
        return result

    def load_conv2d(self, array, filter_value, index, shape, *, group=1, pad, stride, dilation):
        self._need_arg(array)
        self._need_tensor(filter_value)
        coords = self._coords(index)
        self._need_shape(shape)
        self._int_tuple("pad", pad, 4)
        self._int_tuple("stride", stride, 2, positive=True)
        self._int_tuple("dilation", dilation, 2, positive=True)
        if group <= 0:
            raise ValueError("xt.load_conv2d requires group to be positive")
        if array.array.ndim != 4:
            raise ValueError("xt.load_conv2d requires a rank-4 source memref")
        if len(filter_value.shape) != 4:
            raise ValueError("xt.load_conv2d requires a rank-4 filter tensor")
        if len(coords) != 4 or len(shape) != 4:
            raise ValueError("xt.load_conv2d requires rank-4 index and result shape tuples")
        src_dtype = array.array.dtype
        if src_dtype != filter_value.dtype or src_dtype not in (int8, *_NARROW_FLOATS):
            raise TypeError(
                "xt.load_conv2d requires int8, float16 or bfloat16 source/filter of one dtype"
            )
        if array.array.shape[3] != filter_value.shape[2]:
            raise ValueError("xt.load_conv2d requires source/filter channel dimensions to match")
        if shape[3] > filter_value.shape[3]:
            raise ValueError(
                "xt.load_conv2d result channel dimension must not exceed filter output channels"
            )
        result = self._value("load_conv", shape, float32)
        self.ops.append(
            _LoadConv2D(result, array, filter_value, coords, group, pad, stride, dilation)
        )
        self.load_counts[array.index] += 1
        return result

    def store(self, array, index, tile) -> None:
        self._need_arg(array)
        coords = self._coords(index)
        if not isinstance(tile, TensorValue):
            raise TypeError("xt.store expects a tensor value")
        if array.array.ndim != len(tile.shape):
            raise ValueError("xt.store requires tile rank to match the destination array rank")
        if len(coords) != len(tile.shape):
            raise ValueError("xt.store requires index rank to match the destination array rank")
        self.ops.append(_Store(array, coords, tile))
        self.store_counts[array.index] += 1

    # -- compute ----------------------------------------------------------

    def _unary(self, op_name: str, value, stem: str) -> TensorValue:
        self._need_tensor(value)
        result = self._value(stem, value.shape, value.dtype)
        self.ops.append(_Compute(op_name, result, (value,)))
        return result

    def _binary(self, op_name: str, lhs, rhs, stem: str) -> TensorValue:
        self._need_tensor(lhs)
        self._need_tensor(rhs)
        if lhs.dtype != rhs.dtype:
            raise TypeError("binary xtile ops require matching dtypes")
        same_rank = len(lhs.shape) == len(rhs.shape)
        if lhs.shape != rhs.shape and not (
            same_rank and all(r in (1, l) for l, r in zip(lhs.shape, rhs.shape))
        ):
            raise ValueError(
                "binary xtile ops require equal or rowwise-broadcast-compatible shapes"
            )
        result = self._value(stem, lhs.shape, lhs.dtype)
        self.ops.append(_Compute(op_name, result, (lhs, rhs)))
        return result

    def _reduce(self, op_name: str, value, stem: str, axis: int) -> TensorValue:
        self._need_tensor(value)
        if len(value.shape) != 2:
            raise ValueError("xt.max and xt.sum currently support rank-2 tensors only")
        if not isinstance(axis, int):
            raise TypeError("axis must be an integer")
        rank = len(value.shape)
        if not -rank <= axis < rank:
            raise ValueError("axis must be in range [-rank, rank)")
        axis %= rank
        shape = tuple(1 if d == axis else n for d, n in enumerate(value.shape))
        result = self._value(stem, shape, value.dtype)
        self.ops.append(_Compute(op_name, result, (value,), axis=axis))
        return result

    def reduce_max(self, value, axis: int = -1) -> TensorValue:
        return self._reduce("xt.reduce_max", value, "row_max", axis)

    def reduce_sum(self, value, axis: int = -1) -> TensorValue:
        return self._reduce("xt.reduce_sum", value, "row_sum", axis)

    def add(self, lhs, rhs):
        return self._binary("xt.add", lhs, rhs, "sum")

    def sub(self, lhs, rhs):
        return self._binary("xt.sub", lhs, rhs, "shifted")

    def mul(self, lhs, rhs):
        return self._binary("xt.mul", lhs, rhs, "normalized")

    def truediv(self, lhs, rhs):
        self._need_tensor(lhs)
        self._need_tensor(rhs)
        return self.mul(lhs, self.reciprocal(rhs))

    def exp(self, v):
        return self._unary("xt.exp", v, "exp")

    def cos(self, v):
        return self._unary("xt.cos", v, "cos")

    def sin(self, v):
        return self._unary("xt.sin", v, "sin")

    def reciprocal(self, v):
        return self._unary("xt.reciprocal", v, "inv_sum")

    def rsqrt(self, v):
        return self._unary("xt.rsqrt", v, "rsqrt")

    def sigmoid(self, v):
        return self._unary("xt.sigmoid", v, "sigmoid")

    def tanh(self, v):
        return self._unary("xt.tanh", v, "tanh")

    def silu(self, v):
        return self._unary("xt.silu", v, "silu")

    def matmul(self, lhs, rhs) -> TensorValue:
        self._need_tensor(lhs)
        self._need_tensor(rhs)
        if len(lhs.shape) != 2 or len(rhs.shape) != 2:
            raise ValueError("xt.matmul currently supports rank-2 tensors only")
        if lhs.shape[1] != rhs.shape[0]:
            raise ValueError("xt.matmul requires lhs inner dimension to match rhs outer dimension")
        if lhs.dtype == rhs.dtype and lhs.dtype in (int8, *_NARROW_FLOATS):
            out_dtype = float32
        elif lhs.dtype == rhs.dtype:
            out_dtype = lhs.dtype
        else:
            raise TypeError("xt.matmul requires matching dtypes or int8 inputs")
        result = self._value("matmul", (lhs.shape[0], rhs.shape[1]), out_dtype)
        self.ops.append(_Compute("xt.matmul", result, (lhs, rhs)))
        return result

    def mma(self, lhs, rhs, acc) -> TensorValue:
        for v in (lhs, rhs, acc):
            self._need_tensor(v)
        if len(lhs.shape) != 2 or len(rhs.shape) != 2 or len(acc.shape) != 2:
            raise ValueError("xt.mma currently supports rank-2 tensors only")
        if lhs.dtype != int8 or rhs.dtype != int8:
            raise TypeError("xt.mma requires int8 lhs and rhs tensors")
        if acc.dtype != float32:
            raise TypeError("xt.mma currently requires a float32 accumulator")
        if lhs.shape[1] != rhs.shape[0]:
            raise ValueError("xt.mma requires lhs inner dimension to match rhs outer dimension")
        if acc.shape != (lhs.shape[0], rhs.shape[1]):
            raise ValueError("xt.mma accumulator shape must match the matmul result shape")
        result = self._value("mma", acc.shape, acc.dtype)
        self.ops.append(_Compute("xt.mma", result, (lhs, rhs, acc)))
        return result

    def astype(self, value, dtype) -> TensorValue:
        self._need_tensor(value)
        if not isinstance(dtype, DType):
            raise TypeError("xt.astype requires an xtile dtype")
        if value.dtype == dtype:
            return value
        if value.dtype == int8 and dtype == float32:
            op_name = "xt.itof"
        elif value.dtype == float32 and dtype == int8:
            op_name = "xt.ftoi"
        else:
            raise TypeError("xt.astype only supports int8<->float32 conversions")
        result = self._value("cast", value.shape, dtype)
        self.ops.append(_Compute(op_name, result, (value,)))
        return result

    def reshape(self, value, shape) -> TensorValue:
        self._need_tensor(value)
        self._need_shape(shape)
        if _numel(value.shape) != _numel(shape):
            raise ValueError("xt.reshape requires the same number of elements")
        result = self._value("reshape", shape, value.dtype)
        self.ops.append(_Compute("xt.reshape", result, (value,)))
        return result

    def transpose(self, value) -> TensorValue:
        self._need_tensor(value)
        if len(value.shape) != 3:
            raise ValueError("xt.transpose currently supports rank-3 tensors only")
        b, m, n = value.shape
        result = self._value("transpose", (b, n, m), value.dtype)
        self.ops.append(_Compute("xt.transpose", result, (value,)))
        return result

    # -- operators of a language model's layer (extension) ------------------

    @staticmethod
    def _number(op: str, name: str, value: object, positive: bool = True) -> float:
        if isinstance(value, bool) or not isinstance(value, (int, float)):
            raise TypeError(f"{op} requires {name} to be a number")
        if not math.isfinite(value) or value < 0 or (positive and value == 0) or value > 3.4028234663852886e38:
            raise ValueError(f"{op} requires {name} to be finite and {'positive' if positive else 'non-negative'}")
        return float(value)

    def rms_norm(self, value, gamma, eps: float = 1e-6, dtype: DType | None = None) -> TensorValue:
        self._need_tensor(value)
        self._need_tensor(gamma)
        dtype = value.dtype if dtype is None else dtype
        if len(value.shape) != 2:
            raise ValueError("xt.rms_norm currently supports rank-2 tensors only")
        if gamma.shape != (1, value.shape[1]):
            raise ValueError("xt.rms_norm requires a (1, C) gamma matching the value's columns")
        if value.dtype not in _FLOATS or gamma.dtype not in _FLOATS or dtype not in _FLOATS:
            raise TypeError("xt.rms_norm requires float32, float16 or bfloat16 tensors and result")
        eps = self._number("xt.rms_norm", "eps", eps, positive=False)
        result = self._value("rms", value.shape, dtype)
        self.ops.append(_Operator("xt.rms_norm", result, (value, gamma), (("eps", _float_text(eps)),)))
        return result

    def row_scale(self, value) -> TensorValue:
        self._need_tensor(value)
        if len(value.shape) != 2:
            raise ValueError("xt.row_scale currently supports rank-2 tensors only")
        if value.dtype not in _FLOATS:
            raise TypeError("xt.row_scale requires a float32, float16 or bfloat16 tensor")
        result = self._value("row_scale", (value.shape[0], 1), float32)
        self.ops.append(_Operator("xt.row_scale", result, (value,)))
        return result

    def quantize(self, value, scale) -> TensorValue:
        self._need_tensor(value)
        self._need_tensor(scale)
        if len(value.shape) != 2:
            raise ValueError("xt.quantize currently supports rank-2 tensors only")
        if scale.shape != (value.shape[0], 1):
            raise ValueError("xt.quantize requires a (R, 1) scale matching the value's rows")
        if value.dtype not in _FLOATS or scale.dtype != float32:
            raise TypeError("xt.quantize requires a float tensor and a float32 scale")
        result = self._value("quantized", value.shape, int8)
        self.ops.append(_Operator("xt.quantize", result, (value, scale)))
        return result

    def matmul_q4(self, value, weight, scales, row_scale=None, dtype: DType = float32) -> TensorValue:
        operands = (value, weight, scales) if row_scale is None else (value, weight, scales, row_scale)
        for v in operands:
            self._need_tensor(v)
        if any(len(v.shape) != 2 for v in operands):
            raise ValueError("xt.matmul_q4 currently supports rank-2 tensors only")
        (m, k), (n, half) = value.shape, weight.shape
        if value.dtype not in (int8, *_NARROW_FLOATS) or weight.dtype != int8 or scales.dtype not in _FLOATS:
            raise TypeError("xt.matmul_q4 requires an int8, float16 or bfloat16 value, int8 weights and float scales")
        if dtype not in _FLOATS:
            raise TypeError("xt.matmul_q4 requires a float32, float16 or bfloat16 result")
        if k != 2 * half:
            raise ValueError("xt.matmul_q4 requires two weights a byte: weight columns half the value's")
        if scales.shape[0] != n or k % scales.shape[1] or (k // scales.shape[1]) % 32:
            raise ValueError("xt.matmul_q4 requires (N, K / G) scales for groups of G weights, G a multiple of 32")
        if row_scale is not None and (row_scale.shape != (m, 1) or row_scale.dtype != float32):
            raise ValueError("xt.matmul_q4 requires a float32 (M, 1) row scale")
        result = self._value("matmul", (m, n), dtype)
        self.ops.append(_Operator("xt.matmul_q4", result, operands))
        return result

    def _float_rows(self, op: str, value) -> None:
        self._need_tensor(value)
        if len(value.shape) != 2:
            raise ValueError(f"{op} currently supports rank-2 tensors only")
        if value.dtype not in _FLOATS:
            raise TypeError(f"{op} requires a float32, float16 or bfloat16 tensor")
        if value.shape[1] % 32:
            raise ValueError(f"{op} requires rows of whole blocks of 32")

    def _mx4_rows(self, op: str, value, scale) -> tuple[int, int]:
        """(rows, values a row) of packed rows and their scales."""
        self._need_tensor(value)
        self._need_tensor(scale)
        if len(value.shape) != 2 or len(scale.shape) != 2:
            raise ValueError(f"{op} currently supports rank-2 tensors only")
        if value.dtype != int8 or scale.dtype != int8:
            raise TypeError(f"{op} requires int8 rows and scales, as quantize_mx4 and mx4_scale give them")
        if value.shape[1] % 16 or scale.shape != (value.shape[0], value.shape[1] // 16):
            raise ValueError(f"{op} requires (R, C / 2) rows with (R, C / 32) scales")
        return value.shape[0], 2 * value.shape[1]

    def mx4_scale(self, value) -> TensorValue:
        self._float_rows("xt.mx4_scale", value)
        result = self._value("mx4_scale", (value.shape[0], value.shape[1] // 32), int8)
        self.ops.append(_Operator("xt.mx4_scale", result, (value,)))
        return result

    def quantize_mx4(self, value, scale) -> TensorValue:
        self._float_rows("xt.quantize_mx4", value)
        self._need_tensor(scale)
        if scale.shape != (value.shape[0], value.shape[1] // 32) or scale.dtype != int8:
            raise ValueError("xt.quantize_mx4 requires the int8 (R, C / 32) scale of mx4_scale")
        result = self._value("quantized", (value.shape[0], value.shape[1] // 2), int8)
        self.ops.append(_Operator("xt.quantize_mx4", result, (value, scale)))
        return result

    def dequantize_mx4(self, value, scale, dtype: DType = float32) -> TensorValue:
        shape = self._mx4_rows("xt.dequantize_mx4", value, scale)
        if dtype not in _FLOATS:
            raise TypeError("xt.dequantize_mx4 requires a float32, float16 or bfloat16 result")
        result = self._value("values", shape, dtype)
        self.ops.append(_Operator("xt.dequantize_mx4", result, (value, scale)))
        return result

    def matmul_mx4(self, value, value_scale, weight, weight_scale, dtype: DType = float32) -> TensorValue:
        m, k = self._mx4_rows("xt.matmul_mx4", value, value_scale)
        n, wk = self._mx4_rows("xt.matmul_mx4", weight, weight_scale)
        if dtype not in _FLOATS:
            raise TypeError("xt.matmul_mx4 requires a float32, float16 or bfloat16 result")
        if k != wk:
            raise ValueError("xt.matmul_mx4 requires value and weight rows of one length")
        result = self._value("matmul", (m, n), dtype)
        self.ops.append(_Operator("xt.matmul_mx4", result, (value, value_scale, weight, weight_scale)))
        return result

    def sample(self, logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None) -> TensorValue:
        extras = (temperature, top_k, top_p, min_p)
        for t in (logits, uniform, *(e for e in extras if e is not None)):
            self._need_tensor(t)
        if len(logits.shape) != 2:
            raise ValueError("xt.sample currently supports rank-2 tensors only")
        if logits.dtype not in _FLOATS:
            raise TypeError("xt.sample requires float32, float16 or bfloat16 logits")
        rows = (logits.shape[0], 1)
        for name, t in zip(("uniform", "temperature", "top_k", "top_p", "min_p"), (uniform, *extras)):
            dtype = int32 if name == "top_k" else float32
            if t is not None and (t.shape != rows or t.dtype != dtype):
                raise ValueError(f"xt.sample requires {name} of shape {rows} and dtype {dtype.name}")
        present = ", ".join("1" if e is not None else "0" for e in extras)
        result = self._value("token", rows, int32)
        operands = (logits, uniform, *(e for e in extras if e is not None))
        self.ops.append(_Operator("xt.sample", result, operands, (("extras", f"array<i32: {present}>"),)))
        return result

    def attend(self, q, k, v, scale, cap=None, causal=False, window=None, slopes=None, start=None, length=None,
               prefix=None, q_docs=None, k_docs=None, parents=None) -> TensorValue:
        extras = (slopes, start, length, prefix, q_docs, k_docs)
        if parents is not None:
            extras = (*extras, parents)
        for t in (q, k, v, *(e for e in extras if e is not None)):
            self._need_tensor(t)
        if q.dtype not in _NARROW_FLOATS or k.dtype != q.dtype or v.dtype != q.dtype:
            raise TypeError("xt.attend requires float16 or bfloat16 tensors of one dtype")
        if len(k.shape) != 2 or k.shape != v.shape:
            raise ValueError("xt.attend requires (keys, D) key and value tensors of one shape")
        nk, d = k.shape
        if len(q.shape) == 3 and q.shape[2] == d:
            heads, rows = q.shape[0], q.shape[1]
        elif len(q.shape) == 2 and q.shape[1] % d == 0:
            heads, rows = q.shape[1] // d, q.shape[0]
        else:
            raise ValueError("xt.attend requires a (heads, rows, D) or (rows, heads * D) query tensor")
        if (q_docs is None) != (k_docs is None):
            raise ValueError("xt.attend requires q_docs and k_docs together")
        if parents is not None and (causal or prefix is not None or q_docs is not None):
            raise ValueError("xt.attend takes parents without causal, prefix, q_docs and k_docs")
        wants = ((1, heads), (1, 1), (1, 1), (1, 1), (1, rows), (1, nk), (1, rows))
        for name, t, shape in zip(("slopes", "start", "length", "prefix", "q_docs", "k_docs", "parents"), extras, wants):
            dtype = float32 if name == "slopes" else int32
            if t is not None and (t.shape != shape or t.dtype != dtype):
                raise ValueError(f"xt.attend requires {name} of shape {shape} and dtype {dtype.name}")
        attrs = [("scale", _float_text(self._number("xt.attend", "scale", scale)))]
        if cap is not None:
            attrs.append(("cap", _float_text(self._number("xt.attend", "cap", cap))))
        if not isinstance(causal, bool):
            raise TypeError("xt.attend requires causal to be True or False")
        if causal:
            attrs.append(("causal", "true"))
        if window is not None:
            if isinstance(window, bool) or not isinstance(window, int):
                raise TypeError("xt.attend requires window to be an integer")
            if not 0 < window < 2**31:
                raise ValueError("xt.attend requires window to be positive and below 2**31")
            attrs.append(("window", f"{window} : i64"))
        present = ", ".join("1" if e is not None else "0" for e in extras)
        attrs.append(("extras", f"array<i32: {present}>"))
        result = self._value("attend", q.shape, q.dtype)
        operands = (q, k, v, *(e for e in extras if e is not None))
        self.ops.append(_Operator("xt.attend", result, operands, tuple(attrs)))
        return result

    # -- emission ---------------------------------------------------------

    def _arg_names(self) -> dict[int, str]:
        """Loaded-only arrays are input/inputN, stored-only output/outputN."""
        names: dict[int, str] = {}
        n_in = n_out = 0
        for arg in self.kernel_args:
            if not isinstance(arg, KernelArg):
                continue
            loads, stores = self.load_counts[arg.index], self.store_counts[arg.index]
            if loads and not stores:
                n_in += 1
                names[arg.index] = "input" if n_in == 1 else f"input{n_in}"
            elif stores and not loads:
                n_out += 1
                names[arg.index] = "output" if n_out == 1 else f"output{n_out}"
            else:
                names[arg.index] = arg.python_name
        return names

    def emit_function_asm(self) -> str:
        names = self._arg_names()
        params = ", ".join(
            f"%{names[a.index]}: {_memref_type(a.array)}"
            for a in self.kernel_args
            if isinstance(a, KernelArg)
        )
        attrs = ["xt.grid = array<i32: " + ", ".join(map(str, self.grid)) + ">"]
        if self.double_buffering:
            attrs.append("xt.double_buffering = 1 : i32")
        out = [f"func.func @{self.kernel_name}({params}) attributes {{{', '.join(attrs)}}} {{"]
        if self.used_block_ids:
            out.append("  %bid:3 = xt.get_tile_block_id : i32, i32, i32")
        if self._constants:
            out.extend(
                f"  {name} = arith.constant {value} : i32"
                for value, name in sorted(self._constants.items())
            )
            out.append("")
        out.extend("  " + op.render(names) for op in self.ops)
        out.append("  func.return")
        out.append("}")
        return "\n".join(out)


def _numel(shape: Sequence[int]) -> int:
    n = 1
    for d in shape:
        n *= d
    return n


# ---------------------------------------------------------------------------
# module-level API (valid only while a kernel is being converted)
# ---------------------------------------------------------------------------

_ACTIVE_TRACE: TraceContext | None = None


def _trace(what: str) -> TraceContext:
    if _ACTIVE_TRACE is None:
        raise RuntimeError(f"xt.{what} may only be used while converting a kernel")
    return _ACTIVE_TRACE


def kernel(fn: Callable[..., object]) -> KernelFunction:
    return KernelFunction(fn)


def bid(dim: int) -> BlockId:
    return _trace("bid").bid(dim)


def load(array, *, index, shape, shared=None) -> TensorValue:
    return _trace("load").load(array, index, shape, shared)


def load_conv2d(array, filter_value, *, index, shape, group=1, pad, stride, dilation):
    return _trace("load_conv2d").load_conv2d(
        array, filter_value, index, shape, group=group, pad=pad, stride=stride, dilation=dilation
    )


def store(array, *, index, tile) -> None:
    _trace("store").store(array, index, tile)


def max(input_value, axis: int = -1):  # noqa: A001 - mirrors the reference name
    return _trace("max").reduce_max(input_value, axis=axis)


def sum(input_value, axis: int = -1):  # noqa: A001 - mirrors the reference name
    return _trace("sum").reduce_sum(input_value, axis=axis)


def sub(lhs, rhs):
    return _trace("sub").sub(lhs, rhs)


def add(lhs, rhs):
    return _trace("add").add(lhs, rhs)


def mul(lhs, rhs):
    return _trace("mul").mul(lhs, rhs)


def truediv(lhs, rhs):
    ctx = _trace("truediv")
    if not isinstance(rhs, TensorValue):
        raise TypeError("xt.truediv currently requires a tensor rhs")
    return ctx.truediv(lhs, rhs)


def exp(v):
    return _trace("exp").exp(v)


def cos(v):
    return _trace("cos").cos(v)


def sin(v):
    return _trace("sin").sin(v)


def reciprocal(v):
    return _trace("reciprocal").reciprocal(v)


def rsqrt(v):
    return _trace("rsqrt").rsqrt(v)


def sigmoid(v):
    return _trace("sigmoid").sigmoid(v)


def tanh(v):
    return _trace("tanh").tanh(v)


def silu(v):
    return _trace("silu").silu(v)


def matmul(lhs, rhs):
    return _trace("matmul").matmul(lhs, rhs)


def mma(lhs, rhs, acc):
    return _trace("mma").mma(lhs, rhs, acc)


def astype(input_value, *, dtype):
    return _trace("astype").astype(input_value, dtype)


def reshape(input_value, *, shape):
    return _trace("reshape").reshape(input_value, shape)


def transpose(input_value):
    return _trace("transpose").transpose(input_value)


def rms_norm(value, gamma, *, eps: float = 1e-6, dtype: DType | None = None):
    """`value / sqrt(mean(value ** 2) + eps) * gamma`, row by row: a (R, C) tile and
    a (1, C) gamma.  Held in 32 bits, rounded once where it is stored."""
    return _trace("rms_norm").rms_norm(value, gamma, eps=eps, dtype=dtype)


def row_scale(value):
    """(R, 1) float32 scales of a tile's rows in 8 bits: the largest magnitude of
    a row over 127."""
    return _trace("row_scale").row_scale(value)


def quantize(value, scale):
    """`value / scale` to the nearest int8 (half to even), at most 127 in
    magnitude; 0 in rows whose scale is 0 and where the quotient is NaN."""
    return _trace("quantize").quantize(value, scale)


def matmul_q4(value, weight, scales, *, row_scale=None, dtype: DType = float32):
    """`value @ w.T` with 4-bit weights: value (M, K), weight (N, K / 2) int8 as
    `pack_q4` lays them out, scales (N, K / G) with one scale a group of G weights
    of a row.  `row_scale` (M, 1) multiplies the rows of the result: with the int8
    rows of `quantize` it is their scale.  Sums are held in 32 bits, of values up to
    2**115; a row of `value` with an infinity or NaN is NaN."""
    return _trace("matmul_q4").matmul_q4(value, weight, scales, row_scale=row_scale, dtype=dtype)


def mx4_scale(value):
    """(R, C / 32) int8 scales of rows in microscaled 4-bit floating point: of each
    block of 32 neighbours the byte e + 127 (0 to 254 unsigned) of the power 2**e that
    the block's values are multiples of, e = floor(log2(largest magnitude)) - 2, at
    least -127; 0 for a block of zeros, 255 for one with an infinity or NaN."""
    return _trace("mx4_scale").mx4_scale(value)


def quantize_mx4(value, scale):
    """(R, C / 2) int8 rows: `value / 2**e` of each block of 32, with the `scale` that
    mx4_scale gave for them, to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4 and 6 with a
    sign (halfway to the one whose last bit is 0; magnitudes above 6 are 6).  Two
    values a byte, the first in the lower half: sign, two bits of exponent, one of
    mantissa.  All 0 in blocks with an infinity or NaN."""
    return _trace("quantize_mx4").quantize_mx4(value, scale)


def dequantize_mx4(value, scale, *, dtype: DType = float32):
    """The (R, C) values of rows of quantize_mx4 and their scales, rounded once to
    `dtype`; NaN in blocks whose scale is 255."""
    return _trace("dequantize_mx4").dequantize_mx4(value, scale, dtype=dtype)


def matmul_mx4(value, value_scale, weight, weight_scale, *, dtype: DType = float32):
    """`value @ weight.T` of rows in microscaled 4-bit floating point: value (M, K / 2)
    and weight (N, K / 2) with scales (M, K / 32) and (N, K / 32), as quantize_mx4
    and mx4_scale give them.  Sums are held in 32 bits (parts of one past float32's largest
    make infinities or NaN); a row with a scale of 255 is NaN."""
    return _trace("matmul_mx4").matmul_mx4(value, value_scale, weight, weight_scale, dtype=dtype)


def sample(logits, uniform, *, temperature=None, top_k=None, top_p=None, min_p=None):
    """(R, 1) int32 tokens, one drawn from each row of (R, V) logits.

    A token's weight is `exp((logit - largest) / temperature)`; temperatures of 0
    or less, and NaN, leave the largest logits alone, and logits of plus infinity
    leave nothing but themselves.  Tokens are ordered by logit, the largest first,
    equal ones by index.  Of the order's beginning remain: the first `top_k` tokens
    (0 or less: all); of those the fewest whose weights reach `top_p` of their total
    (1 or more, and NaN: all; at least one); and those whose weight is at least
    `min_p` of the largest (above 1: as 1; NaN: as 0).  The result is the first whose
    weights, summed in that order, exceed `uniform` times the sum of what remains:
    `uniform` is held within 0 and what is just below 1, NaN as 0.

    Weights are whole numbers of units in 64 bits, and their sums exact: 2**S units are
    the largest's, S = 61 less the bits of V - 1 and at most 50 (44 for 131072 logits).
    Each is off by half a unit and 3e-13 of itself at most, so a token below half a
    unit is never drawn.  V such tokens are less than 2**-24 of the largest's weight,
    the step of a float32 uniform next to 1, up to 2**19 logits, and 2**-18 at 2**22,
    the most that the kernel takes.  Logits of NaN count as minus infinity, and a row of nothing
    else gives -1.  All but the logits are (R, 1) tiles, float32 or, top_k, int32."""
    return _trace("sample").sample(logits, uniform, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)


def attend(q, k, v, *, scale, cap=None, causal=False, window=None, slopes=None, start=None, length=None, prefix=None,
           q_docs=None, k_docs=None, parents=None):
    """`softmax(scores) v` over the keys that each query row sees.

    q is (heads, rows, D) or (rows, heads * D); its heads share k and v, (keys,
    D).  Row t of q is at position `start + t` (start: a (1, 1) int32 tile, 0
    without it), key j at position j.  The score of a pair is `scale * q . k`,
    with `cap` `cap * tanh(score / cap)`, less `slopes[head] * distance` with
    `slopes`, a (1, heads) float32 tile.  Row at p sees key j when all hold:
    j < length (a (1, 1) int32 tile); their documents are equal (q_docs (1,
    rows), k_docs (1, keys), int32); and j < prefix (a (1, 1) int32 tile), or
    j <= p if `causal` and p - j < window if `window` is given.  Rows that see
    nothing, or only scores of minus infinity, are 0.  What hidden keys and
    values hold, NaN included, has no effect.  Scores, maxima, totals and sums are held
    in 32 bits; a softmax weight is rounded to v's type, in its product with v and in the
    total alike.

    With `parents`, a (1, rows) int32 tile, the rows are a tree of drafted tokens
    that follows the keys before `start`, and key start + u is drafted token u's.
    parents[t] is the drafted token that t continues, one before t; any other
    value is none: t continues the keys before `start`.  Row t is at position
    start + its depth (the number of its ancestors), key start + u at that of token
    u.  Of the drafted tokens a row sees its ancestors and itself (under `window`
    and `length` as above), of the keys behind them none.  Not with `causal`,
    `prefix` or documents."""
    return _trace("attend").attend(q, k, v, scale, cap=cap, causal=causal, window=window, slopes=slopes, start=start,
                                   length=length, prefix=prefix, q_docs=q_docs, k_docs=k_docs, parents=parents)


def convert(kernel_fn, *, args, grid, double_buffering, parse_module):
    """Trace `kernel_fn` once and hand the emitted text to `parse_module`."""
    global _ACTIVE_TRACE
    if not isinstance(kernel_fn, KernelFunction):
        raise TypeError("xt.convert expects a function decorated with @xt.kernel")
    trace = TraceContext(kernel_fn, args, grid, double_buffering)
    outer = _ACTIVE_TRACE
    _ACTIVE_TRACE = trace
    try:
        returned = kernel_fn.fn(*trace.trace_arguments())
    finally:
        _ACTIVE_TRACE = outer
    if returned is not None:
        raise ValueError("xt.kernel functions must not return a value")
    return parse_module(trace.emit_function_asm())
