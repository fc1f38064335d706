"""Mirror of rew's eager ``{.rewOp.}`` procs used on the hot path.

Each function validates like the reference op, then calls ``dispatchEager``
with the same op name and the same stringly-typed attrs in the same wire
format, so the native backend sees exactly what rew would send it:

* ``joinInts`` lists "[a,b]" (src/rew/ops/linalg.nim:21-29, reduce.nim:87-92)
* Nim seq reprs "@[a, b]" for reshape/transpose/slice/iota shapes
  (src/rew/ops/shape.nim:41, 73; concat.nim:94-96; shape.nim:316-320)
* dtype names "float32" for astype (unary.nim:125), "dtInt32" for iota
"""
from __future__ import annotations

from ctypes import c_float
from dataclasses import dataclass
from functools import lru_cache
from math import copysign, prod
from typing import NamedTuple, Sequence

import numpy as np

from . import jit as _jit
from .eager import (DType, Device, Tensor, TensorError, defaultDevice, dispatchEager,
                    fromHost)


def _join(xs: Sequence[int]) -> str:
    return "[" + ",".join(str(int(x)) for x in xs) + "]"


def _nimseq(xs: Sequence[int]) -> str:
    return "@[" + ", ".join(str(int(x)) for x in xs) + "]"


def _one(op, operands, attrs=()):
    if _jit._tls.__dict__.get("trace") is not None:   # trace mode: build the op
        return _jit.traceOp(op, operands, attrs)[0]
    outs = dispatchEager(op, operands, attrs)
    assert len(outs) == 1, f"{op}: eager backend returned wrong arity"
    return outs[0]


def _same(a: Tensor, b: Tensor, op: str):
    # src/rew/ops/arith.nim:21-28
    if a.device != b.device:
        raise TensorError(f"{op}: device mismatch")
    if a.dtype != b.dtype:
        raise TensorError(f"{op}: dtype mismatch ({a.dtype.enum_name} vs {b.dtype.enum_name})")
    if a.shape != b.shape:
        raise TensorError(f"{op}: shape mismatch")


# ---- literals (src/rew/ops/literal.nim:56-194) -------------------------------------

def constant(dtype: DType, shape: Sequence[int], data, device: Device | None = None) -> Tensor:
    if _jit.currentMode() == "trace":
        return _jit.traceConstant(dtype, shape, data)
    return fromHost(np.asarray(data), dtype=dtype, shape=shape, device=device)


def scalarF32(v: float, device: Device | None = None) -> Tensor:
    if _jit.currentMode() == "trace":
        return _jit.traceConstant(DType.FLOAT32, (), np.float32(v))
    return fromHost(np.array(v, dtype=np.float32), DType.FLOAT32, (), device)


def scalarI32(v: int, device: Device | None = None) -> Tensor:
    if _jit.currentMode() == "trace":
        return _jit.traceConstant(DType.INT32, (), np.int32(v))
    return fromHost(np.array(v, dtype=np.int32), DType.INT32, (), device)


def constantF32(shape: Sequence[int], data, device: Device | None = None) -> Tensor:
    a = np.asarray(data, dtype=np.float32)
    n = int(np.prod(shape)) if len(shape) else 1
    if a.size != n:
        raise TensorError(f"constantF32: data length {a.size} does not match shape product {n}")
    if _jit.currentMode() == "trace":
        return _jit.traceConstant(DType.FLOAT32, shape, a)
    return fromHost(a, DType.FLOAT32, shape, device)


def zeros(shape: Sequence[int], dtype: DType = DType.FLOAT32,
          device: Device | None = None) -> Tensor:
    """A zero scalar constant broadcast to `shape` (src/rew/ops/factory.nim:17-24)."""
    scalar = constant(dtype, [], np.zeros(1, np.float32), device)
    if len(shape) == 0:
        return scalar
    return broadcastTo(scalar, list(shape), [])


def zerosLike(t: Tensor, dtype: DType | None = None) -> Tensor:
    """src/rew/ops/factory.nim:26-28."""
    return zeros(t.shape, t.dtype if dtype is None else dtype, t.device)


# ---- elementwise (src/rew/ops/arith.nim, unary.nim) ---------------------------------

def _binary(name):
    def f(a: Tensor, b: Tensor) -> Tensor:
        _same(a, b, name)
        return _one(name, [a, b])
    f.__name__ = name
    return f


add = _binary("add")
sub = _binary("sub")
mul = _binary("mul")
divide = _binary("divide")
maximum = _binary("maximum")
minimum = _binary("minimum")
power = _binary("power")
remainder = _binary("remainder")
atan2 = _binary("atan2")
bitwiseAnd = _binary("bitwiseAnd")
bitwiseOr = _binary("bitwiseOr")
bitwiseXor = _binary("bitwiseXor")


def _unary(name):
    def f(a: Tensor) -> Tensor:
        return _one(name, [a])
    f.__name__ = name
    return f


neg = _unary("neg")
abs_ = _unary("abs")
exp = _unary("exp")
log = _unary("log")
sqrt = _unary("sqrt")
rsqrt = _unary("rsqrt")
tanh = _unary("tanh")
logistic = _unary("logistic")
sine = _unary("sine")
cosine = _unary("cosine")
floor = _unary("floor")
ceil = _unary("ceil")
sign = _unary("sign")
isFinite = _unary("isFinite")
cbrt = _unary("cbrt")
expm1 = _unary("expm1")
log1p = _unary("log1p")
tan = _unary("tan")
roundNearestAfz = _unary("roundNearestAfz")
roundNearestEven = _unary("roundNearestEven")
bitwiseNot = _unary("bitwiseNot")


def astype(a: Tensor, dtype: DType) -> Tensor:
    return _one("astype", [a], [("dtype", DType(dtype).rew_name)])


def clamp(lo: Tensor, x: Tensor, hi: Tensor) -> Tensor:
    return _one("clamp", [lo, x, hi])


# ---- shape ops (src/rew/ops/shape.nim, concat.nim, linalg.nim) ----------------------

def reshape(a: Tensor, newShape: Sequence[int]) -> Tensor:
    for d in newShape:
        if d <= 0:
            raise TensorError(f"reshape: shape contains non-positive dim {d}")
    n = 1
    for d in newShape:
        n *= d
    if n != a.numElements:
        raise TensorError(
            f"reshape: element count mismatch — operand has {a.numElements} elements, "
            f"target shape has {n}")
    return _one("reshape", [a], [("shape", _nimseq(newShape))])


def transpose(a: Tensor, permutation: Sequence[int]) -> Tensor:
    if len(permutation) != len(a.shape):
        raise TensorError(
            f"transpose: permutation length {len(permutation)} does not match operand rank "
            f"{len(a.shape)}")
    if sorted(permutation) != list(range(len(a.shape))):
        raise TensorError("transpose: invalid permutation")
    return _one("transpose", [a], [("permutation", _nimseq(permutation))])


def broadcastTo(t: Tensor, outputShape: Sequence[int],
                broadcastDimensions: Sequence[int]) -> Tensor:
    if len(broadcastDimensions) != len(t.shape):
        raise TensorError("broadcastTo: broadcastDimensions length must match operand rank")
    for i, od in enumerate(broadcastDimensions):
        if t.shape[i] != 1 and t.shape[i] != outputShape[od]:
            raise TensorError("broadcastTo: operand dim is not 1 and does not match")
    return _one("broadcastTo", [t], [("output_shape", _join(outputShape)),
                                     ("broadcast_dimensions", _join(broadcastDimensions))])


def slice_(t: Tensor, startIndices: Sequence[int], limitIndices: Sequence[int],
           strides: Sequence[int] = ()) -> Tensor:
    rank = len(t.shape)
    if len(startIndices) != rank or len(limitIndices) != rank:
        raise TensorError(f"slice: index arrays must match operand rank {rank}")
    st = list(strides) if len(strides) else [1] * rank
    for i in range(rank):
        if (startIndices[i] < 0 or limitIndices[i] > t.shape[i]
                or startIndices[i] >= limitIndices[i] or st[i] <= 0):
            raise TensorError(f"slice: invalid bounds at dim {i}")
    return _one("slice", [t], [("start_indices", _nimseq(startIndices)),
                               ("limit_indices", _nimseq(limitIndices)),
                               ("strides", _nimseq(st))])


def concat(tensors: Sequence[Tensor], dimension: int) -> Tensor:
    if not tensors:
        raise TensorError("concat: empty input list")
    return _one("concat", list(tensors), [("dimension", str(dimension))])


def iota(dtype: DType, shape: Sequence[int], dimension: int,
         device: Device | None = None) -> Tensor:
    if dtype == DType.BOOL:
        raise TensorError("iota: bool dtype is not supported")
    if dimension < 0 or dimension >= len(shape):
        raise TensorError(f"iota: dimension {dimension} out of range for rank {len(shape)}")
    d = device or defaultDevice()
    return _one("iota", [], [("dtype", DType(dtype).enum_name), ("shape", _nimseq(shape)),
                             ("dimension", str(dimension)), ("device", str(d))])


def unsqueeze(a: Tensor, dim: int) -> Tensor:
    s = list(a.shape)
    s.insert(dim, 1)
    return reshape(a, s)


def compare(lhs: Tensor, rhs: Tensor, direction: str) -> Tensor:
    if direction not in ("LT", "LE", "GT", "GE", "EQ", "NE"):
        raise TensorError(f"compare: invalid direction '{direction}'")
    return _one("compare", [lhs, rhs], [("comparison_direction", direction)])


def select(pred: Tensor, onTrue: Tensor, onFalse: Tensor) -> Tensor:
    if pred.dtype != DType.BOOL:
        raise TensorError(f"select: pred must be bool, got {pred.dtype.enum_name}")
    return _one("select", [pred, onTrue, onFalse])


# ---- reductions (src/rew/ops/reduce.nim:93-225) --------------------------------------

def _norm_dims(op: str, rank: int, dims: Sequence[int]) -> list[int]:
    out = []
    for d in dims:
        p = d + rank if d < 0 else d
        if p < 0 or p >= rank:
            raise TensorError(f"{op}: dim {d} out of range for rank {rank}")
        if p in out:
            raise TensorError(f"{op}: dim {d} repeated")
        out.append(p)
    return out


def _reduction(op: str, t: Tensor, dims: Sequence[int]) -> Tensor:
    rd = _norm_dims(op, len(t.shape), dims)
    if t.dtype != DType.FLOAT32:
        raise TensorError(f"{op}: v1 supports only float32 (got {t.dtype.enum_name})")
    return _one(op, [t], [("dims", _join(rd))])


def reduceSum(t: Tensor, dims: Sequence[int]) -> Tensor:
    return _reduction("reduceSum", t, dims)


def reduceMax(t: Tensor, dims: Sequence[int]) -> Tensor:
    return _reduction("reduceMax", t, dims)


def reduceMin(t: Tensor, dims: Sequence[int]) -> Tensor:
    return _reduction("reduceMin", t, dims)


def reduceProd(t: Tensor, dims: Sequence[int]) -> Tensor:
    return _reduction("reduceProd", t, dims)


def reduceMean(t: Tensor, dims: Sequence[int]) -> Tensor:
    # src/rew/ops/reduce.nim:132-150: reduceSum then divide by broadcast n.
    rd = _norm_dims("reduceMean", len(t.shape), dims)
    summed = reduceSum(t, rd)
    n = 1
    for d in rd:
        n *= t.shape[d]
    if n <= 0:
        raise TensorError(f"reduceMean: empty reduction (n = {n})")
    divisor = scalarF32(float(n), t.device)
    if len(summed.shape) == 0:
        return divide(summed, divisor)
    return divide(summed, broadcastTo(divisor, summed.shape, []))


def argmax(t: Tensor, dim: int) -> Tensor:
    """Index of the maximum along ``dim``; ties go to the smallest index.

    rew's composite (src/rew/ops/reduce.nim:202-225) raises at its int32
    ``reduceMin`` (fp32-only guard, reduce.nim:66-69); the backend runs the
    documented semantics as one native op instead, including the
    composite's NaN behaviour (a row containing NaN yields int32.high).
    """
    pos = dim + len(t.shape) if dim < 0 else dim
    if pos < 0 or pos >= len(t.shape):
        raise TensorError(f"argmax: dim {dim} out of range for rank {len(t.shape)}")
    if _jit.currentMode() == "trace":
        # rew's composite, which stops at the int32 reduceMin as rew's does
        m = reduceMax(t, [pos])
        mask = compare(t, broadcastTo(m, t.shape, [i for i in range(len(t.shape)) if i != pos]),
                       "EQ")
        ids = iota(DType.INT32, t.shape, pos, t.device)
        big = broadcastTo(scalarI32(2**31 - 1, t.device), t.shape, [])
        return reduceMin(select(mask, ids, big), [pos])
    return _one("argmax", [t], [("dimension", str(pos))])


def topK(operand: Tensor, k: int, dimension: int = -1, largest: bool = True):
    """(values, indices) of the k largest along the last dim, largest first,
    ties to the lower index (src/rew/ops/sort.nim:36-90 semantics; eager here,
    trace-only in the reference)."""
    if k <= 0:
        raise TensorError(f"topK: k must be positive, got {k}")
    rank = len(operand.shape)
    d = dimension + rank if dimension < 0 else dimension
    if k > operand.shape[d]:
        raise TensorError(f"topK: k {k} > dim size {operand.shape[d]}")
    if _jit.currentMode() == "trace":
        return _jit.traceTopK(operand, k, d, largest)
    outs = dispatchEager("topK", [operand], [("k", str(k)), ("dimension", str(d)),
                                             ("largest", "true" if largest else "false")])
    return outs[0], outs[1]


def sort(operand: Tensor, dimension: int = -1, isStable: bool = False,
         comparator: str = "LT", *others: Tensor):
    """Sorts along ``dimension`` (src/rew/ops/sort.nim:13-33).  rew takes the
    comparator as a builder callback; here it is the one compare direction
    such a callback emits on the operand pair ("LT"/"LE" ascending, "GT"/"GE"
    descending).  ``others`` are permuted along with ``operand`` (the
    multi-operand form of stablehlo.sort).  Trace-only in the reference; the
    backend also runs it eagerly (stable, NaN last)."""
    if comparator not in ("LT", "LE", "GT", "GE"):
        raise TensorError(f"sort: comparator must be LT, LE, GT or GE, got '{comparator}'")
    rank = len(operand.shape)
    d = dimension + rank if dimension < 0 else dimension
    if d < 0 or d >= rank:
        raise TensorError(f"sort: dimension {dimension} out of range for rank {rank}")
    ins = [operand, *others]
    if _jit.currentMode() == "trace":
        res = _jit.traceSort(ins, d, isStable, comparator)
    else:
        res = dispatchEager("sort", ins, [("dimension", str(d)),
                                          ("comparison_direction", comparator),
                                          ("is_stable", "true" if isStable else "false")])
    return res[0] if not others else res


@dataclass
class GatherDimensionNumbers:
    """src/rew/stablehlo/ops.nim:60-68."""
    offsetDims: Sequence[int]
    collapsedSliceDims: Sequence[int]
    startIndexMap: Sequence[int]
    indexVectorDim: int
    operandBatchingDims: Sequence[int] = ()
    startIndicesBatchingDims: Sequence[int] = ()


@dataclass
class ScatterDimensionNumbers:
    """src/rew/stablehlo/ops.nim:70-77."""
    updateWindowDims: Sequence[int]
    insertedWindowDims: Sequence[int]
    scatterDimsToOperandDims: Sequence[int]
    indexVectorDim: int
    inputBatchingDims: Sequence[int] = ()
    scatterIndicesBatchingDims: Sequence[int] = ()


def gather(operand: Tensor, startIndices: Tensor, dims: GatherDimensionNumbers,
           sliceSizes: Sequence[int], resultShape: Sequence[int],
           indicesAreSorted: bool = False) -> Tensor:
    """stablehlo.gather (src/rew/ops/gather.nim:10-28).  Trace-only in the
    reference; the backend also runs it eagerly (start indices clamped)."""
    if _jit.currentMode() == "trace":
        return _jit.traceGather(operand, startIndices, dims, sliceSizes, resultShape,
                                indicesAreSorted)
    out = _one("gather", [operand, startIndices], [
        ("offset_dims", _join(dims.offsetDims)),
        ("collapsed_slice_dims", _join(dims.collapsedSliceDims)),
        ("operand_batching_dims", _join(dims.operandBatchingDims)),
        ("start_indices_batching_dims", _join(dims.startIndicesBatchingDims)),
        ("start_index_map", _join(dims.startIndexMap)),
        ("index_vector_dim", str(dims.indexVectorDim)),
        ("slice_sizes", _join(sliceSizes))])
    if list(out.shape) != list(resultShape):
        raise TensorError(f"gather: resultShape {list(resultShape)} does not match the "
                          f"dimension numbers ({list(out.shape)})")
    return out


_UPDATES = ("replace", "add", "maximum", "minimum", "multiply")


def scatter(inputs: Sequence[Tensor], scatterIndices: Tensor, updates: Sequence[Tensor],
            dims: ScatterDimensionNumbers, updateComputation: str = "add",
            indicesAreSorted: bool = False, uniqueIndices: bool = False) -> list:
    """stablehlo.scatter (src/rew/ops/scatter.nim:10-39).  rew takes the update
    computation as a builder callback; here it names the one op such a
    callback emits on (current, update): "add", "maximum", "minimum",
    "multiply", or "replace" (the callback returns the update).  Updates of
    one element in several places combine in an unspecified order (atomics).
    Trace-only in the reference; the backend also runs one-input scatters
    eagerly."""
    if not inputs or len(inputs) != len(updates):
        raise TensorError("scatter: inputs and updates must have the same non-zero length")
    if updateComputation not in _UPDATES:
        raise TensorError(f"scatter: update computation must be one of {_UPDATES}")
    if _jit.currentMode() == "trace":
        return _jit.traceScatter(list(inputs), scatterIndices, list(updates), dims,
                                 updateComputation, indicesAreSorted, uniqueIndices)
    if len(inputs) != 1:
        raise TensorError("scatter: the backend runs one-input scatters only")
    return [_one("scatter", [inputs[0], scatterIndices, updates[0]], [
        ("update_window_dims", _join(dims.updateWindowDims)),
        ("inserted_window_dims", _join(dims.insertedWindowDims)),
        ("input_batching_dims", _join(dims.inputBatchingDims)),
        ("scatter_indices_batching_dims", _join(dims.scatterIndicesBatchingDims)),
        ("scatter_dims_to_operand_dims", _join(dims.scatterDimsToOperandDims)),
        ("index_vector_dim", str(dims.indexVectorDim)),
        ("update_computation", updateComputation)])]


def indexSelect(operand: Tensor, index: Tensor, dim: int = 0, batchDims: int = 0) -> Tensor:
    """src/rew/ops/gather.nim:55-81: torch_index_select in trace mode; the
    backend also runs it eagerly (as torchIndexSelect)."""
    if dim < 0 or dim >= len(operand.shape):
        raise TensorError(f"indexSelect: dim {dim} out of range for operand rank "
                          f"{len(operand.shape)}")
    return torchIndexSelect(operand, index, dim, batchDims)


# ---- linear algebra (src/rew/ops/linalg.nim:204-256, 432-461) -------------------------

def dotGeneral(a: Tensor, b: Tensor, lhsBatching: Sequence[int], rhsBatching: Sequence[int],
               lhsContracting: Sequence[int], rhsContracting: Sequence[int]) -> Tensor:
    if a.dtype != b.dtype:
        raise TensorError(
            f"dotGeneral: dtype mismatch ({a.dtype.enum_name} vs {b.dtype.enum_name})")
    return _one("dotGeneral", [a, b], [("lhs_batching", _join(lhsBatching)),
                                       ("rhs_batching", _join(rhsBatching)),
                                       ("lhs_contracting", _join(lhsContracting)),
                                       ("rhs_contracting", _join(rhsContracting))])


def matmul(a: Tensor, b: Tensor) -> Tensor:
    if len(a.shape) != 2 or len(b.shape) != 2:
        raise TensorError(
            f"matmul: expected rank-2 operands, got shapes {list(a.shape)} and {list(b.shape)}")
    if a.shape[1] != b.shape[0]:
        raise TensorError(f"matmul: inner dim mismatch — {list(a.shape)} * {list(b.shape)}")
    return dotGeneral(a, b, [], [], [1], [0])


def dot(a: Tensor, b: Tensor) -> Tensor:
    return _one("dot", [a, b])


def torchIndexSelect(operand: Tensor, index: Tensor, dim: int, batchDims: int) -> Tensor:
    if index.dtype not in (DType.INT8, DType.INT16, DType.INT32, DType.INT64, DType.UINT8,
                           DType.UINT16, DType.UINT32, DType.UINT64):
        raise TensorError("torchIndexSelect: index must be an integer tensor")
    return _one("torchIndexSelect", [operand, index], [("dim", str(dim)),
                                                        ("batch_dims", str(batchDims))])


# ---- shape, dynamic and linear-algebra ops outside the configs -------------------------
# src/rew/ops/shape.nim:108-475, ops/distributed.nim:11-35, ops/linalg.nim:177-202

_INT_DTYPES = {DType.INT4, DType.INT8, DType.INT16, DType.INT32, DType.INT64, DType.UINT4,
               DType.UINT8, DType.UINT16, DType.UINT32, DType.UINT64}


def getDimensionSize(a: Tensor, dimension: int) -> Tensor:
    if dimension < 0 or dimension >= len(a.shape):
        raise TensorError(f"getDimensionSize: dimension {dimension} out of range for rank "
                          f"{len(a.shape)}")
    return _one("getDimensionSize", [a], [("dimension", str(dimension))])


def pad(a: Tensor, paddingValue: Tensor, edgePaddingLow: Sequence[int],
        edgePaddingHigh: Sequence[int], interiorPadding: Sequence[int]) -> Tensor:
    if paddingValue.dtype != a.dtype or len(paddingValue.shape) != 0:
        raise TensorError(f"pad: paddingValue must be scalar with dtype {a.dtype.rew_name}")
    rank = len(a.shape)
    if not (len(edgePaddingLow) == len(edgePaddingHigh) == len(interiorPadding) == rank):
        raise TensorError(f"pad: padding arrays must match operand rank {rank}")
    for i, d in enumerate(a.shape):
        if interiorPadding[i] < 0:
            raise TensorError(f"pad: interior padding at dim {i} must be non-negative")
        if d + edgePaddingLow[i] + edgePaddingHigh[i] + max(d - 1, 0) * interiorPadding[i] < 0:
            raise TensorError(f"pad: result dimension {i} is negative")
    return _one("pad", [a, paddingValue], [("edge_padding_low", _nimseq(edgePaddingLow)),
                                           ("edge_padding_high", _nimseq(edgePaddingHigh)),
                                           ("interior_padding", _nimseq(interiorPadding))])


def _start_indices(a: Tensor, startIndices: Sequence[Tensor], op: str):
    if len(startIndices) != len(a.shape):
        raise TensorError(f"{op}: start index count {len(startIndices)} must match operand "
                          f"rank {len(a.shape)}")
    for i, idx in enumerate(startIndices):
        if idx.device != a.device:
            raise TensorError(f"{op}: device mismatch")
        if idx.dtype not in _INT_DTYPES or len(idx.shape) != 0:
            raise TensorError(f"{op}: start index #{i} must be an integer scalar")


def dynamicSlice(a: Tensor, startIndices: Sequence[Tensor], sliceSizes: Sequence[int]) -> Tensor:
    _start_indices(a, startIndices, "dynamicSlice")
    if len(sliceSizes) != len(a.shape):
        raise TensorError(f"dynamicSlice: sliceSizes length {len(sliceSizes)} must match "
                          f"operand rank {len(a.shape)}")
    for i, s in enumerate(sliceSizes):
        if s < 0 or s > a.shape[i]:
            raise TensorError(f"dynamicSlice: slice size {s} out of range for dim {i}")
    return _one("dynamicSlice", [a, *startIndices], [("slice_sizes", _nimseq(sliceSizes))])


def dynamicUpdateSlice(a: Tensor, update: Tensor, startIndices: Sequence[Tensor]) -> Tensor:
    if update.dtype != a.dtype:
        raise TensorError("dynamicUpdateSlice: update dtype must match operand dtype")
    if len(update.shape) != len(a.shape):
        raise TensorError("dynamicUpdateSlice: update rank must match operand rank")
    for i, (u, d) in enumerate(zip(update.shape, a.shape)):
        if u > d:
            raise TensorError(f"dynamicUpdateSlice: update dim {i} exceeds operand dim")
    _start_indices(a, startIndices, "dynamicUpdateSlice")
    return _one("dynamicUpdateSlice", [a, update, *startIndices])


def replicaId(device: Device | None = None) -> Tensor:
    return _one("replicaId", [], [("device", str(device or defaultDevice()))])


def partitionId(device: Device | None = None) -> Tensor:
    return _one("partitionId", [], [("device", str(device or defaultDevice()))])


def setDimensionSize(a: Tensor, size: Tensor, dimension: int) -> Tensor:
    if dimension < 0 or dimension >= len(a.shape):
        raise TensorError(f"setDimensionSize: dimension {dimension} out of range for rank "
                          f"{len(a.shape)}")
    if size.dtype not in _INT_DTYPES or len(size.shape) != 0:
        raise TensorError("setDimensionSize: size must be an integer scalar")
    return _one("setDimensionSize", [a, size], [("dimension", str(dimension))])


def dynamicReshape(a: Tensor, outputShape: Tensor, resultShape: Sequence[int]) -> Tensor:
    if outputShape.dtype not in _INT_DTYPES or tuple(outputShape.shape) != (len(resultShape),):
        raise TensorError(f"dynamicReshape: outputShape must be an integer vector of length "
                          f"{len(resultShape)}")
    if any(d < 0 for d in resultShape):
        raise TensorError("dynamicReshape: result shape contains negative dim")
    if int(np.prod(resultShape, dtype=np.int64)) != int(np.prod(a.shape, dtype=np.int64)):
        raise TensorError("dynamicReshape: result element count does not match operand")
    return _one("dynamicReshape", [a, outputShape], [("result_shape", _nimseq(resultShape))])


def dynamicIota(dtype: DType, outputShape: Tensor, resultShape: Sequence[int],
                dimension: int) -> Tensor:
    if dtype == DType.BOOL:
        raise TensorError("dynamicIota: bool dtype is not supported")
    if outputShape.dtype not in _INT_DTYPES or tuple(outputShape.shape) != (len(resultShape),):
        raise TensorError(f"dynamicIota: outputShape must be an integer vector of length "
                          f"{len(resultShape)}")
    if dimension < 0 or dimension >= len(resultShape):
        raise TensorError(f"dynamicIota: dimension {dimension} out of range for rank "
                          f"{len(resultShape)}")
    return _one("dynamicIota", [outputShape], [("dtype", DType(dtype).enum_name),
                                                ("result_shape", _nimseq(resultShape)),
                                                ("dimension", str(dimension))])


def cholesky(a: Tensor, lower: bool = True) -> Tensor:
    if a.dtype not in (DType.FLOAT16, DType.BFLOAT16, DType.FLOAT32, DType.FLOAT64):
        raise TensorError(f"cholesky: operand must be floating point, got {a.dtype.rew_name}")
    if len(a.shape) < 2:
        raise TensorError(f"cholesky: operand rank must be at least 2, got {len(a.shape)}")
    if a.shape[-1] != a.shape[-2]:
        raise TensorError(f"cholesky: innermost matrix dimensions must be square, got "
                          f"{list(a.shape)}")
    return _one("cholesky", [a], [("lower", "true" if lower else "false")])


# ---- batch norm (src/rew/ops/normalization.nim:40-205) ----------------------------------

def _bn_feature_index(operand: Tensor, featureIndex: int, op: str) -> list:
    if operand.dtype not in (DType.FLOAT16, DType.BFLOAT16, DType.FLOAT32, DType.FLOAT64):
        raise TensorError(f"{op}: operand must be floating point, got {operand.dtype.rew_name}")
    if featureIndex < 0 or featureIndex >= len(operand.shape):
        raise TensorError(f"{op}: featureIndex {featureIndex} out of range for rank "
                          f"{len(operand.shape)}")
    return [operand.shape[featureIndex]]


def _bn_feature(operand: Tensor, t: Tensor, name: str, fshape, op: str):
    if t.device != operand.device:
        raise TensorError(f"{op}: device mismatch")
    if t.dtype != operand.dtype:
        raise TensorError(f"{op}: {name} dtype {t.dtype.rew_name} differs from operand dtype "
                          f"{operand.dtype.rew_name}")
    if list(t.shape) != list(fshape):
        raise TensorError(f"{op}: {name} shape {list(t.shape)} must be {list(fshape)}")


def _bn_attrs(epsilon: float, featureIndex: int):
    return [("epsilon", repr(float(np.float32(epsilon)))), ("feature_index", str(featureIndex))]


def batchNormInference(operand: Tensor, scale: Tensor, offset: Tensor, mean: Tensor,
                       variance: Tensor, epsilon: float, featureIndex: int) -> Tensor:
    fs = _bn_feature_index(operand, featureIndex, "batchNormInference")
    for t, nm in ((scale, "scale"), (offset, "offset"), (mean, "mean"), (variance, "variance")):
        _bn_feature(operand, t, nm, fs, "batchNormInference")
    return _one("batchNormInference", [operand, scale, offset, mean, variance],
                _bn_attrs(epsilon, featureIndex))


def batchNormTraining(operand: Tensor, scale: Tensor, offset: Tensor, epsilon: float,
                      featureIndex: int):
    """(output, batchMean, batchVar)."""
    fs = _bn_feature_index(operand, featureIndex, "batchNormTraining")
    for t, nm in ((scale, "scale"), (offset, "offset")):
        _bn_feature(operand, t, nm, fs, "batchNormTraining")
    outs = dispatchEager("batchNormTraining", [operand, scale, offset],
                         _bn_attrs(epsilon, featureIndex))
    assert len(outs) == 3, "batchNormTraining: eager backend returned wrong arity"
    return tuple(outs)


def batchNormGrad(operand: Tensor, scale: Tensor, mean: Tensor, variance: Tensor,
                  gradOutput: Tensor, epsilon: float, featureIndex: int):
    """(gradOperand, gradScale, gradOffset)."""
    fs = _bn_feature_index(operand, featureIndex, "batchNormGrad")
    if gradOutput.dtype != operand.dtype or list(gradOutput.shape) != list(operand.shape):
        raise TensorError("batchNormGrad: gradOutput type must match operand type")
    for t, nm in ((scale, "scale"), (mean, "mean"), (variance, "variance")):
        _bn_feature(operand, t, nm, fs, "batchNormGrad")
    outs = dispatchEager("batchNormGrad", [operand, scale, mean, variance, gradOutput],
                         _bn_attrs(epsilon, featureIndex))
    assert len(outs) == 3, "batchNormGrad: eager backend returned wrong arity"
    return tuple(outs)


# ---- einsum and the shape-operand ops (src/rew/ops/linalg.nim, shape.nim) -----------

def _join_ints(xs: Sequence[int]) -> str:
    """joinInts (src/rew/ops/linalg.nim:21-29): "[a,b,c]"."""
    return "[" + ",".join(str(int(x)) for x in xs) + "]"


def einsum(a: Tensor, b: Tensor, config: str, outputShape: Sequence[int]) -> Tensor:
    """src/rew/ops/linalg.nim:378-403 (TensorFlow einsum grammar, explicit result shape)."""
    if a.device != b.device:
        raise TensorError("einsum: device mismatch")
    if a.dtype != b.dtype:
        raise TensorError(f"einsum: dtype mismatch ({a.dtype.rew_name} vs {b.dtype.rew_name})")
    if not config:
        raise TensorError("einsum: config must not be empty")
    return _one("einsum", [a, b], [("einsum_config", config),
                                   ("output_shape", _join_ints(outputShape))])


def unaryEinsum(a: Tensor, config: str, outputShape: Sequence[int]) -> Tensor:
    """src/rew/ops/linalg.nim:405-430."""
    if not config:
        raise TensorError("unaryEinsum: config must not be empty")
    return _one("unaryEinsum", [a], [("einsum_config", config),
                                     ("output_shape", _join_ints(outputShape))])


def dynamicBroadcastInDim(t: Tensor, outputDimensions: Tensor, resultShape: Sequence[int],
                          broadcastDimensions: Sequence[int],
                          knownExpandingDimensions: Sequence[int] = (),
                          knownNonexpandingDimensions: Sequence[int] = ()) -> Tensor:
    """src/rew/ops/linalg.nim:288-326."""
    if outputDimensions.dtype not in _INT_DTYPES or \
            tuple(outputDimensions.shape) != (len(resultShape),):
        raise TensorError("dynamicBroadcastInDim: outputDimensions must be an integer vector "
                          f"of length {len(resultShape)}")
    return _one("dynamicBroadcastInDim", [t, outputDimensions],
                [("result_shape", _join_ints(resultShape)),
                 ("broadcast_dimensions", _join_ints(broadcastDimensions)),
                 ("known_expanding_dimensions", _join_ints(knownExpandingDimensions)),
                 ("known_nonexpanding_dimensions", _join_ints(knownNonexpandingDimensions))])


def dynamicPad(a: Tensor, paddingValue: Tensor, edgePaddingLow: Tensor,
               edgePaddingHigh: Tensor, interiorPadding: Tensor,
               resultShape: Sequence[int]) -> Tensor:
    """src/rew/ops/shape.nim:395-441."""
    if paddingValue.dtype != a.dtype or len(paddingValue.shape) != 0:
        raise TensorError(f"dynamicPad: paddingValue must be scalar with dtype {a.dtype.rew_name}")
    for name, t in (("edgePaddingLow", edgePaddingLow), ("edgePaddingHigh", edgePaddingHigh),
                    ("interiorPadding", interiorPadding)):
        if t.dtype not in _INT_DTYPES or tuple(t.shape) != (len(a.shape),):
            raise TensorError(f"dynamicPad: {name} must be an integer vector of length "
                              f"{len(a.shape)}")
    return _one("dynamicPad", [a, paddingValue, edgePaddingLow, edgePaddingHigh, interiorPadding],
                [("result_shape", _nimseq(resultShape))])


def realDynamicSlice(a: Tensor, startIndices: Tensor, limitIndices: Tensor, strides: Tensor,
                     resultShape: Sequence[int]) -> Tensor:
    """src/rew/ops/shape.nim:477-517."""
    for name, t in (("startIndices", startIndices), ("limitIndices", limitIndices),
                    ("strides", strides)):
        if t.dtype not in _INT_DTYPES or tuple(t.shape) != (len(a.shape),):
            raise TensorError(f"realDynamicSlice: {name} must be an integer vector of length "
                              f"{len(a.shape)}")
    return _one("realDynamicSlice", [a, startIndices, limitIndices, strides],
                [("result_shape", _nimseq(resultShape))])


def triangularSolve(a: Tensor, b: Tensor, leftSide: bool = True, lower: bool = True,
                    unitDiagonal: bool = False, transposeA: str = "NO_TRANSPOSE") -> Tensor:
    """src/rew/ops/linalg.nim:350-376 (transposeA: NO_TRANSPOSE, TRANSPOSE or ADJOINT)."""
    if a.device != b.device:
        raise TensorError("triangularSolve: device mismatch")
    return _one("triangularSolve", [a, b],
                [("left_side", "true" if leftSide else "false"),
                 ("lower", "true" if lower else "false"),
                 ("unit_diagonal", "true" if unitDiagonal else "false"),
                 ("transpose_a", transposeA)])


# ---- complex parts and the Fourier transform ----------------------------------------

def complex(real: Tensor, imag: Tensor) -> Tensor:  # noqa: A001 (rew's name)
    """src/rew/ops/arith.nim:86-106: float32 / float64 parts -> complex64 / complex128."""
    if real.dtype not in (DType.FLOAT32, DType.FLOAT64):
        raise TensorError(f"complex: operands must be float32 or float64, got {real.dtype.rew_name}")
    return _one("complex", [real, imag])


def real(a: Tensor) -> Tensor:
    """src/rew/ops/unary.nim:184-202."""
    return _one("real", [a])


def imag(a: Tensor) -> Tensor:
    """src/rew/ops/unary.nim:204-224."""
    return _one("imag", [a])


def fft(a: Tensor, fftType: str, fftLength: Sequence[int]) -> Tensor:
    """src/rew/ops/linalg.nim:328-348 (fftType FFT, IFFT, RFFT or IRFFT)."""
    return _one("fft", [a], [("fft_type", fftType), ("fft_length", _join_ints(fftLength))])


# ---- sequences of unequal lengths and their paged cache ---------------------------------
# Backend extensions without a counterpart in the reference, eager only.  Rows of
# all sequences lie one after another (no padding): sequence s owns rows
# [starts[s], starts[s + 1]).  Lengths and tables are device tensors that no call
# reads back; values out of range never reach memory outside the tensors: starts are
# clamped into the rows, and one below an earlier one counts as that one.  Fewer than
# 2^20 sequences, and at most about 2^23 / kvHeads of them.

def _packed_call(op: str, operands, attrs, nouts: int) -> list:
    if _jit.currentMode() == "trace":
        raise TensorError(f"{op}: eager only (it has no StableHLO form)")
    d = operands[0].device
    for t in operands:
        if t.device is not d and t.device != d:
            raise TensorError(f"{op}: device mismatch")
    outs = dispatchEager(op, operands, attrs)
    assert len(outs) == nouts, f"{op}: eager backend returned wrong arity"
    return outs


def _check_i32(op: str, t: Tensor, name: str, shape) -> None:
    """`shape`: the extents, None where any will do."""
    if t.dtype != DType.INT32 or t.shape != shape and (
            len(t.shape) != len(shape) or
            any(w is not None and w != d for w, d in zip(shape, t.shape))):
        want = ["*" if w is None else w for w in shape]
        raise TensorError(f"{op}: {name} must be int32 {want}, got {t.dtype.rew_name} "
                          f"{list(t.shape)}")


def _check_heads(op: str, q: Tensor, dtype: DType, kvHeads: int, headDim: int) -> None:
    if len(q.shape) != 3:
        raise TensorError(f"{op}: q must be [tokens, heads, headDim], got {list(q.shape)}")
    if q.dtype != dtype:
        raise TensorError(f"{op}: dtype mismatch ({q.dtype.enum_name} vs {dtype.enum_name})")
    if q.shape[2] != headDim:
        raise TensorError(f"{op}: head dims of q and k differ ({q.shape[2]} and {headDim})")
    if kvHeads < 1 or q.shape[1] < 1 or q.shape[1] % kvHeads:
        raise TensorError(f"{op}: {q.shape[1]} query heads do not divide among {kvHeads} "
                          "KV heads")


def _check_packed(op: str, q: Tensor, k: Tensor, v: Tensor, starts: Tensor) -> None:
    if len(k.shape) != 3 or k.shape != v.shape or k.dtype != v.dtype:
        raise TensorError(f"{op}: k and v must be [tokens, kvHeads, headDim] of one dtype, got "
                          f"{list(k.shape)} and {list(v.shape)}")
    _check_heads(op, q, k.dtype, k.shape[1], k.shape[2])
    if q.shape[0] != k.shape[0]:
        raise TensorError(f"{op}: q has {q.shape[0]} tokens, k has {k.shape[0]}")
    _check_i32(op, starts, "starts", (None,))
    if starts.shape[0] < 1:
        raise TensorError(f"{op}: starts must hold at least one value")


def _check_pages(op: str, kPages: Tensor, vPages: Tensor) -> int:
    if len(kPages.shape) != 4 or kPages.shape != vPages.shape or kPages.dtype != vPages.dtype:
        raise TensorError(f"{op}: kPages and vPages must be [pages, kvHeads, pageSize, headDim] "
                          f"of one dtype, got {list(kPages.shape)} and {list(vPages.shape)}")
    return _check_page_size(op, kPages.shape[2])


def _check_page_size(op: str, page: int) -> int:
    if page < 1 or page > 65536 or page & (page - 1):
        raise TensorError(f"{op}: page size {page} must be a power of two from 1 to 65536")
    return page


def _attn_attrs(op: str, causal: bool, scale: float) -> list:
    with np.errstate(over="ignore", under="ignore"):
        value = float(np.float32(scale))
    if not 0.0 <= value < float("inf") or (value == 0.0) != (scale == 0.0):
        raise TensorError(f"{op}: scale must be 0 or a positive float32, got {scale}")
    return [("causal", "true" if causal else "false"), ("scale", repr(value))]


class PackedStats(NamedTuple):
    """What ``packedAttention`` leaves for its gradient, beside its result."""
    lse: Tensor   # float32 [tokens, heads]: log of the row's sum of exponentials, -inf for
                  # a row of no sequence
    rest: Tensor  # int8 [tokens, heads, headDim]: what rounding took from the result, in
                  # 1/127 of half a step (bfloat16 2^-8, float16 2^-11) of the row's largest
                  # (float16: of 2^-14 at least)


def packedAttention(q: Tensor, k: Tensor, v: Tensor, starts: Tensor, causal: bool = True,
                    scale: float = 0.0, withLse: bool = False):
    """softmax(scale q k^T) v within each of the packed sequences.

    ``q`` [tokens, heads, headDim]; ``k``, ``v`` [tokens, kvHeads, headDim] (head h reads
    KV head h / (heads / kvHeads)); bfloat16 or float16; headDim 32, 64 or 128; ``starts``
    int32 [sequences + 1] (one below an earlier one counts as that one).  ``causal``: a row
    sees the rows of its sequence up to itself (unlike ``nn.makeCausalMask``, whose
    orientation is the reference's); otherwise all of them.  ``scale`` 0: 1 / sqrt(headDim).
    The softmax is float32; the probabilities are rounded to the operands' dtype before the
    second product, the result once.  A row of no sequence (before ``starts[0]``, behind
    ``starts[-1]``) gives zeros, and so does one whose every score is -infinity.  What a row
    does not see does not reach its result, infinities and NaN included.

    ``withLse``: (out, stats), the ``PackedStats`` that ``packedAttentionGrad`` takes."""
    _check_packed("packedAttention", q, k, v, starts)
    attrs = _attn_attrs("packedAttention", causal, scale)
    attrs.append(("stats", "true" if withLse else "false"))
    res = _packed_call("packedAttention", [q, k, v, starts], attrs, 3 if withLse else 1)
    return (res[0], PackedStats(res[1], res[2])) if withLse else res[0]


def packedAttentionGrad(q: Tensor, k: Tensor, v: Tensor, starts: Tensor, out: Tensor,
                        stats: PackedStats, gradOut: Tensor, causal: bool = True,
                        scale: float = 0.0):
    """(gradQ, gradK, gradV) of ``packedAttention(q, k, v, starts, causal, scale)`` for the
    gradient ``gradOut`` of its result, given its ``out`` and ``stats``.  gradK and gradV are
    summed over the query heads of each KV head; sums are float32 in a fixed order.  What a row
    does not see takes no part, infinities and NaN included: under causality those of a token's
    k and v do not reach gradQ of the rows before it, those of its q and gradOut not gradK and
    gradV of the keys behind it.  Those of gradOut reach gradV in their own columns only."""
    op = "packedAttentionGrad"
    _check_packed(op, q, k, v, starts)
    for t, name in ((out, "out"), (gradOut, "gradOut")):
        if t.dtype != q.dtype or t.shape != q.shape:
            raise TensorError(f"{op}: {name} must have q's dtype and shape")
    lse, rest = stats
    if lse.dtype != DType.FLOAT32 or lse.shape != q.shape[:2]:
        raise TensorError(f"{op}: lse must be float32 [tokens, heads]")
    if rest.dtype != DType.INT8 or rest.shape != q.shape:
        raise TensorError(f"{op}: rest must be int8 of q's shape")
    return tuple(_packed_call(op, [q, k, v, starts, out, lse, rest, gradOut],
                              _attn_attrs(op, causal, scale), 3))


class PagedStep(NamedTuple):
    """The tables of one serving step (``pagedBlockTables``), all int32."""
    blockTable: Tensor  # [requests, blocks]
    slots: Tensor       # [tokens]
    positions: Tensor   # [tokens]
    starts: Tensor      # [requests + 1]
    lens: Tensor        # [requests]
    taken: Tensor       # [1]


def pagedBlockTables(cachedLens: Tensor, newLens: Tensor, blockTable: Tensor,
                     freePages: Tensor, pageSize: int, tokens: int) -> PagedStep:
    """The tables of a serving step that adds ``newLens[r]`` tokens to request r, which has
    ``cachedLens[r]`` tokens in the pages ``blockTable[r]`` (all int32; blockTable
    [requests, blocks]).  Requests that need more pages take them from the front of
    ``freePages``, in request order.  ``tokens``: the sum of newLens, or more.

    Returns (blockTable, slots, positions, starts, lens, taken), all int32:

    * blockTable [requests, blocks]: the pages each request had, then the new ones; -1 behind
      them, and where freePages ran out;
    * slots [tokens]: the cache row page * pageSize + offset of each new token (requests one
      after another), -1 for a token without a page and behind the last token;
    * positions [tokens]: its position in its request (0 behind the last token);
    * starts [requests + 1]: the first new token of each request, then their number;
    * lens [requests]: cachedLens + newLens;
    * taken [1]: the pages needed (more than freePages holds: they ran out).

    Negative lengths count as 0."""
    op = "pagedBlockTables"
    _check_page_size(op, pageSize)
    _check_i32(op, blockTable, "blockTable", (None, None))
    r = blockTable.shape[0]
    _check_i32(op, cachedLens, "cachedLens", (r,))
    _check_i32(op, newLens, "newLens", (r,))
    _check_i32(op, freePages, "freePages", (None,))
    if tokens < 0:
        raise TensorError(f"{op}: tokens must be non-negative, got {tokens}")
    return PagedStep(*_packed_call(op, [cachedLens, newLens, blockTable, freePages],
                                   [("page_size", str(pageSize)), ("tokens", str(tokens))], 6))


def pagedCacheWrite(kPages: Tensor, vPages: Tensor, k: Tensor, v: Tensor,
                    slots: Tensor) -> None:
    """Writes rows t of ``k`` and ``v`` [tokens, kvHeads, headDim] into row ``slots[t]`` of the
    pages [pages, kvHeads, pageSize, headDim], in place: page slots[t] / pageSize, row
    slots[t] % pageSize of every KV head.  A negative slot, or one past the pages, writes
    nothing.  Slots must be distinct: of two tokens in one slot either may stay, in parts.

    The one op that changes its operands: the pages must come from ``eager.empty``, and no
    tensor that shares their memory (a reshape of them) may be alive.  What was recorded before
    reads the old rows, what is recorded later the new ones."""
    op = "pagedCacheWrite"
    _check_pages(op, kPages, vPages)
    if len(k.shape) != 3 or k.shape != v.shape or k.dtype != v.dtype:
        raise TensorError(f"{op}: k and v must be [tokens, kvHeads, headDim] of one dtype, got "
                          f"{list(k.shape)} and {list(v.shape)}")
    if k.dtype != kPages.dtype or k.shape[1] != kPages.shape[1] or k.shape[2] != kPages.shape[3]:
        raise TensorError(f"{op}: rows {k.dtype.rew_name} {list(k.shape)} do not fit pages "
                          f"{kPages.dtype.rew_name} {list(kPages.shape)}")
    _check_i32(op, slots, "slots", (k.shape[0],))
    _packed_call(op, [kPages, vPages, k, v, slots], [], 0)


def pagedAttention(q: Tensor, kPages: Tensor, vPages: Tensor, blockTable: Tensor,
                   starts: Tensor, lens: Tensor, causal: bool = True, scale: float = 0.0,
                   maxNew: int = 0) -> Tensor:
    """Attention of each request's new tokens over its cached keys and values.

    ``q`` [tokens, heads, headDim]: request r's n = starts[r + 1] - starts[r] rows from
    starts[r], at positions lens[r] - n and on.  Its ``lens[r]`` keys (the new tokens' own
    among them, written before by ``pagedCacheWrite``) lie in the pages ``blockTable[r]``:
    key j in row j % pageSize of page blockTable[r, j / pageSize].  ``causal``: a row sees
    the keys up to its own position; otherwise all ``lens[r]``.  A key without a valid page
    is not seen, and a row that sees none, or belongs to no request, gives zeros.  One token
    per request is a decode step, a whole prompt over an empty cache a prefill, and requests
    of both kinds may be mixed.  dtypes, head dims, scale and rounding as in
    ``packedAttention``.

    ``maxNew``: at least the largest n, if the caller knows it (0: not); it chooses the
    kernels, and with them the order of sums, never what is computed."""
    op = "pagedAttention"
    _check_pages(op, kPages, vPages)
    _check_heads(op, q, kPages.dtype, kPages.shape[1], kPages.shape[3])
    _check_i32(op, blockTable, "blockTable", (None, None))
    _check_i32(op, starts, "starts", (blockTable.shape[0] + 1,))
    _check_i32(op, lens, "lens", (blockTable.shape[0],))
    if maxNew < 0:
        raise TensorError(f"{op}: maxNew must be non-negative, got {maxNew}")
    attrs = _attn_attrs(op, causal, scale) + [("max_new", str(maxNew))]
    return _packed_call(op, [q, kPages, vPages, blockTable, starts, lens], attrs, 1)[0]


# ---- the ends of a training step ------------------------------------------------------
# Backend extensions without a counterpart in the reference, eager only: embedding
# rows, layer norm and the loss over the vocabulary, each with its gradients.  Sums are
# float32 in a fixed order (the same call gives the same bits) and every result is
# rounded once.  Ids and targets are device tensors that no call reads back.

_ROW_DTYPES = (DType.FLOAT32, DType.BFLOAT16, DType.FLOAT16)


@lru_cache(maxsize=256)
def _float_text(op: str, name: str, value: float, sign: float, positive: bool) -> tuple:
    v = c_float(value).value  # (rounded to float32, to infinity past its range)
    if not abs(v) < float("inf") or positive and not v > 0.0:
        raise TensorError(f"{op}: {name} must be a {'positive' if positive else 'finite'} "
                          f"float32, got {value}")
    return name, repr(v)


def _float_attr(op: str, name: str, value: float, positive: bool = False) -> tuple:
    return _float_text(op, name, value, copysign(1.0, value), positive)  # (0.0 == -0.0)


def _check_rows(op: str, t: Tensor) -> None:
    if t.dtype not in _ROW_DTYPES:
        raise TensorError(f"{op}: only float32, bfloat16 or float16, got {t.dtype.rew_name}")


def _check_ids(op: str, ids: Tensor, width: int) -> None:
    if ids.dtype != DType.INT32:
        raise TensorError(f"{op}: ids must be an int32 tensor, got {ids.dtype.rew_name}")
    if not 1 <= width <= 2 ** 20:
        raise TensorError(f"{op}: rows must have 1 to 2^20 values, got {width}")


def embedding(weight: Tensor, ids: Tensor, scale: float = 1.0) -> Tensor:
    """scale * weight[ids]: rows of ``weight`` [vocab, embed] (float32, bfloat16 or float16)
    for int32 ``ids`` of any shape; [*ids.shape, embed].  The product is float32, rounded once.
    An id outside [0, vocab) (padding: -1) gives zeros, unlike ``torchIndexSelect``, which
    clamps it."""
    op = "embedding"
    if len(weight.shape) != 2 or weight.shape[0] < 1:
        raise TensorError(f"{op}: weight must be [vocab, embed], got {list(weight.shape)}")
    _check_rows(op, weight)
    _check_ids(op, ids, weight.shape[1])
    return _packed_call(op, [weight, ids], [_float_attr(op, "scale", scale)], 1)[0]


def embeddingGrad(ids: Tensor, gradOut: Tensor, vocab: int, scale: float = 1.0) -> Tensor:
    """The gradient [vocab, embed] of ``embedding``'s weight for the gradient ``gradOut``
    [*ids.shape, embed] of its result: row v is scale times the sum of gradOut over the places
    of ids that hold v, in their order (rows of many places: in parts), zeros where none does.
    Places with an id outside [0, vocab) take no part, whatever their gradOut.  Fewer than
    2^30 places."""
    op = "embeddingGrad"
    if len(gradOut.shape) < 1 or tuple(gradOut.shape[:-1]) != tuple(ids.shape):
        raise TensorError(f"{op}: gradOut must be [*ids.shape, embed], got "
                          f"{list(gradOut.shape)} for ids {list(ids.shape)}")
    _check_rows(op, gradOut)
    _check_ids(op, ids, gradOut.shape[-1])
    if vocab < 1:
        raise TensorError(f"{op}: vocab must be positive, got {vocab}")
    if prod(ids.shape) >= 2 ** 30:
        raise TensorError(f"{op}: fewer than 2^30 ids, got {list(ids.shape)}")
    return _packed_call(op, [ids, gradOut], [("vocab", str(int(vocab))),
                                             _float_attr(op, "scale", scale)], 1)[0]


class NormStats(NamedTuple):
    """What ``layerNorm`` leaves for its gradient, beside its result (float32, the shape of
    x without the normalised dims)."""
    mean: Tensor
    rstd: Tensor  # 1 / sqrt(variance + eps)


def _check_norm(op: str, x: Tensor, gamma: Tensor) -> tuple:
    _check_rows(op, x)
    if gamma.dtype not in (x.dtype, DType.FLOAT32):
        raise TensorError(f"{op}: gamma must have x's dtype or float32, got "
                          f"{gamma.dtype.rew_name}")
    lead = len(x.shape) - len(gamma.shape)
    if len(gamma.shape) < 1 or lead < 0 or x.shape[lead:] != gamma.shape:
        raise TensorError(f"{op}: gamma {list(gamma.shape)} must be the last dims of x "
                          f"{list(x.shape)}")
    if 0 in gamma.shape:
        raise TensorError(f"{op}: rows must have at least one value")
    return x.shape[:lead]


def layerNorm(x: Tensor, gamma: Tensor, beta: Tensor, eps: float = 1e-5,
              withStats: bool = False):
    """gamma * (x - mean) / sqrt(variance + eps) + beta over the last dims of ``x`` (float32,
    bfloat16 or float16), those of ``gamma`` and ``beta`` (of x's dtype or float32).  The
    arithmetic is float32 and the result, of x's dtype, rounded once.

    ``withStats``: (y, stats), the ``NormStats`` that ``layerNormGrad`` takes."""
    op = "layerNorm"
    _check_norm(op, x, gamma)
    if beta.dtype != gamma.dtype or beta.shape != gamma.shape:
        raise TensorError(f"{op}: beta must have gamma's dtype and shape")
    attrs = [_float_attr(op, "eps", eps, positive=True),
             ("stats", "true" if withStats else "false")]
    res = _packed_call(op, [x, gamma, beta], attrs, 3 if withStats else 1)
    return (res[0], NormStats(res[1], res[2])) if withStats else res[0]


def layerNormGrad(x: Tensor, gamma: Tensor, stats: NormStats, gradOut: Tensor):
    """(gradX, gradGamma, gradBeta) of ``layerNorm(x, gamma, beta, eps)`` for the gradient
    ``gradOut`` of its result, given its ``stats``: gradX of x's dtype, the others of
    gamma's, summed over all rows."""
    op = "layerNormGrad"
    rows = _check_norm(op, x, gamma)
    mean, rstd = stats
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        if t.dtype != DType.FLOAT32 or t.shape != rows:
            raise TensorError(f"{op}: {name} must be float32 {list(rows)}")
    if gradOut.dtype != x.dtype or gradOut.shape != x.shape:
        raise TensorError(f"{op}: gradOut must have x's dtype and shape")
    return tuple(_packed_call(op, [x, gamma, mean, rstd, gradOut], [], 3))


def _check_head(op: str, x: Tensor, weight: Tensor, targets: Tensor, tied: bool) -> None:
    if len(x.shape) != 2 or len(weight.shape) != 2:
        raise TensorError(f"{op}: x must be [tokens, embed] and weight of rank 2, got "
                          f"{list(x.shape)} and {list(weight.shape)}")
    if x.dtype != weight.dtype:
        raise TensorError(f"{op}: dtype mismatch ({x.dtype.enum_name} vs "
                          f"{weight.dtype.enum_name})")
    if x.dtype not in (DType.BFLOAT16, DType.FLOAT16):
        raise TensorError(f"{op}: only bfloat16 or float16, got {x.dtype.rew_name}")
    if weight.shape[1 if tied else 0] != x.shape[1]:
        raise TensorError(f"{op}: x {list(x.shape)} and weight {list(weight.shape)} "
                          f"({'[vocab, embed]' if tied else '[embed, vocab]'}) differ in embed")
    if not all(1 <= d <= 2 ** 21 for d in weight.shape):
        raise TensorError(f"{op}: embed and vocab must be 1 to 2^21, got {list(weight.shape)}")
    if x.shape[0] >= 2 ** 30:
        raise TensorError(f"{op}: fewer than 2^30 tokens, got {x.shape[0]}")
    _check_i32(op, targets, "targets", (x.shape[0],))


def linearCrossEntropy(x: Tensor, weight: Tensor, targets: Tensor, tied: bool = False,
                       withLse: bool = False):
    """The cross entropy of softmax(x weight) and ``targets`` [tokens], float32 [tokens], not
    reduced: log sum_v exp z[t, v] - z[t, targets[t]], z the logits.  ``x`` [tokens, embed];
    ``weight`` [embed, vocab] as ``nn.Linear``'s or, ``tied``, [vocab, embed] as
    ``nn.Embedding``'s; both bfloat16 or float16.  A target outside [0, vocab) (padding: -1)
    gives 0.  The logits are float32, never rounded and never stored.

    ``withLse``: (loss, lse), the float32 [tokens] that ``linearCrossEntropyGrad`` takes."""
    op = "linearCrossEntropy"
    _check_head(op, x, weight, targets, tied)
    res = _packed_call(op, [x, weight, targets],
                       [("tied", "true" if tied else "false"),
                        ("stats", "true" if withLse else "false")], 2 if withLse else 1)
    return tuple(res) if withLse else res[0]


def linearCrossEntropyGrad(x: Tensor, weight: Tensor, targets: Tensor, lse: Tensor,
                           gradLoss: Tensor, tied: bool = False):
    """(gradX, gradWeight) of ``linearCrossEntropy(x, weight, targets, tied)`` for the gradient
    ``gradLoss`` (float32 [tokens]: 1 / tokens for the mean) of its result, given its ``lse``,
    of the dtypes of x and weight.  The logits are formed anew, a piece of the vocabulary at a
    time.  Their gradient is rounded once to x's dtype for the two products, relative to the
    largest |gradLoss|, whose scale is applied to the float32 sums (float16 loses what is below
    2^-39 of it); with up to 32 tokens what that rounding leaves is kept too.  lse's own
    rounding, a step of its size, is a relative error of every probability.  Tokens without a
    target in [0, vocab) take no part, whatever their x and gradLoss: their gradX is 0."""
    op = "linearCrossEntropyGrad"
    _check_head(op, x, weight, targets, tied)
    for t, name in ((lse, "lse"), (gradLoss, "gradLoss")):
        if t.dtype != DType.FLOAT32 or t.shape != (x.shape[0],):
            raise TensorError(f"{op}: {name} must be float32 [{x.shape[0]}]")
    return tuple(_packed_call(op, [x, weight, targets, lse, gradLoss],
                              [("tied", "true" if tied else "false")], 2))
