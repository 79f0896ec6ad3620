"""Newton-Schulz on device matrices that the caller owns: ``vb_orthogonalize`` and
``vb_muon_multi_tensor_step`` over a plan.

    plan = NewtonSchulzPlan([w.shape for w in weights], [(3.4445, -4.7750, 2.0315)] * 5)
    plan.orthogonalize(updates, out)                      # out[i] = O(updates[i])
    plan.muon_step(weights, grads, velocities, lr=2e-4, momentum=0.95, weight_decay=0.1,
                   scales=[0.2 * max(w.shape) ** 0.5 for w in weights])

The counterpart in the reference is Muon::step's loop over parameters with newton_schulz
(src/nn/optim/muon.rs:50-163); ``multi_tensor_step`` is the sibling for Adam and SGD.  Matrices are
torch tensors (or anything with ``data_ptr()``, ``stride()``, ``shape`` and ``dtype``, or with
``__cuda_array_interface__``) of the engine's device, in any strides.  Work is enqueued on the engine's stream:
order other streams' producers and consumers against it, for instance by running them under
``torch.cuda.stream(torch.cuda.ExternalStream(engine.stream))``.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence, Union

from . import _lib
from ._lib import VB_NS_F16, call
from .optim import Engine, default_engine, muon_dims

__all__ = ["NewtonSchulzPlan", "MatrixList", "plan_newton_schulz"]

DTYPES = {"float32": 0, "<f4": 0, "bfloat16": 1, "float16": 2, "<f2": 2}


def _describe(x):
    """(address, shape, strides in elements, dtype) of a device array."""
    if hasattr(x, "data_ptr"):
        if not getattr(x, "is_cuda", True):
            raise ValueError("matrices must be in device memory")
        return x.data_ptr(), tuple(x.shape), tuple(x.stride()), str(x.dtype).rpartition(".")[2]
    if hasattr(x, "__cuda_array_interface__"):
        d = x.__cuda_array_interface__
        shape, kind, strides = tuple(d["shape"]), d["typestr"], d.get("strides")
        if kind not in DTYPES:
            raise TypeError(f"matrices are float32, bfloat16 or float16, not {kind}")
        if strides is None:
            strides, run = [0] * len(shape), 1
            for k in range(len(shape) - 1, -1, -1):
                strides[k], run = run, run * shape[k]
        else:
            size = int(kind[-1])
            if any(s % size for s in strides):
                raise ValueError("strides must be whole elements")
            strides = [s // size for s in strides]
        return int(d["data"][0]), shape, tuple(strides), kind
    raise TypeError(f"not a device matrix: {type(x).__name__}")


def _two_strides(shape, strides):
    """Row and column stride of the 2-D view (shape[0], product of the rest) of an array."""
    if len(shape) < 2:
        return (strides[0] if shape else 1), 1
    run, col = 1, 1
    first = True
    for k in range(len(shape) - 1, 0, -1):
        if shape[k] == 1:
            continue
        if first:
            col, run, first = strides[k], strides[k] * shape[k], False
        elif strides[k] == run:
            run *= shape[k]
        else:
            raise ValueError(f"an array of shape {shape} with strides {strides} has no view as a matrix")
    return strides[0], col


class MatrixList:
    """The device arrays of every matrix of a plan (``vb_ns_matrices_create``): checked once, used in any
    number of calls.  Keeps the arrays alive."""

    def __init__(self, plan: "NewtonSchulzPlan", arrays: Sequence):
        self._h = C.c_void_p()
        self._arrays = list(arrays)
        self.plan = plan
        n = len(plan.dims)
        if len(self._arrays) != n:
            raise ValueError(f"the plan has {n} matrices, the list {len(self._arrays)}")
        pointers, strides = (C.c_void_p * max(n, 1))(), (C.c_int64 * max(2 * n, 1))()
        kind = None
        for i, x in enumerate(self._arrays):
            if x is None:
                continue
            at, shape, st, k = _describe(x)
            if k not in DTYPES:
                raise TypeError(f"matrices are float32, bfloat16 or float16, not {k}")
            if muon_dims(shape) != plan.dims[i]:
                raise ValueError(f"matrix {i} of the plan is {plan.dims[i]}, the array {shape}")
            if kind is not None and DTYPES[k] != kind:
                raise TypeError("the arrays of a list have one dtype")
            kind = DTYPES[k]
            pointers[i] = at or None
            strides[2 * i], strides[2 * i + 1] = _two_strides(shape, st)
        call("vb_ns_matrices_create", plan._h, kind or 0, pointers, strides, C.byref(self._h))

    def close(self) -> None:
        if self._h:
            call("vb_ns_matrices_destroy", self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


Arrays = Union[MatrixList, Sequence]


class NewtonSchulzPlan:
    """Schedule and workspace to orthogonalise matrices of the given shapes together
    (``vb_ns_plan_create``).  ``coefficients``: one (a, b, c) per step of
    ``X <- a X + b (X X^T) X + c (X X^T)^2 X``; the reference's iteration (src/nn/optim/muon.rs:67-100) is
    ``[(1.5, -0.5, 0.0)] * ns_steps``.  ``ns_mode``: ``VB_NS_F16`` or ``VB_NS_F32_TC``."""

    def __init__(self, shapes, coefficients: Sequence[Sequence[float]], eps: float = 1e-7, ns_mode: int = VB_NS_F16,
                 engine: Optional[Engine] = None):
        self._h = C.c_void_p()
        self.engine = engine if engine is not None else default_engine()
        self.dims = [muon_dims(s) for s in shapes]
        flat = [float(v) for step in coefficients for v in step]
        if any(len(step) != 3 for step in coefficients):
            raise ValueError("every step has three coefficients")
        n = len(self.dims)
        rows = (C.c_int64 * max(n, 1))(*[d[0] for d in self.dims])
        cols = (C.c_int64 * max(n, 1))(*[d[1] for d in self.dims])
        call("vb_ns_plan_create", self.engine._h, n, rows, cols, len(coefficients),
             (C.c_float * max(len(flat), 1))(*flat), float(eps), int(ns_mode), C.byref(self._h))

    def close(self) -> None:
        if self._h:
            call("vb_ns_plan_destroy", self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def workspace_bytes(self) -> int:
        n = C.c_size_t()
        call("vb_ns_plan_workspace", self._h, C.byref(n))
        return int(n.value)

    @property
    def flops(self) -> float:
        """FLOPs of the products that one call launches."""
        f = C.c_double()
        call("vb_ns_plan_flops", self._h, C.byref(f))
        return float(f.value)

    def matrices(self, arrays: Sequence) -> MatrixList:
        """A list of device arrays to pass to the calls below as often as wanted; ``None`` marks an absent gradient."""
        return MatrixList(self, arrays)

    def _list(self, x: Arrays) -> MatrixList:
        return x if isinstance(x, MatrixList) else MatrixList(self, x)

    def orthogonalize(self, inputs: Arrays, outputs: Arrays) -> None:
        """``outputs[i] = O(inputs[i])``; an output may be its input."""
        a, b = self._list(inputs), self._list(outputs)
        call("vb_orthogonalize", self._h, a._h, b._h)

    def muon_step(self, params: Arrays, grads: Arrays, velocities: Arrays, *, lr: float, momentum: float = 0.95,
                  nesterov: bool = True, weight_decay: float = 0.0, scales: Optional[Sequence[float]] = None) -> None:
        """``v <- momentum v + g;  p <- p (1 - lr weight_decay) - lr scales[i] O(g + momentum v)`` (without Nesterov:
        ``O(v)``).  Matrices whose gradient is ``None`` are left as they are."""
        p, g, v = self._list(params), self._list(grads), self._list(velocities)
        n = len(self.dims)
        if scales is not None and len(scales) != n:
            raise ValueError(f"the plan has {n} matrices, scales {len(scales)}")
        hp = _lib.MuonStepParams(lr, momentum, weight_decay, int(bool(nesterov)))
        call("vb_muon_multi_tensor_step", self._h, C.byref(hp), p._h, g._h, v._h,
             (C.c_float * n)(*scales) if scales is not None else None)


def plan_newton_schulz(rows: int, cols: int, coefficients: Sequence[Sequence[float]], ns_mode: int = VB_NS_F16):
    """The products a plan runs for one matrix (``vb_plan_newton_schulz``, no device needed): a list of
    dicts with the buffers and factors of ``D = e E + f F + g A B'``, and the factor of the last one's D."""
    flat = [float(v) for step in coefficients for v in step]
    co = (C.c_float * max(len(flat), 1))(*flat)
    n, scale = C.c_int64(), C.c_double()
    call("vb_plan_newton_schulz", rows, cols, len(coefficients), co, int(ns_mode), 0, C.byref(n), None, None, C.byref(scale))
    ints, doubles = (C.c_int32 * (9 * n.value))(), (C.c_double * (3 * n.value))()
    call("vb_plan_newton_schulz", rows, cols, len(coefficients), co, int(ns_mode), n.value, C.byref(n), ints, doubles, C.byref(scale))
    names = ("stage", "A", "B", "E", "F", "D", "scale_power", "update", "gram")
    return [dict(zip(names, ints[9 * k:9 * k + 9]), **dict(zip("efg", doubles[3 * k:3 * k + 3])))
            for k in range(n.value)], scale.value
