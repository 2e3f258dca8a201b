"""ctypes binding of the sm_100a runtime's C ABI.

The v1 half mirrors ArcQML's safe FFI facade ``arcqml-runtime-sys``
(``crates/arcqml-runtime-sys/src/lib.rs:123-336``): the same function names, argument meaning and
error behaviour (a non-zero status becomes ``RuntimeError`` carrying the runtime's thread-local
message, read as in ``last_error`` at ``lib.rs:330-336``). The v2 half drives device-resident
states held in torch CUDA tensors (``complex128``, ``[batch, 2^n]``).

There is no CPU fallback: importing this module loads ``libarcqml_runtime_private.so`` and fails
loudly if it is missing.
"""
from __future__ import annotations

import ctypes as C
import os
import struct
from bisect import bisect_left
from typing import Optional, Sequence

import numpy as np

from .circuit import PlanOp

ABI_VERSION = 1
_HERE = os.path.dirname(os.path.abspath(__file__))
# ARCQML_RUNTIME_LIB may name another build of the same C ABI (e.g. an instrumented one).
LIB_PATH = os.environ.get("ARCQML_RUNTIME_LIB") or os.path.join(_HERE, "libarcqml_runtime_private.so")


class RuntimeError(Exception):  # noqa: A001 - mirrors arcqml_runtime_sys::RuntimeError
    """A failed runtime call; ``str(e)`` is the runtime's message."""

    def message(self) -> str:
        return str(self)


class C128(C.Structure):
    _fields_ = [("re", C.c_double), ("im", C.c_double)]


class GateDescriptor(C.Structure):
    _fields_ = [
        ("abi_version", C.c_uint32),
        ("opcode", C.c_uint32),
        ("arity", C.c_size_t),
        ("parameters", C.c_double * 3),
        ("matrix", C.c_void_p),
        ("matrix_len", C.c_size_t),
        ("name", C.c_void_p),
        ("name_len", C.c_size_t),
    ]


class DerivativeMatrixHandle(C.Structure):
    _fields_ = [("data", C.POINTER(C128)), ("len", C.c_size_t), ("capacity", C.c_size_t)]


class ParameterBindingDescriptor(C.Structure):
    _fields_ = [("parameter_slot", C.c_size_t), ("parent_index", C.c_size_t)]


class OperationDescriptor(C.Structure):
    _fields_ = [
        ("gate", GateDescriptor),
        ("qubits", C.POINTER(C.c_size_t)),
        ("qubits_len", C.c_size_t),
        ("parameters", C.POINTER(ParameterBindingDescriptor)),
        ("parameters_len", C.c_size_t),
    ]


class CircuitPlanHandle(C.Structure):
    _fields_ = [("opaque", C.c_void_p)]


class ObservableHandle(C.Structure):
    _fields_ = [("opaque", C.c_void_p)]


V1_SYMBOLS = (
    "arcqml_rt_abi_version", "arcqml_rt_v1_apply_gate", "arcqml_rt_v1_apply_adjoint_gate",
    "arcqml_rt_v1_parameter_derivative_into", "arcqml_rt_v1_derivative_matrix_create",
    "arcqml_rt_v1_derivative_matrix_apply", "arcqml_rt_v1_derivative_matrix_destroy",
    "arcqml_rt_v1_circuit_plan_create", "arcqml_rt_v1_circuit_plan_create_empty",
    "arcqml_rt_v1_circuit_plan_push", "arcqml_rt_v1_circuit_plan_apply",
    "arcqml_rt_v1_adjoint_backward", "arcqml_rt_v1_circuit_plan_destroy", "arcqml_rt_last_error",
)

_P, _S, _I32, _D = C.c_void_p, C.c_size_t, C.c_int32, C.c_double
# (result type, argument types) of every entry point the binding calls
SIGNATURES = {
    "arcqml_rt_abi_version": (C.c_uint32, []),
    "arcqml_rt_v1_apply_gate": (_I32, [_P, _S, _S, _P, _P, _S]),
    "arcqml_rt_v1_apply_adjoint_gate": (_I32, [_P, _S, _S, _P, _P, _S]),
    "arcqml_rt_v1_parameter_derivative_into": (_I32, [_P, _S, _P, _S, _P, _P, _S, _S]),
    "arcqml_rt_v1_derivative_matrix_create": (_I32, [_P, _S, _P]),
    "arcqml_rt_v1_derivative_matrix_apply": (_I32, [_P, _S, _P, _P, _S]),
    "arcqml_rt_v1_derivative_matrix_destroy": (None, [_P]),
    "arcqml_rt_v1_circuit_plan_create": (_I32, [_P, _S, _P]),
    "arcqml_rt_v1_circuit_plan_create_empty": (_I32, [_S, _P]),
    "arcqml_rt_v1_circuit_plan_push": (_I32, [_P, _P]),
    "arcqml_rt_v1_circuit_plan_apply": (_I32, [_P, _P, _S, _S]),
    "arcqml_rt_v1_adjoint_backward": (_I32, [_P, _P, _P, _S, _P, _S, _D, _P, _S, _P, _S]),
    "arcqml_rt_v1_circuit_plan_destroy": (None, [_P]),
    "arcqml_rt_last_error": (_S, [_P, _S]),
    "arcqml_rt_v2_observable_create": (_I32, [_S, _P, _P, _P, _S, _P]),
    "arcqml_rt_v2_observable_destroy": (None, [_P]),
    "arcqml_rt_v2_plan_apply": (_I32, [_P, _P, _S, _S, _P]),
    "arcqml_rt_v2_apply_gate": (_I32, [_P, _S, _S, _P, _P, _S, _I32, _P]),
    "arcqml_rt_v2_parameter_derivative": (_I32, [_P, _P, _S, _S, _P, _P, _S, _S, _P]),
    "arcqml_rt_v2_expectation": (_I32, [_P, _P, _S, _S, _P, _P]),
    "arcqml_rt_v2_observable_tile_passes": (_I32, [_P, _S, _P]),
    "arcqml_rt_v2_expectation_and_apply": (_I32, [_P, _P, _P, _S, _S, _P, _P]),
    "arcqml_rt_v2_expectation_and_accumulate": (_I32, [_P, _P, _P, _S, _S, _P, _P]),
    "arcqml_rt_v2_sample": (_I32, [_P, _S, C.c_uint64, C.c_uint64, _P, _P, _P]),
    "arcqml_rt_v2_shard_slices": (_I32, [_P, _S, _P, _S, C.c_uint64, C.c_uint64, C.c_uint64, _P,
                                        _I32, _P]),
    "arcqml_rt_v2_small_run": (_I32, [_P, _P, _P, _S, _P, _S, _P, _S, _P, _P, _P]),
    "arcqml_rt_v2_plan_emulate": (_I32, [_P, _P, _S, _I32, _P, _P, _S, _P, _S]),
    "arcqml_rt_v2_plan_schedule_export": (_I32, [_P, _S, _I32, _P, _S, _P, _S, _P]),
    "arcqml_rt_v2_probabilities": (_I32, [_P, _S, _S, _P, _P]),
    "arcqml_rt_v2_marginal_probabilities": (_I32, [_P, _S, _S, _P, _S, _P, _P]),
    "arcqml_rt_v2_bloch_vector": (_I32, [_P, _S, _S, _S, _P, _P]),
    "arcqml_rt_v2_overlap": (_I32, [_P, _P, _S, _S, _P, _P]),
    "arcqml_rt_v2_probability_cotangent": (_I32, [_P, _S, _S, _P, _S, _P, _P, _P]),
    "arcqml_rt_v2_scaled_copy": (_I32, [_P, _S, _S, _P, _P, _P]),
    "arcqml_rt_v2_small_adam": (_I32, [_P, _P, _P, _S, _P, _P, _S, _P, _P, C.c_uint64, _S, _D,
                                      _D, _D, _D, _D, _P, _P]),
    "arcqml_rt_v2_shard_slices_from": (_I32, [_P, _S, _P, _S, C.c_uint64, C.c_uint64, _P, _P]),
    "arcqml_rt_v2_shard_swap_nccl": (_I32, [_P, _S, _P, _P, _S, _P, _P, _S, _P]),
    "arcqml_rt_v2_peer_buffer_create": (_I32, [_S, _P, _P]),
    "arcqml_rt_v2_peer_buffer_open": (_I32, [_P, _P]),
    "arcqml_rt_v2_peer_buffer_close": (_I32, [_P]),
    "arcqml_rt_v2_peer_buffer_destroy": (_I32, [_P]),
    "arcqml_rt_v2_adjoint_backward": (_I32, [_P, _P, _P, _S, _S, _P, _P, _S, _P, _S, _P]),
    "arcqml_rt_v2_gradient_workspace": (_S, [_P, _S]),
    "arcqml_rt_v2_adam_workspace": (_S, [_P, _S]),
    "arcqml_rt_v2_gradient_norm": (_I32, [_P, _S, _P, _P, _S, _P]),
    "arcqml_rt_v2_clip_gradients": (_I32, [_P, _S, _D, _P, _P, _P, _S, _P]),
    "arcqml_rt_v2_adam_step": (_I32, [_P, _P, _P, _P, _P, _S, _P, _P, _P, _P, _P, _S, _P]),
    "arcqml_rt_v2_embedding_lookup_workspace": (_S, [_P, _S, _P]),
    "arcqml_rt_v2_embedding_gradient_workspace": (_S, [_P, C.c_uint64, _P]),
    "arcqml_rt_v2_embedding_lookup": (_I32, [_P, _P, _S, _P, _P, _P, _S, _P]),
    "arcqml_rt_v2_embedding_gradient": (_I32, [_P, _P, _P, _P, _P, _P, _S, _P]),
    "arcqml_rt_v2_orthogonalize_workspace": (_S, [_P, _S]),
    "arcqml_rt_v2_orthogonalize": (_I32, [_P, _P, _S, _I32, _D, _P, _S, _P]),
    "arcqml_rt_v2_muon_step": (_I32, [_P, _P, _P, _S, _P, _P, _S, _P]),
    "arcqml_rt_v2_norms": (_I32, [_P, _S, _S, _P, _P]),
    "arcqml_rt_v2_norms_noalloc": (_I32, [_P, _S, _S, _P, _P]),
    "arcqml_rt_v2_set_basis_state": (_I32, [_P, _S, _S, C.c_uint64, _P]),
    "arcqml_rt_v2_plan_set_parameters": (_I32, [_P, _P, _S]),
    "arcqml_rt_v2_plan_len": (_S, [_P]),
    "arcqml_rt_v2_plan_schedule_stats": (_I32, [_P, _S, _I32, _P, _P, _P]),
    "arcqml_rt_v2_profile_enable": (None, [_I32]),
    "arcqml_rt_v2_profile_read": (_I32, [C.c_uint32, _P, _P, _P]),
    "arcqml_rt_v2_launch_count": (C.c_uint64, []),
    "arcqml_rt_v2_jit_info": (_S, [_P, _P, _P, _P, _S]),
    "arcqml_rt_v2_plan_jit_check": (_I32, [_P, _S, _I32, _P, _P, _P, _S]),
}

_lib = None


def load():
    """Loads the runtime library (once). Raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError(
            f"{LIB_PATH} is missing: build it with `python -m arcqml_b200.build` "
            "(the statevector path has no CPU fallback)")
    L = C.CDLL(LIB_PATH)
    for name, (res, args) in SIGNATURES.items():
        f = getattr(L, name)
        f.restype = res
        f.argtypes = args
    _lib = L
    return L


def last_error() -> str:
    L = load()
    n = L.arcqml_rt_last_error(None, 0)
    buf = (C.c_uint8 * (n + 1))()
    L.arcqml_rt_last_error(buf, n + 1)
    return bytes(buf[:n]).decode("utf-8", errors="replace")


def _status(code: int) -> None:
    if code != 0:
        raise RuntimeError(last_error())


def ensure_compatible() -> None:
    actual = load().arcqml_rt_abi_version()
    if actual != ABI_VERSION:
        raise RuntimeError(f"ArcQML runtime ABI mismatch: expected {ABI_VERSION}, got {actual}")


# ------------------------------------------------------------------ descriptors


class _Keep:
    """Owns the ctypes buffers a descriptor points into."""

    def __init__(self):
        self.items = []

    def add(self, x):
        self.items.append(x)
        return x


def gate_descriptor(opcode: int, arity: int, params=(0.0, 0.0, 0.0), matrix=None,
                    name: str = "", keep: Optional[_Keep] = None,
                    abi_version: int = ABI_VERSION) -> GateDescriptor:
    keep = keep if keep is not None else _Keep()
    g = GateDescriptor()
    g.abi_version = abi_version
    g.opcode = opcode
    g.arity = arity
    p = list(params) + [0.0] * (3 - len(params))
    for i in range(3):
        g.parameters[i] = float(p[i])
    if matrix is not None:
        m = keep.add(np.ascontiguousarray(np.asarray(matrix, dtype=np.complex128).ravel()))
        g.matrix = m.ctypes.data
        g.matrix_len = m.size
    if name:
        nb = keep.add(C.create_string_buffer(name.encode()))
        g.name = C.addressof(nb)
        g.name_len = len(name.encode())
    return g


def _op_descriptor(op: PlanOp, keep: _Keep) -> OperationDescriptor:
    d = OperationDescriptor()
    d.gate = gate_descriptor(op.opcode, len(op.qubits), op.params, op.matrix, op.name, keep)
    q = keep.add((C.c_size_t * max(1, len(op.qubits)))(*op.qubits))
    d.qubits = C.cast(q, C.POINTER(C.c_size_t))
    d.qubits_len = len(op.qubits)
    b = keep.add((ParameterBindingDescriptor * 3)())
    for i, (slot, parent) in enumerate(op.bindings):
        b[i].parameter_slot = slot
        b[i].parent_index = parent
    d.parameters = C.cast(b, C.POINTER(ParameterBindingDescriptor))
    d.parameters_len = len(op.bindings)
    return d


def _state_ptr(a: np.ndarray):
    if a.dtype != np.complex128 or not a.flags.c_contiguous:
        raise TypeError("amplitudes must be a C-contiguous complex128 array")
    return a.ctypes.data


def _qubits(qubits: Sequence[int]):
    return (C.c_size_t * max(1, len(qubits)))(*[int(q) for q in qubits])


# ------------------------------------------------------------------ v1 (host buffers)


def apply_gate(amplitudes: np.ndarray, num_qubits: int, gate: GateDescriptor,
               qubits: Sequence[int]) -> None:
    """arcqml_runtime_sys::apply_gate (lib.rs:137-153): in place."""
    _status(load().arcqml_rt_v1_apply_gate(_state_ptr(amplitudes), amplitudes.size, num_qubits,
                                          C.byref(gate), _qubits(qubits), len(qubits)))


def apply_adjoint_gate(amplitudes: np.ndarray, num_qubits: int, gate: GateDescriptor,
                       qubits: Sequence[int]) -> None:
    """arcqml_runtime_sys::apply_adjoint_gate (lib.rs:155-171): in place."""
    _status(load().arcqml_rt_v1_apply_adjoint_gate(_state_ptr(amplitudes), amplitudes.size,
                                                  num_qubits, C.byref(gate), _qubits(qubits),
                                                  len(qubits)))


def parameter_derivative_into(inp: np.ndarray, out: np.ndarray, gate: GateDescriptor,
                              qubits: Sequence[int], parameter_slot: int) -> None:
    """arcqml_runtime_sys::parameter_derivative_into (lib.rs:173-192)."""
    _status(load().arcqml_rt_v1_parameter_derivative_into(
        _state_ptr(inp), inp.size, _state_ptr(out), out.size, C.byref(gate), _qubits(qubits),
        len(qubits), parameter_slot))


class DerivativeMatrix:
    """arcqml_runtime_sys::DerivativeMatrix (lib.rs:194-232)."""

    def __init__(self, gate: GateDescriptor, parameter_slot: int):
        self.raw = DerivativeMatrixHandle()
        _status(load().arcqml_rt_v1_derivative_matrix_create(C.byref(gate), parameter_slot,
                                                           C.byref(self.raw)))

    @classmethod
    def create(cls, gate: GateDescriptor, parameter_slot: int) -> "DerivativeMatrix":
        return cls(gate, parameter_slot)

    def matrix(self) -> np.ndarray:
        n = self.raw.len
        dim = int(round(np.sqrt(n)))
        flat = np.ctypeslib.as_array(C.cast(self.raw.data, C.POINTER(C.c_double)), shape=(2 * n,))
        return (flat[0::2] + 1j * flat[1::2]).reshape(dim, dim).copy()

    def apply(self, amplitudes: np.ndarray, qubits: Sequence[int]) -> None:
        _status(load().arcqml_rt_v1_derivative_matrix_apply(
            _state_ptr(amplitudes), amplitudes.size, C.byref(self.raw), _qubits(qubits),
            len(qubits)))

    def __del__(self):
        if _lib is not None and getattr(self, "raw", None) is not None:
            _lib.arcqml_rt_v1_derivative_matrix_destroy(C.byref(self.raw))


class CircuitPlan:
    """arcqml_runtime_sys::CircuitPlan (lib.rs:234-320)."""

    def __init__(self, raw: CircuitPlanHandle):
        self.raw = raw

    @classmethod
    def create(cls, operations: Sequence[PlanOp]) -> "CircuitPlan":
        ensure_compatible()
        keep = _Keep()
        arr = (OperationDescriptor * max(1, len(operations)))()
        for i, op in enumerate(operations):
            arr[i] = _op_descriptor(op, keep)
        raw = CircuitPlanHandle()
        _status(load().arcqml_rt_v1_circuit_plan_create(arr, len(operations), C.byref(raw)))
        return cls(raw)

    @classmethod
    def with_capacity(cls, operation_capacity: int) -> "CircuitPlan":
        ensure_compatible()
        raw = CircuitPlanHandle()
        _status(load().arcqml_rt_v1_circuit_plan_create_empty(operation_capacity, C.byref(raw)))
        return cls(raw)

    @classmethod
    def compile(cls, ops: Sequence[PlanOp]) -> "CircuitPlan":
        """RuntimeCircuitPlan::compile: one push per operation, descriptors from temporaries."""
        plan = cls.with_capacity(len(ops))
        for op in ops:
            plan.push(op)
        return plan

    def push(self, op: PlanOp) -> None:
        keep = _Keep()
        d = _op_descriptor(op, keep)
        _status(load().arcqml_rt_v1_circuit_plan_push(C.byref(self.raw), C.byref(d)))
        del keep  # the runtime deep-copied everything

    def apply(self, amplitudes: np.ndarray, num_qubits: int) -> None:
        _status(load().arcqml_rt_v1_circuit_plan_apply(C.byref(self.raw), _state_ptr(amplitudes),
                                                      amplitudes.size, num_qubits))

    def adjoint_backward(self, forward_state: np.ndarray, adjoint_state: np.ndarray,
                         derivative_state: np.ndarray, num_qubits: int, upstream: float,
                         parameter_requires_grad: np.ndarray, gradients: np.ndarray) -> None:
        if not (forward_state.size == adjoint_state.size == derivative_state.size):
            raise RuntimeError("adjoint buffers must have identical lengths")
        req = np.ascontiguousarray(parameter_requires_grad, dtype=np.uint8)
        if gradients.dtype != np.float64 or not gradients.flags.c_contiguous:
            raise TypeError("gradients must be a C-contiguous float64 array")
        _status(load().arcqml_rt_v1_adjoint_backward(
            C.byref(self.raw), _state_ptr(forward_state), _state_ptr(adjoint_state),
            forward_state.size, _state_ptr(derivative_state), num_qubits, float(upstream),
            req.ctypes.data, req.size, gradients.ctypes.data, gradients.size))

    # -- v2 extensions on the same plan -------------------------------------------
    def set_parameters(self, parent_values: np.ndarray) -> None:
        v = np.ascontiguousarray(parent_values, dtype=np.float64)
        _status(load().arcqml_rt_v2_plan_set_parameters(C.byref(self.raw), v.ctypes.data, v.size))

    def jit_check(self, num_qubits: int, adjoint: bool = False) -> dict:
        """Compiles the run-time kernels of this plan's fused passes (NVRTC only, no GPU):
        {compiled, eligible, message}."""
        c, e = C.c_uint64(), C.c_uint64()
        buf = C.create_string_buffer(4096)
        _status(load().arcqml_rt_v2_plan_jit_check(C.byref(self.raw), num_qubits, int(adjoint),
                                                   C.byref(c), C.byref(e), buf, 4096))
        return {"compiled": int(c.value), "eligible": int(e.value),
                "message": buf.value.decode("utf-8", errors="replace")}

    def __len__(self) -> int:
        return load().arcqml_rt_v2_plan_len(C.byref(self.raw))

    def schedule_stats(self, num_qubits: int, adjoint: bool = False) -> dict:
        """Fused-pass schedule size for an n-qubit state (host only)."""
        a, b, c = C.c_uint64(), C.c_uint64(), C.c_uint64()
        _status(load().arcqml_rt_v2_plan_schedule_stats(C.byref(self.raw), num_qubits,
                                                        int(adjoint), C.byref(a), C.byref(b),
                                                        C.byref(c)))
        return {"passes": a.value, "sub_blocks": b.value, "gates": c.value}

    def __del__(self):
        if _lib is not None and getattr(self, "raw", None) is not None:
            _lib.arcqml_rt_v1_circuit_plan_destroy(C.byref(self.raw))


# ------------------------------------------------------------------ v2 (device states)


def _stream_ptr(stream) -> Optional[int]:
    if stream is None:
        import torch
        return torch.cuda.current_stream().cuda_stream
    return int(stream)


def _dev_ptr(t) -> int:
    import torch
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == torch.complex128
            and t.is_contiguous()):
        raise TypeError("device amplitudes must be a contiguous complex128 CUDA tensor")
    return t.data_ptr()


def _dev_ptr_f64(t) -> int:
    import torch
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == torch.float64
            and t.is_contiguous()):
        raise TypeError("device values must be a contiguous float64 CUDA tensor")
    return t.data_ptr()


def _rows(t, num_qubits: int) -> int:
    dim = 1 << num_qubits
    if t.numel() % dim != 0 or t.numel() == 0:
        raise RuntimeError(f"device state of {t.numel()} amplitudes is not [batch, {dim}]")
    return t.numel() // dim


class Observable:
    """Compiled Pauli observable on the runtime (arcqml_rt_v2_observable_*)."""

    def __init__(self, num_qubits: int, coefficients, flip_masks, phase_masks):
        c = np.ascontiguousarray(coefficients, dtype=np.float64)
        f = np.ascontiguousarray(flip_masks, dtype=np.uint64)
        p = np.ascontiguousarray(phase_masks, dtype=np.uint64)
        if not (c.size == f.size == p.size):
            raise ValueError("term arrays differ in length")
        self.num_qubits = num_qubits
        self.raw = ObservableHandle()
        _status(load().arcqml_rt_v2_observable_create(num_qubits, c.ctypes.data, f.ctypes.data,
                                                      p.ctypes.data, c.size, C.byref(self.raw)))

    @classmethod
    def from_sparse_pauli_op(cls, op) -> "Observable":
        c, f, p = op.masks()
        return cls(op.num_qubits, c, f, p)

    def expectation(self, state, num_qubits: int, stream=None) -> np.ndarray:
        b = _rows(state, num_qubits)
        out = np.zeros(b, dtype=np.float64)
        _status(load().arcqml_rt_v2_expectation(C.byref(self.raw), _dev_ptr(state), b, num_qubits,
                                                out.ctypes.data, _stream_ptr(stream)))
        return out

    def expectation_and_apply(self, state, out_state, num_qubits: int, stream=None) -> np.ndarray:
        b = _rows(state, num_qubits)
        vals = np.zeros(b, dtype=np.float64)
        _status(load().arcqml_rt_v2_expectation_and_apply(
            C.byref(self.raw), _dev_ptr(state), _dev_ptr(out_state), b, num_qubits,
            vals.ctypes.data, _stream_ptr(stream)))
        return vals

    def tile_passes(self, num_qubits: int) -> int:
        """Passes over 12-qubit tiles this observable takes on a num_qubits state (0: the gather
        kernel evaluates it)."""
        v = C.c_uint32()
        _status(load().arcqml_rt_v2_observable_tile_passes(C.byref(self.raw), num_qubits,
                                                           C.byref(v)))
        return int(v.value)

    def expectation_and_accumulate(self, state, out_state, num_qubits: int,
                                   stream=None) -> np.ndarray:
        """out_state += H psi; returns <psi|H|psi> per row."""
        b = _rows(state, num_qubits)
        vals = np.zeros(b, dtype=np.float64)
        _status(load().arcqml_rt_v2_expectation_and_accumulate(
            C.byref(self.raw), _dev_ptr(state), _dev_ptr(out_state), b, num_qubits,
            vals.ctypes.data, _stream_ptr(stream)))
        return vals

    def __del__(self):
        if _lib is not None and getattr(self, "raw", None) is not None:
            _lib.arcqml_rt_v2_observable_destroy(C.byref(self.raw))


def plan_apply_device(plan: CircuitPlan, state, num_qubits: int, stream=None) -> None:
    b = _rows(state, num_qubits)
    _status(load().arcqml_rt_v2_plan_apply(C.byref(plan.raw), _dev_ptr(state), b, num_qubits,
                                           _stream_ptr(stream)))


def apply_gate_device(state, num_qubits: int, gate: GateDescriptor, qubits, adjoint=False,
                      stream=None) -> None:
    b = _rows(state, num_qubits)
    _status(load().arcqml_rt_v2_apply_gate(_dev_ptr(state), b, num_qubits, C.byref(gate),
                                           _qubits(qubits), len(qubits), int(adjoint),
                                           _stream_ptr(stream)))


def parameter_derivative_device(inp, out, num_qubits: int, gate: GateDescriptor, qubits, slot,
                                stream=None) -> None:
    b = _rows(inp, num_qubits)
    _status(load().arcqml_rt_v2_parameter_derivative(
        _dev_ptr(inp), _dev_ptr(out), b, num_qubits, C.byref(gate), _qubits(qubits), len(qubits),
        slot, _stream_ptr(stream)))


def adjoint_backward_device(plan: CircuitPlan, psi, lam, num_qubits: int, upstream,
                            requires_grad, num_gradients: int, stream=None) -> np.ndarray:
    b = _rows(psi, num_qubits)
    up = np.ascontiguousarray(np.broadcast_to(np.asarray(upstream, dtype=np.float64), (b,)))
    req = np.ascontiguousarray(requires_grad, dtype=np.uint8)
    grads = np.zeros(num_gradients, dtype=np.float64)
    _status(load().arcqml_rt_v2_adjoint_backward(
        C.byref(plan.raw), _dev_ptr(psi), _dev_ptr(lam), b, num_qubits, up.ctypes.data,
        req.ctypes.data, req.size, grads.ctypes.data, grads.size, _stream_ptr(stream)))
    return grads


SMALL_MAX_QUBITS = 10


def small_run_device(plan: CircuitPlan, observable: "Observable", initial_state, num_qubits: int,
                     requires_grad, num_gradients: int, lambda0=None, stream=None):
    """One-kernel forward + <H> + adjoint (upstream 1) of a small single state; returns
    (value, gradients). initial_state: device tensor or None for |0...0>; lambda0: optional
    device tensor receiving lambda at the start of the circuit."""
    req = np.ascontiguousarray(requires_grad, dtype=np.uint8)
    grads = np.zeros(num_gradients, dtype=np.float64)
    value = C.c_double()
    _status(load().arcqml_rt_v2_small_run(
        C.byref(plan.raw), C.byref(observable.raw),
        None if initial_state is None else _dev_ptr(initial_state), num_qubits,
        req.ctypes.data, req.size, grads.ctypes.data, grads.size, C.byref(value),
        None if lambda0 is None else _dev_ptr(lambda0), _stream_ptr(stream)))
    return float(value.value), grads


class AdamState:
    """Moments of the device optimizer loop (per parent index) and the steps taken so far."""

    def __init__(self, num_parameters: int):
        self.m = np.zeros(num_parameters, dtype=np.float64)
        self.v = np.zeros(num_parameters, dtype=np.float64)
        self.step = 0

    def update(self, values, grads, lr: float = 0.05, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 0.0) -> np.ndarray:
        """One f64 Adam step on the host (crates/arcqml-optim/src/adam.rs:190-240: coupled L2
        weight decay, bias-corrected moments); advances the moments in place and returns the
        new values. The same update the device loop (`small_adam_device`) applies per step."""
        x = np.asarray(values, dtype=np.float64)
        g = np.asarray(grads, dtype=np.float64)
        if x.shape != self.m.shape or g.shape != self.m.shape:
            raise ValueError("values and grads must match the AdamState size")
        self.step += 1
        b1, b2 = float(betas[0]), float(betas[1])
        a = g + weight_decay * x
        self.m = b1 * self.m + (1.0 - b1) * a
        self.v = b2 * self.v + (1.0 - b2) * (a * a)
        m_hat = self.m / (1.0 - b1 ** self.step)
        v_hat = self.v / (1.0 - b2 ** self.step)
        return x - lr * m_hat / (np.sqrt(v_hat) + eps)


def small_adam_device(plan: CircuitPlan, observable: "Observable", num_qubits: int, parameters,
                      requires_grad, steps: int, lr: float = 0.05,
                      betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0,
                      initial_state=None, state: "AdamState" = None, stream=None):
    """`steps` Adam steps of <H> in one launch (arcqml_rt_v2_small_adam): per step forward, <H>,
    adjoint gradient and the f64 Adam update on the device. parameters and requires_grad are
    indexed by parent (entry 0: the initial-state slot). Returns (energies before each update,
    parameters after the last one); `state` (AdamState) is advanced in place when given."""
    req = np.ascontiguousarray(requires_grad, dtype=np.uint8)
    params = np.array(parameters, dtype=np.float64, copy=True)
    if params.shape != req.shape:
        raise ValueError("parameters and requires_grad must have the same length")
    energies = np.zeros(max(int(steps), 0), dtype=np.float64)
    if state is not None and (state.m.size != params.size or state.v.size != params.size):
        raise ValueError("AdamState size does not match the parameters")
    _status(load().arcqml_rt_v2_small_adam(
        C.byref(plan.raw), C.byref(observable.raw),
        None if initial_state is None else _dev_ptr(initial_state), num_qubits,
        req.ctypes.data, params.ctypes.data, params.size,
        None if state is None else state.m.ctypes.data,
        None if state is None else state.v.ctypes.data,
        0 if state is None else int(state.step), int(steps), float(lr), float(betas[0]),
        float(betas[1]), float(eps), float(weight_decay),
        energies.ctypes.data if energies.size else None, _stream_ptr(stream)))
    if state is not None:
        state.step += int(steps)
    return energies, params


# ------------------------------------------------------------------ training over many tensors

NO_TENSOR = 4
_TENSOR = np.dtype([("data", np.uint64), ("length", np.uint64), ("dtype", np.uint32),
                    ("reserved", np.uint32)])  # ArcqmlTensor
_MATRIX = np.dtype([("data", np.uint64), ("rows", np.uint64), ("columns", np.uint64),
                    ("dtype", np.uint32), ("reserved", np.uint32)])  # ArcqmlMatrix


class AdamOptions(C.Structure):
    _fields_ = [("learning_rate", C.c_double), ("beta1", C.c_double), ("beta2", C.c_double),
                ("epsilon", C.c_double), ("weight_decay", C.c_double), ("max_norm", C.c_double),
                ("decoupled", C.c_int32), ("reserved", C.c_int32)]


_tensor_types = {}


def _tensor_kinds() -> dict:
    """torch dtype -> (code of the components, components per element, bytes per element)."""
    if not _tensor_types:
        import torch
        _tensor_types.update({
            torch.float64: (0, 1, 8), torch.float32: (1, 1, 4), torch.bfloat16: (2, 1, 2),
            torch.float16: (3, 1, 2), torch.complex128: (0, 2, 16), torch.complex64: (1, 2, 8)})
    return _tensor_types


def _kind_of(torch, t) -> str:
    """What a tensor list is told that it cannot take."""
    if torch is not None and not isinstance(t, torch.Tensor):
        return type(t).__name__
    lazy = [bit for bit, on in (("conj", t.is_conj()), ("neg", t.is_neg())) if on]
    return (f"{t.dtype} on {t.device}" + (f" laid out as {t.layout}" if str(t.layout) != "torch.strided" else "")
            + (f" with its lazy {' and '.join(lazy)} bit set (resolve_conj, resolve_neg)" if lazy else ""))


def _layout(t):
    """None for a contiguous tensor, (shape, strides) for another one that fills its memory without
    gaps or overlap; anything else is refused."""
    if t.is_contiguous():
        return None
    size = 1
    for stride, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != size:
            raise TypeError("tensors must fill their memory without gaps or overlap: got shape "
                            f"{list(t.shape)} with strides {list(t.stride())}")
        size *= n
    return tuple((n, st) for n, st in zip(t.shape, t.stride()) if n != 1)


class TensorList:
    """The tensors of a model, or their gradients, as the calls below take them: floating or complex
    CUDA tensors of one device (or one such tensor); None where a parameter has no gradient. Checking
    a list and writing it down costs about two microseconds per tensor: a training loop whose tensors
    stay keeps its lists. Every call reads the tensors' addresses anew, and one that has moved (a new
    ``.data``) is checked and written down again. For tensors that change shape or type where they are (a
    view of their own memory), or that are resized, they or their storage (``resize_``), a new list is
    made: reading shapes as well would double a call's time. A list keeps its tensors' memory alive."""

    def __init__(self, tensors):
        import torch
        self.tensors = (tensors,) if isinstance(tensors, torch.Tensor) else tuple(tensors)
        self._present = [t for t in self.tensors if t is not None]
        self._write_down()

    def __len__(self) -> int:
        return len(self.tensors)

    def __reduce__(self):  # a copy is written down anew
        return TensorList, (self.tensors,)

    def _write_down(self) -> None:
        import torch
        kinds = _tensor_kinds()
        rows, layouts, spans, devices = [], [], [], set()
        for i, t in enumerate(self.tensors):
            if t is None:
                rows.append((0, 0, NO_TENSOR, 0))
                layouts.append(None)
                continue
            kind = kinds.get(t.dtype) if isinstance(t, torch.Tensor) else None
            if kind is None or not t.is_cuda or t.layout != torch.strided or t.is_conj() or \
                    t.is_neg():
                raise TypeError("a tensor list takes dense float64, float32, bfloat16, float16 and "
                                f"complex CUDA tensors or None: place {i} holds {_kind_of(torch, t)}")
            layouts.append(None if t.is_contiguous() else _layout(t))
            devices.add(t.get_device())
            at, n = t.data_ptr(), t.numel()
            rows.append((at, n * kind[1], kind[0], 0))
            if n:
                spans.append((at, at + n * kind[2]))
        if len(devices) > 1:
            raise TypeError("the tensors of a list must be on one device")
        # With the memory held, a tensor at the address it had is in the memory it had: nothing else
        # can have been put there since.
        self._held = [t.detach() for t in self._present]
        self.device_index = devices.pop() if devices else None
        self._blank = None if self.device_index is None else torch.empty(
            0, dtype=torch.float64, device=self.device_index)
        self._table = np.array(rows or [(0, 0, NO_TENSOR, 0)], dtype=_TENSOR)
        self._address = self._table.ctypes.data
        self._words = load().arcqml_rt_v2_gradient_workspace(self._address, len(rows))
        self._adam_words = load().arcqml_rt_v2_adam_workspace(self._address, len(rows))
        self._layouts, self._spans, self._apart = layouts, spans, None
        self._shapes = [None if t is None else t.shape for t in self.tensors]
        self._pointers = [r[0] for r in rows if r[2] != NO_TENSOR]
        self._roots = self._matrices = None
        self._state = object()  # another one whenever the list is written down

    def _current(self, torch, device: int) -> int:
        """Address of the table, after a look at the tensors' addresses and the current device."""
        if list(map(torch.Tensor.data_ptr, self._present)) != self._pointers:
            self._write_down()
        if self.device_index != device and self.device_index is not None:
            raise RuntimeError(f"the tensors are on cuda:{self.device_index} and the current device "
                               f"is cuda:{device}")
        return self._address

    def _check_apart(self, name: str) -> None:
        """Refuses a list that is written to when two of its tensors share memory."""
        if self._apart is None:
            self._apart = _spans_apart(self._spans)
        if not self._apart:
            raise RuntimeError(f"{name} share memory: each may be in the list once")

    def _as_matrices(self, name: str) -> int:
        """Address of the list as a table of matrices (ArcqmlMatrix); refuses what is none."""
        if self._matrices is None:
            rows = []
            for i, t in enumerate(self.tensors):
                if t is None:
                    rows.append((0, 0, 0, NO_TENSOR, 0))
                    continue
                code, parts, _ = _tensor_kinds()[t.dtype]
                if t.dim() != 2 or parts != 1 or code == 0 or self._layouts[i] is not None:
                    raise TypeError(f"{name} are float32, bfloat16 or float16 matrices, row-major: place {i} "
                                    f"holds {_kind_of(None, t)} of shape {list(t.shape)} with strides "
                                    f"{list(t.stride())}")
                rows.append((t.data_ptr(), t.shape[0], t.shape[1], code, 0))
            self._matrices = np.array(rows or [(0, 0, 0, NO_TENSOR, 0)], dtype=_MATRIX)
            self._matrix_words = load().arcqml_rt_v2_orthogonalize_workspace(
                self._matrices.ctypes.data, len(rows))
        return self._matrices.ctypes.data

    def _written(self, torch) -> None:
        """Tells autograd that the tensors changed."""
        if self._roots is None:
            # the tensors whose version counters stand for all: views share their base's
            roots = [t._base if t._is_view() else t for t in self._present]
            self._roots = list({id(t): t for t in roots}.values())
        torch.autograd.graph.increment_version(self._roots)


def _spans_apart(spans) -> bool:
    """Whether no two of the (first, end) address ranges overlap."""
    spans = sorted(spans)
    return all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))


def _edges(spans):
    """The starts, and behind a 0 the ends, of (first, end) ranges that are sorted and apart."""
    return [s[0] for s in spans], [0] + [s[1] for s in spans]


def _check_outside(name: str, spans, edges, of: str) -> None:
    """Refuses (first, end) ranges that overlap one of those whose ``_edges`` are given."""
    starts, ends = edges
    for first, end in spans:
        # of the ranges that start before this one's end, the last one ends last
        if ends[bisect_left(starts, end)] > first:
            raise RuntimeError(f"{name} shares memory with {of}")


def _tensor_list(tensors) -> TensorList:
    return tensors if isinstance(tensors, TensorList) else TensorList(tensors)


def _call_memory(torch, device: int, blank, stream, words: int, norm: bool):
    """(stream, norm, scratch) of one call. All of it is allocated for the call alone, on its stream,
    so calls on other streams and captured graphs share nothing."""
    if stream is not None:
        with torch.cuda.stream(torch.cuda.ExternalStream(int(stream))):
            return (int(stream),) + _call_memory(torch, device, blank, None, words, norm)[1:]
    # the raw handle: a Stream object costs as much as the launch
    raw = torch._C._cuda_getCurrentRawStream(device)
    if blank is None:  # a list without tensors
        blank = torch.empty(0, dtype=torch.float64, device=device)
    return raw, blank.new_empty(()) if norm else None, blank.new_empty(words) if words else None


def _scalar_ptr(torch, device: int, t) -> int:
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == torch.float64
            and t.numel() == 1 and t.get_device() == device and not t.is_neg()):
        raise TypeError("a given norm must be one float64 on the current CUDA device, its lazy neg bit "
                        "not set")
    return t.data_ptr()


def gradient_norm_device(gradients, stream=None):
    """The 2-norm over every element of every tensor of `gradients` (a TensorList, or a sequence of
    CUDA tensors and None) as a float64 CUDA scalar (arcqml_rt_v2_gradient_norm). Nothing is read
    back: the norm can go into the calls below, or its square into an all-reduce. With `stream` the
    call runs on that stream and its result is ready there, here and below."""
    import torch
    g = _tensor_list(gradients)
    device = torch.cuda.current_device()
    table = g._current(torch, device)
    on, out, ws = _call_memory(torch, device, g._blank, stream, g._words, True)
    _status(load().arcqml_rt_v2_gradient_norm(table, len(g), out.data_ptr(),
                                              None if ws is None else ws.data_ptr(), g._words, on))
    return out


def clip_gradients_device(gradients, max_norm: float, norm=None, stream=None):
    """Scales `gradients` in place by min(1, max_norm / (n + 1e-6)) with n their global norm, or
    `norm` (a float64 CUDA scalar: over several lists, or over ranks), and returns n
    (arcqml_rt_v2_clip_gradients). No two gradients, nor the given norm and one, may share memory."""
    import torch
    g = _tensor_list(gradients)
    device = torch.cuda.current_device()
    table = g._current(torch, device)
    g._check_apart("the gradients")
    given = None if norm is None else _scalar_ptr(torch, device, norm)
    if given is not None and any(first < given + 8 and given < end for first, end in g._spans):
        raise RuntimeError("the given norm shares memory with the gradients")
    on, out, ws = _call_memory(torch, device, g._blank, stream, g._words, True)
    _status(load().arcqml_rt_v2_clip_gradients(table, len(g), float(max_norm), given,
                                               out.data_ptr(),
                                               None if ws is None else ws.data_ptr(), g._words, on))
    g._written(torch)
    return out


class _Moments(list):
    """The tensors of a written-down list. Another tensor put in a place would not be seen by the steps,
    so that is refused. Copies and pickles are plain lists."""

    def _refuse(self, *args, **kwargs):
        raise TypeError("moments are written in place (state.m[i].copy_(...)) or assigned as a whole "
                        "(state.m = [...])")

    __setitem__ = __delitem__ = __iadd__ = __imul__ = _refuse
    append = clear = extend = insert = pop = remove = reverse = sort = _refuse

    def __reduce__(self):
        return list, (list(self),)


class DeviceAdamState:
    """Moments and step count of Adam over device tensors (``adam_step_device``): ``m`` and ``v``
    hold one tensor per parameter, of its shape and strides, in float32 (float64 or complex128 for
    float64 and complex128 parameters, complex64 for complex64 ones); ``step`` is an int64 CUDA
    scalar with the steps taken. They start at zero, or continue the ones given. Saved ones go on in an
    existing state when they are copied into its tensors (``state.step.copy_``) or, for the moments,
    when whole lists are assigned."""

    def __init__(self, parameters, m=None, v=None, step=0):
        import torch
        p = _tensor_list(parameters)
        if len(p._present) != len(p):
            raise TypeError("a parameter list has no empty places")
        device = torch.device("cuda", torch.cuda.current_device() if p.device_index is None
                              else p.device_index)
        if isinstance(step, torch.Tensor):
            if step.dtype != torch.int64 or step.numel() != 1 or step.device != device:
                raise TypeError(f"the step count must be one int64 on {device}")
            self._step = step
        else:
            if int(step) < 0:
                raise ValueError("the step count must not be negative")
            self._step = torch.full((), int(step), dtype=torch.int64, device=device)
        self._m = self._fitting("first", self._zeros(p) if m is None else m, p)
        self._v = self._fitting("second", self._zeros(p) if v is None else v, p)
        self._checked = self._gradients = None

    @property
    def m(self):
        return _Moments(self._m.tensors)

    @m.setter
    def m(self, tensors):
        self._m = self._fitting("first", tensors, self._m)

    @property
    def v(self):
        return _Moments(self._v.tensors)

    @v.setter
    def v(self, tensors):
        self._v = self._fitting("second", tensors, self._v)

    @property
    def step(self):
        return self._step

    @staticmethod
    def _fitting(name: str, tensors, like: TensorList) -> TensorList:
        x = TensorList(tensors)
        if x._shapes != like._shapes or x._layouts != like._layouts:
            raise ValueError(f"the {name} moments must have the parameters' shapes and strides")
        return x

    @staticmethod
    def _zeros(p: TensorList):
        import torch
        wide = {torch.bfloat16: torch.float32, torch.float16: torch.float32}
        return [torch.zeros_like(t, dtype=wide.get(t.dtype, t.dtype)) for t in p.tensors]


def adam_step_device(parameters, gradients, state: DeviceAdamState, lr: float = 0.05,
                     betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0,
                     decoupled: bool = False, max_norm: float = None, norm=None, copies=None,
                     stream=None):
    """One Adam step over `parameters` (arcqml_rt_v2_adam_step), in place, with the update of
    ``AdamState.update``: coupled L2 weight decay, or with `decoupled` the decay applied to the
    parameter itself. With `max_norm` the gradients enter the step scaled as
    ``clip_gradients_device`` scales them (they stay as they are) and their global norm is returned;
    `norm` gives that norm instead. A parameter whose gradient is None is left as it is. `copies`
    (bfloat16 or float16 tensors, or None, one per parameter) receive the new values of float32
    parameters. What is written (parameters, moments, copies, the step count) may share no memory with
    anything else here; gradients may share theirs. The step count is on the device: a captured step
    counts on when it is replayed (`lr` and the other numbers stay those of the capture)."""
    import torch
    p, g, m, v = _tensor_list(parameters), _tensor_list(gradients), state._m, state._v
    c = None if copies is None else _tensor_list(copies)
    if len(p._present) != len(p):
        raise TypeError("a parameter list has no empty places")
    device = torch.cuda.current_device()
    if max_norm is None:
        if norm is not None:
            raise ValueError("a given norm needs max_norm")
        max_norm, given = -1.0, None
    else:
        max_norm, given = float(max_norm), None if norm is None else _scalar_ptr(torch, device, norm)
        if not max_norm >= 0.0:
            raise ValueError("the maximum norm must be finite and not negative")
    if state._step.get_device() != device:
        raise RuntimeError(f"the step count is on {state._step.device} and the current device is "
                           f"cuda:{device}")
    tables = [x._current(torch, device) for x in (p, g, m, v)]
    tables.append(None if c is None else c._current(torch, device))
    # the lists are held against one another once, and again when one is written down anew
    states = (p._state, m._state, v._state, None if c is None else c._state)
    if states != state._checked:
        for name, x in (("moments", m), ("moments", v), ("copies", c)):
            if x is not None:
                _check_places(name, x, p)
        at = state._step.data_ptr()
        written = sorted([s for x in (p, m, v, c) if x is not None for s in x._spans]
                         + [(at, at + 8)])
        if not _spans_apart(written):
            raise RuntimeError("the parameters, moments, copies and step count share memory")
        state._checked, state._gradients, state._written = states, None, _edges(written)
    # what other places read while one place is written
    written = "the parameters, moments, copies or step count"
    if state._gradients is not g._state:
        _check_places("gradients", g, p)
        _check_outside("a gradient", g._spans, state._written, written)
        state._gradients = g._state
    if given is not None:
        _check_outside("the given norm", [(given, given + 8)], state._written, written)
    options = AdamOptions(lr, betas[0], betas[1], eps, weight_decay, max_norm, bool(decoupled), 0)
    on, out, ws = _call_memory(torch, device, p._blank, stream, p._adam_words, max_norm >= 0.0)
    _status(load().arcqml_rt_v2_adam_step(
        *tables, len(p), state._step.data_ptr(), C.byref(options), given,
        None if out is None else out.data_ptr(), None if ws is None else ws.data_ptr(),
        p._adam_words, on))
    p._written(torch)
    if c is not None:
        c._written(torch)
    return out


def _check_places(name: str, x: TensorList, p: TensorList) -> None:
    """x has one place per parameter, and its tensors have the parameters' shapes and strides."""
    if len(x) != len(p):
        raise ValueError(f"{len(p)} parameters and {len(x)} {name}")
    for i, t in enumerate(x.tensors):
        if t is not None and (x._layouts[i], x._shapes[i]) != (p._layouts[i], p._shapes[i]):
            raise ValueError(f"{name} and parameters differ in shape or strides at place {i}")


# ------------------------------------------------------------------ matrices, orthogonalised updates


class MuonOptions(C.Structure):
    _fields_ = [("learning_rate", C.c_double), ("momentum", C.c_double), ("weight_decay", C.c_double),
                ("epsilon", C.c_double), ("nesterov", C.c_int32), ("steps", C.c_int32)]


def orthogonalize_device(matrices, steps: int = 5, eps: float = 1e-7, out=None, stream=None):
    """`matrices` (a TensorList or a sequence of row-major float32, bfloat16 or float16 CUDA matrices, or
    None) with their singular values pushed towards 1 (arcqml_rt_v2_orthogonalize): X = u / (|u| + eps),
    then `steps` times X <- a X + (b A + c A^2) X with A = X X^T. The results are new matrices of the same
    types, or `out` (`matrices` themselves, or others that share no memory with them). X keeps 22 bits, products
    carry 22 (11 of bfloat16 matrices of more than 128 rows and columns), summed in float32. A matrix of zeros
    stays zero."""
    import torch
    x = _tensor_list(matrices)
    device = torch.cuda.current_device()
    x._current(torch, device)
    table = x._as_matrices("the matrices")
    given = out is not None
    if given:
        y = _tensor_list(out)
        y._current(torch, device)
        _check_places("outputs", y, x)
        y._check_apart("the outputs")
        if y._pointers == x._pointers:
            x._check_apart("the matrices")
        else:
            _check_outside("an output", y._spans, _edges(_merged(x._spans)), "a matrix")
        if [a is None for a in x.tensors] != [b is None for b in y.tensors]:
            raise ValueError("outputs and matrices must have the same empty places")
    on, ws = _scratch(torch, device, x._matrix_words, stream)
    if given:
        outputs, to = list(y.tensors), y._as_matrices("the outputs")
    else:  # of the matrices' shapes and types: their table with other addresses
        outputs = _on_stream(torch, stream, lambda: [
            None if t is None else torch.empty_like(t) for t in x.tensors])
        rows = x._matrices.copy()
        rows["data"][:len(outputs)] = [0 if t is None else t.data_ptr() for t in outputs]
        to = rows.ctypes.data
    _status(load().arcqml_rt_v2_orthogonalize(table, to, len(x), int(steps), float(eps),
                                              None if ws is None else ws.data_ptr(), x._matrix_words, on))
    if given:
        y._written(torch)
    return outputs


class DeviceMuonState:
    """Momentum of ``muon_step_device``: one float32 tensor per parameter, of its shape. It starts at zero,
    or continues the one given. A saved one goes on in an existing state when it is copied into its tensors
    or assigned as a whole."""

    def __init__(self, parameters, momentum=None):
        import torch
        p = _tensor_list(parameters)
        if len(p._present) != len(p):
            raise TypeError("a parameter list has no empty places")
        p._as_matrices("the parameters")
        zeros = [torch.zeros_like(t, dtype=torch.float32) for t in p.tensors] if momentum is None else momentum
        self._momentum = self._fitting(zeros, p)
        self._checked = self._gradients = None

    @property
    def momentum(self):
        return _Moments(self._momentum.tensors)

    @momentum.setter
    def momentum(self, tensors):
        self._momentum = self._fitting(tensors, self._momentum)

    @staticmethod
    def _fitting(tensors, like: TensorList) -> TensorList:
        x = TensorList(tensors)
        if x._shapes != like._shapes or len(x._present) != len(x):
            raise ValueError("the momentum must have the parameters' shapes")
        x._as_matrices("the momentum")
        if any(_tensor_kinds()[t.dtype][0] != 1 for t in x.tensors):  # (matrices of one component)
            raise TypeError("the momentum must be float32")
        return x


def muon_step_device(parameters, gradients, state: DeviceMuonState, lr: float = 0.02, momentum: float = 0.95,
                     nesterov: bool = True, weight_decay: float = 0.0, steps: int = 5, eps: float = 1e-7,
                     stream=None) -> None:
    """One step over `parameters` (row-major float32, bfloat16 or float16 CUDA matrices) in place, whose
    update is orthogonalised (arcqml_rt_v2_muon_step): m <- momentum m + (1 - momentum) g; u = m, or
    momentum m + (1 - momentum) g with `nesterov`; p <- (1 - lr weight_decay) p - lr sqrt(max(1, rows /
    columns)) X(u), X as ``orthogonalize_device`` forms it with the precision of the parameter's type. A
    parameter whose gradient is None is left as it is. Parameters and momentum may share no memory with
    anything else here; gradients may share theirs."""
    import torch
    p, g, m = _tensor_list(parameters), _tensor_list(gradients), state._momentum
    if len(p._present) != len(p):
        raise TypeError("a parameter list has no empty places")
    device = torch.cuda.current_device()
    for x in (p, g, m):
        x._current(torch, device)
    tables = [x._as_matrices(name) for x, name in ((p, "the parameters"), (g, "the gradients"),
                                                   (m, "the momentum"))]
    # held against one another once, and again when a list is written down anew
    if state._checked != (p._state, m._state):
        _check_places("momenta", m, p)
        written = sorted(p._spans + m._spans)
        if not _spans_apart(written):
            raise RuntimeError("the parameters and momentum share memory")
        state._checked, state._gradients, state._written = (p._state, m._state), None, _edges(written)
    if state._gradients is not g._state:
        _check_places("gradients", g, p)
        _check_outside("a gradient", g._spans, state._written, "the parameters or momentum")
        state._gradients = g._state
    options = MuonOptions(lr, momentum, weight_decay, eps, bool(nesterov), int(steps))
    on, ws = _scratch(torch, device, p._matrix_words, stream)
    _status(load().arcqml_rt_v2_muon_step(*tables, len(p), C.byref(options),
                                          None if ws is None else ws.data_ptr(), p._matrix_words, on))
    p._written(torch)


def _merged(spans):
    """(first, end) ranges sorted, those that overlap put together."""
    out = []
    for first, end in sorted(spans):
        if out and first < out[-1][1]:
            out[-1] = (out[-1][0], max(end, out[-1][1]))
        else:
            out.append((first, end))
    return out


def _on_stream(torch, stream, make):
    if stream is None:
        return make()
    with torch.cuda.stream(torch.cuda.ExternalStream(int(stream))):
        return make()


def _scratch(torch, device: int, words: int, stream):
    """(stream, scratch) of one call, allocated for it alone on its stream."""
    on = torch._C._cuda_getCurrentRawStream(device) if stream is None else int(stream)
    if not words:
        return on, None
    return on, _on_stream(torch, stream, lambda: torch.empty(words, dtype=torch.float64, device=device))


# ------------------------------------------------------------------ tables looked up by index


# ArcqmlRows and ArcqmlEmbeddingOptions as bytes: a ctypes structure costs three times as much to fill
_EMBEDDING_ROWS, _EMBEDDING_OPTIONS = struct.Struct("=QQQQII").pack, struct.Struct("=dqii").pack


def _embedding_rows(torch, t, outer: int, name: str, device: int):
    """A tensor as rows, its first `outer` dimensions counting them, the others a row: (rows, elements of a
    row, the tensor as ArcqmlRows)."""
    kind = _tensor_kinds().get(t.dtype) if isinstance(t, torch.Tensor) else None
    if kind is None or not t.is_cuda or t.layout != torch.strided or t.is_conj() or t.is_neg():
        raise TypeError(f"{name} must be a dense float64, float32, bfloat16, float16 or complex CUDA tensor: "
                        f"got {_kind_of(torch, t)}")
    if t.get_device() != device:
        raise RuntimeError(f"{name} is on cuda:{t.get_device()} and the current device is cuda:{device}")
    shape = t.shape
    if len(shape) <= outer:
        raise TypeError(f"{name} has no dimension for its rows' elements: its shape is {list(shape)}")
    width, rows, step = 1, 1, None
    if t.is_contiguous():
        for n in shape[:outer]:
            rows *= n
        for n in shape[outer:]:
            width *= n
        step = width
    else:
        strides, fits = t.stride(), True
        for n, st in zip(reversed(shape[outer:]), reversed(strides[outer:])):
            fits = fits and (n == 1 or st == width)
            width *= n
        for n, st in zip(reversed(shape[:outer]), reversed(strides[:outer])):
            if n != 1:
                fits = fits and (step is None or st == step * rows)
                step = st if step is None else step
            rows *= n
        if not fits and rows and width:
            raise TypeError(f"{name} must have rows without gaps at equal distances: got shape {list(shape)} "
                            f"with strides {list(strides)}")
        step = width if step is None else step
    code, parts, _ = kind
    return rows, width * parts, _EMBEDDING_ROWS(t.data_ptr(), rows, width * parts, step * parts, code, 0)


def _embedding_call(torch, indices, scale, normalize, padding, device: int):
    """The options of a call (ArcqmlEmbeddingOptions), after a look at its indices."""
    kind = indices.dtype if isinstance(indices, torch.Tensor) and indices.is_cuda else None
    if kind != torch.int64 and kind != torch.int32:
        raise TypeError("indices must be an int64 or int32 CUDA tensor")
    if indices.get_device() != device:
        raise RuntimeError(f"the indices are on cuda:{indices.get_device()} and the current device is "
                           f"cuda:{device}")
    if padding is None:
        padding = -1
    elif not 0 <= padding < 1 << 63:
        raise ValueError("the padding index must not be negative, and fit into 8 bytes")
    return _EMBEDDING_OPTIONS(scale, padding, bool(normalize), 8 if kind == torch.int64 else 4)


def embedding_lookup_device(table, indices, scale: float = 1.0, normalize: bool = False, padding=None,
                            stream=None):
    """Rows of `table` ([rows, ...], rows without gaps) picked by `indices` (int64 or int32 CUDA tensor):
    ``scale * table[indices]`` of shape [*indices.shape, ...], with `normalize` each row over its 2-norm
    (states from trained amplitudes; a row of zeros stays zero) (arcqml_rt_v2_embedding_lookup). Places
    whose index is `padding` are zero. An index outside the table gives NaN: refusing it would wait for the
    device."""
    import torch
    if stream is not None:
        with torch.cuda.stream(torch.cuda.ExternalStream(int(stream))):
            return embedding_lookup_device(table, indices, scale, normalize, padding)
    device = torch.cuda.current_device()
    _, width, rows = _embedding_rows(torch, table, 1, "the table", device)
    options = _embedding_call(torch, indices, scale, normalize, padding, device)
    if not indices.is_contiguous():
        indices = indices.contiguous()
    out = table.new_empty(indices.shape + table.shape[1:])
    n = indices.numel()
    if n and width:
        lib, ws, words = load(), None, 0
        if normalize:
            words = lib.arcqml_rt_v2_embedding_lookup_workspace(rows, n, options)
            ws = torch.empty(words, dtype=torch.float64, device=table.device) if words else None
        kind = _tensor_kinds()[out.dtype][0]
        _status(lib.arcqml_rt_v2_embedding_lookup(
            rows, indices.data_ptr(), n, options, _EMBEDDING_ROWS(out.data_ptr(), n, width, width, kind, 0),
            None if ws is None else ws.data_ptr(), words, torch._C._cuda_getCurrentRawStream(device)))
    return out


def embedding_gradient_device(gradient, indices, rows: int, scale: float = 1.0, table=None, padding=None,
                              stream=None):
    """The gradient of a table of `rows` rows from `gradient` ([*indices.shape, ...]), the gradient of its
    lookup by `indices` (arcqml_rt_v2_embedding_gradient): for each row `scale` times the sum over its places,
    zeros where there is none. With `table` the lookup was a normalised one of that table, and the sum is
    taken through the rows' norms. A row's places are added in their order: equal inputs give equal bits."""
    import torch
    if stream is not None:
        with torch.cuda.stream(torch.cuda.ExternalStream(int(stream))):
            return embedding_gradient_device(gradient, indices, rows, scale, table, padding)
    device = torch.cuda.current_device()
    options = _embedding_call(torch, indices, scale, table is not None, padding, device)
    outer = indices.dim()
    if not isinstance(gradient, torch.Tensor) or gradient.shape[:outer] != indices.shape:
        raise ValueError("the gradient must have a row for each index")
    _, width, g = _embedding_rows(torch, gradient, outer, "the gradient", device)
    rows = int(rows)
    if rows < 0:
        raise ValueError("a table has no negative number of rows")
    shape = (rows,) + gradient.shape[outer:]
    t = None
    if table is not None:
        _, _, t = _embedding_rows(torch, table, 1, "the table", device)
        if table.dtype != gradient.dtype or table.shape != shape:
            raise ValueError(f"the table must be {gradient.dtype} of shape {list(shape)}")
    if not indices.is_contiguous():
        indices = indices.contiguous()
    out = gradient.new_empty(shape)
    if rows and width:
        lib = load()
        words = lib.arcqml_rt_v2_embedding_gradient_workspace(g, rows, options)
        ws = torch.empty(words, dtype=torch.float64, device=out.device) if words else None
        kind = _tensor_kinds()[out.dtype][0]
        _status(lib.arcqml_rt_v2_embedding_gradient(
            g, indices.data_ptr(), options, t, _EMBEDDING_ROWS(out.data_ptr(), rows, width, width, kind, 0),
            None if ws is None else ws.data_ptr(), words, torch._C._cuda_getCurrentRawStream(device)))
    return out


def norms_device(state, num_qubits: int, stream=None) -> np.ndarray:
    b = _rows(state, num_qubits)
    out = np.zeros(b, dtype=np.float64)
    _status(load().arcqml_rt_v2_norms(_dev_ptr(state), b, num_qubits, out.ctypes.data,
                                      _stream_ptr(stream)))
    return out


def norms_device_noalloc(state, num_qubits: int, stream=None) -> np.ndarray:
    """Row norms through the entry point that allocates no device memory (see its header)."""
    b = _rows(state, num_qubits)
    out = np.zeros(b, dtype=np.float64)
    _status(load().arcqml_rt_v2_norms_noalloc(_dev_ptr(state), b, num_qubits, out.ctypes.data,
                                              _stream_ptr(stream)))
    return out


def set_basis_state_device(state, num_qubits: int, index: int = 0, stream=None) -> None:
    b = _rows(state, num_qubits)
    _status(load().arcqml_rt_v2_set_basis_state(_dev_ptr(state), b, num_qubits, index,
                                                _stream_ptr(stream)))


# ------------------------------------------------------------------ kernel timing

PROFILE_CATEGORIES = ("gate", "fused_forward", "fused_adjoint", "adjoint_step", "observable",
                      "other", "shard_slices")


def sample_indices_device(state, num_qubits: int, shots: int, seed: int, stream=None):
    """Basis index of every shot (numpy uint64) and the state's norm squared; see
    arcqml_rt_v2_sample (bit-exact with the reference's sample_counts)."""
    out = np.zeros(max(int(shots), 1), dtype=np.uint64)
    norm = C.c_double()
    _status(load().arcqml_rt_v2_sample(_dev_ptr(state), num_qubits, int(shots),
                                       int(seed) & ((1 << 64) - 1), out.ctypes.data,
                                       C.byref(norm), _stream_ptr(stream)))
    return out[:int(shots)], float(norm.value)


def shard_slices(shard, num_local_qubits: int, positions: Sequence[int], chunk_begin: int,
                 chunk_len: int, skip_value: int, staging, unpack: bool, stream=None) -> None:
    """Moves slices of a shard to (unpack=False) or from (unpack=True) contiguous staging
    blocks, one block per slice value other than ``skip_value`` (see arcqml_rt_v2_shard_slices)."""
    pos = (C.c_uint32 * len(positions))(*positions)
    _status(load().arcqml_rt_v2_shard_slices(
        _dev_ptr(shard), num_local_qubits, pos, len(positions), chunk_begin, chunk_len,
        skip_value, _dev_ptr(staging), int(bool(unpack)), _stream_ptr(stream)))


def shard_slices_from(shard, num_local_qubits: int, positions: Sequence[int], chunk_begin: int,
                      chunk_len: int, sources: Sequence[Optional[int]], stream=None) -> None:
    """Gathers slice value y of a chunk from device address sources[y] (None: skip) into the
    shard (see arcqml_rt_v2_shard_slices_from)."""
    pos = (C.c_uint32 * len(positions))(*positions)
    src = (C.c_void_p * len(sources))(*[s if s else None for s in sources])
    _status(load().arcqml_rt_v2_shard_slices_from(
        _dev_ptr(shard), num_local_qubits, pos, len(positions), chunk_begin, chunk_len, src,
        _stream_ptr(stream)))


def shard_swap_nccl(shard, num_local_qubits: int, global_bits: Sequence[int],
                    local_positions: Sequence[int], nccl_comm: int, staging,
                    stream=None) -> None:
    """Swaps the global qubits at rank bits global_bits[i] with the shard's local positions
    local_positions[i] over a raw NCCL communicator (arcqml_rt_v2_shard_swap_nccl); staging is a
    complex128 CUDA tensor of scratch amplitudes."""
    gb = (C.c_uint32 * len(global_bits))(*global_bits)
    lp = (C.c_uint32 * len(local_positions))(*local_positions)
    _status(load().arcqml_rt_v2_shard_swap_nccl(
        _dev_ptr(shard), num_local_qubits, gb, lp, len(global_bits), C.c_void_p(nccl_comm),
        _dev_ptr(staging), staging.numel(), _stream_ptr(stream)))


def shard_slices_ptr(shard, num_local_qubits: int, positions: Sequence[int], chunk_begin: int,
                     chunk_len: int, skip_value: int, staging_address: int, unpack: bool,
                     stream=None) -> None:
    """shard_slices with the staging buffer given as a raw device address."""
    pos = (C.c_uint32 * len(positions))(*positions)
    _status(load().arcqml_rt_v2_shard_slices(
        _dev_ptr(shard), num_local_qubits, pos, len(positions), chunk_begin, chunk_len,
        skip_value, C.c_void_p(staging_address), int(bool(unpack)), _stream_ptr(stream)))


class PeerBuffer:
    """A device buffer other processes of the node can map (CUDA IPC)."""

    def __init__(self, nbytes: int):
        ptr = C.c_void_p()
        self.handle = (C.c_uint8 * 64)()
        _status(load().arcqml_rt_v2_peer_buffer_create(nbytes, C.byref(ptr), self.handle))
        self.address = int(ptr.value)
        self.nbytes = nbytes

    def handle_bytes(self) -> bytes:
        return bytes(self.handle)

    @staticmethod
    def open(handle: bytes) -> int:
        ptr = C.c_void_p()
        h = (C.c_uint8 * 64)(*handle)
        _status(load().arcqml_rt_v2_peer_buffer_open(h, C.byref(ptr)))
        return int(ptr.value)

    @staticmethod
    def close(address: int) -> None:
        _status(load().arcqml_rt_v2_peer_buffer_close(C.c_void_p(address)))

    def destroy(self) -> None:
        if self.address:
            _status(load().arcqml_rt_v2_peer_buffer_destroy(C.c_void_p(self.address)))
            self.address = 0


def profile_enable(on: bool = True) -> None:
    """Bracket the runtime's kernel launches with CUDA events (resets the totals)."""
    load().arcqml_rt_v2_profile_enable(int(on))


def profile_read() -> dict:
    """{category: (launches, total_ms, algorithmic_bytes)} since the last profile_enable."""
    out = {}
    for i, name in enumerate(PROFILE_CATEGORIES):
        n = C.c_uint64()
        ms = C.c_double()
        by = C.c_double()
        _status(load().arcqml_rt_v2_profile_read(i, C.byref(n), C.byref(ms), C.byref(by)))
        out[name] = (int(n.value), float(ms.value), float(by.value))
    return out


def launch_count() -> int:
    return int(load().arcqml_rt_v2_launch_count())


def jit_info() -> dict:
    """Run-time compiled pass kernels: {compiled, launches, fallbacks, last_error}."""
    c, l, f = C.c_uint64(), C.c_uint64(), C.c_uint64()
    buf = C.create_string_buffer(4096)
    load().arcqml_rt_v2_jit_info(C.byref(c), C.byref(l), C.byref(f), buf, 4096)
    return {"compiled": int(c.value), "launches": int(l.value), "fallbacks": int(f.value),
            "last_error": buf.value.decode("utf-8", errors="replace")}


def plan_emulate(plan: CircuitPlan, state, num_qubits: int, adjoint: bool = False, lam=None,
                 requires_grad=None, num_gradients: int = 0):
    """The engine's fused-pass schedule run on the CPU (arcqml_rt_v2_plan_emulate): returns the
    new state, or (psi, lambda, gradients) for the adjoint sweep. numpy complex128 inputs."""
    a = np.ascontiguousarray(state, dtype=np.complex128).copy()
    if not adjoint:
        _status(load().arcqml_rt_v2_plan_emulate(C.byref(plan.raw), a.ctypes.data, num_qubits, 0,
                                                 None, None, 0, None, 0))
        return a
    lm = np.ascontiguousarray(lam, dtype=np.complex128).copy()
    req = np.ascontiguousarray(requires_grad, dtype=np.uint8)
    grads = np.zeros(num_gradients, dtype=np.float64)
    _status(load().arcqml_rt_v2_plan_emulate(C.byref(plan.raw), a.ctypes.data, num_qubits, 1,
                                             lm.ctypes.data, req.ctypes.data, req.size,
                                             grads.ctypes.data, grads.size))
    return a, lm, grads


def plan_structure_key(ops: Sequence[PlanOp]) -> tuple:
    """What a plan holds besides its bound parameter values: per operation the opcode, qubits,
    parameter bindings, constant slot values and custom matrix. Plans with equal keys differ
    only in values that CircuitPlan.set_parameters replaces."""
    key = []
    for o in ops:
        bound = {slot for slot, _ in o.bindings}
        fixed = tuple(v for i, v in enumerate(o.params) if i not in bound)
        mat = None if o.matrix is None else np.asarray(o.matrix, dtype=np.complex128).tobytes()
        key.append((o.opcode, tuple(o.qubits), tuple(o.bindings), fixed, mat))
    return tuple(key)


def plan_bound_values(ops: Sequence[PlanOp]) -> Optional[np.ndarray]:
    """The parent values the operations' bindings carry (index = parent), for
    CircuitPlan.set_parameters; None when one parent carries two different values."""
    vals = {}
    for o in ops:
        for slot, parent in o.bindings:
            v = float(o.params[slot])
            if vals.setdefault(int(parent), v) != v:
                return None
    out = np.zeros(max(vals) + 1 if vals else 0)
    for p, v in vals.items():
        out[p] = v
    return out


def plan_schedule_export(plan: CircuitPlan, num_qubits: int, adjoint: bool = False,
                         requires_grad=None) -> bytes:
    """The engine's fused-pass schedule for the plan, serialised (arcqml_rt_v2_plan_schedule_export)."""
    req = np.ascontiguousarray([] if requires_grad is None else requires_grad, dtype=np.uint8)
    rp = req.ctypes.data if req.size else None
    size = C.c_size_t()
    _status(load().arcqml_rt_v2_plan_schedule_export(C.byref(plan.raw), num_qubits, int(adjoint),
                                                     rp, req.size, None, 0, C.byref(size)))
    buf = (C.c_uint8 * max(1, size.value))()
    _status(load().arcqml_rt_v2_plan_schedule_export(C.byref(plan.raw), num_qubits, int(adjoint),
                                                     rp, req.size, buf, size.value, C.byref(size)))
    return bytes(buf)[:size.value]


def plan_schedule_summary(plan: CircuitPlan, num_qubits: int, adjoint: bool = False,
                          requires_grad=None) -> dict:
    """Counts over the engine's fused-pass schedule (plan_schedule_export): passes, ops executed,
    rotation ops (one-qubit RX/RY forms and one-qubit phase diagonals, the ops whose FP64 work
    the scaled forms make one FMA per amplitude component), gradient rows and the further
    parameters that merged rotations add to a row. Layouts: arcqml_b200/csrc/fused.h."""
    blob = plan_schedule_export(plan, num_qubits, adjoint, requires_grad)
    off = 0

    def u32():
        nonlocal off
        v = int.from_bytes(blob[off:off + 4], "little")
        off += 4
        return v

    out = {"passes": 0, "ops": 0, "rotations": 0, "rows": 0, "aliases": 0, "custom": 0}
    for _ in range(u32()):
        if not u32():
            u32()
            out["custom"] += 1
            continue
        out["passes"] += 1
        off += 48                       # PassHeader
        nsub = u32()
        off += 24 * nsub                # SubBlocks
        nops = u32()
        for i in range(nops):           # FOp: kind at byte 0, code at byte 28
            kind, code = blob[off + 64 * i], blob[off + 64 * i + 28]
            if kind in (1, 2) or (kind == 3 and code in (4, 5)):
                out["rotations"] += 1
        out["ops"] += nops
        off += 64 * nops
        nmat = u32()
        off += 16 * nmat                # matrix entries
        rows = u32()
        out["rows"] += rows
        off += 8 * rows
        nal = u32()
        out["aliases"] += nal
        off += 16 * nal
        ncode = u32()
        off += ncode                    # compiled source
    if off != len(blob):
        raise RuntimeError("schedule export: unexpected length")
    return out


# ---------------------------------------------------------------- state analysis


def _selection(qubits):
    q = np.ascontiguousarray([int(x) for x in qubits], dtype=np.uintp)
    return q, (q.ctypes.data if q.size else None)


def probabilities_device(state, num_qubits: int, out=None, stream=None):
    """|psi_i|^2 of every row (arcqml_rt_v2_probabilities): a float64 CUDA tensor shaped like
    the state."""
    import torch
    b = _rows(state, num_qubits)
    if out is None:
        out = torch.empty(state.shape, dtype=torch.float64, device=state.device)
    _status(load().arcqml_rt_v2_probabilities(_dev_ptr(state), b, num_qubits, _dev_ptr_f64(out),
                                              _stream_ptr(stream)))
    return out


def marginal_probabilities_device(state, num_qubits: int, qubits, out=None, stream=None):
    """Marginal probabilities of the selected qubits (highest selected qubit as the most
    significant output bit) for every row: float64 CUDA tensor [2^k] or [batch, 2^k]."""
    import torch
    b = _rows(state, num_qubits)
    q, qp = _selection(qubits)
    if qp is None:  # empty selection: rejected by the runtime with the reference's message
        q = np.zeros(1, dtype=np.uintp)
        qp = q.ctypes.data
        q = q[:0]
    if out is None:
        shape = (1 << q.size,) if state.dim() == 1 else (b, 1 << q.size)
        out = torch.empty(shape, dtype=torch.float64, device=state.device)
    _status(load().arcqml_rt_v2_marginal_probabilities(
        _dev_ptr(state), b, num_qubits, qp, q.size, _dev_ptr_f64(out), _stream_ptr(stream)))
    return out


def bloch_vector_device(state, num_qubits: int, qubit: int, stream=None) -> np.ndarray:
    """(<X>, <Y>, <Z>) of one qubit per row: numpy [3] or [batch, 3]."""
    b = _rows(state, num_qubits)
    out = np.zeros((b, 3), dtype=np.float64)
    _status(load().arcqml_rt_v2_bloch_vector(_dev_ptr(state), b, num_qubits, int(qubit),
                                             out.ctypes.data, _stream_ptr(stream)))
    return out[0] if state.dim() == 1 else out


def overlap_device(lhs, rhs, num_qubits: int, stream=None):
    """<lhs|rhs> per row: a complex (1-D states) or a numpy complex array [batch]."""
    b = _rows(lhs, num_qubits)
    if rhs.shape != lhs.shape:
        raise RuntimeError("overlap of states with different shapes")
    out = np.zeros((b, 2), dtype=np.float64)
    _status(load().arcqml_rt_v2_overlap(_dev_ptr(lhs), _dev_ptr(rhs), b, num_qubits,
                                        out.ctypes.data, _stream_ptr(stream)))
    z = out[:, 0] + 1j * out[:, 1]
    return complex(z[0]) if lhs.dim() == 1 else z


def probability_cotangent_device(state, num_qubits: int, upstream, qubits=None, out=None,
                                 stream=None):
    """lambda_i = upstream[bin(i)] psi_i per row (arcqml_rt_v2_probability_cotangent): the
    adjoint sweep's lambda for an upstream gradient of the (marginal) probabilities; qubits=None
    for the full probability vector. upstream: float64 CUDA tensor [batch, 2^k] (or [2^k])."""
    import torch
    b = _rows(state, num_qubits)
    if qubits is None:
        q, qp, k = None, None, num_qubits
    else:
        # an explicit empty selection keeps a non-null pointer: the runtime rejects it
        q = np.ascontiguousarray([int(x) for x in qubits] or [0], dtype=np.uintp)
        qp, k = q.ctypes.data, len(list(qubits))
    if upstream.numel() != b << k:
        raise RuntimeError(f"upstream has {upstream.numel()} values, expected {b << k}")
    if out is None:
        out = torch.empty_like(state)
    _status(load().arcqml_rt_v2_probability_cotangent(
        _dev_ptr(state), b, num_qubits, qp, 0 if qubits is None else k, _dev_ptr_f64(upstream),
        _dev_ptr(out), _stream_ptr(stream)))
    return out


def scaled_copy_device(state, num_qubits: int, factors, out=None, stream=None):
    """out[row] = factors[row] * state[row] with complex factors (arcqml_rt_v2_scaled_copy)."""
    import torch
    b = _rows(state, num_qubits)
    f = np.asarray(factors, dtype=np.complex128).reshape(-1)
    if f.size == 1 and b > 1:
        f = np.full(b, f[0])
    if f.size != b:
        raise RuntimeError(f"{f.size} factors for {b} rows")
    fr = np.ascontiguousarray(np.stack([f.real, f.imag], axis=1).reshape(-1))
    if out is None:
        out = torch.empty_like(state)
    _status(load().arcqml_rt_v2_scaled_copy(_dev_ptr(state), b, num_qubits, fr.ctypes.data,
                                            _dev_ptr(out), _stream_ptr(stream)))
    return out
