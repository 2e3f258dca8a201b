"""Optimizers for hybrid models: ``Adam`` over circuits' parameters and device tensors together, ``Muon`` over
the matrices of the network beside them.

A model whose circuit is fed by a classical network, or starts from trained states, has its
parameters in two places: the circuit's on the host (``Circuit.parameters``, bound into plans) and
the others in CUDA tensors. ``Adam`` takes both, clips by the global norm of all their gradients and
updates them in one ``runtime.adam_step_device``; the update is that of ``runtime.AdamState.update``
(``crates/arcqml-optim/src/adam.rs:190-240``). Gradients are read where the backward passes leave
them: ``Parameter.grad`` (``RunResult.backward``, ``StateVectorSimulator.gradient``,
``UnitaryLoss.backward``) and ``Tensor.grad``. ``RunResult.backward``'s initial-state gradient is in
torch's convention for complex tensors, so a network that made the states gets its gradients by
``states.backward(initial_state_grad)``. Amplitudes are trained the same way, through the normalisation that
makes states of them: a step on normalised states themselves would leave them unnormalised, which
``BatchStateVectorSimulator.from_device_state`` does not check (``embedding.lookup`` with ``normalize`` does
both for a table of amplitudes).
"""
from __future__ import annotations

import numpy as np

from . import runtime as rt


class _CircuitParameters:
    """The trained parameters of one type of a circuit, as a vector on the device for the step. The
    host's values are the ones that count: they go up with the gradients and come back."""

    def __init__(self, parameters, dtype):
        import torch
        self.parameters = parameters
        n = len(parameters)
        self.host = torch.zeros((2, n), dtype=dtype, pin_memory=True)
        self.device = torch.zeros((2, n), dtype=dtype, device="cuda")
        self.values, self.gradient = self.device[0], self.device[1]

    def upload(self) -> bool:
        """False when there is no gradient at all."""
        grads = [getattr(p, "grad", None) for p in self.parameters]
        missing = sum(g is None for g in grads)
        if missing == len(grads):
            return False
        if missing:
            raise ValueError(f"{missing} of a circuit's {len(grads)} trained parameters have no "
                             "gradient")
        h = self.host.numpy()
        h[0] = [p.f64() for p in self.parameters]
        h[1] = grads
        self.device.copy_(self.host, non_blocking=True)
        return True

    def download(self) -> None:
        """Starts the copy; ``take`` reads it after the stream has been waited for."""
        self.host[0].copy_(self.values, non_blocking=True)

    def take(self) -> None:
        for p, x in zip(self.parameters, self.host[0].tolist()):
            p.value = x


def _resolved(gradient):
    """A gradient with its values in memory: autograd leaves a complex one conjugated by a bit alone
    when the loss took its tensor's conjugate."""
    if gradient is None or not (gradient.is_conj() or gradient.is_neg()):
        return gradient
    return gradient.resolve_conj().resolve_neg()


class Adam:
    """Adam over ``circuits`` (the parameters with ``requires_grad`` that they have now) and
    ``tensors`` (floating or complex CUDA tensors that autograd leaves gradients in, or one such
    tensor). ``weight_decay`` is coupled (added to the gradient, as in the reference) unless
    ``decoupled``; ``max_norm`` clips by the global norm of all gradients. A tensor without gradient,
    and a circuit without any, stays as it is and out of the norm. The moments and the step count are
    ``state`` (``runtime.DeviceAdamState``), the circuits' vectors first."""

    def __init__(self, circuits=(), tensors=(), lr: float = 0.05, betas=(0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 0.0, decoupled: bool = False,
                 max_norm: float = None):
        import torch
        self.lr, self.betas, self.eps = lr, betas, eps
        self.weight_decay, self.decoupled, self.max_norm = weight_decay, decoupled, max_norm
        self._tensors = (tensors,) if isinstance(tensors, torch.Tensor) else tuple(tensors)
        for i, t in enumerate(self._tensors):
            if t is None:
                raise TypeError("the tensors to train must not be None")
            if isinstance(t, torch.Tensor) and not (t.is_leaf or t.retains_grad):
                raise ValueError(f"the tensor to train at place {i} was computed from others: its "
                                 "gradient would go to them")
        parts = []
        for c in circuits:
            for name, dtype in (("f64", torch.float64), ("f32", torch.float32)):
                trained = [p for p in c.parameters if p.requires_grad and p.dtype == name]
                if trained:
                    parts.append((trained, dtype))
        everything = [id(p) for trained, _ in parts for p in trained]
        if len(set(everything)) != len(everything):
            raise ValueError("a circuit parameter may be trained once")
        if not parts and not self._tensors:
            raise ValueError("there is nothing to train")
        rt.TensorList(self._tensors)._check_apart("the tensors")
        self._circuits = [_CircuitParameters(p, d) for p, d in parts]
        self._parameters = rt.TensorList([c.values for c in self._circuits] + list(self._tensors))
        self.state = rt.DeviceAdamState(self._parameters)

    @property
    def tensors(self) -> tuple:
        """The trained tensors. Others need an optimizer, and moments, of their own."""
        return self._tensors

    def zero_grad(self) -> None:
        for c in self._circuits:
            for p in c.parameters:
                p.grad = None
        for t in self._tensors:
            t.grad = None

    def step(self):
        """One step. Returns the gradients' norm before clipping (a float64 CUDA scalar), or None
        without ``max_norm``. Waits for the step only to bring circuits' parameters back."""
        import torch
        has = [c.upload() for c in self._circuits]
        grads = [c.gradient if h else None for c, h in zip(self._circuits, has)]
        grads += [t.grad for t in self._tensors]
        # a new list every step: one that is kept would keep the gradients' memory
        try:
            grads = rt.TensorList(grads)
        except TypeError:  # what it refuses may only have to be resolved; looking first costs more
            grads = rt.TensorList([_resolved(g) for g in grads])
        norm = rt.adam_step_device(self._parameters, grads, self.state, lr=self.lr,
                                   betas=self.betas, eps=self.eps, weight_decay=self.weight_decay,
                                   decoupled=self.decoupled, max_norm=self.max_norm)
        moved = [c for c, h in zip(self._circuits, has) if h]
        for c in moved:
            c.download()
        if moved:
            torch.cuda.current_stream().synchronize()
        for c in moved:
            c.take()
        return norm


class Muon:
    """Momentum steps whose update is orthogonalised (``runtime.muon_step_device``), over the matrices of a
    network (row-major float32, bfloat16 or float16 CUDA leaves, or one of them). Vectors, tables, circuits'
    parameters and amplitudes go into an ``Adam`` of their own. A matrix without gradient stays as it is. The
    momentum is ``state`` (``runtime.DeviceMuonState``)."""

    def __init__(self, matrices, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.0, steps: int = 5, eps: float = 1e-7):
        import torch
        self.lr, self.momentum, self.nesterov = lr, momentum, nesterov
        self.weight_decay, self.steps, self.eps = weight_decay, steps, eps
        self._matrices = (matrices,) if isinstance(matrices, torch.Tensor) else tuple(matrices)
        if not self._matrices:
            raise ValueError("there is nothing to train")
        for i, t in enumerate(self._matrices):
            if t is None:
                raise TypeError("the matrices to train must not be None")
            if isinstance(t, torch.Tensor) and not (t.is_leaf or t.retains_grad):
                raise ValueError(f"the matrix to train at place {i} was computed from others: its "
                                 "gradient would go to them")
        self._parameters = rt.TensorList(self._matrices)
        self._parameters._check_apart("the matrices")
        self.state = rt.DeviceMuonState(self._parameters)

    @property
    def matrices(self) -> tuple:
        """The trained matrices. Others need an optimizer, and momentum, of their own."""
        return self._matrices

    def zero_grad(self) -> None:
        for t in self._matrices:
            t.grad = None

    def step(self) -> None:
        """One step. Nothing is waited for."""
        # a new list every step: one that is kept would keep the gradients' memory
        grads = rt.TensorList([t.grad for t in self._matrices])
        rt.muon_step_device(self._parameters, grads, self.state, lr=self.lr, momentum=self.momentum,
                            nesterov=self.nesterov, weight_decay=self.weight_decay, steps=self.steps,
                            eps=self.eps)
