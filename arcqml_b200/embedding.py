"""Tables looked up by index: token embeddings of a hybrid model's network, and states made of trained
amplitudes.

``lookup`` picks rows of a table and is differentiable in it; with ``normalize`` each row comes divided by its
norm, so that a table of amplitudes gives states. ``BatchStateVectorSimulator.from_table`` makes a batch of
such states; the table gets its gradient by ``sim.states.backward(initial_state_grad)`` with the
initial-state gradient of ``RunResult.backward`` (in torch's convention for complex tensors).
"""
from __future__ import annotations

from . import runtime as rt


def _function():
    import torch

    class Lookup(torch.autograd.Function):
        @staticmethod
        def forward(ctx, table, indices, scale, normalize, padding):
            ctx.scale, ctx.padding, ctx.normalize = scale, padding, normalize
            ctx.rows, ctx.inner = table.shape[0], table.dim() - 1
            ctx.save_for_backward(indices, *((table,) if normalize else ()))
            return rt.embedding_lookup_device(table.detach(), indices, scale=scale, normalize=normalize,
                                              padding=padding)

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, gradient):
            indices = ctx.saved_tensors[0]
            table = ctx.saved_tensors[1].detach() if ctx.normalize else None
            gradient = gradient.resolve_conj().resolve_neg()
            rows = gradient.shape[indices.dim():]
            # a loss may leave a gradient that is expanded or permuted: rows are laid out
            if not _rows_fit(gradient, indices.dim()):
                gradient = gradient.contiguous()
            return (rt.embedding_gradient_device(gradient, indices, ctx.rows, scale=ctx.scale, table=table,
                                                 padding=ctx.padding).reshape((ctx.rows,) + tuple(rows)),
                    None, None, None, None)

    return Lookup


def _rows_fit(t, outer: int) -> bool:
    """Whether the gradient's rows have no gaps and lie one after the other (or are one row, expanded)."""
    width = 1
    for n, st in zip(reversed(t.shape[outer:]), reversed(t.stride()[outer:])):
        if n != 1 and st != width:
            return False
        width *= n
    outside = [(n, st) for n, st in zip(t.shape[:outer], t.stride()[:outer]) if n != 1]
    if all(st == 0 for _, st in outside):
        return True
    for n, st in reversed(outside):
        if st != width:
            return False
        width *= n
    return True


_lookup = None


def lookup(table, indices, scale: float = 1.0, normalize: bool = False, padding=None):
    """``scale * table[indices]`` (``runtime.embedding_lookup_device``), differentiable in `table`
    ([rows, ...], rows without gaps; float64, float32, bfloat16, float16 or complex). `indices`: int64 or int32
    CUDA tensor. With `normalize` each row is divided by its 2-norm first, and the gradient goes through the
    norm. Places whose index is `padding` are zero and get no gradient; an index outside the table gives NaN.
    Gradients of gradients are not supported."""
    global _lookup
    if _lookup is None:
        _lookup = _function()
    return _lookup.apply(table, indices, float(scale), bool(normalize), padding)
