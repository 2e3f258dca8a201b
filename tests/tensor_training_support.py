"""The gradient norm, clipping and the Adam step over lists of tensors, in 64 bits, with bounds on
what a computation in a type's own precision may be off by.

u is half a step of a type, relative (torch.finfo(t).eps / 2): f64 2^-53, f32 2^-24, f16 2^-11,
bf16 2^-8. Bounds are first order in u, counted operation by operation, and then widened by half for
the products of roundings and the 64-bit side's own error."""
import math

import numpy as np
import torch

U64, U32 = 2.0 ** -53, 2.0 ** -24
TINY = {torch.float64: 2.0 ** -1074, torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133,
        torch.float16: 2.0 ** -24}  # the smallest positive value: an absolute step near zero


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def components(t):
    """The components of a tensor in the order of its memory, as float64 on the host."""
    if t.is_complex():
        t = torch.view_as_real(t)
    if not t.is_contiguous():  # a permutation of a contiguous tensor: put the memory's order back
        order = sorted(range(t.dim()), key=lambda d: (-t.stride(d), -t.shape[d]))
        t = t.permute(order)
    return t.detach().to(torch.float64).reshape(-1).cpu().numpy()


def real_type(t):
    return {torch.complex128: torch.float64, torch.complex64: torch.float32}.get(t.dtype, t.dtype)


def norm64(tensors):
    """Every square is rounded once (u) and fsum adds exactly."""
    parts = [components(t) for t in tensors if t is not None]
    return math.sqrt(math.fsum(float(x) for p in parts for x in p * p))


def norm_bound(count):
    """Relative: each of `count` squares enters a chain of at most count + 40 fused operations (the
    blocks' sums included), each off by u; the root halves that and adds one rounding."""
    return 1.5 * ((count + 40) / 2 + 2) * U64


def clip_factor(norm, max_norm):
    f = max_norm / (norm + 1e-6)
    return 1.0 if f > 1.0 else f


def clip64(t, factor, count):
    """(clipped values, bound). f64: the factor's error (the norm's, an addition, a division) and one
    product. Other types: the factor rounded to f32, the product in f32, one rounding to the type."""
    x, kind = components(t), real_type(t)
    y = x * factor
    rel = norm_bound(count) + 3 * U64
    if kind == torch.float64:
        rel += U64
    else:
        rel += 2 * U32 + (half_step(kind) if kind != torch.float32 else 0.0)
    return y, 1.5 * rel * np.abs(y) + 2 * TINY[kind]


def adam64(p, g, m, v, t, lr, b1, b2, eps, wd, decoupled, factor, u, factor_rel):
    """One step on float64 arrays: (p, m, v) and their bounds for a computation whose operations and
    constants are off by u each; factor_rel: the relative error of the clip factor."""
    a = factor * g
    a_err = (factor_rel + 2 * u) * np.abs(a)
    a_abs = np.abs(a)
    if not decoupled:
        a_abs = a_abs + np.abs(wd * p)
        a = a + wd * p
        a_err = a_err + 3 * u * a_abs  # decay's rounding, its product, the sum
    m2 = b1 * m + (1 - b1) * a
    m_err = 2 * u * np.abs(b1 * m) + (1 - b1) * (a_err + 2 * u * np.abs(a)) + u * (
        np.abs(b1 * m) + (1 - b1) * np.abs(a))
    v2 = b2 * v + (1 - b2) * a * a
    v_err = 2 * u * b2 * v + (1 - b2) * (2 * a_err * np.abs(a) + a_err * a_err + 3 * u * a * a) + u * v2
    bc1, bc2 = 1.0 - b1 ** t, 1.0 - b2 ** t
    bc_err = 4 * U64  # the power within two steps and the difference, absolute (powers are below 1)
    root = np.sqrt(v2 / bc2)
    with np.errstate(divide="ignore", invalid="ignore"):
        root_err = np.where(root > 0, 0.5 * (v_err / bc2) / np.maximum(root, 1e-300), 0.0)
    # near zero the root of the error bounds the error of the root
    root_err = np.minimum(root_err, np.sqrt(v_err / bc2)) + (bc_err / bc2 + 4 * u) * root
    den = root + eps
    den_err = root_err + 2 * u * den
    step = lr * (m2 / bc1) / den
    step_err = lr / bc1 * (m_err / den + np.abs(m2) * den_err / (den * den)) + (
        bc_err / bc1 + 5 * u) * np.abs(step)
    x = p * (1 - lr * wd) if decoupled else p
    p2 = x - step
    p_err = step_err + 3 * u * np.abs(x) + u * (np.abs(x) + np.abs(step))
    return p2, m2, v2, 1.5 * p_err, 1.5 * m_err, 1.5 * v_err


def assert_within(got, want, bound, what):
    off = np.abs(got - want)
    bad = ~(off <= bound)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], want[bad][:4], bound[bad][:4])
