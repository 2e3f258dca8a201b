"""Lookups, their gradient and orthogonalised updates in 64 bits, with what a computation in a type's own
precision may be off by. u is half a step of a type (torch.finfo(t).eps / 2)."""
import math

import torch

A, B, C = 3.4445, -4.7750, 2.0315
U32 = 2.0 ** -24


def half_step(dtype):
    real = {torch.complex128: torch.float64, torch.complex64: torch.float32}.get(dtype, dtype)
    return torch.finfo(real).eps / 2


def parts(t):
    """[rows, width] of the components in 64 bits."""
    t = torch.view_as_real(t.resolve_conj()) if t.is_complex() else t
    return t.reshape(t.shape[0], -1).to(torch.float64) if t.shape[0] else t.new_zeros((0, 1)).double()


def lookup64(table, index, scale, normalize, padding):
    t = parts(table)
    if normalize:
        norm = t.square().sum(1, keepdim=True).sqrt()
        t = torch.where(norm > 0, t / norm, t)
    inside = (index >= 0) & (index < len(t))
    out = t[index.clamp(0, max(0, len(t) - 1))] * scale
    out[~inside] = math.nan
    if padding is not None:
        out[index == padding] = 0.0
    return out


def lookup_bound(want, table, normalize):
    """The factor is f64 (a root, a division; a sum of squares whose relative error is at most width u64) and the
    product is rounded once; without a norm the scale is rounded to f32 for the types below f64."""
    u = half_step(table.dtype)
    width = parts(table[:1]).shape[1]
    rel = u + (2.0 ** -53 * (width / 2 + 6) if normalize else 2.0 ** -53 if u == 2.0 ** -53 else 2 * U32)
    tiny = {2.0 ** -11: 2.0 ** -24}.get(u, 2.0 ** -133 if u == 2.0 ** -8 else 0.0)
    return 1.5 * rel * want.abs() + tiny


def gradient64(g, index, rows, scale, table, padding):
    """(gradient, bound). The k places of a row enter a chain of k additions in the wide type, each off by its
    u of a running sum that is below the sum of magnitudes; the scale, its product and the rounding add three.
    Through a norm: s' = (s - t <t, s> / <t, t>) / |t|, products in f64, so the sum's error goes through a
    projection (never longer than it) and each component moves by at most the row's whole error."""
    x = parts(g)
    keep = (index >= 0) & (index < rows)
    if padding is not None:
        keep &= index != padding
    s = x.new_zeros((rows, x.shape[1])).index_add_(0, index[keep], x[keep]) * scale
    size = x.new_zeros((rows, x.shape[1])).index_add_(0, index[keep], x[keep].abs()) * abs(scale)
    count = torch.zeros(rows, dtype=torch.float64).index_add_(
        0, index[keep], torch.ones(int(keep.sum()), dtype=torch.float64))[:, None]
    u = half_step(g.dtype)
    wide = 2.0 ** -53 if u == 2.0 ** -53 else U32
    tiny = {2.0 ** -11: 2.0 ** -24}.get(u, 2.0 ** -133 if u == 2.0 ** -8 else 0.0)
    bound = (count + 3) * wide * size
    if table is not None:
        t = parts(table)
        tt = t.square().sum(1, keepdim=True)
        norm = tt.sqrt()
        along = (t * s).sum(1, keepdim=True) / tt
        row = bound.square().sum(1, keepdim=True).sqrt() + 2.0 ** -53 * (t.shape[1] + 8) * s.square().sum(
            1, keepdim=True).sqrt()
        s, bound = (s - t * along) / norm, row / norm
        s[tt[:, 0] == 0], bound[tt[:, 0] == 0] = 0.0, 0.0
    bound[count[:, 0] == 0] = 0.0
    return s, 1.5 * (bound + u * s.abs()) + tiny * (count > 0)


# ------------------------------------------------------------------ orthogonalisation


def polynomial64(u, steps=5, eps=1e-7, rounded=None, seed=0):
    """The definition in 64 bits; with `rounded` = (bits of the products' operands) a model of a computation
    that rounds X, A and P to that many bits, the diagonals of A and P to 24, and sums products in f32 with an
    error of one f32 step per 16 terms of a chain (of a running sum that grows evenly: half of it on average, in
    one direction)."""
    gen = torch.Generator().manual_seed(seed)
    u = u.to(torch.float64)
    flip = u.shape[0] > u.shape[1]
    x = u.mT if flip else u

    def operand(t):
        if rounded is None:
            return t
        scale = torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=1e-300))) + 1 - rounded)
        return torch.round(t / scale) * scale

    def product(l, r):
        p = l @ r
        if rounded is None:
            return p
        steps_ = l.shape[1] / 16 + 2
        noise = torch.randn(p.shape, generator=gen, dtype=torch.float64)
        return p * (1.0 - 2.0 ** -23 * steps_ / 2) + 2.0 ** -24 * math.sqrt(steps_) * noise * p.abs()

    x = operand(x / (x.square().sum().sqrt() + eps))
    for _ in range(steps):
        if rounded is None:
            a = x @ x.mT
            x = A * x + (B * a + C * (a @ a)) @ x
            continue
        a = product(x, x.mT)
        d = a.diagonal().clone()
        a = operand(a - torch.diag(d))
        s = product(a, a)
        p = B * a + C * (s + (d[:, None] + d) * a)
        e = B * d + C * (s.diagonal() + d * d)
        p = operand(p - torch.diag(p.diagonal()))
        x = operand((A + e)[:, None] * x + product(p, x))
    return x.mT if flip else x


def operand_bits(dtype):
    return 11 if dtype == torch.bfloat16 else 22


def polynomial_bound(u, steps=5, out=None):
    """(result in 64 bits, Frobenius distance that a computation with the type's operands may have from it):
    four times the largest of what three models of its roundings have, f32's own rounding of X and the norm
    (4 u32 |X|), and the rounding to the type."""
    u = u.detach().cpu()
    want = polynomial64(u, steps)
    models = [polynomial64(u, steps, rounded=operand_bits(out or u.dtype), seed=s) for s in range(3)]
    far = max(float((m - want).norm()) for m in models)
    return want, 4 * far + (4 * U32 + half_step(out or u.dtype)) * float(want.norm()) + 1e-30


def assert_near(got, want, bound, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), what
    off = float((got.detach().cpu().double() - want).norm())
    assert off <= bound, (what, off, bound)
