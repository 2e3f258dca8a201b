"""bf16 matrices of few singular values orthogonalised, on a B200. The polynomial takes small singular values up by as
much as 3.4445 a step, 485 times in five, and with them what X's own roundings leave where there are none."""
import math

import pytest
import torch

import matrix_table_support as ms

pytestmark = pytest.mark.gpu


def rounded(t, bits):
    scale = torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=1e-300))) + 1 - bits)
    return torch.round(t / scale) * scale


def bound_of(u, steps=5):
    """As ms.polynomial_bound, with a model of what the calls are documented to do: X and (up to 128 rows or columns)
    everything in 22 bits, else products from operands of 11; the diagonals of A and P in 24. X starts as the matrix times
    a power of two. Four times what the model is off by, f32's rounding of X, and the type's of the result."""
    want = ms.polynomial64(u, steps)
    bits = 22 if min(u.shape) <= 128 else 11
    x = u.double().mT if u.shape[0] > u.shape[1] else u.double()
    first = 2.0 ** -(math.floor(math.log2(float(x.norm()))) + 1)
    ratio = first * (float(x.norm()) + 1e-7)
    x = rounded(x * first, 22)
    for _ in range(steps):
        h = rounded(x, bits)
        a = h @ h.mT
        d = a.diagonal().clone()
        a = rounded(a - torch.diag(d), bits)
        s = a @ a
        b, c = ms.B / ratio ** 2, ms.C / ratio ** 4
        p = b * a + c * (s + (d[:, None] + d) * a)
        e = b * d + c * (s.diagonal() + d * d)
        x = rounded(((ms.A + e)[:, None] * x + rounded(p - torch.diag(p.diagonal()), bits) @ h) / ratio, 22)
        ratio = 1.0
    x = x.mT if u.shape[0] > u.shape[1] else x
    far = float((x - want).norm())
    return want, 4 * far + (4 * ms.U32 + ms.half_step(u.dtype)) * float(want.norm())


def product(m, n, rank, seed, scale=1e-3):
    g = torch.Generator().manual_seed(seed)
    return ((torch.randn(m, rank, generator=g, dtype=torch.float64) @ torch.randn(
        rank, n, generator=g, dtype=torch.float64)) * scale).bfloat16()


@pytest.mark.parametrize("shape", [(300, 260), (700, 129), (1024, 1024), (130, 2000)])
@pytest.mark.parametrize("rank", [1, 3, 16, 64])
def test_low_rank(runtime, shape, rank):
    u = product(*shape, rank, rank)
    got, = runtime.orthogonalize_device([u.cuda()])
    want, bound = bound_of(u)
    # (says something: X in 11 bits came out 0.017 to 0.097 off. The model alone gives at most 4 x 0.00278 + 0.0039)
    assert bound < 0.016 * float(want.norm())
    ms.assert_near(got, want, bound, (shape, rank))


@pytest.mark.parametrize("shape", [(2, 2), (3, 3), (4, 4), (8, 8), (30, 30), (4, 300), (4, 1000), (100, 257), (128, 600)])
def test_few_rows(runtime, shape):
    """Sixty matrices of each shape, full and of rank 2: no singular value is evened out by many others."""
    u = [product(*shape, rank, 100 * i + rank) for i in range(30) for rank in (2, max(shape))]
    for i, (a, b) in enumerate(zip(runtime.orthogonalize_device([x.cuda() for x in u]), u)):
        want, bound = bound_of(b)
        assert bound < 0.006 * float(want.norm())
        ms.assert_near(a, want, bound, (shape, i))


def test_step_of_low_rank(runtime):
    """The same by way of the momentum, the parameter's update apart from its own rounding: parameters of zeros."""
    shapes = [(300, 260), (40, 40)]
    g = [product(*s, 4, i) for i, s in enumerate(shapes)]
    p = [torch.zeros(s, dtype=torch.bfloat16, device="cuda") for s in shapes]
    runtime.muon_step_device(p, [x.cuda() for x in g], runtime.DeviceMuonState(p), lr=1.0, momentum=0.0)
    for a, b in zip(p, g):
        want, bound = bound_of(b)
        rate = math.sqrt(max(1.0, b.shape[0] / b.shape[1]))
        ms.assert_near(a, -rate * want, rate * bound * 1.01, tuple(b.shape))


@pytest.mark.parametrize("eps", [1e-7, 1e-3, 1.0, 1e30])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(20, 30), (300, 260)])
def test_large_epsilons(runtime, eps, dtype, shape):
    """X starts far below 1 and stays what u / (|u| + eps) makes of it, down to a multiple a^5 of the matrix."""
    u = torch.randn(shape, generator=torch.Generator().manual_seed(7), dtype=torch.float64).mul(1e-2).to(dtype)
    got, = runtime.orthogonalize_device([u.cuda()], eps=eps)
    want = ms.polynomial64(u, eps=eps)
    most = 2e-3 + ms.half_step(dtype) if dtype == torch.bfloat16 else 1e-5
    assert float((got.cpu().double() - want).norm()) <= most * float(want.norm())
