"""Rows and columns orthogonalised, on a B200. A = X X^T is one number there, so the result is the update times a
number: off by the result's rounding alone."""
import math

import pytest
import torch

import matrix_table_support as ms

pytestmark = pytest.mark.gpu

LENGTHS = [1, 2, 7, 8, 9, 80, 255, 257, 1000, 8191, 100_003]


def make(shape, dtype, seed, scale=1e-3):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * scale).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("steps, eps", [(1, 1e-7), (5, 1e-7), (7, 1e-3), (5, 0.0)])
def test_rows_and_columns(runtime, dtype, steps, eps):
    """Half a step of the type (a rounding to f32 before it, for the 16-bit types: by 2^-13 of theirs or less), and
    what f64 makes of a number that each step may move by three times its error: below 3^7 2^-53 (n / 2 + 8)."""
    shapes = [(1, n) for n in LENGTHS] + [(n, 1) for n in LENGTHS]
    for scale in (1e-3, 1e-8, 30.0):
        u = [make(s, dtype, i, scale) for i, s in enumerate(shapes)]
        got = runtime.orthogonalize_device([x.cuda() for x in u], steps=steps, eps=eps)
        tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134
        for x, y in zip(u, got):
            want = ms.polynomial64(x, steps, eps) if x.any() or eps else x.double()
            rel = ms.half_step(dtype) * (1 + 2.0 ** -12) + 3.0 ** 7 * 2.0 ** -53 * (x.numel() / 2 + 8)
            assert ((y.cpu().double() - want).abs() <= rel * want.abs() + tiny).all(), (tuple(x.shape), scale)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("gradient", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nesterov", [True, False])
def test_steps_of_rows(runtime, dtype, gradient, nesterov):
    """u is formed in f32: off by 4 u32 of the magnitudes that enter it, here all of one row's scale, so the result by
    some 8 u32 of the largest of them (each of the five steps passes an error of the norm on, times three at most,
    and that error is the entries' averaged). Then two f32 roundings and the type's."""
    shapes = [(1, 80), (300, 1), (1, 1), (1, 5000)]
    p = [make(s, dtype, i, 0.1).cuda() for i, s in enumerate(shapes)]
    g = [make(s, gradient, 10 + i).cuda() for i, s in enumerate(shapes)]
    m = [make(s, torch.float32, 20 + i, 5e-4).cuda() for i, s in enumerate(shapes)]
    state = runtime.DeviceMuonState(p, momentum=[x.clone() for x in m])
    before = [x.cpu().double() for x in p]
    runtime.muon_step_device(p, g, state, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=0.1)
    for x, old, y, z, moved in zip(p, before, g, m, state.momentum):
        y, z = y.cpu().double(), z.cpu().double()
        m2 = 0.9 * z + 0.1 * y
        assert ((moved.cpu().double() - m2).abs() <= 6 * ms.U32 * (z.abs() + y.abs())).all()
        u = 0.9 * m2 + 0.1 * y if nesterov else m2
        rate = 0.02 * math.sqrt(max(1.0, x.shape[0] / x.shape[1]))
        result = ms.polynomial64(u)
        want = 0.998 * old - rate * result
        size = float((z.abs() + y.abs()).norm() / u.norm())
        bound = (ms.half_step(x.dtype) + 2 * ms.U32) * (want.abs() + rate * result.abs()) + \
            rate * 8 * ms.U32 * size * (1 + 3.0 ** 5 / math.sqrt(x.numel())) * float(result.abs().max()) + 2.0 ** -25
        assert ((x.cpu().double() - want).abs() <= 1.5 * bound).all(), tuple(x.shape)


def test_values_and_places(runtime):
    """In place, unaligned, NaN and infinities, beside other matrices and without scratch."""
    flat = make((20_000,), torch.float32, 1).cuda()
    row, column = flat[1:5002].view(1, 5001), flat[7001:7801].view(800, 1)
    want = [x.clone() for x in runtime.orthogonalize_device([row.clone(), column.clone()])]
    before = flat.clone()
    got = runtime.orthogonalize_device([row, column], out=[row, column])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(flat[:1], before[:1]) and torch.equal(flat[5002:7001], before[5002:7001])
    assert torch.equal(flat[7801:], before[7801:])
    for bad in (math.nan, math.inf):
        x, y = make((1, 3000), torch.float32, 2).cuda(), make((300, 200), torch.float32, 3).cuda()
        alone, = runtime.orthogonalize_device([y])
        x[0, 7] = bad
        a, b = runtime.orthogonalize_device([x, y])
        assert torch.isnan(a).all() and torch.equal(b, alone)
    rows = runtime.TensorList([make((1, 100_000), torch.float32, 4).cuda()])
    runtime.orthogonalize_device(rows)
    assert rows._matrix_words == 0
