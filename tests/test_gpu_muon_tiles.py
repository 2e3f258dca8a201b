"""Orthogonalisation of matrices that take several tiles, on a B200: single blocks and pairs, tiles cut along
their depth, edges inside tiles, lists of mixed depths; against 64 bits as in test_gpu_muon.py."""
import pytest
import torch

import matrix_table_support as ms

pytestmark = pytest.mark.gpu


def make(shape, dtype, seed, scale=1e-3):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * scale).to(dtype)


def check(runtime, matrices, steps=5):
    got = runtime.orthogonalize_device([u.cuda() for u in matrices], steps=steps)
    again = runtime.orthogonalize_device([u.cuda() for u in matrices], steps=steps)
    for a, b, u in zip(got, again, matrices):
        assert torch.equal(a, b)  # parts of tiles are added in one order
        ms.assert_near(a, *ms.polynomial_bound(u, steps), tuple(u.shape))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(129, 4000), (8191, 140), (256, 8192), (512, 6000), (513, 2047), (1290, 1300),
                                   (129, 513), (256, 512), (257, 513)])
def test_one_matrix(runtime, dtype, shape):
    check(runtime, [make(shape, dtype, sum(shape))])


@pytest.mark.parametrize("n", [513, 527, 528, 575, 576, 577, 640, 1023, 1024, 1025])
def test_columns_around_blocks(runtime, n):
    check(runtime, [make((130, n), torch.float16, n), make((n, 200), torch.bfloat16, n)], steps=3)


def test_mixed_depths(runtime):
    shapes = [(300, 5000), (1024, 1024), (1000, 260), (1024, 1024), (140, 900), (700, 2100), (64, 30), (2, 3000)]
    check(runtime, [make(s, torch.float32, i) for i, s in enumerate(shapes)])
    check(runtime, [make(s, (torch.bfloat16, torch.float16)[i % 2], i) for i, s in enumerate(shapes)])


def test_many_in_several_launches(runtime):
    """More matrices than a launch takes, in two precisions."""
    u = [make((130 + i % 7, 131 + i % 11), (torch.float32, torch.bfloat16)[i % 2], i) for i in range(150)]
    got = runtime.orthogonalize_device([x.cuda() for x in u], steps=2)
    for i in range(0, 150, 13):
        ms.assert_near(got[i], *ms.polynomial_bound(u[i], 2), i)
    for x, y in zip(u, got):
        one, = runtime.orthogonalize_device([x.cuda()], steps=2)
        assert float((one.float() - y.float()).norm()) <= 2 * ms.half_step(x.dtype) * float(y.float().norm()) + (
            1e-5 if x.dtype == torch.float32 else 2e-3) * float(y.float().norm())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_small_matrices_of_every_edge(runtime, dtype):
    sizes = (1, 2, 7, 8, 15, 16, 17, 31, 33, 63, 64, 65, 112, 127, 128)
    widths = sizes + (129, 255, 256) + ((257, 511, 512) if dtype == torch.bfloat16 else ())
    u = [make((m, n) if (m + n) % 2 else (n, m), dtype, m * 1000 + n) for m in sizes for n in widths if m <= n]
    got = runtime.orthogonalize_device([x.cuda() for x in u])
    for a, b in zip(got, u):
        ms.assert_near(a, *ms.polynomial_bound(b), tuple(b.shape))


@pytest.mark.parametrize("shape", [(300, 420), (90, 100), (700, 260)])
@pytest.mark.parametrize("norm", [1e-30, 1e-12, 3e-8, 1e-7, 5e-7, 1.0, 1e30])
def test_norms_around_epsilon(runtime, shape, norm):
    """X is u / (|u| + 1e-7) also where epsilon is most of that, or nearly all."""
    u = make(shape, torch.float64, 3)
    u = (u / u.norm() * norm).float()
    check(runtime, [u])
    out, = runtime.orthogonalize_device([u.cuda()], eps=0.0)
    want = ms.polynomial64(u, eps=0.0)
    assert float((out.cpu().double() - want).norm()) <= 1e-5 * float(want.norm())


def test_singular_values(runtime):
    """What the operator is for: singular values from 1 down to 0.01 of the largest end up between 0.6 and
    1.25 (the polynomial's range over five steps), in the same singular directions."""
    g = torch.Generator().manual_seed(1)
    q, _ = torch.linalg.qr(torch.randn(200, 200, generator=g, dtype=torch.float64))
    r, _ = torch.linalg.qr(torch.randn(340, 200, generator=g, dtype=torch.float64))
    s = torch.logspace(0, -2, 200, dtype=torch.float64)
    u = (q * s) @ r.mT
    x = runtime.orthogonalize_device([u.float().cuda()])[0].cpu().double()
    core = q.mT @ x @ r
    assert float((core - torch.diag(core.diagonal())).norm()) < 1e-4 * float(core.norm())
    assert 0.6 < float(core.diagonal().min()) and float(core.diagonal().max()) < 1.25


def test_a_step_over_large_matrices(runtime):
    """The fused last phase on both orientations and types, against orthogonalising and stepping apart."""
    shapes = [(600, 1100), (1100, 600), (513, 515)]
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        p = [make(s, dtype, i, 0.05).cuda() for i, s in enumerate(shapes)]
        g = [make(s, torch.float32, 9 + i).cuda() for i, s in enumerate(shapes)]
        before = [x.clone() for x in p]
        runtime.muon_step_device(p, g, runtime.DeviceMuonState(p), lr=0.1, momentum=0.0, nesterov=False, weight_decay=0.5)
        x = runtime.orthogonalize_device([y.to(dtype) if dtype != torch.bfloat16 else y for y in g])
        for a, b, c in zip(p, before, x):
            want = b.double() * 0.95 - 0.1 * max(1.0, b.shape[0] / b.shape[1]) ** 0.5 * c.double()
            scale = float(want.norm())
            # the 11-bit operands of bf16 parameters, and their own rounding; f16's gradient was rounded first
            most = {torch.float32: 1e-6, torch.bfloat16: 3e-3, torch.float16: 1e-3}[dtype]
            assert float((a.double() - want).norm()) <= most * scale, (dtype, tuple(b.shape))
