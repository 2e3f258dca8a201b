"""Matrices orthogonalised by Newton-Schulz products and the momentum step with them, on a B200: against 64
bits, within what a 64-bit model of the products' roundings is off by."""
import math

import pytest
import torch

import matrix_table_support as ms

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(1, 1), (1, 7), (9, 1), (3, 5), (16, 16), (64, 48), (80, 64), (10, 300), (127, 129), (128, 128), (129, 127),
          (200, 100), (256, 256), (257, 300), (64, 1000), (700, 130), (384, 520)]


def make(shape, dtype, seed, scale=1e-3):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * scale).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize(runtime, dtype, shape):
    u = make(shape, dtype, sum(shape))
    got, = runtime.orthogonalize_device([u.cuda()])
    assert got.dtype == dtype
    ms.assert_near(got, *ms.polynomial_bound(u), shape)


@pytest.mark.parametrize("steps", [1, 2, 7])
def test_steps(runtime, steps):
    u = [make(s, torch.float32, 3) for s in ((5, 70), (150, 140), (300, 520))]
    for a, b in zip(runtime.orthogonalize_device([x.cuda() for x in u], steps=steps), u):
        ms.assert_near(a, *ms.polynomial_bound(b, steps), (steps, b.shape))


def test_a_list_of_all_kinds(runtime):
    """Many matrices of different shapes and types in one call, empty places and empty matrices among them."""
    u = []
    for i in range(70):
        shape = SHAPES[i % len(SHAPES)] if i % 9 else (i, 0)
        u.append(None if i % 11 == 5 else make(shape, TYPES[i % 3], i))
    got = runtime.orthogonalize_device([None if x is None else x.cuda() for x in u])
    for i, (a, b) in enumerate(zip(got, u)):
        assert (a is None) == (b is None)
        if b is not None and b.numel():
            ms.assert_near(a, *ms.polynomial_bound(b), i)
        elif b is not None:
            assert a.shape == b.shape
    assert runtime.orthogonalize_device([]) == []


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1024, 1000), (600, 2100)])
def test_larger(runtime, dtype, shape):
    u = make(shape, dtype, 5)
    got, = runtime.orthogonalize_device([u.cuda()])
    ms.assert_near(got, *ms.polynomial_bound(u), shape)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(40, 60), (300, 260)])
def test_values(runtime, dtype, shape):
    """Rank one, equal rows, huge and tiny entries, zeros; a NaN or infinity stays in its own matrix."""
    base = make(shape, torch.float64, 1)
    cases = [base[:1].expand(shape).contiguous(), base[:, :1] * base[:1] * 1e6, base * 1e30, base * 1e-30 + 0.0,
             torch.zeros(shape, dtype=torch.float64), torch.eye(*shape, dtype=torch.float64)]
    u = [c.to(dtype) for c in cases]
    bad = [base.to(dtype), base.to(dtype)]
    bad[0][1, 2], bad[1][3, 4] = math.nan, math.inf
    got = runtime.orthogonalize_device([x.cuda() for x in u + bad])
    for i, (a, b) in enumerate(zip(got, u)):
        ms.assert_near(a, *ms.polynomial_bound(b), i)
    assert not got[4].any()
    assert torch.isnan(got[-2]).all() and torch.isnan(got[-1]).all()


def test_output_in_place(runtime):
    u = [make(s, torch.float32, 2).cuda() for s in ((30, 40), (200, 190))]
    want = runtime.orthogonalize_device(u)
    out = [torch.empty_like(x) for x in u]
    got = runtime.orthogonalize_device(u, out=out)
    assert all(a is b for a, b in zip(got, out)) and all(torch.equal(a, b) for a, b in zip(out, want))
    before = u[0]._version
    runtime.orthogonalize_device(u, out=u)
    assert all(torch.equal(a, b) for a, b in zip(u, want)) and u[0]._version > before


def test_unaligned_and_views(runtime):
    flat = make((60_000,), torch.bfloat16, 3).cuda()
    u = [flat[1:1 + 33 * 65].view(33, 65), flat[7:7 + 200 * 133].view(200, 133), flat[3:4].view(1, 1)]
    got = runtime.orthogonalize_device(u)
    want = runtime.orthogonalize_device([x.clone() for x in u])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(runtime):
    ok = make((8, 6), torch.float32, 1).cuda()
    for bad in (ok.double(), ok.to(torch.complex64), ok[0], ok.t(), ok.view(2, 4, 6)):
        with pytest.raises(TypeError, match="row-major"):
            runtime.orthogonalize_device([ok, bad])
    for bad in (ok[:, :3], ok.cpu(), 3):
        with pytest.raises(TypeError):
            runtime.orthogonalize_device([bad])
    for steps in (0, 21):
        with pytest.raises(runtime.RuntimeError, match="steps"):
            runtime.orthogonalize_device([ok], steps=steps)
    for eps in (-1.0, math.nan):
        with pytest.raises(runtime.RuntimeError, match="epsilon"):
            runtime.orthogonalize_device([ok], eps=eps)
    with pytest.raises(ValueError):
        runtime.orthogonalize_device([ok], out=[ok.t().contiguous()])
    with pytest.raises(runtime.RuntimeError, match="type"):
        runtime.orthogonalize_device([ok], out=[ok.bfloat16()])
    both = make((2, 8, 6), torch.float32, 1).cuda()
    with pytest.raises(runtime.RuntimeError, match="share"):
        runtime.orthogonalize_device([both[0], both[1]], out=[both[1], both[0]])
    with pytest.raises(runtime.RuntimeError, match="share memory"):
        runtime.orthogonalize_device([ok, ok], out=[both[0], both[0]])


# ------------------------------------------------------------------ the step


def step64(p, g, m, lr, beta, nesterov, wd, steps):
    """(parameter, momentum, their bounds): momentum in f32 (three roundings), the rest by the model."""
    p64, g64, m64 = (x.cpu().double() for x in (p, g, m))
    m2 = beta * m64 + (1 - beta) * g64
    m_bound = 1.5 * 4 * ms.U32 * ((beta * m64).abs() + ((1 - beta) * g64).abs())
    u = (beta * m2 + (1 - beta) * g64 if nesterov else m2)
    x, far = ms.polynomial_bound(u, steps, out=p.dtype)
    # u itself is off by a few f32 roundings, which the polynomial passes on by at most its first steps' growth
    far += 8 * ms.U32 * ms.A ** min(steps, 5) * float(u.norm()) / max(float(u.norm()), 1e-30)
    rate = lr * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
    want = (1 - lr * wd) * p64 - rate * x
    return want, m2, rate * far + (3 * ms.U32 + ms.half_step(p.dtype)) * float(
        (p64.norm() + rate * x.norm())), m_bound


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gradient", TYPES)
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step(runtime, dtype, gradient, nesterov):
    shapes = [(64, 16), (16, 64), (1, 80), (130, 200), (300, 257), (5, 1), (520, 90)]
    p = [make(s, dtype, i, 0.1).cuda() for i, s in enumerate(shapes)]
    g = [make(s, gradient, 10 + i).cuda() for i, s in enumerate(shapes)]
    m = [make(s, torch.float32, 20 + i, 5e-4).cuda() for i, s in enumerate(shapes)]
    want = [step64(a, b, c, 0.02, 0.9, nesterov, 0.1, 5) for a, b, c in zip(p, g, m)]
    state = runtime.DeviceMuonState(p, momentum=m)
    assert runtime.muon_step_device(p, g, state, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=0.1) is None
    for i, (a, c, (pw, mw, p_bound, m_bound)) in enumerate(zip(p, state.momentum, want)):
        ms.assert_near(a, pw, p_bound, (i, "parameter"))
        assert ((c.cpu().double() - mw).abs() <= m_bound).all(), (i, "momentum")


def test_missing_gradients_and_state(runtime):
    p = [make((20, 30), torch.float32, i, 0.1).cuda() for i in range(3)]
    keep = [x.clone() for x in p]
    state = runtime.DeviceMuonState(p)
    g = make((20, 30), torch.float32, 9).cuda()
    runtime.muon_step_device(p, [None, g, None], state)
    assert torch.equal(p[0], keep[0]) and torch.equal(p[2], keep[2]) and not torch.equal(p[1], keep[1])
    assert not state.momentum[0].any() and torch.allclose(state.momentum[1], 0.05 * g, rtol=1e-6)
    with pytest.raises(TypeError):
        state.momentum[0] = g
    saved = [x.clone() for x in state.momentum]
    runtime.muon_step_device(p, [g, g, g], state)
    again = [x.clone() for x in p]
    for x, y in zip(p, keep):
        x.copy_(y)
    runtime.muon_step_device(p, [None, g, None], runtime.DeviceMuonState(p))
    state.momentum = saved
    runtime.muon_step_device(p, [g, g, g], state)
    assert all(torch.equal(a, b) for a, b in zip(p, again))
    # a gradient of zeros: decay alone
    z = [torch.zeros_like(x) for x in p]
    before = [x.clone() for x in p]
    runtime.muon_step_device(p, z, runtime.DeviceMuonState(p), lr=0.5, weight_decay=0.5)
    assert all(torch.equal(a, b * 0.75) for a, b in zip(p, before))


def test_step_refusals(runtime):
    p = [make((8, 6), torch.float32, 1).cuda()]
    g = [make((8, 6), torch.float32, 2).cuda()]
    state = runtime.DeviceMuonState(p)
    for bad in ({"lr": math.nan}, {"momentum": 1.0}, {"momentum": -0.1}, {"weight_decay": math.inf}, {"steps": 0}):
        with pytest.raises(runtime.RuntimeError):
            runtime.muon_step_device(p, g, state, **bad)
    with pytest.raises(ValueError):
        runtime.muon_step_device(p, [g[0][:4]], state)
    with pytest.raises(TypeError, match="row-major"):
        runtime.muon_step_device(p, [g[0].double()], state)
    for shared in (p, list(state.momentum)):
        with pytest.raises(runtime.RuntimeError, match="shares memory"):
            runtime.muon_step_device(p, shared, state)
    with pytest.raises(runtime.RuntimeError, match="share memory"):
        runtime.muon_step_device(p, g, runtime.DeviceMuonState(p, momentum=p))
    with pytest.raises(ValueError):
        runtime.DeviceMuonState(p, momentum=[p[0][:4]])
    with pytest.raises(TypeError):
        runtime.DeviceMuonState(p, momentum=[p[0].bfloat16()])
    with pytest.raises(TypeError):
        runtime.DeviceMuonState([make((8,), torch.float32, 1).cuda()])
    from arcqml_b200.optim import Muon
    with pytest.raises(ValueError, match="nothing"):
        Muon([])
    with pytest.raises(runtime.RuntimeError, match="share memory"):
        Muon([p[0], p[0]])
    with pytest.raises(ValueError, match="computed from others"):
        Muon([p[0].clone().requires_grad_(True) * 2])


def test_captured_on_two_streams(runtime):
    """Two captured steps over lists of their own, replayed at once on two streams, against eager ones."""
    shapes = [(64, 48), (200, 300), (129, 140), (700, 256)]
    runs = []
    for k in range(2):
        p = [make(s, torch.float32, 7 * k + i, 0.1).cuda() for i, s in enumerate(shapes)]
        g = [make(s, torch.float32, 50 + 7 * k + i).cuda() for i, s in enumerate(shapes)]
        twin = [x.clone() for x in p]
        state, twin_state = runtime.DeviceMuonState(p), runtime.DeviceMuonState(twin)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            runtime.muon_step_device(p, g, state)
        runs.append((graph, p, g, twin, twin_state, state))
    streams = [torch.cuda.Stream() for _ in runs]
    for _ in range(4):
        for (graph, *_), s in zip(runs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, p, g, twin, twin_state, _ in runs:
        for _ in range(4):
            runtime.muon_step_device(twin, g, twin_state)
        assert all(torch.equal(a, b) for a, b in zip(p, twin))


def test_given_stream_and_threads(runtime):
    import threading
    u = [make(s, torch.float32, i).cuda() for i, s in enumerate(((70, 60), (256, 400), (500, 200)))]
    want = runtime.orthogonalize_device(u)
    torch.cuda.synchronize()
    failed = []

    def work():
        s = torch.cuda.Stream()
        for _ in range(5):
            got = runtime.orthogonalize_device(u, stream=s.cuda_stream)
            s.synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want)):
                failed.append(1)

    threads = [threading.Thread(target=work) for _ in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed


def test_a_hybrid_models_step(runtime):
    """Tokens -> embeddings -> a linear map -> normalised states -> a circuit; Muon on the map, Adam on the
    table and the circuit. The step on the map against 64 bits from the same gradients."""
    import numpy as np
    from arcqml_b200 import Circuit, SparsePauliOp
    from arcqml_b200.embedding import lookup
    from arcqml_b200.optim import Adam, Muon
    from arcqml_b200.simulator import BatchStateVectorSimulator
    n, batch = 3, 12
    table = make((20, 8), torch.float32, 1, 1.0).cuda().requires_grad_(True)
    w = make((8, 2 << n), torch.float32, 2, 0.3).cuda().requires_grad_(True)
    c = Circuit(n)
    for q in range(n):
        c.append("ry", (q,), c.add_parameter(0.3 + q))
    c.append("cnot", (0, 1)).append("cnot", (1, 2))
    h = SparsePauliOp(n)
    h.add_term(1.0, [(0, "Z")]).add_term(0.5, [(1, "X"), (2, "Z")])
    tokens = torch.randint(0, 20, (batch,), generator=torch.Generator().manual_seed(3)).cuda()
    muon, adam = Muon(w, lr=0.05), Adam([c], [table], lr=0.01, max_norm=1.0)
    for _ in range(3):
        muon.zero_grad()
        adam.zero_grad()
        x = lookup(table, tokens, scale=2.0, padding=0)
        z = torch.view_as_complex((x @ w).double().reshape(batch, 1 << n, 2)) + 0.1
        states = z / z.abs().square().sum(1, keepdim=True).sqrt()
        sim = BatchStateVectorSimulator.from_device_state(n, states.detach().contiguous(), requires_grad=True)
        r = sim.run(c, h)
        _, initial = r.backward(np.full(batch, 1.0 / batch))
        states.backward(initial)
        assert not table.grad[0].any() and table.grad.abs().sum() > 0
        before, moment = w.detach().clone(), muon.state.momentum[0].clone()
        want, m2, bound, m_bound = step64(before, w.grad, moment, 0.05, 0.95, True, 0.0, 5)
        old = table.detach().clone()
        muon.step()
        adam.step()
        ms.assert_near(w, want, bound, "map")
        assert ((muon.state.momentum[0].cpu().double() - m2).abs() <= m_bound).all()
        assert not torch.equal(old, table)
