"""Training a circuit together with the network that feeds it (needs a B200): gradients against
differences of the loss, and the steps against 64 bits."""
import numpy as np
import pytest
import torch

import tensor_training_support as ts
from arcqml_b200 import Circuit, SparsePauliOp

pytestmark = pytest.mark.gpu

N, ROWS = 3, 5


class Model:
    """A linear map of x to normalised amplitudes, a circuit, <Z0 + X1 Z2 / 2>, half-MSE."""

    def __init__(self, seed, weight_type=torch.float64):
        g = torch.Generator().manual_seed(seed)
        self.w = torch.randn(4, 2 << N, generator=g, dtype=torch.float64).to(weight_type).cuda()
        self.b = torch.randn(2 << N, generator=g, dtype=torch.float64).cuda()
        self.x = torch.randn(ROWS, 4, generator=g, dtype=torch.float64).cuda()
        self.w.requires_grad_(True)
        self.b.requires_grad_(True)
        rng = np.random.default_rng(seed)
        self.y = np.sign(rng.normal(size=ROWS))
        c = self.circuit = Circuit(N)
        for q in range(N):
            c.append("ry", (q,), c.add_parameter(float(rng.uniform(-3, 3)), "f32" if q == 1 else "f64"))
        c.append("cnot", (0, 1)).append("cnot", (1, 2))
        for q in range(N):
            theta = c.add_parameter(float(rng.uniform(-3, 3)), requires_grad=q != 2)
            c.append("rz", (q,), theta).append("ry", (q,), theta)
        self.h = SparsePauliOp(N)
        self.h.add_term(1.0, [(0, "Z")]).add_term(0.5, [(1, "X"), (2, "Z")])

    def states(self):
        z = (self.x.to(self.w.dtype) @ self.w).double() + self.b
        z = torch.view_as_complex(z.reshape(ROWS, 1 << N, 2))
        return z / z.abs().square().sum(dim=1, keepdim=True).sqrt()

    def _simulator(self, states, requires_grad):
        from arcqml_b200.simulator import BatchStateVectorSimulator
        return BatchStateVectorSimulator.from_device_state(N, states.detach().contiguous(),
                                                           requires_grad=requires_grad)

    def loss(self):
        with torch.no_grad():
            r = self._simulator(self.states(), False).run(self.circuit, self.h, grad=False)
        return float(np.mean(0.5 * (r.values - self.y) ** 2))

    def backward(self):
        states = self.states()
        r = self._simulator(states, True).run(self.circuit, self.h)
        _, state_grad = r.backward((r.values - self.y) / ROWS)
        states.backward(state_grad)


def test_gradients_against_differences(runtime):
    """Central differences of an f64 loss of order 1: h^2 / 6 of a third derivative of order 10,
    and 2^-53 / h of rounding; the f32 parameter's own rounding bounds what h it can move by."""
    m = Model(1)
    m.backward()
    h = 1e-5
    bound = 10 * h * h + 100 * ts.U64 / h
    for t in (m.w, m.b):
        flat, grad = t.detach().view(-1), t.grad.view(-1)
        for i in range(0, flat.numel(), 7):
            was = float(flat[i])
            flat[i] = was + h
            up = m.loss()
            flat[i] = was - h
            down = m.loss()
            flat[i] = was
            assert abs((up - down) / (2 * h) - float(grad[i])) <= bound
    for p in m.circuit.parameters:
        if not p.requires_grad:
            assert getattr(p, "grad", None) is None
            continue
        was, step = p.value, h if p.dtype == "f64" else 2.0 ** -10
        base = p.f64()
        p.value = base + step
        up, at_up = m.loss(), p.f64()
        p.value = base - step
        down, at_down = m.loss(), p.f64()
        p.value = was
        d = (up - down) / (at_up - at_down)
        # the f32 gradient is rounded; its points lie evenly to half a step of f32 (values below 4)
        rough = bound if p.dtype == "f64" else 10 * step * step + 4 * ts.U32 * (1 + 4 / step * 1e-3)
        assert abs(d - p.grad) <= rough, (p, d)


@pytest.mark.parametrize("decoupled", [False, True])
@pytest.mark.parametrize("weight_type", [torch.float64, torch.float32])
def test_steps_of_a_hybrid_model(runtime, weight_type, decoupled):
    from arcqml_b200.optim import Adam
    m = Model(2, weight_type)
    frozen = m.circuit.parameters[5].value
    opt = Adam([m.circuit], [m.w, m.b], lr=0.02, weight_decay=0.01, decoupled=decoupled,
               max_norm=0.05)
    f64 = [p for p in m.circuit.parameters if p.requires_grad and p.dtype == "f64"]
    f32 = [p for p in m.circuit.parameters if p.requires_grad and p.dtype == "f32"]
    for t in range(1, 5):
        opt.zero_grad()
        m.backward()
        parts = [(np.array([p.f64() for p in g]), np.array([p.grad for p in g])) for g in (f64, f32)]
        parts += [(ts.components(x), ts.components(x.grad)) for x in (m.w, m.b)]
        moments = [(ts.components(a), ts.components(b)) for a, b in zip(opt.state.m, opt.state.v)]
        norm = opt.step()
        count = sum(g.size for _, g in parts)
        want = float(np.sqrt(sum(float(np.sum(g * g)) for _, g in parts)))
        assert abs(float(norm) - want) <= 2 * ts.norm_bound(count) * want
        assert int(opt.state.step) == t
        got = [np.array([p.value for p in g]) for g in (f64, f32)]
        got += [ts.components(x) for x in (m.w, m.b)]
        kinds = [torch.float64, torch.float32, weight_type, torch.float64]
        for (p, g), (a, b), x, kind in zip(parts, moments, got, kinds):
            u = ts.U64 if kind == torch.float64 else ts.U32
            p2, _, _, bound, _, _ = ts.adam64(p, g, a, b, t, 0.02, 0.9, 0.999, 1e-8, 0.01, decoupled,
                                              ts.clip_factor(want, 0.05), u,
                                              2 * ts.norm_bound(count) + 3 * ts.U64)
            ts.assert_within(x, p2, bound, (t, kind))
    assert m.circuit.parameters[5].value == frozen
    assert all(p.value == float(np.float32(p.value)) for p in f32)


def test_parts_without_gradients_stay(runtime):
    from arcqml_b200.optim import Adam
    m = Model(3)
    opt = Adam([m.circuit], [m.w, m.b])
    m.backward()
    m.w.grad = None
    for p in m.circuit.parameters:
        p.grad = None
    values, w, b = m.circuit.parameter_values(), m.w.detach().clone(), m.b.detach().clone()
    assert opt.step() is None and int(opt.state.step) == 1
    assert np.array_equal(m.circuit.parameter_values(), values) and torch.equal(m.w.detach(), w)
    assert not torch.equal(m.b.detach(), b)
    m.circuit.parameters[0].grad = 1.0
    with pytest.raises(ValueError, match="trained parameters have no gradient"):
        opt.step()
    assert int(opt.state.step) == 1
    for bad, match in [(dict(), "nothing to train"),
                       (dict(circuits=[m.circuit, m.circuit]), "trained once"),
                       (dict(tensors=[None]), "must not be None")]:
        with pytest.raises((TypeError, ValueError), match=match):
            Adam(**bad)
    with pytest.raises(runtime.RuntimeError, match="share memory"):
        Adam(tensors=[m.b, m.b])
    # a circuit alone, and its steps against the host's update
    opt = Adam([m.circuit], lr=0.1)
    trained = [p for p in m.circuit.parameters if p.requires_grad and p.dtype == "f64"]
    host = runtime.AdamState(len(trained))
    x = np.array([p.value for p in trained])
    rng = np.random.default_rng(0)
    for t in range(1, 6):
        for p in m.circuit.parameters:
            p.grad = float(rng.normal())
        x = host.update(x, [p.grad for p in trained], lr=0.1)
        opt.step()
        # as test_adam_matches_the_hosts_update: |step| below 4 lr, |x| below 5
        assert np.max(np.abs(np.array([p.value for p in trained]) - x)) <= t * (
            0.1 * 4 * (2 * 4 * ts.U64 / 1e-3 + 8 * ts.U64) + 8 * ts.U64 * 5)


def test_complex_leaves_whose_gradients_are_conjugated(runtime):
    """The amplitudes that normalised states are made from, and leaves that enter by their conjugate:
    autograd conjugates the gradient by a bit alone where the strides allow it. Steps against 64 bits."""
    from arcqml_b200.optim import Adam
    g = torch.Generator(device="cuda").manual_seed(4)

    def normal(*shape):
        return torch.randn(*shape, dtype=torch.complex128, device="cuda", generator=g)

    x, z = normal(ROWS, 1 << N).requires_grad_(True), normal(4, 6).t().requires_grad_(True)
    target, other = normal(ROWS, 1 << N), normal(6, 4)
    c64 = normal(7).to(torch.complex64).requires_grad_(True)
    w, third = normal(4, 6).t().requires_grad_(True), normal(4, 6).t()
    opt = Adam(tensors=[x, z, c64, w], lr=0.02, weight_decay=0.01, max_norm=0.5)
    for t in range(1, 4):
        opt.zero_grad()
        states = x / x.abs().square().sum(dim=1, keepdim=True).sqrt()
        overlap = (target.conj() * states).sum(dim=1).abs().square().sum()
        (overlap + (z.conj() * other).real.sum() + c64.conj().real.sum()
         + (third.mH @ w.conj()).sum().abs()).backward()
        assert w.grad.is_conj() and w.grad.stride() == w.stride()
        old = [[ts.components(u.resolve_conj()) for u in (a, a.grad, m, v)]
               for a, m, v in zip(opt.tensors, opt.state.m, opt.state.v)]
        norm = opt.step()
        count = sum(o[0].size for o in old)
        want = float(np.sqrt(sum(float(np.sum(o[1] * o[1])) for o in old)))
        assert abs(float(norm) - want) <= 2 * ts.norm_bound(count) * want
        for a, m, v, o in zip(opt.tensors, opt.state.m, opt.state.v, old):
            u = ts.U64 if a.dtype == torch.complex128 else ts.U32
            p2, m2, v2, pe, me, ve = ts.adam64(*o, t, 0.02, 0.9, 0.999, 1e-8, 0.01, False,
                                               ts.clip_factor(want, 0.5), u,
                                               2 * ts.norm_bound(count) + 3 * ts.U64)
            tiny = ts.TINY[ts.real_type(a)]
            for got, value, bound in ((a, p2, pe), (m, m2, me), (v, v2, ve)):
                ts.assert_within(ts.components(got), value, bound + 4 * tiny, (t, a.dtype))
