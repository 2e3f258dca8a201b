"""A batch of states picked from a table keeps the table's rows and their gradient apart from what a circuit
makes of the states, on a B200."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def circuit():
    from arcqml_b200 import Circuit
    c = Circuit(2)
    return c.append("ry", (0,), c.add_parameter(0.4)).append("cnot", (0, 1)).append("rx", (1,), c.add_parameter(1.1))


def table():
    g = torch.Generator().manual_seed(4)
    return (torch.randn((3, 4), generator=g, dtype=torch.complex128) + 1.0).cuda()


INDEX = [2, 0, 2, 2, 0]


def test_an_applied_circuit_leaves_the_rows(runtime):
    from arcqml_b200.simulator import BatchStateVectorSimulator
    t, index = table(), torch.tensor(INDEX).cuda()
    sim = BatchStateVectorSimulator.from_table(2, t, index)
    rows = sim.states.clone()
    own = BatchStateVectorSimulator.from_device_state(2, rows.clone())
    for _ in range(2):
        sim.apply_circuit(circuit())
        own.apply_circuit(circuit())
        assert torch.equal(sim.states, rows)
        assert torch.equal(sim.state, own.state) and not torch.equal(sim.state, rows)


def test_a_circuit_is_not_applied_behind_the_tables_gradient(runtime):
    """The gradient of evolved states is not that of the rows."""
    import numpy as np
    from arcqml_b200 import SparsePauliOp
    from arcqml_b200.simulator import BatchStateVectorSimulator, SimError
    h = SparsePauliOp(2)
    h.add_term(1.0, [(0, "Z")]).add_term(0.5, [(1, "X")])
    index, weight = torch.tensor(INDEX).cuda(), np.array([1.0, -0.5, 0.25, 2.0, 1.0])
    grads = []
    for applied in (False, True):
        t = table().requires_grad_(True)
        sim = BatchStateVectorSimulator.from_table(2, t, index)
        rows = sim.states.detach().clone()
        if applied:
            with pytest.raises(SimError, match="no_grad"):
                sim.apply_circuit(circuit())
            assert torch.equal(sim.states, rows) and torch.equal(sim.state, rows)
        _, initial = sim.run(circuit(), h).backward(weight)
        # the states in a loss of their own beside the circuit's
        torch.autograd.backward([sim.states, sim.states.abs().square()[:, 0].sum()], [initial, None])
        grads.append(t.grad)
    assert grads[0].abs().sum() > 0 and torch.equal(*grads)
    with torch.no_grad():
        sim = BatchStateVectorSimulator.from_table(2, t, index)
    sim.apply_circuit(circuit())
    assert torch.equal(sim.states, rows)
