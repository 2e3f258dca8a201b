"""What a training program does with the state and the lists of the tensor operators between its
steps (needs a B200)."""
import copy
import pickle

import pytest
import torch

pytestmark = pytest.mark.gpu


def normal(n, seed, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(n, generator=g, device="cuda", dtype=dtype)


def test_assigned_moments_are_the_ones_that_the_step_takes(runtime):
    """A run that goes on from saved moments and one that was never stopped are equal bit by bit."""
    p, q = [normal(300, 1), normal(80, 2, torch.float64)], [normal(300, 3), normal(80, 4, torch.float64)]
    state = runtime.DeviceAdamState(p)
    for _ in range(3):
        runtime.adam_step_device(p, q, state)
    saved = [[t.clone() for t in x] for x in (p, state.m, state.v)]
    runtime.adam_step_device(p, q, state)

    by_list = runtime.DeviceAdamState(saved[0])
    runtime.adam_step_device([t.clone() for t in saved[0]], q, by_list)  # used before, other moments
    by_list.m, by_list.v = [t.clone() for t in saved[1]], tuple(t.clone() for t in saved[2])
    by_list.step.fill_(3)
    p2 = [t.clone() for t in saved[0]]
    runtime.adam_step_device(p2, q, by_list)
    in_place = runtime.DeviceAdamState(saved[0])
    for mine, old in zip(in_place.m + in_place.v, saved[1] + saved[2]):
        mine.copy_(old)
    in_place.step.copy_(torch.tensor(3))
    p3 = [t.clone() for t in saved[0]]
    runtime.adam_step_device(p3, q, in_place)
    for other, params in ((by_list, p2), (in_place, p3)):
        assert int(other.step) == 4
        for a, b in zip(p + state.m + state.v, params + other.m + other.v):
            assert torch.equal(a, b)


def test_moments_cannot_be_replaced_unseen(runtime):
    p = [normal(30, 1), normal(40, 2)]
    state = runtime.DeviceAdamState(p)
    t = torch.zeros(30, device="cuda")
    for change in (lambda m: m.__setitem__(0, t), lambda m: m.append(t), lambda m: m.pop(),
                   lambda m: m.clear(), lambda m: m.__delitem__(0), lambda m: m.extend([t]),
                   lambda m: m.insert(0, t), lambda m: m.reverse()):
        for moments in (state.m, state.v):
            with pytest.raises(TypeError, match="assigned as a whole"):
                change(moments)
    with pytest.raises(TypeError, match="assigned as a whole"):
        state.m += [t]
    for bad in ([t], [t, t], [t, None], [t[:29], torch.zeros(40, device="cuda")]):
        with pytest.raises(ValueError, match="first moments"):
            state.m = bad
        with pytest.raises(ValueError, match="second moments"):
            state.v = bad
    # assigned moments are held against the parameters like any others
    q = [normal(30, 3), normal(40, 4)]
    state.m = [p[0], torch.zeros(40, device="cuda")]
    with pytest.raises(runtime.RuntimeError, match="share memory"):
        runtime.adam_step_device(p, q, state)
    state.m = [torch.zeros(n, device="cuda", dtype=torch.float64) for n in (30, 40)]
    with pytest.raises(runtime.RuntimeError, match="first moment"):
        runtime.adam_step_device(p, q, state)
    assert int(state.step) == 0
    state.m = [torch.zeros_like(x) for x in p]
    runtime.adam_step_device(p, q, state)
    assert int(state.step) == 1 and all(bool((m != 0).all()) for m in state.m)


def test_copies_of_moments_are_plain_lists(runtime):
    state = runtime.DeviceAdamState([normal(30, 1)])
    for other in (copy.copy(state.m), copy.deepcopy(state.m), pickle.loads(pickle.dumps(state.m))):
        assert type(other) is list and torch.equal(other[0], state.m[0])
        other[0] = None
    assert state.m[0] is not None


def test_an_optimizers_tensors_cannot_be_replaced_unseen(runtime):
    """A tensor put in another's place would have its gradient applied to the other one."""
    from arcqml_b200.optim import Adam
    a, b = (torch.zeros(3, device="cuda").requires_grad_(True) for _ in range(2))
    opt = Adam(tensors=[a])
    with pytest.raises(TypeError):
        opt.tensors[0] = b
    with pytest.raises(AttributeError):
        opt.tensors = [b]
    with pytest.raises(AttributeError):
        opt.tensors.append(b)
    assert len(opt.tensors) == 1 and opt.tensors[0] is a
    b.grad = torch.ones(3, device="cuda")
    opt.step()
    assert bool((a == 0).all()) and bool((b == 0).all())
    a.grad = torch.ones(3, device="cuda")
    opt.step()
    assert bool((a < 0).all()) and bool((b == 0).all())


def test_an_optimizer_of_one_tensor(runtime):
    from arcqml_b200.optim import Adam
    w = torch.ones(4, 3, device="cuda", requires_grad=True)
    opt = Adam(tensors=w, lr=0.5)
    (w * w).sum().backward()
    opt.step()
    # the first step moves each value by lr against its gradient's sign, to a rounding of 1 / (1 + eps)
    assert len(opt.tensors) == 1 and bool(((w - 0.5).abs() <= 1e-6).all())
    assert opt.state.m[0].shape == (4, 3)


def test_gradients_share_no_memory_with_what_the_step_writes(runtime):
    """One block would read what another writes. Gradients may share memory with one another."""
    n = 3000
    flat = normal(8 * n, 11)
    p, g, m, v = [flat[:n]], [flat[n:2 * n]], [flat[2 * n:3 * n]], [flat[3 * n:4 * n].abs_()]
    c = [torch.zeros(n, device="cuda", dtype=torch.bfloat16)]
    count = torch.zeros(2, dtype=torch.int64, device="cuda")
    state = runtime.DeviceAdamState(p, m=m, v=v, step=count[1])
    was = flat.clone()

    def refused(match, **kw):
        kw = {"grads": g, "norm": None, "copies": c, **kw}
        with pytest.raises(runtime.RuntimeError, match=match):
            runtime.adam_step_device(p, kw["grads"], state, copies=kw["copies"], norm=kw["norm"],
                                     max_norm=None if kw["norm"] is None else 1.0)
        assert torch.equal(flat, was) and count.tolist() == [0, 0]

    for at in (0, 1, n - 1, n + 1, 2 * n - 1, 3 * n - 1, 4 * n - 1):
        refused("a gradient shares memory", grads=[flat[at:at + n]])
    refused("a gradient shares memory", grads=c)  # one bucket for gradients and copies
    norm = flat[:2 * n].view(torch.float64)
    refused("the given norm shares memory", norm=norm[0])
    refused("the given norm shares memory", norm=flat[2 * n:4 * n].view(torch.float64)[-1])
    refused("copies and step count share memory", copies=[flat[n // 2:n].view(torch.bfloat16)])
    refused("a gradient shares memory", copies=[flat[3 * n // 2:2 * n].view(torch.bfloat16)])
    # right beside what is written, and twice the same gradient
    runtime.adam_step_device(p, g, state, copies=c, max_norm=1.0, norm=norm[n // 2])
    assert count.tolist() == [0, 1]
    two = runtime.DeviceAdamState([flat[:n], flat[4 * n:5 * n]])
    runtime.adam_step_device([flat[:n], flat[4 * n:5 * n]], [g[0], g[0]], two)
    assert torch.equal(two.m[0], two.m[1])
    # a list that was taken once is looked at again when the state is another one
    kept = runtime.TensorList(g)
    runtime.adam_step_device(p, kept, state)
    state.m = [flat[n + 1:2 * n + 1]]
    was = flat.clone()
    with pytest.raises(runtime.RuntimeError, match="a gradient shares memory"):
        runtime.adam_step_device(p, kept, state)
    assert torch.equal(flat, was)
    one = count.view(torch.float64)
    with pytest.raises(runtime.RuntimeError, match="share memory"):
        runtime.adam_step_device([one], [torch.zeros_like(one)],
                                 runtime.DeviceAdamState([one], step=count[0]))
    # clipping: the given norm
    grads = [torch.ones(10, dtype=torch.float64, device="cuda") for _ in range(3)]
    for bad in (grads[0][0], grads[1][9], grads[2][4]):
        with pytest.raises(runtime.RuntimeError, match="the given norm shares memory"):
            runtime.clip_gradients_device(grads, 1.0, norm=bad)
    assert all(bool((t == 1).all()) for t in grads)


def test_a_given_norm_that_is_negated_by_a_bit_alone(runtime):
    """Its memory holds the negative of its value."""
    t = torch.ones(10, dtype=torch.float64, device="cuda")
    norm = torch.tensor([1 - 4j], dtype=torch.complex128, device="cuda").conj().imag[0]
    assert norm.is_neg() and float(norm) == 4.0
    with pytest.raises(TypeError, match="neg bit"):
        runtime.clip_gradients_device([t], 2.0, norm=norm)
    with pytest.raises(TypeError, match="neg bit"):
        runtime.adam_step_device([t], [t.clone()], runtime.DeviceAdamState([t]), max_norm=2.0, norm=norm)
    assert bool((t == 1).all())
    assert float(runtime.clip_gradients_device([t], 2.0, norm=norm.resolve_neg())) == 4.0
