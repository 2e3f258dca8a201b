"""Extreme values, and lists that take several launches, for the tensor operators against 64 bits
(needs a B200)."""
import pytest
import torch

import tensor_training_support as ts
from test_gpu_tensor_training import TYPES, check_norm, gen, normal, run_adam

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [300, 600_000], ids=["short", "long"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1e18, 3e19, 5e20])
def test_large_gradients_in_the_first_steps(runtime, dtype, n, size):
    """Their second moments are within f32's range, those divided by 1 - beta2^t are not."""
    grads = [(torch.rand(n, generator=gen(1), device="cuda") * 0.25 + 0.75).to(TYPES[dtype]) * size]
    params = [normal((n,), TYPES[dtype], gen(2))]
    was = params[0].clone()
    run_adam(runtime, params, grads, lr=0.5)
    # the first step is lr, for bf16 rounded: half a step of values below 8
    assert bool(((was.double() - params[0].double()) - 0.5).abs().max() <= 8 * ts.half_step(TYPES[dtype]))
    run_adam(runtime, params, grads, lr=0.5, betas=(0.9, 0.9999), wd=0.01, decoupled=True)


@pytest.mark.parametrize("n", [300, 600_000], ids=["short", "long"])
def test_epsilon_below_the_types_range(runtime, n):
    """A zero gradient moves nothing with any epsilon above 0; others move as without one."""
    for dtype in ("f32", "bf16", "f64"):
        params = [normal((n,), TYPES[dtype], gen(3))]
        grads = [normal((n,), TYPES[dtype], gen(4))]
        grads[0][::3] = 0.0
        was = params[0].clone()
        run_adam(runtime, params, grads, eps=1e-50)
        assert torch.equal(params[0][::3], was[::3])
        run_adam(runtime, params, grads, eps=2.0 ** -149)
        # the square of this epsilon, which the bounds above divide by, is 0: the formula's 0 / 1e-300
        was = params[0].clone()
        runtime.adam_step_device(params, [torch.zeros_like(was)], runtime.DeviceAdamState(params),
                                 eps=1e-300)
        assert torch.equal(params[0], was)


def placed(tensors, starts):
    """Copies of the tensors in new memory, tensor i starting starts[i] elements behind 512 bytes."""
    out = []
    for t, start in zip(tensors, starts):
        flat = torch.empty(start + t.numel(), dtype=t.dtype, device="cuda")
        out.append(flat[start:].copy_(t))
    return out


@pytest.mark.parametrize("lengths", [[5, 3001, 64], [1_000_003, 5, 262_144]], ids=["short", "long"])
@pytest.mark.parametrize("dtype", ["f64", "f32", "bf16"])
def test_equal_values_that_start_alike_give_equal_bits(runtime, dtype, lengths):
    """In other memory too. Other starts within 16 bytes add in another order: the same to the bound."""
    kind = TYPES[dtype]
    step = 16 // torch.empty((), dtype=kind).element_size()
    g = gen(6)
    params, grads = ([normal((n,), kind, g) for n in lengths] for _ in range(2))
    long = runtime.TensorList(params)._adam_words > 0
    assert long == (sum(lengths) > 100_000)

    def results(starts):
        q = placed(grads, starts)
        norm = runtime.gradient_norm_device(q)
        check_norm(norm, grads)
        p = placed(params, starts)
        state = runtime.DeviceAdamState(p)
        inside = runtime.adam_step_device(p, q, state, max_norm=0.5)
        check_norm(inside, grads)
        clipped = runtime.clip_gradients_device(q, 0.5)
        check_norm(clipped, grads)
        return [norm, inside, clipped] + p + q + state.m + state.v

    for starts in ([0, 0, 0], [1, step - 1, 0]):
        first = results(starts)
        again = results([s + k * step for s, k in zip(starts, (1, 0, 5))])
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    results([1, 0, 1])
