"""Extreme values, and lists that take several launches, for the tensor operators against 64 bits
(needs a B200)."""
import pytest
import torch

import tensor_training_support as ts
from test_gpu_tensor_training import TYPES, gen, normal, run_adam

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
