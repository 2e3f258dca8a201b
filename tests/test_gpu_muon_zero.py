"""Matrices of zeros orthogonalised without an epsilon, on a B200."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_zeros_stay_zeros(runtime, dtype):
    """X is 0 / 0 by the formula; the documented result is zeros, and a step is the decay alone. A NaN still
    reaches its whole matrix."""
    shapes = [(1, 1), (5, 3), (40, 60), (300, 260), (130, 1000)]
    for eps in (0.0, 1e-7):
        u = [torch.zeros(s, dtype=dtype, device="cuda") for s in shapes]
        bad = [torch.zeros(s, dtype=dtype, device="cuda") for s in shapes]
        for x in bad:
            x[0, 0] = float("nan")
        got = runtime.orthogonalize_device(u + bad, eps=eps)
        assert not any(x.any() for x in got[:len(u)])
        assert all(torch.isnan(x).all() for x in got[len(u):])
        p = [torch.ones(s, dtype=dtype, device="cuda") for s in shapes]
        runtime.muon_step_device(p, u, runtime.DeviceMuonState(p), lr=0.5, weight_decay=0.5, eps=eps)
        assert all((x == 0.75).all() for x in p)
