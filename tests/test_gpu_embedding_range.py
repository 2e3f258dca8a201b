"""Rows whose squares leave f64's range, normalised and with their gradient, on a B200: against the same rows
scaled by powers of two in 64 bits."""
import numpy as np
import pytest
import torch

import matrix_table_support as ms

pytestmark = pytest.mark.gpu

# powers of two of the rows: their entries' squares (or the sums of them) leave f64 below -511 and above 511, the
# entries themselves are below its normal range at -1060
POWERS = [-1060, -800, -530, -511, -450, 0, 450, 505, 511, 800, 1018]


def rows_of(dtype, width, seed):
    """(table, the same rows without their powers): every entry a whole multiple of 2^-12, so that scaling is exact
    but at -1060, where the scaled rows are read back."""
    g = torch.Generator().manual_seed(seed)
    parts = width * (2 if dtype == torch.complex128 else 1)
    x = torch.round(torch.randn((len(POWERS), parts), generator=g, dtype=torch.float64).clamp(-4, 4) * 4096) / 4096
    x[:, 0] = 1.5
    power = np.array(POWERS)[:, None]
    scaled = np.ldexp(x.numpy(), power)
    back = np.ldexp(scaled, -power)

    def typed(a):
        t = torch.from_numpy(a)
        return torch.view_as_complex(t.reshape(len(POWERS), width, 2)) if dtype == torch.complex128 else t
    return typed(scaled), typed(back)


@pytest.mark.parametrize("dtype", [torch.float64, torch.complex128])
@pytest.mark.parametrize("width", [1, 3, 40, 700, 1500, 3001, 9000, 70_000])
def test_normalised_rows(runtime, dtype, width):
    table, plain = rows_of(dtype, width, width)
    index = torch.arange(len(POWERS)).flip(0).repeat(2)
    got = ms.parts(runtime.embedding_lookup_device(table.cuda(), index.cuda(), scale=0.75, normalize=True).cpu())
    want = ms.lookup64(plain, index, 0.75, True, None)
    assert ((got - want).abs() <= ms.lookup_bound(want, plain, True)).all()


@pytest.mark.parametrize("dtype", [torch.float64, torch.complex128])
@pytest.mark.parametrize("width, places", [(2, 40), (40, 40), (700, 40), (1900, 40), (9000, 40), (3, 5000), (40, 5000),
                                           (33_000, 1100), (2, 140_000)])
def test_gradient_through_norms(runtime, dtype, width, places):
    """A row 2^p times as large has a gradient 2^-p times as large: at both ends of the range with gradients that
    keep it in f64."""
    table, plain = rows_of(dtype, width, width + 1)
    g = torch.Generator().manual_seed(places)
    index = torch.randint(0, len(POWERS) - 1, (places,), generator=g)  # none of the last row
    upstream = torch.randn((places, width), generator=g, dtype=dtype)
    want, bound = ms.gradient64(upstream, index, len(POWERS), 0.75, plain, None)
    for power in (-100, 400):
        x = torch.view_as_real(upstream) if dtype == torch.complex128 else upstream
        x = torch.from_numpy(np.ldexp(x.numpy(), power))
        x = torch.view_as_complex(x) if dtype == torch.complex128 else x
        got = ms.parts(runtime.embedding_gradient_device(x.cuda(), index.cuda(), len(POWERS), scale=0.75,
                                                         table=table.cuda()).cpu())
        for r, p in enumerate(POWERS):
            if not -960 < power - p < 990:  # the result leaves f64
                continue
            off = np.ldexp(got[r].numpy(), p - power) - want[r].numpy()
            assert (np.abs(off) <= bound[r].numpy()).all(), (power, p)
        assert not got[-1].any()


@pytest.mark.parametrize("width", [3, 700, 3001, 70_000])
def test_rows_of_zeros_and_infinities(runtime, width):
    """Beside rows out of the range: zeros stay zeros, an infinity is NaN in its place and zeros beside it."""
    table, _ = rows_of(torch.float64, width, 5)
    table[1] = 0
    table[2, 0] = float("inf")
    table[3, 1] = float("nan")
    index = torch.tensor([1, 2, 3])
    got = runtime.embedding_lookup_device(table.cuda(), index.cuda(), normalize=True).cpu()
    assert not got[0].any() and torch.isnan(got[1, 0]) and not got[1, 1:].any() and torch.isnan(got[2]).all()
    for n in (3, 3000):
        x = index.repeat(n // 3)
        got = runtime.embedding_gradient_device(torch.ones((n, width), dtype=torch.float64).cuda(), x.cuda(),
                                                len(POWERS), table=table.cuda()).cpu()
        assert not got[1].any() and torch.isnan(got[3]).all()
