"""The gradient of more places than one cluster sorts, on a B200: every type, through the norm and not, rows of many
widths, with rows that no place points to and one that many do; against 64 bits as in test_gpu_embedding.py."""
import math

import pytest
import torch

import matrix_table_support as ms

pytestmark = pytest.mark.gpu


def check(runtime, dtype, places, rows, width, normalize, seed, start=0):
    gen = torch.Generator().manual_seed(seed)
    wide = torch.complex128 if dtype in (torch.complex64, torch.complex128) else torch.float64
    g = (torch.randn((places, width + start), generator=gen, dtype=wide) * 0.1).to(dtype)
    table = torch.randn((rows, width + start), generator=gen, dtype=wide).to(dtype)
    # every third row: the first of them has about a tenth of the places
    x = torch.exp(torch.rand(places, generator=gen, dtype=torch.float64) * math.log(rows / 3 + 1)) - 1
    index = (x.long() * 3).clamp(0, rows - 1)
    v, t = g[:, start:], table[:, start:]
    gd, td = g.cuda()[:, start:], table.cuda()[:, start:]
    got = runtime.embedding_gradient_device(gd, index.cuda(), rows, scale=0.5, table=td if normalize else None, padding=3)
    want, bound = ms.gradient64(v, index, rows, 0.5, t if normalize else None, 3)
    off = (ms.parts(got.cpu()) - want).abs()
    assert (off <= bound).all(), (float(off.max()), float((off - bound).max()))
    assert not got[1::3].any() and not got[2::3].any() and not got[3:4].any()
    assert torch.equal(got, runtime.embedding_gradient_device(gd, index.cuda(), rows, scale=0.5,
                                                              table=td if normalize else None, padding=3))


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16, torch.float16, torch.complex128,
                                   torch.complex64])
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("places, rows, width", [(131_073, 5000, 24), (300_000, 700, 10), (200_001, 150_001, 5),
                                                 (131_073, 300, 257)])
def test_types(runtime, dtype, normalize, places, rows, width):
    check(runtime, dtype, places, rows, width, normalize, places + width)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("start, width", [(1, 64), (3, 128), (1, 7)])
def test_rows_that_start_anywhere(runtime, dtype, start, width):
    check(runtime, dtype, 140_000, 900, width, True, width, start)
    check(runtime, dtype, 140_000, 900, width, False, width, start)


@pytest.mark.parametrize("rows", [1, 511, 512, 262_143, 262_145])
def test_rows_around_the_sorts_digits(runtime, rows):
    check(runtime, torch.bfloat16, 131_500, rows, 4, rows % 2 == 1, rows)
