"""The gradient of a table whose rows are as long as memory takes them, on a B200."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, width", [(torch.float16, 65_535 * 1024 - 1), (torch.float16, 65_535 * 1024 + 1),
                                          (torch.bfloat16, 80_000_003)])
def test_rows_of_many_pieces(runtime, dtype, width):
    """Rows that take more blocks than a grid has in its second dimension: pieces of 1024 accesses, of one
    element each where the width is odd. Two places of one row, and a row without any: the sum of two numbers is
    one addition in f32, rounded once."""
    g = torch.empty((2, width), dtype=dtype, device="cuda").normal_(generator=torch.Generator(
        device="cuda").manual_seed(width))
    got = runtime.embedding_gradient_device(g, torch.tensor([1, 1], device="cuda"), 2)
    assert not got[0].any()
    assert torch.equal(got[1], (g[0].float() + g[1].float()).to(dtype))
