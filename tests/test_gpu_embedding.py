"""Lookups in a table and their gradient on a B200: each call against 64 bits with bounds counted per
operation, over types, widths, indices and layouts."""
import math

import pytest
import torch

import matrix_table_support as ms

pytestmark = pytest.mark.gpu

TYPES = [torch.float64, torch.float32, torch.bfloat16, torch.float16, torch.complex128, torch.complex64]


def make(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    wide = {torch.complex128: torch.complex128, torch.complex64: torch.complex128}.get(dtype, torch.float64)
    return (torch.randn(shape, generator=g, dtype=wide) * scale).to(dtype)


def indices(n, rows, seed, kind=torch.int64, skewed=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.rand(n, generator=g, dtype=torch.float64)
    x = torch.exp(x * math.log(rows + 1)) - 1 if skewed else x * rows
    return x.long().clamp(0, max(0, rows - 1)).to(kind)


def check_lookup(runtime, table, index, scale=1.0, normalize=False, padding=None):
    got = runtime.embedding_lookup_device(table.cuda(), index.cuda(), scale=scale, normalize=normalize,
                                          padding=padding)
    assert got.dtype == table.dtype and got.shape == index.shape + table.shape[1:]
    flat = index.reshape(-1).long()
    want = ms.lookup64(table, flat, scale, normalize, padding)
    bound = ms.lookup_bound(want, table, normalize)
    x = ms.parts(got.cpu().reshape((flat.numel(),) + table.shape[1:]))
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(x), nan)
    assert ((x - want).abs()[~nan] <= bound[~nan]).all(), float((x - want).abs()[~nan].max())


def check_gradient(runtime, g, index, rows, scale=1.0, table=None, padding=None):
    got = runtime.embedding_gradient_device(g.cuda(), index.cuda(), rows, scale=scale,
                                            table=None if table is None else table.cuda(), padding=padding)
    inner = g.shape[index.dim():]
    assert got.dtype == g.dtype and got.shape == (rows,) + inner
    flat = index.reshape(-1).long()
    want, bound = ms.gradient64(g.reshape((flat.numel(),) + inner), flat, rows, scale, table, padding)
    off = (ms.parts(got.cpu()) - want).abs()
    assert (off <= bound).all(), (float(off.max()), float((off - bound).max()))
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, width, n", [(1, 1, 1), (7, 3, 5), (61, 16, 256), (5, 33, 300), (1000, 97, 300),
                                            (33, 1024, 50), (3, 2500, 17), (2, 40_001, 3), (129, 4, 5000)])
def test_lookup(runtime, dtype, rows, width, n):
    table, index = make((rows, width), dtype, rows + width), indices(n, rows, n, torch.int32 if n % 2 else torch.int64)
    for scale, normalize, padding in ((1.0, False, None), (0.3, False, 0), (1.0, True, None), (2.5, True, rows - 1)):
        check_lookup(runtime, table, index, scale, normalize, padding)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, width, n", [(1, 1, 1), (7, 3, 5), (61, 16, 256), (5, 33, 300), (1000, 97, 300),
                                            (33, 1024, 50), (3, 2500, 17), (2, 40_001, 3), (129, 4, 5000),
                                            (600, 8, 2049), (1, 5, 4100)])
def test_gradient(runtime, dtype, rows, width, n):
    table, g = make((rows, width), dtype, rows), make((n, width), dtype, n, 0.1)
    for k, (scale, normalize, padding) in enumerate(((1.0, False, None), (0.3, False, 0), (1.5, True, None),
                                                     (1.0, True, rows - 1))):
        index = indices(n, rows, n + k, torch.int32 if n % 2 else torch.int64, k % 2 == 1)
        check_gradient(runtime, g, index, rows, scale, table if normalize else None, padding)


@pytest.mark.parametrize("rows", [511, 512, 513, 262_143, 262_144, 300_001])
def test_gradient_of_many_rows(runtime, rows):
    """Rows on both sides of the sort's digits."""
    g = make((3000, 2), torch.float32, rows)
    check_gradient(runtime, g, indices(3000, rows, rows), rows)
    check_gradient(runtime, g, torch.full((3000,), rows - 1), rows, padding=0)


@pytest.mark.parametrize("n", [1024, 1025, 8192, 8193, 20_000, 131_072, 131_073, 300_000])
def test_gradient_of_many_places(runtime, n):
    g = make((n, 3), torch.float32, n)
    check_gradient(runtime, g, indices(n, 700, n, skewed=True), 700, 0.5)
    check_gradient(runtime, g, torch.zeros(n, dtype=torch.int64), 3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.complex64])
@pytest.mark.parametrize("n", [40, 3000])
def test_rows_that_start_anywhere(runtime, dtype, n):
    """Views whose rows start off the accesses' boundaries, through the norm too, against their copies."""
    wide, g = make((20, 300), dtype, 1).cuda(), make((n, 300), dtype, 2).cuda()
    x = indices(n, 20, 3).cuda()
    for start, width in ((1, 64), (3, 128), (5, 200), (1, 7)):
        t, v = wide[:, start:start + width], g[:, start:start + width]
        for table in (None, t):
            got = runtime.embedding_gradient_device(v, x, 20, table=table)
            assert torch.equal(got, runtime.embedding_gradient_device(
                v.contiguous(), x, 20, table=None if table is None else table.contiguous()))
        index = x.cpu().long()
        check_gradient(runtime, v.cpu(), index, 20, table=t.cpu().contiguous())
        check_lookup(runtime, t.cpu().contiguous(), index, 0.5, True)


def test_indices_outside_and_padding(runtime):
    table = make((10, 6), torch.float32, 1)
    index = torch.tensor([0, -1, 10, 9, 3, 2 ** 40, -2 ** 40, 3, 9])
    check_lookup(runtime, table, index)
    check_lookup(runtime, table, index, normalize=True, padding=3)
    check_lookup(runtime, table, index, padding=2 ** 40)
    g = make((9, 6), torch.float32, 2)
    check_gradient(runtime, g, index, 10)
    check_gradient(runtime, g, index, 10, table=table, padding=3)
    check_gradient(runtime, g, torch.full((9,), -5), 10)
    check_gradient(runtime, g, torch.full((9,), 4), 10, padding=4)


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.complex128])
@pytest.mark.parametrize("width", [8, 5000, 70_000])
def test_rows_of_zeros_and_extreme_rows(runtime, dtype, width):
    table = make((6, width), dtype, 3)
    table[1] = 0
    table[2] *= 1e-30
    table[4] *= 1e30
    index = torch.tensor([0, 1, 2, 3, 4, 5, 1])
    check_lookup(runtime, table, index, normalize=True)
    check_gradient(runtime, make((7, width), dtype, 4), index, 6, table=table)
    table[3, 1] = math.nan
    table[5, 0] = math.inf
    got = runtime.embedding_lookup_device(table.cuda(), index.cuda(), normalize=True).cpu()
    assert torch.isnan(got[3]).all() and torch.isnan(got[5, :1]).all()
    assert torch.isfinite(torch.view_as_real(got[[0, 1, 2, 4, 6]]) if got.is_complex() else got[[0, 1, 2, 4, 6]]).all()


def test_shapes_and_layouts(runtime):
    table = make((9, 4, 6), torch.float32, 5).cuda()
    index = indices(24, 9, 6).reshape(2, 3, 4)
    check_lookup(runtime, table.cpu(), index)
    wide = make((9, 40), torch.float32, 7).cuda()
    for view in (wide[:, 3:20], wide[::2, :32], wide[:, 1:2], wide[:1].expand(5, 40)):
        x = indices(11, view.shape[0], 8).cuda()
        for normalize in (False, True):
            got = runtime.embedding_lookup_device(view, x, normalize=normalize)
            assert torch.equal(got, runtime.embedding_lookup_device(view.contiguous(), x, normalize=normalize))
    turned = index.cuda().permute(2, 0, 1)
    assert torch.equal(runtime.embedding_lookup_device(table, turned),
                       runtime.embedding_lookup_device(table, turned.contiguous()))
    g = make((30, 40), torch.bfloat16, 9).cuda()
    for view in (g[:, 5:37], g[::3], g[:1].expand(12, 40), g[:, 7:8]):
        x = indices(view.shape[0], 5, 10).cuda()
        assert torch.equal(runtime.embedding_gradient_device(view, x, 5),
                           runtime.embedding_gradient_device(view.contiguous(), x, 5))
    check_gradient(runtime, make((2, 3, 4, 4, 6), torch.float64, 11), index, 9)


def test_nothing_to_do(runtime):
    table = make((4, 3), torch.float32, 1).cuda()
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert runtime.embedding_lookup_device(table, none).shape == (0, 3)
    got = runtime.embedding_gradient_device(table[:0], none, 4)
    assert got.shape == (4, 3) and not got.any()
    got = runtime.embedding_gradient_device(table[:0], none, 4, table=table)
    assert got.shape == (4, 3) and not got.any()
    assert runtime.embedding_lookup_device(table[:, :0], none + 1).shape == (0, 0)
    x = torch.tensor([0, 1], device="cuda")
    assert runtime.embedding_lookup_device(table[:, :0], x).shape == (2, 0)
    assert torch.isnan(runtime.embedding_lookup_device(table[:0], x)).all()
    assert runtime.embedding_gradient_device(table[:2], x, 0).shape == (0, 3)


def test_equal_bits(runtime):
    """Hot rows over several chunks, run again and replayed: no order is left open."""
    g = make((20_011, 130), torch.bfloat16, 1).cuda()
    x = indices(20_011, 3000, 2, skewed=True).cuda()
    want = runtime.embedding_gradient_device(g, x, 3000)
    for _ in range(3):
        assert torch.equal(want, runtime.embedding_gradient_device(g, x, 3000))


def test_captured_and_on_other_streams(runtime):
    table = make((50, 64), torch.complex128, 1).cuda()
    x = indices(70, 50, 2).cuda()
    g = make((70, 64), torch.complex128, 3).cuda()

    def both():
        return (runtime.embedding_lookup_device(table, x, normalize=True),
                runtime.embedding_gradient_device(g, x, 50, table=table))

    want = [t.clone() for t in both()]
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both()
        graphs.append((graph, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(3):
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = runtime.embedding_gradient_device(g, x, 50, table=table, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(got, want[1])
    # new values, replayed
    table.mul_(1.5).add_(0.1)
    x.copy_(x.flip(0))
    torch.cuda.synchronize()
    graphs[0][0].replay()
    assert all(torch.equal(a, b) for a, b in zip(graphs[0][1], both()))


def test_large_offsets(runtime):
    """A table and gradient of more than 2^32 bytes and elements past 2^31."""
    rows, width = 70_000, 32_768
    table = torch.empty((rows, width), dtype=torch.bfloat16, device="cuda")
    picked = torch.tensor([0, 65_535, 65_536, rows - 1], device="cuda")
    values = make((4, width), torch.bfloat16, 1).cuda()
    table[picked] = values
    assert torch.equal(runtime.embedding_lookup_device(table, picked), values)
    got = runtime.embedding_gradient_device(values, picked, rows)
    assert torch.equal(got[picked], values)
    assert not got[65_500:65_535].any() and not got[rows - 9:rows - 1].any() and not got[1:9].any()
    x = torch.full((rows,), 2, device="cuda")
    x[-2:] = torch.tensor([1, 0], device="cuda")
    table[:-2] = 0
    table[rows - 2:] = values[:2]
    got = runtime.embedding_gradient_device(table, x, 3)
    assert torch.equal(got[0], values[1]) and torch.equal(got[1], values[0]) and not got[2].any()


def test_refusals(runtime):
    table = make((5, 4), torch.float32, 1).cuda()
    x = torch.tensor([1, 2], device="cuda")
    for bad in (table.cpu(), table.int(), [1.0], table.to_sparse()):
        with pytest.raises(TypeError, match="the table must be a dense"):
            runtime.embedding_lookup_device(bad, x)
    with pytest.raises(TypeError, match="lazy conj"):
        runtime.embedding_lookup_device(table.to(torch.complex64).conj(), x)
    with pytest.raises(TypeError, match="rows without gaps"):
        runtime.embedding_lookup_device(table[:, ::2], x)
    with pytest.raises(TypeError, match="no dimension"):
        runtime.embedding_lookup_device(table[0], x)
    for bad in (x.cpu(), x.float(), x.to(torch.int16), [1, 2]):
        with pytest.raises(TypeError, match="indices must be"):
            runtime.embedding_lookup_device(table, bad)
    with pytest.raises(ValueError, match="padding"):
        runtime.embedding_lookup_device(table, x, padding=-1)
    for scale in (math.nan, math.inf):
        with pytest.raises(runtime.RuntimeError, match="scale must be finite"):
            runtime.embedding_lookup_device(table, x, scale=scale)
    with pytest.raises(ValueError, match="a row for each index"):
        runtime.embedding_gradient_device(table, x, 5)
    with pytest.raises(ValueError, match="the table must be"):
        runtime.embedding_gradient_device(table[:2], x, 6, table=table)
    with pytest.raises(ValueError, match="the table must be"):
        runtime.embedding_gradient_device(table[:2].double(), x, 5, table=table)
    with pytest.raises(ValueError, match="negative"):
        runtime.embedding_gradient_device(table[:2], x, -1)
    with pytest.raises(TypeError, match="equal distances"):
        runtime.embedding_gradient_device(make((2, 3, 4), torch.float32, 1).cuda().permute(1, 0, 2), x.expand(3, 2), 5)


# ------------------------------------------------------------------ through autograd and a circuit


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("normalize", [False, True])
def test_autograd(runtime, dtype, normalize):
    from arcqml_b200.embedding import lookup
    table = make((11, 12), dtype, 1).cuda().requires_grad_(True)
    index = indices(30, 11, 2).reshape(5, 6).cuda()
    upstream = make((5, 6, 12), dtype, 3).cuda()
    out = lookup(table, index, 0.7, normalize, padding=2)
    out.backward(upstream)
    want = runtime.embedding_gradient_device(upstream, index, 11, 0.7, table.detach() if normalize else None, 2)
    assert torch.equal(table.grad, want)
    # a sum's gradient is one number, expanded
    table.grad = None
    lookup(table, index, 0.7, normalize).real.sum().backward()
    ones = torch.ones((5, 6, 12), dtype=dtype, device="cuda")
    want = runtime.embedding_gradient_device(ones, index, 11, 0.7, table.detach() if normalize else None)
    assert torch.equal(table.grad, want)
    with torch.no_grad():
        assert not lookup(table, index).requires_grad


@pytest.mark.parametrize("dtype", [torch.float64, torch.complex128])
@pytest.mark.parametrize("normalize", [False, True])
def test_gradient_against_differences(runtime, dtype, normalize):
    """Central differences of a smooth f64 loss: h^2 / 6 of a third derivative (below 1e3 here, rows of
    norm 0.5 and more) and 1e-16 / h of rounding: below 1e-6 for h = 1e-5."""
    from arcqml_b200.embedding import lookup
    table = make((5, 4), dtype, 8)
    table[:, 0] += 2.0
    index = torch.tensor([0, 3, 3, 1, 3, 4]).cuda()
    w = make((6, 4), dtype, 9).cuda()

    def loss(t):
        x = lookup(t, index, 1.3, normalize, padding=1)
        return ((x * w).real.sum(dim=1)).square().sum() + (x.abs() ** 2 if x.is_complex() else x ** 2)[:, 0].sum()

    t = table.cuda().requires_grad_(True)
    loss(t).backward()
    g = ms.parts(t.grad.cpu())
    flat = torch.view_as_real(table) if table.is_complex() else table
    flat = flat.reshape(5, -1)
    h = 1e-5
    for r in range(5):
        for k in range(flat.shape[1]):
            values = []
            for sign in (1, -1):
                moved = flat.clone()
                moved[r, k] += sign * h
                moved = torch.view_as_complex(moved.reshape(5, -1, 2)) if table.is_complex() else moved
                values.append(float(loss(moved.cuda())))
            assert abs((values[0] - values[1]) / (2 * h) - float(g[r, k])) < 1e-6, (r, k)


def test_double_backward_is_refused(runtime):
    from arcqml_b200.embedding import lookup
    table = make((5, 4), torch.float64, 1).cuda().requires_grad_(True)
    out = lookup(table, torch.tensor([1, 2]).cuda(), normalize=True)
    g, = torch.autograd.grad(out.square().sum(), table, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_states_of_a_table_in_a_circuit(runtime):
    """<Z0 + X1> of a trained circuit on states picked from a table of amplitudes: the table's gradient against
    differences of the loss (as above: below 1e-6)."""
    import numpy as np
    from arcqml_b200 import Circuit, SparsePauliOp
    from arcqml_b200.simulator import BatchStateVectorSimulator, SimError
    c = Circuit(2)
    c.append("ry", (0,), c.add_parameter(0.4)).append("cnot", (0, 1)).append("rx", (1,), c.add_parameter(1.1))
    h = SparsePauliOp(2)
    h.add_term(1.0, [(0, "Z")]).add_term(0.5, [(1, "X")])
    amplitudes = make((3, 4), torch.complex128, 4) + 1.0
    index = torch.tensor([2, 0, 2, 2, 0]).cuda()
    weight = np.array([1.0, -0.5, 0.25, 2.0, 1.0])

    def loss(a):
        sim = BatchStateVectorSimulator.from_table(2, a, index)
        return float(np.sum(weight * sim.run(c, h, grad=False).values))

    table = amplitudes.cuda().requires_grad_(True)
    sim = BatchStateVectorSimulator.from_table(2, table, index)
    assert np.allclose(np.linalg.norm(sim.amplitudes(), axis=1), 1.0, atol=1e-14)
    _, initial = sim.run(c, h).backward(weight)
    sim.states.backward(initial)
    g = torch.view_as_real(table.grad.cpu())
    assert not g[1].any()
    step = 1e-5
    for r in range(3):
        for k in range(4):
            for part, unit in ((0, 1.0), (1, 1j)):
                pair = []
                for sign in (1, -1):
                    moved = amplitudes.clone()
                    moved[r, k] += sign * step * unit
                    pair.append(loss(moved.cuda()))
                assert abs((pair[0] - pair[1]) / (2 * step) - float(g[r, k, part])) < 1e-6, (r, k, part)
    for bad in ((1, table, index), (2, table.real, index), (2, table, index.reshape(1, -1)), (2, table, index[:0])):
        with pytest.raises(SimError):
            BatchStateVectorSimulator.from_table(*bad)
