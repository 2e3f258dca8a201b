"""The gradient norm, clipping and the Adam step over many device tensors against 64 bits (needs a
B200)."""
import math

import numpy as np
import pytest
import torch

import tensor_training_support as ts

pytestmark = pytest.mark.gpu

TYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16,
         "c128": torch.complex128, "c64": torch.complex64}
# lengths around vectors (2, 4, 8 elements), a block's share, the chunks, and empty tensors
LENGTHS = {"one": [1], "short": [1, 2, 3, 5, 7, 8, 9, 0, 15, 16, 17, 31, 33],
           "chunks": [2047, 2048, 2049, 8191, 8192, 8193, 16385],
           "large": [1_000_003, 70_001, 5, 262_144]}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(shape, dtype, g, scale=1.0):
    """Values of `dtype`; complex ones with two components."""
    kind = {torch.complex128: torch.float64, torch.complex64: torch.float32}.get(dtype, dtype)
    if dtype.is_complex:
        t = torch.randn(*shape, 2, generator=g, device="cuda", dtype=kind) * scale
        return torch.view_as_complex(t)
    return (torch.randn(tuple(shape), generator=g, device="cuda", dtype=torch.float64) * scale).to(kind)


def views(lengths, dtype, g, offset, scale=1.0):
    """Tensors of the lengths as views of one buffer without gaps, the first `offset` elements in."""
    flat = normal((offset + sum(lengths) + 1,), dtype, g, scale)
    out, at = [], offset
    for n in lengths:
        out.append(flat[at:at + n])
        at += n
    return flat, out


def count(tensors):
    return sum(t.numel() * (2 if t.is_complex() else 1) for t in tensors if t is not None)


def check_norm(got, tensors):
    want = ts.norm64(tensors)
    assert abs(float(got) - want) <= ts.norm_bound(count(tensors)) * want


@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_and_clip(runtime, dtype, lengths, offset):
    g = gen(11 + offset)
    flat, grads = views(LENGTHS[lengths], TYPES[dtype], g, offset)
    before = flat.clone()
    norm = runtime.gradient_norm_device(grads)
    assert norm.dtype == torch.float64 and norm.shape == () and norm.is_cuda
    check_norm(norm, grads)
    assert torch.equal(torch.view_as_real(flat) if flat.is_complex() else flat,
                       torch.view_as_real(before) if flat.is_complex() else before)
    want = ts.norm64(grads)
    for max_norm in (0.37 * want, 2.0 * want, 0.0):
        work = flat.clone()
        at, mine = offset, []
        for n in LENGTHS[lengths]:
            mine.append(work[at:at + n])
            at += n
        got = runtime.clip_gradients_device(mine, max_norm)
        check_norm(got, grads)
        factor = ts.clip_factor(want, max_norm)
        for a, b in zip(mine, grads):
            y, bound = ts.clip64(b, factor, count(grads))
            ts.assert_within(ts.components(a), y, bound, (dtype, max_norm))
        # what lies around the tensors is left alone
        assert torch.equal(work[:offset], before[:offset]) and torch.equal(work[at:], before[at:])


def test_norm_of_mixed_types_strides_and_empty_places(runtime):
    g = gen(5)
    a = normal((5, 7, 3), torch.float32, g).permute(2, 0, 1)
    b = normal((40, 30), torch.bfloat16, g).t()
    c = normal((3, 64), torch.complex128, g)
    d = torch.tensor(2.5, dtype=torch.float64, device="cuda")
    e = torch.empty((0, 4), device="cuda")
    grads = [a, None, b, c, d, e, normal((1, 9, 1), torch.float16, g)]
    check_norm(runtime.gradient_norm_device(grads), grads)
    kept = [None if t is None else t.clone() for t in grads]
    want = ts.norm64(grads)
    runtime.clip_gradients_device(grads, 0.1)
    for x, y in zip(grads, kept):
        if x is not None:
            z, bound = ts.clip64(y, ts.clip_factor(want, 0.1), count(kept))
            ts.assert_within(ts.components(x), z, bound, x.dtype)
    for nothing in ([], [None, None], [e]):
        assert float(runtime.gradient_norm_device(nothing)) == 0.0
        assert float(runtime.clip_gradients_device(nothing, 1.0)) == 0.0


@pytest.mark.parametrize("tensors", [64, 65, 511, 512, 513, 1100, 1500, 1501])
def test_lists_longer_than_one_launch(runtime, tensors):
    g = gen(tensors)
    lengths = [1 + (i * 37) % 201 for i in range(tensors)]
    flat, grads = views(lengths, torch.float32, g, 0)
    check_norm(runtime.gradient_norm_device(grads), grads)
    params = [normal((n,), torch.float32, g) for n in lengths]
    run_adam(runtime, params, grads, max_norm=0.5)


def test_large_and_tiny_values(runtime):
    """f32 squares leave the range of f32: the sum is in f64."""
    for scale in (1e30, 1e-30):
        t = torch.full((1000,), scale, dtype=torch.float32, device="cuda")
        check_norm(runtime.gradient_norm_device([t]), [t])
    t = torch.full((9,), 2.0 ** -149, dtype=torch.float32, device="cuda")  # subnormals count
    check_norm(runtime.gradient_norm_device([t]), [t])
    t = torch.full((9,), 2.0 ** -133, dtype=torch.bfloat16, device="cuda")
    check_norm(runtime.gradient_norm_device([t]), [t])
    t = torch.full((70000,), 65504.0, dtype=torch.float16, device="cuda")
    check_norm(runtime.gradient_norm_device([t]), [t])
    t = torch.full((7,), torch.finfo(torch.bfloat16).max, dtype=torch.bfloat16, device="cuda")
    check_norm(runtime.gradient_norm_device([t]), [t])


@pytest.mark.parametrize("dtype", ["f64", "f32", "bf16", "f16"])
@pytest.mark.parametrize("place", [0, 4, 8197])
def test_infinities_and_nan(runtime, dtype, place):
    kind = TYPES[dtype]
    for bad in (math.inf, -math.inf, math.nan):
        t = normal((9000,), kind, gen(3))
        t[place] = bad
        other = normal((77,), torch.float32, gen(4))
        norm = runtime.clip_gradients_device([t, other], 1.0)
        if math.isnan(bad):
            assert math.isnan(float(norm)) and t.isnan().all() and other.isnan().all()
        else:  # the factor is 0, and infinity times 0 is NaN
            assert float(norm) == math.inf and other.eq(0).all()
            assert t[place].isnan() and int(t.isnan().sum()) == 1
            assert t.nan_to_num(0.0).eq(0).all()


@pytest.mark.parametrize("n", [300, 3_000_000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_factors_below_the_normal_range(runtime, dtype, n):
    """Gradients near the type's largest values, and a small maximum: the factor is subnormal in
    f32, the results are not."""
    kind = TYPES[dtype]
    t = (torch.rand(n, generator=gen(9), device="cuda") + 0.5).to(kind) * 1e38
    was = t.clone()
    want = ts.norm64([was])
    runtime.clip_gradients_device([t], 1e-2)
    y, bound = ts.clip64(was, ts.clip_factor(want, 1e-2), n)
    assert ts.clip_factor(want, 1e-2) < 2.0 ** -126 and y.min() > 2.0 ** -120
    ts.assert_within(ts.components(t), y, bound, dtype)
    run_adam(runtime, [torch.zeros(n, dtype=kind, device="cuda")], [was], max_norm=1e-2)


def test_one_tensor_in_place_of_a_list(runtime):
    t = normal((60, 70), torch.float32, gen(6))
    check_norm(runtime.gradient_norm_device(t), [t])
    check_norm(runtime.clip_gradients_device(t[3], 1e9), [t[3]])


def test_equal_inputs_give_equal_bits(runtime):
    _, grads = views([300_001, 17, 5_000_000], torch.bfloat16, gen(8), 1)
    first = runtime.gradient_norm_device(grads)
    for _ in range(5):
        assert torch.equal(runtime.gradient_norm_device(grads), first)


def test_clip_with_a_given_norm(runtime):
    t = normal((1000,), torch.float64, gen(2))
    was = t.clone()
    norm = torch.tensor(50.0, dtype=torch.float64, device="cuda")
    out = runtime.clip_gradients_device([t], 5.0, norm=norm)
    assert float(out) == 50.0
    ts.assert_within(ts.components(t), ts.components(was) * (5.0 / (50.0 + 1e-6)),
                     6 * ts.U64 * np.abs(ts.components(was)), "given")
    for bad in (torch.tensor(1.0, device="cuda"), torch.tensor(1.0, dtype=torch.float64), 1.0,
                torch.ones(2, dtype=torch.float64, device="cuda")):
        with pytest.raises(TypeError, match="given norm"):
            runtime.clip_gradients_device([t], 5.0, norm=bad)


def run_adam(runtime, params, grads, m=None, v=None, step=0, lr=0.01, betas=(0.9, 0.999), eps=1e-8,
             wd=0.0, decoupled=False, max_norm=None, copies=None, steps=1, norm=None):
    """Runs `steps` steps, each checked against 64 bits from the values before it."""
    state = runtime.DeviceAdamState(params, m=m, v=v, step=step)
    total = count(grads)
    for k in range(steps):
        olds = [[ts.components(t) for t in x] for x in (params, state.m, state.v)]
        out = runtime.adam_step_device(params, grads, state, lr=lr, betas=betas, eps=eps,
                                       weight_decay=wd, decoupled=decoupled, max_norm=max_norm,
                                       copies=copies, norm=norm)
        assert int(state.step) == step + k + 1
        factor, rel = 1.0, 0.0
        if max_norm is None:
            assert out is None
        else:
            n = ts.norm64(grads) if norm is None else float(norm)
            assert abs(float(out) - n) <= ts.norm_bound(total) * n
            factor, rel = ts.clip_factor(n, max_norm), ts.norm_bound(total) + 3 * ts.U64
        for i, (p, g) in enumerate(zip(params, grads)):
            kind = ts.real_type(p)
            if g is None:
                for t, o in zip((p, state.m[i], state.v[i]), (x[i] for x in olds)):
                    assert np.array_equal(ts.components(t), o)
                continue
            u = ts.U64 if kind == torch.float64 else ts.U32
            p2, m2, v2, pe, me, ve = ts.adam64(
                olds[0][i], ts.components(g), olds[1][i], olds[2][i], step + k + 1, lr, betas[0],
                betas[1], eps, wd, decoupled, factor, u, rel)
            tiny = ts.TINY[torch.float64 if kind == torch.float64 else torch.float32]
            ts.assert_within(ts.components(state.m[i]), m2, me + 4 * tiny, ("m", i, p.dtype))
            ts.assert_within(ts.components(state.v[i]), v2, ve + 4 * tiny, ("v", i, p.dtype))
            if kind in (torch.bfloat16, torch.float16):
                pe = pe + ts.half_step(kind) * (np.abs(p2) + pe) + ts.TINY[kind]
            ts.assert_within(ts.components(p), p2, pe + 4 * tiny, ("p", i, p.dtype))
            if copies is not None and copies[i] is not None:
                # the copy is the f32 value rounded once
                assert torch.equal(copies[i], p.to(copies[i].dtype))
    return state


MIXES = [("f64", "f64"), ("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("c128", "c128"),
         ("c64", "c64"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "f32"), ("f16", "f32"),
         ("bf16", "f16"), ("f16", "bf16")]


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("types", MIXES, ids=lambda m: "-".join(m))
def test_adam_types_and_lengths(runtime, types, lengths):
    g = gen(21)
    p_type, g_type = TYPES[types[0]], TYPES[types[1]]
    params = [normal((n,), p_type, g) for n in LENGTHS[lengths]]
    grads = [normal((n,), g_type, g, 0.1) for n in LENGTHS[lengths]]
    run_adam(runtime, params, grads, steps=3, wd=0.01, max_norm=0.2)
    run_adam(runtime, params, grads, step=40, wd=0.1, decoupled=True)


@pytest.mark.parametrize("offsets", [(0, 0), (0, 1), (1, 0), (1, 1), (3, 3), (3, 2), (5, 1)])
@pytest.mark.parametrize("types", [("f64", "f64"), ("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16")],
                         ids=lambda m: "-".join(m))
def test_adam_views_at_any_offset(runtime, types, offsets):
    g = gen(31)
    lengths = [1, 6, 8191, 3, 20_000]
    flat_p, params = views(lengths, TYPES[types[0]], g, offsets[0])
    flat_g, grads = views(lengths, TYPES[types[1]], g, offsets[1])
    copies, flat_c = None, None
    if types == ("f32", "bf16"):
        flat_c, copies = views(lengths, torch.bfloat16, g, offsets[1])
        ends = flat_c[:offsets[1]].clone(), flat_c[-1:].clone()
    first, last, kept = flat_p[:offsets[0]].clone(), flat_p[-1:].clone(), flat_g.clone()
    run_adam(runtime, params, grads, max_norm=1.0, wd=0.02, copies=copies)
    # moments that start elsewhere in their vectors
    _, m = views(lengths, TYPES[types[0]] if types[0] == "f64" else torch.float32, g, 2, 0.1)
    v = [t.abs() for t in views(lengths, m[0].dtype, g, 0, 0.01)[1]]
    run_adam(runtime, params, grads, m=m, v=v, step=7, copies=copies)
    assert torch.equal(flat_p[:offsets[0]], first) and torch.equal(flat_p[-1:], last)
    assert torch.equal(flat_g, kept)
    if copies:
        assert torch.equal(flat_c[:offsets[1]], ends[0]) and torch.equal(flat_c[-1:], ends[1])


def test_adam_mixed_list_with_copies_strides_and_missing_gradients(runtime):
    g = gen(41)
    params = [normal((80,), torch.float64, g), normal((33, 65), torch.float32, g).t(),
              normal((4, 128), torch.complex128, g), normal((9,), torch.bfloat16, g),
              normal((7, 3), torch.float32, g), torch.empty((0, 3), device="cuda"),
              torch.tensor(0.5, device="cuda")]
    grads = [normal(p.shape, p.dtype, g, 0.1) for p in params]
    grads[1] = normal((33, 65), torch.bfloat16, g).t()
    grads[4] = None
    copies = [None, torch.zeros((33, 65), dtype=torch.bfloat16, device="cuda").t(), None, None, None,
              torch.empty((0, 3), dtype=torch.float16, device="cuda"),
              torch.zeros((), dtype=torch.float16, device="cuda")]
    run_adam(runtime, params, grads, max_norm=0.1, wd=0.01, decoupled=True, copies=copies, steps=2)
    run_adam(runtime, [], [], max_norm=1.0)
    run_adam(runtime, params[4:5], [None])


def test_adam_zero_gradient_zero_moments_and_extreme_values(runtime):
    p = [normal((100,), torch.float32, gen(1)), normal((100,), torch.float64, gen(1))]
    zero = [torch.zeros_like(t) for t in p]
    was = [t.clone() for t in p]
    run_adam(runtime, p, zero, max_norm=1.0)
    assert all(torch.equal(a, b) for a, b in zip(p, was))  # 0 / (0 + eps)
    run_adam(runtime, p, [t * 1e15 for t in was], max_norm=1e-3)
    run_adam(runtime, p, [t * 0.1 for t in was], betas=(0.0, 0.0), lr=0.0)


def test_adam_matches_the_hosts_update(runtime):
    """f64: the same operations in the same order as AdamState.update; the device's power may differ
    by a step, which bc_err in the bound counts."""
    g = np.random.default_rng(3)
    x, host = g.normal(size=300), runtime.AdamState(300)
    p = [torch.from_numpy(x.copy()).cuda()]
    state = runtime.DeviceAdamState(p)
    for t in range(1, 30):
        grad = g.normal(size=300)
        x = host.update(x, grad, lr=0.03, weight_decay=0.01)
        runtime.adam_step_device(p, [torch.from_numpy(grad).cuda()], state, lr=0.03,
                                 weight_decay=0.01)
        # per step: 4 u / bc2 relative in the root at most (bc2 >= 1e-3 t), half of it in the step of
        # at most lr * 4, plus a few roundings of |x| <= 5
        bound = t * (0.03 * 4 * (2 * 4 * ts.U64 / 1e-3 + 8 * ts.U64) + 8 * ts.U64 * 5)
        assert np.max(np.abs(p[0].cpu().numpy() - x)) <= bound


def test_given_norm_goes_over_several_lists(runtime):
    g = gen(51)
    params = [normal((50,), torch.float32, g), normal((60,), torch.float64, g)]
    grads = [normal((50,), torch.float32, g), normal((60,), torch.float64, g)]
    norm = runtime.gradient_norm_device(grads)
    run_adam(runtime, params[:1], grads[:1], max_norm=0.5, norm=norm)
    run_adam(runtime, params[1:], grads[1:], max_norm=0.5, norm=norm)


def test_moved_tensors_are_found_and_lists_can_be_kept(runtime):
    g = gen(61)
    p = [torch.nn.Parameter(normal((500,), torch.float32, g)), normal((30,), torch.float32, g)]
    grads = [normal((500,), torch.float32, g), normal((30,), torch.float32, g)]
    pl, gl = runtime.TensorList(p), runtime.TensorList(grads)
    check_norm(runtime.gradient_norm_device(gl), grads)
    grads[0].data = normal((700,), torch.float64, g)
    check_norm(runtime.gradient_norm_device(gl), grads)
    state = runtime.DeviceAdamState(pl)
    with pytest.raises(ValueError, match="differ in shape"):
        runtime.adam_step_device(pl, gl, state)
    grads[0].data = normal((500,), torch.float32, g)
    p[0].data = normal((500,), torch.float32, g)
    was = p[0].detach().clone()
    runtime.adam_step_device(pl, gl, state)
    assert not torch.equal(p[0].detach(), was)


def test_autograd_sees_the_change(runtime):
    p = torch.nn.Parameter(torch.randn(100, device="cuda"))
    loss = (p * p).sum()
    grads = [torch.randn(100, device="cuda")]
    runtime.adam_step_device([p], grads, runtime.DeviceAdamState([p]))
    with pytest.raises(Exception, match="modified by an inplace operation"):
        loss.backward()


def test_streams_and_threads(runtime):
    import threading
    g = gen(71)
    sets = [[normal((n, 1000), torch.float32, g) for n in (30, 70, 1)] for _ in range(4)]
    wants = [ts.norm64(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None] * len(sets)

    def work(k):
        for _ in range(20):
            got[k] = runtime.gradient_norm_device(sets[k], stream=streams[k].cuda_stream)
        streams[k].synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(sets))]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for k, want in enumerate(wants):
        assert abs(float(got[k]) - want) <= ts.norm_bound(count(sets[k])) * want
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        norm = runtime.gradient_norm_device(sets[0])
    s.synchronize()
    assert abs(float(norm) - wants[0]) <= ts.norm_bound(count(sets[0])) * wants[0]
    norm = runtime.gradient_norm_device(sets[0], stream=0)
    torch.cuda.synchronize()
    assert abs(float(norm) - wants[0]) <= ts.norm_bound(count(sets[0])) * wants[0]


def test_captured_steps_count_on(runtime):
    """Two captured steps over their own models, replayed in turn and together."""
    def model(seed):
        g = gen(seed)
        p = [normal((3000,), torch.float32, g), normal((81,), torch.float64, g)]
        q = [normal((3000,), torch.float32, g), normal((81,), torch.float64, g)]
        return p, q, runtime.DeviceAdamState(p)

    def step(p, q, state):
        return runtime.adam_step_device(p, q, state, lr=0.01, weight_decay=0.01, max_norm=1.0)

    models, twins, graphs, norms = [], [], [], []
    for seed in (81, 82):
        models.append(model(seed))
        twins.append(model(seed))
        step(*model(seed))  # loads the kernels
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norms.append(step(*models[-1]))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(6):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (p, q, state), twin, norm in zip(models, twins, norms):
        for _ in range(6):
            want = step(*twin)
        assert int(state.step) == 6 and torch.equal(norm, want)
        assert all(torch.equal(a, b) for a, b in zip(p + state.m + state.v,
                                                     twin[0] + twin[2].m + twin[2].v))


@pytest.mark.parametrize("op", ["norm", "clip", "adam"])
def test_tensors_of_more_than_32_bits_of_elements(runtime, op):
    n = (1 << 32) + 4097
    t = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    t[:3] = 3.0
    t[-2:] = 4.0
    t[1 << 32] = -2.0
    want = math.sqrt(3 * 9 + 2 * 16 + 4)
    if op == "norm":
        assert abs(float(runtime.gradient_norm_device([t])) - want) <= 4 * ts.U64 * want
    elif op == "clip":
        runtime.clip_gradients_device([t], want / 2 * (1 + 1e-6))
        assert t[0] == 1.5 and t[-1] == 2.0 and t[1 << 32] == -1.0 and t[5] == 0.0
    else:
        p = torch.ones(n, dtype=torch.bfloat16, device="cuda")
        runtime.adam_step_device([p], [t], runtime.DeviceAdamState([p]), lr=0.5)
        # the first step moves each parameter with a gradient by lr against its sign
        assert p[0] == 0.5 and p[-1] == 0.5 and p[-2] == 0.5 and p[1 << 32] == 1.5
        assert p[5] == 1.0 and p[(1 << 32) - 1] == 1.0


def test_refusals_on_the_device(runtime):
    a = torch.randn(100, device="cuda")
    with pytest.raises(TypeError, match="without gaps"):
        runtime.gradient_norm_device([a[::2]])
    with pytest.raises(TypeError, match="without gaps"):
        runtime.gradient_norm_device([torch.ones(1, device="cuda").expand(4)])
    with pytest.raises(TypeError, match="place 1"):
        runtime.gradient_norm_device([a, torch.ones(3, dtype=torch.int64, device="cuda")])
    with pytest.raises(TypeError, match="place 0"):
        runtime.gradient_norm_device([torch.ones(3)])
    with pytest.raises(TypeError, match="place 0"):
        runtime.gradient_norm_device([torch.ones(3, dtype=torch.complex64, device="cuda").conj()])
    for two in ([a, a], [a, a[50:]], [a[:60], a[59:]]):
        assert float(runtime.gradient_norm_device(two)) > 0  # read twice is fine
        with pytest.raises(runtime.RuntimeError, match="share memory"):
            runtime.clip_gradients_device(two, 1.0)
    assert float(runtime.clip_gradients_device([a[:60], a[60:]], 1e9)) > 0
    for bad in (-1.0, math.inf, math.nan):
        with pytest.raises((ValueError, runtime.RuntimeError), match="norm must be finite"):
            runtime.clip_gradients_device([a], bad)
        with pytest.raises((ValueError, runtime.RuntimeError), match="norm must be finite"):
            runtime.adam_step_device([a], [a.clone()], runtime.DeviceAdamState([a]), max_norm=bad)
    state = runtime.DeviceAdamState([a])
    before = a.clone()
    for kw, match in [(dict(lr=math.nan), "hyperparameters"), (dict(betas=(1.0, 0.9)), "hyperparameters"),
                      (dict(betas=(0.9, -0.1)), "hyperparameters"), (dict(eps=-1e-8), "hyperparameters"),
                      (dict(weight_decay=math.inf), "hyperparameters"),
                      (dict(norm=torch.ones((), dtype=torch.float64, device="cuda")), "needs max_norm")]:
        with pytest.raises((ValueError, runtime.RuntimeError), match=match):
            runtime.adam_step_device([a], [before.clone()], state, **kw)
    for grads, match in [([], "1 parameters and 0"), ([before[:99].clone()], "differ in shape"),
                         ([before.double()], "f64"), ([before.view(10, 10)], "differ in shape")]:
        with pytest.raises((ValueError, runtime.RuntimeError), match=match):
            runtime.adam_step_device([a], grads, state)
    with pytest.raises(runtime.RuntimeError, match="copy"):
        runtime.adam_step_device([a], [before.clone()], state, copies=[torch.zeros_like(a)])
    with pytest.raises((runtime.RuntimeError, TypeError), match="missing|empty"):
        runtime.adam_step_device([None], [before.clone()], state)
    with pytest.raises(runtime.RuntimeError, match="share memory"):
        runtime.adam_step_device([a, a], [before.clone(), before.clone()],
                                 runtime.DeviceAdamState([a, a]))
    z = torch.zeros(100, device="cuda")
    for m, v in (([z], [z]), ([a], [z]), ([z], [a])):
        with pytest.raises(runtime.RuntimeError, match="share memory"):
            runtime.adam_step_device([a], [before.clone()], runtime.DeviceAdamState([a], m=m, v=v))
    with pytest.raises(ValueError, match="moments"):
        runtime.DeviceAdamState([a], m=[torch.zeros(99, device="cuda")])
    with pytest.raises(runtime.RuntimeError, match="first moment"):
        s = runtime.DeviceAdamState([a], m=[torch.zeros(100, dtype=torch.float64, device="cuda")])
        runtime.adam_step_device([a], [before.clone()], s)
    with pytest.raises(TypeError, match="step count"):
        runtime.DeviceAdamState([a], step=torch.zeros((), device="cuda"))
    assert torch.equal(a, before) and int(state.step) == 0


def test_captured_long_lists(runtime):
    """The launches of a list that takes several, captured and replayed against calls."""
    def model():
        g = gen(91)
        p = [normal((700_001,), torch.float32, g), normal((300_000,), torch.float64, g),
             normal((90_000,), torch.bfloat16, g)]
        return p, [normal(t.shape, t.dtype, g) for t in p], runtime.DeviceAdamState(p)

    def step(p, q, state):
        norm = runtime.clip_gradients_device(q, 50.0)
        return norm, runtime.adam_step_device(p, q, state, lr=0.01, max_norm=1.0)

    a, b = model(), model()
    step(*model())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*a)
    for _ in range(5):
        graph.replay()
    torch.cuda.synchronize()
    for _ in range(5):
        want = step(*b)
    assert int(a[2].step) == 5 and all(torch.equal(x, y) for x, y in zip(got, want))
    assert all(torch.equal(x, y) for x, y in zip(a[0] + a[1] + a[2].m + a[2].v,
                                                 b[0] + b[1] + b[2].m + b[2].v))


@pytest.mark.parametrize("narrow", [100_000, 3_000_000])
def test_mixed_long_lists(runtime, narrow):
    """f64 tensors and others in one launch."""
    g = gen(95)
    params = [normal((400_003,), torch.float64, g), normal((narrow + 1,), torch.float32, g),
              normal((20_001,), torch.bfloat16, g), normal((300, 128), torch.complex128, g)]
    grads = [normal(p.shape, p.dtype, g, 0.1) for p in params]
    run_adam(runtime, params, grads, max_norm=1.0, wd=0.01, steps=2)
    check_norm(runtime.gradient_norm_device(grads), grads)
    run_adam(runtime, params, [None, None] + grads[2:], max_norm=1.0)


def test_a_list_keeps_its_memory(runtime):
    """Memory that a list has written down is not given to another tensor while the list lives, so
    an address that is met again is the same memory."""
    p = torch.nn.Parameter(torch.ones(1 << 20, device="cuda"))
    pl = runtime.TensorList([p])
    at = p.data_ptr()
    p.data = torch.empty(0, device="cuda")  # the parameter's memory would be free now
    others = [torch.empty(1 << 20, device="cuda") for _ in range(4)]
    assert at not in [t.data_ptr() for t in others]
    del others
    p.data = torch.full((1 << 10,), 2.0, device="cuda")
    assert abs(float(runtime.gradient_norm_device(pl)) - 64.0) <= 1e-12  # sqrt(1024 * 4)


def test_copies_of_lists_and_states_are_their_own(runtime):
    import copy
    g = gen(97)
    p, q = [normal((300,), torch.float32, g)], [normal((300,), torch.float32, g)]
    state = runtime.DeviceAdamState(p)
    runtime.adam_step_device(p, q, state)
    other, ql = copy.deepcopy(state), copy.deepcopy(runtime.TensorList(q))
    assert ql.tensors[0].data_ptr() != q[0].data_ptr()
    check_norm(runtime.gradient_norm_device(ql), q)
    p2 = [p[0].clone()]
    for _ in range(3):
        runtime.adam_step_device(p, q, state)
        runtime.adam_step_device(p2, ql, other)
    assert torch.equal(p[0], p2[0]) and torch.equal(state.v[0], other.v[0])
    assert state.v[0].data_ptr() != other.v[0].data_ptr() and int(other.step) == 4
    with pytest.raises(AttributeError):
        state.step = 5


def test_no_momentum(runtime):
    g = gen(98)
    p, q = [normal((3000,), torch.float32, g)], [normal((3000,), torch.float32, g)]
    run_adam(runtime, p, q, betas=(0.0, 0.0), lr=0.1, steps=2)
    run_adam(runtime, p, q, betas=(0.0, 0.999), lr=0.1, eps=1e-3, wd=0.1, max_norm=1.0)


@pytest.mark.parametrize("n", [262_144, 262_145])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_both_sides_of_the_short_list(runtime, dtype, n):
    g = gen(99)
    p, q = [normal((n,), TYPES[dtype], g)], [normal((n,), TYPES[dtype], g)]
    run_adam(runtime, p, q, max_norm=1.0, wd=0.01)
    # 2.5, 4 and 6 MB of gradients, and a little more
    for big in (5 * n // 2, 4 * n, 6 * n):
        t = normal((big,), torch.float32, g)
        check_norm(runtime.gradient_norm_device([t]), [t])
        was, norm = t.clone(), ts.norm64([t])
        runtime.clip_gradients_device([t], 3.0)
        y, bound = ts.clip64(was, ts.clip_factor(norm, 3.0), big)
        ts.assert_within(ts.components(t), y, bound, "clip")


def test_launches_are_counted_and_timed(runtime):
    g = gen(101)
    short, long = [normal((100,), torch.float32, g)], [normal((3_000_000,), torch.float32, g)]
    runtime.gradient_norm_device(long)
    for grads, launches, nbytes in ((short, 1, 400.0), (long, 2, 12e6)):
        before = runtime.launch_count()
        runtime.profile_enable(True)
        runtime.gradient_norm_device(grads)
        other = runtime.profile_read()["other"]
        runtime.profile_enable(False)
        assert runtime.launch_count() - before == launches and other[0] == launches
        assert nbytes <= other[2] <= nbytes + 1e4
