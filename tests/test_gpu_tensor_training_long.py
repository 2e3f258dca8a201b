"""The tensor operators over lists that take several launches, at the offsets, given norms, values,
streams and captured graphs that the short lists are tested with, against 64 bits (needs a B200).

Every list of parameters here is asserted to need scratch, which a list of one launch does not."""
import math
import threading

import numpy as np
import pytest
import torch

import tensor_training_support as ts
from test_gpu_tensor_training import TYPES, check_norm, count, gen, normal, run_adam, views

pytestmark = pytest.mark.gpu

# few tensors that are large, and more than one launch takes at once of short ones
LENGTHS = {"large": [1, 6, 8191, 3, 800_003], "many": [1 + (i * 61) % 7001 for i in range(130)]}


def assert_long(runtime, params, grads=()):
    assert runtime.TensorList(params)._adam_words > 0
    for g in grads:
        assert runtime.TensorList(g)._words > 0


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("offsets", [(0, 0), (0, 1), (1, 0), (1, 1), (3, 3), (3, 2), (5, 1)])
@pytest.mark.parametrize("types", [("f64", "f64"), ("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"),
                                   ("f32", "f16")], ids=lambda m: "-".join(m))
def test_views_at_any_offset(runtime, types, offsets, lengths):
    g = gen(31)
    lengths = LENGTHS[lengths]
    flat_p, params = views(lengths, TYPES[types[0]], g, offsets[0])
    flat_g, grads = views(lengths, TYPES[types[1]], g, offsets[1])
    copies, flat_c = None, torch.zeros(0, device="cuda")
    if types[0] == "f32" and types[1] != "f32":
        flat_c, copies = views(lengths, TYPES[types[1]], g, offsets[1])
    assert_long(runtime, params)
    ends = [(f[:o].clone(), f[-1:].clone()) for f, o in ((flat_p, offsets[0]), (flat_c, offsets[1]))]
    kept = flat_g.clone()
    run_adam(runtime, params, grads, max_norm=1.0, wd=0.02, copies=copies)
    # moments that start elsewhere in their vectors, copies at some places only
    wide = TYPES[types[0]] if types[0] == "f64" else torch.float32
    flat_m, m = views(lengths, wide, g, 2, 0.1)
    flat_v, v = views(lengths, wide, g, 1, 0.1)
    flat_v.abs_()
    ends += [(f[:o].clone(), f[-1:].clone()) for f, o in ((flat_m, 2), (flat_v, 1))]
    if copies:
        copies[1::2] = [None] * len(copies[1::2])
    run_adam(runtime, params, grads, m=m, v=v, step=7, copies=copies, decoupled=True, wd=0.1)
    for (first, last), flat in zip(ends, (flat_p, flat_c, flat_m, flat_v)):
        assert torch.equal(flat[:len(first)], first) and torch.equal(flat[-1:], last)
    assert torch.equal(flat_g, kept)


def test_strides_empty_places_and_missing_gradients(runtime):
    g = gen(41)
    params = [normal((800, 512), torch.float32, g).t(), normal((81,), torch.float64, g),
              torch.empty((0, 3), device="cuda"), normal((3, 1024), torch.complex128, g),
              normal((7, 3), torch.float32, g), normal((90_001,), torch.bfloat16, g)]
    grads = [normal((800, 512), torch.float16, g).t()] + [normal(p.shape, p.dtype, g) for p in params[1:]]
    grads[4] = None
    copies = [torch.zeros((800, 512), dtype=torch.float16, device="cuda").t(), None,
              torch.empty((0, 3), dtype=torch.bfloat16, device="cuda"), None,
              torch.zeros((7, 3), dtype=torch.bfloat16, device="cuda"), None]
    assert_long(runtime, params)
    copies_kept = copies[4].clone()
    # a place without a gradient has its copy left alone as well: it is compared by itself
    state = runtime.DeviceAdamState(params)
    old = [ts.components(x[4]) for x in (params, state.m, state.v)]
    runtime.adam_step_device(params, grads, state, max_norm=0.1, copies=copies)
    assert all(np.array_equal(ts.components(x[4]), o) for x, o in zip((params, state.m, state.v), old))
    assert torch.equal(copies[4], copies_kept) and torch.equal(copies[0], params[0].to(torch.float16))
    run_adam(runtime, params, grads, max_norm=0.1, wd=0.01, copies=copies[:4] + [None] * 2, steps=2)
    run_adam(runtime, params, [None] * 6, max_norm=1.0)
    assert int(state.step) == 1


@pytest.mark.parametrize("lengths", LENGTHS)
def test_given_norm(runtime, lengths):
    """The launches without a sum before them."""
    g = gen(51)
    for p_type, g_type in (("f32", "f32"), ("f64", "f64"), ("f32", "bf16")):
        params = [normal((n,), TYPES[p_type], g) for n in LENGTHS[lengths]]
        grads = [normal((n,), TYPES[g_type], g) for n in LENGTHS[lengths]]
        assert_long(runtime, params, [grads] if lengths == "many" or g_type != "bf16" else [])
        norm = torch.tensor(50.0, dtype=torch.float64, device="cuda")
        run_adam(runtime, params, grads, max_norm=0.5, norm=norm, steps=2)
        was = [t.clone() for t in grads]
        out = runtime.clip_gradients_device(grads, 5.0, norm=norm)
        assert float(out) == 50.0
        for a, b in zip(grads, was):
            y, bound = ts.clip64(b, 5.0 / (50.0 + 1e-6), 1)
            ts.assert_within(ts.components(a), y, bound, (g_type, "clip"))
        # a norm that keeps the gradients as they are
        was = [t.clone() for t in grads]
        runtime.clip_gradients_device(grads, 60.0, norm=norm)
        assert all(torch.equal(a, b) for a, b in zip(grads, was))


@pytest.mark.parametrize("dtype", ["f64", "f32", "bf16", "f16"])
@pytest.mark.parametrize("place", [0, 1_000_001, 2_999_999])
def test_infinities_and_nan(runtime, dtype, place):
    kind = TYPES[dtype]
    other_kind = torch.float64 if dtype == "f64" else torch.float32
    for bad in (math.inf, -math.inf, math.nan):
        t, other = normal((3_000_000,), kind, gen(3)), normal((77,), other_kind, gen(4))
        t[place] = bad
        params = [normal((3_000_000,), kind, gen(5)), normal((77,), other_kind, gen(6))]
        assert_long(runtime, params, [[t, other]])
        was = [p.clone() for p in params]
        # without clipping the bad element alone is lost
        plain = [p.clone() for p in params]
        runtime.adam_step_device(plain, [t, other], runtime.DeviceAdamState(plain))
        assert bool(plain[0][place].isnan()) and int(plain[0].isnan().sum()) == 1
        assert not bool(plain[1].isnan().any())
        norm = runtime.adam_step_device(params, [t, other], runtime.DeviceAdamState(params), max_norm=1.0)
        clip = runtime.clip_gradients_device([t, other], 1.0)
        if math.isnan(bad):
            assert math.isnan(float(norm)) and math.isnan(float(clip))
            assert all(bool(x.isnan().all()) for x in params + [t, other])
        else:  # the factor is 0, and infinity times 0 is NaN
            assert float(norm) == math.inf and float(clip) == math.inf
            assert bool(params[0][place].isnan()) and int(params[0].isnan().sum()) == 1
            was[0][place] = params[0][place] = 0.0
            assert all(torch.equal(a, b) for a, b in zip(params, was))
            assert bool(other.eq(0).all()) and bool(t[place].isnan()) and int(t.isnan().sum()) == 1
            assert bool(t.nan_to_num(0.0).eq(0).all())


def model(seed):
    """More tensors than the smallest table holds, of all types, their gradients and state."""
    g = gen(seed)
    p = [normal((400_003,), torch.float32, g), normal((150_001,), torch.float64, g),
         normal((90_000,), torch.bfloat16, g)] + [normal((n,), torch.float32, g) for n in range(1, 70)]
    q = [normal((n.numel(),), n.dtype, g) for n in p]
    return p, q, runtime_state(p)


def runtime_state(p):
    from arcqml_b200 import runtime as rt
    assert_long(rt, p)
    return rt.DeviceAdamState(p)


def step(runtime, p, q, state, stream=None):
    """The norm by itself, clipping, and a step that clips again: every kind of launch and its scratch."""
    first = runtime.gradient_norm_device(q, stream=stream)
    clipped = runtime.clip_gradients_device(q, 300.0, stream=stream)
    return [first, clipped, runtime.adam_step_device(p, q, state, lr=0.01, weight_decay=0.01, max_norm=1.0,
                                                     stream=stream)]


def assert_equal_models(got, want, norms, want_norms):
    for a, b in zip(got[0] + got[1] + got[2].m + got[2].v + norms,
                    want[0] + want[1] + want[2].m + want[2].v + want_norms):
        assert torch.equal(a, b)


def test_streams_and_threads(runtime):
    """Calls that overlap have scratch of their own."""
    models, twins = [model(s) for s in (71, 72, 73, 74)], [model(s) for s in (71, 72, 73, 74)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in models]
    got, errors = [None] * len(models), []

    def work(k):
        try:
            for i in range(12):
                # by the argument and by the current stream
                if i % 2:
                    got[k] = step(runtime, *models[k], stream=streams[k].cuda_stream)
                else:
                    with torch.cuda.stream(streams[k]):
                        got[k] = step(runtime, *models[k])
            streams[k].synchronize()
        except Exception as e:  # raised in the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(models))]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors
    for mine, twin, norms in zip(models, twins, got):
        for _ in range(12):
            want = step(runtime, *twin)
        assert int(mine[2].step) == 12
        assert_equal_models(mine, twin, norms, want)


def test_captured_graphs_replayed_together(runtime):
    models, twins, graphs, norms = [], [], [], []
    step(runtime, *model(80))  # loads the kernels
    for seed in (81, 82):
        models.append(model(seed))
        twins.append(model(seed))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norms.append(step(runtime, *models[-1]))
        graphs.append(graph)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(8):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for mine, twin, got in zip(models, twins, norms):
        for _ in range(8):
            want = step(runtime, *twin)
        assert int(mine[2].step) == 8
        assert_equal_models(mine, twin, got, want)


def test_16_bit_buckets_of_many_tensors(runtime):
    """Gradients without gaps at odd offsets, copies on their own: what a network in 16 bits keeps."""
    g = gen(91)
    lengths = [3 + (i * 7919) % 20_011 for i in range(200)]
    for grad in ("bf16", "f16"):
        params = [normal((n,), torch.float32, g) for n in lengths]
        _, grads = views(lengths, TYPES[grad], g, 1)
        copies = [torch.zeros(n, dtype=TYPES[grad], device="cuda") for n in lengths]
        assert_long(runtime, params, [grads])
        check_norm(runtime.gradient_norm_device(grads), grads)
        run_adam(runtime, params, grads, max_norm=1.0, wd=0.1, decoupled=True, copies=copies, steps=2)
        assert count(grads) == sum(lengths)
