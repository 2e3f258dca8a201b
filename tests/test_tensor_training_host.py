"""Checks of the gradient norm, clipping and Adam step entry points that need no GPU: every refusal
comes before a CUDA call, so the tables here hold addresses that are never read."""
import ctypes as C

import numpy as np
import pytest
import torch


def table(runtime, *rows):
    t = np.zeros(max(1, len(rows)), dtype=runtime._TENSOR)
    for i, r in enumerate(rows):
        t[i] = r
    return t


class Call:
    """Calls the C entry points with host arrays as stand-ins for device memory."""

    def __init__(self, runtime):
        self.rt, self.lib = runtime, runtime.load()
        self.ws = np.zeros(1 << 15, dtype=np.float64)
        at = (-self.ws.ctypes.data // 8) % 2
        self.ws = self.ws[at:]
        self.norm = np.zeros(1)
        self.step = np.zeros(1, dtype=np.int64)

    def norm_of(self, t, n=None, norm=True, ws=True, words=None):
        return self.lib.arcqml_rt_v2_gradient_norm(
            None if t is None else t.ctypes.data, len(t) if n is None else n,
            self.norm.ctypes.data if norm else None, self.ws.ctypes.data if ws else None,
            self.ws.size if words is None else words, None)

    def clip(self, t, max_norm):
        return self.lib.arcqml_rt_v2_clip_gradients(t.ctypes.data, len(t), max_norm, None, None,
                                                    self.ws.ctypes.data, self.ws.size, None)

    def adam(self, p, g, m, v, copies=None, step=True, options=(1e-3, .9, .999, 1e-8, 0., -1., 0, 0)):
        o = None if options is None else self.rt.AdamOptions(*options)
        at = lambda x: None if x is None else x.ctypes.data  # noqa: E731
        return self.lib.arcqml_rt_v2_adam_step(
            at(p), at(g), at(m), at(v), at(copies), 1, self.step.ctypes.data if step else None,
            None if o is None else C.byref(o), None, None, self.ws.ctypes.data, self.ws.size, None)

    def message(self, status, match):
        assert status == 1
        assert match in self.rt.last_error(), self.rt.last_error()


@pytest.fixture
def call(runtime):
    return Call(runtime)


def test_malformed_lists(runtime, call):
    ok = (64, 10, 1, 0)
    call.message(call.norm_of(None, n=2), "gradient list is null")
    call.message(call.norm_of(table(runtime, ok, (64, 10, 5, 0))), "gradient tensor 1 has an unknown type")
    call.message(call.norm_of(table(runtime, (64, 10, 1, 7))), "reserved")
    call.message(call.norm_of(table(runtime, (0, 10, 1, 0))), "gradient tensor 0 is null")
    for address, dtype in ((66, 1), (68, 0), (65, 2), (65, 3)):
        call.message(call.norm_of(table(runtime, (address, 10, dtype, 0))), "not aligned")
    call.message(call.norm_of(table(runtime, (64, 1 << 41, 1, 0))), "too long")
    call.message(call.norm_of(table(runtime, *[(64, (1 << 40) - 1, 1, 0)] * 40)), "too many elements")
    call.message(call.norm_of(table(runtime, ok), norm=False), "norm pointer is null")
    # a list that one launch does not take needs scratch
    for long in (table(runtime, *[ok] * 2000), table(runtime, (64, 1 << 30, 1, 0))):
        need = runtime.load().arcqml_rt_v2_gradient_workspace(long.ctypes.data, len(long))
        assert need > 0
        call.message(call.norm_of(long, ws=False), "workspace is null")
        call.message(call.norm_of(long, words=need - 1), "too small")
    assert runtime.load().arcqml_rt_v2_gradient_workspace(table(runtime, ok).ctypes.data, 1) == 0
    call.message(call.clip(table(runtime, ok), -1.0), "finite and not negative")
    call.message(call.clip(table(runtime, ok), float("nan")), "finite and not negative")
    call.message(call.clip(table(runtime, ok), float("inf")), "finite and not negative")


def test_adam_lists_that_do_not_match(runtime, call):
    p = table(runtime, (64, 10, 2, 0))
    g = table(runtime, (128, 10, 2, 0))
    m = table(runtime, (256, 10, 1, 0))
    f64 = table(runtime, (256, 10, 0, 0))
    none = table(runtime, (0, 0, 4, 0))
    short = table(runtime, (128, 9, 2, 0))
    call.message(call.adam(None, g, m, m), "parameter list is null")
    call.message(call.adam(p, None, m, m), "gradient list is null")
    call.message(call.adam(p, g, None, m), "first moment list is null")
    call.message(call.adam(p, g, m, None), "second moment list is null")
    call.message(call.adam(none, g, m, m), "parameter tensor 0 is missing")
    call.message(call.adam(p, short, m, m), "differs in length")
    call.message(call.adam(p, f64, m, m), "gradient tensor 0 is f64")
    call.message(call.adam(f64, g, f64, f64), "gradient tensor 0 is f64")
    call.message(call.adam(p, g, f64, m), "first moment tensor 0 differs")
    call.message(call.adam(p, g, m, g), "second moment tensor 0 differs")
    call.message(call.adam(p, g, m, none), "second moment tensor 0 differs")
    call.message(call.adam(p, g, m, m, copies=g), "copy tensor 0 is not a 16-bit copy")
    call.message(call.adam(m, m, m, m, copies=m), "copy tensor 0 is not a 16-bit copy")
    call.message(call.adam(m, m, m, m, copies=short), "copy tensor 0 differs in length")
    call.message(call.adam(p, g, m, m, step=False), "step counter is null")
    call.message(call.adam(p, g, m, m, options=None), "options are null")
    good = [1e-3, .9, .999, 1e-8, 0., -1., 0, 0]
    for i, bad in ((0, float("inf")), (1, 1.0), (1, -0.1), (1, float("nan")), (2, 1.0), (3, -1.0),
                   (4, float("nan"))):
        o = list(good)
        o[i] = bad
        call.message(call.adam(p, g, m, m, options=o), "invalid Adam hyperparameters")
    for i, bad in ((6, 2), (7, 1)):
        o = list(good)
        o[i] = bad
        call.message(call.adam(p, g, m, m, options=o), "invalid Adam options")
    for bad in (float("nan"), float("inf"), -float("inf")):
        o = list(good)
        o[5] = bad
        call.message(call.adam(p, g, m, m, options=o), "maximum norm must be finite")
    assert call.step[0] == 0


def test_table_layout_matches_the_header(runtime, tmp_path):
    import os
    import subprocess
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    src = tmp_path / "probe.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "arcqml_runtime_v2.h"\n'
                   'int main(void) { printf("%zu %zu %zu %zu %zu %zu %d\\n", sizeof(ArcqmlTensor), '
                   'offsetof(ArcqmlTensor, length), offsetof(ArcqmlTensor, dtype), '
                   'sizeof(ArcqmlAdamOptions), offsetof(ArcqmlAdamOptions, max_norm), '
                   'offsetof(ArcqmlAdamOptions, decoupled), ARCQML_NO_TENSOR); return 0; }\n')
    exe = tmp_path / "probe"
    subprocess.run(["/usr/bin/gcc", "-I", include, str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()]
    t, o = runtime._TENSOR, runtime.AdamOptions
    assert got == [t.itemsize, t.fields["length"][1], t.fields["dtype"][1], C.sizeof(o),
                   o.max_norm.offset, o.decoupled.offset, runtime.NO_TENSOR]


def test_lists_refuse_what_is_not_on_the_device(runtime):
    for bad in (torch.ones(3), np.ones(3), 1.0):
        with pytest.raises(TypeError, match="place 0"):
            runtime.TensorList([bad])
    assert len(runtime.TensorList([])) == 0 and len(runtime.TensorList([None])) == 1


def test_layouts(runtime):
    x = torch.zeros(4, 5, 6)
    assert runtime._layout(x) is None and runtime._layout(torch.zeros(())) is None
    assert runtime._layout(x.permute(2, 0, 1)) == ((6, 1), (4, 30), (5, 6))
    assert runtime._layout(x[:, :1].permute(2, 0, 1)[:, :1]) is None  # one row of 6
    assert runtime._layout(torch.zeros(0, 3)) is None
    for bad in (x[:, ::2], x[:, :, 1:], x[1:, 1:], torch.zeros(1).expand(3),
                torch.zeros(10).as_strided((3, 3), (1, 1)), x.permute(2, 0, 1)[:, ::2]):
        with pytest.raises(TypeError, match="without gaps"):
            runtime._layout(bad)


def test_shared_memory_is_found(runtime):
    apart = runtime._spans_apart
    assert apart([]) and apart([(64, 80)]) and apart([(80, 96), (64, 80)])
    assert not apart([(76, 92), (64, 80)]) and not apart([(64, 80), (64, 80)])
    assert not apart([(64, 200), (70, 80), (200, 300)])


def test_hybrid_optimizer_refusals(runtime):
    from arcqml_b200 import Circuit
    from arcqml_b200.optim import Adam
    c = Circuit(2)
    c.append("ry", (0,), c.add_parameter(0.5, requires_grad=False))
    for bad in (dict(), dict(circuits=[c]), dict(circuits=[Circuit(1)])):
        with pytest.raises(ValueError, match="nothing to train"):
            Adam(**bad)
    c.append("ry", (1,), c.add_parameter(0.5))
    with pytest.raises(ValueError, match="trained once"):
        Adam([c, c])
    with pytest.raises(TypeError, match="must not be None"):
        Adam([c], [None])
    with pytest.raises(TypeError, match="place 0"):
        Adam([c], [torch.ones(3)])


def test_hybrid_optimizer_takes_no_computed_tensors(runtime):
    """Their gradients go to the tensors that they were computed from: they would never move."""
    from arcqml_b200.optim import Adam
    w = torch.ones(4, 3, requires_grad=True)
    for bad in ([2 * w], w.unbind(), [w[0]], [torch.ones(2), w.t()]):
        with pytest.raises(ValueError, match="computed from others"):
            Adam(tensors=bad)
    # what keeps its gradient, and one tensor by itself, get as far as the check of the device
    kept = 2 * w
    kept.retain_grad()
    for tensors in ([kept], w):
        with pytest.raises(TypeError, match="place 0"):
            Adam(tensors=tensors)


def test_what_is_read_lies_outside_what_is_written(runtime):
    def outside(name, spans, taken, of):
        runtime._check_outside(name, spans, runtime._edges(taken), of)

    taken = [(64, 80), (80, 96), (128, 200), (1000, 1001)]
    for free in ([], [(0, 64)], [(96, 128)], [(200, 300), (96, 100), (96, 100)], [(1001, 1 << 62)]):
        outside("a", free, taken, "b")
        outside("a", free, [], "b")
    for bad in ((0, 65), (64, 80), (79, 81), (95, 96), (95, 300), (127, 129), (130, 140), (199, 1000),
                (0, 2000), (1000, 1001)):
        with pytest.raises(runtime.RuntimeError, match="a shares memory with b"):
            outside("a", [(96, 128), bad], taken, "b")


def test_conjugated_gradients(runtime):
    """Autograd leaves the gradient of a conjugated leaf with its conj bit set, unless it has to copy it
    into the leaf's strides. Lists name the bit; the optimizer resolves it, in the gradient's strides."""
    from arcqml_b200.optim import _resolved
    for shape, order, lazy in (((5,), (0,), True), ((3, 4), (0, 1), True), ((3, 4), (1, 0), False)):
        g = torch.Generator().manual_seed(3)
        x = torch.randn(shape, dtype=torch.complex128, generator=g).permute(order)
        y = torch.randn(x.shape, dtype=torch.complex128, generator=g)
        x.requires_grad_(True)
        (x.conj() * y).real.sum().backward()
        assert x.grad.is_conj() == lazy and x.grad.stride() == x.stride()
        if lazy:
            with pytest.raises(TypeError, match="torch.complex128 on cpu with its lazy conj bit"):
                runtime.TensorList([x.grad])
        z = _resolved(x.grad)
        assert not z.is_conj() and z.stride() == x.grad.stride()
        # d Re(conj(x) y) / d conj(x), doubled: y
        assert torch.equal(z, y)
        assert _resolved(z) is z
    z = _resolved(y.mH)
    assert not z.is_conj() and z.stride() == y.mH.stride() and torch.equal(z, y.mH)
    neg = torch.ones(3, dtype=torch.complex64).conj().imag
    assert neg.is_neg() and not _resolved(neg).is_neg()
    with pytest.raises(TypeError, match="lazy neg bit"):
        runtime.TensorList([neg])
    assert _resolved(None) is None
    with pytest.raises(TypeError, match="laid out as torch.sparse_coo"):
        runtime.TensorList([torch.eye(3).to_sparse()])
