"""Checks of the lookup, orthogonalisation and Muon entry points that need no GPU: every refusal comes before a
CUDA call, so the tables here hold addresses that are never read."""
import ctypes as C
import math

import numpy as np
import pytest
import torch


class Call:
    """Calls the C entry points with host arrays as stand-ins for device memory."""

    def __init__(self, runtime):
        self.rt, self.lib = runtime, runtime.load()
        self.ws = np.zeros(1 << 15, dtype=np.float64)
        at = (-self.ws.ctypes.data // 8) % 2
        self.ws = self.ws[at:]

    def rows(self, data=64, rows=10, width=4, stride=None, dtype=1, reserved=0):
        return self.rt._EMBEDDING_ROWS(data, rows, width, width if stride is None else stride, dtype, reserved)

    def options(self, scale=1.0, padding=-1, normalize=0, index_bytes=8):
        return self.rt._EMBEDDING_OPTIONS(scale, padding, normalize, index_bytes)

    def lookup(self, table=None, indices=64, count=3, options=None, output=None, ws=True, words=None):
        return self.lib.arcqml_rt_v2_embedding_lookup(
            table or self.rows(), indices, count, options or self.options(), output or self.rows(rows=count),
            self.ws.ctypes.data if ws else None, self.ws.size if words is None else words, None)

    def gradient(self, gradient=None, indices=64, options=None, table=None, output=None, ws=True, words=None):
        return self.lib.arcqml_rt_v2_embedding_gradient(
            gradient or self.rows(rows=3), indices, options or self.options(), table, output or self.rows(),
            self.ws.ctypes.data if ws else None, self.ws.size if words is None else words, None)

    def matrices(self, *rows):
        t = np.zeros(max(1, len(rows)), dtype=self.rt._MATRIX)
        for i, r in enumerate(rows):
            t[i] = r
        return t

    def orthogonalize(self, x, y=None, n=None, steps=5, eps=1e-7, ws=True, words=None):
        y = x if y is None else y
        return self.lib.arcqml_rt_v2_orthogonalize(
            None if x is None else x.ctypes.data, None if y is None else y.ctypes.data, len(x) if n is None else n,
            steps, eps, self.ws.ctypes.data if ws else None, self.ws.size if words is None else words, None)

    def muon(self, p, g, m, options=(0.02, 0.95, 0.0, 1e-7, 1, 5), ws=True):
        o = None if options is None else self.rt.MuonOptions(*options)
        return self.lib.arcqml_rt_v2_muon_step(
            p.ctypes.data, g.ctypes.data, m.ctypes.data, len(p), None if o is None else C.byref(o),
            self.ws.ctypes.data if ws else None, self.ws.size, None)

    def message(self, status, match):
        assert status == 1
        assert match in self.rt.last_error(), self.rt.last_error()


@pytest.fixture
def call(runtime):
    return Call(runtime)


@pytest.mark.parametrize("entry", ["lookup", "gradient"])
def test_malformed_rows_and_options(call, entry):
    run = getattr(call, entry)
    name = {"lookup": "table", "gradient": "gradient"}[entry]
    n = 10 if entry == "lookup" else 3
    for bad, match in ((dict(dtype=4), "unknown type"), (dict(reserved=1), "reserved"), (dict(rows=1 << 31), "too many rows"),
                       (dict(width=0), "without elements"), (dict(width=1 << 30), "too long"),
                       (dict(stride=1 << 40), "too far apart"), (dict(data=0), "is null"), (dict(data=66), "not aligned")):
        call.message(run(**{name: call.rows(**{"rows": n, **bad})}), f"the embedding's {name}")
        assert match in call.rt.last_error(), call.rt.last_error()
    for scale in (math.nan, math.inf):
        call.message(run(options=call.options(scale=scale)), "scale must be finite")
    call.message(run(options=call.options(normalize=2)), "normalize is 0 or 1")
    call.message(run(options=call.options(index_bytes=2)), "4 or 8 bytes")
    call.message(run(indices=0), "indices are null")
    call.message(run(indices=68), "indices are not aligned")
    wrong = [dict(dtype=2), dict(width=5), dict(stride=8)] + ([dict(rows=4)] if entry == "lookup" else [])
    for bad in wrong:
        call.message(run(output=call.rows(**{"rows": 3, **bad})), "output")
    for null in range(2):
        args = [call.rows(), call.options(), call.rows(rows=3)]
        args[2 * null] = None
        call.message(call.lib.arcqml_rt_v2_embedding_lookup(args[0], 64, 3, args[1], args[2], None, 0, None), "null")
    call.message(call.lib.arcqml_rt_v2_embedding_gradient(call.rows(), 64, None, None, call.rows(), None, 0, None),
                 "options are null")


def test_lookup_counts_and_scratch(call):
    call.message(call.lookup(count=1 << 31, output=call.rows(rows=1)), "too many")
    wide = call.rows(width=40_000)
    need = call.lib.arcqml_rt_v2_embedding_lookup_workspace(wide, 3, call.options(normalize=1))
    assert need > 0
    assert call.lib.arcqml_rt_v2_embedding_lookup_workspace(wide, 3, call.options()) == 0
    for ws, words, match in ((False, None, "workspace is null"), (True, need - 1, "too small")):
        call.message(call.lookup(table=wide, output=call.rows(rows=3, width=40_000), options=call.options(normalize=1),
                                 ws=ws, words=words), match)


def test_gradient_tables_and_scratch(call):
    normal = call.options(normalize=1)
    call.message(call.gradient(options=normal), "table is null")
    call.message(call.gradient(table=call.rows()), "not normalised")
    for bad in (dict(rows=9), dict(width=5), dict(dtype=2)):
        call.message(call.gradient(options=normal, table=call.rows(**bad)), "type and shape")
    many = call.rows(rows=5000)
    need = call.lib.arcqml_rt_v2_embedding_gradient_workspace(many, 10, call.options())
    assert need > 0 and call.lib.arcqml_rt_v2_embedding_gradient_workspace(call.rows(), 10, call.options()) == 0
    for ws, words, match in ((False, None, "workspace is null"), (True, need - 1, "too small")):
        call.message(call.gradient(gradient=many, ws=ws, words=words), match)


def test_malformed_matrices(call):
    ok = (64, 4, 5, 1, 0)
    call.message(call.orthogonalize(None, n=2), "input list is null")
    for bad, match in (((64, 4, 5, 0, 0), "f64"), ((64, 4, 5, 5, 0), "unknown type"), ((64, 4, 5, 1, 1), "reserved"),
                       ((64, 1 << 24, 5, 1, 0), "too large"), ((64, 1 << 20, 1 << 20, 1, 0), "too large"),
                       ((0, 4, 5, 1, 0), "is null"), ((66, 4, 5, 1, 0), "not aligned")):
        call.message(call.orthogonalize(call.matrices(ok, bad)), "input matrix 1")
        assert match in call.rt.last_error()
    for steps in (0, -1, 21):
        call.message(call.orthogonalize(call.matrices(ok), steps=steps), "1 to 20")
    for eps in (-1e-9, math.nan, math.inf):
        call.message(call.orthogonalize(call.matrices(ok), eps=eps), "epsilon")
    for other in ((64, 5, 4, 1, 0), (64, 4, 5, 2, 0), (0, 0, 0, 4, 0)):
        call.message(call.orthogonalize(call.matrices(ok), call.matrices(other)), "output matrix 0 differs")
    large = call.matrices((64, 300, 500, 1, 0))
    need = call.lib.arcqml_rt_v2_orthogonalize_workspace(large.ctypes.data, 1)
    small = call.matrices(ok)
    assert need > 0 and call.lib.arcqml_rt_v2_orthogonalize_workspace(small.ctypes.data, 1) == 0
    call.message(call.orthogonalize(large, ws=False), "workspace is null")
    call.message(call.orthogonalize(large, words=100), "too small")
    assert call.lib.arcqml_rt_v2_orthogonalize(None, None, 0, 5, 1e-7, None, 0, None) == 0


def test_muon_lists_that_do_not_match(call):
    p, none = (64, 4, 5, 2, 0), (0, 0, 0, 4, 0)
    m = (128, 4, 5, 1, 0)
    call.message(call.muon(call.matrices(none), call.matrices(p), call.matrices(m)), "parameter matrix 0 is missing")
    call.message(call.muon(call.matrices(p), call.matrices((64, 5, 4, 2, 0)), call.matrices(m)), "gradient matrix 0 differs")
    for bad in ((128, 4, 5, 2, 0), (128, 5, 4, 1, 0), none):
        call.message(call.muon(call.matrices(p), call.matrices(p), call.matrices(bad)), "momentum matrix 0")
    for bad in ((math.nan, 0.9, 0, 1e-7, 1, 5), (0.1, 1.0, 0, 1e-7, 1, 5), (0.1, -0.1, 0, 1e-7, 1, 5),
                (0.1, 0.9, math.inf, 1e-7, 1, 5), (0.1, 0.9, 0, 1e-7, 2, 5)):
        call.message(call.muon(call.matrices(p), call.matrices(p), call.matrices(m), bad), "invalid Muon")
    call.message(call.muon(call.matrices(p), call.matrices(p), call.matrices(m), (0.1, 0.9, 0, 1e-7, 1, 0)), "1 to 20")
    call.message(call.muon(call.matrices(p), call.matrices(p), call.matrices(m), None), "options are null")
    # nothing to do: no gradient
    assert call.muon(call.matrices(p), call.matrices(none), call.matrices(none), ws=False) == 0


def test_scratch_of_a_list_bounds_that_of_its_parts(call):
    """Launches take what fits into the scratch; a list without some of its gradients needs no more."""
    rng = np.random.default_rng(5)
    lib = call.lib
    for _ in range(20):
        rows = [(64, int(rng.integers(1, 9000)), int(rng.integers(1, 9000)), int(rng.integers(1, 4)), 0)
                for _ in range(int(rng.integers(1, 90)))]
        full = call.matrices(*rows)
        each = [lib.arcqml_rt_v2_orthogonalize_workspace(call.matrices(r).ctypes.data, 1) for r in rows]
        assert lib.arcqml_rt_v2_orthogonalize_workspace(full.ctypes.data, len(rows)) >= max(each)


def test_host_tensors_are_refused(runtime):
    from arcqml_b200.optim import Muon
    x = torch.zeros(4, 5)
    for make in (lambda: runtime.TensorList([x]), lambda: runtime.orthogonalize_device([x]), lambda: Muon([x]),
                 lambda: runtime.DeviceMuonState([x])):
        with pytest.raises(TypeError):
            make()


# ------------------------------------------------------------------ who takes which tile


def cuts(classes, units, parts):
    """The kernels' shares of the tiles left over, restated: (runs per unit, steps left, tiles with a cut)."""
    left = [0]
    for has, depth in classes:
        left.append(left[-1] + has % units * max(16, depth))
    total = left[-1]
    snap = 8 if parts else 1 << 40
    runs = max(1, min(units, total // max(16, (classes[0][1] + 5) // 6))) if parts else units

    def cut(u):
        if u >= runs:
            return total
        at = u * total // runs
        if at == 0:
            return 0
        c = max(i for i in range(len(classes)) if left[i] <= at)
        depth = classes[c][1]
        w = max(16, depth)
        past = (at - left[c]) % w
        if past < snap and past < w - past:
            return at - past
        return at + w - past if past < snap or past + snap > depth else at

    return [cut(u) for u in range(units + 1)], left


@pytest.mark.parametrize("seed", range(8))
def test_every_step_of_every_tile_is_taken_once(seed):
    rng = np.random.default_rng(seed)
    for _ in range(150):
        units = int(rng.choice([74, 148]))
        depths = sorted(rng.choice(np.arange(1, 140), int(rng.integers(1, 6)), replace=False).tolist(), reverse=True)
        classes = [(int(rng.choice([1, 2, 3, 10, 36, 136, 300])), int(d)) for d in depths]
        parts = bool(rng.integers(2))
        bounds, left = cuts(classes, units, parts)
        assert bounds == sorted(bounds) and bounds[0] == 0 and bounds[-1] == left[-1]
        for c, (has, depth) in enumerate(classes):
            w = max(16, depth)
            for k in range(has % units):
                start = left[c] + k * w
                inner = [b for b in bounds if start < b < start + w]
                assert all(b - start < depth for b in inner)
                assert parts or not inner
                # parts: of 8 steps or more, and no more than the slots of a unit can hold (its first and last)
                edges = sorted({0, *[b - start for b in inner], depth})
                assert all(b - a >= min(8, depth) for a, b in zip(edges, edges[1:])), (edges, depth)
                assert len(edges) - 1 <= 14
