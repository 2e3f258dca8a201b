"""Work over the tensors of a hybrid model: the global norm of its gradients, clipping by that norm,
and the Adam step with the clip factor folded in.

A case's tensors are up to three parts, as a model that feeds a circuit has them:
  weights   `tensors` tensors of `dtype` with `elements` elements in all, of uneven sizes (`layout` seeds
            the sizes); with `packed` the gradients are views of one buffer without gaps (as a
            bucket of an all-reduce holds them: odd offsets), else each starts on its own 512 bytes
  circuit   `circuit` float64 circuit parameters in one tensor
  states    a [`rows`, 2^`qubits`] complex128 tensor: amplitudes, or their gradient
"""
import math
import random

import torch

own = False

BETAS = (0.9, 0.999)
EPS = 1e-8
TYPES = {"float64": torch.float64, "float32": torch.float32, "bfloat16": torch.bfloat16,
         "float16": torch.float16}
STEPS_TAKEN = 99


def _case(name, op, dtype="", tensors=0, elements=0, layout=0, packed=False, circuit=0, rows=0,
          qubits=0, **more):
    return dict({"name": name} if name else {}, op=op, dtype=dtype, tensors=tensors,
                elements=elements, layout=layout, packed=packed, circuit=circuit, rows=rows,
                qubits=qubits, **more)


def _adam(clip, decoupled, grad="", copy=False, decay=0.01):
    """`clip`: the maximum norm (0: none); `grad`: the weights' gradient type where it is not the
    weights' own; `copy`: a copy of the updated weights in the gradients' type."""
    return {"max_norm": clip, "decoupled": decoupled, "grad": grad, "copy": copy, "lr": 1e-3,
            "decay": decay}


def listed():
    return [
        # the gradient of the 4-qubit VQE's 8 parameters: a call's latency
        _case("norm_circuit_8", "norm", circuit=8),
        # the batched QNN: 80 circuit parameters, a small encoder, the gradient of 1024 10-qubit states
        _case("norm_hybrid", "norm", "float32", 6, 42_017, 1, circuit=80, rows=1024, qubits=10),
        # the gradient of one 28-qubit state (4 GB)
        _case("norm_state_28q", "norm", rows=1, qubits=28),
        # a large classical half, its gradients in one all-reduce bucket
        _case("norm_bf16_packed", "norm", "bfloat16", 300, 251_000_003, 2, packed=True),
        # a small encoder's gradients
        _case("clip_encoder", "clip", "float32", 8, 42_017, 3, max_norm=2.0),
        # many short tensors: launches and bookkeeping
        _case("clip_many_short", "clip", "float32", 600, 1_300_001, 4, max_norm=10.0),
        # a 26-qubit state's gradient with its circuit's 1280 parameters
        _case("clip_state_26q", "clip", circuit=1280, rows=1, qubits=26, max_norm=100.0),
        # a 16-bit bucket
        _case("clip_bf16_packed", "clip", "bfloat16", 150, 120_000_007, 5, packed=True, max_norm=50.0),
        # the 32-qubit circuit's 1280 parameters, Adam with coupled decay, no clipping
        _case("adam_circuit_1280", "adam", circuit=1280, **_adam(0.0, False)),
        # the batched QNN's circuit, its encoder and trained input states together, clipped
        _case("adam_hybrid", "adam", "float32", 6, 42_017, 6, circuit=80, rows=1024, qubits=10,
              **_adam(1.0, False, decay=0.0)),
        # float32 weights and gradients, clipped, decoupled decay
        _case("adam_f32_400m", "adam", "float32", 200, 400_000_009, 7, **_adam(1.0, True)),
        # float32 weights behind a bfloat16 copy that the network runs on, bfloat16 gradients in a bucket
        _case("adam_master_bf16", "adam", "float32", 150, 150_000_011, 8, packed=True,
              **_adam(1.0, True, grad="bfloat16", copy=True)),
    ]


def draw(rng):
    def size(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    op = rng.choice(["norm", "clip", "adam"])
    most = {"norm": 300_000_000, "clip": 150_000_000, "adam": 120_000_000}[op]
    parts = rng.choice(["weights", "weights", "circuit", "states", "all"])
    case = {"circuit": size(1, 5000) if parts in ("circuit", "all") else 0}
    if parts in ("states", "all"):
        case["rows"] = rng.choice([1, size(2, 2000)])
        case["qubits"] = rng.randint(1, int(math.log2(most / 8 / case["rows"])))
    if parts in ("weights", "all"):
        case["tensors"] = size(1, 600)
        case["elements"] = size(case["tensors"], most)
        # 16-bit gradients that are clipped again and again in place would fall below float16's range
        case["dtype"] = rng.choice(["float32", "bfloat16"] if op == "clip" else
                                   ["float32", "bfloat16", "float16"])
        case["packed"] = rng.random() < 0.5
        case["layout"] = rng.randrange(1 << 20)
    if op == "clip":
        case["max_norm"] = round(0.3 * math.sqrt(_numel(_case("", op, **case))), 3)
    if op == "adam":
        clip = rng.choice([0.0, 1.0])
        mixed = case.get("dtype") == "float32" and rng.random() < 0.5
        grad = rng.choice(["bfloat16", "float16"]) if mixed else ""
        case.update(_adam(clip, rng.random() < 0.5, grad, mixed and rng.random() < 0.7,
                          rng.choice([0.0, 0.01, 0.1])))
    return _case("", op, **case)


def _sizes(case):
    """The sizes of the weights: uneven, at least 1 each, `elements` in all."""
    n = case["tensors"]
    if not n:
        return []
    rng = random.Random(case["layout"])
    share = [math.exp(rng.gauss(0.0, 1.5)) for _ in range(n)]
    scale = (case["elements"] - n) / sum(share)
    sizes = [1 + int(s * scale) for s in share]
    sizes[-1] += case["elements"] - sum(sizes)
    return sizes


def _numel(case):
    return case["elements"] + case["circuit"] + 2 * (case["rows"] << case["qubits"])


def _parts(case):
    """(part, type of the parameters) of the parts that the case has."""
    found = [("weights", TYPES[case["dtype"]])] if case["tensors"] else []
    found += [("circuit", torch.float64)] if case["circuit"] else []
    return found + ([("states", torch.complex128)] if case["rows"] else [])


class _Buffers:
    """One buffer for each part of a case, and the tensors as views of them."""

    def __init__(self, case, fill, types, packed):
        self.flat, self.tensors = {}, []
        for part, kind in types:
            if part == "weights":
                sizes = _sizes(case)
                step = 1 if packed else 512 // torch.empty((), dtype=kind).element_size()
                starts, at = [], 0
                for n in sizes:
                    starts.append(at)
                    at += -(-n // step) * step
                flat = torch.zeros(at, dtype=kind, device="cuda")
                views = [flat[s:s + n] for s, n in zip(starts, sizes)]
                if packed:
                    fill(flat)
                else:
                    [fill(v) for v in views]
            else:
                shape = (case["circuit"],) if part == "circuit" else (case["rows"], 1 << case["qubits"])
                flat = torch.empty(shape, dtype=kind, device="cuda")
                fill(torch.view_as_real(flat) if flat.is_complex() else flat)
                views = [flat]
            self.flat[part] = flat
            self.tensors += views


def _wide(kind):
    return kind if kind in (torch.float64, torch.complex128) else torch.float32


def _tensors(case, seed):
    """Everything that the case's path reads and writes, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(scale):
        return lambda t: t.normal_(0.0, scale, generator=gen)

    parts = _parts(case)
    state = {"op": case["op"], "case": case}
    if case["op"] != "adam":
        state["gradients"] = _Buffers(case, normal(1.0), parts, case["packed"])
        state["max_norm"] = case.get("max_norm", 0.0)
        return state
    thin = TYPES[case["grad"]] if case["grad"] else None
    grads = [(p, thin if thin and p == "weights" else k) for p, k in parts]
    wide = [(p, _wide(k)) for p, k in parts]
    state["parameters"] = _Buffers(case, normal(0.5), parts, False)
    state["gradients"] = _Buffers(case, normal(0.02), grads, case["packed"])
    state["m"] = _Buffers(case, normal(0.01), wide, False)
    state["v"] = _Buffers(case, lambda t: t.uniform_(1e-4, 1e-3, generator=gen), wide, False)
    state["copies"] = _Buffers(case, lambda t: t.zero_(), grads[:1], False) if case["copy"] else None
    state["step"] = torch.full((), STEPS_TAKEN, dtype=torch.int64, device="cuda")
    return state


def prepare(case, seed):
    state = _tensors(case, seed)
    if own:
        # what a training program keeps between its steps: the tensor lists, the optimizer's state
        from arcqml_b200 import runtime as rt
        state["gradient_list"] = rt.TensorList(state["gradients"].tensors)
        if case["op"] == "adam":
            state["parameter_list"] = rt.TensorList(state["parameters"].tensors)
            state["adam"] = rt.DeviceAdamState(state["parameter_list"], m=state["m"].tensors,
                                               v=state["v"].tensors, step=state["step"])
            # only the weights (the first tensors) have copies
            state["copy_list"] = None
            if case["copy"]:
                copies = state["copies"].tensors
                rest = len(state["parameters"].tensors) - len(copies)
                state["copy_list"] = rt.TensorList(copies + [None] * rest)
    return state


def _real(t):
    return torch.view_as_real(t) if t.is_complex() else t


def _plain_norm(tensors):
    squares = [_real(t).double().square().sum() for t in tensors]
    return torch.stack(squares).sum().sqrt()


def _plain_factor(norm, max_norm):
    return torch.clamp(max_norm / (norm + 1e-6), max=1.0)


def _plain_clip(tensors, max_norm):
    norm = _plain_norm(tensors)
    factor = _plain_factor(norm, max_norm)
    for t in map(_real, tensors):
        if t.dtype == torch.float64:
            t.mul_(factor)
        else:
            t.copy_(t.float() * factor.float())
    return norm


def _plain_adam(state):
    case, step = state["case"], state["step"]
    norm = _plain_norm(state["gradients"].tensors) if case["max_norm"] else None
    factor = _plain_factor(norm, case["max_norm"]) if case["max_norm"] else None
    step.add_(1)
    bc = [1.0 - torch.pow(b, step.double()) for b in BETAS]
    copies = state["copies"].tensors if state["copies"] else []
    lists = [state[k].tensors for k in ("parameters", "gradients", "m", "v")]
    for i, (p, g, m, v) in enumerate(zip(*lists)):
        p, g, m, v = _real(p), _real(g), _real(m), _real(v)
        kind = m.dtype
        x, g = p.to(kind), g.to(kind)
        if factor is not None:
            g = g * factor.to(kind)
        if not case["decoupled"]:
            g = g + case["decay"] * x
        m.copy_(BETAS[0] * m + (1.0 - BETAS[0]) * g)
        v.copy_(BETAS[1] * v + (1.0 - BETAS[1]) * g * g)
        update = (m / bc[0].to(kind)) / ((v / bc[1].to(kind)).sqrt() + EPS)
        if case["decoupled"]:
            x = x * (1.0 - case["lr"] * case["decay"])
        x = x - case["lr"] * update
        p.copy_(x)
        if i < len(copies):
            copies[i].copy_(x)
    return norm


def run(state):
    op, case = state["op"], state["case"]
    if op == "norm":
        if own:
            from arcqml_b200 import runtime as rt
            return rt.gradient_norm_device(state["gradient_list"])
        return _plain_norm(state["gradients"].tensors)
    if op == "clip":
        if own:
            from arcqml_b200 import runtime as rt
            norm = rt.clip_gradients_device(state["gradient_list"], state["max_norm"])
        else:
            norm = _plain_clip(state["gradients"].tensors, state["max_norm"])
        # the next pass has the same gradients, scaled: a threshold that falls keeps it a pass that scales
        state["max_norm"] *= 0.999
        return {"norm": norm, "gradients": state["gradients"].flat}
    if own:
        from arcqml_b200 import runtime as rt
        norm = rt.adam_step_device(state["parameter_list"], state["gradient_list"], state["adam"],
                                   lr=case["lr"], betas=BETAS, eps=EPS, weight_decay=case["decay"],
                                   decoupled=case["decoupled"], max_norm=case["max_norm"] or None,
                                   copies=state["copy_list"])
    else:
        norm = _plain_adam(state)
    out = {"parameters": state["parameters"].flat, "m": state["m"].flat, "v": state["v"].flat,
           "step": state["step"]}
    if norm is not None:
        out["norm"] = norm
    if state["copies"]:
        out["copies"] = state["copies"].flat
    return out


def work(case):
    """Each tensor read once and written once where it changes."""
    size = {k: torch.empty((), dtype=t).element_size() for k, t in TYPES.items()}
    n64 = case["circuit"] + 2 * (case["rows"] << case["qubits"])
    n, total = case["elements"], case["elements"] + n64
    weight = size[case["dtype"]] if case["dtype"] else 0
    if case["op"] == "norm":
        return {"bytes": n * weight + n64 * 8, "flops": 2 * total}
    if case["op"] == "clip":
        return {"bytes": 2 * (n * weight + n64 * 8), "flops": 3 * total}
    grad = size[case["grad"]] if case["grad"] else weight
    each = 2 * weight + grad + 4 * 4 + (grad if case["copy"] else 0)
    return {"bytes": n * each + n64 * 7 * 8, "flops": (14 if case["max_norm"] else 12) * total}


def exact(case, seed):
    """From the definitions, part by part in 64 bits (a gap between two tensors holds zeros)."""
    s = _tensors(case, seed)
    g = {p: _real(t).to(torch.float64) for p, t in s["gradients"].flat.items()}
    norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(t)) ** 2 for t in g.values()))
    if case["op"] == "norm":
        return torch.tensor(norm, dtype=torch.float64)
    clipped = min(1.0, case["max_norm"] / (norm + 1e-6)) if case["max_norm"] else 1.0

    def shaped(t, like):
        return torch.view_as_complex(t) if like.is_complex() else t

    if case["op"] == "clip":
        return {"norm": torch.tensor(norm, dtype=torch.float64),
                "gradients": {p: shaped(t * clipped, s["gradients"].flat[p]) for p, t in g.items()}}
    t = STEPS_TAKEN + 1
    out = {"parameters": {}, "m": {}, "v": {}, "step": None}
    if case["max_norm"]:
        out["norm"] = torch.tensor(norm, dtype=torch.float64)
    if case["copy"]:
        out["copies"] = {}
    for part, kind in _parts(case):
        like = s["parameters"].flat[part]
        if part == "weights" and case["packed"]:
            # the gradients lie without gaps, the others each on its own 512 bytes
            spread = torch.zeros(like.numel(), dtype=torch.float64, device="cuda")
            sizes, at, to = _sizes(case), 0, 0
            step = 512 // like.element_size()
            for n in sizes:
                spread[to:to + n] = g[part][at:at + n]
                at, to = at + n, to + -(-n // step) * step
            a = spread * clipped
        else:
            a = _same_places(case, part, g[part], like, s["gradients"].flat[part]) * clipped
        x = _real(like).to(torch.float64)
        m = _same_places(case, part, _real(s["m"].flat[part]).double(), like, s["m"].flat[part])
        v = _same_places(case, part, _real(s["v"].flat[part]).double(), like, s["v"].flat[part])
        if not case["decoupled"]:
            a = a + case["decay"] * x
        m = BETAS[0] * m + (1.0 - BETAS[0]) * a
        v = BETAS[1] * v + (1.0 - BETAS[1]) * a * a
        down = 1.0 - case["lr"] * case["decay"] if case["decoupled"] else 1.0
        rate = case["lr"] / (1.0 - BETAS[0] ** t)
        x = x * down - rate * m / (torch.sqrt(v) / math.sqrt(1.0 - BETAS[1] ** t) + EPS)
        out["parameters"][part] = shaped(x, like)
        out["m"][part] = shaped(_other_places(case, part, m, like, s["m"].flat[part]), like)
        out["v"][part] = shaped(_other_places(case, part, v, like, s["v"].flat[part]), like)
        if part == "weights" and case["copy"]:
            out["copies"][part] = _other_places(case, part, x, like, s["copies"].flat[part])
    return out


def _moved(case, flat, of, to):
    """The weights' values from a buffer of element size `of` to the places of one of size `to`."""
    if of == to:
        return flat
    sizes, a, b, start = _sizes(case), 512 // of, 512 // to, [0, 0]
    moved = torch.zeros(sum(-(-n // b) * b for n in sizes), dtype=flat.dtype, device=flat.device)
    for n in sizes:
        moved[start[1]:start[1] + n] = flat[start[0]:start[0] + n]
        start = [start[0] + -(-n // a) * a, start[1] + -(-n // b) * b]
    return moved


def _same_places(case, part, values, like, at):
    return _moved(case, values, at.element_size(), like.element_size()) if part == "weights" else values


def _other_places(case, part, values, like, at):
    return _moved(case, values, like.element_size(), at.element_size()) if part == "weights" else values
