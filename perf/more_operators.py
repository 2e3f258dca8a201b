"""Work of a hybrid model's training around its circuit: rows of a table looked up by index (token
embeddings, or states made of trained amplitudes), that lookup's gradient, matrices orthogonalised by
Newton-Schulz products, and the momentum step that updates weights with them.

  lookup     out[i] = scale * table[index[i]], or with `normalize` scale * table[index[i]] / |table[index[i]]|;
             zeros where the index is `padding` (-1: no such index)
  gradient   of a loss's table, from the gradient of out: for each row of the table the sum over its
             places, in 32 bits or more, and through the norm where rows are normalised
  orthogonalize
             X <- u / (|u| + 1e-7), then `steps` times X <- a X + (b A + c A^2) X with A = X X^T
             (the polynomial pushes every singular value towards 1)
  muon       m <- 0.95 m + 0.05 g;  u = 0.95 m + 0.05 g;  p <- (1 - lr decay) p - lr s X(u), with
             s = sqrt(max(1, rows / columns))

`shapes` lists matrices as rows x columns, with * for how many."""
import math

import torch

own = False

A, B, C = 3.4445, -4.7750, 2.0315
EPS, BETA = 1e-7, 0.95
TYPES = {"float64": torch.float64, "float32": torch.float32, "bfloat16": torch.bfloat16,
         "float16": torch.float16, "complex128": torch.complex128, "complex64": torch.complex64}


def _table(name, op, dtype, places, rows, width, scale=1.0, normalize=False, padding=-1, skewed=False):
    return dict({"name": name} if name else {}, op=op, dtype=dtype, places=places, rows=rows, width=width,
                scale=scale, normalize=normalize, padding=padding, skewed=skewed)


def _matrices(name, op, dtype, shapes, gradient="", lr=0.0, decay=0.0, steps=5):
    return dict({"name": name} if name else {}, op=op, dtype=dtype, shapes=shapes, gradient=gradient, lr=lr,
                decay=decay, steps=steps)


def listed():
    return [
        # a batch of 4-qubit states from trained amplitudes: a call's latency
        _table("lookup_states_4q", "lookup", "complex128", 256, 61, 16, normalize=True),
        # the batched QNN's 1024 10-qubit states, picked from a table of 4096
        _table("lookup_states_10q", "lookup", "complex128", 1024, 4096, 1024, normalize=True),
        # tokens of a large classical half, embeddings times the root of their width
        _table("lookup_bf16_64k", "lookup", "bfloat16", 65_536, 50_021, 1024, 32.0, padding=0, skewed=True),
        # a small encoder's tokens
        _table("gradient_f32_small", "gradient", "float32", 300, 1000, 97, padding=0, skewed=True),
        # the QNN's initial-state gradient into the table of amplitudes
        _table("gradient_states_10q", "gradient", "complex128", 1024, 509, 1024, normalize=True),
        # the tokens' gradient, a few of them in most places
        _table("gradient_bf16_128k", "gradient", "bfloat16", 131_071, 50_021, 1024, 32.0, padding=0,
               skewed=True),
        # an encoder that feeds the QNN's 80 angles
        _matrices("orthogonalize_encoder", "orthogonalize", "float32", "64x16*2,80x64,10x80,1x80"),
        # 16-bit updates of a middle-sized network
        _matrices("orthogonalize_bf16", "orthogonalize", "bfloat16", "2048x2048*2,1000x4096,8192x512"),
        # one large 32-bit matrix
        _matrices("orthogonalize_f32_large", "orthogonalize", "float32", "4096x8191"),
        # a step of that encoder
        _matrices("muon_encoder", "muon", "float32", "64x16*2,80x64,10x80,1x80", "float32", 0.02),
        # float32 weights of a network of many layers
        _matrices("muon_f32_layers", "muon", "float32", "1024x1024*16,4096x1024*4,1024x4096*4", "float32",
                  0.02, 0.01),
        # large 16-bit weights
        _matrices("muon_bf16_large", "muon", "bfloat16", "4096x4096*4,2048x8192*2,8192x2048*2", "bfloat16",
                  0.02, 0.1),
    ]


def draw(rng):
    """Tables of 1 to 150,000 rows, 1 to 131,071 places and rows of up to 1 MB; up to 40 matrices of 1 to
    8192 rows or columns."""
    def size(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    op = rng.choice(["lookup", "gradient", "orthogonalize", "muon"])
    if op in ("lookup", "gradient"):
        states = rng.random() < 0.4
        dtype = rng.choice(["complex128", "complex64"] if states else
                           ["float32", "bfloat16", "float16", "float64"])
        width = 1 << rng.randint(1, 16) if states else size(1, 4096)
        # a real row of one or two numbers has next to nothing left to turn by
        normalize = states or (dtype in ("float32", "float64") and width > 3 and rng.random() < 0.3)
        most = 2 ** 28 // (width * (16 if dtype == "complex128" else 8))
        rows = size(1, max(1, min(150_000, most)))
        places = size(1, max(1, min(131_071, most)))
        return _table("", op, dtype, places, rows, width, rng.choice([1.0, 0.125, math.sqrt(width)]), normalize,
                      rng.choice([-1, 0, rows - 1]), rng.random() < 0.7)
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    left, shapes = 2.5e12, []
    for _ in range(rng.choice([1, 2, 3, 5])):
        m, n = size(1, 4096), size(1, 8192)
        times = size(1, 8)
        while times * _products(m, n, 5) > left and m > 1:
            m, n, times = max(1, m // 2), max(1, n // 2), max(1, times // 2)
        left -= times * _products(m, n, 5)
        shapes.append(f"{m}x{n}*{times}")
    gradient = dtype if rng.random() < 0.6 else rng.choice(["float32", "bfloat16", "float16"])
    muon = op == "muon"
    return _matrices("", op, dtype, ",".join(shapes), gradient if muon else "",
                     rng.choice([0.002, 0.02]) if muon else 0.0, rng.choice([0.0, 0.01, 0.1]) if muon else 0.0)


def _shapes(case):
    found = []
    for part in case["shapes"].split(","):
        shape, _, times = part.partition("*")
        found += [tuple(int(n) for n in shape.split("x"))] * int(times or 1)
    return found


def _products(rows, columns, steps):
    """Operations of the products, each symmetric one counted once."""
    m, n = min(rows, columns), max(rows, columns)
    return steps * (3 * m * m * n + m ** 3)


def _buffer(shapes, dtype, fill):
    """One buffer, and matrices as views of it that each start on 512 bytes."""
    step = 512 // torch.empty((), dtype=dtype).element_size()
    starts, at = [], 0
    for m, n in shapes:
        starts.append(at)
        at += -(-m * n // step) * step
    flat = torch.zeros(at, dtype=dtype, device="cuda")
    views = [flat[s:s + m * n].view(m, n) for s, (m, n) in zip(starts, shapes)]
    for v in views:
        fill(v)
    return flat, views


def _inputs(case, seed):
    """Everything that the case's path reads, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(scale):
        def fill(t):
            t = torch.view_as_real(t) if t.is_complex() else t
            return t.normal_(0.0, scale, generator=gen)
        return fill

    state = {"op": case["op"], "case": case}
    if case["op"] in ("lookup", "gradient"):
        rows, width, places = case["rows"], case["width"], case["places"]
        chance = torch.rand(places, device="cuda", dtype=torch.float64, generator=gen)
        # skewed: the i-th row comes up about 1 / i as often as the first, as words do
        index = torch.exp(chance * math.log(rows + 1)) - 1 if case["skewed"] else chance * rows
        state["index"] = index.long().clamp_(0, rows - 1)
        if case["op"] == "lookup" or case["normalize"]:
            state["table"] = torch.empty(rows, width, dtype=dtype, device="cuda")
            normal(0.02 if not case["normalize"] else 1.0)(state["table"])
        if case["op"] == "gradient":
            state["gradient"] = torch.empty(places, width, dtype=dtype, device="cuda")
            normal(1e-2)(state["gradient"])
        return state
    shapes = _shapes(case)
    if case["op"] == "orthogonalize":
        state["matrices"] = _buffer(shapes, dtype, normal(1e-3))[1]
        return state
    state["flat"], state["parameters"] = _buffer(shapes, dtype, lambda t: normal(t.shape[1] ** -0.5)(t))
    state["gradients"] = _buffer(shapes, TYPES[case["gradient"]], normal(1e-3))[1]
    state["momentum_flat"], state["momentum"] = _buffer(shapes, torch.float32, normal(5e-4))
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    if own and case["op"] == "muon":
        # what a training program keeps between its steps: the lists and the optimizer's state
        from arcqml_b200 import runtime as rt
        state["parameter_list"] = rt.TensorList(state["parameters"])
        state["gradient_list"] = rt.TensorList(state["gradients"])
        state["muon"] = rt.DeviceMuonState(state["parameter_list"], momentum=state["momentum"])
    if own and case["op"] == "orthogonalize":
        from arcqml_b200 import runtime as rt
        state["matrix_list"] = rt.TensorList(state["matrices"])
    return state


def _wide(t):
    return t.float() if t.dtype in (torch.bfloat16, torch.float16) else t


def _norms(t):
    return (torch.view_as_real(t).flatten(1) if t.is_complex() else t).square().sum(1, keepdim=True).sqrt()


def _plain_lookup(state):
    case, index, table = state["case"], state["index"], state["table"]
    x = _wide(table[index])
    if case["normalize"]:
        x = x / _norms(x)
    return (x * (index != case["padding"])[:, None] * case["scale"]).to(table.dtype)


def _plain_gradient(state):
    case, index, g = state["case"], state["index"], state["gradient"]
    x = _wide(g) * (index != case["padding"])[:, None] * case["scale"]
    x = torch.view_as_real(x) if x.is_complex() else x
    total = torch.zeros((case["rows"],) + x.shape[1:], dtype=x.dtype, device="cuda").index_add_(0, index, x)
    if case["normalize"]:
        table = state["table"]
        t = torch.view_as_real(table) if table.is_complex() else _wide(table)
        t, s = t.reshape(case["rows"], -1), total.reshape(case["rows"], -1)
        norm = t.square().sum(1, keepdim=True).sqrt()
        t = t / norm
        total = ((s - t * (t * s).sum(1, keepdim=True)) / norm).reshape(total.shape)
    return torch.view_as_complex(total) if g.is_complex() else total.to(g.dtype)


def _plain_polynomial(u, steps):
    """In 32 bits."""
    flip = u.shape[0] > u.shape[1]
    x = u.mT if flip else u
    x = x / (x.square().sum().sqrt() + EPS)
    for _ in range(steps):
        a = x @ x.mT
        x = A * x + (B * a + C * (a @ a)) @ x
    return x.mT if flip else x


def _plain_muon(state):
    case = state["case"]
    for p, g, m in zip(state["parameters"], state["gradients"], state["momentum"]):
        g = g.float()
        m.copy_(BETA * m + (1.0 - BETA) * g)
        x = _plain_polynomial(BETA * m + (1.0 - BETA) * g, case["steps"])
        rate = case["lr"] * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
        p.copy_(p.float() * (1.0 - case["lr"] * case["decay"]) - rate * x)


def run(state):
    op, case = state["op"], state["case"]
    padding = case["padding"] if case.get("padding", -1) >= 0 else None
    if op == "lookup":
        if own:
            from arcqml_b200 import runtime as rt
            return rt.embedding_lookup_device(state["table"], state["index"], scale=case["scale"],
                                              normalize=case["normalize"], padding=padding)
        return _plain_lookup(state)
    if op == "gradient":
        if own:
            from arcqml_b200 import runtime as rt
            return rt.embedding_gradient_device(state["gradient"], state["index"], case["rows"],
                                                scale=case["scale"], padding=padding,
                                                table=state["table"] if case["normalize"] else None)
        return _plain_gradient(state)
    if op == "orthogonalize":
        if own:
            from arcqml_b200 import runtime as rt
            return rt.orthogonalize_device(state["matrix_list"], steps=case["steps"])
        return [_plain_polynomial(u.float(), case["steps"]).to(u.dtype).contiguous() for u in state["matrices"]]
    if own:
        from arcqml_b200 import runtime as rt
        rt.muon_step_device(state["parameter_list"], state["gradient_list"], state["muon"], lr=case["lr"],
                            momentum=BETA, nesterov=True, weight_decay=case["decay"], steps=case["steps"])
    else:
        _plain_muon(state)
    return {"parameters": state["flat"], "momentum": state["momentum_flat"]}


def _distinct(case):
    """Rows of the table that come up, on average."""
    rows, places = case["rows"], case["places"]
    if not case["skewed"]:
        return rows * -math.expm1(places * math.log1p(-1.0 / rows)) if rows > 1 else 1.0
    v = torch.arange(rows, dtype=torch.float64)
    chance = torch.log1p(1.0 / (v + 1.0)) / math.log(rows + 1)
    return float((1.0 - torch.exp(places * torch.log1p(-chance.clamp(max=1.0 - 1e-12)))).sum())


def work(case):
    size = {k: torch.empty((), dtype=t).element_size() for k, t in TYPES.items()}
    if case["op"] in ("lookup", "gradient"):
        row = case["width"] * size[case["dtype"]]
        parts = case["width"] * (2 if case["dtype"].startswith("complex") else 1)
        read = 8 * case["places"]
        if case["op"] == "lookup":
            return {"bytes": read + row * (_distinct(case) + case["places"]),
                    "flops": parts * case["places"] * (3 if case["normalize"] else 1)}
        bytes_ = read + row * (case["places"] + case["rows"])
        if case["normalize"]:
            bytes_ += row * _distinct(case)
        return {"bytes": bytes_, "flops": parts * (case["places"] + (6 * _distinct(case) if case["normalize"] else 0))}
    shapes, each = _shapes(case), size[case["dtype"]]
    elements = sum(m * n for m, n in shapes)
    moved = 2 * each if case["op"] == "orthogonalize" else 2 * each + 8 + size[case["gradient"]]
    return {"bytes": elements * moved, "flops": sum(_products(m, n, case["steps"]) for m, n in shapes)}


def _exact_polynomial(u, steps):
    """All factors commute with u u^T: their product is formed apart from u."""
    flip = u.shape[0] > u.shape[1]
    u = u.mT if flip else u
    u = u / (torch.linalg.matrix_norm(u) + EPS)
    gram = u @ u.mT
    one = torch.eye(len(gram), dtype=torch.float64, device="cuda")
    whole = one
    for _ in range(steps):
        factor = A * one + gram @ (B * one + C * gram)
        whole = factor @ whole
        gram = factor @ gram @ factor
    x = whole @ u
    return x.mT.contiguous() if flip else x


def exact(case, seed):
    """From the definitions, in 64 bits."""
    s = _inputs(case, seed)
    if case["op"] in ("lookup", "gradient"):
        index, rows, wide = s["index"], case["rows"], torch.float64
        table = s.get("table")
        if table is not None:
            t = torch.view_as_real(table).flatten(1).to(wide) if table.is_complex() else table.to(wide)
            norm = torch.linalg.vector_norm(t, dim=1, keepdim=True)
        if case["op"] == "lookup":
            out = (t / norm if case["normalize"] else t)[index] * case["scale"]
            out[index == case["padding"]] = 0.0
        else:
            g = s["gradient"]
            g = torch.view_as_real(g).flatten(1) if g.is_complex() else g
            # places in the order of their rows; each row's sum lies between two running sums
            order = torch.argsort(index, stable=True)
            ends = torch.cumsum(torch.bincount(index, minlength=rows), 0)
            out = torch.empty(rows, g.shape[1], dtype=wide, device="cuda")
            for at in range(0, g.shape[1], 1024):
                run_ = torch.zeros(len(index) + 1, min(1024, g.shape[1] - at), dtype=wide, device="cuda")
                torch.cumsum(g[order, at:at + 1024].to(wide), 0, out=run_[1:])
                out[:, at:at + 1024] = run_[ends] - run_[ends - torch.bincount(index, minlength=rows)]
            out *= case["scale"]
            if case["padding"] >= 0:
                out[case["padding"]] = 0.0
            if case["normalize"]:
                unit = t / norm
                out = (out - unit * (unit * out).sum(1, keepdim=True)) / norm
        return torch.view_as_complex(out.view(len(out), -1, 2)) if case["dtype"].startswith("complex") else out
    if case["op"] == "orthogonalize":
        return [_exact_polynomial(u.to(torch.float64), case["steps"]) for u in s["matrices"]]
    out = {"parameters": torch.zeros(s["flat"].shape, dtype=torch.float64, device="cuda"),
           "momentum": torch.zeros(s["momentum_flat"].shape, dtype=torch.float64, device="cuda")}
    places = {"parameters": s["flat"], "momentum": s["momentum_flat"]}
    for p, g, m in zip(s["parameters"], s["gradients"], s["momentum"]):
        g, moved = g.to(torch.float64), m.to(torch.float64)
        moved = BETA * moved + (1.0 - BETA) * g
        x = _exact_polynomial(BETA * moved + (1.0 - BETA) * g, case["steps"])
        rate = case["lr"] * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
        new = p.to(torch.float64) * (1.0 - case["lr"] * case["decay"]) - rate * x
        for name, view, value in (("parameters", p, new), ("momentum", m, moved)):
            at = (view.data_ptr() - places[name].data_ptr()) // view.element_size()
            out[name][at:at + view.numel()] = value.reshape(-1)
    return out
