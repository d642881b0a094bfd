"""What the adapter and gradient-norm operators are measured on: cases, inputs,
one pass, and the same pass in plain torch.

Three operators, called as a user of ``fp_emulation`` calls them:

* ``serve``: ``adapter_matmul(x, A, B, rows, base, scale)`` without gradients:
  every row of a batch adds the low-rank product of its own adapter to the
  output of the projection that all rows share;
* ``train``: the same call recorded by autograd, and its backward pass (the
  gradients of the input and of both adapter factors);
* ``clip``: the global norm over a list of gradients of any sizes and types, and
  the gradients scaled to at most a given norm (``clip_grads``), or in place
  over parameters (``clip_grad_norm_``).

``own`` selects the framework's calls; otherwise ``run`` uses elementary torch
operations in 32 bits (64 for float64 data and for long sums).
"""
import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DTYPES = {"float64": torch.float64, "float32": torch.float32, "float16": torch.float16,
           "bfloat16": torch.bfloat16}
_EPS = 1e-6  # added to the norm before the division, as torch.nn.utils does


def _package():
    path = os.path.join(_ROOT, "fp-emulation_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import fp_emulation

    return fp_emulation


# ----------------------------------------------------------------- cases ----

def _adapters(name, op, dtype, rows, n, fan_in, fan_out, rank, order="mixed", idle=0.0, scale="one"):
    """``order``: "runs" (the rows of one request stand together) or "mixed" (any
    order); ``idle``: the share of rows that no adapter serves; ``scale``: one
    factor for all adapters, or one for each."""
    case = {"op": op, "dtype": dtype, "rows": rows, "adapters": n, "in": fan_in, "out": fan_out, "rank": rank,
            "order": order, "idle": idle, "scale": scale}
    if name:
        case["name"] = name
    return case


def _clip(name, kind, dtype, layers, width, norm=2.0, clipped=True, inplace=False):
    """``kind`` names the list of tensors: see ``_shapes``."""
    case = {"op": "clip", "kind": kind, "dtype": dtype, "layers": layers, "width": width, "norm": norm,
            "clipped": clipped, "inplace": inplace}
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # One point asked of one member of a family of 256-wide physics networks in float64.
        _adapters("serve_f64_1row", "serve", "float64", 1, 16, 256, 256, 8),
        # A decoding step: 32 sequences, each with an adapter of its own, beside a 4096-wide projection.
        _adapters("serve_bf16_32rows", "serve", "bfloat16", 32, 64, 4096, 4096, 16, scale="each"),
        # A small batch of evaluations, many adapters, some rows on the plain model, float64.
        _adapters("serve_f64_200rows", "serve", "float64", 200, 24, 4096, 4096, 16, idle=0.1),
        # The whole 16384-row batch of the 4096-wide float64 network, eight adapters in runs.
        _adapters("serve_f64_16384rows", "serve", "float64", 16384, 8, 4096, 4096, 16, order="runs"),
        # Prompts of sixteen requests in one batch, rank 64, half precision.
        _adapters("serve_f16_prompts", "serve", "float16", 16384, 16, 4096, 8192, 64, order="runs", scale="each"),
        # Nothing even: odd widths, odd rank, rows in any order, a fifth of them idle, float32.
        _adapters("serve_f32_odd", "serve", "float32", 5001, 7, 1000, 777, 12, idle=0.2),
        # Fine-tuning ten members of the physics family on their 40 x 40 grids at once.
        _adapters("train_f64_grid", "train", "float64", 16000, 10, 256, 256, 4, order="runs"),
        # Fine-tuning four adapters together on long sequences, bfloat16.
        _adapters("train_bf16_long", "train", "bfloat16", 16384, 4, 4096, 4096, 32, order="runs"),
        # A small odd training batch in float32, rows in any order.
        _adapters("train_f32_odd", "train", "float32", 3333, 6, 1023, 515, 20, idle=0.1, scale="each"),
        # The gradients of one physics network (2-256-256-256-1, float64).
        _clip("clip_f64_small", "network", "float64", 3, 256),
        # A converted model: float64 layers, float32 norms, bfloat16 embedding, many tensors; in bounds, in place.
        _clip("clip_mixed_in_bounds", "mixed", "float64", 24, 1024, clipped=False, inplace=True),
        # A large model's gradients in bfloat16, scaled.
        _clip("clip_bf16_large", "network", "bfloat16", 18, 4096),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["serve", "serve", "train", "clip"])
    dtype = rng.choice(list(_DTYPES))
    if op == "clip":
        kind = rng.choice(["network", "adapters", "mixed"])
        width = _spread(rng, 17, 4096)
        inplace = rng.random() < 0.25
        most = 48 if inplace else 14  # a list that comes back tensor by tensor stays below 60 of them
        layers = _spread(rng, 1, max(1, min(most, (1 << 26) // (width + 8) ** 2)))
        # An in-place call that scales would hand its next pass other gradients: in bounds, they stay.
        return _clip(None, kind, dtype, layers, width, rng.choice([2.0, 2.0, 2.0, 1.0, math.inf]), not inplace, inplace)
    fan_in, fan_out = _spread(rng, 32, 4096), _spread(rng, 32, 4096)
    if rng.random() < 0.6:  # widths of models are mostly multiples of 64
        fan_in, fan_out = max(64, fan_in // 64 * 64), max(64, fan_out // 64 * 64)
    rank = rng.choice([4, 8, 16, 32, 64]) if rng.random() < 0.6 else _spread(rng, 1, 64)
    rows = _spread(rng, 1, 8192 if op == "serve" else 6000)
    return _adapters(None, op, dtype, rows, _spread(rng, 1, 64), fan_in, fan_out, rank,
                     rng.choice(["runs", "mixed"]), rng.choice([0.0, 0.0, 0.1, 0.5]), rng.choice(["one", "each"]))


# ---------------------------------------------------------------- inputs ----

def _busy(case):
    """How many rows have an adapter."""
    return max(1, case["rows"] - int(case["rows"] * case["idle"]))


def _index(case, gen):
    """One adapter per row, -1 for none; every adapter has a row where there are rows enough."""
    rows, n, busy = case["rows"], case["adapters"], _busy(case)
    order = torch.randperm(n, generator=gen, device="cuda")
    if busy <= n:
        ids = order[:busy]
    else:
        ids = torch.cat([order, torch.randint(n, (busy - n,), generator=gen, device="cuda")])
    ids = torch.cat([ids, torch.full((rows - busy,), -1, dtype=ids.dtype, device="cuda")])
    if case["order"] == "runs":
        return torch.sort(ids)[0].to(torch.int32)
    return ids[torch.randperm(rows, generator=gen, device="cuda")].to(torch.int32)


def _shapes(case):
    """The tensors of a model: (shape, type)."""
    width, layers, dtype = case["width"], case["layers"], case["dtype"]
    if case["kind"] == "network":  # a first and a last layer, square layers between, all with a bias
        dims = [2] + [width] * layers + [1]
        out = []
        for a, b in zip(dims, dims[1:]):
            out += [((b, a), dtype), ((b,), dtype)]
        return out
    if case["kind"] == "adapters":  # two low-rank factors a layer
        return [shape for _ in range(layers) for shape in (((8, 16, width), dtype), ((8, width, 16), dtype))]
    out = [((8 * width, width), "bfloat16")]  # an embedding, then float64 layers with float32 norms between
    for _ in range(layers):
        out += [((width,), "float32"), ((width,), "float32"), ((width, width), "float64"), ((width,), "float64")]
    return out


def _packed(tensors):
    """One buffer for each type that holds its tensors end to end, and the views of them."""
    flat, place = {}, {}
    for dtype in dict.fromkeys(t.dtype for t in tensors):
        flat[dtype] = torch.cat([t.flatten() for t in tensors if t.dtype == dtype])
        place[dtype] = 0
    views = []
    for t in tensors:
        at = place[t.dtype]
        views.append(flat[t.dtype][at:at + t.numel()].view(t.shape))
        place[t.dtype] = at + t.numel()
    return list(flat.values()), views


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, dtype, std=1.0):
        t = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float64 if dtype == torch.float64 else
                        torch.float32)
        return t.mul_(std).to(dtype)

    if case["op"] == "clip":
        shapes = _shapes(case)
        count = sum(math.prod(shape) for shape, _ in shapes)
        # Gradients of about this norm before clipping to 1 (layers differ by some powers of two).
        target = {2.0: count ** -0.5, 1.0: 1.0 / count, math.inf: 0.3}[case["norm"]] * (6.0 if case["clipped"] else 0.02)
        grads = [normal(shape, _DTYPES[dtype], target * 2.0 ** (i % 5 - 2)) for i, (shape, dtype) in enumerate(shapes)]
        state = {"case": case, "grads": grads}
        if case["inplace"]:
            # The gradients are views of one packed buffer for each type, as a training loop
            # that reduces them between GPUs keeps them; the buffers are what the pass returns.
            flat, views = _packed(grads)
            state["flat"], state["grads"] = flat, views
            state["params"] = [torch.nn.Parameter(torch.empty_like(g)) for g in views]
            for p, g in zip(state["params"], views):
                p.grad = g
        return state

    dtype = _DTYPES[case["dtype"]]
    rows, n, k, m, r = (case[key] for key in ("rows", "adapters", "in", "out", "rank"))
    index = _index(case, gen)
    state = {
        "case": case, "index": index,
        "x": normal((rows, k), dtype),
        "A": normal((n, r, k), dtype, k ** -0.5),
        "B": normal((n, m, r), dtype, r ** -0.5),
        "base": normal((rows, m), dtype),
    }
    if case["scale"] == "each":
        state["scale"] = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64) + 0.5
    else:
        state["scale"] = 2.0
    if case["op"] == "train":
        state["dy"] = normal((rows, m), dtype, 0.01)
        for key in ("x", "A", "B"):
            state[key].requires_grad_(True)
    if own:
        state["rows"] = _package().prepare_rows(index, n)  # made once a batch, used by every layer
    return state


# ------------------------------------------------------------- one pass ----

def run(state):
    case = state["case"]
    if case["op"] == "clip":
        return _run_clip(state, case)
    if own:
        fp = _package()
        if case["op"] == "serve":
            return fp.adapter_matmul(state["x"], state["A"], state["B"], state["rows"], base=state["base"],
                                     scale=state["scale"])
        y = fp.adapter_matmul(state["x"], state["A"], state["B"], state["rows"], base=state["base"],
                              scale=state["scale"])
        return (y.detach(),) + torch.autograd.grad(y, (state["x"], state["A"], state["B"]), state["dy"])
    return _plain_adapters(state, case)


def _run_clip(state, case):
    grads, norm_type = state["grads"], case["norm"]
    if own:
        fp = _package()
        if case["inplace"]:
            return state["flat"], fp.clip_grad_norm_(state["params"], 1.0, norm_type)
        return fp.clip_grads(grads, 1.0, norm_type)
    wide = [g if g.dtype == torch.float64 else g.float() for g in grads]
    if norm_type == math.inf:
        norm = torch.stack([g.abs().max().double() for g in wide]).max()
    elif norm_type == 1.0:
        norm = torch.stack([g.abs().sum(dtype=torch.float64) for g in wide]).sum()
    else:
        norm = torch.stack([(g * g).sum(dtype=torch.float64) for g in wide]).sum().sqrt()
    factor = torch.clamp(1.0 / (norm + _EPS), max=1.0)
    if any(g.dtype == torch.float64 for g in grads):
        total = norm
    else:
        total, factor = norm.float(), factor.float()
    out = [(w * (factor if w.dtype == torch.float64 else factor.float())).to(g.dtype) for w, g in zip(wide, grads)]
    if case["inplace"]:
        for g, o in zip(grads, out):
            g.copy_(o)
        return state["flat"], total
    return out, total


def _plain_adapters(state, case):
    dtype = _DTYPES[case["dtype"]]
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    index, scale = state["index"].long(), state["scale"]
    x, A, B, base = (state[key].detach().to(wide) for key in ("x", "A", "B", "base"))
    y = base.clone()
    train = case["op"] == "train"
    if train:
        dy = state["dy"].to(wide)
        dx, dA, dB = torch.zeros_like(x), torch.zeros_like(A), torch.zeros_like(B)
    for i in range(case["adapters"]):
        picked = torch.nonzero(index == i).flatten()
        if picked.numel() == 0:
            continue
        s = scale if isinstance(scale, float) else scale[i].to(wide)
        xi = x[picked]
        u = (xi @ A[i].T) * s
        y[picked] += u @ B[i].T
        if train:
            gi = dy[picked]
            v = (gi @ B[i]) * s
            dx[picked] = v @ A[i]
            dA[i] = v.T @ xi
            dB[i] = gi.T @ u
    if train:
        return y.to(dtype), dx.to(dtype), dA.to(dtype), dB.to(dtype)
    return y.to(dtype)


# ------------------------------------------------------ work and results ----

def work(case):
    if case["op"] == "clip":
        size = {"float64": 8, "float32": 4, "float16": 2, "bfloat16": 2}
        total = sum(math.prod(shape) * size[dtype] for shape, dtype in _shapes(case))
        count = sum(math.prod(shape) for shape, _ in _shapes(case))
        # Gradients in bounds are read and stay as they are; scaled ones are read and written.
        return {"bytes": total * (2 if case["clipped"] else 1), "flops": count * (3 if case["clipped"] else 2)}
    e = {"float64": 8, "float32": 4, "float16": 2, "bfloat16": 2}[case["dtype"]]
    rows, n, k, m, r = (case[key] for key in ("rows", "adapters", "in", "out", "rank"))
    busy = _busy(case)
    used = min(n, busy)
    if case["op"] == "serve":
        return {"bytes": e * (busy * k + 2 * rows * m + used * r * (k + m)) + 4 * rows,
                "flops": 2 * busy * r * (k + m)}
    # x, base, dy and the factors read; y, dx and the factors' gradients written.
    return {"bytes": e * (busy * k + 2 * rows * m + busy * m + rows * k + (used + n) * r * (k + m)) + 4 * rows,
            "flops": 6 * busy * r * (k + m)}


def exact(case, seed):
    """The definition in 64 bits: row by row sums over the row's own adapter, all rows of a
    block at once with the factors gathered per row; gradients as sums over a one-hot choice."""
    state = prepare(case, seed)
    if case["op"] == "clip":
        p = case["norm"]
        flat = [g.to(torch.float64).flatten() for g in state["grads"]]
        per = torch.stack([torch.linalg.vector_norm(f, p) for f in flat])
        norm = torch.linalg.vector_norm(per, p)
        coef = min(1.0, 1.0 / (float(norm) + _EPS))
        if case["inplace"]:
            return [f.to(torch.float64) * coef for f in state["flat"]], norm
        return [(f * coef).view_as(g) for f, g in zip(flat, state["grads"])], norm
    x, A, B, base = (state[key].detach().to(torch.float64) for key in ("x", "A", "B", "base"))
    index = state["index"].long()
    n = case["adapters"]
    scale = state["scale"]
    s = torch.full((n,), scale, dtype=torch.float64, device="cuda") if isinstance(scale, float) else scale
    choice = torch.nn.functional.one_hot(index.clamp(min=0), n).to(torch.float64) * (index >= 0).unsqueeze(1)
    s_row = choice @ s
    # u[t, j] = sum over i of choice[t, i] x[t] . A[i, j]: all adapters' products, then the row's own one.
    rows, r = case["rows"], case["rank"]
    y = base.clone()
    u = torch.empty((rows, r), dtype=torch.float64, device="cuda")
    block = max(1, (1 << 25) // (n * max(r, 1)))
    for a in range(0, rows, block):
        b = min(rows, a + block)
        every = torch.einsum("tk,njk->tnj", x[a:b], A)
        u[a:b] = torch.einsum("tnj,tn->tj", every, choice[a:b]) * s_row[a:b, None]
        spread = (choice[a:b, :, None] * u[a:b, None, :]).reshape(b - a, n * r)
        y[a:b] += spread @ B.permute(0, 2, 1).reshape(n * r, -1)
    if case["op"] == "serve":
        return y
    dy = state["dy"].to(torch.float64)
    v = torch.empty_like(u)
    dx = torch.empty_like(x)
    dA, dB = torch.zeros_like(A), torch.zeros_like(B)
    for a in range(0, rows, block):
        b = min(rows, a + block)
        every = torch.einsum("tm,nmj->tnj", dy[a:b], B)
        v[a:b] = torch.einsum("tnj,tn->tj", every, choice[a:b]) * s_row[a:b, None]
        spread = (choice[a:b, :, None] * v[a:b, None, :]).reshape(b - a, n * r)
        dx[a:b] = spread @ A.reshape(n * r, -1)
        dA += (spread.T @ x[a:b]).view_as(dA)
        held = (choice[a:b, :, None] * u[a:b, None, :]).reshape(b - a, n * r)
        dB += (held.T @ dy[a:b]).view(n, r, -1).permute(0, 2, 1)
    return y, dx, dA, dB
