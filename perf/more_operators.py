"""Products in 8-bit integers and tokens sorted by expert, at the sizes that serving and training programs call them with.

* ``matmul``  -- ``int8_matmul``: a product of int8 rows with a scale per token (or one for all) and int8 weights with a scale per output
  channel, and a bias.
* ``quant``   -- ``quant_int8``: rows in int8 with a scale each, in front of such a product.
* ``ragged``  -- ``ragged_int8_matmul``: the product over the segments of rows that belong to experts.
* ``route``   -- ``moe_sort``, ``moe_permute``, ``moe_unpermute``: tokens sorted by expert and back with the router's weights, and, in
  training, their gradients.
* ``layer``   -- ``int8_moe``: a layer of experts in int8 out of all of these and ``silu_mul_quant_int8``.

With ``own`` false the operators are computed in their plain form, in float32; with ``own`` true by the framework.  Layer sizes are
those of ``tilegym_amd.workloads`` or generic.
"""

from __future__ import annotations

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
INT8_MAX = 127.0


# ---------------------------------------------------------------------------- cases
def _matmul(name, m, n, k, dtype="bf16", bias=False, per_token=True):
    """per_token False: one scale for all rows of a."""
    return {"name": name, "op": "matmul", "m": m, "n": n, "k": k, "dtype": dtype, "bias": bias, "per_token": per_token}


def _quant(name, rows, k, dtype="bf16"):
    return {"name": name, "op": "quant", "rows": rows, "k": k, "dtype": dtype}


def _experts(name, op, tokens, experts, top_k, hidden, dtype="bf16", skew=0.5, **more):
    """skew: standard deviation of the experts' popularity, in the router's logits (which have 1)."""
    return {"name": name, "op": op, "tokens": tokens, "experts": experts, "top_k": top_k, "hidden": hidden, "dtype": dtype, "skew": skew, **more}


def listed():
    return [
        # sixteen sequences decoding: a QKV projection, bound by its weight
        _matmul("matmul_16", 16, 6144, 4096),
        # a chunk of a prompt, an odd number of rows, in an f16 model whose projections have a bias
        _matmul("matmul_333", 333, 5120, 12288, dtype="f16", bias=True),
        # a full prefill batch in front of a SwiGLU
        _matmul("matmul_8192", 8192, 28672, 4096),
        # one sequence decoding: in front of a projection; a launch and little else
        _quant("quant_1", 1, 4096),
        # a prompt's activations in front of a down projection
        _quant("quant_5000", 5000, 14336, dtype="f16"),
        # forty tokens decoding: every expert has a few rows, and its whole weight to read
        _experts("ragged_40", "ragged", 40, 64, 6, 2048, n=2816),
        # a chunk of a prompt: about a hundred rows an expert, unevenly
        _experts("ragged_1000", "ragged", 1000, 64, 6, 2048, n=2816, skew=1.0),
        # sixteen tokens decoding: to the experts and back
        _experts("route_16", "route", 16, 64, 6, 2048, grad=False, absent=0.0),
        # a training step's batch, its gradients with it
        _experts("route_4096", "route", 4096, 64, 6, 2048, grad=True, absent=0.0),
        # a training step on one of two ranks: half of the experts are elsewhere; float32
        _experts("route_3001", "route", 3001, 32, 8, 4096, dtype="f32", grad=True, absent=0.5),
        # eight sequences decoding through a layer of experts
        _experts("layer_8", "layer", 8, 64, 6, 2048, inter=1408),
        # a prefill batch through it
        _experts("layer_4096", "layer", 4096, 64, 6, 2048, inter=1408),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    """One more case: rows from one to a full batch, layers from narrow ones to wide ones, few experts and many, every type."""
    while True:
        op = rng.choice(("matmul", "matmul", "matmul", "quant", "ragged", "ragged", "route", "route", "layer"))
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        if op == "matmul":
            odd = rng.random() < 0.15  # sizes that are no multiples of anything
            m, n, k = _log_int(rng, 1, 8192), _log_int(rng, 500, 28672), _log_int(rng, 500, 16384)
            if not odd:
                n, k = n // 16 * 16 + 16, k // 64 * 64 + 64
            elif m * n * k > 1 << 34:
                continue
            if m * n * k <= 8192 * 28672 * 4096:
                return {"op": op, "m": m, "n": n, "k": k, "dtype": dtype, "bias": rng.random() < 0.3, "per_token": rng.random() < 0.8}
            continue
        if op == "quant":
            case = {"op": op, "rows": _log_int(rng, 1, 16384), "k": _log_int(rng, 16, 16384), "dtype": dtype}
            if rng.random() < 0.8:
                case["k"] = case["k"] // 16 * 16 + 16
            if case["rows"] * case["k"] <= 5000 * 14336:
                return case
            continue
        case = {"op": op, "tokens": _log_int(rng, 1, 4096), "experts": rng.choice((4, 8, 16, 32, 64, 128)), "top_k": rng.choice((1, 2, 2, 4, 6, 8)),
                "hidden": 64 * _log_int(rng, 4, 80), "dtype": dtype, "skew": rng.choice((0.0, 0.5, 1.0))}
        rows = case["tokens"] * case["top_k"]
        if case["top_k"] > case["experts"]:
            continue
        if op == "route":
            case["grad"] = rng.random() < 0.6
            case["absent"] = rng.choice((0.0, 0.0, 0.5))
            if rows * case["hidden"] * SIZE[dtype] > 4096 * 8 * 4096 * 2:
                continue
            return case
        if op == "layer":
            if dtype == "f32":
                case["dtype"] = "bf16"
            case["inter"] = 64 * _log_int(rng, 4, 64)
            width = 2 * case["inter"]
        else:
            case["n"] = width = 32 * _log_int(rng, 8, 160)
        # the plain form's padded rows and its weights in 32 bits
        if rows * width * case["hidden"] > 24576 * 2816 * 2048 or case["experts"] * width * case["hidden"] > 64 * 2816 * 2048:
            continue
        if case["experts"] * rows * max(width, case["hidden"]) > 1 << 32:
            continue
        return case


# ---------------------------------------------------------------------------- states
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _activations(shape, g, dtype):
    """Normal values, of which one in a thousand is twenty times as large."""
    x = torch.randn(shape, generator=g, device="cuda")
    return torch.where(torch.rand(shape, generator=g, device="cuda") < 1e-3, x * 20, x).to(dtype)


def _codes(shape, g):
    """What a per-row quantizer makes of normal values: most of them within a third of the range."""
    out = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat = out.view(-1)
    for part in flat.split(1 << 27):
        part.copy_((torch.randn(part.shape, generator=g, device="cuda") * 32).round_().clamp_(-INT8_MAX, INT8_MAX))
    return out


def _scales(shape, g, around):
    return around * torch.exp(0.5 * torch.randn(shape, generator=g, device="cuda"))


def _routing(case, g):
    """(ids, weights) of a router's top k: distinct experts per token, weights that add up to one."""
    T, E = case["tokens"], case["experts"]
    local = E if not case.get("absent") else round(E / (1.0 - case["absent"]))  # experts on all ranks; ours are the first E
    logits = torch.randn((T, local), generator=g, device="cuda") + case["skew"] * torch.randn((1, local), generator=g, device="cuda")
    top = logits.topk(case["top_k"], 1)
    return top.indices.to(torch.int32), torch.softmax(top.values, 1)


def prepare(case, seed):
    g, op = _generator(seed), case["op"]
    t = TYPES[case["dtype"]]
    state = {"case": case}
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        state.update(a=_codes((m, k), g), b=_codes((n, k), g), scale_a=_scales(m if case["per_token"] else 1, g, 0.03), scale_b=_scales(n, g, 1e-3), bias=None)
        if case["bias"]:
            state["bias"] = torch.randn(n, generator=g, device="cuda").to(t)
        return state
    if op == "quant":
        state["x"] = _activations((case["rows"], case["k"]), g, t)
        return state
    E, H = case["experts"], case["hidden"]
    ids, weights = _routing(case, g)
    if op == "ragged":
        count = torch.bincount(ids.flatten(), minlength=E)
        indptr = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
        indptr[1:] = torch.cumsum(count, 0)
        rows = ids.numel()
        state.update(a=_codes((rows, H), g), b=_codes((E, case["n"], H), g), scale_a=_scales(rows, g, 0.03), scale_b=_scales((E, case["n"]), g, 1e-3),
                     indptr=indptr, longest=int(count.max()))
        return state
    state.update(ids=ids, weights=weights, x=_activations((case["tokens"], H), g, t))
    if op == "route":
        # what the experts make of their rows; in training, the gradients that come from the layer behind and from the experts
        state["made"] = torch.randn((ids.numel(), H), generator=g, device="cuda").to(t)
        if case["grad"]:
            state["grad"] = torch.randn((case["tokens"], H), generator=g, device="cuda").to(t)
            state["grad_made"] = torch.randn((ids.numel(), H), generator=g, device="cuda").to(t)
    if op == "layer":
        inter = case["inter"]
        state.update(w1=_codes((E, 2 * inter, H), g), w2=_codes((E, H, inter), g), s1=_scales((E, 2 * inter), g, 1.0 / (32 * math.sqrt(H))),
                     s2=_scales((E, H), g, 1.0 / (32 * math.sqrt(inter))), longest=int(torch.bincount(ids.flatten(), minlength=E).max()))
    return state


# ---------------------------------------------------------------------------- plain forms
def _plain_matmul(state):
    y = torch.matmul(state["a"].float(), state["b"].float().t()) * state["scale_a"][:, None] * state["scale_b"]
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(TYPES[state["case"]["dtype"]])


def _plain_quantizer(x):
    scale = x.abs().amax(-1) / INT8_MAX
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    return (x / scale[..., None]).round().clamp(-INT8_MAX, INT8_MAX), scale


def _plain_quant(state):
    q, scale = _plain_quantizer(state["x"].float())
    return {"q": q.to(torch.int8), "scales": scale}


def _plain_segments(a, scale_a, b, scale_b, indptr, longest):
    """Rows (codes in float32) times their expert's weight: the experts' rows side by side, padded to the longest."""
    row = torch.arange(a.shape[0], device="cuda")
    expert = torch.searchsorted(indptr[1:].long(), row, right=True)
    at = row - indptr.long()[expert]
    padded = torch.zeros((b.shape[0], longest, a.shape[1]), device="cuda")
    padded[expert, at] = a
    y = torch.bmm(b.float(), padded.transpose(1, 2).contiguous())  # (expert, n, row)
    return y.transpose(1, 2)[expert, at] * scale_a[:, None] * scale_b[expert]


def _plain_ragged(state):
    y = _plain_segments(state["a"].float(), state["scale_a"], state["b"], state["scale_b"], state["indptr"], state["longest"])
    return y.to(TYPES[state["case"]["dtype"]])


def _plain_sort(ids, experts):
    """indptr, the row of each slot (below zero, -1 - row, where its expert is not here), the slot of each row."""
    flat = ids.flatten().long()
    flat = torch.where((flat < 0) | (flat >= experts), torch.full_like(flat, experts), flat)
    slots = torch.sort(flat, stable=True).indices
    indptr = torch.zeros(experts + 1, dtype=torch.long, device="cuda")
    indptr[1:] = torch.cumsum(torch.bincount(flat, minlength=experts + 1)[:experts], 0)
    rows = torch.empty_like(slots)
    rows[slots] = torch.arange(slots.numel(), device="cuda")
    return indptr, torch.where(flat < experts, rows, -1 - rows).view(ids.shape), slots


def _plain_route(state):
    case, k, t = state["case"], state["case"]["top_k"], TYPES[state["case"]["dtype"]]
    indptr, row, slots = _plain_sort(state["ids"], case["experts"])
    x, w = state["x"].float(), state["weights"]
    live = (torch.arange(slots.numel(), device="cuda") < indptr[-1])[:, None]
    here, place = (row >= 0)[..., None], torch.where(row >= 0, row, -1 - row)
    rows = torch.where(live, x[slots // k], torch.zeros((), device="cuda")).to(t)
    back = state["made"].float()[place]  # (token, k, element)
    out = {"indptr": indptr.int(), "row": row.int(), "slots": slots.int(), "rows": rows}
    out["out"] = torch.where(here, back * w[..., None], torch.zeros((), device="cuda")).sum(1).to(t)
    if case["grad"]:
        g = state["grad"].float()
        out["grad_made"] = torch.where(live, g[slots // k] * w.flatten()[slots][:, None], torch.zeros((), device="cuda")).to(t)
        out["grad_weights"] = torch.where(here[..., 0], (back * g[:, None]).sum(-1), torch.zeros_like(w))
        out["grad_x"] = torch.where(here, state["grad_made"].float()[place], torch.zeros((), device="cuda")).sum(1).to(t)
    return out


def _plain_layer(state):
    case, k = state["case"], state["case"]["top_k"]
    indptr, row, slots = _plain_sort(state["ids"], case["experts"])
    q, scale = _plain_quantizer(state["x"].float())
    token = slots // k
    h = _plain_segments(q[token], scale[token], state["w1"], state["s1"], indptr, state["longest"])
    h = h.to(state["x"].dtype).float()  # (the first product's output is of the layer's type)
    gate, up = h[:, :case["inter"]], h[:, case["inter"]:]
    q, scale = _plain_quantizer(gate / (1 + torch.exp(-gate)) * up)
    y = _plain_segments(q, scale, state["w2"], state["s2"], indptr, state["longest"])
    return (y[row] * state["weights"][..., None]).sum(1).to(state["x"].dtype)


# ---------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if not own:
        return {"matmul": _plain_matmul, "quant": _plain_quant, "ragged": _plain_ragged, "route": _plain_route, "layer": _plain_layer}[case["op"]](state)
    from tilegym_amd import ops

    t = TYPES[case["dtype"]]
    if case["op"] == "matmul":
        return ops.int8_matmul(state["a"], state["b"], state["scale_a"], state["scale_b"], bias=state["bias"], out_dtype=t)
    if case["op"] == "quant":
        q, scales = ops.quant_int8(state["x"])
        return {"q": q, "scales": scales}
    if case["op"] == "ragged":
        return ops.ragged_int8_matmul(state["a"], state["b"], state["scale_a"], state["scale_b"], state["indptr"], out_dtype=t)
    if case["op"] == "layer":
        return ops.int8_moe(state["x"], state["w1"], state["w2"], state["s1"], state["s2"], state["weights"], state["ids"])
    order = ops.moe_sort(state["ids"], case["experts"])
    out = {"indptr": order.indptr, "row": order.rows, "slots": order.slots, "rows": ops.moe_permute(state["x"], order),
           "out": ops.moe_unpermute(state["made"], order, state["weights"])}
    if case["grad"]:
        out["grad_made"], out["grad_weights"] = ops.moe_unpermute_backward(state["grad"], state["made"], order, state["weights"])
        out["grad_x"] = ops.moe_permute_backward(state["grad_made"], order)
    return out


# ---------------------------------------------------------------------------- what a pass cannot do without
def _experts_used(case):
    """How many experts have rows, on average, where all are as popular."""
    return case["experts"] * (1.0 - (1.0 - case["top_k"] / case["experts"]) ** case["tokens"])


def work(case):
    size, op = SIZE[case["dtype"]], case["op"]
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + m * n * size + 4 * (m + n) + (n * size if case["bias"] else 0), "flops": 2 * m * n * k}
    if op == "quant":
        return {"bytes": case["rows"] * (case["k"] * (size + 1) + 4), "flops": 3 * case["rows"] * case["k"]}
    rows, H = case["tokens"] * case["top_k"], case["hidden"]
    if op == "ragged":
        n = case["n"]
        return {"bytes": _experts_used(case) * n * (H + 4) + rows * (H + 4 + n * size), "flops": 2 * rows * n * H}
    if op == "layer":
        inter = case["inter"]
        return {"bytes": _experts_used(case) * 3 * inter * H + 2 * case["tokens"] * H * size + 8 * rows, "flops": 6 * rows * inter * H}
    there = rows * (1.0 - case["absent"])  # slots whose expert is here
    token, row = case["tokens"] * H * size, rows * H * size
    moved = 12 * rows + token + row + there * H * size + token  # sort, permute (all rows are written), unpermute
    if case["grad"]:
        moved += token + there * H * size + row + 8 * rows + there * H * size + token
    return {"bytes": moved, "flops": there * H * (6 if case["grad"] else 2)}


# ---------------------------------------------------------------------------- in 64 bits
def _exact_codes(x):
    """What a row's codes stand for."""
    step = x.abs().max(-1, keepdim=True).values / 127
    step = step.masked_fill(step == 0, 1.0)
    return torch.round(x / step) * step


def _exact_layer(state):
    case = state["case"]
    ids, w, inter = state["ids"].long(), state["weights"].double(), case["inter"]
    x = _exact_codes(state["x"].double())
    out = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        token, slot = torch.nonzero(ids == e, as_tuple=True)
        if token.numel():
            h = x[token] @ (state["w1"][e].double() * state["s1"][e].double()[:, None]).t()
            h = h.to(state["x"].dtype).double()
            act = _exact_codes(torch.sigmoid(h[:, :inter]) * h[:, :inter] * h[:, inter:])
            y = act @ (state["w2"][e].double() * state["s2"][e].double()[:, None]).t()
            out.index_add_(0, token, y * w[token, slot][:, None])
    return out


def _exact_route(state):
    case, ids, w, x = state["case"], state["ids"].long(), state["weights"].double(), state["x"].double()
    rows = torch.zeros((ids.numel(), case["hidden"]), dtype=torch.float64, device="cuda")
    result = {"indptr": None, "row": None, "slots": None, "rows": rows, "out": torch.zeros_like(x)}
    made = state["made"].double()
    if case["grad"]:
        g, grad_made = state["grad"].double(), state["grad_made"].double()
        result.update(grad_made=torch.zeros_like(rows), grad_weights=torch.zeros_like(w), grad_x=torch.zeros_like(x))
    first = 0
    for e in range(case["experts"]):
        token, slot = torch.nonzero(ids == e, as_tuple=True)
        last, weight = first + token.numel(), w[token, slot][:, None]
        rows[first:last] = x[token]
        result["out"].index_add_(0, token, weight * made[first:last])
        if case["grad"]:
            result["grad_made"][first:last] = weight * g[token]
            result["grad_weights"][token, slot] = (g[token] * made[first:last]).sum(1)
            result["grad_x"].index_add_(0, token, grad_made[first:last])
        first = last
    return result


def exact(case, seed):
    state, op = prepare(case, seed), case["op"]
    if op == "matmul":
        out = (state["a"].double() * state["scale_a"].double()[:, None]) @ (state["b"].double() * state["scale_b"].double()[:, None]).t()
        return out if state["bias"] is None else out + state["bias"].double()
    if op == "quant":
        return {"q": None, "scales": state["x"].double().abs().max(1).values.div(127)}
    if op == "ragged":
        out = torch.empty((state["a"].shape[0], case["n"]), dtype=torch.float64, device="cuda")
        ends = state["indptr"].tolist()
        for e, (lo, hi) in enumerate(zip(ends, ends[1:])):
            out[lo:hi] = (state["a"][lo:hi].double() * state["scale_a"][lo:hi, None].double()) @ (state["b"][e].double() * state["scale_b"][e].double()[:, None]).t()
        return out
    return _exact_layer(state) if op == "layer" else _exact_route(state)
