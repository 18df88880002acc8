"""The operators around a decoder layer's FP8 projections, at the sizes that serving programs call them with.

* ``norm``      -- ``rms_norm_quant``: root-mean-square norm with the residual's addition, the output in e4m3 with a scale per group
  (what a block-scaled projection takes) or with a given per-tensor scale.
* ``append``    -- ``kv_cache_append``: rotary positions on the new tokens' q and k, and k and v written to a paged e4m3 cache with a
  scale per page and head.
* ``read``      -- ``kv_cache_read``: a cache's tokens as plain rows.
* ``attention`` -- ``kv_cache_attention``: causal attention of the new tokens over that cache, whole, or in a window with
  a few first tokens that stay visible.

With ``own`` false the operators are computed in their plain form, in float32 (the rotary table is made in float64); with ``own``
true by the framework.  Layer sizes are those of ``tilegym_amd.workloads`` or generic.
"""

from __future__ import annotations

import math

import torch

own = False

FP8 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
E4M3_MAX = 448.0
MIN_EXPONENT, MAX_EXPONENT = -40, 40  # of a page's scale
EPS = 1e-5


# ---------------------------------------------------------------------------- cases
def _norm(name, rows, hidden, dtype="bf16", group=128, residual=True):
    """group 0: one given scale for the whole tensor."""
    return {"name": name, "op": "norm", "rows": rows, "hidden": hidden, "dtype": dtype, "group": group, "residual": residual}


def _cached(name, op, batch, new, len_lo, len_hi, dtype="bf16", kv_heads=8, group=4, dim=128, page=64, **more):
    """batch sequences of len_lo .. len_hi tokens, spread evenly; `new` of them new in all sequences together."""
    return {"name": name, "op": op, "batch": batch, "new": new, "len_lo": len_lo, "len_hi": len_hi, "dtype": dtype, "kv_heads": kv_heads,
            "group": group, "dim": dim, "page": page, **more}


def listed():
    return [
        # one sequence decoding: in front of a layer's QKV projection; a launch and little else
        _norm("norm_1", 1, 4096),
        # a chunk of a prompt in a wider f16 model, an odd number of rows
        _norm("norm_777", 777, 5120, dtype="f16"),
        # a full prefill batch in front of a projection with a per-tensor scale
        _norm("norm_8192", 8192, 4096, group=0),
        # sixteen sequences decoding: one token each into pages that are partly full
        _cached("append_16", "append", 16, 16, 100, 2000, rotary=128, interleaved=False),
        # five prompts (or chunks of prompts) of uneven lengths, half of the head rotated in neighbouring pairs
        _cached("append_4096", "append", 5, 4096, 300, 3000, rotary=64, interleaved=True),
        # a prefix of one conversation, read back for another use of its tokens
        _cached("read_500", "read", 1, 0, 500, 500, kv_heads=8),
        # the caches of eight long conversations moved out
        _cached("read_100000", "read", 8, 0, 5000, 20000, dtype="f16", page=16),
        # one sequence decoding over a short context: latency
        _cached("decode_1", "attention", 1, 1, 777, 777, dtype="f16", window=0, sinks=0),
        # a batch decoding in continuous batching: lengths between a short prompt and a long document
        _cached("decode_64", "attention", 64, 64, 100, 8000, window=0, sinks=0),
        # eight long conversations that attend to the last 4096 tokens and to the first 4, multi-query heads
        _cached("window_8", "attention", 8, 8, 20000, 40000, kv_heads=2, group=16, page=16, window=4096, sinks=4),
        # five drafted tokens verified in each of sixteen sequences
        _cached("verify_16", "attention", 16, 80, 500, 4000, page=32, window=0, sinks=0),
        # prompts of uneven lengths, the first parts of which are in the cache already
        _cached("prefill_4096", "attention", 3, 4096, 1500, 4500, window=0, sinks=0),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    """One more case: rows and tokens from one to a full batch, contexts from a few tokens to long ones, every type and layout."""
    while True:
        op = rng.choice(("norm", "norm", "append", "append", "read", "attention", "attention", "attention"))
        if op == "norm":
            group = rng.choice((0, 16, 32, 64, 128, 128, 128))
            hidden = 128 * _log_int(rng, 4, 128)
            case = {"op": op, "rows": _log_int(rng, 1, 8192), "hidden": hidden, "dtype": rng.choice(("bf16", "bf16", "f16", "f32")), "group": group,
                    "residual": rng.random() < 0.7}
            if case["rows"] * hidden <= 8192 * 4096:
                return case
            continue
        dim = rng.choice((64, 128, 128, 256))
        case = {"op": op, "batch": _log_int(rng, 1, 64), "dtype": rng.choice(("bf16", "bf16", "f16")), "kv_heads": rng.choice((1, 2, 4, 8)),
                "group": rng.choice((1, 2, 4, 5, 8, 16)), "dim": dim, "page": rng.choice((16, 32, 64, 64, 128))}
        if op == "read":
            case["dtype"] = rng.choice(("bf16", "f16", "f32"))
        case["len_hi"] = _log_int(rng, 1, 40000)
        case["len_lo"] = rng.randint(max(1, case["len_hi"] // 8), case["len_hi"])
        tokens = case["batch"] * case["len_hi"]
        if tokens * case["kv_heads"] * dim > (100000 if op == "read" else 64 * 8000) * 8 * 128:
            continue
        kind = rng.random()
        if op == "read":
            case["new"] = 0
        elif kind < 0.4:
            case["new"] = case["batch"]
        elif kind < 0.6:
            case["new"] = case["batch"] * min(case["len_lo"], rng.randint(2, 16))
        else:
            case["new"] = min(_log_int(rng, 1, 4096), case["batch"] * case["len_lo"])
        if op == "append":
            case["rotary"] = rng.choice((dim, dim, dim // 2, 32))
            case["interleaved"] = rng.random() < 0.4
            if case["new"] * case["kv_heads"] * case["group"] * dim > 4096 * 32 * 128 or tokens * case["kv_heads"] * dim > 64 * 2000 * 8 * 128:
                continue
        if op == "attention":
            windowed = rng.random() < 0.4
            case["window"] = _log_int(rng, 1, 8192) if windowed else 0
            case["sinks"] = rng.choice((0, 1, 4, 77)) if windowed else 0
            largest = 4096 * 3200 * 32 * 128
            if case["new"] * case["len_hi"] * case["kv_heads"] * case["group"] * dim > largest:
                continue
            # the plain form's score matrix
            if case["batch"] * -(-case["new"] // case["batch"]) * 2 * case["len_hi"] * case["kv_heads"] * case["group"] > 2 ** 30:
                continue
        return case


def _lengths(case):
    """(new tokens, length with them) of each sequence: whole numbers that the case alone fixes, uneven where it says so."""
    batch, lo, hi = case["batch"], case["len_lo"], case["len_hi"]
    lens = [hi if batch == 1 else lo + round((hi - lo) * ((i * 0.6180339887 + 0.3) % 1.0)) for i in range(batch)]
    new = [case["new"] // batch] * batch
    new[-1] += case["new"] - sum(new)
    # every second sequence hands a third of its new tokens to the one before it, where both have room
    for i in range(1, batch, 2):
        give = min(new[i] // 3, max(0, lens[i - 1] - new[i - 1]))
        new[i] -= give
        new[i - 1] += give
    lens = [max(a, b) for a, b in zip(lens, new)]
    return new, lens


# ---------------------------------------------------------------------------- states
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _cache(case, lens, g):
    """A pool with a tenth more pages than are in use, in no order; pages hold codes of normal values, scales of a few binades."""
    batch, page, heads, dim = case["batch"], case["page"], case["kv_heads"], case["dim"]
    used = [-(-n // page) for n in lens]
    pages = sum(used) + sum(used) // 10 + 1
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    width = max(used)
    count = torch.tensor(used, device="cuda")
    first = torch.cumsum(count, 0) - count
    column = torch.arange(width, device="cuda")
    at = first[:, None] + column[None, :]
    table = torch.where(column[None, :] < count[:, None], order[at.clamp(max=pages - 1)], torch.full_like(at, -1, dtype=torch.int32))

    def codes(shape):
        out = torch.empty(shape, dtype=FP8, device="cuda")
        for part in out.split(max(1, (1 << 27) // (heads * page * dim))):
            part.copy_((torch.randn(part.shape, generator=g, device="cuda") * 100).clamp(-E4M3_MAX, E4M3_MAX))
        return out

    def scales():
        return torch.exp2(torch.randint(-8, -5, (pages, heads), generator=g, device="cuda").float())

    return {"k": codes((pages, heads, page, dim)), "v": codes((pages, heads, dim, page)), "k_scale": scales(), "v_scale": scales()}, table


def rotary_table(positions, rotary, base=500000.0):
    """cos and sin of every position's angles, side by side: angles in float64, entries in float32."""
    freq = base ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq[None, :]
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "norm":
        t, shape = TYPES[case["dtype"]], (case["rows"], case["hidden"])
        x = torch.randn(shape, generator=g, device="cuda")
        x = torch.where(torch.rand(shape, generator=g, device="cuda") < 1e-3, x * 20, x)  # (activations have outliers)
        state = {"x": x.to(t), "weight": (1 + 0.2 * torch.randn(case["hidden"], generator=g, device="cuda")).to(t), "residual": None, "scale": None}
        if case["residual"]:
            state["residual"] = (3 * torch.randn(shape, generator=g, device="cuda")).to(t)
        if not case["group"]:
            state["scale"] = torch.tensor([0.03], device="cuda")  # calibrated: the largest values saturate
        return {"case": case, **state}
    new, lens = _lengths(case)
    cache, table = _cache(case, lens, g)
    state = {"case": case, "cache": cache, "table": table, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    if case["op"] == "read":
        indptr = [0]
        for n in lens:
            indptr.append(indptr[-1] + n)
        state.update(indptr=torch.tensor(indptr, dtype=torch.int32, device="cuda"), total=indptr[-1])
        return state
    indptr = [0]
    for n in new:
        indptr.append(indptr[-1] + n)
    t, heads, total, dim = TYPES[case["dtype"]], case["kv_heads"], indptr[-1], case["dim"]
    q_heads = heads * case["group"]
    # q, k and v as the QKV projection leaves them: side by side in one row per token
    qkv = torch.randn((total, q_heads + 2 * heads, dim), generator=g, device="cuda")
    qkv = (qkv * torch.exp2(torch.randint(-2, 3, (1, q_heads + 2 * heads, 1), generator=g, device="cuda").float())).to(t)
    state.update(indptr=torch.tensor(indptr, dtype=torch.int32, device="cuda"), q=qkv[:, :q_heads], k=qkv[:, q_heads:q_heads + heads],
                 v=qkv[:, q_heads + heads:], longest=max(new))
    if case["op"] == "append":
        state["rope"] = rotary_table(table.shape[1] * case["page"], case["rotary"])
    return state


# ---------------------------------------------------------------------------- plain forms
def _plain_norm(state):
    case, x, w = state["case"], state["x"].float(), state["weight"].float()
    if state["residual"] is not None:
        x = x + state["residual"].float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    out = {}
    if state["residual"] is not None:
        out["residual"] = x.to(state["x"].dtype)
    if case["group"]:
        groups = y.unflatten(-1, (-1, case["group"]))
        scale = groups.abs().amax(-1) / E4M3_MAX
        scale = torch.where(scale == 0, torch.ones_like(scale), scale)
        out["q"] = (groups / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).flatten(-2).to(FP8)
        out["scales"] = scale
    else:
        out["q"] = (y / state["scale"]).clamp(-E4M3_MAX, E4M3_MAX).to(FP8)
    return out


def _token_places(state):
    """For each new token: its sequence, its position, its page and its place in the page."""
    indptr, lens, page = state["indptr"].long(), state["lens"].long(), state["case"]["page"]
    token = torch.arange(state["q"].shape[0], device="cuda")
    seq = torch.searchsorted(indptr[1:], token, right=True)
    position = lens[seq] - (indptr[seq + 1] - token)
    return seq, position, state["table"].long()[seq, position // page], position % page


def _rotated(x, cos, sin, interleaved):
    half = cos.shape[-1]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, rest], -1)


def _page_scale(amax):
    """The smallest power of two that brings amax within e4m3's range."""
    mantissa, exponent = torch.frexp(amax)
    exponent = exponent - 9 + (mantissa > 0.875)  # 448 = 0.875 * 2^9
    exponent = torch.where(amax == 0, torch.full_like(exponent, MIN_EXPONENT), exponent)
    return torch.exp2(exponent.clamp(MIN_EXPONENT, MAX_EXPONENT).to(amax.dtype))


def _plain_append(state):
    case, cache = state["case"], state["cache"]
    seq, position, page, slot = _token_places(state)
    half = case["rotary"] // 2
    cos, sin = state["rope"][position, None, :half], state["rope"][position, None, half:]
    q = _rotated(state["q"].float(), cos, sin, case["interleaved"])
    k = _rotated(state["k"].float(), cos, sin, case["interleaved"])
    v = state["v"].float()
    pages, heads = cache["k_scale"].shape
    # slots of a touched page that hold earlier tokens
    kept = torch.full((pages,), case["page"], device="cuda").scatter_reduce(0, page, slot, "amin")
    touched = torch.zeros(pages, dtype=torch.bool, device="cuda").index_fill(0, page, True)
    place = torch.arange(case["page"], device="cuda")
    earlier = touched[:, None] & (place[None, :] < kept[:, None])
    for name, x, shape in (("k", k, (pages, 1, -1, 1)), ("v", v, (pages, 1, 1, -1))):
        codes, old = cache[name], cache[name + "_scale"]
        need = torch.zeros((pages, heads), device="cuda").scatter_reduce(0, page[:, None].expand(-1, heads), x.abs().amax(-1), "amax")
        scale = _page_scale(need)
        scale = torch.where((kept > 0)[:, None], torch.maximum(scale, old), scale)
        scale = torch.where(touched[:, None], scale, old)
        moved = (codes.float() * (old / scale)[:, :, None, None]).to(FP8)
        codes.copy_(torch.where(earlier.view(shape).expand_as(codes), moved.view(torch.uint8), codes.view(torch.uint8)).view(FP8))
        new = (x / scale[page][..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(FP8).view(torch.uint8)
        if name == "k":
            codes.view(torch.uint8)[page, :, slot] = new
        else:
            codes.view(torch.uint8)[page, :, :, slot] = new
        old.copy_(scale)
    return {"q": q.to(state["q"].dtype), **cache}


def _gathered(state, name):
    """One of a cache's halves as (sequence, head, token, element), in float32."""
    cache, table = state["cache"], state["table"].long().clamp(min=0)
    x = cache[name][table].float() * cache[name + "_scale"][table][..., None, None]
    if name == "v":
        x = x.transpose(-1, -2)
    return x.transpose(1, 2).flatten(2, 3)


def _plain_read(state):
    lens, t = state["lens"].long(), TYPES[state["case"]["dtype"]]
    live = torch.arange(state["table"].shape[1] * state["case"]["page"], device="cuda")[None, :] < lens[:, None]
    return {name: _gathered(state, name).transpose(1, 2)[live].to(t) for name in ("k", "v")}


def _plain_attention(state):
    case, q = state["case"], state["q"]
    seq, position, _, _ = _token_places(state)
    row = torch.arange(q.shape[0], device="cuda") - state["indptr"].long()[seq]
    k, v = _gathered(state, "k"), _gathered(state, "v")
    batch, heads, dim = case["batch"], case["kv_heads"], case["dim"]
    padded = torch.zeros((batch, state["longest"], heads, case["group"], dim), device="cuda")
    padded[seq, row] = q.float().unflatten(1, (heads, case["group"]))
    at = torch.full((batch, state["longest"]), -1, dtype=torch.long, device="cuda")
    at[seq, row] = position
    padded = padded.permute(0, 2, 1, 3, 4).flatten(2, 3)  # (sequence, kv head, row and head of the group, element)
    scores = torch.matmul(padded, k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(dim))
    key = torch.arange(k.shape[2], device="cuda")
    seen = key[None, None, :] <= at[..., None]
    if case["window"]:
        seen = seen & ((at[..., None] - key < case["window"]) | (key < case["sinks"]))
    seen = seen[:, None, :, None, :].expand(-1, 1, -1, case["group"], -1).flatten(2, 3)
    scores = scores.masked_fill_(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    scores = scores.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores, v) / torch.where(total == 0, torch.ones_like(total), total)
    out = out.unflatten(2, (state["longest"], case["group"])).permute(0, 2, 1, 3, 4).flatten(2, 3)
    return out[seq, row].to(q.dtype)


# ---------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if not own:
        return {"norm": _plain_norm, "append": _plain_append, "read": _plain_read, "attention": _plain_attention}[case["op"]](state)
    from tilegym_amd import ops

    if case["op"] == "norm":
        got = ops.rms_norm_quant(state["x"], state["weight"], EPS, residual=state["residual"], group_size=case["group"] or None, scale=state["scale"])
        out = {"q": got[0]}
        if case["group"]:
            out["scales"] = got[1]
        if case["residual"]:
            out["residual"] = got[2]
        return out
    cache = ops.KVCache(**state["cache"])
    if case["op"] == "append":
        q = ops.kv_cache_append(cache, state["k"], state["v"], state["table"], state["lens"], state["indptr"], q=state["q"], rope=state["rope"],
                                interleaved=case["interleaved"])
        return {"q": q, **state["cache"]}
    if case["op"] == "read":
        k, v = ops.kv_cache_read(cache, state["table"], state["indptr"], state["total"], out_dtype=TYPES[case["dtype"]])
        return {"k": k, "v": v}
    return ops.kv_cache_attention(state["q"], cache, state["table"], state["lens"], state["indptr"], window=case["window"], sink_tokens=case["sinks"])


# ---------------------------------------------------------------------------- what a pass cannot do without
def _seen_by(case, n, length):
    """(key, query) pairs that one sequence's n new tokens see, and the keys that any of them sees."""
    window, sinks = case["window"], case["sinks"]
    if not window:
        return n * (length - n) + n * (n + 1) // 2, length
    pairs = 0
    for p in range(length - n, length):
        recent = min(window, p + 1)
        pairs += recent + min(sinks, p + 1 - recent)
    first = max(0, length - n - window + 1)
    return pairs, length - first + min(sinks, first)


def work(case):
    if case["op"] == "norm":
        n, size = case["rows"] * case["hidden"], SIZE[case["dtype"]]
        moved = n * size * (3 if case["residual"] else 1) + n + case["hidden"] * size + (4 * n // case["group"] if case["group"] else 4)
        return {"bytes": moved, "flops": 6 * n}
    new, lens = _lengths(case)
    heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    size = SIZE[case["dtype"]]
    if case["op"] == "read":
        return {"bytes": sum(lens) * 2 * heads * dim * (1 + size) + sum(-(-n // page) for n in lens) * (8 * heads + 4), "flops": sum(lens) * 2 * heads * dim}
    total, q_heads = sum(new), heads * case["group"]
    if case["op"] == "append":
        moved = total * dim * (2 * q_heads * size + 2 * heads * (size + 1)) + total * 4 * case["rotary"]
        return {"bytes": moved, "flops": total * (q_heads + heads) * 3 * case["rotary"] + total * 4 * heads * dim}
    pairs, keys = (sum(x) for x in zip(*(_seen_by(case, n, length) for n, length in zip(new, lens) if n)))
    return {"bytes": keys * heads * 2 * dim + keys // page * heads * 8 + 2 * total * q_heads * dim * size, "flops": 4 * pairs * q_heads * dim}


# ---------------------------------------------------------------------------- in 64 bits
def _exact_norm(state):
    case = state["case"]
    total = state["x"].double() if state["residual"] is None else state["x"].double() + state["residual"].double()
    power = total.square().sum(-1, keepdim=True) / case["hidden"]
    y = state["weight"].double() * (total / (power + EPS).sqrt())
    out = {"residual": total} if case["residual"] else {}
    if not case["group"]:
        return {**out, "q": (y / state["scale"].double()).clamp(-E4M3_MAX, E4M3_MAX)}
    blocks = y.reshape(case["rows"], -1, case["group"])
    scales = blocks.abs().max(-1).values / E4M3_MAX
    return {**out, "q": (blocks / scales.masked_fill(scales == 0, 1.0)[..., None]).reshape(y.shape), "scales": scales.masked_fill(scales == 0, 1.0)}


def _turn(x, row, interleaved):
    """The rotary rule on one sequence's tokens (tokens, heads, elements) with their table rows, as a product of complex numbers."""
    r = row.shape[1]
    turn = torch.complex(row[:, : r // 2].double(), row[:, r // 2:].double())[:, None, :]
    x = x.double()
    if interleaved:
        y = torch.view_as_real(torch.complex(x[..., 0:r:2], x[..., 1:r:2]) * turn).reshape(*x.shape[:2], r)
    else:
        y = torch.complex(x[..., : r // 2], x[..., r // 2: r]) * turn
        y = torch.cat([y.real, y.imag], -1)
    return torch.cat([y, x[..., r:]], -1)


def _exact_append(state):
    case, P = state["case"], state["case"]["page"]
    new, lens = _lengths(case)
    out = {name: t.double() for name, t in state["cache"].items()}
    q_out = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda")
    table, at = state["table"].tolist(), 0
    for b, n in enumerate(new):
        start = lens[b] - n
        rows = state["rope"][start:lens[b]]
        q_out[at:at + n] = _turn(state["q"][at:at + n], rows, case["interleaved"])
        k, v = _turn(state["k"][at:at + n], rows, case["interleaved"]), state["v"][at:at + n].double()
        for first in range(start // P * P, lens[b], P):
            lo, hi, page = max(first, start), min(first + P, lens[b]), table[b][first // P]
            for name, x in (("k", k[lo - start:hi - start]), ("v", v[lo - start:hi - start])):
                codes, scale = out[name][page], out[name + "_scale"][page]
                if name == "v":
                    codes = codes.transpose(1, 2)
                top = x.abs().amax((0, 2))
                need = torch.exp2(torch.ceil(torch.log2(top / E4M3_MAX)).clamp(MIN_EXPONENT, MAX_EXPONENT))
                chosen = torch.maximum(need, scale) if lo > first else need
                codes[:, : lo - first] *= (scale / chosen)[:, None, None]
                codes[:, lo - first:hi - first] = (x / chosen[None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).transpose(0, 1)
                scale.copy_(chosen)
        at += n
    return {"q": q_out, **out}


def _sequence(state, b, length, name):
    """(heads, tokens, elements) of one sequence's keys or values."""
    P = state["case"]["page"]
    pages = state["table"][b, : -(-length // P)].long()
    x = state["cache"][name][pages].double() * state["cache"][name + "_scale"][pages].double()[:, :, None, None]
    x = x.permute(1, 0, 2, 3) if name == "k" else x.permute(1, 0, 3, 2)
    return x.reshape(x.shape[0], -1, state["case"]["dim"])[:, :length]


def _exact_read(state):
    _, lens = _lengths(state["case"])
    return {name: torch.cat([_sequence(state, b, n, name).transpose(0, 1) for b, n in enumerate(lens)]) for name in ("k", "v")}


def _exact_attention(state):
    case = state["case"]
    new, lens = _lengths(case)
    out, at = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda"), 0
    for b, (n, length) in enumerate(zip(new, lens)):
        if not n:
            continue
        k, v = _sequence(state, b, length, "k"), _sequence(state, b, length, "v")
        p = torch.arange(length - n, length, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")[None, :]
        hidden = j > p
        if case["window"]:
            hidden = hidden | ((j <= p - case["window"]) & (j >= case["sinks"]))
        for h in range(case["kv_heads"] * case["group"]):
            s = state["q"][at:at + n, h].double() @ k[h // case["group"]].t().contiguous() / math.sqrt(case["dim"])
            out[at:at + n, h] = torch.softmax(s.masked_fill(hidden, float("-inf")), -1) @ v[h // case["group"]]
        at += n
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"norm": _exact_norm, "append": _exact_append, "read": _exact_read, "attention": _exact_attention}[case["op"]](state)
