"""The int8 products and the routing as programs call them: through torch's dispatcher, with gradients under capture, over operands past 32-bit offsets, from
several graphs and streams, and over drawn sizes."""

import gc
import random

import pytest
import torch

from oracle import int8_reference as R
from tilegym_amd import _lib, ops

from .test_int8_ops import BF16, F16, F32, bits, codes, gen, near, routing, scales


def test_sort_refuses_a_workspace_that_is_too_small():
    d, L, i32 = _lib._desc, _lib.load(), torch.int32
    n, experts = 40000, 8
    need = L.tg_moe_sort_workspace_bytes(n, experts)
    assert need >= 4 * (experts + 1) and L.tg_moe_sort_workspace_bytes(100, experts) == 0 and L.tg_moe_sort_workspace_bytes(n, 0) == 0
    ids, ptr, slots = torch.zeros(n, 1, dtype=i32), torch.zeros(experts + 1, dtype=i32), torch.zeros(n, dtype=i32)

    def rc(ws):
        return L.tg_moe_sort(d(ids), experts, d(ptr), d(slots), d(slots), d(ws), 9999, 0)

    assert rc(None) == -6 and rc(torch.zeros(need - 1, dtype=torch.uint8)) == -6
    assert rc(torch.zeros(need + 8, dtype=torch.uint8)[8:]) == -6  # not at a 16-byte address
    assert rc(torch.zeros(need, dtype=torch.uint8)) == -4          # everything is in order up to the device


def test_tensors_without_elements_are_contiguous():
    """Whatever their strides: an expanded gradient of no tokens, say."""
    d = _lib._desc
    x = torch.zeros(1, 1).expand(0, 16)
    assert x.stride() == (0, 0) or x.is_contiguous()
    assert _lib.load().tg_int8_quant(d(torch.zeros(0, 16, dtype=torch.int8)), d(torch.zeros(0)), d(x), None, 0, 9999, 0) == 0


def test_more_rows_of_experts_than_are_counted_are_refused():
    import ctypes
    one, (cfg, n) = torch.zeros(1, dtype=torch.int8), _lib.make_cfg(None)

    def rc(m):
        def desc(t, *shape):
            d = _lib.make_tensor_desc(t)
            d.ndim = len(shape)
            for i, size in enumerate(shape):
                d.shape[i], d.strides[i] = size, 1
                for other in shape[i + 1:]:
                    d.strides[i] *= other
            return ctypes.byref(d)
        f32 = torch.zeros(1)
        return _lib.load().tg_int8_ragged_gemm(desc(torch.zeros(1, dtype=BF16), m, 8), desc(one, m, 16), desc(one, 2, 8, 16), desc(f32, 1), desc(f32, 1),
                                               desc(torch.zeros(1, dtype=torch.int32), 3), cfg, n, 9999, 0)

    assert rc(2 ** 29 - 1) == -4 and rc(2 ** 29) == -6  # (nothing is read: the device is refused behind all sizes)


def test_leaf_held():
    """What a capture asks about a leaf: whether a graph that still lives adds to its gradient."""
    _lib.load()
    if _lib.native is None:
        pytest.skip("needs the native module")
    x = torch.zeros(3, requires_grad=True)
    assert not _lib.native.leaf_held(x)
    y = x * 2
    assert _lib.native.leaf_held(x) and not _lib.native.leaf_held(torch.zeros(3))
    del y
    assert not _lib.native.leaf_held(x)


# ---------------------------------------------------------------------------- torch's dispatcher
def test_operators_infer_shapes_through_torchs_dispatcher():
    from torch._subclasses.fake_tensor import FakeTensorMode

    t = torch.ops.tilegym_hip
    with FakeTensorMode():
        e = lambda *s, dtype=BF16: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731
        i8, i32 = dict(dtype=torch.int8), dict(dtype=torch.int32)
        c = t.int8_gemm(e(2, 5, 64, **i8), e(24, 64, **i8), e(2, 5, dtype=F32), e(24, dtype=F32), None, F16)
        assert c.shape == (2, 5, 24) and c.dtype == F16
        c = t.int8_ragged_gemm(e(10, 64, **i8), e(4, 24, 64, **i8), e(10, dtype=F32), e(4, 24, dtype=F32), e(5, **i32), BF16)
        assert c.shape == (10, 24) and c.dtype == BF16
        for got, q_shape in ((t.int8_quant(e(2, 5, 64)), (2, 5, 64)), (t.int8_silu_mul_quant(e(2, 5, 64)), (2, 5, 32))):
            assert got[0].shape == q_shape and got[0].dtype == torch.int8 and got[1].shape == (2, 5) and got[1].dtype == F32
        order = t.moe_sort(e(7, 3, dtype=torch.int64), 9)
        assert [tuple(x.shape) for x in order] == [(10,), (7, 3), (21,)] and all(x.dtype == torch.int32 for x in order)
        rows = order[1]
        q, s = t.int8_permute_quant(e(7, 40), rows)
        assert q.shape == (21, 40) and s.shape == (21,)
        there = t.moe_permute(e(7, 40), rows)
        assert there.shape == (21, 40) and t.moe_unpermute(there, rows, None).shape == (7, 40)
        gx, gw = t.moe_unpermute_backward(e(7, 40), there, rows, e(7, 3, dtype=F32))
        assert gx.shape == (21, 40) and gx.dtype == BF16 and gw.shape == (7, 3) and gw.dtype == F32
        for bad in (lambda: t.int8_gemm(e(2, 64, **i8), e(24, 32, **i8), e(2, dtype=F32), e(24, dtype=F32), None, F16), lambda: t.int8_silu_mul_quant(e(2, 63)),
                    lambda: t.moe_permute(e(6, 40), rows), lambda: t.moe_unpermute(e(7, 40), rows, None)):
            with pytest.raises(ValueError):
                bad()
    with pytest.raises(NotImplementedError):
        t.int8_quant(torch.zeros(2, 8))


@pytest.mark.gpu
def test_operators_through_torchs_dispatcher(device):
    """The bits of the direct calls, and the same gradients."""
    tokens, experts, k, h = 40, 8, 3, 256
    t = torch.ops.tilegym_hip
    ids, x = routing(tokens, experts, k, 1, absent=True).to(device), torch.randn(tokens, h, generator=gen(2)).to(BF16).to(device)
    w, g = torch.rand(tokens, k, generator=gen(3)).to(device), torch.randn(tokens, h, generator=gen(4)).to(BF16).to(device)
    b, sb = codes((experts, 64, h), 5).to(device), scales((experts, 64), 6).to(device)
    order = ops.moe_sort(ids, experts)
    assert all(torch.equal(a, o) for a, o in zip(t.moe_sort(ids, experts), order))
    q, s = ops.moe_permute_quant_int8(x, order)
    assert all(torch.equal(a, o) for a, o in zip(t.int8_permute_quant(x, order.rows), (q, s)))
    live = int(order.indptr[-1])
    y = t.int8_ragged_gemm(q, b, s, sb, order.indptr, BF16)
    assert torch.equal(bits(y[:live]), bits(ops.ragged_int8_matmul(q, b, s, sb, order.indptr)[:live])) and not bool(y[live:].any())
    assert torch.equal(t.int8_gemm(q, b[0], s, sb[0], None, F32), ops.int8_matmul(q, b[0], s, sb[0], out_dtype=F32))
    for got, want in ((t.int8_quant(x), ops.quant_int8(x)), (t.int8_silu_mul_quant(x), ops.silu_mul_quant_int8(x))):
        assert all(torch.equal(a, o) for a, o in zip(got, want))

    grads = []
    for permute, unpermute in ((lambda v: ops.moe_permute(v, order), lambda v, u: ops.moe_unpermute(v, order, u)),
                               (lambda v: t.moe_permute(v, order.rows), lambda v, u: t.moe_unpermute(v, order.rows, u))):
        xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
        out = unpermute(permute(xl), wl)
        plain = unpermute(permute(xl), None)
        grads.append((out.detach(), plain.detach(), *torch.autograd.grad((out, plain), (xl, wl), (g, g))))
    assert all(torch.equal(a, o) for a, o in zip(*grads))
    torch.library.opcheck(t.moe_permute.default, (x.clone().requires_grad_(), order.rows))
    torch.library.opcheck(t.moe_unpermute.default, (ops.moe_permute(x, order).requires_grad_(), order.rows, w.clone().requires_grad_()))


# ---------------------------------------------------------------------------- gradients
@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("t", [BF16, F32])
def test_autograd_is_the_backward_operators(device, monkeypatch, native, t):
    """In native code and without it: the gradients' bits, expanded and strided gradients, each input alone, what a second derivative and a changed input do."""
    if not native:
        monkeypatch.setattr(_lib, "native_path", lambda: False)
    tokens, experts, k, h = 37, 8, 3, 72
    order = ops.moe_sort(routing(tokens, experts, k, 1, absent=True).to(device), experts)
    x = torch.randn(tokens, h, generator=gen(2)).to(t).to(device).requires_grad_()
    y = torch.randn(tokens * k, h, generator=gen(3)).to(t).to(device).requires_grad_()
    w = torch.rand(tokens, k, generator=gen(4)).to(device).requires_grad_()
    g = torch.randn(tokens, h, generator=gen(5)).to(t).to(device)
    gr = torch.randn(tokens * k, h, generator=gen(6)).to(t).to(device)
    with torch.no_grad():
        want_y, want_w = ops.moe_unpermute_backward(g, y, order, w)
        want_x, want_plain = ops.moe_permute_backward(gr, order), ops.moe_permute(g, order)
    there, back = ops.moe_permute(x, order), ops.moe_unpermute(y, order, w)
    assert there.requires_grad and back.requires_grad and there.grad_fn is not None
    assert torch.equal(bits(there.detach()), bits(ops.moe_permute(x.detach(), order)))
    assert torch.equal(torch.autograd.grad(there, x, gr, retain_graph=True)[0], want_x)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(back, (y, w), g, retain_graph=True), (want_y, want_w)))
    assert torch.equal(torch.autograd.grad(ops.moe_unpermute(y, order), y, g)[0], want_plain)
    assert torch.equal(torch.autograd.grad(ops.moe_unpermute(y.detach(), order, w), w, g)[0], want_w)
    assert torch.equal(torch.autograd.grad(ops.moe_unpermute(y, order, w.detach()), y, g)[0], want_y)
    strided = g.t().contiguous().t()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(back, (y, w), strided, retain_graph=True), (want_y, want_w)))
    one = torch.ones((), dtype=t, device=device)
    assert torch.equal(torch.autograd.grad(there, x, one.expand_as(there), retain_graph=True)[0], ops.moe_permute_backward(torch.ones_like(gr), order))
    with torch.no_grad():
        assert not ops.moe_permute(x, order).requires_grad and not ops.moe_unpermute(y, order, w).requires_grad
    # no second derivative: an error, not a wrong number
    for out, leaf, grad in ((there, x, gr), (back, y, g), (back, w, g)):
        (first,) = torch.autograd.grad(out, leaf, grad.clone().requires_grad_(), create_graph=True)
        assert first.requires_grad
        with pytest.raises(RuntimeError, match="differentiate"):
            first.float().sum().backward()
        with pytest.raises(RuntimeError):
            torch.autograd.grad(first.float().sum(), leaf)
    # what the backward pass reads has been changed
    out = ops.moe_unpermute(y, order, w)
    with torch.no_grad():
        y.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    for call in (lambda: ops.moe_permute(x[1:], order), lambda: ops.moe_permute(x.t().contiguous().t(), order), lambda: ops.moe_unpermute(y, order, w[:, :2]),
                 lambda: ops.moe_unpermute(y[1:], order), lambda: ops.moe_unpermute(y, order, w.cpu())):
        with pytest.raises((ValueError, _lib.TileGymHipError)):
            call()


# ---------------------------------------------------------------------------- gradients under capture
@pytest.mark.gpu
def test_forward_and_backward_captured(device):
    """A training step's forward and backward passes in one graph, replayed over new inputs with eager steps between; while an eager graph of a leaf
    lives, the capture is refused."""
    tokens, experts, k, h = 30, 8, 2, 128
    order = ops.moe_sort(routing(tokens, experts, k, 1).to(device), experts)
    x = torch.randn(tokens, h, generator=gen(1)).to(device).requires_grad_()
    w = torch.rand(tokens, k, generator=gen(2)).to(device).requires_grad_()
    g = torch.randn(tokens, h, generator=gen(3)).to(device)

    def step():
        return torch.autograd.grad(ops.moe_unpermute(ops.moe_permute(x, order) * 2, order, w), (x, w), g)

    held = ops.moe_permute(x, order), ops.moe_unpermute(ops.moe_permute(x.detach(), order), order, w)
    torch.cuda.synchronize()
    for call in (lambda: ops.moe_permute(x, order), lambda: ops.moe_unpermute(ops.moe_permute(g, order), order, w)):
        with pytest.raises(RuntimeError, match="eager graph of this leaf"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                torch.zeros(1, device=device)
                call()
    del held
    gc.collect()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = step()
    for seed in range(4, 8):
        with torch.no_grad():
            x.copy_(torch.randn(tokens, h, generator=gen(seed)))
            w.copy_(torch.rand(tokens, k, generator=gen(seed + 1)))
            g.copy_(torch.randn(tokens, h, generator=gen(seed + 2)))
        graph.replay()
        got = [t.clone() for t in grads]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------- several graphs
@pytest.mark.gpu
def test_two_graphs_replayed_at_once(device):
    """Graphs captured on one stream and replayed on two keep their scratch memory (a split K's partial sums, a long sort's counts) apart."""
    a, b = [codes((20, 4096), s).to(device) for s in (1, 2)], codes((256, 4096), 3).to(device)
    one = torch.full((1,), 0.01, device=device)
    ids = [torch.randint(0, 16, (20000, 2), generator=gen(s), dtype=torch.int32).to(device) for s in (4, 5)]
    cfg = dict(KERNEL="tiled", BLOCK_M=32, BLOCK_N=64, SPLIT_K=8)

    def run(i):
        return [(ops.int8_matmul(a[i], b, one, one, kernel_configs=cfg), *ops.moe_sort(ids[i], 16)) for _ in range(4)]

    want = [[[t.clone() for t in r] for r in run(i)] for i in (0, 1)]
    assert _lib.last_config() is not None and _lib.load().tg_moe_sort_workspace_bytes(40000, 16) > 0
    graphs, held = [], []
    for i in (0, 1):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(run(i))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for h, w in zip(held, want):
            assert all(torch.equal(x, y) for r, s in zip(h, w) for x, y in zip(r, s))


# ---------------------------------------------------------------------------- offsets past 32 bits
@pytest.mark.gpu
def test_rows_past_32_bit_offsets(device):
    """2.3 GB of rows against a small weight, and outputs of as many bytes: the last rows are those of a call over them alone."""
    k, n = 16384, 256
    m = 140_000
    a = torch.randint(-128, 128, (m, k), dtype=torch.int8, device=device)
    b, sa, sb = codes((n, k), 2).to(device), scales(m, 3).to(device), scales(n, 4).to(device)
    last = slice(m - 300, m)
    want = ops.int8_matmul(a[last].contiguous(), b, sa[last].contiguous(), sb)
    assert torch.equal(ops.int8_matmul(a, b, sa, sb)[last], want)
    for cfg in (dict(KERNEL="tiled", BLOCK_M=256, BLOCK_N=128), dict(KERNEL="fallback")):
        assert torch.equal(ops.int8_matmul(a, b, sa, sb, kernel_configs=cfg)[last], want)
    indptr = torch.tensor([0, 100, m - 300, m], dtype=torch.int32, device=device)
    b3, sb3 = torch.stack([b.flip(0), b.flip(1), b]), torch.stack([sb, sb, sb])
    for cfg in (None, dict(KERNEL="tiled", BLOCK_M=192, BLOCK_N=192), dict(KERNEL="tiled", BLOCK_M=256, BLOCK_N=256)):
        assert torch.equal(ops.ragged_int8_matmul(a, b3, sa, sb3, indptr, kernel_configs=cfg)[last], want)
    del a, b3
    # a weight of more bytes, its last rows
    b = torch.randint(-128, 128, (m, k), dtype=torch.int8, device=device)
    x, one = codes((40, k), 5).to(device), torch.full((1,), 0.01, device=device)
    want = ops.int8_matmul(x, b[last].contiguous(), one, sa[last].contiguous())
    assert torch.equal(ops.int8_matmul(x, b, one, sa)[:, last], want)
    assert torch.equal(ops.int8_matmul(x[:9], b, one, sa)[:, last], want[:9])
    # experts whose weights lie past them: rows of the last one
    e = torch.tensor([0] * 140 + [40], dtype=torch.int32, device=device)
    w = b.view(140, 1000, k)
    want = ops.int8_matmul(x, w[-1].contiguous(), one, one)
    for rows in (40, 7):
        e[-1] = rows
        assert torch.equal(ops.ragged_int8_matmul(x[:rows].contiguous(), w, one, one, e), want[:rows])


@pytest.mark.gpu
def test_routing_past_32_bit_offsets(device):
    tokens, k, h = 70_000, 8, 4096  # 560 000 rows of 4096
    ids = torch.randint(0, 64, (tokens, k), dtype=torch.int32, device=device)
    order = ops.moe_sort(ids, 64)
    x = torch.randint(0, 256, (tokens, 1), device=device).to(BF16).expand(tokens, h).contiguous()
    there = ops.moe_permute(x, order)
    slots = order.slots.long()
    assert torch.equal(there[:, 0], x[slots // k, 0]) and torch.equal(there[:, -1], x[slots // k, -1])
    q, s = ops.moe_permute_quant_int8(x, order)
    want = ops.quant_int8(x)
    assert torch.equal(q[:, -1], want[0][slots // k, -1]) and torch.equal(s, want[1][slots // k])
    w = torch.ones(tokens, k, device=device)
    assert torch.equal(ops.moe_unpermute(there, order, w), x * k)
    gx, gw = ops.moe_unpermute_backward(x, there, order, w)
    assert torch.equal(gx[:, -1], there[:, -1])
    assert torch.equal(gw, (x[:, :1].float() ** 2 * h).expand(tokens, k))  # (sums of equal powers of 2 ** 12 products: exact)
    q, s = ops.silu_mul_quant_int8(there)
    assert torch.equal(q[-5:], ops.silu_mul_quant_int8(there[-5:].contiguous())[0])


# ---------------------------------------------------------------------------- routings a router can make
@pytest.mark.gpu
@pytest.mark.parametrize("t", [BF16, F32])
def test_an_expert_twice_and_ids_past_32_bits(device, t):
    """A token that is sent to one expert in several slots, with weights of zero, below zero and infinite; ids whose low 32 bits are an expert's."""
    tokens, experts, k, h = 60, 6, 4, 136
    ids = torch.randint(0, experts, (tokens, k), generator=gen(1))
    ids[::3] = ids[::3, :1]                                        # four times the same
    ids[5, 1], ids[6, 2], ids[7, 0], ids[8] = 2 ** 32 + 1, -2 ** 33 + 2, 2 ** 62, -2 ** 63
    order = ops.moe_sort(ids.to(device), experts)
    indptr, rows, slots = R.ref_sort(ids, experts)
    assert order.indptr.tolist() == indptr and order.rows.flatten().tolist() == rows and order.slots.tolist() == slots
    rows = order.rows.cpu()
    assert [int((rows[i] < 0).sum()) for i in (5, 6, 7, 8)] == [1, 1, 1, 4]
    x = torch.randn(tokens, h, generator=gen(2)).to(t)
    there = ops.moe_permute(x.to(device), order)
    assert torch.equal(bits(there), bits(R.ref_permute(x, rows).to(t)))
    w = torch.randn(tokens, k, generator=gen(3))
    w[::4] = 0
    w[5, 1], w[8, 0] = float("nan"), float("inf")                  # of pairs without an expert
    y = torch.randn(tokens * k, h, generator=gen(4)).to(t)
    exact, size = R.ref_unpermute(y, rows, w)
    near(ops.moe_unpermute(y.to(device), order, w.to(device)), exact, size, t, k)
    assert not bool(ops.moe_unpermute(y.to(device), order, w.to(device))[8].any())
    g = torch.randn(tokens, h, generator=gen(5)).to(t)
    gx, gw = ops.moe_unpermute_backward(g.to(device), y.to(device), order, w.to(device))
    ex, ew, size = R.ref_unpermute_backward(g, y, rows, w)
    near(gx, ex, ex.abs(), t, 1)
    near(gw, ew, size, F32, h / 64 + 16)
    # an infinite weight of a pair that has an expert shows in its token, and there alone
    w[3, 0] = float("inf")
    out = ops.moe_unpermute(y.to(device), order, w.to(device))
    assert not bool(out[3].isfinite().any()) and bool(out[:3].isfinite().all()) and bool(out[4:].isfinite().all())


# ---------------------------------------------------------------------------- the layer in one call
@pytest.mark.gpu
@pytest.mark.parametrize("tokens,experts,k,h,i,dtype", [(1, 4, 2, 64, 32, BF16), (9, 64, 6, 256, 100, F16), (33, 8, 2, 250, 64, BF16), (700, 16, 4, 512, 192, BF16), (5000, 8, 6, 64, 48, F16)])
def test_layer_in_one_call_is_its_operators(device, monkeypatch, tokens, experts, k, h, i, dtype):
    x = torch.randn(tokens, h, generator=gen(1)).to(dtype).to(device)
    w1, w2 = codes((experts, 2 * i, h), 2).to(device), codes((experts, h, i), 3).to(device)
    s1, s2 = scales((experts, 2 * i), 4).to(device) / 50, scales((experts, h), 5).to(device)
    for absent, wt, it in ((False, F32, torch.int32), (True, BF16, torch.int64)):
        ids, w = routing(tokens, experts, k, 6, absent, dtype=it).to(device), torch.rand(tokens, k, generator=gen(7)).to(wt).to(device)
        got = ops.int8_moe(x, w1, w2, s1, s2, w, ids)
        order = ops.moe_sort(ids, experts)
        q, s = ops.moe_permute_quant_int8(x, order)
        q, s = ops.silu_mul_quant_int8(ops.ragged_int8_matmul(q, w1, s, s1, order.indptr, out_dtype=dtype))
        want = ops.moe_unpermute(ops.ragged_int8_matmul(q, w2, s, s2, order.indptr, out_dtype=dtype), order, w)
        assert torch.equal(bits(got), bits(want))
        with monkeypatch.context() as m:
            m.setattr(_lib, "native_path", lambda: False)
            assert torch.equal(bits(ops.int8_moe(x, w1, w2, s1, s2, w, ids)), bits(want))
    for bad in (dict(w2=w2[:-1]), dict(w1_scale=s1[:1, :3].contiguous()), dict(topk_weights=w[:, :1].contiguous()), dict(w1=w1[:, :-2].contiguous())):
        args = {**dict(hidden_states=x, w1=w1, w2=w2, w1_scale=s1, w2_scale=s2, topk_weights=w, topk_ids=ids), **bad}
        with pytest.raises((ValueError, _lib.TileGymHipError)):
            ops.int8_moe(**args)


# ---------------------------------------------------------------------------- nothing to do
@pytest.mark.gpu
def test_empty_sizes(device):
    f32 = lambda *s: torch.ones(*s, device=device)  # noqa: E731
    i8 = lambda *s: torch.zeros(*s, dtype=torch.int8, device=device)  # noqa: E731
    for tokens, k, h in ((0, 2, 64), (3, 0, 64), (3, 2, 0), (0, 0, 0)):
        order = ops.moe_sort(torch.zeros(tokens, k, dtype=torch.int32, device=device), 4)
        assert order.indptr.tolist() == [0] + [tokens * k] * 4
        x, y, w = f32(tokens, h), f32(tokens * k, h), f32(tokens, k)
        assert torch.equal(ops.moe_permute(x, order), y)
        assert torch.equal(ops.moe_unpermute(y, order), x * k) and torch.equal(ops.moe_unpermute(y, order, w), x * k)
        gx, gw = ops.moe_unpermute_backward(x, y, order, w)
        assert torch.equal(gx, y) and torch.equal(gw, w * h)
        if h:
            q, s = ops.moe_permute_quant_int8(x, order)
            assert q.shape == (tokens * k, h) and s.shape == (tokens * k,)
            xl = x.clone().requires_grad_()
            ops.moe_unpermute(ops.moe_permute(xl, order), order, w).sum().backward()
            assert torch.equal(xl.grad, x * k)
    assert ops.int8_matmul(i8(0, 64), i8(24, 64), f32(1), f32(24)).shape == (0, 24)
    assert ops.int8_matmul(i8(5, 64), i8(0, 64), f32(5), f32(1)).shape == (5, 0)
    assert ops.ragged_int8_matmul(i8(0, 64), i8(4, 24, 64), f32(0), f32(4, 24), torch.zeros(5, dtype=torch.int32, device=device)).shape == (0, 24)
    out = torch.full((6, 24), 3.0, dtype=BF16, device=device)
    ops.ragged_int8_matmul(i8(6, 64), i8(0, 24, 64), f32(6), f32(1), torch.zeros(1, dtype=torch.int32, device=device), out=out)
    assert bool((out == 3).all())  # rows of no expert, as there is none
    assert ops.quant_int8(f32(0, 64))[1].shape == (0,) and ops.silu_mul_quant_int8(f32(0, 64))[0].shape == (0, 32)
    none = torch.zeros(0, 2, dtype=torch.int32, device=device)
    assert ops.int8_moe(f32(0, 64).to(BF16), i8(4, 64, 64), i8(4, 64, 32), f32(4, 64), f32(4, 64), f32(0, 2), none).shape == (0, 64)
    # a layer none of whose experts is here; it has no gradient, in the router's weights either
    ids = torch.full((5, 2), -1, dtype=torch.int32, device=device)
    made = ops.int8_moe(f32(5, 64).to(BF16), i8(4, 64, 64), i8(4, 64, 32), f32(4, 64), f32(4, 64), f32(5, 2).requires_grad_(), ids)
    assert not bool(made.any()) and not made.requires_grad


@pytest.mark.gpu
def test_forced_streaming_over_more_passes_than_a_grid_has(device):
    """2^20 rows and more of few experts: the streaming form does not take them, the call still answers."""
    rows = 65600 * 16
    a, b = torch.randint(-128, 128, (rows, 16), dtype=torch.int8, device=device), codes((2, 8, 16), 1).to(device)
    sa, sb = torch.rand(rows, device=device), scales((2, 8), 2).to(device)
    ptr = torch.tensor([0, 100, rows], dtype=torch.int32, device=device)
    got = ops.ragged_int8_matmul(a, b, sa, sb, ptr, kernel_configs=dict(KERNEL="stream"))
    assert _lib.last_config()["KERNEL"] != 3
    assert torch.equal(bits(got[:100]), bits(_exact(a[:100], b[0], sa[:100], sb[0], BF16)))
    assert torch.equal(bits(got[100:]), bits(_exact(a[100:], b[1], sa[100:], sb[1], BF16)))


@pytest.mark.gpu
def test_experts_beyond_the_limit_are_refused(device):
    """Without an allocation of their number."""
    ids = torch.zeros(3, 2, dtype=torch.int32, device=device)
    for experts in (513, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 4, 10 ** 12, -1):
        before = torch.cuda.memory_allocated()
        with pytest.raises((_lib.TileGymHipError, OverflowError)):
            ops.moe_sort(ids, experts)
        assert torch.cuda.memory_allocated() == before


# ---------------------------------------------------------------------------- many rows
@pytest.mark.gpu
@pytest.mark.parametrize("k", [8, 500, 512, 1000, 1024, 1408, 1536, 2041, 2048])
@pytest.mark.parametrize("t", [BF16, F16, F32])
def test_quantizers_of_many_rows(device, k, t):
    """Rows enough for a wave each, of up to 256 vectors; the odd ones element by element."""
    rows = 2051
    x = torch.randn(rows, k, generator=gen(k)).to(t)
    x[5], x[6, k // 3], x[7, 0] = 0, float("nan"), float("inf")
    wq, ws = R.ref_quant(x)
    q, s = ops.quant_int8(x.to(device))
    assert torch.equal(q.cpu(), wq) and torch.equal(bits(s.nan_to_num(-1)), bits(ws.nan_to_num(-1)))
    order = ops.moe_sort(routing(rows, 16, 3, k, absent=True).to(device), 16)
    q, s = ops.moe_permute_quant_int8(x.to(device), order)
    live, slots = int(order.indptr[-1]), order.slots.cpu().long()
    token = slots[:live] // 3
    assert torch.equal(q[:live].cpu(), wq[token]) and torch.equal(bits(s[:live].nan_to_num(-1)), bits(ws[token].nan_to_num(-1)))
    assert not bool(q[live:].any()) and bool((s[live:] == 1).all())
    # the activation: the codes of few rows are those of many
    both = torch.randn(rows, 2 * k, generator=gen(k + 1)).to(t).to(device)
    q, s = ops.silu_mul_quant_int8(both)
    for part in (slice(0, 40), slice(1000, 1333), slice(rows - 1, rows)):
        pq, ps = ops.silu_mul_quant_int8(both[part].contiguous())
        assert torch.equal(q[part], pq) and torch.equal(bits(s[part]), bits(ps))


# ---------------------------------------------------------------------------- drawn sizes
def _exact(a, b, sa, sb, t):
    """The kernels' fp32 steps on the exact sum, on the GPU (sums of integers below 2^31 are exact in float64)."""
    return ((a.double() @ b.double().t()).float() * sa[:, None] * sb).to(t)


@pytest.mark.gpu
def test_drawn_products(device):
    rng = random.Random(3)
    for i in range(60):
        m = rng.choice((1, 2, 13, 16, 17, 31, 32, 33, 70, 150, 333, 700, 1500, 4000))
        n, k = rng.choice((8, 64, 72, 500, 1000, 2000, 4104)), rng.choice((16, 144, 256, 1000, 1024, 2064, 4096))
        t = rng.choice((BF16, F16, F32))
        a, b = codes((m, k), i).to(device), codes((n, k), i + 1).to(device)
        sa, sb = scales(m, i + 2).to(device), scales(n, i + 3).to(device)
        got = ops.int8_matmul(a, b, sa, sb, out_dtype=t)
        assert torch.equal(bits(got), bits(_exact(a, b, sa, sb, t))), (m, n, k, t, _lib.last_config())


@pytest.mark.gpu
def test_lengths_of_no_vectors_split(device):
    """Few tiles of the kernel that takes any length: its K is split, in parts that end inside a row's last bytes."""
    seen = set()
    for m, n, k in ((1, 4478, 3250), (2, 70, 7822), (64, 65, 4001), (65, 130, 2047), (200, 60, 16001), (30, 501, 1027), (513, 100, 4097), (5, 1, 131071)):
        a, b = codes((m, k), m).to(device), codes((n, k), n).to(device)
        sa, sb = scales(m, 3).to(device), scales(n, 4).to(device)
        for t in (BF16, F32):
            assert torch.equal(bits(ops.int8_matmul(a, b, sa, sb, out_dtype=t)), bits(_exact(a, b, sa, sb, t))), (m, n, k)
            got = _lib.last_config()
            assert got["KERNEL"] == 0
            seen.add(got["SPLIT_K"])
        bias = torch.randn(n, generator=gen(5)).to(device)
        exact = (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double() + bias.double()
        got = ops.int8_matmul(a, b, sa, sb, bias=bias, out_dtype=F32).double()
        # the sum's conversion, its product with the token's scale, the multiply-add
        assert bool(((got - exact).abs() <= 3.01 * 2.0 ** -24 * (exact.abs() + 2 * bias.double().abs())).all())
    assert 1 in seen and max(seen) > 8


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [9, 10, 11, 17, 19, 20, 33, 34, 35, 41, 42, 49, 50, 57])
def test_splits_that_do_not_divide_the_length(device, steps):
    """Every part of a split K has a share of it, whatever the scratch memory held: lengths that eight parts, or four, would leave one of empty."""
    k, seen = 128 * steps, set()
    for m, n in ((1, 72), (8, 64), (17, 64), (20, 130), (33, 256), (65, 128), (100, 256), (256, 64), (400, 64)):
        a, b = codes((m, k), m).to(device), codes((n, k), n).to(device)
        sa, sb = scales(m, 3).to(device), scales(n, 4).to(device)
        want = bits(_exact(a, b, sa, sb, BF16))
        for cfg in (None, dict(KERNEL="fallback"), dict(KERNEL="tiled", BLOCK_M=64, BLOCK_N=64, SPLIT_K=8), dict(KERNEL="stream", SPLIT_K=4)):
            dirty = [torch.full((16 << i,), 0x55, dtype=torch.uint8, device=device) for i in range(10, 18)]
            del dirty  # (the allocator's free blocks, of the scratch memory's sizes too)
            assert torch.equal(bits(ops.int8_matmul(a, b, sa, sb, kernel_configs=cfg)), want), (m, n, k, cfg, _lib.last_config())
            seen.add(_lib.last_config()["SPLIT_K"])
    assert max(seen) > 1


@pytest.mark.gpu
def test_drawn_products_over_experts(device):
    rng = random.Random(4)
    for i in range(40):
        experts, rows = rng.choice((1, 3, 8, 60, 130)), rng.choice((1, 10, 100, 500, 3000, 9000))
        n, k = rng.choice((8, 64, 264, 500, 1408)), rng.choice((16, 256, 400, 1024, 1408))
        ids = torch.randint(-1, experts, (rows, 1), generator=gen(i), dtype=torch.int32).to(device)
        if rng.random() < 0.3:
            ids[:rows // 2] = 0
        order = ops.moe_sort(ids, experts)
        a, b = codes((rows, k), i).to(device), codes((experts, n, k), i + 1).to(device)
        sa, sb = scales(rows, i + 2).to(device), scales((experts, n), i + 3).to(device)
        out = torch.full((rows, n), 5.0, dtype=BF16, device=device)
        ops.ragged_int8_matmul(a, b, sa, sb, order.indptr, out=out)
        ptr = order.indptr.tolist()
        for e in range(experts):
            part = slice(ptr[e], ptr[e + 1])
            assert torch.equal(bits(out[part]), bits(_exact(a[part], b[e], sa[part], sb[e], BF16))), (experts, rows, n, k, e, _lib.last_config())
        assert bool((out[ptr[-1]:] == 5).all())
