"""What the ways to the experts and back do with derivatives that they do not have."""

import gc
import os

import pytest
import torch
from torch.autograd import forward_ad

from tilegym_amd import _lib, ops

from .test_int8_ops import gen, routing


def _order(tokens, k):
    rows = torch.arange(tokens * k, dtype=torch.int32).view(tokens, k)
    return ops.MoeOrder(torch.tensor([0, tokens * k], dtype=torch.int32), rows, rows.flatten())


def _refusals(order, x, y, w, dual):
    t = torch.ops.tilegym_hip
    calls = [lambda: ops.moe_permute(dual(x), order), lambda: ops.moe_unpermute(dual(y), order), lambda: ops.moe_unpermute(dual(y), order, w),
             lambda: ops.moe_unpermute(y, order, dual(w))]
    calls += [lambda: ops.moe_permute_backward(dual(y), order), lambda: ops.moe_unpermute_backward(dual(x), y, order, w), lambda: ops.moe_unpermute_backward(x, dual(y), order, w),
              lambda: ops.moe_unpermute_backward(x, y, order, dual(w))]
    if x.is_cuda:
        calls += [lambda: t.moe_permute(dual(x), order.rows), lambda: t.moe_unpermute(y, order.rows, dual(w))]
    for call in calls:
        with pytest.raises(NotImplementedError):
            call()


def test_forward_mode_is_refused():
    """Not a value without its tangent; in front of everything else that is looked at."""
    x, y, w = torch.zeros(3, 8), torch.zeros(6, 8), torch.ones(3, 2)
    with forward_ad.dual_level():
        for leaf in (False, True):
            _refusals(_order(3, 2), x, y, w, lambda v: forward_ad.make_dual(v.clone().requires_grad_(leaf), torch.ones_like(v)))
            with torch.no_grad(), pytest.raises(NotImplementedError):
                ops.moe_permute(forward_ad.make_dual(x, torch.ones_like(x)), _order(3, 2))
        for call in (lambda: ops.moe_permute(x, _order(3, 2)), lambda: ops.moe_unpermute(y, _order(3, 2), w)):
            with pytest.raises(RuntimeError, match="HIP device"):  # (tensors without a tangent go on to the check of their device)
                call()


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_forward_mode_is_refused_on_a_device(device, monkeypatch, native):
    if not native:
        monkeypatch.setattr(_lib, "native_path", lambda: False)
    order = ops.moe_sort(routing(5, 4, 2, 1).to(device), 4)
    x, y, w = (torch.randn(*s, generator=gen(i)).to(device) for i, s in enumerate(((5, 64), (10, 64), (5, 2))))
    with forward_ad.dual_level():
        for leaf in (False, True):
            _refusals(order, x, y, w, lambda v: forward_ad.make_dual(v.clone().requires_grad_(leaf), torch.ones_like(v)))
        assert torch.equal(ops.moe_unpermute(ops.moe_permute(x, order), order), 2 * x)
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda v: ops.moe_permute(v, order), (x,), (x,))


# ---------------------------------------------------------------------------- leaves under capture
def test_leaves_without_a_device():
    """No capture is asked for where no device has been used: shapes of graphs are inferred, and tensors of the host are refused for what they are."""
    import subprocess
    import sys
    code = """
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from tilegym_amd import ops
t = torch.ops.tilegym_hip
with FakeTensorMode():
    x, rows = torch.empty(7, 40, device="cuda", requires_grad=True), torch.empty(7, 3, dtype=torch.int32, device="cuda")
    w = torch.empty(7, 3, device="cuda", requires_grad=True)
    y = t.moe_unpermute(t.moe_permute(x, rows), rows, w)
    assert y.shape == (7, 40) and y.requires_grad
assert not torch.cuda.is_initialized()
rows = torch.zeros(2, 1, dtype=torch.int32)
try:
    ops.moe_permute(torch.zeros(2, 8, requires_grad=True), ops.MoeOrder(rows, rows, rows))
except RuntimeError as e:
    assert "HIP device" in str(e), e
else:
    raise AssertionError
"""
    # (a process of its own: the others' may have used a device)
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=110, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.gpu
def test_leaf_held_by_stream(device):
    """A leaf is held by a graph that lives on another stream than the current one, and not by one on the same."""
    x, side = torch.zeros(3, device=device, requires_grad=True), torch.cuda.Stream()
    held = _lib.native.leaf_held
    assert not held(x)
    y = x * 2
    assert not held(x)
    with torch.cuda.stream(side):
        assert held(x)
    del y
    with torch.cuda.stream(side):
        assert not held(x)
        y = x * 2
        assert not held(x)
    assert held(x)


def _captured(step, leaves, inputs):
    """The step's gradients, captured and replayed over new inputs with eager steps between, against the eager ones."""
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
            for i, t in enumerate(leaves + inputs):
                t.copy_(torch.rand(t.shape, generator=gen(10 * seed + i)))
        graph.replay()
        got = [v.clone() for v in grads]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_a_leaf_used_twice_in_a_captured_step(device):
    """A residual beside the experts, weights that two layers share: the second use finds the first one's graph, on the stream of the capture."""
    tokens, experts, k, h = 30, 8, 2, 128
    order = ops.moe_sort(routing(tokens, experts, k, 1).to(device), experts)
    x = torch.randn(tokens, h, generator=gen(1)).to(device).requires_grad_()
    w = torch.rand(tokens, k, generator=gen(2)).to(device).requires_grad_()
    g = torch.randn(tokens, h, generator=gen(3)).to(device)

    def step():
        made = x * 2 + ops.moe_unpermute(ops.moe_permute(x, order) * 3, order, w)
        made = made + ops.moe_unpermute(ops.moe_permute(made, order) * 2, order, w)
        return torch.autograd.grad(made, (x, w), g)

    _captured(step, [x, w], [g])


@pytest.mark.gpu
def test_captures_through_torchs_dispatcher(device):
    """As the direct calls: while an eager graph of a leaf lives on another stream the capture is refused (the refused ones run no backward pass); without one a
    step is captured."""
    t = torch.ops.tilegym_hip
    tokens, experts, k, h = 30, 8, 2, 128
    rows = ops.moe_sort(routing(tokens, experts, k, 1).to(device), experts).rows
    x = torch.randn(tokens, h, generator=gen(1)).to(device).requires_grad_()
    w = torch.rand(tokens, k, generator=gen(2)).to(device).requires_grad_()
    g = torch.randn(tokens, h, generator=gen(3)).to(device)
    held = t.moe_permute(x, rows), t.moe_unpermute(t.moe_permute(g, rows), rows, w)
    torch.cuda.synchronize()
    for call in (lambda: t.moe_permute(x, rows), lambda: t.moe_unpermute(t.moe_permute(g, rows), rows, w)):
        with pytest.raises(RuntimeError, match="eager graph of this leaf"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                torch.zeros(1, device=device)
                call()
    del held
    gc.collect()

    def step():
        made = x * 2 + t.moe_unpermute(t.moe_permute(x, rows) * 3, rows, w)
        return torch.autograd.grad(t.moe_unpermute(t.moe_permute(made, rows) * 2, rows, w), (x, w), g)

    _captured(step, [x, w], [g])


@pytest.mark.gpu
def test_an_eager_graph_on_the_capturing_stream(device):
    """What is documented beside the refusal: a leaf whose eager graph lives on the stream that captures is taken, forwards and backwards."""
    tokens, experts, k, h = 30, 8, 2, 128
    order = ops.moe_sort(routing(tokens, experts, k, 1).to(device), experts)
    x = torch.randn(tokens, h, generator=gen(1)).to(device).requires_grad_()
    w = torch.rand(tokens, k, generator=gen(2)).to(device).requires_grad_()
    g = torch.randn(tokens, h, generator=gen(3)).to(device)

    def step():
        return torch.autograd.grad(ops.moe_unpermute(ops.moe_permute(x, order) * 2, order, w), (x, w), g)

    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        want = step()
        held = ops.moe_permute(x, order), ops.moe_unpermute(ops.moe_permute(g, order), order, w)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        grads = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, want))
        for t in grads:
            t.zero_()
    assert held[0].requires_grad and held[1].requires_grad
