"""Gradients through the MXFP4 operators: recorded where there is one, in the Python and the C++ layer alike, and refused
at the backward pass where there is none."""

import pytest
import torch

from pulsarlm_amd import _host, ops
from tests import _mxfp4 as mx

pytestmark = pytest.mark.gpu

# The two layers, by (linear, its gradient, gated block, its gradient, W4A4 linear, W4A4 block).
PYTHON = (ops.gemm_mxfp4_cuda, ops.gemm_mxfp4_grad_cuda, ops.gated_mxfp4_cuda, ops.gated_mxfp4_grad_cuda, ops.gemm_mxfp4_w4a4_cuda,
          ops.mlp_mxfp4_w4a4_cuda)
HOST = (_host.gemm_mxfp4_cuda, _host.gemm_mxfp4_grad_cuda, lambda x, g, u, i, keep_gate_up=False:
        _host.gated_mxfp4_cuda(x, *g, *u, i, keep_gate_up)[slice(None) if keep_gate_up else 0],
        lambda dh, gu, g, u, k: _host.gated_mxfp4_grad_cuda(dh, gu, *g, *u, k), _host.gemm_mxfp4_w4a4_cuda,
        lambda x, g, u, d, i: _host.mlp_mxfp4_w4a4_cuda(x, *g, *u, *d, i))
LAYERS = pytest.mark.parametrize("layer", [PYTHON, HOST], ids=["python", "host"])


def parts(m, n=96, k=160, dtype=torch.bfloat16):
    return (mx.rows(m, k, dtype, seed=1), mx.rows(m, n, dtype, seed=2), mx.Weight(n, k, seed=3).packed, mx.Weight(n, k, seed=4).packed,
            mx.Weight(k, n, seed=5).packed)


def leaf(x):
    return x.clone().requires_grad_()


@LAYERS
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("m", [1, 70])
def test_linear_and_gated_record_their_gradient(m, dtype, layer):
    linear, linear_grad, gated, gated_grad, _, _ = layer
    x, dy, wg, wu, _ = parts(m, dtype=mx.DT[dtype])
    n, k = 96, 160
    at = leaf(x)
    y = linear(at, *wg, n)
    assert y.requires_grad and torch.equal(y, linear(x, *wg, n))
    y.backward(dy)
    assert torch.equal(at.grad, linear_grad(dy, *wg, k))
    # What autograd hands on is not always contiguous: a sum's gradient is one value, expanded.
    at = leaf(x)
    linear(at, *wg, n).sum().backward()
    assert torch.equal(at.grad, linear_grad(torch.ones_like(dy), *wg, k))

    h0, gate_up0 = gated(x, wg, wu, n, keep_gate_up=True)
    expected = gated_grad(dy, gate_up0, wg, wu, k)
    for keep in (False, True):
        at = leaf(x)
        out = gated(at, wg, wu, n, keep_gate_up=keep)
        h = out[0] if keep else out
        if keep:
            assert torch.equal(out[1], gate_up0) and not out[1].requires_grad
        assert h.requires_grad and torch.equal(h, h0)
        h.backward(dy)
        assert torch.equal(at.grad, expected)


@LAYERS
def test_feed_forward_block_through_autograd(layer):
    """x used twice, through gated and down products and past them: the gradients of both ways meet in x."""
    linear, linear_grad, gated, gated_grad, _, _ = layer
    m, n, k = 40, 96, 160
    x, _, wg, wu, wd = parts(m)
    dy = mx.rows(m, k, torch.bfloat16, seed=9)
    at = leaf(x)
    (at + linear(gated(at, wg, wu, n), *wd, k)).backward(dy)
    _, gate_up = gated(x, wg, wu, n, keep_gate_up=True)
    assert torch.equal(at.grad, dy + gated_grad(linear_grad(dy, *wd, n), gate_up, wg, wu, k))


class Stop(torch.autograd.Function):
    """A user's own function that hands no gradient back."""

    @staticmethod
    def forward(ctx, y):
        return y.clone()

    @staticmethod
    def backward(ctx, dy):
        return None


@LAYERS
def test_no_gradient_from_above_is_none_below(layer):
    linear, _, gated, _, _, _ = layer
    x, dy, wg, wu, _ = parts(20)
    for f in (lambda x: linear(x, *wg, 96), lambda x: gated(x, wg, wu, 96)):
        at = leaf(x)
        Stop.apply(f(at)).backward(dy)
        assert at.grad is None or not at.grad.any()


@LAYERS
def test_nothing_is_recorded_unasked(layer):
    linear, _, gated, _, w4a4, mlp = layer
    n, k = 96, 160
    x, _, wg, wu, wd = parts(20)
    calls = (lambda x: linear(x, *wg, n), lambda x: gated(x, wg, wu, n), lambda x: w4a4(x, *wg, n), lambda x: mlp(x, wg, wu, wd, n))
    for f in calls:
        assert not f(x).requires_grad
        with torch.no_grad():
            y = f(leaf(x))
        assert not y.requires_grad and torch.equal(y, f(x))


@LAYERS
def test_what_has_no_gradient_says_so(layer):
    linear, linear_grad, gated, gated_grad, w4a4, mlp = layer
    n, k = 96, 160
    x, dy, wg, wu, wd = parts(20)
    _, gate_up = gated(x, wg, wu, n, keep_gate_up=True)
    for op, f, t in (("gemm_mxfp4_w4a4", lambda x: w4a4(x, *wg, n), x), ("mlp_mxfp4_w4a4", lambda x: mlp(x, wg, wu, wd, n), x),
                     ("gemm_mxfp4_grad", lambda d: linear_grad(d, *wg, k), dy),
                     ("gated_mxfp4_grad", lambda d: gated_grad(d, gate_up, wg, wu, k), dy)):
        y = f(leaf(t))
        assert y.requires_grad and torch.equal(y, f(t))
        with pytest.raises(RuntimeError, match=f"{op}: has no gradient"):
            y.sum().backward()
    # Neither have the gradients: a second derivative is refused.
    for f in (lambda x: linear(x, *wg, n), lambda x: gated(x, wg, wu, n)):
        at = leaf(x)
        d = leaf(dy)
        dx, = torch.autograd.grad(f(at), at, d, create_graph=True)
        with pytest.raises(RuntimeError):
            dx.sum().backward()


def test_out_records_nothing():
    x, dy, wg, _, _ = parts(4)
    for f, t, n in ((ops.gemm_mxfp4_cuda, x, 96), (ops.gemm_mxfp4_w4a4_cuda, x, 96), (ops.gemm_mxfp4_grad_cuda, dy, 160)):
        out = torch.empty(4, n, dtype=t.dtype, device="cuda")
        with pytest.raises(RuntimeError, match="out records no gradient"):
            f(leaf(t), *wg, n, out=out)
        with torch.no_grad():
            assert f(leaf(t), *wg, n, out=out) is out


@LAYERS
def test_refusals_come_through(layer):
    linear, _, gated, _, w4a4, _ = layer
    x, _, wg, wu, _ = parts(4)
    for f, op in ((lambda x: linear(x, *wg, 96), "gemm_mxfp4"), (lambda x: gated(x, wg, wu, 96), "gated_mxfp4"),
                  (lambda x: w4a4(x, *wg, 96), "gemm_mxfp4_w4a4")):
        for bad in (x[0], x.t(), x.float()):
            with pytest.raises(RuntimeError, match=f"{op}: x must be"):
                f(leaf(bad) if bad.is_contiguous() else bad.detach().requires_grad_())


def test_linear_mxfp4_records():
    w = mx.Weight(96, 160, seed=3)
    x = mx.rows(6, 160, torch.bfloat16, seed=1).view(2, 3, 160)
    dy = mx.rows(6, 96, torch.bfloat16, seed=2)
    at = leaf(x)
    _host.linear.mxfp4(*w.plain, False).apply(at).backward(dy.view(2, 3, 96))
    assert torch.equal(at.grad.view(6, 160), ops.gemm_mxfp4_grad_cuda(dy, *w.packed, 160))


@LAYERS
def test_captured_step_and_another_stream(layer):
    """A captured step with its backward pass, replayed between eager ones of another leaf; and one on a side stream."""
    linear, _, gated, _, _, _ = layer
    n, k = 544, 1056
    x, _, wg, wu, wd = parts(40, n, k)
    dy = mx.rows(40, k, torch.bfloat16, seed=9)

    def step(at):
        y = linear(gated(at, wg, wu, n), *wd, k)
        return y.detach(), torch.autograd.grad(y, at, dy)[0]

    expected = step(leaf(x))
    torch.cuda.synchronize()
    held, stream, graph = leaf(x), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step(held)
    for _ in range(3):
        for o in out:
            o.fill_(float("nan"))
        graph.replay()
        again = step(leaf(x))
        torch.cuda.synchronize()
        for o, a, e in zip(out, again, expected):
            assert torch.equal(o, e) and torch.equal(a, e)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        aside = step(leaf(x))
    stream.synchronize()
    for a, e in zip(aside, expected):
        assert torch.equal(a, e)
