"""Gradients of the expert products as a program's own operations hand them over, in the Python and the C++ layer."""

import pytest
import torch

from pulsarlm_amd import _host, ops
from tests import _dense as dense

pytestmark = pytest.mark.gpu

LAYERS = pytest.mark.parametrize("layer", [ops, _host], ids=["python", "host"])


@LAYERS
@pytest.mark.parametrize("before", [1, 3, 8])
def test_a_gradient_that_begins_at_any_element(before, layer):
    """Joined to a tensor of odd length, the output's gradient is a part of a longer one, contiguous and not aligned."""
    counts, n, k = [9, 0, 31], 72, 64
    rows, off = sum(counts), dense.offsets([9, 0, 31])
    x, w, dy = dense.values((rows, k), torch.bfloat16, 1), dense.values((3, n, k), torch.bfloat16, 2), dense.values((rows, n), torch.bfloat16, 3)
    a, b, aux = x.clone().requires_grad_(), w.clone().requires_grad_(), torch.ones(before, dtype=x.dtype, device="cuda")
    joined = torch.cat([aux, layer.grouped_gemm_cuda(a, b, off).flatten()])
    joined.backward(torch.cat([aux, dy.flatten()]))
    assert torch.equal(a.grad, layer.grouped_gemm_grad_x_cuda(dy, w, off)) and torch.equal(b.grad, layer.grouped_gemm_grad_w_cuda(dy, x, off))


@LAYERS
def test_an_activation_without_a_gradient_says_so(layer):
    """Between two expert products, and at the router: no gradient is left out in silence."""
    counts, hidden, inter = [9, 0, 31], 64, 72
    x, off = dense.values((40, hidden), torch.bfloat16, 1), dense.offsets(counts)
    up, down = (dense.values(s, torch.bfloat16, 2).requires_grad_() for s in ((3, 2 * inter, hidden), (3, hidden, inter)))
    y = layer.grouped_gemm_cuda(layer.silu_mul_cuda(layer.grouped_gemm_cuda(x, up, off)), down, off)
    with torch.no_grad():
        assert torch.equal(y, layer.grouped_gemm_cuda(layer.silu_mul_cuda(layer.grouped_gemm_cuda(x, up, off)), down, off))
    with pytest.raises(RuntimeError, match="silu_mul: has no gradient"):
        y.float().sum().backward()
    logits = dense.values((40, 8), torch.float32, 3)
    want = layer.route_top_k_cuda(logits, 2)
    weights, chosen = layer.route_top_k_cuda(logits.clone().requires_grad_(), 2)
    assert torch.equal(weights, want[0]) and torch.equal(chosen, want[1]) and weights.requires_grad and not chosen.requires_grad
    with pytest.raises(RuntimeError, match="route_top_k: has no gradient"):
        weights.sum().backward()


def test_what_records_nothing_keeps_no_graph():
    x, logits = dense.values((5, 16), torch.bfloat16, 1).requires_grad_(), dense.values((5, 8), torch.float32, 2).requires_grad_()
    with torch.no_grad():
        assert not ops.silu_mul_cuda(x).requires_grad and not ops.route_top_k_cuda(logits, 2)[0].requires_grad
    assert ops.route_top_k_cuda(logits, 2, experts_i32=True)[1].dtype is torch.int32
    assert not ops.silu_mul_cuda(x.detach()).requires_grad and not ops.route_top_k_cuda(logits.detach(), 2)[0].requires_grad
