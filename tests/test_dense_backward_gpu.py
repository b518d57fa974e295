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
