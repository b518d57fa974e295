"""MXFP4 operands, outputs and kept sums past 2^31 elements and 2^32 bytes: samples against float64."""

import pytest
import torch

from pulsarlm_amd import ops
from tests import _mxfp4 as mx

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


def sample(m):
    return torch.tensor([0, 1, m // 2, (1 << 31) // 16400, m - 129, m - 2, m - 1], device="cuda")


def test_many_rows():
    m, n, k = 140001, 16400, 64  # 2.3e9 outputs
    w, wu = mx.Weight(n, k, seed=1), mx.Weight(n, k, seed=2)
    g = torch.Generator("cuda").manual_seed(0)
    x = torch.randn(m, k, generator=g, device="cuda", dtype=torch.bfloat16)
    at = sample(m)
    mx.within(ops.gemm_mxfp4_cuda(x, *w.packed, n)[at], *mx.product(x[at].double(), w.dense), "W4A16")
    mx.within(ops.gemm_mxfp4_w4a4_cuda(x, *w.packed, n)[at], *mx.product(mx.rounded(x[at]), w.dense), "W4A4")
    h, gate_up = ops.gated_mxfp4_cuda(x, w.packed, wu.packed, n, keep_gate_up=True)
    ref, err, _, _ = mx.gated(x[at].double(), w.dense, wu.dense)
    mx.within(h[at], ref, err, "h")
    mx.within(gate_up[at], *mx.product(x[at].double(), torch.cat([w.dense, wu.dense])), "gate_up")
    # h serves as dy; N is not whole steps, so that its rows are copied first.
    dx = ops.gemm_mxfp4_grad_cuda(h, *w.packed, k)
    mx.within(dx[at], *mx.product(h[at].double(), w.dense.t()), "dx")
    dx = ops.gated_mxfp4_grad_cuda(h, gate_up, w.packed, wu.packed, k)
    d, gu = h[at].double(), gate_up[at].double()
    dg, du = mx.gated_factors(d, gu[:, :n], gu[:, n:])
    own = [mx.half(torch.bfloat16) * f.abs() + 2.0**-19 * d.abs() * v * (1 + gu[:, :n].abs()) for f, v in ((dg, gu[:, n:].abs()), (du, 1.0))]
    err = sum(e @ w_.dense.abs() + (2 * n + 8) * 2.0**-23 * ((f.abs() + e) @ w_.dense.abs()) for e, f, w_ in zip(own, (dg, du), (w, wu)))
    mx.within(dx[at], dg @ w.dense + du @ wu.dense, err, "gated dx")


def test_a_weight_past_4_gib():
    """Few rows and many against a weight of 4.6 GB, forward and back, and its repack and inverse."""
    n, k = 1 << 19, 17440
    g = torch.Generator("cuda").manual_seed(0)
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=g)
    scale = torch.randint(118, 122, (n, k // 32), dtype=torch.uint8, device="cuda", generator=g)
    weight = ops.repack_mxfp4_cuda(codes, scale)
    at = torch.tensor([0, 17, n // 2 - 1, n // 2, n - 130, n - 1], device="cuda")
    dense = ops.dequantize_mxfp4_cuda(codes[at].contiguous(), scale[at].contiguous(), torch.float32)
    whole = ops.dequantize_mxfp4_cuda(codes, scale, torch.bfloat16)  # 18 GB: past 2^33 elements
    assert torch.equal(whole[at].float(), dense)
    dense = dense.double()
    for m in (1, 20, 300):
        x = mx.rows(m, k, torch.bfloat16, seed=m)
        mx.within(ops.gemm_mxfp4_cuda(x, *weight, n)[:, at], *mx.product(x.double(), dense), "W4A16")
        mx.within(ops.gemm_mxfp4_w4a4_cuda(x, *weight, n)[:, at], *mx.product(mx.rounded(x), dense), "W4A4")
        dy = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
        dy[:, at] = mx.rows(m, at.numel(), torch.bfloat16, seed=m + 1)
        ref, err = mx.product(dy[:, at].double(), dense.t())
        mx.within(ops.gemm_mxfp4_grad_cuda(dy, *weight, k), ref, err, "dx")  # zeros add no error
    requantized = ops.quantize_mxfp4_cuda(whole)
    back = ops.dequantize_mxfp4_cuda(requantized[0], requantized[1], torch.bfloat16)
    for rows in range(0, n, n // 8):  # a block without 4 or 6 takes a lower scale: the same values
        assert torch.equal(back[rows : rows + n // 8], whole[rows : rows + n // 8])
