"""The C++ host layer's MXFP4 operators: the same bits as pulsarlm_amd.ops, and linear::mxfp4 on a 3-D input."""

import pytest
import torch

from pulsarlm_amd import _host, ops
from tests import _mxfp4 as mx

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 20, 300])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_host_layer_matches_ops(m, dtype):
    dt, n, k = mx.DT[dtype], 96, 160
    wg, wu, wd = mx.Weight(n, k, seed=1), mx.Weight(n, k, seed=2), mx.Weight(k, n, seed=3)
    for w in (wg, wu, wd):
        for a, b in zip(_host.repack_mxfp4_cuda(*w.plain), w.packed):
            assert torch.equal(a, b)
    x, dh = mx.rows(m, k, dt, seed=4), mx.rows(m, n, dt, seed=5)
    for a, b in zip(_host.quantize_mxfp4_cuda(x), ops.quantize_mxfp4_cuda(x)):
        assert torch.equal(a, b)
    assert torch.equal(_host.dequantize_mxfp4_cuda(*wg.plain, dt), ops.dequantize_mxfp4_cuda(*wg.plain, dt))
    assert torch.equal(_host.gemm_mxfp4_cuda(x, *wg.packed, n), ops.gemm_mxfp4_cuda(x, *wg.packed, n))
    assert torch.equal(_host.gemm_mxfp4_w4a4_cuda(x, *wg.packed, n), ops.gemm_mxfp4_w4a4_cuda(x, *wg.packed, n))
    assert torch.equal(_host.gemm_mxfp4_grad_cuda(dh, *wg.packed, k), ops.gemm_mxfp4_grad_cuda(dh, *wg.packed, k))
    h, gate_up = _host.gated_mxfp4_cuda(x, *wg.packed, *wu.packed, n, True)
    h2, gate_up2 = ops.gated_mxfp4_cuda(x, wg.packed, wu.packed, n, keep_gate_up=True)
    assert torch.equal(h, h2) and torch.equal(gate_up, gate_up2)
    assert torch.equal(_host.gated_mxfp4_cuda(x, *wg.packed, *wu.packed, n, False)[0], h)
    assert torch.equal(_host.gated_mxfp4_grad_cuda(dh, gate_up, *wg.packed, *wu.packed, k),
                       ops.gated_mxfp4_grad_cuda(dh, gate_up, wg.packed, wu.packed, k))
    assert torch.equal(_host.mlp_mxfp4_w4a4_cuda(x, *wg.packed, *wu.packed, *wd.packed, n),
                       ops.mlp_mxfp4_w4a4_cuda(x, wg.packed, wu.packed, wd.packed, n))


def test_linear_mxfp4():
    n, k = 72, 160
    w = mx.Weight(n, k, seed=1)
    x = mx.rows(6, k, torch.bfloat16, seed=2).view(2, 3, k)
    y = _host.linear.mxfp4(*w.plain, False).apply(x)
    assert y.shape == (2, 3, n)
    mx.within(y.view(6, n), *mx.product(x.view(6, k).double(), w.dense), "linear")
    y = _host.linear.mxfp4(*w.plain, True).apply(x)
    mx.within(y.view(6, n), *mx.product(mx.rounded(x.view(6, k)), w.dense), "linear, W4A4")


def test_host_layer_refuses():
    w = mx.Weight(96, 160, seed=1)
    x = mx.rows(4, 160, torch.bfloat16, seed=2)
    with pytest.raises(RuntimeError, match="gemm_mxfp4: weight has the wrong size"):
        _host.gemm_mxfp4_cuda(x, *w.packed, 300)
    with pytest.raises(RuntimeError, match="gemm_mxfp4_w4a4: x must be contiguous"):
        _host.gemm_mxfp4_w4a4_cuda(x.t(), *w.packed, 96)
    with pytest.raises(RuntimeError, match="gemm_mxfp4: x must be a CUDA fp16 or bf16"):
        _host.gemm_mxfp4_cuda(x.float(), *w.packed, 96)
    with pytest.raises(RuntimeError, match="repack_mxfp4: scale must be"):
        _host.repack_mxfp4_cuda(w.plain[0], w.plain[1][:, :3].contiguous())
    with pytest.raises(RuntimeError, match="gated_mxfp4_grad: gate_up must be contiguous fp32"):
        _host.gated_mxfp4_grad_cuda(x[:, :96].contiguous(), x, *w.packed, *w.packed, 160)
    with pytest.raises(RuntimeError, match="mlp_mxfp4_w4a4: weight has the wrong size"):
        _host.mlp_mxfp4_w4a4_cuda(x, *w.packed, *w.packed, *w.packed, 96)
