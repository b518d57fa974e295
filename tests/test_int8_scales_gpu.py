"""8-bit products under scales from one end of fp32 to the other: only a result that is out of range itself may pass it,
whichever of its two scales is the large one."""

import pytest
import torch

from pulsarlm_amd import ops
from tests import _dense as dense

pytestmark = pytest.mark.gpu

# The kernel for few rows, tiles that store whole lines or not (N), and a sum in parts.
KERNELS = ["r16", "r64", "t0", "t5", "t5,4"]
# Token's and channel's; a sum of 512 products of codes is up to 2^23, and these results lie well within bf16's range.
PAIRS = [(1e36, 1e-36), (1e-36, 1e36), (1e-20, 1e35), (1e38, 1e-41), (1e-41, 1e38), (1e-43, 1e33), (3e38, 2e-38)]


def full(rows, value):
    return torch.full((rows,), value, dtype=torch.float32, device="cuda")


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("token,channel", PAIRS)
def test_product(token, channel, kernel, tuning_env):
    tuning_env("PLM_DENSE", kernel)
    for n in (40, 37):
        q, w = dense.codes(20, 512, 1), dense.codes(n, 512, 2)
        xs, ws = full(20, token), full(n, channel)
        y = ops.gemm_int8_cuda(q, xs, w, ws)
        assert y.isfinite().all()
        dense.within(y, *dense.int8_product(q, xs, w, ws), f"N {n}")


@pytest.mark.parametrize("kernel", [None, "r16", "t0", "t5"])
@pytest.mark.parametrize("top,channel", [(1e38, 1e-36), (1e-12, 1e36), (1e-13, 1e33)])
def test_16_bit_tokens(top, channel, kernel, tuning_env):
    """Tokens' scales as the quantizer makes them, the product dense and by expert."""
    tuning_env("PLM_DENSE", kernel)
    n, k = 40, 64
    w, ws = dense.codes(2 * n, k, 2).view(2, n, k), full(2 * n, channel).view(2, n)
    for counts in ([1, 2], [0, 30]):
        rows = sum(counts)
        x = (dense.values((rows, k), torch.float32, 1).clamp(-4, 4) / 4 * top).bfloat16()
        q, xs = (t.cuda() for t in dense.quantize(x))
        dense.within(ops.gemm_int8_w8a8_cuda(x, w[0], ws[0]), *dense.int8_product(q, xs, w[0], ws[0]), "dense")
        y = ops.grouped_gemm_int8_cuda(x, w, ws, dense.offsets(counts))
        for e, lo, hi in dense.by_expert(counts):
            dense.within(y[lo:hi], *dense.int8_product(q[lo:hi], xs[lo:hi], w[e], ws[e]), f"expert {e}")


@pytest.mark.parametrize("kernel", ["r16", "t0", "t5,4"])
def test_scales_that_are_not_numbers(kernel, tuning_env):
    """What is out of range, infinite, NaN or zero goes into the results of its row and channel, as in the formula."""
    tuning_env("PLM_DENSE", kernel)
    q, w = torch.ones(6, 512, dtype=torch.int8, device="cuda"), torch.ones(40, 512, dtype=torch.int8, device="cuda")
    q[5] = 0
    xs, ws = full(6, 2.0), full(40, 0.5)
    xs[1], xs[2], xs[3], xs[4] = float("inf"), float("nan"), 0.0, 3e38
    ws[1], ws[2], ws[3], ws[4] = float("inf"), float("nan"), 0.0, -3e38
    y = ops.gemm_int8_cuda(q, xs, w, ws).double()
    want = ((512.0 * (q[:, :1] != 0).double()) * xs.double()[:, None] * ws.double()).expand(6, 40)
    want = torch.where(want.abs() > 3.4e38, want.sign() * float("inf"), want)
    assert torch.equal(y.isnan(), want.isnan())
    assert torch.equal(y.isinf(), want.isinf()) and torch.equal(y.sign()[y.isinf()], want.sign()[want.isinf()])
    ok = want.isfinite()
    assert ((y - want).abs()[ok] <= 2.0**-8 * want.abs()[ok]).all()
