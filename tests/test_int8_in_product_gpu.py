"""Tokens quantized inside the product, on the kernel that does so: one to four rows, in rows of one and two strips a
workgroup, with values that wait in registers and values that are read again, up to the most codes that it keeps."""

import pytest
import torch

from pulsarlm_amd import ops
from tests import _dense as dense

pytestmark = pytest.mark.gpu

# One strip of 16 columns a workgroup (eight wavefronts, 4096 pieces of eight values a row wait) and two (four; 2048).
# Rows of one wavefront in four, in two and all of them.
SIZES = [(1, 72, 16), (1, 72, 16384), (1, 72, 16400), (1, 72, 65536), (2, 72, 8208), (2, 72, 32768), (3, 72, 2720), (4, 72, 2048),
         (1, 4112, 4096), (1, 6144, 4096), (1, 4100, 8192), (1, 4100, 8208), (1, 4100, 65536), (2, 4100, 4096), (2, 6144, 4112), (2, 4100, 32768),
         (3, 4100, 2720), (4, 4112, 2048), (4, 4100, 16)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_the_same_as_quantized_before(m, n, k, dtype, tuning_env):
    tuning_env("PLM_DENSE", "r16")
    x, w, ws = dense.values((m, k), dense.DT[dtype], m + k), dense.codes(n, k, 2, low=-128), dense.scales(n, 3)
    x[0, k - 1] = 30.0  # the row's largest, in its last piece
    if m > 2:
        x[2] = 0
    y = ops.gemm_int8_w8a8_cuda(x, w, ws)
    q, xs = dense.quantize(x)
    dense.within(y, *dense.int8_product(q.cuda(), xs.cuda(), w, ws))
    assert torch.equal(y, ops.gemm_int8_cuda(*ops.quantize_rows_int8_cuda(x), w, ws, x.dtype))


@pytest.mark.parametrize("n", [72, 4100])
@pytest.mark.parametrize("m,k", [(1, 65536), (2, 32768), (3, 2720), (4, 2048)])
def test_a_row_that_is_not_finite(m, k, n, tuning_env):
    tuning_env("PLM_DENSE", "r16")
    x, w, ws = dense.values((m, k), torch.bfloat16, 1), dense.codes(n, k, 2), dense.scales(n, 3)
    clean = ops.gemm_int8_w8a8_cuda(x, w, ws)
    x[m - 1, k - 1] = float("nan")
    y = ops.gemm_int8_w8a8_cuda(x, w, ws)
    assert y[m - 1].isnan().all() and torch.equal(y[: m - 1], clean[: m - 1])
