"""W8A8 products of one to four rows: the plan counts the launch that quantizes them, and no plan changes a result."""

import pytest
import torch

from pulsarlm_amd import _lib, ops
from tests import _dense as dense

pytestmark = pytest.mark.gpu


def product(x, w, ws, room):
    lib, y = _lib.load(), torch.empty(x.shape[0], w.shape[0], dtype=x.dtype, device="cuda")
    _lib.check(lib.plm_gemm_int8_w8a8(x.data_ptr(), _lib.PLM_BF16, w.data_ptr(), ws.data_ptr(), x.shape[0], w.shape[0], x.shape[1], y.data_ptr(),
                                      room.data_ptr(), room.numel(), torch.cuda.current_stream().cuda_stream))
    return y


# Through tiles, with a launch more and some with a third, these took 1.1 to 1.9 times as long.
@pytest.mark.parametrize("m,n,k", [(1, 512, 512), (1, 1024, 1024), (1, 4096, 1024), (2, 4096, 512), (4, 256, 1024), (1, 256, 8192), (3, 12288, 1024)])
def test_a_few_tokens_are_quantized_inside(m, n, k):
    """Nothing is written to the workspace: no codes for another launch."""
    x, w, ws = dense.values((m, k), torch.bfloat16, 1), dense.codes(n, k, 2), dense.scales(n, 3)
    room = torch.full((_lib.load().plm_gemm_int8_w8a8_workspace_bytes(m, n, k),), 0x5A, dtype=torch.uint8, device="cuda")
    y = product(x, w, ws, room)
    assert (room == 0x5A).all()
    q, xs = dense.quantize(x)
    dense.within(y, *dense.int8_product(q.cuda(), xs.cuda(), w, ws))


@pytest.mark.parametrize("m,n,k", [(1, 1024, 1024), (2, 4096, 512), (4, 520, 1040), (1, 256, 16384), (2, 256, 16384), (1, 12288, 1024), (5, 512, 512)])
def test_any_alignment_of_x_in_one_workspace(m, n, k):
    """x that is not 16-byte aligned is quantized by a launch of its own, under another plan; one workspace serves both."""
    w, ws = dense.codes(n, k, 2), dense.scales(n, 3)
    room = dense.values((1, 1 + m * k), torch.bfloat16, 1).view(-1)
    x = room[1:].view(m, k)
    y = ops.gemm_int8_w8a8_cuda(x, w, ws)
    assert torch.equal(y, ops.gemm_int8_w8a8_cuda(x.clone(), w, ws))
    q, xs = dense.quantize(x)
    dense.within(y, *dense.int8_product(q.cuda(), xs.cuda(), w, ws))
    lib = _lib.load()
    need = lib.plm_gemm_int8_w8a8_workspace_bytes(m, n, k)
    assert need >= m * k + 4 * m + lib.plm_gemm_int8_workspace_bytes(m, n, k)
    spare = torch.empty(need, dtype=torch.uint8, device="cuda")
    assert torch.equal(product(x, w, ws, spare), y) and torch.equal(product(x.clone(), w, ws, spare), y)
