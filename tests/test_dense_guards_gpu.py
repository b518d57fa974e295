"""The grouped products write their outputs and nothing beside them: each output inside a larger buffer of a known value,
from one tile in all on."""

import pytest
import torch

from pulsarlm_amd import _lib
from tests import _dense as dense

pytestmark = pytest.mark.gpu

BF, GUARD = _lib.PLM_BF16, 7.0


def stream():
    return torch.cuda.current_stream().cuda_stream


def guarded(shape, call):
    """What call(pointer) leaves in a tensor of `shape` that has 64 of its own sizes on both sides."""
    size = shape.numel()
    room = torch.full((129 * size,), GUARD, dtype=torch.bfloat16, device="cuda")
    _lib.check(call(room.data_ptr() + 64 * size * 2))
    assert (room[: 64 * size] == GUARD).all() and (room[65 * size :] == GUARD).all()
    return room[64 * size : 65 * size].view(shape)


def sizes(experts):
    counts = [(11 * i + 3 * experts) % 29 for i in range(experts)]
    counts[-1] += 1
    return counts


@pytest.mark.parametrize("kernel", [None, "t0", "t3", "t5"])
@pytest.mark.parametrize("experts", [1, 2, 3, 4, 5, 9])
def test_gradients(experts, kernel, tuning_env):
    tuning_env("PLM_DENSE", kernel)
    lib, counts = _lib.load(), sizes(experts)
    rows, off = sum(counts), dense.offsets(sizes(experts))
    for n, k in ((8, 8), (64, 64), (8, 200), (128, 64), (64, 136), (200, 72), (200, 200)):
        dy, x = dense.values((rows, n), torch.bfloat16, 1), dense.values((rows, k), torch.bfloat16, 2)
        w = dense.values((experts, n, k), torch.bfloat16, 3)
        dw = guarded(w.shape, lambda to: lib.plm_grouped_gemm_grad_w(dy.data_ptr(), x.data_ptr(), BF, off.data_ptr(), experts, rows, n, k, to, stream()))
        dense.within(dw, *dense.grad_w(dy, x, counts), f"dw {n} {k}")
        dx = guarded(x.shape, lambda to: lib.plm_grouped_gemm_grad_x(dy.data_ptr(), BF, w.data_ptr(), off.data_ptr(), experts, rows, n, k, to, 1, stream()))
        dense.within(dx, *dense.grad_x(dy, w, counts), f"dx {n} {k}")


@pytest.mark.parametrize("kernel", [None, "r16", "r64", "t0", "t3", "t5"])
@pytest.mark.parametrize("experts", [1, 2, 3, 9])
def test_products(experts, kernel, tuning_env):
    tuning_env("PLM_DENSE", kernel)
    lib, counts = _lib.load(), sizes(experts)
    rows, off = sum(counts), dense.offsets(sizes(experts))
    for n, k in ((1, 16), (8, 208), (130, 64), (200, 80)):
        x, w = dense.values((rows, k), torch.bfloat16, 1), dense.values((experts, n, k), torch.bfloat16, 2)
        shape = torch.Size((rows, n))
        y = guarded(shape, lambda to: lib.plm_grouped_gemm_16(x.data_ptr(), BF, w.data_ptr(), off.data_ptr(), experts, rows, n, k, to, 1, stream()))
        dense.within(y, *dense.grouped(x, w, counts), f"y {n} {k}")
        w8, ws = dense.codes(experts * n, k, 3).view(experts, n, k), dense.scales(experts * n, 4).view(experts, n)
        size = lib.plm_grouped_gemm_int8_workspace_bytes(rows, n, k)
        room = torch.empty(size, dtype=torch.uint8, device="cuda")
        y = guarded(shape, lambda to: lib.plm_grouped_gemm_int8(x.data_ptr(), BF, w8.data_ptr(), ws.data_ptr(), off.data_ptr(), experts, rows, n, k, to, 1,
                                                                room.data_ptr(), size, stream()))
        q, xs = (t.cuda() for t in dense.quantize(x))
        for e, lo, hi in dense.by_expert(counts):
            dense.within(y[lo:hi], *dense.int8_product(q[lo:hi], xs[lo:hi], w8[e], ws[e]), f"8 bits {n} {k}, expert {e}")
