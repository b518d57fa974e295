"""The products and the quantizer write their outputs and nothing beside them: each output inside a larger buffer of a known
value, from one tile in all on, and a workspace of the size that the query names inside one, too."""

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


def guarded_bytes(size, call):
    """call(pointer) on `size` bytes, 256-byte aligned, between two times 4 KiB; those bytes."""
    room = torch.full((size + 8192 + 256,), 0x5A, dtype=torch.uint8, device="cuda")
    at = 4096 + -(room.data_ptr() + 4096) % 256
    _lib.check(call(room.data_ptr() + at))
    assert (room[:at] == 0x5A).all() and (room[at + size :] == 0x5A).all()
    return room[at : at + size]


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


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 16), (3, 7), (5, 1024), (2, 8200), (7, 20000), (130, 72)])
def test_quantizer(m, k, dtype):
    lib, x = _lib.load(), dense.values((m, k), dense.DT[dtype], 1)
    kind, q, s = {"bf16": _lib.PLM_BF16, "fp32": _lib.PLM_FP32}[dtype], *dense.quantize(x)
    scale = torch.empty(m, device="cuda")
    codes = guarded_bytes(m * k, lambda to: lib.plm_quantize_rows_int8(x.data_ptr(), kind, m, k, to, scale.data_ptr(), stream()))
    assert torch.equal(codes.view(torch.int8).view(m, k).cpu(), q)
    to_scale = guarded_bytes(4 * m, lambda to: lib.plm_quantize_rows_int8(x.data_ptr(), kind, m, k, codes.data_ptr(), to, stream()))
    assert torch.equal(to_scale.view(torch.float32).cpu(), s) and torch.equal(scale.cpu(), s)
    back = guarded_bytes(x.nbytes, lambda to: lib.plm_dequantize_rows_int8(codes.data_ptr(), scale.data_ptr(), m, k, to, kind, stream()))
    assert torch.equal(back.view(x.dtype).view(m, k).cpu(), (q.float() * s[:, None]).to(x.dtype))


@pytest.mark.parametrize("kernel", [None, "r16", "r64", "t0", "t3", "t5", "t2,3", "t5,4"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (2, 8, 208), (3, 200, 2720), (20, 37, 528), (70, 136, 1040), (1, 4100, 64)])
def test_dense_products(m, n, k, kernel, tuning_env):
    tuning_env("PLM_DENSE", kernel)
    lib = _lib.load()
    x, w, ws = dense.values((m, k), torch.bfloat16, 1), dense.codes(n, k, 2), dense.scales(n, 3)
    q, xs = (t.cuda() for t in dense.quantize(x))
    want, shape = dense.int8_product(q, xs, w, ws), torch.Size((m, n))
    size = lib.plm_gemm_int8_workspace_bytes(m, n, k)

    def on_codes(to):
        guarded_bytes(size, lambda ws8: lib.plm_gemm_int8(q.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), m, n, k, to, BF, ws8, size, stream()))
        return _lib.PLM_OK

    dense.within(guarded(shape, on_codes), *want, "codes")
    size8 = lib.plm_gemm_int8_w8a8_workspace_bytes(m, n, k)

    def on_x(to):
        guarded_bytes(size8, lambda ws8: lib.plm_gemm_int8_w8a8(x.data_ptr(), BF, w.data_ptr(), ws.data_ptr(), m, n, k, to, ws8, size8, stream()))
        return _lib.PLM_OK

    dense.within(guarded(shape, on_x), *want, "w8a8")
