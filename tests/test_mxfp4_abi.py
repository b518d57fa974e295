"""Refusals of the MXFP4 entry points, on the CPU: every argument error is reported with the operation's name
before any device work; and the sizes of the packed forms."""

import ctypes

import pytest
import torch

from pulsarlm_amd import _lib, ops

D = ctypes.c_void_p(4096)
ODD = ctypes.c_void_p(4097)
BF, F32 = _lib.PLM_BF16, _lib.PLM_FP32
BIG = 1 << 40


def call(name, *args):
    lib = _lib.load()
    return getattr(lib, name)(*args), lib.plm_last_error().decode()


def quantize(x=D, dt=BF, m=4, k=64, codes=D, scale=D):
    return call("plm_quantize_mxfp4", x, dt, m, k, codes, scale, None)


def dequantize(codes=D, scale=D, m=4, k=64, out=D, dt=BF):
    return call("plm_dequantize_mxfp4", codes, scale, m, k, out, dt, None)


def repack(codes=D, scale=D, n=48, k=64, w=D, s=D):
    return call("plm_repack_mxfp4", codes, scale, n, k, w, s, None)


def gemm(x=D, dt=BF, w=D, s=D, m=4, n=48, k=64, y=D):
    return call("plm_gemm_mxfp4", x, dt, w, s, m, n, k, y, None)


def w4a4(x=D, dt=BF, w=D, s=D, m=4, n=48, k=64, y=D, ws=D, size=BIG):
    return call("plm_gemm_mxfp4_w4a4", x, dt, w, s, m, n, k, y, ws, size, None)


def grad(dy=D, dt=BF, w=D, s=D, m=4, n=48, k=64, dx=D, ws=D, size=BIG):
    return call("plm_gemm_mxfp4_grad", dy, dt, w, s, m, n, k, dx, ws, size, None)


def gated(x=D, dt=BF, w=D, s=D, w1=D, s1=D, m=4, n=48, k=64, h=D, gate_up=None):
    return call("plm_gated_mxfp4", x, dt, w, s, w1, s1, m, n, k, h, gate_up, None)


def gated_grad(dh=D, gate_up=D, dt=BF, w=D, s=D, w1=D, s1=D, m=4, n=48, k=64, dx=D, ws=D, size=BIG):
    return call("plm_gated_mxfp4_grad", dh, gate_up, dt, w, s, w1, s1, m, n, k, dx, ws, size, None)


def mlp(x=D, dt=BF, w=D, s=D, w1=D, s1=D, w2=D, s2=D, m=4, n=96, k=64, y=D, ws=D, size=BIG):
    return call("plm_mlp_mxfp4_w4a4", x, dt, w, s, w1, s1, w2, s2, m, n, k, y, ws, size, None)


PRODUCTS = {gemm: "gemm_mxfp4", w4a4: "gemm_mxfp4_w4a4", grad: "gemm_mxfp4_grad", gated: "gated_mxfp4", gated_grad: "gated_mxfp4_grad",
            mlp: "mlp_mxfp4_w4a4"}


@pytest.mark.parametrize("f", PRODUCTS, ids=PRODUCTS.values())
@pytest.mark.parametrize("args,msg", [
    ({"dt": F32}, "x must be fp16 or bf16"),
    ({"dt": 7}, "x must be fp16 or bf16"),
    ({"m": -1}, "sizes must be non-negative"),
    ({"n": -32}, "sizes must be non-negative"),
    ({"k": -32}, "sizes must be non-negative"),
    ({"k": 80}, "K must be a multiple of 32"),
    ({"k": (1 << 19) + 32}, "N and K must be at most 2^19"),
    ({"n": (1 << 19) + 32}, "N and K must be at most 2^19"),
    ({"m": (1 << 24) + 1}, "M must be at most 2^24"),
    ({"m": 1 << 20, "k": 1 << 17}, "M must be at most 2^24"),
    ({"w": None}, "null pointer"),
    ({"s": None}, "null pointer"),
    ({"w": ODD}, "weight must be 16-byte aligned"),
    ({"s": ODD}, "scale must be 4-byte aligned"),
])
def test_products_refuse(f, args, msg):
    rc, said = f(**args)
    assert rc == _lib.PLM_ERR_INVALID and said.startswith(f"{PRODUCTS[f]}: {msg}"), said


@pytest.mark.parametrize("f,args,msg", [
    (gemm, {"x": None}, "null pointer"), (gemm, {"x": ODD}, "x must be 16-byte aligned"), (gemm, {"y": None}, "null pointer"),
    (gemm, {"y": ODD}, "y must be 2-byte aligned"), (w4a4, {"x": ctypes.c_void_p(4104)}, "x must be 16-byte aligned"),
    (w4a4, {"ws": ODD}, "workspace must be 256-byte aligned"), (gated, {"w1": None}, "null pointer"),
    (gated, {"gate_up": ctypes.c_void_p(4098)}, "gate_up must be 4-byte aligned"), (gated, {"s1": ODD}, "scale must be 4-byte aligned"),
    (mlp, {"n": 48}, "the intermediate size must be a multiple of 32"), (mlp, {"w2": None}, "null pointer"),
    (grad, {"dx": ctypes.c_void_p(4100)}, "dx must be 8-byte aligned"), (grad, {"dy": None}, "dy must be 2-byte aligned"),
    (grad, {"dx": None}, "dx must be 8-byte aligned"), (gated_grad, {"gate_up": None}, "dh must be 2-byte"),
    (gated_grad, {"gate_up": ctypes.c_void_p(4098)}, "dh must be 2-byte and gate_up 4-byte aligned"),
])
def test_pointers_refused(f, args, msg):
    rc, said = f(**args)
    assert rc == _lib.PLM_ERR_INVALID and said.startswith(f"{PRODUCTS[f]}: {msg}"), said


@pytest.mark.parametrize("f", [w4a4, mlp, gated_grad])
def test_workspace_refused(f):
    for args in ({"ws": None}, {"size": 0}):
        rc, said = f(**args)
        assert rc == _lib.PLM_ERR_WORKSPACE and "workspace of" in said


def test_quantizer_and_repack_refuse():
    for f, args, msg in ((quantize, {"dt": 9}, "quantize_mxfp4: x must be fp32, fp16 or bf16"), (quantize, {"k": 48}, "quantize_mxfp4: K must be a multiple of 32"),
                         (quantize, {"x": ODD}, "quantize_mxfp4: x must be 16-byte aligned"), (quantize, {"codes": ODD}, "quantize_mxfp4: codes must be 4-byte"),
                         (quantize, {"m": -1}, "quantize_mxfp4: sizes must be non-negative"), (quantize, {"scale": None}, "quantize_mxfp4: null pointer"),
                         (quantize, {"m": 1 << 31}, "quantize_mxfp4: sizes must be below 2^30"),
                         (dequantize, {"dt": 9}, "dequantize_mxfp4: out dtype must be"), (dequantize, {"out": ODD}, "dequantize_mxfp4: out must be 16-byte"),
                         (dequantize, {"k": 33}, "dequantize_mxfp4: K must be a multiple of 32"), (dequantize, {"codes": None}, "dequantize_mxfp4: null pointer"),
                         (repack, {"k": 48}, "repack_mxfp4: K must be a multiple of 32"), (repack, {"n": 1 << 20}, "repack_mxfp4: N and K must be at most 2^19"),
                         (repack, {"codes": ODD}, "repack_mxfp4: codes and weight_out must be 16-byte"), (repack, {"s": ODD}, "repack_mxfp4: scale_out must be 4-byte"),
                         (repack, {"w": None}, "repack_mxfp4: null pointer")):
        rc, said = f(**args)
        assert rc == _lib.PLM_ERR_INVALID and said.startswith(msg), said


def test_empty_calls_do_no_device_work():
    for f in (gemm, w4a4, gated):
        assert f(m=0, x=None, w=None, s=None)[0] == _lib.PLM_OK and f(n=0, x=None)[0] == _lib.PLM_OK
    for f in (grad, gated_grad, mlp):
        assert f(m=0, dt=BF, w=None)[0] == _lib.PLM_OK and f(k=0, w=None)[0] == _lib.PLM_OK
    assert quantize(m=0, x=None)[0] == quantize(k=0, x=None)[0] == dequantize(m=0, out=None)[0] == repack(n=0, w=None)[0] == _lib.PLM_OK


def test_sizes():
    lib = _lib.load()
    assert lib.plm_mxfp4_weight_bytes(4096, 4096) == 4096 * 4096 // 2
    assert lib.plm_mxfp4_scale_bytes(4096, 4096) == 4096 * 4096 // 32
    assert lib.plm_mxfp4_weight_bytes(17, 160) == 2 * 2 * 1024 and lib.plm_mxfp4_scale_bytes(17, 160) == 2 * 256 and lib.plm_mxfp4_scale_bytes(65, 160) == 4 * 256
    assert lib.plm_mxfp4_weight_bytes(-1, 32) == -1 and lib.plm_mxfp4_scale_bytes(4, -32) == -1
    assert lib.plm_gemm_mxfp4_w4a4_workspace_bytes(0, 4, 64) == lib.plm_mlp_mxfp4_w4a4_workspace_bytes(4, 0, 64) == 0
    assert lib.plm_gemm_mxfp4_w4a4_workspace_bytes(300, 48, 1056) >= 300 * 1056 // 2 + 300 * 1056 // 32


def test_python_refuses_host_tensors_and_wrong_shapes():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    w, s = torch.zeros(48 * 128 // 8, dtype=torch.int32), torch.zeros(1, 1, 64, dtype=torch.int32)
    c, b = torch.zeros(48, 32, dtype=torch.uint8), torch.zeros(48, 2, dtype=torch.uint8)
    for op, f in (("quantize_mxfp4", lambda: ops.quantize_mxfp4_cuda(x)), ("dequantize_mxfp4", lambda: ops.dequantize_mxfp4_cuda(c, b)),
                  ("repack_mxfp4", lambda: ops.repack_mxfp4_cuda(c, b)), ("gemm_mxfp4", lambda: ops.gemm_mxfp4_cuda(x, w, s, 48)),
                  ("gemm_mxfp4_w4a4", lambda: ops.gemm_mxfp4_w4a4_cuda(x, w, s, 48)),
                  ("gemm_mxfp4_grad", lambda: ops.gemm_mxfp4_grad_cuda(x, w, s, 48)),
                  ("gated_mxfp4", lambda: ops.gated_mxfp4_cuda(x, (w, s), (w, s), 48)),
                  ("gated_mxfp4_grad", lambda: ops.gated_mxfp4_grad_cuda(x, x, (w, s), (w, s), 64)),
                  ("mlp_mxfp4_w4a4", lambda: ops.mlp_mxfp4_w4a4_cuda(x, (w, s), (w, s), (w, s), 48))):
        with pytest.raises(RuntimeError, match=f"^{op}: .*CUDA"):
            f()


def test_python_and_library_agree_on_the_scales():
    lib = _lib.load()
    for n in (0, 1, 16, 63, 64, 65, 200, 4096):
        for k in (0, 32, 128, 160, 544, 4128):
            g, t, lanes = ops._mx_scale_shape(n, k)
            assert 4 * g * t * lanes == lib.plm_mxfp4_scale_bytes(n, k)


QUERIES = ["plm_gemm_mxfp4_w4a4_workspace_bytes", "plm_mlp_mxfp4_w4a4_workspace_bytes", "plm_gemm_mxfp4_grad_workspace_bytes",
           "plm_gated_mxfp4_grad_workspace_bytes"]


@pytest.mark.parametrize("name", QUERIES)
def test_workspace_queries_take_any_sizes(name):
    """Sizes that the call refuses need no workspace; the sizes are multiplied only once they are known to be small."""
    query = getattr(_lib.load(), name)
    for huge in (1 << 25, 1 << 32, 1 << 40, (1 << 63) - 1):
        for sizes in ((huge, 64, 64), (64, huge, 64), (64, 64, huge), (huge, huge, 64), (huge, 64, huge), (64, huge, huge), (huge, huge, huge)):
            assert query(*sizes) == 0, sizes
    assert query(1 << 24, 64, 64) > 0  # the largest M
    assert query(1 << 17, 1 << 19, 1 << 19) > 0


def test_layout_queries_take_any_sizes():
    lib = _lib.load()
    for n, k in ((1 << 62, 1 << 62), ((1 << 19) + 1, 32), (16, (1 << 19) + 32), ((1 << 63) - 1, 1)):
        assert lib.plm_mxfp4_weight_bytes(n, k) == lib.plm_mxfp4_scale_bytes(n, k) == -1
    assert lib.plm_mxfp4_weight_bytes(1 << 19, 1 << 19) == 1 << 37


def test_gradient_needs_no_room_for_a_dy_that_it_reads_in_place():
    lib = _lib.load()
    for m, n, k in ((4096, 24576, 4096), (1, 64, 32), (2000, 4096, 4096), (333, 5000, 4128), (8200, 4300, 96)):
        every, aligned = lib.plm_gemm_mxfp4_grad_workspace_bytes(m, n, k), lib.plm_gemm_mxfp4_grad_aligned_workspace_bytes(m, n, k)
        copy = -(-m * -(-n // 64) * 64 * 2 // 256) * 256
        assert every - aligned == (copy if n % 64 == 0 else 0) and every >= copy
    assert lib.plm_gemm_mxfp4_grad_aligned_workspace_bytes(4096, 24576, 4096) == 0  # one round of tiles, unsplit
    assert lib.plm_gemm_mxfp4_grad_aligned_workspace_bytes(0, 64, 64) == lib.plm_gemm_mxfp4_grad_aligned_workspace_bytes(1 << 40, 64, 1 << 40) == 0
    # What is missing is said for the dy at hand: an aligned one asks for less.
    need = lib.plm_gemm_mxfp4_grad_workspace_bytes(1, 64, 32)
    rc, said = grad(dy=ctypes.c_void_p(4098), m=1, n=64, k=32, ws=None, size=0)
    assert rc == _lib.PLM_ERR_WORKSPACE and f"workspace of {need} bytes" in said
