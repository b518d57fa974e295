"""Refusals of the int8 and expert entry points, on the CPU: every argument error is reported with the operation's name
before any device work."""

import ctypes

import pytest
import torch

from pulsarlm_amd import _host, _lib, ops

D = ctypes.c_void_p(4096)
ODD = ctypes.c_void_p(4097)
TWO = ctypes.c_void_p(4098)
BF, F32 = _lib.PLM_BF16, _lib.PLM_FP32
BIG = 1 << 40


def call(name, *args):
    lib = _lib.load()
    return getattr(lib, name)(*args), lib.plm_last_error().decode()


def quantize(x=D, dt=BF, m=4, k=64, codes=D, scale=D):
    return call("plm_quantize_rows_int8", x, dt, m, k, codes, scale, None)


def dequantize(codes=D, scale=D, m=4, k=64, out=D, dt=BF):
    return call("plm_dequantize_rows_int8", codes, scale, m, k, out, dt, None)


def gemm(x=D, xs=D, w=D, s=D, m=4, n=48, k=64, y=D, dt=BF, ws=D, size=BIG):
    return call("plm_gemm_int8", x, xs, w, s, m, n, k, y, dt, ws, size, None)


def w8a8(x=D, dt=BF, w=D, s=D, m=4, n=48, k=64, y=D, ws=D, size=BIG):
    return call("plm_gemm_int8_w8a8", x, dt, w, s, m, n, k, y, ws, size, None)


def grouped8(x=D, dt=BF, w=D, s=D, off=D, e=4, m=40, n=48, k=64, y=D, rest=1, ws=D, size=BIG):
    return call("plm_grouped_gemm_int8", x, dt, w, s, off, e, m, n, k, y, rest, ws, size, None)


def grouped(x=D, dt=BF, w=D, off=D, e=4, m=40, n=48, k=64, y=D, rest=1):
    return call("plm_grouped_gemm_16", x, dt, w, off, e, m, n, k, y, rest, None)


def grad_x(x=D, dt=BF, w=D, off=D, e=4, m=40, n=48, k=64, y=D, rest=1):
    return call("plm_grouped_gemm_grad_x", x, dt, w, off, e, m, n, k, y, rest, None)


def grad_w(dy=D, x=D, dt=BF, off=D, e=4, m=40, n=48, k=64, y=D):
    return call("plm_grouped_gemm_grad_w", dy, x, dt, off, e, m, n, k, y, None)


INT8 = {gemm: "gemm_int8", w8a8: "gemm_int8_w8a8", grouped8: "grouped_gemm_int8"}
EXPERTS = {grouped8: "grouped_gemm_int8", grouped: "grouped_gemm", grad_x: "grouped_gemm_grad_x", grad_w: "grouped_gemm_grad_w"}
ALL = {**INT8, **EXPERTS}


def refused(f, args, msg):
    rc, said = f(**args)
    assert rc == _lib.PLM_ERR_INVALID and said.startswith(f"{ALL[f]}: {msg}"), said


@pytest.mark.parametrize("f", ALL, ids=ALL.values())
@pytest.mark.parametrize("args,msg", [
    ({"dt": F32}, ""),
    ({"dt": 7}, ""),
    ({"m": -1}, "sizes must be non-negative"),
    ({"n": -32}, "sizes must be non-negative"),
    ({"k": -32}, "sizes must be non-negative"),
    ({"k": (1 << 19) + 32}, "N and K must be at most 2^19"),
    ({"n": (1 << 19) + 32}, "N and K must be at most 2^19"),
    ({"m": 1 << 24}, ""),
    ({"m": 1 << 62}, ""),
    ({"m": 1 << 20, "n": 1 << 17}, ""),
    ({"k": 68}, ""),
    ({"y": None}, "null pointer"),
    ({"x": None}, "null pointer"),
])
def test_products_refuse(f, args, msg):
    refused(f, args, msg)


@pytest.mark.parametrize("f", INT8, ids=INT8.values())
def test_int8_products_refuse(f):
    for args, msg in (({"k": 72}, "K must be a multiple of 16"), ({"k": 131072}, "K must be at most 131056"), ({"w": TWO}, "weight must be 16-byte"),
                      ({"s": TWO}, "scale must be 4-byte"), ({"w": None}, "null pointer"), ({"s": None}, "null pointer"), ({"y": ODD}, "y must be 2-byte")):
        refused(f, args, msg)
    refused(f, {"x": ODD}, "codes must be 16-byte" if f is gemm else "x must be 2-byte")
    refused(gemm, {"xs": TWO}, "x_scale must be 4-byte")


@pytest.mark.parametrize("f", EXPERTS, ids=EXPERTS.values())
def test_expert_products_refuse(f):
    for args, msg in (({"e": 0}, "n_experts must be in [1, 4096]"), ({"e": 4097}, "n_experts must be in [1, 4096]"), ({"off": None}, "offsets must be"),
                      ({"off": TWO}, "offsets must be"), ({"e": 4096, "n": 1 << 17, "k": 64}, "n_experts N K must be at most"),
                      ({"e": 4096, "n": 1 << 15, "k": 1 << 13}, "n_experts N K must be at most"), ({"e": 4096, "n": 64, "k": 1 << 17, "m": 4}, "")):
        refused(f, args, msg)
    if f in (grad_x, grad_w):
        refused(f, {"n": 44}, "N and K must be multiples of 8")
    if f is not grouped8:
        refused(f, {"x": ctypes.c_void_p(4104)}, "dy must be 16-byte" if f is grad_x else "x must be 16-byte")
    if f in (grouped, grad_x):
        refused(f, {"w": TWO}, "weight must be 16-byte")
        refused(f, {"w": None}, "null pointer")
    refused(grad_w, {"dy": ctypes.c_void_p(4104)}, "dy must be 16-byte")


@pytest.mark.parametrize("f", [w8a8, grouped8])
def test_workspace_refused(f):
    for args in ({"ws": None}, {"size": 0}):
        rc, said = f(**args)
        assert rc == _lib.PLM_ERR_WORKSPACE and "workspace of" in said
    refused(f, {"ws": ctypes.c_void_p(4096 + 64)}, "workspace must be 256-byte aligned")


def test_a_split_sum_needs_its_room():
    lib = _lib.load()
    m, n, k = 64, 4096, 12288
    need = lib.plm_gemm_int8_workspace_bytes(m, n, k)
    assert need > 0 and need % (m * n * 4) == 0
    rc, said = gemm(m=m, n=n, k=k, ws=None, size=0)
    assert rc == _lib.PLM_ERR_WORKSPACE and f"workspace of {need} bytes" in said
    rc, said = gemm(m=m, n=n, k=k, size=need - 1)
    assert rc == _lib.PLM_ERR_WORKSPACE
    assert lib.plm_gemm_int8_w8a8_workspace_bytes(m, n, k) >= need + m * k + 4 * m
    assert lib.plm_gemm_int8_workspace_bytes(4096, 24576, 4096) == 0


def test_quantizer_refuses():
    for f, args, msg in ((quantize, {"dt": 9}, "quantize_rows_int8: x must be fp32, fp16 or bf16"), (quantize, {"m": -1}, "quantize_rows_int8: M must be"),
                         (quantize, {"k": (1 << 28) + 1}, "quantize_rows_int8: M must be"), (quantize, {"m": 1 << 24}, "quantize_rows_int8: M must be"),
                         (quantize, {"x": ODD}, "quantize_rows_int8: x must be 2-byte"), (quantize, {"x": TWO, "dt": F32}, "quantize_rows_int8: x must be 4-byte"),
                         (quantize, {"scale": TWO}, "quantize_rows_int8: scale must be 4-byte"), (quantize, {"codes": None}, "quantize_rows_int8: null pointer"),
                         (dequantize, {"dt": 9}, "dequantize_rows_int8: out must be fp32"), (dequantize, {"out": ODD}, "dequantize_rows_int8: out must be 2-byte"),
                         (dequantize, {"m": 1 << 24}, "dequantize_rows_int8: M must be"), (dequantize, {"scale": None}, "dequantize_rows_int8: null pointer")):
        rc, said = f(**args)
        assert rc == _lib.PLM_ERR_INVALID and said.startswith(msg), said


def test_empty_calls_do_no_device_work():
    for f in (gemm, w8a8, grouped8, grouped):
        assert f(m=0, x=None, w=None)[0] == f(n=0, x=None, w=None, y=None)[0] == _lib.PLM_OK
    assert grad_x(m=0, x=None)[0] == grad_x(k=0, x=None)[0] == grad_w(n=0, y=None)[0] == grad_w(k=0, y=None)[0] == _lib.PLM_OK
    assert quantize(m=0, x=None)[0] == dequantize(m=0, out=None)[0] == dequantize(k=0, codes=None)[0] == _lib.PLM_OK


@pytest.mark.parametrize("name", ["plm_gemm_int8_workspace_bytes", "plm_gemm_int8_w8a8_workspace_bytes", "plm_grouped_gemm_int8_workspace_bytes"])
def test_workspace_queries_take_any_sizes(name):
    """Sizes that the call refuses need no workspace; the sizes are multiplied only once they are known to be small."""
    query = getattr(_lib.load(), name)
    for huge in (1 << 25, 1 << 32, 1 << 40, (1 << 63) - 1, -1, -(1 << 63)):
        for sizes in ((huge, 64, 64), (64, huge, 64), (64, 64, huge), (huge, huge, 64), (huge, 64, huge), (64, huge, huge), (huge, huge, huge)):
            assert query(*sizes) == 0, sizes
    for sizes in (((1 << 24) - 1, 64, 64), (1 << 17, 1 << 19, 131056), (1, 1 << 19, 131056), (1, 1, 16)):
        assert query(*sizes) >= 0


def test_python_refuses_host_tensors_and_wrong_shapes():
    x, c, s = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4)
    w, off = torch.zeros(2, 48, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    for mod in (ops, _host):
        for op, f in (("quantize_rows_int8", lambda: mod.quantize_rows_int8_cuda(x)), ("dequantize_rows_int8", lambda: mod.dequantize_rows_int8_cuda(c, s, torch.float32)),
                      ("gemm_int8", lambda: mod.gemm_int8_cuda(c, s, c, s, torch.bfloat16)), ("gemm_int8_w8a8", lambda: mod.gemm_int8_w8a8_cuda(x, c, s)),
                      ("grouped_gemm_int8", lambda: mod.grouped_gemm_int8_cuda(x, c[None], s[None], off)), ("grouped_gemm", lambda: mod.grouped_gemm_cuda(x, w, off)),
                      ("grouped_gemm_grad_x", lambda: mod.grouped_gemm_grad_x_cuda(x, w, off)), ("grouped_gemm_grad_w", lambda: mod.grouped_gemm_grad_w_cuda(x, x, off))):
            with pytest.raises(RuntimeError, match=f"^{op}: .*CUDA"):
                f()
