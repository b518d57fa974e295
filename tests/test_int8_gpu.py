"""The 8-bit operators on the GPU against float64: the row quantizer, its inverse, and the products with a scale for each
token and channel."""

import numpy as np
import pytest
import torch

from pulsarlm_amd import ops
from tests import _dense as dense

pytestmark = pytest.mark.gpu

# The kernels that a call can run on: by the rule, each block of the kernel for few rows, each tile shape.
KERNELS = [None, "r16", "r32", "r64", *(f"t{i}" for i in range(6)), "t0,3", "t2,2", "t3,5", "t4,16", "t5,4"]


def check_quantizer(x):
    codes, scale = ops.quantize_rows_int8_cuda(x)
    q, s = dense.quantize(x)
    assert torch.equal(scale.cpu().view(torch.int32)[~s.isnan()], s.view(torch.int32)[~s.isnan()])
    assert torch.equal(scale.cpu().isnan(), s.isnan())
    assert torch.equal(codes.cpu(), q)
    return codes, scale


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("m,k", [(1, 4096), (1, 1), (3, 7), (5, 33), (300, 520), (600, 1288), (2, 70000), (513, 24)])
def test_quantizer(m, k, dtype):
    check_quantizer(dense.values((m, k), dense.DT[dtype], seed=m + k))


def test_quantizer_without_columns_or_rows():
    codes, scale = ops.quantize_rows_int8_cuda(torch.empty(3, 0, dtype=torch.bfloat16, device="cuda"))
    assert codes.shape == (3, 0) and torch.equal(scale.cpu(), dense.row_scale(torch.zeros(3, 1)))
    codes, scale = ops.quantize_rows_int8_cuda(torch.empty(0, 16, dtype=torch.bfloat16, device="cuda"))
    assert codes.shape == (0, 16) and scale.shape == (0,)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("k", [64, 61])
def test_quantizer_rows_apart(k, dtype):
    """Zeros, the largest and the smallest magnitudes, values that are not finite: each row by itself."""
    dt = dense.DT[dtype]
    x = dense.values((12, k), dt, seed=3)
    info = torch.finfo(dt)
    x[1] = 0
    x[2] = info.max
    x[3] = -info.max * x[3].abs().float().div(8).clamp(max=1).to(dt)
    x[4] *= info.tiny
    x[5, k - 1] = float("inf")
    x[6, 0] = float("-inf")
    x[7, 5] = float("nan")
    x[8] = -0.0
    x[9, 7] = info.max
    codes, scale = check_quantizer(x)
    assert scale[5:8].isnan().all() and not codes[5:8].any() and not codes[1].any()


def test_quantizer_ties_go_to_the_even_code():
    """Scale 1: halves are ties. Scales of three bits more: exact ties at other places."""
    halves = torch.arange(-126.5, 127, 1.0)
    x = torch.cat([halves, torch.tensor([127.0, -127.0])]).repeat(3, 1) * torch.tensor([[1.0], [0.125], [24.0]])
    codes, scale = check_quantizer(x.cuda())
    assert scale.tolist() == [1.0, 0.125, 24.0]
    assert not (codes[:, :254] % 2).any()


@pytest.mark.parametrize("top", [1.0, 3.0, 0.7, 5e4, 1e-3])
def test_quantizer_next_to_every_border(top):
    """fp32 values on both sides of every border between two codes."""
    s = np.float32(top) / np.float32(127)
    border = ((np.arange(-127, 127) + 0.5) * np.float64(s)).astype(np.float32)
    near = np.concatenate([border, np.nextafter(border, np.float32(np.inf)), np.nextafter(border, np.float32(-np.inf)), [np.float32(top)]])
    check_quantizer(torch.from_numpy(near.astype(np.float32))[None].cuda())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("top", [1.0, 0.9453125, 113.0, 2.0**-9 * 1.7])
def test_quantizer_every_16_bit_value(top, dtype):
    dt = dense.DT[dtype]
    v = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dt)
    v = v[v.isfinite()]
    v = v[v.abs() <= top]
    check_quantizer(torch.cat([v, torch.tensor([top], dtype=dt)])[None].cuda())


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("at", [1, 4])
def test_quantizer_unaligned(at, dtype):
    m, k = 5, 48
    x = dense.values((1, at + m * k), dense.DT[dtype], seed=1).view(-1)[at:].view(m, k)
    check_quantizer(x)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("m,k,at", [(1, 16, 0), (7, 33, 0), (300, 4096, 0), (5, 48, 3), (20000, 16, 0)])
def test_dequantizer(m, k, at, dtype):
    dt = dense.DT[dtype]
    codes = dense.codes(1, at + m * k, seed=m, low=-128).view(-1)[at:].view(m, k)
    scale = dense.scales(m, seed=k)
    out = ops.dequantize_rows_int8_cuda(codes, scale, dt)
    assert out.dtype == dt and torch.equal(out, (codes.float() * scale[:, None]).to(dt))


def test_quantized_and_back():
    x = dense.values((40, 200), torch.float32, seed=1)
    codes, scale = ops.quantize_rows_int8_cuda(x)
    back = ops.dequantize_rows_int8_cuda(codes, scale, torch.float32)
    # Half a code's step, and the product's rounding.
    assert ((back - x).abs() <= 0.5 * scale[:, None] * (1 + 2.0**-20) + 2.0**-24 * back.abs()).all()


def check_product(m, n, k, dtype, seed=0, out=None):
    q, xs, w, ws = dense.codes(m, k, seed + 1, low=-128), dense.scales(m, seed + 2), dense.codes(n, k, seed + 3, low=-128), dense.scales(n, seed + 4)
    y = ops.gemm_int8_cuda(q, xs, w, ws, dtype, out=out)
    dense.within(y, *dense.int8_product(q, xs, w, ws), f"{m} {n} {k}")
    return y


@pytest.mark.parametrize("m", [1, 2, 15, 17, 33, 64, 65, 130, 300])
@pytest.mark.parametrize("n,k", [(1, 16), (7, 48), (130, 144), (520, 1040), (64, 4128)])
def test_product(m, n, k):
    check_product(m, n, k, torch.bfloat16 if (m + n) % 2 else torch.float16)


@pytest.mark.parametrize("kernel", KERNELS[1:])
@pytest.mark.parametrize("m,n,k", [(1, 260, 128), (64, 24, 400), (257, 515, 272), (300, 264, 16), (129, 1000, 640)])
def test_product_on_every_kernel(m, n, k, kernel, tuning_env):
    tuning_env("PLM_DENSE", kernel)
    if kernel[0] == "r" and int(kernel[1:]) < 64 and m > 257:
        m = 200  # several row blocks all the same
    check_product(m, n, k, torch.bfloat16)


@pytest.mark.parametrize("kernel", ["r16", "r64", "t0", "t4"])
@pytest.mark.parametrize("at", [1, 4])
def test_product_into_an_unaligned_out(at, kernel, tuning_env):
    tuning_env("PLM_DENSE", kernel)
    m, n = 70, 136
    room = torch.full((m * n + 16,), 7.0, dtype=torch.bfloat16, device="cuda")
    y = check_product(m, n, 256, torch.bfloat16, out=room[at : at + m * n].view(m, n))
    assert y.data_ptr() == room.data_ptr() + 2 * at
    assert (room[:at] == 7).all() and (room[at + m * n :] == 7).all()


@pytest.mark.parametrize("m", [2, 100])
def test_product_of_the_largest_codes(m):
    """128 * 128 * 131056 is the largest sum of 31 bits."""
    n, k = 24, 131056
    q, w = torch.full((m, k), -128, dtype=torch.int8, device="cuda"), torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    xs, ws = dense.scales(m, 1) * 1e-4, dense.scales(n, 2)
    y = ops.gemm_int8_cuda(q, xs, w, ws, torch.float16)
    dense.within(y, *dense.int8_product(q, xs, w, ws))


def test_product_scales_at_the_ends_of_fp32():
    """Sums beyond fp32's range with one scale that come back with the other."""
    q, w = dense.codes(20, 64, 1), dense.codes(40, 64, 2)
    xs, ws = torch.full((20,), 1e36, device="cuda"), torch.full((40,), 1e-36, device="cuda")
    dense.within(ops.gemm_int8_cuda(q, xs, w, ws), *dense.int8_product(q, xs, w, ws))
    xs[3], xs[4] = float("nan"), 0.0
    y = ops.gemm_int8_cuda(q, xs, w, ws)
    assert y[3].isnan().all() and not y[4].any() and y[5:].isfinite().all()


@pytest.mark.parametrize("n", [0, 5])
@pytest.mark.parametrize("m", [0, 4])
@pytest.mark.parametrize("k", [0, 32])
def test_empty_sizes(m, n, k):
    x = torch.randn(m, k, device="cuda").bfloat16()
    w, s = torch.ones(n, k, dtype=torch.int8, device="cuda"), torch.ones(n, device="cuda")
    y = ops.gemm_int8_w8a8_cuda(x, w, s)
    z = ops.gemm_int8_cuda(*ops.quantize_rows_int8_cuda(x), w, s)
    assert y.shape == z.shape == (m, n) and (k > 0 or (not y.any() and not z.any()))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("m,n,k", [(1, 100, 4096), (3, 520, 144), (16, 64, 2048), (40, 130, 1040), (333, 500, 4128), (700, 264, 512)])
def test_w8a8(m, n, k, dtype):
    x = dense.values((m, k), dense.DT[dtype], seed=m)
    x[0, : k // 2] = 0
    w, ws = dense.codes(n, k, 3), dense.scales(n, 4)
    y = ops.gemm_int8_w8a8_cuda(x, w, ws)
    q, xs = ops.quantize_rows_int8_cuda(x)
    assert y.dtype == x.dtype and torch.equal(y, ops.gemm_int8_cuda(q, xs, w, ws, x.dtype))
    q, xs = dense.quantize(x)
    dense.within(y, *dense.int8_product(q.cuda(), xs.cuda(), w, ws))


@pytest.mark.parametrize("m,k", [(1, 16), (1, 65536), (1, 65552), (2, 32768), (2, 32784), (3, 2720), (3, 2736), (4, 2048), (4, 2064), (5, 1024)])
def test_w8a8_where_the_product_quantizes_and_where_not(m, k):
    x, w, ws = dense.values((m, k), torch.bfloat16, 1), dense.codes(72, k, 2), dense.scales(72, 3)
    x[-1] = 0
    q, xs = ops.quantize_rows_int8_cuda(x)
    y = ops.gemm_int8_w8a8_cuda(x, w, ws)
    dense.within(y, *dense.int8_product(q, xs, w, ws))
    assert not y[-1].any()


@pytest.mark.parametrize("m", [3, 100])
def test_w8a8_keeps_rows_apart(m):
    """A row that is not finite is NaN, the others do not change."""
    n, k = 72, 256
    x, w, ws = dense.values((m, k), torch.bfloat16, 1), dense.codes(n, k, 2), dense.scales(n, 3)
    y = ops.gemm_int8_w8a8_cuda(x, w, ws)
    x[1, 7] = float("inf")
    z = ops.gemm_int8_w8a8_cuda(x, w, ws)
    assert z[1].isnan().all() and torch.equal(z[0], y[0]) and torch.equal(z[2:], y[2:])


def test_w8a8_unaligned_x():
    m, n, k = 20, 72, 64
    x = dense.values((1, 3 + m * k), torch.bfloat16, 1).view(-1)[3:].view(m, k)
    w, ws = dense.codes(n, k, 2), dense.scales(n, 3)
    assert torch.equal(ops.gemm_int8_w8a8_cuda(x, w, ws), ops.gemm_int8_w8a8_cuda(x.clone(), w, ws))


@pytest.mark.parametrize("m", [1, 40, 300])
def test_captured_and_on_two_streams(m):
    """A captured call replayed over new inputs, with eager calls and synchronizations between; and eager calls on two
    streams at once: each has its own scratch."""
    n, k = 264, 512
    w, ws = dense.codes(n, k, 2), dense.scales(n, 3)
    inputs = [dense.values((m, k), torch.bfloat16, s) for s in range(4)]
    expected = [ops.gemm_int8_w8a8_cuda(x, w, ws) for x in inputs]
    x = inputs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.gemm_int8_w8a8_cuda(x, w, ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.gemm_int8_w8a8_cuda(x, w, ws)
    for new, want in zip(inputs, expected):
        x.copy_(new)
        graph.replay()
        ops.gemm_int8_w8a8_cuda(inputs[1], w, ws)
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            got.append(ops.gemm_int8_w8a8_cuda(inputs[i % 4], w, ws))
    torch.cuda.synchronize()
    assert all(torch.equal(g, expected[i % 4]) for i, g in enumerate(got))
