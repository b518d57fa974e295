"""8-bit and expert products whose operands or outputs pass 2^31 elements and 2^32 bytes: samples against float64."""

import pytest
import torch

from pulsarlm_amd import ops
from tests import _dense as dense

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


def device_codes(shape, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randint(-127, 128, shape, generator=g, dtype=torch.int8, device="cuda")


def device_values(shape, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, dtype=torch.bfloat16, device="cuda")


def test_quantizer():
    m, k = 140001, 16400  # 2.3e9 values
    x = device_values((m, k), 1)
    codes, scale = ops.quantize_rows_int8_cuda(x)
    back = ops.dequantize_rows_int8_cuda(codes, scale, torch.bfloat16)
    at = torch.tensor([0, 1, m // 2, (1 << 31) // k, m - 2, m - 1], device="cuda")
    q, s = dense.quantize(x[at])
    assert torch.equal(codes[at].cpu(), q) and torch.equal(scale[at].cpu(), s)
    assert torch.equal(back[at].cpu(), (q.float() * s[:, None]).bfloat16())


def test_quantizer_of_more_rows_than_a_grid_of_wide_workgroups():
    m, k = (1 << 22) + 3, 8200  # 69 GB
    x = torch.zeros((m, k), dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 1 << 21, (1 << 22) - 1, 1 << 22, m - 1], device="cuda")
    x[at] = device_values((5, k), 1)
    codes, scale = ops.quantize_rows_int8_cuda(x)
    q, s = dense.quantize(x[at])
    assert torch.equal(codes[at].cpu(), q) and torch.equal(scale[at].cpu(), s)
    others = torch.ones(m, dtype=torch.bool, device="cuda")
    others[at] = False
    assert (scale[others] == dense.row_scale(torch.zeros(1, 8))[0].item()).all()
    used = torch.cat([part.view(torch.int64).any(dim=1) for part in codes.split(1 << 19)])
    assert torch.equal(used.nonzero()[:, 0], at)


def test_rows():
    m, n, k = 140001, 16400, 64  # 2.3e9 outputs
    q, xs, w, ws = device_codes((m, k), 1), dense.scales(m, 2), device_codes((n, k), 3), dense.scales(n, 4)
    at = torch.tensor([0, 1, m // 2, (1 << 31) // n, m - 129, m - 2, m - 1], device="cuda")
    y = ops.gemm_int8_cuda(q, xs, w, ws)
    dense.within(y[at], *dense.int8_product(q[at], xs[at], w, ws))


def test_a_weight():
    n, k = 1 << 19, 8208  # 4.3e9 codes
    w, ws = device_codes((n, k), 1), dense.scales(n, 2)
    at = torch.tensor([0, 17, n // 2 - 1, n // 2, n - 130, n - 1], device="cuda")
    for m in (1, 20, 300):
        x = dense.values((m, k), torch.bfloat16, 3)
        q, xs = dense.quantize(x)
        y = ops.gemm_int8_w8a8_cuda(x, w, ws)
        dense.within(y[:, at], *dense.int8_product(q.cuda(), xs.cuda(), w[at], ws[at]), f"{m} rows")


def test_many_rows_of_experts():
    """x, y and dy of 2.3e9 values: forward and both gradients, the weights' over sums that begin past 2^31 elements."""
    counts = [5000, 0, 134801, 200]
    rows, n, k = 140001, 16400, 72
    w, off = dense.values((4, n, k), torch.bfloat16, 1), dense.offsets(counts)
    x = device_values((rows, k), 2)
    y = ops.grouped_gemm_cuda(x, w, off)
    at = torch.tensor([0, 4999, 5000, (1 << 31) // n, 139800, 139801, 140000], device="cuda")
    for r in at.tolist():
        e = 0 if r < 5000 else 2 if r < 139801 else 3
        a, b = x[r:r + 1].double(), w[e].double()
        dense.within(y[r:r + 1], a @ b.t(), dense.sums(k) * (a.abs() @ b.abs().t()), f"row {r}")
    dx = ops.grouped_gemm_grad_x_cuda(y, w, off)
    for r in at.tolist():
        e = 0 if r < 5000 else 2 if r < 139801 else 3
        a, b = y[r:r + 1].double(), w[e].double()
        dense.within(dx[r:r + 1], a @ b, dense.sums(n) * (a.abs() @ b.abs()), f"row {r}")
    dw = ops.grouped_gemm_grad_w_cuda(y, x, off)
    assert not dw[1].any()
    cols = torch.tensor([0, 1, n // 2, n - 1], device="cuda")
    for e, lo, hi in dense.by_expert(counts):
        a, b = y[lo:hi][:, cols].double().t().contiguous(), x[lo:hi].double()
        dense.within(dw[e][cols], a @ b, dense.sums(hi - lo) * (a.abs() @ b.abs()), f"dw of {e}")


def test_experts_past_4_gib():
    """16-bit experts of 4.3e9 values in all, and 8-bit ones; few rows and many."""
    experts, n, k = 64, 8200, 8192
    w = torch.empty(experts, n, k, dtype=torch.bfloat16, device="cuda")
    for e in range(experts):
        w[e] = device_values((n, k), e)
    for counts in ([0] * 60 + [1, 0, 3, 7], [0] * 60 + [100, 30, 0, 300]):
        rows, off = sum(counts), dense.offsets(counts)
        x, dy = dense.values((rows, k), torch.bfloat16, 1), dense.values((rows, n), torch.bfloat16, 2)
        y, dx = ops.grouped_gemm_cuda(x, w, off), ops.grouped_gemm_grad_x_cuda(dy, w, off)
        dw = ops.grouped_gemm_grad_w_cuda(dy, x, off)
        for e, lo, hi in dense.by_expert(counts)[60:]:
            a, d, b = x[lo:hi].double(), dy[lo:hi].double(), w[e].double()
            dense.within(y[lo:hi], a @ b.t(), dense.sums(k) * (a.abs() @ b.abs().t()), f"y of {e}")
            dense.within(dx[lo:hi], d @ b, dense.sums(n) * (d.abs() @ b.abs()), f"dx of {e}")
            dense.within(dw[e], d.t() @ a, dense.sums(hi - lo) * (d.abs().t() @ a.abs()), f"dw of {e}")
        assert not dw[:60].any()
        del dw
    w8, ws = device_codes((experts, n, k), 5), torch.rand(experts, n, device="cuda") * 0.01
    for counts in ([0] * 60 + [1, 0, 3, 7], [0] * 60 + [100, 30, 0, 300]):
        x = dense.values((sum(counts), k), torch.bfloat16, 1)
        y = ops.grouped_gemm_int8_cuda(x, w8, ws, dense.offsets(counts))
        q, xs = (t.cuda() for t in dense.quantize(x))
        for e, lo, hi in dense.by_expert(counts)[60:]:
            dense.within(y[lo:hi], *dense.int8_product(q[lo:hi], xs[lo:hi], w8[e], ws[e]), f"8-bit expert {e}")
