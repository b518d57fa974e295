"""Products of more tiles than the GPU holds at once, so that a workgroup takes several in turn: against float64, on every
tile shape."""

import random

import pytest
import torch

from pulsarlm_amd import ops
from tests import _dense as dense

pytestmark = pytest.mark.gpu

TILES = [f"t{i}" for i in range(6)]


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


# N a multiple of 8, of 4 and odd: three ways of storing; one to five stages of the sum, fewer than are in flight and more.
@pytest.mark.parametrize("kernel", TILES)
@pytest.mark.parametrize("m,n,k", [(4097, 4360, 64), (4100, 4364, 144), (4300, 4361, 528)])
def test_dense(m, n, k, kernel, tuning_env):
    tuning_env("PLM_DENSE", kernel)
    q, xs, w, ws = dense.codes(m, k, 1, low=-128), dense.scales(m, 2), dense.codes(n, k, 3, low=-128), dense.scales(n, 4)
    dense.within(ops.gemm_int8_cuda(q, xs, w, ws), *dense.int8_product(q, xs, w, ws), kernel)


def test_more_turns_than_a_workgroup_keeps(tuning_env):
    """33489 tiles of 64 x 64: past 64 for each of the workgroups that are resident."""
    tuning_env("PLM_DENSE", "t5")
    m = n = 11700
    q, xs, w, ws = dense.codes(m, 48, 1), dense.scales(m, 2), dense.codes(n, 48, 3), dense.scales(n, 4)
    y = ops.gemm_int8_cuda(q, xs, w, ws)
    for lo in range(0, m, 2340):
        dense.within(y[lo:lo + 2340], *dense.int8_product(q[lo:lo + 2340], xs[lo:lo + 2340], w, ws), f"rows from {lo}")


def uneven(experts, rows):
    """Most experts have a few rows, some none, one a third of all."""
    rng = random.Random(experts)
    counts = [rng.choice([0, 1, 5, 40, 2 * rows // (3 * experts)]) for _ in range(experts)]
    counts[experts // 3] = rows - sum(counts)
    assert counts[experts // 3] > 0
    return counts


# Up to 64 experts, whose products' tiles go by their rows, and more.
@pytest.mark.parametrize("kernel", [None, *TILES])
@pytest.mark.parametrize("experts,rows,n,k", [(40, 3000, 2056, 520), (130, 4500, 1288, 72)])
def test_experts(experts, rows, n, k, kernel, tuning_env):
    tuning_env("PLM_DENSE", kernel)
    counts, spare = uneven(experts, rows), 700
    x, dy = dense.values((rows + spare, k), torch.bfloat16, 1), dense.values((rows + spare, n), torch.bfloat16, 3)
    x[rows:], dy[rows:] = float("nan"), float("inf")
    w, off = dense.values((experts, n, k), torch.bfloat16, 2, scale=k**-0.5), dense.offsets(counts)
    y, dx, dw = ops.grouped_gemm_cuda(x, w, off), ops.grouped_gemm_grad_x_cuda(dy, w, off), ops.grouped_gemm_grad_w_cuda(dy, x, off)
    for what, got, (ref, err) in (("y", y, dense.grouped(x[:rows], w, counts)), ("dx", dx, dense.grad_x(dy[:rows], w, counts))):
        dense.within(got[:rows], ref, err, what)
        assert not got[rows:].any(), what
    for e, lo, hi in dense.by_expert(counts):
        a, b = dy[lo:hi].double(), x[lo:hi].double()
        dense.within(dw[e], a.t() @ b, dense.sums(hi - lo) * (a.abs().t() @ b.abs()), f"dw of {e}")


@pytest.mark.parametrize("kernel", [None, *TILES])
@pytest.mark.parametrize("experts,rows,n,k", [(40, 3000, 2056, 528), (130, 4500, 1285, 80)])
def test_8_bit_experts(experts, rows, n, k, kernel, tuning_env):
    tuning_env("PLM_DENSE", kernel)
    counts, spare = uneven(experts, rows), 700
    x = dense.values((rows + spare, k), torch.float16, 1)
    x[rows:] = float("nan")
    w, ws = dense.codes(experts * n, k, 2).view(experts, n, k), dense.scales(experts * n, 3).view(experts, n)
    y = ops.grouped_gemm_int8_cuda(x, w, ws, dense.offsets(counts))
    q, xs = (t.cuda() for t in dense.quantize(x))
    for e, lo, hi in dense.by_expert(counts):
        dense.within(y[lo:hi], *dense.int8_product(q[lo:hi], xs[lo:hi], w[e], ws[e]), f"expert {e}")
    assert not y[rows:].any()


def test_the_same_bits_on_every_call():
    counts = uneven(40, 3000)
    k, n = 520, 2056
    x, dy, w = dense.values((3000, k), torch.bfloat16, 1), dense.values((3000, n), torch.bfloat16, 3), dense.values((40, n, k), torch.bfloat16, 2)
    off, first = dense.offsets(counts), None
    for _ in range(4):
        out = ops.grouped_gemm_cuda(x, w, off), ops.grouped_gemm_grad_x_cuda(dy, w, off), ops.grouped_gemm_grad_w_cuda(dy, x, off)
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(first, out))


@pytest.mark.parametrize("kernel", [None, "t0", "t2", "t5"])
@pytest.mark.parametrize("experts", [1, 2, 7, 8, 9, 31, 32, 33, 39, 40, 63, 64, 65, 127, 128, 129, 257])
def test_weights_gradient_of_any_number_of_experts(experts, kernel, tuning_env):
    """Their tiles are shared out by expert from some number on, and by their rows up to another."""
    tuning_env("PLM_DENSE", kernel)
    rng = random.Random(experts)
    counts = [rng.choice([0, 1, 3, 70, 130]) for _ in range(experts)]
    rows, n, k = sum(counts), 520, 264
    dy, x = dense.values((rows + 5, n), torch.bfloat16, 1), dense.values((rows + 5, k), torch.bfloat16, 2)
    dw = ops.grouped_gemm_grad_w_cuda(dy, x, dense.offsets(counts))
    dense.within(dw, *dense.grad_w(dy[:rows], x[:rows], counts), kernel)
