"""Products grouped by expert with ragged sizes on the GPU against float64: 8-bit and 16-bit experts, and the 16-bit ones'
gradients."""

import numpy as np
import pytest
import torch

from pulsarlm_amd import ops
from tests import _dense as dense

pytestmark = pytest.mark.gpu

KERNELS = [None, "r16", "r32", "r64", *(f"t{i}" for i in range(6))]
# Rows of each expert: none, one, whole and part blocks; one expert; more experts than a wavefront's lanes.
COUNTS = {
    "few": [3, 0, 1, 17],
    "one": [70],
    "blocks": [256, 0, 257, 255, 1, 64, 128],
    "ends empty": [0, 0, 5, 40, 0],
    "none": [0, 0, 0],
    "many": [(7 * i) % 5 for i in range(200)],
    "skewed": [1, 600, 0, 2, 33],
}


def inputs(counts, n, k, dtype, spare=0, seed=0):
    rows = sum(counts) + spare
    x = dense.values((rows, k), dtype, seed + 1)
    w = dense.values((len(counts), n, k), dtype, seed + 2, scale=k**-0.5)
    dy = dense.values((rows, n), dtype, seed + 3)
    if spare:  # a padded batch's spare rows hold anything
        x[-spare:], dy[-spare:] = float("nan"), float("inf")
    return x, w, dy, dense.offsets(counts)


def check(counts, n, k, dtype, spare=0):
    x, w, dy, off = inputs(counts, n, k, dtype, spare)
    end = sum(counts)
    y, dx, dw = ops.grouped_gemm_cuda(x, w, off), ops.grouped_gemm_grad_x_cuda(dy, w, off), ops.grouped_gemm_grad_w_cuda(dy, x, off)
    for what, got, (ref, err) in (("y", y, dense.grouped(x[:end], w, counts)), ("dx", dx, dense.grad_x(dy[:end], w, counts))):
        dense.within(got[:end], ref, err, what)
        assert not got[end:].any(), what
    dense.within(dw, *dense.grad_w(dy[:end], x[:end], counts), "dw")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("spare", [0, 37])
@pytest.mark.parametrize("counts", COUNTS)
def test_16_bit_experts(counts, spare, dtype):
    check(COUNTS[counts], 72, 136, dense.DT[dtype], spare)


@pytest.mark.parametrize("kernel", KERNELS[1:])
@pytest.mark.parametrize("counts,n,k", [("blocks", 264, 520), ("few", 8, 8), ("skewed", 520, 200), ("many", 136, 72)])
def test_16_bit_experts_on_every_kernel(counts, n, k, kernel, tuning_env):
    tuning_env("PLM_DENSE", kernel)
    check(COUNTS[counts], n, k, torch.bfloat16, spare=19)


@pytest.mark.parametrize("n,k", [(8, 2080), (1000, 16), (5, 64), (33, 128)])
def test_odd_output_sizes(n, k):
    counts = COUNTS["skewed"]
    x, w, _, off = inputs(counts, n, k, torch.bfloat16)
    dense.within(ops.grouped_gemm_cuda(x, w, off), *dense.grouped(x, w, counts))


def check_int8(counts, n, k, dtype, spare=0):
    rows, end = sum(counts) + spare, sum(counts)
    x = dense.values((rows, k), dtype, 1)
    x[end:] = float("nan")
    w, ws = dense.codes(len(counts) * n, k, 2).view(-1, n, k), dense.scales(len(counts) * n, 3).view(-1, n)
    y = ops.grouped_gemm_int8_cuda(x, w, ws, dense.offsets(counts))
    q, xs = (t.cuda() for t in dense.quantize(x))
    for e, lo, hi in dense.by_expert(counts):
        dense.within(y[lo:hi], *dense.int8_product(q[lo:hi], xs[lo:hi], w[e], ws[e]), f"expert {e}")
    assert not y[end:].any()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("spare", [0, 37])
@pytest.mark.parametrize("counts", COUNTS)
def test_8_bit_experts(counts, spare, dtype):
    check_int8(COUNTS[counts], 72, 144, dense.DT[dtype], spare)


@pytest.mark.parametrize("kernel", KERNELS[1:])
@pytest.mark.parametrize("counts,n,k", [("blocks", 264, 528), ("few", 5, 16), ("skewed", 520, 208), ("many", 130, 64)])
def test_8_bit_experts_on_every_kernel(counts, n, k, kernel, tuning_env):
    tuning_env("PLM_DENSE", kernel)
    check_int8(COUNTS[counts], n, k, torch.float16, spare=19)


def both(counts, n, k, spare, seed=0):
    """The two forward operators as f(offsets, out) with rows of their own, and their outputs' shape."""
    rows = sum(counts) + spare
    x = dense.values((rows, k), torch.bfloat16, seed + 1)
    w16 = dense.values((len(counts), n, k), torch.bfloat16, seed + 2)
    w8, ws = dense.codes(len(counts) * n, k, seed + 3).view(-1, n, k), dense.scales(len(counts) * n, seed + 4).view(-1, n)
    return (lambda off, out=None: ops.grouped_gemm_cuda(x, w16, off, out=out),
            lambda off, out=None: ops.grouped_gemm_int8_cuda(x, w8, ws, off, out=out)), (rows, n)


@pytest.mark.parametrize("kernel", [None, "r16", "t0", "t4"])
def test_rows_past_the_last_expert_stay_in_out(kernel, tuning_env):
    tuning_env("PLM_DENSE", kernel)
    counts = [5, 0, 300, 2]
    fs, shape = both(counts, 40, 64, spare=100)
    off, end = dense.offsets(counts), sum(counts)
    for f in fs:
        out = torch.full(shape, 7.0, dtype=torch.bfloat16, device="cuda")
        assert f(off, out) is out
        assert (out[end:] == 7).all() and torch.equal(out[:end], f(off)[:end])


@pytest.mark.parametrize("kernel", [None, "t0", "t4", "r16"])
@pytest.mark.parametrize("bad,counts", [([10, 4, 25, 30], [10, 0, 15, 5]), ([-5, 12, 90, 20], [0, 12, 28, 0]), ([40, 40, 1, -7], [40, 0, 0, 0]),
                                        ([2**31 - 1, 0, -(2**31), 3], [40, 0, 0, 0])])
def test_offsets_that_are_none(bad, counts, kernel, tuning_env):
    """Taken within the rows, and no less than an earlier one: never two experts' rows at once."""
    tuning_env("PLM_DENSE", kernel)
    fs, _ = both([10] * 4, 40, 64, spare=0)
    off = torch.tensor(bad, dtype=torch.int32, device="cuda")
    for f in fs:
        assert torch.equal(f(off), f(dense.offsets(counts)))
    x, w, dy, _ = inputs([10] * 4, 40, 64, torch.bfloat16)
    assert torch.equal(ops.grouped_gemm_grad_x_cuda(dy, w, off), ops.grouped_gemm_grad_x_cuda(dy, w, dense.offsets(counts)))
    assert torch.equal(ops.grouped_gemm_grad_w_cuda(dy, x, off), ops.grouped_gemm_grad_w_cuda(dy, x, dense.offsets(counts)))


def test_experts_do_not_meet():
    """What is not finite in one expert's rows or weight stays with it."""
    counts, n, k = [30, 41, 5, 60], 72, 64
    x, w, dy, off = inputs(counts, n, k, torch.bfloat16)
    clean = ops.grouped_gemm_cuda(x, w, off), ops.grouped_gemm_grad_x_cuda(dy, w, off), ops.grouped_gemm_grad_w_cuda(dy, x, off)
    x[35], dy[40], w[1, 3, 3] = float("nan"), float("inf"), float("nan")
    dirty = ops.grouped_gemm_cuda(x, w, off), ops.grouped_gemm_grad_x_cuda(dy, w, off), ops.grouped_gemm_grad_w_cuda(dy, x, off)
    for c, d in zip(clean[:2], dirty[:2]):
        assert torch.equal(c[:30], d[:30]) and torch.equal(c[71:], d[71:])
    assert torch.equal(clean[2][[0, 2, 3]], dirty[2][[0, 2, 3]]) and dirty[2][1].isnan().any()


def test_most_experts():
    """4096 experts, of which a few have rows, past the first chunks of their scan."""
    counts = [0] * 4096
    counts[0], counts[63], counts[64], counts[2500], counts[4095] = 3, 1, 20, 2, 9
    check(counts, 8, 16, torch.bfloat16, spare=5)
    check_int8(counts, 8, 16, torch.bfloat16, spare=5)


@pytest.mark.parametrize("rows,n,k", [(0, 8, 16), (12, 0, 16), (12, 8, 0), (0, 0, 0)])
def test_empty_sizes(rows, n, k):
    x, dy = torch.ones(rows, k, device="cuda").bfloat16(), torch.ones(rows, n, device="cuda").bfloat16()
    w, off = torch.ones(3, n, k, device="cuda").bfloat16(), torch.tensor([rows // 2] * 2 + [rows], dtype=torch.int32, device="cuda")
    y, dx, dw = ops.grouped_gemm_cuda(x, w, off), ops.grouped_gemm_grad_x_cuda(dy, w, off), ops.grouped_gemm_grad_w_cuda(dy, x, off)
    assert y.shape == (rows, n) and dx.shape == (rows, k) and dw.shape == (3, n, k)
    assert not dw.any() if rows == 0 else True
    assert not y.any() and not dx.any()
    z = ops.grouped_gemm_int8_cuda(x, w.to(torch.int8), torch.ones(3, n, device="cuda"), off)
    assert z.shape == (rows, n) and not z.any()


def test_gradients_against_differences():
    """The products are linear in x and in W: with small integers, whose sums all three types hold, the difference along a
    direction is the gradient's product with it, to the bit."""
    counts, n, k = [20, 0, 33, 7], 104, 96
    g = torch.Generator().manual_seed(1)

    def small(*shape):
        return torch.randint(-1, 2, shape, generator=g).bfloat16().cuda()

    off, rows = dense.offsets(counts), sum(counts)
    x, vx, w, vw, dy = small(rows, k), small(rows, k), small(4, n, k), small(4, n, k), small(rows, n)
    dx, dw = ops.grouped_gemm_grad_x_cuda(dy, w, off), ops.grouped_gemm_grad_w_cuda(dy, x, off)

    def f(x, w):
        return (ops.grouped_gemm_cuda(x, w, off).double() * dy.double()).sum()

    assert (f(x + vx, w) - f(x - vx, w)) / 2 == (dx.double() * vx.double()).sum() != 0
    assert (f(x, w + vw) - f(x, w - vw)) / 2 == (dw.double() * vw.double()).sum() != 0


@pytest.mark.parametrize("kernel", [None, "t0"])
def test_captured_with_other_offsets_on_each_replay(kernel, tuning_env):
    """The experts' sizes are read on the device: a captured step follows its offsets' values."""
    tuning_env("PLM_DENSE", kernel)
    n, k, rows = 72, 64, 300
    x, w, dy, _ = inputs([rows, 0, 0, 0, 0], n, k, torch.bfloat16)
    w8, ws = dense.codes(5 * n, k, 2).view(5, n, k), dense.scales(5 * n, 3).view(5, n)
    off = dense.offsets([rows, 0, 0, 0, 0])

    def step(off):
        return (ops.grouped_gemm_cuda(x, w, off), ops.grouped_gemm_grad_x_cuda(dy, w, off), ops.grouped_gemm_grad_w_cuda(dy, x, off),
                ops.grouped_gemm_int8_cuda(x, w8, ws, off))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(off)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(off)
    for counts in ([0, 1, 200, 0, 99], [60] * 5, [0, 0, 0, 0, 10], [299, 1, 0, 0, 0]):
        off.copy_(dense.offsets(counts))
        graph.replay()
        want = step(dense.offsets(counts))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), counts


def test_same_bits_on_every_call():
    counts, n, k = [300, 1, 0, 517], 520, 264
    x, w, dy, off = inputs(counts, n, k, torch.bfloat16)
    first = None
    for _ in range(5):
        out = ops.grouped_gemm_cuda(x, w, off), ops.grouped_gemm_grad_x_cuda(dy, w, off), ops.grouped_gemm_grad_w_cuda(dy, x, off)
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(first, out))


def test_on_two_streams_at_once():
    """Calls on other streams than the tensors' own, each with scratch of its own."""
    counts, n, k = [60, 0, 211, 5], 264, 144
    x, w, dy, off = inputs(counts, n, k, torch.bfloat16)
    w8, ws = dense.codes(4 * n, k, 2).view(4, n, k), dense.scales(4 * n, 3).view(4, n)

    def step():
        return (ops.grouped_gemm_cuda(x, w, off), ops.grouped_gemm_grad_x_cuda(dy, w, off), ops.grouped_gemm_grad_w_cuda(dy, x, off),
                ops.grouped_gemm_int8_cuda(x, w8, ws, off))

    want = step()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(10):
        with torch.cuda.stream(streams[i % 2]):
            got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_a_weight_shared_by_every_expert():
    """A broadcast weight: refused as it is, and its gradient the sum of the copies'."""
    counts, n, k = [7, 30, 0, 63], 40, 64
    x, _, dy, off = inputs(counts, n, k, torch.bfloat16)
    one = dense.values((1, n, k), torch.float32, 5).requires_grad_()
    with pytest.raises(RuntimeError, match="weight must be contiguous"):
        ops.grouped_gemm_cuda(x, one.detach().bfloat16().expand(4, n, k), off)
    y = ops.grouped_gemm_cuda(x, one.bfloat16().expand(4, n, k).contiguous(), off)
    y.backward(dy)
    ref = dy.double().t() @ x.double()
    # Each expert's sum rounded to bf16, then three additions of them, rounded as well: six half steps of what they add up to.
    bound = dense.sums(100) * (dy.double().abs().t() @ x.double().abs())
    parts = sum((dy[lo:hi].double().t() @ x[lo:hi].double()).abs() for _, lo, hi in dense.by_expert(counts))
    assert ((one.grad[0].double() - ref).abs() <= bound + 6 * 2.0**-8 * (parts + bound)).all()
