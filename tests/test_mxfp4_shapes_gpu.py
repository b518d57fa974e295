"""The MXFP4 products at sizes that take each of their kernels' shapes (on 256 CUs), unaligned outputs, operands
that are not contiguous, work on two streams at once, and what the Python layer refuses."""

import numpy as np
import pytest
import torch

from pulsarlm_amd import ops
from tests import _mxfp4 as mx
from tests.test_mxfp4_gpu import mlp_reference

pytestmark = pytest.mark.gpu

BOTH = pytest.mark.parametrize("dtype", ["bf16", "fp16"])
K = 1184  # ten K tiles, the last one a quarter full: turns of every stage count, and a last turn that is not whole

# Every tile shape with 16-bit x, once where whole rows leave and once where they cannot.
TILES_W4A16 = [(33, 33), (33, 8), (4125, 65), (4125, 104), (4125, 200), (3288, 264), (3381, 200), (2668, 264), (3629, 513), (3629, 520),
               (3598, 1034), (3598, 1032), (3598, 2050), (3598, 2056), (3846, 2050), (3846, 2056), (1924, 6100), (1924, 6104)]


@BOTH
@pytest.mark.parametrize("m,n", TILES_W4A16)
def test_tiles_w4a16(m, n, dtype):
    w, x = mx.Weight(n, K, seed=n), mx.rows(m, K, mx.DT[dtype], seed=m)
    mx.within(ops.gemm_mxfp4_cuda(x, *w.packed, n), *mx.product(x.double(), w.dense), "W4A16")


@BOTH
@pytest.mark.parametrize("m,n", [(33, 33), (33, 8), (3598, 513), (3598, 520), (3598, 1034), (3598, 1032), (3846, 2050), (3846, 2056),
                                 (2575, 6100), (2575, 6104)])
def test_tiles_w4a4(m, n, dtype):
    w, x = mx.Weight(n, K, seed=n), mx.rows(m, K, mx.DT[dtype], seed=m)
    mx.within(ops.gemm_mxfp4_w4a4_cuda(x, *w.packed, n), *mx.product(mx.rounded(x), w.dense), "W4A4")


@BOTH
@pytest.mark.parametrize("m,n", [(33, 8), (4125, 40), (3381, 104), (4125, 104), (3629, 264), (3598, 521), (3598, 1032), (3846, 1030),
                                 (281, 12200), (405, 12202)])
def test_tiles_gated(m, n, dtype):
    wg, wu, x = mx.Weight(n, K, seed=n), mx.Weight(n, K, seed=n + 1), mx.rows(m, K, mx.DT[dtype], seed=m)
    ref, err, _, _ = mx.gated(x.double(), wg.dense, wu.dense)
    h, gate_up = ops.gated_mxfp4_cuda(x, wg.packed, wu.packed, n, keep_gate_up=True)
    mx.within(h, ref, err, "h")
    assert torch.equal(h, ops.gated_mxfp4_cuda(x, wg.packed, wu.packed, n))
    for part, w in ((gate_up[:, :n], wg), (gate_up[:, n:], wu)):
        mx.within(part, *mx.product(x.double(), w.dense), "gate_up")


@pytest.mark.parametrize("m,n", [(33, 32), (343, 5504), (777, 5024), (901, 4064)])
def test_tiles_gated_codes(m, n):
    k = 416
    wg, wu, wd = mx.Weight(n, k, seed=1), mx.Weight(n, k, seed=2), mx.Weight(k, n, seed=3)
    x = mx.rows(m, k, torch.bfloat16, seed=m)
    y = ops.mlp_mxfp4_w4a4_cuda(x, wg.packed, wu.packed, wd.packed, n)
    part = torch.arange(0, m, 7, device="cuda")  # rows do not meet
    mx.within(y[part], *mlp_reference(x[part], wg, wu, wd), "mlp")


# One, two and four strips of weights in a workgroup; x staged, through the ring (16 rows of K 2080 and more than
# 16 rows), quantized in the kernel, and as codes in one, two and four row blocks.
@pytest.mark.parametrize("n", [200, 4200, 8300, 16500])
@pytest.mark.parametrize("m,k", [(1, 544), (5, 544), (16, 2080), (8, 4128), (20, 1184), (32, 544)])
def test_rows_strips(m, n, k):
    w, x = mx.Weight(n, k, seed=n), mx.rows(m, k, torch.bfloat16, seed=m)
    mx.within(ops.gemm_mxfp4_cuda(x, *w.packed, n), *mx.product(x.double(), w.dense), "W4A16")
    mx.within(ops.gemm_mxfp4_w4a4_cuda(x, *w.packed, n), *mx.product(mx.rounded(x), w.dense), "W4A4")


# x as codes in one row block (K too long to be quantized in the kernel), two and four strips, and in a whole second block.
@pytest.mark.parametrize("m,n,k", [(16, 4200, 8224), (16, 8300, 4128), (9, 4200, 12320), (32, 4200, 8224), (17, 8300, 160)])
def test_rows_codes_blocks(m, n, k):
    w, x = mx.Weight(n, k, seed=n), mx.rows(m, k, torch.bfloat16, seed=m)
    mx.within(ops.gemm_mxfp4_w4a4_cuda(x, *w.packed, n), *mx.product(mx.rounded(x), w.dense), "W4A4")


@pytest.mark.parametrize("m", [1, 20])
def test_rows_gated_strips(m):
    n, k = 4200, 544
    wg, wu, x = mx.Weight(n, k, seed=1), mx.Weight(n, k, seed=2), mx.rows(m, k, torch.bfloat16, seed=m)
    ref, err, _, _ = mx.gated(x.double(), wg.dense, wu.dense)
    mx.within(ops.gated_mxfp4_cuda(x, wg.packed, wu.packed, n), ref, err, "h")


# K in parts whose sums a second kernel adds (N a multiple of 4), whole, and in parts of which the last is shorter.
@BOTH
@pytest.mark.parametrize("m,n,k", [(33, 48, 8224), (64, 4200, 8224), (33, 50, 8224), (48, 2052, 17408), (70, 100, 4128)])
def test_k_split(m, n, k, dtype):
    w, x = mx.Weight(n, k, seed=n), mx.rows(m, k, mx.DT[dtype], seed=m)
    y = ops.gemm_mxfp4_w4a4_cuda(x, *w.packed, n)
    mx.within(y, *mx.product(mx.rounded(x), w.dense), "W4A4")
    assert torch.equal(y, ops.gemm_mxfp4_w4a4_cuda(x, *w.packed, n))
    # Where y is not aligned for it, K is not split: another order of the sums.
    room = torch.full((m * n + 8,), 7.0, dtype=x.dtype, device="cuda")
    mx.within(ops.gemm_mxfp4_w4a4_cuda(x, *w.packed, n, out=room[1 : 1 + m * n].view(m, n)), *mx.product(mx.rounded(x), w.dense), "W4A4")
    assert (room[0] == 7).all() and (room[1 + m * n :] == 7).all()


def test_k_split_in_a_graph():
    """Two captured graphs with scratch of their own, replayed in turn with eager work between them."""
    n, k = 96, 8224
    w = mx.Weight(n, k, seed=1)
    xs = [mx.rows(m, k, torch.bfloat16, seed=m) for m in (40, 64)]
    expected = [ops.gemm_mxfp4_w4a4_cuda(x, *w.packed, n) for x in xs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.gemm_mxfp4_w4a4_cuda(x, *w.packed, n))
        graphs.append(g)
    for _ in range(3):
        for o in outs:
            o.zero_()
        for g in graphs:
            g.replay()
        again = ops.gemm_mxfp4_w4a4_cuda(xs[0], *w.packed, n)
        torch.cuda.synchronize()
        for o, e in zip(outs, expected):
            assert torch.equal(o, e)
        assert torch.equal(again, expected[0])


@pytest.mark.parametrize("m", [8, 40])
@pytest.mark.parametrize("n,k", [(96, 8224), (8224, 96)])
def test_rows_mlp_long(m, n, k):
    wg, wu, wd = mx.Weight(n, k, seed=1), mx.Weight(n, k, seed=2), mx.Weight(k, n, seed=3)
    x = mx.rows(m, k, torch.bfloat16, seed=m)
    mx.within(ops.mlp_mxfp4_w4a4_cuda(x, wg.packed, wu.packed, wd.packed, n), *mlp_reference(x, wg, wu, wd), "mlp")


# Tiles of 64, 128 and 256 rows; unsplit, split evenly, and with a last part that is shorter.
@BOTH
@pytest.mark.parametrize("m,n,k", [(1, 33, 96), (333, 2113, 4128), (1, 1057, 96), (1001, 33, 4128), (4100, 2113, 544), (8200, 2113, 96),
                                   (2049, 33, 4128), (8200, 4300, 544), (8200, 4300, 96)])
def test_gradient_plans(m, n, k, dtype):
    w, dy = mx.Weight(n, k, seed=n), mx.rows(m, n, mx.DT[dtype], seed=m)
    dx = ops.gemm_mxfp4_grad_cuda(dy, *w.packed, k)
    mx.within(dx, *mx.product(dy.double(), w.dense.t()), "dx")
    assert torch.equal(dx, ops.gemm_mxfp4_grad_cuda(dy, *w.packed, k))


@pytest.mark.parametrize("m", [1, 20, 70, 300])
@pytest.mark.parametrize("offset", [1, 4])
def test_outputs_at_any_element(m, offset):
    """An output that is not 16-byte aligned, inside a larger buffer whose rest stays as it is."""
    n, k = 88, 160
    w, x = mx.Weight(n, k, seed=1), mx.rows(m, k, torch.bfloat16, seed=2)
    for f in (ops.gemm_mxfp4_cuda, ops.gemm_mxfp4_w4a4_cuda):
        room = torch.full((m * n + 16,), 7.0, dtype=torch.bfloat16, device="cuda")
        f(x, *w.packed, n, out=room[offset : offset + m * n].view(m, n))
        assert torch.equal(room[offset : offset + m * n].view(m, n), f(x, *w.packed, n))
        assert (room[:offset] == 7).all() and (room[offset + m * n :] == 7).all()


@pytest.mark.parametrize("m", [1, 100])
def test_gradient_of_unaligned_rows(m):
    """dy at an element that is not 16-byte aligned is copied first, also where N is whole steps."""
    n, k = 128, 160
    w, dy = mx.Weight(n, k, seed=1), mx.rows(m, n, torch.bfloat16, seed=2)
    room = torch.empty(m * n + 8, dtype=torch.bfloat16, device="cuda")
    for offset in (1, 4):
        at = room[offset : offset + m * n].view(m, n)
        at.copy_(dy)
        assert torch.equal(ops.gemm_mxfp4_grad_cuda(at, *w.packed, k), ops.gemm_mxfp4_grad_cuda(dy, *w.packed, k))


def test_plain_weights_need_not_be_contiguous():
    """Codes and scales that are both views with strides: the copies made of them are apart."""
    for n, k in ((64, 64), (96, 1056), (300, 4096)):
        w = mx.Weight(n, k, seed=n)
        codes, scale = w.plain
        views = codes.t().contiguous().t(), scale.t().contiguous().t()
        for a, b in zip(ops.repack_mxfp4_cuda(*views), w.packed):
            assert torch.equal(a, b)
        assert torch.equal(ops.dequantize_mxfp4_cuda(*views, torch.float32).double(), w.dense)


@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("lowest,power", [(0, 100), (249, -60)])
def test_smallest_and_largest_scales(lowest, power, m):
    """Weights that are subnormal in bf16, and ones at its upper end."""
    n, k = 48, 288
    w = mx.Weight(n, k, seed=1)
    byte = np.random.default_rng(2).integers(lowest, lowest + 4, w.byte.shape, dtype=np.uint8)
    dense = torch.from_numpy(mx.values(w.code, byte)).cuda()
    packed = ops.repack_mxfp4_cuda(w.plain[0], torch.from_numpy(byte).cuda())
    x, dy = (torch.ldexp(mx.rows(m, c, torch.bfloat16, seed=c).double(), torch.tensor(power)).to(torch.bfloat16) for c in (k, n))
    mx.within(ops.gemm_mxfp4_cuda(x, *packed, n), *mx.product(x.double(), dense), "W4A16")
    mx.within(ops.gemm_mxfp4_w4a4_cuda(x, *packed, n), *mx.product(mx.rounded(x), dense), "W4A4")
    mx.within(ops.gemm_mxfp4_grad_cuda(dy, *packed, k), *mx.product(dy.double(), dense.t()), "dx")


def test_two_streams_at_once():
    """Calls with scratch of their own on two streams, of one weight, without a wait between them."""
    n, k = 544, 1056
    wg, wu, wd = mx.Weight(n, k, seed=1), mx.Weight(n, k, seed=2), mx.Weight(k, n, seed=3)
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    xs = [mx.rows(m, k, torch.bfloat16, seed=m) for m in (300, 200)]
    dhs = [mx.rows(x.shape[0], n, torch.bfloat16, seed=9) for x in xs]

    def step(x, dh):
        _, gate_up = ops.gated_mxfp4_cuda(x, wg.packed, wu.packed, n, keep_gate_up=True)
        return (ops.mlp_mxfp4_w4a4_cuda(x, wg.packed, wu.packed, wd.packed, n), ops.gemm_mxfp4_w4a4_cuda(x, *wg.packed, n),
                ops.gated_mxfp4_grad_cuda(dh, gate_up, wg.packed, wu.packed, k))

    expected = [step(x, dh) for x, dh in zip(xs, dhs)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(xs[i], dhs[i]))
    torch.cuda.synchronize()
    for results, e in zip(got, expected):
        for r in results:
            assert all(torch.equal(a, b) for a, b in zip(r, e))


def test_refusals():
    n, k = 96, 160
    w, x = mx.Weight(n, k, seed=1), mx.rows(4, k, torch.bfloat16, seed=2)
    weight, scale = w.packed
    dh, gate_up = mx.rows(4, n, torch.bfloat16, seed=3), torch.zeros(4, 2 * n, device="cuda")
    for f, args, message in (
        (ops.quantize_mxfp4_cuda, (x.cpu(),), "must be a CUDA"),
        (ops.quantize_mxfp4_cuda, (x.double(),), "must be a CUDA"),
        (ops.quantize_mxfp4_cuda, (x.t(),), "must be contiguous"),
        (ops.quantize_mxfp4_cuda, (x[:, :40].contiguous(),), "K must be a multiple of 32"),
        (ops.quantize_mxfp4_cuda, (torch.empty(65, dtype=torch.bfloat16, device="cuda")[1:].view(2, 32),), "16-byte aligned"),
        (ops.dequantize_mxfp4_cuda, (w.plain[0], w.plain[1][:, 1:]), "scale must be"),
        (ops.dequantize_mxfp4_cuda, (w.plain[0], w.plain[1], torch.int32), "dtype must be"),
        (ops.repack_mxfp4_cuda, (w.plain[0], w.plain[1].cpu()), "must be on one CUDA device"),
        (ops.repack_mxfp4_cuda, (w.plain[0].int(), w.plain[1]), "codes must be uint8"),
        (ops.gemm_mxfp4_cuda, (x.float(), weight, scale, n), "must be a CUDA fp16 or bf16"),
        (ops.gemm_mxfp4_cuda, (x[0], weight, scale, n), "must be contiguous"),
        (ops.gemm_mxfp4_cuda, (x, weight.cpu(), scale, n), "must be on one device"),
        (ops.gemm_mxfp4_cuda, (x, weight.short(), scale, n), "must be contiguous int32"),
        (ops.gemm_mxfp4_cuda, (x, weight, scale, n + 16), "weight has the wrong size"),
        (ops.gemm_mxfp4_cuda, (x, weight, scale[:, :1].contiguous(), n), "scale has the wrong shape"),
        (ops.gemm_mxfp4_cuda, (x, weight, scale, -1), "must be non-negative"),
        (ops.gemm_mxfp4_cuda, (x, weight, scale, n, torch.empty(4, n + 1, dtype=x.dtype, device="cuda")), "out must be"),
        (ops.gemm_mxfp4_w4a4_cuda, (x, weight, scale, n, torch.empty(4, n, device="cuda")), "out must be"),
        (ops.gemm_mxfp4_grad_cuda, (dh, weight, scale, k + 1), "K must be a multiple of 32"),
        (ops.gemm_mxfp4_grad_cuda, (dh, weight, scale, k + 128), "weight has the wrong size"),
        (ops.gated_mxfp4_cuda, (x, w.packed, w.packed, 500), "weight has the wrong size"),
        (ops.gated_mxfp4_grad_cuda, (dh, gate_up.bfloat16(), w.packed, w.packed, k), "gate_up must be"),
        (ops.gated_mxfp4_grad_cuda, (dh, gate_up[:2], w.packed, w.packed, k), "gate_up must be"),
        (ops.mlp_mxfp4_w4a4_cuda, (x, w.packed, w.packed, w.packed, 40), "must be a multiple of 32"),
        (ops.mlp_mxfp4_w4a4_cuda, (x, w.packed, w.packed, w.packed, n), "weight has the wrong size"),
    ):
        with pytest.raises((ValueError, RuntimeError), match=message):
            f(*args)
