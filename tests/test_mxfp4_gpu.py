"""The MXFP4 operators against float64 on the GPU: the quantizer bit for bit, the products, the gated block, its
gradient (against the formula and against differences) and the whole block, over sizes where tiles end early."""

import numpy as np
import pytest
import torch

from pulsarlm_amd import _lib, ops
from tests import _mxfp4 as mx

pytestmark = pytest.mark.gpu

BOTH = pytest.mark.parametrize("dtype", ["bf16", "fp16"])


def every_bf16_block():
    """All finite bf16 values in blocks of 32 under block maxima of many sizes."""
    bits = np.arange(65536, dtype=np.uint32)
    v = (bits << 16).view(np.float32)
    v = v[np.isfinite(v)].astype(np.float64)
    v = v[np.argsort(np.abs(v), kind="stable")]
    return v[: v.size // 32 * 32].reshape(-1, 32)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("m,k", [(1, 32), (1, 4096), (3, 96), (17, 544), (300, 1056)])
def test_quantize_is_exact(m, k, dtype):
    x = mx.rows(m, k, mx.DT[dtype], seed=m + k)
    codes, scale = ops.quantize_mxfp4_cuda(x)
    code, byte = mx.quantize(x.double().cpu().numpy())
    assert np.array_equal(scale.cpu().numpy(), byte)
    assert np.array_equal(codes.cpu().numpy(), mx.pack(code))
    for out in mx.DT.values():
        back = ops.dequantize_mxfp4_cuda(codes, scale, out)
        assert back.dtype == out
        assert torch.equal(back.double().cpu(), torch.from_numpy(mx.values(code, byte)).to(out).double())


def test_quantize_every_bf16_value():
    rng = np.random.default_rng(0)
    v = every_bf16_block()
    wide = v[rng.permutation(v.shape[0])].copy()
    wide[:, 0] *= 1.0  # blocks of near magnitudes
    mixed = v.reshape(-1)[rng.permutation(v.size)].reshape(-1, 32)  # blocks of far ones
    for block in (wide, mixed):
        x = torch.from_numpy(block).to(torch.bfloat16).cuda()
        codes, scale = ops.quantize_mxfp4_cuda(x)
        code, byte = mx.quantize(block)
        assert np.array_equal(scale.cpu().numpy(), byte)
        # Zero has a sign in either; the sign of a value that rounds to zero is kept.
        assert np.array_equal(codes.cpu().numpy(), mx.pack(code))


def test_ties_go_to_the_even_code():
    v = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 7.0] * 2)
    codes, scale = ops.quantize_mxfp4_cuda(torch.from_numpy(v[None]).float().cuda())
    assert scale.item() == 127
    got = ops.dequantize_mxfp4_cuda(codes, scale, torch.float32).cpu().numpy()[0]
    assert got.tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, -0.0, -1.0, -1.0, -2.0, -2.0, -4.0, -4.0, 6.0] * 2


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_infinity_and_nan_make_their_block_nan(bad, dtype):
    x = mx.rows(3, 128, mx.DT[dtype], seed=1)
    x[1, 70] = bad
    codes, scale = ops.quantize_mxfp4_cuda(x)
    assert (scale.cpu().numpy() == 255).tolist() == [[False] * 4, [False, False, True, False], [False] * 4]
    back = ops.dequantize_mxfp4_cuda(codes, scale, torch.float32)
    assert back.isnan().sum() == 32 and back[1, 64:96].isnan().all()


def test_quantize_empty():
    for shape in ((0, 64), (4, 0)):
        codes, scale = ops.quantize_mxfp4_cuda(torch.empty(shape, device="cuda"))
        assert codes.shape == (shape[0], shape[1] // 2) and scale.shape == (shape[0], shape[1] // 32)
        assert ops.dequantize_mxfp4_cuda(codes, scale).shape == shape


# Rows on either side of every kernel's limits, N and K off the tiles.
SIZES = [(1, 16, 32), (1, 200, 4128), (2, 33, 96), (5, 257, 1056), (7, 1, 160), (16, 48, 4096), (16, 100, 12288), (17, 200, 544),
         (31, 16, 128), (33, 65, 1056), (64, 130, 160), (65, 200, 544), (129, 257, 96), (200, 333, 1056), (300, 31, 2080)]
# Enough work tiles for the 256 x 256 shape, off its edges.
WIDE = [(3850, 4200, 544), (4096, 4096, 160)]


@BOTH
@pytest.mark.parametrize("m,n,k", SIZES + WIDE)
def test_gemm(m, n, k, dtype):
    dt = mx.DT[dtype]
    w, x = mx.Weight(n, k, seed=n), mx.rows(m, k, dt, seed=m)
    ref, err = mx.product(x.double(), w.dense)
    mx.within(ops.gemm_mxfp4_cuda(x, *w.packed, n), ref, err, "W4A16")
    ref, err = mx.product(mx.rounded(x), w.dense)
    mx.within(ops.gemm_mxfp4_w4a4_cuda(x, *w.packed, n), ref, err, "W4A4")


@BOTH
@pytest.mark.parametrize("m,n,k", SIZES + WIDE[:1])
def test_gated(m, n, k, dtype):
    dt = mx.DT[dtype]
    wg, wu, x = mx.Weight(n, k, seed=n), mx.Weight(n, k, seed=n + 1), mx.rows(m, k, dt, seed=m)
    ref, err, g, u = mx.gated(x.double(), wg.dense, wu.dense)
    h = ops.gated_mxfp4_cuda(x, wg.packed, wu.packed, n)
    mx.within(h, ref, err, "h")
    h2, gate_up = ops.gated_mxfp4_cuda(x, wg.packed, wu.packed, n, keep_gate_up=True)
    assert torch.equal(h, h2)
    for part, w in ((gate_up[:, :n], wg), (gate_up[:, n:], wu)):
        mx.within(part, *mx.product(x.double(), w.dense), "gate_up")


@BOTH
@pytest.mark.parametrize("m,n,k", SIZES + WIDE[:1])
def test_gradients(m, n, k, dtype):
    dt = mx.DT[dtype]
    wg, wu = mx.Weight(n, k, seed=n), mx.Weight(n, k, seed=n + 1)
    dy = mx.rows(m, n, dt, seed=m)
    ref, err = mx.product(dy.double(), wg.dense.t())
    mx.within(ops.gemm_mxfp4_grad_cuda(dy, *wg.packed, k), ref, err, "dx")
    g = torch.Generator("cuda").manual_seed(m)
    gate_up = 3 * torch.randn(m, 2 * n, generator=g, device="cuda")
    dg, du = mx.gated_factors(dy.double(), gate_up[:, :n].double(), gate_up[:, n:].double())
    ref = dg @ wg.dense + du @ wu.dense
    # The factors are rounded to 16 bits: by half a step, and their own arithmetic by a few 2^-23 of the terms'
    # magnitude (|1 + g (1 - s)| <= 1 + |g|).
    own = [mx.half(dt) * f.abs() + mx.tiny(dt) + 2.0**-19 * (dy.double().abs() * v.abs() * (1 + gate_up[:, :n].double().abs()))
           for f, v in ((dg, gate_up[:, n:].double()), (du, torch.ones_like(du)))]
    err = sum(e @ w.dense.abs() + (2 * n + 8) * 2.0**-23 * ((f.abs() + e) @ w.dense.abs()) for e, f, w in zip(own, (dg, du), (wg, wu)))
    mx.within(ops.gated_mxfp4_grad_cuda(dy, gate_up, wg.packed, wu.packed, k), ref, err, "gated dx")


def test_gradient_against_differences():
    """<dx, v> against the central difference of sum(dh h(x + t v)) in float64, through the kernels' own forward."""
    m, n, k = 20, 96, 160
    wg, wu = mx.Weight(n, k, seed=1), mx.Weight(n, k, seed=2)
    x, v = mx.rows(m, k, torch.bfloat16, seed=3) * 0.25, mx.rows(m, k, torch.bfloat16, seed=4).double()
    dh = mx.rows(m, n, torch.bfloat16, seed=5)
    h, gate_up = ops.gated_mxfp4_cuda(x, wg.packed, wu.packed, n, keep_gate_up=True)
    dx = ops.gated_mxfp4_grad_cuda(dh, gate_up, wg.packed, wu.packed, k)

    def loss(t):
        return (dh.double() * mx.gated(x.double() + t * v, wg.dense, wu.dense)[0]).sum().item()

    t = 1e-5
    slope = (loss(t) - loss(-t)) / (2 * t)
    # The factors and dx are rounded to bf16; g and u are off by what `gated` bounds (1e-4 covers it here).
    _, _, g, u = mx.gated(x.double(), wg.dense, wu.dense)
    r = mx.half(torch.bfloat16)
    dg, du = mx.gated_factors(dh.double(), g, u)
    eg, eu = r * dg.abs() + 1e-4 * dh.double().abs() * (1 + u.abs()), r * du.abs() + 1e-4 * dh.double().abs()
    ref = dg @ wg.dense + du @ wu.dense
    bound = ((eg @ wg.dense.abs() + eu @ wu.dense.abs() + r * ref.abs()) * v.abs()).sum().item()
    assert abs((dx.double() * v).sum().item() - slope) <= bound + 1e-4 * abs(slope)
    assert bound < 2 * (ref * v).abs().sum().item()  # and that says something


def mlp_reference(x, wg, wu, wd):
    """(y, bound): h within its error of a border between codes may go to either."""
    h, e, _, _ = mx.gated(mx.rounded(x), wg.dense, wu.dense)
    hn, en = h.cpu().numpy(), e.cpu().numpy()
    lo, hi = np.abs(hn) - en, np.abs(hn) + en
    shape = hn.shape[0], -1, 32
    base = mx.values(*mx.quantize(hn))
    spread = np.zeros_like(hn)
    for top in (np.maximum(lo, 0).reshape(shape).max(axis=-1), hi.reshape(shape).max(axis=-1)):
        byte = mx.scale_byte(top)
        for side in (hn - en, hn, hn + en):
            q = mx.values(mx.encode(side.reshape(shape), byte).reshape(hn.shape), byte)
            spread = np.maximum(spread, np.abs(q - base))
    q, s = torch.from_numpy(base).to(x.device), torch.from_numpy(spread).to(x.device)
    y, err = mx.product(q, wd.dense)
    return y, err + s @ wd.dense.abs().t()


MLP = [(1, 32, 32), (1, 96, 544), (3, 544, 96), (16, 1056, 160), (17, 160, 1056), (48, 544, 544), (65, 96, 288), (200, 1056, 544),
       (300, 544, 1056)]


@BOTH
@pytest.mark.parametrize("m,n,k", MLP)
def test_mlp_w4a4(m, n, k, dtype):
    dt = mx.DT[dtype]
    wg, wu, wd = mx.Weight(n, k, seed=1), mx.Weight(n, k, seed=2), mx.Weight(k, n, seed=3)
    x = mx.rows(m, k, dt, seed=m)
    mx.within(ops.mlp_mxfp4_w4a4_cuda(x, wg.packed, wu.packed, wd.packed, n), *mlp_reference(x, wg, wu, wd), "mlp")


def test_mlp_w4a4_wide():
    m, n, k = 3850, 2112, 2080
    wg, wu, wd = mx.Weight(n, k, seed=1), mx.Weight(n, k, seed=2), mx.Weight(k, n, seed=3)
    x = mx.rows(m, k, torch.bfloat16, seed=m)
    y = ops.mlp_mxfp4_w4a4_cuda(x, wg.packed, wu.packed, wd.packed, n)
    part = torch.arange(0, m, 37, device="cuda")  # rows do not meet
    ref, err = mlp_reference(x[part], wg, wu, wd)
    mx.within(y[part], ref, err, "mlp")


@pytest.mark.parametrize("m", [1, 40, 300])
def test_nan_and_infinity_stay_in_their_rows(m):
    n, k = 96, 160  # K ends inside a tile: what is read past it must not meet the NaN
    w, x = mx.Weight(n, k, seed=1), mx.rows(m + 1, k, torch.bfloat16, seed=2)
    x[m, 3] = float("nan")
    x[m, 100] = float("inf")
    wu = mx.Weight(n, k, seed=5)
    wd = mx.Weight(k, n, seed=6)
    for f in (lambda x: ops.gemm_mxfp4_cuda(x, *w.packed, n), lambda x: ops.gemm_mxfp4_w4a4_cuda(x, *w.packed, n),
              lambda x: ops.gated_mxfp4_cuda(x, w.packed, wu.packed, n),
              lambda x: ops.mlp_mxfp4_w4a4_cuda(x, w.packed, wu.packed, wd.packed, n)):
        y = f(x)
        assert y[m].isnan().all()
        assert y[:m].isfinite().all()
    dy = mx.rows(m + 1, n, torch.bfloat16, seed=3)
    dy[m, 5] = float("nan")
    dx = ops.gemm_mxfp4_grad_cuda(dy, *w.packed, k)
    assert dx[m].isnan().all() and dx[:m].isfinite().all()


def test_nan_scale_makes_its_weight_row_nan():
    n, k = 40, 160
    w = mx.Weight(n, k, seed=1)
    codes, scale = w.plain
    scale = scale.clone()
    scale[17, 4] = 255
    packed = ops.repack_mxfp4_cuda(codes, scale)
    for m in (1, 40, 300):
        x = mx.rows(m, k, torch.bfloat16, seed=2)
        for y in (ops.gemm_mxfp4_cuda(x, *packed, n), ops.gemm_mxfp4_w4a4_cuda(x, *packed, n)):
            assert y[:, 17].isnan().all()
            assert y[:, torch.arange(n, device="cuda") != 17].isfinite().all()


def test_rows_past_the_last_are_left():
    """Nothing is written outside the output (it lies inside a larger buffer)."""
    n, k = 50, 160
    w, wu = mx.Weight(n, k, seed=1), mx.Weight(n, k, seed=2)
    for m in (1, 20, 70, 130):
        x = mx.rows(m, k, torch.bfloat16, seed=2)
        for f in (ops.gemm_mxfp4_cuda, ops.gemm_mxfp4_w4a4_cuda):
            room = torch.full((m + 2, n), 7.0, dtype=torch.bfloat16, device="cuda")
            f(x, *w.packed, n, out=room[1:-1])
            assert torch.equal(room[1:-1], f(x, *w.packed, n))
            assert (room[0] == 7).all() and (room[-1] == 7).all()


def test_empty_sizes():
    w = mx.Weight(48, 64, seed=1)
    x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    assert ops.gemm_mxfp4_cuda(x, *w.packed, 48).shape == (0, 48)
    assert ops.gemm_mxfp4_w4a4_cuda(x, *w.packed, 48).shape == (0, 48)
    assert ops.gemm_mxfp4_grad_cuda(x[:, :48].contiguous(), *w.packed, 64).shape == (0, 64)
    none = ops.repack_mxfp4_cuda(torch.empty(0, 32, dtype=torch.uint8, device="cuda"), torch.empty(0, 2, dtype=torch.uint8, device="cuda"))
    some = mx.rows(5, 64, torch.bfloat16, seed=1)
    assert ops.gemm_mxfp4_cuda(some, *none, 0).shape == (5, 0)
    dx = ops.gemm_mxfp4_grad_cuda(torch.empty(5, 0, dtype=torch.bfloat16, device="cuda"), *none, 64)
    assert dx.shape == (5, 64) and not dx.any()
    flat = ops.repack_mxfp4_cuda(torch.empty(48, 0, dtype=torch.uint8, device="cuda"), torch.empty(48, 0, dtype=torch.uint8, device="cuda"))
    no_k = torch.empty(5, 0, dtype=torch.bfloat16, device="cuda")
    for y in (ops.gemm_mxfp4_cuda(no_k, *flat, 48), ops.gemm_mxfp4_w4a4_cuda(no_k, *flat, 48), ops.gated_mxfp4_cuda(no_k, flat, flat, 48)):
        assert y.shape == (5, 48) and not y.any()
    wd = ops.repack_mxfp4_cuda(torch.empty(64, 0, dtype=torch.uint8, device="cuda"), torch.empty(64, 0, dtype=torch.uint8, device="cuda"))
    assert not ops.mlp_mxfp4_w4a4_cuda(some, none, none, wd, 0).any()


def test_results_repeat_bit_for_bit():
    n, k = 544, 1056
    wg, wu, wd = mx.Weight(n, k, seed=1), mx.Weight(n, k, seed=2), mx.Weight(k, n, seed=3)
    for m in (1, 40, 300):
        x, dh = mx.rows(m, k, torch.bfloat16, seed=2), mx.rows(m, n, torch.bfloat16, seed=3)
        h, gate_up = ops.gated_mxfp4_cuda(x, wg.packed, wu.packed, n, keep_gate_up=True)
        for f in (lambda: ops.gemm_mxfp4_cuda(x, *wg.packed, n), lambda: ops.gemm_mxfp4_w4a4_cuda(x, *wg.packed, n),
                  lambda: ops.mlp_mxfp4_w4a4_cuda(x, wg.packed, wu.packed, wd.packed, n),
                  lambda: ops.gated_mxfp4_grad_cuda(dh, gate_up, wg.packed, wu.packed, k)):
            first = f()
            for _ in range(3):
                assert torch.equal(first, f())


def test_graph_and_streams():
    """A captured training step and serving step, replayed between eager work of other sizes, on another stream."""
    n, k = 544, 1056
    wg, wu, wd = mx.Weight(n, k, seed=1), mx.Weight(n, k, seed=2), mx.Weight(k, n, seed=3)
    for m in (2, 40, 300):
        x, dh = mx.rows(m, k, torch.bfloat16, seed=2), mx.rows(m, n, torch.bfloat16, seed=3)

        def step():
            h, gate_up = ops.gated_mxfp4_cuda(x, wg.packed, wu.packed, n, keep_gate_up=True)
            dx = ops.gated_mxfp4_grad_cuda(dh, gate_up, wg.packed, wu.packed, k)
            y = ops.gemm_mxfp4_cuda(h, *wd.packed, k)
            return h, dx, y, ops.mlp_mxfp4_w4a4_cuda(x, wg.packed, wu.packed, wd.packed, n), ops.gemm_mxfp4_w4a4_cuda(x, *wg.packed, n)

        expected = step()
        torch.cuda.synchronize()
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step()
        big = mx.rows(333, k, torch.bfloat16, seed=9)
        for _ in range(3):
            for o in out:
                o.fill_(float("nan"))
            graph.replay()
            ops.mlp_mxfp4_w4a4_cuda(big, wg.packed, wu.packed, wd.packed, n)
            torch.cuda.synchronize()
            for o, e in zip(out, expected):
                assert torch.equal(o, e)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            again = step()
        stream.synchronize()
        for o, e in zip(again, expected):
            assert torch.equal(o, e)


def test_weights_quantized_here_run_the_block():
    """As a user has it: dense weights quantized and repacked, the forward in 16 bits, its gradient and the 4-bit form."""
    g = torch.Generator("cuda").manual_seed(0)
    m, n, k = 33, 256, 192
    dense = [torch.randn(*s, generator=g, device="cuda") / s[1] ** 0.5 for s in ((n, k), (n, k), (k, n))]
    plain = [ops.quantize_mxfp4_cuda(w) for w in dense]
    wg, wu, wd = (ops.repack_mxfp4_cuda(*p) for p in plain)
    vg, vu, vd = (ops.dequantize_mxfp4_cuda(*p, torch.float32).double() for p in plain)
    x = mx.rows(m, k, torch.bfloat16, seed=1)
    h, gate_up = ops.gated_mxfp4_cuda(x, wg, wu, n, keep_gate_up=True)
    ref, err, _, _ = mx.gated(x.double(), vg, vu)
    mx.within(h, ref, err, "h")
    mx.within(ops.gemm_mxfp4_cuda(h, *wd, k), *mx.product(h.double(), vd), "y")
    dy = mx.rows(m, k, torch.bfloat16, seed=2)
    dh = ops.gemm_mxfp4_grad_cuda(dy, *wd, n)
    mx.within(dh, *mx.product(dy.double(), vd.t()), "dh")
    assert ops.gated_mxfp4_grad_cuda(dh, gate_up, wg, wu, k).shape == (m, k)
    assert ops.mlp_mxfp4_w4a4_cuda(x, wg, wu, wd, n).shape == (m, k)


def test_workspace_is_required():
    lib = _lib.load()
    w, x = mx.Weight(48, 64, seed=1), mx.rows(20, 64, torch.bfloat16, seed=1)
    y = torch.empty(20, 48, dtype=torch.bfloat16, device="cuda")
    need = lib.plm_gemm_mxfp4_w4a4_workspace_bytes(20, 48, 64)
    assert need > 0
    for ws, size in ((None, 0), (x, need - 1)):
        rc = lib.plm_gemm_mxfp4_w4a4(x.data_ptr(), _lib.PLM_BF16, w.packed[0].data_ptr(), w.packed[1].data_ptr(), 20, 48, 64, y.data_ptr(),
                                     None if ws is None else ws.data_ptr(), size, None)
        assert rc == _lib.PLM_ERR_WORKSPACE and b"gemm_mxfp4_w4a4: workspace of" in lib.plm_last_error()
