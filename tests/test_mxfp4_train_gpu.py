"""The MXFP4 operators in training, where the 16-bit type's range or a term of the gradient could get lost."""

import pytest
import torch

from pulsarlm_amd import ops
from tests import _mxfp4 as mx

pytestmark = pytest.mark.gpu


def shifted(n, k, seed, power):
    """A random weight times 2^power: (dense float64, packed)."""
    w = mx.Weight(n, k, seed=seed)
    return torch.ldexp(w.dense, torch.tensor(power)), ops.repack_mxfp4_cuda(w.plain[0], w.plain[1] + power)


def fp16_gradient(dh, gate_up, wg, wu):
    """(dx, bound) in float64. A factor is rounded to 11 bits of its own or, below 2^-14 of its row's largest in [2^14, 2^15),
    to fp16's subnormal steps: half a step is 2^-25 there, 2^-39 of the row's largest. Its own arithmetic is off by a
    few 2^-23 of the terms' magnitude (|1 + g (1 - s)| <= 1 + |g|)."""
    n = dh.shape[1]
    d, g, u = dh.double(), gate_up[:, :n].double(), gate_up[:, n:].double()
    dg, du = mx.gated_factors(d, g, u)
    top = torch.maximum(dg.abs().amax(dim=1), du.abs().amax(dim=1))[:, None]
    own = [mx.half(torch.float16) * f.abs() + 2.0**-39 * top + 2.0**-19 * d.abs() * v * (1 + g.abs()) for f, v in ((dg, u.abs()), (du, 1.0))]
    err = sum(e @ w.abs() + (2 * n + 8) * 2.0**-23 * ((f.abs() + e) @ w.abs()) for e, f, w in zip(own, (dg, du), (wg, wu)))
    return dg @ wg + du @ wu, err, top


# Rows of one and several tiles, unsplit and split sums, N of whole 16-byte pieces and not, past what a workgroup
# holds, and more rows than workgroups.
FACTORS = [(1, 96, 160), (3, 4096, 160), (70, 33, 96), (300, 520, 1056), (2100, 264, 288), (2, 12331, 96), (5, 16504, 96), (20000, 88, 32)]


@pytest.mark.parametrize("m,n,k", FACTORS)
def test_fp16_factors_beyond_the_type(m, n, k):
    """dh u s (1 + g (1 - s)) passes 65504 where dx, through small weights, is an ordinary number."""
    (dg, pg), (du, pu) = shifted(n, k, 1, -9), shifted(n, k, 2, -9)
    r = torch.Generator("cuda").manual_seed(m)
    dh = (64 * torch.randn(m, n, generator=r, device="cuda")).half()
    gate_up = torch.randn(m, 2 * n, generator=r, device="cuda") * torch.tensor([3.0, 3000.0], device="cuda").repeat_interleave(n)
    ref, err, top = fp16_gradient(dh, gate_up, dg, du)
    assert (top > 65504).all() and (ref.abs() + err < 65504).all()
    mx.within(ops.gated_mxfp4_grad_cuda(dh, gate_up, pg, pu, k), ref, err, "dx")


@pytest.mark.parametrize("m,n,k", FACTORS)
def test_fp16_factors_below_the_type(m, n, k):
    """Factors among fp16's subnormals, whose dx through large weights is not."""
    (dg, pg), (du, pu) = shifted(n, k, 1, 10), shifted(n, k, 2, 10)
    r = torch.Generator("cuda").manual_seed(m)
    dh = (2.0**-12 * torch.randn(m, n, generator=r, device="cuda")).half()
    gate_up = 2.0**-8 * torch.randn(m, 2 * n, generator=r, device="cuda")
    ref, err, top = fp16_gradient(dh, gate_up, dg, du)
    assert (top < 2.0**-14).all()
    mx.within(ops.gated_mxfp4_grad_cuda(dh, gate_up, pg, pu, k), ref, err, "dx")


def test_fp16_factors_of_every_row_apart():
    """Rows of very different size, of zeros, and with infinity and NaN, in one call: each as if it were alone."""
    m, n, k = 40, 96, 160
    (dg, pg), (du, pu) = shifted(n, k, 1, -9), shifted(n, k, 2, -9)
    r = torch.Generator("cuda").manual_seed(3)
    power = torch.arange(m, device="cuda") % 20 - 10.0
    dh = (torch.randn(m, n, generator=r, device="cuda") * torch.exp2(power)[:, None]).half()
    dh[7] = 0
    gate_up = torch.randn(m, 2 * n, generator=r, device="cuda") * torch.exp2(power)[:, None]
    dh[11, 5], gate_up[13, n + 3], gate_up[17, 2] = float("nan"), float("inf"), float("nan")
    odd = torch.tensor([11, 13, 17], device="cuda")
    dx = ops.gated_mxfp4_grad_cuda(dh, gate_up, pg, pu, k)
    assert not dx[7].any() and not dx[odd].isfinite().any()
    rest = torch.tensor([i for i in range(m) if i not in (11, 13, 17)], device="cuda")
    ref, err, _ = fp16_gradient(dh[rest], gate_up[rest], dg, du)
    mx.within(dx[rest], ref, err, "dx")
    for i in range(m):
        alone = ops.gated_mxfp4_grad_cuda(dh[i : i + 1], gate_up[i : i + 1], pg, pu, k)
        assert torch.equal(alone.view(torch.int16), dx[i : i + 1].view(torch.int16)) or i in (11, 13, 17)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("m,n,k", [(20, 96, 160), (70, 520, 288)])
def test_gated_gradient_is_the_slope(m, n, k, dtype):
    """<dx, v> against the central difference of sum(dh h(x + t v)), h in float64 and differentiated by nothing but
    that, along a v in which every term of the gradient counts: a dx without one is told apart."""
    dt = mx.DT[dtype]
    wg, wu = mx.Weight(n, k, seed=1), mx.Weight(n, k, seed=2)
    x, dh = mx.rows(m, k, dt, seed=3) * 0.25, mx.rows(m, n, dt, seed=5)
    _, gate_up = ops.gated_mxfp4_cuda(x, wg.packed, wu.packed, n, keep_gate_up=True)
    dx = ops.gated_mxfp4_grad_cuda(dh, gate_up, wg.packed, wu.packed, k)
    check = Slope(x, dh, wg.dense, wu.dense, dt)
    assert check.accepts(dx.double())
    for without in check.incomplete():
        assert not check.accepts(without)


class Slope:
    def __init__(self, x, dh, wg, wu, dt):
        x, d = x.double(), dh.double()
        g, u = x @ wg.t(), x @ wu.t()
        s = torch.sigmoid(g)
        dg, du = mx.gated_factors(d, g, u)
        self.ref = dg @ wg + du @ wu
        # dx without its up term, its gate term, the factor 1 + g (1 - s), and the part g (1 - s) of it.
        self.others = [dg @ wg, du @ wu, (d * u) @ wg + du @ wu, (d * u * s) @ wg + du @ wu]
        self.v = self.ref / self.ref.abs().max()

        def loss(t):
            gt, ut = (x + t * self.v) @ wg.t(), (x + t * self.v) @ wu.t()
            return (d * gt / (1 + torch.exp(-gt)) * ut).sum().item()

        # t^2 / 6 of the third derivative and 2^-53 of the losses' terms over t: 1e-5 of the slope leaves room for both.
        t = 1e-4
        self.slope = (loss(t) - loss(-t)) / (2 * t)
        # A factor is rounded by at most half a step of its size and meets v through its weight row, dx likewise. g, u and dx
        # are sums in 32 bits, off by less than 600 2^-23 of magnitudes some 10 times their own: 2^-10 of the terms.
        rounding = (dg * (self.v @ wg.t())).abs().sum() + (du * (self.v @ wu.t())).abs().sum() + (self.ref * self.v).abs().sum()
        terms = ((dg.abs() @ wg.abs() + du.abs() @ wu.abs()) * self.v.abs()).sum()
        self.bound = (mx.half(dt) * rounding + 2.0**-10 * terms).item() + 1e-5 * abs(self.slope)

    def accepts(self, dx):
        return abs((dx * self.v).sum().item() - self.slope) <= self.bound

    def incomplete(self):
        return [torch.zeros_like(self.ref), *self.others]


@pytest.mark.parametrize("m,n,k", [(1, 64, 96), (333, 4096, 4128), (300, 256, 1056), (70, 33, 96)])
def test_linear_gradient_in_the_workspace_it_asks_for(m, n, k):
    """Exactly the bytes of either query, with a guard behind them; the same dx from an aligned dy and one that is copied."""
    from pulsarlm_amd import _lib

    lib, w, dy = _lib.load(), mx.Weight(n, k, seed=1), mx.rows(m, n, torch.bfloat16, seed=2)
    room = torch.empty(m * n + 8, dtype=torch.bfloat16, device="cuda")
    apart = room[1 : 1 + m * n].view(m, n).copy_(dy)
    results = []
    for rows, need in ((dy, lib.plm_gemm_mxfp4_grad_aligned_workspace_bytes(m, n, k)), (dy, lib.plm_gemm_mxfp4_grad_workspace_bytes(m, n, k)),
                       (apart, lib.plm_gemm_mxfp4_grad_workspace_bytes(m, n, k))):
        ws = torch.full((need + 256,), 77, dtype=torch.uint8, device="cuda")
        dx = torch.full((m, k), float("nan"), dtype=torch.bfloat16, device="cuda")
        _lib.check(lib.plm_gemm_mxfp4_grad(rows.data_ptr(), _lib.PLM_BF16, w.packed[0].data_ptr(), w.packed[1].data_ptr(), m, n, k,
                                           dx.data_ptr(), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
        assert (ws[need:] == 77).all()
        results.append(dx)
    mx.within(results[0], *mx.product(dy.double(), w.dense.t()), "dx")
    assert torch.equal(results[0], results[1]) and torch.equal(results[0], results[2])
    assert torch.equal(results[0], ops.gemm_mxfp4_grad_cuda(dy, *w.packed, k)) and torch.equal(results[0], ops.gemm_mxfp4_grad_cuda(apart, *w.packed, k))


def test_linear_gradient_takes_no_scratch_for_rows_in_place():
    """What a call takes from the allocator, over its output."""
    m, n, k = 8192, 4096, 4096
    w, dy = mx.Weight(n, k, seed=1), torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    dx = torch.empty(m, k, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops.gemm_mxfp4_grad_cuda(dy, *w.packed, k, out=dx)
    assert torch.cuda.max_memory_allocated() - before < 2 * m * n
