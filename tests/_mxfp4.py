"""MXFP4 restated in float64 with numpy and torch, for the tests: the format, the quantizer, the products, the
gated block and its gradient, and bounds on what correct kernels may differ by.

Bounds: a product of 16-bit values is exact in fp32, a sum of K of them in any order is off by at most
K 2^-23 of the sum of magnitudes (2^-24 a rounding, twice that for a truncating adder), and the result is
rounded once, by at most half a step of its type (`half`)."""

from __future__ import annotations

import numpy as np
import torch

from pulsarlm_amd import ops

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the smallest subnormal step: what rounding is off by near zero."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def scale_byte(amax):
    """float64 amax per block -> byte."""
    with np.errstate(divide="ignore"):
        e = np.frexp(amax)[1] - 1
    b = np.clip(e - 2 + 127, 0, 254)
    b = np.where(amax == 0, 0, b)
    return np.where(np.isfinite(amax), b, 255).astype(np.uint8)


def encode(v, byte):
    """float64 values [..., 32] under scale bytes [...] -> codes 0..15; the nearest value, ties to the even code."""
    a = np.abs(np.ldexp(v, 127 - byte.astype(np.int64)[..., None]))
    d = np.abs(np.minimum(a, 6.0)[..., None] - E2M1)
    near = d.min(axis=-1, keepdims=True)
    # Among equally near codes the even one.
    code = np.where(d == near, np.arange(8) + 100 * (np.arange(8) % 2), 1000).argmin(axis=-1)
    return (code | (np.signbit(v) << 3)).astype(np.uint8)


def quantize(x):
    """float64 [M, K] -> (codes 0..15 [M, K], bytes [M, K/32])."""
    b = x.reshape(x.shape[0], -1, 32)
    amax = np.where(np.isnan(b).any(axis=-1), np.nan, np.abs(b).max(axis=-1, initial=0))
    byte = scale_byte(amax)
    code = np.where((byte == 255)[..., None], 0, encode(np.where(np.isfinite(b), b, 0.0), byte))
    return code.reshape(x.shape).astype(np.uint8), byte


def values(code, byte):
    v = E2M1[code & 7] * np.where(code & 8, -1.0, 1.0)
    s = np.where(byte == 255, np.nan, np.exp2(byte.astype(np.float64) - 127))
    return (v.reshape(*byte.shape, 32) * s[..., None]).reshape(code.shape)


def pack(code):
    return np.ascontiguousarray(code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8)


class Weight:
    """A random MXFP4 weight [N, K]: dense float64 on the GPU, and its repacked form."""

    def __init__(self, n, k, seed, spread=3, device="cuda"):
        rng = np.random.default_rng(seed)
        self.code = rng.integers(0, 16, (n, k), dtype=np.uint8)
        self.byte = rng.integers(127 - 5 - spread, 127 - 5 + 1, (n, k // 32), dtype=np.uint8)
        self.dense = torch.from_numpy(values(self.code, self.byte)).to(device)
        self.plain = torch.from_numpy(pack(self.code)).to(device), torch.from_numpy(self.byte).to(device)
        self.packed = ops.repack_mxfp4_cuda(*self.plain) if device == "cuda" else None


def rows(m, k, dtype, seed, device="cuda"):
    """Activations with loud channels and a block of zeros, in dtype."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g, dtype=torch.float64) * torch.exp(0.7 * torch.randn(k, generator=g, dtype=torch.float64))
    if k >= 64:
        x[0, 32:64] = 0
    return x.to(dtype).to(device)


def rounded(x):
    """Q(x) in float64 on x's device."""
    return torch.from_numpy(values(*quantize(x.double().cpu().numpy()))).to(x.device)


def product(x, w):
    """(x @ w^T, its sums' error bound) in float64."""
    return x @ w.t(), (x.shape[1] + 8) * 2.0**-23 * (x.abs() @ w.abs().t())


def silu(g):
    return g / (1 + torch.exp(-g))


def gated(x, wg, wu):
    """(h, bound of its error before the last rounding, g, u): |silu'| <= 1.1; exp2 and the reciprocal are off by
    a few 2^-23, the exponent's rounding by |g| 2^-23 of exp(-g)."""
    g, eg = product(x, wg)
    u, eu = product(x, wu)
    h = silu(g) * u
    return h, 1.1 * eg * (u.abs() + eu) + silu(g).abs() * eu + (g.abs() + 8) * 2.0**-22 * h.abs(), g, u


def gated_factors(dh, g, u):
    """(d gate, d up) in float64."""
    s = torch.sigmoid(g)
    return dh * u * s * (1 + g * (1 - s)), dh * g * s


def within(y, ref, error, what=""):
    """y (16 or 32 bits) against float64 ref: `error` before, half a step for the last rounding."""
    h, t = half(y.dtype), tiny(y.dtype)
    bound = error + h * (ref.abs() + error) + t
    bad = ~((y.double() - ref).abs() <= bound)
    over = torch.finfo(y.dtype).max
    bad &= ~((ref.abs() + error >= over * (1 - h)) & (y.double().abs() >= over))  # beyond the type: infinity
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first {bad.nonzero()[0].tolist()}: " \
                          f"{y[tuple(bad.nonzero()[0])].item()} for {ref[tuple(bad.nonzero()[0])].item()} +- {bound[tuple(bad.nonzero()[0])].item()}"
