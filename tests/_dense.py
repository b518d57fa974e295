"""The operators on unpacked weights restated in float64, for the tests: the 8-bit row quantizer, products with scales for
each token and channel, products by expert and their gradients, and bounds on what correct kernels may differ by.

Bounds: an 8-bit product's sum is exact; it is converted to fp32 and multiplied by two scales, 2^-24 each, and rounded once
(_mxfp4.within counts that). 16-bit products are bounded as _mxfp4.product."""

from __future__ import annotations

import numpy as np
import torch

from tests import _mxfp4 as mx

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def row_scale(x):
    """fp32 [M] of x [M, K] on the CPU, by IEEE division; NaN for rows that are not finite."""
    x = x.float().cpu().numpy()
    top = np.abs(x).max(axis=1, initial=0)
    with np.errstate(invalid="ignore"):
        s = (np.maximum(top, np.float32(1e-12)) / np.float32(127)).astype(np.float32)
    return torch.from_numpy(np.where(np.isfinite(x).all(axis=1), s, np.float32(np.nan)))


def quantize(x):
    """(codes int8 [M, K], scale fp32 [M]) on the CPU: nearest to the quotient, ties to even, decided in float64."""
    scale = row_scale(x)
    q = torch.round(x.double().cpu() / scale.double()[:, None])  # half to even
    return torch.nan_to_num(q, nan=0.0, posinf=0.0, neginf=0.0).to(torch.int8), scale


def codes(m, k, seed, low=-127):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(low, 128, (m, k), generator=g, dtype=torch.int8).cuda()


def scales(m, seed):
    g = torch.Generator().manual_seed(seed)
    return (0.02 * torch.rand(m, generator=g) + 1e-4).cuda()


def int8_product(q, xs, w, ws):
    """(y, its error before the last rounding) in float64."""
    y = (q.double() @ w.double().t()) * xs.double()[:, None] * ws.double()
    return y, 4 * 2.0**-24 * y.abs()


def ends_of(counts):
    return np.cumsum(counts).astype(np.int32)


def offsets(counts, device="cuda"):
    return torch.from_numpy(ends_of(counts)).to(device)


def by_expert(counts):
    """(expert, first row, past its last)."""
    ends = ends_of(counts).tolist()
    return [(e, hi - c, hi) for e, (c, hi) in enumerate(zip(counts, ends))]


def values(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(shape, generator=g)).to(dtype).cuda()


def sums(k):
    """What a sum of k products is off by, of the sum of their magnitudes."""
    return (k + 8) * 2.0**-23


def grouped(x, w, counts):
    """(y, error bound); rows past the last expert's are zero."""
    y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device=x.device)
    e = torch.zeros_like(y)
    for i, lo, hi in by_expert(counts):
        a, b = x[lo:hi].double(), w[i].double()
        y[lo:hi] = a @ b.t()
        e[lo:hi] = sums(x.shape[1]) * (a.abs() @ b.abs().t())
    return y, e


def grad_x(dy, w, counts):
    return grouped(dy, w.transpose(1, 2), counts)


def grad_w(dy, x, counts):
    w = torch.zeros(len(counts), dy.shape[1], x.shape[1], dtype=torch.float64, device=x.device)
    err = torch.zeros_like(w)
    for i, lo, hi in by_expert(counts):
        a, b = dy[lo:hi].double(), x[lo:hi].double()
        w[i] = a.t() @ b
        err[i] = sums(hi - lo) * (a.abs().t() @ b.abs())
    return w, err


within = mx.within
