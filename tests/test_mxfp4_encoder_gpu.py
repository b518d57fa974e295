"""The MXFP4 encoder, bit for bit: each value under scales above its own, and the neighbours of every border."""

import numpy as np
import pytest
import torch

from pulsarlm_amd import ops
from tests import _mxfp4 as mx

pytestmark = pytest.mark.gpu


def same(block, dtype):
    x = torch.from_numpy(block).to(dtype).cuda()
    assert torch.equal(x.double().cpu(), torch.from_numpy(block))
    codes, scale = ops.quantize_mxfp4_cuda(x)
    code, byte = mx.quantize(block)
    assert np.array_equal(scale.cpu().numpy(), byte)
    assert np.array_equal(codes.cpu().numpy(), mx.pack(code))
    return byte


@pytest.mark.parametrize("above", range(12))
def test_every_bf16_value_under_a_louder_one(above):
    """All finite bf16 values, 31 near ones to a block, whose first value is 2^above times as loud: under twelve scales
    each goes through every code from the largest down to zero."""
    v = (np.arange(65536, dtype=np.uint32) << 16).view(np.float32)
    v = v[np.isfinite(v)].astype(np.float64)
    v = v[np.argsort(np.abs(v), kind="stable")]
    v = np.concatenate([v, v[: -v.size % 31]]).reshape(-1, 31)
    top = np.abs(v).max(axis=1)
    e = np.frexp(top)[1] - 1 + above
    loud = np.ldexp(1.0, np.clip(e, -133, 127)) * np.where(np.arange(v.shape[0]) % 2, -1.0, 1.0)
    block = np.concatenate([loud[:, None], v], axis=1)
    byte = same(block, torch.bfloat16)[:, 0]
    inside = (e <= 127) & (e - 2 + 127 >= 0) & (top > 0)
    assert inside.sum() > 1800 and np.array_equal(byte[inside], (e - 2 + 127)[inside])


@pytest.mark.parametrize("byte", [0, 1, 2, 3, 20, 60, 110, 126, 127, 128, 150, 200, 250, 252])
def test_fp32_neighbours_of_the_borders(byte):
    """Each border between two codes, and the fp32 numbers next to it, under one scale."""
    unit = np.float32(2.0) ** np.float32(byte - 127)
    at = [np.float32(b) * unit for b in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0)]
    near = [s * f(b) for b in at for s in (np.float32(1), np.float32(-1))
            for f in (lambda b: b, lambda b: np.nextafter(b, np.float32(0)), lambda b: np.nextafter(b, np.float32(np.inf)))]
    near += [np.float32(0), -np.float32(0)] * 4  # 62 in all
    loud = np.float32(7.5) * unit
    block = np.array([[loud, *near[:31]], [loud, *near[31:]]], dtype=np.float32).astype(np.float64)
    assert (same(block, torch.float32) == byte).all()
