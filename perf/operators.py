"""Operators on microscaled 4-bit (MXFP4) weights: quantisation, the linear product with 16-bit and with
4-bit activations, its input gradient, and the gated feed-forward block forward, backward and as a whole.

``listed()`` gives fixed cases, ``draw(rng)`` more of the same ranges; ``prepare`` makes inputs from a seed,
``run`` is one pass (plain torch in 32 bits, or the framework's kernels where ``own`` is true), ``work`` its
unavoidable bytes and operations and ``exact`` the same outputs in float64.

The format: 32 consecutive K values share a scale 2^(b - 127), b one byte, and are e2m1 codes (+-0, 0.5,
1, 1.5, 2, 3, 4, 6), two to a byte, the lower K in the low half. Quantisation takes b = floor(log2(amax)) - 2
+ 127 and rounds to nearest, ties to the even code, saturating at 6.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _case(name, kind, m, n, k, dtype="bf16"):
    return {"name": name, "kind": kind, "m": m, "n": n, "k": k, "dtype": dtype}


# n: output features of the product; of the gated block, its intermediate size.
def listed():
    return [
        # One token's activations before a projection: the quantiser alone, where latency counts.
        _case("quantize_m1", "quantize", 1, 0, 4096),
        # A prefill chunk's activations before the down projection.
        _case("quantize_m4096", "quantize", 4096, 0, 12288),
        # One user's token through the qkv projection (Qwen3-8B sizes), 16-bit activations.
        _case("linear_m1", "linear", 1, 6144, 4096),
        # A short ragged prompt in fp16; N and K off the tile sizes.
        _case("linear_m333", "linear", 333, 5000, 4128, "fp16"),
        # Adapter training on a frozen linear: the product and the gradient of its input.
        _case("linear_train_m2000", "linear_train", 2000, 4096, 4096),
        # A small server's decode batch through a wide projection, 4-bit activations.
        _case("linear_w4a4_m12", "linear_w4a4", 12, 24576, 4096),
        # A full prefill chunk through the widest projection, 4-bit activations.
        _case("linear_w4a4_m4096", "linear_w4a4", 4096, 24576, 4096),
        # One user's token through gate, up and activation.
        _case("gated_m1", "gated", 1, 12288, 4096),
        # A training micro-batch through the gated block and back, off the tile sizes.
        _case("gated_train_m1001", "gated_train", 1001, 4864, 2080),
        # A large training micro-batch (Qwen3-8B sizes).
        _case("gated_train_m4096", "gated_train", 4096, 12288, 4096),
        # Decode of a busy server through the whole feed-forward block, 4-bit activations (Qwen3-27B-like layer).
        _case("mlp_w4a4_m48", "mlp_w4a4", 48, 17408, 5120),
        # Its prefill at Qwen3-8B sizes.
        _case("mlp_w4a4_m4096", "mlp_w4a4", 4096, 12288, 4096),
    ]


_KINDS = ("quantize", "linear", "linear_train", "linear_w4a4", "gated", "gated_train", "mlp_w4a4")


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(_KINDS)
    most = max(work(c)["flops"] for c in listed() if c["kind"].split("_")[0] == kind.split("_")[0])
    while True:
        m = _log_int(rng, 256, 4096) if kind.endswith("train") else _log_int(rng, 1, 4096)
        n, k = _log_int(rng, 512, 24576), 32 * _log_int(rng, 16, 384)
        dtype = rng.choice(["bf16", "bf16", "fp16"])
        if kind == "quantize":
            n, dtype = 0, rng.choice(["bf16", "fp16", "fp32"])
        elif kind.startswith(("gated", "mlp")):
            n = _log_int(rng, 512, 17408)
            if kind.startswith("mlp"):
                n = (n + 31) // 32 * 32  # the down projection's K
        c = {"kind": kind, "m": m, "n": n, "k": k, "dtype": dtype}
        if work(c)["flops"] <= most:
            return c


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _pack(code):
    return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous()


def _quantize(x):
    """fp32 [M, K] -> (codes 0..15 uint8 [M, K], scale bytes uint8 [M, K/32])."""
    m, k = x.shape
    b = x.view(m, k // 32, 32)
    e = torch.frexp(b.abs().amax(dim=2))[1] - 3  # amax = f 2^e', f in [0.5, 1): floor(log2) = e' - 1
    e = e.clamp(-127, 127)
    v = torch.ldexp(b, -e[:, :, None]).abs()
    q = torch.where(v < 2, torch.round(2 * v) / 2, torch.where(v < 4, torch.round(v), 2 * torch.round(v / 2)))
    q = q.clamp(max=6.0)
    code = torch.where(q < 2, 2 * q, torch.where(q < 4, q + 2, q / 2 + 4)).to(torch.uint8)
    code = code | (torch.signbit(b).to(torch.uint8) << 3)
    return code.view(m, k), (e + 127).to(torch.uint8)


def _values(code, scale):
    """(codes [M, K], scale bytes) -> the fp32 values they stand for."""
    lut = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), dtype=torch.float32, device=code.device)
    m, k = code.shape
    v = lut[code.to(torch.int32)].view(m, k // 32, 32)
    return torch.ldexp(v, (scale.to(torch.int32) - 127)[:, :, None]).view(m, k)


def _unpack(codes):
    return torch.stack((codes & 15, codes >> 4), dim=2).view(codes.shape[0], -1)


def _weight_shapes(case):
    n, k = case["n"], case["k"]
    kind = case["kind"]
    if kind == "quantize":
        return []
    if kind.startswith("linear"):
        return [(n, k)]
    return [(n, k), (n, k)] + ([(k, n)] if kind == "mlp_w4a4" else [])


def _inputs(case, seed):
    """(x, [(packed codes, scale bytes) per weight], gradient of the output or None)."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]
    m, k = case["m"], case["k"]
    # Activations with a few loud channels, as a transformer's are.
    x = torch.randn(m, k, generator=g, device="cuda") * torch.exp(0.7 * torch.randn(k, generator=g, device="cuda"))
    weights = []
    for rows, cols in _weight_shapes(case):
        w = torch.randn(rows, cols, generator=g, device="cuda") * (0.7 / math.sqrt(cols))
        code, scale = _quantize(w)
        weights.append((_pack(code), scale))
        del w, code
    grad = None
    if case["kind"].endswith("train"):
        grad = (torch.randn(m, case["n"], generator=g, device="cuda") * 0.02).to(dt)
    return x.to(dt), weights, grad


def prepare(case, seed):
    x, weights, grad = _inputs(case, seed)
    state = {"case": case, "x": x, "grad": grad, "weights": weights}
    if own:
        from pulsarlm_amd import ops

        state["ops"] = ops
        state["weights"] = [ops.repack_mxfp4_cuda(codes, scale) for codes, scale in weights]
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def _run_own(state):
    ops, case, x, w, grad = state["ops"], state["case"], state["x"], state["weights"], state["grad"]
    kind, n, k = case["kind"], case["n"], case["k"]
    if kind == "quantize":
        codes, scale = ops.quantize_mxfp4_cuda(x)
        return ops.dequantize_mxfp4_cuda(codes, scale, torch.float32)
    if kind == "linear":
        return ops.gemm_mxfp4_cuda(x, *w[0], n)
    if kind == "linear_train":
        return ops.gemm_mxfp4_cuda(x, *w[0], n), ops.gemm_mxfp4_grad_cuda(grad, *w[0], k)
    if kind == "linear_w4a4":
        return ops.gemm_mxfp4_w4a4_cuda(x, *w[0], n)
    if kind == "gated":
        return ops.gated_mxfp4_cuda(x, w[0], w[1], n)
    if kind == "gated_train":
        h, gate_up = ops.gated_mxfp4_cuda(x, w[0], w[1], n, keep_gate_up=True)
        return h, ops.gated_mxfp4_grad_cuda(grad, gate_up, w[0], w[1], k)
    return ops.mlp_mxfp4_w4a4_cuda(x, w[0], w[1], w[2], n)


def _run_plain(state):
    case, dt = state["case"], state["x"].dtype
    kind = case["kind"]
    x = state["x"].float()
    if kind == "quantize":
        return _values(*_quantize(x))
    if kind.endswith("w4a4"):
        x = _values(*_quantize(x))
    w = [_values(_unpack(codes), scale) for codes, scale in state["weights"]]
    if kind.startswith("linear"):
        y = (x @ w[0].t()).to(dt)
        return (y, (state["grad"].float() @ w[0]).to(dt)) if kind == "linear_train" else y
    g, u = x @ w[0].t(), x @ w[1].t()
    s = 1.0 / (1.0 + torch.exp(-g))
    h = g * s * u
    if kind == "gated":
        return h.to(dt)
    if kind == "gated_train":
        dh = state["grad"].float()
        dx = (dh * u * s * (1.0 + g * (1.0 - s))) @ w[0] + (dh * g * s) @ w[1]
        return h.to(dt), dx.to(dt)
    return (_values(*_quantize(h)) @ w[2].t()).to(dt)


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# ---------------------------------------------------------------------------
# Work
# ---------------------------------------------------------------------------


def work(case):
    kind, m, n, k, e = case["kind"], case["m"], case["n"], case["k"], _SIZE[case["dtype"]]
    if kind == "quantize":
        # x in, values out (4 bytes each); the largest magnitude and one product a value.
        return {"bytes": m * k * (e + 4.0), "flops": 2.0 * m * k}
    weight = n * k * (0.5 + 1.0 / 32)
    if kind == "linear_train":
        return {"bytes": weight + 2.0 * e * m * (k + n), "flops": 4.0 * m * n * k}
    if kind.startswith("linear"):
        return {"bytes": weight + float(e) * m * (k + n), "flops": 2.0 * m * n * k}
    if kind == "gated":
        return {"bytes": 2 * weight + float(e) * m * (k + n), "flops": 4.0 * m * n * k}
    if kind == "gated_train":
        return {"bytes": 2 * weight + 2.0 * e * m * (k + n), "flops": 8.0 * m * n * k}
    return {"bytes": 3 * weight + 2.0 * e * m * k, "flops": 6.0 * m * n * k}


# ---------------------------------------------------------------------------
# The definition in float64
# ---------------------------------------------------------------------------


def _round64(x):
    """Each value of float64 [M, K] as quantisation keeps it: the midpoints between codes that it passes are counted."""
    blocks = x.reshape(x.shape[0], -1, 32)
    top = blocks.abs().amax(dim=-1, keepdim=True)
    unit = torch.exp2((torch.floor(torch.log2(top)) - 2.0).clamp(-127.0, 127.0))
    a = blocks.abs() / unit
    code = torch.zeros_like(a, dtype=torch.int64)
    # A tie goes to the even one of codes i and i + 1.
    for i, mid in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
        code += (a > mid) if i % 2 == 0 else (a >= mid)
    value = torch.tensor(_E2M1, dtype=torch.float64, device=x.device).take(code)
    return (torch.sign(blocks) * value * unit).reshape(x.shape)


def _dense64(codes, scale):
    """float64 [N, K] of a packed weight."""
    table = torch.tensor(_E2M1, dtype=torch.float64, device=codes.device)
    out = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
    for half in (0, 1):
        c = ((codes >> (4 * half)) & 15).long()
        out[:, half::2] = table[c & 7] * (1.0 - 2.0 * (c >> 3).double())
    return out * torch.exp2(scale.double() - 127.0).repeat_interleave(32, dim=1)


def exact(case, seed):
    x, weights, grad = _inputs(case, seed)
    x = x.double()
    kind = case["kind"]
    if kind == "quantize" or kind.endswith("w4a4"):
        x = _round64(x)
    if kind == "quantize":
        return x
    w = [_dense64(codes, scale) for codes, scale in weights]
    if kind == "linear_train":
        return torch.matmul(x, w[0].t()), torch.matmul(grad.double(), w[0])
    if kind.startswith("linear"):
        return torch.matmul(x, w[0].t())
    g, u = torch.matmul(x, w[0].t()), torch.matmul(x, w[1].t())
    silu = g * torch.sigmoid(g)
    h = silu * u
    if kind == "gated":
        return h
    if kind == "gated_train":
        dh = grad.double()
        slope = torch.sigmoid(g) * (1.0 + g - silu)  # d silu / d g
        return h, torch.matmul(dh * u * slope, w[0]) + torch.matmul(dh * silu, w[1])
    return torch.matmul(_round64(h), w[2].t())
