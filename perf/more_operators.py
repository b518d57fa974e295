"""Operators on 8-bit integer weights and on experts: the row quantizer, the 8-bit product with a scale for each
token and channel, and products grouped by expert with ragged sizes, in 8 bits and in 16 bits with both gradients.

``listed()`` gives fixed cases, ``draw(rng)`` more of the same ranges; ``prepare`` makes inputs from a seed,
``run`` is one pass (plain torch in 32 bits, or the framework's kernels where ``own`` is true), ``work`` its
unavoidable bytes and operations and ``exact`` the same outputs in float64.

The format: a row's scale is s = max(amax, 1e-12) / 127 in fp32, its codes the integers nearest to x / s, ties to
even. A grouped call's rows are sorted by expert: expert e has rows offsets[e - 1] to offsets[e]; rows past the last
expert's belong to none and give zeros.
"""

from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def _case(name, kind, m, n, k, dtype="bf16", experts=0, spare=0):
    """m rows, of which the last `spare` belong to no expert; n output and k input features."""
    return {"name": name, "kind": kind, "m": m, "n": n, "k": k, "dtype": dtype, "experts": experts, "spare": spare}


def listed():
    return [
        # One token's activations before a projection: the quantizer alone, where latency counts.
        _case("quantize_m1", "quantize", 1, 0, 4096),
        # A prefill chunk's activations before the down projection.
        _case("quantize_m4096", "quantize", 4096, 0, 12288),
        # One user's token through the qkv projection (Qwen3-8B sizes), quantized on the way.
        _case("w8a8_m1", "w8a8", 1, 6144, 4096),
        # A short ragged prompt in fp16; N and K off the tile sizes.
        _case("w8a8_m333", "w8a8", 333, 5000, 4128, "fp16"),
        # A full prefill chunk through the widest projection.
        _case("w8a8_m4096", "w8a8", 4096, 24576, 4096),
        # A server's decode batch through the down projection, quantized by what came before it.
        _case("codes_m16", "codes", 16, 4096, 12288),
        # A prefill chunk through the output projection, quantized by what came before it.
        _case("codes_m2000", "codes", 2000, 4096, 4096),
        # Decode of 8 tokens, 8 experts each of 128 (Qwen3-30B-A3B sizes): gate and up of the 8-bit experts.
        _case("w8a8_grouped_t8", "w8a8_grouped", 64, 1536, 2048, experts=128),
        # Its prefill chunk of 4096 tokens.
        _case("w8a8_grouped_t4096", "w8a8_grouped", 32768, 1536, 2048, experts=128),
        # The decode step with 16-bit experts.
        _case("grouped_t8", "grouped", 64, 1536, 2048, experts=128),
        # Training a few wide experts on a small padded batch, off the tile sizes.
        _case("grouped_train_m1001", "grouped_train", 1001, 4864, 2080, "fp16", experts=8, spare=23),
        # A training micro-batch of 4096 tokens through the down projections of 128 experts.
        _case("grouped_train_t4096", "grouped_train", 32768, 2048, 768, experts=128),
    ]


_KINDS = ("quantize", "w8a8", "codes", "w8a8_grouped", "grouped", "grouped_train")


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(_KINDS)
    like = "w8a8" if kind == "codes" else "grouped_train" if kind == "grouped" else kind
    most = [work(c) for c in listed() if c["kind"] == like]
    most = {key: max(w[key] for w in most) for key in ("bytes", "flops")}
    while True:
        c = {"kind": kind, "m": _log_int(rng, 1, 4096), "n": _log_int(rng, 512, 24576), "k": 16 * _log_int(rng, 32, 1088),
             "dtype": rng.choice(["bf16", "bf16", "fp16"]), "experts": 0, "spare": 0}
        if kind == "quantize":
            c["n"], c["dtype"] = 0, rng.choice(["bf16", "fp16", "fp32"])
        elif "grouped" in kind:
            c["experts"] = _log_int(rng, 4, 128)
            c["m"] = _log_int(rng, 256 if kind == "grouped_train" else 4, 32768)
            c["spare"] = rng.choice([0, 0, c["m"] // 20])
            unit = 16 if kind == "w8a8_grouped" else 8
            c["n"], c["k"] = 8 * _log_int(rng, 64, 640), unit * _log_int(rng, 512 // unit, 5120 // unit)
        w = work(c)
        if w["flops"] <= most["flops"] and w["bytes"] <= most["bytes"]:
            return c


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _used(case):
    """How many of the experts get rows: a router's choice leaves some out."""
    rows, experts = case["m"] - case["spare"], case["experts"]
    return min(experts - experts // 20, -(-7 * rows // 10))


def _ends(case, seed):
    """The rows' inclusive ends by expert, unevenly shared."""
    rng = random.Random(int(seed) * 1000003 + case["experts"])
    rows, used = case["m"] - case["spare"], _used(case)
    chosen = rng.sample(range(case["experts"]), used)
    count = [0] * case["experts"]
    share = [math.exp(rng.gauss(0.0, 0.8)) for _ in chosen]
    for e, s in zip(chosen, share):
        count[e] = 1 + int((rows - used) * s / sum(share))
    for _ in range(rows - sum(count)):
        count[rng.choice(chosen)] += 1
    ends = []
    for c in count:
        ends.append(c + (ends[-1] if ends else 0))
    return ends


def _quantize(x):
    """[M, K] -> (codes fp32 [M, K], scale fp32 [M])."""
    top = x.float().abs().amax(dim=1).clamp(min=1e-12)
    scale = top / torch.full_like(top, 127.0)  # a quotient by a number is a product with its reciprocal, off by a rounding
    # The quotient in 64 bits: in 32 it rounds onto the border between two codes from both sides.
    return torch.round(x.double() / scale.double()[:, None]).float(), scale


def _weight(g, rows, cols):
    """An 8-bit weight and its channels' scales."""
    w = torch.randn(rows, cols, generator=g, device="cuda") * (0.7 / math.sqrt(cols))
    scale = w.abs().amax(dim=1) / 127.0
    return torch.round(w / scale[:, None]).to(torch.int8), scale


def _inputs(case, seed):
    """Everything that the pass starts from, by name."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    kind, m, n, k, experts, dt = case["kind"], case["m"], case["n"], case["k"], case["experts"], _DTYPES[case["dtype"]]
    # Activations with a few loud channels, as a transformer's are.
    loud = torch.exp(0.7 * torch.randn(k, generator=g, device="cuda"))
    x = (torch.randn(m, k, generator=g, device="cuda") * loud).to(dt)
    made = {"x": x}
    if kind == "codes":
        codes, scale = _quantize(x)
        made = {"codes": codes.to(torch.int8), "x_scale": scale}
    if kind in ("w8a8", "codes"):
        made["weight"], made["scale"] = _weight(g, n, k)
    if experts:
        made["ends"] = _ends(case, seed)
        made["offsets"] = torch.tensor(made["ends"], dtype=torch.int32, device="cuda")
    if kind == "w8a8_grouped":
        made["weight"] = torch.empty(experts, n, k, dtype=torch.int8, device="cuda")
        made["scale"] = torch.empty(experts, n, device="cuda")
        for e in range(experts):
            made["weight"][e], made["scale"][e] = _weight(g, n, k)
    elif kind.startswith("grouped"):
        made["weight"] = torch.empty(experts, n, k, dtype=dt, device="cuda")
        for e in range(experts):
            made["weight"][e] = torch.randn(n, k, generator=g, device="cuda") * (0.7 / math.sqrt(k))
    if kind == "grouped_train":
        made["grad"] = (torch.randn(m, n, generator=g, device="cuda") * 0.02).to(dt)
    return made


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if own:
        from pulsarlm_amd import ops

        state["ops"] = ops
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def _run_own(s):
    ops, kind = s["ops"], s["case"]["kind"]
    if kind == "quantize":
        codes, scale = ops.quantize_rows_int8_cuda(s["x"])
        return ops.dequantize_rows_int8_cuda(codes, scale, torch.float32), scale
    if kind == "w8a8":
        return ops.gemm_int8_w8a8_cuda(s["x"], s["weight"], s["scale"])
    if kind == "codes":
        return ops.gemm_int8_cuda(s["codes"], s["x_scale"], s["weight"], s["scale"], _DTYPES[s["case"]["dtype"]])
    if kind == "w8a8_grouped":
        return ops.grouped_gemm_int8_cuda(s["x"], s["weight"], s["scale"], s["offsets"])
    y = ops.grouped_gemm_cuda(s["x"], s["weight"], s["offsets"])
    if kind == "grouped":
        return y
    return (y, ops.grouped_gemm_grad_x_cuda(s["grad"], s["weight"], s["offsets"]),
            ops.grouped_gemm_grad_w_cuda(s["grad"], s["x"], s["offsets"]))


def _each(ends):
    """(expert, its first row, past its last one) of the experts that have rows."""
    return [(e, lo, hi) for e, (lo, hi) in enumerate(zip([0] + ends[:-1], ends)) if hi > lo]


def _run_plain(s):
    case = s["case"]
    kind, dt = case["kind"], _DTYPES[case["dtype"]]
    if kind == "quantize":
        codes, scale = _quantize(s["x"])
        return codes * scale[:, None], scale
    if kind in ("w8a8", "codes"):
        x, xs = (s["codes"].float(), s["x_scale"]) if kind == "codes" else _quantize(s["x"])
        return ((x @ s["weight"].float().t()) * s["scale"] * xs[:, None]).to(dt)
    y = torch.zeros(case["m"], case["n"], dtype=dt, device=s["x"].device)
    if kind == "w8a8_grouped":
        x, xs = _quantize(s["x"])
        for e, lo, hi in _each(s["ends"]):
            y[lo:hi] = (x[lo:hi] @ s["weight"][e].float().t()) * s["scale"][e] * xs[lo:hi, None]
        return y
    x, w = s["x"].float(), s["weight"]
    for e, lo, hi in _each(s["ends"]):
        y[lo:hi] = x[lo:hi] @ w[e].float().t()
    if kind == "grouped":
        return y
    dy = s["grad"].float()
    dx, dw = torch.zeros_like(s["x"]), torch.zeros_like(w)
    for e, lo, hi in _each(s["ends"]):
        dx[lo:hi] = dy[lo:hi] @ w[e].float()
        dw[e] = dy[lo:hi].t() @ x[lo:hi]
    return y, dx, dw


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------
# Work
# ---------------------------------------------------------------------------


def work(case):
    kind, m, n, k, size = case["kind"], case["m"], case["n"], case["k"], _SIZE[case["dtype"]]
    if kind == "quantize":
        # x in, values (4 bytes each) and scales out; the largest magnitude and one quotient a value.
        return {"bytes": m * k * (size + 4.0) + 4.0 * m, "flops": 2.0 * m * k}
    rows = m - case["spare"]
    weights = _used(case) if case["experts"] else 1  # an expert without rows is not read
    flops = 2.0 * rows * n * k
    if kind == "codes":
        return {"bytes": m * k + 4.0 * m + n * k + 4.0 * n + 2.0 * m * n, "flops": flops}
    if kind.startswith("w8a8"):
        return {"bytes": 2.0 * rows * k + weights * (n * k + 4.0 * n) + 2.0 * m * n, "flops": flops}
    if kind == "grouped":
        return {"bytes": 2.0 * (rows * k + weights * n * k + m * n), "flops": flops}
    return {"bytes": 2.0 * (rows * k + rows * n + weights * n * k + m * n + m * k + case["experts"] * n * k), "flops": 3.0 * flops}


# ---------------------------------------------------------------------------
# The definition in float64
# ---------------------------------------------------------------------------


def _round64(x):
    """(integers, scales) in float64 of float64 rows; a scale is kept in 32 bits."""
    top = torch.maximum(x.abs().max(dim=1, keepdim=True).values, torch.full((), 1e-12, dtype=torch.float64, device=x.device))
    scale = torch.div(top, torch.full_like(top, 127.0)).to(torch.float32).to(torch.float64)
    low = torch.floor(x / scale)
    part = x / scale - low
    up = (part > 0.5) | ((part == 0.5) & (torch.remainder(low, 2.0) == 1.0))
    return low + up.to(torch.float64), scale


def exact(case, seed):
    made = _inputs(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        q, scale = _round64(made["x"].double())
        return q * scale, scale[:, 0]
    if kind == "codes":
        left = made["codes"].double() * made["x_scale"].double().unsqueeze(1)
    elif kind.startswith("w8a8"):
        q, scale = _round64(made["x"].double())
        left = q * scale
    else:
        left = made["x"].double()
    if not case["experts"]:
        return torch.matmul(left, (made["weight"].double() * made["scale"].double().unsqueeze(1)).t())
    # A row's expert: how many experts end at it or before it.
    expert = (made["offsets"].unsqueeze(0) <= torch.arange(case["m"], device="cuda").unsqueeze(1)).sum(dim=1)
    y = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
    dx = torch.zeros(case["m"], case["k"], dtype=torch.float64, device="cuda")
    dw = torch.zeros(made["weight"].shape, dtype=torch.float64, device="cuda") if kind == "grouped_train" else None
    for e in range(case["experts"]):
        at = torch.nonzero(expert == e)[:, 0]
        w = made["weight"][e].double()
        if kind == "w8a8_grouped":
            w = w * made["scale"][e].double().unsqueeze(1)
        y.index_copy_(0, at, torch.matmul(left[at], w.t()))
        if kind == "grouped_train":
            grad = made["grad"][at].double()
            dx.index_copy_(0, at, torch.matmul(grad, w))
            dw[e] = torch.matmul(grad.t(), left[at])
    return (y, dx, dw) if kind == "grouped_train" else y
