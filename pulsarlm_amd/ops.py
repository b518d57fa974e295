"""Tensor-level ops over the C ABI, mirroring pulsarlm-core's quant-linear ops.

Same names, argument meaning and error behaviour as the reference's
``pulsarlm-core/inc/pulsarlm/kernels/ops.hpp:299-332``:

* ``repack_int4_marlin_cuda(weight_packed, weight_scale, block_n, group_size)``
  -> ``(weight_marlin, scale_marlin)``
* ``repack_fp8_marlin_cuda(weight, weight_scale, block_n, group_size)``
* ``gemm_int4_marlin_cuda(x, weight_marlin, scale_marlin, n, block_n, group_size)``
* ``gemm_fp8_marlin_cuda(...)``

``weight_marlin`` is an opaque 1-D int32 tensor in the plm tile layout (the
reference's is also opaque, marlin.cu:21-30); ``scale_marlin`` keeps the scale's
source dtype, shaped [strips, groups, cols]. Errors raise ``RuntimeError`` with
the reference's ``"<op>: ..."`` message style. Work is enqueued on torch's
current stream of the tensors' device; nothing synchronizes.
"""

from __future__ import annotations

import contextlib
import threading

import torch

from . import _lib

_DTYPES = {torch.bfloat16: _lib.PLM_BF16, torch.float16: _lib.PLM_FP16, torch.float32: _lib.PLM_FP32}


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _stream(device: torch.device) -> int:
    """The current stream's handle. Without the Stream object and the device guard below, a call at
    N 1024, K 2048, M 1 takes 9.2 us instead of 14.5. The raw handle's function is not public: where
    torch has it under no such name, the Stream object is made."""
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    if raw is None or device.index is None or not torch.cuda.is_initialized():
        return torch.cuda.current_stream(device).cuda_stream
    return raw(device.index)


_no_switch = contextlib.nullcontext()


def _on(device: torch.device):
    """torch.cuda.device(device), where the device is not the current one already."""
    if device.index is not None and torch.cuda.is_initialized() and torch.cuda.current_device() == device.index:
        return _no_switch
    return torch.cuda.device(device)


def _require(cond: bool, op: str, msg: str) -> None:
    if not cond:
        raise RuntimeError(f"{op}: {msg}")


def _call(fn_name: str, *args) -> None:
    lib = _lib.load()
    _lib.check(getattr(lib, fn_name)(*args))


# ---------------------------------------------------------------------------
# Workspace: one zero-initialised buffer per (device, stream). The kernels leave
# their arrival counters at zero, so reuse by calls ordered on one stream is safe.
# ---------------------------------------------------------------------------
_ws_lock = threading.Lock()
_ws: dict[tuple[int, int], torch.Tensor] = {}


def workspace(device: torch.device, nbytes: int) -> torch.Tensor | None:
    if nbytes <= 0:
        return None
    key = (device.index if device.index is not None else torch.cuda.current_device(), _stream(device))
    with _ws_lock:
        buf = _ws.get(key)
        if buf is None or buf.numel() < nbytes:
            size = max(nbytes, 1 << 20)
            buf = torch.zeros(size, dtype=torch.uint8, device=device)
            _ws[key] = buf
        return buf


# ---------------------------------------------------------------------------
# Repack
# ---------------------------------------------------------------------------


def _scale_shape(n: int, k: int, block_n: int, group_size: int):
    strips = -(-n // 16)
    ktiles = -(-k // 128)
    groups = -(-(ktiles * 128) // group_size)
    cols = 1 if block_n % 16 == 0 else 16
    return strips, groups, cols


def _repack(op: str, fmt: int, weight: torch.Tensor, n: int, k: int, weight_scale: torch.Tensor, block_n: int,
            group_size: int):
    _require(weight.is_cuda and weight_scale.is_cuda, op, "inputs must be CUDA tensors")
    _require(block_n > 0, op, "block_n must be positive")
    _require(group_size > 0 and group_size % 16 == 0, op, "group_size must be a positive multiple of 16")
    _require(k % group_size == 0, op, "K must be a multiple of group_size")
    rows = -(-n // block_n)
    _require(weight_scale.dim() == 2 and tuple(weight_scale.shape) == (rows, k // group_size), op,
             "weight_scale must be [ceil(N / block_n), K / group_size]")
    _require(weight_scale.dtype in _DTYPES, op, "weight_scale must be fp32, fp16 or bf16")
    src = weight.contiguous()
    scale = weight_scale.contiguous()
    lib = _lib.load()
    wbytes = lib.plm_weight_bytes(fmt, n, k)
    w_out = torch.empty(max(wbytes // 4, 0), dtype=torch.int32, device=weight.device)
    s_out = torch.empty(_scale_shape(n, k, block_n, group_size), dtype=scale.dtype, device=weight.device)
    fn = "plm_repack_int4" if fmt == _lib.PLM_INT4 else "plm_repack_fp8"
    with _on(weight.device):
        _call(fn, _ptr(src), _ptr(scale), _DTYPES[scale.dtype], n, k, block_n, group_size, _ptr(w_out), _ptr(s_out),
              _stream(weight.device))
    return w_out, s_out


def repack_int4_marlin_cuda(weight_packed: torch.Tensor, weight_scale: torch.Tensor, block_n: int, group_size: int):
    """int32 [N, K/8] LSB-first int4 + scales [ceil(N/bn), K/g] -> (weight, scale) in the plm layout
    (ops.hpp:306-311; marlin.cu:601-620)."""
    _require(weight_packed.dtype == torch.int32 and weight_packed.dim() == 2, "repack_int4_marlin",
             "weight_packed must be int32 [N, K/8]")
    n, k = weight_packed.shape[0], weight_packed.shape[1] * 8
    return _repack("repack_int4_marlin", _lib.PLM_INT4, weight_packed, n, k, weight_scale, block_n, group_size)


def repack_fp8_marlin_cuda(weight: torch.Tensor, weight_scale: torch.Tensor, block_n: int, group_size: int):
    """float8_e4m3fn [N, K] + scales -> (weight, scale) in the plm layout (ops.hpp:313-314; marlin.cu:622-629)."""
    _require(weight.dtype == torch.float8_e4m3fn and weight.dim() == 2, "repack_fp8_marlin",
             "weight must be float8_e4m3fn [N, K]")
    n, k = weight.shape
    return _repack("repack_fp8_marlin", _lib.PLM_FP8, weight.view(torch.uint8), n, k, weight_scale, block_n,
                   group_size)


def convert_marlin_cuda(fmt: str, weight_marlin: torch.Tensor, scale_marlin: torch.Tensor, n: int, k: int,
                        block_n: int, group_size: int):
    """Reference Marlin (words, fp32 [K/g, ceil(N/bn)] scales) -> plm layout (fp32 scales)."""
    op = "convert_marlin"
    f = _lib.PLM_INT4 if fmt == "int4" else _lib.PLM_FP8
    _require(weight_marlin.dtype == torch.int32 and scale_marlin.dtype == torch.float32, op,
             "weight_marlin must be int32 and scale_marlin fp32")
    lib = _lib.load()
    w_out = torch.empty(lib.plm_weight_bytes(f, n, k) // 4, dtype=torch.int32, device=weight_marlin.device)
    s_out = torch.empty(_scale_shape(n, k, block_n, group_size), dtype=torch.float32, device=weight_marlin.device)
    with _on(weight_marlin.device):
        _call("plm_convert_marlin", f, _ptr(weight_marlin.contiguous()), _ptr(scale_marlin.contiguous()), n, k,
              block_n, group_size, _ptr(w_out), _ptr(s_out), _stream(weight_marlin.device))
    return w_out, s_out


def dequant_marlin_cuda(fmt: str, weight_marlin: torch.Tensor, scale_marlin: torch.Tensor, n: int, k: int,
                        block_n: int, group_size: int, dtype=torch.bfloat16) -> torch.Tensor:
    """Dense [N, K] round(q * round(scale)) in ``dtype`` from the plm layout."""
    f = _lib.PLM_INT4 if fmt == "int4" else _lib.PLM_FP8
    out = torch.empty((n, k), dtype=dtype, device=weight_marlin.device)
    with _on(weight_marlin.device):
        _call("plm_dequant", f, _ptr(weight_marlin), _ptr(scale_marlin), _DTYPES[scale_marlin.dtype], n, k, block_n,
              group_size, _ptr(out), _DTYPES[dtype], _stream(weight_marlin.device))
    return out


# ---------------------------------------------------------------------------
# GEMM
# ---------------------------------------------------------------------------


def _gemm_checks(op: str, fmt: int, x: torch.Tensor, weight_marlin: torch.Tensor, scale_marlin: torch.Tensor, n: int,
                 block_n: int, group_size: int):
    """gemm<fmt> checks, marlin.cu:547-571."""
    _require(x.is_cuda and weight_marlin.is_cuda and scale_marlin.is_cuda, op, "all inputs must be CUDA tensors")
    _require(x.dtype in (torch.float16, torch.bfloat16), op, "x must be fp16 or bf16")
    _require(x.dim() == 2 and x.is_contiguous(), op, "x must be a contiguous [M, K]")
    _require(weight_marlin.dtype == torch.int32, op, "weight_marlin must be int32")
    _require(scale_marlin.dtype in _DTYPES, op, "scale_marlin must be fp32, fp16 or bf16")
    _require(block_n > 0, op, "block_n must be positive")
    _require(group_size > 0 and group_size % 16 == 0, op, "group_size must be a positive multiple of 16")
    k = x.shape[1]
    _require(k % group_size == 0, op, "K must be a multiple of group_size")
    _require(tuple(scale_marlin.shape) == _scale_shape(n, k, block_n, group_size), op,
             "scale_marlin has the wrong shape for this N, K, block_n and group_size")
    _require(weight_marlin.numel() * 4 == _lib.weight_bytes(fmt, n, k), op,
             "weight_marlin has the wrong size for this shape")


def _gemm(op: str, fmt: int, x, weight_marlin, scale_marlin, n: int, block_n: int, group_size: int,
          out: torch.Tensor | None = None) -> torch.Tensor:
    _gemm_checks(op, fmt, x, weight_marlin, scale_marlin, n, block_n, group_size)
    m, k = x.shape
    y = out if out is not None else torch.empty((m, n), dtype=x.dtype, device=x.device)
    if m == 0 or n == 0:
        return y
    ws = workspace(x.device, _lib.gemm_workspace_bytes(fmt, m, n, k))
    with _on(x.device):
        _call("plm_gemm", fmt, _ptr(x), _DTYPES[x.dtype], _ptr(weight_marlin.contiguous()),
              _ptr(scale_marlin.contiguous()), _DTYPES[scale_marlin.dtype], m, n, k, block_n, group_size, _ptr(y),
              _ptr(ws), 0 if ws is None else ws.numel(), _stream(x.device))
    return y


def gemm_int4_marlin_cuda(x, weight_marlin, scale_marlin, n: int, block_n: int, group_size: int, out=None):
    """y [M, N] = x [M, K] @ dequant(W)^T (ops.hpp:316-323; marlin.cu:631-640)."""
    return _gemm("gemm_int4_marlin", _lib.PLM_INT4, x, weight_marlin, scale_marlin, n, block_n, group_size, out)


def gemm_fp8_marlin_cuda(x, weight_marlin, scale_marlin, n: int, block_n: int, group_size: int, out=None):
    """fp8 W8A16 form (ops.hpp:325-332; marlin.cu:642-651)."""
    return _gemm("gemm_fp8_marlin", _lib.PLM_FP8, x, weight_marlin, scale_marlin, n, block_n, group_size, out)


def quantize_rows_e4m3_cuda(x: torch.Tensor):
    """Per-row dynamic e4m3 quantization: (codes uint8 [M, K], scale fp32 [M]),
    scale = max(amax, 1e-12) / 448 (the test_qwen3_5.cpp:301-311 rule per row)."""
    op = "quantize_rows_e4m3"
    _require(x.is_cuda and x.dtype in (torch.float16, torch.bfloat16), op, "x must be a CUDA fp16/bf16 tensor")
    _require(x.dim() == 2 and x.is_contiguous(), op, "x must be a contiguous [M, K]")
    m, k = x.shape
    codes = torch.empty((m, k), dtype=torch.uint8, device=x.device)
    scale = torch.empty((m,), dtype=torch.float32, device=x.device)
    with _on(x.device):
        _call("plm_quantize_rows_e4m3", _ptr(x), _DTYPES[x.dtype], m, k, _ptr(codes), _ptr(scale),
              _stream(x.device))
    return codes, scale


def gemm_fp8_w8a8_cuda(x, weight_marlin, scale_marlin, n: int, block_n: int, group_size: int, out=None):
    """W8A8: x quantized per row to e4m3, fp8 x fp8 MFMA with fp32 block scales
    (no reference counterpart; the reference's fp8 GEMM is W8A16)."""
    op = "gemm_fp8_w8a8"
    _gemm_checks(op, _lib.PLM_FP8, x, weight_marlin, scale_marlin, n, block_n, group_size)
    _require(group_size % 128 == 0, op, "group_size must be a multiple of 128 for the fp8 MFMA")
    m, k = x.shape
    y = out if out is not None else torch.empty((m, n), dtype=x.dtype, device=x.device)
    if m == 0 or n == 0:
        return y
    ws = workspace(x.device, _lib.gemm_w8a8_workspace_bytes(m, n, k))
    with _on(x.device):
        _call("plm_gemm_w8a8", _ptr(x), _DTYPES[x.dtype], _ptr(weight_marlin.contiguous()),
              _ptr(scale_marlin.contiguous()), _DTYPES[scale_marlin.dtype], m, n, k, block_n, group_size, _ptr(y),
              _ptr(ws), 0 if ws is None else ws.numel(), _stream(x.device))
    return y


# ---------------------------------------------------------------------------
# MoE: experts repacked back to back, grouped GEMM, routed experts
# ---------------------------------------------------------------------------


def repack_int4_experts(weight_packed: torch.Tensor, weight_scale: torch.Tensor, group_size: int):
    """[E, N, K/8] int32 + [E, N, K/g] scales -> per-expert plm layouts back to back:
    (weights int32 [E * words], scales [E, strips, groups, 16])."""
    op = "repack_int4_experts"
    _require(weight_packed.dim() == 3 and weight_scale.dim() == 3, op, "expected [E, N, K/8] and [E, N, K/g]")
    e = weight_packed.shape[0]
    ws, ss = [], []
    for i in range(e):
        w, s = repack_int4_marlin_cuda(weight_packed[i], weight_scale[i], 1, group_size)
        ws.append(w)
        ss.append(s)
    return torch.cat(ws), torch.stack(ss)


def grouped_gemm_int4_cuda(x: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, offsets: torch.Tensor, n: int,
                           group_size: int, out=None) -> torch.Tensor:
    """Rows [offsets[e-1], offsets[e]) of x times expert e's W^T (one at::_grouped_mm of
    paged_forward.cpp:124-125, int4 experts)."""
    op = "grouped_gemm"
    _require(x.is_cuda and x.dim() == 2 and x.is_contiguous() and x.dtype in (torch.float16, torch.bfloat16), op,
             "x must be a contiguous CUDA [rows, K] fp16/bf16")
    _require(offsets.dtype == torch.int32 and offsets.dim() == 1, op, "offsets must be int32 [E]")
    rows, k = x.shape
    e = offsets.shape[0]
    lib = _lib.load()
    _require(weight.numel() * 4 == e * lib.plm_weight_bytes(_lib.PLM_INT4, n, k), op, "weight has the wrong size")
    y = out if out is not None else torch.empty((rows, n), dtype=x.dtype, device=x.device)
    if rows == 0 or n == 0:
        return y
    ws = workspace(x.device, lib.plm_grouped_gemm_workspace_bytes(rows, e))
    with _on(x.device):
        _call("plm_grouped_gemm", _lib.PLM_INT4, _ptr(x), _DTYPES[x.dtype], _ptr(weight), _ptr(scale),
              _DTYPES[scale.dtype], _ptr(offsets.contiguous()), e, rows, n, k, 1, group_size, _ptr(y), _ptr(ws),
              ws.numel(), _stream(x.device))
    return y


def routed_experts_int4_cuda(h: torch.Tensor, top_experts: torch.Tensor, top_weights: torch.Tensor,
                             gate_up: tuple, down: tuple, intermediate: int, group_size: int):
    """routed_experts (paged_forward.cpp:108-130) with int4 experts and SiLU:
    returns (out [T, H] in h's dtype, offsets int32 [E])."""
    op = "routed_experts"
    _require(h.is_cuda and h.dim() == 2 and h.dtype in (torch.float16, torch.bfloat16), op,
             "h must be a CUDA [T, H] fp16/bf16 tensor")
    t, hidden = h.shape
    top_k = top_experts.shape[-1]
    e = gate_up[1].shape[0]
    experts = top_experts.to(torch.int32).contiguous()
    weights = top_weights.to(torch.float32).contiguous()
    out = torch.empty_like(h)
    offsets = torch.empty((e,), dtype=torch.int32, device=h.device)
    lib = _lib.load()
    ws = workspace(h.device, lib.plm_moe_workspace_bytes(t, top_k, e, hidden, intermediate))
    with _on(h.device):
        _call("plm_moe", _ptr(h.contiguous()), _DTYPES[h.dtype], _ptr(experts), _ptr(weights), t, top_k, e, hidden,
              intermediate, _ptr(gate_up[0]), _ptr(gate_up[1]), _ptr(down[0]), _ptr(down[1]),
              _DTYPES[gate_up[1].dtype], group_size, _ptr(offsets), _ptr(out), _ptr(ws),
              0 if ws is None else ws.numel(), _stream(h.device))
    return out, offsets


def route_top_k_cuda(logits: torch.Tensor, k: int, experts_i32: bool = False):
    """route_top_k_cuda (ops.hpp:37-40): (weights fp32 [T, k], experts int64 [T, k]) for
    logits [T, E] whose rows may lie apart (unit column stride); experts_i32 gives int32
    experts (what routed_experts_int4_cuda / plm_moe take) instead. Has no gradient: a backward pass that reaches the
    weights raises."""
    op = "route_top_k"
    if _records(logits):
        return _MxNoGradient.apply(op, lambda: route_top_k_cuda(logits, k, experts_i32), logits)
    _require(logits.is_cuda and logits.dim() == 2 and logits.stride(1) == 1, op,
             "logits must be CUDA [tokens, experts], each row contiguous")
    _require(logits.dtype in _DTYPES, op, "logits must be fp32, fp16 or bf16")
    t, e = logits.shape
    weights = torch.empty((t, k), dtype=torch.float32, device=logits.device)
    chosen = torch.empty((t, k), dtype=torch.int32 if experts_i32 else torch.int64, device=logits.device)
    stride = logits.stride(0) if t > 1 else e
    with _on(logits.device):
        _call("plm_route_top_k", _ptr(logits), _DTYPES[logits.dtype], t, e, stride, k, _ptr(weights),
              None if experts_i32 else _ptr(chosen), _ptr(chosen) if experts_i32 else None, _stream(logits.device))
    return weights, chosen


def silu_mul_cuda(x: torch.Tensor) -> torch.Tensor:
    """silu_mul_cuda (ops.hpp:42-43): silu(x[:, :n]) * x[:, n:], silu rounded to the dtype. Has no
    gradient: a backward pass that reaches it raises."""
    op = "silu_mul"
    if _records(x):
        return _MxNoGradient.apply(op, lambda: silu_mul_cuda(x), x)
    _require(x.is_cuda and x.dim() == 2 and x.is_contiguous() and x.size(1) % 2 == 0, op,
             "x must be contiguous CUDA [tokens, 2 * n]")
    _require(x.dtype in _DTYPES, op, "x must be fp32, fp16 or bf16")
    t, n = x.size(0), x.size(1) // 2
    y = torch.empty((t, n), dtype=x.dtype, device=x.device)
    with _on(x.device):
        _call("plm_silu_mul", _ptr(x), _DTYPES[x.dtype], t, n, _ptr(y), _stream(x.device))
    return y


def moe_block_int4_cuda(h: torch.Tensor, router_logits: torch.Tensor, top_k: int, gate_up: tuple, down: tuple,
                        intermediate: int, group_size: int):
    """The routed-experts half of a MoE block from the router's logits: route_top_k (int32
    experts) then routed_experts with int4 experts and SiLU (qwen4_exp.cpp:542 followed by
    paged_forward.cpp:108-130), all enqueued on the current stream with no host sync.
    Returns (out [T, H], offsets int32 [E], top_weights fp32 [T, k], top_experts int32 [T, k])."""
    weights, experts = route_top_k_cuda(router_logits, top_k, experts_i32=True)
    out, offsets = routed_experts_int4_cuda(h, experts, weights, gate_up, down, intermediate, group_size)
    return out, offsets, weights, experts


def _gemm_int4_plain(op: str, x: torch.Tensor, weight_packed: torch.Tensor, weight_scale: torch.Tensor,
                     group_size: int, num_splits: int) -> torch.Tensor:
    _require(x.is_cuda and x.dim() == 2 and x.dtype in (torch.float16, torch.bfloat16), op,
             "x must be a CUDA [M, K] fp16/bf16 tensor")
    _require(weight_packed.dtype == torch.int32 and weight_packed.dim() == 2, op, "weight_packed must be int32 [N, K/8]")
    m, k = x.shape
    n = weight_packed.shape[0]
    _require(weight_packed.shape[1] * 8 == k, op, "weight_packed must be [N, K/8]")
    _require(weight_scale.dim() == 2 and tuple(weight_scale.shape) == (n, k // group_size) if group_size > 0 else False,
             op, "weight_scale must be [N, K/group_size]")
    scale = weight_scale.to(torch.float32).contiguous()
    y = torch.empty((m, n), dtype=x.dtype, device=x.device)
    lib = _lib.load()
    nbytes = lib.plm_gemm_int4_plain_workspace_bytes(m, n, k, num_splits)
    ws = torch.empty((nbytes,), dtype=torch.uint8, device=x.device) if nbytes > 0 else None
    with _on(x.device):
        _call("plm_gemm_int4_plain", _ptr(x.contiguous()), _DTYPES[x.dtype], _ptr(weight_packed.contiguous()),
              _ptr(scale), m, n, k, group_size, num_splits, _ptr(y), _ptr(ws), 0 if ws is None else ws.numel(),
              _stream(x.device))
    return y


def gemm_int4_cuda(x: torch.Tensor, weight_packed: torch.Tensor, weight_scale: torch.Tensor, group_size: int):
    """gemm_int4_cuda (ops.hpp:272-285): the non-repacked int4 GEMM, W = round(fp32(q * scale))."""
    return _gemm_int4_plain("gemm_int4", x, weight_packed, weight_scale, group_size, 0)


def gemm_int4_split_cuda(x: torch.Tensor, weight_packed: torch.Tensor, weight_scale: torch.Tensor, group_size: int,
                         num_splits: int):
    """gemm_int4_split_cuda (ops.hpp:287-297): the same with the K split forced to num_splits (>= 1)."""
    _require(num_splits >= 1, "gemm_int4", "num_splits must be >= 1")
    return _gemm_int4_plain("gemm_int4", x, weight_packed, weight_scale, group_size, num_splits)


# ---------------------------------------------------------------------------
# MXFP4: microscaled 4-bit floating point (no reference counterpart). 32 consecutive K values share a scale
# 2^(b - 127) and are e2m1 codes; plain form: codes uint8 [M, K/2] (lower K in the low half), scale uint8 [M, K/32].
# ---------------------------------------------------------------------------


def _mx_contiguous(op: str, name: str, x: torch.Tensor, dtypes) -> None:
    if not (x.is_cuda and x.dtype in dtypes):
        _require(False, op, f"{name} must be a CUDA {'fp32, ' if len(dtypes) > 2 else ''}fp16 or bf16 tensor")
    if not (x.dim() == 2 and x.is_contiguous()):
        _require(False, op, f"{name} must be contiguous [rows, columns]")


_HALF = (torch.float16, torch.bfloat16)


def quantize_mxfp4_cuda(x: torch.Tensor):
    """x [M, K] (fp32, fp16 or bf16, K a multiple of 32) -> (codes uint8 [M, K/2], scale uint8 [M, K/32]): scale byte
    floor(log2(amax)) - 2 + 127 per block of 32, codes to nearest (ties to the even code), saturating at 6. A block
    with an infinity or NaN gets scale byte 255, which reads as NaN."""
    op = "quantize_mxfp4"
    _mx_contiguous(op, "x", x, _DTYPES)
    m, k = x.shape
    _require(k % 32 == 0, op, "K must be a multiple of 32")
    codes = torch.empty((m, k // 2), dtype=torch.uint8, device=x.device)
    scale = torch.empty((m, k // 32), dtype=torch.uint8, device=x.device)
    with _on(x.device):
        _call("plm_quantize_mxfp4", _ptr(x), _DTYPES[x.dtype], m, k, _ptr(codes), _ptr(scale), _stream(x.device))
    return codes, scale


def _mx_plain(op: str, codes: torch.Tensor, scale: torch.Tensor):
    _require(codes.is_cuda and scale.is_cuda and codes.device == scale.device, op, "codes and scale must be on one CUDA device")
    _require(codes.dtype == torch.uint8 and scale.dtype == torch.uint8 and codes.dim() == 2 and scale.dim() == 2, op,
             "codes must be uint8 [N, K/2] and scale uint8 [N, K/32]")
    n, k = codes.shape[0], 2 * codes.shape[1]
    _require(k % 32 == 0, op, "K must be a multiple of 32")
    _require(tuple(scale.shape) == (n, k // 32), op, "scale must be [N, K/32]")
    return n, k


def dequantize_mxfp4_cuda(codes: torch.Tensor, scale: torch.Tensor, dtype=torch.bfloat16) -> torch.Tensor:
    """The values [M, K] that codes and scale stand for: exact in bf16 and fp32, rounded once to fp16."""
    op = "dequantize_mxfp4"
    m, k = _mx_plain(op, codes, scale)
    _require(dtype in _DTYPES, op, "dtype must be fp32, fp16 or bf16")
    out = torch.empty((m, k), dtype=dtype, device=codes.device)
    codes, scale = codes.contiguous(), scale.contiguous()  # both live until the call: copies do not share memory
    with _on(codes.device):
        _call("plm_dequantize_mxfp4", _ptr(codes), _ptr(scale), m, k, _ptr(out), _DTYPES[dtype], _stream(codes.device))
    return out


def repack_mxfp4_cuda(codes: torch.Tensor, scale: torch.Tensor):
    """An MXFP4 weight [N, K] (codes uint8 [N, K/2], scale uint8 [N, K/32]) for the products: (weight int32 1-D,
    scale int32 [groups, K tiles, 64]), opaque, the plm tile layout of the format."""
    op = "repack_mxfp4"
    n, k = _mx_plain(op, codes, scale)
    _require(max(n, k) <= 1 << 19, op, "N and K must be at most 2^19")
    weight = torch.empty((_lib.mxfp4_bytes("mxfp4_weight_bytes", n, k) // 4,), dtype=torch.int32, device=codes.device)
    packed = torch.empty(_mx_scale_shape(n, k), dtype=torch.int32, device=codes.device)
    codes, scale = codes.contiguous(), scale.contiguous()
    with _on(codes.device):
        _call("plm_repack_mxfp4", _ptr(codes), _ptr(scale), n, k, _ptr(weight), _ptr(packed), _stream(codes.device))
    return weight, packed


def _mx_scale_shape(n: int, k: int):
    return -(-n // 64), -(-k // 128), 64


def _mx_weight(op: str, x: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, n: int, k: int) -> None:
    _require(n >= 0 and k >= 0, op, "sizes must be non-negative")
    at = x.get_device()
    _require(weight.get_device() == at and scale.get_device() == at, op, "x and the weights must be on one device")
    _require(weight.dtype is torch.int32 and scale.dtype is torch.int32 and weight.is_contiguous() and scale.is_contiguous(), op,
             "weight and scale must be contiguous int32, as repack_mxfp4 returns them")
    _require(weight.numel() * 4 == _lib.mxfp4_bytes("mxfp4_weight_bytes", n, k), op, "weight has the wrong size for this shape")
    _require(scale.shape == _mx_scale_shape(n, k), op, "scale has the wrong shape for this N and K")


def _mx_scratch(name: str, x: torch.Tensor, *sizes: int) -> torch.Tensor | None:
    """Scratch of one call, from torch's allocator: a captured call's belongs to its graph."""
    nbytes = _lib.mxfp4_bytes(name + "_workspace_bytes", *sizes)
    return torch.empty((nbytes,), dtype=torch.uint8, device=x.device) if nbytes > 0 else None


def _mx_out(op: str, x: torch.Tensor, shape, out: torch.Tensor | None) -> torch.Tensor:
    if out is None:
        return x.new_empty(shape)
    _require(out.dtype == x.dtype and out.device == x.device and tuple(out.shape) == shape and out.is_contiguous(), op,
             f"out must be contiguous {list(shape)} of x's dtype and device")
    return out


class _MxLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, scale, n):
        y = gemm_mxfp4_cuda(x, weight, scale, n)
        ctx.save_for_backward(weight, scale)
        ctx.k = x.shape[1]
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        return gemm_mxfp4_grad_cuda(dy.contiguous(), *ctx.saved_tensors, ctx.k), None, None, None


class _MxGated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, gate_scale, up, up_scale, intermediate):
        h, gate_up = gated_mxfp4_cuda(x, (gate, gate_scale), (up, up_scale), intermediate, keep_gate_up=True)
        ctx.mark_non_differentiable(gate_up)
        ctx.set_materialize_grads(False)  # no zeros for gate_up's
        ctx.save_for_backward(gate_up, gate, gate_scale, up, up_scale)
        ctx.k = x.shape[1]
        return h, gate_up

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, _):
        if dh is None:
            return (None,) * 6
        gate_up, gate, gate_scale, up, up_scale = ctx.saved_tensors
        return gated_mxfp4_grad_cuda(dh.contiguous(), gate_up, (gate, gate_scale), (up, up_scale), ctx.k), *(None,) * 5


class _MxNoGradient(torch.autograd.Function):
    """call(): an output in x's graph whose gradient is asked for in vain, and says so then."""

    @staticmethod
    def forward(ctx, op, call, *inputs):
        ctx.op = op
        return call()

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.op}: has no gradient")


def _mx_records(x: torch.Tensor) -> bool:
    return x.requires_grad and torch.is_grad_enabled()


def _records(*inputs: torch.Tensor) -> bool:
    return torch.is_grad_enabled() and any(t.requires_grad for t in inputs)


def _mx_x(op: str, x: torch.Tensor):
    _mx_contiguous(op, "x", x, _HALF)
    _require(x.shape[1] % 32 == 0, op, "K must be a multiple of 32")
    return x.shape


def gemm_mxfp4_cuda(x: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, n: int, out=None) -> torch.Tensor:
    """y [M, N] = x [M, K] @ W^T with an MXFP4 weight (repack_mxfp4_cuda) and 16-bit x, fp32 sums. out may not overlap x.
    Differentiable in x, without out, by gemm_mxfp4_grad_cuda."""
    op = "gemm_mxfp4"
    if _mx_records(x):
        _require(out is None, op, "out records no gradient")
        return _MxLinear.apply(x, weight, scale, n)
    m, k = _mx_x(op, x)
    _mx_weight(op, x, weight, scale, n, k)
    y = _mx_out(op, x, (m, n), out)
    with _on(x.device):
        _call("plm_gemm_mxfp4", _ptr(x), _DTYPES[x.dtype], _ptr(weight), _ptr(scale), m, n, k, _ptr(y), _stream(x.device))
    return y


def gemm_mxfp4_w4a4_cuda(x: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, n: int, out=None) -> torch.Tensor:
    """W4A4: the same with x quantized as by quantize_mxfp4_cuda, on the fp4 matrix instruction. Has no gradient: a
    backward pass that reaches it raises."""
    op = "gemm_mxfp4_w4a4"
    if _mx_records(x):
        _require(out is None, op, "out records no gradient")
        return _MxNoGradient.apply(op, lambda: gemm_mxfp4_w4a4_cuda(x, weight, scale, n), x)
    m, k = _mx_x(op, x)
    _mx_weight(op, x, weight, scale, n, k)
    y = _mx_out(op, x, (m, n), out)
    ws = _mx_scratch(op, x, m, n, k)
    with _on(x.device):
        _call("plm_gemm_mxfp4_w4a4", _ptr(x), _DTYPES[x.dtype], _ptr(weight), _ptr(scale), m, n, k, _ptr(y), _ptr(ws),
              0 if ws is None else ws.numel(), _stream(x.device))
    return y


def gemm_mxfp4_grad_cuda(dy: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, k: int, out=None) -> torch.Tensor:
    """The gradient of gemm_mxfp4_cuda's x: dx [M, K] = dy [M, N] @ W. Has none of its own."""
    op = "gemm_mxfp4_grad"
    if _mx_records(dy):
        _require(out is None, op, "out records no gradient")
        return _MxNoGradient.apply(op, lambda: gemm_mxfp4_grad_cuda(dy, weight, scale, k), dy)
    _mx_contiguous(op, "dy", dy, _HALF)
    _require(k % 32 == 0, op, "K must be a multiple of 32")
    m, n = dy.shape
    _mx_weight(op, dy, weight, scale, n, k)
    dx = _mx_out(op, dy, (m, k), out)
    ws = _mx_scratch(op if dy.data_ptr() % 16 else "gemm_mxfp4_grad_aligned", dy, m, n, k)
    with _on(dy.device):
        _call("plm_gemm_mxfp4_grad", _ptr(dy), _DTYPES[dy.dtype], _ptr(weight), _ptr(scale), m, n, k, _ptr(dx), _ptr(ws),
              0 if ws is None else ws.numel(), _stream(dy.device))
    return dx


def gated_mxfp4_cuda(x: torch.Tensor, gate: tuple, up: tuple, intermediate: int, keep_gate_up: bool = False):
    """h [M, I] = silu(x @ Wgate^T) * (x @ Wup^T) in one kernel, from fp32 sums; gate and up are (weight, scale) pairs
    of repack_mxfp4_cuda. keep_gate_up: (h, gate_up fp32 [M, 2 I]), what gated_mxfp4_grad_cuda takes. h is differentiable
    in x by that (gate_up is kept then in either case), gate_up is not."""
    op = "gated_mxfp4"
    if _mx_records(x):
        h, gate_up = _MxGated.apply(x, *gate, *up, intermediate)
        return (h, gate_up) if keep_gate_up else h
    m, k = _mx_x(op, x)
    for w in (gate, up):
        _mx_weight(op, x, w[0], w[1], intermediate, k)
    h = torch.empty((m, intermediate), dtype=x.dtype, device=x.device)
    gate_up = torch.empty((m, 2 * intermediate), dtype=torch.float32, device=x.device) if keep_gate_up else None
    with _on(x.device):
        _call("plm_gated_mxfp4", _ptr(x), _DTYPES[x.dtype], _ptr(gate[0]), _ptr(gate[1]), _ptr(up[0]), _ptr(up[1]), m,
              intermediate, k, _ptr(h), _ptr(gate_up), _stream(x.device))
    return (h, gate_up) if keep_gate_up else h


def gated_mxfp4_grad_cuda(dh: torch.Tensor, gate_up: torch.Tensor, gate: tuple, up: tuple, hidden: int) -> torch.Tensor:
    """The gradient of gated_mxfp4_cuda's x [M, hidden] from dh [M, I] and the gate_up that it kept, d gate and d up rounded
    to dh's type for the products (in fp16 after a power of two a row that keeps them in range). Has none of its own."""
    op = "gated_mxfp4_grad"
    if _mx_records(dh) or _mx_records(gate_up):
        return _MxNoGradient.apply(op, lambda: gated_mxfp4_grad_cuda(dh, gate_up, gate, up, hidden), dh, gate_up)
    _mx_contiguous(op, "dh", dh, _HALF)
    _require(hidden % 32 == 0, op, "K must be a multiple of 32")
    m, n = dh.shape
    _require(gate_up.dtype == torch.float32 and gate_up.device == dh.device and tuple(gate_up.shape) == (m, 2 * n) and
             gate_up.is_contiguous(), op, "gate_up must be contiguous fp32 [M, 2 I] on dh's device")
    for w in (gate, up):
        _mx_weight(op, dh, w[0], w[1], n, hidden)
    dx = torch.empty((m, hidden), dtype=dh.dtype, device=dh.device)
    ws = _mx_scratch(op, dh, m, n, hidden)
    with _on(dh.device):
        _call("plm_gated_mxfp4_grad", _ptr(dh), _ptr(gate_up), _DTYPES[dh.dtype], _ptr(gate[0]), _ptr(gate[1]), _ptr(up[0]),
              _ptr(up[1]), m, n, hidden, _ptr(dx), _ptr(ws), 0 if ws is None else ws.numel(), _stream(dh.device))
    return dx


def mlp_mxfp4_w4a4_cuda(x: torch.Tensor, gate: tuple, up: tuple, down: tuple, intermediate: int) -> torch.Tensor:
    """The feed-forward block with 4-bit activations: y [M, K] = Q(h) @ Wdown^T, h = silu(g) u of Q(x), Q as
    quantize_mxfp4_cuda; h is quantized from its fp32 values. Wgate, Wup [I, K], Wdown [K, I]; I a multiple of 32. Has no
    gradient: a backward pass that reaches it raises."""
    op = "mlp_mxfp4_w4a4"
    if _mx_records(x):
        return _MxNoGradient.apply(op, lambda: mlp_mxfp4_w4a4_cuda(x, gate, up, down, intermediate), x)
    m, k = _mx_x(op, x)
    _require(intermediate % 32 == 0, op, "the intermediate size must be a multiple of 32")
    for w in (gate, up):
        _mx_weight(op, x, w[0], w[1], intermediate, k)
    _mx_weight(op, x, down[0], down[1], k, intermediate)
    y = torch.empty_like(x)
    ws = _mx_scratch(op, x, m, intermediate, k)
    with _on(x.device):
        _call("plm_mlp_mxfp4_w4a4", _ptr(x), _DTYPES[x.dtype], _ptr(gate[0]), _ptr(gate[1]), _ptr(up[0]), _ptr(up[1]),
              _ptr(down[0]), _ptr(down[1]), m, intermediate, k, _ptr(y), _ptr(ws), 0 if ws is None else ws.numel(),
              _stream(x.device))
    return y


# ---------------------------------------------------------------------------
# 8-bit integers with a scale for each token and channel, and experts in 8 and 16 bits (formats that the reference has no
# kernels of its own for). Weights are row-major and read in place: int8 [N, K] with scale fp32 [N], or 16-bit; by expert
# [E, N, K]. A grouped call's rows are sorted by expert, offsets int32 [E] their inclusive ends, as in grouped_gemm_int4_cuda.
# Operands of the products begin at 16 bytes (16-bit x of an 8-bit product: at any element), outputs at any element. An out may not
# overlap an input.
# ---------------------------------------------------------------------------


def quantize_rows_int8_cuda(x: torch.Tensor):
    """x [M, K] (fp32, fp16 or bf16; tokens, or a weight's output channels) -> (codes int8 [M, K], scale fp32 [M]): scale
    max(amax, 1e-12) / 127, codes the integers nearest to x / scale, ties to even. A row with an infinity or NaN gets scale
    NaN and codes 0. Has no gradient: a backward pass that reaches it raises."""
    op = "quantize_rows_int8"
    if _mx_records(x):
        return _MxNoGradient.apply(op, lambda: quantize_rows_int8_cuda(x), x)
    _mx_contiguous(op, "x", x, _DTYPES)
    m, k = x.shape
    codes = torch.empty((m, k), dtype=torch.int8, device=x.device)
    scale = torch.empty((m,), dtype=torch.float32, device=x.device)
    with _on(x.device):
        _call("plm_quantize_rows_int8", _ptr(x), _DTYPES[x.dtype], m, k, _ptr(codes), _ptr(scale), _stream(x.device))
    return codes, scale


def _int8_codes(op: str, name: str, codes: torch.Tensor, scale: torch.Tensor, dim: int) -> None:
    if not (codes.is_cuda and codes.dtype is torch.int8 and codes.dim() == dim and codes.is_contiguous()):
        _require(False, op, f"{name} must be a contiguous CUDA int8 tensor of {dim} dimensions")
    if not (scale.dtype is torch.float32 and scale.get_device() == codes.get_device() and scale.shape == codes.shape[:-1] and scale.is_contiguous()):
        _require(False, op, f"{name}'s scale must be contiguous fp32, one for each row, on its device")


def dequantize_rows_int8_cuda(codes: torch.Tensor, scale: torch.Tensor, dtype=torch.bfloat16) -> torch.Tensor:
    """The values [M, K] that codes and scale stand for: their product in fp32, rounded to dtype. Has no gradient."""
    op = "dequantize_rows_int8"
    if _mx_records(scale):
        return _MxNoGradient.apply(op, lambda: dequantize_rows_int8_cuda(codes, scale, dtype), scale)
    _int8_codes(op, "codes", codes, scale, 2)
    _require(dtype in _DTYPES, op, "dtype must be fp32, fp16 or bf16")
    m, k = codes.shape
    out = torch.empty((m, k), dtype=dtype, device=codes.device)
    with _on(codes.device):
        _call("plm_dequantize_rows_int8", _ptr(codes), _ptr(scale), m, k, _ptr(out), _DTYPES[dtype], _stream(codes.device))
    return out


def _int8_out(op: str, like: torch.Tensor, dtype, shape, out: torch.Tensor | None) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=dtype, device=like.device)
    _require(out.dtype == dtype and out.device == like.device and tuple(out.shape) == shape and out.is_contiguous(), op,
             f"out must be contiguous {list(shape)} of type {dtype} on the inputs' device")
    return out


def gemm_int8_cuda(codes: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, dtype=torch.bfloat16,
                   out=None) -> torch.Tensor:
    """y [M, N] = x_scale[m] scale[n] sum_k codes[m, k] weight[n, k] in dtype (fp16 or bf16), the sums exact: int8 codes
    [M, K] and x_scale fp32 [M] as quantize_rows_int8_cuda makes them, weight int8 [N, K] and scale fp32 [N]. K a multiple of
    16. Has no gradient."""
    op = "gemm_int8"
    if _records(x_scale, scale):
        _require(out is None, op, "out records no gradient")
        return _MxNoGradient.apply(op, lambda: gemm_int8_cuda(codes, x_scale, weight, scale, dtype), x_scale, scale)
    _int8_codes(op, "codes", codes, x_scale, 2)
    _int8_codes(op, "weight", weight, scale, 2)
    m, k = codes.shape
    n = weight.shape[0]
    _require(weight.shape[1] == k and weight.get_device() == codes.get_device(), op, "weight must be [N, K] for codes [M, K], on their device")
    _require(dtype in _HALF, op, "dtype must be fp16 or bf16")
    y = _int8_out(op, codes, dtype, (m, n), out)
    ws = _mx_scratch(op, codes, m, n, k)
    with _on(codes.device):
        _call("plm_gemm_int8", _ptr(codes), _ptr(x_scale), _ptr(weight), _ptr(scale), m, n, k, _ptr(y), _DTYPES[dtype], _ptr(ws),
              0 if ws is None else ws.numel(), _stream(codes.device))
    return y


def gemm_int8_w8a8_cuda(x: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, out=None) -> torch.Tensor:
    """W8A8: gemm_int8_cuda with 16-bit x [M, K], quantized on the way as by quantize_rows_int8_cuda; y in x's type. out may
    not overlap x. Has no gradient: a backward pass that reaches it raises."""
    op = "gemm_int8_w8a8"
    if _records(x, scale):
        _require(out is None, op, "out records no gradient")
        return _MxNoGradient.apply(op, lambda: gemm_int8_w8a8_cuda(x, weight, scale), x, scale)
    _mx_contiguous(op, "x", x, _HALF)
    _int8_codes(op, "weight", weight, scale, 2)
    m, k = x.shape
    n = weight.shape[0]
    _require(weight.shape[1] == k and weight.get_device() == x.get_device(), op, "weight must be [N, K] for x [M, K], on its device")
    y = _mx_out(op, x, (m, n), out)
    ws = _mx_scratch(op, x, m, n, k)
    with _on(x.device):
        _call("plm_gemm_int8_w8a8", _ptr(x), _DTYPES[x.dtype], _ptr(weight), _ptr(scale), m, n, k, _ptr(y), _ptr(ws),
              0 if ws is None else ws.numel(), _stream(x.device))
    return y


def _expert_offsets(op: str, x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> None:
    _require(weight.get_device() == x.get_device() and offsets.get_device() == x.get_device(), op, "x, weight and offsets must be on one device")
    if not (offsets.dtype is torch.int32 and offsets.shape == weight.shape[:1] and offsets.is_contiguous()):
        _require(False, op, "offsets must be contiguous int32 [E]")


def grouped_gemm_int8_cuda(x: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, offsets: torch.Tensor, out=None) -> torch.Tensor:
    """Rows [offsets[e-1], offsets[e]) of x times expert e's W^T, W8A8 as gemm_int8_w8a8_cuda: weight int8 [E, N, K], scale
    fp32 [E, N]. Rows past the last expert's are left as they were in out, and zero in a new tensor. Has no gradient: a
    backward pass that reaches it raises."""
    op = "grouped_gemm_int8"
    if _records(x, scale):
        _require(out is None, op, "out records no gradient")
        return _MxNoGradient.apply(op, lambda: grouped_gemm_int8_cuda(x, weight, scale, offsets), x, scale)
    _mx_contiguous(op, "x", x, _HALF)
    _int8_codes(op, "weight", weight, scale, 3)
    _expert_offsets(op, x, weight, offsets)
    rows, k = x.shape
    e, n = scale.shape
    _require(weight.shape[2] == k, op, "weight must be [E, N, K] for x [rows, K]")
    y = _mx_out(op, x, (rows, n), out)
    ws = _mx_scratch(op, x, rows, n, k)
    with _on(x.device):
        _call("plm_grouped_gemm_int8", _ptr(x), _DTYPES[x.dtype], _ptr(weight), _ptr(scale), _ptr(offsets), e, rows, n, k, _ptr(y),
              int(out is None), _ptr(ws), 0 if ws is None else ws.numel(), _stream(x.device))
    return y


class _Grouped(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, offsets):
        ctx.save_for_backward(x, weight, offsets)
        return grouped_gemm_cuda(x, weight, offsets)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, offsets = ctx.saved_tensors
        dy = dy.contiguous()
        if dy.data_ptr() % 16 != 0:  # a part of a longer gradient (torch.cat's), from any element on
            dy = dy.clone()
        dx = grouped_gemm_grad_x_cuda(dy, weight, offsets) if ctx.needs_input_grad[0] else None
        dw = grouped_gemm_grad_w_cuda(dy, x, offsets) if ctx.needs_input_grad[1] else None
        return dx, dw, None


def _expert_weight(op: str, x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> None:
    if not (weight.dim() == 3 and weight.dtype == x.dtype and weight.is_contiguous()):
        _require(False, op, "weight must be contiguous [E, N, K] of the rows' type")
    _expert_offsets(op, x, weight, offsets)


def grouped_gemm_cuda(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, out=None) -> torch.Tensor:
    """Rows [offsets[e-1], offsets[e]) of x [rows, K] times expert e's W^T, 16-bit weight [E, N, K] of x's type (one
    at::_grouped_mm of paged_forward.cpp:124-125), fp32 sums. Rows past the last expert's are left as they were in out, and
    zero in a new tensor. K a multiple of 8, for the gradients N, too. Differentiable in x and weight, without out."""
    op = "grouped_gemm"
    if _records(x, weight):
        _require(out is None, op, "out records no gradient")
        _require(weight.dim() != 3 or weight.shape[1] % 8 == 0, op, "N must be a multiple of 8 for the gradients")
        return _Grouped.apply(x, weight, offsets)
    _mx_contiguous(op, "x", x, _HALF)
    _expert_weight(op, x, weight, offsets)
    rows, k = x.shape
    e, n = weight.shape[:2]
    _require(weight.shape[2] == k, op, "weight must be [E, N, K] for x [rows, K]")
    y = _mx_out(op, x, (rows, n), out)
    with _on(x.device):
        _call("plm_grouped_gemm_16", _ptr(x), _DTYPES[x.dtype], _ptr(weight), _ptr(offsets), e, rows, n, k, _ptr(y), int(out is None), _stream(x.device))
    return y


def grouped_gemm_grad_x_cuda(dy: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """The gradient of grouped_gemm_cuda's x: dx [rows, K] = dy [rows, N] W_e, zero past the last expert's rows. N and K
    multiples of 8. Has none of its own."""
    op = "grouped_gemm_grad_x"
    if _records(dy, weight):
        return _MxNoGradient.apply(op, lambda: grouped_gemm_grad_x_cuda(dy, weight, offsets), dy, weight)
    _mx_contiguous(op, "dy", dy, _HALF)
    _expert_weight(op, dy, weight, offsets)
    rows, n = dy.shape
    e, k = weight.shape[0], weight.shape[2]
    _require(weight.shape[1] == n, op, "weight must be [E, N, K] for dy [rows, N]")
    dx = dy.new_empty((rows, k))
    with _on(dy.device):
        _call("plm_grouped_gemm_grad_x", _ptr(dy), _DTYPES[dy.dtype], _ptr(weight), _ptr(offsets), e, rows, n, k, _ptr(dx), 1, _stream(dy.device))
    return dx


def grouped_gemm_grad_w_cuda(dy: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """The gradient of grouped_gemm_cuda's weight: dw [E, N, K], expert e's the sum over its rows of dy[r, n] x[r, k], zero
    for an expert without rows. N and K multiples of 8. Has none of its own."""
    op = "grouped_gemm_grad_w"
    if _records(dy, x):
        return _MxNoGradient.apply(op, lambda: grouped_gemm_grad_w_cuda(dy, x, offsets), dy, x)
    _mx_contiguous(op, "dy", dy, _HALF)
    _mx_contiguous(op, "x", x, _HALF)
    _require(x.dtype == dy.dtype and x.shape[0] == dy.shape[0], op, "dy and x must have one type and as many rows")
    _require(offsets.dim() == 1, op, "offsets must be contiguous int32 [E]")
    e, (rows, n), k = offsets.shape[0], dy.shape, x.shape[1]
    dw = dy.new_empty((e, n, k))
    _expert_offsets(op, dy, dw, offsets)
    _require(x.get_device() == dy.get_device(), op, "dy, x and offsets must be on one device")
    with _on(dy.device):
        _call("plm_grouped_gemm_grad_w", _ptr(dy), _ptr(x), _DTYPES[dy.dtype], _ptr(offsets), e, rows, n, k, _ptr(dw), _stream(dy.device))
    return dw
