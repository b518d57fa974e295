"""The int8 and expert operators as a user's program runs them together, in the Python and the C++ layer: experts between
a router and the sum of their outputs, trained and served, and gradients that autograd records or refuses."""

import pytest
import torch

from pulsarlm_amd import _host, ops
from tests import _dense as dense

pytestmark = pytest.mark.gpu

LAYERS = pytest.mark.parametrize("layer", [ops, _host], ids=["python", "host"])


def leaf(x):
    return x.clone().requires_grad_()


def parts(counts, n=72, k=64, dtype=torch.bfloat16):
    rows = sum(counts)
    return (dense.values((rows, k), dtype, 1), dense.values((len(counts), n, k), dtype, 2), dense.values((rows, n), dtype, 3), dense.offsets(counts))


@pytest.mark.parametrize("m", [1, 20, 300])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_host_layer_matches_ops(m, dtype):
    dt, n, k = dense.DT[dtype], 96, 160
    x, w, ws = dense.values((m, k), dt, 1), dense.codes(n, k, 2), dense.scales(n, 3)
    for a, b in zip(_host.quantize_rows_int8_cuda(x), ops.quantize_rows_int8_cuda(x)):
        assert torch.equal(a, b)
    q = ops.quantize_rows_int8_cuda(x)
    assert torch.equal(_host.dequantize_rows_int8_cuda(*q, dt), ops.dequantize_rows_int8_cuda(*q, dt))
    assert torch.equal(_host.gemm_int8_cuda(*q, w, ws, dt), ops.gemm_int8_cuda(*q, w, ws, dt))
    assert torch.equal(_host.gemm_int8_w8a8_cuda(x, w, ws), ops.gemm_int8_w8a8_cuda(x, w, ws))
    counts = [m // 2, 0, m - m // 2]
    x, w16, dy, off = parts(counts, dtype=dt)
    w8, ws8 = dense.codes(3 * 72, 64, 4).view(3, 72, 64), dense.scales(3 * 72, 5).view(3, 72)
    assert torch.equal(_host.grouped_gemm_int8_cuda(x, w8, ws8, off), ops.grouped_gemm_int8_cuda(x, w8, ws8, off))
    assert torch.equal(_host.grouped_gemm_cuda(x, w16, off), ops.grouped_gemm_cuda(x, w16, off))
    assert torch.equal(_host.grouped_gemm_grad_x_cuda(dy, w16, off), ops.grouped_gemm_grad_x_cuda(dy, w16, off))
    assert torch.equal(_host.grouped_gemm_grad_w_cuda(dy, x, off), ops.grouped_gemm_grad_w_cuda(dy, x, off))


def test_linear_int8():
    n, k = 72, 160
    w, ws = dense.codes(n, k, 1), dense.scales(n, 2)
    x = dense.values((6, k), torch.bfloat16, 3).view(2, 3, k)
    y = _host.linear.int8(w, ws[:, None]).apply(x)
    assert y.shape == (2, 3, n) and torch.equal(y.view(6, n), ops.gemm_int8_w8a8_cuda(x.view(6, k), w, ws))
    with pytest.raises(RuntimeError, match="linear: codes must be int8"):
        _host.linear.int8(w.float(), ws)


@LAYERS
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_experts_record_their_gradients(dtype, layer):
    counts = [30, 0, 41, 1]
    x, w, dy, off = parts(counts, dtype=dense.DT[dtype])
    dx, dw = layer.grouped_gemm_grad_x_cuda(dy, w, off), layer.grouped_gemm_grad_w_cuda(dy, x, off)
    a, b = leaf(x), leaf(w)
    y = layer.grouped_gemm_cuda(a, b, off)
    assert y.requires_grad and torch.equal(y, layer.grouped_gemm_cuda(x, w, off))
    y.backward(dy)
    assert torch.equal(a.grad, dx) and torch.equal(b.grad, dw)
    # One of them alone, and a sum's gradient, which is one value, expanded.
    a = leaf(x)
    layer.grouped_gemm_cuda(a, w, off).sum().backward()
    assert torch.equal(a.grad, layer.grouped_gemm_grad_x_cuda(torch.ones_like(dy), w, off))
    b = leaf(w)
    layer.grouped_gemm_cuda(x, b, off).backward(dy)
    assert torch.equal(b.grad, dw)
    with torch.no_grad():
        assert not layer.grouped_gemm_cuda(leaf(x), leaf(w), off).requires_grad
    # Second derivatives are refused.
    a, d = leaf(x), leaf(dy)
    g, = torch.autograd.grad(layer.grouped_gemm_cuda(a, w, off), a, d, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@LAYERS
def test_what_has_no_gradient_says_so(layer):
    counts, n, k = [8, 12], 72, 64
    x, w16, dy, off = parts(counts)
    w, ws = dense.codes(n, k, 4), dense.scales(n, 5)
    w8, ws8 = dense.codes(2 * n, k, 6).view(2, n, k), dense.scales(2 * n, 7).view(2, n)
    q, xs = layer.quantize_rows_int8_cuda(x)
    bf = torch.bfloat16
    for op, f, t in (("quantize_rows_int8", lambda x: layer.quantize_rows_int8_cuda(x)[1], x), ("gemm_int8_w8a8", lambda x: layer.gemm_int8_w8a8_cuda(x, w, ws), x),
                     ("gemm_int8_w8a8", lambda s: layer.gemm_int8_w8a8_cuda(x, w, s), ws), ("dequantize_rows_int8", lambda s: layer.dequantize_rows_int8_cuda(q, s, bf), xs),
                     ("gemm_int8", lambda s: layer.gemm_int8_cuda(q, s, w, ws, bf), xs), ("gemm_int8", lambda s: layer.gemm_int8_cuda(q, xs, w, s, bf), ws),
                     ("grouped_gemm_int8", lambda x: layer.grouped_gemm_int8_cuda(x, w8, ws8, off), x), ("grouped_gemm_int8", lambda s: layer.grouped_gemm_int8_cuda(x, w8, s, off), ws8),
                     ("grouped_gemm_grad_x", lambda d: layer.grouped_gemm_grad_x_cuda(d, w16, off), dy), ("grouped_gemm_grad_x", lambda w: layer.grouped_gemm_grad_x_cuda(dy, w, off), w16),
                     ("grouped_gemm_grad_w", lambda d: layer.grouped_gemm_grad_w_cuda(d, x, off), dy), ("grouped_gemm_grad_w", lambda x: layer.grouped_gemm_grad_w_cuda(dy, x, off), x)):
        y = f(leaf(t))
        assert y.requires_grad and torch.equal(y, f(t)), op
        with pytest.raises(RuntimeError, match=f"{op}: has no gradient"):
            y.sum().backward()
    assert not layer.quantize_rows_int8_cuda(leaf(x))[0].requires_grad


def test_out_records_nothing():
    counts = [8, 12]
    x, w, _, off = parts(counts)
    w8, ws8 = dense.codes(2 * 72, 64, 6).view(2, 72, 64), dense.scales(2 * 72, 7).view(2, 72)
    out = torch.empty(20, 72, dtype=x.dtype, device="cuda")
    for f in (lambda x, out: ops.grouped_gemm_cuda(x, w, off, out=out), lambda x, out: ops.grouped_gemm_int8_cuda(x, w8, ws8, off, out=out),
              lambda x, out: ops.gemm_int8_w8a8_cuda(x, w8[0], ws8[0], out=out)):
        with pytest.raises(RuntimeError, match="out records no gradient"):
            f(leaf(x), out)
        with torch.no_grad():
            assert f(leaf(x), out) is out


@LAYERS
def test_refusals_come_through(layer):
    counts = [8, 12]
    x, w, dy, off = parts(counts)
    c, s = layer.quantize_rows_int8_cuda(x)
    for f, msg in ((lambda: layer.grouped_gemm_cuda(x.t(), w, off), "grouped_gemm: x must be contiguous"),
                   (lambda: layer.grouped_gemm_cuda(x, w.half(), off), "grouped_gemm: weight must be contiguous"),
                   (lambda: layer.grouped_gemm_cuda(x, w.transpose(1, 2), off), "grouped_gemm: weight must be contiguous"),
                   (lambda: layer.grouped_gemm_cuda(x, w, off.long()), "grouped_gemm: offsets must be contiguous int32"),
                   (lambda: layer.grouped_gemm_cuda(x, w, off[:1]), "grouped_gemm: offsets must be contiguous int32"),
                   (lambda: layer.grouped_gemm_cuda(x, w, off.cpu()), "grouped_gemm: x, weight and offsets must be on one device"),
                   (lambda: layer.grouped_gemm_cuda(x[:, :56].contiguous(), w, off), "grouped_gemm: weight must be"),
                   (lambda: layer.grouped_gemm_cuda(leaf(x), w[:, :70].contiguous(), off), "grouped_gemm: N must be a multiple of 8"),
                   (lambda: layer.grouped_gemm_grad_w_cuda(dy, x[:4], off), "grouped_gemm_grad_w: dy and x must have"),
                   (lambda: layer.grouped_gemm_grad_x_cuda(x, w, off), "grouped_gemm_grad_x: weight must be"),
                   (lambda: layer.gemm_int8_cuda(c, s[:3], c, s, torch.bfloat16), "gemm_int8: codes's scale must be"),
                   (lambda: layer.gemm_int8_cuda(c, s, c, s, torch.float32), "gemm_int8: dtype must be"),
                   (lambda: layer.gemm_int8_w8a8_cuda(x, c[:, :48].contiguous(), s), "gemm_int8_w8a8: weight must be"),
                   (lambda: layer.gemm_int8_w8a8_cuda(x.float(), c, s), "gemm_int8_w8a8: x must be"),
                   (lambda: layer.gemm_int8_w8a8_cuda(x, c, s.double()), "gemm_int8_w8a8: weight's scale must be")):
        with pytest.raises(RuntimeError, match=msg):
            f()


def routed(t, hidden, experts, top_k, seed):
    """Tokens sent to their experts: (x [T * k, H] sorted by expert, weights, where each came from, offsets)."""
    x = dense.values((t, hidden), torch.bfloat16, seed)
    weights, chosen = ops.route_top_k_cuda(dense.values((t, experts), torch.float32, seed + 1), top_k)
    order = torch.argsort(chosen.view(-1), stable=True)
    counts = torch.bincount(chosen.view(-1), minlength=experts)
    return x, weights.view(-1)[order], order // top_k, counts.cumsum(0).int(), counts.tolist()


@pytest.mark.parametrize("t", [1, 37, 400])
def test_experts_between_a_router_and_their_sum(t):
    """A block of 16-bit experts forward and backward, against float64; and the same experts in 8 bits."""
    hidden, inter, experts, top_k = 128, 96, 10, 2
    x, weights, token, off, counts = routed(t, hidden, experts, top_k, seed=t)
    gate_up, down = dense.values((experts, 2 * inter, hidden), torch.bfloat16, 5, hidden**-0.5), dense.values((experts, hidden, inter), torch.bfloat16, 6, inter**-0.5)

    def block(x, gate_up, down, product):
        rows = product(x[token], gate_up)
        h = torch.nn.functional.silu(rows[:, :inter].float()) * rows[:, inter:].float()
        y = product(h.to(x.dtype), down).float() * weights[:, None]
        return torch.zeros_like(x, dtype=torch.float32).index_add(0, token, y)

    leaves = [leaf(v) for v in (x, gate_up, down)]
    out = block(*leaves, lambda x, w: ops.grouped_gemm_cuda(x, w, off))
    grad = dense.values((t, hidden), torch.float32, 9)
    out.backward(grad)

    exact = [v.double().requires_grad_() for v in (x, gate_up, down)]
    rows = torch.cat([exact[0][token][lo:hi] @ exact[1][e].t() for e, lo, hi in dense.by_expert(counts)])
    h = torch.nn.functional.silu(rows[:, :inter]) * rows[:, inter:]
    y = torch.cat([h[lo:hi] @ exact[2][e].t() for e, lo, hi in dense.by_expert(counts)]) * weights[:, None].double()
    want = torch.zeros(t, hidden, dtype=torch.float64, device="cuda").index_add(0, token, y)
    want.backward(grad.double())

    # A chain of five bf16 roundings, each off by at most half a step (2^-8) of its value: relative to the whole tensor's
    # size their sum is below 6 * 2^-8.
    def off_by(got, ref):
        return ((got.double() - ref).norm() / ref.norm()).item()

    assert off_by(out, want) < 6 * 2.0**-8
    for got, ref in zip(leaves, exact):
        assert off_by(got.grad, ref.grad) < 6 * 2.0**-8

    # In 8 bits: weights and tokens are off by half a code's step each, amax / 254 of values whose root mean square is at
    # least amax / 6 for these rows of at most 128 normal values: 6 / 254 / sqrt(3) a factor, four factors in the block.
    def quantized(w):
        q, s = ops.quantize_rows_int8_cuda(w.reshape(-1, w.shape[2]))
        return q.view(w.shape), s.view(w.shape[:2])

    got = block(x, quantized(gate_up), quantized(down), lambda x, w: ops.grouped_gemm_int8_cuda(x, *w, off))
    assert off_by(got, want) < 4 * 6 / 254 / 3**0.5 + 6 * 2.0**-8


@pytest.mark.parametrize("m", [1, 3, 100])
def test_a_layer_of_8_bit_linears(m):
    """One quantization of a token for two projections, and the second linear on the first's output."""
    hidden, inter = 256, 192
    x = dense.values((m, hidden), torch.bfloat16, 1)
    w = [ops.quantize_rows_int8_cuda(dense.values(s, torch.float32, 2 + i, s[1] ** -0.5)) for i, s in enumerate(((inter, hidden), (inter, hidden), (hidden, inter)))]
    q, xs = ops.quantize_rows_int8_cuda(x)
    g, u = (ops.gemm_int8_cuda(q, xs, *v, torch.bfloat16) for v in w[:2])
    for y, v in ((g, w[0]), (u, w[1])):
        dense.within(y, *dense.int8_product(q, xs, *v))
        assert torch.equal(y, ops.gemm_int8_w8a8_cuda(x, *v))
    h = ops.silu_mul_cuda(torch.cat([g, u], dim=1))
    y = ops.gemm_int8_w8a8_cuda(h, *w[2])
    hq, hs = dense.quantize(h)
    dense.within(y, *dense.int8_product(hq.cuda(), hs.cuda(), *w[2]))


def test_a_training_step_captured():
    """Forward and both gradients in a graph, replayed over new rows and sizes with eager steps between."""
    counts, n, k = [40, 0, 60], 72, 64
    x, w, dy, off = parts(counts)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.grouped_gemm_cuda(a, b, off), (a, b), dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.grouped_gemm_cuda(a, b, off)
        da, db = torch.autograd.grad(y, (a, b), dy)
    for seed, new in enumerate(([40, 0, 60], [1, 99, 0], [0, 0, 100])):
        with torch.no_grad():
            a.copy_(dense.values(x.shape, x.dtype, 10 + seed))
        off.copy_(dense.offsets(new))
        graph.replay()
        fresh = a.detach().clone()
        want = ops.grouped_gemm_cuda(fresh, w, off), ops.grouped_gemm_grad_x_cuda(dy, w, off), ops.grouped_gemm_grad_w_cuda(dy, fresh, off)
        torch.cuda.synchronize()
        assert all(torch.equal(g, e) for g, e in zip((y, da, db), want)), new
