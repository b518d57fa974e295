// Implementation of pulsarlm_ops.hpp over the C ABI. Argument checks restate those of
// gemm<fmt> / repack<fmt> (pulsarlm-core/src/kernels/marlin.cu:395-445,538-576); the C
// ABI checks them again and reports anything it rejects through plm_last_error().
#include "pulsarlm_ops.hpp"

// PyTorch-ROCm tensors report device type "cuda"; the masquerading guard and stream
// accessors take that device type.
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <torch/csrc/autograd/custom_function.h>

#include <algorithm>
#include <functional>
#include <map>
#include <mutex>
#include <string>
#include <utility>

#include "pulsarlm_amd.h"

namespace pulsarlm {
namespace {

plm_dtype dtype_of(const char* op, at::ScalarType t) {
    switch (t) {
        case at::kBFloat16: return PLM_BF16;
        case at::kHalf: return PLM_FP16;
        case at::kFloat: return PLM_FP32;
        default: TORCH_CHECK(false, op, ": unsupported dtype ", t);
    }
}

void check_rc(int rc) {
    TORCH_CHECK(rc == PLM_OK, plm_last_error());
}

void* stream_of(const at::Tensor& t) {
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

std::vector<int64_t> scale_shape(int64_t n, int64_t k, int64_t block_n, int64_t group_size) {
    const int64_t strips = ceil_div(n, 16), ktiles = ceil_div(k, 128);
    return {strips, ceil_div(ktiles * 128, group_size), block_n % 16 == 0 ? 1 : 16};
}

// One zero-initialised workspace per (device, stream): the kernels leave the split-K
// counters at its front at zero, so calls ordered on one stream can share it.
std::mutex ws_mutex;
std::map<std::pair<int, void*>, at::Tensor> ws_cache;

at::Tensor workspace(const at::Tensor& like, int64_t bytes) {
    if (bytes <= 0) return at::Tensor();
    std::lock_guard<std::mutex> lock(ws_mutex);
    auto key = std::make_pair(static_cast<int>(like.device().index()), stream_of(like));
    auto it = ws_cache.find(key);
    if (it == ws_cache.end() || it->second.numel() < bytes) {
        at::Tensor buf = at::zeros({std::max<int64_t>(bytes, 1 << 20)}, like.options().dtype(at::kByte));
        ws_cache[key] = buf;
        return buf;
    }
    return it->second;
}

void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

std::tuple<at::Tensor, at::Tensor> repack(const char* op, plm_format fmt, const at::Tensor& weight, int64_t n,
                                          int64_t k, const at::Tensor& weight_scale, int64_t block_n,
                                          int64_t group_size) {
    TORCH_CHECK(weight.is_cuda() && weight_scale.is_cuda(), op, ": inputs must be CUDA tensors");
    TORCH_CHECK(block_n > 0, op, ": block_n must be positive");
    TORCH_CHECK(group_size > 0 && group_size % 16 == 0, op, ": group_size must be a positive multiple of 16");
    TORCH_CHECK(k % group_size == 0, op, ": K must be a multiple of group_size");
    TORCH_CHECK(weight_scale.dim() == 2 && weight_scale.size(0) == ceil_div(n, block_n) &&
                    weight_scale.size(1) == k / group_size,
                op, ": weight_scale must be [ceil(N / block_n), K / group_size]");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(weight.device());
    const at::Tensor src = weight.contiguous();
    const at::Tensor scale = weight_scale.contiguous();
    at::Tensor w = at::empty({plm_weight_bytes(fmt, n, k) / 4}, weight.options().dtype(at::kInt));
    at::Tensor s = at::empty(scale_shape(n, k, block_n, group_size), scale.options());
    const plm_dtype sd = dtype_of(op, scale.scalar_type());
    const int rc = fmt == PLM_INT4
                       ? plm_repack_int4(static_cast<const int32_t*>(src.data_ptr()), scale.data_ptr(), sd, n, k,
                                         block_n, group_size, w.data_ptr(), s.data_ptr(), stream_of(weight))
                       : plm_repack_fp8(static_cast<const uint8_t*>(src.data_ptr()), scale.data_ptr(), sd, n, k,
                                        block_n, group_size, w.data_ptr(), s.data_ptr(), stream_of(weight));
    check_rc(rc);
    return {w, s};
}

void gemm_checks(const char* op, plm_format fmt, const at::Tensor& x, const at::Tensor& weight_marlin,
                 const at::Tensor& scale_marlin, int64_t n, int64_t block_n, int64_t group_size) {
    TORCH_CHECK(x.is_cuda() && weight_marlin.is_cuda() && scale_marlin.is_cuda(), op,
                ": all inputs must be CUDA tensors");
    TORCH_CHECK(x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16, op, ": x must be fp16 or bf16");
    TORCH_CHECK(x.dim() == 2 && x.is_contiguous(), op, ": x must be a contiguous [M, K]");
    TORCH_CHECK(weight_marlin.scalar_type() == at::kInt, op, ": weight_marlin must be int32");
    TORCH_CHECK(block_n > 0, op, ": block_n must be positive");
    TORCH_CHECK(group_size > 0 && group_size % 16 == 0, op, ": group_size must be a positive multiple of 16");
    const int64_t k = x.size(1);
    TORCH_CHECK(k % group_size == 0, op, ": K must be a multiple of group_size");
    TORCH_CHECK(scale_marlin.sizes().vec() == scale_shape(n, k, block_n, group_size), op,
                ": scale_marlin has the wrong shape for this N, K, block_n and group_size");
    TORCH_CHECK(weight_marlin.numel() * 4 == plm_weight_bytes(fmt, n, k), op,
                ": weight_marlin has the wrong size for this shape");
}

at::Tensor gemm(const char* op, plm_format fmt, bool w8a8, const at::Tensor& x, const at::Tensor& weight_marlin,
                const at::Tensor& scale_marlin, int64_t n, int64_t block_n, int64_t group_size) {
    gemm_checks(op, fmt, x, weight_marlin, scale_marlin, n, block_n, group_size);
    at::Tensor y = at::empty({x.size(0), n}, x.options());
    if (x.size(0) == 0 || n == 0) return y;
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    const int64_t m = x.size(0), k = x.size(1);
    const at::Tensor w = weight_marlin.contiguous(), s = scale_marlin.contiguous();
    const plm_dtype sd = dtype_of(op, s.scalar_type());
    const plm_dtype xd = dtype_of(op, x.scalar_type());
    if (w8a8) {
        at::Tensor ws = workspace(x, plm_gemm_w8a8_workspace_bytes(m, n, k));
        check_rc(plm_gemm_w8a8(x.data_ptr(), xd, w.data_ptr(), s.data_ptr(), sd, m, n, k, block_n, group_size,
                               y.data_ptr(), ptr(ws), ws.defined() ? ws.numel() : 0, stream_of(x)));
    } else {
        at::Tensor ws = workspace(x, plm_gemm_workspace_bytes(fmt, m, n, k));
        check_rc(plm_gemm(fmt, x.data_ptr(), xd, w.data_ptr(), s.data_ptr(), sd, m, n, k, block_n, group_size,
                          y.data_ptr(), ptr(ws), ws.defined() ? ws.numel() : 0, stream_of(x)));
    }
    return y;
}

}  // namespace

std::tuple<at::Tensor, at::Tensor> repack_int4_marlin_cuda(const at::Tensor& weight_packed,
                                                           const at::Tensor& weight_scale, int64_t block_n,
                                                           int64_t group_size) {
    TORCH_CHECK(weight_packed.scalar_type() == at::kInt && weight_packed.dim() == 2,
                "repack_int4_marlin: weight_packed must be int32 [N, K/8]");
    return repack("repack_int4_marlin", PLM_INT4, weight_packed, weight_packed.size(0), weight_packed.size(1) * 8,
                  weight_scale, block_n, group_size);
}

std::tuple<at::Tensor, at::Tensor> repack_fp8_marlin_cuda(const at::Tensor& weight, const at::Tensor& weight_scale,
                                                          int64_t block_n, int64_t group_size) {
    TORCH_CHECK(weight.scalar_type() == at::kFloat8_e4m3fn && weight.dim() == 2,
                "repack_fp8_marlin: weight must be float8_e4m3fn [N, K]");
    return repack("repack_fp8_marlin", PLM_FP8, weight, weight.size(0), weight.size(1), weight_scale, block_n,
                  group_size);
}

at::Tensor gemm_int4_marlin_cuda(const at::Tensor& x, const at::Tensor& weight_marlin, const at::Tensor& scale_marlin,
                                 int64_t n, int64_t block_n, int64_t group_size) {
    return gemm("gemm_int4_marlin", PLM_INT4, false, x, weight_marlin, scale_marlin, n, block_n, group_size);
}

at::Tensor gemm_fp8_marlin_cuda(const at::Tensor& x, const at::Tensor& weight_marlin, const at::Tensor& scale_marlin,
                                int64_t n, int64_t block_n, int64_t group_size) {
    return gemm("gemm_fp8_marlin", PLM_FP8, false, x, weight_marlin, scale_marlin, n, block_n, group_size);
}

at::Tensor gemm_fp8_w8a8_cuda(const at::Tensor& x, const at::Tensor& weight_marlin, const at::Tensor& scale_marlin,
                              int64_t n, int64_t block_n, int64_t group_size) {
    TORCH_CHECK(group_size % 128 == 0, "gemm_fp8_w8a8: group_size must be a multiple of 128 for the fp8 MFMA");
    return gemm("gemm_fp8_w8a8", PLM_FP8, true, x, weight_marlin, scale_marlin, n, block_n, group_size);
}

std::tuple<at::Tensor, at::Tensor> quantize_rows_e4m3_cuda(const at::Tensor& x) {
    const char* op = "quantize_rows_e4m3";
    TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.is_contiguous(), op, ": x must be a contiguous CUDA [M, K]");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    at::Tensor codes = at::empty({x.size(0), x.size(1)}, x.options().dtype(at::kByte));
    at::Tensor scale = at::empty({x.size(0)}, x.options().dtype(at::kFloat));
    check_rc(plm_quantize_rows_e4m3(x.data_ptr(), dtype_of(op, x.scalar_type()), x.size(0), x.size(1),
                                    static_cast<uint8_t*>(codes.data_ptr()), static_cast<float*>(scale.data_ptr()),
                                    stream_of(x)));
    return {codes, scale};
}

std::tuple<at::Tensor, at::Tensor> convert_marlin_cuda(const std::string& format, const at::Tensor& weight_marlin,
                                                       const at::Tensor& scale_marlin, int64_t n, int64_t k,
                                                       int64_t block_n, int64_t group_size) {
    const char* op = "convert_marlin";
    TORCH_CHECK(format == "int4" || format == "fp8", op, ": format must be int4 or fp8");
    TORCH_CHECK(weight_marlin.scalar_type() == at::kInt && scale_marlin.scalar_type() == at::kFloat, op,
                ": weight_marlin must be int32 and scale_marlin fp32");
    const plm_format fmt = format == "int4" ? PLM_INT4 : PLM_FP8;
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(weight_marlin.device());
    at::Tensor w = at::empty({plm_weight_bytes(fmt, n, k) / 4}, weight_marlin.options());
    at::Tensor s = at::empty(scale_shape(n, k, block_n, group_size), scale_marlin.options());
    const at::Tensor wm = weight_marlin.contiguous(), sm = scale_marlin.contiguous();
    check_rc(plm_convert_marlin(fmt, static_cast<const int32_t*>(wm.data_ptr()), static_cast<const float*>(sm.data_ptr()),
                                n, k, block_n, group_size, w.data_ptr(), s.data_ptr(), stream_of(weight_marlin)));
    return {w, s};
}

at::Tensor dequant_marlin_cuda(const std::string& format, const at::Tensor& weight_marlin,
                               const at::Tensor& scale_marlin, int64_t n, int64_t k, int64_t block_n,
                               int64_t group_size, at::ScalarType dtype) {
    const char* op = "dequant";
    TORCH_CHECK(format == "int4" || format == "fp8", op, ": format must be int4 or fp8");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(weight_marlin.device());
    at::Tensor out = at::empty({n, k}, weight_marlin.options().dtype(dtype));
    check_rc(plm_dequant(format == "int4" ? PLM_INT4 : PLM_FP8, weight_marlin.data_ptr(), scale_marlin.data_ptr(),
                         dtype_of(op, scale_marlin.scalar_type()), n, k, block_n, group_size, out.data_ptr(),
                         dtype_of(op, dtype), stream_of(weight_marlin)));
    return out;
}

std::tuple<at::Tensor, at::Tensor> repack_int4_experts_cuda(const at::Tensor& weight_packed,
                                                            const at::Tensor& weight_scale, int64_t group_size) {
    TORCH_CHECK(weight_packed.dim() == 3 && weight_scale.dim() == 3,
                "repack_int4_experts: expected [E, N, K/8] weights and [E, N, K/g] scales");
    std::vector<at::Tensor> ws, ss;
    for (int64_t e = 0; e < weight_packed.size(0); ++e) {
        auto [w, s] = repack_int4_marlin_cuda(weight_packed[e], weight_scale[e], 1, group_size);
        ws.push_back(w);
        ss.push_back(s);
    }
    return {at::cat(ws), at::stack(ss)};
}

at::Tensor grouped_gemm_int4_cuda(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& scale,
                                  const at::Tensor& offsets, int64_t n, int64_t group_size) {
    const char* op = "grouped_gemm";
    TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.is_contiguous(), op, ": x must be a contiguous CUDA [rows, K]");
    TORCH_CHECK(offsets.scalar_type() == at::kInt && offsets.dim() == 1, op, ": offsets must be int32 [E]");
    const int64_t rows = x.size(0), k = x.size(1), e = offsets.size(0);
    TORCH_CHECK(weight.numel() * 4 == e * plm_weight_bytes(PLM_INT4, n, k), op, ": weight has the wrong size");
    at::Tensor y = at::empty({rows, n}, x.options());
    if (rows == 0 || n == 0) return y;
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    at::Tensor ws = workspace(x, plm_grouped_gemm_workspace_bytes(rows, e));
    const at::Tensor off = offsets.contiguous();
    check_rc(plm_grouped_gemm(PLM_INT4, x.data_ptr(), dtype_of(op, x.scalar_type()), weight.data_ptr(),
                              scale.data_ptr(), dtype_of(op, scale.scalar_type()),
                              static_cast<const int32_t*>(off.data_ptr()), e, rows, n, k, 1, group_size, y.data_ptr(),
                              ptr(ws), ws.numel(), stream_of(x)));
    return y;
}

std::tuple<at::Tensor, at::Tensor> routed_experts_int4_cuda(const at::Tensor& h, const at::Tensor& top_experts,
                                                            const at::Tensor& top_weights,
                                                            const at::Tensor& gate_up_weight,
                                                            const at::Tensor& gate_up_scale,
                                                            const at::Tensor& down_weight,
                                                            const at::Tensor& down_scale, int64_t intermediate,
                                                            int64_t group_size) {
    const char* op = "routed_experts";
    TORCH_CHECK(h.is_cuda() && h.dim() == 2, op, ": h must be a CUDA [T, H] tensor");
    TORCH_CHECK(top_experts.sizes() == top_weights.sizes() && top_experts.dim() == 2, op,
                ": top_experts and top_weights must be [T, top_k]");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(h.device());
    const int64_t t = h.size(0), hidden = h.size(1), top_k = top_experts.size(1), e = gate_up_scale.size(0);
    const at::Tensor hc = h.contiguous();
    const at::Tensor experts = top_experts.to(at::kInt).contiguous();
    const at::Tensor weights = top_weights.to(at::kFloat).contiguous();
    at::Tensor out = at::empty_like(hc);
    at::Tensor offsets = at::empty({e}, h.options().dtype(at::kInt));
    at::Tensor ws = workspace(h, plm_moe_workspace_bytes(t, top_k, e, hidden, intermediate));
    check_rc(plm_moe(hc.data_ptr(), dtype_of(op, h.scalar_type()), static_cast<const int32_t*>(experts.data_ptr()),
                     static_cast<const float*>(weights.data_ptr()), t, top_k, e, hidden, intermediate,
                     gate_up_weight.data_ptr(), gate_up_scale.data_ptr(), down_weight.data_ptr(),
                     down_scale.data_ptr(), dtype_of(op, gate_up_scale.scalar_type()), group_size,
                     static_cast<int32_t*>(offsets.data_ptr()), out.data_ptr(), ptr(ws), ws.defined() ? ws.numel() : 0,
                     stream_of(h)));
    return {out, offsets};
}

std::tuple<at::Tensor, at::Tensor> route_top_k_cuda(const at::Tensor& logits, int64_t k) {
    const char* op = "route_top_k";
    TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.stride(1) == 1, op,
                ": logits must be CUDA [tokens, experts], each row contiguous");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(logits.device());
    const int64_t tokens = logits.size(0), experts = logits.size(1);
    at::Tensor weights = at::empty({tokens, k}, logits.options().dtype(at::kFloat));
    at::Tensor chosen = at::empty({tokens, k}, logits.options().dtype(at::kLong));
    check_rc(plm_route_top_k(logits.data_ptr(), dtype_of(op, logits.scalar_type()), tokens, experts,
                             tokens > 1 ? logits.stride(0) : experts, k, static_cast<float*>(weights.data_ptr()),
                             static_cast<int64_t*>(chosen.data_ptr()), nullptr, stream_of(logits)));
    return {weights, chosen};
}

at::Tensor silu_mul_cuda(const at::Tensor& x) {
    const char* op = "silu_mul";
    TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.is_contiguous() && x.size(1) % 2 == 0, op,
                ": x must be contiguous CUDA [tokens, 2 * n]");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    const int64_t tokens = x.size(0), n = x.size(1) / 2;
    at::Tensor y = at::empty({tokens, n}, x.options());
    check_rc(plm_silu_mul(x.data_ptr(), dtype_of(op, x.scalar_type()), tokens, n, y.data_ptr(), stream_of(x)));
    return y;
}

namespace {
at::Tensor gemm_int4_plain(const char* op, const at::Tensor& x, const at::Tensor& weight_packed,
                           const at::Tensor& weight_scale, int64_t group_size, int64_t num_splits) {
    TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.is_contiguous(), op, ": x must be a contiguous CUDA [M, K] tensor");
    TORCH_CHECK(weight_packed.is_cuda() && weight_packed.scalar_type() == at::kInt && weight_packed.dim() == 2 &&
                    weight_packed.is_contiguous(),
                op, ": weight_packed must be contiguous CUDA int32 [N, K/8]");
    const int64_t m = x.size(0), k = x.size(1), n = weight_packed.size(0);
    TORCH_CHECK(weight_packed.size(1) * 8 == k, op, ": weight_packed must be [N, K/8]");
    TORCH_CHECK(group_size > 0 && weight_scale.dim() == 2 && weight_scale.size(0) == n &&
                    weight_scale.size(1) * group_size == k,
                op, ": weight_scale must be [N, K/group_size]");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    const at::Tensor scale = weight_scale.to(at::kFloat).contiguous();
    at::Tensor y = at::empty({m, n}, x.options());
    const int64_t nbytes = plm_gemm_int4_plain_workspace_bytes(m, n, k, num_splits);
    at::Tensor ws = nbytes > 0 ? at::empty({nbytes}, x.options().dtype(at::kByte)) : at::Tensor();
    check_rc(plm_gemm_int4_plain(x.data_ptr(), dtype_of(op, x.scalar_type()),
                                 static_cast<const int32_t*>(weight_packed.data_ptr()),
                                 static_cast<const float*>(scale.data_ptr()), m, n, k, group_size, num_splits,
                                 y.data_ptr(), ptr(ws), ws.defined() ? ws.numel() : 0, stream_of(x)));
    return y;
}
}  // namespace

at::Tensor gemm_int4_cuda(const at::Tensor& x, const at::Tensor& weight_packed, const at::Tensor& weight_scale,
                          int64_t group_size) {
    return gemm_int4_plain("gemm_int4", x, weight_packed, weight_scale, group_size, 0);
}

at::Tensor gemm_int4_split_cuda(const at::Tensor& x, const at::Tensor& weight_packed,
                                const at::Tensor& weight_scale, int64_t group_size, int64_t num_splits) {
    TORCH_CHECK(num_splits >= 1, "gemm_int4: num_splits must be >= 1");
    return gemm_int4_plain("gemm_int4", x, weight_packed, weight_scale, group_size, num_splits);
}

namespace {

void mx_rows(const char* op, const char* name, const at::Tensor& x) {
    TORCH_CHECK(x.is_cuda() && (x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16), op, ": ", name,
                " must be a CUDA fp16 or bf16 tensor");
    TORCH_CHECK(x.dim() == 2 && x.is_contiguous(), op, ": ", name, " must be contiguous [rows, columns]");
}

std::pair<int64_t, int64_t> mx_plain(const char* op, const at::Tensor& codes, const at::Tensor& scale) {
    TORCH_CHECK(codes.is_cuda() && scale.is_cuda() && codes.device() == scale.device(), op,
                ": codes and scale must be on one CUDA device");
    TORCH_CHECK(codes.scalar_type() == at::kByte && scale.scalar_type() == at::kByte && codes.dim() == 2 && scale.dim() == 2, op,
                ": codes must be uint8 [N, K/2] and scale uint8 [N, K/32]");
    const int64_t n = codes.size(0), k = 2 * codes.size(1);
    TORCH_CHECK(k % 32 == 0, op, ": K must be a multiple of 32");
    TORCH_CHECK(scale.size(0) == n && scale.size(1) == k / 32, op, ": scale must be [N, K/32]");
    return {n, k};
}

std::vector<int64_t> mx_scale_shape(int64_t n, int64_t k) { return {ceil_div(n, 64), ceil_div(k, 128), 64}; }

void mx_weight(const char* op, const at::Tensor& x, const at::Tensor& weight, const at::Tensor& scale, int64_t n, int64_t k) {
    TORCH_CHECK(n >= 0 && k >= 0, op, ": sizes must be non-negative");
    TORCH_CHECK(weight.device() == x.device() && scale.device() == x.device(), op, ": x and the weights must be on one device");
    TORCH_CHECK(weight.scalar_type() == at::kInt && scale.scalar_type() == at::kInt && weight.is_contiguous() && scale.is_contiguous(),
                op, ": weight and scale must be contiguous int32, as repack_mxfp4 returns them");
    TORCH_CHECK(weight.numel() * 4 == plm_mxfp4_weight_bytes(n, k), op, ": weight has the wrong size for this shape");
    TORCH_CHECK(scale.sizes().vec() == mx_scale_shape(n, k), op, ": scale has the wrong shape for this N and K");
}

// Scratch of one call, from the caching allocator: a captured call's belongs to its graph.
at::Tensor mx_scratch(const at::Tensor& x, int64_t bytes) {
    return bytes > 0 ? at::empty({bytes}, x.options().dtype(at::kByte)) : at::Tensor();
}
size_t mx_bytes(const at::Tensor& t) { return t.defined() ? static_cast<size_t>(t.numel()) : 0; }

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool mx_records(const at::Tensor& x) { return x.requires_grad() && at::GradMode::is_enabled(); }

struct mx_linear : torch::autograd::Function<mx_linear> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight, const at::Tensor& scale, int64_t n) {
        at::Tensor y = gemm_mxfp4_cuda(x, weight, scale, n);
        ctx->save_for_backward({weight, scale});
        ctx->saved_data["k"] = x.size(1);
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list dy) {
        const variable_list w = ctx->get_saved_variables();
        return {gemm_mxfp4_grad_cuda(dy[0].contiguous(), w[0], w[1], ctx->saved_data["k"].toInt()), {}, {}, {}};
    }
};

struct mx_gated : torch::autograd::Function<mx_gated> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& gate_weight, const at::Tensor& gate_scale,
                                 const at::Tensor& up_weight, const at::Tensor& up_scale, int64_t intermediate) {
        auto [h, gate_up] = gated_mxfp4_cuda(x, gate_weight, gate_scale, up_weight, up_scale, intermediate, true);
        ctx->mark_non_differentiable({gate_up});
        ctx->set_materialize_grads(false);  // no zeros for gate_up's
        ctx->save_for_backward({gate_up, gate_weight, gate_scale, up_weight, up_scale});
        ctx->saved_data["k"] = x.size(1);
        return {h, gate_up};
    }
    static variable_list backward(AutogradContext* ctx, variable_list dh) {
        if (!dh[0].defined()) return variable_list(6);
        const variable_list w = ctx->get_saved_variables();
        return {gated_mxfp4_grad_cuda(dh[0].contiguous(), w[0], w[1], w[2], w[3], w[4], ctx->saved_data["k"].toInt()), {}, {}, {}, {}, {}};
    }
};

// call(): an output in the graph of its two inputs (or one, twice) whose gradient is asked for in vain, and says so then.
struct mx_no_gradient : torch::autograd::Function<mx_no_gradient> {
    static at::Tensor forward(AutogradContext* ctx, const char* op, const std::function<at::Tensor()>& call, const at::Tensor&,
                              const at::Tensor&) {
        ctx->saved_data["op"] = std::string(op);
        return call();
    }
    static variable_list backward(AutogradContext* ctx, const variable_list&) {
        TORCH_CHECK(false, ctx->saved_data["op"].toStringRef(), ": has no gradient");
    }
};

}  // namespace

std::tuple<at::Tensor, at::Tensor> quantize_mxfp4_cuda(const at::Tensor& x) {
    const char* op = "quantize_mxfp4";
    TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.is_contiguous(), op, ": x must be a contiguous CUDA [M, K]");
    TORCH_CHECK(x.size(1) % 32 == 0, op, ": K must be a multiple of 32");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    at::Tensor codes = at::empty({x.size(0), x.size(1) / 2}, x.options().dtype(at::kByte));
    at::Tensor scale = at::empty({x.size(0), x.size(1) / 32}, x.options().dtype(at::kByte));
    check_rc(plm_quantize_mxfp4(x.data_ptr(), dtype_of(op, x.scalar_type()), x.size(0), x.size(1),
                                static_cast<uint8_t*>(codes.data_ptr()), static_cast<uint8_t*>(scale.data_ptr()), stream_of(x)));
    return {codes, scale};
}

at::Tensor dequantize_mxfp4_cuda(const at::Tensor& codes, const at::Tensor& scale, at::ScalarType dtype) {
    const char* op = "dequantize_mxfp4";
    const auto [m, k] = mx_plain(op, codes, scale);
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(codes.device());
    const at::Tensor c = codes.contiguous(), s = scale.contiguous();
    at::Tensor out = at::empty({m, k}, codes.options().dtype(dtype));
    check_rc(plm_dequantize_mxfp4(static_cast<const uint8_t*>(c.data_ptr()), static_cast<const uint8_t*>(s.data_ptr()), m, k,
                                  out.data_ptr(), dtype_of(op, dtype), stream_of(codes)));
    return out;
}

std::tuple<at::Tensor, at::Tensor> repack_mxfp4_cuda(const at::Tensor& codes, const at::Tensor& scale) {
    const auto [n, k] = mx_plain("repack_mxfp4", codes, scale);
    TORCH_CHECK(std::max(n, k) <= int64_t{1} << 19, "repack_mxfp4: N and K must be at most 2^19");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(codes.device());
    const at::Tensor c = codes.contiguous(), s = scale.contiguous();
    at::Tensor weight = at::empty({plm_mxfp4_weight_bytes(n, k) / 4}, codes.options().dtype(at::kInt));
    at::Tensor packed = at::empty(mx_scale_shape(n, k), codes.options().dtype(at::kInt));
    check_rc(plm_repack_mxfp4(static_cast<const uint8_t*>(c.data_ptr()), static_cast<const uint8_t*>(s.data_ptr()), n, k,
                              weight.data_ptr(), packed.data_ptr(), stream_of(codes)));
    return {weight, packed};
}

at::Tensor gemm_mxfp4_cuda(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& scale, int64_t n) {
    const char* op = "gemm_mxfp4";
    if (mx_records(x)) return mx_linear::apply(x, weight, scale, n);
    mx_rows(op, "x", x);
    mx_weight(op, x, weight, scale, n, x.size(1));
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    at::Tensor y = at::empty({x.size(0), n}, x.options());
    check_rc(plm_gemm_mxfp4(x.data_ptr(), dtype_of(op, x.scalar_type()), weight.data_ptr(), scale.data_ptr(), x.size(0), n, x.size(1),
                            y.data_ptr(), stream_of(x)));
    return y;
}

at::Tensor gemm_mxfp4_w4a4_cuda(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& scale, int64_t n) {
    const char* op = "gemm_mxfp4_w4a4";
    if (mx_records(x)) return mx_no_gradient::apply(op, [&] { return gemm_mxfp4_w4a4_cuda(x, weight, scale, n); }, x, x);
    mx_rows(op, "x", x);
    mx_weight(op, x, weight, scale, n, x.size(1));
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    at::Tensor y = at::empty({x.size(0), n}, x.options());
    const at::Tensor ws = mx_scratch(x, plm_gemm_mxfp4_w4a4_workspace_bytes(x.size(0), n, x.size(1)));
    check_rc(plm_gemm_mxfp4_w4a4(x.data_ptr(), dtype_of(op, x.scalar_type()), weight.data_ptr(), scale.data_ptr(), x.size(0), n,
                                 x.size(1), y.data_ptr(), ptr(ws), mx_bytes(ws), stream_of(x)));
    return y;
}

at::Tensor gemm_mxfp4_grad_cuda(const at::Tensor& dy, const at::Tensor& weight, const at::Tensor& scale, int64_t k) {
    const char* op = "gemm_mxfp4_grad";
    if (mx_records(dy)) return mx_no_gradient::apply(op, [&] { return gemm_mxfp4_grad_cuda(dy, weight, scale, k); }, dy, dy);
    mx_rows(op, "dy", dy);
    mx_weight(op, dy, weight, scale, dy.size(1), k);
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(dy.device());
    at::Tensor dx = at::empty({dy.size(0), k}, dy.options());
    const auto bytes = reinterpret_cast<uintptr_t>(dy.data_ptr()) % 16 == 0 ? plm_gemm_mxfp4_grad_aligned_workspace_bytes
                                                                            : plm_gemm_mxfp4_grad_workspace_bytes;
    const at::Tensor ws = mx_scratch(dy, bytes(dy.size(0), dy.size(1), k));
    check_rc(plm_gemm_mxfp4_grad(dy.data_ptr(), dtype_of(op, dy.scalar_type()), weight.data_ptr(), scale.data_ptr(), dy.size(0),
                                 dy.size(1), k, dx.data_ptr(), ptr(ws), mx_bytes(ws), stream_of(dy)));
    return dx;
}

std::tuple<at::Tensor, at::Tensor> gated_mxfp4_cuda(const at::Tensor& x, const at::Tensor& gate_weight, const at::Tensor& gate_scale,
                                                    const at::Tensor& up_weight, const at::Tensor& up_scale,
                                                    int64_t intermediate, bool keep_gate_up) {
    const char* op = "gated_mxfp4";
    if (mx_records(x)) {
        const variable_list out = mx_gated::apply(x, gate_weight, gate_scale, up_weight, up_scale, intermediate);
        return {out[0], keep_gate_up ? out[1] : at::Tensor()};
    }
    mx_rows(op, "x", x);
    mx_weight(op, x, gate_weight, gate_scale, intermediate, x.size(1));
    mx_weight(op, x, up_weight, up_scale, intermediate, x.size(1));
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    at::Tensor h = at::empty({x.size(0), intermediate}, x.options());
    at::Tensor gate_up = keep_gate_up ? at::empty({x.size(0), 2 * intermediate}, x.options().dtype(at::kFloat)) : at::Tensor();
    check_rc(plm_gated_mxfp4(x.data_ptr(), dtype_of(op, x.scalar_type()), gate_weight.data_ptr(), gate_scale.data_ptr(),
                             up_weight.data_ptr(), up_scale.data_ptr(), x.size(0), intermediate, x.size(1), h.data_ptr(),
                             static_cast<float*>(ptr(gate_up)), stream_of(x)));
    return {h, gate_up};
}

at::Tensor gated_mxfp4_grad_cuda(const at::Tensor& dh, const at::Tensor& gate_up, const at::Tensor& gate_weight,
                                 const at::Tensor& gate_scale, const at::Tensor& up_weight, const at::Tensor& up_scale,
                                 int64_t hidden) {
    const char* op = "gated_mxfp4_grad";
    if (mx_records(dh) || mx_records(gate_up))
        return mx_no_gradient::apply(
            op, [&] { return gated_mxfp4_grad_cuda(dh, gate_up, gate_weight, gate_scale, up_weight, up_scale, hidden); }, dh, gate_up);
    mx_rows(op, "dh", dh);
    const int64_t m = dh.size(0), n = dh.size(1);
    TORCH_CHECK(gate_up.scalar_type() == at::kFloat && gate_up.device() == dh.device() && gate_up.dim() == 2 && gate_up.size(0) == m &&
                    gate_up.size(1) == 2 * n && gate_up.is_contiguous(),
                op, ": gate_up must be contiguous fp32 [M, 2 I] on dh's device");
    mx_weight(op, dh, gate_weight, gate_scale, n, hidden);
    mx_weight(op, dh, up_weight, up_scale, n, hidden);
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(dh.device());
    at::Tensor dx = at::empty({m, hidden}, dh.options());
    const at::Tensor ws = mx_scratch(dh, plm_gated_mxfp4_grad_workspace_bytes(m, n, hidden));
    check_rc(plm_gated_mxfp4_grad(dh.data_ptr(), static_cast<const float*>(gate_up.data_ptr()), dtype_of(op, dh.scalar_type()),
                                  gate_weight.data_ptr(), gate_scale.data_ptr(), up_weight.data_ptr(), up_scale.data_ptr(), m, n, hidden,
                                  dx.data_ptr(), ptr(ws), mx_bytes(ws), stream_of(dh)));
    return dx;
}

at::Tensor mlp_mxfp4_w4a4_cuda(const at::Tensor& x, const at::Tensor& gate_weight, const at::Tensor& gate_scale,
                               const at::Tensor& up_weight, const at::Tensor& up_scale, const at::Tensor& down_weight,
                               const at::Tensor& down_scale, int64_t intermediate) {
    const char* op = "mlp_mxfp4_w4a4";
    if (mx_records(x))
        return mx_no_gradient::apply(
            op,
            [&] { return mlp_mxfp4_w4a4_cuda(x, gate_weight, gate_scale, up_weight, up_scale, down_weight, down_scale, intermediate); }, x,
            x);
    mx_rows(op, "x", x);
    const int64_t m = x.size(0), k = x.size(1);
    mx_weight(op, x, gate_weight, gate_scale, intermediate, k);
    mx_weight(op, x, up_weight, up_scale, intermediate, k);
    mx_weight(op, x, down_weight, down_scale, k, intermediate);
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    at::Tensor y = at::empty({m, k}, x.options());
    const at::Tensor ws = mx_scratch(x, plm_mlp_mxfp4_w4a4_workspace_bytes(m, intermediate, k));
    check_rc(plm_mlp_mxfp4_w4a4(x.data_ptr(), dtype_of(op, x.scalar_type()), gate_weight.data_ptr(), gate_scale.data_ptr(),
                                up_weight.data_ptr(), up_scale.data_ptr(), down_weight.data_ptr(), down_scale.data_ptr(), m,
                                intermediate, k, y.data_ptr(), ptr(ws), mx_bytes(ws), stream_of(x)));
    return y;
}

}  // namespace pulsarlm
