// linear over the pulsarlm_amd ops: the reference's dense/fp8 linear
// (pulsarlm-core/src/engine/model/linear.cpp:14-41) plus int4, MXFP4 and int8 alternatives.
// Quantized weights are repacked once, at construction, as the reference does.
#include "linear.hpp"

#include <utility>
#include <vector>

#include "pulsarlm_ops.hpp"

namespace pulsarlm {

linear::linear(std::variant<at::Tensor, quant_weight, mxfp4_weight, int8_weight> weight) : weight(std::move(weight)) {}

linear linear::dense(at::Tensor weight) { return linear(std::move(weight)); }

linear linear::fp8(const at::Tensor& weight, const at::Tensor& scale, std::int64_t block_n, std::int64_t group_size) {
    auto [w, s] = repack_fp8_marlin_cuda(weight, scale, block_n, group_size);
    return linear(quant_weight{std::move(w), std::move(s), weight.size(0), block_n, group_size, true});
}

linear linear::fp8_rows(const at::Tensor& weight, const at::Tensor& weight_scale_inv, std::int64_t block_n,
                        std::int64_t block_k, const at::Tensor& row_order) {
    TORCH_CHECK(row_order.dim() == 1 && row_order.size(0) == weight.size(0),
                "linear: row_order must hold one index per weight row");
    const at::Tensor order = row_order.to(weight.device(), at::kLong);
    const at::Tensor row_scale =
        weight_scale_inv.to(weight.device()).repeat_interleave(block_n, 0).narrow(0, 0, weight.size(0));
    const at::Tensor rows = weight.view(at::kByte).index_select(0, order).view(at::kFloat8_e4m3fn);
    return fp8(rows, row_scale.index_select(0, order).contiguous(), 1, block_k);
}

linear linear::int4(const at::Tensor& weight_packed, const at::Tensor& scale, std::int64_t block_n,
                    std::int64_t group_size) {
    auto [w, s] = repack_int4_marlin_cuda(weight_packed, scale, block_n, group_size);
    return linear(quant_weight{std::move(w), std::move(s), weight_packed.size(0), block_n, group_size, false});
}

linear linear::mxfp4(const at::Tensor& codes, const at::Tensor& scale, bool w4a4) {
    auto [w, s] = repack_mxfp4_cuda(codes, scale);
    return linear(mxfp4_weight{std::move(w), std::move(s), codes.size(0), w4a4});
}

linear linear::int8(const at::Tensor& codes, const at::Tensor& scale) {
    TORCH_CHECK(codes.scalar_type() == at::kChar && codes.dim() == 2 && scale.scalar_type() == at::kFloat && scale.numel() == codes.size(0),
                "linear: codes must be int8 [N, K] and scale fp32 [N]");
    return linear(int8_weight{codes.contiguous(), scale.reshape({-1}).contiguous()});
}

at::Tensor linear::apply(const at::Tensor& x) const {
    if (const auto* dense = std::get_if<at::Tensor>(&weight)) return at::linear(x, *dense);
    std::vector<std::int64_t> sizes = x.sizes().vec();
    const at::Tensor rows = x.reshape({-1, sizes.back()}).contiguous();
    if (const auto* mx = std::get_if<mxfp4_weight>(&weight)) {
        sizes.back() = mx->n;
        return (mx->w4a4 ? gemm_mxfp4_w4a4_cuda(rows, mx->weight, mx->scale, mx->n) : gemm_mxfp4_cuda(rows, mx->weight, mx->scale, mx->n))
            .view(sizes);
    }
    if (const auto* w8 = std::get_if<int8_weight>(&weight)) {
        sizes.back() = w8->codes.size(0);
        return gemm_int8_w8a8_cuda(rows, w8->codes, w8->scale).view(sizes);
    }
    const quant_weight& w = std::get<quant_weight>(weight);
    sizes.back() = w.n;
    const at::Tensor y = w.fp8 ? gemm_fp8_marlin_cuda(rows, w.weight_marlin, w.scale_marlin, w.n, w.block_n, w.group_size)
                               : gemm_int4_marlin_cuda(rows, w.weight_marlin, w.scale_marlin, w.n, w.block_n,
                                                       w.group_size);
    return y.view(sizes);
}

}  // namespace pulsarlm
