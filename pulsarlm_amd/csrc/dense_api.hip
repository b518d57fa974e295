// C entry points of the products on unpacked weights: 8-bit integers with scales for each token and channel, 16-bit
// experts and their gradients. Argument checks, the workspace of tokens quantized on the way, and the choice between the
// kernel for few rows and the tiles.
#include "dense_gemm.hpp"

namespace plm {

int zero_output(const char* op, void* y, int64_t m, int64_t n, hipStream_t s);
void launch_dequantize_int8(const int8_t* codes, const float* scale, int64_t m, int64_t k, void* out, plm_dtype dtype, hipStream_t s);

namespace {

bool sixteen(plm_dtype t) { return t == PLM_BF16 || t == PLM_FP16; }

// These keep offsets of one workgroup below kOOB, and the numbers of 64 x 64 tiles within 31 bits.
bool takes_rows(int64_t rows, int64_t n, int64_t k) { return rows <= kDenseMaxRows && rows * std::max(n, k) <= (int64_t{1} << 36); }
int check_sizes(const char* op, const char* m, int64_t rows, int64_t n, int64_t k) {
    PLM_CHECK_ARG(rows >= 0 && n >= 0 && k >= 0, op, "sizes must be non-negative");
    PLM_CHECK_ARG(n <= kDenseMaxSize && k <= kDenseMaxSize, op, "N and K must be at most 2^19");
    PLM_CHECK_ARG(takes_rows(rows, n, k), op, "%s must be below 2^24, %s N and %s K at most 2^36", m, m, m);
    return PLM_OK;
}
// What a workspace query counts: sizes that a call takes, and works on.
bool counts(int64_t m, int64_t n, int64_t k) { return m > 0 && n > 0 && k > 0 && k <= kInt8MaxK && n <= kDenseMaxSize && takes_rows(m, n, k); }
int check_int8(const char* op, int64_t k) {
    PLM_CHECK_ARG(k % 16 == 0, op, "K must be a multiple of 16");
    PLM_CHECK_ARG(k <= kInt8MaxK, op, "K must be at most 131056");
    return PLM_OK;
}
int check_experts(const char* op, int64_t experts, int64_t n, int64_t k) {
    PLM_CHECK_ARG(experts > 0 && experts <= kMaxExperts, op, "n_experts must be in [1, 4096]");
    PLM_CHECK_ARG(experts * n * k <= int64_t{1} << 38 && experts * std::max(n, k) <= int64_t{1} << 28, op,
                  "n_experts N K must be at most 2^38, n_experts N and n_experts K at most 2^28");
    return PLM_OK;
}
int check_offsets(const char* op, const int32_t* offsets) {
    PLM_CHECK_ARG(offsets != nullptr && aligned(offsets, 4), op, "offsets must be a 4-byte aligned pointer");
    return PLM_OK;
}
int check_pointer(const char* op, const char* name, const void* p, size_t align, bool used = true) {
    if (!used) return PLM_OK;
    PLM_CHECK_ARG(p != nullptr, op, "null pointer");
    PLM_CHECK_ARG(aligned(p, align), op, "%s must be %zu-byte aligned", name, align);
    return PLM_OK;
}

dense_product product(dense_type type, const void* p, const void* q, void* y, bool bf16, int64_t rows, int64_t cols, int64_t depth) {
    dense_product d{};
    d.type = type;
    d.p = p, d.q = q, d.y = y;
    d.bf16 = bf16;
    d.rows = rows, d.cols = cols, d.depth = depth;
    d.experts = 1;
    return d;
}
// The dense 8-bit product, and the workspace of a split sum's parts.
int64_t partial_bytes(int64_t m, int64_t n, int64_t k, bool to_quantize = false) {
    dense_product p = product(kInt8, nullptr, nullptr, nullptr, true, m, n, k);
    p.to_quantize = to_quantize;
    return dense_partial_bytes(plan_dense(p, kDense, true, true), m, n);
}
// p.plan is set.
void run_int8(dense_product p, void* partial, hipStream_t s) {
    if (p.plan.rows_block > 0) return launch_dense_rows(p, kDense, s);
    p.partial = static_cast<i32x4_t*>(partial);
    launch_tiles_int8(p, kDense, s);
    if (p.plan.splits > 1) launch_combine_int8(p, s);
}

// 16-bit experts, forward.
int run_experts(const char* op, dense_product p, const int32_t* offsets, int64_t experts, int zero_rest, hipStream_t s) {
    p.offsets = offsets, p.experts = experts, p.zero_rest = zero_rest != 0;
    p.plan = plan_dense(p, kByRows, true, false);
    if (p.plan.rows_block > 0) launch_dense_rows(p, kByRows, s);
    else launch_tiles_16(p, s);
    PLM_HIP_LAUNCH_CHECK(op);
    return PLM_OK;
}

// Tokens quantized on the way: [codes][scales] in a workspace.
int64_t codes_bytes(int64_t m, int64_t k) { return round_up(m * k, 256); }
int64_t tokens_bytes(int64_t m, int64_t k) { return codes_bytes(m, k) + round_up(m * 4, 256); }
int check_workspace(const char* op, const void* workspace, size_t have, int64_t need) {
    if (need == 0) return PLM_OK;
    if (workspace == nullptr || static_cast<int64_t>(have) < need) {
        set_error(op, "workspace of %lld bytes required, %zu given", static_cast<long long>(need), have);
        return PLM_ERR_WORKSPACE;
    }
    PLM_CHECK_ARG(aligned(workspace, 256), op, "workspace must be 256-byte aligned");
    return PLM_OK;
}

}  // namespace
}  // namespace plm

using namespace plm;

extern "C" {

int plm_quantize_rows_int8(const void* x, plm_dtype x_dtype, int64_t m, int64_t k, int8_t* codes, float* x_scale, void* stream) {
    const char* op = "quantize_rows_int8";
    clear_error();
    PLM_CHECK_ARG(x_dtype == PLM_BF16 || x_dtype == PLM_FP16 || x_dtype == PLM_FP32, op, "x must be fp32, fp16 or bf16");
    PLM_CHECK_ARG(m >= 0 && k >= 0 && m <= kDenseMaxRows && k <= int64_t{1} << 28, op, "M must be below 2^24, K at most 2^28");
    if (m == 0) return PLM_OK;
    if (int rc = check_pointer(op, "x", x, dtype_size(x_dtype), k > 0)) return rc;
    if (int rc = check_pointer(op, "codes", codes, 1, k > 0)) return rc;
    if (int rc = check_pointer(op, "scale", x_scale, 4)) return rc;
    launch_quantize_int8(x, x_dtype, m, k, codes, x_scale, as_stream(stream));
    PLM_HIP_LAUNCH_CHECK(op);
    return PLM_OK;
}

int plm_dequantize_rows_int8(const int8_t* codes, const float* x_scale, int64_t m, int64_t k, void* out, plm_dtype out_dtype, void* stream) {
    const char* op = "dequantize_rows_int8";
    clear_error();
    PLM_CHECK_ARG(out_dtype == PLM_BF16 || out_dtype == PLM_FP16 || out_dtype == PLM_FP32, op, "out must be fp32, fp16 or bf16");
    PLM_CHECK_ARG(m >= 0 && k >= 0 && m <= kDenseMaxRows && k <= int64_t{1} << 28, op, "M must be below 2^24, K at most 2^28");
    if (m == 0 || k == 0) return PLM_OK;
    if (int rc = check_pointer(op, "codes", codes, 1)) return rc;
    if (int rc = check_pointer(op, "scale", x_scale, 4)) return rc;
    if (int rc = check_pointer(op, "out", out, dtype_size(out_dtype))) return rc;
    launch_dequantize_int8(codes, x_scale, m, k, out, out_dtype, as_stream(stream));
    PLM_HIP_LAUNCH_CHECK(op);
    return PLM_OK;
}

int64_t plm_gemm_int8_workspace_bytes(int64_t m, int64_t n, int64_t k) { return counts(m, n, k) ? partial_bytes(m, n, k) : 0; }

int plm_gemm_int8(const int8_t* codes, const float* x_scale, const int8_t* weight, const float* scale, int64_t m, int64_t n, int64_t k,
                  void* y, plm_dtype y_dtype, void* workspace, size_t workspace_bytes, void* stream) {
    const char* op = "gemm_int8";
    clear_error();
    PLM_CHECK_ARG(sixteen(y_dtype), op, "y must be fp16 or bf16");
    if (int rc = check_sizes(op, "M", m, n, k)) return rc;
    if (int rc = check_int8(op, k)) return rc;
    if (m == 0 || n == 0) return PLM_OK;
    hipStream_t s = as_stream(stream);
    if (int rc = check_pointer(op, "y", y, 2)) return rc;
    if (k == 0) return zero_output(op, y, m, n, s);
    if (int rc = check_pointer(op, "codes", codes, 16)) return rc;
    if (int rc = check_pointer(op, "weight", weight, 16)) return rc;
    if (int rc = check_pointer(op, "x_scale", x_scale, 4)) return rc;
    if (int rc = check_pointer(op, "scale", scale, 4)) return rc;
    if (int rc = check_workspace(op, workspace, workspace_bytes, partial_bytes(m, n, k))) return rc;
    dense_product p = product(kInt8, codes, weight, y, y_dtype == PLM_BF16, m, n, k);
    p.p_scale = x_scale, p.q_scale = scale;
    p.plan = plan_dense(p, kDense, true, true);
    run_int8(p, workspace, s);
    PLM_HIP_LAUNCH_CHECK(op);
    return PLM_OK;
}

int64_t plm_gemm_int8_w8a8_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    // Of both plans, one for x that is 16-byte aligned and one for x that is not.
    return counts(m, n, k) ? tokens_bytes(m, k) + std::max(partial_bytes(m, n, k, true), partial_bytes(m, n, k)) : 0;
}

int plm_gemm_int8_w8a8(const void* x, plm_dtype x_dtype, const int8_t* weight, const float* scale, int64_t m, int64_t n, int64_t k, void* y,
                       void* workspace, size_t workspace_bytes, void* stream) {
    const char* op = "gemm_int8_w8a8";
    clear_error();
    PLM_CHECK_ARG(sixteen(x_dtype), op, "x must be fp16 or bf16");
    if (int rc = check_sizes(op, "M", m, n, k)) return rc;
    if (int rc = check_int8(op, k)) return rc;
    if (m == 0 || n == 0) return PLM_OK;
    hipStream_t s = as_stream(stream);
    if (int rc = check_pointer(op, "y", y, 2)) return rc;
    if (k == 0) return zero_output(op, y, m, n, s);
    if (int rc = check_pointer(op, "x", x, 2)) return rc;
    if (int rc = check_pointer(op, "weight", weight, 16)) return rc;
    if (int rc = check_pointer(op, "scale", scale, 4)) return rc;
    dense_product p = product(kInt8, x, weight, y, x_dtype == PLM_BF16, m, n, k);
    p.q_scale = scale, p.to_quantize = aligned(x, 16);
    p.plan = plan_dense(p, kDense, true, true);
    if (int rc = check_workspace(op, workspace, workspace_bytes, tokens_bytes(m, k) + dense_partial_bytes(p.plan, m, n))) return rc;
    if (dense_rows_quantizes(p, p.plan.rows_block)) {
        launch_dense_rows_quantize(p, s);
        PLM_HIP_LAUNCH_CHECK(op);
        return PLM_OK;
    }
    auto* codes = static_cast<int8_t*>(workspace);
    auto* x_scale = reinterpret_cast<float*>(codes + codes_bytes(m, k));
    launch_quantize_int8(x, x_dtype, m, k, codes, x_scale, s);
    p.p = codes, p.p_scale = x_scale;
    run_int8(p, codes + tokens_bytes(m, k), s);
    PLM_HIP_LAUNCH_CHECK(op);
    return PLM_OK;
}

int64_t plm_grouped_gemm_int8_workspace_bytes(int64_t rows, int64_t n, int64_t k) { return counts(rows, n, k) ? tokens_bytes(rows, k) : 0; }

int plm_grouped_gemm_int8(const void* x, plm_dtype x_dtype, const int8_t* weight, const float* scale, const int32_t* offsets,
                          int64_t n_experts, int64_t rows, int64_t n, int64_t k, void* y, int zero_rest, void* workspace,
                          size_t workspace_bytes, void* stream) {
    const char* op = "grouped_gemm_int8";
    clear_error();
    PLM_CHECK_ARG(sixteen(x_dtype), op, "x must be fp16 or bf16");
    if (int rc = check_sizes(op, "rows", rows, n, k)) return rc;
    if (int rc = check_int8(op, k)) return rc;
    if (int rc = check_experts(op, n_experts, n, k)) return rc;
    if (rows == 0 || n == 0) return PLM_OK;
    hipStream_t s = as_stream(stream);
    if (int rc = check_pointer(op, "y", y, 2)) return rc;
    if (int rc = check_pointer(op, "x", x, 2, k > 0)) return rc;
    if (int rc = check_pointer(op, "weight", weight, 16, k > 0)) return rc;
    if (int rc = check_pointer(op, "scale", scale, 4)) return rc;
    if (int rc = check_offsets(op, offsets)) return rc;
    if (k == 0) return run_experts(op, product(x_dtype == PLM_BF16 ? kBf16 : kFp16, x, weight, y, x_dtype == PLM_BF16, rows, n, k), offsets, n_experts, zero_rest, s);
    if (int rc = check_workspace(op, workspace, workspace_bytes, tokens_bytes(rows, k))) return rc;
    auto* codes = static_cast<int8_t*>(workspace);
    auto* x_scale = reinterpret_cast<float*>(codes + codes_bytes(rows, k));
    launch_quantize_int8(x, x_dtype, rows, k, codes, x_scale, s);
    dense_product p = product(kInt8, codes, weight, y, x_dtype == PLM_BF16, rows, n, k);
    p.p_scale = x_scale, p.q_scale = scale;
    p.offsets = offsets, p.experts = n_experts, p.zero_rest = zero_rest != 0;
    p.plan = plan_dense(p, kByRows, true, false);
    if (p.plan.rows_block > 0) launch_dense_rows(p, kByRows, s);
    else launch_tiles_int8(p, kByRows, s);
    PLM_HIP_LAUNCH_CHECK(op);
    return PLM_OK;
}

int plm_grouped_gemm_16(const void* x, plm_dtype dtype, const void* weight, const int32_t* offsets, int64_t n_experts, int64_t rows, int64_t n,
                        int64_t k, void* y, int zero_rest, void* stream) {
    const char* op = "grouped_gemm";
    clear_error();
    PLM_CHECK_ARG(sixteen(dtype), op, "x must be fp16 or bf16");
    if (int rc = check_sizes(op, "rows", rows, n, k)) return rc;
    PLM_CHECK_ARG(k % 8 == 0, op, "K must be a multiple of 8");
    if (int rc = check_experts(op, n_experts, n, k)) return rc;
    if (rows == 0 || n == 0) return PLM_OK;
    if (int rc = check_pointer(op, "y", y, 2)) return rc;
    if (int rc = check_pointer(op, "x", x, 16, k > 0)) return rc;
    if (int rc = check_pointer(op, "weight", weight, 16, k > 0)) return rc;
    if (int rc = check_offsets(op, offsets)) return rc;
    return run_experts(op, product(dtype == PLM_BF16 ? kBf16 : kFp16, x, weight, y, dtype == PLM_BF16, rows, n, k), offsets, n_experts, zero_rest,
                       as_stream(stream));
}

int plm_grouped_gemm_grad_x(const void* dy, plm_dtype dtype, const void* weight, const int32_t* offsets, int64_t n_experts, int64_t rows,
                            int64_t n, int64_t k, void* dx, int zero_rest, void* stream) {
    const char* op = "grouped_gemm_grad_x";
    clear_error();
    PLM_CHECK_ARG(sixteen(dtype), op, "dy must be fp16 or bf16");
    if (int rc = check_sizes(op, "rows", rows, n, k)) return rc;
    PLM_CHECK_ARG(n % 8 == 0 && k % 8 == 0, op, "N and K must be multiples of 8");
    if (int rc = check_experts(op, n_experts, n, k)) return rc;
    if (rows == 0 || k == 0) return PLM_OK;
    if (int rc = check_pointer(op, "dx", dx, 2)) return rc;
    if (int rc = check_pointer(op, "dy", dy, 16, n > 0)) return rc;
    if (int rc = check_pointer(op, "weight", weight, 16, n > 0)) return rc;
    if (int rc = check_offsets(op, offsets)) return rc;
    dense_product p = product(dtype == PLM_BF16 ? kBf16 : kFp16, dy, weight, dx, dtype == PLM_BF16, rows, k, n);
    p.offsets = offsets, p.experts = n_experts, p.zero_rest = zero_rest != 0;
    p.plan = plan_dense(p, kByRows, false, false);
    launch_tiles_grad_x(p, as_stream(stream));
    PLM_HIP_LAUNCH_CHECK(op);
    return PLM_OK;
}

int plm_grouped_gemm_grad_w(const void* dy, const void* x, plm_dtype dtype, const int32_t* offsets, int64_t n_experts, int64_t rows, int64_t n,
                            int64_t k, void* dw, void* stream) {
    const char* op = "grouped_gemm_grad_w";
    clear_error();
    PLM_CHECK_ARG(sixteen(dtype), op, "dy and x must be fp16 or bf16");
    if (int rc = check_sizes(op, "rows", rows, n, k)) return rc;
    PLM_CHECK_ARG(n % 8 == 0 && k % 8 == 0, op, "N and K must be multiples of 8");
    if (int rc = check_experts(op, n_experts, n, k)) return rc;
    if (n == 0 || k == 0) return PLM_OK;
    if (int rc = check_pointer(op, "dw", dw, 2)) return rc;
    if (int rc = check_pointer(op, "dy", dy, 16, rows > 0)) return rc;
    if (int rc = check_pointer(op, "x", x, 16, rows > 0)) return rc;
    if (int rc = check_offsets(op, offsets)) return rc;
    dense_product p = product(dtype == PLM_BF16 ? kBf16 : kFp16, dy, x, dw, dtype == PLM_BF16, n, k, rows);
    p.offsets = offsets, p.experts = n_experts;
    p.plan = plan_dense(p, kByRanges, false, false);
    launch_tiles_grad_w(p, as_stream(stream));
    PLM_HIP_LAUNCH_CHECK(op);
    return PLM_OK;
}

}  // extern "C"
