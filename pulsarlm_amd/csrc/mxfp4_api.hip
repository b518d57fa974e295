// C entry points of the MXFP4 products: argument checks, workspaces, and the choice between the kernel for
// few rows (mxfp4_rows.hip) and the tiles (mxfp4_tiles.hpp). The reference has no 4-bit floating point.
#include "mxfp4.hpp"

namespace plm {

int zero_output(const char* op, void* y, int64_t m, int64_t n, hipStream_t s);
void launch_mx_tiles_w4a16(const mx_product& p, hipStream_t s);
void launch_mx_tiles_w4a4(const mx_product& p, hipStream_t s);
int64_t mx_tiles_w4a4_bytes(int64_t m, int64_t n, int64_t k);
int64_t mx_grad_bytes(int64_t m, int64_t n, int64_t k, bool gated, bool dy_aligned);
int launch_mx_grad(const char* op, bool gated, bool bf16, const void* dy, const void* gate_up, const mx_matrix& w0, const mx_matrix& w1,
                   int64_t m, int64_t n, int64_t k, void* dx, void* workspace, hipStream_t s);

namespace {

mx_matrix matrix(const void* codes, const void* scale) {
    return {static_cast<const uint8_t*>(codes), static_cast<const uint32_t*>(scale)};
}

// A grid of at most 2^32 work-items, and offsets of one workgroup below kOOB.
bool takes_rows(int64_t m, int64_t n, int64_t k) { return m <= (int64_t{1} << 24) && m * std::max(n, k) <= (int64_t{1} << 36); }
bool takes(int64_t m, int64_t n, int64_t k) { return n <= kMxMaxSize && k <= kMxMaxSize && takes_rows(m, n, k); }
// What a workspace query counts: sizes that a call takes, and works on.
bool counts(int64_t m, int64_t n, int64_t k) { return m > 0 && n > 0 && k > 0 && takes(m, n, k); }
int check_sizes(const char* op, plm_dtype x_dtype, int64_t m, int64_t n, int64_t k) {
    PLM_CHECK_ARG(x_dtype == PLM_BF16 || x_dtype == PLM_FP16, op, "x must be fp16 or bf16");
    PLM_CHECK_ARG(m >= 0 && n >= 0 && k >= 0, op, "sizes must be non-negative");
    PLM_CHECK_ARG(k % kMxBlock == 0, op, "K must be a multiple of 32");
    PLM_CHECK_ARG(n <= kMxMaxSize && k <= kMxMaxSize, op, "N and K must be at most 2^19");
    PLM_CHECK_ARG(takes_rows(m, n, k), op, "M must be at most 2^24, M N and M K at most 2^36");
    return PLM_OK;
}
int check_weight(const char* op, const void* weight, const void* scale) {
    PLM_CHECK_ARG(weight && scale, op, "null pointer");
    PLM_CHECK_ARG(aligned(weight, 16), op, "weight must be 16-byte aligned");
    PLM_CHECK_ARG(aligned(scale, 4), op, "scale must be 4-byte aligned");
    return PLM_OK;
}
// x [M, K] and y; with K == 0 x has no element.
int check_rows(const char* op, const void* x, int64_t k, const void* y) {
    PLM_CHECK_ARG((x || k == 0) && y, op, "null pointer");
    PLM_CHECK_ARG(aligned(x, 16), op, "x must be 16-byte aligned");
    PLM_CHECK_ARG(aligned(y, 2), op, "y must be 2-byte aligned");
    return PLM_OK;
}
int check_workspace(const char* op, const void* workspace, size_t have, int64_t need) {
    if (need == 0) return PLM_OK;
    if (workspace == nullptr || static_cast<int64_t>(have) < need) {
        set_error(op, "workspace of %lld bytes required, %zu given", static_cast<long long>(need), have);
        return PLM_ERR_WORKSPACE;
    }
    PLM_CHECK_ARG(aligned(workspace, 256), op, "workspace must be 256-byte aligned");
    return PLM_OK;
}

// Codes of [M, K] in a workspace: [tiles][scales]. After them, the sums of K splits.
struct codes_room {
    int64_t tiles, total;
};
codes_room room(int64_t m, int64_t k) {
    const mx_dims d = make_mx_dims(m, k);
    return {d.tile_bytes(), d.tile_bytes() + round_up(d.scale_bytes(), 1024)};
}
struct codes_at {
    uint8_t* codes;
    uint32_t* scale;
    mx_matrix in() const { return {codes, scale}; }
};
codes_at place(void* base, int64_t offset, const codes_room& r) {
    auto* p = static_cast<uint8_t*>(base) + offset;
    return {p, reinterpret_cast<uint32_t*>(p + r.tiles)};
}

void run_w4a16(const mx_product& p, hipStream_t s) {
    if (!launch_mx_rows(p, false, s)) launch_mx_tiles_w4a16(p, s);
}
// x quantized in the kernel where that can be, else to `to` first.
void run_w4a4(mx_product p, const codes_at& to, hipStream_t s) {
    if (launch_mx_rows(p, true, s)) return;
    launch_mx_quantize_tiles(p.x16, p.bf16, p.m, p.k, to.codes, to.scale, s);
    p.xq = to.in();
    if (!launch_mx_rows(p, false, s)) launch_mx_tiles_w4a4(p, s);
}

mx_product product(const void* x, plm_dtype x_dtype, const mx_matrix& w0, const mx_matrix& w1, int64_t m, int64_t n, int64_t k,
                   mx_epilogue epilogue, const mx_output& out) {
    mx_product p{};
    p.x16 = static_cast<const uint16_t*>(x);
    p.w0 = w0;
    p.w1 = w1;
    p.m = m, p.n = n, p.k = k;
    p.bf16 = x_dtype == PLM_BF16;
    p.epilogue = epilogue;
    p.out = out;
    return p;
}

}  // namespace
}  // namespace plm

using namespace plm;

extern "C" {

int plm_gemm_mxfp4(const void* x, plm_dtype x_dtype, const void* weight, const void* scale, int64_t m, int64_t n, int64_t k, void* y,
                   void* stream) {
    const char* op = "gemm_mxfp4";
    clear_error();
    if (int rc = check_sizes(op, x_dtype, m, n, k)) return rc;
    if (m == 0 || n == 0) return PLM_OK;
    hipStream_t s = as_stream(stream);
    if (int rc = check_rows(op, x, k, y)) return rc;
    if (k == 0) return zero_output(op, y, m, n, s);
    if (int rc = check_weight(op, weight, scale)) return rc;
    run_w4a16(product(x, x_dtype, matrix(weight, scale), {}, m, n, k, kMxPlain, mx_make_output(y, nullptr, n)), s);
    PLM_HIP_LAUNCH_CHECK(op);
    return PLM_OK;
}

int64_t plm_gemm_mxfp4_w4a4_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    return counts(m, n, k) ? room(m, k).total + mx_tiles_w4a4_bytes(m, n, k) : 0;
}

int plm_gemm_mxfp4_w4a4(const void* x, plm_dtype x_dtype, const void* weight, const void* scale, int64_t m, int64_t n, int64_t k, void* y,
                        void* workspace, size_t workspace_bytes, void* stream) {
    const char* op = "gemm_mxfp4_w4a4";
    clear_error();
    if (int rc = check_sizes(op, x_dtype, m, n, k)) return rc;
    if (m == 0 || n == 0) return PLM_OK;
    hipStream_t s = as_stream(stream);
    if (int rc = check_rows(op, x, k, y)) return rc;
    if (k == 0) return zero_output(op, y, m, n, s);
    if (int rc = check_weight(op, weight, scale)) return rc;
    if (int rc = check_workspace(op, workspace, workspace_bytes, plm_gemm_mxfp4_w4a4_workspace_bytes(m, n, k))) return rc;
    const codes_room r = room(m, k);
    mx_product p = product(x, x_dtype, matrix(weight, scale), {}, m, n, k, kMxPlain, mx_make_output(y, nullptr, n));
    p.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + r.total);
    run_w4a4(p, place(workspace, 0, r), s);
    PLM_HIP_LAUNCH_CHECK(op);
    return PLM_OK;
}

int plm_gated_mxfp4(const void* x, plm_dtype x_dtype, const void* gate_weight, const void* gate_scale, const void* up_weight,
                    const void* up_scale, int64_t m, int64_t n, int64_t k, void* h, float* gate_up, void* stream) {
    const char* op = "gated_mxfp4";
    clear_error();
    if (int rc = check_sizes(op, x_dtype, m, n, k)) return rc;
    if (m == 0 || n == 0) return PLM_OK;
    hipStream_t s = as_stream(stream);
    if (int rc = check_rows(op, x, k, h)) return rc;
    PLM_CHECK_ARG(aligned(gate_up, 4), op, "gate_up must be 4-byte aligned");
    if (k == 0) {
        if (gate_up != nullptr)
            if (int rc = zero_output(op, gate_up, m, 4 * n, s)) return rc;
        return zero_output(op, h, m, n, s);
    }
    if (int rc = check_weight(op, gate_weight, gate_scale)) return rc;
    if (int rc = check_weight(op, up_weight, up_scale)) return rc;
    run_w4a16(product(x, x_dtype, matrix(gate_weight, gate_scale), matrix(up_weight, up_scale), m, n, k, kMxGated, mx_make_output(h, gate_up, n)),
              s);
    PLM_HIP_LAUNCH_CHECK(op);
    return PLM_OK;
}

int64_t plm_mlp_mxfp4_w4a4_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    return counts(m, n, k) ? room(m, k).total + room(m, n).total + mx_tiles_w4a4_bytes(m, k, n) : 0;
}

int plm_mlp_mxfp4_w4a4(const void* x, plm_dtype x_dtype, const void* gate_weight, const void* gate_scale, const void* up_weight,
                       const void* up_scale, const void* down_weight, const void* down_scale, int64_t m, int64_t n, int64_t k, void* y,
                       void* workspace, size_t workspace_bytes, void* stream) {
    const char* op = "mlp_mxfp4_w4a4";
    clear_error();
    if (int rc = check_sizes(op, x_dtype, m, n, k)) return rc;
    PLM_CHECK_ARG(n % kMxBlock == 0, op, "the intermediate size must be a multiple of 32");
    if (m == 0 || k == 0) return PLM_OK;
    hipStream_t s = as_stream(stream);
    if (int rc = check_rows(op, x, k, y)) return rc;
    if (n == 0) return zero_output(op, y, m, k, s);
    if (int rc = check_weight(op, gate_weight, gate_scale)) return rc;
    if (int rc = check_weight(op, up_weight, up_scale)) return rc;
    if (int rc = check_weight(op, down_weight, down_scale)) return rc;
    if (int rc = check_workspace(op, workspace, workspace_bytes, plm_mlp_mxfp4_w4a4_workspace_bytes(m, n, k))) return rc;
    const codes_room xr = room(m, k), hr = room(m, n);
    const codes_at xq = place(workspace, 0, xr), hq = place(workspace, xr.total, hr);
    const mx_dims hd = make_mx_dims(m, n);
    mx_output act = mx_make_output(nullptr, nullptr, n);
    act.codes = hq.codes;
    act.scale = reinterpret_cast<uint8_t*>(hq.scale);
    act.ktiles = static_cast<int>(hd.ktiles);
    run_w4a4(product(x, x_dtype, matrix(gate_weight, gate_scale), matrix(up_weight, up_scale), m, n, k, kMxGatedCodes, act), xq, s);
    PLM_HIP_LAUNCH_CHECK(op);
    mx_product down = product(nullptr, x_dtype, matrix(down_weight, down_scale), {}, m, k, n, kMxPlain, mx_make_output(y, nullptr, k));
    down.xq = hq.in();
    down.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + xr.total + hr.total);
    if (!launch_mx_rows(down, false, s)) launch_mx_tiles_w4a4(down, s);
    PLM_HIP_LAUNCH_CHECK(op);
    return PLM_OK;
}

int64_t plm_gemm_mxfp4_grad_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    return counts(m, n, k) ? mx_grad_bytes(m, n, k, false, false) : 0;
}
int64_t plm_gemm_mxfp4_grad_aligned_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    return counts(m, n, k) ? mx_grad_bytes(m, n, k, false, true) : 0;
}
int64_t plm_gated_mxfp4_grad_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    return counts(m, n, k) ? mx_grad_bytes(m, n, k, true, true) : 0;
}

int plm_gemm_mxfp4_grad(const void* dy, plm_dtype dtype, const void* weight, const void* scale, int64_t m, int64_t n, int64_t k, void* dx,
                        void* workspace, size_t workspace_bytes, void* stream) {
    const char* op = "gemm_mxfp4_grad";
    clear_error();
    if (int rc = check_sizes(op, dtype, m, n, k)) return rc;
    if (m == 0 || k == 0) return PLM_OK;
    hipStream_t s = as_stream(stream);
    PLM_CHECK_ARG(dx && aligned(dx, 8), op, "dx must be 8-byte aligned");
    if (n == 0) return zero_output(op, dx, m, k, s);
    PLM_CHECK_ARG(dy && aligned(dy, 2), op, "dy must be 2-byte aligned");
    if (int rc = check_weight(op, weight, scale)) return rc;
    if (int rc = check_workspace(op, workspace, workspace_bytes, mx_grad_bytes(m, n, k, false, aligned(dy, 16)))) return rc;
    return launch_mx_grad(op, false, dtype == PLM_BF16, dy, nullptr, matrix(weight, scale), matrix(weight, scale), m, n, k, dx, workspace, s);
}

int plm_gated_mxfp4_grad(const void* dh, const float* gate_up, plm_dtype dtype, const void* gate_weight, const void* gate_scale,
                         const void* up_weight, const void* up_scale, int64_t m, int64_t n, int64_t k, void* dx, void* workspace,
                         size_t workspace_bytes, void* stream) {
    const char* op = "gated_mxfp4_grad";
    clear_error();
    if (int rc = check_sizes(op, dtype, m, n, k)) return rc;
    if (m == 0 || k == 0) return PLM_OK;
    hipStream_t s = as_stream(stream);
    PLM_CHECK_ARG(dx && aligned(dx, 8), op, "dx must be 8-byte aligned");
    if (n == 0) return zero_output(op, dx, m, k, s);
    PLM_CHECK_ARG(dh && gate_up && aligned(dh, 2) && aligned(gate_up, 4), op, "dh must be 2-byte and gate_up 4-byte aligned");
    if (int rc = check_weight(op, gate_weight, gate_scale)) return rc;
    if (int rc = check_weight(op, up_weight, up_scale)) return rc;
    if (int rc = check_workspace(op, workspace, workspace_bytes, plm_gated_mxfp4_grad_workspace_bytes(m, n, k))) return rc;
    return launch_mx_grad(op, true, dtype == PLM_BF16, dh, gate_up, matrix(gate_weight, gate_scale), matrix(up_weight, up_scale), m, n, k, dx,
                          workspace, s);
}

}  // extern "C"
