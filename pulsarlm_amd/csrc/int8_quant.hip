// Rows of 8-bit integers: quantizer (tokens' activations, a weight's output channels; the rule: int8_rows.hpp) and its
// inverse.
// What bounds it: memory. M = 4096, K 12288, bf16, x and codes not in the caches: quantizer 30 us, 5.0 TB/s; back to fp32 43 us,
// 5.9 TB/s.
#include <algorithm>

#include "dense_gemm.hpp"
#include "int8_rows.hpp"

namespace plm {

namespace {

// Eight consecutive values.
template <plm_dtype D> struct eight {
    u32x4_t v[D == PLM_FP32 ? 2 : 1];
};
template <plm_dtype D> __device__ __forceinline__ eight<D> load_eight(const uint8_t* row, int64_t chunk, bool in) {
    eight<D> e{};
    if (in) {
        const u32x4_t* p = reinterpret_cast<const u32x4_t*>(row + chunk * (D == PLM_FP32 ? 32 : 16));
        e.v[0] = p[0];
        if constexpr (D == PLM_FP32) e.v[1] = p[1];
    }
    return e;
}
// The running largest magnitude: fp32 bits, or those of both halves of a dword.
template <plm_dtype D> __device__ __forceinline__ uint32_t top_of(const eight<D>& e, uint32_t top) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (D == PLM_FP32) top = max(top, max(e.v[0][i] & 0x7fffffffu, e.v[1][i] & 0x7fffffffu));
        else top = top_16(top, e.v[0][i]);
    }
    return top;
}
template <plm_dtype D> __device__ __forceinline__ uint2 codes_of(const eight<D>& e, const int8_scale& k) {
    if (!k.finite) return make_uint2(0u, 0u);
    float x[8];
    if constexpr (D == PLM_FP32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(e.v[i >> 2][i & 3]);
    } else {
        eight_values<D == PLM_BF16>(e.v[0], x);
    }
    uint32_t w[2];
    int8_codes<8>(x, k, w);
    return make_uint2(w[0], w[1]);
}

__device__ __forceinline__ uint32_t wave_top(uint32_t top) {
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), s)));
    return top;
}

// T threads a row, ROWS rows a workgroup (T == 64: a wavefront each, which needs no barrier). The first CAP chunks of
// eight a thread wait in registers for the row's largest; what is past them is read again.
template <plm_dtype D, int T, int ROWS, int CAP>
__global__ void __launch_bounds__(T * ROWS) quantize_int8_kernel(const uint8_t* __restrict__ x, int64_t m, int64_t k, int8_t* __restrict__ codes,
                                                                 float* __restrict__ scale) {
    static_assert(ROWS == 1 || T == 64, "rows of a wavefront each");
    __shared__ uint32_t part[T / 64];
    const int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / T, chunks = k >> 3;
    const int at = threadIdx.x % T;
    if (ROWS > 1 && row >= m) return;
    const uint8_t* from = x + row * k * (D == PLM_FP32 ? 4 : 2);
    uint2* to = reinterpret_cast<uint2*>(codes + row * k);
    eight<D> held[CAP];
#pragma unroll
    for (int c = 0; c < CAP; ++c) held[c] = load_eight<D>(from, at + c * T, at + c * T < chunks);
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < CAP; ++c) top = top_of(held[c], top);
    for (int64_t c = at + CAP * T; c < chunks; c += T) top = top_of(load_eight<D>(from, c, true), top);
    if constexpr (D != PLM_FP32) top = top_bits<D == PLM_BF16>(top);
    top = wave_top(top);
    if constexpr (T > 64) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < T / 64; ++w) top = max(top, part[w]);
    }
    const int8_scale s = make_int8_scale(top);
    if (at == 0) scale[row] = s.s;
#pragma unroll
    for (int c = 0; c < CAP; ++c)
        if (at + c * T < chunks) to[at + c * T] = codes_of(held[c], s);
    for (int64_t c = at + CAP * T; c < chunks; c += T) to[c] = codes_of(load_eight<D>(from, c, true), s);
}

template <plm_dtype D> __device__ __forceinline__ float load_one(const void* x, int64_t at) {
    if constexpr (D == PLM_FP32) return static_cast<const float*>(x)[at];
    else return from_bits16<D == PLM_BF16>(static_cast<const uint16_t*>(x)[at]);
}
// Any K and alignment, a value at a time.
template <plm_dtype D>
__global__ void __launch_bounds__(256) quantize_int8_any_kernel(const void* __restrict__ x, int64_t k, int8_t* __restrict__ codes,
                                                                float* __restrict__ scale) {
    __shared__ uint32_t part[4];
    const int64_t row = blockIdx.x;
    uint32_t top = 0;
    for (int64_t i = threadIdx.x; i < k; i += 256) top = max(top, int8_magnitude(load_one<D>(x, row * k + i)));
    top = wave_top(top);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    const int8_scale s = make_int8_scale(max(max(part[0], part[1]), max(part[2], part[3])));
    if (threadIdx.x == 0) scale[row] = s.s;
    for (int64_t i = threadIdx.x; i < k; i += 256) {
        const float v[4] = {load_one<D>(x, row * k + i), 0.f, 0.f, 0.f};
        uint32_t code[1] = {0};
        if (s.finite) int8_codes<4>(v, s, code);
        codes[row * k + i] = static_cast<int8_t>(code[0]);
    }
}

template <plm_dtype D> void launch_quantize(const void* x, int64_t m, int64_t k, int8_t* codes, float* scale, hipStream_t s) {
    const unsigned grid = static_cast<unsigned>(m);
    const auto* bytes = static_cast<const uint8_t*>(x);
    if (k % 8 != 0 || !aligned(x, 16) || !aligned(codes, 8)) {
        quantize_int8_any_kernel<D><<<grid, 256, 0, s>>>(x, k, codes, scale);
        return;
    }
    // As many threads a row as hold it in two chunks each: fewer hold more each and have fewer rows in flight, more spend
    // their time on the row's maximum. bf16, x not in the caches, us: M = 4096, K 4096 with 64, 128, 256, 512 and 1024 threads
    // that hold the row 16.2, 13.4, 12.1, 13.1 and 18.9; K 12288 with 256, 512 and 1024 30.3, 28.4 and 29.7; M = 32768, K 1024 with
    // 64, 128 and 256 19.3, 22.0 and 31.3; M = 333, K 12288 with 256, 512 and 1024 8.7, 7.0 and 6.4. A wavefront's rows need no barrier: four of them
    // a workgroup. More rows than a grid of such workgroups has: 256 threads each, which read the rest of a row twice.
    const int64_t chunks = k / 8;
    if (chunks <= 64 * 2) quantize_int8_kernel<D, 64, 4, 2><<<static_cast<unsigned>(ceil_div(m, 4)), 256, 0, s>>>(bytes, m, k, codes, scale);
    else if (chunks <= 128 * 2) quantize_int8_kernel<D, 128, 1, 2><<<grid, 128, 0, s>>>(bytes, m, k, codes, scale);
    else if (chunks <= 256 * 2 || !dense_grid_fits(m, 1024)) quantize_int8_kernel<D, 256, 1, 2><<<grid, 256, 0, s>>>(bytes, m, k, codes, scale);
    else if (chunks <= 512 * 2) quantize_int8_kernel<D, 512, 1, 2><<<grid, 512, 0, s>>>(bytes, m, k, codes, scale);
    else if (chunks <= 1024 * 2) quantize_int8_kernel<D, 1024, 1, 2><<<grid, 1024, 0, s>>>(bytes, m, k, codes, scale);
    else quantize_int8_kernel<D, 1024, 1, 4><<<grid, 1024, 0, s>>>(bytes, m, k, codes, scale);
}

// Items of N codes, 16 bytes of output (or one value, where rows are not whole items or not aligned): four a thread, a
// workgroup's width apart, so that a wavefront's loads and stores are contiguous. INDEX: 32 bits where the items fit, for
// the division by the items of a row.
template <plm_dtype D, int N, typename INDEX>
__global__ void __launch_bounds__(256) dequantize_int8_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scale, INDEX items,
                                                              INDEX per_row, void* __restrict__ out) {
    constexpr int EACH = 4;
    const INDEX first = static_cast<INDEX>(blockIdx.x) * (256 * EACH) + threadIdx.x;
    uint32_t c[EACH][N == 8 ? 2 : 1];
    float s[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const INDEX i = first + e * 256;
        if (i >= items) continue;
        if constexpr (N == 8) {
            const uint2 w = reinterpret_cast<const uint2*>(codes)[i];
            c[e][0] = w.x, c[e][1] = w.y;
        } else if constexpr (N == 4) {
            c[e][0] = reinterpret_cast<const uint32_t*>(codes)[i];
        } else {
            c[e][0] = static_cast<uint8_t>(codes[i]);
        }
        s[e] = scale[i / per_row];
    }
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const INDEX i = first + e * 256;
        if (i >= items) continue;
        float f[N];
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = static_cast<float>(static_cast<int8_t>(c[e][j >> 2] >> (8 * (j & 3)))) * s[e];
        if constexpr (N == 8) reinterpret_cast<u32x4_t*>(out)[i] = u32x4_t{pack2<D == PLM_BF16>(f[0], f[1]), pack2<D == PLM_BF16>(f[2], f[3]), pack2<D == PLM_BF16>(f[4], f[5]), pack2<D == PLM_BF16>(f[6], f[7])};
        else if constexpr (N == 4) reinterpret_cast<f32x4_t*>(out)[i] = f32x4_t{f[0], f[1], f[2], f[3]};
        else if constexpr (D == PLM_FP32) static_cast<float*>(out)[i] = f[0];
        else static_cast<uint16_t*>(out)[i] = static_cast<uint16_t>(to_bits16<D == PLM_BF16>(f[0]));
    }
}

template <plm_dtype D, int N> void launch_items(const int8_t* codes, const float* scale, int64_t m, int64_t k, void* out, hipStream_t s) {
    // Whole rows at a time, as many as a grid holds.
    const int64_t most = std::max<int64_t>(1, (int64_t{1} << 33) / k);
    for (int64_t row = 0; row < m; row += most) {
        const int64_t rows = std::min(most, m - row), items = rows * k / N, at = row * k;
        const unsigned grid = static_cast<unsigned>(ceil_div(items, 1024));
        void* to = static_cast<uint8_t*>(out) + at * (D == PLM_FP32 ? 4 : 2);
        if (items < int64_t{1} << 31) dequantize_int8_kernel<D, N, uint32_t><<<grid, 256, 0, s>>>(codes + at, scale + row, items, k / N, to);
        else dequantize_int8_kernel<D, N, uint64_t><<<grid, 256, 0, s>>>(codes + at, scale + row, items, k / N, to);
    }
}
template <plm_dtype D> void launch_dequantize(const int8_t* codes, const float* scale, int64_t m, int64_t k, void* out, hipStream_t s) {
    constexpr int N = D == PLM_FP32 ? 4 : 8;
    if (k % N == 0 && aligned(codes, N) && aligned(out, 16)) launch_items<D, N>(codes, scale, m, k, out, s);
    else launch_items<D, 1>(codes, scale, m, k, out, s);
}

}  // namespace

void launch_quantize_int8(const void* x, plm_dtype dtype, int64_t m, int64_t k, int8_t* codes, float* scale, hipStream_t s) {
    if (dtype == PLM_FP32) launch_quantize<PLM_FP32>(x, m, k, codes, scale, s);
    else if (dtype == PLM_BF16) launch_quantize<PLM_BF16>(x, m, k, codes, scale, s);
    else launch_quantize<PLM_FP16>(x, m, k, codes, scale, s);
}
void launch_dequantize_int8(const int8_t* codes, const float* scale, int64_t m, int64_t k, void* out, plm_dtype dtype, hipStream_t s) {
    if (dtype == PLM_FP32) launch_dequantize<PLM_FP32>(codes, scale, m, k, out, s);
    else if (dtype == PLM_BF16) launch_dequantize<PLM_BF16>(codes, scale, m, k, out, s);
    else launch_dequantize<PLM_FP16>(codes, scale, m, k, out, s);
}

}  // namespace plm
