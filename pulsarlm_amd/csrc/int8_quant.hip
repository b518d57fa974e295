// Rows of 8-bit integers: quantizer (tokens' activations, a weight's output channels) and its inverse.
//
// s = max(amax, 1e-12) / 127 in fp32, q the integer nearest to x / s, ties to even, of the exact quotient: the fp32
// quotient of a value next to the border between two codes can round onto the border. With q0 = rint(x * (1 / s)), off by
// at most one, r = x - q0 s is exact in fp32 wherever |r| is near s / 2 (x, q0 s and so r are multiples of s's last bit,
// of s / 2's where q0 = 0), and says on which side of the border x lies.
// A row with an infinity or NaN gets s = NaN and codes 0: every product with it is NaN.
// What bounds it: memory. M = 4096, K 12288, bf16.
#include <algorithm>

#include "dense_gemm.hpp"

namespace plm {

namespace {

// Magnitude bits, ordered as the values; infinity is 0x7f800000 and NaNs lie above.
__device__ __forceinline__ uint32_t magnitude(float f) { return __float_as_uint(f) & 0x7fffffffu; }

struct row_scale {
    float s, inv, half;  // inv == 0: a row that is not finite
};
__device__ __forceinline__ row_scale make_row_scale(uint32_t top) {
    if (top >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.f, 0.f};
    const float s = fmaxf(__uint_as_float(top), 1e-12f) / 127.f;
    return {s, 1.f / s, 0.5f * s};
}
__device__ __forceinline__ int quantized(float x, const row_scale& k) {
    if (k.inv == 0.f) return 0;
    float q = rintf(x * k.inv);
    const float r = fmaf(-q, k.s, x), a = fabsf(r);
    const bool odd = static_cast<int>(q) & 1;
    if (a > k.half || (a == k.half && odd)) q += copysignf(1.f, r);
    return static_cast<int>(q);
}

// Eight consecutive values.
template <plm_dtype D> struct eight {
    u32x4_t v[D == PLM_FP32 ? 2 : 1];
    __device__ __forceinline__ float get(int i) const {
        if constexpr (D == PLM_FP32) return __uint_as_float(v[i >> 2][i & 3]);
        else return from_bits16<D == PLM_BF16>((v[0][i >> 1] >> (16 * (i & 1))) & 0xffffu);
    }
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
template <plm_dtype D> __device__ __forceinline__ uint32_t top_of(const eight<D>& e, uint32_t top) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, magnitude(e.get(i)));
    return top;
}
template <plm_dtype D> __device__ __forceinline__ uint2 codes_of(const eight<D>& e, const row_scale& k) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i >> 2] |= (static_cast<uint32_t>(quantized(e.get(i), k)) & 0xffu) << (8 * (i & 3));
    return make_uint2(w[0], w[1]);
}

template <int T> __device__ __forceinline__ uint32_t block_top(uint32_t top, uint32_t* part) {
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), s)));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < T / 64; ++w) top = max(top, part[w]);
    return top;
}

// A workgroup a row. The first CAP chunks of eight a thread wait in registers for the row's largest; what is past them
// is read again.
template <plm_dtype D, int T, int CAP>
__global__ void __launch_bounds__(T) quantize_int8_kernel(const uint8_t* __restrict__ x, int64_t k, int8_t* __restrict__ codes,
                                                          float* __restrict__ scale) {
    __shared__ uint32_t part[T / 64];
    const int64_t row = blockIdx.x, chunks = k >> 3;
    const uint8_t* from = x + row * k * (D == PLM_FP32 ? 4 : 2);
    uint2* to = reinterpret_cast<uint2*>(codes + row * k);
    eight<D> held[CAP];
#pragma unroll
    for (int c = 0; c < CAP; ++c) held[c] = load_eight<D>(from, threadIdx.x + c * T, threadIdx.x + c * T < chunks);
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < CAP; ++c) top = top_of(held[c], top);
    for (int64_t c = threadIdx.x + CAP * T; c < chunks; c += T) top = top_of(load_eight<D>(from, c, true), top);
    const row_scale s = make_row_scale(block_top<T>(top, part));
    if (threadIdx.x == 0) scale[row] = s.s;
#pragma unroll
    for (int c = 0; c < CAP; ++c)
        if (threadIdx.x + c * T < chunks) to[threadIdx.x + c * T] = codes_of(held[c], s);
    for (int64_t c = threadIdx.x + CAP * T; c < chunks; c += T) to[c] = codes_of(load_eight<D>(from, c, true), s);
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
    for (int64_t i = threadIdx.x; i < k; i += 256) top = max(top, magnitude(load_one<D>(x, row * k + i)));
    const row_scale s = make_row_scale(block_top<256>(top, part));
    if (threadIdx.x == 0) scale[row] = s.s;
    for (int64_t i = threadIdx.x; i < k; i += 256) codes[row * k + i] = static_cast<int8_t>(quantized(load_one<D>(x, row * k + i), s));
}

template <plm_dtype D> void launch_quantize(const void* x, int64_t m, int64_t k, int8_t* codes, float* scale, hipStream_t s) {
    const unsigned grid = static_cast<unsigned>(m);
    const auto* bytes = static_cast<const uint8_t*>(x);
    if (k % 8 != 0 || !aligned(x, 16) || !aligned(codes, 8)) {
        quantize_int8_any_kernel<D><<<grid, 256, 0, s>>>(x, k, codes, scale);
        return;
    }
    // Few rows: many threads each, for loads in flight; many rows fill the GPU by themselves.
    constexpr int CAP = D == PLM_FP32 ? 4 : 8;
    if (m < 2 * cu_count()) quantize_int8_kernel<D, 1024, CAP / 2><<<grid, 1024, 0, s>>>(bytes, k, codes, scale);
    else quantize_int8_kernel<D, 256, CAP><<<grid, 256, 0, s>>>(bytes, k, codes, scale);
}

// Sixteen codes a thread, or one.
template <plm_dtype D, bool WIDE>
__global__ void __launch_bounds__(256) dequantize_int8_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scale, int64_t total,
                                                              int64_t k, void* __restrict__ out) {
    constexpr int N = WIDE ? 16 : 1;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total / N; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t at = i * N;
        const float s = scale[at / k];
        if constexpr (WIDE) {
            const u32x4_t c = *reinterpret_cast<const u32x4_t*>(codes + at);
            float f[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) f[j] = static_cast<float>(static_cast<int8_t>(c[j >> 2] >> (8 * (j & 3)))) * s;
            if constexpr (D == PLM_FP32) {
#pragma unroll
                for (int j = 0; j < 4; ++j) reinterpret_cast<f32x4_t*>(static_cast<float*>(out) + at)[j] = f32x4_t{f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]};
            } else {
                u32x4_t* to = reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(out) + at);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float* g = f + 8 * j;
                    to[j] = u32x4_t{pack2<D == PLM_BF16>(g[0], g[1]), pack2<D == PLM_BF16>(g[2], g[3]), pack2<D == PLM_BF16>(g[4], g[5]), pack2<D == PLM_BF16>(g[6], g[7])};
                }
            }
        } else {
            const float f = static_cast<float>(codes[at]) * s;
            if constexpr (D == PLM_FP32) static_cast<float*>(out)[at] = f;
            else static_cast<uint16_t*>(out)[at] = static_cast<uint16_t>(to_bits16<D == PLM_BF16>(f));
        }
    }
}

template <plm_dtype D> void launch_dequantize(const int8_t* codes, const float* scale, int64_t m, int64_t k, void* out, hipStream_t s) {
    const int64_t total = m * k;
    const bool wide = k % 16 == 0 && aligned(codes, 16) && aligned(out, 16);
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ceil_div(total / (wide ? 16 : 1), 256), int64_t{64} * cu_count()));
    if (wide) dequantize_int8_kernel<D, true><<<grid, 256, 0, s>>>(codes, scale, total, k, out);
    else dequantize_int8_kernel<D, false><<<grid, 256, 0, s>>>(codes, scale, total, k, out);
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
