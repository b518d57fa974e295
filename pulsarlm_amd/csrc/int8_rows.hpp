// The rule of the 8-bit row quantizer: s = max(amax, 1e-12) / 127 in fp32, q the integer nearest to x / s, ties to even,
// of the exact quotient: the fp32 quotient of a value next to the border between two codes can round onto the border. With
// q0 = rint(x * (1 / s)), off by at most one, r = x - q0 s is exact in fp32 wherever |r| is near s / 2 (x, q0 s and so r
// are multiples of s's last bit, of s / 2's where q0 = 0), and says on which side of the border x lies. |r| < s / 2 almost
// always, so that eight values check their largest |r| and seldom look further: 4 operations a value and the packing.
// A row with an infinity or NaN gets s = NaN and codes 0: every product with it is NaN.
#pragma once

#include "plm_common.hpp"

namespace plm {

namespace {

// Magnitude bits, ordered as the values; infinity is 0x7f800000 and NaNs lie above.
__device__ __forceinline__ uint32_t int8_magnitude(float f) { return __float_as_uint(f) & 0x7fffffffu; }

struct int8_scale {
    float s, inv, half;
    bool finite;
};
__device__ __forceinline__ int8_scale make_int8_scale(uint32_t top) {
    if (top >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.f, 0.f, false};
    const float s = fmaxf(__uint_as_float(top), 1e-12f) / 127.f;
    return {s, 1.f / s, 0.5f * s, true};
}

// Added to a number of magnitude below 2^22, 1.5 * 2^23 leaves the nearest integer, ties to even, in the low bits.
constexpr float kInt8Magic = 12582912.f;

// The codes of N values (4 or 8) of a row that is finite, four to a dword.
template <int N> __device__ __forceinline__ void int8_codes(const float (&x)[N], const int8_scale& k, uint32_t (&codes)[N / 4]) {
    float u[N], worst = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        u[i] = fmaf(x[i], k.inv, kInt8Magic);
        worst = fmaxf(worst, fabsf(fmaf(kInt8Magic - u[i], k.s, x[i])));
    }
    if (worst >= k.half) {  // a tie, or a quotient rounded over the border
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float r = fmaf(kInt8Magic - u[i], k.s, x[i]), a = fabsf(r);
            if (a > k.half || (a == k.half && (__float_as_uint(u[i]) & 1u))) u[i] += copysignf(1.f, r);
        }
    }
#pragma unroll
    for (int d = 0; d < N / 4; ++d) {
        const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(u[4 * d + 1]), __float_as_uint(u[4 * d]), 0x0c0c0400);
        const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(u[4 * d + 3]), __float_as_uint(u[4 * d + 2]), 0x04000c0c);
        codes[d] = lo | hi;
    }
}

// The largest magnitude of 16-bit values, two to a dword, as running maxima of both halves; and its fp32 bits.
typedef __attribute__((ext_vector_type(2))) uint16_t u16x2_t;
__device__ __forceinline__ uint32_t top_16(uint32_t top, uint32_t two) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, top), __builtin_bit_cast(u16x2_t, two & 0x7fff7fffu)));
}
template <bool BF16> __device__ __forceinline__ uint32_t top_bits(uint32_t top) {
    return int8_magnitude(from_bits16<BF16>(max(top & 0xffffu, top >> 16)));
}
// Eight 16-bit values in fp32.
template <bool BF16> __device__ __forceinline__ void eight_values(const u32x4_t& v, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = from_bits16<BF16>(v[i] & 0xffffu), x[2 * i + 1] = from_bits16<BF16>(v[i] >> 16);
}

}  // namespace

}  // namespace plm
