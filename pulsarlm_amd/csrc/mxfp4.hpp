// MXFP4: microscaled 4-bit weights and activations. 32 consecutive K values share a scale
// 2^(b - 127), b one byte (255: NaN), and are e2m1 codes (+-0, 0.5, 1, 1.5, 2, 3, 4, 6).
//
// Tile layout, for weights and for quantized activations alike: [16-row strips][K tiles of 128][1 KiB],
// lane r + 16 g of a tile holding the 16 bytes of row r's block g. That is at once one coalesced
// 16-byte load per lane, the operand of v_mfma_scale_f32_16x16x128_f8f6f4 (whose lane group g carries
// block g, with the block's scale in a byte of the lane's scale register) and, word j converted with
// that one scale, the operand of v_mfma_f32_16x16x32 for K = 32 g + 8 j + 0..7. The scales are
// [groups of 4 strips][K tiles][64 lanes] dwords, byte j that of the group's strip j: one load serves a
// wavefront's four strips, and the matrix instruction picks the byte. Padding rows of a weight, and columns
// past K, hold code and scale 0.
#pragma once

#include <algorithm>

#include "plm_common.hpp"

namespace plm {

constexpr int kMxBlock = 32;
constexpr int64_t kMxMaxSize = int64_t{1} << 19;  // N, K: the byte offsets of one workgroup's buffers stay below kOOB

struct mx_dims {
    int64_t strips, ktiles, groups;  // groups of 4 strips
    int64_t tile_bytes() const { return strips * ktiles * kSubTileBytes; }
    int64_t scale_bytes() const { return groups * ktiles * 256; }
};
inline mx_dims make_mx_dims(int64_t rows, int64_t k) {
    mx_dims d;
    d.strips = ceil_div(rows, kTileN);
    d.ktiles = ceil_div(k, kTileK);
    d.groups = ceil_div(d.strips, 4);
    return d;
}

// A matrix in the tile layout.
struct mx_matrix {
    const uint8_t* codes;
    const uint32_t* scale;
};

__device__ __forceinline__ float mx_scale(uint32_t byte) { return __uint_as_float(byte << 23); }  // 0: read as 2^-127 by the converts

// Eight codes (a word, lowest K first) times their scale: exact in bf16, rounded once to fp16.
template <bool BF16> __device__ __forceinline__ u32x4_t mx_decode(uint32_t w, float s) {
    u32x4_t r;
    if constexpr (BF16) {
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1));
        r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2));
        r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3));
    } else {
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 0));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 1));
        r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 2));
        r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 3));
    }
    return r;
}

// Magnitudes are compared as integers: NaN above infinity above every number.
__device__ __forceinline__ uint32_t mx_magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// Scale byte of a block from its largest magnitude: floor(log2) - 2 + 127, at least 0; infinity or NaN in
// the block makes it 255, which reads as NaN.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t magnitude) {
    const uint32_t e = magnitude >> 23;
    return e == 255u ? 255u : (e < 2u ? 0u : e - 2u);
}
// Codes of eight values under scale byte b: round to nearest, ties to the even code, saturating at 6
// (tests: every bf16 value under twelve scales, and the fp32 numbers on either side of each border).
__device__ __forceinline__ uint32_t mx_encode8(const float (&v)[8], uint32_t b) {
    const float s = mx_scale(b);
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], s, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], s, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], s, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], s, 3);
    return b == 255u ? 0u : q;
}

// 16 x 16 x 128 product of e2m1 operands (16 bytes and a scale register per lane); byte SA / SB of the
// scale registers is used.
template <int SA, int SB>
__device__ __forceinline__ f32x4_t mx_mfma(u32x4_t a, uint32_t sa, u32x4_t b, uint32_t sb, f32x4_t c) {
    const i32x8_t av = __builtin_bit_cast(i32x8_t, u32x8_cat(a, u32x4_t{0, 0, 0, 0}));
    const i32x8_t bv = __builtin_bit_cast(i32x8_t, u32x8_cat(b, u32x4_t{0, 0, 0, 0}));
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, SA, static_cast<int>(sa), SB,
                                                            static_cast<int>(sb));
}

// silu(g) u from the 32-bit sums. 1 / (1 + e^-g) by the hardware's exp2 and reciprocal, each within an ulp
// or two of 32 bits (and zero below 2^-126, g < -87.3): the caller rounds to 16 bits or to e2m1 codes.
__device__ __forceinline__ float mx_sigmoid(float g) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.44269504088896341f));
}
__device__ __forceinline__ float mx_gated(float g, float u) { return g * mx_sigmoid(g) * u; }

// How an output tile leaves: 16-bit sums; h = silu(g) u in 16 bits, with [g | u] kept where asked; or h
// as e2m1 codes in the tile layout, the next product's activations.
enum mx_epilogue { kMxPlain, kMxGated, kMxGatedCodes };

struct mx_output {
    uint16_t* y;         // [M, N], kMxGated: h
    float* gate_up;      // kMxGated: [g | u] [M, 2 N], or null
    uint8_t* codes;      // kMxGatedCodes
    uint8_t* scale;
    int n, ktiles;       // columns; K tiles of the codes' layout
    bool wide;               // four columns a store: N % 4 == 0 and 8-byte aligned pointers
    bool lines;              // eight: N % 8 == 0 and y 16-byte aligned
};

template <bool BF16> __device__ __forceinline__ void mx_store4(uint16_t* p, int col, int n, bool wide, const float (&v)[4]) {
    if (wide) {
        if (col < n) *reinterpret_cast<uint2*>(p) = make_uint2(pack2<BF16>(v[0], v[1]), pack2<BF16>(v[2], v[3]));
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (col + r < n) p[r] = static_cast<uint16_t>(to_bits16<BF16>(v[r]));
    }
}

// Columns col .. col + 3 of one row.
template <bool BF16> __device__ __forceinline__ void mx_store_plain(const mx_output& o, int64_t row, int col, const f32x4_t& v) {
    const float f[4] = {v[0], v[1], v[2], v[3]};
    mx_store4<BF16>(o.y + row * o.n + col, col, o.n, o.wide, f);
}
// [g | u] of columns col .. col + 3 of one row, where the caller keeps them.
__device__ __forceinline__ void mx_store_gate_up(const mx_output& o, int64_t row, int col, const f32x4_t& g, const f32x4_t& u) {
    // Kept in 32 bits: rounded to 16 they cost the gradient as much as its own last rounding does (its error
    // against float64 is 3.0e-3 with bf16 g and u, 2.3e-3 with these; one bf16 rounding is 1.7e-3).
    if (o.gate_up != nullptr) {
        float* p = o.gate_up + row * 2 * o.n + col;
        if (o.wide) {
            if (col < o.n) *reinterpret_cast<f32x4_t*>(p) = g, *reinterpret_cast<f32x4_t*>(p + o.n) = u;
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (col + r < o.n) p[r] = g[r], p[o.n + r] = u[r];
        }
    }
}
__device__ __forceinline__ f32x4_t mx_gated4(const f32x4_t& g, const f32x4_t& u) {
    return f32x4_t{mx_gated(g[0], u[0]), mx_gated(g[1], u[1]), mx_gated(g[2], u[2]), mx_gated(g[3], u[3])};
}
// One block of 32 columns (slices 2 block and 2 block + 1 of 16) of 16 rows, held by a wavefront: lane
// r + 16 g has row r's columns 4 g .. 4 g + 3 of either slice. All 64 lanes take part.
__device__ __forceinline__ void mx_store_codes(const mx_output& o, int strip, int block, const f32x4_t (&g)[2], const f32x4_t (&u)[2]) {
    const int lane = __lane_id();
    float h[8];
    uint32_t top = 0;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        h[r] = mx_gated(g[r >> 2][r & 3], u[r >> 2][r & 3]);
        top = max(top, mx_magnitude(h[r]));
    }
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16)));
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
    const uint32_t b = mx_scale_byte(top);
    const uint32_t q = mx_encode8(h, b);
    const int64_t tile = static_cast<int64_t>(strip) * o.ktiles + (block >> 2);
    const int at = (lane & 15) + 16 * (block & 3);
    uint16_t* c = reinterpret_cast<uint16_t*>(o.codes + tile * kSubTileBytes + at * 16) + (lane >> 4);
    c[0] = static_cast<uint16_t>(q);
    c[4] = static_cast<uint16_t>(q >> 16);
    uint8_t* s = o.scale + ((static_cast<int64_t>(strip >> 2) * o.ktiles + (block >> 2)) * 64 + at) * 4 + (strip & 3);
    if (lane < 16) *s = static_cast<uint8_t>(b);
    if (32 * (block + 1) >= o.n) {  // the last tile's blocks past the end are read, too
        for (int e = (block & 3) + 1; e < 4; ++e) {
            c += 16 * 8;
            s += 16 * 4;
            c[0] = 0;
            c[4] = 0;
            if (lane < 16) *s = 0;
        }
    }
}

inline mx_output mx_make_output(void* y, void* gate_up, int64_t n) {
    mx_output o{};
    o.y = static_cast<uint16_t*>(y);
    o.gate_up = static_cast<float*>(gate_up);
    o.n = static_cast<int>(n);
    o.lines = n % 8 == 0 && aligned(y, 16);
    o.wide = n % 4 == 0 && aligned(y, 8) && aligned(gate_up, 16);
    return o;
}

// 16-bit x [M, K] to the tile layout.
void launch_mx_quantize_tiles(const void* x, bool bf16, int64_t m, int64_t k, uint8_t* codes, uint32_t* scale, hipStream_t s);

// The products. x16 is the 16-bit x [M, K], or xq its codes; w1 is null for plain products.
struct mx_product {
    const uint16_t* x16;
    mx_matrix xq;
    mx_matrix w0, w1;
    int64_t m, n, k;
    float* partial;  // W4A4, plain: room for the sums of K splits (mx_tiles_w4a4_bytes), or null
    bool bf16;
    mx_epilogue epilogue;
    mx_output out;
};
// out[i] = sum over s of partial[s][i], in order of s; count a multiple of 4, out 8-byte aligned.
void launch_mx_combine(bool bf16, const float* partial, int64_t count, int splits, uint16_t* out, hipStream_t s);
// The kernel for few rows: true where it has launched. quantize_x: it quantizes x16 itself.
bool launch_mx_rows(const mx_product& p, bool quantize_x, hipStream_t s);

}  // namespace plm
