// Microscaled 4-bit floating point: the storage of an operand and the rounding to it, shared by the
// quantizer and the product.
//
// An operand [rows, K] is stored as
//   codes  [rows, pitch]  two e2m1 codes a byte, the even column in the low nibble, zero behind K
//   scales [ceil(rows / 128)][groups][512]  one byte a block, in tiles of 128 rows x 4 blocks: the byte of
//          (row r of the tile, block j of the group) sits at (r % 32) * 16 + (r / 32) * 4 + j.
// A tile is what one tcgen05.cp of 32 x 128 bits moves into tensor memory, and what the tensor core reads
// from there: 32 lanes x 4 columns, a column holding the four scales of 32 rows.  `groups` covers K rounded
// up to 256 columns (one 128-byte row of codes in shared memory); the scales behind K are zero, because the
// product multiplies them with zero codes and a NaN there would spread.
#pragma once

#include "common.cuh"

namespace samq {
namespace fp4 {

constexpr int KPAD = 256;                       // columns that a pipeline stage of the product covers
constexpr int TILE_ROWS = 128;
constexpr int TILE_BYTES = 512;

// columns per scale
__host__ __device__ constexpr int block_of(int fmt) { return fmt == SAMQ_FP4_MX ? 32 : 16; }
// scale tiles per 256 columns: 2 or 4
__host__ __device__ constexpr int groups_per_kpad(int fmt) { return KPAD / (4 * block_of(fmt)); }
inline int64_t groups_of(int fmt, int64_t K) { return (K + KPAD - 1) / KPAD * groups_per_kpad(fmt); }
inline bool known_format(int fmt) { return fmt == SAMQ_FP4_MX || fmt == SAMQ_FP4_NV; }
// a power of two for which neither the scales nor their reciprocals leave the normal range
inline bool good_global_scale(float g) {
    return g >= 5.42101086e-20f /* 2^-64 */ && g <= 1.84467441e19f /* 2^64 */ && (__builtin_bit_cast(uint32_t, g) & 0x7FFFFFu) == 0;
}

// Eight values to eight e2m1 codes, v[0] in the low nibble: round to nearest, ties to the even code,
// magnitudes beyond 6 become 6 (the conversion instruction's definition).
__device__ __forceinline__ uint32_t pack_e2m1x8(const float* v) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
// the magnitude bits and sign of a 4-bit code as the float it stands for
__device__ __forceinline__ float e2m1_value(uint32_t code) {
    // 0, .5, 1, 1.5, 2, 3, 4, 6 : doubled they are the integers of this table, four bits each
    const float mag = 0.5f * (float)((0xC8643210u >> (4 * (code & 7u))) & 15u);
    return (code & 8u) ? -mag : mag;
}

// Scale of a block from its largest magnitude, given as the bits of |x| (compared as integers, so that a NaN
// or an infinity in the block wins): the stored byte and the scale itself.  A block that is not finite gets
// the format's NaN byte, and the product of anything with it is NaN.
struct Scale { uint32_t byte; float value; };

template <int FMT>
__device__ __forceinline__ Scale block_scale(uint32_t amax_bits, float global_scale) {
    Scale s;
    const bool finite = amax_bits < 0x7F800000u;
    if constexpr (FMT == SAMQ_FP4_MX) {
        // 2^(floor(log2 amax) - 2): the exponent field less two, so that amax lands in [4, 8); zero and
        // subnormal blocks take the smallest scale, 2^-127
        const int e = (int)(amax_bits >> 23) - 2;
        s.byte = finite ? (uint32_t)max(e, 0) : 0xFFu;
        s.value = __uint_as_float(s.byte > 0 ? s.byte << 23 : 0x00400000u);
    } else {
        // amax / (6 g) to e4m3, at most 448, and at least its smallest value 2^-9 (the block's own values are
        // then still resolved below the point where the scale alone would round to zero).  6 g has few
        // significant bits, so the correctly rounded quotient never reaches a tie that amax itself missed.
        const float q = __fdiv_rn(__uint_as_float(amax_bits), 6.0f * global_scale);
        uint16_t two;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(0.0f), "f"(q));
        s.byte = finite ? max((uint32_t)two & 0x7Fu, 1u) : 0x7Fu;
        const uint32_t e = s.byte >> 3, m = s.byte & 7u;
        const float v = e ? __uint_as_float(((e + 120u) << 23) | (m << 20)) : (float)m * 0x1p-9f;
        s.value = finite ? v * global_scale : __uint_as_float(0x7FC00000u);
    }
    if (!finite) s.value = __uint_as_float(0x7FC00000u);
    return s;
}

// x / scale for a finite block.  mxfp4: a product with the exact reciprocal.  nvfp4: the correctly rounded
// quotient (a scale has four significant bits and a border between codes three, so a quotient that rounds to a
// border lies on it).
template <int FMT>
struct ToCode {
    Divider d;
    float inv;
    __device__ __forceinline__ explicit ToCode(const Scale& s) {
        if constexpr (FMT == SAMQ_FP4_MX) inv = __uint_as_float((254u - s.byte) << 23);
        else d = make_divider(s.value);
    }
    __device__ __forceinline__ float operator()(float x) const {
        if constexpr (FMT == SAMQ_FP4_MX) return x * inv;
        else return copysignf(div_exact(x, d), x);        // the correction step loses the sign of -0
    }
};

}  // namespace fp4
}  // namespace samq
