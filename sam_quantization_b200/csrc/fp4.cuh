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
#include <type_traits>

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
inline int check_global_scale(int fmt, float g) {
    if (!good_global_scale(g)) return fail(SAMQ_ERR_BAD_ARG, "global_scale must be a power of two between 2^-64 and 2^64");
    if (fmt == SAMQ_FP4_MX && g != 1.0f) return fail(SAMQ_ERR_BAD_ARG, "mxfp4 has no global scale: its block scales reach every exponent");
    return SAMQ_OK;
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
// the eight values of eight codes
__device__ __forceinline__ void unpack_e2m1x8(uint32_t codes, float2 (&v)[4]) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(codes));
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
}

// Sixteen columns of a row as the threads hold them: packed pairs of a 16-bit type, or fp32.
template <typename T> struct Chunk {
    uint32_t w[8];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 0;
    }
    __device__ __forceinline__ void set(int i, T v) {
        const uint32_t b = *reinterpret_cast<const uint16_t*>(&v);
        w[i >> 1] = (i & 1) ? (w[i >> 1] & 0xFFFFu) | (b << 16) : b;
    }
    __device__ __forceinline__ float2 pair(int i) const {
        if constexpr (sizeof(T) == 2) {
            if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            else return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
        }
    }
    // values that bfloat16 holds exactly
    __device__ __forceinline__ void set_pair(int i, float2 v) { w[i] = (__float_as_uint(v.x) >> 16) | (__float_as_uint(v.y) & 0xFFFF0000u); }
    // the largest |x| as fp32 bits; a NaN or an infinity counts as larger than every number
    __device__ __forceinline__ uint32_t amax_bits() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
        m = max(m & 0xFFFFu, m >> 16);
        if constexpr (std::is_same<T, __half>::value) {
            const uint16_t h = (uint16_t)m;
            return __float_as_uint(__half2float(*reinterpret_cast<const __half*>(&h)));
        } else {
            return m << 16;
        }
    }
};
template <> struct Chunk<float> {
    float f[16];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = 0.0f;
    }
    __device__ __forceinline__ void set(int i, float v) { f[i] = v; }
    __device__ __forceinline__ float2 pair(int i) const { return make_float2(f[2 * i], f[2 * i + 1]); }
    __device__ __forceinline__ void set_pair(int i, float2 v) { f[2 * i] = v.x; f[2 * i + 1] = v.y; }
    __device__ __forceinline__ uint32_t amax_bits() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(f[i]) & 0x7FFFFFFFu);
        return m;
    }
};

// 32 bytes in one access (the address on 32 bytes)
__device__ __forceinline__ void load32(const void* p, uint32_t* w) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p));
}
__device__ __forceinline__ void store32(void* p, const uint32_t* w) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

// how a row's chunks may be accessed: by 32 bytes, by 16, or element by element
enum Access { BY_ELEMENT = 0, BY_16 = 1, BY_32 = 2 };
inline int row_access(const void* base, int64_t ld_bytes) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(base) | (uintptr_t)ld_bytes;
    return (a & 31) == 0 ? BY_32 : (a & 15) == 0 ? BY_16 : BY_ELEMENT;
}

// `n` (1 to 16) columns at x, zeros behind them
template <typename T>
__device__ __forceinline__ void load_chunk(Chunk<T>& c, const T* x, int n, int access) {
    constexpr int WORDS = 16 * (int)sizeof(T) / 4;
    uint32_t* w = reinterpret_cast<uint32_t*>(&c);
    if (n >= 16 && access == BY_32) {
#pragma unroll
        for (int i = 0; i < WORDS; i += 8) load32(reinterpret_cast<const uint32_t*>(x) + i, w + i);
    } else if (n >= 16 && access == BY_16) {
#pragma unroll
        for (int i = 0; i < WORDS; i += 4) *reinterpret_cast<uint4*>(w + i) = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(x) + i);
    } else {
        c.zero();
#pragma unroll
        for (int i = 0; i < 16; ++i) if (i < n) c.set(i, x[i]);
    }
}

// Scale of a block from its largest magnitude, given as the bits of |x| (compared as integers, so that a NaN
// or an infinity in the block wins): the stored byte and the scale itself.  A block that is not finite gets
// the format's NaN byte, and the product of anything with it is NaN.
struct Scale { uint32_t byte; float value; };

template <int FMT>
__device__ __forceinline__ Scale block_scale(uint32_t amax_bits, float global_scale, float inv_global_scale) {
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
        // then still resolved below the point where the scale alone would round to zero).  6 has few
        // significant bits, so the correctly rounded quotient never reaches a tie that amax itself missed.
        // g is a power of two: amax / g is exact, and a sixth of it is one correctly rounded quotient by a constant.  Beyond
        // 6 * 448 the scale saturates; a is held there, since the correction of an infinite a would be a NaN.
        const float a = fminf(__uint_as_float(amax_bits) * inv_global_scale, 2688.0f);
        const float sixth = 1.0f / 6.0f;
        const float q0 = a * sixth;
        const float q = fmaf(fmaf(-q0, 6.0f, a), sixth, q0);
        uint16_t two;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(0.0f), "f"(q));
        s.byte = finite ? max((uint32_t)two & 0x7Fu, 1u) : 0x7Fu;
        uint32_t h;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)s.byte));
        s.value = __low2float(*reinterpret_cast<const __half2*>(&h)) * global_scale;
    }
    if (!finite) s.value = __uint_as_float(0x7FC00000u);
    return s;
}

// x / scale for a finite block, two values at a time.  mxfp4: a product with the exact reciprocal.  nvfp4: Markstein's
// correction of an approximate quotient, y = y0 + (x - y0 s) / s: exact where x / s is a number of few bits, so on every
// border between codes, and a correct rounding elsewhere up to 2^-45; a scale has four significant bits and a border
// three, so a value beside a border stays beside it.  The correction loses the sign of -0, which is put back; and it needs
// a quotient within fp32 (see hold_far).
template <int FMT>
struct ToCode {
    float2 s2, inv2;
    __device__ __forceinline__ explicit ToCode(const Scale& s) {
        float inv;
        if constexpr (FMT == SAMQ_FP4_MX) inv = __uint_as_float((254u - s.byte) << 23);
        else asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s.value));
        inv2 = make_float2(inv, inv);
        s2 = make_float2(-s.value, -s.value);
    }
    __device__ __forceinline__ float2 operator()(float2 x) const {
        if constexpr (FMT == SAMQ_FP4_MX) return __fmul2_rn(x, inv2);
        const float2 y0 = __fmul2_rn(x, inv2);
        const float2 y = __ffma2_rn(__ffma2_rn(y0, s2, x), inv2, y0);
        return make_float2(copysignf(y.x, x.x), copysignf(y.y, x.y));
    }
};

// The codes of a chunk under its block's scale, eight a word; zero where the block is not finite.
template <int FMT, typename T>
__device__ __forceinline__ uint2 encode_chunk(const Chunk<T>& c, const Scale& s, bool finite) {
    const ToCode<FMT> to_code(s);
    float v[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 y = to_code(c.pair(i));
        v[2 * i] = y.x; v[2 * i + 1] = y.y;
    }
    const uint2 q = make_uint2(pack_e2m1x8(v), pack_e2m1x8(v + 8));
    return finite ? q : make_uint2(0u, 0u);
}

// An nvfp4 block far beyond the largest scale: x / s may leave fp32.  Magnitudes from 6 s on have the same code, so they are
// held at 8 s.  Only where the largest scale 448 g is below 1, since |x| < 2^128, and not in fp16, whose values end at 2^16:
// the branch is the same in the whole grid (a bound on every element would cost 32768 x 5120 bf16 a seventh of its time).
template <int FMT, typename T>
__device__ __forceinline__ void hold_far(Chunk<T>& c, const Scale& s, float global_scale) {
    if constexpr (FMT == SAMQ_FP4_NV && !std::is_same<T, __half>::value) {
        if (global_scale < 0x1p-8f) {
            const float most = 8.0f * s.value;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 x = c.pair(i);
                c.set_pair(i, make_float2(fminf(fmaxf(x.x, -most), most), fminf(fmaxf(x.y, -most), most)));
            }
        }
    }
}

}  // namespace fp4
}  // namespace samq
