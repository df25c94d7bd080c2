// RMS norm of the residual stream with an 8-bit output.
//
//   h = T(x + residual)                      the new residual stream, rounded as it is stored
//   y = h * rsqrt(mean(h^2) + eps) * w       fp32, never rounded to the tensor type
//   s = max(max|y|, 1e-5) / q_max            one scale per row
//   q = round_half_even(y / s)
//
// One pass: a row stays in registers between the two reductions (sum of squares, largest magnitude).  Bound: HBM,
// 2 + 2 + 2 + 1 bytes an element of a 16-bit type (x, residual, h, q), 2 more for the dequantized values.  A row is kept
// in its own type (60 registers instead of 110 of fp32: 66.3 -> 61.5 us).  Measured, 32768 x 1280 fp16 with residual and
// values: 61.5 us, 6.1 TB/s; without either 28.6; 1278 columns (4-byte accesses) 74, 1279 80; bfloat16 within 6 % of these.
#include "common.cuh"
#include <float.h>
#include <type_traits>

namespace samq {

namespace {

struct RmsNormParams {
    const void* x; int64_t ldx;
    const void* residual; int64_t ldr;
    const void* weight;
    void* residual_out; int64_t ldo;
    int8_t* q; float* scale; void* fq;
    int64_t M; int K;
    float eps, inv_k, qmax;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// the larger of a and |b|; a NaN wins
__device__ __forceinline__ float max_abs_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
    return r;
}

template <int BYTES> struct RawOf;
template <> struct RawOf<16> { using type = uint4; };
template <> struct RawOf<8>  { using type = uint2; };
template <> struct RawOf<4>  { using type = uint32_t; };
template <> struct RawOf<2>  { using type = uint16_t; };
template <> struct RawOf<1>  { using type = uint8_t; };

// E elements of a row in the tensor type, loaded and stored at once, widened to fp32 pairs where they are used (E = 1: the
// second of the pair is 0)
template <typename T, int E> struct Vec {
    static constexpr int P = E == 1 ? 1 : E / 2;
    using Raw = typename RawOf<E * (int)sizeof(T)>::type;
    union { Raw raw; T t[E]; };
    __device__ __forceinline__ Vec() {}
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int j = 0; j < E; ++j) t[j] = Elem<T>::down(0.0f);
    }
    __device__ __forceinline__ void load(const T* p) {
        raw = *reinterpret_cast<const Raw*>(p);
    }
    __device__ __forceinline__ void load_each(const T* p) {
#pragma unroll
        for (int j = 0; j < E; ++j) t[j] = p[j];
    }
    __device__ __forceinline__ void store(T* p) const {
        *reinterpret_cast<Raw*>(p) = raw;
    }
    __device__ __forceinline__ float2 pair(int i) const {
        if constexpr (E == 1) return make_float2(Elem<T>::up(t[0]), 0.0f);
        else return make_float2(Elem<T>::up(t[2 * i]), Elem<T>::up(t[2 * i + 1]));
    }
    __device__ __forceinline__ void set(int i, float2 v) {
        if constexpr (E == 1) t[0] = Elem<T>::down(v.x);
        else if constexpr (std::is_same<T, __half>::value) *reinterpret_cast<__half2*>(t + 2 * i) = __float22half2_rn(v);
        else if constexpr (std::is_same<T, __nv_bfloat16>::value) *reinterpret_cast<__nv_bfloat162*>(t + 2 * i) = __float22bfloat162_rn(v);
        else { t[2 * i] = v.x; t[2 * i + 1] = v.y; }
    }
};

// a barrier of the RW warps of a block's `sub`-th row, and of what they have stored (numbers known when compiled: a block whose
// barriers go by a register reserves all sixteen, and only four such fit an SM)
template <int RW>
__device__ __forceinline__ void row_sync(int sub) {
    if constexpr (RW == 1) __syncwarp();
    else if (RW > 2 || sub == 0) asm volatile("bar.sync 1, %0;" ::"n"(RW * 32) : "memory");
    else asm volatile("bar.sync 2, %0;" ::"n"(RW * 32) : "memory");
}
// the sum (or the largest, of values that are not negative) over the threads of a row; `red`: RW floats of the row
template <int RW, bool MAX>
__device__ __forceinline__ float row_reduce(float v, int sub, int t, float* red) {
    v = MAX ? __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v))) : warp_sum(v);
    if constexpr (RW > 1) {
        row_sync<RW>(sub);                                         // `red` has been read
        if ((t & 31) == 0) red[t >> 5] = v;
        row_sync<RW>(sub);
        v = red[0];
#pragma unroll 1
        for (int w = 1; w < RW; ++w) v = MAX ? max_abs_nan(v, red[w]) : v + red[w];
    }
    return v;
}

// A row whose squares leave fp32, or lose bits below it where eps does not cover them, and a row of zeros without an eps (which
// stays one).  y does not change when h is scaled by a power of two and eps by its square, so the row is brought to where
// its largest element, or the root of eps, is near 1.  It is read again, element by element: kept out of the kernel's
// registers (in line, the branch took ordinary rows of bfloat16 from 64 to 80).
template <typename T, int RW>
__device__ __noinline__ void scaled_row(const RmsNormParams p, int64_t row, int sub, int t, float* red) {
    constexpr int T_ROW = RW * 32;
    const T* h = p.residual != nullptr ? static_cast<const T*>(p.residual_out) + row * p.ldo : static_cast<const T*>(p.x) + row * p.ldx;
    const T* w = static_cast<const T*>(p.weight);
    row_sync<RW>(sub);                                             // the row's sums with the residual have been stored
    float m = 0.0f;
#pragma unroll 1
    for (int k = t; k < p.K; k += T_ROW) m = fmaxf(m, fabsf(Elem<T>::up(h[k])));
    m = row_reduce<RW, true>(m, sub, t, red);
    float c = 1.0f;                                                // 2^-126 to 2^126; an infinity stays one, and its row ends as NaN
    if (m > 0.0f && m <= FLT_MAX) c = __uint_as_float((254u - min(max(__float_as_uint(fmaxf(m, sqrtf(p.eps))) >> 23, 1u), 253u)) << 23);
    float sum = 0.0f;
#pragma unroll 1
    for (int k = t; k < p.K; k += T_ROW) { const float f = Elem<T>::up(h[k]) * c; sum = fmaf(f, f, sum); }
    const float mean = fmaf(row_reduce<RW, false>(sum, sub, t, red), p.inv_k, p.eps * c * c);
    const float u = mean == 0.0f ? 0.0f : rsqrtf(mean);
    float amax = 0.0f;
#pragma unroll 1
    for (int k = t; k < p.K; k += T_ROW) amax = max_abs_nan(amax, Elem<T>::up(h[k]) * c * u * Elem<T>::up(w[k]));
    amax = row_reduce<RW, true>(fabsf(amax), sub, t, red);
    const bool finite = __float_as_uint(amax) < 0x7F800000u;
    const float s = finite ? __fdiv_rn(fmaxf(amax, 1e-5f), p.qmax) : __uint_as_float(0x7FC00000u);
    if (t == 0 && p.scale != nullptr) p.scale[row] = s;
#pragma unroll 1
    for (int k = t; k < p.K; k += T_ROW) {
        const float q = rintf(__fdiv_rn(Elem<T>::up(h[k]) * c * u * Elem<T>::up(w[k]), s));
        if (p.q != nullptr) p.q[row * (int64_t)p.K + k] = (int8_t)(finite ? (int)q : 0);
        if (p.fq != nullptr) static_cast<T*>(p.fq)[row * (int64_t)p.K + k] = Elem<T>::down(q * s);
    }
}

// E elements a load (the widest that every row of every tensor starts on), NV loads a thread, RW warps a row.
// ODD (E = 2): an odd number of columns side by side.  Even rows start on a pair, odd rows one element before one; so the
// pairs of an odd row begin at its second element, and each row has one element left, its first or its last, which its last
// thread takes.
template <typename T, int E, int NV, int RW, bool RES, bool ODD>
__global__ void __launch_bounds__(RW >= 4 ? RW * 32 : 128, 1)
rms_norm_quant_kernel(const RmsNormParams p)
{
    using V = Vec<T, E>;
    constexpr int P = V::P;
    constexpr int ROWS = RW >= 4 ? 1 : 4 / RW;     // rows of a block
    constexpr int T_ROW = RW * 32;                 // threads of a row
    __shared__ float red_sum[RW > 1 ? ROWS * RW : 1];
    __shared__ float red_max[RW > 1 ? ROWS * RW : 1];
    const int sub = threadIdx.x / T_ROW, t = threadIdx.x % T_ROW;
    const int64_t row = (int64_t)blockIdx.x * ROWS + sub;
    // loads of this thread; rows behind the last one only keep the barriers company
    const int nv = row < p.M ? (p.K / E - t + T_ROW - 1) / T_ROW : 0;
    const int start = t * E + (ODD ? (int)(row & 1) : 0);          // column of the first load
    const bool extra = ODD && t == T_ROW - 1 && row < p.M;         // this thread has the row's single element
    const int alone = (row & 1) ? 0 : p.K - 1;

    V h[NV];
    {
        const T* x = static_cast<const T*>(p.x) + row * p.ldx + start;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            h[v].zero();
            if (v < nv) h[v].load(x + v * T_ROW * E);
        }
    }
    float h1 = 0.0f, y1 = 0.0f;                                    // of the single element
    if (extra) h1 = Elem<T>::up(static_cast<const T*>(p.x)[row * p.ldx + alone]);
    if constexpr (RES) {
        const T* res = static_cast<const T*>(p.residual) + row * p.ldr + start;
        T* h_out = static_cast<T*>(p.residual_out) + row * p.ldo + start;
        V r[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (v < nv) r[v].load(res + v * T_ROW * E);
        if (extra) {
            const T sum1 = Elem<T>::down(h1 + Elem<T>::up(static_cast<const T*>(p.residual)[row * p.ldr + alone]));
            static_cast<T*>(p.residual_out)[row * p.ldo + alone] = sum1;
            h1 = Elem<T>::up(sum1);
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (v >= nv) continue;
#pragma unroll
            for (int i = 0; i < P; ++i) h[v].set(i, __fadd2_rn(h[v].pair(i), r[v].pair(i)));     // rounded as it is stored
            h[v].store(h_out + v * T_ROW * E);
        }
    }
    float2 sum2 = make_float2(ODD ? h1 * h1 : 0.0f, 0.0f);
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const float2 f = h[v].pair(i);
            sum2 = __ffma2_rn(f, f, sum2);
        }
    float sum = warp_sum(sum2.x + sum2.y);
    if constexpr (RW > 1) {
        if ((t & 31) == 0) red_sum[sub * RW + (t >> 5)] = sum;
        __syncthreads();
        sum = red_sum[sub * RW];
#pragma unroll
        for (int w = 1; w < RW; ++w) sum += red_sum[sub * RW + w];
    }
    const float u = rsqrtf(fmaf(sum, p.inv_k, p.eps));
    const float2 u2 = make_float2(u, u);

    float amax = 0.0f;
    if (extra) {
        y1 = h1 * u * Elem<T>::up(static_cast<const T*>(p.weight)[alone]);
        amax = max_abs_nan(amax, y1);
    }
    float2 y[NV][P];
    const T* w = static_cast<const T*>(p.weight) + start;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        if (v >= nv) continue;
        V wv;
        if constexpr (ODD) wv.load_each(w + v * T_ROW * E);
        else wv.load(w + v * T_ROW * E);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            y[v][i] = __fmul2_rn(__fmul2_rn(h[v].pair(i), u2), wv.pair(i));
            amax = max_abs_nan(amax, y[v][i].x);
            if constexpr (E > 1) amax = max_abs_nan(amax, y[v][i].y);
        }
    }
    // non-negative floats and NaNs order as integers do
    amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax) & 0x7FFFFFFFu));
    if constexpr (RW > 1) {
        if ((t & 31) == 0) red_max[sub * RW + (t >> 5)] = amax;
        __syncthreads();
        amax = red_max[sub * RW];
#pragma unroll
        for (int k = 1; k < RW; ++k) amax = max_abs_nan(amax, red_max[sub * RW + k]);
    }
    if (row >= p.M) return;
    // The squares have left fp32 (u = 0), or are so small that some may have been lost and eps does not hide it.  All threads of a
    // row take the same way; the rows of a block share no barrier from here on.
    if (u == 0.0f || u > 0x1p35f) {
        scaled_row<T, RW>(p, row, sub, t, red_max + sub * RW);
        return;
    }
    // a row with a NaN or an infinity has a NaN scale and zero codes
    const bool finite = (__float_as_uint(amax) & 0x7FFFFFFFu) < 0x7F800000u;
    const float s = finite ? __fdiv_rn(fmaxf(amax, 1e-5f), p.qmax) : __uint_as_float(0x7FC00000u);
    if (t == 0 && p.scale != nullptr) p.scale[row] = s;
    // y / s, correctly rounded (a multiply by the reciprocal and one correction), plus 1.5 * 2^23: the sum rounds the
    // quotient half to even to an integer, whose low byte is the code.  |y / s| <= q_max (1 + 2^-23), so none is clamped.
    const float inv = finite ? __frcp_rn(s) : 0.0f;
    const float2 inv2 = make_float2(inv, inv), ns2 = make_float2(-s, -s), magic2 = make_float2(kRoundMagic, kRoundMagic);
    const float2 s2 = make_float2(s, s), nmagic2 = make_float2(-kRoundMagic, -kRoundMagic);
    int8_t* q_out = p.q == nullptr ? nullptr : p.q + row * (int64_t)p.K + start;
    T* fq = p.fq == nullptr ? nullptr : static_cast<T*>(p.fq) + row * (int64_t)p.K + start;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        if (v >= nv) continue;
        const int c = v * T_ROW * E;
        uint32_t code[2 * P];
        V o;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const float2 y0 = __fmul2_rn(y[v][i], inv2);
            const float2 z = __ffma2_rn(__ffma2_rn(y0, ns2, y[v][i]), inv2, y0);
            const float2 m = __fadd2_rn(z, magic2);
            code[2 * i] = finite ? __float_as_uint(m.x) : 0u;
            code[2 * i + 1] = finite ? __float_as_uint(m.y) : 0u;
            o.set(i, __fmul2_rn(__fadd2_rn(m, nmagic2), s2));
        }
        if (q_out != nullptr) {
            if constexpr (E == 1) {
                q_out[c] = (int8_t)(code[0] & 0xFFu);
            } else if constexpr (E == 2) {
                *reinterpret_cast<uint16_t*>(q_out + c) = (uint16_t)__byte_perm(code[0], code[1], 0x0040);
            } else {
                uint32_t word[E / 4];
#pragma unroll
                for (int k = 0; k < E / 4; ++k)
                    word[k] = __byte_perm(__byte_perm(code[4 * k], code[4 * k + 1], 0x0040), __byte_perm(code[4 * k + 2], code[4 * k + 3], 0x0040), 0x5410);
                if constexpr (E == 8) *reinterpret_cast<uint2*>(q_out + c) = make_uint2(word[0], word[1]);
                else *reinterpret_cast<uint32_t*>(q_out + c) = word[0];
            }
        }
        if (fq != nullptr) o.store(fq + c);
    }
    if (extra) {
        const float y0 = y1 * inv, m = fmaf(fmaf(y0, -s, y1), inv, y0) + kRoundMagic;
        if (p.q != nullptr) p.q[row * (int64_t)p.K + alone] = (int8_t)(finite ? __float_as_uint(m) & 0xFFu : 0u);
        if (p.fq != nullptr) static_cast<T*>(p.fq)[row * (int64_t)p.K + alone] = Elem<T>::down((m - kRoundMagic) * s);
    }
}

template <typename T, int E, int NV, int RW, bool ODD = false>
int launch(const RmsNormParams& p, cudaStream_t st) {
    constexpr int ROWS = RW >= 4 ? 1 : 4 / RW;
    const int64_t blocks = (p.M + ROWS - 1) / ROWS;
    if (blocks > 2147483647LL) return fail(SAMQ_ERR_TOO_LARGE, "RMS norm of %lld rows is too large", (long long)p.M);
    const int threads = RW >= 4 ? RW * 32 : 128;
    if (p.residual != nullptr) rms_norm_quant_kernel<T, E, NV, RW, true, ODD><<<(unsigned)blocks, threads, 0, st>>>(p);
    else rms_norm_quant_kernel<T, E, NV, RW, false, ODD><<<(unsigned)blocks, threads, 0, st>>>(p);
    SAMQ_CUDA_TRY(cudaGetLastError());
    return SAMQ_OK;
}

// The fewest warps whose threads hold the row in NV loads each, 1 to 32.
template <typename T, int E, int NV, bool ODD = false>
int launch_warps(int64_t loads, const RmsNormParams& p, cudaStream_t st) {
    if (loads <= 32 * NV) return launch<T, E, NV, 1, ODD>(p, st);
    if (loads <= 64 * NV) return launch<T, E, NV, 2, ODD>(p, st);
    if (loads <= 128 * NV) return launch<T, E, NV, 4, ODD>(p, st);
    if (loads <= 256 * NV) return launch<T, E, NV, 8, ODD>(p, st);
    if (loads <= 512 * NV) return launch<T, E, NV, 16, ODD>(p, st);
    return launch<T, E, NV, 32, ODD>(p, st);
}

// `e` elements: the widest access for all rows; odd: all rows as ODD needs them (see the caller)
template <typename T>
int launch_rms_norm(const RmsNormParams& p, int e, bool odd, cudaStream_t st) {
    constexpr int E = Elem<T>::kPerVec;
    // 5 vectors: 1280 columns of a 16-bit type are one warp's, with no lane idle
    if (e == E && p.K <= 1024 * 5 * E) return launch_warps<T, E, 5>(p.K / E, p, st);
    // narrower accesses: more warps a row and fewer elements each
    if constexpr (E == 8) { if (e == 4) return launch_warps<T, 4, 8>(p.K / 4, p, st); }
    if (e >= 2 && p.K <= 1024 * 8 * 2) return launch_warps<T, 2, 8>(p.K / 2, p, st);
    // odd widths: pairs once single elements take more than a warp a row.  us, elements / pairs, fp16: 65536 x 255 38.9 / 45.0,
    // 32768 x 301 34.8 / 26.6, 32768 x 1279 131 / 82, 8192 x 8191 250 / 182
    if constexpr (sizeof(T) == 2) { if (odd && p.K > 256 && p.K < 1024 * 8 * 2) return launch_warps<T, 2, 8, true>(p.K / 2, p, st); }
    if (p.K <= 1024 * 8) return launch_warps<T, 1, 8>(p.K, p, st);
    return launch<T, 1, 32, 32>(p, st);
}

}  // namespace

int rms_norm_quant_dispatch(const void* x, const void* residual, const void* weight, int dtype, int64_t M, int64_t K,
                            int64_t ldx, int64_t ldr, float eps, int n_bits, void* residual_out, int64_t ldo,
                            int8_t* q, float* scale, void* fq, void* stream)
{
    if (M < 0 || K <= 0) return fail(SAMQ_ERR_BAD_ARG, "bad shape M=%lld K=%lld", (long long)M, (long long)K);
    if (dtype != SAMQ_F16 && dtype != SAMQ_BF16 && dtype != SAMQ_F32) return fail(SAMQ_ERR_BAD_ARG, "unknown dtype %d", dtype);
    if (n_bits < 2 || n_bits > 8) return fail(SAMQ_ERR_BAD_ARG, "n_bits must lie between 2 and 8, got %d", n_bits);
    if (!(eps >= 0.0f)) return fail(SAMQ_ERR_BAD_ARG, "eps must not be negative");
    if (K > 32768) return fail(SAMQ_ERR_TOO_LARGE, "RMS norm holds a row in registers: K=%lld is beyond 32768", (long long)K);
    if (M == 0) return SAMQ_OK;
    if (x == nullptr || weight == nullptr) return fail(SAMQ_ERR_BAD_ARG, "x and weight must not be null");
    if ((residual == nullptr) != (residual_out == nullptr)) return fail(SAMQ_ERR_BAD_ARG, "residual and residual_out come together");
    if (ldx < K || (residual != nullptr && (ldr < K || ldo < K))) return fail(SAMQ_ERR_BAD_ARG, "leading dimension smaller than K");
    const size_t esz = dtype == SAMQ_F32 ? 4 : 2;
    const uintptr_t all = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(weight) |
                          reinterpret_cast<uintptr_t>(residual_out) | reinterpret_cast<uintptr_t>(fq);
    if (all & (esz - 1)) return fail(SAMQ_ERR_ALIGNMENT, "tensors must be aligned to their elements");
    RmsNormParams p;
    p.x = x; p.ldx = ldx; p.residual = residual; p.ldr = residual ? ldr : 0; p.weight = weight;
    p.residual_out = residual_out; p.ldo = residual ? ldo : 0; p.q = q; p.scale = scale; p.fq = fq;
    p.M = M; p.K = (int)K; p.eps = eps; p.inv_k = 1.0f / (float)K; p.qmax = (float)((1 << (n_bits - 1)) - 1);
    // Every address and pitch that a row starts by, in bytes of the tensor type (the codes' scaled to it): the largest power of
    // two that divides them all is the widest access, up to 16 bytes.
    const uintptr_t starts = all | reinterpret_cast<uintptr_t>(q) * esz | (uintptr_t)((K | ldx | p.ldr | p.ldo) * (int64_t)esz) | 16;
    const int e = (int)((starts & (~starts + 1)) / esz);
    const uintptr_t bases = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(residual_out) |
                            reinterpret_cast<uintptr_t>(fq) | reinterpret_cast<uintptr_t>(q) * 2;
    const bool odd = (bases & 3) == 0 && (K & ldx & (residual ? ldr & ldo : 1) & 1) != 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
    case SAMQ_F16:  return launch_rms_norm<__half>(p, e, odd, st);
    case SAMQ_BF16: return launch_rms_norm<__nv_bfloat16>(p, e, odd, st);
    default:        return launch_rms_norm<float>(p, e, odd, st);
    }
}

}  // namespace samq
