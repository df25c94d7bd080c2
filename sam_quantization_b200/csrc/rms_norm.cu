// RMS norm of the residual stream with an 8-bit output.
//
//   h = T(x + residual)                      the new residual stream, rounded as it is stored
//   y = h * rsqrt(mean(h^2) + eps) * w       fp32, never rounded to the tensor type
//   s = max(max|y|, 1e-5) / q_max            one scale per row
//   q = round_half_even(y / s)
//
// One pass: a row stays in registers between the two reductions (sum of squares, largest magnitude).  Bound: HBM,
// 2 + 2 + 2 + 1 bytes an element of a 16-bit type (x, residual, h, q), 2 more for the dequantized values.
#include "common.cuh"

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
    int vec;                                       // every row of every tensor starts on 16 bytes and K fills vectors
};

// sum and integer maximum over the `warps` warps that share a row
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ uint32_t warp_umax(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

template <typename T, int E>
__device__ __forceinline__ void load_vec(const T* p, float (&f)[E]) {
    if constexpr (E == 1) {
        f[0] = Elem<T>::up(*p);
    } else {
        T t[E];
        *reinterpret_cast<uint4*>(t) = *reinterpret_cast<const uint4*>(p);
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = Elem<T>::up(t[e]);
    }
}
template <typename T, int E>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[E]) {
    if constexpr (E == 1) {
        *p = Elem<T>::down(f[0]);
    } else {
        T t[E];
#pragma unroll
        for (int e = 0; e < E; ++e) t[e] = Elem<T>::down(f[e]);
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(t);
    }
}

// E elements a load (a 16-byte vector, or one where rows are not aligned), NV loads a thread, RW warps a row.
template <typename T, int E, int NV, int RW>
__global__ void __launch_bounds__(RW >= 8 ? RW * 32 : 256)
rms_norm_quant_kernel(const RmsNormParams p)
{
    constexpr int ROWS = RW >= 8 ? 1 : 8 / RW;     // rows of a block
    constexpr int T_ROW = RW * 32;                 // threads of a row
    __shared__ float red_sum[RW > 1 ? ROWS * RW : 1];
    __shared__ uint32_t red_max[RW > 1 ? ROWS * RW : 1];
    const int sub = threadIdx.x / T_ROW, t = threadIdx.x % T_ROW;
    const int64_t row = (int64_t)blockIdx.x * ROWS + sub;
    const bool row_ok = row < p.M;                 // rows behind the last one only keep the barriers company

    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* res = static_cast<const T*>(p.residual) + row * p.ldr;
    T* h_out = static_cast<T*>(p.residual_out) + row * p.ldo;
    float h[NV][E];
    float sum = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = (v * T_ROW + t) * E;
#pragma unroll
        for (int e = 0; e < E; ++e) h[v][e] = 0.0f;
        if (row_ok && c < p.K) load_vec<T, E>(x + c, h[v]);
    }
    if (p.residual != nullptr) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * T_ROW + t) * E;
            if (!(row_ok && c < p.K)) continue;
            float r[E];
            load_vec<T, E>(res + c, r);
#pragma unroll
            for (int e = 0; e < E; ++e) h[v][e] = round_to<T>(h[v][e] + r[e]);
            store_vec<T, E>(h_out + c, h[v]);
        }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < E; ++e) sum = fmaf(h[v][e], h[v][e], sum);
    sum = warp_sum(sum);
    if constexpr (RW > 1) {
        if ((t & 31) == 0) red_sum[sub * RW + (t >> 5)] = sum;
        __syncthreads();
        sum = red_sum[sub * RW];
#pragma unroll
        for (int w = 1; w < RW; ++w) sum += red_sum[sub * RW + w];
    }
    const float u = rsqrtf(fmaf(sum, p.inv_k, p.eps));

    uint32_t amax_bits = 0;
    const T* w = static_cast<const T*>(p.weight);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = (v * T_ROW + t) * E;
        if (!(row_ok && c < p.K)) continue;
        float wv[E];
        load_vec<T, E>(w + c, wv);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            h[v][e] = h[v][e] * u * wv[e];
            amax_bits = max(amax_bits, __float_as_uint(h[v][e]) & 0x7FFFFFFFu);   // as integers: a NaN wins
        }
    }
    amax_bits = warp_umax(amax_bits);
    if constexpr (RW > 1) {
        if ((t & 31) == 0) red_max[sub * RW + (t >> 5)] = amax_bits;
        __syncthreads();
        amax_bits = red_max[sub * RW];
#pragma unroll
        for (int k = 1; k < RW; ++k) amax_bits = max(amax_bits, red_max[sub * RW + k]);
    }
    if (!row_ok) return;
    const float amax = __uint_as_float(amax_bits);
    // a row with a NaN or an infinity has a NaN scale and zero codes
    const bool finite = amax_bits < 0x7F800000u;
    const float s = finite ? __fdiv_rn(fmaxf(amax, 1e-5f), p.qmax) : __uint_as_float(0x7FC00000u);
    if (t == 0 && p.scale != nullptr) p.scale[row] = s;
    const Divider d = make_divider(s);
    int8_t* q_out = p.q == nullptr ? nullptr : p.q + row * (int64_t)p.K;
    T* fq = p.fq == nullptr ? nullptr : static_cast<T*>(p.fq) + row * (int64_t)p.K;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = (v * T_ROW + t) * E;
        if (c >= p.K) continue;
        float q[E];
#pragma unroll
        for (int e = 0; e < E; ++e) q[e] = finite ? rint_small(div_exact(h[v][e], d), h[v][e]) : 0.0f;
        if (q_out != nullptr) {
            if constexpr (E == 1) {
                q_out[c] = (int8_t)code_byte(q[0], p.qmax);
            } else {
                uint32_t word[E / 4];
#pragma unroll
                for (int k = 0; k < E / 4; ++k) {
                    word[k] = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) word[k] |= code_byte(q[4 * k + e], p.qmax) << (8 * e);
                }
                if constexpr (E == 8) *reinterpret_cast<uint2*>(q_out + c) = make_uint2(word[0], word[1]);
                else *reinterpret_cast<uint32_t*>(q_out + c) = word[0];
            }
        }
        if (fq != nullptr) {
#pragma unroll
            for (int e = 0; e < E; ++e) q[e] *= s;
            store_vec<T, E>(fq + c, q);
        }
    }
}

template <typename T, int E, int NV, int RW>
int launch(const RmsNormParams& p, cudaStream_t st) {
    constexpr int ROWS = RW >= 8 ? 1 : 8 / RW;
    const int64_t blocks = (p.M + ROWS - 1) / ROWS;
    if (blocks > 2147483647LL) return fail(SAMQ_ERR_TOO_LARGE, "RMS norm of %lld rows is too large", (long long)p.M);
    rms_norm_quant_kernel<T, E, NV, RW><<<(unsigned)blocks, RW >= 8 ? RW * 32 : 256, 0, st>>>(p);
    SAMQ_CUDA_TRY(cudaGetLastError());
    return SAMQ_OK;
}

// The fewest warps whose threads hold the row in NV loads each, 1 to 32.
template <typename T, int E, int NV>
int launch_warps(int64_t loads, const RmsNormParams& p, cudaStream_t st) {
    if (loads <= 32 * NV) return launch<T, E, NV, 1>(p, st);
    if (loads <= 64 * NV) return launch<T, E, NV, 2>(p, st);
    if (loads <= 128 * NV) return launch<T, E, NV, 4>(p, st);
    if (loads <= 256 * NV) return launch<T, E, NV, 8>(p, st);
    if (loads <= 512 * NV) return launch<T, E, NV, 16>(p, st);
    return launch<T, E, NV, 32>(p, st);
}

template <typename T>
int launch_rms_norm(const RmsNormParams& p, cudaStream_t st) {
    constexpr int E = Elem<T>::kPerVec;
    // 5 vectors: 1280 columns of a 16-bit type are one warp's, with no lane idle
    if (p.vec) return launch_warps<T, E, 5>(p.K / E, p, st);
    return launch_warps<T, 1, 32>(p.K, p, st);
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
    const int64_t vec = 16 / (int64_t)esz;
    p.vec = (all & 15) == 0 && K % vec == 0 && ldx % vec == 0 && p.ldr % vec == 0 && p.ldo % vec == 0 &&
            (reinterpret_cast<uintptr_t>(q) & (vec - 1)) == 0 && K <= 1024 * 5 * vec;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
    case SAMQ_F16:  return launch_rms_norm<__half>(p, st);
    case SAMQ_BF16: return launch_rms_norm<__nv_bfloat16>(p, st);
    default:        return launch_rms_norm<float>(p, st);
    }
}

}  // namespace samq
