// Quantization to microscaled 4-bit floating point (mxfp4 / nvfp4), the operand format of samq_gemm_fp4.
//
//   mxfp4 : s = 2^(floor(log2 max|x|) - 2) per 32 columns          code = e2m1(x / s)
//   nvfp4 : s = e4m3(max|x| / (6 g)) * g   per 16 columns, g a power of two
//
// Bound: HBM (a row of K 16-bit values is 2K bytes in and K/2 + K/16 or K/32 out, plus 2K for the values).
#include "fp4.cuh"

namespace samq {

namespace {

using namespace fp4;

constexpr int CHUNK = 16;                        // columns of one thread: a block of nvfp4, half of one of mxfp4
constexpr int WARPS = 8;

struct QuantFp4Params {
    const void* x; int64_t ldx;
    int64_t M; int64_t K;
    float global_scale;
    uint8_t* codes; int64_t ldq;
    uint8_t* scales; int64_t groups;
    void* fq;
    int col_blocks;
    int vec_x, vec_q, vec_fq;                    // rows start on 16 (8 for the codes) bytes: vectors may be used
};

template <typename T>
__device__ __forceinline__ void load_chunk(const T* p, float (&f)[CHUNK]) {
    constexpr int E = Elem<T>::kPerVec;
#pragma unroll
    for (int v = 0; v < CHUNK / E; ++v) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + v);
        T t[E];
        *reinterpret_cast<uint4*>(t) = u;
#pragma unroll
        for (int e = 0; e < E; ++e) f[v * E + e] = Elem<T>::up(t[e]);
    }
}

// A warp takes the rows that share 32 (nvfp4) or 16 (mxfp4) bytes of a scale tile, so that its scales leave as
// whole pieces: nvfp4 8 rows (r, r + 1, each + 0, 32, 64, 96) x 4 chunks, mxfp4 4 rows (r + 0, 32, 64, 96) x 8 chunks.
template <typename T, int FMT, bool FQ>
__global__ void __launch_bounds__(WARPS * 32)
quant_fp4_kernel(const QuantFp4Params p)
{
    constexpr int LANES = FMT == SAMQ_FP4_MX ? 8 : 4;              // threads of four blocks: one word of scales
    constexpr int ROWS = 32 / LANES;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row_unit = blockIdx.x / p.col_blocks;
    const int64_t group = (int64_t)(blockIdx.x % p.col_blocks) * WARPS + warp;
    if (group >= p.groups) return;                                 // whole warps
    constexpr int UNITS = 128 / ROWS;                              // row units of a tile
    const int64_t tile = row_unit / UNITS;
    const int sub = lane / LANES;
    const int r = FMT == SAMQ_FP4_MX ? (int)(row_unit % UNITS) + 32 * sub
                                     : 2 * (int)(row_unit % UNITS) + (sub >> 2) + 32 * (sub & 3);
    const int64_t row = tile * TILE_ROWS + r;
    const int64_t col = (group * LANES + lane % LANES) * CHUNK;
    const bool row_ok = row < p.M;

    float f[CHUNK];
    const T* x = static_cast<const T*>(p.x) + row * p.ldx + col;
    const bool whole = col + CHUNK <= p.K;
    if (row_ok && whole && p.vec_x) {
        load_chunk<T>(x, f);
    } else {
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) f[i] = (row_ok && col + i < p.K) ? Elem<T>::up(x[i]) : 0.0f;
    }
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < CHUNK; ++i) amax = max(amax, __float_as_uint(f[i]) & 0x7FFFFFFFu);
    if constexpr (FMT == SAMQ_FP4_MX) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    const Scale s = block_scale<FMT>(amax, p.global_scale);
    const ToCode<FMT> to_code(s);
    const bool finite = amax < 0x7F800000u;
    float v[CHUNK];
#pragma unroll
    for (int i = 0; i < CHUNK; ++i) v[i] = finite ? to_code(f[i]) : 0.0f;
    const uint2 q = make_uint2(pack_e2m1x8(v), pack_e2m1x8(v + 8));

    // the word of four scales is put together by the group's first lane; blocks behind K and rows behind M are zero
    const int64_t block_col = col / block_of(FMT) * block_of(FMT);
    const uint32_t byte = (row_ok && block_col < p.K) ? s.byte : 0u;
    constexpr int STEP = LANES / 4;
    uint32_t word = byte << (8 * ((lane % LANES) / STEP));
#pragma unroll
    for (int o = STEP; o < LANES; o <<= 1) word |= __shfl_xor_sync(0xffffffffu, word, o);
    if (lane % LANES == 0)
        *reinterpret_cast<uint32_t*>(p.scales + (tile * p.groups + group) * TILE_BYTES + (r & 31) * 16 + (r >> 5) * 4) = word;
    if (!row_ok) return;

    const int64_t cbyte = col / 2;
    if (cbyte < p.ldq) {
        uint8_t* o = p.codes + row * p.ldq + cbyte;
        if (p.vec_q && cbyte + 8 <= p.ldq) {
            *reinterpret_cast<uint2*>(o) = q;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) if (cbyte + i < p.ldq) o[i] = (uint8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
        }
    }
    if constexpr (FQ) {
        T* o = static_cast<T*>(p.fq) + row * p.K + col;
        T t[CHUNK];
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
            const uint32_t c = ((i < 8 ? q.x : q.y) >> (4 * (i & 7))) & 15u;
            t[i] = Elem<T>::down(e2m1_value(c) * s.value);
        }
        if (whole && p.vec_fq) {
            constexpr int E = Elem<T>::kPerVec;
#pragma unroll
            for (int k = 0; k < CHUNK / E; ++k) reinterpret_cast<uint4*>(o)[k] = *reinterpret_cast<const uint4*>(t + k * E);
        } else {
#pragma unroll
            for (int i = 0; i < CHUNK; ++i) if (col + i < p.K) o[i] = t[i];
        }
    }
}

template <typename T, int FMT>
int launch_quant_fp4(const QuantFp4Params& p, cudaStream_t st) {
    constexpr int ROWS = FMT == SAMQ_FP4_MX ? 4 : 8;
    const int64_t units = (p.M + TILE_ROWS - 1) / TILE_ROWS * (TILE_ROWS / ROWS);
    const int64_t blocks = units * p.col_blocks;
    if (blocks > 2147483647LL) return fail(SAMQ_ERR_TOO_LARGE, "quantization to 4 bits: %lld x %lld is too large", (long long)p.M, (long long)p.K);
    if (p.fq != nullptr) quant_fp4_kernel<T, FMT, true><<<(unsigned)blocks, WARPS * 32, 0, st>>>(p);
    else quant_fp4_kernel<T, FMT, false><<<(unsigned)blocks, WARPS * 32, 0, st>>>(p);
    SAMQ_CUDA_TRY(cudaGetLastError());
    return SAMQ_OK;
}

template <typename T>
int launch_quant_fp4(int fmt, const QuantFp4Params& p, cudaStream_t st) {
    return fmt == SAMQ_FP4_MX ? launch_quant_fp4<T, SAMQ_FP4_MX>(p, st) : launch_quant_fp4<T, SAMQ_FP4_NV>(p, st);
}

}  // namespace

int quant_fp4_dispatch(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, int fmt, float global_scale,
                       uint8_t* codes, int64_t ldq, uint8_t* scales, void* fq, void* stream)
{
    if (M < 0 || K <= 0) return fail(SAMQ_ERR_BAD_ARG, "bad shape M=%lld K=%lld", (long long)M, (long long)K);
    if (dtype != SAMQ_F16 && dtype != SAMQ_BF16 && dtype != SAMQ_F32) return fail(SAMQ_ERR_BAD_ARG, "unknown dtype %d", dtype);
    if (!fp4::known_format(fmt)) return fail(SAMQ_ERR_BAD_ARG, "unknown 4-bit format %d", fmt);
    if (!fp4::good_global_scale(global_scale)) return fail(SAMQ_ERR_BAD_ARG, "global_scale must be a power of two between 2^-64 and 2^64");
    if (fmt == SAMQ_FP4_MX && global_scale != 1.0f) return fail(SAMQ_ERR_BAD_ARG, "mxfp4 has no global scale: its block scales reach every exponent");
    if (M == 0) return SAMQ_OK;
    if (x == nullptr || codes == nullptr || scales == nullptr) return fail(SAMQ_ERR_BAD_ARG, "x, codes and scales must not be null");
    if (ldx < K) return fail(SAMQ_ERR_BAD_ARG, "ldx smaller than K");
    if (ldq < (K + 1) / 2) return fail(SAMQ_ERR_BAD_ARG, "ldq smaller than the %lld bytes of a row", (long long)((K + 1) / 2));
    if (ldq > fp4::groups_of(fmt, K) * 2 * fp4::block_of(fmt)) return fail(SAMQ_ERR_BAD_ARG, "ldq beyond the columns that the scales cover");
    if (reinterpret_cast<uintptr_t>(scales) & 15) return fail(SAMQ_ERR_ALIGNMENT, "scales must be 16-byte aligned");
    const size_t esz = dtype == SAMQ_F32 ? 4 : 2;
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(fq)) & (esz - 1)) return fail(SAMQ_ERR_ALIGNMENT, "x and fq_out must be aligned to their elements");
    QuantFp4Params p;
    p.x = x; p.ldx = ldx; p.M = M; p.K = K; p.global_scale = global_scale;
    p.codes = codes; p.ldq = ldq; p.scales = scales; p.groups = fp4::groups_of(fmt, K); p.fq = fq;
    p.col_blocks = (int)((p.groups + WARPS - 1) / WARPS);
    p.vec_x = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ldx * esz) % 16 == 0;
    p.vec_q = (reinterpret_cast<uintptr_t>(codes) & 7) == 0 && ldq % 8 == 0;
    p.vec_fq = (reinterpret_cast<uintptr_t>(fq) & 15) == 0 && (K * esz) % 16 == 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
    case SAMQ_F16:  return launch_quant_fp4<__half>(fmt, p, st);
    case SAMQ_BF16: return launch_quant_fp4<__nv_bfloat16>(fmt, p, st);
    default:        return launch_quant_fp4<float>(fmt, p, st);
    }
}

}  // namespace samq
