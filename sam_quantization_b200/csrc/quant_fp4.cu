// Quantization to microscaled 4-bit floating point (mxfp4 / nvfp4), the operand format of samq_gemm_fp4.
//
//   mxfp4 : s = 2^(floor(log2 max|x|) - 2) per 32 columns          code = e2m1(x / s)
//   nvfp4 : s = e4m3(max|x| / (6 g)) * g   per 16 columns, g a power of two
//
// Bound: HBM (a row of K 16-bit values is 2K bytes in and K/2 + K/16 or K/32 out, plus 2K for the values).  Measured with the
// values: 32768 x 5120 bf16 mxfp4 114 us, 6.7 TB/s (above the rate of a copy, 6.55: the last writes are still in L2 at the end);
// nvfp4 127-129, where the instructions of twice the scales count (9 an element); 32768 x 1280 / 1278 / 1279 fp16 nvfp4 35 / 50 / 58 us (see STAGED).
#include "fp4.cuh"

namespace samq {

namespace {

using namespace fp4;

constexpr int CHUNK = 16;                        // columns of one thread: a block of nvfp4, half of one of mxfp4
constexpr int WARPS = 8;

struct QuantFp4Params {
    const void* x; int64_t ldx;
    int64_t M; int64_t K;
    float global_scale, inv_global_scale;
    uint8_t* codes; int64_t ldq;
    uint8_t* scales; int64_t groups;
    void* fq;
    int col_blocks;
    int access_x, access_fq;                     // see Access
    int pairs;                                   // STAGED 16-bit rows start on 4 bytes: two elements an access
    int vec_q;                                   // rows of codes start on 8 bytes
};

// A warp takes the rows that share 32 (nvfp4) or 16 (mxfp4) bytes of a scale tile, so that its scales leave as
// whole pieces: nvfp4 8 rows (r, r + 1, each + 0, 32, 64, 96) x 4 chunks, mxfp4 4 rows (r + 0, 32, 64, 96) x 8 chunks.
// the warp's rows in a tile: `sub` rows behind the unit's first one
template <int FMT>
__device__ __forceinline__ int first_row(int unit) { return FMT == SAMQ_FP4_MX ? unit : 2 * unit; }
template <int FMT>
__device__ __forceinline__ constexpr int row_offset(int sub) { return FMT == SAMQ_FP4_MX ? 32 * sub : (sub >> 2) + 32 * (sub & 3); }
// elements between the chunks of two lanes in shared memory: an odd number of words, so that no two lanes meet in a bank
template <typename T> constexpr int staged_pitch() { return sizeof(T) == 2 ? CHUNK + 2 : CHUNK + 1; }

// STAGED: rows of x or fq that do not start on 16 bytes pass through shared memory
template <typename T, int FMT, bool FQ, bool STAGED>
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
    const int r0 = first_row<FMT>((int)(row_unit % UNITS)), r = r0 + row_offset<FMT>(sub);
    const int64_t row = tile * TILE_ROWS + r;
    const int64_t col = (group * LANES + lane % LANES) * CHUNK;
    const bool row_ok = row < p.M;

    const int left = row_ok ? (int)min((int64_t)CHUNK, p.K - col) : 0;          // columns of the chunk (0 or less: none)
    Chunk<T> x;
    constexpr int STAGED_PITCH = staged_pitch<T>();
    __shared__ __align__(16) T staged[STAGED ? WARPS * 32 * STAGED_PITCH : 1];
    T* const mine = staged + (STAGED ? warp * 32 * STAGED_PITCH : 0);
    constexpr int SPAN = LANES * CHUNK;                            // columns of a row in the warp
    const int64_t first_col = group * SPAN, row0 = tile * TILE_ROWS + r0;
    const int cols = (int)max((int64_t)0, min((int64_t)SPAN, p.K - first_col));       // STAGED: the warp's columns and rows
    const int rows_left = (int)min((int64_t)TILE_ROWS, p.M - row0);
    if constexpr (STAGED) {
        // rows that no vector may start at: the warp reads 32 neighbouring elements an instruction and turns them into
        // its lanes' chunks in shared memory
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const T* src = static_cast<const T*>(p.x) + row0 * p.ldx + first_col + row_offset<FMT>(i) * p.ldx;
            const int in = row_offset<FMT>(i) < rows_left ? cols : 0;
            if (sizeof(T) == 2 && p.pairs) {
#pragma unroll
                for (int j = 0; j < SPAN; j += 64) {
                    const int c = j + 2 * lane;
                    *reinterpret_cast<uint32_t*>(mine + (i * LANES + c / CHUNK) * STAGED_PITCH + c % CHUNK) =
                        c < in ? *reinterpret_cast<const uint32_t*>(src + c) : 0u;
                }
            } else {
#pragma unroll
                for (int j = 0; j < SPAN; j += 32) {
                    const int c = j + lane;
                    mine[(i * LANES + c / CHUNK) * STAGED_PITCH + c % CHUNK] = c < in ? src[c] : Elem<T>::down(0.0f);
                }
            }
        }
        __syncwarp();
        uint32_t* words = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
        for (int i = 0; i < CHUNK * (int)sizeof(T) / 4; ++i) words[i] = reinterpret_cast<const uint32_t*>(mine + lane * STAGED_PITCH)[i];
        __syncwarp();
    } else {
        load_chunk(x, static_cast<const T*>(p.x) + row * p.ldx + col, left, p.access_x);
    }
    uint32_t amax = x.amax_bits();
    if constexpr (FMT == SAMQ_FP4_MX) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    const Scale s = block_scale<FMT>(amax, p.global_scale, p.inv_global_scale);
    hold_far<FMT>(x, s, p.global_scale);
    const uint2 q = encode_chunk<FMT>(x, s, amax < 0x7F800000u);

    // the word of four scales is put together by the group's first lane; blocks behind K and rows behind M are zero
    const int64_t block_col = col / block_of(FMT) * block_of(FMT);
    const uint32_t byte = (row_ok && block_col < p.K) ? s.byte : 0u;
    constexpr int STEP = LANES / 4;
    uint32_t word = byte << (8 * ((lane % LANES) / STEP));
#pragma unroll
    for (int o = STEP; o < LANES; o <<= 1) word |= __shfl_xor_sync(0xffffffffu, word, o);
    if (lane % LANES == 0)
        *reinterpret_cast<uint32_t*>(p.scales + (tile * p.groups + group) * TILE_BYTES + (r & 31) * 16 + (r >> 5) * 4) = word;
    if constexpr (!STAGED) { if (!row_ok) return; }

    const int64_t cbyte = col / 2;
    if (row_ok && cbyte < p.ldq) {
        uint8_t* o = p.codes + row * p.ldq + cbyte;
        if (p.vec_q && cbyte + 8 <= p.ldq) {
            *reinterpret_cast<uint2*>(o) = q;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) if (cbyte + i < p.ldq) o[i] = (uint8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
        }
    }
    if constexpr (FQ) {
        if constexpr (!STAGED) { if (left <= 0) return; }
        T* o = static_cast<T*>(p.fq) + row * p.K + col;
        T t[CHUNK];
        const float2 s2 = make_float2(s.value, s.value);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float2 v[4];
            unpack_e2m1x8(h ? q.y : q.x, v);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 y = __fmul2_rn(v[i], s2);
                if constexpr (std::is_same<T, __half>::value) *reinterpret_cast<__half2*>(t + 8 * h + 2 * i) = __floats2half2_rn(y.x, y.y);
                else if constexpr (std::is_same<T, __nv_bfloat16>::value) *reinterpret_cast<__nv_bfloat162*>(t + 8 * h + 2 * i) = __floats2bfloat162_rn(y.x, y.y);
                else { t[8 * h + 2 * i] = y.x; t[8 * h + 2 * i + 1] = y.y; }
            }
        }
        const uint32_t* w = reinterpret_cast<const uint32_t*>(t);
        constexpr int WORDS = CHUNK * (int)sizeof(T) / 4;
        if constexpr (STAGED) {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) reinterpret_cast<uint32_t*>(mine + lane * STAGED_PITCH)[i] = w[i];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                T* dst = static_cast<T*>(p.fq) + row0 * p.K + first_col + row_offset<FMT>(i) * p.K;
                const int in = row_offset<FMT>(i) < rows_left ? cols : 0;
                if (sizeof(T) == 2 && p.pairs) {
#pragma unroll
                    for (int j = 0; j < SPAN; j += 64) {
                        const int c = j + 2 * lane;
                        if (c < in)
                            *reinterpret_cast<uint32_t*>(dst + c) =
                                *reinterpret_cast<const uint32_t*>(mine + (i * LANES + c / CHUNK) * STAGED_PITCH + c % CHUNK);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < SPAN; j += 32) {
                        const int c = j + lane;
                        if (c < in) dst[c] = mine[(i * LANES + c / CHUNK) * STAGED_PITCH + c % CHUNK];
                    }
                }
            }
        } else if (left >= CHUNK && p.access_fq == BY_32) {
#pragma unroll
            for (int i = 0; i < WORDS; i += 8) store32(reinterpret_cast<uint32_t*>(o) + i, w + i);
        } else if (left >= CHUNK && p.access_fq == BY_16) {
#pragma unroll
            for (int i = 0; i < WORDS; i += 4) *reinterpret_cast<uint4*>(reinterpret_cast<uint32_t*>(o) + i) = *reinterpret_cast<const uint4*>(w + i);
        } else {
#pragma unroll
            for (int i = 0; i < CHUNK; ++i) if (i < left) o[i] = t[i];
        }
    }
}

template <typename T, int FMT>
int launch_quant_fp4(const QuantFp4Params& p, cudaStream_t st) {
    constexpr int ROWS = FMT == SAMQ_FP4_MX ? 4 : 8;
    const int64_t units = (p.M + TILE_ROWS - 1) / TILE_ROWS * (TILE_ROWS / ROWS);
    const int64_t blocks = units * p.col_blocks;
    if (blocks > 2147483647LL) return fail(SAMQ_ERR_TOO_LARGE, "quantization to 4 bits: %lld x %lld is too large", (long long)p.M, (long long)p.K);
    const bool staged = p.access_x == BY_ELEMENT || (p.fq != nullptr && p.access_fq == BY_ELEMENT);
    const unsigned grid = (unsigned)blocks;
    if (p.fq != nullptr) {
        if (staged) quant_fp4_kernel<T, FMT, true, true><<<grid, WARPS * 32, 0, st>>>(p);
        else quant_fp4_kernel<T, FMT, true, false><<<grid, WARPS * 32, 0, st>>>(p);
    } else {
        if (staged) quant_fp4_kernel<T, FMT, false, true><<<grid, WARPS * 32, 0, st>>>(p);
        else quant_fp4_kernel<T, FMT, false, false><<<grid, WARPS * 32, 0, st>>>(p);
    }
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
    if (K > 2147483647LL - 256) return fail(SAMQ_ERR_TOO_LARGE, "K=%lld exceeds 2^31", (long long)K);
    if (dtype != SAMQ_F16 && dtype != SAMQ_BF16 && dtype != SAMQ_F32) return fail(SAMQ_ERR_BAD_ARG, "unknown dtype %d", dtype);
    if (!fp4::known_format(fmt)) return fail(SAMQ_ERR_BAD_ARG, "unknown 4-bit format %d", fmt);
    const int rc = fp4::check_global_scale(fmt, global_scale);
    if (rc != SAMQ_OK || M == 0) return rc;
    if (x == nullptr || codes == nullptr || scales == nullptr) return fail(SAMQ_ERR_BAD_ARG, "x, codes and scales must not be null");
    if (ldx < K) return fail(SAMQ_ERR_BAD_ARG, "ldx smaller than K");
    if (ldq < (K + 1) / 2) return fail(SAMQ_ERR_BAD_ARG, "ldq smaller than the %lld bytes of a row", (long long)((K + 1) / 2));
    if (ldq > fp4::groups_of(fmt, K) * 2 * fp4::block_of(fmt)) return fail(SAMQ_ERR_BAD_ARG, "ldq beyond the columns that the scales cover");
    if (reinterpret_cast<uintptr_t>(scales) & 15) return fail(SAMQ_ERR_ALIGNMENT, "scales must be 16-byte aligned");
    const size_t esz = dtype == SAMQ_F32 ? 4 : 2;
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(fq)) & (esz - 1)) return fail(SAMQ_ERR_ALIGNMENT, "x and fq_out must be aligned to their elements");
    QuantFp4Params p;
    p.x = x; p.ldx = ldx; p.M = M; p.K = K; p.global_scale = global_scale; p.inv_global_scale = 1.0f / global_scale;
    p.codes = codes; p.ldq = ldq; p.scales = scales; p.groups = fp4::groups_of(fmt, K); p.fq = fq;
    p.col_blocks = (int)((p.groups + WARPS - 1) / WARPS);
    p.access_x = row_access(x, ldx * (int64_t)esz);
    p.access_fq = row_access(fq, K * (int64_t)esz);
    p.pairs = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(fq) | (uintptr_t)((ldx | K) * (int64_t)esz)) & 3) == 0;
    p.vec_q = (reinterpret_cast<uintptr_t>(codes) & 7) == 0 && ldq % 8 == 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
    case SAMQ_F16:  return launch_quant_fp4<__half>(fmt, p, st);
    case SAMQ_BF16: return launch_quant_fp4<__nv_bfloat16>(fmt, p, st);
    default:        return launch_quant_fp4<float>(fmt, p, st);
    }
}

}  // namespace samq
