// Pieces shared by the 4-bit product kernels: the block-scaled MMA, the scale copies, tensor maps, and an epilogue
// warp's work on 32 x 64 outputs.
#pragma once

#include "fp4.cuh"
#include "gemm_common.cuh"

namespace samq {
namespace fp4 {

using namespace sm100;
using namespace gemm;

constexpr int UKB = 32;                          // bytes of codes along K of one MMA: 64 columns

// Instruction descriptor of the block-scaled kinds: B's scale id in [4,6); A, B = e2m1 (1) in [7,10) and [10,12);
// both K-major; N >> 3 in [17,23); scale type in bit 23 (0 ue4m3, 1 ue8m0); M >> 7 in [27,29); A's scale id in [29,31).
__host__ __device__ constexpr uint32_t instr_desc(int fmt, int m, int n, uint32_t sf_id) {
    return (sf_id << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) |
           ((fmt == SAMQ_FP4_MX ? 1u : 0u) << 23) | ((uint32_t)(m >> 7) << 27) | (sf_id << 29);
}

#define SAMQ_MMA_FP4(GROUP, KIND)                                                                                     \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                                   \
                 "tcgen05.mma.cta_group::" GROUP "." KIND " [%0], %1, %2, %3, [%4], [%5], p;\n\t}"                    \
                 ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory")

// CTAS = 1, or 2 for a pair of CTAs (issued by the leader)
template <int FMT, int CTAS>
__device__ __forceinline__ void mma_fp4(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if constexpr (FMT == SAMQ_FP4_MX) {
        if constexpr (CTAS == 1) SAMQ_MMA_FP4("1", "kind::mxf4.block_scale.scale_vec::2X");
        else SAMQ_MMA_FP4("2", "kind::mxf4.block_scale.scale_vec::2X");
    } else {
        if constexpr (CTAS == 1) SAMQ_MMA_FP4("1", "kind::mxf4nvf4.block_scale.scale_vec::4X");
        else SAMQ_MMA_FP4("2", "kind::mxf4nvf4.block_scale.scale_vec::4X");
    }
}
#undef SAMQ_MMA_FP4

// 32 rows x 16 bytes of shared memory to four columns of tensor memory, repeated in all four lane quadrants; with
// CTAS = 2 in both CTAs of the pair, each from its own shared memory
template <int CTAS>
__device__ __forceinline__ void tmem_copy_scales(uint32_t tmem, uint64_t desc) {
    if constexpr (CTAS == 1) asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
    else asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
// rows of 16 bytes, no swizzle, eight rows (128 bytes) a core matrix
__device__ __forceinline__ uint64_t scale_desc(uint32_t smem_addr) {
    uint64_t d = (uint64_t)((smem_addr >> 4) & 0x3FFFu);
    d |= (uint64_t)(128 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    return d;
}

// ---- the epilogue of one warp: 32 rows x 64 columns -----------------------------------------------------
constexpr int EPI_COLS = 64;
constexpr int STAGING_BYTES = 32 * 128;          // per warp: 32 rows x 128 bytes, 128-byte swizzle

struct EpiParams {
    int M, N;
    float alpha;
    const void* bias;
    const void* residual; int64_t ldr;
    void* out; int64_t ldo;
    int tma_out;                                  // out is described by a tensor map (16-byte rows); else element stores
    int tma_res;                                  // the residual too
};

// byte of element `col` of row `row` in a staging buffer (the 128-byte swizzle of the tensor maps)
__device__ __forceinline__ uint32_t staged(int row, uint32_t byte) {
    return (uint32_t)row * 128u + (byte ^ ((uint32_t)(row & 7) << 4));
}

__device__ __forceinline__ float max0_nan(float x) {
    float r;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(x));
    return r;
}
// gelu_erf of two values in the fewest operations a result: with v = max(-|x|, -6.08), 2^Q(v) = Phi(v) and
// gelu(x) = max(x, 0) + v * Phi(v).  Q is gelu_erf's polynomial with the odd coefficients' signs turned.  v loses a NaN, the
// other maximum keeps it.
__device__ __forceinline__ float2 gelu_pair(float2 x) {
    const float2 v = make_float2(fmaxf(-fabsf(x.x), -6.08f), fmaxf(-fabsf(x.y), -6.08f));
    float2 q = make_float2(3.586083039e-05f, 3.586083039e-05f);
    q = __ffma2_rn(q, v, make_float2(7.942179800e-04f, 7.942179800e-04f));
    q = __ffma2_rn(q, v, make_float2(8.166280575e-03f, 8.166280575e-03f));
    q = __ffma2_rn(q, v, make_float2(5.355186760e-02f, 5.355186760e-02f));
    q = __ffma2_rn(q, v, make_float2(-4.586586654e-01f, -4.586586654e-01f));
    q = __ffma2_rn(q, v, make_float2(1.151242375e+00f, 1.151242375e+00f));
    q = __ffma2_rn(q, v, make_float2(-9.999881387e-01f, -9.999881387e-01f));
    float2 h;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(h.x) : "f"(q.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(h.y) : "f"(q.y));
    return __ffma2_rn(v, h, make_float2(max0_nan(x.x), max0_nan(x.y)));
}

template <typename OutT, bool GELU, bool RES>
struct EpiWarp {
    static constexpr int PASS_COLS = 128 / (int)sizeof(OutT);       // columns of a staging row: 64, or 32 of fp32
    static constexpr int PASSES = EPI_COLS / PASS_COLS;
    const EpiParams& p;
    const CUtensorMap* map_out;
    const CUtensorMap* map_res;
    uint8_t* staging;                              // STAGING_BYTES, 1024-byte aligned
    float* bias;                                   // EPI_COLS floats of the warp's own
    uint32_t res_bar; uint32_t res_phase;          // of the residual's TMA loads
    volatile uint32_t* abort_flag;
    int lane;

    __device__ __forceinline__ void load_residual(int row0, int col) {
        // the staging buffer is free once the previous tile's store has read it
        if (lane == 0) {
            bulk_wait_read0();
            fence_async_smem();
            mbar_expect_tx(res_bar, STAGING_BYTES);
            tma_load_2d(smem_u32(staging), map_res, res_bar, col, row0);
        }
    }
    // rows that no tensor map describes: element loads, a row's columns side by side in the warp
    __device__ __forceinline__ void fetch_residual(int row0, int col) {
        if (lane == 0) bulk_wait_read0();
        __syncwarp();
        const OutT* res = static_cast<const OutT*>(p.residual) + (int64_t)row0 * p.ldr + col + lane;
#pragma unroll 8
        for (int i = 0; i < 32; ++i)
#pragma unroll
            for (int j = 0; j < PASS_COLS; j += 32)
                if (row0 + i < p.M && col + j + lane < p.N)
                    *reinterpret_cast<OutT*>(staging + staged(i, (j + lane) * sizeof(OutT))) = res[(int64_t)i * p.ldr + j];
        __syncwarp();
    }
    // What does not depend on the accumulator: the bias of the columns, and the residual's first box under way.
    __device__ __forceinline__ void before(int row0, int col0) {
#pragma unroll
        for (int j = 0; j < EPI_COLS; j += 32) {
            const int n = col0 + j + lane;
            bias[j + lane] = (p.bias != nullptr && n < p.N) ? OutOps<OutT>::up(static_cast<const OutT*>(p.bias)[n]) : 0.0f;
        }
        __syncwarp();
        if constexpr (RES) {
            if (col0 < p.N && row0 < p.M) {
                if (p.tma_res) load_residual(row0, col0);
                else fetch_residual(row0, col0);
            }
        }
    }
    // acc: the 64 accumulator columns of this lane's row
    __device__ __forceinline__ bool finish(int row0, int col0, uint32_t (&acc)[EPI_COLS]) {
        if (row0 >= p.M) return true;
#pragma unroll
        for (int ps = 0; ps < PASSES; ++ps) {
            const int col = col0 + ps * PASS_COLS;
            if (col >= p.N) break;                                  // warp-uniform
            float y[PASS_COLS];
#pragma unroll
            for (int j = 0; j < PASS_COLS; j += 4) {
                const float4 b = *reinterpret_cast<const float4*>(bias + ps * PASS_COLS + j);
                const float2 a = make_float2(p.alpha, p.alpha);
                const int k = ps * PASS_COLS + j;
                const float2 lo = __ffma2_rn(make_float2(__uint_as_float(acc[k]), __uint_as_float(acc[k + 1])), a, make_float2(b.x, b.y));
                const float2 hi = __ffma2_rn(make_float2(__uint_as_float(acc[k + 2]), __uint_as_float(acc[k + 3])), a, make_float2(b.z, b.w));
                y[j] = lo.x; y[j + 1] = lo.y; y[j + 2] = hi.x; y[j + 3] = hi.y;
            }
            if constexpr (GELU) {
#pragma unroll
                for (int j = 0; j < PASS_COLS; j += 2) {
                    const float2 g = gelu_pair(make_float2(y[j], y[j + 1]));
                    y[j] = g.x; y[j + 1] = g.y;
                }
            }
            constexpr int PER16 = 16 / (int)sizeof(OutT);
            bool staging_free = false;
            if constexpr (RES) {
                if (p.tma_res) {
                    if (ps > 0) load_residual(row0, col);
                    const bool ok = mbar_wait_warp(res_bar, res_phase, abort_flag);
                    res_phase ^= 1u;
                    if (!ok) return false;
                } else if (ps > 0) {
                    fetch_residual(row0, col);
                }
                staging_free = true;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    OutT t[PER16];
                    *reinterpret_cast<uint4*>(t) = *reinterpret_cast<const uint4*>(staging + staged(lane, j * 16));
#pragma unroll
                    for (int e = 0; e < PER16; ++e) y[j * PER16 + e] += OutOps<OutT>::up(t[e]);
                }
            }
            if (!staging_free) {
                if (lane == 0) bulk_wait_read0();                   // the previous store has left the buffer
                __syncwarp();
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                OutT t[PER16];
#pragma unroll
                for (int e = 0; e < PER16; e += 2) {
                    if constexpr (sizeof(OutT) == 4) { t[e] = y[j * PER16 + e]; t[e + 1] = y[j * PER16 + e + 1]; }
                    else if constexpr (std::is_same<OutT, __half>::value)
                        *reinterpret_cast<__half2*>(t + e) = __floats2half2_rn(y[j * PER16 + e], y[j * PER16 + e + 1]);
                    else *reinterpret_cast<__nv_bfloat162*>(t + e) = __floats2bfloat162_rn(y[j * PER16 + e], y[j * PER16 + e + 1]);
                }
                *reinterpret_cast<uint4*>(staging + staged(lane, j * 16)) = *reinterpret_cast<const uint4*>(t);
            }
            if (p.tma_out) {
                fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                    tma_store_2d(map_out, smem_u32(staging), col, row0);
                    bulk_commit();
                }
            } else {
                __syncwarp();
                OutT* out = static_cast<OutT*>(p.out) + (int64_t)row0 * p.ldo + col;
#pragma unroll 8
                for (int i = 0; i < 32; ++i)
#pragma unroll
                    for (int j = 0; j < PASS_COLS; j += 32)
                        if (row0 + i < p.M && col + j + lane < p.N)
                            out[(int64_t)i * p.ldo + j + lane] = *reinterpret_cast<const OutT*>(staging + staged(i, (j + lane) * sizeof(OutT)));
                __syncwarp();
            }
        }
        return true;
    }
};

// 64 accumulator columns of this lane's row
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t (&r)[EPI_COLS]) {
    uint32_t (&lo)[32] = *reinterpret_cast<uint32_t (*)[32]>(r);
    uint32_t (&hi)[32] = *reinterpret_cast<uint32_t (*)[32]>(r + 32);
    tmem_ld32(taddr, lo);
    tmem_ld32(taddr + 32, hi);
    tmem_ld_wait();
}

// ---- host side ---------------------------------------------------------------------------------------------
// scale tiles as rows of 512 bytes (128 words); a box is the `box_tiles` tiles of one stage
inline int make_scale_map(CUtensorMap* map, const uint8_t* scales, int64_t tiles, int box_tiles) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) return fail(SAMQ_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    cuuint64_t dims[2] = {(cuuint64_t)(TILE_BYTES / 4), (cuuint64_t)tiles};
    cuuint64_t strides[1] = {(cuuint64_t)TILE_BYTES};
    cuuint32_t box[2] = {(cuuint32_t)(TILE_BYTES / 4), (cuuint32_t)box_tiles};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<uint8_t*>(scales), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(SAMQ_ERR_CUDA, "cuTensorMapEncodeTiled (scales) failed with CUresult %d", (int)r);
    return SAMQ_OK;
}
// [M, N] rows of `esize`-byte elements, boxes of 32 rows x 128 bytes, 128-byte swizzle
inline int make_row_map(CUtensorMap* map, const void* base, int64_t M, int64_t N, int64_t ld, int esize) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) return fail(SAMQ_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)M};
    cuuint64_t strides[1] = {(cuuint64_t)(ld * esize)};
    cuuint32_t box[2] = {(cuuint32_t)(128 / esize), 32u};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(map, esize == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(base), dims,
                    strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(SAMQ_ERR_CUDA, "cuTensorMapEncodeTiled (rows) failed with CUresult %d", (int)r);
    return SAMQ_OK;
}

// the call, checked and with its tensor maps, as the kernels take it
struct Fp4Call {
    const uint8_t* A; int64_t lda; const uint8_t* a_scales;
    const uint8_t* W; int64_t ldw; const uint8_t* w_scales;
    int64_t M, N, K;
    int fmt, out_dtype, gelu;
    EpiParams epi;
    CUtensorMap map_out, map_res;
    int32_t* status;
    cudaStream_t stream;
};

int gemm_fp4_pair(const Fp4Call& c);

}  // namespace fp4
}  // namespace samq
