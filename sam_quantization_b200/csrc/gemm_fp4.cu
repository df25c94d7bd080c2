// Product of two microscaled 4-bit operands on the tensor cores, with the linear layer's epilogue.
//
//   acc[m,n] = sum over blocks b of sa[m,b] * sw[n,b] * sum_{k in b} a[m,k] * w[n,k]
//   y[m,n]   = act(alpha * acc[m,n] + bias[n]) + residual[m,n]
//
// tcgen05.mma with block scaling (kind::mxf4 for mxfp4, kind::mxf4nvf4 for nvfp4) takes K = 64 columns an
// instruction: 32 bytes of codes from shared memory (128-byte swizzle, as the int8 product) and the scales of both
// operands from tensor memory, where tcgen05.cp puts a stage's tiles before its MMAs.  Accumulators are fp32.
#include "fp4_gemm.cuh"

namespace samq {

using namespace fp4;

namespace {

// 256 x 192 tiles from which the pair kernel has enough to do
constexpr int PAIR_MIN_TILES = 32;

constexpr int BM = 128;
constexpr int BN = 128;
constexpr int STAGES = 4;
constexpr int A_BYTES = BM * BK;                 // BK = 128 bytes = 256 columns
constexpr int B_BYTES = BN * BK;
constexpr int EPI_WARPS = 4;
constexpr int THREADS = 64 + EPI_WARPS * 32;
constexpr int TMEM_COLS = 256;
constexpr int SFA_COL = BN;                      // scale columns behind the accumulator

struct __align__(8) Control {
    uint64_t full[STAGES];
    uint64_t empty[STAGES];
    uint64_t acc_full;
    uint32_t tmem_base;
    uint32_t abort_flag;
};

template <int FMT> struct Shape {
    static constexpr int GROUPS = groups_per_kpad(FMT);        // scale tiles of an operand's 128 rows a stage
    static constexpr int SF_BYTES = GROUPS * TILE_BYTES;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + 2 * SF_BYTES;
    static constexpr int SFB_COL = SFA_COL + 4 * GROUPS;
    static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE_BYTES + BN * sizeof(float) + sizeof(Control);
};

struct Fp4Params {
    int M, N, K;
    const uint8_t* a_scales;
    const uint8_t* w_scales;
    int groups;
    float alpha;
    const void* bias;
    const void* residual; int64_t ldr;
    void* out; int64_t ldo;
    int gelu;
    int vec_ok;
    int32_t* status;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

template <typename OutT, int FMT>
__global__ void __launch_bounds__(THREADS, 1)
gemm_fp4_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const Fp4Params p)
{
    using S = Shape<FMT>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    uint8_t* tiles = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
    uint8_t* sf = tiles + (size_t)STAGES * (A_BYTES + B_BYTES);
    float* bias_s = reinterpret_cast<float*>(sf + (size_t)STAGES * 2 * S::SF_BYTES);
    Control* ctl = reinterpret_cast<Control*>(bias_s + BN);
    volatile uint32_t* abort_flag = &ctl->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int k_blocks = (p.K + KPAD - 1) / KPAD;
    const int n_blocks = (p.N + BN - 1) / BN;
    const int mt = blockIdx.x / n_blocks, nt = blockIdx.x % n_blocks;
    const int m0 = mt * BM, n0 = nt * BN;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(smem_u32(&ctl->full[s]), 1); mbar_init(smem_u32(&ctl->empty[s]), 1); }
        mbar_init(smem_u32(&ctl->acc_full), 1);
        ctl->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&ctl->tmem_base)), "r"((uint32_t)TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = ctl->tmem_base;

    if (warp == 0) {
        if (lane == 0) {
            bool ok = true;
            for (int kb = 0; kb < k_blocks; ++kb) {
                const int st = kb % STAGES;
                if (!mbar_wait(smem_u32(&ctl->empty[st]), ((kb / STAGES) & 1) ^ 1u, abort_flag)) { ok = false; break; }
                const uint32_t bar = smem_u32(&ctl->full[st]);
                const uint32_t sa = smem_u32(tiles + (size_t)st * (A_BYTES + B_BYTES));
                const uint32_t ss = smem_u32(sf + (size_t)st * 2 * S::SF_BYTES);
                mbar_expect_tx(bar, S::STAGE_BYTES);
                tma_load_2d(sa, &map_a, bar, kb * BK, m0);
                tma_load_2d(sa + A_BYTES, &map_w, bar, kb * BK, n0);
                bulk_load(ss, p.a_scales + ((int64_t)mt * p.groups + kb * S::GROUPS) * TILE_BYTES, S::SF_BYTES, bar);
                bulk_load(ss + S::SF_BYTES, p.w_scales + ((int64_t)nt * p.groups + kb * S::GROUPS) * TILE_BYTES, S::SF_BYTES, bar);
            }
            if (!ok) {
                const long long t0 = clock64();
                while (clock64() - t0 < 2000000LL) { }              // copies in flight land before the CTA retires
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            bool ok = true;
            for (int kb = 0; kb < k_blocks; ++kb) {
                const int st = kb % STAGES;
                if (!mbar_wait(smem_u32(&ctl->full[st]), (kb / STAGES) & 1, abort_flag)) { ok = false; break; }
                tcgen05_fence_after();
                const uint32_t sa = smem_u32(tiles + (size_t)st * (A_BYTES + B_BYTES));
                const uint32_t ss = smem_u32(sf + (size_t)st * 2 * S::SF_BYTES);
#pragma unroll
                for (int g = 0; g < S::GROUPS; ++g) {
                    tmem_copy_scales<1>(tmem + SFA_COL + 4 * g, scale_desc(ss + g * TILE_BYTES));
                    tmem_copy_scales<1>(tmem + S::SFB_COL + 4 * g, scale_desc(ss + S::SF_BYTES + g * TILE_BYTES));
                }
                const uint64_t adesc = make_smem_desc(sa), bdesc = make_smem_desc(sa + A_BYTES);
#pragma unroll
                for (int k = 0; k < BK / UKB; ++k) {
                    // mxfp4: a word of four scales serves two MMAs, the second taking its upper half (scale id 2)
                    const int g = FMT == SAMQ_FP4_MX ? k / 2 : k;
                    const uint32_t id = FMT == SAMQ_FP4_MX ? 2u * (k & 1) : 0u;
                    mma_fp4<FMT, 1>(tmem, adesc + (uint64_t)(k * (UKB >> 4)), bdesc + (uint64_t)(k * (UKB >> 4)), instr_desc(FMT, BM, BN, id),
                                 tmem + SFA_COL + 4 * g, tmem + S::SFB_COL + 4 * g, (kb | k) != 0 ? 1u : 0u);
                }
                tcgen05_commit(smem_u32(&ctl->empty[st]));
            }
            if (ok) tcgen05_commit(smem_u32(&ctl->acc_full));
        }
    } else {
        const int quad = warp & 3;
        const int tid = threadIdx.x - 64;
        const OutT* bias = static_cast<const OutT*>(p.bias);
        bias_s[tid] = (bias != nullptr && n0 + tid < p.N) ? OutOps<OutT>::up(bias[n0 + tid]) : 0.0f;
        asm volatile("bar.sync 1, %0;" ::"r"(EPI_WARPS * 32) : "memory");
        if (mbar_wait(smem_u32(&ctl->acc_full), 0, abort_flag)) {
            tcgen05_fence_after();
            const int row = m0 + quad * 32 + lane;
#pragma unroll 1
            for (int c = 0; c < BN / 32; ++c) {
                const int n_first = n0 + c * 32;
                if (n_first >= p.N) break;                              // warp-uniform
                uint32_t r[32];
                tmem_ld32(tmem + ((uint32_t)(quad * 32) << 16) + c * 32, r);
                tmem_ld_wait();
                float y[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) y[j] = fmaf(__uint_as_float(r[j]), p.alpha, bias_s[c * 32 + j]);
                if (p.gelu) gelu32(y);
                if (row < p.M) {
                    const int n_valid = min(32, p.N - n_first);
                    if (p.residual != nullptr) {
                        const OutT* res = static_cast<const OutT*>(p.residual) + (int64_t)row * p.ldr + n_first;
#pragma unroll
                        for (int j = 0; j < 32; ++j) if (j < n_valid) y[j] += OutOps<OutT>::up(res[j]);
                    }
                    OutT* o = static_cast<OutT*>(p.out) + (int64_t)row * p.ldo + n_first;
                    if (p.vec_ok && n_valid == 32) {
                        constexpr int NVEC = 32 * sizeof(OutT) / 16;
                        uint4 packed[NVEC];
                        OutOps<OutT>::pack32(y, packed);
#pragma unroll
                        for (int j = 0; j < NVEC; ++j) reinterpret_cast<uint4*>(o)[j] = packed[j];
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; ++j) if (j < n_valid) o[j] = OutOps<OutT>::down(y[j]);
                    }
                }
            }
        }
        tcgen05_fence_before();
    }
    __syncthreads();
    tcgen05_fence_after();
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)TMEM_COLS) : "memory");
    }
    if (threadIdx.x == 0 && ctl->abort_flag != 0 && p.status != nullptr) atomicExch(p.status, 1);
}

template <typename OutT, int FMT>
int launch(const CUtensorMap& ma, const CUtensorMap& mw, const Fp4Params& p, cudaStream_t st) {
    SAMQ_CUDA_TRY(cudaFuncSetAttribute(gemm_fp4_kernel<OutT, FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<FMT>::SMEM));
    const int64_t tiles = (int64_t)((p.M + BM - 1) / BM) * ((p.N + BN - 1) / BN);
    if (tiles > 2147483647LL) return fail(SAMQ_ERR_TOO_LARGE, "product of %d x %d outputs is too large", p.M, p.N);
    gemm_fp4_kernel<OutT, FMT><<<(unsigned)tiles, THREADS, Shape<FMT>::SMEM, st>>>(ma, mw, p);
    SAMQ_CUDA_TRY(cudaGetLastError());
    return SAMQ_OK;
}

template <typename OutT>
int launch(int fmt, const CUtensorMap& ma, const CUtensorMap& mw, const Fp4Params& p, cudaStream_t st) {
    return fmt == SAMQ_FP4_MX ? launch<OutT, SAMQ_FP4_MX>(ma, mw, p, st) : launch<OutT, SAMQ_FP4_NV>(ma, mw, p, st);
}

}  // namespace

int gemm_fp4_dispatch(const uint8_t* A, int64_t lda, const uint8_t* a_scales, const uint8_t* W, int64_t ldw, const uint8_t* w_scales,
                      int64_t M, int64_t N, int64_t K, int fmt, float alpha, const void* bias, const void* residual, int64_t ldr,
                      int activation, void* out, int out_dtype, int64_t ldo, int32_t* status, void* stream)
{
    if (M < 0 || N <= 0 || K <= 0) return fail(SAMQ_ERR_BAD_ARG, "bad GEMM shape M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
    if (!known_format(fmt)) return fail(SAMQ_ERR_BAD_ARG, "unknown 4-bit format %d", fmt);
    if (activation != SAMQ_ACT_NONE && activation != SAMQ_ACT_GELU) return fail(SAMQ_ERR_BAD_ARG, "unknown activation %d", activation);
    if (out_dtype != SAMQ_F16 && out_dtype != SAMQ_BF16 && out_dtype != SAMQ_F32) return fail(SAMQ_ERR_BAD_ARG, "unknown out_dtype %d", out_dtype);
    if (M == 0) return SAMQ_OK;
    if (A == nullptr || W == nullptr || a_scales == nullptr || w_scales == nullptr || out == nullptr)
        return fail(SAMQ_ERR_BAD_ARG, "operands, scales and out must not be null");
    if (M > 2147483647LL - 256 || N > 2147483647LL - 256 || K > 2147483647LL - 256) return fail(SAMQ_ERR_TOO_LARGE, "GEMM dimension exceeds 2^31");
    if (lda < (K + 1) / 2 || ldw < (K + 1) / 2 || ldo < N || (residual != nullptr && ldr < N))
        return fail(SAMQ_ERR_BAD_ARG, "leading dimension smaller than the row");
    if ((lda & 15) || (ldw & 15) || ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(W) |
         reinterpret_cast<uintptr_t>(a_scales) | reinterpret_cast<uintptr_t>(w_scales)) & 15))
        return fail(SAMQ_ERR_ALIGNMENT, "4-bit operands need 16-byte aligned bases and row strides (lda=%lld ldw=%lld)", (long long)lda, (long long)ldw);
    const size_t esz = out_dtype == SAMQ_F32 ? 4 : 2;
    if ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(residual)) & (esz - 1))
        return fail(SAMQ_ERR_ALIGNMENT, "out, bias and residual must be aligned to their elements");
    Fp4Call c;
    c.A = A; c.lda = lda; c.a_scales = a_scales; c.W = W; c.ldw = ldw; c.w_scales = w_scales;
    c.M = M; c.N = N; c.K = K; c.fmt = fmt; c.out_dtype = out_dtype; c.gelu = activation == SAMQ_ACT_GELU;
    c.status = status; c.stream = static_cast<cudaStream_t>(stream);
    c.epi.M = (int)M; c.epi.N = (int)N; c.epi.alpha = alpha; c.epi.bias = bias; c.epi.residual = residual; c.epi.ldr = ldr;
    c.epi.out = out; c.epi.ldo = ldo;
    c.epi.tma_out = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && (ldo * esz) % 16 == 0;
    c.epi.tma_res = residual != nullptr && (reinterpret_cast<uintptr_t>(residual) & 15) == 0 && (ldr * esz) % 16 == 0;
    if ((M + 255) / 256 * ((N + 191) / 192) >= PAIR_MIN_TILES) {
        memset(&c.map_out, 0, sizeof(c.map_out));
        memset(&c.map_res, 0, sizeof(c.map_res));
        int rc = SAMQ_OK;
        if (c.epi.tma_out) rc = make_row_map(&c.map_out, out, M, N, ldo, (int)esz);
        if (rc == SAMQ_OK && c.epi.tma_res) rc = make_row_map(&c.map_res, residual, M, N, ldr, (int)esz);
        return rc != SAMQ_OK ? rc : gemm_fp4_pair(c);
    }
    CUtensorMap ma, mw;
    int rc = make_operand_map(&ma, reinterpret_cast<const int8_t*>(A), M, (K + 1) / 2, lda, BM);
    if (rc != SAMQ_OK) return rc;
    rc = make_operand_map(&mw, reinterpret_cast<const int8_t*>(W), N, (K + 1) / 2, ldw, BN);
    if (rc != SAMQ_OK) return rc;
    Fp4Params p;
    p.M = (int)M; p.N = (int)N; p.K = (int)K; p.a_scales = a_scales; p.w_scales = w_scales;
    p.groups = (int)groups_of(fmt, K); p.alpha = alpha; p.bias = bias; p.residual = residual; p.ldr = ldr;
    p.out = out; p.ldo = ldo; p.gelu = activation == SAMQ_ACT_GELU; p.status = status;
    p.vec_ok = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && (ldo * esz) % 16 == 0;
    cudaStream_t st = c.stream;
    switch (out_dtype) {
    case SAMQ_F16:  return launch<__half>(fmt, ma, mw, p, st);
    case SAMQ_BF16: return launch<__nv_bfloat16>(fmt, ma, mw, p, st);
    default:        return launch<float>(fmt, ma, mw, p, st);
    }
}

}  // namespace samq
