// The 4-bit product for few rows (a token, a few tokens, a window) and the checks and dispatch of samq_gemm_fp4 and
// samq_linear_fp4.
//
// Few rows leave the output too small for the device, and the weight's bytes and the latency of one pass are what counts.
// So the operands change places: 128 rows of W are the M side of the MMA, the T <= 128 rows of the activation its N side
// (T a multiple of 8: one token costs an eighth of an N = 64 MMA), and a cluster of S CTAs splits K, each CTA with its
// own range of 256-column blocks and all of its loads in flight at once.  The S partial tiles meet in distributed shared
// memory: after a cluster barrier every CTA sums a share of the rows over the S copies in rank order (the result does
// not depend on timing), finishes them and stores them.
//
// samq_linear_fp4 also quantizes here: the four epilogue warps round the CTA's K range of the activation to codes and
// scales straight into the shared-memory layout that the MMA reads, which saves a launch and the trip through memory.
// Every N tile repeats that work, so it is for at most 32 rows.
#include "fp4_gemm.cuh"

namespace samq {

using namespace fp4;

namespace {

constexpr int BW = 128;                          // rows of W of a CTA
constexpr int MAX_T = 128;                       // rows of the activation of a CTA
constexpr int STAGES = 4;
constexpr int MAX_SPLIT = 8;
constexpr int W_BYTES = BW * BK;
constexpr int EPI_WARPS = 4;
constexpr int EPI_THREADS = EPI_WARPS * 32;
constexpr int THREADS = 64 + EPI_THREADS;
constexpr int FUSED_MAX_ROWS = SAMQ_LINEAR_FP4_MAX_ROWS;

struct __align__(8) Control {
    uint64_t full[STAGES];
    uint64_t empty[STAGES];
    uint64_t acc_full;
    uint32_t tmem_base;
    uint32_t abort_flag;
};

struct SmallParams {
    int M, N, K;
    int T;                                        // rows of the activation in a tile, a multiple of 8
    int groups;
    const uint8_t* a_scales;                      // unless the kernel quantizes
    const uint8_t* w_scales;
    const void* x; int64_t ldx; int access_x;     // the activation, if the kernel quantizes it
    int tmem_cols;
    float alpha;
    const void* bias;
    const void* residual; int64_t ldr;
    void* out; int64_t ldo;
    int gelu;
    int32_t* status;
};

template <int FMT> struct Shape {
    static constexpr int GROUPS = groups_per_kpad(FMT);
    static constexpr int SF_BYTES = GROUPS * TILE_BYTES;
    static constexpr int SF_COLS = 8 * GROUPS;                     // columns of tensor memory for one stage's scales
};
template <int FMT>
__host__ __device__ constexpr int stage_bytes(int T) { return W_BYTES + T * BK; }
template <int FMT>
size_t smem_bytes(int T) { return 1024 + (size_t)STAGES * (stage_bytes<FMT>(T) + 2 * Shape<FMT>::SF_BYTES) + sizeof(Control); }

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t cluster_nctas() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
    return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t cluster_addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
    return v;
}

// QUANT: the activation is `x` of type OutT, quantized here; otherwise codes and scales are loaded.
template <typename OutT, int FMT, bool QUANT>
__global__ void __launch_bounds__(THREADS)
gemm_fp4_small_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const SmallParams p)
{
    using S = Shape<FMT>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    uint8_t* tiles = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
    const int st_bytes = stage_bytes<FMT>(p.T);
    uint8_t* sf = tiles + (size_t)STAGES * st_bytes;
    Control* ctl = reinterpret_cast<Control*>(sf + (size_t)STAGES * 2 * S::SF_BYTES);
    float* partial = reinterpret_cast<float*>(tiles);                   // [T][128], once the stages are done with
    volatile uint32_t* abort_flag = &ctl->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = (int)cluster_nctas(), rank = (int)cluster_ctarank();
    const int nt = blockIdx.x / split, mt = blockIdx.y;
    const int n0 = nt * BW, m0 = mt * MAX_T;
    const int k_blocks = (p.K + KPAD - 1) / KPAD;
    const int kb_first = rank * (k_blocks / split) + min(rank, k_blocks % split);
    const int kb_count = k_blocks / split + (rank < k_blocks % split ? 1 : 0);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(smem_u32(&ctl->full[s]), QUANT ? 1 + EPI_THREADS : 1); mbar_init(smem_u32(&ctl->empty[s]), 1); }
        mbar_init(smem_u32(&ctl->acc_full), 1);
        ctl->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&ctl->tmem_base)), "r"((uint32_t)p.tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = ctl->tmem_base;

    if (warp == 0) {
        bool ok = true;
        for (int i = 0; i < kb_count; ++i) {
            const int s = i % STAGES, kb = kb_first + i;
            ok = mbar_wait(smem_u32(&ctl->empty[s]), ((i / STAGES) & 1) ^ 1u, abort_flag);
            if (!ok) break;
            if (elect_one()) {
                const uint32_t bar = smem_u32(&ctl->full[s]);
                const uint32_t sw = smem_u32(tiles + (size_t)s * st_bytes);
                const uint32_t ss = smem_u32(sf + (size_t)s * 2 * S::SF_BYTES);
                mbar_expect_tx(bar, W_BYTES + S::SF_BYTES + (QUANT ? 0 : p.T * BK + S::SF_BYTES));
                tma_load_2d(sw, &map_w, bar, kb * BK, n0);
                bulk_load(ss, p.w_scales + ((int64_t)nt * p.groups + kb * S::GROUPS) * TILE_BYTES, S::SF_BYTES, bar);
                if constexpr (!QUANT) {
                    tma_load_2d(sw + W_BYTES, &map_a, bar, kb * BK, m0);
                    bulk_load(ss + S::SF_BYTES, p.a_scales + ((int64_t)mt * p.groups + kb * S::GROUPS) * TILE_BYTES, S::SF_BYTES, bar);
                }
            }
            __syncwarp();
        }
        if (!ok) {
            const long long t0 = clock64();
            while (clock64() - t0 < 2000000LL) { }                  // copies in flight land before the CTA retires
        }
    } else if (warp == 1) {
        bool ok = true;
        const uint32_t idesc_n = (uint32_t)p.T;
        for (int i = 0; i < kb_count; ++i) {
            const int s = i % STAGES;
            ok = mbar_wait(smem_u32(&ctl->full[s]), (i / STAGES) & 1, abort_flag);
            if (!ok) break;
            tcgen05_fence_after();
            const uint32_t sw = smem_u32(tiles + (size_t)s * st_bytes);
            const uint32_t ss = smem_u32(sf + (size_t)s * 2 * S::SF_BYTES);
            const uint32_t sf_w = tmem + (uint32_t)p.T + (uint32_t)((i & 1) * S::SF_COLS);
            const uint32_t sf_a = sf_w + 4 * S::GROUPS;
            const uint64_t wdesc = make_smem_desc(sw), adesc = make_smem_desc(sw + W_BYTES);
            if (elect_one()) {
#pragma unroll
                for (int g = 0; g < S::GROUPS; ++g) {
                    tmem_copy_scales<1>(sf_w + 4 * g, scale_desc(ss + g * TILE_BYTES));
                    tmem_copy_scales<1>(sf_a + 4 * g, scale_desc(ss + S::SF_BYTES + g * TILE_BYTES));
                }
#pragma unroll
                for (int k = 0; k < BK / UKB; ++k) {
                    // mxfp4: a word of four scales serves two MMAs, the second taking its upper half (scale id 2)
                    const int g = FMT == SAMQ_FP4_MX ? k / 2 : k;
                    const uint32_t id = FMT == SAMQ_FP4_MX ? 2u * (k & 1) : 0u;
                    mma_fp4<FMT, 1>(tmem, wdesc + (uint64_t)(k * (UKB >> 4)), adesc + (uint64_t)(k * (UKB >> 4)),
                                    instr_desc(FMT, BW, 0, id) | ((idesc_n >> 3) << 17), sf_w + 4 * g, sf_a + 4 * g, (i | k) != 0 ? 1u : 0u);
                }
                tcgen05_commit(smem_u32(&ctl->empty[s]));
                if (i == kb_count - 1) tcgen05_commit(smem_u32(&ctl->acc_full));
            }
            __syncwarp();
        }
    } else {
        const int quad = warp & 3;
        if constexpr (QUANT) {
            // the CTA's columns of the activation, 16 a thread and step, into the operand layout (128-byte swizzle) and its
            // scale tile; rows behind M are zero
            constexpr int CHUNKS = KPAD / 16;                       // of a row and stage
            const int tid = threadIdx.x - 64;
            bool ok = true;
            for (int i = 0; i < kb_count && ok; ++i) {
                const int s = i % STAGES, kb = kb_first + i;
                ok = mbar_wait(smem_u32(&ctl->empty[s]), ((i / STAGES) & 1) ^ 1u, abort_flag);
                if (!ok) break;
                uint8_t* codes = tiles + (size_t)s * st_bytes + W_BYTES;
                uint8_t* scales = sf + (size_t)s * 2 * S::SF_BYTES + S::SF_BYTES;
                for (int c = tid; c < p.T * CHUNKS; c += EPI_THREADS) {
                    const int r = c / CHUNKS, j = c % CHUNKS, col = kb * KPAD + j * 16;
                    Chunk<OutT> x;
                    load_chunk(x, static_cast<const OutT*>(p.x) + (int64_t)(m0 + r) * p.ldx + col, m0 + r < p.M ? min(16, p.K - col) : 0, p.access_x);
                    uint32_t amax = x.amax_bits();
                    if constexpr (FMT == SAMQ_FP4_MX) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                    const Scale sc = block_scale<FMT>(amax, 1.0f, 1.0f);
                    *reinterpret_cast<uint2*>(codes + staged(r, j * 8)) = encode_chunk<FMT>(x, sc, amax < 0x7F800000u);
                    const int block = j * 16 / block_of(FMT);
                    if (FMT == SAMQ_FP4_NV || (j & 1) == 0)
                        scales[(block / 4) * TILE_BYTES + r * 16 + (block & 3)] = (uint8_t)(kb * KPAD + block * block_of(FMT) < p.K ? sc.byte : 0u);
                }
                fence_async_smem();
                mbar_arrive(smem_u32(&ctl->full[s]));
            }
        }
        if (mbar_wait(smem_u32(&ctl->acc_full), 0, abort_flag)) {
            tcgen05_fence_after();
            for (int c = 0; c < p.T; c += 8) {
                uint32_t r[8];
                asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                             : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                             : "r"(tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)c));
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 8; ++j) partial[(c + j) * BW + quad * 32 + lane] = __uint_as_float(r[j]);
            }
        }
        tcgen05_fence_before();
    }
    __syncthreads();
    tcgen05_fence_after();
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)p.tmem_cols) : "memory");
    }
    if (split > 1) cluster_sync();                                  // every CTA's partial sums are in its shared memory
    if (warp >= 2) {
        const int col = (warp & 3) * 32 + lane, n = n0 + col;
        if (n < p.N) {
            const float bias = p.bias != nullptr ? OutOps<OutT>::up(static_cast<const OutT*>(p.bias)[n]) : 0.0f;
            const uint32_t base = smem_u32(partial);
            const int rows = min(p.T, p.M - m0);
            for (int r = rank; r < rows; r += split) {              // the ranks share the rows
                float v[MAX_SPLIT];
#pragma unroll
                for (int q = 0; q < MAX_SPLIT; ++q)
                    v[q] = q < split ? ld_cluster(map_to_cta(base + (uint32_t)(r * BW + col) * 4u, (uint32_t)q)) : 0.0f;
                float y = v[0];
#pragma unroll
                for (int q = 1; q < MAX_SPLIT; ++q) y += v[q];
                y = fmaf(y, p.alpha, bias);
                if (p.gelu) y = gelu_erf(y);
                const int64_t m = m0 + r;
                if (p.residual != nullptr) y += OutOps<OutT>::up(static_cast<const OutT*>(p.residual)[m * p.ldr + n]);
                static_cast<OutT*>(p.out)[m * p.ldo + n] = OutOps<OutT>::down(y);
            }
        }
    }
    if (threadIdx.x == 0 && ctl->abort_flag != 0 && p.status != nullptr) atomicExch(p.status, 1);
    __syncwarp();
    if (split > 1) cluster_sync();                                  // nobody reads a retired CTA's shared memory
}

template <typename OutT, int FMT, bool QUANT>
int launch_small(const Fp4Call& c, SmallParams& p, const CUtensorMap& ma, const CUtensorMap& mw) {
    auto kernel = gemm_fp4_small_kernel<OutT, FMT, QUANT>;
    // the largest tile's shared memory, set once per device
    static thread_local bool ready[64] = {false};
    int dev = 0;
    SAMQ_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        SAMQ_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes<FMT>(MAX_T)));
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    const int64_t n_tiles = (c.N + BW - 1) / BW, m_tiles = (c.M + MAX_T - 1) / MAX_T;
    const int64_t k_blocks = (c.K + KPAD - 1) / KPAD;
    // split K until about two small CTAs or one large one sit on every SM
    const int64_t room = (p.T <= 32 ? 2 : 1) * sm_count() / (n_tiles * m_tiles);
    int split = (int)(room < 1 ? 1 : room > MAX_SPLIT ? MAX_SPLIT : room);
    if (split > k_blocks) split = (int)k_blocks;
    if (n_tiles * split > 2147483647LL || m_tiles > 65535) return fail(SAMQ_ERR_TOO_LARGE, "product of %lld x %lld outputs is too large", (long long)c.M, (long long)c.N);
    const int cols = p.T + 2 * Shape<FMT>::SF_COLS;
    p.tmem_cols = cols <= 64 ? 64 : cols <= 128 ? 128 : 256;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)split; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(n_tiles * split), (unsigned)m_tiles);
    cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = smem_bytes<FMT>(p.T); cfg.stream = c.stream;
    cfg.attrs = attr; cfg.numAttrs = 1;
    SAMQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, ma, mw, p));
    return SAMQ_OK;
}

// x != nullptr: quantize it in the kernel
int gemm_fp4_small(const Fp4Call& c, const void* x, int64_t ldx) {
    SmallParams p;
    p.M = (int)c.M; p.N = (int)c.N; p.K = (int)c.K;
    p.T = c.M >= MAX_T ? MAX_T : (int)((c.M + 7) / 8 * 8);
    p.groups = (int)groups_of(c.fmt, c.K); p.a_scales = c.a_scales; p.w_scales = c.w_scales;
    const size_t esz = c.out_dtype == SAMQ_F32 ? 4 : 2;
    p.x = x; p.ldx = ldx; p.access_x = row_access(x, ldx * (int64_t)esz);
    p.alpha = c.epi.alpha; p.bias = c.epi.bias; p.residual = c.epi.residual; p.ldr = c.epi.ldr; p.out = c.epi.out; p.ldo = c.epi.ldo;
    p.gelu = c.gelu; p.status = c.status;
    CUtensorMap ma, mw;
    const int64_t row_bytes = (c.K + 1) / 2;
    int rc = make_operand_map(&mw, reinterpret_cast<const int8_t*>(c.W), c.N, row_bytes, c.ldw, BW);
    if (rc == SAMQ_OK && x == nullptr) rc = make_operand_map(&ma, reinterpret_cast<const int8_t*>(c.A), c.M, row_bytes, c.lda, p.T);
    if (rc != SAMQ_OK) return rc;
    if (x != nullptr) ma = mw;                                      // not used
    const bool mx = c.fmt == SAMQ_FP4_MX;
#define SAMQ_SMALL(T)                                                                                                        \
    (x != nullptr ? (mx ? launch_small<T, SAMQ_FP4_MX, true>(c, p, ma, mw) : launch_small<T, SAMQ_FP4_NV, true>(c, p, ma, mw)) \
                  : (mx ? launch_small<T, SAMQ_FP4_MX, false>(c, p, ma, mw) : launch_small<T, SAMQ_FP4_NV, false>(c, p, ma, mw)))
    switch (c.out_dtype) {
    case SAMQ_F16:  return SAMQ_SMALL(__half);
    case SAMQ_BF16: return SAMQ_SMALL(__nv_bfloat16);
    default:        return SAMQ_SMALL(float);
    }
#undef SAMQ_SMALL
}

// 256 x 192 tiles from which the pair kernel has enough to do
constexpr int PAIR_MIN_TILES = 32;

// What both entry points check: everything but the activation.
int check_call(Fp4Call& c, int64_t M, int64_t N, int64_t K, int fmt, const uint8_t* W, int64_t ldw, const uint8_t* w_scales, float alpha,
               const void* bias, const void* residual, int64_t ldr, int activation, void* out, int out_dtype, int64_t ldo,
               int32_t* status, void* stream)
{
    if (M < 0 || N <= 0 || K <= 0) return fail(SAMQ_ERR_BAD_ARG, "bad GEMM shape M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
    if (!known_format(fmt)) return fail(SAMQ_ERR_BAD_ARG, "unknown 4-bit format %d", fmt);
    if (activation != SAMQ_ACT_NONE && activation != SAMQ_ACT_GELU) return fail(SAMQ_ERR_BAD_ARG, "unknown activation %d", activation);
    if (out_dtype != SAMQ_F16 && out_dtype != SAMQ_BF16 && out_dtype != SAMQ_F32) return fail(SAMQ_ERR_BAD_ARG, "unknown out_dtype %d", out_dtype);
    if (M > 2147483647LL - 256 || N > 2147483647LL - 256 || K > 2147483647LL - 256) return fail(SAMQ_ERR_TOO_LARGE, "GEMM dimension exceeds 2^31");
    if (M == 0) return SAMQ_OK;
    if (W == nullptr || w_scales == nullptr || out == nullptr) return fail(SAMQ_ERR_BAD_ARG, "operands, scales and out must not be null");
    if (ldw < (K + 1) / 2 || ldo < N || (residual != nullptr && ldr < N)) return fail(SAMQ_ERR_BAD_ARG, "leading dimension smaller than the row");
    if ((ldw & 15) || ((reinterpret_cast<uintptr_t>(W) | reinterpret_cast<uintptr_t>(w_scales)) & 15))
        return fail(SAMQ_ERR_ALIGNMENT, "4-bit operands need 16-byte aligned bases and row strides (ldw=%lld)", (long long)ldw);
    const size_t esz = out_dtype == SAMQ_F32 ? 4 : 2;
    if ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(residual)) & (esz - 1))
        return fail(SAMQ_ERR_ALIGNMENT, "out, bias and residual must be aligned to their elements");
    c.A = nullptr; c.lda = 0; c.a_scales = nullptr; c.W = W; c.ldw = ldw; c.w_scales = w_scales;
    c.M = M; c.N = N; c.K = K; c.fmt = fmt; c.out_dtype = out_dtype; c.gelu = activation == SAMQ_ACT_GELU;
    c.status = status; c.stream = static_cast<cudaStream_t>(stream);
    c.epi.M = (int)M; c.epi.N = (int)N; c.epi.alpha = alpha; c.epi.bias = bias; c.epi.residual = residual; c.epi.ldr = ldr;
    c.epi.out = out; c.epi.ldo = ldo;
    c.epi.tma_out = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && (ldo * esz) % 16 == 0;
    c.epi.tma_res = residual != nullptr && (reinterpret_cast<uintptr_t>(residual) & 15) == 0 && (ldr * esz) % 16 == 0;
    return SAMQ_OK;
}

}  // namespace

int gemm_fp4_dispatch(const uint8_t* A, int64_t lda, const uint8_t* a_scales, const uint8_t* W, int64_t ldw, const uint8_t* w_scales,
                      int64_t M, int64_t N, int64_t K, int fmt, float alpha, const void* bias, const void* residual, int64_t ldr,
                      int activation, void* out, int out_dtype, int64_t ldo, int32_t* status, void* stream)
{
    Fp4Call c;
    int rc = check_call(c, M, N, K, fmt, W, ldw, w_scales, alpha, bias, residual, ldr, activation, out, out_dtype, ldo, status, stream);
    if (rc != SAMQ_OK || M == 0) return rc;
    if (A == nullptr || a_scales == nullptr) return fail(SAMQ_ERR_BAD_ARG, "operands, scales and out must not be null");
    if (lda < (K + 1) / 2) return fail(SAMQ_ERR_BAD_ARG, "leading dimension smaller than the row");
    if ((lda & 15) || ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(a_scales)) & 15))
        return fail(SAMQ_ERR_ALIGNMENT, "4-bit operands need 16-byte aligned bases and row strides (lda=%lld)", (long long)lda);
    c.A = A; c.lda = lda; c.a_scales = a_scales;
    if (M <= MAX_T || (M + 255) / 256 * ((N + 191) / 192) < PAIR_MIN_TILES) return gemm_fp4_small(c, nullptr, 0);
    const int esz = out_dtype == SAMQ_F32 ? 4 : 2;
    memset(&c.map_out, 0, sizeof(c.map_out));
    memset(&c.map_res, 0, sizeof(c.map_res));
    if (c.epi.tma_out) rc = make_row_map(&c.map_out, out, M, N, ldo, esz);
    if (rc == SAMQ_OK && c.epi.tma_res) rc = make_row_map(&c.map_res, residual, M, N, ldr, esz);
    return rc != SAMQ_OK ? rc : gemm_fp4_pair(c);
}

int linear_fp4_dispatch(const void* x, int dtype, int64_t ldx, const uint8_t* W, int64_t ldw, const uint8_t* w_scales,
                        int64_t M, int64_t N, int64_t K, int fmt, float alpha, const void* bias, const void* residual, int64_t ldr,
                        int activation, void* out, int64_t ldo, int32_t* status, void* stream)
{
    Fp4Call c;
    int rc = check_call(c, M, N, K, fmt, W, ldw, w_scales, alpha, bias, residual, ldr, activation, out, dtype, ldo, status, stream);
    if (rc != SAMQ_OK) return rc;
    if (M > FUSED_MAX_ROWS) return fail(SAMQ_ERR_TOO_LARGE, "the one-kernel 4-bit linear takes at most %d rows, got %lld", FUSED_MAX_ROWS, (long long)M);
    if (M == 0) return SAMQ_OK;
    if (x == nullptr) return fail(SAMQ_ERR_BAD_ARG, "x must not be null");
    if (ldx < K) return fail(SAMQ_ERR_BAD_ARG, "ldx smaller than K");
    if (reinterpret_cast<uintptr_t>(x) & (dtype == SAMQ_F32 ? 3 : 1)) return fail(SAMQ_ERR_ALIGNMENT, "x must be aligned to its elements");
    return gemm_fp4_small(c, x, ldx);
}

}  // namespace samq
