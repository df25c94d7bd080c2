// The 4-bit product for many rows: a persistent kernel on CTA pairs (tcgen05 cta_group::2).
//
// A pair owns a 256-row tile of 256 or 192 columns.  Each CTA loads its own 128 rows of A with their scales, half of the
// W tile's rows and the scales of the whole W tile, a stage of 256 columns of K at a time.  The leader issues a stage's four
// MMAs (M = 256, N = the tile's columns, K = 64).
//
// The scales reach tensor memory by tcgen05.cp, 12 copies of 512 bytes a stage for nvfp4 and 6 for mxfp4.  In the MMA thread
// their issue would add to the MMAs'; a warp of its own issues them, into a ring of two to four stages behind the
// accumulators.  (Every issuing loop runs in a whole warp with one elected lane: from divergent code each of these
// instructions takes about 50 clocks.  32768 x 5120 x 5120 nvfp4 / mxfp4: copies in the MMA thread 530 / 420 us, beside it
// 685 / 502 from divergent loops, 371 / 326 from warp-uniform ones.)
//
// What bounds the kernel beside the power limit is the traffic between L2 and the SMs, about 45 bytes a clock and SM.
//   K <= 1280 (RESIDENT): the A tile of a pair stays in shared memory, the pair walks along consecutive N tiles of its
//     rows, and a stage is W's part only: 192 columns, two whole accumulators.  1280 -> 5120: 153 -> 134 us (sustained).
//   else: 256 columns, 14 % less traffic a product than 192.  The two accumulators and the scale ring do not fit tensor memory
//     side by side: the second accumulator shares its first columns with the first one's last, and its MMAs start when the
//     epilogue warps that hold those columns have read them.  5120 -> 1280 nvfp4 111 -> 98 us, mxfp4 96 -> 94.
//
// The epilogue warps (32 rows x 64 columns each) read their columns at once and hand them back before they compute.
// The residual comes in by TMA into the warp's staging buffer while the tile is computed, the result leaves from there
// by TMA.  Every wait is bounded.
#include "fp4_gemm.cuh"

namespace samq {
namespace fp4 {

namespace {

constexpr int BM = 128;                          // rows of A of a CTA
constexpr int A_BYTES = BM * BK;
constexpr int FIRST_EPI_WARP = 4;                // TMA, MMA, scale copies, one idle
constexpr int RESIDENT_BLOCKS = 5;               // blocks of 256 columns of a resident A tile
constexpr int TMEM_COLS = 512;
constexpr int MAX_STAGES = 5, MAX_UNITS = 4, MAX_EPI_WARPS = 16;

// The two shapes: RESIDENT with 192-column tiles, else 256.
template <int FMT, bool RESIDENT> struct Shape {
    static constexpr int BN = RESIDENT ? 192 : 256;                // columns of the pair's tile
    static constexpr int BNH = BN / 2;                             // rows of W of a CTA
    static constexpr int STAGES = RESIDENT ? 5 : 4;
    static constexpr int EPI_WARPS = 4 * (BN / EPI_COLS);
    static constexpr int THREADS = (FIRST_EPI_WARP + EPI_WARPS) * 32;
    static constexpr int GROUPS = groups_per_kpad(FMT);            // scale tiles of 128 rows a stage
    static constexpr int UNIT_COLS = 12 * GROUPS;                  // a buffer of the ring: per group 4 columns for A, 8 for W
    static constexpr int UNITS = !RESIDENT ? 3 : FMT == SAMQ_FP4_MX ? 4 : 2;
    static constexpr int SF_COL = TMEM_COLS - UNITS * UNIT_COLS;   // the ring of scale columns behind the accumulators
    static constexpr int ACC1_COL = SF_COL - BN;                   // the second accumulator ends there
    static constexpr int SHARED_COLS = BN > ACC1_COL ? BN - ACC1_COL : 0;      // columns that both accumulators use
    static constexpr int SHARED_GROUPS = (SHARED_COLS + EPI_COLS - 1) / EPI_COLS;
    static constexpr int B_BYTES = BNH * BK;
    static constexpr int SFA_BYTES = GROUPS * TILE_BYTES;
    static constexpr int SFB_BYTES = 2 * GROUPS * TILE_BYTES;      // W's rows lie in two tiles of 128
    static constexpr int A_BLOCK_BYTES = A_BYTES + SFA_BYTES;
    static constexpr int W_BLOCK_BYTES = B_BYTES + SFB_BYTES;
    static_assert(UNITS <= STAGES && UNITS <= MAX_UNITS, "a buffer's last stage is waited for by its place in the ring of stages");
    static_assert(SFB_BYTES % 128 == 0 && ACC1_COL >= 0, "layout");
    static constexpr int A_BLOCKS = RESIDENT ? RESIDENT_BLOCKS : STAGES;       // one a stage, or all of a resident tile
};

struct __align__(8) Control {
    uint64_t full[MAX_STAGES];
    uint64_t empty[MAX_STAGES];
    uint64_t acc_full[2];
    uint64_t acc_empty[2];
    uint64_t shared_empty;                        // the columns that the two accumulators share
    uint64_t sf_ready[MAX_UNITS];                         // scale columns written (the leader's only)
    uint64_t res[MAX_EPI_WARPS];
    uint64_t a_full[RESIDENT_BLOCKS];             // RESIDENT: blocks of A loaded / no longer read
    uint64_t a_empty[RESIDENT_BLOCKS];
    uint32_t tmem_base;
    uint32_t abort_flag;
};

template <int FMT, bool RESIDENT>
constexpr size_t smem_bytes() {
    using S = Shape<FMT, RESIDENT>;
    return 1024 + (size_t)S::A_BLOCKS * S::A_BLOCK_BYTES + (size_t)S::STAGES * S::W_BLOCK_BYTES +
           (size_t)S::EPI_WARPS * (STAGING_BYTES + EPI_COLS * sizeof(float)) + sizeof(Control);
}

struct PairParams {
    EpiParams epi;
    int K, groups;
    int32_t* status;
};

// The tiles of a pair in order, without a division per tile.  RESIDENT: consecutive tiles, so that A changes seldom; else
// the pairs work side by side.
template <bool RESIDENT, int BN>
struct TileWalk {
    int n_blocks, left, m, n, step_m, step_n;
    bool first = true;                            // nothing of the pair's rows has been done before
    __device__ __forceinline__ TileWalk(int num_tiles, int n_blocks_, int pair, int num_pairs) : n_blocks(n_blocks_) {
        const int begin = RESIDENT ? (int)((int64_t)num_tiles * pair / num_pairs) : pair;
        left = RESIDENT ? (int)((int64_t)num_tiles * (pair + 1) / num_pairs) - begin : (num_tiles - pair + num_pairs - 1) / num_pairs;
        m = begin / n_blocks; n = begin % n_blocks;
        step_m = RESIDENT ? 0 : num_pairs / n_blocks; step_n = RESIDENT ? 1 : num_pairs % n_blocks;
    }
    // Columns of the tile's MMA: the last tile of a row is only as wide as it has to be (1280 columns are six tiles of 192
    // and one of 128), in steps of 32 of which each CTA holds half.
    __device__ __forceinline__ int width(int N) const { return min(BN, (N - n * BN + 31) / 32 * 32); }
    __device__ __forceinline__ bool more() const { return left > 0; }
    __device__ __forceinline__ void next() {
        --left; first = false;
        m += step_m; n += step_n;
        if (n >= n_blocks) { n -= n_blocks; ++m; }
    }
    __device__ __forceinline__ bool new_rows() const { return first || n == 0; }                  // RESIDENT
    __device__ __forceinline__ bool rows_done() const { return left > 1 && n == n_blocks - 1; }
};

template <typename OutT, int FMT, bool GELU, bool RES, bool RESIDENT>
__global__ void __launch_bounds__(Shape<FMT, RESIDENT>::THREADS, 1)
gemm_fp4_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                     const __grid_constant__ CUtensorMap map_sfa, const __grid_constant__ CUtensorMap map_sfw,
                     const __grid_constant__ CUtensorMap map_out, const __grid_constant__ CUtensorMap map_res,
                     const __grid_constant__ PairParams p)
{
    using S = Shape<FMT, RESIDENT>;
    constexpr int BN = S::BN, STAGES = S::STAGES, EPI_WARPS = S::EPI_WARPS, B_BYTES = S::B_BYTES;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    uint8_t* tiles = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);              // 1024-byte aligned
    uint8_t* w_tiles = tiles + (size_t)S::A_BLOCKS * A_BYTES;                     // all of these 1024-byte aligned
    uint8_t* staging = w_tiles + (size_t)STAGES * B_BYTES;
    uint8_t* sfa_s = staging + (size_t)EPI_WARPS * STAGING_BYTES;
    uint8_t* sfw_s = sfa_s + (size_t)S::A_BLOCKS * S::SFA_BYTES;
    float* bias_s = reinterpret_cast<float*>(sfw_s + (size_t)STAGES * S::SFB_BYTES);
    Control* ctl = reinterpret_cast<Control*>(bias_s + EPI_WARPS * EPI_COLS);
    volatile uint32_t* abort_flag = &ctl->abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();                       // 0 = leader of the pair
    const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
    const int m_blocks = (p.epi.M + 2 * BM - 1) / (2 * BM);
    const int n_blocks = (p.epi.N + BN - 1) / BN;
    const int k_blocks = (p.K + KPAD - 1) / KPAD;
    const int num_tiles = m_blocks * n_blocks;
    TileWalk<RESIDENT, BN> walk(num_tiles, n_blocks, pair, num_pairs);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(smem_u32(&ctl->full[s]), 1); mbar_init(smem_u32(&ctl->empty[s]), 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(smem_u32(&ctl->acc_full[b]), 1); mbar_init(smem_u32(&ctl->acc_empty[b]), 2 * EPI_WARPS); }
        mbar_init(smem_u32(&ctl->shared_empty), 2 * 4 * (S::SHARED_GROUPS > 0 ? S::SHARED_GROUPS : 1));
        for (int u = 0; u < S::UNITS; ++u) mbar_init(smem_u32(&ctl->sf_ready[u]), 1);
        for (int w = 0; w < EPI_WARPS; ++w) mbar_init(smem_u32(&ctl->res[w]), 1);
        for (int b = 0; b < RESIDENT_BLOCKS; ++b) { mbar_init(smem_u32(&ctl->a_full[b]), 1); mbar_init(smem_u32(&ctl->a_empty[b]), 1); }
        ctl->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&ctl->tmem_base)), "r"((uint32_t)TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    cluster_sync();                                                // both CTAs' barriers exist before any remote arrival
    tcgen05_fence_after();
    const uint32_t tmem = ctl->tmem_base;

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        int stage = 0; uint32_t phase = 0, a_phase = 1;
        bool ok = true;
        for (; walk.more() && ok; walk.next()) {
            const int mt = walk.m * 2 + (int)rank;                         // this CTA's 128-row tile of A
            const int n0 = walk.n * BN;
            const int nt = n0 / TILE_ROWS;                                 // first of W's two scale tiles
            const int w_rows = walk.width(p.epi.N) / 2;                    // of W in this CTA (a whole box is loaded)
            const bool load_a = RESIDENT && walk.new_rows();
            for (int kb = 0; kb < k_blocks; ++kb) {
                if (load_a) ok = mbar_wait_warp(smem_u32(&ctl->a_empty[kb]), a_phase, abort_flag);
                ok = ok && mbar_wait_warp(smem_u32(&ctl->empty[stage]), phase ^ 1u, abort_flag);
                if (!ok) break;
                if (elect_one()) {
                    const uint32_t bar = smem_u32(&ctl->full[stage]), leader_bar = map_to_cta(bar, 0);
                    if (load_a || !RESIDENT) {
                        const int ab = RESIDENT ? kb : stage;
                        const uint32_t a_bar = RESIDENT ? smem_u32(&ctl->a_full[kb]) : bar;
                        const uint32_t a_leader = RESIDENT ? map_to_cta(a_bar, 0) : leader_bar;
                        if (RESIDENT && rank == 0) mbar_expect_tx(a_bar, 2 * S::A_BLOCK_BYTES);       // bytes of both CTAs
                        if (!RESIDENT && rank == 0) mbar_expect_tx(bar, 2 * (S::A_BLOCK_BYTES + S::W_BLOCK_BYTES));
                        tma_load_2d_pair(smem_u32(tiles + (size_t)ab * A_BYTES), &map_a, a_leader, kb * BK, mt * BM);
                        tma_load_2d_pair(smem_u32(sfa_s + (size_t)ab * S::SFA_BYTES), &map_sfa, a_leader, 0, mt * p.groups + kb * S::GROUPS);
                    }
                    if (RESIDENT && rank == 0) mbar_expect_tx(bar, 2 * S::W_BLOCK_BYTES);
                    const uint32_t ss = smem_u32(sfw_s + (size_t)stage * S::SFB_BYTES);
                    tma_load_2d_pair(smem_u32(w_tiles + (size_t)stage * B_BYTES), &map_w, leader_bar, kb * BK, n0 + (int)rank * w_rows);
                    tma_load_2d_pair(ss, &map_sfw, leader_bar, 0, nt * p.groups + kb * S::GROUPS);
                    tma_load_2d_pair(ss + S::SFB_BYTES / 2, &map_sfw, leader_bar, 0, (nt + 1) * p.groups + kb * S::GROUPS);
                }
                __syncwarp();
                if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            }
            if (load_a) a_phase ^= 1u;
        }
        // every stage has been handed back: no completion from the leader's MMAs can still be on its way to this CTA's
        // barriers when the CTA retires
        for (int s = 0; s < STAGES && ok; ++s) {
            ok = mbar_wait_warp(smem_u32(&ctl->empty[stage]), phase ^ 1u, abort_flag);
            if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
        if (!ok) {
            const long long t0 = clock64();
            while (clock64() - t0 < 2000000LL) { }                  // copies in flight land before the CTA retires
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        if (rank == 0) {
            int stage = 0; uint32_t phase = 0;
            int acc = 0; uint32_t acc_phase = 0;
            int unit = 0; uint32_t unit_phase = 0, a_phase = 1, shared_phase = 1;
            bool ok = true;
            for (; walk.more() && ok; walk.next()) {
                const bool wait_a = RESIDENT && walk.new_rows(), free_a = RESIDENT && walk.rows_done();
                if (wait_a) a_phase ^= 1u;
                // the buffer itself (two tiles ago) and the columns that the previous tile's buffer shares with it
                if (!mbar_wait_warp(smem_u32(&ctl->acc_empty[acc]), acc_phase ^ 1u, abort_flag)) break;
                if (S::SHARED_COLS > 0 && !mbar_wait_warp(smem_u32(&ctl->shared_empty), shared_phase, abort_flag)) break;
                shared_phase ^= 1u;
                const uint32_t tmem_d = tmem + (uint32_t)(acc * S::ACC1_COL);
                // an odd tile of 192 rows begins in the middle of a scale tile: skip its first 64 rows, two columns
                const uint32_t idesc_n = (uint32_t)(walk.width(p.epi.N) >> 3) << 17;
                const uint32_t sf_shift = BN % TILE_ROWS != 0 ? (uint32_t)(walk.n & 1) * 2u : 0u;
                for (int kb = 0; kb < k_blocks; ++kb) {
                    ok = mbar_wait_warp(smem_u32(&ctl->full[stage]), phase, abort_flag) &&
                         (!wait_a || mbar_wait_warp(smem_u32(&ctl->a_full[kb]), a_phase, abort_flag)) &&
                         mbar_wait_warp(smem_u32(&ctl->sf_ready[unit]), unit_phase, abort_flag);
                    if (!ok) break;
                    tcgen05_fence_after();
                    const uint64_t adesc = make_smem_desc(smem_u32(tiles + (size_t)(RESIDENT ? kb : stage) * A_BYTES));
                    const uint64_t bdesc = make_smem_desc(smem_u32(w_tiles + (size_t)stage * B_BYTES));
                    const uint32_t sfa = tmem + S::SF_COL + (uint32_t)(unit * S::UNIT_COLS);
                    const uint32_t sfb = sfa + 4 * S::GROUPS + sf_shift;
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < BK / UKB; ++k) {
                            // mxfp4: a word of four scales serves two MMAs, the second taking its upper half (scale id 2)
                            const int g = FMT == SAMQ_FP4_MX ? k / 2 : k;
                            const uint32_t id = FMT == SAMQ_FP4_MX ? 2u * (k & 1) : 0u;
                            mma_fp4<FMT, 2>(tmem_d, adesc + (uint64_t)(k * (UKB >> 4)), bdesc + (uint64_t)(k * (UKB >> 4)),
                                            instr_desc(FMT, 2 * BM, 0, id) | idesc_n, sfa + 4 * g, sfb + 8 * g, (kb | k) != 0 ? 1u : 0u);
                        }
                        if (free_a) tcgen05_commit_both(smem_u32(&ctl->a_empty[kb]));
                        tcgen05_commit_both(smem_u32(&ctl->empty[stage]));
                        if (kb == k_blocks - 1) tcgen05_commit_both(smem_u32(&ctl->acc_full[acc]));
                    }
                    __syncwarp();
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                    if (++unit == S::UNITS) { unit = 0; unit_phase ^= 1u; }
                }
                if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
            }
        }
    } else if (warp == 2) {
        // ---------------- scale copies ----------------
        if (rank == 0) {
            int stage = 0; uint32_t phase = 0;
            int unit = 0;
            int old_stage = 0; uint32_t old_phase = 0;             // the stage that last used the buffer
            int filled = 0;
            uint32_t a_phase = 1;
            bool ok = true;
            for (; walk.more() && ok; walk.next()) {
                const bool wait_a = RESIDENT && walk.new_rows();
                if (wait_a) a_phase ^= 1u;
                for (int kb = 0; kb < k_blocks; ++kb) {
                    ok = mbar_wait_warp(smem_u32(&ctl->full[stage]), phase, abort_flag) &&
                         (!wait_a || mbar_wait_warp(smem_u32(&ctl->a_full[kb]), a_phase, abort_flag));
                    if (ok && filled == S::UNITS) {
                        ok = mbar_wait_warp(smem_u32(&ctl->empty[old_stage]), old_phase, abort_flag);
                        if (++old_stage == STAGES) { old_stage = 0; old_phase ^= 1u; }
                    } else {
                        ++filled;
                    }
                    if (!ok) break;
                    tcgen05_fence_after();
                    const uint32_t sa = smem_u32(sfa_s + (size_t)(RESIDENT ? kb : stage) * S::SFA_BYTES);
                    const uint32_t sw = smem_u32(sfw_s + (size_t)stage * S::SFB_BYTES);
                    const uint32_t sfa = tmem + S::SF_COL + (uint32_t)(unit * S::UNIT_COLS);
                    const uint32_t sfb = sfa + 4 * S::GROUPS;
                    if (elect_one()) {
#pragma unroll
                        for (int g = 0; g < S::GROUPS; ++g) {
                            tmem_copy_scales<2>(sfa + 4 * g, scale_desc(sa + g * TILE_BYTES));
                            tmem_copy_scales<2>(sfb + 8 * g, scale_desc(sw + g * TILE_BYTES));
                            tmem_copy_scales<2>(sfb + 8 * g + 4, scale_desc(sw + S::SFB_BYTES / 2 + g * TILE_BYTES));
                        }
                        tcgen05_commit_pair(smem_u32(&ctl->sf_ready[unit]));
                    }
                    __syncwarp();
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                    if (++unit == S::UNITS) unit = 0;
                }
            }
        }
    } else if (warp >= FIRST_EPI_WARP) {
        // ---------------- epilogue ----------------
        const int ew = warp - FIRST_EPI_WARP;
        const int quad = warp & 3;                                  // TMEM lane quadrant this warp may read
        const int cg = ew >> 2;                                     // which 64 columns
        EpiWarp<OutT, GELU, RES> epi{p.epi, &map_out, &map_res, staging + (size_t)ew * STAGING_BYTES, bias_s + ew * EPI_COLS,
                                     smem_u32(&ctl->res[ew]), 0u, abort_flag, lane};
        int acc = 0; uint32_t acc_phase = 0;
        for (; walk.more(); walk.next()) {
            const int row0 = walk.m * (2 * BM) + (int)rank * BM + quad * 32;
            const int col0 = walk.n * BN + cg * EPI_COLS;
            epi.before(row0, col0);
            if (!mbar_wait_warp(smem_u32(&ctl->acc_full[acc]), acc_phase, abort_flag)) break;
            tcgen05_fence_after();
            uint32_t r[EPI_COLS];
            tmem_ld64(tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc * S::ACC1_COL + cg * EPI_COLS), r);
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) {
                // the last groups of the first buffer and the first ones of the second hold the shared columns
                if (S::SHARED_GROUPS > 0 && (acc == 0 ? cg >= BN / EPI_COLS - S::SHARED_GROUPS : cg < S::SHARED_GROUPS))
                    mbar_arrive_remote(map_to_cta(smem_u32(&ctl->shared_empty), 0));
                mbar_arrive_remote(map_to_cta(smem_u32(&ctl->acc_empty[acc]), 0));
            }
            if (!epi.finish(row0, col0, r)) break;
            if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
        }
        if (lane == 0) bulk_wait0();                                // this warp's stores have completed
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    cluster_sync();                                   // no remote arrival or MMA read of the peer is still in flight
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)TMEM_COLS) : "memory");
    }
    if (threadIdx.x == 0 && ctl->abort_flag != 0 && p.status != nullptr) atomicExch(p.status, 1);
}

template <typename OutT, int FMT, bool GELU, bool RES, bool RESIDENT>
int launch(const Fp4Call& c, const CUtensorMap& ma, const CUtensorMap& mw, const CUtensorMap& msa, const CUtensorMap& msw, const PairParams& p) {
    auto kernel = gemm_fp4_pair_kernel<OutT, FMT, GELU, RES, RESIDENT>;
    constexpr size_t SMEM = smem_bytes<FMT, RESIDENT>();
    SAMQ_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM));
    using S = Shape<FMT, RESIDENT>;
    static_assert(SMEM <= 227 * 1024, "shared memory");
    const int64_t tiles = ((c.M + 2 * BM - 1) / (2 * BM)) * ((c.N + S::BN - 1) / S::BN);
    if (tiles > 2147483647LL - 256) return fail(SAMQ_ERR_TOO_LARGE, "product of %lld x %lld outputs is too large", (long long)c.M, (long long)c.N);
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.blockDim = dim3(S::THREADS); cfg.dynamicSmemBytes = SMEM; cfg.stream = c.stream;
    cfg.attrs = attr; cfg.numAttrs = 1;
    // how many pairs the device can hold at once (GPCs with an odd number of SMs leave one out)
    static thread_local int pairs_cached[64] = {0};
    int dev = 0;
    SAMQ_CUDA_TRY(cudaGetDevice(&dev));
    int max_pairs = (dev >= 0 && dev < 64) ? pairs_cached[dev] : 0;
    if (max_pairs == 0) {
        cfg.gridDim = dim3(2 * (sm_count() / 2));
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) { (void)cudaGetLastError(); n = sm_count() / 2 - 4; }
        max_pairs = n;
        if (dev >= 0 && dev < 64) pairs_cached[dev] = n;
    }
    const int pairs = tiles < max_pairs ? (int)tiles : max_pairs;
    cfg.gridDim = dim3(2 * pairs);
    SAMQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, ma, mw, msa, msw, c.map_out, c.map_res, p));
    return SAMQ_OK;
}

template <typename OutT, int FMT, bool RESIDENT>
int launch(const Fp4Call& c) {
    CUtensorMap ma, mw, msa, msw;
    const int64_t row_bytes = (c.K + 1) / 2;
    int rc = make_operand_map(&ma, reinterpret_cast<const int8_t*>(c.A), c.M, row_bytes, c.lda, BM);
    if (rc == SAMQ_OK) rc = make_operand_map(&mw, reinterpret_cast<const int8_t*>(c.W), c.N, row_bytes, c.ldw, Shape<FMT, RESIDENT>::BNH);
    const int64_t groups = groups_of(FMT, c.K);
    if (rc == SAMQ_OK) rc = make_scale_map(&msa, c.a_scales, (c.M + TILE_ROWS - 1) / TILE_ROWS * groups, Shape<FMT, RESIDENT>::GROUPS);
    if (rc == SAMQ_OK) rc = make_scale_map(&msw, c.w_scales, (c.N + TILE_ROWS - 1) / TILE_ROWS * groups, Shape<FMT, RESIDENT>::GROUPS);
    if (rc != SAMQ_OK) return rc;
    PairParams p;
    p.epi = c.epi; p.K = (int)c.K; p.groups = (int)groups; p.status = c.status;
    const bool res = c.epi.residual != nullptr;
    if (c.gelu && res) return launch<OutT, FMT, true, true, RESIDENT>(c, ma, mw, msa, msw, p);
    if (c.gelu) return launch<OutT, FMT, true, false, RESIDENT>(c, ma, mw, msa, msw, p);
    if (res) return launch<OutT, FMT, false, true, RESIDENT>(c, ma, mw, msa, msw, p);
    return launch<OutT, FMT, false, false, RESIDENT>(c, ma, mw, msa, msw, p);
}

template <typename OutT>
int launch(const Fp4Call& c) {
    if (c.K <= RESIDENT_BLOCKS * KPAD) return c.fmt == SAMQ_FP4_MX ? launch<OutT, SAMQ_FP4_MX, true>(c) : launch<OutT, SAMQ_FP4_NV, true>(c);
    return c.fmt == SAMQ_FP4_MX ? launch<OutT, SAMQ_FP4_MX, false>(c) : launch<OutT, SAMQ_FP4_NV, false>(c);
}

}  // namespace

int gemm_fp4_pair(const Fp4Call& c) {
    switch (c.out_dtype) {
    case SAMQ_F16:  return launch<__half>(c);
    case SAMQ_BF16: return launch<__nv_bfloat16>(c);
    default:        return launch<float>(c);
    }
}

}  // namespace fp4
}  // namespace samq
