// The 4-bit product for few rows (a token, a few tokens, a window) and the checks and dispatch of samq_gemm_fp4 and
// samq_linear_fp4.
//
// Few rows leave the output too small for the device, and the weight's bytes and the latency of one pass are what counts.
// So the operands change places: 128 rows of W are the M side of the MMA, the T <= 128 rows of the activation its N side
// (T a multiple of 8: one token costs an eighth of an N = 64 MMA), and a cluster of S CTAs splits K, each CTA with its
// own range of 256-column blocks and all of its loads in flight at once.  The S partial tiles are joined by rows: a CTA
// owns a share of them; every CTA pushes its sums of a row into the owner's shared memory (st.async, counted by the
// owner's barrier), and the owner adds the S copies in rank order (the result does not depend on timing), finishes
// the row and stores it.  Nothing waits for the whole cluster but the first push, for a barrier that all have passed at
// their start; pulling the sums after a cluster barrier and a second one before the exit took 4000 of 7400 clocks.
//
// samq_linear_fp4 also quantizes here: the epilogue warps round the CTA's K range of the activation to codes and
// scales straight into the shared-memory layout that the MMA reads, which saves a launch and the trip through memory.
// Every N tile repeats that work, so it is for at most 32 rows.
//
// Measured (20 calls in a captured graph, behind a flush of L2, on up to six weights in turn): 8 x 3840 x 1280 5.3 us, 1 x 5120 x
// 1280 with the quantization 5.9, 196 x 2304 x 768 5.3: the latency of one pass (loads 1.1 us, stores 0.4, the rest launch and
// set-up); 1 x 40000 x 5120 from memory 28 us, 4.1 TB/s.
#include "fp4_gemm.cuh"
#include <float.h>

namespace samq {

using namespace fp4;

namespace {

constexpr int BW = 128;                          // rows of W of a CTA
constexpr int MAX_T = 128;                       // rows of the activation of a CTA
constexpr int MIN_STAGES = 3, MAX_STAGES = 8;    // as many as leave room for two CTAs on an SM
constexpr int MAX_SPLIT = 8;                    // the portable cluster size
constexpr int W_BYTES = BW * BK;
constexpr int EPI_WARPS = 8;                     // two for each quarter of the 128 columns, taking turns by 16 rows
constexpr int EPI_THREADS = EPI_WARPS * 32;
constexpr int THREADS = 64 + EPI_THREADS;
constexpr int FUSED_MAX_ROWS = SAMQ_LINEAR_FP4_ONE_KERNEL_ROWS, FUSED_MOST = SAMQ_LINEAR_FP4_ONE_KERNEL_WORK;

struct __align__(8) Control {
    uint64_t full[MAX_STAGES];
    uint64_t empty[MAX_STAGES];
    uint64_t acc_full;
    uint64_t joined;                              // the sums of this CTA's rows have arrived from every CTA
    uint32_t tmem_base;
    uint32_t abort_flag;
};

struct SmallParams {
    int M, N, K;
    int T;                                        // rows of the activation in a tile, a multiple of 8
    int stages;
    int groups;
    const uint8_t* a_scales;                      // unless the kernel quantizes
    const uint8_t* w_scales;
    const void* x; int64_t ldx; int access_x;     // the activation, if the kernel quantizes it
    float x_global_scale, inv_x_global_scale;
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
inline int tile_rows(int64_t M) { return M >= MAX_T ? MAX_T : (int)((M + 7) / 8 * 8); }
// rows of a tile that one of `split` CTAs owns, at most
__host__ __device__ inline int owned_rows(int rows, int split) { return (rows + split - 1) / split; }
constexpr size_t HALF_SM = 112 * 1024;           // shared memory of one of two CTAs on an SM
inline size_t joined_bytes(int T, int split) { return split > 1 ? (size_t)split * owned_rows(T, split) * BW * sizeof(float) : 0; }
template <int FMT>
int stages_of(int T, int split) {
    const int n = (int)((HALF_SM - 2048 - (T <= 32 ? joined_bytes(T, split) : 0)) / (stage_bytes<FMT>(T) + 2 * Shape<FMT>::SF_BYTES));
    return n < MIN_STAGES ? MIN_STAGES : n > MAX_STAGES ? MAX_STAGES : n;
}
template <int FMT>
size_t smem_bytes(int T, int stages, int split) {
    return 1024 + (size_t)stages * (stage_bytes<FMT>(T) + 2 * Shape<FMT>::SF_BYTES) + joined_bytes(T, split) + sizeof(Control);
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t cluster_nctas() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
    return r;
}
// one value into another CTA's shared memory, counted by a barrier there
__device__ __forceinline__ void push_async(uint32_t cluster_addr, float v, uint32_t cluster_bar) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];"
                 ::"r"(cluster_addr), "r"(__float_as_uint(v)), "r"(cluster_bar) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr));
    tmem_ld_wait();
}

// The residual under up to 16 neighbouring rows of output column n from row m on, asked for before the sums are there: its
// way from memory is a good part of a small call (2777 x 1001 x 1283, 176 CTAs of 4 x 16 rows a warp: 14.3 -> 12.0 us).
template <typename OutT, bool RES>
__device__ __forceinline__ void load_residual(const SmallParams& p, int n, int64_t m, int count, OutT (&r)[16]) {
    if (!RES || n >= p.N) return;
    const OutT* res = static_cast<const OutT*>(p.residual) + m * p.ldr + n;
#pragma unroll
    for (int j = 0; j < 16; ++j)
        if (j < count) { r[j] = *res; res += p.ldr; }
}
// those rows' outputs: the sums in y
template <typename OutT, bool RES>
__device__ __forceinline__ void finish_rows(const SmallParams& p, int n, float bias, int64_t m, int count, float (&y)[16], const OutT (&r)[16]) {
    OutT* out = static_cast<OutT*>(p.out) + m * p.ldo + n;
    const bool all = count >= 16;                                   // the same in all threads, as the other branches here
#pragma unroll
    for (int j = 0; j < 16; ++j) y[j] = fmaf(y[j], p.alpha, bias);
    if (p.gelu) {
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
            const float2 g = gelu_pair(make_float2(y[j], y[j + 1]));
            y[j] = g.x; y[j + 1] = g.y;
        }
    }
    if (RES) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (all || j < count) y[j] += OutOps<OutT>::up(r[j]);
    }
    if (all) {
#pragma unroll
        for (int j = 0; j < 16; ++j) { *out = OutOps<OutT>::down(y[j]); out += p.ldo; }
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (j < count) { *out = OutOps<OutT>::down(y[j]); out += p.ldo; }
    }
}

// Quantization of `blocks` k-blocks of the activation's `rows` rows from kb on, into the operand layout (128-byte swizzle) and
// scale tiles of as many stages of the ring from `stage` on.  (What the tile's other rows hold only meets output rows that do
// not exist.)  Sixteen threads take the chunks of 16 columns of one row and block; 16 rows at a time, BATCH times: the loads
// of a batch are under way together, and may be while a stage is waited for.
constexpr int BATCH = 4;
constexpr int BATCH_ROWS = EPI_THREADS / 16;
struct RowOf {                                   // idx = block * rows + row, for idx < 2048 and rows <= 32
    int rows, inv;
    __device__ __forceinline__ explicit RowOf(int rows_) : rows(rows_), inv((65536 + rows_ - 1) / rows_) {}
    __device__ __forceinline__ int block(int idx) const { return (idx * inv) >> 16; }
};

template <typename T>
__device__ __forceinline__ void load_batch(const SmallParams& p, const RowOf& of, int m0, int kb, int blocks, int first, int tid, Chunk<T> (&x)[BATCH]) {
    const int total = blocks * of.rows;
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
        if (first + u * BATCH_ROWS >= total) break;                // the same in all threads; those behind the end repeat the last row
        const int idx = min(first + u * BATCH_ROWS + (tid >> 4), total - 1), b = of.block(idx), r = idx - b * of.rows;
        const int col = (kb + b) * KPAD + (tid & 15) * 16;
        load_chunk(x[u], static_cast<const T*>(p.x) + (int64_t)(m0 + r) * p.ldx + col, min(16, p.K - col), p.access_x);
    }
}
template <typename T, int FMT>
__device__ __forceinline__ void quantize_batch(const SmallParams& p, const RowOf& of, int kb, int blocks, int first, int tid, int stage,
                                               const Chunk<T> (&x)[BATCH], uint8_t* tiles, int st_bytes, uint8_t* sf) {
    const int total = blocks * of.rows, j = tid & 15, block = j * 16 / block_of(FMT);
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
        if (first + u * BATCH_ROWS >= total) break;
        const int idx = min(first + u * BATCH_ROWS + (tid >> 4), total - 1), b = of.block(idx), r = idx - b * of.rows;
        const int s = stage + b < p.stages ? stage + b : stage + b - p.stages;
        uint32_t amax = x[u].amax_bits();
        if constexpr (FMT == SAMQ_FP4_MX) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        const Scale sc = block_scale<FMT>(amax, p.x_global_scale, p.inv_x_global_scale);
        Chunk<T> held = x[u];
        hold_far<FMT>(held, sc, p.x_global_scale);
        *reinterpret_cast<uint2*>(tiles + (size_t)s * st_bytes + W_BYTES + r * BK + ((uint32_t)(j * 8) ^ ((uint32_t)(r & 7) << 4))) =
            encode_chunk<FMT>(held, sc, amax < 0x7F800000u);
        if (FMT == SAMQ_FP4_NV || (j & 1) == 0)
            sf[(size_t)(2 * s + 1) * Shape<FMT>::SF_BYTES + (block / 4) * TILE_BYTES + r * 16 + (block & 3)] =
                (uint8_t)((kb + b) * KPAD + block * block_of(FMT) < p.K ? sc.byte : 0u);
    }
}

// QUANT: the activation is `x` of type OutT, quantized here; otherwise codes and scales are loaded.  RES: with a residual
// (whose registers cost a call without one 0.3 us).
template <typename OutT, int FMT, bool QUANT, bool RES>
__global__ void __launch_bounds__(THREADS, 2)
gemm_fp4_small_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const SmallParams p)
{
    using S = Shape<FMT>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    uint8_t* tiles = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
    const int st_bytes = stage_bytes<FMT>(p.T);
    const int stages = p.stages;
    uint8_t* sf = tiles + (size_t)stages * st_bytes;
    const int split = (int)cluster_nctas(), rank = (int)cluster_ctarank();
    float* joined = reinterpret_cast<float*>(sf + (size_t)stages * 2 * S::SF_BYTES);     // [split][own_max][128]
    Control* ctl = reinterpret_cast<Control*>(joined + (split > 1 ? split * owned_rows(p.T, split) * BW : 0));
    volatile uint32_t* abort_flag = &ctl->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nt = blockIdx.x / split, mt = blockIdx.y;
    const int n0 = nt * BW, m0 = mt * MAX_T;
    const int k_blocks = (p.K + KPAD - 1) / KPAD;
    const int kb_first = rank * (k_blocks / split) + min(rank, k_blocks % split);
    const int kb_count = k_blocks / split + (rank < k_blocks % split ? 1 : 0);

    auto load_stage = [&](int i) {                                  // by one thread
        const int s = i % stages, kb = kb_first + i;
        const uint32_t bar = smem_u32(&ctl->full[s]);
        const uint32_t sw = smem_u32(tiles + (size_t)s * st_bytes), ss = smem_u32(sf + (size_t)s * 2 * S::SF_BYTES);
        mbar_expect_tx(bar, W_BYTES + S::SF_BYTES + (QUANT ? 0 : p.T * BK + S::SF_BYTES));
        tma_load_2d(sw, &map_w, bar, kb * BK, n0);
        bulk_load(ss, p.w_scales + ((int64_t)nt * p.groups + kb * S::GROUPS) * TILE_BYTES, S::SF_BYTES, bar);
        if constexpr (!QUANT) {
            tma_load_2d(sw + W_BYTES, &map_a, bar, kb * BK, m0);
            bulk_load(ss + S::SF_BYTES, p.a_scales + ((int64_t)mt * p.groups + kb * S::GROUPS) * TILE_BYTES, S::SF_BYTES, bar);
        }
    };
    const int rows = min(p.T, p.M - m0);
    const int own_max = owned_rows(rows, split);
    const int owned = max(0, min(own_max, rows - rank * own_max));  // rows of this CTA, from rank * own_max on

    // The set-up of the roles runs side by side: the first warp makes the barriers, lets the others pass and sends the first
    // loads off, the second allocates tensor memory, the others quantize as many blocks as there are stages.
    if (warp == 0) {
        if (elect_one()) {
            for (int s = 0; s < stages; ++s) { mbar_init(smem_u32(&ctl->full[s]), QUANT ? 1 + EPI_THREADS : 1); mbar_init(smem_u32(&ctl->empty[s]), 1); }
            mbar_init(smem_u32(&ctl->acc_full), 1);
            mbar_init(smem_u32(&ctl->joined), 1);
            ctl->abort_flag = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            if (split > 1) mbar_expect_tx(smem_u32(&ctl->joined), (uint32_t)(split * owned * BW) * 4u);
        }
        __syncwarp();
        asm volatile("bar.arrive 1, %0;" ::"r"(THREADS) : "memory");
        if (elect_one()) {
            for (int i = 0; i < min(kb_count, stages); ++i) load_stage(i);
        }
        __syncwarp();
    } else if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&ctl->tmem_base)), "r"((uint32_t)p.tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else if constexpr (QUANT) {
        const int tid = threadIdx.x - 64, blocks = min(kb_count, stages);
        const RowOf of(rows);
        for (int first = 0; first < blocks * rows; first += BATCH * BATCH_ROWS) {
            Chunk<OutT> x[BATCH];
            load_batch(p, of, m0, kb_first, blocks, first, tid, x);
            quantize_batch<OutT, FMT>(p, of, kb_first, blocks, first, tid, 0, x, tiles, st_bytes, sf);
        }
        fence_async_smem();
    }
    if (warp > 0) {
        tcgen05_fence_before();
        asm volatile("bar.sync 1, %0;" ::"r"(THREADS) : "memory");
        tcgen05_fence_after();
    }
    if (split > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");    // this CTA's barriers exist
    const uint32_t tmem = warp > 0 ? ctl->tmem_base : 0u;          // (the first warp has not waited for it, and does not need it)

    if (warp == 0) {
        bool ok = true;
        for (int i = stages; i < kb_count; ++i) {
            ok = mbar_wait_warp(smem_u32(&ctl->empty[i % stages]), ((i / stages) & 1) ^ 1u, abort_flag);
            if (!ok) break;
            if (elect_one()) load_stage(i);
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
            const int s = i % stages;
            ok = mbar_wait_warp(smem_u32(&ctl->full[s]), (i / stages) & 1, abort_flag);
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
        if constexpr (QUANT) {
            const int tid = threadIdx.x - 64;
            for (int i = 0; i < min(kb_count, stages); ++i) mbar_arrive(smem_u32(&ctl->full[i]));
            // the others a few blocks at a time: half of the ring, and no more than one batch
            const int group = max(1, min(stages / 2, BATCH * BATCH_ROWS / rows));
            const RowOf of(rows);
            bool ok = true;
            for (int i = stages; i < kb_count && ok; i += group) {
                const int blocks = min(group, kb_count - i);
                Chunk<OutT> x[BATCH];
                load_batch(p, of, m0, kb_first + i, blocks, 0, tid, x);
                for (int k = i; k < i + blocks && ok; ++k) ok = mbar_wait_warp(smem_u32(&ctl->empty[k % stages]), ((k / stages) & 1) ^ 1u, abort_flag);
                if (!ok) break;
                quantize_batch<OutT, FMT>(p, of, kb_first + i, blocks, 0, tid, i % stages, x, tiles, st_bytes, sf);
                fence_async_smem();
                for (int k = i; k < i + blocks; ++k) mbar_arrive(smem_u32(&ctl->full[k % stages]));
            }
        }
    }
    // all warps: the others' first pushes may come once every CTA of the cluster has made its barriers
    __syncwarp();
    if (split > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (warp >= 2) {
        const int col = (warp & 3) * 32 + lane, n = n0 + col;
        const uint32_t acc = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const float bias = (p.bias != nullptr && n < p.N) ? OutOps<OutT>::up(static_cast<const OutT*>(p.bias)[n]) : 0.0f;
        const int turn = 16 * ((warp - 2) >> 2);                    // this warp's rows: every second sixteen
        const int first_row = split == 1 ? m0 : m0 + rank * own_max, mine = split == 1 ? rows : owned;
        OutT res[2][16] = {};                                       // of this turn and the next
        load_residual<OutT, RES>(p, n, first_row + turn, mine - turn, res[0]);
        load_residual<OutT, RES>(p, n, first_row + turn + 32, mine - turn - 32, res[1]);
        if (mbar_wait_warp(smem_u32(&ctl->acc_full), 0, abort_flag)) {
            tcgen05_fence_after();
            if (split == 1) {
                for (int c = turn; c < rows; c += 64) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int at = c + 32 * h;
                        if (at >= rows) break;
                        uint32_t r[16];
                        tmem_ld16(acc + (uint32_t)at, r);
                        float y[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) y[j] = __uint_as_float(r[j]);
                        if (n < p.N) finish_rows<OutT, RES>(p, n, bias, m0 + at, rows - at, y, res[h]);
                        load_residual<OutT, RES>(p, n, m0 + at + 64, rows - at - 64, res[h]);
                    }
                }
            } else {
                const uint32_t bar = smem_u32(&ctl->joined);
                const uint32_t to = smem_u32(joined + rank * own_max * BW + col);
                for (int c = turn; c < rows; c += 32) {
                    uint32_t r[16];
                    tmem_ld16(acc + (uint32_t)c, r);
                    int owner = c / own_max, k = c % own_max;
                    uint32_t at = map_to_cta(to + (uint32_t)(k * BW) * 4u, (uint32_t)owner), at_bar = map_to_cta(bar, (uint32_t)owner);
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        if (c + j >= rows) break;
                        push_async(at, __uint_as_float(r[j]), at_bar);
                        at += BW * 4u;
                        if (++k == own_max && c + j + 1 < rows) {
                            k = 0; ++owner;
                            at = map_to_cta(to, (uint32_t)owner); at_bar = map_to_cta(bar, (uint32_t)owner);
                        }
                    }
                }
                if (turn < owned && mbar_wait_cluster(bar, 0, abort_flag) && n < p.N) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {                   // two turns at most: half of 128 rows
                        const int k = turn + 32 * h;
                        if (k >= owned) break;
                        const float* from = joined + k * BW + col;
                        float y[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) y[j] = 0.0f;
                        for (int q = 0; q < split; ++q, from += own_max * BW) {
#pragma unroll
                            for (int j = 0; j < 16; ++j) if (k + j < owned) y[j] += from[j * BW];
                        }
                        finish_rows<OutT, RES>(p, n, bias, first_row + k, owned - k, y, res[h]);
                    }
                }
                static_assert(MAX_T / 2 <= 64, "rows of one of two CTAs in two turns");
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
    if (threadIdx.x == 0 && ctl->abort_flag != 0 && p.status != nullptr) atomicExch(p.status, 1);
    // A CTA has its rows once every other has pushed them, and nobody reads or writes its memory after that; one that gave
    // up stays until the others have left or given up too.
    __syncwarp();
    if (split > 1 && *abort_flag != 0) cluster_sync();
}

// as much shared memory as the largest tile takes
constexpr size_t SMEM_MOST = 227 * 1024;

// How many clusters of `split` CTAs, two an SM, are on the device at once: fewer than its CTAs divided by `split`, since a
// cluster stays within one of the device's groups of SMs.  The runtime answers for one CTA an SM (15 clusters of eight, 22 of
// six, 33 of four), the same for every form of the kernel; a property of the device, asked for once.
int active_clusters(int split) {
    static thread_local int known[64][MAX_SPLIT + 1] = {};
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return 2 * (sm_count() / split); }
    if (known[dev][split] > 0) return known[dev][split];
    auto kernel = gemm_fp4_small_kernel<__half, SAMQ_FP4_NV, true, false>;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)split; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)split); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = HALF_SM + HALF_SM / 2;
    cfg.attrs = attr; cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_MOST) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        return 2 * (sm_count() / split);
    }
    return known[dev][split] = 2 * n;
}

// Split K while SMs are idle, but leave a CTA four blocks of 256 columns at least: of five blocks two CTAs gain nothing (us, whole /
// in two: 1 x 3840 x 1280 4.9 / 4.9, 8 x 3840 x 1280 5.3 / 5.6, 64 x 1280 x 2048 6.6 / 7.0), of twenty five gain much (1 x 1280 x
// 5120 10.6 / 5.8 in five).  The border is not the best everywhere: shares of two blocks take 1 x 1280 x 2560 from 6.0 in two
// to 4.9 in five.  All clusters are on the device at once: 1 x 5120 x 10240 takes 10.7 us in six and 13.4 in seven, 30 of whose 40
// clusters fit.
int split_of(const Fp4Call& c, int T) {
    const int64_t tiles = (c.N + BW - 1) / BW * ((c.M + MAX_T - 1) / MAX_T), k_blocks = (c.K + KPAD - 1) / KPAD;
    const int64_t room = (T <= 32 ? 2 : 1) * (int64_t)sm_count() / tiles;
    const int64_t most = k_blocks / 4 < room ? k_blocks / 4 : room;
    int split = (int)(most < 1 ? 1 : most > MAX_SPLIT ? MAX_SPLIT : most);
    while (split > 1 && tiles > active_clusters(split) / (T <= 32 ? 1 : 2)) --split;
    return split;
}

template <typename OutT, int FMT, bool QUANT, bool RES>
int launch_small(const Fp4Call& c, SmallParams& p, const CUtensorMap& ma, const CUtensorMap& mw) {
    auto kernel = gemm_fp4_small_kernel<OutT, FMT, QUANT, RES>;
    static thread_local bool ready[64] = {false};
    int dev = 0;
    SAMQ_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        SAMQ_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_MOST));
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    const int64_t n_tiles = (c.N + BW - 1) / BW, m_tiles = (c.M + MAX_T - 1) / MAX_T;
    const int split = split_of(c, p.T);
    p.stages = stages_of<FMT>(p.T, split);
    if (n_tiles * split > 2147483647LL || m_tiles > 65535) return fail(SAMQ_ERR_TOO_LARGE, "product of %lld x %lld outputs is too large", (long long)c.M, (long long)c.N);
    const int cols = p.T + 2 * Shape<FMT>::SF_COLS;
    p.tmem_cols = cols <= 64 ? 64 : cols <= 128 ? 128 : 256;
    const dim3 grid((unsigned)(n_tiles * split), (unsigned)m_tiles);
    const size_t smem = smem_bytes<FMT>(p.T, p.stages, split);
    static_assert(1024 + MIN_STAGES * (stage_bytes<FMT>(MAX_T) + 2 * Shape<FMT>::SF_BYTES) + (MAX_T + MAX_SPLIT) * BW * 4 + sizeof(Control) <= SMEM_MOST &&
                  HALF_SM + (MAX_T + MAX_SPLIT) * BW * 4 + sizeof(Control) <= SMEM_MOST, "the largest tiles and their joined rows");
    if (split == 1) {
        kernel<<<grid, THREADS, smem, c.stream>>>(ma, mw, p);
        SAMQ_CUDA_TRY(cudaGetLastError());
        return SAMQ_OK;
    }
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)split; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.gridDim = grid; cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = c.stream;
    cfg.attrs = attr; cfg.numAttrs = 1;
    SAMQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, ma, mw, p));
    return SAMQ_OK;
}

template <typename OutT>
int launch_form(int form, const Fp4Call& c, SmallParams& p, const CUtensorMap& ma, const CUtensorMap& mw) {
    switch (form) {
    case 0:  return launch_small<OutT, SAMQ_FP4_NV, false, false>(c, p, ma, mw);
    case 1:  return launch_small<OutT, SAMQ_FP4_NV, false, true>(c, p, ma, mw);
    case 2:  return launch_small<OutT, SAMQ_FP4_MX, false, false>(c, p, ma, mw);
    case 3:  return launch_small<OutT, SAMQ_FP4_MX, false, true>(c, p, ma, mw);
    case 4:  return launch_small<OutT, SAMQ_FP4_NV, true, false>(c, p, ma, mw);
    case 5:  return launch_small<OutT, SAMQ_FP4_NV, true, true>(c, p, ma, mw);
    case 6:  return launch_small<OutT, SAMQ_FP4_MX, true, false>(c, p, ma, mw);
    default: return launch_small<OutT, SAMQ_FP4_MX, true, true>(c, p, ma, mw);
    }
}

// x != nullptr: quantize it in the kernel, under x_global_scale
int gemm_fp4_small(const Fp4Call& c, const void* x, int64_t ldx, float x_global_scale) {
    SmallParams p;
    p.M = (int)c.M; p.N = (int)c.N; p.K = (int)c.K;
    p.T = tile_rows(c.M);
    p.groups = (int)groups_of(c.fmt, c.K); p.a_scales = c.a_scales; p.w_scales = c.w_scales;
    const size_t esz = c.out_dtype == SAMQ_F32 ? 4 : 2;
    p.x = x; p.ldx = ldx; p.access_x = row_access(x, ldx * (int64_t)esz);
    p.x_global_scale = x_global_scale; p.inv_x_global_scale = 1.0f / x_global_scale;
    p.alpha = c.epi.alpha; p.bias = c.epi.bias; p.residual = c.epi.residual; p.ldr = c.epi.ldr; p.out = c.epi.out; p.ldo = c.epi.ldo;
    p.gelu = c.gelu; p.status = c.status;
    CUtensorMap ma, mw;
    const int64_t row_bytes = (c.K + 1) / 2;
    int rc = make_operand_map(&mw, reinterpret_cast<const int8_t*>(c.W), c.N, row_bytes, c.ldw, BW);
    if (rc == SAMQ_OK && x == nullptr) rc = make_operand_map(&ma, reinterpret_cast<const int8_t*>(c.A), c.M, row_bytes, c.lda, p.T);
    if (rc != SAMQ_OK) return rc;
    if (x != nullptr) ma = mw;                                      // not used
    const int form = (x != nullptr ? 4 : 0) + (c.fmt == SAMQ_FP4_MX ? 2 : 0) + (p.residual != nullptr ? 1 : 0);
    switch (c.out_dtype) {
    case SAMQ_F16:  return launch_form<__half>(form, c, p, ma, mw);
    case SAMQ_BF16: return launch_form<__nv_bfloat16>(form, c, p, ma, mw);
    default:        return launch_form<float>(form, c, p, ma, mw);
    }
}

// What both entry points check: everything but the activation.
int check_call(Fp4Call& c, int64_t M, int64_t N, int64_t K, int fmt, const uint8_t* W, int64_t ldw, const uint8_t* w_scales, float alpha,
               const void* bias, const void* residual, int64_t ldr, int activation, void* out, int out_dtype, int64_t ldo,
               int32_t* status, void* stream)
{
    if (M < 0 || N <= 0 || K <= 0) return fail(SAMQ_ERR_BAD_ARG, "bad GEMM shape M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
    if (!known_format(fmt)) return fail(SAMQ_ERR_BAD_ARG, "unknown 4-bit format %d", fmt);
    if (activation != SAMQ_ACT_NONE && activation != SAMQ_ACT_GELU) return fail(SAMQ_ERR_BAD_ARG, "unknown activation %d", activation);
    if (out_dtype != SAMQ_F16 && out_dtype != SAMQ_BF16 && out_dtype != SAMQ_F32) return fail(SAMQ_ERR_BAD_ARG, "unknown out_dtype %d", out_dtype);
    if (!(fabsf(alpha) <= FLT_MAX)) return fail(SAMQ_ERR_BAD_ARG, "alpha, the product of the global scales, must be finite");
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

// the product of a checked call whose activation is set
int run_gemm(Fp4Call& c) {
    // The small kernel while all of its CTAs are on the device at once (two an SM), and for a single tile of rows, of
    // which the pair kernel would compute two.  us, small / pair: 2048 x 2304 x 768 (288 CTAs) 7.1 / 8.6, 512 x 5120 x
    // 1280 (160) 7.7 / 8.1, 1000 x 5120 x 1280 (320) 11.6 / 10.1, 200 x 20000 x 768 (314) 9.7 / 8.6, 2048 x 5120 x 5120
    // (640) 35.8 / 31.6, 100 x 20000 x 5120 (157) 14.4 / 22.4, 300 x 1280 x 5120 (30) 10.1 / 13.6.  The rule does not ask for K:
    // 2048 x 2304 x 2560 10.4 / 10.8, but at K = 5120 the small kernel's 128 x 128 tiles lose some (2048 x 2304 15.4 / 14.6, 1500 x
    // 2560 15.2 / 14.4, 1000 x 2560 14.6 / 13.9).
    if (c.M <= MAX_T || (c.M + MAX_T - 1) / MAX_T * ((c.N + BW - 1) / BW) <= 2 * sm_count()) return gemm_fp4_small(c, nullptr, 0, 1.0f);
    const int esz = c.out_dtype == SAMQ_F32 ? 4 : 2;
    int rc = SAMQ_OK;
    memset(&c.map_out, 0, sizeof(c.map_out));
    memset(&c.map_res, 0, sizeof(c.map_res));
    if (c.epi.tma_out) rc = make_row_map(&c.map_out, c.epi.out, c.M, c.N, c.epi.ldo, esz);
    if (rc == SAMQ_OK && c.epi.tma_res) rc = make_row_map(&c.map_res, c.epi.residual, c.M, c.N, c.epi.ldr, esz);
    return rc != SAMQ_OK ? rc : gemm_fp4_pair(c);
}

// Whether the layer quantizes its activation in the product's kernel.  Every CTA quantizes all rows of its share of K: where
// that is much, and there is a workspace, the quantizer runs first.  us, one kernel / two: 32 rows, 1280 -> 5120 (a share of 5
// blocks) 8.2 / 7.0, but the second launch costs the host 3 us; 32, 5120 -> 10240 (7) 17.3 / 13.7; 8, 10240 -> 10240 (14)
// 17.1 / 18.4, 16 20.7 / 18.2; 8, 5120 -> 20000 (20) 18.5 / 17.4; 1, 10240 -> 20000 (40) 32.3 / 26.8; 32, 5120 -> 20000 33.1 / 17.0.
bool one_kernel(const Fp4Call& c, int dtype, bool has_workspace) {
    if (c.M > FUSED_MAX_ROWS || dtype != c.out_dtype) return false;
    const int64_t k_blocks = (c.K + KPAD - 1) / KPAD;
    if (!has_workspace || (c.M + 8) * k_blocks <= FUSED_MOST) return true;
    const int split = split_of(c, tile_rows(c.M));
    return (c.M + 8) * ((k_blocks + split - 1) / split) <= FUSED_MOST;
}

}  // namespace

size_t linear_fp4_workspace(int fmt, int64_t M, int64_t K);

int linear_fp4_kernels(int fmt, int dtype, int out_dtype, int64_t M, int64_t N, int64_t K, size_t workspace_bytes) {
    Fp4Call c;
    c.M = M; c.N = N; c.K = K; c.fmt = fmt; c.out_dtype = out_dtype;
    return one_kernel(c, dtype, workspace_bytes >= linear_fp4_workspace(fmt, M, K)) ? 1 : 2;
}

int quant_fp4_dispatch(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, int fmt, float global_scale,
                       uint8_t* codes, int64_t ldq, uint8_t* scales, void* fq, void* stream);

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
    return run_gemm(c);
}

// codes of whole 16-byte rows, then the scales
size_t linear_fp4_workspace(int fmt, int64_t M, int64_t K) {
    return (size_t)M * ((K + 31) / 32 * 16) + (size_t)((M + TILE_ROWS - 1) / TILE_ROWS * groups_of(fmt, K)) * TILE_BYTES;
}

int linear_fp4_dispatch(const void* x, int dtype, int64_t ldx, float x_global_scale, const uint8_t* W, int64_t ldw, const uint8_t* w_scales,
                        int64_t M, int64_t N, int64_t K, int fmt, float alpha, const void* bias, const void* residual, int64_t ldr,
                        int activation, void* out, int out_dtype, int64_t ldo, void* workspace, size_t workspace_bytes,
                        int32_t* status, void* stream)
{
    Fp4Call c;
    int rc = check_global_scale(fmt, x_global_scale);
    if (rc != SAMQ_OK) return rc;
    rc = check_call(c, M, N, K, fmt, W, ldw, w_scales, alpha * x_global_scale, bias, residual, ldr, activation, out, out_dtype, ldo, status, stream);
    if (rc != SAMQ_OK) return rc;
    if (dtype != SAMQ_F16 && dtype != SAMQ_BF16 && dtype != SAMQ_F32) return fail(SAMQ_ERR_BAD_ARG, "unknown dtype %d", dtype);
    if (M == 0) return SAMQ_OK;
    if (x == nullptr) return fail(SAMQ_ERR_BAD_ARG, "x must not be null");
    if (ldx < K) return fail(SAMQ_ERR_BAD_ARG, "ldx smaller than K");
    if (reinterpret_cast<uintptr_t>(x) & (dtype == SAMQ_F32 ? 3 : 1)) return fail(SAMQ_ERR_ALIGNMENT, "x must be aligned to its elements");
    const int64_t pitch = (K + 31) / 32 * 16;
    const size_t need = linear_fp4_workspace(fmt, M, K);
    if (one_kernel(c, dtype, workspace != nullptr && workspace_bytes >= need)) return gemm_fp4_small(c, x, ldx, x_global_scale);
    if (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))
        return fail(SAMQ_ERR_WORKSPACE, "the 4-bit linear needs %zu bytes of 16-byte aligned workspace", need);
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    uint8_t* scales = codes + (size_t)M * pitch;
    rc = quant_fp4_dispatch(x, dtype, M, K, ldx, fmt, x_global_scale, codes, pitch, scales, nullptr, stream);
    if (rc != SAMQ_OK) return rc;
    c.A = codes; c.lda = pitch; c.a_scales = scales;
    return run_gemm(c);
}

}  // namespace samq
