// Products of 8-bit integers with a scale for each token and one for each output channel, on the tensor cores of sm_100a:
//   C[t, n] = epilogue(a_scale[t] w_scale[n] sum_k A[t, k] W[n, k])
// The sums are 32-bit integers in tensor memory (`tcgen05.mma.kind::i8`, 32 entries of K an instruction) and exact (K up to 131,071: 128 * 128 * K stays
// below 2^31), so a row's result does not depend on how K is cut, nor on the other rows.  The scaling is (sum * a_scale) * w_scale in float32.
// Epilogues: store (float32 or bfloat16), add into float32 C, gated (W holds N gate rows, then N up rows; see GluRule).
//
// Operand tiles of 128 entries of K (128 bytes a row, 128-byte swizzle) come into shared memory by TMA through a ring of stages guarded by mbarriers; one
// thread issues the copies, one the MMAs, the other warps drain the accumulators.  Two kernels:
//   few tokens    the 128-row side holds weight rows, the other 16 to 128 tokens; K is cut over a cluster of up to 8 CTAs, whose partial sums meet
//                 through distributed shared memory (gemm_q8_few_kernel).  Bound by the weights' way from memory.
//   many tokens   persistent pairs of CTAs (cta_group::2) on tiles of 256 tokens (gemm_q8_pair_kernel).  Bound by the tensor cores.
// Rows, tokens and K beyond the matrices are zeros by TMA and masked in the epilogue.  Every wait on an mbarrier is bounded (see tc_common.cuh).
#include "tc_common.cuh"

#include <type_traits>

namespace {

enum { EPI_STORE = 0, EPI_ACCUMULATE = 1, EPI_GATED = 2 };
constexpr int MAX_K = 131071, BLOCK_K = 128, UMMA_K = 32, TILE_M = 128, MAX_STAGES = 12;
constexpr int A_TILE_BYTES = TILE_M * BLOCK_K;
// instruction descriptor: D 32-bit integers, A and B signed 8-bit integers, both K-major
__host__ __device__ constexpr uint32_t idesc_q8(int m, int n) { return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

struct GemmQ8Params {
    void* C;
    const float *a_scale, *w_scale;
    long ldc;
    int T, N, K;
    int bn, stages, splits, k_blocks_per_split;
    int early;               // the weights were complete before the kernel in front was launched
    int tma_out;             // many tokens: C leaves by TMA
    int* status;
    GluRule glu;
    uint32_t wait_limit;     // FAULT: tries of a wait before it gives up,
    int withhold_block;      // and a k block whose copies are announced and never made
};
// FAULT: kernels for hymt2_gemm_q8_debug, whose waits have a limit of the launch's (read from the arguments it costs every wait of every launch: 2,048 x 2,048
// for a token 4.2 us against 4.0) and which copy every block but one.
template <bool FAULT> __device__ __forceinline__ uint32_t wait_limit(const GemmQ8Params& p) { return FAULT ? p.wait_limit : WAIT_LIMIT; }
template <bool FAULT> __device__ __forceinline__ uint32_t landing_limit(const GemmQ8Params& p) { return FAULT ? p.wait_limit : 1u << 16; }

__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// x sigmoid(alpha x).  The drain of a gated tile is bound by its instructions (2,048 x 6,144 gated x 2,048 into bfloat16 takes 54 us with an exact division and
// exponential, 39 with approximate ones), so the reciprocal is the hardware's approximate one (a step of float32).  The exponential is too where the result becomes
// bfloat16: it is off by 2^-22 and by 2^-24 of its argument's size, where that rounding is 2^-9.  What stays float32 has expf, so that far negative gates are as
// good as near ones (8 half steps in all; the form with a division, common.cuh's silu_mul, 6): that product takes 43.2 us for 42.5, with the division 51.
template <typename TC> __device__ __forceinline__ float swish(float x, float alpha) {
    float r;
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.0f + (sizeof(TC) == 4 ? expf(-alpha * x) : __expf(-alpha * x))));
    return x * r;
}
// glu_at of common.cuh, but a NaN stays one under the clamps: it says that the row held one before it became integers
template <typename TC> __device__ __forceinline__ float gated_at(const GluRule& r, float g, float u, int n, int N) {
    if (r.bias) { g = __fadd_rn(g, r.bias[n]); u = __fadd_rn(u, r.bias[N + n]); }
    if (r.kind == GLU_SILU) return swish<TC>(g, 1.0f) * u;
    g = min_nan(g, r.limit);
    u = min_nan(max_nan(u, -r.limit), r.limit);
    return swish<TC>(g, r.alpha) * (u + 1.0f);
}
// (products of their own and no FMA with what follows: both kernels give the same bits)
__device__ __forceinline__ float scaled(int sum, float a, float w) { return __fmul_rn(__fmul_rn((float)sum, a), w); }

__device__ __forceinline__ void umma_q8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_q8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_pair_commit(uint32_t bar) {      // the barrier at this place in both CTAs
    asm volatile(
        "{\n\t.reg .b16 both;\n\tmov.b16 both, 3;\n\t"
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], both;\n\t}" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t even_bar, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(dst), "l"((uint64_t)map), "r"(even_bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void mbar_arrive_even(uint32_t even_bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(even_bar) : "memory");
}
// A look at a barrier that does not wait.  The roles look at the next stage's barrier in front of this stage's work, so that the answer's way (a
// few hundred cycles under load) passes behind that work, and wait only where the look saw nothing.
__device__ __forceinline__ bool mbar_look(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// A warp reads N columns from each of two places of its 32 lanes of tensor memory, one row a thread.
template <int N> __device__ __forceinline__ void tmem_load_two(uint32_t at_a, uint32_t at_b, float* a, float* b);
template <> __device__ __forceinline__ void tmem_load_two<16>(uint32_t at_a, uint32_t at_b, float* a, float* b) {
    uint32_t *r = reinterpret_cast<uint32_t*>(a), *q = reinterpret_cast<uint32_t*>(b);
    asm volatile(            // (both addresses are read before a result may take their registers)
        "{\n\t.reg .b32 from_a, from_b;\n\tmov.b32 from_a, %32;\n\tmov.b32 from_b, %33;\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [from_a];\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [from_b];\n\t"
        "tcgen05.wait::ld.sync.aligned;\n\t}"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]), "=r"(q[4]), "=r"(q[5]), "=r"(q[6]), "=r"(q[7]),
          "=r"(q[8]), "=r"(q[9]), "=r"(q[10]), "=r"(q[11]), "=r"(q[12]), "=r"(q[13]), "=r"(q[14]), "=r"(q[15])
        : "r"(at_a), "r"(at_b) : "memory");
}
template <> __device__ __forceinline__ void tmem_load_two<32>(uint32_t at_a, uint32_t at_b, float* a, float* b) {
    uint32_t *r = reinterpret_cast<uint32_t*>(a), *q = reinterpret_cast<uint32_t*>(b);
    asm volatile(            // (both addresses are read before a result may take their registers)
        "{\n\t.reg .b32 from_a, from_b;\n\tmov.b32 from_a, %64;\n\tmov.b32 from_b, %65;\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [from_a];\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
        "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [from_b];\n\t"
        "tcgen05.wait::ld.sync.aligned;\n\t}"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
          "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]), "=r"(q[4]), "=r"(q[5]), "=r"(q[6]), "=r"(q[7]),
          "=r"(q[8]), "=r"(q[9]), "=r"(q[10]), "=r"(q[11]), "=r"(q[12]), "=r"(q[13]), "=r"(q[14]), "=r"(q[15]),
          "=r"(q[16]), "=r"(q[17]), "=r"(q[18]), "=r"(q[19]), "=r"(q[20]), "=r"(q[21]), "=r"(q[22]), "=r"(q[23]),
          "=r"(q[24]), "=r"(q[25]), "=r"(q[26]), "=r"(q[27]), "=r"(q[28]), "=r"(q[29]), "=r"(q[30]), "=r"(q[31])
        : "r"(at_a), "r"(at_b) : "memory");
}
__device__ __forceinline__ int4 ld_cluster_s32x4(uint32_t local_addr, uint32_t rank) {
    const float4 v = ld_cluster_f32x4(local_addr, rank);
    return make_int4(__float_as_int(v.x), __float_as_int(v.y), __float_as_int(v.z), __float_as_int(v.w));
}

// --------------------------------------------------------------------------------------------
// Few tokens: a CTA computes 128 weight rows (gated: 128 gate and 128 up rows) x BN tokens over its cut of K.
// --------------------------------------------------------------------------------------------
__host__ __device__ constexpr int few_warps(int bn) { return bn >= 64 ? 8 : 4; }      // that drain the sums (behind warp 0, TMA, and warp 1, MMAs)
constexpr int MAX_RANKS = 8;           // a portable cluster

template <int BN, int EPI, typename TC, bool FAULT = false>
__global__ void __launch_bounds__(64 + 32 * few_warps(BN))
gemm_q8_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, GemmQ8Params p) {
    constexpr int NUM_ACC = EPI == EPI_GATED ? 2 : 1;
    constexpr int STAGE_BYTES = NUM_ACC * A_TILE_BYTES + BN * BLOCK_K;
    constexpr int ACC_COLS = NUM_ACC * BN;
    constexpr int TMEM_COLS = ACC_COLS <= 32 ? 32 : ACC_COLS;        // 32, 64, 128 or 256
    constexpr uint32_t IDESC = idesc_q8(TILE_M, BN);
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * MAX_STAGES + 1];
    __shared__ uint32_t tmem_base_s;
    __shared__ int abort_s;
    const uint32_t tiles = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, stages = p.stages;
    const uint32_t full0 = smem_u32(&bars[0]), empty0 = smem_u32(&bars[MAX_STAGES]), done_bar = smem_u32(&bars[2 * MAX_STAGES]);
    volatile int* abort_flag = &abort_s;
    const int num_k_blocks = (p.K + BLOCK_K - 1) / BLOCK_K;
    const int kb_begin = blockIdx.z * p.k_blocks_per_split;
    const int my_blocks = max(0, min(num_k_blocks, kb_begin + p.k_blocks_per_split) - kb_begin);
    const int n0 = blockIdx.x * TILE_M, t0 = blockIdx.y * BN;

    if (threadIdx.x == 32) {            // the maps are on their way while the barriers are made
        for (const CUtensorMap* map : {&map_w, &map_a}) asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)map) : "memory");
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; s++) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        mbar_init(done_bar, 1);
        abort_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    // Tensor memory is taken once the kernel in front is through (a CTA of that one may have yet to take its own), and the next kernel released behind that.
    uint32_t tmem_base = 0;
    if (warp >= 1) {
        pdl_wait();
        if (warp == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
            pdl_launch_dependents();
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        asm volatile("bar.sync 2, %0;" ::"n"(32 + 32 * few_warps(BN)) : "memory");
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        tmem_base = tmem_base_s;
    }

    int issued = 0;                     // k blocks that were announced (in the thread that copies)
    if (warp == 0 && elect_one()) {
        auto load_weights = [&](int i) {
            const uint32_t bar = full0 + 8 * (i % stages), dst = tiles + (i % stages) * STAGE_BYTES;
            const int k = (kb_begin + i) * BLOCK_K;
            if (FAULT && kb_begin + i == p.withhold_block) return;
            tma_load_2d(dst, &map_w, bar, k, n0);
            if (NUM_ACC == 2) tma_load_2d(dst + A_TILE_BYTES, &map_w, bar, k, p.N + n0);
        };
        auto load_tokens = [&](int i) {
            if (FAULT && kb_begin + i == p.withhold_block) return;
            tma_load_2d(tiles + (i % stages) * STAGE_BYTES + NUM_ACC * A_TILE_BYTES, &map_a, full0 + 8 * (i % stages), (kb_begin + i) * BLOCK_K, t0);
        };
        // the first ring of weights before the wait for the kernel in front, where they do not come from it
        const int ahead = min(stages, my_blocks);
        if (!p.early) pdl_wait();
        for (int i = 0; i < ahead; i++) {
            mbar_expect_tx(full0 + 8 * i, STAGE_BYTES);
            load_weights(i);
        }
        if (p.early) pdl_wait();
        for (int i = 0; i < ahead; i++) load_tokens(i);
        issued = ahead;
        for (int i = ahead; i < my_blocks; i++) {
            const int s = i % stages;
            if (!mbar_wait(empty0 + 8 * s, ((i / stages) & 1) ^ 1, abort_flag, p.status, 151, wait_limit<FAULT>(p))) break;
            mbar_expect_tx(full0 + 8 * s, STAGE_BYTES);
            load_weights(i);
            load_tokens(i);
            issued = i + 1;
        }
    } else if (warp == 1 && elect_one()) {
        constexpr uint64_t K_STEP = UMMA_K >> 4, A2_STEP = A_TILE_BYTES >> 4, B_STEP = (NUM_ACC * A_TILE_BYTES) >> 4;
        const uint64_t desc0 = desc_k_major(tiles);
        uint32_t s = 0, phase = 0;
        bool seen = false;
        for (int i = 0; i < my_blocks; i++) {
            if (!seen && !mbar_wait(full0 + 8 * s, phase, abort_flag, p.status, 152, wait_limit<FAULT>(p))) {
                __threadfence_block();          // whoever meets the barrier below also meets the abort flag
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint64_t adesc = desc0 + (uint64_t)s * (uint64_t)(STAGE_BYTES >> 4), bdesc = adesc + B_STEP;
            const uint32_t s_next = s + 1 == (uint32_t)stages ? 0 : s + 1, phase_next = s_next ? phase : phase ^ 1;
            seen = mbar_look(full0 + 8 * s_next, phase_next);       // (behind the last block nothing comes of it)
#pragma unroll
            for (int k = 0; k < BLOCK_K / UMMA_K; k++) {
                umma_q8(tmem_base, adesc + k * K_STEP, bdesc + k * K_STEP, IDESC, i > 0 || k > 0);
                if (NUM_ACC == 2) umma_q8(tmem_base + BN, adesc + A2_STEP + k * K_STEP, bdesc + k * K_STEP, IDESC, i > 0 || k > 0);
            }
            umma_commit(empty0 + 8 * s);
            s = s_next;
            phase = phase_next;
        }
        umma_commit(done_bar);
    } else if (warp >= 2) {
        const int quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
        TC* C = (TC*)p.C;
        const int cols = min(BN, p.T - t0);
        // a lane of the fold has four neighbouring weight rows
        const int n4 = n0 + 4 * lane;
        float sw[NUM_ACC][4];
#pragma unroll
        for (int h = 0; h < NUM_ACC; h++)
#pragma unroll
            for (int i = 0; i < 4; i++) sw[h][i] = n4 + i < p.N ? p.w_scale[(size_t)h * p.N + n4 + i] : 0.f;
        const bool vec = n4 + 4 <= p.N && (p.ldc & 3) == 0 && ((uintptr_t)C & (4 * sizeof(TC) - 1)) == 0;

        // (done_bar completes for an issuer that gave up too, once the MMAs that it did issue are through.  One answer for the warp: a load of tensor memory
        // takes all of it)
        const bool done = my_blocks > 0 ? mbar_wait(done_bar, 0, abort_flag, p.status, 153, wait_limit<FAULT>(p)) : true;
        const bool ok = __all_sync(0xffffffffu, done && !*abort_flag);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        // the sums -> this CTA's shared memory (the ring is free now), [column][row]
        constexpr int CH = BN >= 32 ? 32 : 16, GROUPS = few_warps(BN) / 4;
        const int group = (warp - 2) >> 2;
#pragma unroll 1
        for (int h = 0; h < NUM_ACC; h++)
#pragma unroll 1
            for (int c = group * CH; c < cols; c += GROUPS * CH) {
                float g[CH];
                if (ok && my_blocks > 0) {
                    if constexpr (CH == 32) tmem_load32(lane_addr + h * BN + c, g);
                    else tmem_load16(lane_addr + h * BN + c, g);
                } else {
#pragma unroll
                    for (int j = 0; j < CH; j++) g[j] = 0.f;
                }
#pragma unroll
                for (int j = 0; j < CH; j++)
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(tiles + ((h * BN + c + j) * TILE_M + row) * 4), "f"(g[j]) : "memory");
            }
        __syncwarp();
        if (p.splits > 1) cluster_sync_all();
        else asm volatile("bar.sync 1, %0;" ::"n"(32 * few_warps(BN)) : "memory");
        // Where one of the cluster's CTAs gave up, the tile becomes NaN: every wait lies in front of this barrier, so the ranks' abort flags say it.  They are asked
        // for in front of the sums and looked at behind them, by a factor and not a branch (64 tokens, 2,048 x 2,048: 4.8 us, with a branch 4.9, without either 4.7).
        int gave_up = 0;
        if (p.splits == 1) gave_up = *abort_flag;
        else if (lane < p.splits)
            asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(gave_up) : "r"(at_rank(smem_u32(&abort_s), lane)) : "memory");
        // every CTA of the cluster takes a share of the tokens, adds all ranks' sums for them and writes them out; a warp has a token, a lane four
        // weight rows.  The way to another CTA's memory is long (one token at a time took 170 ns a token), so the sums of U tokens and R ranks are
        // asked for together: many tokens a warp where there are few ranks, and the other way round.
        constexpr int WARPS = few_warps(BN);
        const int share = (cols + p.splits - 1) / p.splits;
        const int c_begin = (int)blockIdx.z * share, c_end = min(cols, c_begin + share);
        auto fold = [&](auto tokens, auto ranks) {
            constexpr int U = decltype(tokens)::value, R = decltype(ranks)::value;
#pragma unroll 1
            for (int c0 = c_begin + warp - 2; c0 < c_end; c0 += WARPS * U) {
                int4 part[U][R][NUM_ACC];
                float sa[U];
                [[maybe_unused]] float old[EPI == EPI_ACCUMULATE ? U : 1][4];       // what is added to: asked for with the sums, not behind them
#pragma unroll
                for (int k = 0; k < U; k++) {
                    const int c = c0 + k * WARPS;
                    sa[k] = c < c_end ? p.a_scale[t0 + c] : 0.f;
                    if constexpr (EPI == EPI_ACCUMULATE) {
                        const float* at = (const float*)C + (size_t)(t0 + c) * p.ldc + n4;
                        if (vec && c < c_end) {
                            const float4 v = *reinterpret_cast<const float4*>(at);
                            old[k][0] = v.x; old[k][1] = v.y; old[k][2] = v.z; old[k][3] = v.w;
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; i++) old[k][i] = c < c_end && n4 + i < p.N ? at[i] : 0.f;
                        }
                    }
#pragma unroll
                    for (int r = 0; r < R; r++)
#pragma unroll
                        for (int h = 0; h < NUM_ACC; h++) {
                            const uint32_t at = tiles + ((h * BN + c) * TILE_M + 4 * lane) * 4;
                            part[k][r][h] = make_int4(0, 0, 0, 0);
                            if (c < c_end && r < p.splits) {
                                if constexpr (R == 1)
                                    asm volatile("ld.shared.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(part[k][r][h].x), "=r"(part[k][r][h].y),
                                                 "=r"(part[k][r][h].z), "=r"(part[k][r][h].w) : "r"(at) : "memory");
                                else part[k][r][h] = ld_cluster_s32x4(at, r);
                            }
                        }
                }
                const bool none = __any_sync(0xffffffffu, gave_up);
#pragma unroll
                for (int k = 0; k < U; k++) {
                    const int c = c0 + k * WARPS;
                    if (c >= c_end) break;
                    float y[NUM_ACC][4];
                    if (none) sa[k] = __uint_as_float(0x7fc00000u);
#pragma unroll
                    for (int h = 0; h < NUM_ACC; h++) {
                        int4 sum = part[k][0][h];
#pragma unroll
                        for (int r = 1; r < R; r++) { sum.x += part[k][r][h].x; sum.y += part[k][r][h].y; sum.z += part[k][r][h].z; sum.w += part[k][r][h].w; }
                        y[h][0] = scaled(sum.x, sa[k], sw[h][0]); y[h][1] = scaled(sum.y, sa[k], sw[h][1]);
                        y[h][2] = scaled(sum.z, sa[k], sw[h][2]); y[h][3] = scaled(sum.w, sa[k], sw[h][3]);
                    }
                    TC* dst = C + (size_t)(t0 + c) * p.ldc + n4;
                    if constexpr (EPI == EPI_GATED) {
#pragma unroll
                        for (int i = 0; i < 4; i++) if (n4 + i < p.N) y[0][i] = gated_at<TC>(p.glu, y[0][i], y[1][i], n4 + i, p.N);
                    }
                    if constexpr (EPI == EPI_ACCUMULATE) {
#pragma unroll
                        for (int i = 0; i < 4; i++) y[0][i] = __fadd_rn(old[k][i], y[0][i]);
                    }
                    if (vec) {
                        if constexpr (sizeof(TC) == 4) *reinterpret_cast<float4*>(dst) = make_float4(y[0][0], y[0][1], y[0][2], y[0][3]);
                        else {
                            __nv_bfloat162 h[2] = {__floats2bfloat162_rn(y[0][0], y[0][1]), __floats2bfloat162_rn(y[0][2], y[0][3])};
                            *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(h);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (n4 + i < p.N) dst[i] = from_float<TC>(y[0][i]);
                    }
                }
            }
        };
        if (p.splits == 1) fold(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
        else if (p.splits == 2) fold(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{});
        else if (p.splits <= 4) fold(std::integral_constant<int, 2>{}, std::integral_constant<int, 4>{});
        else fold(std::integral_constant<int, 1>{}, std::integral_constant<int, MAX_RANKS>{});
        __syncwarp();
    }
    // Where a role gave up, copies may be in flight: they must land before the CTA's shared memory goes away.  (Looked at once every wait of the CTA is behind
    // it, while the sums are folded; a wait for the copies in every launch took 2,048 x 2,048 for a token from 4.0 to 4.4 us.)
    auto landed = [&] {
        if (warp == 0 && *abort_flag)
            for (int i = max(0, issued - stages); i < issued; i++)
                for (uint32_t t = 0; t < landing_limit<FAULT>(p) && !mbar_try_wait(full0 + 8 * (i % stages), (i / stages) & 1); t++) {}
        __syncwarp();
    };
    if (p.splits > 1) {         // no CTA leaves before its peers have read its sums; the other warps come to both barriers too
        __syncwarp();
        if (warp < 2) {
            cluster_sync_all();
            landed();
        }
        cluster_sync_all();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (p.splits == 1) landed();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
    }
}

// --------------------------------------------------------------------------------------------
// Many tokens: persistent pairs of CTAs walk tiles of 256 tokens x bn weight rows (gated: bn / 2 gate and bn / 2 up rows), token tiles fastest.  A CTA holds
// its 128 tokens and half of the weight rows; the even CTA issues the MMAs of both.  Two accumulators in tensor memory alternate.
// --------------------------------------------------------------------------------------------
constexpr int PAIR_THREADS = 320;      // warp 0 TMA, warp 1 MMAs, warps 2 to 9 the sums: each has 32 tokens and every other piece of columns
constexpr int PAIR_BN = 256;           // the widest tile: the accumulators lie so many columns apart
constexpr int PIECE_BYTES = 64;        // a token's piece of output columns: 32 of bfloat16, 16 of float32
constexpr int OUT_BUFFER = 32 * PIECE_BYTES, OUT_BYTES = 8 * 2 * OUT_BUFFER;   // a warp has two buffers that TMA writes out

template <int EPI, typename TC, bool FAULT = false>
__global__ void __launch_bounds__(PAIR_THREADS, 1)
gemm_q8_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_c,
                    GemmQ8Params p) {
    constexpr bool GATED = EPI == EPI_GATED;
    constexpr int PIECE = PIECE_BYTES / (int)sizeof(TC);
    const int bn = p.bn, B_TILE_BYTES = bn / 2 * BLOCK_K, STAGE_BYTES = A_TILE_BYTES + B_TILE_BYTES;
    const int OUT_COLS = GATED ? bn / 2 : bn;
    const uint32_t IDESC = idesc_q8(2 * TILE_M, bn);
    const int pair = blockIdx.x / 2, pairs = gridDim.x / 2, rank = blockIdx.x % 2;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * MAX_STAGES + 4];
    __shared__ uint32_t tmem_base_s;
    __shared__ int abort_s;
    const uint32_t tiles = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, stages = p.stages;
    const uint32_t full0 = smem_u32(&bars[0]), empty0 = smem_u32(&bars[MAX_STAGES]);
    const uint32_t acc_full0 = smem_u32(&bars[2 * MAX_STAGES]), acc_empty0 = acc_full0 + 16;
    volatile int* abort_flag = &abort_s;
    const int num_k_blocks = (p.K + BLOCK_K - 1) / BLOCK_K;
    const int tiles_t = (p.T + 2 * TILE_M - 1) / (2 * TILE_M), tiles_n = (p.N + OUT_COLS - 1) / OUT_COLS, num_tiles = tiles_t * tiles_n;

    if (threadIdx.x == 32) {            // the maps are on their way while the barriers are made
        for (const CUtensorMap* map : {&map_w, &map_a}) asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)map) : "memory");
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; s++) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(acc_full0 + 8 * b, 1);
            mbar_init(acc_empty0 + 8 * b, 16);      // the warps of both CTAs
        }
        abort_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(2 * PAIR_BN) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync_all();                 // both CTAs' barriers and tensor memory are there
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = tmem_base_s;
    // (behind the allocation: a CTA of the next kernel cannot have taken this one's tensor memory; and beside this kernel's shared memory no CTA of the one in
    // front fits that has yet to take its own)
    pdl_launch_dependents();

    if (warp == 0 && elect_one()) {
        uint32_t s = 0, round = 0;
        const uint32_t even_full0 = at_rank(full0, 0);
        bool first = true, seen = false;
        if (!p.early) pdl_wait();
        for (int tile = pair; tile < num_tiles && !*abort_flag; tile += pairs) {
            const int a_row = (tile % tiles_t) * 2 * TILE_M + rank * TILE_M;
            // the even CTA brings the first half of the weight rows, the odd one the second; of gated rows the gates and the ups
            const int w_row = (tile / tiles_t) * OUT_COLS + rank * (GATED ? p.N : bn / 2);
            for (int kb = 0; kb < num_k_blocks; kb++) {
                if (round > 0 && !seen && !mbar_wait(empty0 + 8 * s, (round & 1) ^ 1, abort_flag, p.status, 151, wait_limit<FAULT>(p))) break;
                const uint32_t bar = even_full0 + 8 * s, a_dst = tiles + s * STAGE_BYTES;
                const uint32_t s_next = s + 1 == (uint32_t)stages ? 0 : s + 1, round_next = s_next ? round : round + 1;
                seen = round_next > 0 && mbar_look(empty0 + 8 * s_next, (round_next & 1) ^ 1);
                if (rank == 0) mbar_expect_tx(full0 + 8 * s, 2 * STAGE_BYTES);
                if (!FAULT || kb != p.withhold_block) tma_load_2d_pair(a_dst + A_TILE_BYTES, &map_w, bar, kb * BLOCK_K, w_row);
                if (first && p.early) pdl_wait();
                first = false;
                if (!FAULT || kb != p.withhold_block) tma_load_2d_pair(a_dst, &map_a, bar, kb * BLOCK_K, a_row);
                s = s_next;
                round = round_next;
            }
        }
        // copies (both CTAs' are counted here) must land before the shared memory goes away, whatever became of the roles that wait for them
        if (rank == 0)
            for (int back = 0; back < stages && (round > 0 || s > 0); back++) {
                if (s == 0) { s = stages; round--; }
                s--;
                for (uint32_t t = 0; t < landing_limit<FAULT>(p) && !mbar_try_wait(full0 + 8 * s, round & 1); t++) {}
            }
    } else if (warp == 1 && rank == 0 && elect_one()) {
        const uint64_t desc0 = desc_k_major(tiles);
        uint32_t s = 0, phase = 0;
        bool seen = false;
        int j = 0;
        for (int tile = pair; tile < num_tiles; tile += pairs, j++) {
            const int buf = j & 1;
            if (j >= 2 && !mbar_wait(acc_empty0 + 8 * buf, (uint32_t)(((j >> 1) - 1) & 1), abort_flag, p.status, 154, wait_limit<FAULT>(p))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            bool ok = true;
            for (int kb = 0; kb < num_k_blocks; kb++) {
                if (!seen && !(ok = mbar_wait(full0 + 8 * s, phase, abort_flag, p.status, 152, wait_limit<FAULT>(p)))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t adesc = desc0 + (uint64_t)s * (uint64_t)(STAGE_BYTES >> 4), bdesc = adesc + (A_TILE_BYTES >> 4);
                const uint32_t s_next = s + 1 == (uint32_t)stages ? 0 : s + 1, phase_next = s_next ? phase : phase ^ 1;
                seen = mbar_look(full0 + 8 * s_next, phase_next);
#pragma unroll
                for (int k = 0; k < BLOCK_K / UMMA_K; k++)
                    umma_q8_pair(tmem_base + buf * PAIR_BN, adesc + k * (UMMA_K >> 4), bdesc + k * (UMMA_K >> 4), IDESC, kb > 0 || k > 0);
                umma_pair_commit(empty0 + 8 * s);
                s = s_next;
                phase = phase_next;
            }
            if (!ok) break;
            umma_pair_commit(acc_full0 + 8 * buf);
        }
    } else if (warp >= 2) {
        const int quarter = warp & 3, side = (warp - 2) >> 2;
        const uint32_t stage_out = tiles + stages * STAGE_BYTES + (warp - 2) * 2 * OUT_BUFFER;
        pdl_wait();             // C may still be in use by the kernel in front, and the scales come from it
        TC* C = (TC*)p.C;
        const bool plain = p.glu.kind == GLU_SILU && !p.glu.bias;
        int j = 0, used = 0;
        // the token's scale, and the scale of one column of a piece a lane (gated: of its gate and its up row): fetched a tile and a piece ahead.  (Plain
        // loads: the kernel in front may have been writing them when this one was started, so they are not read-only data, and stay behind the wait.)
        auto first_token = [&](int tile) { return (tile % tiles_t) * 2 * TILE_M + rank * TILE_M + quarter * 32; };
        auto token_scale = [&](int tile) {
            const int t = first_token(tile) + lane;
            return tile < num_tiles && t < p.T ? p.a_scale[t] : 0.f;
        };
        auto column_scale = [&](int tile, int c, int h) {
            const int n = (tile / tiles_t) * OUT_COLS + c + lane;
            return tile < num_tiles && c < OUT_COLS && lane < PIECE && n < p.N ? p.w_scale[(size_t)h * p.N + n] : 0.f;
        };
        float sa_next = token_scale(pair), ws_next = column_scale(pair, side * PIECE, 0), us_next = GATED ? column_scale(pair, side * PIECE, 1) : 0.f;
        for (int tile = pair; tile < num_tiles; tile += pairs, j++) {
            const int buf = j & 1;
            const int t_first = first_token(tile);
            const int n_first = (tile / tiles_t) * OUT_COLS;
            const float sa = sa_next;
            float ws = ws_next, us = us_next;
            sa_next = token_scale(tile + pairs);
            ws_next = column_scale(tile + pairs, side * PIECE, 0);
            if constexpr (GATED) us_next = column_scale(tile + pairs, side * PIECE, 1);
            const bool landed = mbar_wait(acc_full0 + 8 * buf, (uint32_t)((j >> 1) & 1), abort_flag, p.status, 153, wait_limit<FAULT>(p));
            if (!__all_sync(0xffffffffu, landed)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16) + buf * PAIR_BN;
#pragma unroll 1
            for (int c = side * PIECE; c < OUT_COLS; c += 2 * PIECE) {
                const int n = n_first + c;
                if (n >= p.N || t_first >= p.T) break;               // (the same for the whole warp)
                float y[PIECE], u[GATED ? PIECE : 1];
                if constexpr (GATED) tmem_load_two<PIECE>(lane_addr + c, lane_addr + bn / 2 + c, y, u);
                else if constexpr (PIECE == 32) tmem_load32(lane_addr + c, y);
                else tmem_load16(lane_addr + c, y);
                // the piece's scales go round the warp through the buffer that its output will fill (32 shuffles a piece took longer than the products);
                // TMA has read what lay there two pieces ago
                const uint32_t out = stage_out + (used & 1) * OUT_BUFFER;
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                __syncwarp();
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(out + lane * 4), "f"(ws) : "memory");
                if constexpr (GATED) asm volatile("st.shared.f32 [%0], %1;" ::"r"(out + 128 + lane * 4), "f"(us) : "memory");
                __syncwarp();
                ws = column_scale(tile, c + 2 * PIECE, 0);
                if constexpr (GATED) us = column_scale(tile, c + 2 * PIECE, 1);
                auto scale_all = [&](float* v, uint32_t at) {
#pragma unroll
                    for (int q = 0; q < PIECE; q += 4) {
                        float s4[4];
                        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(s4[0]), "=f"(s4[1]), "=f"(s4[2]), "=f"(s4[3]) : "r"(at + q * 4) : "memory");
#pragma unroll
                        for (int i = 0; i < 4; i++) v[q + i] = scaled(__float_as_int(v[q + i]), sa, s4[i]);
                    }
                };
                scale_all(y, out);
                if constexpr (GATED) {
                    scale_all(u, out + 128);
                    if (plain) {
#pragma unroll
                        for (int q = 0; q < PIECE; q++) y[q] = swish<TC>(y[q], 1.0f) * u[q];
                    } else {
#pragma unroll
                        for (int q = 0; q < PIECE; q++) y[q] = n + q < p.N ? gated_at<TC>(p.glu, y[q], u[q], n + q, p.N) : 0.f;
                    }
                }
                // the token's 64 bytes, its 16-byte pieces where the 64-byte swizzle has them
                __syncwarp();
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const uint32_t at = out + lane * PIECE_BYTES + ((q ^ ((lane >> 1) & 3)) << 4);
                    uint32_t w[4];
                    if constexpr (sizeof(TC) == 4) {
#pragma unroll
                        for (int i = 0; i < 4; i++) w[i] = __float_as_uint(y[4 * q + i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const __nv_bfloat162 h = __floats2bfloat162_rn(y[8 * q + 2 * i], y[8 * q + 2 * i + 1]);
                            w[i] = *reinterpret_cast<const uint32_t*>(&h);
                        }
                    }
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                }
                if (p.tma_out) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        if constexpr (EPI == EPI_ACCUMULATE)
                            asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2}], [%3];"
                                         ::"l"((uint64_t)&map_c), "r"(n), "r"(t_first), "r"(out) : "memory");
                        else
                            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];"
                                         ::"l"((uint64_t)&map_c), "r"(n), "r"(t_first), "r"(out) : "memory");
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                    used++;
                } else {
                    // rows that TMA does not write: a row's columns side by side, so that an access meets a few sectors and not 32 (4,076 x 4,353 x 768 25 us,
                    // with the reads out of shared memory one behind the other 34, and 4,352 columns by TMA 19)
                    __syncwarp();
                    constexpr int ROWS = 32 / PIECE, BATCH = 8;            // rows an access, accesses whose reads are under way together
                    const int col = lane % PIECE, first = lane / PIECE, at = col * (int)sizeof(TC);
                    const int rows = n + col < p.N ? p.T - t_first - first : 0;
                    TC* dst = C + (size_t)(t_first + first) * p.ldc + n + col;
#pragma unroll
                    for (int i0 = 0; i0 < 32 / ROWS; i0 += BATCH) {
                        TC v[BATCH];
#pragma unroll
                        for (int i = 0; i < BATCH; i++) {
                            const int row = (i0 + i) * ROWS;                // (row + first has the same place in the swizzle)
                            const uint32_t from = out + (row + first) * PIECE_BYTES + ((((at >> 4) ^ ((row >> 1) & 3)) << 4) | (at & 15));
                            if constexpr (sizeof(TC) == 4) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[i]) : "r"(from) : "memory");
                            else {
                                unsigned short h;
                                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(from) : "memory");
                                v[i] = __ushort_as_bfloat16(h);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < BATCH; i++, dst += ROWS * p.ldc) {
                            if ((i0 + i) * ROWS >= rows) continue;
                            // (added in memory, once a place: a read of the old value would be waited for row by row.  5,734 x 13,459 x 6,344 took
                            // 1.1 ms so, and takes 0.44)
                            if constexpr (EPI == EPI_ACCUMULATE) asm volatile("red.global.add.f32 [%0], %1;" ::"l"(dst), "f"(v[i]) : "memory");
                            else *dst = v[i];
                        }
                    }
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive_even(at_rank(acc_empty0 + 8 * buf, 0));
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");      // what left by TMA is in memory
        __syncwarp();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    __syncwarp();
    cluster_sync_all();                 // neither CTA leaves while the other may still arrive at its barriers
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2 * PAIR_BN) : "memory");
    }
}

// --------------------------------------------------------------------------------------------
// host side
// --------------------------------------------------------------------------------------------
// [rows, cols] 8-bit integers, rows ld bytes apart: boxes of 128 columns x box_rows rows, 128-byte swizzle, zeros outside the matrix
bool make_map_q8(CUtensorMap* map, const void* base, long rows, long cols, long ld, int box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
    cuuint32_t box[2] = {BLOCK_K, (cuuint32_t)box_rows}, elem[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// the output [rows, cols]: boxes of 64 bytes x 32 rows, 64-byte swizzle
bool make_map_out(CUtensorMap* map, void* base, bool bf16, long rows, long cols, long ld) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const int size = bf16 ? 2 : 4;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * size};
    cuuint32_t box[2] = {(cuuint32_t)(PIECE_BYTES / size), 32}, elem[2] = {1, 1};
    return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, base, dims, strides, box, elem,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Plan {
    bool few;
    int bn, stages, splits, k_blocks_per_split;
    int tiles_n, tiles_t, ctas;
    size_t smem;
    double cost;             // ns
};

// What decides between the kernels, widths and cuts: estimates of a call's time in ns, fitted to sweeps of 4 to 6,000 tokens over eleven weights of 1,000 x 500
// to 28,672 x 4,096 with every cut, and pairs of 64, 128, 192 and 256 weight rows.  Against every cut and every width that it may choose (20 numbers of tokens
// from 1 to 6,000) its choice was within 4 % of the best one at 186 of 220 products, within 10 % at 211 and within 19 % at all.
// A CTA of the few-token kernel takes 200 ns a k block as long as its SM takes in less than 145 bytes a ns; partial sums cost by the number of ranks, and more
// where more tokens are folded.  A pair by itself takes 1.07 ns a k block and weight row, and no less than its tiles' way from L2 (165 ns); with all SMs at
// work (power, L2) 115 ns and 0.76 ns a weight row.
constexpr double BYTES_NS = 6500.0, SM_BYTES_NS = 145.0, FEW_BLOCK_NS = 200.0, PAIR_BLOCK_NS = 165.0, PAIR_COLUMN_NS = 1.07, PAIR_BUSY_NS = 115.0,
                 PAIR_BUSY_COLUMN_NS = 0.76, PAIR_TILE_NS = 600.0;

// clusters of c CTAs lie inside one GPC, whose SMs they seldom fill: the CTAs that are on the device at one time with one on an SM (of 148)
constexpr int RESIDENT[MAX_RANKS] = {148, 144, 132, 128, 120, 104, 104, 104};

bool plan_few(Plan& pl, int T, int N, int K, bool gated, int sm_count, int bn, int want) {
    const int k_blocks = (K + BLOCK_K - 1) / BLOCK_K;
    pl.few = true;
    pl.bn = bn;
    pl.tiles_n = (N + TILE_M - 1) / TILE_M;
    pl.tiles_t = (T + bn - 1) / bn;
    pl.k_blocks_per_split = (k_blocks + want - 1) / want;
    pl.splits = (k_blocks + pl.k_blocks_per_split - 1) / pl.k_blocks_per_split;
    if (want > 1 && (pl.splits != want || pl.k_blocks_per_split < 2)) return false;
    const long ctas = (long)pl.tiles_n * pl.tiles_t * pl.splits, one = (long)RESIDENT[pl.splits - 1] * sm_count / 148;
    if (pl.splits > 1 && ctas > 2 * one) return false;       // a second wave of clusters costs a call's whole latency again
    if (pl.tiles_t > 65535 || ctas > 2147483647L) return false;
    pl.ctas = (int)ctas;
    const int acc = gated ? 2 : 1, stage = acc * A_TILE_BYTES + bn * BLOCK_K, sums = acc * bn * TILE_M * 4;
    int stages = (ctas <= one ? 200 : 110) * 1024 / stage;     // an SM's whole memory, or half where two CTAs share one
    stages = stages > MAX_STAGES ? MAX_STAGES : stages > pl.k_blocks_per_split ? pl.k_blocks_per_split : stages;
    pl.stages = stages < 2 ? 2 : stages;
    const size_t ring = (size_t)pl.stages * stage;
    pl.smem = (ring > (size_t)sums ? ring : (size_t)sums) + 1024;
    const double on_sm = ctas <= one ? 1 : pl.splits > 1 ? 2 : (double)((ctas + sm_count - 1) / sm_count);
    const double block = stage / SM_BYTES_NS * on_sm > FEW_BLOCK_NS ? stage / SM_BYTES_NS * on_sm : FEW_BLOCK_NS;
    const double memory = ((double)acc * N * K + (double)T * K) / BYTES_NS, stream = pl.k_blocks_per_split * block + (memory < 4000 ? 0.5 * memory : 2000.0);
    const int columns = T < bn ? T : bn;
    const double start = bn <= 32 ? (gated ? 3900 : 3400) : (gated ? 5600 : 3600) + (columns > 64 ? (columns - 64) * (gated ? 50.0 : 20.0) : 0.0);
    const double waves = pl.splits == 1 && ctas > one ? (double)ctas / one : 1.0, tokens = 100.0 * (pl.tiles_t - 1);
    const double fold = (pl.splits - 1) * (bn == 16 ? 100.0 : bn == 32 ? 200.0 : 450.0);
    pl.cost = start * waves + tokens + fold + (stream > memory ? stream : memory);
    return true;
}

void plan_pairs(Plan& pl, int T, int N, int K, bool gated, int sm_count, int bn) {
    const int k_blocks = (K + BLOCK_K - 1) / BLOCK_K, out = gated ? bn / 2 : bn, pairs = sm_count / 2;
    pl.few = false;
    pl.bn = bn;
    pl.splits = 1;
    pl.k_blocks_per_split = k_blocks;
    pl.tiles_n = (N + out - 1) / out;
    pl.tiles_t = (T + 2 * TILE_M - 1) / (2 * TILE_M);
    const long tiles = (long)pl.tiles_n * pl.tiles_t, waves = (tiles + pairs - 1) / pairs;
    pl.ctas = 2 * (int)(tiles < pairs ? tiles : pairs);
    const int stage = A_TILE_BYTES + bn / 2 * BLOCK_K, stages = (225 * 1024 - OUT_BYTES) / stage;
    pl.stages = stages > MAX_STAGES ? MAX_STAGES : stages;
    pl.smem = (size_t)pl.stages * stage + OUT_BYTES + 1024;
    const double alone = PAIR_COLUMN_NS * bn > PAIR_BLOCK_NS ? PAIR_COLUMN_NS * bn : PAIR_BLOCK_NS, together = PAIR_BUSY_NS + PAIR_BUSY_COLUMN_NS * bn;
    const double busy = tiles < pairs ? (double)tiles / pairs : 1.0, block = alone + (together - alone) * busy;
    const double memory = ((gated ? 2.0 : 1.0) * N * K + (double)T * K) / BYTES_NS, stream = waves * (k_blocks * block + PAIR_TILE_NS);
    pl.cost = 2500.0 + 10.0 * bn + (stream > memory ? stream : memory);
}

constexpr long MOST_TILES = 1L << 30;      // (they are counted in an int, some beyond the last)
constexpr int FEW_MOST_TOKENS = 512;       // from here on pairs were the faster ones at every size swept

Plan make_plan(int T, int N, int K, bool gated, int sm_count) {
    Plan best{}, pl{};
    best.cost = 1e300;
    if (T <= FEW_MOST_TOKENS) {
        const int narrowest = T <= 16 ? 16 : T <= 32 ? 32 : 64, widest = T <= 64 ? narrowest : 128;
        for (int bn = narrowest; bn <= widest; bn *= 2)
            for (int splits = MAX_RANKS; splits >= 1; splits--)
                if (plan_few(pl, T, N, K, gated, sm_count, bn, splits) && pl.cost < best.cost) best = pl;
    }
    if (T > 64)
        for (int bn = PAIR_BN; bn >= 64; bn -= gated ? 64 : 32) {      // (a piece of 32 output columns at a time)
            plan_pairs(pl, T, N, K, gated, sm_count, bn);
            if (pl.cost < best.cost) best = pl;
        }
    return best;
}

int sm_count_of_current_device() {
    static int cached[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return 148;
    if (!cached[dev]) cudaDeviceGetAttribute(&cached[dev], cudaDevAttrMultiProcessorCount, dev);
    return cached[dev] > 0 ? cached[dev] : 148;
}

template <auto KERNEL, typename... Args>
int launch_cluster(dim3 grid, int threads, dim3 cluster, size_t smem, cudaStream_t stream, Args... args) {
    static bool configured[64] = {};       // per kernel and device
    int dev = 0;
    cudaGetDevice(&dev);
    cudaError_t e = cudaSuccess;
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024);
        if (e == cudaSuccess && dev >= 0 && dev < 64) configured[dev] = true;
    }
    if (e == cudaSuccess) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = grid;
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = hymt2_pdl_enabled() ? 1 : 0;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = cluster.x;
        attr[1].val.clusterDim.y = cluster.y;
        attr[1].val.clusterDim.z = cluster.z;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        e = cudaLaunchKernelEx(&cfg, KERNEL, args...);
    }
    if (e != cudaSuccess) { hymt2_set_error("gemm_q8_tc: %s", cudaGetErrorString(e)); return HYMT2_ERR_LAUNCH; }
    return hymt2_check_launch("gemm_q8_tc");
}

template <int EPI, typename TC, bool FAULT = false>
int run(const void* A, const void* W, long lda, long ldw, GemmQ8Params p, const Plan& pl, cudaStream_t stream) {
    CUtensorMap ma, mw, mc{};
    const long w_rows = EPI == EPI_GATED ? 2L * p.N : p.N;
    HYMT2_REQUIRE(make_map_q8(&ma, A, p.T, p.K, lda, pl.few ? pl.bn : TILE_M) && make_map_q8(&mw, W, w_rows, p.K, ldw, pl.few ? TILE_M : pl.bn / 2),
                  "gemm_q8_tc: cuTensorMapEncodeTiled refused the operands");
    if (pl.few) {
        const dim3 grid(pl.tiles_n, pl.tiles_t, pl.splits), cluster(1, 1, pl.splits);
        const int threads = 64 + 32 * few_warps(pl.bn);
        if constexpr (FAULT) {
            HYMT2_REQUIRE(pl.bn == 16, "gemm_q8_debug: at most 16 tokens, or many");
            return launch_cluster<gemm_q8_few_kernel<16, EPI, TC, true>>(grid, threads, cluster, pl.smem, stream, mw, ma, p);
        } else switch (pl.bn) {
            case 16: return launch_cluster<gemm_q8_few_kernel<16, EPI, TC>>(grid, threads, cluster, pl.smem, stream, mw, ma, p);
            case 32: return launch_cluster<gemm_q8_few_kernel<32, EPI, TC>>(grid, threads, cluster, pl.smem, stream, mw, ma, p);
            case 64: return launch_cluster<gemm_q8_few_kernel<64, EPI, TC>>(grid, threads, cluster, pl.smem, stream, mw, ma, p);
            default: return launch_cluster<gemm_q8_few_kernel<128, EPI, TC>>(grid, threads, cluster, pl.smem, stream, mw, ma, p);
        }
    }
    // (TMA writes whole pieces of 16 bytes: where the last of a row is not whole, it would write what lies between the rows)
    p.tma_out = (uintptr_t)p.C % 16 == 0 && p.ldc * (long)sizeof(TC) % 16 == 0 && p.N * (long)sizeof(TC) % 16 == 0;
    if (p.tma_out) HYMT2_REQUIRE(make_map_out(&mc, p.C, sizeof(TC) == 2, p.T, p.N, p.ldc), "gemm_q8_tc: cuTensorMapEncodeTiled refused the output");
    return launch_cluster<gemm_q8_pair_kernel<EPI, TC, FAULT>>(dim3(pl.ctas), PAIR_THREADS, dim3(2, 1, 1), pl.smem, stream, ma, mw, mc, p);
}

}  // namespace

// How a product of T tokens, N outputs (gated: of 2N weight rows) and K would be run on a device of sm_count SMs (0: the current one): out[0] the kernel for few
// tokens, [1] the tile's other side (tokens, or a pair's weight rows), [2] stages of the ring, [3] the cut of K, [4] k blocks of a part, [5] CTAs, [6] bytes of
// shared memory.  Nothing is launched.  (A device has room for a pair of CTAs.)
HYMT2_API int hymt2_gemm_q8_describe(int T, int N, int K, int gated, int sm_count, long* out) {
    HYMT2_REQUIRE(T > 0 && N > 0 && K > 0 && K <= MAX_K && sm_count != 1 && out, "gemm_q8_describe: bad arguments");
    const Plan pl = make_plan(T, N, K, gated != 0, sm_count > 0 ? sm_count : sm_count_of_current_device());
    const long v[7] = {pl.few, pl.bn, pl.stages, pl.splits, pl.k_blocks_per_split, pl.ctas, (long)pl.smem};
    for (int i = 0; i < 7; i++) out[i] = v[i];
    return HYMT2_OK;
}

// C[T, N] (ldc) = epilogue(A[T, K] (lda) · W[N, K]^T (ldw)) with the scales of A's rows and W's; gated: W has 2N rows.  weights_settled: W and its
// scales were complete before the kernel in front of this one was launched, so they are fetched while that one still runs.
HYMT2_API int hymt2_gemm_q8_tc(void* C, int c_dtype, const void* A, const float* a_scale, const void* W, const float* w_scale, int T, int N, int K,
                               long lda, long ldw, long ldc, int epilogue, int weights_settled, int* status, cudaStream_t stream, int glu_kind,
                               float glu_limit, float glu_alpha, const float* glu_bias) {
    if (T == 0 || N == 0) return HYMT2_OK;
    HYMT2_REQUIRE(T > 0 && N > 0 && K > 0 && K <= MAX_K, "gemm_q8_tc: bad sizes T=%d N=%d K=%d (K is at most %d)", T, N, K, MAX_K);
    HYMT2_REQUIRE(lda % 16 == 0 && ldw % 16 == 0 && (uintptr_t)A % 16 == 0 && (uintptr_t)W % 16 == 0, "gemm_q8_tc: rows must start on 16 bytes");
    HYMT2_REQUIRE(epilogue >= 0 && epilogue <= 2 && (c_dtype == HYMT2_F32 || (c_dtype == HYMT2_BF16 && epilogue != EPI_ACCUMULATE)),
                  "gemm_q8_tc: epilogue %d with output type %d is not built", epilogue, c_dtype);
    HYMT2_REQUIRE(status != nullptr, "gemm_q8_tc: a status word is needed");
    const Plan pl = make_plan(T, N, K, epilogue == EPI_GATED, sm_count_of_current_device());
    HYMT2_REQUIRE((long)pl.tiles_t * pl.tiles_n <= MOST_TILES, "gemm_q8_tc: too many tiles");
    const GemmQ8Params p{C, a_scale, w_scale, ldc, T, N, K, pl.bn, pl.stages, pl.splits, pl.k_blocks_per_split, weights_settled, 0, status,
                         GluRule{glu_kind, glu_limit, glu_alpha, glu_bias}, WAIT_LIMIT, -1};
    if (epilogue == EPI_ACCUMULATE) return run<EPI_ACCUMULATE, float>(A, W, lda, ldw, p, pl, stream);
    if (epilogue == EPI_STORE)
        return c_dtype == HYMT2_F32 ? run<EPI_STORE, float>(A, W, lda, ldw, p, pl, stream) : run<EPI_STORE, __nv_bfloat16>(A, W, lda, ldw, p, pl, stream);
    return c_dtype == HYMT2_F32 ? run<EPI_GATED, float>(A, W, lda, ldw, p, pl, stream) : run<EPI_GATED, __nv_bfloat16>(A, W, lda, ldw, p, pl, stream);
}

// The same product with a fault put in on purpose, for a test of the waits: the copies of k block `withhold_block` are announced and never made, and every
// wait gives up after `wait_limit` tries (a few thousand: milliseconds).  The waits for that block, for the stages behind it and for the sums then run out: a
// CTA whose wait does writes 151, 152 or 153 into the status word and raises its abort flag, every role leaves its loop, every CTA comes to the cluster's
// barriers, C's tile is NaN (few tokens) or left as it was, copies in flight land, tensor memory is freed and the kernel returns.  Only sums added into float32 and
// gated products into bfloat16, of up to 16 tokens or of many, on at most 8 CTAs are taken.
HYMT2_API int hymt2_gemm_q8_debug(void* C, int c_dtype, const void* A, const float* a_scale, const void* W, const float* w_scale, int T, int N, int K,
                                  long lda, long ldw, long ldc, int epilogue, int* status, cudaStream_t stream, int wait_limit, int withhold_block) {
    HYMT2_REQUIRE(T > 0 && N > 0 && K > 0 && K <= MAX_K && status != nullptr, "gemm_q8_debug: bad sizes T=%d N=%d K=%d", T, N, K);
    HYMT2_REQUIRE(wait_limit > 0 && wait_limit <= (1 << 16), "gemm_q8_debug: wait_limit %d must be in [1, 65536]", wait_limit);
    HYMT2_REQUIRE(withhold_block >= 0 && withhold_block < (K + BLOCK_K - 1) / BLOCK_K, "gemm_q8_debug: K has no block %d", withhold_block);
    const Plan pl = make_plan(T, N, K, epilogue == EPI_GATED, sm_count_of_current_device());
    HYMT2_REQUIRE(pl.ctas <= MAX_RANKS, "gemm_q8_debug: at most %d CTAs", MAX_RANKS);
    const GemmQ8Params p{C, a_scale, w_scale, ldc, T, N, K, pl.bn, pl.stages, pl.splits, pl.k_blocks_per_split, 0, 0, status, GluRule{}, (uint32_t)wait_limit,
                         withhold_block};
    if (epilogue == EPI_ACCUMULATE && c_dtype == HYMT2_F32) return run<EPI_ACCUMULATE, float, true>(A, W, lda, ldw, p, pl, stream);
    if (epilogue == EPI_GATED && c_dtype == HYMT2_BF16) return run<EPI_GATED, __nv_bfloat16, true>(A, W, lda, ldw, p, pl, stream);
    HYMT2_REQUIRE(false, "gemm_q8_debug: epilogue %d with output type %d is not built", epilogue, c_dtype);
}
