// Products of 8-bit integers with a scale for each token and one for each output channel:
//   C[t, n] = epilogue(a_scale[t] w_scale[n] sum_k A[t, k] W[n, k])
// The sums are 32-bit integers and exact (K up to 131,071: 128 * 128 * K stays below 2^31), so a row's result does not depend on how K is cut,
// nor on the other rows.  Epilogues: store (float32 or bfloat16), add into float32 C, gated (W holds N gate rows, then N up rows).
#include "common.cuh"

namespace {

enum { EPI_STORE = 0, EPI_ACCUMULATE = 1, EPI_GATED = 2 };
constexpr int MAX_K = 131071, TILE = 64, TILE_K = 64;

struct GemmQ8Params {
    void* C;
    const int8_t *A, *W;
    const float *a_scale, *w_scale;
    long lda, ldw, ldc;
    int T, N, K;
    GluRule glu;
};

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
// glu_at of common.cuh, but a NaN stays one under the clamps: it says that the row held one before it became integers
__device__ __forceinline__ float gated_at(const GluRule& r, float g, float u, int n, int N) {
    if (r.bias) { g += r.bias[n]; u += r.bias[N + n]; }
    if (r.kind == GLU_SILU) return silu_mul(g, u);
    g = min_nan(g, r.limit);
    u = min_nan(max_nan(u, -r.limit), r.limit);
    return g / (1.0f + expf(-r.alpha * g)) * (u + 1.0f);
}

template <int EPI, typename TC>
__global__ void gemm_q8_kernel(GemmQ8Params p) {
    __shared__ int a_s[TILE][TILE_K / 4 + 1], w_s[2][TILE][TILE_K / 4 + 1];
    constexpr int PARTS = EPI == EPI_GATED ? 2 : 1;
    pdl_wait();
    pdl_launch_dependents();
    const int t0 = blockIdx.x * TILE, n0 = blockIdx.y * TILE;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    int acc[PARTS][4][4] = {};
    auto word = [&](const int8_t* m, long ld, long row, bool in, int k) {
        int v = 0;
        if (in && k < p.K) {
            v = *reinterpret_cast<const int*>(m + row * ld + k);          // (rows lie on 16 bytes, so the word is the matrix's own memory)
            if (k + 4 > p.K) v &= (1 << (8 * (p.K - k))) - 1;
        }
        return v;
    };
    for (int k0 = 0; k0 < p.K; k0 += TILE_K) {
        for (int i = threadIdx.x; i < TILE * TILE_K / 4; i += 256) {
            const int row = i / (TILE_K / 4), k = i % (TILE_K / 4);
            a_s[row][k] = word(p.A, p.lda, t0 + row, t0 + row < p.T, k0 + 4 * k);
            for (int h = 0; h < PARTS; h++) w_s[h][row][k] = word(p.W, p.ldw, (long)h * p.N + n0 + row, n0 + row < p.N, k0 + 4 * k);
        }
        __syncthreads();
        for (int k = 0; k < TILE_K / 4; k++)
            for (int i = 0; i < 4; i++)
                for (int h = 0; h < PARTS; h++)
                    for (int j = 0; j < 4; j++) acc[h][i][j] = __dp4a(a_s[ty * 4 + i][k], w_s[h][tx * 4 + j][k], acc[h][i][j]);
        __syncthreads();
    }
    TC* C = (TC*)p.C;
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) {
            const int t = t0 + ty * 4 + i, n = n0 + tx * 4 + j;
            if (t >= p.T || n >= p.N) continue;
            const float y = (float)acc[0][i][j] * p.a_scale[t] * p.w_scale[n];
            TC* dst = C + (size_t)t * p.ldc + n;
            if (EPI == EPI_STORE) *dst = from_float<TC>(y);
            else if (EPI == EPI_ACCUMULATE) *dst = from_float<TC>(to_float(*dst) + y);
            else *dst = from_float<TC>(gated_at(p.glu, y, (float)acc[PARTS - 1][i][j] * p.a_scale[t] * p.w_scale[p.N + n], n, p.N));
        }
}

}  // namespace

// C[T, N] (ldc) = epilogue(A[T, K] (lda) · W[N, K]^T (ldw)) with the scales of A's rows and W's; gated: W has 2N rows.
HYMT2_API int hymt2_gemm_q8_tc(void* C, int c_dtype, const void* A, const float* a_scale, const void* W, const float* w_scale, int T, int N, int K,
                               long lda, long ldw, long ldc, int epilogue, int* status, cudaStream_t stream, int glu_kind, float glu_limit,
                               float glu_alpha, const float* glu_bias) {
    if (T == 0 || N == 0) return HYMT2_OK;
    HYMT2_REQUIRE(T > 0 && N > 0 && K > 0 && K <= MAX_K, "gemm_q8_tc: bad sizes T=%d N=%d K=%d (K is at most %d)", T, N, K, MAX_K);
    HYMT2_REQUIRE(lda % 16 == 0 && ldw % 16 == 0 && (uintptr_t)A % 16 == 0 && (uintptr_t)W % 16 == 0, "gemm_q8_tc: rows must start on 16 bytes");
    const GemmQ8Params p{C, (const int8_t*)A, (const int8_t*)W, a_scale, w_scale, lda, ldw, ldc, T, N, K, GluRule{glu_kind, glu_limit, glu_alpha, glu_bias}};
    const dim3 grid((T + TILE - 1) / TILE, (N + TILE - 1) / TILE);
    if (epilogue == EPI_ACCUMULATE) {
        HYMT2_REQUIRE(c_dtype == HYMT2_F32, "gemm_q8_tc: sums are added into float32 only");
        launch_pdl(gemm_q8_kernel<EPI_ACCUMULATE, float>, grid, dim3(256), 0, stream, p);
    } else if (epilogue == EPI_STORE) {
        HYMT2_DISPATCH_DTYPE(c_dtype, TC, (launch_pdl(gemm_q8_kernel<EPI_STORE, TC>, grid, dim3(256), 0, stream, p)));
    } else {
        HYMT2_REQUIRE(epilogue == EPI_GATED, "gemm_q8_tc: unknown epilogue %d", epilogue);
        HYMT2_DISPATCH_DTYPE(c_dtype, TC, (launch_pdl(gemm_q8_kernel<EPI_GATED, TC>, grid, dim3(256), 0, stream, p)));
    }
    return hymt2_check_launch("gemm_q8_tc");
}
