// Rows of 8-bit integers with a float32 scale each, and what makes and reads them:
//   q = 127 x / max|x|, rounded to the nearest whole number (ties to even),  s = max|x| / 127;   a row stands for q s
//   quantize_q8     the rows of a matrix (activations; a weight matrix, whose rows are output channels)
//   dequantize_q8   q s again
//   rmsnorm_q8      t = x + add (kept in x's type), r = 1 / sqrt(mean(t^2) + eps): q and s of the rows t gain, s times r.  r is the same for
//                   the whole row, so it changes no integer and goes into the scale.
// A row that holds a NaN or an infinity gets the scale NaN and zeros: whatever is computed from it is NaN.  A row of zeros gets the scale 0.
// The whole numbers are exact: the quotient of the numbers as they are stored, not of rounded ones, decides (q8_settle).
#include "common.cuh"

namespace {

struct RowCode {
    float f, inv, top;    // a power of two that keeps what follows in range; 127 / (max|x| f); max|x| f
    float s;              // the scale
    bool none;            // zeros: nothing in the row, or nothing that is a number
};

// `bits`: of the largest |x|, as an unsigned number, which orders infinity and NaN above all others
__device__ __forceinline__ RowCode row_code(uint32_t bits) {
    RowCode c;
    const float top = __uint_as_float(bits);
    c.none = bits == 0 || bits >= 0x7f800000u;
    c.f = top > 0x1p100f ? 0x1p-60f : top < 0x1p-60f ? 0x1p90f : 1.0f;
    c.top = top * c.f;
    c.inv = 127.0f / c.top;
    c.s = bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : top / 127.0f;
    return c;
}

// t = x inv is within 127 * 2^-23 = 1.6e-5 of the quotient v = 127 x / top, so the nearest whole number of t is that of v unless t lies within
// 2e-5 of a border b (a whole number and a half).  There the sign of 127 x - b top decides: 127 x is hi + lo without an error, hi - b top is
// a multiple of half of top's last place and small, so both differences are exact.
constexpr float NEAR_BORDER = 0.49998f;
__device__ __noinline__ float q8_settle(float x, float r, float e, float top) {
    const float b = r + copysignf(0.5f, e);
    const float hi = 127.0f * x, lo = fmaf(127.0f, x, -hi);
    const float d = fmaf(-b, top, hi) + lo;
    return d == 0.f ? rintf(b) : d > 0.f ? b + 0.5f : b - 0.5f;
}
__device__ __forceinline__ int8_t q8_of(float x, const RowCode& c) {
    if (c.none) return 0;
    const float v = x * c.f, t = v * c.inv;
    float r = rintf(t);
    if (fabsf(t - r) > NEAR_BORDER) r = q8_settle(v, r, t - r, c.top);
    return (int8_t)(int)r;
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t block_umax(uint32_t v, uint32_t* scratch) {
    v = __reduce_max_sync(0xffffffffu, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    for (int w = 0; w < (int)(blockDim.x >> 5); w++) v = max(v, scratch[w]);
    return v;
}

template <typename TX>
__global__ void quantize_q8_kernel(int8_t* q, long ldq, float* scale, const TX* x, long ldx, int width) {
    __shared__ uint32_t most_s[32];
    pdl_wait();
    pdl_launch_dependents();
    const size_t r = blockIdx.x;
    const TX* src = x + r * ldx;
    uint32_t most = 0;
    for (int i = threadIdx.x; i < width; i += blockDim.x) most = max(most, abs_bits(to_float(src[i])));
    const RowCode c = row_code(block_umax(most, most_s));
    for (int i = threadIdx.x; i < width; i += blockDim.x) q[r * ldq + i] = q8_of(to_float(src[i]), c);
    if (threadIdx.x == 0) scale[r] = c.s;
}

template <typename TY>
__global__ void dequantize_q8_kernel(TY* y, long ldy, const int8_t* q, long ldq, const float* scale, int width) {
    pdl_wait();
    pdl_launch_dependents();
    const size_t r = blockIdx.x;
    const float s = scale[r];
    for (int i = threadIdx.x; i < width; i += blockDim.x) y[r * ldy + i] = from_float<TY>((float)q[r * ldq + i] * s);
}

struct NormQ8Params {
    int8_t* q;
    float* scale;
    const void *x, *add;
    void* total;
    const void* gain;
    long ldq, ldx, ldadd, ldt;
    int width;
    float eps;
};

template <typename TX, typename TA, typename TG>
__global__ void rmsnorm_q8_kernel(NormQ8Params p) {
    __shared__ uint32_t most_s[32];
    __shared__ float sum_s[33];
    pdl_wait();
    pdl_launch_dependents();
    const size_t r = blockIdx.x;
    const TX* x = (const TX*)p.x + r * p.ldx;
    const TA* add = p.add ? (const TA*)p.add + r * p.ldadd : nullptr;
    TX* total = p.total ? (TX*)p.total + r * p.ldt : nullptr;
    const TG* gain = (const TG*)p.gain;
    auto at = [&](int i) { return add ? to_float(from_float<TX>(to_float(x[i]) + to_float(add[i]))) : to_float(x[i]); };
    uint32_t most = 0;
    float ss = 0.f;
    for (int i = threadIdx.x; i < p.width; i += blockDim.x) {
        const float t = at(i);
        ss = fmaf(t, t, ss);
        most = max(most, abs_bits(t * to_float(gain[i])));
    }
    const RowCode c = row_code(block_umax(most, most_s));
    const float scale = 1.0f / sqrtf(block_sum(ss, sum_s) / (float)p.width + p.eps);
    for (int i = threadIdx.x; i < p.width; i += blockDim.x) {
        const float t = at(i);
        p.q[r * p.ldq + i] = q8_of(t * to_float(gain[i]), c);
        if (total) total[i] = from_float<TX>(t);        // (x itself may be the place: entry i is not read again)
    }
    if (threadIdx.x == 0) p.scale[r] = c.s * scale;
}

inline int row_threads(int width) { return width >= 2048 ? 256 : width >= 512 ? 128 : 32; }

}  // namespace

HYMT2_API int hymt2_quantize_q8(void* q, long ldq, float* scale, const void* x, int x_dtype, long ldx, int rows, int width, cudaStream_t stream) {
    if (rows == 0) return HYMT2_OK;
    HYMT2_REQUIRE(rows > 0 && width > 0 && ldq >= width && ldx >= width, "quantize_q8: bad sizes rows=%d width=%d", rows, width);
    HYMT2_DISPATCH_DTYPE(x_dtype, TX, (launch_pdl(quantize_q8_kernel<TX>, dim3(rows), dim3(row_threads(width)), 0, stream, (int8_t*)q, ldq, scale,
                                                  (const TX*)x, ldx, width)));
    return hymt2_check_launch("quantize_q8");
}

HYMT2_API int hymt2_dequantize_q8(void* y, int y_dtype, long ldy, const void* q, long ldq, const float* scale, int rows, int width, cudaStream_t stream) {
    if (rows == 0) return HYMT2_OK;
    HYMT2_REQUIRE(rows > 0 && width > 0 && ldq >= width && ldy >= width, "dequantize_q8: bad sizes rows=%d width=%d", rows, width);
    HYMT2_DISPATCH_DTYPE(y_dtype, TY, (launch_pdl(dequantize_q8_kernel<TY>, dim3(rows), dim3(row_threads(width)), 0, stream, (TY*)y, ldy,
                                                  (const int8_t*)q, ldq, scale, width)));
    return hymt2_check_launch("dequantize_q8");
}

// x, add (or null), total (or null; it may be x): [rows, width] with rows ld* entries apart; gain [width].
HYMT2_API int hymt2_rmsnorm_q8(void* q, long ldq, float* scale, const void* x, int x_dtype, long ldx, const void* add, int add_dtype, long ldadd,
                               void* total, long ldt, const void* gain, int gain_dtype, int rows, int width, float eps, cudaStream_t stream) {
    if (rows == 0) return HYMT2_OK;
    HYMT2_REQUIRE(rows > 0 && width > 0 && ldq >= width && ldx >= width, "rmsnorm_q8: bad sizes rows=%d width=%d", rows, width);
    HYMT2_REQUIRE(!total || add, "rmsnorm_q8: the sums have a place, but nothing is added");
    const NormQ8Params p{(int8_t*)q, scale, x, add, total, gain, ldq, ldx, ldadd, ldt, width, eps};
    HYMT2_DISPATCH_DTYPE(x_dtype, TX, HYMT2_DISPATCH_DTYPE(add_dtype, TA, HYMT2_DISPATCH_DTYPE(gain_dtype, TG,
        (launch_pdl(rmsnorm_q8_kernel<TX, TA, TG>, dim3(rows), dim3(row_threads(width)), 0, stream, p)))));
    return hymt2_check_launch("rmsnorm_q8");
}
