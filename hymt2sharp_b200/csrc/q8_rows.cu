// Rows of 8-bit integers with a float32 scale each, and what makes and reads them:
//   q = 127 x / max|x|, rounded to the nearest whole number (ties to even),  s = max|x| / 127;   a row stands for q s
//   quantize_q8     the rows of a matrix (activations; a weight matrix, whose rows are output channels)
//   dequantize_q8   q s again
//   rmsnorm_q8      t = x + add (kept in x's type), r = 1 / sqrt(mean(t^2) + eps): q and s of the rows t gain, s times r.  r is the same for
//                   the whole row, so it changes no integer and goes into the scale.
// A row that holds a NaN or an infinity gets the scale NaN and zeros: whatever is computed from it is NaN.  A row of zeros gets the scale 0.
// The whole numbers are exact: the quotient of the numbers as they are stored, not of rounded ones, decides (q8_of).
#include "common.cuh"

// Each kernel waits for the one in front before it releases the one behind it: that one may take tensor memory which one in front has yet to take.
namespace {

struct RowCode {
    float f, inv, low, top;   // a power of two that keeps what follows in range; about 127 / (max|x| f), and what that leaves of it; max|x| f
    bool none;                // zeros: nothing in the row, or nothing that is a number
};

// `top`: the largest |x|, infinity and NaN included
__device__ __forceinline__ RowCode row_code(float top) {
    RowCode c;
    c.none = !(top < __uint_as_float(0x7f800000u)) || top == 0.f;
    c.f = top > 0x1p100f ? 0x1p-60f : top < 0x1p-60f ? 0x1p90f : 1.0f;
    c.top = top * c.f;
    asm("rcp.approx.f32 %0, %1;" : "=f"(c.inv) : "f"(c.top));
    c.low = c.inv;
    c.inv *= 127.0f;
    c.low *= __fmaf_rn(-c.inv, c.top, 127.0f);
    return c;
}
__device__ __forceinline__ float row_scale(float top) { return top < __uint_as_float(0x7f800000u) ? top / 127.0f : __uint_as_float(0x7fc00000u); }

// x inv is within 127 (2^-23 + 2^-24) = 2.3e-5 of the quotient 127 x / top (the approximate reciprocal's last place, a rounding), so the nearest whole
// number r of the one is that of the other unless the quotient lies within 3e-5 of a border b (a whole number and a half).  There the sign of
// 127 x - b top decides: 127 x is hi + lo without an error, hi - b top is a multiple of half of top's last place and small, so both differences are exact.
constexpr float NEAR_BORDER = 0.49997f;
// Adding 1.5 * 2^23 rounds to a whole number (ties to even), whose two's complement then fills the lowest bits.
constexpr float WHOLE = 12582912.0f;
// entries x (times c.f) of a row that is all numbers -> the whole numbers, in the lowest bytes
template <int V> __device__ __forceinline__ void q8_of(const float (&x)[V], const RowCode& c, uint32_t (&code)[V]) {
    float far = 0.f;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const float w = __fmaf_rn(x[i], c.inv, WHOLE);
        code[i] = __float_as_uint(w);
        far = fmaxf(far, fabsf(__fmaf_rn(x[i], c.inv, WHOLE - w)));
    }
    if (far > NEAR_BORDER) {      // (3e-5 on each side of a border: one float32 in 17,000, eight of them one time in 2,100)
#pragma unroll
        for (int i = 0; i < V; i++) {
            const float r = __uint_as_float(code[i]) - WHOLE, e = __fmaf_rn(x[i], c.inv, -r);
            if (fabsf(e) > NEAR_BORDER) {
                const float b = r + copysignf(0.5f, e), hi = 127.0f * x[i], d = __fmaf_rn(-b, c.top, hi) + __fmaf_rn(127.0f, x[i], -hi);
                code[i] = __float_as_uint((d == 0.f ? rintf(b) : d > 0.f ? b + 0.5f : b - 0.5f) + WHOLE);
            }
        }
    }
}
// The same for bfloat16 entries, without a special case: 127 x / top is x (inv + low) within 4e-12, summed so that t is that rounded once.  A border is a
// float32, so a quotient on one stays there (then ties go to even), and one of bfloat16 numbers that is not on a border is 2^-17 away from it at least
// (1 / (2 * 255 * 2^8)), twice what the rounding of t moves.
template <int V> __device__ __forceinline__ void q8_of_short(const float (&x)[V], const RowCode& c, uint32_t (&code)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) {
        const float p = __fmul_rn(x[i], c.inv), t = __fadd_rn(p, __fmaf_rn(x[i], c.low, __fmaf_rn(x[i], c.inv, -p)));
        code[i] = __float_as_uint(__fadd_rn(t, WHOLE));
    }
}
__device__ __forceinline__ uint32_t pack4(const uint32_t* c) { return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410); }

__device__ __forceinline__ float max_abs(float m, float x) {        // a NaN stays
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(x)));
    return r;
}
__device__ __forceinline__ float warp_max_bits(float m) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m))); }   // (not negative: as bits)

// A row is held in registers by the threads that share it, CH groups of 8 neighbouring entries each: WARP: a warp a row, several rows a block (up to
// 1,024 entries: no barrier); else a block a row.  Rows move 16 bytes at a time.  SHIFT: a row may begin anywhere (rows of odd length lie so); a thread then
// puts its entries together from the aligned pieces around them, and pieces to write from its own entries and its neighbour's (4,000 x 7,169 bfloat16 to
// integers 27 us, with one entry an access 69; a gain that does not start on 16 bytes is read entry by entry, out of the caches).
template <bool WARP> struct Place {
    size_t row;
    int tid, threads;
    bool in;
    __device__ Place(int rows) {
        if (WARP) { row = (size_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); tid = threadIdx.x & 31; threads = 32; }
        else { row = blockIdx.x; tid = threadIdx.x; threads = blockDim.x; }
        in = row < (size_t)rows;
    }
};

// eight entries as they are stored
template <typename T> struct Eight { uint32_t w[2 * (int)sizeof(T)]; };
// words of the byte stream `from` that begin m bytes (below 16) behind its start
template <int N> __device__ __forceinline__ void shifted_words(const uint32_t (&from)[N + 4], uint32_t m, uint32_t (&to)[N]) {
    const uint32_t bits = (m & 3) * 8;
    switch (m >> 2) {                   // (the same for a whole row)
        case 0:
#pragma unroll
            for (int i = 0; i < N; i++) to[i] = __funnelshift_r(from[i], from[i + 1], bits);
            break;
        case 1:
#pragma unroll
            for (int i = 0; i < N; i++) to[i] = __funnelshift_r(from[i + 1], from[i + 2], bits);
            break;
        case 2:
#pragma unroll
            for (int i = 0; i < N; i++) to[i] = __funnelshift_r(from[i + 2], from[i + 3], bits);
            break;
        default:
#pragma unroll
            for (int i = 0; i < N; i++) to[i] = __funnelshift_r(from[i + 3], from[i + 4], bits);
    }
}
// What may be read of a matrix around one of its rows, in bytes from the row's begin: from -front up to back (16 bytes each way at most).
struct Around { int front, back; };
template <bool SHIFT> __device__ __forceinline__ Around around(long row, long rows, long ld, int width, int size) {
    if (!SHIFT) return Around{0, width * size};
    const long front = row * ld * size, back = (rows - 1 - row) * ld * size;
    return Around{front < 16 ? (int)front : 16, width * size + (back < 16 ? (int)back : 16)};
}
// Entries at .. at + 7 of a row as the aligned pieces that hold them (pieces that the matrix does not hold whole are read entry by entry), and those entries
// out of the pieces, zeros behind the row's end.  (Two steps, so that all of a thread's reads are under way before it waits for one.)
template <bool SHIFT, typename T> struct Pieces {
    static constexpr int SIZE = (int)sizeof(T), COUNT = SIZE / 2 + (SHIFT ? 1 : 0);
    uint32_t w[4 * COUNT];
};
template <bool SHIFT, typename T> __device__ __forceinline__ void fetch8(const T* row, int at, int width, const Around& matrix, Pieces<SHIFT, T>& p) {
    using P = Pieces<SHIFT, T>;
    const int m = SHIFT ? (int)((uintptr_t)row & 15) : 0, begin = at * P::SIZE - m;
#pragma unroll
    for (int k = 0; k < P::COUNT; k++) {
        const int b = begin + 16 * k;
        if (b >= width * P::SIZE || (SHIFT && k + 1 == P::COUNT && m == 0)) {       // (nothing of the entries is there)
#pragma unroll
            for (int i = 0; i < 4; i++) p.w[4 * k + i] = 0;
        } else if (b >= -matrix.front && b + 16 <= matrix.back) {
            const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(row) + b);
            p.w[4 * k] = v.x; p.w[4 * k + 1] = v.y; p.w[4 * k + 2] = v.z; p.w[4 * k + 3] = v.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int n = at - m / P::SIZE + (16 * k + 4 * i) / P::SIZE;         // the entry that word i begins with
                if constexpr (P::SIZE == 2) {
                    const unsigned short* r = reinterpret_cast<const unsigned short*>(row);
                    p.w[4 * k + i] = (n >= 0 && n < width ? (uint32_t)r[n] : 0u) | (n + 1 >= 0 && n + 1 < width ? (uint32_t)r[n + 1] << 16 : 0u);
                } else p.w[4 * k + i] = n >= 0 && n < width ? __float_as_uint(row[n]) : 0u;
            }
        }
    }
}
template <bool SHIFT, typename T> __device__ __forceinline__ void settle8(const Pieces<SHIFT, T>& p, const T* row, int at, int width, Eight<T>& e) {
    constexpr int SIZE = (int)sizeof(T), WORDS = 2 * SIZE;
    if constexpr (SHIFT) shifted_words<WORDS>(p.w, (uint32_t)((uintptr_t)row & 15), e.w);
    else {
#pragma unroll
        for (int i = 0; i < WORDS; i++) e.w[i] = p.w[i];
    }
    if (SHIFT && at + 8 > width) {
#pragma unroll
        for (int i = 0; i < WORDS; i++) {
            if constexpr (SIZE == 2) e.w[i] = at + 2 * i + 1 < width ? e.w[i] : at + 2 * i < width ? e.w[i] & 0xffffu : 0u;
            else e.w[i] = at + i < width ? e.w[i] : 0u;
        }
    }
}
// the entries as float32, and the largest of `most` and their sizes (a bfloat16's bits are the upper half of the float32's; sizes are compared two at a time)
template <typename T> __device__ __forceinline__ void floats8(const Eight<T>& e, float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = __uint_as_float(e.w[i] << 16);
            v[2 * i + 1] = __uint_as_float(e.w[i] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = __uint_as_float(e.w[i]);
    }
}
template <typename T> __device__ __forceinline__ float most8(const Eight<T>& e, float most) {
    if constexpr (sizeof(T) == 2) {
        uint32_t m = e.w[0] & 0x7fff7fffu;
#pragma unroll
        for (int i = 1; i < 4; i++) m = __vmaxu2(m, e.w[i] & 0x7fff7fffu);
        return __uint_as_float(max(__float_as_uint(most), max(m << 16, m & 0xffff0000u)));
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) most = max_abs(most, __uint_as_float(e.w[i]));
        return most;
    }
}
template <bool SHIFT, typename T> __device__ __forceinline__ void settle8(const Pieces<SHIFT, T>& p, const T* row, int at, int width, float (&v)[8]) {
    Eight<T> e;
    settle8<SHIFT>(p, row, at, width, e);
    floats8(e, v);
}
// Writes entries at .. at + 7 of a row, as far as the row goes.  SHIFT: a whole warp calls it, with neighbouring entries in neighbouring lanes; a lane writes
// the aligned pieces that begin in its entries (the last one with its neighbour's first entries), and what no such piece covers one by one.
template <bool SHIFT, typename T> __device__ __forceinline__ void store8(T* row, int at, int width, const float (&v)[8]) {
    constexpr int SIZE = (int)sizeof(T), PIECES = SIZE / 2, WORDS = 4 * PIECES, PER = 16 / SIZE;
    Eight<T> e;
#pragma unroll
    for (int i = 0; i < WORDS; i++) {
        if constexpr (SIZE == 2) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            e.w[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else e.w[i] = __float_as_uint(v[i]);
    }
    auto singly = [&](int from, int to) {
#pragma unroll
        for (int i = 0; i < 8; i++) if (i >= from && i < to && at + i < width) row[at + i] = from_float<T>(v[i]);
    };
    const uint32_t m = SHIFT ? (uint32_t)((uintptr_t)(row + at) & 15) : 0;
    if (m == 0) {
        if (at + 8 <= width) {
#pragma unroll
            for (int k = 0; k < PIECES; k++) reinterpret_cast<uint4*>(row + at)[k] = make_uint4(e.w[4 * k], e.w[4 * k + 1], e.w[4 * k + 2], e.w[4 * k + 3]);
        } else singly(0, 8);
        return;
    }
    if constexpr (SHIFT) {
        const int head = 16 - (int)m, lane = threadIdx.x & 31;       // bytes in front of the first aligned piece
        uint32_t s[WORDS + 4], piece[WORDS];
#pragma unroll
        for (int i = 0; i < WORDS; i++) s[i] = e.w[i];
#pragma unroll
        for (int i = 0; i < 4; i++) s[WORDS + i] = __shfl_down_sync(0xffffffffu, e.w[i], 1);
        shifted_words<WORDS>(s, head, piece);
        if (at >= width) return;
        const long mine = (long)at * SIZE, end = (long)width * SIZE;
        uint4* to = reinterpret_cast<uint4*>(reinterpret_cast<char*>(row + at) + head);
        if (lane == 0 || mine + head > end) singly(0, head / SIZE);       // (else the lane below writes them)
#pragma unroll
        for (int k = 0; k < PIECES; k++) {
            const bool whole = mine + head + 16 * (k + 1) <= end && (k + 1 < PIECES || lane < 31);
            if (whole) to[k] = make_uint4(piece[4 * k], piece[4 * k + 1], piece[4 * k + 2], piece[4 * k + 3]);
            else singly(head / SIZE + k * PER, k + 1 < PIECES ? head / SIZE + (k + 1) * PER : 8);
        }
    }
}
template <bool SHORT> __device__ __forceinline__ void store_codes(int8_t* row, int at, int width, float (&v)[8], const RowCode& code) {
    uint32_t w[8];
    if (code.none) {
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = 0;
    } else {
        if (code.f != 1.0f) {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] *= code.f;
        }
        if constexpr (SHORT) q8_of_short(v, code, w);
        else q8_of(v, code, w);
    }
    if (at + 8 <= width) *reinterpret_cast<uint2*>(row + at) = make_uint2(pack4(w), pack4(w + 4));
    else {
#pragma unroll
        for (int i = 0; i < 8; i++) if (at + i < width) row[at + i] = (int8_t)w[i];
    }
}

// The largest |x| and (SUM) the sum of the squares over the threads of a row.  Sums in a fixed order.
template <bool WARP, bool SUM> __device__ __forceinline__ void over_row(float& most, float& ss, float2* scratch) {
    most = warp_max_bits(most);
    if (SUM) ss = warp_sum(ss);
    if (WARP) return;
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) scratch[threadIdx.x >> 5] = make_float2(most, ss);
    __syncthreads();
    const float2 mine = lane < warps ? scratch[lane] : make_float2(0.f, 0.f);
    most = warp_max_bits(mine.x);
    if (SUM) ss = warp_sum(mine.y);
}

// MOST: the threads of a block at most; 256: a warp a row.  (Blocks an SM that the registers are to leave room for, compiled for one and as here: 8,192 x 14,336
// bfloat16, three blocks of 448 threads, 81 and 72 us; 256 x 8,192, 4.4 and 3.4.)
constexpr int quantize_blocks(int ch, int most, bool shift, int size) {
    return most == 256 || (ch == 4 && most == 1024) ? 1 : ch == 4 ? (size == 2 && !shift ? 3 : 2) : shift ? 1 : 2;
}
template <typename TX, int CH, int MOST, bool SHIFT>
__global__ void __launch_bounds__(MOST, quantize_blocks(CH, MOST, SHIFT, sizeof(TX)))
quantize_q8_kernel(int8_t* q, long ldq, float* scale, const TX* x, long ldx, int rows, int width) {
    constexpr bool WARP = MOST == 256;
    __shared__ float2 scratch[32];
    pdl_wait();
    pdl_launch_dependents();
    const Place<WARP> at(rows);
    if (!at.in) return;
    const TX* src = x + at.row * ldx;
    const Around matrix = around<SHIFT>(at.row, rows, ldx, width, sizeof(TX));
    Eight<TX> x8[CH];             // (as they are stored: half the registers of float32 for bfloat16)
    Pieces<SHIFT, TX> pieces[CH];
    float most = 0.f, none = 0.f;
#pragma unroll
    for (int c = 0; c < CH; c++) fetch8<SHIFT>(src, 8 * (c * at.threads + at.tid), width, matrix, pieces[c]);
#pragma unroll
    for (int c = 0; c < CH; c++) {
        settle8<SHIFT>(pieces[c], src, 8 * (c * at.threads + at.tid), width, x8[c]);
        most = most8(x8[c], most);
    }
    over_row<WARP, false>(most, none, scratch);
    const RowCode code = row_code(most);
#pragma unroll
    for (int c = 0; c < CH; c++) {
        float v[8];
        floats8(x8[c], v);
        store_codes<sizeof(TX) == 2>(q + at.row * ldq, 8 * (c * at.threads + at.tid), width, v, code);
    }
    if (at.tid == 0) scale[at.row] = row_scale(most);
}

struct NormQ8Params {
    int8_t* q;
    float* scale;
    const void *x, *add;
    void* total;
    const void* gain;
    long ldq, ldx, ldadd, ldt;
    int rows, width;
    float eps;
};

template <typename TX, typename TA, typename TG, int CH, bool WARP, bool SHIFT>
__global__ void __launch_bounds__(WARP ? 256 : 1024, !WARP && CH == 1 && !SHIFT ? 2 : 1) rmsnorm_q8_kernel(NormQ8Params p) {
    __shared__ float2 scratch[32];
    pdl_wait();
    pdl_launch_dependents();
    const Place<WARP> at(p.rows);
    if (!at.in) return;
    const TX* x = (const TX*)p.x + at.row * p.ldx;
    const TA* add = (const TA*)p.add + at.row * p.ldadd;
    const TG* gain = (const TG*)p.gain;
    float v[CH][8], most = 0.f, ss = 0.f;
    Pieces<SHIFT, TX> px[CH];
    Pieces<SHIFT, TA> pa[CH];
    Pieces<false, TG> pg[CH];
    auto begin = [&](int c) { return 8 * (c * at.threads + at.tid); };
    const Around of_x = around<SHIFT>(at.row, p.rows, p.ldx, p.width, sizeof(TX)), of_add = around<SHIFT>(at.row, p.rows, p.ldadd, p.width, sizeof(TA)),
                 of_gain{0, (uintptr_t)gain % 16 == 0 ? p.width * (int)sizeof(TG) : 0};     // (a gain that begins elsewhere goes entry by entry)
#pragma unroll
    for (int c = 0; c < CH; c++) {
        fetch8<SHIFT>(x, begin(c), p.width, of_x, px[c]);
        if (p.add) fetch8<SHIFT>(add, begin(c), p.width, of_add, pa[c]);
        fetch8<false>(gain, begin(c), p.width, of_gain, pg[c]);
    }
#pragma unroll
    for (int c = 0; c < CH; c++) {
        settle8<SHIFT>(px[c], x, begin(c), p.width, v[c]);
        if (p.add) {
            float a[8];
            settle8<SHIFT>(pa[c], add, begin(c), p.width, a);
#pragma unroll
            for (int i = 0; i < 8; i++) v[c][i] = to_float(from_float<TX>(v[c][i] + a[i]));   // (as the rows are kept: what a later reader finds is normed)
            if (p.total) store8<SHIFT>((TX*)p.total + at.row * p.ldt, begin(c), p.width, v[c]);
        }
        float g[8];
        settle8<false>(pg[c], gain, begin(c), p.width, g);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            ss = fmaf(v[c][i], v[c][i], ss);
            v[c][i] *= g[i];
            most = max_abs(most, v[c][i]);
        }
    }
    over_row<WARP, true>(most, ss, scratch);
    const RowCode code = row_code(most);
#pragma unroll
    for (int c = 0; c < CH; c++) store_codes<false>(p.q + at.row * p.ldq, begin(c), p.width, v[c], code);
    if (at.tid == 0) p.scale[at.row] = row_scale(most) * (1.0f / sqrtf(ss / (float)p.width + p.eps));
}

// Rows that the registers of 1,024 threads do not hold (four groups a thread of quantize_q8, two of rmsnorm_q8) are read twice, the second time out of L2.
constexpr int LONGEST_HELD = 32768, LONGEST_NORMED = 16384;

template <typename TX, bool SHIFT>
__global__ void __launch_bounds__(1024) quantize_q8_long_kernel(int8_t* q, long ldq, float* scale, const TX* x, long ldx, int width) {
    __shared__ float2 scratch[32];
    pdl_wait();
    pdl_launch_dependents();
    const TX* src = x + (size_t)blockIdx.x * ldx;
    const Around matrix = around<SHIFT>(blockIdx.x, gridDim.x, ldx, width, sizeof(TX));
    float most = 0.f, none = 0.f;
    for (int c = 0; c * 8192 < width; c++) {
        Pieces<SHIFT, TX> pieces;
        float v[8];
        fetch8<SHIFT>(src, 8 * (c * 1024 + (int)threadIdx.x), width, matrix, pieces);
        settle8<SHIFT>(pieces, src, 8 * (c * 1024 + (int)threadIdx.x), width, v);
#pragma unroll
        for (int i = 0; i < 8; i++) most = max_abs(most, v[i]);
    }
    over_row<false, false>(most, none, scratch);
    const RowCode code = row_code(most);
    for (int c = 0; c * 8192 < width; c++) {
        Pieces<SHIFT, TX> pieces;
        float v[8];
        fetch8<SHIFT>(src, 8 * (c * 1024 + (int)threadIdx.x), width, matrix, pieces);
        settle8<SHIFT>(pieces, src, 8 * (c * 1024 + (int)threadIdx.x), width, v);
        store_codes<sizeof(TX) == 2>(q + (size_t)blockIdx.x * ldq, 8 * (c * 1024 + (int)threadIdx.x), width, v, code);
    }
    if (threadIdx.x == 0) scale[blockIdx.x] = row_scale(most);
}

template <typename TX, typename TA, typename TG, bool SHIFT>
__global__ void __launch_bounds__(1024) rmsnorm_q8_long_kernel(NormQ8Params p) {
    __shared__ float2 scratch[32];
    pdl_wait();
    pdl_launch_dependents();
    const size_t r = blockIdx.x;
    const TX* x = (const TX*)p.x + r * p.ldx;
    const TA* add = p.add ? (const TA*)p.add + r * p.ldadd : nullptr;
    TX* total = p.total ? (TX*)p.total + r * p.ldt : nullptr;
    const TG* gain = (const TG*)p.gain;
    const Around of_x = around<SHIFT>(r, p.rows, p.ldx, p.width, sizeof(TX)), of_add = around<SHIFT>(r, p.rows, p.ldadd, p.width, sizeof(TA)),
                 of_gain{0, (uintptr_t)gain % 16 == 0 ? p.width * (int)sizeof(TG) : 0};     // (a gain that begins elsewhere goes entry by entry)
    auto begin = [&](int c) { return 8 * (c * 1024 + (int)threadIdx.x); };
    auto read = [&](int c, float (&v)[8], float (&g)[8]) {
        Pieces<SHIFT, TX> px;
        Pieces<SHIFT, TA> pa;
        Pieces<false, TG> pg;
        fetch8<SHIFT>(x, begin(c), p.width, of_x, px);
        if (add) fetch8<SHIFT>(add, begin(c), p.width, of_add, pa);
        fetch8<false>(gain, begin(c), p.width, of_gain, pg);
        settle8<SHIFT>(px, x, begin(c), p.width, v);
        if (add) {
            float a[8];
            settle8<SHIFT>(pa, add, begin(c), p.width, a);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = to_float(from_float<TX>(v[i] + a[i]));
        }
        settle8<false>(pg, gain, begin(c), p.width, g);
    };
    float v[8], g[8], most = 0.f, ss = 0.f;
    for (int c = 0; c * 8192 < p.width; c++) {
        read(c, v, g);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            ss = fmaf(v[i], v[i], ss);
            most = max_abs(most, v[i] * g[i]);
        }
    }
    over_row<false, true>(most, ss, scratch);
    const RowCode code = row_code(most);
    for (int c = 0; c * 8192 < p.width; c++) {
        read(c, v, g);
        if (total) store8<SHIFT>(total, begin(c), p.width, v);        // (x itself may be the place: these entries are not read again)
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] *= g[i];
        store_codes<false>(p.q + r * p.ldq, begin(c), p.width, v, code);
    }
    if (threadIdx.x == 0) p.scale[r] = row_scale(most) * (1.0f / sqrtf(ss / (float)p.width + p.eps));
}

// A warp takes pieces of 4 x 32 groups of a row: of 16 output bytes, or (SHIFT) of 8 entries.
template <typename TY, bool SHIFT>
__global__ void __launch_bounds__(256) dequantize_q8_kernel(TY* y, long ldy, const int8_t* q, long ldq, const float* scale, int rows, int width, int pieces) {
    constexpr int V = SHIFT ? 8 : 16 / (int)sizeof(TY), GROUPS = 4, STEP = GROUPS * 32 * V;
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const long all = (long)rows * pieces, step = (long)gridDim.x * (blockDim.x >> 5);
    for (long i = (long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); i < all; i += step) {
        const long r = i / pieces;
        const int from = (int)(i - r * pieces) * STEP;
        const int8_t* src = q + r * ldq;
        TY* dst = y + r * ldy;
        const float s = scale[r];
        Pack<int8_t, V> p[GROUPS];
#pragma unroll
        for (int g = 0; g < GROUPS; g++) {
            const int at = from + (g * 32 + lane) * V;
            if (from + g * 32 * V >= width) break;
            if (at + V <= width) {
                if constexpr (V == 8) *reinterpret_cast<uint2*>(p[g].v) = *reinterpret_cast<const uint2*>(src + at);
                else *reinterpret_cast<uint32_t*>(p[g].v) = *reinterpret_cast<const uint32_t*>(src + at);
            } else if (at < width) {
#pragma unroll
                for (int k = 0; k < V; k++) p[g].v[k] = at + k < width ? src[at + k] : (int8_t)0;
            }
        }
#pragma unroll
        for (int g = 0; g < GROUPS; g++) {
            const int at = from + (g * 32 + lane) * V;
            if (from + g * 32 * V >= width) break;          // (the whole warp)
            if constexpr (SHIFT) {
                float v[8];
#pragma unroll
                for (int k = 0; k < 8; k++) v[k] = (float)p[g].v[k] * s;
                store8<true>(dst, at, width, v);
            } else if (at + V <= width) {
                Pack<TY, V> o;
#pragma unroll
                for (int k = 0; k < V; k++) o.v[k] = from_float<TY>((float)p[g].v[k] * s);
                store_pack<TY, V>(dst + at, o);
            } else if (at < width)
                for (int k = 0; k < V; k++) if (at + k < width) dst[at + k] = from_float<TY>((float)p[g].v[k] * s);
        }
    }
}

inline bool whole(const void* p, long ld, int size) { return (uintptr_t)p % 16 == 0 && ld * size % 16 == 0; }

// How a row is shared: groups of 8 entries a thread, a warp or a block a row, threads of a block.  Four groups a thread where there are more rows than two
// blocks an SM, so that what a thread does once a row costs less (8,192 x 14,336 bfloat16 72 us, with two groups 82; 8,192 x 8,192 40, with two 45, with one
// 60); fewer where a row's own way counts (64 x 4,096 1.6 us with one group or two, 1.7 with four; 16 x 14,336 2.2, with four 2.3).  A norm takes one group as
// far as 512 threads go, then two (float32 and bfloat16 added: 8,192 x 4,096 56 us, with two 62; 8,192 x 6,144 84 us, with one 89; 4,000 x 7,169 65, with one
// 103; 8,192 x 8,192 115, with one 110).
struct Share { int ch, threads, blocks; bool warp; };
constexpr int FEW_ROWS = 296;
Share share_of(int rows, int width, bool norm) {
    const int groups = (width + 7) / 8;
    if (groups <= 128) return Share{groups <= 32 ? 1 : groups <= 64 ? 2 : 4, 256, (rows + 7) / 8, true};
    // (a norm's sums are added in an order that the share decides, so its share hangs on the width alone)
    const int ch = !norm && (rows > FEW_ROWS || groups > 2048) ? 4 : groups <= (norm ? 512 : 1024) ? 1 : 2;
    return Share{ch, ((groups + ch - 1) / ch + 31) / 32 * 32, rows, false};
}

template <typename TX, bool SHIFT>
int run_quantize(const Share& s, int8_t* q, long ldq, float* scale, const TX* x, long ldx, int rows, int width, cudaStream_t stream) {
#define HYMT2_RUN(CH, MOST) launch_pdl(quantize_q8_kernel<TX, CH, MOST, SHIFT>, dim3(s.blocks), dim3(s.threads), 0, stream, q, ldq, scale, x, ldx, rows, width)
    if (s.warp) s.ch == 1 ? HYMT2_RUN(1, 256) : s.ch == 2 ? HYMT2_RUN(2, 256) : HYMT2_RUN(4, 256);
    else s.ch == 1 ? HYMT2_RUN(1, 1024) : s.ch == 2 ? HYMT2_RUN(2, 1024) : s.threads <= 512 ? HYMT2_RUN(4, 512) : HYMT2_RUN(4, 1024);
#undef HYMT2_RUN
    return hymt2_check_launch("quantize_q8");
}
template <typename TX, typename TA, typename TG, bool SHIFT>
int run_norm(const Share& s, const NormQ8Params& p, cudaStream_t stream) {
#define HYMT2_RUN(CH, WARP) launch_pdl(rmsnorm_q8_kernel<TX, TA, TG, CH, WARP, SHIFT>, dim3(s.blocks), dim3(s.threads), 0, stream, p)
    if (s.warp) s.ch == 1 ? HYMT2_RUN(1, true) : s.ch == 2 ? HYMT2_RUN(2, true) : HYMT2_RUN(4, true);
    else s.ch == 1 ? HYMT2_RUN(1, false) : HYMT2_RUN(2, false);
#undef HYMT2_RUN
    return hymt2_check_launch("rmsnorm_q8");
}

constexpr int MOST_Q8 = 1 << 28;        // rows, entries of a row: a row's bytes are counted in an int

}  // namespace

HYMT2_API int hymt2_quantize_q8(void* q, long ldq, float* scale, const void* x, int x_dtype, long ldx, int rows, int width, cudaStream_t stream) {
    if (rows == 0) return HYMT2_OK;
    HYMT2_REQUIRE(rows > 0 && rows <= MOST_Q8 && width > 0 && width <= MOST_Q8 && ldq >= width && ldx >= width, "quantize_q8: bad sizes rows=%d width=%d", rows, width);
    HYMT2_REQUIRE((uintptr_t)q % 16 == 0 && ldq % 16 == 0, "quantize_q8: rows of integers must start on 16 bytes");
    HYMT2_DISPATCH_DTYPE(x_dtype, TX, {
        const bool shift = !whole(x, ldx, sizeof(TX));
        if (width > LONGEST_HELD) {
            launch_pdl(shift ? quantize_q8_long_kernel<TX, true> : quantize_q8_long_kernel<TX, false>, dim3(rows), dim3(1024), 0, stream, (int8_t*)q, ldq,
                       scale, (const TX*)x, ldx, width);
            return hymt2_check_launch("quantize_q8");
        }
        const Share s = share_of(rows, width, false);
        if (shift) return run_quantize<TX, true>(s, (int8_t*)q, ldq, scale, (const TX*)x, ldx, rows, width, stream);
        return run_quantize<TX, false>(s, (int8_t*)q, ldq, scale, (const TX*)x, ldx, rows, width, stream);
    });
}

HYMT2_API int hymt2_dequantize_q8(void* y, int y_dtype, long ldy, const void* q, long ldq, const float* scale, int rows, int width, cudaStream_t stream) {
    if (rows == 0) return HYMT2_OK;
    HYMT2_REQUIRE(rows > 0 && rows <= MOST_Q8 && width > 0 && width <= MOST_Q8 && ldq >= width && ldy >= width, "dequantize_q8: bad sizes rows=%d width=%d", rows, width);
    HYMT2_REQUIRE((uintptr_t)q % 16 == 0 && ldq % 16 == 0, "dequantize_q8: rows of integers must start on 16 bytes");
    HYMT2_DISPATCH_DTYPE(y_dtype, TY, {
        const bool shift = !whole(y, ldy, sizeof(TY));
        const int step = shift ? 1024 : 2048 / (int)sizeof(TY), pieces = (width + step - 1) / step;
        const long blocks = ((long)rows * pieces + 7) / 8;
        const dim3 grid((unsigned)(blocks < 148 * 64 ? blocks : 148 * 64));
        launch_pdl(shift ? dequantize_q8_kernel<TY, true> : dequantize_q8_kernel<TY, false>, grid, dim3(256), 0, stream, (TY*)y, ldy, (const int8_t*)q, ldq, scale,
                   rows, width, pieces);
    });
    return hymt2_check_launch("dequantize_q8");
}

// x, add (or null), total (or null; it may be x): [rows, width] with rows ld* entries apart; gain [width].
HYMT2_API int hymt2_rmsnorm_q8(void* q, long ldq, float* scale, const void* x, int x_dtype, long ldx, const void* add, int add_dtype, long ldadd,
                               void* total, long ldt, const void* gain, int gain_dtype, int rows, int width, float eps, cudaStream_t stream) {
    if (rows == 0) return HYMT2_OK;
    HYMT2_REQUIRE(rows > 0 && rows <= MOST_Q8 && width > 0 && width <= MOST_Q8 && ldq >= width && ldx >= width, "rmsnorm_q8: bad sizes rows=%d width=%d", rows, width);
    HYMT2_REQUIRE((uintptr_t)q % 16 == 0 && ldq % 16 == 0, "rmsnorm_q8: rows of integers must start on 16 bytes");
    HYMT2_REQUIRE(!total || add, "rmsnorm_q8: the sums have a place, but nothing is added");
    const NormQ8Params p{(int8_t*)q, scale, x, add, total, gain, ldq, ldx, ldadd, ldt, rows, width, eps};
    HYMT2_DISPATCH_DTYPE(x_dtype, TX, HYMT2_DISPATCH_DTYPE(add_dtype, TA, HYMT2_DISPATCH_DTYPE(gain_dtype, TG, {
        const bool shift = !whole(x, ldx, sizeof(TX)) || (add && !whole(add, ldadd, sizeof(TA))) || (total && !whole(total, ldt, sizeof(TX))) ||
                           (uintptr_t)gain % 16 != 0;
        const Share s = share_of(rows, width, true);
        if (width > LONGEST_NORMED) {
            launch_pdl(shift ? rmsnorm_q8_long_kernel<TX, TA, TG, true> : rmsnorm_q8_long_kernel<TX, TA, TG, false>, dim3(rows), dim3(1024), 0, stream, p);
            return hymt2_check_launch("rmsnorm_q8");
        }
        return shift ? run_norm<TX, TA, TG, true>(s, p, stream) : run_norm<TX, TA, TG, false>(s, p, stream);
    })));
}
