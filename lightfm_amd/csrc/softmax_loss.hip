// softmax_loss.hip -- softmax cross entropy over the whole catalogue with its gradient, without keeping the logits.
//
//   s[n, v] = <x[n], w[v]> + b[v],  lse[n] = log sum_v exp s[n, v],  loss[n] = g[n] (lse[n] - s[n, t[n]])
//   q[n, v] = g[n] (exp(s[n, v] - lse[n]) - [v = t[n]]),  dx = q w,  dw = q^T x,  db[v] = sum_n q[n, v]
//
// Two sweeps over the [rows, vocab] plane, each of which makes the scores in registers on the matrix cores and drops them:
//
//   rows_kernel   a wave owns 32 rows x (in registers) and streams the table through LDS.  dx needs no second look at
//                 the scores: sum_v p w is a mean weighted by the softmax, accumulated beside the running maximum and sum
//                 (rescaled when the maximum grows), so ONE sweep gives lse and dx -- 4 rows vocab d operations.
//   table_kernel  a wave owns 32 rows of the table and streams x; with lse known it forms q and accumulates dw and db.
//
// Both sweeps compute the score tile transposed to what they own: S = streamed tile (rows of the result) x owned rows
// (columns = lanes).  A lane then holds 16 scores of ONE owned row, the softmax statistics stay in the lane (one exchange
// between the two half-waves per tile), and -- the order of the summation index being free -- the lane's 16 values are
// exactly the operand that the second product needs: no trip through LDS.  The streamed tile's other operand shape is
// read with the transposing LDS load (ds_read_b64_tr_b16).
//
// float32 operands: x = 2^-k (hi + lo) with hi, lo in float16 and k from the largest magnitude, a product is hi hi + hi lo +
// lo hi on the float16 matrix pipe.  An operand keeps 22 bits (and a floor of 2^-39 of the largest magnitude), the product
// left out is 2^-22 of the term: the size of float32's own rounding over a sum, at a third of the float16 rate instead of the
// float32 pipe's 1/16.  The probabilities that enter the second product are split the same way.  Those of dw, scaled so that the
// largest weight is 2^14, are off by 2^-38 of it at most, so a probability below 2^-17 or so has fewer bits than float32's; those
// of dx, scaled so that the largest of a row is 2^7 or more, by 2^-32 of that.
// Half-precision operands are multiplied as they are; their probabilities are rounded once to the operands' type, to nearest: at
// most 2^-8 (bfloat16) or 2^-11 (float16) relative, as much as the result's own rounding -- where one term rules a sum the two
// add up.  Of float16's, those below 2^-21 of a row's largest (dx) or 2^-27 of the largest weight (dw) are subnormal: off by
// 2^-32 and 2^-38 of these.  All sums, maxima and statistics are float32.
#include "ops_common.hpp"

#include <math.h>

namespace lfm {
namespace ops {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <typename E> struct Half;
template <> struct Half<bf16_t> { typedef bf16_t x8 __attribute__((ext_vector_type(8))); typedef bf16_t x4 __attribute__((ext_vector_type(4))); };
template <> struct Half<f16_t> { typedef f16_t x8 __attribute__((ext_vector_type(8))); typedef f16_t x4 __attribute__((ext_vector_type(4))); };

__device__ inline f32x16 mfma(Half<bf16_t>::x8 a, Half<bf16_t>::x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ inline f32x16 mfma(Half<f16_t>::x8 a, Half<f16_t>::x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// Four rows of one column: the 16 lanes of a group point at 4 rows x 16 columns (lane i: row i / 4, columns 4 (i % 4) ..),
// lane i receives column i.
template <typename E>
__device__ inline typename Half<E>::x4 read_column(const E *p)
{
    const s16x4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(E *)p);
    return __builtin_bit_cast(typename Half<E>::x4, r);
}

__device__ inline float half_wave_max(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const unsigned low = r[0], high = r[1];
    return fmaxf(__uint_as_float(low), __uint_as_float(high));
}

__device__ inline float half_wave_sum(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const unsigned low = r[0], high = r[1];
    return __uint_as_float(low) + __uint_as_float(high);
}

// in pairs: long sums of these are then as many times shorter
__device__ inline float sum16(const float (&q)[16])
{
    float a[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = q[2 * j] + q[2 * j + 1];
    return ((a[0] + a[1]) + (a[2] + a[3])) + ((a[4] + a[5]) + (a[6] + a[7]));
}

__device__ inline float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
// probabilities enter rows_kernel's second product as 2^7 p: with the maximum up to 8 binades behind they reach 2^15,
// and what float16 cannot hold below is 2^-32 of the largest
constexpr float P_SHIFT = 7.0f, LAG = 8.0f;
// exp2(s c - m c) as one multiply-add is off by the rounding of m c: with |m c| up to this, as much as s itself
constexpr float FAR = 512.0f;
constexpr int K_MOST = 60;  // see Scales
constexpr int MAX_PARTS = 512;  // of an operand in largest_kernel (128: 24380 x 169 float32 takes 100 us instead of 82)

// Powers of two that bring the operands into float16's range (all 0 for half-precision operands).
struct Scales {
    int kx, kw;   // x 2^kx, w 2^kw are what the products see
    int eg;       // 2^eg >= the largest |g|
    int pad;
};

struct Derived {
    float c;      // matrix units -> base-2 logarithms
    int k;        // score = matrix units * 2^-k
    float owned;  // factor of the owned operand
    float low;    // stands for "lowest score" in matrix units: c * low is finite
};

// The bias enters the products in matrix units, b 2^k, which has to stay finite: where kx + kw > K_MOST the scores are
// below 2^-20 and the owned operand of the first product (not the streamed one, which the second product needs at full
// size) gives up the difference.
__device__ inline Derived derive(const Scales *s)
{
    const int k = s ? s->kx + s->kw : 0;
    Derived d;
    d.k = k > K_MOST ? K_MOST : k;
    d.owned = k > K_MOST ? ldexpf(1.0f, K_MOST - k) : 1.0f;
    d.c = ldexpf(LOG2E, -d.k);
    d.low = -3.3e38f / fmaxf(d.c, 1.0f);
    return d;
}

// A row without a target that does not fit x's scale has one of its own: `code` = OWN_SCALE + k, the score being matrix units 2^-k,
// and no factor.  Beside 0, x's scale, it can be NOT_FINITE: then the row's scores are not wanted.  Loss of 4096 rows x 20011 x 64,
// a third of them such rows: 88 us, without any 63 (scored one by one in the join: 6100).
constexpr int16_t OWN_SCALE = 1024, NOT_FINITE = 0x7fff;

__device__ inline bool has_own_scale(int16_t code) { return code != 0 && code != NOT_FINITE; }

__device__ inline Derived derived_from(float c)
{
    int e;
    frexpf(c, &e);  // c = LOG2E 2^-k
    return {c, 1 - e, 1.0f, -3.3e38f / fmaxf(c, 1.0f)};
}

__device__ inline Derived derive_row(const Derived &all, int16_t code)
{
    return has_own_scale(code) ? derived_from(ldexpf(LOG2E, OWN_SCALE - code)) : all;
}

__device__ inline float bias_units(float b, const Derived &d)
{
    return fabsf(b) < INFINITY ? fminf(fmaxf(ldexpf(b, d.k), d.low), -d.low) : b;
}

// An item whose bias is -inf is not there: its row is not looked at, whatever it holds.
__device__ inline bool removed(const float *bias, int64_t v) { return bias && bias[v] == -INFINITY; }

__device__ inline int64_t target_of(const lfm_softmax_args &a, int64_t n)
{
    const int64_t t = a.id_bytes == 8 ? ((const int64_t *)a.targets)[n] : (int64_t)((const int32_t *)a.targets)[n];
    return (uint64_t)t < (uint64_t)a.vocab ? t : -1;
}

// -------------------------------------------------------------- operands ---

// Largest finite magnitudes: `parts` blocks for x (rows with a target, and behind the others' the rows without one; all rows'
// codes are cleared on the way), as many for w (float32 operands alone), as many for g.  Threads take four columns of a row each,
// LOAD (4, 2, 1) of them at once.
template <typename T, int LOAD>
__global__ __launch_bounds__(256) void largest_kernel(lfm_softmax_args a, int parts, float *largest, int tensors, int16_t *codes)
{
    const int which = blockIdx.x / parts, part = blockIdx.x % parts;
    float m = 0.0f, rest = 0.0f;  // rest: rows of x without a target
    if (which < 2 && tensors == 3) {
        const T *p = (const T *)(which ? a.table : a.hidden);
        const int64_t rows = which ? a.vocab : a.rows, stride = which ? a.table_stride : a.hidden_stride;
        const int groups = (a.d + 3) / 4, per = 256 / groups, tr = (int)threadIdx.x / groups, c = ((int)threadIdx.x - tr * groups) * 4;
        auto look = [&](float v, bool counts) {
            const float s = fabsf(v) < INFINITY ? fabsf(v) : 0.0f;
            m = fmaxf(m, counts ? s : 0.0f);
            rest = fmaxf(rest, counts ? 0.0f : s);
        };
        const int64_t step = (int64_t)parts * per;
        if (tr < per)
#pragma unroll 4
            for (int64_t r = (int64_t)part * per + tr; r < rows; r += step) {
                bool counts = true;
                if (!which) {
                    if (c == 0) codes[r] = 0;
                    counts = target_of(a, r) >= 0;
                } else if (removed(a.bias, r))
                    continue;
                const T *q = p + r * stride + c;
#pragma unroll
                for (int j = 0; j < 4; j += LOAD) {
                    if (c + j >= a.d) break;
                    const Vec<T, LOAD> v = *(const Vec<T, LOAD> *)(q + j);
#pragma unroll
                    for (int i = 0; i < LOAD; ++i) look((float)v.v[i], counts);
                }
            }
    } else {
        for (int64_t i = (int64_t)part * 256 + threadIdx.x; i < a.rows; i += (int64_t)parts * 256) {
            if (target_of(a, i) < 0) continue;
            const float v = a.weights ? fabsf(a.weights[i]) : 1.0f;
            if (v < INFINITY) m = fmaxf(m, v);
        }
    }
    for (int o = 32; o; o >>= 1) {
        m = fmaxf(m, __shfl_xor(m, o));
        rest = fmaxf(rest, __shfl_xor(rest, o));
    }
    __shared__ float s[2][4];
    if ((threadIdx.x & 63) == 0) {
        s[0][threadIdx.x >> 6] = m;
        s[1][threadIdx.x >> 6] = rest;
    }
    __syncthreads();
    const int i = threadIdx.x;
    if (i == 0 || (i == 1 && which == 0 && tensors == 3))
        largest[i ? tensors * parts + part : (int)blockIdx.x] = fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3]));
}

// k with max 2^k in [2^13, 2^14); 0 for an empty or all-zero operand
__device__ inline int exponent_for(float largest)
{
    if (!(largest > 0.0f)) return 0;
    int e;
    frexpf(largest, &e);  // largest in [2^(e-1), 2^e)
    return 14 - e;
}

struct PackArgs {
    lfm_softmax_args a;
    const float *largest;  // parts values for x, w, g and x's rows without a target (or for g alone), or NULL: no scales are wanted
    int parts, tensors;
    Scales *scales;
    void *x, *w;           // packed, NULL: that operand is used where it is
    int16_t *codes;        // [rows], see OWN_SCALE
};

// The scale of a row without a target that is far larger than the rows with one: every thread of the row reads the whole row
// (from the caches), so that such rows need no pass of their own and cost the others nothing.
template <typename T, int LOAD>
__device__ inline int16_t own_scale(const T *row, int d, int kx, int kw, int &k)
{
    float m = 0.0f;
    bool finite = true;
    for (int c = 0; c < d; c += LOAD) {
        const Vec<T, LOAD> v = *(const Vec<T, LOAD> *)(row + c);
#pragma unroll
        for (int i = 0; i < LOAD; ++i) {
            const float s = fabsf((float)v.v[i]);
            finite &= s < INFINITY;
            m = fmaxf(m, s);
        }
    }
    const int kr = exponent_for(m);
    if (!finite || !(m > 0.0f) || kr >= kx - 1) return 0;  // (up to twice x's largest still fits)
    k = kr + kw > K_MOST ? K_MOST - kw : kr;
    return (int16_t)(OWN_SCALE + k + kw);
}

// Rows of x and w to the padded, split form, zeros behind d: per row and chunk of `width` columns [hi: width | lo: width]
// (width = dp up to 256 columns, 256 beyond).  A thread makes 8 elements and reads LOAD (4, 2, 1) of them at once.
template <typename T, typename E, int NS, int LOAD>
__global__ __launch_bounds__(256) void pack_kernel(PackArgs p, int dp, int width)
{
    __shared__ float ms[4];
    int kx = 0, kw = 0;
    bool large = false;  // a row without a target does not fit x's scale
    if (p.largest) {
        const int which = threadIdx.x >> 6, lane = threadIdx.x & 63;
        float m = 0.0f;
        if (p.tensors == 3 || which == 2)
            for (int i = lane; i < p.parts; i += 64) m = fmaxf(m, p.largest[(p.tensors == 3 ? which : 0) * p.parts + i]);
        for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        if (lane == 0) ms[which] = m;
        __syncthreads();
        // the rows with a target set x's scale; where none holds anything, the others do
        kx = exponent_for(ms[0] > 0.0f ? ms[0] : ms[3]);
        kw = exponent_for(ms[1]);
        large = !(ldexpf(ms[3], kx) < 65504.0f);
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            Scales s = {kx, kw, ms[2] > 0.0f ? 14 - exponent_for(ms[2]) : 0, 0};
            *p.scales = s;
        }
    }
    typedef typename Half<E>::x8 x8;
    const int chunks = dp / 8, per = 256 / chunks, tr = (int)threadIdx.x / chunks, c = ((int)threadIdx.x - tr * chunks) * 8;
    const int64_t xr = p.x ? p.a.rows : 0, n = xr + (p.w ? p.a.vocab : 0);
    const int at = (c / width) * (NS * width) + c % width;
    if (tr >= per) return;
    for (int64_t i = (int64_t)blockIdx.x * per + tr; i < n; i += (int64_t)gridDim.x * per) {
        const bool is_x = i < xr;
        const int64_t r = is_x ? i : i - xr;
        const T *src = is_x ? (const T *)p.a.hidden + r * p.a.hidden_stride : (const T *)p.a.table + r * p.a.table_stride;
        E *dst = (E *)(is_x ? p.x : p.w) + r * (NS * dp) + at;
        const bool gone = !is_x && removed(p.a.bias, r);
        T v[8];
#pragma unroll
        for (int q = 0; q < 8; q += LOAD) {
            Vec<T, LOAD> part = {};
            if (!gone && c + q < p.a.d) part = *(const Vec<T, LOAD> *)(src + c + q);
#pragma unroll
            for (int j = 0; j < LOAD; ++j) v[q + j] = part.v[j];
        }
        x8 hi, lo;
        if (NS == 1) {
#pragma unroll
            for (int j = 0; j < 8; ++j) hi[j] = (E)v[j];
        } else {
            int k = is_x ? kx : kw;
            if (large && is_x && target_of(p.a, r) < 0) {
                const int16_t code = own_scale<T, LOAD>(src, p.a.d, kx, kw, k);
                if (code && c == 0) p.codes[r] = code;
            }
            bool fits = true;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float f = ldexpf((float)v[j], k);
                if (is_x && !(fabsf(f) < 65504.0f)) { fits = false; f = 0.0f; }
                hi[j] = (E)f;
                lo[j] = (E)(f - (float)hi[j]);
            }
            if (is_x && !fits) p.codes[r] = NOT_FINITE;
            *(x8 *)(dst + width) = lo;
        }
        *(x8 *)dst = hi;
    }
}

// ------------------------------------------------------------- the sweeps ---

// Streams rows of NS DP halves into LDS, BV at a time, double-buffered through registers: the loads of the next tile are in
// flight while this one is used.
// LDS has 64 banks and serves the 16-byte reads of 16 lanes, or the 8-byte reads of 32, at once.  The products read a tile
// in two ways: 16 bytes of 16 neighbouring rows, and (transposing) 64 bytes of 4 neighbouring rows.  Both are free of
// conflicts when a row takes NS DP + 8 halves (4 banks more than a multiple of 64, times an odd number) and the rows of a
// group of 16 are stored transposed as a 4 x 4 square: neighbours then lie 16 banks apart, and all 16 rows 4 banks apart.
__host__ __device__ constexpr int slot_of(int r) { return (r & ~15) | ((r & 3) << 2) | ((r >> 2) & 3); }

template <typename E, int NS, int DP>
struct Tile {
    static constexpr int BV = NS * DP <= 128 ? 64 : 32, ROW = NS * DP + 8, CHUNKS = NS * DP / 8, PER = BV * CHUNKS / 256;
    static constexpr int SIZE = BV * ROW;
    uint4 held[PER];

    __device__ static inline int row_of(int q) { return (q * 256 + (int)threadIdx.x) / CHUNKS; }
    // the tile's first row is row0 < rows; rows behind the last are zeros
    __device__ inline void fetch(const E *p, int64_t ld, int64_t row0, int64_t rows)
    {
        const E *base = p + row0 * ld;  // the same for all lanes
        const uint32_t ld32 = (uint32_t)ld;
        if (row0 + BV <= rows) {
#pragma unroll
            for (int q = 0; q < PER; ++q) held[q] = *(const uint4 *)(base + ((uint32_t)row_of(q) * ld32 + (uint32_t)((q * 256 + threadIdx.x) % CHUNKS) * 8u));
        } else {
#pragma unroll
            for (int q = 0; q < PER; ++q) {
                held[q] = make_uint4(0, 0, 0, 0);
                if (row0 + row_of(q) < rows) held[q] = *(const uint4 *)(base + ((uint32_t)row_of(q) * ld32 + (uint32_t)((q * 256 + threadIdx.x) % CHUNKS) * 8u));
            }
        }
    }
    __device__ inline void store(E *tile) const
    {
#pragma unroll
        for (int q = 0; q < PER; ++q) *(uint4 *)(tile + slot_of(row_of(q)) * ROW + (q * 256 + (int)threadIdx.x) % CHUNKS * 8) = held[q];
    }
};

template <typename E, int NS, int DP>
__device__ inline void load_owned(typename Half<E>::x8 (&f)[NS][DP / 16], const E *p, int64_t ld, int64_t row, int64_t rows, float factor)
{
    typedef typename Half<E>::x8 x8;
    const bool there = row < rows;
    const E *q = p + (there ? row : 0) * ld + ((threadIdx.x & 63) >> 5) * 8;
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) f[s][k] = there ? *(const x8 *)(q + s * DP + k * 16) : (x8)((E)0.0f);
    if (NS == 2 && factor != 1.0f) {  // (a power of two that float16 need not hold: what vanishes does not show in a score)
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) f[s][k] *= (E)factor;
    }
}

// The two shapes in which a block of 32 streamed rows (from row r0 of the tile) enters the products.
template <typename E, int NS, int DP>
struct ScoreOperand {  // rows of the block: lane = row, 8 columns at a time
    typename Half<E>::x8 v[NS][DP / 16];

    __device__ inline void read(const E *tile, int r0)
    {
        const int lane = threadIdx.x & 63;
        const E *p = tile + (r0 + slot_of(lane & 31)) * Tile<E, NS, DP>::ROW + (lane >> 5) * 8;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) v[s][k] = *(const typename Half<E>::x8 *)(p + s * DP + k * 16);
    }
};

template <typename E, int NS, int DP>
struct SumOperand {  // columns of the block: lane = column, the rows in the order in which a lane holds its scores
    typename Half<E>::x8 v[NS][2][DP / 32];

    __device__ inline void read(const E *tile, int r0)
    {
        typedef typename Half<E>::x4 x4;
        constexpr int ROW = Tile<E, NS, DP>::ROW;
        const int lane = threadIdx.x & 63;
        // rows 8 e + 4 (lane / 32) + 0 .. 3 of a group of 16, e = 0, 1
        const E *p = tile + (r0 + (lane >> 5) + ((lane & 15) >> 2) * 4) * ROW + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int b = 0; b < DP / 32; ++b) {
                    const x4 lo = read_column(p + s * DP + k * 16 * ROW + b * 32), hi = read_column(p + s * DP + (k * 16 + 2) * ROW + b * 32);
                    v[s][k][b] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                }
    }
};

// acc += block x owned rows
template <typename E, int NS, int DP>
__device__ inline void scores(f32x16 &acc, const typename Half<E>::x8 (&own)[NS][DP / 16], const ScoreOperand<E, NS, DP> &a)
{
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
        acc = mfma(a.v[0][k], own[0][k], acc);
        if (NS == 2) {
            acc = mfma(a.v[NS - 1][k], own[0][k], acc);
            acc = mfma(a.v[0][k], own[NS - 1][k], acc);
        }
    }
}

// Eight float32 values to a matrix operand: rounded to nearest (bf16, f16), or split into two float16 (hi towards zero, two
// values per instruction; the remainder is exact and keeps 11 bits more, to nearest).
__device__ inline Half<bf16_t>::x8 round_values(const float (&v)[8], Half<bf16_t>::x8)
{
    Half<bf16_t>::x8 r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (bf16_t)v[j];
    return r;
}

__device__ inline Half<f16_t>::x8 round_values(const float (&v)[8], Half<f16_t>::x8)
{
    Half<f16_t>::x8 r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (f16_t)v[j];
    return r;
}

__device__ inline Half<f16_t>::x8 cut_values(const float (&v)[8])
{
    typedef __fp16 fp16x2 __attribute__((ext_vector_type(2)));
    union { fp16x2 p[4]; Half<f16_t>::x8 r; } u;
#pragma unroll
    for (int j = 0; j < 4; ++j) u.p[j] = __builtin_amdgcn_cvt_pkrtz(v[2 * j], v[2 * j + 1]);
    return u.r;
}

template <typename E, int NS>
struct Values {  // the probabilities of 32 streamed rows as matrix operands
    typename Half<E>::x8 v[NS][2];

    __device__ inline void pack(const float (&q)[16])
    {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float part[8], rest[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) part[j] = q[8 * k + j];
            if constexpr (NS == 2) {
                v[0][k] = cut_values(part);
#pragma unroll
                for (int j = 0; j < 8; ++j) rest[j] = __builtin_fmaf((float)v[0][k][j], -1.0f, part[j]);
                v[NS - 1][k] = round_values(rest, typename Half<E>::x8());
            } else
                v[0][k] = round_values(part, typename Half<E>::x8());
        }
    }
};

// out[d, owned] += block^T x values
template <typename E, int NS, int DP>
__device__ inline void accumulate(f32x16 (&out)[DP / 32], const Values<E, NS> &p, const SumOperand<E, NS, DP> &a)
{
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int b = 0; b < DP / 32; ++b) {
            out[b] = mfma(a.v[0][k][b], p.v[0][k], out[b]);
            if (NS == 2) {
                out[b] = mfma(a.v[NS - 1][k][b], p.v[0][k], out[b]);
                out[b] = mfma(a.v[0][k][b], p.v[NS - 1][k], out[b]);
            }
        }
}

// The plane of (owned rows, streamed tiles) is cut into as many equal pieces as blocks fit on the card, whatever the sizes: a
// block takes `tiles` consecutive tiles, the last of one owner and the first of the next among them.
struct Pieces {
    uint32_t owners, tiles, blocks;  // owners * tiles units, dealt to `blocks` blocks

    __host__ __device__ inline uint64_t begin(uint32_t block) const
    {
        const uint64_t units = (uint64_t)owners * tiles;
        if ((units * (blocks + 1)) >> 32 == 0) return (uint32_t)(units * block) / blocks;
        return units * block / blocks;
    }
    __host__ __device__ inline uint32_t block_of(uint64_t unit) const
    {
        const uint64_t units = (uint64_t)owners * tiles, at = (unit + 1) * blocks - 1;
        if ((units * blocks) >> 32 == 0) return (uint32_t)at / (uint32_t)units;  // (a 64-bit division takes microseconds)
        return (uint32_t)(at / units);
    }
    __host__ __device__ inline uint32_t owner_of(uint64_t unit) const
    {
        return unit >> 32 == 0 ? (uint32_t)unit / tiles : (uint32_t)(unit / tiles);
    }
    __host__ __device__ inline uint32_t first_block(uint32_t owner) const { return block_of((uint64_t)owner * tiles); }
    __host__ __device__ inline uint32_t last_block(uint32_t owner) const { return block_of((uint64_t)owner * tiles + tiles - 1); }
    // most blocks that one owner is spread over
    __host__ __device__ inline uint32_t most() const { return (blocks + owners - 1) / owners + 1; }
};

struct SweepArgs {
    const void *x, *w;      // packed or in place
    int64_t ldx, ldw;       // halves per row
    int64_t rows, vocab;
    const float *bias;
    const Scales *scales;
    const int16_t *codes;   // rows_kernel, NS == 2: see OWN_SCALE
    const void *targets;    // rows_kernel: [rows], id_bytes wide
    int id_bytes;
    Pieces pieces;
    int d, dp;
    int chunks;             // of 256 columns (WIDE; else 1): the second product's columns are blockIdx.y's
    // rows_kernel: per chunk, part and row, the row's target left out (the parts of a row are the blocks of its owner)
    float *pm, *pl, *po;    // maximum (matrix units), sum of 2^7 p; per part and row: sum of 2^7 p w [dp]
    int parts;
    // table_kernel: per row
    const float *row_max, *row_rate, *row_weight;  // maximum (matrix units; +inf: no target), 2^shift g / sum, 2^shift g (1 - p[target])
    const int32_t *row_target;
    void *dw;               // table rows that one block has to itself
    float *db, *pw, *pb;    // the others': per block its first and its last owner, [128][dp], [128]
    int aligned;            // rows of dw can be written four elements at a time
    int shifted;            // q is scaled by 2^(14 - eg): 0 no (bfloat16), 1 with eg = 0, 2 with eg of scales
};

// WIDE: more than 256 columns, taken 256 at a time.  The scores add up over the chunks (the owned operand is read again for
// each, from the caches); a block accumulates the second product of one chunk, blockIdx.y's, which it streams last.  The
// scores' work is repeated for every chunk of the result, and the owned operand read again for every tile: gradients of 8192 x 26744
// x 512 take 11.8 ms in float32 and 6.0 in bfloat16, where 256 columns take 3.6 and 0.86.
template <typename E, int NS, int DP, bool WIDE>
struct Stream {
    typedef Tile<E, NS, DP> Tl;
    static constexpr int BLOCKS = Tl::BV / 32;
    int chunks, first;
    __device__ inline explicit Stream(int chunks_) : chunks(WIDE ? chunks_ : 1), first(WIDE ? (int)blockIdx.y + 1 : 0) {}
    __device__ inline int offset(int j) const { return WIDE ? ((first + j) % chunks) * (NS * DP) : 0; }  // of the j-th chunk
};

// Registers that a block's operands take: the owned rows and the scores' operand ns dp / 4 each, with the sums their operand as many
// and the result dp / 2.
constexpr int registers_for(int ns, int dp, bool sums) { return ns * dp / 2 + (sums ? ns * dp / 4 + dp / 2 : 0); }

// Two waves per SIMD while that leaves room for them, one beyond.  With the sums 192 (float32 x 96) fits 256 registers, up to 9
// of them spilled; at 240 (half precision x 192) the sweeps spilled 39 and 75 as two waves, and one is as fast where the sweeps
// are long and faster where they are not (gradients, bfloat16, two waves and one, us: 8192 x 26744 x 192 740 and 747, 2048 x 26744 x
// 192 239 and 226, 1003 x 50021 x 136 232 and 221, 512 x 200003 x 192 418 and 401, 300 x 3000 x 192 51 and 43).  Without the sums
// more than two would fit at small widths.  float32 beyond 128 columns does not fit one wave either: the rows' sweep spills 16, 312
// and 68 registers at 192, 256 and more columns.
constexpr int waves_for(int ns, int dp, bool sums) { return registers_for(ns, dp, sums) > (sums ? 200 : 128) ? 1 : 2; }

// A wave's 32 rows x 32 columns of a result on their way to memory: the products leave a lane 4 neighbouring columns of its row,
// which written as they are make 16-byte pieces (2-byte ones where rows are not aligned); by way of LDS a row's 32 columns
// are written by neighbouring lanes.
struct Strip {
    float v[32][36];

    __device__ inline void write(const f32x16 &out)
    {
        const int lane = threadIdx.x & 63;
        settle();  // (what was read before)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *(float4 *)&v[lane & 31][8 * g + 4 * (lane >> 5)] = make_float4(out[4 * g], out[4 * g + 1], out[4 * g + 2], out[4 * g + 3]);
        settle();
    }
    // the order of a wave's own accesses
    __device__ static inline void settle() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }
    __device__ static inline int row4(int i) { return i * 8 + ((threadIdx.x & 63) >> 3); }
    __device__ static inline int column4() { return (threadIdx.x & 7) * 4; }
    __device__ inline float4 read4(int i) const { return *(const float4 *)&v[row4(i)][column4()]; }
};

// Bound by the matrix pipe and the exponentials together: a block of 32 x 32 scores costs 4 DP matrix cycles per product and
// about as many for its 16 exponentials, maxima, sums and roundings at DP = 128, which overlap only across the two waves of a
// SIMD (one wave: 1.5 times the time; three: the operands spill).  8192 x 200003 x 128 bfloat16: 0.96 ms with the gradient,
// 880 TFLOP/s, where a product of 8192^3 by the library reaches 1137; 8192 x 26744 x 64 float32: 0.20 ms (280 TFLOP/s, each of
// them three float16 products; the float32 pipe reaches 150).
template <typename E, int NS, int DP, bool GRAD, bool WIDE>
__global__ __launch_bounds__(256, WIDE ? 1 : waves_for(NS, DP, GRAD)) void rows_kernel(SweepArgs a)
{
    typedef Tile<E, NS, DP> Tl;
    typedef Stream<E, NS, DP, WIDE> St;
    static_assert(!WIDE || St::BLOCKS == 1, "a chunk per tile");
    __shared__ __attribute__((aligned(16))) E tile[2][Tl::SIZE];
    __shared__ __attribute__((aligned(16))) float sb[2][Tl::BV];
    __shared__ __attribute__((aligned(16))) float raw[2][NS == 2 ? Tl::BV : 4];  // the biases themselves
    __shared__ uint64_t gone[2];  // removed items of a tile
    __shared__ __attribute__((aligned(16))) Strip strips[GRAD ? 4 : 1];
    const Derived all = derive(NS == 2 ? a.scales : nullptr);
    const St sm(a.chunks);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    uint64_t unit = a.pieces.begin(blockIdx.x);
    const uint64_t end = a.pieces.begin(blockIdx.x + 1);
    while (unit < end) {
        const uint32_t owner = a.pieces.owner_of(unit), t0 = (uint32_t)(unit - (uint64_t)owner * a.pieces.tiles);
        const uint64_t left = end - unit;
        const int nt = (int)(a.pieces.tiles - t0 < left ? a.pieces.tiles - t0 : left);
        unit += nt;
        const int64_t n = (int64_t)owner * 128 + wave * 32 + (lane & 31);
        const Derived dv = NS == 2 ? derive_row(all, n < a.rows ? a.codes[n] : (int16_t)0) : all;
        const bool other_units = NS == 2 && __any(dv.c != all.c);
        typename Half<E>::x8 own[NS][DP / 16];
        if (!WIDE) load_owned<E, NS, DP>(own, (const E *)a.x, a.ldx, n, a.rows, dv.owned);
        const int64_t at = n >= a.rows ? -1 : a.id_bytes == 8 ? ((const int64_t *)a.targets)[n] : (int64_t)((const int32_t *)a.targets)[n];
        const uint32_t target = (uint64_t)at < (uint64_t)a.vocab ? (uint32_t)at : 0xc0000000u;  // (no row of the table)
        f32x16 out[DP / 32];
        float m = dv.low * 1.01f, l = 0.0f;
        if (GRAD)
#pragma unroll
            for (int b = 0; b < DP / 32; ++b) out[b] = (f32x16)(0.0f);

        Tl t;
        float next_bias = 0.0f, next_raw = 0.0f;
        bool next_gone = false;
        auto fetch = [&](int i, int j) {
            const int64_t r = (int64_t)(t0 + i) * Tl::BV, v = r + threadIdx.x;
            t.fetch((const E *)a.w + sm.offset(j), a.ldw, r, a.vocab);
            if (j == 0 && threadIdx.x < Tl::BV) {
                next_raw = v >= a.vocab ? -INFINITY : a.bias ? a.bias[v] : 0.0f;
                next_bias = bias_units(next_raw, all);
                next_gone = v < a.vocab && next_bias == -INFINITY;
            }
        };
        auto store = [&](int i, int j, int buf) {
            t.store(tile[buf]);
            if (j == 0 && threadIdx.x < Tl::BV) {
                sb[i & 1][threadIdx.x] = next_bias;
                if (NS == 2) raw[i & 1][threadIdx.x] = next_raw;
                const uint64_t mask = __ballot(next_gone);
                if (threadIdx.x == 0) gone[i & 1] = mask;
            }
        };
        // the rows of removed items, where the tile has any (split operands: pack_kernel has seen to it)
        auto clear_removed = [&](int i, int buf) {
            if (NS == 2) return;
            const uint64_t mask = gone[i & 1];
            if (mask == 0) return;
#pragma unroll
            for (int q = 0; q < Tl::PER; ++q)
                if ((mask >> Tl::row_of(q)) & 1u) *(uint4 *)(tile[buf] + slot_of(Tl::row_of(q)) * Tl::ROW + (q * 256 + (int)threadIdx.x) % Tl::CHUNKS * 8) = make_uint4(0, 0, 0, 0);
            __syncthreads();
        };
        __syncthreads();  // (the owner before is done with the tiles)
        fetch(0, 0);
        store(0, 0, 0);
        __syncthreads();
        clear_removed(0, 0);
        int buf = 0;
        for (int i = 0; i < nt; ++i) {
            if (!WIDE && i + 1 < nt) fetch(i + 1, 0);
#pragma unroll
            for (int blk = 0; blk < St::BLOCKS; ++blk) {
                ScoreOperand<E, NS, DP> so;
                SumOperand<E, NS, DP> to;
                f32x16 s;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const float4 b = *(const float4 *)&sb[i & 1][blk * 32 + 8 * g + 4 * h];
                    s[4 * g + 0] = b.x;
                    s[4 * g + 1] = b.y;
                    s[4 * g + 2] = b.z;
                    s[4 * g + 3] = b.w;
                }
                if (other_units) {  // a wave in some; what it needs is made here, not kept in registers
                    float c = dv.c;
                    asm volatile("" : "+v"(c));
                    const Derived units = derived_from(c);
#pragma unroll
                    for (int j = 0; j < 16; ++j) s[j] = bias_units(raw[i & 1][blk * 32 + 8 * (j / 4) + 4 * h + j % 4], units);
                }
                if (WIDE) {
                    for (int j = 0; j < sm.chunks; ++j) {
                        load_owned<E, NS, DP>(own, (const E *)a.x + sm.offset(j), a.ldx, n, a.rows, dv.owned);
                        const bool last = j + 1 == sm.chunks;
                        if (!last || i + 1 < nt) fetch(last ? i + 1 : i, last ? 0 : j + 1);
                        so.read(tile[buf], 0);
                        scores<E, NS, DP>(s, own, so);
                        if (last) break;
                        store(i, j + 1, buf ^ 1);
                        __syncthreads();
                        buf ^= 1;
                        clear_removed(i, buf);
                    }
                    if (GRAD) to.read(tile[buf], 0);
                } else {
                    so.read(tile[buf], blk * 32);
                    scores<E, NS, DP>(s, own, so);
                    if (GRAD) to.read(tile[buf], blk * 32);
                }
                // the target's own score is left to the join, in float32: what remains is not a difference of near-equals
                const uint32_t hit = target - ((t0 + i) * (uint32_t)Tl::BV + blk * 32u);
                if (__any(hit < 32u)) {  // one block in some
#pragma unroll
                    for (int j = 0; j < 16; ++j) s[j] = hit == 8u * (j / 4) + 4u * h + j % 4 ? -INFINITY : s[j];
                }
                float mx = s[0];
#pragma unroll
                for (int j = 1; j < 16; ++j) mx = fmaxf(mx, s[j]);
                mx = half_wave_max(mx);
                const bool grows = (mx - m) * dv.c > LAG;
                if (__any(grows)) {  // seldom after the first blocks; by row, so that no row's bits depend on its neighbours
                    const float up = grows ? mx : m, f = exp2_fast((m - up) * dv.c);
                    m = up;
                    l *= f;
                    if (GRAD)
#pragma unroll
                        for (int b = 0; b < DP / 32; ++b) out[b] *= f;
                }
                float base = P_SHIFT - m * dv.c;
                const bool far = fabsf(m * dv.c) > FAR;
                if (__any(far)) {  // the rounding of m c would show: subtract first
                    s -= far ? m : 0.0f;
                    base = far ? P_SHIFT : base;
                }
                float q[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) q[j] = exp2_fast(__builtin_fmaf(s[j], dv.c, base));
                l += sum16(q);
                if (GRAD) {
                    Values<E, NS> p;
                    p.pack(q);
                    accumulate<E, NS, DP>(out, p, to);
                }
            }
            if (i + 1 < nt) store(i + 1, 0, buf ^ 1);
            __syncthreads();
            buf ^= 1;
            if (i + 1 < nt) clear_removed(i + 1, buf);
        }
        const float sum = half_wave_sum(l);
        const int64_t part = (int64_t)(blockIdx.x - a.pieces.first_block(owner)) * a.rows;
        if (h == 0 && n < a.rows) {
            const int64_t to = part + n + (WIDE ? (int64_t)blockIdx.y * a.parts * a.rows : 0);
            a.pm[to] = m;
            a.pl[to] = sum;
        }
        if (GRAD)
#pragma unroll
            for (int b = 0; b < DP / 32; ++b) {
                Strip *strip = &strips[wave];
                strip->write(out[b]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int64_t r = (int64_t)owner * 128 + wave * 32 + strip->row4(i);
                    if (r < a.rows) *(float4 *)(a.po + (part + r) * a.dp + (WIDE ? (int)blockIdx.y * DP : 0) + b * 32 + strip->column4()) = strip->read4(i);
                }
            }
    }
}

// What table_kernel needs to know of the rows of a tile
template <int BV>
struct RowFacts {
    float m[BV];        // -maximum in base 2 (0 where FAR is about the row)
    float rate[BV];     // 2^shift g / sum
    float weight[BV];   // 2^shift g (1 - p[target])
    float far[BV];      // the maximum in matrix units where FAR is about the row, else 0
    int32_t target[BV];
};

// Bound like rows_kernel, with more to do per score: maximum, rate and target of a score's row come from LDS.  8192 x 200003 x
// 128 bfloat16: 1.13 ms, 740 TFLOP/s; 8192 x 26744 x 64 float32: 0.23 ms.
// ONE: all rows are one tile, which stays in LDS over the owners: few rows, and what counts is how the table is read and dw written
// (whole calls in us, the general form and this one: 2 x 178913 x 98 bfloat16 110 and 78, 24 x 211856 x 65 float16 100 and 76, 1 x
// 24380 x 169 float32 77 and 68).  With more tiles the detour by LDS costs registers in the sweep and gains nothing.
template <typename T, typename E, int NS, int DP, bool WIDE, bool ONE>
__global__ __launch_bounds__(256, WIDE ? 1 : waves_for(NS, DP, true)) void table_kernel(SweepArgs a)
{
    typedef Tile<E, NS, DP> Tl;
    typedef Stream<E, NS, DP, WIDE> St;
    static_assert(!WIDE || (St::BLOCKS == 1 && !ONE), "a chunk per tile");
    __shared__ __attribute__((aligned(16))) E tile[ONE ? 1 : 2][Tl::SIZE];
    __shared__ __attribute__((aligned(16))) RowFacts<Tl::BV> facts[ONE ? 1 : 2];
    __shared__ __attribute__((aligned(16))) Strip strips[ONE ? 4 : 1];
    const Derived dv = derive(NS == 2 ? a.scales : nullptr);
    const St sm(a.chunks);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int shift = a.shifted == 2 ? a.scales->eg - 14 : a.shifted ? -14 : 0, kx = NS == 2 ? a.scales->kx : 0;
    const int c0 = WIDE ? (int)blockIdx.y * DP : 0;
    const uint64_t begin = a.pieces.begin(blockIdx.x), end = a.pieces.begin(blockIdx.x + 1);
    uint64_t unit = begin;
    while (unit < end) {
        const uint32_t owner = a.pieces.owner_of(unit), t0 = (uint32_t)(unit - (uint64_t)owner * a.pieces.tiles);
        const uint64_t left = end - unit;
        const int nt = (int)(a.pieces.tiles - t0 < left ? a.pieces.tiles - t0 : left);
        unit += nt;
        const int32_t w0 = (int32_t)(owner * 128 + wave * 32);
        const int64_t v = (int64_t)w0 + (lane & 31);
        typename Half<E>::x8 own[NS][DP / 16];
        const float bias = a.bias && v < a.vocab ? bias_units(a.bias[v], dv) : 0.0f;
        const int64_t have = NS == 1 && bias == -INFINITY ? 0 : a.vocab;  // a removed item's row: zeros
        if (!WIDE) load_owned<E, NS, DP>(own, (const E *)a.w, a.ldw, v, have, dv.owned);
        float db = 0.0f;
        f32x16 out[DP / 32];
#pragma unroll
        for (int b = 0; b < DP / 32; ++b) out[b] = (f32x16)(0.0f);

        Tl t;
        bool keep[Tl::PER];
        float next_m = 0.0f, next_r = 0.0f, next_g = 0.0f;
        int32_t next_t = -1;
        auto fetch = [&](int i, int j) {
            const int64_t r = (int64_t)(t0 + i) * Tl::BV;
            t.fetch((const E *)a.x + sm.offset(j), a.ldx, r, a.rows);
#pragma unroll
            for (int k = 0; k < Tl::PER; ++k) {
                const int64_t n = r + Tl::row_of(k);
                keep[k] = n < a.rows && a.row_target[n] >= 0;
            }
            if (j == 0 && threadIdx.x < Tl::BV) {
                const int64_t n = r + threadIdx.x;
                const bool ok = n < a.rows;
                next_m = ok ? a.row_max[n] : INFINITY;
                next_r = ok ? a.row_rate[n] : 0.0f;
                next_g = ok ? a.row_weight[n] : 0.0f;
                next_t = ok ? a.row_target[n] : -1;
            }
        };
        auto store = [&](int i, int j, int buf) {
#pragma unroll
            for (int k = 0; k < Tl::PER; ++k)  // a row without a target is not read: zeros in its place
                if (!keep[k]) t.held[k] = make_uint4(0, 0, 0, 0);
            t.store(tile[buf]);
            if (j == 0 && threadIdx.x < Tl::BV) {
                const bool far = fabsf(next_m * dv.c) > FAR && next_m < INFINITY;
                RowFacts<Tl::BV> &f = facts[i & 1];
                f.m[threadIdx.x] = far ? 0.0f : -next_m * dv.c;
                f.far[threadIdx.x] = far ? next_m : 0.0f;
                f.rate[threadIdx.x] = next_r;
                f.weight[threadIdx.x] = next_g;
                f.target[threadIdx.x] = next_t;
            }
        };
        if (!ONE || unit == begin + 1) {
            __syncthreads();  // (the owner before is done with the tiles)
            fetch(0, 0);
            store(0, 0, 0);
            __syncthreads();
        }
        int buf = 0;
        for (int i = 0; i < nt; ++i) {
            if (!WIDE && !ONE && i + 1 < nt) fetch(i + 1, 0);
            const RowFacts<Tl::BV> &f = facts[i & 1];
#pragma unroll
            for (int blk = 0; blk < St::BLOCKS; ++blk) {
                ScoreOperand<E, NS, DP> so;
                SumOperand<E, NS, DP> to;
                f32x16 s = (f32x16)(bias);
                const int r0 = blk * 32;
                const int32_t mine = f.target[r0 + (lane & 31)] - w0;
                const float fars = f.far[r0 + (lane & 31)];
                if (WIDE) {
                    for (int j = 0; j < sm.chunks; ++j) {
                        load_owned<E, NS, DP>(own, (const E *)a.w + sm.offset(j), a.ldw, v, have, dv.owned);
                        const bool last = j + 1 == sm.chunks;
                        if (!last || i + 1 < nt) fetch(last ? i + 1 : i, last ? 0 : j + 1);
                        so.read(tile[buf], 0);
                        scores<E, NS, DP>(s, own, so);
                        if (last) break;
                        store(i, j + 1, buf ^ 1);
                        __syncthreads();
                        buf ^= 1;
                    }
                    to.read(tile[buf], 0);
                } else {
                    so.read(tile[buf], r0);
                    scores<E, NS, DP>(s, own, so);
                    to.read(tile[buf], r0);
                }
                // Where a row's target is among the owned table rows q is -g (1 - p), formed from the sum over the other
                // items: popular items are targets in every block, so this has to be cheap.  A lane collects the rows
                // whose target is its own table row as bits.
                uint32_t hits = 0, any = (uint32_t)__ballot((uint32_t)mine < 32u);  // (both half-waves say the same)
                for (uint32_t rows = any; rows; rows &= rows - 1) {
                    const int r = __ffs(rows) - 1;
                    hits |= (lane & 31) == __builtin_amdgcn_readlane(mine, r) ? 1u << r : 0u;
                }
                if (__any(fars != 0.0f)) {  // see FAR
#pragma unroll
                    for (int j = 0; j < 16; ++j) s[j] -= f.far[r0 + 8 * (j / 4) + 4 * h + j % 4];
                }
                float q[16];
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int r = r0 + 8 * g + 4 * h;
                    const float4 mm = *(const float4 *)&f.m[r], rr = *(const float4 *)&f.rate[r];
                    const float ms[4] = {mm.x, mm.y, mm.z, mm.w}, rs[4] = {rr.x, rr.y, rr.z, rr.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) q[4 * g + j] = exp2_fast(__builtin_fmaf(s[4 * g + j], dv.c, ms[j])) * rs[j];
                }
                if (any) {
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const float4 ww = *(const float4 *)&f.weight[r0 + 8 * g + 4 * h];
                        const float ws[4] = {ww.x, ww.y, ww.z, ww.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) q[4 * g + j] = (hits >> (4 * h)) & (1u << (8 * g + j)) ? -ws[j] : q[4 * g + j];
                    }
                }
                db += sum16(q);
                Values<E, NS> p;
                p.pack(q);
                accumulate<E, NS, DP>(out, p, to);
            }
            if (ONE) break;
            if (i + 1 < nt) store(i + 1, 0, buf ^ 1);
            __syncthreads();
            buf ^= 1;
        }
        const float total = half_wave_sum(db);
        if constexpr (ONE) {
            if (a.db && h == 0 && v < a.vocab) a.db[v] = ldexpf(total, shift);
            Strip *strip = &strips[wave];
#pragma unroll
            for (int b = 0; b < DP / 32; ++b) {
                strip->write(out[b]);
                if (a.aligned) {
                    const int c = b * 32 + strip->column4();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int64_t to = (int64_t)w0 + strip->row4(i);
                        const float4 f = strip->read4(i);
                        const float o[4] = {f.x, f.y, f.z, f.w};
                        Vec<T, 4> r;
#pragma unroll
                        for (int k = 0; k < 4; ++k) r.v[k] = (T)ldexpf(o[k], shift - kx);
                        if (to < a.vocab && c < a.d) *(Vec<T, 4> *)((T *)a.dw + to * a.d + c) = r;
                    }
                } else {
                    const int c = b * 32 + (lane & 31);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int64_t to = (int64_t)w0 + 2 * i + h;
                        const float f = strip->v[2 * i + h][lane & 31];
                        if (to < a.vocab && c < a.d) ((T *)a.dw)[to * a.d + c] = (T)ldexpf(f, shift - kx);
                    }
                }
            }
            continue;
        }
        const uint32_t b0 = a.pieces.first_block(owner), b1 = a.pieces.last_block(owner);
        if (b0 != b1) {  // shared with other blocks: the block's first owner, or its last
            const int64_t part = 2 * (int64_t)blockIdx.x + (begin > (uint64_t)owner * a.pieces.tiles ? 0 : 1);
            const int64_t at = part * 128 + (v - (int64_t)owner * 128);
            if (h == 0 && c0 == 0) a.pb[at] = total;
#pragma unroll
            for (int b = 0; b < DP / 32; ++b)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *(float4 *)(a.pw + at * a.dp + c0 + b * 32 + 8 * g + 4 * h) =
                        make_float4(out[b][4 * g], out[b][4 * g + 1], out[b][4 * g + 2], out[b][4 * g + 3]);
            continue;
        }
        if (v >= a.vocab) continue;
        if (a.db && h == 0 && c0 == 0) a.db[v] = ldexpf(total, shift);
        T *row = (T *)a.dw + v * a.d;
#pragma unroll
        for (int b = 0; b < DP / 32; ++b)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = c0 + b * 32 + 8 * g + 4 * h;
                Vec<T, 4> o;
#pragma unroll
                for (int j = 0; j < 4; ++j) o.v[j] = (T)ldexpf(out[b][4 * g + j], shift - kx);
                if (a.aligned && c < a.d) *(Vec<T, 4> *)(row + c) = o;
                else
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (c + j < a.d) row[c + j] = o.v[j];
            }
    }
}

// ---------------------------------------------------------------- few rows ---

// Without the gradient and with up to FEW float32 rows the table is read once, as it is, and multiplied in float32: the
// matrix form reads it twice and writes it once before it begins.  `lanes` neighbouring lanes own a table row, VEC elements
// each and step.  Bound by reading the table with one row, by the products and exponentials with more.  A block leaves the
// maximum and the sum of its part of the table for each row, like rows_kernel.  Measured (us for 1 / 2 / 4 / 8 rows, with the join;
// matrix form in brackets): 26744 x 64 9.9 / 11.7 / 15.2 / 17.2 (23), 200003 x 128 26 / 36 / 57 / 96 (84), 60000 x 50 12 / 15 / 22 / 35 (31),
// 59803 x 51 16 / 23 / 37 / 65 (33), 100000 x 301 37 / 48 / 72 / 123 (226): up to four rows, and up to eight where the table is small
// or wider than a chunk.  Half-precision tables need no packing where their rows are 16-byte aligned, and the matrix form is then the
// faster one from one row on (26744 x 64: 10.5).
constexpr int FEW = 8;

bool takes_few(int64_t rows, int64_t vocab, int d, int dtype, bool grad)
{
    if (grad || dtype != LFM_F32) return false;
    return rows <= 4 || (rows <= FEW && (d > 256 || (d % 4 == 0 && vocab * d <= 4000000)));
}

template <int VEC, int ROWS>
__global__ __launch_bounds__(256) void few_rows_kernel(SweepArgs a, const float *hidden, const float *table, int lanes_log2)
{
    constexpr int U = ROWS > 4 ? 2 : 4;  // table rows in flight
    __shared__ __attribute__((aligned(16))) float xs[ROWS][LFM_MAX_COMPONENTS];
    __shared__ float ms[ROWS][4], ls[ROWS][4];
    __shared__ int64_t ts[ROWS];
    const Derived dv = derive(nullptr);
    const int lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1), group = threadIdx.x >> lanes_log2, groups = 256 >> lanes_log2;
    const int rows = (int)a.rows;
    for (int i = threadIdx.x; i < ROWS * a.d; i += 256) {
        const int r = i / a.d, c = i - r * a.d;
        xs[r][c] = r < rows ? hidden[r * a.ldx + c] : 0.0f;
    }
    if (threadIdx.x < ROWS) {
        const int n = threadIdx.x;
        ts[threadIdx.x] = (int)threadIdx.x >= rows ? -1 : a.id_bytes == 8 ? ((const int64_t *)a.targets)[n] : (int64_t)((const int32_t *)a.targets)[n];
    }
    __syncthreads();
    float m[ROWS], l[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        m[r] = dv.low * 1.01f;
        l[r] = 0.0f;
    }
    const int64_t lo = a.vocab * blockIdx.x / gridDim.x, hi = a.vocab * (blockIdx.x + 1) / gridDim.x;
    for (int64_t v0 = lo + group; v0 < hi; v0 += (int64_t)U * groups) {
        float s[U][ROWS], b[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t v = v0 + (int64_t)u * groups;
            b[u] = v >= hi ? -INFINITY : a.bias ? bias_units(a.bias[v], dv) : 0.0f;
#pragma unroll
            for (int r = 0; r < ROWS; ++r) s[u][r] = 0.0f;
        }
        for (int c = lane * VEC; c < a.d; c += lanes * VEC) {
            Vec<float, VEC> w[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t v = v0 + (int64_t)u * groups;
                w[u] = *(const Vec<float, VEC> *)(table + (v < hi ? v : v0) * a.ldw + c);
                if (b[u] == -INFINITY) w[u] = {};  // a removed item, or none
            }
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const float x = xs[r][c + k];
#pragma unroll
                    for (int u = 0; u < U; ++u) s[u][r] = __builtin_fmaf(x, w[u].v[k], s[u][r]);
                }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t v = v0 + (int64_t)u * groups;
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                for (int o = lanes >> 1; o; o >>= 1) s[u][r] += __shfl_xor(s[u][r], o);
                const float score = v == ts[r] ? -INFINITY : s[u][r] + b[u];  // the target is left to the join
                const float up = fmaxf(m[r], score);
                l[r] = l[r] * exp2_fast((m[r] - up) * LOG2E) + exp2_fast((score - up) * LOG2E + P_SHIFT);
                m[r] = up;
            }
        }
    }
    // a wave's groups, then the block's waves
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        for (int o = lanes; o < 64; o <<= 1) {
            const float mo = __shfl_xor(m[r], o), lo2 = __shfl_xor(l[r], o), up = fmaxf(m[r], mo);
            l[r] = l[r] * exp2_fast((m[r] - up) * LOG2E) + lo2 * exp2_fast((mo - up) * LOG2E);
            m[r] = up;
        }
        if ((threadIdx.x & 63) == 0) {
            ms[r][threadIdx.x >> 6] = m[r];
            ls[r][threadIdx.x >> 6] = l[r];
        }
    }
    __syncthreads();
    if ((int)threadIdx.x < rows) {
        const int r = threadIdx.x;
        float mm = ms[r][0], ll = ls[r][0];
        for (int w = 1; w < 4; ++w) {
            const float up = fmaxf(mm, ms[r][w]);
            ll = ll * exp2_fast((mm - up) * LOG2E) + ls[r][w] * exp2_fast((ms[r][w] - up) * LOG2E);
            mm = up;
        }
        a.pm[(int64_t)blockIdx.x * a.rows + r] = mm;
        a.pl[(int64_t)blockIdx.x * a.rows + r] = ll;
    }
}

// ------------------------------------------------------------------- joins ---

struct JoinArgs {
    lfm_softmax_args a;
    const Scales *scales;
    const int16_t *codes;
    Pieces pieces;
    int parts, dp, ns, grad, shifted;
    int few;                // few_rows_kernel: every row has `parts` parts
    int aligned;            // rows of d_hidden can be written four elements at a time
    const float *pm, *pl, *po;
    float *row_max, *row_rate, *row_weight;
    int32_t *row_target;
};

// Sums and maxima over the lanes that share a row: 16 neighbouring ones, or the block's 256
template <int LANES>
__device__ inline float row_sum(float v, float *shared)
{
    for (int o = LANES < 64 ? LANES / 2 : 32; o; o >>= 1) v += __shfl_xor(v, o);
    if (LANES < 64) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    return shared[0] + shared[1] + shared[2] + shared[3];
}

template <int LANES>
__device__ inline float row_max(float v, float *shared)
{
    for (int o = LANES < 64 ? LANES / 2 : 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    if (LANES < 64) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(shared[0], shared[1]), fmaxf(shared[2], shared[3]));
}

// Joins the parts of the table, finishes lse, loss, dx, and leaves table_kernel what it needs.  LANES lanes per row: 16 where
// there are rows enough to fill the card or little to join, a block's 256 (which share the parts, too) elsewhere; with very few the
// columns of dx are dealt to blockIdx.y, each of which makes the row's statistics for itself.
template <typename T, int LANES>
__global__ __launch_bounds__(256) void join_rows_kernel(JoinArgs j)
{
    __shared__ float shared[4];
    __shared__ __attribute__((aligned(16))) float4 sums[LANES == 256 ? 256 : 1];
    const lfm_softmax_args &a = j.a;
    const int64_t n = (int64_t)blockIdx.x * (256 / LANES) + (LANES == 256 ? 0 : threadIdx.x / LANES);
    const int lane = threadIdx.x % LANES;
    if (n >= a.rows) return;  // (with 256 lanes: nobody; with 16: all of a row's)
    const int16_t code = j.ns == 2 ? j.codes[n] : (int16_t)0;
    const Derived dv = derive_row(derive(j.ns == 2 ? j.scales : nullptr), code);
    const uint32_t owner = (uint32_t)(n / 128);
    const int splits = j.few ? j.parts : (int)(j.pieces.last_block(owner) - j.pieces.first_block(owner)) + 1;
    const int64_t t = target_of(a, n);
    const float g = t < 0 ? 0.0f : a.weights ? a.weights[n] : 1.0f;
    const T *x = (const T *)a.hidden + n * a.hidden_stride;
    const T *wt = (const T *)a.table + (t < 0 ? 0 : t) * a.table_stride;
    const bool out = t >= 0 && removed(a.bias, t);  // its score is -inf, whatever its row holds
    float m = -INFINITY, l = 0.0f, st = 0.0f;
#pragma unroll 4
    for (int s = lane; s < splits; s += LANES) m = fmaxf(m, j.pm[(int64_t)s * a.rows + n]);
    if (t >= 0 && !out)
        for (int c = lane; c < a.d; c += LANES) st = __builtin_fmaf((float)x[c], (float)wt[c], st);
    m = row_max<LANES>(m, shared);
#pragma unroll 4
    for (int s = lane; s < splits; s += LANES)
        l += j.pl[(int64_t)s * a.rows + n] * exp2_fast((j.pm[(int64_t)s * a.rows + n] - m) * dv.c);
    l = row_sum<LANES>(l, shared);
    st = row_sum<LANES>(st, shared);
    // l = sum without the target (times 2^7, about m).  With the target's score st and everything about the larger of the two:
    // 1 - p[target] = l / (l + e), loss = log1p(l / e): nothing is lost where p[target] is near 1.
    float e = 0.0f, loss = 0.0f;
    if (t >= 0) {
        if (a.bias) st += a.bias[t];
        const float su = bias_units(st, dv);  // (not only a bias: any score)
        const float up = fmaxf(m, su);
        e = exp2_fast((su - up) * dv.c + P_SHIFT);
        l *= exp2_fast((m - up) * dv.c);
        m = up;
        // a score below the products' range (a mask) is cut there, which a probability of 0 does not show, but the loss would
        const float behind = su <= dv.low && m > su ? ldexpf(m, -dv.k) - st : ldexpf(m - su, -dv.k);
        loss = st == -INFINITY ? INFINITY : l <= e ? log1pf(l / e) : behind + (logf(l + e) - P_SHIFT * LN2);
    }
    const float sum = l + e;
    // (m says nothing about a row of NaN, which no maximum takes in: its sum does)
    float lse = sum != sum ? sum : sum == 0.0f ? -INFINITY : m <= dv.low * 0.999f ? -3.402823466e38f : ldexpf(m, -dv.k) + (logf(sum) - P_SHIFT * LN2);
    const float other = sum == 0.0f ? 1.0f : l / sum;  // 1 - p[target]
    const bool odd = code == NOT_FINITE;
    if (odd) lse = NAN;
    if (odd && t >= 0) loss = NAN;
    loss = t < 0 ? 0.0f : g * loss;
    if (lane == 0 && blockIdx.y == 0) {
        a.lse[n] = lse;
        a.loss[n] = loss;
    }
    if (!j.grad) return;
    const bool lost = odd && t >= 0;  // not finite: its gradients are not either
    if (lane == 0 && blockIdx.y == 0) {
        const int shift = j.shifted == 2 ? 14 - j.scales->eg : j.shifted ? 14 : 0;
        const float gs = ldexpf(g, shift);
        j.row_target[n] = (int32_t)t;
        j.row_max[n] = t < 0 ? INFINITY : m;
        j.row_rate[n] = lost ? NAN : t < 0 || sum == 0.0f ? 0.0f : gs * exp2_fast(P_SHIFT) / sum;
        j.row_weight[n] = gs * other;
    }
    const int kw = j.ns == 2 ? j.scales->kw : 0;
    // four columns per lane; with 256 lanes `groups` of them share a column's parts
    const int span = LANES == 256 ? j.dp / (int)gridDim.y : j.dp, c_begin = LANES == 256 ? (int)blockIdx.y * span : 0;
    const int columns = span / 4, groups = LANES == 256 ? 256 / columns : 1, group = LANES == 256 ? lane / columns : 0;
    const int c_first = c_begin + (LANES == 256 ? lane - group * columns : lane) * 4;
    for (int c = c_first; c < c_begin + span; c += (LANES == 256 ? columns : LANES) * 4) {
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (t >= 0 && c < a.d && group < groups) {
            const float *pm = j.pm + (int64_t)(c >> 8) * j.parts * a.rows;  // the maxima that chunk c / 256 went by
#pragma unroll 4
            for (int s = group; s < splits; s += groups) {
                const int64_t at = (int64_t)s * a.rows + n;
                const float4 p = *(const float4 *)(j.po + at * j.dp + c);
                const float f = exp2_fast((pm[at] - m) * dv.c);
                o.x = __builtin_fmaf(p.x, f, o.x);
                o.y = __builtin_fmaf(p.y, f, o.y);
                o.z = __builtin_fmaf(p.z, f, o.z);
                o.w = __builtin_fmaf(p.w, f, o.w);
            }
        }
        if (LANES == 256) {
            sums[lane] = o;
            __syncthreads();
            if (group) break;
            for (int q = 1; q < groups; ++q) {
                const float4 p = sums[lane + q * columns];
                o.x += p.x;
                o.y += p.y;
                o.z += p.z;
                o.w += p.w;
            }
        }
        if (c >= a.d) continue;
        const float ov[4] = {o.x, o.y, o.z, o.w};
        Vec<T, 4> r;
        T *to = (T *)a.d_hidden + n * a.d + c;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float v = 0.0f;
            if (t >= 0 && c + k < a.d) {
                v = sum == 0.0f ? 0.0f : ldexpf(ov[k] / sum, -kw);
                const float wv = (float)wt[c + k];
                v = lost ? NAN : g * (v - other * (out && !(fabsf(wv) < INFINITY) ? 0.0f : wv));
            }
            r.v[k] = (T)v;
        }
        if (j.aligned) *(Vec<T, 4> *)to = r;
        else
            for (int k = 0; k < 4; ++k)
                if (c + k < a.d) to[k] = r.v[k];
    }
}

// dw and db of the table rows that several blocks share, added in the order of the blocks: block (owner, 32 columns, 32 rows), or,
// where there are more owners than blocks, (boundary between two blocks, ...): the others have a block to themselves.
template <typename T>
__global__ __launch_bounds__(256) void join_table_kernel(SweepArgs a, int ns)
{
    uint32_t owner = blockIdx.x, b0 = blockIdx.x;
    if (a.pieces.owners > a.pieces.blocks) {  // (an owner lies in two blocks at most)
        const uint64_t boundary = a.pieces.begin(b0 + 1);
        owner = a.pieces.owner_of(boundary);
        if (boundary == (uint64_t)owner * a.pieces.tiles) return;
    } else
        b0 = a.pieces.first_block(owner);
    const uint32_t b1 = a.pieces.last_block(owner);
    if (b0 == b1) return;
    const int shift = a.shifted == 2 ? a.scales->eg - 14 : a.shifted ? -14 : 0, kx = ns == 2 ? a.scales->kx : 0;
    const int64_t first = 2 * (int64_t)b0 + 1;  // the others began inside the owner
    auto part = [&](uint32_t b) { return b == b0 ? first : 2 * (int64_t)b; };
    const int c = (int)blockIdx.y * 32 + (threadIdx.x & 7) * 4;
    const int r = (int)blockIdx.z * 32 + (threadIdx.x >> 3);
    const int64_t v = (int64_t)owner * 128 + r;
    if (v < a.vocab && c < a.d) {
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (uint32_t b = b0; b <= b1; ++b) {
            const float4 p = *(const float4 *)(a.pw + (part(b) * 128 + r) * a.dp + c);
            s.x += p.x;
            s.y += p.y;
            s.z += p.z;
            s.w += p.w;
        }
        const float o[4] = {s.x, s.y, s.z, s.w};
        T *to = (T *)a.dw + v * a.d + c;
        Vec<T, 4> ov;
#pragma unroll
        for (int j = 0; j < 4; ++j) ov.v[j] = (T)ldexpf(o[j], shift - kx);
        if (a.aligned) *(Vec<T, 4> *)to = ov;
        else
            for (int j = 0; j < 4; ++j)
                if (c + j < a.d) to[j] = ov.v[j];
    }
    if (a.db && blockIdx.y == 0 && (threadIdx.x & 7) == 0 && v < a.vocab) {
        float t = 0.0f;
        for (uint32_t b = b0; b <= b1; ++b) t += a.pb[part(b) * 128 + r];
        a.db[v] = ldexpf(t, shift);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void clear_kernel(T *p, int64_t n, float *q, int64_t m)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        p[i] = (T)0.0f;
        if (q && i < m) q[i] = 0.0f;  // (m <= n)
    }
}

// -------------------------------------------------------------------- host ---

struct Plan {
    int dp, ns;
    int chunks;             // of 256 columns
    Pieces rows, table;
    int few;                // blocks over the table of the few-rows form, 0: the matrix form
};

int width_for(int d)
{
    const int widths[] = {32, 64, 96, 128, 192, 256};
    for (int w : widths)
        if (d <= w) return w;
    return (d + 255) / 256 * 256;
}

// As many blocks as run at once, with two exceptions.  A block of a single tile is mostly prologue and parts to join: up to
// twice as many tiles as the card has compute units are dealt two to a block (gradients of 5276 rows x 712 items x 16 float32: 69 ->
// 55 us, 3660 x 806 x 188 float16: 115 -> 100).  And where there are nearly as many owners as blocks would be, each has a block
// to itself and nothing is joined, if what the other slots then leave undone, tiles (slots - owners) / slots, is less than the
// join costs, `idle` tiles.  Calls with the gradients, blocks dealt and owners to themselves (us; 512 slots, 256 for 128 columns of float32):
//   table's sweep   1003 rows (16 tiles) x 391 owners x 100 float16 124 and 109; 2000 (32) x 391 x 32 float16 103 and 101; 2228 (35) x
//                   420 x 19 float32 159 and 162; 1003 (32) x 210 x 128 float32 163 and 162; 4096 (64) x 450 x 64 float32 420 and
//                   422; 8192 (128) x 64 bfloat16, 391 owners 342 and 379, 480 411 and 416, 511 435 and 429: even from 4 to 12
//   rows' sweep     (its join remains, with less to add) 500 items (8 tiles) x 368 owners x 64 bfloat16 109 and 110; 1682 (27) x 409 x 64
//                   float32 230 and 231; its loss alone x 450 84 and 85; 8000 (125) x 486 260 and 262: even from 2 to 5
constexpr int IDLE_TABLE = 7, IDLE_ROWS = 3;

Pieces pieces_for(int64_t owned, int64_t streamed, int bv, int64_t slots, int idle)
{
    Pieces p;
    p.owners = (uint32_t)ceil_div(owned < 1 ? 1 : owned, 128);
    p.tiles = (uint32_t)ceil_div(streamed < 1 ? 1 : streamed, bv);
    const uint64_t units = (uint64_t)p.owners * p.tiles;
    uint64_t blocks = units / 2 > p.owners ? units / 2 : p.owners;
    if (blocks < 256) blocks = units < 256 ? units : 256;
    if (blocks > (uint64_t)slots) blocks = slots;
    if (p.owners <= blocks && (uint64_t)p.owners * 100 >= blocks * 70 && p.tiles * (blocks - p.owners) <= idle * blocks) blocks = p.owners;
    p.blocks = (uint32_t)blocks;
    return p;
}

Plan plan_for(int64_t rows, int64_t vocab, int d, int dtype, bool grad)
{
    Plan p;
    p.dp = width_for(d);
    p.ns = dtype == LFM_F32 ? 2 : 1;
    p.chunks = p.dp > 256 ? p.dp / 256 : 1;
    const int w = p.dp > 256 ? 256 : p.dp, bv = p.ns * w <= 128 ? 64 : 32;
    // slots: blocks that run at once on the card's 256 compute units
    p.rows = pieces_for(rows, vocab, bv, 256 * (p.chunks > 1 ? 1 : waves_for(p.ns, w, grad)), IDLE_ROWS);
    p.few = 0;
    if (takes_few(rows, vocab, d, dtype, grad)) {
        const int64_t want = ceil_div(vocab, 16);  // (a block's lane groups have a few table rows each)
        p.few = (int)(want < 1024 ? want : 1024);
    }
    p.table = pieces_for(vocab, rows, bv, 256 * (p.chunks > 1 ? 1 : waves_for(p.ns, w, true)), IDLE_TABLE);
    return p;
}

struct Space {
    Scales *scales;
    float *largest;
    int16_t *codes;
    void *x, *w;
    float *pm, *pl, *po, *pw, *pb;
    float *row_max, *row_rate, *row_weight;
    int32_t *row_target;
    int64_t bytes;
};

// Sized for the case that both operands have to be packed: whether they have to depends on addresses and strides.
Space space_for(const Plan &p, int64_t rows, int64_t vocab, bool grad, void *ws)
{
    Carver c(ws);
    Space s = {};
    if (p.few) {
        s.pm = c.take<float>(rows * p.few);
        s.pl = c.take<float>(rows * p.few);
        s.bytes = c.used;
        return s;
    }
    s.scales = c.take<Scales>(1);
    s.largest = c.take<float>(4 * MAX_PARTS);
    s.codes = c.take<int16_t>(rows);
    s.x = c.take<uint16_t>(rows * p.ns * p.dp);
    s.w = c.take<uint16_t>(vocab * p.ns * p.dp);
    const int64_t parts = rows * p.rows.most(), shared = (int64_t)p.table.blocks * 2 * 128;
    s.pm = c.take<float>(parts * p.chunks);
    s.pl = c.take<float>(parts * p.chunks);
    s.po = c.take<float>(grad ? parts * p.dp : 0);
    s.pw = c.take<float>(grad ? shared * p.dp : 0);
    s.pb = c.take<float>(grad ? shared : 0);
    s.row_max = c.take<float>(grad ? rows : 0);
    s.row_rate = c.take<float>(grad ? rows : 0);
    s.row_weight = c.take<float>(grad ? rows : 0);
    s.row_target = c.take<int32_t>(grad ? rows : 0);
    s.bytes = c.used;
    return s;
}

template <typename E, int NS, int DP, bool WIDE>
hipError_t sweep_rows(const SweepArgs &s, bool grad, hipStream_t st)
{
    // without the gradient one chunk's sweep does
    if (grad) rows_kernel<E, NS, DP, true, WIDE><<<dim3(s.pieces.blocks, (unsigned)s.chunks), 256, 0, st>>>(s);
    else rows_kernel<E, NS, DP, false, WIDE><<<dim3(s.pieces.blocks), 256, 0, st>>>(s);
    return hipGetLastError();
}

template <typename T, typename E, int NS, int DP, bool WIDE>
hipError_t sweep_table(const SweepArgs &s, hipStream_t st)
{
    if (!WIDE && s.pieces.tiles == 1) table_kernel<T, E, NS, DP, WIDE, !WIDE><<<dim3(s.pieces.blocks), 256, 0, st>>>(s);
    else table_kernel<T, E, NS, DP, WIDE, false><<<dim3(s.pieces.blocks, (unsigned)s.chunks), 256, 0, st>>>(s);
    return hipGetLastError();
}

#define BY_WIDTH(dp, call)                      \
    switch (dp) {                               \
    case 32: e = call(32, false); break;        \
    case 64: e = call(64, false); break;        \
    case 96: e = call(96, false); break;        \
    case 128: e = call(128, false); break;      \
    case 192: e = call(192, false); break;      \
    case 256: e = call(256, false); break;      \
    default: e = call(256, true); break;        \
    }

template <int VEC>
hipError_t launch_few(const SweepArgs &w, const lfm_softmax_args &a, int blocks, hipStream_t st)
{
    int ll = 0;
    while ((1 << ll) * VEC < a.d && ll < 6) ++ll;
    const float *x = (const float *)a.hidden, *t = (const float *)a.table;
    const dim3 grid((unsigned)blocks);
    if (a.rows == 1) few_rows_kernel<VEC, 1><<<grid, 256, 0, st>>>(w, x, t, ll);
    else if (a.rows == 2) few_rows_kernel<VEC, 2><<<grid, 256, 0, st>>>(w, x, t, ll);
    else if (a.rows <= 4) few_rows_kernel<VEC, 4><<<grid, 256, 0, st>>>(w, x, t, ll);
    else few_rows_kernel<VEC, FEW><<<grid, 256, 0, st>>>(w, x, t, ll);
    return hipGetLastError();
}

template <typename T>
hipError_t join_rows(JoinArgs j, int64_t parts, hipStream_t st)
{
    j.aligned = j.a.d % 4 == 0 && ((uintptr_t)j.a.d_hidden & (4 * sizeof(T) - 1)) == 0;
    if (j.a.rows <= 2048 && parts > (j.grad ? 4 : 64)) {
        int slices = j.grad ? j.dp / 32 : 1;  // (with every row's dx in one block 32 rows x 200003 x 128: 14.7 us)
        while (slices > 1 && (j.a.rows * slices > 1024 || j.dp / 32 % slices)) --slices;
        join_rows_kernel<T, 256><<<dim3((unsigned)j.a.rows, (unsigned)slices), 256, 0, st>>>(j);
    }
    else join_rows_kernel<T, 16><<<dim3((unsigned)ceil_div(j.a.rows, 16)), 256, 0, st>>>(j);
    return hipGetLastError();
}

template <typename T, typename E, int NS>
hipError_t run(const lfm_softmax_args &a, bool grad, void *ws, hipStream_t st)
{
    const Plan p = plan_for(a.rows, a.vocab, a.d, a.dtype, grad);
    const Space s = space_for(p, a.rows, a.vocab, grad, ws);
    hipError_t e;
    if (a.rows == 0) {
        if (!grad) return hipSuccess;
        const int64_t blocks = ceil_div(a.vocab * a.d, 256);
        clear_kernel<T><<<dim3((unsigned)(blocks < 8192 ? blocks : 8192)), 256, 0, st>>>((T *)a.d_table, a.vocab * a.d, a.d_bias, a.vocab);
        return hipGetLastError();
    }
    // scales are wanted for float32 operands, and of the weights for float16 gradients
    const bool scales = NS == 2 || (a.dtype == LFM_F16 && a.weights && grad);
    auto in_place = [&](const void *q, int64_t stride) {  // (offsets inside a tile are 32-bit)
        return NS == 1 && a.d == p.dp && stride % 8 == 0 && stride < (1 << 24) && ((uintptr_t)q & 15) == 0;
    };
    const bool x_there = in_place(a.hidden, a.hidden_stride), w_there = in_place(a.table, a.table_stride);
    // both operands can be read four elements at a time
    const bool wide = a.d % 4 == 0 && a.hidden_stride % 4 == 0 && a.table_stride % 4 == 0 &&
                      (((uintptr_t)a.hidden | (uintptr_t)a.table) & (4 * sizeof(T) - 1)) == 0;
    // ... or two
    const bool two = a.d % 2 == 0 && a.hidden_stride % 2 == 0 && a.table_stride % 2 == 0 &&
                     (((uintptr_t)a.hidden | (uintptr_t)a.table) & (2 * sizeof(T) - 1)) == 0;
    SweepArgs w = {};
    w.rows = a.rows;
    w.vocab = a.vocab;
    w.bias = a.bias;
    w.targets = a.targets;
    w.id_bytes = a.id_bytes;
    w.d = a.d;
    w.pm = s.pm;
    w.pl = s.pl;
    JoinArgs j = {};
    j.a = a;
    j.grad = grad ? 1 : 0;
    j.pm = s.pm;
    j.pl = s.pl;
    if (NS == 2 && p.few) {
        w.ldx = a.hidden_stride;
        w.ldw = a.table_stride;
        e = wide ? launch_few<4>(w, a, p.few, st) : two ? launch_few<2>(w, a, p.few, st) : launch_few<1>(w, a, p.few, st);
        if (e != hipSuccess) return e;
        j.ns = 1;
        j.few = 1;
        j.parts = p.few;
        return join_rows<T>(j, p.few, st);
    }
    PackArgs pk = {};
    pk.a = a;
    pk.largest = scales ? s.largest : nullptr;
    pk.tensors = NS == 2 ? 3 : 1;
    pk.scales = s.scales;
    pk.x = x_there ? nullptr : s.x;
    pk.w = w_there ? nullptr : s.w;
    pk.codes = s.codes;
    const int64_t most = NS == 2 ? (a.rows > a.vocab ? a.rows : a.vocab) * a.d : a.rows;
    pk.parts = (int)(ceil_div(most, 4096) < MAX_PARTS ? ceil_div(most, 4096) : MAX_PARTS);
    if (scales) {
        const dim3 grid((unsigned)(pk.tensors * pk.parts));
        if (wide) largest_kernel<T, 4><<<grid, 256, 0, st>>>(a, pk.parts, s.largest, pk.tensors, s.codes);
        else if (two) largest_kernel<T, 2><<<grid, 256, 0, st>>>(a, pk.parts, s.largest, pk.tensors, s.codes);
        else largest_kernel<T, 1><<<grid, 256, 0, st>>>(a, pk.parts, s.largest, pk.tensors, s.codes);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (scales || pk.x || pk.w) {
        const int64_t per = 256 / (p.dp / 8);
        int64_t blocks = ceil_div((pk.x ? a.rows : 0) + (pk.w ? a.vocab : 0), per);
        blocks = blocks < 1 ? 1 : blocks > 4096 ? 4096 : blocks;
        const int width = p.dp < 256 ? p.dp : 256;
        if (wide) pack_kernel<T, E, NS, 4><<<dim3((unsigned)blocks), 256, 0, st>>>(pk, p.dp, width);
        else if (two) pack_kernel<T, E, NS, 2><<<dim3((unsigned)blocks), 256, 0, st>>>(pk, p.dp, width);
        else pack_kernel<T, E, NS, 1><<<dim3((unsigned)blocks), 256, 0, st>>>(pk, p.dp, width);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    w.x = x_there ? a.hidden : s.x;
    w.ldx = x_there ? a.hidden_stride : NS * p.dp;
    w.w = w_there ? a.table : s.w;
    w.ldw = w_there ? a.table_stride : NS * p.dp;
    w.scales = s.scales;
    w.codes = s.codes;
    w.pieces = p.rows;
    w.parts = (int)p.rows.most();
    w.dp = p.dp;
    w.chunks = p.chunks;
    w.po = s.po;
    w.row_max = s.row_max;
    w.row_rate = s.row_rate;
    w.row_weight = s.row_weight;
    w.row_target = s.row_target;
    w.dw = a.d_table;
    w.aligned = a.d % 4 == 0 && ((uintptr_t)a.d_table & (4 * sizeof(T) - 1)) == 0;
    w.db = a.d_bias;
    w.pw = s.pw;
    w.pb = s.pb;
    w.shifted = scales ? 2 : a.dtype == LFM_F16 ? 1 : 0;
#define ROWS(DP, WIDE) sweep_rows<E, NS, DP, WIDE>(w, grad, st)
    BY_WIDTH(p.dp, ROWS)
    if (e != hipSuccess) return e;
    j.scales = s.scales;
    j.codes = s.codes;
    j.pieces = p.rows;
    j.parts = w.parts;
    j.dp = p.dp;
    j.ns = NS;
    j.shifted = w.shifted;
    j.po = s.po;
    j.row_max = s.row_max;
    j.row_rate = s.row_rate;
    j.row_weight = s.row_weight;
    j.row_target = s.row_target;
    if ((e = join_rows<T>(j, w.parts, st)) != hipSuccess || !grad) return e;
    w.pieces = p.table;
#define TABLE(DP, WIDE) sweep_table<T, E, NS, DP, WIDE>(w, st)
    BY_WIDTH(p.dp, TABLE)
    if (e != hipSuccess || p.table.owners % p.table.blocks == 0 || p.table.tiles == 1) return e;  // (no block shares an owner)
    const uint32_t shared = p.table.owners > p.table.blocks ? p.table.blocks - 1 : p.table.owners;
    join_table_kernel<T><<<dim3(shared, (unsigned)(p.dp / 32), 4), 256, 0, st>>>(w, NS);
    return hipGetLastError();
}

}  // namespace

int64_t softmax_workspace(int64_t rows, int64_t vocab, int d, int dtype, bool grad)
{
    return space_for(plan_for(rows, vocab, d, dtype, grad), rows, vocab, grad, nullptr).bytes;
}

hipError_t softmax_loss(const lfm_softmax_args &a, bool grad, void *ws, hipStream_t st)
{
    return a.dtype == LFM_F32 ? run<float, f16_t, 2>(a, grad, ws, st)
         : a.dtype == LFM_BF16 ? run<bf16_t, bf16_t, 1>(a, grad, ws, st) : run<f16_t, f16_t, 1>(a, grad, ws, st);
}

}  // namespace ops
}  // namespace lfm
