// softmax_loss.hip -- softmax cross entropy over the whole catalogue with its gradient, without keeping the logits.
//
//   s[n, v] = <x[n], w[v]> + b[v],  lse[n] = log sum_v exp s[n, v],  loss[n] = g[n] (lse[n] - s[n, t[n]])
//   q[n, v] = g[n] (exp(s[n, v] - lse[n]) - [v = t[n]]),  dx = q w,  dw = q^T x,  db[v] = sum_n q[n, v]
//
// Two sweeps over the [rows, vocab] plane, each of which makes the scores in registers on the matrix cores and drops them:
//
//   rows_kernel   a wave owns 32 CW rows x (in registers) and streams the table through LDS.  dx needs no second look at
//                 the scores: sum_v p w is a mean weighted by the softmax, accumulated beside the running maximum and sum
//                 (rescaled when the maximum grows), so ONE sweep gives lse and dx -- 4 rows vocab d operations.
//   table_kernel  a wave owns 32 CW rows of the table and streams x; with lse known it forms q and accumulates dw and db.
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
// float32 pipe's 1/16.  The probabilities that enter the second product are split the same way.  Half-precision operands
// are multiplied as they are; their probabilities are rounded once to the operands' type (to nearest: 2^-9 / 2^-12
// relative, below the rounding of the result).  All sums, maxima and statistics are float32.
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

__device__ inline float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
// probabilities enter rows_kernel's second product as 2^7 p: with the maximum up to 8 binades behind they reach 2^15,
// and what float16 cannot hold below is 2^-32 of the largest
constexpr float P_SHIFT = 7.0f, LAG = 8.0f;
// exp2(s c - m c) as one multiply-add is off by the rounding of m c: with |m c| up to this, as much as s itself
constexpr float FAR = 512.0f;
constexpr int K_MOST = 60;  // see Scales
constexpr int MAX_PARTS = 128;

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

__device__ inline float bias_units(float b, const Derived &d)
{
    return fabsf(b) < INFINITY ? fminf(fmaxf(ldexpf(b, d.k), d.low), -d.low) : b;
}

__device__ inline int64_t target_of(const lfm_softmax_args &a, int64_t n)
{
    const int64_t t = a.id_bytes == 8 ? ((const int64_t *)a.targets)[n] : (int64_t)((const int32_t *)a.targets)[n];
    return (uint64_t)t < (uint64_t)a.vocab ? t : -1;
}

// -------------------------------------------------------------- operands ---

// Largest finite magnitudes: blocks [0, parts) of x (rows with a target), of w, of g.
template <typename T>
__global__ __launch_bounds__(256) void largest_kernel(lfm_softmax_args a, int parts, float *largest, int tensors)
{
    const int which = blockIdx.x / parts, part = blockIdx.x % parts;
    float m = 0.0f;
    if (which < 2 && tensors == 3) {
        const T *p = (const T *)(which ? a.table : a.hidden);
        const int64_t rows = which ? a.vocab : a.rows, stride = which ? a.table_stride : a.hidden_stride;
        const int64_t n = rows * a.d;
        for (int64_t i = (int64_t)part * 256 + threadIdx.x; i < n; i += (int64_t)parts * 256) {
            const int64_t r = i / a.d;
            if (!which && target_of(a, r) < 0) continue;
            const float v = fabsf((float)p[r * stride + (i - r * a.d)]);
            if (v < INFINITY) m = fmaxf(m, v);
        }
    } else {
        for (int64_t i = (int64_t)part * 256 + threadIdx.x; i < a.rows; i += (int64_t)parts * 256) {
            if (target_of(a, i) < 0) continue;
            const float v = a.weights ? fabsf(a.weights[i]) : 1.0f;
            if (v < INFINITY) m = fmaxf(m, v);
        }
    }
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    __shared__ float s[4];
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) largest[blockIdx.x] = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
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
    const float *largest;  // parts values for x, w and g, or NULL: no scales are wanted
    int parts, tensors;
    Scales *scales;
    void *x, *w;           // packed [rows + the outliers' flags], NULL: that operand is used where it is
    uint8_t *outlier;      // [rows]: the row does not fit x's scale (only a row without a target, or one that is not finite)
};

// Rows of x and w to the padded, split form, zeros behind d: per row and chunk of `width` columns [hi: width | lo: width]
// (width = dp up to 256 columns, 256 beyond).  A thread makes 8 elements.
template <typename T, typename E, int NS>
__global__ __launch_bounds__(256) void pack_kernel(PackArgs p, int dp, int width)
{
    __shared__ int ks[3];
    if (p.largest) {
        if (threadIdx.x < 192) {
            const int which = threadIdx.x >> 6, lane = threadIdx.x & 63;
            float m = 0.0f;
            if (p.tensors == 3 || which == 2)
                for (int i = lane; i < p.parts; i += 64) m = fmaxf(m, p.largest[(p.tensors == 3 ? which : 0) * p.parts + i]);
            for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
            int k = which < 2 ? exponent_for(m) : 14 - exponent_for(m);
            if (which == 2 && !(m > 0.0f)) k = 0;
            if (lane == 0) ks[which] = k;
        }
        __syncthreads();
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            Scales s = {ks[0], ks[1], ks[2], 0};
            *p.scales = s;
        }
    }
    typedef typename Half<E>::x8 x8;
    const int chunks = dp / 8;
    const int64_t xr = p.x ? p.a.rows : 0, wr = p.w ? p.a.vocab : 0, n = (xr + wr) * chunks;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        int64_t r = i / chunks;
        const int c = (int)(i - r * chunks) * 8;
        const bool is_x = r < xr;
        if (!is_x) r -= xr;
        const T *src = is_x ? (const T *)p.a.hidden + r * p.a.hidden_stride : (const T *)p.a.table + r * p.a.table_stride;
        E *dst = (E *)(is_x ? p.x : p.w) + r * (NS * dp) + (c / width) * (NS * width) + c % width;
        x8 hi, lo;
        if (NS == 1) {
#pragma unroll
            for (int j = 0; j < 8; ++j) hi[j] = c + j < p.a.d ? (E)src[c + j] : (E)0.0f;
        } else {
            const int k = ks[is_x ? 0 : 1];
            bool fits = true;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float v = c + j < p.a.d ? ldexpf((float)src[c + j], k) : 0.0f;
                if (is_x && !(fabsf(v) < 65504.0f)) { fits = false; v = 0.0f; }
                hi[j] = (E)v;
                lo[j] = (E)(v - (float)hi[j]);
            }
            if (is_x && !fits) p.outlier[r] = 1;
            *(x8 *)(dst + width) = lo;
        }
        *(x8 *)dst = hi;
    }
}

// ------------------------------------------------------------- the sweeps ---

// Streams `rows` rows of NS DP halves into LDS, BV at a time, double-buffered through registers: the loads of the next
// tile are in flight while this one is used.  A row takes NS DP + 8 halves of LDS: the padding spreads the 16-byte reads of
// 16 neighbouring rows over all banks.
template <typename E, int NS, int DP>
struct Tile {
    static constexpr int BV = NS * DP <= 128 ? 64 : 32, ROW = NS * DP + 8, CHUNKS = NS * DP / 8, PER = BV * CHUNKS / 256;
    static constexpr int SIZE = BV * ROW;
    uint4 held[PER];

    __device__ inline void fetch(const E *p, int64_t ld, int64_t row0, int64_t rows)
    {
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const int i = q * 256 + threadIdx.x, r = i / CHUNKS, c = i % CHUNKS;
            held[q] = make_uint4(0, 0, 0, 0);
            if (row0 + r < rows) held[q] = *(const uint4 *)(p + (row0 + r) * ld + c * 8);
        }
    }
    __device__ inline void store(E *tile) const
    {
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const int i = q * 256 + threadIdx.x, r = i / CHUNKS, c = i % CHUNKS;
            *(uint4 *)(tile + r * ROW + c * 8) = held[q];
        }
    }
};

template <typename E, int NS, int DP>
__device__ inline void load_owned(typename Half<E>::x8 (&f)[NS][DP / 16], const E *p, int64_t ld, int64_t row, int64_t rows, float factor)
{
    typedef typename Half<E>::x8 x8;
    const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
            x8 v = {};
            if (row < rows) v = *(const x8 *)(p + row * ld + s * DP + k * 16 + h * 8);
            if (NS == 2 && factor != 1.0f) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = (E)((float)v[j] * factor);
            }
            f[s][k] = v;
        }
}

// acc += 32 rows of the tile (from row r0) x the owned rows
template <typename E, int NS, int DP, int CW>
__device__ inline void scores(f32x16 (&acc)[CW], const typename Half<E>::x8 (&own)[CW][NS][DP / 16], const E *tile, int r0)
{
    typedef typename Half<E>::x8 x8;
    constexpr int ROW = Tile<E, NS, DP>::ROW;
    const int lane = threadIdx.x & 63;
    const E *p = tile + (r0 + (lane & 31)) * ROW + (lane >> 5) * 8;
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
        const x8 hi = *(const x8 *)(p + k * 16);
#pragma unroll
        for (int w = 0; w < CW; ++w) acc[w] = mfma(hi, own[w][0][k], acc[w]);
        if (NS == 2) {
            const x8 lo = *(const x8 *)(p + DP + k * 16);
#pragma unroll
            for (int w = 0; w < CW; ++w) {
                acc[w] = mfma(lo, own[w][0][k], acc[w]);
                acc[w] = mfma(hi, own[w][NS - 1][k], acc[w]);
            }
        }
    }
}

// out[d, owned] += tile^T x value for 16 rows of the tile (from row r0); v: the lane's 8 values of those rows
template <typename E, int NS, int DP, int CW>
__device__ inline void accumulate(f32x16 (&out)[CW][DP / 32], const float (&v)[CW][8], const E *tile, int r0)
{
    typedef typename Half<E>::x8 x8;
    typedef typename Half<E>::x4 x4;
    constexpr int ROW = Tile<E, NS, DP>::ROW;
    const int lane = threadIdx.x & 63;
    x8 hi[CW], lo[CW];
#pragma unroll
    for (int w = 0; w < CW; ++w)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            hi[w][j] = (E)v[w][j];
            if (NS == 2) lo[w][j] = (E)(v[w][j] - (float)hi[w][j]);
        }
    const E *p = tile + (r0 + 4 * (lane >> 5) + ((lane & 15) >> 2)) * ROW + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) {
        const x4 h0 = read_column(p + b * 32), h1 = read_column(p + 8 * ROW + b * 32);
        const x8 th = __builtin_shufflevector(h0, h1, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
        for (int w = 0; w < CW; ++w) out[w][b] = mfma(th, hi[w], out[w][b]);
        if (NS == 2) {
            const x4 l0 = read_column(p + DP + b * 32), l1 = read_column(p + DP + 8 * ROW + b * 32);
            const x8 tl = __builtin_shufflevector(l0, l1, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
            for (int w = 0; w < CW; ++w) {
                out[w][b] = mfma(tl, hi[w], out[w][b]);
                out[w][b] = mfma(th, lo[w], out[w][b]);
            }
        }
    }
}

struct SweepArgs {
    const void *x, *w;      // packed or in place
    int64_t ldx, ldw;       // halves per row
    int64_t rows, vocab;
    const float *bias;
    const Scales *scales;
    int splits;             // parts of the streamed side
    int d, dp;
    int chunks;             // of 256 columns (WIDE; else 1): the second product's columns are blockIdx.y's
    // rows_kernel: per chunk, part and row
    float *pm, *pl, *po;    // maximum (matrix units), sum of 2^7 p; per part and row: sum of 2^7 p w [dp]
    // table_kernel: per row
    const float *row_max, *row_rate, *row_weight;  // maximum (matrix units; +inf: no target), 2^shift g / sum, 2^shift g
    const int32_t *row_target;
    void *dw;               // one part: the result
    float *db, *pw, *pb;    // several: partial sums per part [vocab][dp], [vocab]
    int shifted;            // q is scaled by 2^(14 - eg): 0 no (bfloat16), 1 with eg = 0, 2 with eg of scales
};

// WIDE: more than 256 columns, taken 256 at a time.  The scores add up over the chunks (the owned operand is read again for
// each, from the caches); a block accumulates the second product of one chunk, the one that it streams last.
template <typename E, int NS, int DP, int CW, bool GRAD, bool WIDE>
__global__ __launch_bounds__(256, GRAD && (NS * DP >= 384 || WIDE) ? 1 : 2) void rows_kernel(SweepArgs a)
{
    typedef Tile<E, NS, DP> Tl;
    typedef typename Half<E>::x8 x8;
    constexpr int VB = Tl::BV / 32;
    __shared__ __attribute__((aligned(16))) E tile[2][Tl::SIZE];
    __shared__ __attribute__((aligned(16))) float sb[2][Tl::BV];
    const Derived dv = derive(NS == 2 ? a.scales : nullptr);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int part = blockIdx.x % a.splits;
    const int64_t n0 = (int64_t)(blockIdx.x / a.splits) * (128 * CW) + wave * (32 * CW) + (lane & 31);
    const int64_t tiles = ceil_div(a.vocab, Tl::BV);
    const int64_t t0 = tiles * part / a.splits, t1 = tiles * (part + 1) / a.splits;

    const int chunks = WIDE ? a.chunks : 1, first = WIDE ? (int)blockIdx.y + 1 : 0;
    auto offset = [&](int j) { return WIDE ? ((first + j) % chunks) * (NS * DP) : 0; };  // of the j-th chunk; the last is blockIdx.y's
    x8 own[CW][NS][DP / 16];
    auto take = [&](int j) {
#pragma unroll
        for (int w = 0; w < CW; ++w) load_owned<E, NS, DP>(own[w], (const E *)a.x + offset(j), a.ldx, n0 + 32 * w, a.rows, dv.owned);
    };
    if (!WIDE) take(0);
    f32x16 out[CW][DP / 32];
    float m[CW], l[CW];
#pragma unroll
    for (int w = 0; w < CW; ++w) {
        m[w] = dv.low * 1.01f;
        l[w] = 0.0f;
        if (GRAD)
#pragma unroll
            for (int b = 0; b < DP / 32; ++b) out[w][b] = (f32x16)(0.0f);
    }

    Tl t;
    float next_bias = 0.0f;
    auto fetch = [&](int64_t i, int j) {
        t.fetch((const E *)a.w + offset(j), a.ldw, i * Tl::BV, a.vocab);
        const int64_t v = i * Tl::BV + threadIdx.x;
        if (j == 0 && threadIdx.x < Tl::BV) next_bias = v >= a.vocab ? -INFINITY : a.bias ? bias_units(a.bias[v], dv) : 0.0f;
    };
    auto store = [&](int64_t i, int j, int buf) {
        t.store(tile[buf]);
        if (j == 0 && threadIdx.x < Tl::BV) sb[(i - t0) & 1][threadIdx.x] = next_bias;
    };
    if (t0 < t1) {
        fetch(t0, 0);
        store(t0, 0, 0);
    }
    __syncthreads();
    int buf = 0;
    for (int64_t i = t0; i < t1; ++i) {
        f32x16 s[VB][CW];
#pragma unroll
        for (int vb = 0; vb < VB; ++vb) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 b = *(const float4 *)&sb[(i - t0) & 1][vb * 32 + 8 * g + 4 * h];
#pragma unroll
                for (int w = 0; w < CW; ++w) {
                    s[vb][w][4 * g + 0] = b.x;
                    s[vb][w][4 * g + 1] = b.y;
                    s[vb][w][4 * g + 2] = b.z;
                    s[vb][w][4 * g + 3] = b.w;
                }
            }
        }
        for (int j = 0; j < chunks - 1; ++j) {  // WIDE: the other chunks first
            take(j);
            fetch(i, j + 1);
#pragma unroll
            for (int vb = 0; vb < VB; ++vb) scores<E, NS, DP, CW>(s[vb], own, tile[buf], vb * 32);
            store(i, j + 1, buf ^ 1);
            __syncthreads();
            buf ^= 1;
        }
        if (WIDE) take(chunks - 1);
        if (i + 1 < t1) fetch(i + 1, 0);
#pragma unroll
        for (int vb = 0; vb < VB; ++vb) scores<E, NS, DP, CW>(s[vb], own, tile[buf], vb * 32);
        bool grows = false;
        float mx[CW];
#pragma unroll
        for (int w = 0; w < CW; ++w) {
            mx[w] = s[0][w][0];
#pragma unroll
            for (int vb = 0; vb < VB; ++vb)
#pragma unroll
                for (int j = 0; j < 16; ++j) mx[w] = fmaxf(mx[w], s[vb][w][j]);
            mx[w] = half_wave_max(mx[w]);
            grows |= (mx[w] - m[w]) * dv.c > LAG;
        }
        if (__any(grows)) {  // seldom after the first tiles; by row, so that no row's bits depend on its neighbours
#pragma unroll
            for (int w = 0; w < CW; ++w) {
                const float up = (mx[w] - m[w]) * dv.c > LAG ? mx[w] : m[w], f = exp2_fast((m[w] - up) * dv.c);
                m[w] = up;
                l[w] *= f;
                if (GRAD)
#pragma unroll
                    for (int b = 0; b < DP / 32; ++b) out[w][b] *= f;
            }
        }
        float base[CW];
        bool far = false;
#pragma unroll
        for (int w = 0; w < CW; ++w) {
            base[w] = P_SHIFT - m[w] * dv.c;
            far |= fabsf(m[w] * dv.c) > FAR;
        }
        if (__any(far)) {  // the rounding of m c would show: subtract first
#pragma unroll
            for (int w = 0; w < CW; ++w) {
                const bool mine = fabsf(m[w] * dv.c) > FAR;
                const float less = mine ? m[w] : 0.0f;
                base[w] = mine ? P_SHIFT : base[w];
#pragma unroll
                for (int vb = 0; vb < VB; ++vb) s[vb][w] -= less;
            }
        }
#pragma unroll
        for (int vb = 0; vb < VB; ++vb)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                float p[CW][8];
#pragma unroll
                for (int w = 0; w < CW; ++w)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        p[w][j] = exp2_fast(__builtin_fmaf(s[vb][w][8 * kb + j], dv.c, base[w]));
                        l[w] += p[w][j];
                    }
                if (GRAD) accumulate<E, NS, DP, CW>(out, p, tile[buf], vb * 32 + kb * 16);
            }
        if (i + 1 < t1) store(i + 1, 0, buf ^ 1);
        __syncthreads();
        buf ^= 1;
    }
#pragma unroll
    for (int w = 0; w < CW; ++w) {
        const int64_t n = n0 + 32 * w;
        const float sum = half_wave_sum(l[w]);
        if (n >= a.rows) continue;
        const int64_t at = (int64_t)part * a.rows + n;
        if (h == 0) {
            const int64_t to = at + (WIDE ? (int64_t)blockIdx.y * a.splits * a.rows : 0);
            a.pm[to] = m[w];
            a.pl[to] = sum;
        }
        if (GRAD)
#pragma unroll
            for (int b = 0; b < DP / 32; ++b)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *(float4 *)(a.po + at * a.dp + (WIDE ? (int)blockIdx.y * DP : 0) + b * 32 + 8 * g + 4 * h) =
                        make_float4(out[w][b][4 * g], out[w][b][4 * g + 1], out[w][b][4 * g + 2], out[w][b][4 * g + 3]);
    }
}

template <typename T, typename E, int NS, int DP, int CW, bool WIDE>
__global__ __launch_bounds__(256, NS * DP >= 256 || DP >= 192 ? 1 : 2) void table_kernel(SweepArgs a)
{
    typedef Tile<E, NS, DP> Tl;
    typedef typename Half<E>::x8 x8;
    constexpr int NB = Tl::BV / 32;
    __shared__ __attribute__((aligned(16))) E tile[2][Tl::SIZE];
    __shared__ __attribute__((aligned(16))) float sm[2][Tl::BV], sr[2][Tl::BV], sg[2][Tl::BV], sf[2][Tl::BV];
    __shared__ __attribute__((aligned(16))) int32_t st[2][Tl::BV];
    const Derived dv = derive(NS == 2 ? a.scales : nullptr);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int part = blockIdx.x % a.splits;
    const int64_t w0 = (int64_t)(blockIdx.x / a.splits) * (128 * CW) + wave * (32 * CW), v0 = w0 + (lane & 31);
    const int64_t tiles = ceil_div(a.rows, Tl::BV);
    const int64_t t0 = tiles * part / a.splits, t1 = tiles * (part + 1) / a.splits;

    const int chunks = WIDE ? a.chunks : 1, first = WIDE ? (int)blockIdx.y + 1 : 0;
    auto offset = [&](int j) { return WIDE ? ((first + j) % chunks) * (NS * DP) : 0; };
    x8 own[CW][NS][DP / 16];
    auto take = [&](int j) {
#pragma unroll
        for (int w = 0; w < CW; ++w) load_owned<E, NS, DP>(own[w], (const E *)a.w + offset(j), a.ldw, v0 + 32 * w, a.vocab, dv.owned);
    };
    if (!WIDE) take(0);
    f32x16 out[CW][DP / 32];
    float bias[CW], db[CW];
#pragma unroll
    for (int w = 0; w < CW; ++w) {
        const int64_t v = v0 + 32 * w;
        bias[w] = a.bias && v < a.vocab ? bias_units(a.bias[v], dv) : 0.0f;
        db[w] = 0.0f;
#pragma unroll
        for (int b = 0; b < DP / 32; ++b) out[w][b] = (f32x16)(0.0f);
    }

    Tl t;
    float next_m = 0.0f, next_r = 0.0f, next_g = 0.0f;
    int32_t next_t = -1;
    auto fetch = [&](int64_t i, int j) {
        t.fetch((const E *)a.x + offset(j), a.ldx, i * Tl::BV, a.rows);
#pragma unroll
        for (int q = 0; q < Tl::PER; ++q) {  // a row without a target is not read: zeros in its place
            const int64_t n = i * Tl::BV + (q * 256 + (int)threadIdx.x) / Tl::CHUNKS;
            if (n < a.rows && a.row_target[n] < 0) t.held[q] = make_uint4(0, 0, 0, 0);
        }
        if (j == 0 && threadIdx.x < Tl::BV) {
            const int64_t n = i * Tl::BV + threadIdx.x;
            const bool ok = n < a.rows;
            next_m = ok ? a.row_max[n] : INFINITY;
            next_r = ok ? a.row_rate[n] : 0.0f;
            next_g = ok ? a.row_weight[n] : 0.0f;
            next_t = ok ? a.row_target[n] : -1;
        }
    };
    auto store = [&](int64_t i, int j, int buf) {
        t.store(tile[buf]);
        if (j == 0 && threadIdx.x < Tl::BV) {
            const int o = (int)(i - t0) & 1;
            const bool far = fabsf(next_m * dv.c) > FAR && next_m < INFINITY;
            sm[o][threadIdx.x] = far ? 0.0f : -next_m * dv.c;
            sf[o][threadIdx.x] = far ? next_m : 0.0f;
            sr[o][threadIdx.x] = next_r;
            sg[o][threadIdx.x] = next_g;
            st[o][threadIdx.x] = next_t;
        }
    };
    if (t0 < t1) {
        fetch(t0, 0);
        store(t0, 0, 0);
    }
    __syncthreads();
    int buf = 0;
    for (int64_t i = t0; i < t1; ++i) {
        const int o = (int)(i - t0) & 1;
        f32x16 s[NB][CW];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int w = 0; w < CW; ++w) s[nb][w] = (f32x16)(bias[w]);
        for (int j = 0; j < chunks - 1; ++j) {  // WIDE: the other chunks first
            take(j);
            fetch(i, j + 1);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) scores<E, NS, DP, CW>(s[nb], own, tile[buf], nb * 32);
            store(i, j + 1, buf ^ 1);
            __syncthreads();
            buf ^= 1;
        }
        if (WIDE) take(chunks - 1);
        if (i + 1 < t1) fetch(i + 1, 0);
        const int32_t mine = st[o][lane & (Tl::BV - 1)];
        const bool hits = __any(mine >= w0 && mine < w0 + 32 * CW);  // a target among this wave's table rows
        const bool far = __any(sf[o][lane & (Tl::BV - 1)] != 0.0f);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            scores<E, NS, DP, CW>(s[nb], own, tile[buf], nb * 32);
            if (far)  // see FAR
#pragma unroll
                for (int w = 0; w < CW; ++w)
#pragma unroll
                    for (int j = 0; j < 16; ++j) s[nb][w][j] -= sf[o][nb * 32 + 8 * (j / 4) + 4 * h + j % 4];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                float q[CW][8];
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const int r = nb * 32 + kb * 16 + 8 * g + 4 * h;
                    const float4 mm = *(const float4 *)&sm[o][r], rr = *(const float4 *)&sr[o][r];
                    const float ms[4] = {mm.x, mm.y, mm.z, mm.w}, rs[4] = {rr.x, rr.y, rr.z, rr.w};
#pragma unroll
                    for (int w = 0; w < CW; ++w)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            q[w][4 * g + j] = exp2_fast(__builtin_fmaf(s[nb][w][8 * kb + 4 * g + j], dv.c, ms[j])) * rs[j];
                    if (hits)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int w = 0; w < CW; ++w)
                                if ((int64_t)st[o][r + j] == v0 + 32 * w) q[w][4 * g + j] -= sg[o][r + j];
                }
#pragma unroll
                for (int w = 0; w < CW; ++w)
#pragma unroll
                    for (int j = 0; j < 8; ++j) db[w] += q[w][j];
                accumulate<E, NS, DP, CW>(out, q, tile[buf], nb * 32 + kb * 16);
            }
        }
        if (i + 1 < t1) store(i + 1, 0, buf ^ 1);
        __syncthreads();
        buf ^= 1;
    }
    const int shift = a.shifted == 2 ? a.scales->eg - 14 : a.shifted ? -14 : 0, kx = NS == 2 ? a.scales->kx : 0;
    const int c0 = WIDE ? (int)blockIdx.y * DP : 0;
#pragma unroll
    for (int w = 0; w < CW; ++w) {
        const int64_t v = v0 + 32 * w;
        const float total = half_wave_sum(db[w]);
        if (v >= a.vocab) continue;
        if (a.splits > 1) {
            const int64_t at = (int64_t)part * a.vocab + v;
            if (h == 0 && c0 == 0) a.pb[at] = total;
#pragma unroll
            for (int b = 0; b < DP / 32; ++b)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *(float4 *)(a.pw + at * a.dp + c0 + b * 32 + 8 * g + 4 * h) =
                        make_float4(out[w][b][4 * g], out[w][b][4 * g + 1], out[w][b][4 * g + 2], out[w][b][4 * g + 3]);
        } else {
            if (a.db && h == 0 && c0 == 0) a.db[v] = ldexpf(total, shift);
            T *row = (T *)a.dw + v * a.d;
#pragma unroll
            for (int b = 0; b < DP / 32; ++b)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int c = c0 + b * 32 + 8 * g + 4 * h;
                    Vec<T, 4> o;
#pragma unroll
                    for (int j = 0; j < 4; ++j) o.v[j] = (T)ldexpf(out[w][b][4 * g + j], shift - kx);
                    if (c + 4 <= a.d && (a.d & 3) == 0) *(Vec<T, 4> *)(row + c) = o;
                    else
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (c + j < a.d) row[c + j] = o.v[j];
                }
        }
    }
}

// ------------------------------------------------------------------- joins ---

struct JoinArgs {
    lfm_softmax_args a;
    const Scales *scales;
    const uint8_t *outlier;
    int splits, dp, ns, grad, shifted;
    const float *pm, *pl, *po;
    float *row_max, *row_rate, *row_weight;
    int32_t *row_target;
};

__device__ inline float wave_sum(float v)
{
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

__device__ inline float wave_max(float v)
{
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

template <typename T>
__device__ inline float dot_lane(const T *x, const T *w, int d)
{
    float s = 0.0f;
    for (int c = 0; c < d; ++c) s = __builtin_fmaf((float)x[c], (float)w[c], s);
    return s;
}

// One wave per row: joins the parts of the table, finishes lse, loss, dx, and leaves table_kernel what it needs.
template <typename T>
__global__ __launch_bounds__(256) void join_rows_kernel(JoinArgs j)
{
    const lfm_softmax_args &a = j.a;
    const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (n >= a.rows) return;
    const int lane = threadIdx.x & 63;
    const Derived dv = derive(j.ns == 2 ? j.scales : nullptr);
    float m = -INFINITY;
    for (int s = lane; s < j.splits; s += 64) m = fmaxf(m, j.pm[(int64_t)s * a.rows + n]);
    m = wave_max(m);
    float l = 0.0f;
    for (int s = lane; s < j.splits; s += 64)
        l += j.pl[(int64_t)s * a.rows + n] * exp2_fast((j.pm[(int64_t)s * a.rows + n] - m) * dv.c);
    l = wave_sum(l);
    const T *x = (const T *)a.hidden + n * a.hidden_stride;
    float lse = l == 0.0f ? -INFINITY : m <= dv.low * 0.999f ? -3.402823466e38f : ldexpf(m, -dv.k) + (logf(l) - P_SHIFT * LN2);
    const bool odd = j.ns == 2 && j.outlier[n];
    if (odd) {  // a row beyond x's scale: not finite, or without a target and far larger than the others
        bool finite = true;
        for (int c = lane; c < a.d; c += 64) finite &= fabsf((float)x[c]) < INFINITY;
        lse = NAN;
        if (__all(finite)) {
            float top = -INFINITY, sum = 0.0f;
            for (int64_t v = lane; v < a.vocab; v += 64) {
                const float s = dot_lane(x, (const T *)a.table + v * a.table_stride, a.d) + (a.bias ? a.bias[v] : 0.0f);
                const float up = fmaxf(top, s);
                if (up > -INFINITY) sum = sum * expf(top - up) + expf(s - up);
                top = up;
            }
            const float up = wave_max(top);
            sum = wave_sum(top > -INFINITY ? sum * expf(top - up) : 0.0f);
            lse = up + logf(sum);
        }
    }
    const int64_t t = target_of(a, n);
    const float g = t < 0 ? 0.0f : a.weights ? a.weights[n] : 1.0f;
    float loss = 0.0f;
    const T *wt = (const T *)a.table + (t < 0 ? 0 : t) * a.table_stride;
    if (t >= 0) {
        float s = 0.0f;
        for (int c = lane; c < a.d; c += 64) s = __builtin_fmaf((float)x[c], (float)wt[c], s);
        s = wave_sum(s);
        if (a.bias) s += a.bias[t];
        loss = s == -INFINITY ? INFINITY : lse - s;
        loss *= g;
    }
    if (lane == 0) {
        a.lse[n] = lse;
        a.loss[n] = loss;
    }
    if (!j.grad) return;
    const bool lost = odd && t >= 0;  // not finite: its gradients are not either
    if (lane == 0) {
        const int shift = j.shifted == 2 ? 14 - j.scales->eg : j.shifted ? 14 : 0;
        const float gs = ldexpf(g, shift);
        j.row_target[n] = (int32_t)t;
        j.row_max[n] = t < 0 ? INFINITY : m;
        j.row_rate[n] = lost ? NAN : t < 0 || l == 0.0f ? 0.0f : gs * exp2_fast(P_SHIFT) / l;
        j.row_weight[n] = gs;
    }
    const int kw = j.ns == 2 ? j.scales->kw : 0;
    for (int c = lane; c < a.d; c += 64) {
        float o = 0.0f;
        if (t >= 0) {
            const float *pm = j.pm + (int64_t)(c >> 8) * j.splits * a.rows;  // the maxima that chunk c / 256 went by
            for (int s = 0; s < j.splits; ++s) {
                const int64_t at = (int64_t)s * a.rows + n;
                o += j.po[at * j.dp + c] * exp2_fast((pm[at] - m) * dv.c);
            }
            o = l == 0.0f ? 0.0f : ldexpf(o / l, -kw);
            o = lost ? NAN : g * (o - (float)wt[c]);
        }
        ((T *)a.d_hidden)[n * a.d + c] = (T)o;
    }
}

// dw and db from the parts of the rows, added in order
template <typename T>
__global__ __launch_bounds__(256) void join_table_kernel(SweepArgs a, int dp, int ns)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, v = i / a.d;
    if (v >= a.vocab) return;
    const int c = (int)(i - v * a.d);
    const int shift = a.shifted == 2 ? a.scales->eg - 14 : a.shifted ? -14 : 0, kx = ns == 2 ? a.scales->kx : 0;
    float s = 0.0f;
    for (int p = 0; p < a.splits; ++p) s += a.pw[((int64_t)p * a.vocab + v) * dp + c];
    ((T *)a.dw)[i] = (T)ldexpf(s, shift - kx);
    if (c == 0 && a.db) {
        float b = 0.0f;
        for (int p = 0; p < a.splits; ++p) b += a.pb[(int64_t)p * a.vocab + v];
        a.db[v] = ldexpf(b, shift);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void clear_kernel(T *p, int64_t n, float *q, int64_t m)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = (T)0.0f;
    if (q && i < m) q[i] = 0.0f;
}

// -------------------------------------------------------------------- host ---

struct Plan {
    int dp, ns, cw;
    int chunks;             // of 256 columns
    int bv;                 // rows of a streamed tile
    int row_splits, table_splits;
    bool largest;           // scales are wanted (float32 operands; float16 with weights)
};

int width_for(int d)
{
    const int widths[] = {32, 64, 96, 128, 192, 256};
    for (int w : widths)
        if (d <= w) return w;
    return (d + 255) / 256 * 256;
}

int splits_for(int64_t owners, int64_t tiles, int64_t slots)
{
    int64_t s = slots / owners;
    if (s < 1) s = 1;
    if (s > 8) s = s / 8 * 8;  // a part of the streamed side then stays with one XCD's L2
    if (s > tiles) s = tiles;
    if (s < 1) s = 1;
    return (int)s;
}

Plan plan_for(int64_t rows, int64_t vocab, int d, int dtype, bool weights)
{
    Plan p;
    p.dp = width_for(d);
    p.ns = dtype == LFM_F32 ? 2 : 1;
    p.cw = 1;
    p.chunks = p.dp > 256 ? p.dp / 256 : 1;
    p.bv = p.ns * p.dp <= 128 ? 64 : 32;
    p.largest = dtype == LFM_F32 || (dtype == LFM_F16 && weights);
    p.row_splits = splits_for(ceil_div(rows < 1 ? 1 : rows, 128 * p.cw), ceil_div(vocab, p.bv), 512);
    p.table_splits = splits_for(ceil_div(vocab, 128 * p.cw), ceil_div(rows < 1 ? 1 : rows, p.bv), 512);
    return p;
}

struct Space {
    Scales *scales;
    float *largest;
    uint8_t *outlier;
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
    Space s;
    s.scales = c.take<Scales>(1);
    s.largest = c.take<float>(3 * MAX_PARTS);
    s.outlier = c.take<uint8_t>(rows);
    s.x = c.take<uint16_t>(rows * p.ns * p.dp);
    s.w = c.take<uint16_t>(vocab * p.ns * p.dp);
    s.pm = c.take<float>(rows * p.row_splits * p.chunks);
    s.pl = c.take<float>(rows * p.row_splits * p.chunks);
    s.po = c.take<float>(grad ? rows * p.row_splits * p.dp : 0);
    s.pw = c.take<float>(grad && p.table_splits > 1 ? vocab * p.table_splits * p.dp : 0);
    s.pb = c.take<float>(grad && p.table_splits > 1 ? vocab * p.table_splits : 0);
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
    const dim3 grid((unsigned)(ceil_div(s.rows, 128) * s.splits), WIDE && grad ? (unsigned)s.chunks : 1);
    if (grad) rows_kernel<E, NS, DP, 1, true, WIDE><<<grid, 256, 0, st>>>(s);
    else rows_kernel<E, NS, DP, 1, false, WIDE><<<grid, 256, 0, st>>>(s);
    return hipGetLastError();
}

template <typename T, typename E, int NS, int DP, bool WIDE>
hipError_t sweep_table(const SweepArgs &s, hipStream_t st)
{
    const dim3 grid((unsigned)(ceil_div(s.vocab, 128) * s.splits), WIDE ? (unsigned)s.chunks : 1);
    table_kernel<T, E, NS, DP, 1, WIDE><<<grid, 256, 0, st>>>(s);
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

template <typename T, typename E, int NS>
hipError_t run(const lfm_softmax_args &a, bool grad, void *ws, hipStream_t st)
{
    const Plan p = plan_for(a.rows, a.vocab, a.d, a.dtype, a.weights != nullptr);
    const Space s = space_for(p, a.rows, a.vocab, grad, ws);
    hipError_t e;
    if (a.rows == 0) {
        if (!grad) return hipSuccess;
        clear_kernel<T><<<dim3((unsigned)ceil_div(a.vocab * a.d, 256)), 256, 0, st>>>((T *)a.d_table, a.vocab * a.d, a.d_bias, a.vocab);
        return hipGetLastError();
    }
    const bool scales = p.largest && (grad || NS == 2);
    auto in_place = [&](const void *q, int64_t stride) { return NS == 1 && a.d == p.dp && stride % 8 == 0 && ((uintptr_t)q & 15) == 0; };
    const bool x_there = in_place(a.hidden, a.hidden_stride), w_there = in_place(a.table, a.table_stride);
    PackArgs pk;
    pk.a = a;
    pk.largest = scales ? s.largest : nullptr;
    pk.tensors = NS == 2 ? 3 : 1;
    pk.scales = s.scales;
    pk.x = x_there ? nullptr : s.x;
    pk.w = w_there ? nullptr : s.w;
    pk.outlier = s.outlier;
    const int64_t most = NS == 2 ? (a.rows > a.vocab ? a.rows : a.vocab) * a.d : a.rows;
    pk.parts = (int)(ceil_div(most, 4096) < MAX_PARTS ? ceil_div(most, 4096) : MAX_PARTS);
    if (scales) {
        largest_kernel<T><<<dim3((unsigned)(pk.tensors * pk.parts)), 256, 0, st>>>(a, pk.parts, s.largest, pk.tensors);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (NS == 2) {
        clear_kernel<uint8_t><<<dim3((unsigned)ceil_div(a.rows, 256)), 256, 0, st>>>(s.outlier, a.rows, nullptr, 0);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (scales || pk.x || pk.w) {
        const int64_t work = ((pk.x ? a.rows : 0) + (pk.w ? a.vocab : 0)) * (p.dp / 8);
        int64_t blocks = ceil_div(work, 256);
        blocks = blocks < 1 ? 1 : blocks > 4096 ? 4096 : blocks;
        pack_kernel<T, E, NS><<<dim3((unsigned)blocks), 256, 0, st>>>(pk, p.dp, p.dp < 256 ? p.dp : 256);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    SweepArgs w;
    w.x = x_there ? a.hidden : s.x;
    w.ldx = x_there ? a.hidden_stride : NS * p.dp;
    w.w = w_there ? a.table : s.w;
    w.ldw = w_there ? a.table_stride : NS * p.dp;
    w.rows = a.rows;
    w.vocab = a.vocab;
    w.bias = a.bias;
    w.scales = s.scales;
    w.splits = p.row_splits;
    w.d = a.d;
    w.dp = p.dp;
    w.chunks = p.chunks;
    w.pm = s.pm;
    w.pl = s.pl;
    w.po = s.po;
    w.row_max = s.row_max;
    w.row_rate = s.row_rate;
    w.row_weight = s.row_weight;
    w.row_target = s.row_target;
    w.dw = a.d_table;
    w.db = a.d_bias;
    w.pw = s.pw;
    w.pb = s.pb;
    w.shifted = scales ? 2 : a.dtype == LFM_F16 ? 1 : 0;
#define ROWS(DP, WIDE) sweep_rows<E, NS, DP, WIDE>(w, grad, st)
    BY_WIDTH(p.dp, ROWS)
    if (e != hipSuccess) return e;
    JoinArgs j;
    j.a = a;
    j.scales = s.scales;
    j.outlier = s.outlier;
    j.splits = p.row_splits;
    j.dp = p.dp;
    j.ns = NS;
    j.grad = grad ? 1 : 0;
    j.shifted = w.shifted;
    j.pm = s.pm;
    j.pl = s.pl;
    j.po = s.po;
    j.row_max = s.row_max;
    j.row_rate = s.row_rate;
    j.row_weight = s.row_weight;
    j.row_target = s.row_target;
    join_rows_kernel<T><<<dim3((unsigned)ceil_div(a.rows, 4)), 256, 0, st>>>(j);
    if ((e = hipGetLastError()) != hipSuccess || !grad) return e;
    w.splits = p.table_splits;
#define TABLE(DP, WIDE) sweep_table<T, E, NS, DP, WIDE>(w, st)
    BY_WIDTH(p.dp, TABLE)
    if (e != hipSuccess || p.table_splits == 1) return e;
    join_table_kernel<T><<<dim3((unsigned)ceil_div(a.vocab * a.d, 256)), 256, 0, st>>>(w, p.dp, NS);
    return hipGetLastError();
}

}  // namespace

int64_t softmax_workspace(int64_t rows, int64_t vocab, int d, int dtype, bool grad)
{
    return space_for(plan_for(rows, vocab, d, dtype, true), rows, vocab, grad, nullptr).bytes;
}

hipError_t softmax_loss(const lfm_softmax_args &a, bool grad, void *ws, hipStream_t st)
{
    return a.dtype == LFM_F32 ? run<float, f16_t, 2>(a, grad, ws, st)
         : a.dtype == LFM_BF16 ? run<bf16_t, bf16_t, 1>(a, grad, ws, st) : run<f16_t, f16_t, 1>(a, grad, ws, st);
}

}  // namespace ops
}  // namespace lfm
