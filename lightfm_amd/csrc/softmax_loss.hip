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

#ifndef LFM_ROWS_WAVES
#define LFM_ROWS_WAVES 2
#endif
#ifndef LFM_TABLE_WAVES
#define LFM_TABLE_WAVES 2
#endif

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
// tile are in flight while this one is used.  A row takes NS DP + 16 halves of LDS: neighbouring rows then start 8 banks
// apart (modulo 64, in some order), which serves the 16-byte reads of 8 rows and the transposing reads of 4 x 32 bytes
// without conflicts.
template <typename E, int NS, int DP>
struct Tile {
    static constexpr int BV = NS * DP <= 128 ? 64 : 32, ROW = NS * DP + 16, CHUNKS = NS * DP / 8, PER = BV * CHUNKS / 256;
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

// Eight float32 values to a matrix operand: rounded to nearest (bf16, f16), or split into two float16 (hi towards zero, two
// values per instruction; the remainder is exact and keeps 11 bits more).
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

template <typename E, int NS, int CW>
struct Values {  // the probabilities of 32 streamed rows as matrix operands
    typename Half<E>::x8 hi[CW][2], lo[NS == 2 ? CW : 1][2];
};

template <typename E, int NS, int CW>
__device__ inline void clear_values(Values<E, NS, CW> &p)
{
#pragma unroll
    for (int w = 0; w < CW; ++w)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            p.hi[w][k] = (typename Half<E>::x8)((E)0.0f);
            if (NS == 2) p.lo[w][k] = (typename Half<E>::x8)((E)0.0f);
        }
}

template <typename E, int NS, int CW>
__device__ inline void pack_values(Values<E, NS, CW> &p, const float (&v)[CW][8], int k)
{
#pragma unroll
    for (int w = 0; w < CW; ++w)
        if constexpr (NS == 2) {
            float rest[8];
            p.hi[w][k] = cut_values(v[w]);
#pragma unroll
            for (int j = 0; j < 8; ++j) rest[j] = __builtin_fmaf((float)p.hi[w][k][j], -1.0f, v[w][j]);
            p.lo[w][k] = cut_values(rest);
        } else
            p.hi[w][k] = round_values(v[w], typename Half<E>::x8());
}

// out[d, owned] += tile^T x values for 32 rows of the tile (from row r0)
template <typename E, int NS, int DP, int CW>
__device__ inline void accumulate(f32x16 (&out)[CW][DP / 32], const Values<E, NS, CW> &p, const E *tile, int r0)
{
    typedef typename Half<E>::x8 x8;
    typedef typename Half<E>::x4 x4;
    constexpr int ROW = Tile<E, NS, DP>::ROW;
    const int lane = threadIdx.x & 63;
    const E *at = tile + (r0 + 4 * (lane >> 5) + ((lane & 15) >> 2)) * ROW + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int b = 0; b < DP / 32; ++b) {
            const E *c = at + k * 16 * ROW + b * 32;
            const x4 h0 = read_column(c), h1 = read_column(c + 8 * ROW);
            const x8 th = __builtin_shufflevector(h0, h1, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
            for (int w = 0; w < CW; ++w) out[w][b] = mfma(th, p.hi[w][k], out[w][b]);
            if (NS == 2) {
                const x4 l0 = read_column(c + DP), l1 = read_column(c + DP + 8 * ROW);
                const x8 tl = __builtin_shufflevector(l0, l1, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                for (int w = 0; w < CW; ++w) {
                    out[w][b] = mfma(tl, p.hi[w][k], out[w][b]);
                    out[w][b] = mfma(th, p.lo[w][k], out[w][b]);
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
    const void *targets;    // rows_kernel: [rows], id_bytes wide
    int id_bytes;
    int splits;             // parts of the streamed side
    int d, dp;
    int chunks;             // of 256 columns (WIDE; else 1): the second product's columns are blockIdx.y's
    // rows_kernel: per chunk, part and row, the row's target left out
    float *pm, *pl, *po;    // maximum (matrix units), sum of 2^7 p; per part and row: sum of 2^7 p w [dp]
    // table_kernel: per row
    const float *row_max, *row_rate, *row_weight;  // maximum (matrix units; +inf: no target), 2^shift g / sum, 2^shift g (1 - p[target])
    const int32_t *row_target;
    void *dw;               // one part: the result
    float *db, *pw, *pb;    // several: partial sums per part [vocab][dp], [vocab]
    int shifted;            // q is scaled by 2^(14 - eg): 0 no (bfloat16), 1 with eg = 0, 2 with eg of scales
};

// Both sweeps are pipelined over blocks of 32 streamed rows: a step makes the scores of block b + 1 and the second product
// of block b - 1 on the matrix cores while the vector units turn the scores of block b into probabilities.  None of the
// three waits for another, so a wave keeps both busy by itself.  Tiles rotate through BUFS buffers of LDS, so that a tile
// is free again two steps after its last score and one barrier per tile does.
template <typename E, int NS, int DP>
struct Rotation {
    static constexpr int BLOCKS = Tile<E, NS, DP>::BV / 32, BUFS = BLOCKS == 2 ? 3 : 4;
    // tiles stored ahead of the first step, before which the next tile is stored
    static constexpr int AHEAD = BLOCKS == 2 ? 1 : 2;
};

// What a step has to hide: one matrix instruction, an LDS read, a few vector instructions, and so on
template <int MATRIX, int VECTOR>
__device__ inline void interleave()
{
#ifndef LFM_NO_INTERLEAVE
#pragma unroll
    for (int i = 0; i < MATRIX; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, VECTOR, 0);
    }
#endif
}

template <typename E, int NS, int DP, int CW, bool GRAD>
__global__ __launch_bounds__(256, (GRAD ? NS * DP >= 384 : NS * DP >= 512) ? 1 : LFM_ROWS_WAVES) void rows_kernel(SweepArgs a)
{
    typedef Tile<E, NS, DP> Tl;
    typedef Rotation<E, NS, DP> Ro;
    typedef typename Half<E>::x8 x8;
    __shared__ __attribute__((aligned(16))) E tile[Ro::BUFS][Tl::SIZE];
    __shared__ __attribute__((aligned(16))) float sb[Ro::BUFS][Tl::BV];
    const Derived dv = derive(NS == 2 ? a.scales : nullptr);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const uint32_t part = blockIdx.x % (uint32_t)a.splits;
    const int64_t n0 = (int64_t)(blockIdx.x / (uint32_t)a.splits) * (128 * CW) + wave * (32 * CW) + (lane & 31);
    const uint32_t tiles = (uint32_t)((a.vocab + Tl::BV - 1) / Tl::BV);
    const uint32_t t0 = (uint32_t)((uint64_t)tiles * part / (uint32_t)a.splits);
    const int nt = (int)((uint64_t)tiles * (part + 1) / (uint32_t)a.splits) - (int)t0;

    x8 own[CW][NS][DP / 16];
    f32x16 out[CW][DP / 32], cur[CW], next[CW];
    Values<E, NS, CW> p;
    float m[CW], l[CW];
    int32_t target[CW];
#pragma unroll
    for (int w = 0; w < CW; ++w) {
        const int64_t n = n0 + 32 * w;
        load_owned<E, NS, DP>(own[w], (const E *)a.x, a.ldx, n, a.rows, dv.owned);
        const int64_t at = n >= a.rows ? -1 : a.id_bytes == 8 ? ((const int64_t *)a.targets)[n] : (int64_t)((const int32_t *)a.targets)[n];
        target[w] = (uint64_t)at < (uint64_t)a.vocab ? (int32_t)at - 4 * h : INT32_MIN / 2;
        m[w] = dv.low * 1.01f;
        l[w] = 0.0f;
        if (GRAD) {
#pragma unroll
            for (int b = 0; b < DP / 32; ++b) out[w][b] = (f32x16)(0.0f);
        }
    }
    clear_values(p);

    Tl t;
    float next_bias = 0.0f;
    auto fetch = [&](int i) {
        const int64_t r = (int64_t)(t0 + i) * Tl::BV;
        t.fetch((const E *)a.w, a.ldw, r, a.vocab);
        const int64_t v = r + threadIdx.x;
        if (threadIdx.x < Tl::BV) next_bias = v >= a.vocab ? -INFINITY : a.bias ? bias_units(a.bias[v], dv) : 0.0f;
    };
    auto store = [&](int buf) {
        t.store(tile[buf]);
        if (threadIdx.x < Tl::BV) sb[buf][threadIdx.x] = next_bias;
    };
    auto score = [&](f32x16 (&s)[CW], int buf, int r0) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float4 b = *(const float4 *)&sb[buf][r0 + 8 * g + 4 * h];
#pragma unroll
            for (int w = 0; w < CW; ++w) {
                s[w][4 * g + 0] = b.x;
                s[w][4 * g + 1] = b.y;
                s[w][4 * g + 2] = b.z;
                s[w][4 * g + 3] = b.w;
            }
        }
        scores<E, NS, DP, CW>(s, own, tile[buf], r0);
    };
    // the step of the block whose first vocabulary row is v: before_* the block before it, after_* the one behind it
    auto step = [&](int32_t v, int before, int before_r, int after, int after_r) {
        // the target's own score is left to the join, in float32: what remains is not a difference of near-equals
        bool here = false;
#pragma unroll
        for (int w = 0; w < CW; ++w) here |= (uint32_t)target[w] + 4 * h - (uint32_t)v < 32u;
        if (__any(here)) {  // one block in some
#pragma unroll
            for (int w = 0; w < CW; ++w)
#pragma unroll
                for (int j = 0; j < 16; ++j) cur[w][j] = (uint32_t)target[w] - (uint32_t)v == 8u * (j / 4) + j % 4 ? -INFINITY : cur[w][j];
        }
        bool grows = false;
        float mx[CW];
#pragma unroll
        for (int w = 0; w < CW; ++w) {
            mx[w] = cur[w][0];
#pragma unroll
            for (int j = 1; j < 16; ++j) mx[w] = fmaxf(mx[w], cur[w][j]);
            mx[w] = half_wave_max(mx[w]);
            grows |= (mx[w] - m[w]) * dv.c > LAG;
        }
        if (__any(grows)) {  // seldom after the first blocks; by row, so that no row's bits depend on its neighbours
            if (GRAD) {
                accumulate<E, NS, DP, CW>(out, p, tile[before], before_r);  // still about the old maximum
                clear_values(p);
            }
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
                cur[w] -= less;
            }
        }
        score(next, after, after_r);
        if (GRAD) accumulate<E, NS, DP, CW>(out, p, tile[before], before_r);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float v8[CW][8];
#pragma unroll
            for (int w = 0; w < CW; ++w)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v8[w][j] = exp2_fast(__builtin_fmaf(cur[w][8 * k + j], dv.c, base[w]));
                    l[w] += v8[w][j];
                }
            if (GRAD) pack_values<E, NS, CW>(p, v8, k);
        }
        constexpr int MATRIX = CW * (NS == 2 ? 3 : 1) * (DP / 16) * (GRAD ? 2 : 1), VECTOR = CW * (GRAD ? NS == 2 ? 96 : 72 : 56);
        interleave<MATRIX, (VECTOR + MATRIX - 1) / MATRIX>();
#pragma unroll
        for (int w = 0; w < CW; ++w) cur[w] = next[w];
    };

    if (nt > 0) {
        fetch(0);
        store(0);
        if (Ro::AHEAD == 2 && nt > 1) {
            fetch(1);
            store(1);
        }
        if (nt > Ro::AHEAD) fetch(Ro::AHEAD);
        __syncthreads();
        score(cur, 0, 0);
    }
    int b0 = 0, b1 = 1, before = 0;  // the buffers of tile i, i + 1, i - 1
    for (int i = 0; i < nt; ++i) {
        int b2 = b1 + 1 == Ro::BUFS ? 0 : b1 + 1;
        const int into = Ro::BLOCKS == 2 ? b1 : b2;
        if (i + Ro::AHEAD < nt) store(into);
        if (i + Ro::AHEAD + 1 < nt) fetch(i + Ro::AHEAD + 1);
        const int32_t v = (int32_t)((t0 + i) * Tl::BV);
        const int after = i + 1 < nt ? b1 : b0;  // (behind the last block: scores that nobody looks at)
        if (Ro::BLOCKS == 2) {
            step(v, before, i ? 32 : 0, b0, 32);
            __syncthreads();
            step(v + 32, b0, 0, after, 0);
        } else {
            step(v, before, 0, after, 0);
            __syncthreads();
        }
        before = b0;
        b0 = b1;
        b1 = b2;
    }
    if (GRAD && nt > 0) accumulate<E, NS, DP, CW>(out, p, tile[before], Tl::BV - 32);
#pragma unroll
    for (int w = 0; w < CW; ++w) {
        const int64_t n = n0 + 32 * w;
        const float sum = half_wave_sum(l[w]);
        if (n >= a.rows) continue;
        const int64_t at = (int64_t)part * a.rows + n;
        if (h == 0) {
            a.pm[at] = m[w];
            a.pl[at] = sum;
        }
        if (GRAD)
#pragma unroll
            for (int b = 0; b < DP / 32; ++b)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *(float4 *)(a.po + at * DP + b * 32 + 8 * g + 4 * h) =
                        make_float4(out[w][b][4 * g], out[w][b][4 * g + 1], out[w][b][4 * g + 2], out[w][b][4 * g + 3]);
    }
}

// Writes a wave's part of dw (or its partial sums) and db
template <typename T, int NS, int DP, int CW>
__device__ inline void write_table(const SweepArgs &a, const f32x16 (&out)[CW][DP / 32], const float (&db)[CW], int64_t v0, int64_t part, int c0)
{
    const int h = (threadIdx.x & 63) >> 5;
    const int shift = a.shifted == 2 ? a.scales->eg - 14 : a.shifted ? -14 : 0, kx = NS == 2 ? a.scales->kx : 0;
#pragma unroll
    for (int w = 0; w < CW; ++w) {
        const int64_t v = v0 + 32 * w;
        const float total = half_wave_sum(db[w]);
        if (v >= a.vocab) continue;
        if (a.splits > 1) {
            const int64_t at = part * a.vocab + v;
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

// What table_kernel needs to know of the rows of a tile
template <int BV>
struct RowFacts {
    float m[BV];        // -maximum in base 2 (0 where FAR is about the row)
    float rate[BV];     // 2^shift g / sum
    float weight[BV];   // 2^shift g (1 - p[target])
    float far[BV];      // the maximum in matrix units where FAR is about the row, else 0
    int32_t target[BV];
};

// The rare part of a block of scores: rows whose target is among the owned table rows leave the sum here and enter it as
// -g (1 - p) x, in float32; rows that FAR is about lose their maximum first.
template <typename E, int NS, int DP, int CW, int BV>
__device__ inline void special_rows(f32x16 (&s)[CW], f32x16 (&out)[CW][DP / 32], float (&db)[CW], const RowFacts<BV> &f, const E *tile, int r0,
                                    int32_t w0, bool hit)
{
    const int lane = threadIdx.x & 63, h = lane >> 5;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const int r = r0 + 8 * (j / 4) + 4 * h + j % 4;
#pragma unroll
        for (int w = 0; w < CW; ++w) s[w][j] = f.target[r] == w0 + (lane & 31) + 32 * w ? -INFINITY : s[w][j] - f.far[r];
    }
    uint32_t hits = (uint32_t)__ballot(hit);  // (the half-waves say the same)
    while (hits) {
        const int r = r0 + __ffs(hits) - 1;
        hits &= hits - 1;
        const int32_t at = f.target[r] - w0 - (lane & 31);
        const float g = f.weight[r];
        const E *x = tile + r * Tile<E, NS, DP>::ROW + 4 * h;
#pragma unroll
        for (int w = 0; w < CW; ++w) {
            const float mg = at == 32 * w ? g : 0.0f;
            if (h == 0) db[w] -= mg;
#pragma unroll
            for (int b = 0; b < DP / 32; ++b)
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int c = b * 32 + 8 * (j / 4) + j % 4;
                    const float xv = NS == 2 ? (float)x[c] + (float)x[(NS - 1) * DP + c] : (float)x[c];
                    out[w][b][j] = __builtin_fmaf(-mg, xv, out[w][b][j]);
                }
        }
    }
}

template <typename T, typename E, int NS, int DP, int CW>
__global__ __launch_bounds__(256, NS * DP >= 384 ? 1 : LFM_TABLE_WAVES) void table_kernel(SweepArgs a)
{
    typedef Tile<E, NS, DP> Tl;
    typedef Rotation<E, NS, DP> Ro;
    typedef typename Half<E>::x8 x8;
    __shared__ __attribute__((aligned(16))) E tile[Ro::BUFS][Tl::SIZE];
    __shared__ __attribute__((aligned(16))) RowFacts<Tl::BV> facts[Ro::BUFS];
    const Derived dv = derive(NS == 2 ? a.scales : nullptr);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const uint32_t part = blockIdx.x % (uint32_t)a.splits;
    const int64_t w0 = (int64_t)(blockIdx.x / (uint32_t)a.splits) * (128 * CW) + wave * (32 * CW), v0 = w0 + (lane & 31);
    const uint32_t tiles = (uint32_t)((a.rows + Tl::BV - 1) / Tl::BV);
    const uint32_t t0 = (uint32_t)((uint64_t)tiles * part / (uint32_t)a.splits);
    const int nt = (int)((uint64_t)tiles * (part + 1) / (uint32_t)a.splits) - (int)t0;

    x8 own[CW][NS][DP / 16];
    f32x16 out[CW][DP / 32], cur[CW], next[CW];
    Values<E, NS, CW> q;
    float bias[CW], db[CW];
#pragma unroll
    for (int w = 0; w < CW; ++w) {
        const int64_t v = v0 + 32 * w;
        load_owned<E, NS, DP>(own[w], (const E *)a.w, a.ldw, v, a.vocab, dv.owned);
        bias[w] = a.bias && v < a.vocab ? bias_units(a.bias[v], dv) : 0.0f;
        db[w] = 0.0f;
#pragma unroll
        for (int b = 0; b < DP / 32; ++b) out[w][b] = (f32x16)(0.0f);
    }
    clear_values(q);

    Tl t;
    bool keep[Tl::PER];
    float next_m = 0.0f, next_r = 0.0f, next_g = 0.0f;
    int32_t next_t = -1;
    auto fetch = [&](int i) {
        const int64_t r = (int64_t)(t0 + i) * Tl::BV;
        t.fetch((const E *)a.x, a.ldx, r, a.rows);
#pragma unroll
        for (int k = 0; k < Tl::PER; ++k) {
            const int64_t n = r + (k * 256 + (int)threadIdx.x) / Tl::CHUNKS;
            keep[k] = n < a.rows && a.row_target[n] >= 0;
        }
        if (threadIdx.x < Tl::BV) {
            const int64_t n = r + threadIdx.x;
            const bool ok = n < a.rows;
            next_m = ok ? a.row_max[n] : INFINITY;
            next_r = ok ? a.row_rate[n] : 0.0f;
            next_g = ok ? a.row_weight[n] : 0.0f;
            next_t = ok ? a.row_target[n] : -1;
        }
    };
    auto store = [&](int buf) {
#pragma unroll
        for (int k = 0; k < Tl::PER; ++k)  // a row without a target is not read: zeros in its place
            if (!keep[k]) t.held[k] = make_uint4(0, 0, 0, 0);
        t.store(tile[buf]);
        if (threadIdx.x < Tl::BV) {
            const bool far = fabsf(next_m * dv.c) > FAR && next_m < INFINITY;
            RowFacts<Tl::BV> &f = facts[buf];
            f.m[threadIdx.x] = far ? 0.0f : -next_m * dv.c;
            f.far[threadIdx.x] = far ? next_m : 0.0f;
            f.rate[threadIdx.x] = next_r;
            f.weight[threadIdx.x] = next_g;
            f.target[threadIdx.x] = next_t;
        }
    };
    auto score = [&](f32x16 (&s)[CW], int buf, int r0) {
#pragma unroll
        for (int w = 0; w < CW; ++w) s[w] = (f32x16)(bias[w]);
        scores<E, NS, DP, CW>(s, own, tile[buf], r0);
    };
    auto step = [&](int here, int r0, int before, int before_r, int after, int after_r) {
        const RowFacts<Tl::BV> &f = facts[here];
        const bool hit = (uint32_t)(f.target[r0 + (lane & 31)] - (int32_t)w0) < 32u * CW;
        if (__any(hit || f.far[r0 + (lane & 31)] != 0.0f))  // seldom
            special_rows<E, NS, DP, CW, Tl::BV>(cur, out, db, f, tile[here], r0, (int32_t)w0, hit);
        score(next, after, after_r);
        accumulate<E, NS, DP, CW>(out, q, tile[before], before_r);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float v8[CW][8];
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const int r = r0 + k * 16 + 8 * g + 4 * h;
                const float4 mm = *(const float4 *)&f.m[r], rr = *(const float4 *)&f.rate[r];
                const float ms[4] = {mm.x, mm.y, mm.z, mm.w}, rs[4] = {rr.x, rr.y, rr.z, rr.w};
#pragma unroll
                for (int w = 0; w < CW; ++w)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float v = exp2_fast(__builtin_fmaf(cur[w][8 * k + 4 * g + j], dv.c, ms[j])) * rs[j];
                        db[w] += v;
                        v8[w][4 * g + j] = v;
                    }
            }
            pack_values<E, NS, CW>(q, v8, k);
        }
        constexpr int MATRIX = 2 * CW * (NS == 2 ? 3 : 1) * (DP / 16), VECTOR = CW * (NS == 2 ? 112 : 88);
        interleave<MATRIX, (VECTOR + MATRIX - 1) / MATRIX>();
#pragma unroll
        for (int w = 0; w < CW; ++w) cur[w] = next[w];
    };

    if (nt > 0) {
        fetch(0);
        store(0);
        if (Ro::AHEAD == 2 && nt > 1) {
            fetch(1);
            store(1);
        }
        if (nt > Ro::AHEAD) fetch(Ro::AHEAD);
        __syncthreads();
        score(cur, 0, 0);
    }
    int b0 = 0, b1 = 1, before = 0;  // the buffers of tile i, i + 1, i - 1
    for (int i = 0; i < nt; ++i) {
        int b2 = b1 + 1 == Ro::BUFS ? 0 : b1 + 1;
        const int into = Ro::BLOCKS == 2 ? b1 : b2;
        if (i + Ro::AHEAD < nt) store(into);
        if (i + Ro::AHEAD + 1 < nt) fetch(i + Ro::AHEAD + 1);
        const int after = i + 1 < nt ? b1 : b0;  // (behind the last block: scores that nobody looks at)
        if (Ro::BLOCKS == 2) {
            step(b0, 0, before, i ? 32 : 0, b0, 32);
            __syncthreads();
            step(b0, 32, b0, 0, after, 0);
        } else {
            step(b0, 0, before, 0, after, 0);
            __syncthreads();
        }
        before = b0;
        b0 = b1;
        b1 = b2;
    }
    if (nt > 0) accumulate<E, NS, DP, CW>(out, q, tile[before], Tl::BV - 32);
    write_table<T, NS, DP, CW>(a, out, db, v0, part, 0);
}

// More than 256 columns, taken 256 at a time.  The scores add up over the chunks (the owned operand is read again for each,
// from the caches); a block accumulates the second product of one chunk, blockIdx.y's, which it streams last.  The work of
// the scores is repeated for every chunk of the result: a width that is rare is not worth a second shape of block.
template <typename E, int NS, bool GRAD>
__global__ __launch_bounds__(256, 1) void wide_rows_kernel(SweepArgs a)
{
    constexpr int DP = 256;
    typedef Tile<E, NS, DP> Tl;
    typedef typename Half<E>::x8 x8;
    static_assert(Tl::BV == 32, "one block of scores per tile");
    __shared__ __attribute__((aligned(16))) E tile[2][Tl::SIZE];
    __shared__ __attribute__((aligned(16))) float sb[2][32];
    const Derived dv = derive(NS == 2 ? a.scales : nullptr);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int part = blockIdx.x % a.splits;
    const int64_t n = (int64_t)(blockIdx.x / a.splits) * 128 + wave * 32 + (lane & 31);
    const int64_t tiles = ceil_div(a.vocab, 32), t0 = tiles * part / a.splits, t1 = tiles * (part + 1) / a.splits;
    const int chunks = a.chunks, first = (int)blockIdx.y + 1;
    auto offset = [&](int j) { return ((first + j) % chunks) * (NS * DP); };  // of the j-th chunk; the last is blockIdx.y's
    f32x16 out[1][DP / 32];
    Values<E, NS, 1> p;
    float m = dv.low * 1.01f, l = 0.0f;
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) out[0][b] = (f32x16)(0.0f);
    const int64_t at = n >= a.rows ? -1 : a.id_bytes == 8 ? ((const int64_t *)a.targets)[n] : (int64_t)((const int32_t *)a.targets)[n];
    const int64_t target = (uint64_t)at < (uint64_t)a.vocab ? at - 4 * h : -1000;
    Tl t;
    float next_bias = 0.0f;
    auto fetch = [&](int64_t i, int j) {
        t.fetch((const E *)a.w + offset(j), a.ldw, i * 32, a.vocab);
        const int64_t v = i * 32 + threadIdx.x;
        if (j == 0 && threadIdx.x < 32) next_bias = v >= a.vocab ? -INFINITY : a.bias ? bias_units(a.bias[v], dv) : 0.0f;
    };
    auto store = [&](int64_t i, int j, int buf) {
        t.store(tile[buf]);
        if (j == 0 && threadIdx.x < 32) sb[(i - t0) & 1][threadIdx.x] = next_bias;
    };
    if (t0 < t1) {
        fetch(t0, 0);
        store(t0, 0, 0);
    }
    __syncthreads();
    int buf = 0;
    for (int64_t i = t0; i < t1; ++i) {
        f32x16 s[1];
#pragma unroll
        for (int j = 0; j < 16; ++j) s[0][j] = sb[(i - t0) & 1][8 * (j / 4) + 4 * h + j % 4];
        for (int j = 0; j < chunks; ++j) {
            x8 own[1][NS][DP / 16];
            load_owned<E, NS, DP>(own[0], (const E *)a.x + offset(j), a.ldx, n, a.rows, dv.owned);
            const bool more = j + 1 < chunks || i + 1 < t1;
            if (more) fetch(j + 1 < chunks ? i : i + 1, j + 1 < chunks ? j + 1 : 0);
            scores<E, NS, DP, 1>(s, own, tile[buf], 0);
            if (j + 1 < chunks) {
                store(i, j + 1, buf ^ 1);
                __syncthreads();
                buf ^= 1;
            }
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) s[0][j] = target - i * 32 == 8 * (j / 4) + j % 4 ? -INFINITY : s[0][j];
        float mx = s[0][0];
#pragma unroll
        for (int j = 1; j < 16; ++j) mx = fmaxf(mx, s[0][j]);
        mx = half_wave_max(mx);
        if (__any((mx - m) * dv.c > LAG)) {
            const float up = (mx - m) * dv.c > LAG ? mx : m, f = exp2_fast((m - up) * dv.c);
            m = up;
            l *= f;
            if (GRAD)
#pragma unroll
                for (int b = 0; b < DP / 32; ++b) out[0][b] *= f;
        }
        const bool far = fabsf(m * dv.c) > FAR;
        const float base = far ? P_SHIFT : P_SHIFT - m * dv.c, less = far ? m : 0.0f;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float v8[1][8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v8[0][j] = exp2_fast(__builtin_fmaf(s[0][8 * k + j] - less, dv.c, base));
                l += v8[0][j];
            }
            if (GRAD) pack_values<E, NS, 1>(p, v8, k);
        }
        if (GRAD) accumulate<E, NS, DP, 1>(out, p, tile[buf], 0);
        if (i + 1 < t1) store(i + 1, 0, buf ^ 1);
        __syncthreads();
        buf ^= 1;
    }
    const float sum = half_wave_sum(l);
    if (n >= a.rows) return;
    const int64_t to = (int64_t)part * a.rows + n;
    if (h == 0) {
        a.pm[to + (int64_t)blockIdx.y * a.splits * a.rows] = m;
        a.pl[to + (int64_t)blockIdx.y * a.splits * a.rows] = sum;
    }
    if (GRAD)
#pragma unroll
        for (int b = 0; b < DP / 32; ++b)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *(float4 *)(a.po + to * a.dp + (int)blockIdx.y * DP + b * 32 + 8 * g + 4 * h) =
                    make_float4(out[0][b][4 * g], out[0][b][4 * g + 1], out[0][b][4 * g + 2], out[0][b][4 * g + 3]);
}

template <typename T, typename E, int NS>
__global__ __launch_bounds__(256, 1) void wide_table_kernel(SweepArgs a)
{
    constexpr int DP = 256;
    typedef Tile<E, NS, DP> Tl;
    typedef typename Half<E>::x8 x8;
    static_assert(Tl::BV == 32, "one block of scores per tile");
    __shared__ __attribute__((aligned(16))) E tile[2][Tl::SIZE];
    __shared__ __attribute__((aligned(16))) RowFacts<32> facts[2];
    const Derived dv = derive(NS == 2 ? a.scales : nullptr);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int part = blockIdx.x % a.splits;
    const int64_t w0 = (int64_t)(blockIdx.x / a.splits) * 128 + wave * 32, v = w0 + (lane & 31);
    const int64_t tiles = ceil_div(a.rows, 32), t0 = tiles * part / a.splits, t1 = tiles * (part + 1) / a.splits;
    const int chunks = a.chunks, first = (int)blockIdx.y + 1;
    auto offset = [&](int j) { return ((first + j) % chunks) * (NS * DP); };
    f32x16 out[1][DP / 32];
    Values<E, NS, 1> q;
    const float bias = a.bias && v < a.vocab ? bias_units(a.bias[v], dv) : 0.0f;
    float db[1] = {0.0f};
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) out[0][b] = (f32x16)(0.0f);
    Tl t;
    bool keep[Tl::PER];
    float next_m = 0.0f, next_r = 0.0f, next_g = 0.0f;
    int32_t next_t = -1;
    auto fetch = [&](int64_t i, int j) {
        t.fetch((const E *)a.x + offset(j), a.ldx, i * 32, a.rows);
#pragma unroll
        for (int k = 0; k < Tl::PER; ++k) {
            const int64_t n = i * 32 + (k * 256 + (int)threadIdx.x) / Tl::CHUNKS;
            keep[k] = n < a.rows && a.row_target[n] >= 0;
        }
        if (j == 0 && threadIdx.x < 32) {
            const int64_t n = i * 32 + threadIdx.x;
            const bool ok = n < a.rows;
            next_m = ok ? a.row_max[n] : INFINITY;
            next_r = ok ? a.row_rate[n] : 0.0f;
            next_g = ok ? a.row_weight[n] : 0.0f;
            next_t = ok ? a.row_target[n] : -1;
        }
    };
    auto store = [&](int64_t i, int j, int buf) {
#pragma unroll
        for (int k = 0; k < Tl::PER; ++k)
            if (!keep[k]) t.held[k] = make_uint4(0, 0, 0, 0);
        t.store(tile[buf]);
        if (j == 0 && threadIdx.x < 32) {
            const bool far = fabsf(next_m * dv.c) > FAR && next_m < INFINITY;
            RowFacts<32> &f = facts[(i - t0) & 1];
            f.m[threadIdx.x] = far ? 0.0f : -next_m * dv.c;
            f.far[threadIdx.x] = far ? next_m : 0.0f;
            f.rate[threadIdx.x] = next_r;
            f.weight[threadIdx.x] = next_g;
            f.target[threadIdx.x] = next_t;
        }
    };
    if (t0 < t1) {
        fetch(t0, 0);
        store(t0, 0, 0);
    }
    __syncthreads();
    int buf = 0;
    for (int64_t i = t0; i < t1; ++i) {
        const RowFacts<32> &f = facts[(i - t0) & 1];
        f32x16 s[1] = {(f32x16)(bias)};
        for (int j = 0; j < chunks; ++j) {
            x8 own[1][NS][DP / 16];
            load_owned<E, NS, DP>(own[0], (const E *)a.w + offset(j), a.ldw, v, a.vocab, dv.owned);
            const bool more = j + 1 < chunks || i + 1 < t1;
            if (more) fetch(j + 1 < chunks ? i : i + 1, j + 1 < chunks ? j + 1 : 0);
            scores<E, NS, DP, 1>(s, own, tile[buf], 0);
            if (j + 1 < chunks) {
                store(i, j + 1, buf ^ 1);
                __syncthreads();
                buf ^= 1;
            }
        }
        const bool hit = (uint32_t)(f.target[lane & 31] - (int32_t)w0) < 32u;
        if (__any(hit || f.far[lane & 31] != 0.0f))
            special_rows<E, NS, DP, 1, 32>(s, out, db, f, tile[buf], 0, (int32_t)w0, hit);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float v8[1][8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int r = k * 16 + 8 * (j / 4) + 4 * h + j % 4;
                v8[0][j] = exp2_fast(__builtin_fmaf(s[0][8 * k + j], dv.c, f.m[r])) * f.rate[r];
                db[0] += v8[0][j];
            }
            pack_values<E, NS, 1>(q, v8, k);
        }
        accumulate<E, NS, DP, 1>(out, q, tile[buf], 0);
        if (i + 1 < t1) store(i + 1, 0, buf ^ 1);
        __syncthreads();
        buf ^= 1;
    }
    write_table<T, NS, DP, 1>(a, out, db, v, part, (int)blockIdx.y * DP);
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
    const int64_t t = target_of(a, n);
    const float g = t < 0 ? 0.0f : a.weights ? a.weights[n] : 1.0f;
    const T *wt = (const T *)a.table + (t < 0 ? 0 : t) * a.table_stride;
    // l = sum without the target (times 2^7, about m).  With the target's score st and everything about the larger of the two:
    // 1 - p[target] = l / (l + e), loss = log1p(l / e): nothing is lost where p[target] is near 1.
    float st = 0.0f, e = 0.0f, loss = 0.0f;
    if (t >= 0) {
        for (int c = lane; c < a.d; c += 64) st = __builtin_fmaf((float)x[c], (float)wt[c], st);
        st = wave_sum(st);
        if (a.bias) st += a.bias[t];
        const float su = bias_units(st, dv);  // (not only a bias: any score)
        const float up = fmaxf(m, su);
        e = exp2_fast((su - up) * dv.c + P_SHIFT);
        const float f = exp2_fast((m - up) * dv.c);
        l *= f;
        m = up;
        loss = st == -INFINITY ? INFINITY : l <= e ? log1pf(l / e) : ldexpf(m - su, -dv.k) + (logf(l + e) - P_SHIFT * LN2);
    }
    const float sum = l + e;
    float lse = sum == 0.0f ? -INFINITY : m <= dv.low * 0.999f ? -3.402823466e38f : ldexpf(m, -dv.k) + (logf(sum) - P_SHIFT * LN2);
    const float other = sum == 0.0f ? 1.0f : l / sum;  // 1 - p[target]
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
    if (odd && t >= 0) loss = NAN;
    loss = t < 0 ? 0.0f : g * loss;
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
        j.row_rate[n] = lost ? NAN : t < 0 || sum == 0.0f ? 0.0f : gs * exp2_fast(P_SHIFT) / sum;
        j.row_weight[n] = gs * other;
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
            o = sum == 0.0f ? 0.0f : ldexpf(o / sum, -kw);
            o = lost ? NAN : g * (o - other * (float)wt[c]);
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
    const unsigned blocks = (unsigned)(ceil_div(s.rows, 128) * s.splits);
    if constexpr (WIDE) {
        if (grad) wide_rows_kernel<E, NS, true><<<dim3(blocks, (unsigned)s.chunks), 256, 0, st>>>(s);
        else wide_rows_kernel<E, NS, false><<<dim3(blocks), 256, 0, st>>>(s);  // without the gradient one chunk's sweep does
    } else {
        if (grad) rows_kernel<E, NS, DP, 1, true><<<dim3(blocks), 256, 0, st>>>(s);
        else rows_kernel<E, NS, DP, 1, false><<<dim3(blocks), 256, 0, st>>>(s);
    }
    return hipGetLastError();
}

template <typename T, typename E, int NS, int DP, bool WIDE>
hipError_t sweep_table(const SweepArgs &s, hipStream_t st)
{
    const unsigned blocks = (unsigned)(ceil_div(s.vocab, 128) * s.splits);
    if constexpr (WIDE) wide_table_kernel<T, E, NS><<<dim3(blocks, (unsigned)s.chunks), 256, 0, st>>>(s);
    else table_kernel<T, E, NS, DP, 1><<<dim3(blocks), 256, 0, st>>>(s);
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
    w.targets = a.targets;
    w.id_bytes = a.id_bytes;
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
