// embedding_ops.hip -- rows of an embedding table times a scale (single ids or weighted bags of ids) and the gradient
// by sorted ids.  Both move memory and compute next to nothing: the lookup reads each picked row and writes each
// output row once; the gradient reads each row of d_out once per id and writes the table's gradient once.
#include "ops_common.hpp"

namespace lfm {
namespace ops {
namespace {

// ------------------------------------------------------------------ lookup ---

// A group of `lanes` (a power of two <= 64) neighbouring lanes owns one output row, VEC elements (16 bytes where the
// addresses allow it) per lane and step: 16 lanes read a row of 64 floats in one access.  Accumulates in float32 in the
// order of the bag and rounds once, after the scale.
template <typename T, typename I, int VEC, bool BAGS>
__global__ __launch_bounds__(256) void lookup_kernel(lfm_lookup_args a, int lanes_log2)
{
    const int64_t t = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x;
    const int64_t row = t >> lanes_log2;
    if (row >= a.rows) return;
    const int lanes = 1 << lanes_log2, lane = (int)(t & (lanes - 1));
    const I *ids = (const I *)a.ids;
    typedef Vec<T, VEC> V;
    int64_t lo = row, hi = row + 1;
    if (BAGS) {  // an indptr that is not monotone inside [0, nnz] never leaves the arrays
        const int64_t l = (int64_t)((const I *)a.indptr)[row], h = (int64_t)((const I *)a.indptr)[row + 1];
        lo = l < 0 ? 0 : (l > a.nnz ? a.nnz : l);
        hi = h > a.nnz ? a.nnz : h;
    }
    const int base = (int)(threadIdx.x & 63) & ~(lanes - 1);  // the group's first lane in its wave
    for (int c0 = 0; c0 < a.d; c0 += lanes * VEC) {
        const int c = c0 + lane * VEC;
        float acc[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] = 0.0f;
        // a bag's ids are read `lanes` at a time and handed round, rows UP at a time: the loads do not wait for each other
        constexpr int UP = BAGS ? 8 : 1;
        for (int64_t j0 = lo; j0 < hi; j0 += lanes) {
            int32_t mine = -1;
            float weight = 0.0f;
            if (j0 + lane < hi) {
                const int64_t id = (int64_t)ids[j0 + lane];
                if ((uint64_t)id < (uint64_t)a.vocab) {
                    mine = (int32_t)id;
                    weight = BAGS && a.values ? a.values[j0 + lane] : 1.0f;
                }
            }
            const int count = hi - j0 < lanes ? (int)(hi - j0) : lanes;
            for (int q0 = 0; q0 < count; q0 += UP) {
                V r[UP];
                float w[UP];
                int32_t id[UP];
#pragma unroll
                for (int q = 0; q < UP; ++q) {
                    id[q] = __shfl(mine, base + (q0 + q < count ? q0 + q : 0));
                    w[q] = __shfl(weight, base + (q0 + q < count ? q0 + q : 0));
                    if (q0 + q >= count) id[q] = -1;
#pragma unroll
                    for (int k = 0; k < VEC; ++k) r[q].v[k] = (T)0.0f;
                    if (id[q] >= 0 && c < a.d) r[q] = *(const V *)((const T *)a.table + id[q] * a.table_stride + c);
                }
#pragma unroll
                for (int q = 0; q < UP; ++q)
                    if (id[q] >= 0)
#pragma unroll
                        for (int k = 0; k < VEC; ++k) acc[k] = fmaf(w[q], (float)r[q].v[k], acc[k]);
            }
        }
        if (c >= a.d) continue;
        V o;
#pragma unroll
        for (int k = 0; k < VEC; ++k) o.v[k] = (T)(acc[k] * a.scale);
        *(V *)((T *)a.out + row * a.d + c) = o;
    }
}

int lanes_for(int d, int vec)
{
    int l = 0;
    while ((1 << l) * vec < d && l < 6) ++l;
    return l;
}

bool aligned(const void *p, int64_t stride, int d, int item, int vec)
{
    return ((uintptr_t)p % (uintptr_t)(item * vec)) == 0 && stride % vec == 0 && d % vec == 0;
}

template <typename T, typename I, int VEC>
hipError_t launch_lookup(const lfm_lookup_args &a, hipStream_t st)
{
    const int ll = lanes_for(a.d, VEC);
    const int64_t blocks = ceil_div(a.rows << ll, 256), most = 1 << 22;  // (a dimension of a launch has fewer than 2^32 threads)
    const dim3 grid((unsigned)(blocks < most ? blocks : most), (unsigned)ceil_div(blocks, most));
    if (a.indptr) lookup_kernel<T, I, VEC, true><<<grid, 256, 0, st>>>(a, ll);
    else lookup_kernel<T, I, VEC, false><<<grid, 256, 0, st>>>(a, ll);
    return hipGetLastError();
}

template <typename T, typename I>
hipError_t lookup_typed(const lfm_lookup_args &a, hipStream_t st)
{
    constexpr int W = 16 / (int)sizeof(T);
    if (aligned(a.table, a.table_stride, a.d, sizeof(T), W) && aligned(a.out, a.d, a.d, sizeof(T), W))
        return launch_lookup<T, I, W>(a, st);
    if (aligned(a.table, a.table_stride, a.d, sizeof(T), W / 2) && aligned(a.out, a.d, a.d, sizeof(T), W / 2))
        return launch_lookup<T, I, W / 2>(a, st);
    if constexpr (W > 4)
        if (aligned(a.table, a.table_stride, a.d, sizeof(T), 2) && aligned(a.out, a.d, a.d, sizeof(T), 2)) return launch_lookup<T, I, 2>(a, st);
    return launch_lookup<T, I, 1>(a, st);
}

// ---------------------------------------------------------------- gradient ---
//
// 1. the ids are sorted by value with their positions, stable: a least-significant-digit radix sort of one to three
//    digits of up to 11 bits (200 003 ids: two digits of 9 bits).  A block owns one contiguous piece of the list, its
//    eight waves one contiguous part of the piece each, so "earlier block, earlier wave, earlier lane" is the order of
//    the positions.  The scatter kernel sums the blocks' digit counts itself (at most 128 blocks): a digit takes two
//    launches, and no count depends on the order in which atomics land.
// 2. the sorted list is cut into chunks of 8 to 32 ids (chunk_for); a lane group sums a chunk's runs of equal ids in float32, in order.  A run inside one chunk is written to its row at once, a run that crosses chunks leaves partial sums.
// 3. the block of the chunk where a crossing run starts adds the run's partial sums, in a fixed order.
// Rows without ids are zero: the first launch fills the output.

constexpr int SORT_WAVES = 8, SORT_THREADS = 64 * SORT_WAVES, MAX_BINS = 2048, MAX_BLOCKS = 128;

struct SortPlan {
    int passes, bits, bins;  // digits, bits of a digit, 1 << bits
    int blocks;
    int64_t items;           // ids of a block, a multiple of SORT_THREADS
};

SortPlan sort_plan(int64_t vocab, int64_t nnz)
{
    SortPlan p;
    int all = 1;
    while (all < 32 && ((uint64_t)vocab >> all) != 0) ++all;  // keys 0 .. vocab (= an id to leave out)
    p.passes = (all + 10) / 11;
    p.bits = (all + p.passes - 1) / p.passes;
    p.bins = 1 << p.bits;
    int64_t want = ceil_div(nnz, 2048);
    if (want < 1) want = 1;
    if (want > MAX_BLOCKS) want = MAX_BLOCKS;
    p.items = ceil_div(ceil_div(nnz, want), SORT_THREADS) * SORT_THREADS;
    if (p.items < SORT_THREADS) p.items = SORT_THREADS;  // no ids at all
    p.blocks = (int)ceil_div(nnz, p.items);
    if (p.blocks < 1) p.blocks = 1;
    return p;
}

template <typename I>
__device__ inline uint32_t key_of(const I *ids, int64_t j, int64_t vocab)
{
    const int64_t id = (int64_t)ids[j];
    return (uint64_t)id < (uint64_t)vocab ? (uint32_t)id : (uint32_t)vocab;
}

// A fill of the output and the bags of all positions by blocks [first, gridDim.x)
template <typename I>
__device__ inline void fill_and_bags(int first, uint4 *fill, int64_t fill_words, char *fill_tail, int fill_tail_bytes, const I *indptr,
                                     int64_t rows, int64_t n, int32_t *bag_of)
{
    const int64_t t = (int64_t)((int)blockIdx.x - first) * blockDim.x + threadIdx.x;
    const int64_t step = (int64_t)((int)gridDim.x - first) * blockDim.x;
    for (int64_t i = t; i < fill_words; i += step) fill[i] = make_uint4(0, 0, 0, 0);
    if (t < fill_tail_bytes) fill_tail[t] = 0;
    if (!indptr) return;
    const double per_id = (double)rows / (double)n;
    for (int64_t j = t; j < n; j += step) {  // the last row whose bag starts at or before j, looked for around where even bags have it
        int64_t lo = 0, hi = rows - 1, at = (int64_t)((double)j * per_id), gap = 1;
        if (at > hi) at = hi;
        if ((int64_t)indptr[at] <= j) {
            lo = at;
            while (lo + gap <= hi && (int64_t)indptr[lo + gap] <= j) {
                lo += gap;
                gap *= 2;
            }
            if (lo + gap - 1 < hi) hi = lo + gap - 1;
        } else {
            hi = at > 0 ? at - 1 : 0;
            while (hi - gap >= 0 && (int64_t)indptr[hi - gap + 1] > j) {
                hi -= gap;
                gap *= 2;
            }
            if (hi - gap + 1 > 0) lo = hi - gap + 1;
        }
        while (lo < hi) {
            const int64_t mid = (lo + hi + 1) >> 1;
            if ((int64_t)indptr[mid] <= j) lo = mid;
            else hi = mid - 1;
        }
        bag_of[j] = (int64_t)indptr[lo] <= j && j < (int64_t)indptr[lo + 1] ? (int32_t)lo : -1;
    }
}

// Short lists are sorted in one launch: an id's place is the number of ids before it (smaller, or equal and earlier), which
// a block counts for 32 ids over the whole list in LDS, eight threads to an id.  n^2 comparisons, but no passes that wait for
// each other: 3 launches for the whole gradient instead of 6.  On the GPU alone (26744 x 64 float32) 2000 ids take 19.8 us, 3000 21.7
// against 27, 4000 26.1 against 28; from 6000 on (31 against 28) the digits are faster.
constexpr int SHORT = 4096, RANKED = 32, RANK_PARTS = 256 / RANKED;

// Ids that a lane group sums one after the other, eight rows in flight: small chunks while there are lanes enough, large ones
// where the parts of runs that cross chunks would cost more than the waiting (26744 x 64 float32 / 400000 x 128 bfloat16, us, 8 | 16 |
// 32 to a chunk: 8000 ids 29 | 31 | 36 / 48 | 53 | 64; 60000 35 | 36 | 40 / 59 | 62 | 72; 180000 48 | 48 | 48 / 92 | 86 | 92; 600000 32
// alone 85 / 144, 16 90 / 158).
int chunk_for(int64_t nnz) { return nnz <= 65536 ? 8 : nnz <= 200000 ? 16 : 32; }

template <typename I>
__global__ __launch_bounds__(256) void rank_kernel(const I *ids, int n, int64_t vocab, int sort_blocks, uint4 *fill, int64_t fill_words,
                                                   char *fill_tail, int fill_tail_bytes, const I *indptr, int64_t rows, int32_t *bag_of,
                                                   uint32_t *keys_out, uint32_t *pos_out)
{
    if ((int)blockIdx.x >= sort_blocks) return fill_and_bags(sort_blocks, fill, fill_words, fill_tail, fill_tail_bytes, indptr, rows, n, bag_of);
    __shared__ __attribute__((aligned(16))) uint32_t keys[SHORT];
    __shared__ uint32_t places[RANK_PARTS][RANKED];
    const int padded = (n + 4 * RANK_PARTS - 1) & ~(4 * RANK_PARTS - 1);  // (at most SHORT)
#pragma unroll 8
    for (int j = threadIdx.x; j < padded; j += 256) keys[j] = j < n ? key_of(ids, j, vocab) : 0xffffffffu;  // (behind every id)
    __syncthreads();
    const int i = (int)blockIdx.x * RANKED + (threadIdx.x & (RANKED - 1)), part = threadIdx.x / RANKED;
    const uint32_t mine = i < n ? keys[i] : 0u;
    uint32_t place = 0;
    const int from = padded / RANK_PARTS * part, to = padded / RANK_PARTS * (part + 1);
    const int before = i & ~3;  // quads wholly before i: equal ids count
#pragma unroll 4
    for (int j = from; j < to; j += 4) {
        const uint4 k = *(const uint4 *)&keys[j];
        const uint32_t limit = mine + (j < before ? 1u : 0u);  // (ids end below 2^31)
        place += (k.x < limit) + (k.y < limit) + (k.z < limit) + (k.w < limit);
        if (j == before) {
#pragma unroll
            for (int q = 0; q < 3; ++q) place += j + q < i && keys[j + q] == mine;
        }
    }
    places[part][threadIdx.x & (RANKED - 1)] = place;
    __syncthreads();
    if (part || i >= n) return;
#pragma unroll
    for (int q = 1; q < RANK_PARTS; ++q) place += places[q][threadIdx.x];
    keys_out[place] = mine;
    pos_out[place] = (uint32_t)i;
}

// Digit counts of every block's piece (blocks [0, sort_blocks)); in the first pass (FIRST) the other blocks fill the
// output with zeros and write the bag of every position.
template <typename I, bool FIRST>
__global__ __launch_bounds__(SORT_THREADS) void count_kernel(const I *ids, const uint32_t *keys, int64_t n, int64_t vocab,
                                                            int shift, int bins, int64_t items, uint32_t *hist,
                                                            int sort_blocks, uint4 *fill, int64_t fill_words,
                                                            char *fill_tail, int fill_tail_bytes, const I *indptr,
                                                            int64_t rows, int32_t *bag_of)
{
    if (FIRST && (int)blockIdx.x >= sort_blocks)
        return fill_and_bags(sort_blocks, fill, fill_words, fill_tail, fill_tail_bytes, indptr, rows, n, bag_of);
    __shared__ uint32_t count[MAX_BINS];
    for (int b = threadIdx.x; b < bins; b += SORT_THREADS) count[b] = 0;
    __syncthreads();
    const int64_t lo = (int64_t)blockIdx.x * items, hi = lo + items < n ? lo + items : n;
    for (int64_t j = lo + threadIdx.x; j < hi; j += SORT_THREADS) {
        const uint32_t k = FIRST ? key_of(ids, j, vocab) : keys[j];
        atomicAdd(&count[(k >> shift) & (uint32_t)(bins - 1)], 1u);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += SORT_THREADS) hist[b * MAX_BLOCKS + (int)blockIdx.x] = count[b];
}

// PER: neighbouring digits whose counts one thread adds up
template <typename I, bool FIRST, int PER>
__global__ __launch_bounds__(SORT_THREADS) void scatter_kernel(const I *ids, const uint32_t *keys, const uint32_t *pos,
                                                              int64_t n, int64_t vocab, int shift, int bits,
                                                              int64_t items, const uint32_t *hist, int blocks,
                                                              uint32_t *keys_out, uint32_t *pos_out)
{
    __shared__ uint32_t count[SORT_WAVES][MAX_BINS];  // per wave: ids of the digit, then where the next one goes
    __shared__ uint32_t wave_sum[SORT_WAVES];
    const int bins = 1 << bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < SORT_WAVES * bins; i += SORT_THREADS) count[i / bins][i % bins] = 0;
    __syncthreads();
    const int64_t part = items / SORT_WAVES;
    const int64_t lo = (int64_t)blockIdx.x * items + wave * part;
    const int64_t hi = lo + part < n ? lo + part : n;
    constexpr int UP = 4;  // ids of a lane in flight
    for (int64_t j0 = lo; j0 < hi; j0 += 64 * UP) {
        uint32_t k[UP];
#pragma unroll
        for (int q = 0; q < UP; ++q) {
            const int64_t j = j0 + q * 64 + lane;
            k[q] = j >= hi ? 0u : FIRST ? key_of(ids, j, vocab) : keys[j];
        }
#pragma unroll
        for (int q = 0; q < UP; ++q)
            if (j0 + q * 64 + lane < hi) atomicAdd(&count[wave][(k[q] >> shift) & (uint32_t)(bins - 1)], 1u);
    }
    uint32_t before[PER], total[PER], sum = 0;
#pragma unroll
    for (int q = 0; q < PER; ++q) before[q] = total[q] = 0;
    const int first = threadIdx.x * PER;
    if (first < bins) {
#pragma unroll
        for (int q = 0; q < PER; ++q) {  // a digit's counts lie together: few, wide loads
            const uint4 *h = (const uint4 *)(hist + (first + q) * MAX_BLOCKS);
#pragma unroll 8
            for (int b = 0; b < blocks; b += 4) {
                const uint4 c = h[b / 4];
                const uint32_t cs[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    total[q] += b + k < blocks ? cs[k] : 0u;
                    before[q] += b + k < (int)blockIdx.x ? cs[k] : 0u;
                }
            }
        }
#pragma unroll
        for (int q = 0; q < PER; ++q) sum += total[q];
    }
    uint32_t scan = sum;  // inclusive scan over the threads
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t up = __shfl_up(scan, o);
        if (lane >= o) scan += up;
    }
    if (lane == 63) wave_sum[wave] = scan;
    __syncthreads();  // also: the waves' counts are complete
    uint32_t at = scan - sum;
    for (int w = 0; w < wave; ++w) at += wave_sum[w];
    if (first < bins) {
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            uint32_t next = at + before[q];
#pragma unroll
            for (int w = 0; w < SORT_WAVES; ++w) {
                const uint32_t c = count[w][first + q];
                count[w][first + q] = next;
                next += c;
            }
            at += total[q];
        }
    }
    __syncthreads();
    for (int64_t j0 = lo; j0 < hi; j0 += 64 * UP) {
        uint32_t k[UP], p[UP];
#pragma unroll
        for (int q = 0; q < UP; ++q) {
            const int64_t j = j0 + q * 64 + lane;
            const bool ok = j < hi;
            k[q] = !ok ? 0u : FIRST ? key_of(ids, j, vocab) : keys[j];
            p[q] = !ok ? 0u : FIRST ? (uint32_t)j : pos[j];
        }
#pragma unroll
        for (int q = 0; q < UP; ++q) {
            const bool ok = j0 + q * 64 + lane < hi;
            const uint32_t digit = (k[q] >> shift) & (uint32_t)(bins - 1);
            uint64_t same = __ballot(ok);  // the lanes with this lane's digit
            if (!same) break;
            for (int b = 0; b < bits; ++b) {
                const uint64_t has = __ballot((digit >> b) & 1u);
                same &= ((digit >> b) & 1u) ? has : ~has;
            }
            const int leader = ok ? __ffsll((unsigned long long)same) - 1 : lane;
            uint32_t base = 0;
            if (ok && lane == leader) base = atomicAdd(&count[wave][digit], (uint32_t)__popcll(same));
            base = __shfl(base, leader);
            if (ok) {
                const uint32_t to = base + (uint32_t)__popcll(same & ((1ull << lane) - 1ull));
                if (to < (uint64_t)n) {
                    keys_out[to] = k[q];
                    pos_out[to] = p[q];
                }
            }
        }
    }
}

struct SumArgs {
    const uint32_t *keys, *pos;
    const int32_t *bag_of;  // or NULL: the position is the row
    const float *values;
    const void *d_out;
    void *out;
    float *head, *tail;     // [chunks, d]: the part of a run that began earlier / that goes on
    int64_t n, vocab, rows, stride;
    int d;
    float scale;
};

template <typename T, int VEC>
__device__ inline void store_row(const SumArgs &a, uint32_t key, int c, const float *acc)
{
    Vec<T, VEC> o;
#pragma unroll
    for (int k = 0; k < VEC; ++k) o.v[k] = (T)(acc[k] * a.scale);
    *(Vec<T, VEC> *)((T *)a.out + (int64_t)key * a.d + c) = o;
}

// A block reads the ids, rows and values of its lane groups' chunks at once (they are pointers to pointers: position, bag,
// row), then each group walks its own.  blockIdx.y: the columns, as many at a time as a group has lanes for.
template <typename T, int VEC, int CHUNK>
__global__ __launch_bounds__(256) void chunk_sum_kernel(SumArgs a, int lanes_log2)
{
    constexpr int MOST = 64 * CHUNK;  // 4 lanes to a group at least
    __shared__ uint32_t keys[MOST + 1];
    __shared__ int32_t rows[MOST];
    __shared__ float values[MOST];
    const int lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1), group = threadIdx.x >> lanes_log2, groups = 256 >> lanes_log2;
    const int64_t first = (int64_t)blockIdx.x * groups * CHUNK;
    const uint32_t none = (uint32_t)a.vocab;
    for (int i = threadIdx.x; i <= groups * CHUNK; i += 256) {
        const int64_t j = first + i;
        const uint32_t key = j < a.n ? a.keys[j] : none;
        keys[i] = key;
        if (i == groups * CHUNK) continue;
        int32_t row = -1;
        float value = 0.0f;
        if (key != none) {
            const uint32_t p = a.pos[j];
            row = a.bag_of ? a.bag_of[p] : (int32_t)p;
            if ((uint64_t)row < (uint64_t)a.rows) value = a.values ? a.values[p] : 1.0f;
            else row = -1;
        }
        rows[i] = row;
        values[i] = value;
    }
    __syncthreads();
    const int lo = group * CHUNK;
    const int64_t chunk = (int64_t)blockIdx.x * groups + group;
    if (first + lo >= a.n) return;
    const int hi = a.n - first < lo + CHUNK ? (int)(a.n - first) : lo + CHUNK;
    const uint32_t earlier = lo ? keys[lo - 1] : first ? a.keys[first - 1] : none, later = keys[hi];
    typedef Vec<T, VEC> V;
    const int c = ((int)blockIdx.y * lanes + lane) * VEC;
    if (c < a.d) {
        float acc[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] = 0.0f;
        uint32_t run = keys[lo];
        bool began = earlier != run || (first == 0 && lo == 0);  // the run's first id is in this chunk
        for (int j0 = lo; j0 < hi; j0 += 8) {
            V r[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) r[q].v[k] = (T)0.0f;
                if (j0 + q < hi && rows[j0 + q] >= 0) r[q] = *(const V *)((const T *)a.d_out + rows[j0 + q] * a.stride + c);
            }
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                if (j0 + q >= hi) break;
                if (keys[j0 + q] != run) {  // the run ends here
                    if (began) {
                        if (run != none) store_row<T, VEC>(a, run, c, acc);
                    } else {
#pragma unroll
                        for (int k = 0; k < VEC; ++k) a.head[chunk * a.d + c + k] = acc[k];
                    }
                    run = keys[j0 + q];
                    began = true;
#pragma unroll
                    for (int k = 0; k < VEC; ++k) acc[k] = 0.0f;
                }
                if (rows[j0 + q] >= 0)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) acc[k] = fmaf(values[j0 + q], (float)r[q].v[k], acc[k]);
            }
        }
        if (run == none) return;
        if (began && later != run) store_row<T, VEC>(a, run, c, acc);
        else {
            float *to = (began ? a.tail : a.head) + chunk * a.d + c;
#pragma unroll
            for (int k = 0; k < VEC; ++k) to[k] = acc[k];
        }
    }
}

// A run that goes on behind its first chunk: its parts are shared by a wave's lane groups, or by a block's where the run is
// long (a popular id), and added in a fixed order.  A block looks at one chunk per wave.
constexpr int LONG_RUN = 64;

template <typename T, int VEC, int CHUNK>
__global__ __launch_bounds__(256) void join_kernel(SumArgs a, int lanes_log2)
{
    __shared__ float sums[256 * VEC];
    __shared__ int64_t parts_of[4];
    const int wave = threadIdx.x >> 6, in_wave = threadIdx.x & 63;
    const int lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1);
    const int64_t chunk0 = (int64_t)blockIdx.x * 4;
    // the parts behind a chunk whose last run starts there and goes on: chunks that begin with the run's id
    int64_t parts = 0;
    const int64_t end = (chunk0 + wave + 1) * CHUNK;
    if (end < a.n) {
        const uint32_t key = a.keys[end - 1];
        const bool earlier = end > CHUNK && a.keys[end - CHUNK] == key && a.keys[end - CHUNK - 1] == key;
        if (key != (uint32_t)a.vocab && !earlier)
            for (int64_t p = 0;; p += 64) {
                const int64_t at = end + (p + in_wave) * CHUNK;
                const uint64_t same = __ballot(at < a.n && a.keys[at] == key);
                parts += __popcll(same);
                if (~same) break;
            }
    }
    if (in_wave == 0) parts_of[wave] = parts;
    __syncthreads();
    for (int w = 0; w < 4; ++w) {
        const int64_t n = parts_of[w], chunk = chunk0 + w;
        const bool together = n > LONG_RUN;
        if (n == 0 || (!together && w != wave)) continue;
        const int groups = (together ? 256 : 64) >> lanes_log2, group = (together ? (int)threadIdx.x : in_wave) >> lanes_log2;
        float *mine = sums + (together ? 0 : wave * 64 * VEC);
        const uint32_t key = a.keys[(chunk + 1) * CHUNK];
        const int64_t share = ceil_div(n, groups);
        const int64_t p0 = group * share < n ? group * share : n, p1 = p0 + share < n ? p0 + share : n;
        const int used = (int)ceil_div(n, share);
        const int c = ((int)blockIdx.y * lanes + lane) * VEC;
        float acc[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] = 0.0f;
        if (c < a.d) {
#pragma unroll 8
            for (int64_t p = p0; p < p1; ++p) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) acc[k] += a.head[(chunk + 1 + p) * a.d + c + k];
            }
        }
        if (together) __syncthreads();
#pragma unroll
        for (int k = 0; k < VEC; ++k) mine[(group * lanes + lane) * VEC + k] = acc[k];
        if (together) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (group == 0 && c < a.d) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[k] = a.tail[chunk * a.d + c + k];
            for (int g = 0; g < used; ++g)
#pragma unroll
                for (int k = 0; k < VEC; ++k) acc[k] += mine[(g * lanes + lane) * VEC + k];
            store_row<T, VEC>(a, key, c, acc);
        }
        if (together) __syncthreads();  // (a wave's own sums use the same places)
    }
}

struct GradSpace {
    uint32_t *keys[2], *pos[2], *hist;
    int32_t *bag_of;
    float *head, *tail;
    int64_t bytes;
};

GradSpace grad_space(int64_t vocab, int64_t nnz, int d, bool bags, void *ws)
{
    Carver c(ws);
    GradSpace s;
    const SortPlan p = sort_plan(vocab, nnz);
    const int64_t chunks = ceil_div(nnz, chunk_for(nnz));
    for (int i = 0; i < 2; ++i) {
        s.keys[i] = c.take<uint32_t>(nnz);
        s.pos[i] = c.take<uint32_t>(nnz);
    }
    s.hist = c.take<uint32_t>((int64_t)MAX_BLOCKS * p.bins);  // [digit][block]
    s.bag_of = c.take<int32_t>(bags ? nnz : 0);
    s.head = c.take<float>(chunks * d);
    s.tail = c.take<float>(chunks * d);
    s.bytes = c.used;
    return s;
}

template <typename T, int VEC, int CHUNK>
hipError_t launch_chunks(const SumArgs &s, hipStream_t st)
{
    int ll = lanes_for(s.d, VEC);
    if (ll < 2) ll = 2;
    const int64_t chunks = ceil_div(s.n, CHUNK);
    const unsigned slices = (unsigned)ceil_div(s.d, (int64_t)VEC << ll);  // (at most 1024)
    chunk_sum_kernel<T, VEC, CHUNK><<<dim3((unsigned)ceil_div(chunks, 256 >> ll), slices), 256, 0, st>>>(s, ll);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || chunks < 2) return e;
    join_kernel<T, VEC, CHUNK><<<dim3((unsigned)ceil_div(chunks, 4), slices), 256, 0, st>>>(s, ll);
    return hipGetLastError();
}

template <typename T, int VEC>
hipError_t launch_sums(const SumArgs &s, hipStream_t st)
{
    switch (chunk_for(s.n)) {
    case 8: return launch_chunks<T, VEC, 8>(s, st);
    case 16: return launch_chunks<T, VEC, 16>(s, st);
    default: return launch_chunks<T, VEC, 32>(s, st);
    }
}

template <typename T>
hipError_t sums_typed(const SumArgs &s, hipStream_t st)
{
    constexpr int W = 16 / (int)sizeof(T);
    if (aligned(s.d_out, s.stride, s.d, sizeof(T), W) && aligned(s.out, s.d, s.d, sizeof(T), W))
        return launch_sums<T, W>(s, st);
    if (aligned(s.d_out, s.stride, s.d, sizeof(T), W / 2) && aligned(s.out, s.d, s.d, sizeof(T), W / 2))
        return launch_sums<T, W / 2>(s, st);
    if constexpr (W > 4)
        if (aligned(s.d_out, s.stride, s.d, sizeof(T), 2) && aligned(s.out, s.d, s.d, sizeof(T), 2)) return launch_sums<T, 2>(s, st);
    return launch_sums<T, 1>(s, st);
}

template <typename I>
hipError_t grad_typed(const lfm_lookup_args &a, void *ws, hipStream_t st)
{
    const SortPlan p = sort_plan(a.vocab, a.nnz);
    const GradSpace s = grad_space(a.vocab, a.nnz, a.d, a.indptr != nullptr, ws);
    const int64_t out_bytes = a.vocab * a.d * dtype_bytes(a.dtype);
    const int64_t words = out_bytes / 16;  // the output is 16-byte aligned (checked by the caller)
    int64_t fill_blocks = ceil_div(words > a.nnz ? words : a.nnz, (int64_t)SORT_THREADS * 4);
    if (fill_blocks < 1) fill_blocks = 1;
    if (fill_blocks > 2048) fill_blocks = 2048;
    const I *ids = (const I *)a.ids;
    hipError_t e;
    const uint32_t *keys = nullptr, *pos = nullptr;
    int at = 0;
    const bool in_one = a.nnz > 0 && a.nnz <= SHORT;
    if (in_one) {
        const int sort_blocks = (int)ceil_div(a.nnz, RANKED);
        rank_kernel<I><<<dim3((unsigned)(sort_blocks + fill_blocks)), 256, 0, st>>>(
            ids, (int)a.nnz, a.vocab, sort_blocks, (uint4 *)a.out, words, (char *)a.out + words * 16, (int)(out_bytes - words * 16),
            (const I *)a.indptr, a.rows, s.bag_of, s.keys[0], s.pos[0]);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        keys = s.keys[0];
        pos = s.pos[0];
    }
    for (int pass = 0; pass < (in_one ? 0 : p.passes); ++pass) {
        const int shift = pass * p.bits;
        if (pass == 0)
            count_kernel<I, true><<<dim3((unsigned)(p.blocks + fill_blocks)), SORT_THREADS, 0, st>>>(
                ids, nullptr, a.nnz, a.vocab, shift, p.bins, p.items, s.hist, p.blocks, (uint4 *)a.out, words,
                (char *)a.out + words * 16, (int)(out_bytes - words * 16), (const I *)a.indptr, a.rows, s.bag_of);
        else
            count_kernel<I, false><<<dim3((unsigned)p.blocks), SORT_THREADS, 0, st>>>(
                ids, keys, a.nnz, a.vocab, shift, p.bins, p.items, s.hist, p.blocks, nullptr, 0, nullptr, 0, nullptr, 0,
                nullptr);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        if (a.nnz == 0) return hipSuccess;
        const int per = p.bins / SORT_THREADS;
#define SCATTER(FIRST, PER)                                                                                               \
    scatter_kernel<I, FIRST, PER><<<dim3((unsigned)p.blocks), SORT_THREADS, 0, st>>>(                                         \
        ids, keys, pos, a.nnz, a.vocab, shift, p.bits, p.items, s.hist, p.blocks, s.keys[at], s.pos[at])
        if (pass == 0) {
            if (per <= 1) SCATTER(true, 1);
            else if (per == 2) SCATTER(true, 2);
            else SCATTER(true, 4);
        } else {
            if (per <= 1) SCATTER(false, 1);
            else if (per == 2) SCATTER(false, 2);
            else SCATTER(false, 4);
        }
#undef SCATTER
        if ((e = hipGetLastError()) != hipSuccess) return e;
        keys = s.keys[at];
        pos = s.pos[at];
        at ^= 1;
    }
    SumArgs sum;
    sum.keys = keys;
    sum.pos = pos;
    sum.bag_of = a.indptr ? s.bag_of : nullptr;
    sum.values = a.values;
    sum.d_out = a.d_out;
    sum.out = a.out;
    sum.head = s.head;
    sum.tail = s.tail;
    sum.n = a.nnz;
    sum.vocab = a.vocab;
    sum.rows = a.rows;
    sum.stride = a.d_out_stride;
    sum.d = a.d;
    sum.scale = a.scale;
    return a.dtype == LFM_F32 ? sums_typed<float>(sum, st)
         : a.dtype == LFM_BF16 ? sums_typed<bf16_t>(sum, st) : sums_typed<f16_t>(sum, st);
}

}  // namespace

hipError_t embedding_lookup(const lfm_lookup_args &a, hipStream_t st)
{
    if (a.rows == 0) return hipSuccess;
    if (a.id_bytes == 8)
        return a.dtype == LFM_F32 ? lookup_typed<float, int64_t>(a, st)
             : a.dtype == LFM_BF16 ? lookup_typed<bf16_t, int64_t>(a, st) : lookup_typed<f16_t, int64_t>(a, st);
    return a.dtype == LFM_F32 ? lookup_typed<float, int32_t>(a, st)
         : a.dtype == LFM_BF16 ? lookup_typed<bf16_t, int32_t>(a, st) : lookup_typed<f16_t, int32_t>(a, st);
}

int64_t embedding_grad_workspace(int64_t rows, int64_t vocab, int64_t nnz, int d, bool bags)
{
    (void)rows;
    return grad_space(vocab, nnz, d, bags, nullptr).bytes;
}

hipError_t embedding_grad(const lfm_lookup_args &a, void *ws, hipStream_t st)
{
    return a.id_bytes == 8 ? grad_typed<int64_t>(a, ws, st) : grad_typed<int32_t>(a, ws, st);
}

}  // namespace ops
}  // namespace lfm
