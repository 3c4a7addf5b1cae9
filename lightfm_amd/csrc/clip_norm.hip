// clip_norm.hip -- the global norm over many tensors and the tensors scaled to at most max_norm.
//
// norm = sqrt(sum over all elements of x^2), y = round(x * min(1, max_norm / norm)).  Every element is read twice and
// written once, which is what bounds it.  The squares are summed in float64: a float32 square overflows at 1.8e19 and a
// float32 running sum of 10^8 squares loses digits, while the card adds float64 faster than it reads float32.  Sums are
// taken in a fixed order (a block's elements, the blocks by index): the same bits every time.
#include "ops_common.hpp"

namespace lfm {
namespace ops {
namespace {

constexpr int GROUP = 64;             // tensors per launch: their table travels in the kernel's arguments
constexpr int64_t PIECE = 32768;      // elements of one tensor that a block takes at a time
constexpr int64_t MAX_GRID = 2048;    // blocks of a launch

struct Table {
    const void *x[GROUP];
    void *out[GROUP];
    int64_t count[GROUP];
    int32_t first_piece[GROUP + 1];   // pieces of the tensors before this one
    uint8_t dtype[GROUP];
    int32_t tensors;
};

__device__ inline int tensor_of(const Table &t, int piece)
{
    int lo = 0, hi = t.tensors - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first_piece[mid] <= piece) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ inline double block_sum(double v, double *shared)
{
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    v = shared[0] + shared[1] + shared[2] + shared[3];
    __syncthreads();
    return v;
}

template <typename T>
__device__ inline double piece_squares(const T *x, int64_t n)
{
    constexpr int W = 16 / (int)sizeof(T);
    typedef Vec<T, W> V;
    double acc[2] = {0.0, 0.0};
    int64_t done = 0;
    if (((uintptr_t)x & 15) == 0) {
        const int64_t words = n / W;
        int64_t i = threadIdx.x;
        for (; i + 3 * 256 < words; i += 4 * 256) {
            V r[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) r[q] = ((const V *)x)[i + q * 256];
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int k = 0; k < W; ++k) {
                    const double v = (double)(float)r[q].v[k];
                    acc[k & 1] = fma(v, v, acc[k & 1]);
                }
        }
        for (; i < words; i += 256) {
            const V r = ((const V *)x)[i];
#pragma unroll
            for (int k = 0; k < W; ++k) {
                const double v = (double)(float)r.v[k];
                acc[k & 1] = fma(v, v, acc[k & 1]);
            }
        }
        done = words * W;
    }
    for (int64_t i = done + threadIdx.x; i < n; i += 256) {
        const double v = (double)(float)x[i];
        acc[0] = fma(v, v, acc[0]);
    }
    return acc[0] + acc[1];
}

__global__ __launch_bounds__(256) void squares_kernel(Table t, double *partial)
{
    __shared__ double shared[4];
    double sum = 0.0;
    const int pieces = t.first_piece[t.tensors];
    for (int p = blockIdx.x; p < pieces; p += gridDim.x) {
        const int i = tensor_of(t, p);
        const int64_t lo = (int64_t)(p - t.first_piece[i]) * PIECE;
        const int64_t n = t.count[i] - lo < PIECE ? t.count[i] - lo : PIECE;
        if (t.dtype[i] == LFM_F32) sum += piece_squares((const float *)t.x[i] + lo, n);
        else if (t.dtype[i] == LFM_BF16) sum += piece_squares((const bf16_t *)t.x[i] + lo, n);
        else sum += piece_squares((const f16_t *)t.x[i] + lo, n);
    }
    sum = block_sum(sum, shared);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
__device__ inline void piece_scale(const T *x, T *y, int64_t n, float f)
{
    constexpr int W = 16 / (int)sizeof(T);
    typedef Vec<T, W> V;
    int64_t done = 0;
    if ((((uintptr_t)x | (uintptr_t)y) & 15) == 0) {
        const int64_t words = n / W;
        int64_t i = threadIdx.x;
        for (; i + 3 * 256 < words; i += 4 * 256) {
            V r[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) r[q] = ((const V *)x)[i + q * 256];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
#pragma unroll
                for (int k = 0; k < W; ++k) r[q].v[k] = (T)((float)r[q].v[k] * f);
                __builtin_nontemporal_store(*(u32x4 *)&r[q], (u32x4 *)y + i + q * 256);
            }
        }
        for (; i < words; i += 256) {
            V r = ((const V *)x)[i];
#pragma unroll
            for (int k = 0; k < W; ++k) r.v[k] = (T)((float)r.v[k] * f);
            ((V *)y)[i] = r;
        }
        done = words * W;
    }
    for (int64_t i = done + threadIdx.x; i < n; i += 256) y[i] = (T)((float)x[i] * f);
}

// A factor below float32's normal numbers (values of 1e30 clipped to 1e-10) would have too few bits as one
template <typename T>
__device__ inline void piece_scale_far(const T *x, T *y, int64_t n, double f)
{
    for (int64_t i = threadIdx.x; i < n; i += 256) y[i] = (T)(float)((double)(float)x[i] * f);
}

template <typename T>
__device__ inline void piece_scale(const T *x, T *y, int64_t n, double f)
{
    if (f < 1.17549435e-38) piece_scale_far(x, y, n, f);
    else piece_scale(x, y, n, (float)f);
}

// Every block adds the partial sums itself (a fixed order) and scales its pieces; block 0 of the first group writes the
// norm.  in_place with a factor of 1: the values stay as they are, there is nothing to write.
__global__ __launch_bounds__(256) void scale_kernel(Table t, const double *partial, int partials, double max_norm,
                                                    float *norm_out, int scale)
{
    __shared__ double shared[4];
    double sum = 0.0;
    for (int i = threadIdx.x; i < partials; i += 256) sum += partial[i];
    sum = block_sum(sum, shared);
    const double norm = sqrt(sum);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    if (!scale) return;
    // a norm that is not finite (an element was not) scales nothing
    const double f = norm > max_norm && norm < HUGE_VAL ? max_norm / norm : 1.0;
    const int pieces = t.first_piece[t.tensors];
    // From the last piece to the first: what the norm read last is still in the 256 MB cache, and the results, stored past it
    // (piece_scale), do not push the first ones out before the next call: 320 M elements of two types 209 + 396 us before, 177 + 408
    // with both, the order alone gains nothing.
    for (int back = blockIdx.x; back < pieces; back += gridDim.x) {
        const int p = pieces - 1 - back;
        const int i = tensor_of(t, p);
        if (f == 1.0 && t.x[i] == t.out[i]) continue;
        const int64_t lo = (int64_t)(p - t.first_piece[i]) * PIECE;
        const int64_t n = t.count[i] - lo < PIECE ? t.count[i] - lo : PIECE;
        if (t.dtype[i] == LFM_F32) piece_scale((const float *)t.x[i] + lo, (float *)t.out[i] + lo, n, f);
        else if (t.dtype[i] == LFM_BF16) piece_scale((const bf16_t *)t.x[i] + lo, (bf16_t *)t.out[i] + lo, n, f);
        else piece_scale((const f16_t *)t.x[i] + lo, (f16_t *)t.out[i] + lo, n, f);
    }
}

int64_t pieces_of(const int64_t *counts, int64_t lo, int64_t hi)
{
    int64_t n = 0;
    for (int64_t i = lo; i < hi; ++i) n += ceil_div(counts[i], PIECE);
    return n;
}

// an empty group still takes one block: its partial sum is 0
int64_t grid_of(int64_t pieces) { return pieces < 1 ? 1 : pieces > MAX_GRID ? MAX_GRID : pieces; }

}  // namespace

int64_t clip_workspace(int64_t n_tensors, const int64_t *counts)
{
    int64_t partials = 1;
    for (int64_t g = 0; g < n_tensors; g += GROUP)
        partials += grid_of(pieces_of(counts, g, g + GROUP < n_tensors ? g + GROUP : n_tensors));
    return align_up(partials * (int64_t)sizeof(double));
}

hipError_t clip_global_norm(int64_t n_tensors, const void *const *x, void *const *out, const int64_t *counts,
                            const int32_t *dtypes, double max_norm, float *norm, void *ws, hipStream_t st)
{
    double *partial = (double *)ws;
    int64_t partials = 0;
    for (int phase = 0; phase < 2; ++phase) {
        const int64_t count = n_tensors < 1 ? 1 : ceil_div(n_tensors, GROUP);
        for (int64_t q = 0; q < count; ++q) {
            const int64_t g = (phase ? count - 1 - q : q) * GROUP;
            Table t;
            t.tensors = (int32_t)(n_tensors - g < GROUP ? n_tensors - g : GROUP);
            t.first_piece[0] = 0;
            for (int i = 0; i < t.tensors; ++i) {
                t.x[i] = x[g + i];
                t.out[i] = out ? out[g + i] : nullptr;
                t.count[i] = counts[g + i];
                t.dtype[i] = (uint8_t)dtypes[g + i];
                t.first_piece[i + 1] = t.first_piece[i] + (int32_t)ceil_div(counts[g + i], PIECE);
            }
            if (t.tensors == 0) {  // no tensors at all: one empty entry
                t.tensors = 1;
                t.x[0] = nullptr;
                t.out[0] = nullptr;
                t.count[0] = 0;
                t.dtype[0] = LFM_F32;
                t.first_piece[1] = 0;
            }
            const int64_t grid = grid_of(t.first_piece[t.tensors]);
            if (phase == 0) {
                squares_kernel<<<dim3((unsigned)grid), 256, 0, st>>>(t, partial + partials);
                partials += grid;
            } else {
                const bool scales = out != nullptr;
                if (scales || g == 0)
                    scale_kernel<<<dim3((unsigned)(scales ? grid : 1)), 256, 0, st>>>(t, partial, (int)partials, max_norm,
                                                                                  g == 0 ? norm : nullptr, scales ? 1 : 0);
            }
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
    }
    return hipSuccess;
}

}  // namespace ops
}  // namespace lfm
