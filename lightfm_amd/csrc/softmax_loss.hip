// softmax_loss.hip -- softmax cross entropy over the whole catalogue with its gradient, without keeping the logits.
#include "ops_common.hpp"

namespace lfm {
namespace ops {
namespace {

template <typename T>
__device__ inline float dot(const float *x, const T *w, int d)
{
    float s = 0.0f;
    for (int c = 0; c < d; ++c) s = fmaf(x[c], (float)w[c], s);
    return s;
}

__device__ inline int64_t target_of(const lfm_softmax_args &a, int64_t n)
{
    const int64_t t = a.id_bytes == 8 ? ((const int64_t *)a.targets)[n] : (int64_t)((const int32_t *)a.targets)[n];
    return (uint64_t)t < (uint64_t)a.vocab ? t : -1;
}

// One block per row: running maximum and sum of the softmax over the vocabulary.
template <typename T>
__global__ __launch_bounds__(256) void loss_kernel(lfm_softmax_args a)
{
    __shared__ float x[LFM_MAX_COMPONENTS], ms[256], ls[256];
    const int64_t n = blockIdx.x;
    for (int c = threadIdx.x; c < a.d; c += 256) x[c] = (float)((const T *)a.hidden)[n * a.hidden_stride + c];
    __syncthreads();
    float m = -INFINITY, l = 0.0f;
    for (int64_t v = threadIdx.x; v < a.vocab; v += 256) {
        const float s = dot(x, (const T *)a.table + v * a.table_stride, a.d) + (a.bias ? a.bias[v] : 0.0f);
        if (s > m) {
            l = l * expf(m - s) + 1.0f;
            m = s;
        } else if (!(s == -INFINITY)) l += expf(s - m);
    }
    ms[threadIdx.x] = m;
    ls[threadIdx.x] = l;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 256; ++i) {
            const float hi = fmaxf(m, ms[i]);
            if (hi == -INFINITY) { l += ls[i]; continue; }
            l = l * expf(m - hi) + ls[i] * expf(ms[i] - hi);
            m = hi;
        }
        const float lse = m + logf(l);
        a.lse[n] = lse;
        const int64_t t = target_of(a, n);
        float loss = 0.0f;
        if (t >= 0) {
            const float s = dot(x, (const T *)a.table + t * a.table_stride, a.d) + (a.bias ? a.bias[t] : 0.0f);
            loss = s == -INFINITY ? INFINITY : lse - s;
            if (a.weights) loss *= a.weights[n];
        }
        a.loss[n] = loss;
    }
}

__device__ inline float residual(float s, float lse, bool hit, float g)
{
    return g * ((s == -INFINITY ? 0.0f : expf(s - lse)) - (hit ? 1.0f : 0.0f));
}

template <typename T>
__global__ __launch_bounds__(256) void hidden_kernel(lfm_softmax_args a)
{
    __shared__ float x[LFM_MAX_COMPONENTS], q[256];
    const int64_t n = blockIdx.x;
    const int64_t t = target_of(a, n);
    const float lse = a.lse[n], g = t < 0 ? 0.0f : a.weights ? a.weights[n] : 1.0f;
    for (int c = threadIdx.x; c < a.d; c += 256) x[c] = (float)((const T *)a.hidden)[n * a.hidden_stride + c];
    __syncthreads();
    float acc[4] = {0, 0, 0, 0};
    for (int64_t v0 = 0; v0 < a.vocab && t >= 0; v0 += 256) {
        const int64_t v = v0 + threadIdx.x;
        q[threadIdx.x] = 0.0f;
        if (v < a.vocab) {
            const float s = dot(x, (const T *)a.table + v * a.table_stride, a.d) + (a.bias ? a.bias[v] : 0.0f);
            q[threadIdx.x] = residual(s, lse, v == t, g);
        }
        __syncthreads();
        const int m = a.vocab - v0 < 256 ? (int)(a.vocab - v0) : 256;
        for (int j = 0; j < m; ++j)
            for (int k = 0; k < 4; ++k) {
                const int c = threadIdx.x + 256 * k;
                if (c < a.d) acc[k] = fmaf(q[j], (float)((const T *)a.table)[(v0 + j) * a.table_stride + c], acc[k]);
            }
        __syncthreads();
    }
    for (int k = 0; k < 4; ++k) {
        const int c = threadIdx.x + 256 * k;
        if (c < a.d) ((T *)a.d_hidden)[n * a.d + c] = (T)acc[k];
    }
}

template <typename T>
__global__ __launch_bounds__(256) void table_kernel(lfm_softmax_args a)
{
    __shared__ float w[LFM_MAX_COMPONENTS], q[256];
    const int64_t v = blockIdx.x;
    for (int c = threadIdx.x; c < a.d; c += 256) w[c] = (float)((const T *)a.table)[v * a.table_stride + c];
    __syncthreads();
    const float b = a.bias ? a.bias[v] : 0.0f;
    float acc[4] = {0, 0, 0, 0}, db = 0.0f;
    for (int64_t n0 = 0; n0 < a.rows; n0 += 256) {
        const int64_t n = n0 + threadIdx.x;
        q[threadIdx.x] = 0.0f;
        if (n < a.rows) {
            const int64_t t = target_of(a, n);
            if (t >= 0)
                q[threadIdx.x] = residual(dot(w, (const T *)a.hidden + n * a.hidden_stride, a.d) + b, a.lse[n], v == t,
                                          a.weights ? a.weights[n] : 1.0f);
        }
        __syncthreads();
        const int m = a.rows - n0 < 256 ? (int)(a.rows - n0) : 256;
        for (int j = 0; j < m; ++j) {
            if (q[j] == 0.0f) continue;  // a row without a target is not read
            db += q[j];
            for (int k = 0; k < 4; ++k) {
                const int c = threadIdx.x + 256 * k;
                if (c < a.d) acc[k] = fmaf(q[j], (float)((const T *)a.hidden)[(n0 + j) * a.hidden_stride + c], acc[k]);
            }
        }
        __syncthreads();
    }
    for (int k = 0; k < 4; ++k) {
        const int c = threadIdx.x + 256 * k;
        if (c < a.d) ((T *)a.d_table)[v * a.d + c] = (T)acc[k];
    }
    if (a.d_bias && threadIdx.x == 0) a.d_bias[v] = db;
}

template <typename T>
hipError_t run(const lfm_softmax_args &a, bool grad, hipStream_t st)
{
    hipError_t e = hipSuccess;
    if (a.rows) {
        loss_kernel<T><<<dim3((unsigned)a.rows), 256, 0, st>>>(a);
        if ((e = hipGetLastError()) != hipSuccess || !grad) return e;
        hidden_kernel<T><<<dim3((unsigned)a.rows), 256, 0, st>>>(a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (grad) table_kernel<T><<<dim3((unsigned)a.vocab), 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace

int64_t softmax_workspace(int64_t, int64_t, int, int, bool) { return 256; }

hipError_t softmax_loss(const lfm_softmax_args &a, bool grad, void *, hipStream_t st)
{
    return a.dtype == LFM_F32 ? run<float>(a, grad, st) : a.dtype == LFM_BF16 ? run<bf16_t>(a, grad, st) : run<f16_t>(a, grad, st);
}

}  // namespace ops
}  // namespace lfm
