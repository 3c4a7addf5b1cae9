// ops_common.hpp -- what the device-memory operators (include/lfm_ops.h) share: element types, wave helpers and the
// host launchers that lfm_ops.hip (the C ABI) and the softmax epochs call.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/lfm_ops.h"

namespace lfm {
namespace ops {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

__host__ __device__ inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t align_up(int64_t n, int64_t a = 256) { return (n + a - 1) / a * a; }
inline int dtype_bytes(int dtype) { return dtype == LFM_F32 ? 4 : 2; }

// Carves a workspace; with base == nullptr it only counts.
struct Carver {
    char *base;
    int64_t used = 0;
    explicit Carver(void *b) : base((char *)b) {}
    template <typename T>
    T *take(int64_t n)
    {
        T *p = base ? (T *)(base + used) : nullptr;
        used += align_up(n * (int64_t)sizeof(T));
        return p;
    }
};

// N elements of T as one memory access
template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
    T v[N];
};

// softmax_loss.hip
int64_t softmax_workspace(int64_t rows, int64_t vocab, int d, int dtype, bool grad);
hipError_t softmax_loss(const lfm_softmax_args &a, bool grad, void *ws, hipStream_t st);
// embedding_ops.hip
hipError_t embedding_lookup(const lfm_lookup_args &a, hipStream_t st);
int64_t embedding_grad_workspace(int64_t rows, int64_t vocab, int64_t nnz, int d, bool bags);
hipError_t embedding_grad(const lfm_lookup_args &a, void *ws, hipStream_t st);
// clip_norm.hip
int64_t clip_workspace(int64_t n_tensors, const int64_t *counts);
hipError_t clip_global_norm(int64_t n_tensors, const void *const *x, void *const *out, const int64_t *counts,
                            const int32_t *dtypes, double max_norm, float *norm, void *ws, hipStream_t st);

}  // namespace ops
}  // namespace lfm
