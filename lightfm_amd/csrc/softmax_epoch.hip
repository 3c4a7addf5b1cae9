// softmax_epoch.hip -- the kernels around the operators in a step of the softmax loss (session.hip:
// lfm_session_epoch_softmax): what a batch trains on, its summed loss, and the optimizer.
#include "kernels.hpp"

namespace lfm {

// ------------------------------------------------------------------ batch ---
// Positions [begin, begin + len) of the shuffle as the operators take them: a user id, a target item (-1 = none: the
// interaction is not a positive, like the Y > 0 test of the ranking losses, PYX:842) and a weight per position.
__global__ __launch_bounds__(256) void softmax_batch_kernel(SoftmaxBatch b)
{
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= b.len) return;
    int r = b.shuffle[b.begin + i];
    if ((uint32_t)r >= (uint32_t)b.n) {  // not a permutation: LFM_ECORRUPT at the end of the epoch (device.hpp: guard_row)
        b.counters[FAULT_SLOT] = 1ull;
        r = 0;
    }
    const int user = b.user_ids[r];
    b.users[i] = user;
    b.targets[i] = b.Y[r] > 0.0f ? b.item_ids[r] : -1;
    b.weights[i] = b.weight[r];
    if (b.first && (uint32_t)user < (uint32_t)b.n_users) atomicMin(&b.first[user], i);
}

__global__ __launch_bounds__(256) void softmax_slots_kernel(SoftmaxBatch b)
{
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= b.len) return;
    const int user = b.users[i];
    b.slots[i] = (uint32_t)user < (uint32_t)b.n_users ? b.first[user] : -1;
}

hipError_t launch_softmax_batch(const SoftmaxBatch &b, hipStream_t st)
{
    const dim3 grid((unsigned)((b.len + 255) / 256));
    softmax_batch_kernel<<<grid, 256, 0, st>>>(b);
    if (b.first) softmax_slots_kernel<<<grid, 256, 0, st>>>(b);
    return hipGetLastError();
}

// ------------------------------------------------------------------ update ---
// One optimizer step over the tables with the batch's summed gradients, and the batch's loss.  Bound by memory: a cell
// reads its gradient and, where that is not zero, reads and writes W and G (and M).
//
// A batch's gradient is a SUM over its interactions (hundreds at the bias of a popular item), so adagrad's accumulator takes
// the gradient in before it divides -- a cell's first step is then at most the learning rate -- where the per-interaction
// kernels divide by the accumulator of the steps before (PYX:443-447).  A cell whose gradient is zero keeps its
// accumulators: rows that no interaction of the batch touches are left as they are, as the per-interaction losses leave them.
struct CellStep {
    float lr, rho, eps, scale, l2;
    int adadelta;
    __device__ __forceinline__ void operator()(float &w, float &acc, float &mom, float g) const
    {
        g = g * scale + l2 * w;
        if (g == 0.0f) return;
        if (adadelta) {
            acc = rho * acc + (1.0f - rho) * (g * g);
            const float step = sqrtf(mom + eps) / sqrtf(acc + eps) * g;
            mom = rho * mom + (1.0f - rho) * (step * step);
            w -= step;
        } else {
            acc += g * g;
            w -= lr * g / sqrtf(acc);
        }
    }
};

__global__ __launch_bounds__(256) void softmax_update_kernel(SoftmaxUpdate u)
{
    CellStep cell{u.lr, u.rho, u.eps, 1.0f, 0.0f, u.adadelta};
    if (u.norm && *u.norm > u.max_norm && *u.norm < __builtin_inff()) cell.scale = u.max_norm / *u.norm;
    const int64_t step = (int64_t)gridDim.x * 256;
    for (int t = 0; t < 3; ++t) {
        const SoftmaxTable &tab = u.table[t];
        cell.l2 = tab.l2;
        const int64_t quads = tab.cells >> 2;
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < quads; i += step) {
            const float4 g = ((const float4 *)tab.g)[i];
            if (tab.l2 == 0.0f && g.x == 0.0f && g.y == 0.0f && g.z == 0.0f && g.w == 0.0f) continue;
            float4 w = ((const float4 *)tab.W)[i], a = ((const float4 *)tab.G)[i], m = {};
            if (u.adadelta) m = ((const float4 *)tab.M)[i];
            cell(w.x, a.x, m.x, g.x);
            cell(w.y, a.y, m.y, g.y);
            cell(w.z, a.z, m.z, g.z);
            cell(w.w, a.w, m.w, g.w);
            ((float4 *)tab.W)[i] = w;
            ((float4 *)tab.G)[i] = a;
            if (u.adadelta) ((float4 *)tab.M)[i] = m;
        }
        if (blockIdx.x == 0 && (int)threadIdx.x < (int)(tab.cells & 3)) {
            const int64_t i = (quads << 2) + threadIdx.x;
            float m = u.adadelta ? tab.M[i] : 0.0f;
            cell(tab.W[i], tab.G[i], m, tab.g[i]);
            if (u.adadelta) tab.M[i] = m;
        }
    }
    if (u.slots) {  // every user of the batch once, at the user's first position
        const SoftmaxTable &tab = u.table[0];
        cell.l2 = 0.0f;
        const int quads = u.d >> 2;  // (rows are padded to a multiple of four)
        for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < (int64_t)u.len * quads; q += step) {
            const int i = (int)(q / quads), c = (int)(q - (int64_t)i * quads);
            if (u.slots[i] != i) continue;
            const int64_t at = (int64_t)u.users[i] * quads + c;
            const float4 g = ((const float4 *)tab.g)[q];
            float4 w = ((const float4 *)tab.W)[at], a = ((const float4 *)tab.G)[at], m = {};
            if (u.adadelta) m = ((const float4 *)tab.M)[at];
            cell(w.x, a.x, m.x, g.x);
            cell(w.y, a.y, m.y, g.y);
            cell(w.z, a.z, m.z, g.z);
            cell(w.w, a.w, m.w, g.w);
            ((float4 *)tab.W)[at] = w;
            ((float4 *)tab.G)[at] = a;
            if (u.adadelta) ((float4 *)tab.M)[at] = m;
            if (c == 0) u.first[u.users[i]] = SOFTMAX_NOBODY;
        }
    }
    if (blockIdx.x == gridDim.x - 1) {  // the batch's loss, in the order of the threads: the same bits every time
        __shared__ double part[256];
        __shared__ int seen[256];
        double sum = 0.0;
        int count = 0;
        for (int i = threadIdx.x; i < u.len; i += 256) {
            sum += (double)u.loss[i];
            count += (uint32_t)u.targets[i] < (uint32_t)u.items;
        }
        part[threadIdx.x] = sum;
        seen[threadIdx.x] = count;
        __syncthreads();
        for (int s = 128; s > 0; s >>= 1) {
            if ((int)threadIdx.x < s) {
                part[threadIdx.x] += part[threadIdx.x + s];
                seen[threadIdx.x] += seen[threadIdx.x + s];
            }
            __syncthreads();
        }
        if (threadIdx.x == 0) {
            u.stats[0] += part[0];
            u.stats[1] += (double)seen[0];
        }
    }
}

hipError_t launch_softmax_update(const SoftmaxUpdate &u, int cus, hipStream_t st)
{
    int64_t most = 1;
    for (const SoftmaxTable &t : u.table) most = std::max(most, t.cells);
    if (u.slots) most = std::max(most, (int64_t)u.len * u.d);
    const int64_t blocks = std::min<int64_t>((most / 4 + 255) / 256 + 1, (int64_t)cus * 8);
    softmax_update_kernel<<<dim3((unsigned)blocks), 256, 0, st>>>(u);
    return hipGetLastError();
}

}  // namespace lfm
