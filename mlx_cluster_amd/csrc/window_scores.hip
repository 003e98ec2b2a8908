// Scores of the skip-gram windows of walks, and their gradient by place.
//
// With U the rows of a walk's M nodes (zeros where there is no node) and
// B[j, j + k] = 1 for the pairs of its windows (j < W = M - C + 1, 1 <= k < C),
//   scores    S = s * B o (U U^T)            a band of the walk's product
//   gradient  dU = (D + D^T) U               D the band of the scores' gradients
// (the table's gradient adds dU up by node, embedding.hip).
#include "train_host.h"

namespace mlxc {

namespace {

constexpr int kWaves = kBlock / kWave;

// One wavefront a window: its first node's row against the rows after it.
template <typename E>
__global__ __launch_bounds__(kBlock) void window_scores_kernel(
    const typename E::S* __restrict__ weight, int64_t row_stride, int32_t dim, Walks walks,
    float scale, float* __restrict__ scores, int64_t* status) {
    const int lane = threadIdx.x % kWave;
    const int64_t W = walks.windows(), total = walks.num_walks * W;
    bool bad = false;
    for (int64_t j = blockIdx.x * static_cast<int64_t>(kWaves) + threadIdx.x / kWave; j < total;
         j += static_cast<int64_t>(gridDim.x) * kWaves) {
        const int64_t first = j / W * walks.walk_nodes + j % W;
        const int64_t u = node_at(walks.nodes, first, bad);
        for (int32_t k = 1; k < walks.ctx; ++k) {
            const int64_t v = node_at(walks.nodes, first + k, bad);
            float s = 0.f;
            if (u >= 0 && v >= 0)
                for (int32_t d = lane; d < dim; d += kWave)
                    s += E::load(weight[u * row_stride + d]) * E::load(weight[v * row_stride + d]);
#pragma unroll
            for (int o = kWave / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, kWave);
            if (lane == 0) scores[j * (walks.ctx - 1) + k - 1] = s * scale;
        }
    }
    report_bad(bad, status);
}

// One wavefront a place: the gradient of its row.
template <typename E>
__global__ __launch_bounds__(kBlock) void window_rows_grad_kernel(
    const float* __restrict__ grad, const typename E::S* __restrict__ weight, int64_t row_stride,
    int32_t dim, Walks walks, float* __restrict__ rows) {
    const int lane = threadIdx.x % kWave;
    const int32_t M = walks.walk_nodes, C = walks.ctx;
    const int64_t W = walks.windows(), total = walks.num_walks * M;
    for (int64_t at = blockIdx.x * static_cast<int64_t>(kWaves) + threadIdx.x / kWave; at < total;
         at += static_cast<int64_t>(gridDim.x) * kWaves) {
        const int64_t n = at / M;
        const int32_t i = static_cast<int32_t>(at % M);
        const int32_t lo = i - C + 1 > 0 ? i - C + 1 : 0;
        const int32_t hi = i + C - 1 < M - 1 ? i + C - 1 : M - 1;
        for (int32_t d = lane; d < dim; d += kWave) {
            float acc = 0.f;
            for (int32_t o = lo; o <= hi; ++o) {
                const int32_t j = i < o ? i : o, k = (i < o ? o : i) - j;
                if (k == 0 || j >= W) continue;
                bool bad = false;
                const int64_t v = node_at(walks.nodes, n * M + o, bad);
                if (v < 0) continue;
                acc += grad[(n * W + j) * (C - 1) + k - 1] * E::load(weight[v * row_stride + d]);
            }
            rows[at * dim + d] = acc;
        }
    }
}

int wave_grid(int64_t waves, int& grid) {
    DeviceInfo info;
    if (int rc = device_info(info)) return rc;
    int64_t blocks = (waves + kWaves - 1) / kWaves;
    if (blocks > info.cus * 64) blocks = info.cus * 64;
    grid = static_cast<int>(blocks < 1 ? 1 : blocks);
    return MLXC_OK;
}

template <typename E>
int scores_typed(const Table& table, const Walks& walks, float scale, float* scores,
                 int64_t* status, hipStream_t stream) {
    int grid;
    if (int rc = wave_grid(walks.num_walks * walks.windows(), grid)) return rc;
    hipLaunchKernelGGL(window_scores_kernel<E>, dim3(grid), dim3(kBlock), 0, stream,
                       static_cast<const typename E::S*>(table.p), table.row_stride, table.dim,
                       walks, scale, scores, status);
    MLXC_HIP_TRY(hipGetLastError());
    return MLXC_OK;
}

template <typename E>
int rows_grad_typed(const float* grad, const Table& table, const Walks& walks, float* rows,
                    hipStream_t stream) {
    int grid;
    if (int rc = wave_grid(walks.count(), grid)) return rc;
    hipLaunchKernelGGL(window_rows_grad_kernel<E>, dim3(grid), dim3(kBlock), 0, stream, grad,
                       static_cast<const typename E::S*>(table.p), table.row_stride, table.dim,
                       walks, rows);
    MLXC_HIP_TRY(hipGetLastError());
    return MLXC_OK;
}

__global__ void clear_status_kernel(int64_t* status) {
    if (threadIdx.x == 0) *status = 0;
}

}  // namespace

int launch_window_scores(const Table& table, const Walks& walks, float scale, float* scores,
                         int64_t* status, hipStream_t stream) {
    if (status) {
        hipLaunchKernelGGL(clear_status_kernel, dim3(1), dim3(kWave), 0, stream, status);
        MLXC_HIP_TRY(hipGetLastError());
    }
    if (walks.num_walks == 0) return MLXC_OK;
    if (table.dtype == MLXC_FLOAT32)
        return scores_typed<F32>(table, walks, scale, scores, status, stream);
    if (table.dtype == MLXC_BFLOAT16)
        return scores_typed<BF16>(table, walks, scale, scores, status, stream);
    return scores_typed<F16>(table, walks, scale, scores, status, stream);
}

int launch_window_rows_grad(const float* grad, const Table& table, const Walks& walks, float* rows,
                            hipStream_t stream) {
    if (walks.num_walks == 0) return MLXC_OK;
    if (table.dtype == MLXC_FLOAT32) return rows_grad_typed<F32>(grad, table, walks, rows, stream);
    if (table.dtype == MLXC_BFLOAT16) return rows_grad_typed<BF16>(grad, table, walks, rows, stream);
    return rows_grad_typed<F16>(grad, table, walks, rows, stream);
}

}  // namespace mlxc
