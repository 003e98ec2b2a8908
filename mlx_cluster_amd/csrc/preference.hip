// Preference loss of paired log ratios, and its gradients.
//
// For a pair with r = the sum (or mean) of values - reference over the places
// that a side's mask leaves, z = beta * (r_chosen - r_rejected):
//   loss      (1 - e) softplus(-z) + e softplus(z),  softplus(x) = max(x, 0) + log1p(exp(-|x|))
//   d loss/dz -(1 - e) sigma(-z) + e sigma(z)
// and a value's gradient is d loss/dz * beta (/ its side's count), negated on
// the rejected side, 0 where it is masked.  A term whose weight is 0 is left
// out, so that an infinite z does not meet it.
#include "train_host.h"

namespace mlxc {

namespace {

constexpr int kWaves = kBlock / kWave;

struct Side {
    const void* values;
    const void* reference;
    const uint8_t* mask;
    int64_t length;
    void* grad;
};

struct PairTerms {
    float loss, slope;  // slope: d loss / d z
};

__device__ __forceinline__ float softplus(float x) {
    return fmaxf(x, 0.f) + log1pf(expf(-fabsf(x)));
}

__device__ __forceinline__ PairTerms pair_terms(float z, float smoothing) {
    PairTerms t{0.f, 0.f};
    if (smoothing < 1.f) {
        t.loss += (1.f - smoothing) * softplus(-z);
        t.slope -= (1.f - smoothing) / (1.f + expf(z));
    }
    if (smoothing > 0.f) {
        t.loss += smoothing * softplus(z);
        t.slope += smoothing / (1.f + expf(-z));
    }
    return t;
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int o = kWave / 2; o > 0; o >>= 1) x += __shfl_xor(x, o, kWave);
    return x;
}

// Writes a row of a side's gradient.
template <typename E>
__device__ __forceinline__ void grad_row(const Side& s, int64_t p, float slope, int lane,
                                         int lanes) {
    typename E::S* g = static_cast<typename E::S*>(s.grad) + p * s.length;
    const uint8_t* m = s.mask ? s.mask + p * s.length : nullptr;
    for (int64_t t = lane; t < s.length; t += lanes) g[t] = E::store(!m || m[t] ? slope : 0.f);
}

// One wavefront a pair; partial[block] <- the sum of its pairs' losses.
template <typename E>
__global__ __launch_bounds__(kBlock) void preference_kernel(Side chosen, Side rejected,
                                                            int64_t pairs, float beta,
                                                            float smoothing, bool normalize,
                                                            float share, float* __restrict__ rewards,
                                                            float* __restrict__ slopes,
                                                            float* __restrict__ partial) {
    __shared__ float part[kWaves];
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
    float loss = 0.f;
    for (int64_t p = blockIdx.x * static_cast<int64_t>(kWaves) + w; p < pairs;
         p += static_cast<int64_t>(gridDim.x) * kWaves) {
        float r[2], per[2];
        for (int s = 0; s < 2; ++s) {
            const Side& x = s ? rejected : chosen;
            const typename E::S* v = static_cast<const typename E::S*>(x.values) + p * x.length;
            const typename E::S* f =
                x.reference ? static_cast<const typename E::S*>(x.reference) + p * x.length : nullptr;
            const uint8_t* m = x.mask ? x.mask + p * x.length : nullptr;
            float sum = 0.f, left = 0.f;
            for (int64_t t = lane; t < x.length; t += kWave) {
                if (m && !m[t]) continue;
                left += 1.f;
                sum += E::load(v[t]) - (f ? E::load(f[t]) : 0.f);
            }
            sum = wave_sum(sum);
            left = wave_sum(left);
            per[s] = normalize ? 1.f / fmaxf(left, 1.f) : 1.f;
            r[s] = beta * (sum * per[s]);
        }
        const PairTerms t = pair_terms(r[0] - r[1], smoothing);
        loss += t.loss;
        const float dz = t.slope * beta * share;
        const float slope[2] = {dz * per[0], -dz * per[1]};
        if (lane == 0) {
            for (int s = 0; s < 2; ++s) {
                if (rewards) rewards[s * pairs + p] = r[s];
                if (slopes) slopes[s * pairs + p] = slope[s];
            }
        }
        if (chosen.grad) grad_row<E>(chosen, p, slope[0], lane, kWave);
        if (rejected.grad) grad_row<E>(rejected, p, slope[1], lane, kWave);
    }
    if (lane == 0) part[w] = loss;
    __syncthreads();
    if (threadIdx.x == 0) {
        float s = 0.f;
        for (int k = 0; k < kWaves; ++k) s += part[k];
        partial[blockIdx.x] = s;
    }
}

// *loss <- share * the sum of n partial sums, in a fixed order.
__global__ __launch_bounds__(kBlock) void loss_sum_kernel(const float* __restrict__ partial, int n,
                                                          float share, float* __restrict__ loss) {
    __shared__ float part[kWaves];
    float s = 0.f;
    for (int k = threadIdx.x; k < n; k += kBlock) s += partial[k];
    s = wave_sum(s);
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        float all = 0.f;
        for (int k = 0; k < kWaves; ++k) all += part[k];
        *loss = all * share;
    }
}

// One wavefront a pair and side.
template <typename E>
__global__ __launch_bounds__(kBlock) void preference_grad_kernel(Side chosen, Side rejected,
                                                                 int64_t pairs,
                                                                 const float* __restrict__ slopes,
                                                                 const float* upstream) {
    const int lane = threadIdx.x % kWave;
    const float up = upstream ? *upstream : 1.f;
    const Side& s = blockIdx.y ? rejected : chosen;
    if (!s.grad) return;
    for (int64_t p = blockIdx.x * static_cast<int64_t>(kWaves) + threadIdx.x / kWave; p < pairs;
         p += static_cast<int64_t>(gridDim.x) * kWaves)
        grad_row<E>(s, p, up * slopes[blockIdx.y * pairs + p], lane, kWave);
}

constexpr int kMaxBlocks = 4096;

int pair_blocks(int64_t pairs) {
    const int64_t b = (pairs + kWaves - 1) / kWaves;
    return static_cast<int>(b < 1 ? 1 : b > kMaxBlocks ? kMaxBlocks : b);
}

Side side(const mlxc_preference_side& s) {
    return Side{s.values, s.reference, s.mask, s.length, s.grad};
}

template <typename E>
int loss_typed(const PreferenceCall& c, float* loss, float* rewards, float* slopes, void* workspace,
               hipStream_t stream) {
    const int blocks = pair_blocks(c.pairs);
    const float share = c.sum || c.pairs == 0 ? 1.f : static_cast<float>(1.0 / c.pairs);
    float* partial = static_cast<float*>(workspace);
    hipLaunchKernelGGL(preference_kernel<E>, dim3(blocks), dim3(kBlock), 0, stream, side(c.side[0]),
                       side(c.side[1]), c.pairs, c.beta, c.smoothing, c.normalize, share, rewards,
                       slopes, partial);
    MLXC_HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL(loss_sum_kernel, dim3(1), dim3(kBlock), 0, stream, partial, blocks, share,
                       loss);
    MLXC_HIP_TRY(hipGetLastError());
    return MLXC_OK;
}

template <typename E>
int grad_typed(const PreferenceCall& c, const float* slopes, const float* upstream,
               hipStream_t stream) {
    hipLaunchKernelGGL(preference_grad_kernel<E>, dim3(pair_blocks(c.pairs), 2), dim3(kBlock), 0,
                       stream, side(c.side[0]), side(c.side[1]), c.pairs, slopes, upstream);
    MLXC_HIP_TRY(hipGetLastError());
    return MLXC_OK;
}

}  // namespace

size_t preference_workspace_bytes(int64_t pairs) {
    return static_cast<size_t>(pair_blocks(pairs)) * sizeof(float);
}

int launch_preference_loss(const PreferenceCall& c, float* loss, float* rewards, float* slopes,
                           void* workspace, hipStream_t stream) {
    if (c.dtype == MLXC_FLOAT32) return loss_typed<F32>(c, loss, rewards, slopes, workspace, stream);
    if (c.dtype == MLXC_BFLOAT16)
        return loss_typed<BF16>(c, loss, rewards, slopes, workspace, stream);
    return loss_typed<F16>(c, loss, rewards, slopes, workspace, stream);
}

int launch_preference_grad(const PreferenceCall& c, const float* slopes, const float* upstream,
                           hipStream_t stream) {
    if (c.pairs == 0) return MLXC_OK;
    if (c.dtype == MLXC_FLOAT32) return grad_typed<F32>(c, slopes, upstream, stream);
    if (c.dtype == MLXC_BFLOAT16) return grad_typed<BF16>(c, slopes, upstream, stream);
    return grad_typed<F16>(c, slopes, upstream, stream);
}

}  // namespace mlxc
