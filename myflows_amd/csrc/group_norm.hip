// Group norm with an activation over channels-last activations (n, positions, channels), and its gradients.
//
// A group is channels / groups neighbouring channels of one sample, over all its positions. With its mean
// and biased variance:
//   xhat = (x - mean) inv_std,  u = gamma xhat + beta,  y = act(u)      inv_std = (variance + eps)^(-1/2)
// and, with du = dy act'(u) and the averages over the group,
//   dgamma[c] = sum du xhat,  dbeta[c] = sum du,
//   dx = inv_std (gamma du - average(gamma du) - xhat average(gamma du xhat)).
// Sums are float32; the variance is a sum of squares about the mean, never a difference of large sums.
#include <algorithm>
#include <cstdint>

#include "common.h"
#include "typed.h"

namespace mfh {
namespace {

constexpr int NORM_THREADS = 256;

__device__ __forceinline__ float block_sum(float v) {
    __shared__ float part[NORM_THREADS];
    __syncthreads();
    part[threadIdx.x] = v;
    __syncthreads();
    for (int half = NORM_THREADS / 2; half > 0; half /= 2) {
        if (static_cast<int>(threadIdx.x) < half) part[threadIdx.x] += part[threadIdx.x + half];
        __syncthreads();
    }
    return part[0];
}

__device__ __forceinline__ float sigmoid_of(float u) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * u));
}
template <int ACT>
__device__ __forceinline__ float activate(float u) {
    if constexpr (ACT == ACT_RELU) return u > 0.0f || u != u ? u : 0.0f;
    if constexpr (ACT == ACT_SILU) return u * sigmoid_of(u);
    return u;
}
// dy act'(u)
template <int ACT>
__device__ __forceinline__ float through(float u, float dy) {
    if constexpr (ACT == ACT_RELU) return u > 0.0f ? dy : 0.0f;
    if constexpr (ACT == ACT_SILU) {
        const float g = sigmoid_of(u);
        return dy * (g * (1.0f + u * (1.0f - g)));
    }
    return dy;
}

template <typename T, int ACT>
__global__ __launch_bounds__(NORM_THREADS) void group_norm_kernel(const T* __restrict__ x, T* __restrict__ y,
                                                                  GroupNormShape s, GroupNormForward f) {
    const int per = s.channels / s.groups, count = s.positions * per;
    const long long n = blockIdx.x / s.groups;
    const int g = blockIdx.x % s.groups;
    const long long base = n * s.positions * s.channels + g * per;
    float sum = 0.0f;
    for (int i = threadIdx.x; i < count; i += NORM_THREADS) sum += static_cast<float>(x[base + (i / per) * static_cast<long long>(s.channels) + i % per]);
    const float mean = block_sum(sum) / count;
    float squares = 0.0f;
    for (int i = threadIdx.x; i < count; i += NORM_THREADS) {
        const float d = static_cast<float>(x[base + (i / per) * static_cast<long long>(s.channels) + i % per]) - mean;
        squares += d * d;
    }
    const float inv_std = 1.0f / sqrtf(block_sum(squares) / count + f.eps);
    if (threadIdx.x == 0) {
        f.mean[blockIdx.x] = mean;
        f.inv_std[blockIdx.x] = inv_std;
    }
    for (int i = threadIdx.x; i < count; i += NORM_THREADS) {
        const long long at = base + (i / per) * static_cast<long long>(s.channels) + i % per;
        const int c = g * per + i % per;
        y[at] = static_cast<T>(activate<ACT>((static_cast<float>(x[at]) - mean) * inv_std * f.gamma[c] + f.beta[c]));
    }
}

template <typename T, int ACT>
__global__ __launch_bounds__(NORM_THREADS) void group_norm_dx_kernel(const T* __restrict__ x, const T* __restrict__ dy,
                                                                     T* dx, GroupNormShape s, GroupNormBackward b) {
    const int per = s.channels / s.groups, count = s.positions * per;
    const long long n = blockIdx.x / s.groups;
    const int g = blockIdx.x % s.groups;
    const long long base = n * s.positions * s.channels + g * per;
    const float mean = b.mean[blockIdx.x], inv_std = b.inv_std[blockIdx.x];
    float first = 0.0f, second = 0.0f;
    for (int i = threadIdx.x; i < count; i += NORM_THREADS) {
        const long long at = base + (i / per) * static_cast<long long>(s.channels) + i % per;
        const int c = g * per + i % per;
        const float hat = (static_cast<float>(x[at]) - mean) * inv_std;
        const float d = through<ACT>(hat * b.gamma[c] + b.beta[c], static_cast<float>(dy[at])) * b.gamma[c];
        first += d;
        second += d * hat;
    }
    first = block_sum(first) / count;
    second = block_sum(second) / count;
    for (int i = threadIdx.x; i < count; i += NORM_THREADS) {
        const long long at = base + (i / per) * static_cast<long long>(s.channels) + i % per;
        const int c = g * per + i % per;
        const float hat = (static_cast<float>(x[at]) - mean) * inv_std;
        const float d = through<ACT>(hat * b.gamma[c] + b.beta[c], static_cast<float>(dy[at])) * b.gamma[c];
        const float v = inv_std * (d - first - hat * second);
        dx[at] = static_cast<T>(b.add_x ? static_cast<float>(dx[at]) + v : v);
    }
}

template <typename T, int ACT>
__global__ __launch_bounds__(NORM_THREADS) void group_norm_params_kernel(const T* __restrict__ x,
                                                                         const T* __restrict__ dy, GroupNormShape s,
                                                                         GroupNormBackward b) {
    const int c = blockIdx.x, g = c / (s.channels / s.groups);
    const float gamma = b.gamma[c], beta = b.beta[c];
    float first = 0.0f, second = 0.0f;
    for (long long i = threadIdx.x; i < s.n * s.positions; i += NORM_THREADS) {
        const long long n = i / s.positions;
        const float hat = (static_cast<float>(x[i * s.channels + c]) - b.mean[n * s.groups + g]) * b.inv_std[n * s.groups + g];
        const float d = through<ACT>(hat * gamma + beta, static_cast<float>(dy[i * s.channels + c]));
        first += d;
        second += d * hat;
    }
    first = block_sum(first);
    second = block_sum(second);
    if (threadIdx.x != 0) return;
    if (b.beta_grad) b.beta_grad[c] = b.add_beta ? b.beta_grad[c] + first : first;
    if (b.gamma_grad) b.gamma_grad[c] = b.add_gamma ? b.gamma_grad[c] + second : second;
}

// Calls f with the element type and activation as types.
template <typename F>
void with_type_and_act(int type, int act, F&& f) {
    with_type(type, [&](auto zero) {
        if (act == ACT_RELU) f(zero, std::integral_constant<int, ACT_RELU>{});
        else if (act == ACT_SILU) f(zero, std::integral_constant<int, ACT_SILU>{});
        else f(zero, std::integral_constant<int, ACT_NONE>{});
    });
}

}  // namespace

std::int64_t group_norm_workspace(const GroupNormShape&, int, bool) { return 0; }

int launch_group_norm_forward(const GroupNormShape& s, int type, const void* x, void* y, const GroupNormForward& f,
                              hipStream_t stream) {
    with_type_and_act(type, f.act, [&](auto zero, auto act) {
        using T = decltype(zero);
        launch(group_norm_kernel<T, decltype(act)::value>, static_cast<unsigned>(s.n * s.groups), NORM_THREADS, 0, stream,
               static_cast<const T*>(x), static_cast<T*>(y), s, f);
    });
    return MFH_CHECK_LAUNCH("group_norm", stream);
}

int launch_group_norm_backward(const GroupNormShape& s, int type, const void* x, const void* dy, void* dx,
                               const GroupNormBackward& b, hipStream_t stream) {
    with_type_and_act(type, b.act, [&](auto zero, auto act) {
        using T = decltype(zero);
        if (dx)
            launch(group_norm_dx_kernel<T, decltype(act)::value>, static_cast<unsigned>(s.n * s.groups), NORM_THREADS, 0,
                   stream, static_cast<const T*>(x), static_cast<const T*>(dy), static_cast<T*>(dx), s, b);
        if (b.gamma_grad || b.beta_grad)
            launch(group_norm_params_kernel<T, decltype(act)::value>, static_cast<unsigned>(s.channels), NORM_THREADS, 0,
                   stream, static_cast<const T*>(x), static_cast<const T*>(dy), s, b);
    });
    return MFH_CHECK_LAUNCH("group_norm_backward", stream);
}

}  // namespace mfh
