// Rows of logits: log probabilities of given tokens with the rows' entropy and top alternatives, the
// distillation loss against a teacher's top logits, and both gradients.
//
// With m = max z, s = sum e^(z - m) of a row:
//   log_sum = m + ln s,  log_prob = (z[t] - m) - ln s,  entropy = ln s - (1/s) sum e^(z - m) (z - m)
//   d log_prob / dz[j] = [j = t] - p[j],  d entropy / dz[j] = -p[j] (ln p[j] + entropy),  p = e^(z - m) / s
// and, with the student's q = softmax(z / T) and the teacher's p over the ids its record holds,
//   row_loss = T^2 sum p (ln p - ln q[id]),  loss = sum w row_loss / sum w,
//   d loss / dz[j] = (w / sum w) T (q[j] - sum over k of p[k] [id[k] = j]).
// A logit of -inf has p = 0 and adds nothing to any sum; a row of nothing else has s = 0: log_sum and
// log_prob -inf, entropy 0, gradient 0. A NaN or +inf makes its row NaN. All sums are float32.
#include <algorithm>
#include <cstdint>

#include "common.h"
#include "typed.h"

namespace mfh {
namespace {

constexpr int ROW_THREADS = 256;
constexpr int MEAN_THREADS = 1024;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LOWEST = -3.402823466e38f;
// e^(z - m) is 0 in float32 from a difference of -104 on; a difference that is multiplied by it is held
// above this, so that -inf (a masked logit, or an overflow) does not make 0 * -inf.
constexpr float DIFFERENCE_FLOOR = -200.0f;

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// The running softmax statistics of a set of logits. m starts at the lowest float, so that a set of -inf
// alone has s = 0. scale = log2(e) / T turns a difference of logits into the exponent of 2.
struct RowStats {
    float m, s, t;  // t = sum e (z - m), for T = 1

    static __device__ __forceinline__ RowStats none() { return {LOWEST, 0.0f, 0.0f}; }

    __device__ __forceinline__ void rescale(float to, float scale) {
        const float d = fmaxf(m - to, DIFFERENCE_FLOOR / scale);
        const float f = exp2_of(d * scale);
        t = f * (t + s * d);
        s *= f;
        m = to;
    }
    __device__ __forceinline__ void add(float z, float scale) {
        const float d = z - m;
        const float e = exp2_of(d * scale);
        s += e;
        t += e * fmaxf(d, DIFFERENCE_FLOOR);
    }
};

// Keys order logits by (value, lower index first) as unsigned 64-bit numbers; -0 counts as 0. NaN is
// never made a key. 0 lies below every key.
__device__ __forceinline__ unsigned long long key_of(float z, int index) {
    const unsigned bits = __float_as_uint(z + 0.0f);
    const unsigned order = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
    return (static_cast<unsigned long long>(order) << 32) | (0xffffffffu - static_cast<unsigned>(index));
}
__device__ __forceinline__ float key_value(unsigned long long key) {
    const unsigned order = static_cast<unsigned>(key >> 32);
    return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ int key_index(unsigned long long key) {
    return static_cast<int>(0xffffffffu - static_cast<unsigned>(key));
}

constexpr float NOT_A_NUMBER = __builtin_nanf("");

// What the last step of a row of log probabilities knows of it (by one thread).
struct RowEnd {
    float m, s, ln_s;
    bool empty;  // no logit above -inf
    __device__ __forceinline__ explicit RowEnd(const RowStats& row) : m(row.m), s(row.s), ln_s(logf(row.s)), empty(row.s == 0.0f) {}
    __device__ __forceinline__ float log_prob(float z) const { return empty ? -INFINITY : (z - m) - ln_s; }
};

template <typename T>
__device__ __forceinline__ void finish_log_probs(const LogProbsForward& f, const T* __restrict__ z, long long r,
                                                 const RowStats& row) {
    const RowEnd end(row);
    f.stats[r] = end.m;
    f.stats[f.rows + r] = end.s;
    f.log_sum[r] = end.empty ? -INFINITY : end.m + end.ln_s;
    f.entropy[r] = end.empty ? 0.0f : end.ln_s - row.t / row.s;
    if (!f.log_prob) return;
    const long long t = whole_at(f.tokens, f.tokens_wide, r);
    f.log_prob[r] = t < 0 ? 0.0f : t >= f.vocab ? NOT_A_NUMBER : end.log_prob(static_cast<float>(z[t]));
}

__device__ __forceinline__ void write_top(const LogProbsForward& f, long long r, int k, unsigned long long key,
                                          const RowStats& row) {
    const long long at = r * f.top + k;
    f.top_ids[at] = key ? key_index(key) : -1;
    f.top_log_probs[at] = key ? RowEnd(row).log_prob(key_value(key)) : NOT_A_NUMBER;
}

// The loss of one row, its targets and weight, by all threads of a workgroup. A row that does not count
// (no id held, weight 0) has loss 0 and weight 0, whatever its logits hold; an id beyond the vocabulary
// makes a counting row's loss and gradient NaN.
template <typename T>
__device__ __forceinline__ void finish_distill(const DistillForward& f, const T* __restrict__ z, long long r,
                                               const RowStats& row) {
    __shared__ long long ids[DISTILL_HELD_MAX];
    __shared__ float probs[DISTILL_HELD_MAX];
    const int lane = threadIdx.x;
    const float inv_t = 1.0f / f.temperature;
    if (lane < 64) {
        const float ln_s = logf(row.s);
        float most = -INFINITY, bad = 0.0f;
        for (int k = lane; k < f.held; k += 64) {
            const long long id = whole_at(f.ids, f.ids_wide, r * f.held + k);
            const float u = id < 0 ? -INFINITY : f.teacher[r * f.held + k] * inv_t;
            ids[k] = id;
            probs[k] = u;
            if (id >= f.vocab) bad = 1.0f;
            most = u > most || u != u ? u : most;
        }
        for (int o = 32; o > 0; o /= 2) {
            const float other = __shfl_xor(most, o);
            most = other > most || other != other ? other : most;
            bad = fmaxf(bad, __shfl_xor(bad, o));
        }
        float sum = 0.0f;
        if (most > -INFINITY || most != most) {
            for (int k = lane; k < f.held; k += 64) sum += exp2_of((probs[k] - most) * LOG2E);
            for (int o = 32; o > 0; o /= 2) sum += __shfl_xor(sum, o);
        }
        const bool counts = sum != 0.0f && (!f.row_weights || f.row_weights[r] != 0.0f);
        const float ln_sum = logf(sum);
        float loss = 0.0f;
        for (int k = lane; k < f.held; k += 64) {
            const float d = probs[k] - most;
            const float p = counts ? exp2_of(d * LOG2E) / sum : 0.0f;
            probs[k] = p;
            if (p == 0.0f || ids[k] >= f.vocab) continue;
            const float log_q = row.s == 0.0f ? -INFINITY : (static_cast<float>(z[ids[k]]) - row.m) * inv_t - ln_s;
            loss += p * (d - ln_sum - log_q);
        }
        for (int o = 32; o > 0; o /= 2) loss += __shfl_xor(loss, o);
        if (lane == 0) {
            const bool poisoned = counts && bad != 0.0f;
            f.row_loss[r] = !counts ? 0.0f : poisoned ? NOT_A_NUMBER : f.temperature * f.temperature * loss;
            f.weights[r] = !counts ? 0.0f : f.row_weights ? f.row_weights[r] : 1.0f;
            f.stats[r] = row.m;
            f.stats[f.rows + r] = poisoned ? NOT_A_NUMBER : row.s;
        }
    }
    __syncthreads();
    // An id that the record holds twice has the sum of its probabilities as its target.
    for (int k = lane; k < f.held; k += blockDim.x) {
        float p = 0.0f;
        for (int other = 0; other < f.held; ++other) p += ids[other] == ids[k] ? probs[other] : 0.0f;
        f.targets[r * f.held + k] = p;
    }
}

// The statistics of a whole row, the same in every thread of the workgroup.
template <typename T>
__device__ __forceinline__ RowStats row_stats(const T* __restrict__ z, int vocab, float scale) {
    __shared__ RowStats part[ROW_THREADS];
    RowStats mine = RowStats::none();
    for (int j = threadIdx.x; j < vocab; j += ROW_THREADS) {
        const float x = static_cast<float>(z[j]);
        if (x > mine.m) mine.rescale(x, scale);
        mine.add(x, scale);
    }
    part[threadIdx.x] = mine;
    __syncthreads();
    for (int half = ROW_THREADS / 2; half > 0; half /= 2) {
        if (static_cast<int>(threadIdx.x) < half) {
            RowStats a = part[threadIdx.x], b = part[threadIdx.x + half];
            const float m = fmaxf(a.m, b.m);
            a.rescale(m, scale);
            b.rescale(m, scale);
            a.s += b.s;
            a.t += b.t;
            part[threadIdx.x] = a;
        }
        __syncthreads();
    }
    return part[0];
}

template <typename T>
__global__ __launch_bounds__(ROW_THREADS) void log_probs_kernel(const T* __restrict__ logits, LogProbsForward f) {
    __shared__ unsigned long long best[ROW_THREADS];
    const long long r = blockIdx.x;
    const T* __restrict__ z = logits + r * f.stride;
    const RowStats row = row_stats(z, f.vocab, LOG2E);
    if (threadIdx.x == 0) finish_log_probs(f, z, r, row);
    unsigned long long last = ~0ull;
    for (int k = 0; k < f.top; ++k) {
        unsigned long long key = 0;
        for (int j = threadIdx.x; j < f.vocab; j += ROW_THREADS) {
            const float x = static_cast<float>(z[j]);
            const unsigned long long c = key_of(x, j);
            if (x == x && c < last && c > key) key = c;
        }
        best[threadIdx.x] = key;
        __syncthreads();
        for (int half = ROW_THREADS / 2; half > 0; half /= 2) {
            if (static_cast<int>(threadIdx.x) < half && best[threadIdx.x + half] > best[threadIdx.x])
                best[threadIdx.x] = best[threadIdx.x + half];
            __syncthreads();
        }
        last = best[0];
        __syncthreads();
        if (threadIdx.x == 0) write_top(f, r, k, last, row);
    }
}

template <typename T>
__global__ __launch_bounds__(ROW_THREADS) void distill_kernel(const T* __restrict__ logits, DistillForward f) {
    const long long r = blockIdx.x;
    const T* __restrict__ z = logits + r * f.stride;
    finish_distill(f, z, r, row_stats(z, f.vocab, LOG2E / f.temperature));
}

template <typename T>
__global__ __launch_bounds__(ROW_THREADS) void log_probs_backward_kernel(const T* __restrict__ logits, T* grad,
                                                                         LogProbsBackward b) {
    const long long r = blockIdx.x;
    const T* __restrict__ z = logits + r * b.stride;
    T* out = grad + r * b.grad_stride;
    const float m = b.stats[r], s = b.stats[b.rows + r], inv = s == 0.0f ? 0.0f : 1.0f / s;
    const long long t = b.log_prob_grad ? whole_at(b.tokens, b.tokens_wide, r) : -1;
    const float factor = b.factor ? b.factor[0] : 1.0f;
    float g = t < 0 || s == 0.0f ? 0.0f : b.scale * factor * b.log_prob_grad[r * b.log_prob_step];
    if (t >= b.vocab) g = NOT_A_NUMBER;
    const float h = b.entropy_grad && s != 0.0f ? factor * b.entropy_grad[r * b.entropy_step] : 0.0f;
    const float c = h != 0.0f ? b.entropy[r] - logf(s) : 0.0f;
    for (int j = threadIdx.x; j < b.vocab; j += ROW_THREADS) {
        const float d = static_cast<float>(z[j]) - m;
        const float p = exp2_of(d * LOG2E) * inv;
        float v = -p * (g + h * (fmaxf(d, DIFFERENCE_FLOOR) + c));
        if (j == t) v += g;
        if (g == 0.0f && h == 0.0f) v = 0.0f;
        out[j] = static_cast<T>(b.add ? static_cast<float>(out[j]) + v : v);
    }
}

template <typename T>
__global__ __launch_bounds__(ROW_THREADS) void distill_backward_kernel(const T* __restrict__ logits, T* grad,
                                                                       DistillBackward b) {
    const long long r = blockIdx.x;
    const T* __restrict__ z = logits + r * b.stride;
    T* out = grad + r * b.grad_stride;
    const float m = b.stats[r], s = b.stats[b.rows + r], inv = s == 0.0f ? 0.0f : 1.0f / s;
    const float scale = LOG2E / b.temperature;
    const float w = b.weights[r];
    const float coef = w == 0.0f ? 0.0f : b.seed[0] * w * b.loss[1] * b.temperature;
    for (int j = threadIdx.x; j < b.vocab; j += ROW_THREADS) {
        float q = exp2_of((static_cast<float>(z[j]) - m) * scale) * inv;
        for (int k = 0; k < b.held; ++k)
            if (whole_at(b.ids, b.ids_wide, r * b.held + k) == j) {
                q -= b.targets[r * b.held + k];
                break;
            }
        const float v = w == 0.0f ? 0.0f : coef * q;
        out[j] = static_cast<T>(b.add ? static_cast<float>(out[j]) + v : v);
    }
}

// out[0] = scale * sum w v / sum w and out[1] = 1 / sum w (both 0 when nothing counts), in FP64: thread t
// adds rows t, t + threads, ... in order, a fixed tree the threads' sums. w is the row's weight, or whether
// its token is given, or 1; a row of weight 0 adds nothing, whatever its value is.
__global__ __launch_bounds__(MEAN_THREADS) void row_mean_kernel(const float* __restrict__ values,
                                                                const float* __restrict__ weights,
                                                                const void* __restrict__ tokens, int tokens_wide,
                                                                long long rows, float scale, float* __restrict__ out) {
    __shared__ double sum[MEAN_THREADS], weight[MEAN_THREADS];
    double a = 0.0, b = 0.0;
    for (long long r = threadIdx.x; r < rows; r += MEAN_THREADS) {
        const float w = weights ? weights[r] : tokens && whole_at(tokens, tokens_wide, r) < 0 ? 0.0f : 1.0f;
        if (w == 0.0f) continue;
        a += static_cast<double>(w) * static_cast<double>(values[r]);
        b += static_cast<double>(w);
    }
    sum[threadIdx.x] = a;
    weight[threadIdx.x] = b;
    __syncthreads();
    for (int half = MEAN_THREADS / 2; half > 0; half /= 2) {
        if (static_cast<int>(threadIdx.x) < half) {
            sum[threadIdx.x] += sum[threadIdx.x + half];
            weight[threadIdx.x] += weight[threadIdx.x + half];
        }
        __syncthreads();
    }
    if (threadIdx.x != 0) return;
    out[0] = weight[0] == 0.0 ? 0.0f : static_cast<float>(scale * sum[0] / weight[0]);
    out[1] = weight[0] == 0.0 ? 0.0f : static_cast<float>(1.0 / weight[0]);
}

}  // namespace

std::int64_t log_probs_workspace(std::int64_t, int, int, int) { return 0; }
std::int64_t distill_workspace(std::int64_t, int, int) { return 0; }

int launch_log_probs(const void* logits, int type, const LogProbsForward& f, hipStream_t stream) {
    if (f.rows == 0) return OK;
    with_type(type, [&](auto zero) {
        using T = decltype(zero);
        launch(log_probs_kernel<T>, static_cast<unsigned>(f.rows), ROW_THREADS, 0, stream, static_cast<const T*>(logits), f);
    });
    return MFH_CHECK_LAUNCH("log_probs", stream);
}

int launch_log_probs_backward(const void* logits, void* grad, int type, const LogProbsBackward& b, hipStream_t stream) {
    if (b.rows == 0) return OK;
    with_type(type, [&](auto zero) {
        using T = decltype(zero);
        launch(log_probs_backward_kernel<T>, static_cast<unsigned>(b.rows), ROW_THREADS, 0, stream,
               static_cast<const T*>(logits), static_cast<T*>(grad), b);
    });
    return MFH_CHECK_LAUNCH("log_probs_backward", stream);
}

int launch_distill(const void* logits, int type, const DistillForward& f, hipStream_t stream) {
    if (f.rows != 0) {
        with_type(type, [&](auto zero) {
            using T = decltype(zero);
            launch(distill_kernel<T>, static_cast<unsigned>(f.rows), ROW_THREADS, 0, stream, static_cast<const T*>(logits), f);
        });
        MFH_TRY(MFH_CHECK_LAUNCH("distill", stream));
    }
    return launch_row_mean(f.row_loss, f.weights, nullptr, 0, f.rows, 1.0f, f.loss, stream);
}

int launch_distill_backward(const void* logits, void* grad, int type, const DistillBackward& b, hipStream_t stream) {
    if (b.rows == 0) return OK;
    with_type(type, [&](auto zero) {
        using T = decltype(zero);
        launch(distill_backward_kernel<T>, static_cast<unsigned>(b.rows), ROW_THREADS, 0, stream,
               static_cast<const T*>(logits), static_cast<T*>(grad), b);
    });
    return MFH_CHECK_LAUNCH("distill_backward", stream);
}

int launch_row_mean(const float* values, const float* weights, const void* tokens, int tokens_wide, std::int64_t rows,
                    float scale, float* out, hipStream_t stream) {
    launch(row_mean_kernel, 1, MEAN_THREADS, 0, stream, values, weights, tokens, tokens_wide, rows, scale, out);
    return MFH_CHECK_LAUNCH("row_mean", stream);
}

}  // namespace mfh
