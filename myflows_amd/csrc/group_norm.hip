// Group norm with an activation over channels-last activations (n, positions, channels), and its gradients.
//
// A group is channels / groups neighbouring channels of one sample, over all its positions. With its mean
// and biased variance:
//   xhat = (x - mean) inv_std,  u = gamma xhat + beta,  y = act(u)      inv_std = (variance + eps)^(-1/2)
// and, with du = dy act'(u) and the averages over the group,
//   dgamma[c] = sum du xhat,  dbeta[c] = sum du,
//   dx = inv_std (gamma du - average(gamma du) - xhat average(gamma du xhat)).
// u is formed as a (x - mean) + beta, a = gamma inv_std, in every pass alike (affine): the backward's ReLU lets
// through exactly what the forward's did.
// Sums are float32; the variance is a sum of squares about a mean, never a difference of large sums. Every
// sum is formed in one fixed order.
//
// Two routes, both bound by HBM (or, in small calls, by latency):
//   * held: a workgroup reads its groups of a sample into registers, once, forms the sums and writes the
//     result from there. One launch forward; backward a second one adds the samples' dgamma and dbeta.
//     64 x 1131 x 64 float32 in 32 groups 12.8 us forward (2.9 TB/s), 13.8 backward (4.0): 256 workgroups, one a
//     CU, whose loads, sums and stores follow one another; the split route took 22.5 and 30;
//   * split: groups that no workgroup holds are summed by runs of positions over many workgroups, the runs
//     joined, and a last launch reads the activations again. It starts with those read last, which a cache
//     still holds. 16 x 16384 x 256 bfloat16: 26 + 42 us forward (5.1 and 6.4 TB/s), 53 + 66 backward (5.0 and 6.1).
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "common.h"
#include "group_norm_plan.h"
#include "typed.h"
#include "wave.h"

namespace mfh {
namespace {

// A plan's block as the kernels take it (GroupNormPlan's fields).
struct Block {
    int per, groups, parts, width, blocks, lanes;
    FastDiv per_div;
};
constexpr int BLOCK_GROUPS_MAX = GROUP_NORM_BLOCK_GROUPS;

// The place of a block: its first channel, its channels and its first group.
struct Place {
    int channel, width, group, part;
};
__device__ __forceinline__ Place place_of(const Block& k, int index) {
    if (k.parts == 1) return {index * k.width, k.width, index * k.groups, 0};
    const int group = index / k.parts, part = index - group * k.parts;
    return {group * k.per + part * k.width, min(k.width, k.per - part * k.width), group, part};
}

// ---- activations -----------------------------------------------------------------------------
// ReLU and no activation are one form: the larger of u and a floor of 0 or -inf (a NaN stays).
__device__ __forceinline__ float sigmoid_of(float u) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * u));
}
template <bool SILU>
__device__ __forceinline__ float activate(float u, float floor) {
    if constexpr (SILU) return u * sigmoid_of(u);
    return u < floor ? floor : u;
}
// u, rounded the same way in every pass.
__device__ __forceinline__ float affine(float less_mean, float a, float beta) { return fmaf(less_mean, a, beta); }
__device__ __forceinline__ float inv_std_of(float squares, float inv_count, float eps) {
    return 1.0f / sqrtf(fmaf(squares, inv_count, eps));
}
// dy act'(u)
template <bool SILU>
__device__ __forceinline__ float through(float u, float dy, float floor) {
    if constexpr (SILU) {
        const float g = sigmoid_of(u);
        return dy * (g * (1.0f + u * (1.0f - g)));
    }
    return u <= floor ? 0.0f : dy;
}

// ---- sums over a block -----------------------------------------------------------------------
// Each thread brings VW columns' sums over its rows. Rows of one wave are joined across its lanes, the rest
// through LDS, part by part in order.
template <int THREADS, int VW>
struct ColumnSums {
    static constexpr int FLOATS = THREADS * VW;

    // Whether a wave's rows are joined across its lanes; parts that a column then has in LDS, and the floats from
    // one part to the next.
    static __device__ __forceinline__ bool joined(const Block& k) { return k.lanes <= 32; }
    static __device__ __forceinline__ int parts(const Block& k) { return joined(k) ? THREADS / 64 : THREADS / k.lanes; }
    static __device__ __forceinline__ int pitch(const Block& k) { return VW * k.lanes; }

    static __device__ __forceinline__ void put(const Block& k, float (&lds)[FLOATS], const float (&mine)[VW]) {
        float v[VW];
#pragma unroll
        for (int i = 0; i < VW; ++i) v[i] = mine[i];
        const int tid = threadIdx.x;
        int part = tid / k.lanes, lane = tid - part * k.lanes;
        if (joined(k)) {
            for (int o = k.lanes; o < 64; o <<= 1)
#pragma unroll
                for (int i = 0; i < VW; ++i) v[i] += __shfl_xor(v[i], o);
            part = tid / 64;
            if ((tid & 63) >= k.lanes) return;
        } else if (part >= parts(k)) {
            return;
        }
        float* to = lds + part * pitch(k) + lane * VW;
#pragma unroll
        for (int i = 0; i < VW; ++i) to[i] = v[i];
    }

    // sums[g] = the sum of group g's columns and parts (a wave a group).
    static __device__ __forceinline__ void groups(const Block& k, int width, const float (&lds)[FLOATS], float* sums) {
        const int wave = threadIdx.x / 64, lane = threadIdx.x & 63, step = pitch(k);
        const int per = k.parts == 1 ? k.per : width, count = parts(k) * per;
        for (int g = wave; g < k.groups; g += THREADS / 64) {
            float s = 0.0f;
            for (int i = lane; i < count; i += 64) {
                const int part = k.parts == 1 ? k.per_div.div(i) : i / per;
                s += lds[part * step + g * per + (i - part * per)];
            }
            s = wave_sum(s);
            if (lane == 0) sums[g] = s;
        }
    }
};

// The group sums of the threads' column sums, for each thread's columns.
template <int THREADS, int VW>
__device__ __forceinline__ void group_sums(const Block& k, int width, float (&lds)[THREADS * VW], float* sums,
                                           const int (&group)[VW], const float (&mine)[VW], float (&result)[VW]) {
    __syncthreads();  // what the last call left is read
    ColumnSums<THREADS, VW>::put(k, lds, mine);
    __syncthreads();
    ColumnSums<THREADS, VW>::groups(k, width, lds, sums);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < VW; ++i) result[i] = sums[group[i]];
}

// A thread's place in a block: its columns, first row and the rows from one of its rows to the next.
template <int THREADS, int VW>
struct Thread {
    int column, row, step;
    bool active;
    int group[VW];  // of the block's groups

    __device__ __forceinline__ Thread(const Block& k, int width) {
        const int tid = threadIdx.x;
        row = tid / k.lanes;
        column = (tid - row * k.lanes) * VW;
        step = THREADS / k.lanes;
        active = column < width && row < step;
#pragma unroll
        for (int i = 0; i < VW; ++i) group[i] = active && k.parts == 1 ? k.per_div.div(column + i) : 0;
    }
    // The values of this thread's columns in an array by channel (0 for an idle thread).
    __device__ __forceinline__ void by_column(const float* __restrict__ values, float (&to)[VW]) const {
#pragma unroll
        for (int i = 0; i < VW; ++i) to[i] = active ? values[column + i] : 0.0f;
    }
    __device__ __forceinline__ void by_group(const float* __restrict__ values, float (&to)[VW]) const {
#pragma unroll
        for (int i = 0; i < VW; ++i) to[i] = active ? values[group[i]] : 0.0f;
    }
};

template <typename T, int VW, int HOLD>
__device__ __forceinline__ void stay_packed(Pack<T, VW> (&held)[HOLD]) {
#pragma unroll
    for (int h = 0; h < HOLD; ++h) held[h].stay_packed();
}

template <typename T, int VW>
__device__ __forceinline__ void add_pack(float (&out)[VW], const T* from) {
    const Pack<T, VW> old = load_pack<T, VW>(from);
#pragma unroll
    for (int i = 0; i < VW; ++i) out[i] += old.at(i);
}

// Neighbouring blocks of a sample share cache lines where a block's row is narrower than one: the workgroups
// are dealt round-robin to the 8 XCDs, so each XCD takes one run of the blocks.
__device__ __forceinline__ unsigned xcd_run(unsigned total) {
    return total % 8 ? blockIdx.x : (blockIdx.x & 7) * (total / 8) + blockIdx.x / 8;
}

// ---- held ------------------------------------------------------------------------------------
template <typename T, int VW, bool SILU, int THREADS, int HOLD>
__global__ __launch_bounds__(THREADS) void held_forward_kernel(const T* __restrict__ x, T* __restrict__ y,
                                                               GroupNormShape s, Block k, GroupNormForward f) {
    __shared__ float lds[THREADS * VW], sums[BLOCK_GROUPS_MAX];
    const unsigned at = xcd_run(gridDim.x), sample = at / static_cast<unsigned>(k.blocks);
    const long long n = sample;
    const Place place = place_of(k, static_cast<int>(at - sample * k.blocks));
    const Thread<THREADS, VW> t(k, place.width);
    const long long base = n * s.positions * s.channels + place.channel + t.column;
    Pack<T, VW> held[HOLD];
    float sum[VW] = {}, mean[VW], squares[VW] = {}, a[VW], beta[VW];
#pragma unroll
    for (int h = 0; h < HOLD; ++h) {
        if (h * t.step >= s.positions) break;
        const int row = t.row + h * t.step;
        if (t.active && row < s.positions) held[h] = load_pack<T, VW>(x + base + row * s.channels);
    }
    t.by_column(f.gamma + place.channel, a);
    t.by_column(f.beta + place.channel, beta);
#pragma unroll
    for (int h = 0; h < HOLD; ++h) {
        if (h * t.step >= s.positions) break;
        if (t.active && t.row + h * t.step < s.positions)
#pragma unroll
            for (int i = 0; i < VW; ++i) sum[i] += held[h].at(i);
    }
    stay_packed(held);
    group_sums<THREADS, VW>(k, place.width, lds, sums, t.group, sum, mean);
    const float inv_count = 1.0f / (static_cast<float>(s.positions) * static_cast<float>(k.per));
#pragma unroll
    for (int i = 0; i < VW; ++i) mean[i] *= inv_count;
    if (static_cast<int>(threadIdx.x) < k.groups) f.mean[n * s.groups + place.group + threadIdx.x] = sums[threadIdx.x] * inv_count;
#pragma unroll
    for (int h = 0; h < HOLD; ++h) {
        if (h * t.step >= s.positions) break;
        if (t.active && t.row + h * t.step < s.positions)
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                const float d = held[h].at(i) - mean[i];
                squares[i] += d * d;
            }
    }
    float variance[VW];
    stay_packed(held);
    group_sums<THREADS, VW>(k, place.width, lds, sums, t.group, squares, variance);
    if (static_cast<int>(threadIdx.x) < k.groups)
        f.inv_std[n * s.groups + place.group + threadIdx.x] = inv_std_of(sums[threadIdx.x], inv_count, f.eps);
#pragma unroll
    for (int i = 0; i < VW; ++i) a[i] *= inv_std_of(variance[i], inv_count, f.eps);
    const float floor = f.act == ACT_RELU ? 0.0f : -INFINITY;
#pragma unroll
    for (int h = 0; h < HOLD; ++h) {
        if (h * t.step >= s.positions) break;
        const int row = t.row + h * t.step;
        if (t.active && row < s.positions) {
            float out[VW];
#pragma unroll
            for (int i = 0; i < VW; ++i) out[i] = activate<SILU>(affine(held[h].at(i) - mean[i], a[i], beta[i]), floor);
            store_pack(y + base + row * s.channels, Pack<T, VW>::of(out));
        }
    }
}

// What the backward forms of an element: xhat and du, with a = gamma inv as in the forward.
template <bool SILU>
struct Backward {
    float hat, du;
    __device__ __forceinline__ Backward(float x, float dy, float mean, float inv, float a, float beta, float floor) {
        const float d = x - mean;
        hat = d * inv;
        du = through<SILU>(affine(d, a, beta), dy, floor);
    }
    // dx from the group's averages of gamma du and gamma du xhat.
    __device__ __forceinline__ float dx(float inv, float a, float average, float average_hat) const {
        return du * a - inv * (average + hat * average_hat);
    }
};

// columns[2 c], columns[2 c + 1] = sum du, sum du xhat of channel c of a sample.
template <typename T, int VW, bool SILU, int THREADS, int HOLD>
__global__ __launch_bounds__(THREADS) void held_backward_kernel(const T* __restrict__ x, const T* __restrict__ dy, T* dx,
                                                                GroupNormShape s, Block k, GroupNormBackward b,
                                                                float* __restrict__ columns) {
    using Sums = ColumnSums<THREADS, VW>;
    __shared__ float first[THREADS * VW], second[THREADS * VW], sums[2][BLOCK_GROUPS_MAX];
    const unsigned at = xcd_run(gridDim.x), sample = at / static_cast<unsigned>(k.blocks);
    const long long n = sample;
    const Place place = place_of(k, static_cast<int>(at - sample * k.blocks));
    const Thread<THREADS, VW> t(k, place.width);
    const long long base = n * s.positions * s.channels + place.channel + t.column;
    Pack<T, VW> held[HOLD], grad[HOLD];
    float mean[VW], inv[VW], a[VW], beta[VW], sum[VW] = {}, product[VW] = {};
#pragma unroll
    for (int h = 0; h < HOLD; ++h) {
        if (h * t.step >= s.positions) break;
        const int row = t.row + h * t.step;
        if (t.active && row < s.positions) {
            held[h] = load_pack<T, VW>(x + base + row * s.channels);
            grad[h] = load_pack<T, VW>(dy + base + row * s.channels);
        }
    }
    t.by_group(b.mean + n * s.groups + place.group, mean);
    t.by_group(b.inv_std + n * s.groups + place.group, inv);
    t.by_column(b.gamma + place.channel, a);
    t.by_column(b.beta + place.channel, beta);
#pragma unroll
    for (int i = 0; i < VW; ++i) a[i] *= inv[i];
    const float floor = b.act == ACT_RELU ? 0.0f : -INFINITY;
    const auto form = [&](int h, int i) {
        return Backward<SILU>(held[h].at(i), grad[h].at(i), mean[i], inv[i], a[i], beta[i], floor);
    };
#pragma unroll
    for (int h = 0; h < HOLD; ++h) {
        if (h * t.step >= s.positions) break;
        if (t.active && t.row + h * t.step < s.positions)
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                const Backward<SILU> e = form(h, i);
                sum[i] += e.du;
                product[i] += e.du * e.hat;
            }
    }
    stay_packed(held);
    stay_packed(grad);
    Sums::put(k, first, sum);
    Sums::put(k, second, product);
    __syncthreads();
    // The columns' sums, weighted by gamma for the groups, take the first part's place.
    const int parts = Sums::parts(k), pitch = Sums::pitch(k);
    for (int c = threadIdx.x; c < place.width; c += THREADS) {
        float d = first[c], p = second[c];
        for (int i = 1; i < parts; ++i) {
            d += first[i * pitch + c];
            p += second[i * pitch + c];
        }
        if (columns) {
            float* to = columns + 2 * (n * s.channels + place.channel + c);
            to[0] = d;
            to[1] = p;
        }
        const float g = b.gamma[place.channel + c];
        first[c] = g * d;
        second[c] = g * p;
    }
    if (!dx) return;
    __syncthreads();
    const int wave = threadIdx.x / 64, lane = threadIdx.x & 63;
    const float inv_count = 1.0f / (static_cast<float>(s.positions) * static_cast<float>(k.per));
    for (int g = wave; g < k.groups; g += THREADS / 64) {
        float d = 0.0f, p = 0.0f;
        for (int c = lane; c < k.per; c += 64) {
            d += first[g * k.per + c];
            p += second[g * k.per + c];
        }
        d = wave_sum(d) * inv_count;
        p = wave_sum(p) * inv_count;
        if (lane == 0) {
            sums[0][g] = d;
            sums[1][g] = p;
        }
    }
    __syncthreads();
    float mean_d[VW], mean_p[VW];
    t.by_group(sums[0], mean_d);
    t.by_group(sums[1], mean_p);
#pragma unroll
    for (int h = 0; h < HOLD; ++h) {
        if (h * t.step >= s.positions) break;
        const int row = t.row + h * t.step;
        if (t.active && row < s.positions) {
            T* to = dx + base + row * s.channels;
            float out[VW];
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                const Backward<SILU> e = form(h, i);
                out[i] = e.dx(inv[i], a[i], mean_d[i], mean_p[i]);
            }
            if (b.add_x) add_pack(out, to);
            store_pack(to, Pack<T, VW>::of(out));
        }
    }
}

// ---- split -----------------------------------------------------------------------------------
constexpr int SPLIT_THREADS = GROUP_NORM_SPLIT_THREADS, SPLIT_AHEAD = GROUP_NORM_SPLIT_AHEAD;

struct Runs {
    int count, rows;  // runs of a sample's positions, and positions of a run
};
struct RunAt {
    long long n;
    int run, begin, end;
    Place place;
};
// The run of a workgroup, forwards through the samples or backwards.
__device__ __forceinline__ RunAt run_at(const Runs& r, const Block& k, int positions, bool backwards) {
    unsigned at = backwards ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
    const unsigned rest = at / static_cast<unsigned>(k.blocks);
    const int block = static_cast<int>(at - rest * k.blocks);
    const unsigned n = rest / static_cast<unsigned>(r.count);
    const int run = static_cast<int>(rest - n * r.count);
    return {n, run, run * r.rows, min(positions, (run + 1) * r.rows), place_of(k, block)};
}

// means and squares [sample][run][group and part]: the mean of a run's values and the squares about it. A
// thread keeps each of its columns' mean and squares, SPLIT_AHEAD rows at a time joined to them by
//   mean += d k / (n + k),  squares += squares' + d^2 n k / (n + k),  d = mean' - mean
// (Chan, Golub and LeVeque, 1983); the threads' are joined about the run's mean.
template <typename T, int VW>
__global__ __launch_bounds__(SPLIT_THREADS) void run_stats_kernel(const T* __restrict__ x, GroupNormShape s, Block k,
                                                                  Runs runs, float* __restrict__ means,
                                                                  float* __restrict__ squares) {
    __shared__ float lds[SPLIT_THREADS * VW], sums[BLOCK_GROUPS_MAX];
    const RunAt r = run_at(runs, k, s.positions, false);
    const Thread<SPLIT_THREADS, VW> t(k, r.place.width);
    const T* __restrict__ from = x + r.n * s.positions * s.channels + r.place.channel + t.column;
    float count = 0.0f, mean[VW] = {}, m2[VW] = {};
    if (t.active) {
        int row = r.begin + t.row;
        for (; row + (SPLIT_AHEAD - 1) * t.step < r.end; row += SPLIT_AHEAD * t.step) {
            Pack<T, VW> packs[SPLIT_AHEAD];
#pragma unroll
            for (int u = 0; u < SPLIT_AHEAD; ++u) packs[u] = load_pack<T, VW>(from + (row + u * t.step) * s.channels);
            const float more = count + SPLIT_AHEAD, share = SPLIT_AHEAD * __builtin_amdgcn_rcpf(more), weight = count * share;
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                float sum = 0.0f, about = 0.0f;
#pragma unroll
                for (int u = 0; u < SPLIT_AHEAD; ++u) sum += packs[u].at(i);
                const float here = sum * (1.0f / SPLIT_AHEAD);
#pragma unroll
                for (int u = 0; u < SPLIT_AHEAD; ++u) {
                    const float d = packs[u].at(i) - here;
                    about += d * d;
                }
                const float d = here - mean[i];
                mean[i] += d * share;
                m2[i] += about + d * d * weight;
            }
            count = more;
        }
        for (; row < r.end; row += t.step) {
            const Pack<T, VW> pack = load_pack<T, VW>(from + row * s.channels);
            const float more = count + 1.0f, share = __builtin_amdgcn_rcpf(more), weight = count * share;
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                const float d = pack.at(i) - mean[i];
                mean[i] += d * share;
                m2[i] += d * d * weight;
            }
            count = more;
        }
    }
    float sum[VW], whole[VW];
#pragma unroll
    for (int i = 0; i < VW; ++i) sum[i] = count * mean[i];
    group_sums<SPLIT_THREADS, VW>(k, r.place.width, lds, sums, t.group, sum, whole);
    const int per = k.parts == 1 ? k.per : r.place.width;
    const float inv_count = 1.0f / (static_cast<float>(r.end - r.begin) * static_cast<float>(per));
    const long long to = (r.n * runs.count + r.run) * s.groups * k.parts + static_cast<long long>(r.place.group) * k.parts + r.place.part;
    if (static_cast<int>(threadIdx.x) < k.groups) means[to + threadIdx.x] = sums[threadIdx.x] * inv_count;
#pragma unroll
    for (int i = 0; i < VW; ++i) {
        const float d = mean[i] - whole[i] * inv_count;
        sum[i] = m2[i] + count * (d * d);
    }
    group_sums<SPLIT_THREADS, VW>(k, r.place.width, lds, sums, t.group, sum, whole);
    if (static_cast<int>(threadIdx.x) < k.groups) squares[to + threadIdx.x] = sums[threadIdx.x];
}

__device__ __forceinline__ float group_sum(float v) {
    __shared__ float part[SPLIT_THREADS / 64];
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x / 64] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int w = 1; w < SPLIT_THREADS / 64; ++w) v += part[w];
    return v;
}

// The runs and parts of each (sample, group) joined: one workgroup each.
__global__ __launch_bounds__(SPLIT_THREADS) void join_stats_kernel(const float* __restrict__ means,
                                                                   const float* __restrict__ squares, GroupNormShape s,
                                                                   Block k, Runs runs, GroupNormForward f) {
    const unsigned sample = blockIdx.x / static_cast<unsigned>(s.groups);
    const int g = static_cast<int>(blockIdx.x - sample * s.groups), pieces = runs.count * k.parts;
    const long long n = sample;
    const auto piece = [&](int i, float& count) {
        const int run = i / k.parts, part = i - run * k.parts;
        const int rows = min(s.positions - run * runs.rows, runs.rows);
        const int columns = k.parts == 1 ? k.per : min(k.width, k.per - part * k.width);
        count = static_cast<float>(rows) * static_cast<float>(columns);
        return ((n * runs.count + run) * s.groups + g) * k.parts + part;
    };
    float sum = 0.0f;
    for (int i = threadIdx.x; i < pieces; i += SPLIT_THREADS) {
        float count;
        const long long from = piece(i, count);
        sum += count * means[from];
    }
    const float inv_count = 1.0f / (static_cast<float>(s.positions) * static_cast<float>(k.per));
    const float mean = group_sum(sum) * inv_count;
    float about = 0.0f;
    for (int i = threadIdx.x; i < pieces; i += SPLIT_THREADS) {
        float count;
        const long long from = piece(i, count);
        const float d = means[from] - mean;
        about += squares[from] + count * (d * d);
    }
    about = group_sum(about);
    if (threadIdx.x != 0) return;
    f.mean[blockIdx.x] = mean;
    f.inv_std[blockIdx.x] = inv_std_of(about, inv_count, f.eps);
}

template <typename T, int VW, bool SILU>
__global__ __launch_bounds__(SPLIT_THREADS) void apply_forward_kernel(const T* __restrict__ x, T* __restrict__ y,
                                                                      GroupNormShape s, Block k, Runs runs,
                                                                      GroupNormForward f) {
    const RunAt r = run_at(runs, k, s.positions, true);
    const Thread<SPLIT_THREADS, VW> t(k, r.place.width);
    if (!t.active) return;
    const long long base = r.n * s.positions * s.channels + r.place.channel + t.column;
    float mean[VW], a[VW], beta[VW], inv[VW];
    t.by_group(f.mean + r.n * s.groups + r.place.group, mean);
    t.by_group(f.inv_std + r.n * s.groups + r.place.group, inv);
    t.by_column(f.gamma + r.place.channel, a);
    t.by_column(f.beta + r.place.channel, beta);
    const float floor = f.act == ACT_RELU ? 0.0f : -INFINITY;
#pragma unroll
    for (int i = 0; i < VW; ++i) a[i] *= inv[i];
    const auto write = [&](int row, const Pack<T, VW>& in) {
        float out[VW];
#pragma unroll
        for (int i = 0; i < VW; ++i) out[i] = activate<SILU>(affine(in.at(i) - mean[i], a[i], beta[i]), floor);
        store_pack(y + base + row * s.channels, Pack<T, VW>::of(out));
    };
    int row = r.begin + t.row;
    for (; row + (SPLIT_AHEAD - 1) * t.step < r.end; row += SPLIT_AHEAD * t.step) {
        Pack<T, VW> packs[SPLIT_AHEAD];
#pragma unroll
        for (int u = 0; u < SPLIT_AHEAD; ++u) packs[u] = load_pack<T, VW>(x + base + (row + u * t.step) * s.channels);
#pragma unroll
        for (int u = 0; u < SPLIT_AHEAD; ++u) write(row + u * t.step, packs[u]);
    }
    for (; row < r.end; row += t.step) write(row, load_pack<T, VW>(x + base + row * s.channels));
}

// run_columns [sample][run][channel][2]: sum du and sum du xhat of a run's positions.
template <typename T, int VW, bool SILU>
__global__ __launch_bounds__(SPLIT_THREADS) void run_gradients_kernel(const T* __restrict__ x, const T* __restrict__ dy,
                                                                      GroupNormShape s, Block k, Runs runs,
                                                                      GroupNormBackward b, float* __restrict__ run_columns) {
    using Sums = ColumnSums<SPLIT_THREADS, VW>;
    __shared__ float first[SPLIT_THREADS * VW], second[SPLIT_THREADS * VW];
    const RunAt r = run_at(runs, k, s.positions, false);
    const Thread<SPLIT_THREADS, VW> t(k, r.place.width);
    const long long base = r.n * s.positions * s.channels + r.place.channel + t.column;
    float mean[VW], inv[VW], a[VW], beta[VW], sum[VW] = {}, product[VW] = {};
    t.by_group(b.mean + r.n * s.groups + r.place.group, mean);
    t.by_group(b.inv_std + r.n * s.groups + r.place.group, inv);
    t.by_column(b.gamma + r.place.channel, a);
    t.by_column(b.beta + r.place.channel, beta);
#pragma unroll
    for (int i = 0; i < VW; ++i) a[i] *= inv[i];
    const float floor = b.act == ACT_RELU ? 0.0f : -INFINITY;
    const auto take = [&](const Pack<T, VW>& in, const Pack<T, VW>& grad) {
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            const Backward<SILU> e(in.at(i), grad.at(i), mean[i], inv[i], a[i], beta[i], floor);
            sum[i] += e.du;
            product[i] += e.du * e.hat;
        }
    };
    if (t.active) {
        int row = r.begin + t.row;
        for (; row + (SPLIT_AHEAD - 1) * t.step < r.end; row += SPLIT_AHEAD * t.step) {
            Pack<T, VW> in[SPLIT_AHEAD], grad[SPLIT_AHEAD];
#pragma unroll
            for (int u = 0; u < SPLIT_AHEAD; ++u) {
                in[u] = load_pack<T, VW>(x + base + (row + u * t.step) * s.channels);
                grad[u] = load_pack<T, VW>(dy + base + (row + u * t.step) * s.channels);
            }
#pragma unroll
            for (int u = 0; u < SPLIT_AHEAD; ++u) take(in[u], grad[u]);
        }
        for (; row < r.end; row += t.step)
            take(load_pack<T, VW>(x + base + row * s.channels), load_pack<T, VW>(dy + base + row * s.channels));
    }
    Sums::put(k, first, sum);
    Sums::put(k, second, product);
    __syncthreads();
    const int parts = Sums::parts(k), pitch = Sums::pitch(k);
    for (int c = threadIdx.x; c < r.place.width; c += SPLIT_THREADS) {
        float d = first[c], p = second[c];
        for (int i = 1; i < parts; ++i) {
            d += first[i * pitch + c];
            p += second[i * pitch + c];
        }
        float* to = run_columns + 2 * ((r.n * runs.count + r.run) * s.channels + r.place.channel + c);
        to[0] = d;
        to[1] = p;
    }
}

// out[outer][j] = the sum over `inner` rows of from[outer][row][j], j < columns: 16 runs of rows a column, each in
// order, then in run order.
constexpr int COLUMN_SPAN = GROUP_NORM_COLUMN_SPAN, COLUMN_RUNS = GROUP_NORM_COLUMN_RUNS;
__device__ __forceinline__ float sum_of_rows(const float* __restrict__ from, long long rows, long long columns, long long j,
                                             float (&lds)[COLUMN_RUNS][COLUMN_SPAN]) {
    const int c = threadIdx.x % COLUMN_SPAN, g = threadIdx.x / COLUMN_SPAN;
    const long long each = (rows + COLUMN_RUNS - 1) / COLUMN_RUNS, last = min(rows, (g + 1) * each);
    float s = 0.0f;
    if (j < columns) {
        long long row = g * each;
        for (; row + 8 <= last; row += 8) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = from[(row + u) * columns + j];
#pragma unroll
            for (int u = 0; u < 8; ++u) s += v[u];
        }
        for (; row < last; ++row) s += from[row * columns + j];
    }
    lds[g][c] = s;
    __syncthreads();
    if (g == 0)
#pragma unroll
        for (int i = 1; i < COLUMN_RUNS; ++i) s += lds[i][c];
    return s;  // of the first COLUMN_SPAN threads
}

__global__ __launch_bounds__(COLUMN_SPAN* COLUMN_RUNS) void join_columns_kernel(const float* __restrict__ run_columns,
                                                                                int runs, int columns, int tiles,
                                                                                float* __restrict__ out) {
    __shared__ float lds[COLUMN_RUNS][COLUMN_SPAN];
    const long long n = blockIdx.x / tiles, j = (blockIdx.x % tiles) * COLUMN_SPAN + threadIdx.x % COLUMN_SPAN;
    const float s = sum_of_rows(run_columns + n * runs * columns, runs, columns, j, lds);
    if (threadIdx.x < COLUMN_SPAN && j < columns) out[n * columns + j] = s;
}

// dbeta and dgamma: the sums of columns [sample][channel][2] over the samples.
__global__ __launch_bounds__(COLUMN_SPAN* COLUMN_RUNS) void parameter_grads_kernel(const float* __restrict__ columns,
                                                                                   GroupNormShape s, GroupNormBackward b) {
    __shared__ float lds[COLUMN_RUNS][COLUMN_SPAN];
    const long long j = static_cast<long long>(blockIdx.x) * COLUMN_SPAN + threadIdx.x % COLUMN_SPAN;
    const float v = sum_of_rows(columns, s.n, 2LL * s.channels, j, lds);
    if (threadIdx.x >= COLUMN_SPAN || j >= 2LL * s.channels) return;
    float* out = j & 1 ? b.gamma_grad : b.beta_grad;
    if (!out) return;
    const bool add = j & 1 ? b.add_gamma : b.add_beta;
    out[j / 2] = add ? out[j / 2] + v : v;
}

template <typename T, int VW, bool SILU>
__global__ __launch_bounds__(SPLIT_THREADS) void apply_backward_kernel(const T* __restrict__ x, const T* __restrict__ dy,
                                                                       T* dx, GroupNormShape s, Block k, Runs runs,
                                                                       GroupNormBackward b,
                                                                       const float* __restrict__ columns) {
    __shared__ float sums[2][BLOCK_GROUPS_MAX];
    const RunAt r = run_at(runs, k, s.positions, true);
    const Thread<SPLIT_THREADS, VW> t(k, r.place.width);
    const int wave = threadIdx.x / 64, lane = threadIdx.x & 63;
    const float inv_count = 1.0f / (static_cast<float>(s.positions) * static_cast<float>(k.per));
    for (int g = wave; g < k.groups; g += SPLIT_THREADS / 64) {
        const int channel = (r.place.group + g) * k.per;
        const float* __restrict__ from = columns + 2 * (r.n * s.channels + channel);
        float d = 0.0f, p = 0.0f;
        for (int c = lane; c < k.per; c += 64) {
            const float gamma = b.gamma[channel + c];
            d += gamma * from[2 * c];
            p += gamma * from[2 * c + 1];
        }
        d = wave_sum(d) * inv_count;
        p = wave_sum(p) * inv_count;
        if (lane == 0) {
            sums[0][g] = d;
            sums[1][g] = p;
        }
    }
    __syncthreads();
    if (!t.active) return;
    const long long base = r.n * s.positions * s.channels + r.place.channel + t.column;
    float mean[VW], inv[VW], a[VW], beta[VW], mean_d[VW], mean_p[VW];
    t.by_group(b.mean + r.n * s.groups + r.place.group, mean);
    t.by_group(b.inv_std + r.n * s.groups + r.place.group, inv);
    t.by_column(b.gamma + r.place.channel, a);
    t.by_column(b.beta + r.place.channel, beta);
#pragma unroll
    for (int i = 0; i < VW; ++i) a[i] *= inv[i];
    t.by_group(sums[0], mean_d);
    t.by_group(sums[1], mean_p);
    const float floor = b.act == ACT_RELU ? 0.0f : -INFINITY;
    const auto write = [&](int row, const Pack<T, VW>& in, const Pack<T, VW>& grad) {
        T* to = dx + base + row * s.channels;
        float out[VW];
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            const Backward<SILU> e(in.at(i), grad.at(i), mean[i], inv[i], a[i], beta[i], floor);
            out[i] = e.dx(inv[i], a[i], mean_d[i], mean_p[i]);
        }
        if (b.add_x) add_pack(out, to);
        store_pack(to, Pack<T, VW>::of(out));
    };
    int row = r.begin + t.row;
    for (; row + (SPLIT_AHEAD - 1) * t.step < r.end; row += SPLIT_AHEAD * t.step) {
        Pack<T, VW> in[SPLIT_AHEAD], grad[SPLIT_AHEAD];
#pragma unroll
        for (int u = 0; u < SPLIT_AHEAD; ++u) {
            in[u] = load_pack<T, VW>(x + base + (row + u * t.step) * s.channels);
            grad[u] = load_pack<T, VW>(dy + base + (row + u * t.step) * s.channels);
        }
#pragma unroll
        for (int u = 0; u < SPLIT_AHEAD; ++u) write(row + u * t.step, in[u], grad[u]);
    }
    for (; row < r.end; row += t.step)
        write(row, load_pack<T, VW>(x + base + row * s.channels), load_pack<T, VW>(dy + base + row * s.channels));
}

// ---- launches --------------------------------------------------------------------------------
Block block_of(const GroupNormPlan& plan) {
    return {plan.per, plan.groups, plan.parts, plan.width, plan.blocks, plan.lanes, FastDiv(plan.per)};
}

// Calls f(first sample, the slice's shape) for each slice of the samples that a launch takes.
template <typename F>
int for_slices(const GroupNormShape& s, std::int64_t slice, F&& f) {
    for (std::int64_t first = 0; first < s.n; first += slice) {
        GroupNormShape part = s;
        part.n = std::min(slice, s.n - first);
        MFH_TRY(f(first, part));
    }
    return OK;
}

// Calls f with the element type, the pack's size and whether the activation is SiLU as types.
template <typename F>
void with_kernel(int type, int vw, int act, F&& f) {
    with_type(type, [&](auto zero) {
        using T = decltype(zero);
        constexpr int WIDE = 16 / sizeof(T);
        const auto packed = [&](auto pack) {
            if (act == ACT_SILU) f(zero, pack, std::true_type{});
            else f(zero, pack, std::false_type{});
        };
        if (vw == WIDE) return packed(std::integral_constant<int, WIDE>{});
        if constexpr (sizeof(T) == 2)
            if (vw == 2) return packed(std::integral_constant<int, 2>{});
        packed(std::integral_constant<int, 1>{});
    });
}

std::int64_t columns_floats(const GroupNormShape& s) { return 2 * s.n * s.channels; }

}  // namespace

std::int64_t group_norm_workspace(const GroupNormShape& s, int type, bool backward) {
    if (s.n == 0) return 0;
    const GroupNormPlan plan = group_norm_plan(s, type_bytes(type), backward);
    const std::int64_t columns = columns_floats(s);
    if (plan.held) return backward ? 4 * columns : 0;
    if (backward) return 4 * columns * (1 + plan.runs);
    return 4 * 2 * s.n * plan.runs * s.groups * plan.parts;
}

int launch_group_norm_forward(const GroupNormShape& s, int type, const void* x, void* y, const GroupNormForward& f,
                              hipStream_t stream) {
    const GroupNormPlan plan = group_norm_plan(s, type_bytes(type), false);
    const Block block = block_of(plan);
    const Runs runs{plan.runs, plan.rows};
    const std::int64_t sample = static_cast<std::int64_t>(s.positions) * s.channels;
    const std::int64_t pieces = static_cast<std::int64_t>(plan.runs) * s.groups * plan.parts;  // of a sample, where split
    return for_slices(s, group_norm_slice(s, plan, false), [&](std::int64_t first, const GroupNormShape& part) -> int {
        const unsigned groups = static_cast<unsigned>(part.n * plan.grid());
        GroupNormForward own = f;
        own.mean += first * s.groups;
        own.inv_std += first * s.groups;
        float* means = plan.held ? nullptr : static_cast<float*>(f.workspace) + first * pieces;
        float* squares = plan.held ? nullptr : means + s.n * pieces;
        with_kernel(type, plan.vw, f.act, [&](auto zero, auto pack, auto silu) {
            using T = decltype(zero);
            constexpr int VW = decltype(pack)::value;
            constexpr int HOLD = group_norm_hold(sizeof(T), VW, false, 256), HOLD_MANY = group_norm_hold(sizeof(T), VW, false, 1024);
            constexpr bool SILU = decltype(silu)::value;
            const T* in = static_cast<const T*>(x) + first * sample;
            T* out = static_cast<T*>(y) + first * sample;
            if (plan.held && plan.threads == 256)
                launch(held_forward_kernel<T, VW, SILU, 256, HOLD>, groups, 256, 0, stream, in, out, part, block, own);
            else if (plan.held)
                launch(held_forward_kernel<T, VW, SILU, 1024, HOLD_MANY>, groups, 1024, 0, stream, in, out, part, block, own);
            else
                launch(run_stats_kernel<T, VW>, groups, SPLIT_THREADS, 0, stream, in, part, block, runs, means, squares);
        });
        MFH_TRY(MFH_CHECK_LAUNCH("group_norm_forward", stream));
        if (plan.held) return OK;
        launch(join_stats_kernel, static_cast<unsigned>(part.n * s.groups), SPLIT_THREADS, 0, stream, means, squares, part,
               block, runs, own);
        MFH_TRY(MFH_CHECK_LAUNCH("group_norm_join", stream));
        with_kernel(type, plan.vw, f.act, [&](auto zero, auto pack, auto silu) {
            using T = decltype(zero);
            launch(apply_forward_kernel<T, decltype(pack)::value, decltype(silu)::value>, groups, SPLIT_THREADS, 0, stream,
                   static_cast<const T*>(x) + first * sample, static_cast<T*>(y) + first * sample, part, block, runs, own);
        });
        return MFH_CHECK_LAUNCH("group_norm_apply", stream);
    });
}

int launch_group_norm_backward(const GroupNormShape& s, int type, const void* x, const void* dy, void* dx,
                               const GroupNormBackward& b, hipStream_t stream) {
    const bool parameters = b.gamma_grad || b.beta_grad;
    float* every = static_cast<float*>(b.workspace);
    if (s.n > 0) {
        const GroupNormPlan plan = group_norm_plan(s, type_bytes(type), true);
        const Block block = block_of(plan);
        const Runs runs{plan.runs, plan.rows};
        const std::int64_t sample = static_cast<std::int64_t>(s.positions) * s.channels;
        MFH_TRY(for_slices(s, group_norm_slice(s, plan, true), [&](std::int64_t first, const GroupNormShape& part) -> int {
            const unsigned groups = static_cast<unsigned>(part.n * plan.grid());
            GroupNormBackward own = b;
            own.mean += first * s.groups;
            own.inv_std += first * s.groups;
            float* columns = every + 2 * first * s.channels;
            float* run_columns = every + columns_floats(s) + 2 * first * plan.runs * s.channels;
            with_kernel(type, plan.vw, b.act, [&](auto zero, auto pack, auto silu) {
                using T = decltype(zero);
                constexpr int VW = decltype(pack)::value;
                constexpr int HOLD = group_norm_hold(sizeof(T), VW, true, 256), HOLD_MANY = group_norm_hold(sizeof(T), VW, true, 1024);
                constexpr bool SILU = decltype(silu)::value;
                const T *in = static_cast<const T*>(x) + first * sample, *grad = static_cast<const T*>(dy) + first * sample;
                T* out = dx ? static_cast<T*>(dx) + first * sample : nullptr;
                if (plan.held && plan.threads == 256)
                    launch(held_backward_kernel<T, VW, SILU, 256, HOLD>, groups, 256, 0, stream, in, grad, out, part, block, own,
                           parameters ? columns : nullptr);
                else if (plan.held)
                    launch(held_backward_kernel<T, VW, SILU, 1024, HOLD_MANY>, groups, 1024, 0, stream, in, grad, out, part,
                           block, own, parameters ? columns : nullptr);
                else
                    launch(run_gradients_kernel<T, VW, SILU>, groups, SPLIT_THREADS, 0, stream, in, grad, part, block, runs,
                           own, run_columns);
            });
            MFH_TRY(MFH_CHECK_LAUNCH("group_norm_backward", stream));
            if (plan.held) return OK;
            const int tiles = static_cast<int>(blocks_for(2LL * s.channels, COLUMN_SPAN));
            launch(join_columns_kernel, static_cast<unsigned>(part.n * tiles), COLUMN_SPAN * COLUMN_RUNS, 0, stream, run_columns,
                   plan.runs, 2 * s.channels, tiles, columns);
            MFH_TRY(MFH_CHECK_LAUNCH("group_norm_join_columns", stream));
            if (!dx) return OK;
            with_kernel(type, plan.vw, b.act, [&](auto zero, auto pack, auto silu) {
                using T = decltype(zero);
                launch(apply_backward_kernel<T, decltype(pack)::value, decltype(silu)::value>, groups, SPLIT_THREADS, 0, stream,
                       static_cast<const T*>(x) + first * sample, static_cast<const T*>(dy) + first * sample,
                       static_cast<T*>(dx) + first * sample, part, block, runs, own, columns);
            });
            return MFH_CHECK_LAUNCH("group_norm_apply_backward", stream);
        }));
    }
    if (!parameters) return OK;
    launch(parameter_grads_kernel, blocks_for(2LL * s.channels, COLUMN_SPAN), COLUMN_SPAN * COLUMN_RUNS, 0, stream, every, s, b);
    return MFH_CHECK_LAUNCH("group_norm_parameter_grads", stream);
}

}  // namespace mfh
