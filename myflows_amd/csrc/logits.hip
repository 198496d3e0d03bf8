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
#include "wave.h"

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

// ---- the pass over a row --------------------------------------------------------------------
// A workgroup takes a run of a row's logits tile by tile, in 16-byte packs: each thread keeps the running
// statistics of its own logits, and the threads' are joined once, at the end of the run. One read of the
// logits, one exp a logit. Bound by HBM for float32; a bfloat16 or float16 logit costs about as many vector
// instructions as the time that its two bytes take allows.
//
// The top alternatives come out of the same read. The k-th largest of the threads' own maxima is at most the
// row's k-th largest logit, so only logits above that threshold can be alternatives: about k of a tile's
// thousands. They are kept in LDS (a list of CANDIDATES), the threshold is raised as the maxima grow, and at
// the end each candidate's rank is counted. A list that overflows (all logits equal, or rising logits) is made
// again by exact_top, which needs no threshold.
constexpr int TILE_PACKS = 4;
constexpr int CANDIDATES = 1024;

struct RowRun {
    long long row;
    int chunk, begin, end;
};

// Where a run's results go when a row is split: statistics and k keys a run, joined by a second launch.
struct RowPartials {
    RowStats* stats;
    unsigned long long* keys;
};

template <int THREADS>
struct TopState {
    unsigned long long candidates[CANDIDATES];
    unsigned long long best[2][TOP_MAX];
    unsigned long long wave_best[THREADS / 64];
    float maxima[2][THREADS];
    int count;
};

template <typename T, int THREADS>
struct RowTile {
    static constexpr int N = 16 / sizeof(T), SIZE = THREADS * TILE_PACKS * N;
    Pack<T, N> packs[TILE_PACKS];

    // Index of element e of pack p of this thread in a tile that starts at base.
    static __device__ __forceinline__ int index(int base, int p, int e) {
        return base + (p * THREADS + static_cast<int>(threadIdx.x)) * N + e;
    }
    __device__ __forceinline__ void load(const T* __restrict__ z, int base) {
#pragma unroll
        for (int p = 0; p < TILE_PACKS; ++p) packs[p] = load_pack<T, N>(z + index(base, p, 0));
    }
    // A tile that the run's end cuts: -inf past the end.
    __device__ __forceinline__ void load_cut(const T* __restrict__ z, int base, int end) {
#pragma unroll
        for (int p = 0; p < TILE_PACKS; ++p) {
            const int at = index(base, p, 0);
            if (at + N <= end) {
                packs[p] = load_pack<T, N>(z + at);
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) packs[p].v[e] = at + e < end ? z[at + e] : static_cast<T>(-INFINITY);
            }
        }
    }
};

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

template <int COUNT>
__device__ __forceinline__ float largest(const float (&x)[COUNT]) {
    float m[2] = {x[0], x[1]};
#pragma unroll
    for (int i = 2; i + 3 < COUNT; i += 4) {
        m[0] = max3(m[0], x[i], x[i + 1]);
        m[1] = max3(m[1], x[i + 2], x[i + 3]);
    }
    static_assert(COUNT % 4 == 0, "pairs of pairs");
    return max3(fmaxf(m[0], m[1]), x[COUNT - 2], x[COUNT - 1]);
}

// A float that at least k of the threads' maxima reach (the k-th largest of them, its low 16 bits cleared
// downwards), -inf where fewer than k lie above that. The same in every thread.
template <int THREADS>
__device__ __forceinline__ float kth_of_maxima(float (&maxima)[THREADS], float mine, int k) {
    constexpr int EACH = THREADS / 64;
    maxima[threadIdx.x] = mine;
    __syncthreads();
    unsigned order[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const unsigned bits = __float_as_uint(maxima[(threadIdx.x & 63) * EACH + i] + 0.0f);
        order[i] = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
    }
    unsigned found = 0;
    for (int bit = 31; bit >= 16; --bit) {
        const unsigned probe = found | (1u << bit);
        int reached = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) reached += __popcll(__ballot(order[i] >= probe));
        if (reached >= k) found = probe;
        if (reached == k) break;
    }
    if (found <= 0x007fffffu) return -INFINITY;  // -inf itself, or nothing
    return __uint_as_float(found & 0x80000000u ? found & 0x7fffffffu : ~found);
}

// The next float below (of a float above -inf).
__device__ __forceinline__ float just_below(float v) {
    const unsigned bits = __float_as_uint(v);
    return __uint_as_float(v > 0.0f ? bits - 1 : v == 0.0f ? 0x80000001u : bits + 1);
}

// The k largest keys of a run in falling order, in best (0 where there are fewer), by k rounds a tile of the
// largest key below the last, for the tiles that hold a key above the k-th best so far.
template <typename T, int THREADS>
__device__ __forceinline__ unsigned long long* exact_top(TopState<THREADS>& top, const T* __restrict__ z,
                                                         const RowRun& run, int k) {
    using Tile = RowTile<T, THREADS>;
    int side = 0;
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < k) top.best[0][threadIdx.x] = 0;
    __syncthreads();
    for (int base = run.begin; base < run.end; base += Tile::SIZE) {
        Tile tile;
        tile.load_cut(z, base, run.end);
        const auto key_at = [&](int p, int e) -> unsigned long long {
            const float x = tile.packs[p].at(e);
            const int at = Tile::index(base, p, e);
            return x == x && at < run.end ? key_of(x, at) : 0;
        };
        const unsigned long long least = top.best[side][k - 1];
        bool above = false;
        for (int p = 0; p < TILE_PACKS; ++p)
            for (int e = 0; e < Tile::N; ++e) above = above || key_at(p, e) > least;
        if (!__syncthreads_or(above)) continue;
        unsigned long long last = ~0ull;
        for (int i = 0; i < k && last; ++i) {
            unsigned long long mine = 0;
            for (int p = 0; p < TILE_PACKS; ++p)
                for (int e = 0; e < Tile::N; ++e) {
                    const unsigned long long key = key_at(p, e);
                    if (key < last && key > mine) mine = key;
                }
            if (static_cast<int>(threadIdx.x) < k) {
                const unsigned long long key = top.best[side][threadIdx.x];
                if (key < last && key > mine) mine = key;
            }
            for (int o = 32; o > 0; o /= 2) {
                const unsigned long long other = __shfl_xor(mine, o);
                if (other > mine) mine = other;
            }
            if constexpr (THREADS > 64) {
                __syncthreads();
                if ((threadIdx.x & 63) == 0) top.wave_best[threadIdx.x / 64] = mine;
                __syncthreads();
                for (int w = 0; w < THREADS / 64; ++w)
                    if (top.wave_best[w] > mine) mine = top.wave_best[w];
            }
            last = mine;
            if (threadIdx.x == 0) top.best[side ^ 1][i] = last;
            if (last == 0 && static_cast<int>(threadIdx.x) > i && static_cast<int>(threadIdx.x) < k)
                top.best[side ^ 1][threadIdx.x] = 0;
        }
        side ^= 1;
        __syncthreads();
    }
    return top.best[side];
}

// Takes every candidate to its rank: emit(rank, key) for the k largest, emit(rank, 0) for those that are missing.
// Fewer than k candidates mean that all logits above -inf are candidates: the first -inf of the run follow.
template <typename T, int THREADS, typename Emit>
__device__ __forceinline__ void emit_top(TopState<THREADS>& top, const T* __restrict__ z, const RowRun& run, int k,
                                         float s, Emit&& emit) {
    __syncthreads();
    const int count = top.count;
    if (count > CANDIDATES || s != s) {  // a NaN among a thread's logits leaves its maximum open
        const unsigned long long* best = exact_top(top, z, run, k);
        if (static_cast<int>(threadIdx.x) < k) emit(static_cast<int>(threadIdx.x), best[threadIdx.x]);
        return;
    }
    for (int i = threadIdx.x; i < count; i += THREADS) {
        const unsigned long long key = top.candidates[i];
        int rank = 0;
        for (int j = 0; j < count; ++j) rank += top.candidates[j] > key;
        if (rank < k) emit(rank, key);
    }
    if (count >= k || threadIdx.x >= 64) return;
    int next = count;
    for (int base = run.begin; base < run.end && next < k; base += 64) {
        const int at = base + static_cast<int>(threadIdx.x);
        const bool ruled = at < run.end && static_cast<float>(z[at]) == -INFINITY;
        const unsigned long long who = __ballot(ruled);
        const int rank = next + __popcll(who & ((1ull << threadIdx.x) - 1));
        if (ruled && rank < k) emit(rank, key_of(-INFINITY, at));
        next += __popcll(who);
    }
    for (int rank = next + static_cast<int>(threadIdx.x); rank < k; rank += 64) emit(rank, 0);
}

// One tile into the thread's statistics and, with TOP, the list of candidates: those above `below`.
template <bool ENTROPY, bool TOP, typename T, int THREADS>
__device__ __forceinline__ void take_tile(const RowTile<T, THREADS>& tile, RowStats& mine, float scale, int base, int end,
                                          TopState<THREADS>* top, int top_k, float& below, int number) {
    using Tile = RowTile<T, THREADS>;
    constexpr int COUNT = TILE_PACKS * Tile::N;
    float x[COUNT];
#pragma unroll
    for (int p = 0; p < TILE_PACKS; ++p)
#pragma unroll
        for (int e = 0; e < Tile::N; ++e) x[p * Tile::N + e] = tile.packs[p].at(e);
    const float tile_max = largest(x);
    const float to = fmaxf(mine.m, tile_max);
    if constexpr (TOP) {
        // The threshold after the first tile, then raised at the tiles 1, 4, 16, ...: each time the candidates
        // to come are at most those of the tiles so far, three times over.
        const bool first = number == 0;
        if (first) {
            const float kth = kth_of_maxima(top->maxima[0], tile_max, top_k);
            below = kth == -INFINITY ? kth : just_below(kth);
        }
        if (tile_max > below) {
#pragma unroll
            for (int i = 0; i < COUNT; ++i)
                if (x[i] > below) {
                    const int slot = atomicAdd(&top->count, 1);
                    if (slot < CANDIDATES)
                        top->candidates[slot] = key_of(x[i], Tile::index(base, i / Tile::N, i % Tile::N));
                }
        }
        if (!first && (number & (number - 1)) == 0 && (__ffs(number) & 1)) {
            const float kth = kth_of_maxima(top->maxima[(__ffs(number) >> 1) + 1 & 1], to > LOWEST ? to : -INFINITY, top_k);
            below = fmaxf(below, kth);
        }
    }
    mine.rescale(to, scale);
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
        const float d = x[i] - mine.m;
        const float e = exp2_of(d * scale);
        mine.s += e;
        if constexpr (ENTROPY) mine.t += e * fmaxf(d, DIFFERENCE_FLOOR);
    }
}

// The statistics of a run, the same in every thread.
template <bool ENTROPY, bool TOP, typename T, int THREADS>
__device__ __forceinline__ RowStats take_run(const T* __restrict__ z, const RowRun& run, float scale, TopState<THREADS>* top,
                                             int top_k) {
    using Tile = RowTile<T, THREADS>;
    __shared__ RowStats waves[THREADS / 64];
    __shared__ float wave_m[THREADS / 64];
    if constexpr (TOP) {
        if (threadIdx.x == 0) top->count = 0;  // before the barrier of the first threshold
    }
    RowStats mine = RowStats::none();
    float below = -INFINITY;
    int base = run.begin, number = 0;
    for (; base + Tile::SIZE <= run.end; base += Tile::SIZE, ++number) {
        Tile tile;
        tile.load(z, base);
        take_tile<ENTROPY, TOP>(tile, mine, scale, base, run.end, top, top_k, below, number);
    }
    if (base < run.end) {
        Tile tile;
        tile.load_cut(z, base, run.end);
        take_tile<ENTROPY, TOP>(tile, mine, scale, base, run.end, top, top_k, below, number);
    }
    float m = wave_max(mine.m);
    if constexpr (THREADS > 64) {
        if ((threadIdx.x & 63) == 0) wave_m[threadIdx.x / 64] = m;
        __syncthreads();
        m = wave_m[0];
#pragma unroll
        for (int w = 1; w < THREADS / 64; ++w) m = fmaxf(m, wave_m[w]);
    }
    mine.rescale(m, scale);
    mine.s = wave_sum(mine.s);
    if constexpr (ENTROPY) mine.t = wave_sum(mine.t);
    if constexpr (THREADS > 64) {
        if ((threadIdx.x & 63) == 0) waves[threadIdx.x / 64] = mine;
        __syncthreads();
        mine = waves[0];
#pragma unroll
        for (int w = 1; w < THREADS / 64; ++w) {
            mine.s += waves[w].s;
            mine.t += waves[w].t;
        }
    }
    return mine;
}

struct RowSplit {
    int chunks, length;  // runs of a row and logits of a run
};

__device__ __forceinline__ RowRun run_of(const RowSplit& split, int vocab) {
    const unsigned row = blockIdx.x / static_cast<unsigned>(split.chunks);
    const int chunk = static_cast<int>(blockIdx.x - row * split.chunks);
    return {row, chunk, chunk * split.length, min(vocab, (chunk + 1) * split.length)};
}

template <typename T, int THREADS, bool TOP>
__global__ __launch_bounds__(THREADS) void log_probs_kernel(const T* __restrict__ logits, LogProbsForward f, RowSplit split,
                                                            RowPartials partials) {
    __shared__ TopState<TOP ? THREADS : 64> top;
    const RowRun run = run_of(split, f.vocab);
    const T* __restrict__ z = logits + run.row * f.stride;
    if constexpr (TOP) {
        const RowStats row = take_run<true, true, T, THREADS>(z, run, LOG2E, &top, f.top);
        if (split.chunks == 1) {
            if (threadIdx.x == 0) finish_log_probs(f, z, run.row, row);
            emit_top(top, z, run, f.top, row.s, [&](int rank, unsigned long long key) { write_top(f, run.row, rank, key, row); });
        } else {
            const long long at = run.row * split.chunks + run.chunk;
            if (threadIdx.x == 0) partials.stats[at] = row;
            emit_top(top, z, run, f.top, row.s,
                     [&](int rank, unsigned long long key) { partials.keys[at * f.top + rank] = key; });
        }
    } else {
        const RowStats row = take_run<true, false, T, THREADS>(z, run, LOG2E, nullptr, 0);
        if (threadIdx.x != 0) return;
        if (split.chunks == 1) finish_log_probs(f, z, run.row, row);
        else partials.stats[run.row * split.chunks + run.chunk] = row;
    }
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void distill_kernel(const T* __restrict__ logits, DistillForward f, RowSplit split,
                                                          RowPartials partials) {
    const RowRun run = run_of(split, f.vocab);
    const T* __restrict__ z = logits + run.row * f.stride;
    const RowStats row = take_run<false, false, T, THREADS>(z, run, LOG2E / f.temperature, nullptr, 0);
    if (split.chunks == 1) finish_distill(f, z, run.row, row);
    else if (threadIdx.x == 0) partials.stats[run.row * split.chunks + run.chunk] = row;
}

// The runs of a row (at most 64) joined by one wave, the same in every lane.
__device__ __forceinline__ RowStats join_runs(const RowStats* __restrict__ stats, int chunks, float scale) {
    const int lane = threadIdx.x & 63;
    RowStats mine = lane < chunks ? stats[lane] : RowStats::none();
    mine.rescale(wave_max(mine.m), scale);
    mine.s = wave_sum(mine.s);
    mine.t = wave_sum(mine.t);
    return mine;
}

constexpr int JOIN_THREADS = 256;
constexpr int SPLIT_MAX = 64;

// The largest 64-bit key that k of the threads' keys reach (0 when fewer than k are above 0).
__device__ __forceinline__ unsigned long long kth_of_keys(unsigned long long (&maxima)[JOIN_THREADS],
                                                          unsigned long long mine, int k) {
    constexpr int EACH = JOIN_THREADS / 64;
    maxima[threadIdx.x] = mine;
    __syncthreads();
    unsigned long long key[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) key[i] = maxima[(threadIdx.x & 63) * EACH + i];
    unsigned long long found = 0;
    for (int bit = 63; bit >= 0; --bit) {
        const unsigned long long probe = found | (1ull << bit);
        int reached = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) reached += __popcll(__ballot(key[i] >= probe));
        if (reached >= k) found = probe;
        if (reached == k) break;
    }
    return found;
}

// Joins a row's runs: one workgroup a row.
template <typename T>
__global__ __launch_bounds__(JOIN_THREADS) void log_probs_join_kernel(const T* __restrict__ logits, LogProbsForward f,
                                                                      RowSplit split, RowPartials partials) {
    __shared__ unsigned long long maxima[JOIN_THREADS], kept[SPLIT_MAX * TOP_MAX];
    __shared__ int count;
    const long long r = blockIdx.x;
    const RowStats row = join_runs(partials.stats + r * split.chunks, split.chunks, LOG2E);
    if (threadIdx.x == 0) {
        finish_log_probs(f, logits + r * f.stride, r, row);
        count = 0;
    }
    if (f.top == 0) return;
    const unsigned long long* __restrict__ keys = partials.keys + r * split.chunks * f.top;
    const int total = split.chunks * f.top;
    unsigned long long mine = 0;
    for (int i = threadIdx.x; i < total; i += JOIN_THREADS) mine = max(mine, keys[i]);
    const unsigned long long least = max(kth_of_keys(maxima, mine, f.top), 1ull);
    for (int i = threadIdx.x; i < total; i += JOIN_THREADS)
        if (keys[i] >= least) kept[atomicAdd(&count, 1)] = keys[i];
    __syncthreads();
    for (int i = threadIdx.x; i < count; i += JOIN_THREADS) {
        int rank = 0;
        for (int j = 0; j < count; ++j) rank += kept[j] > kept[i];
        if (rank < f.top) write_top(f, r, rank, kept[i], row);
    }
    for (int k = count + threadIdx.x; k < f.top; k += JOIN_THREADS) write_top(f, r, k, 0, row);
}

template <typename T>
__global__ __launch_bounds__(64) void distill_join_kernel(const T* __restrict__ logits, DistillForward f, RowSplit split,
                                                          RowPartials partials) {
    const long long r = blockIdx.x;
    finish_distill(f, logits + r * f.stride, r,
                   join_runs(partials.stats + r * split.chunks, split.chunks, LOG2E / f.temperature));
}

// ---- the gradients --------------------------------------------------------------------------
// A workgroup forms GRAD_PACKS packs a thread of one row's gradient: every logit is read once and every
// gradient written once, p formed again from the row's m and s. Bound by HBM.
constexpr int GRAD_THREADS = 256, GRAD_PACKS = 4;

template <typename T>
struct GradSpan {
    static constexpr int N = 16 / sizeof(T), SIZE = GRAD_THREADS * GRAD_PACKS * N;
};

// Reads the packs of a span, forms value(logit, index) and writes it (added to what is there with ADD).
// Before the first write of the workgroup `between` runs.
template <bool ADD, typename T, typename Value, typename Between>
__device__ __forceinline__ void form_span(const T* z, T* out, int first, int vocab, Value&& value, Between&& between) {
    constexpr int N = GradSpan<T>::N;
    const int base = first + static_cast<int>(threadIdx.x) * N;
    Pack<T, N> in[GRAD_PACKS], old[ADD ? GRAD_PACKS : 1];
#pragma unroll
    for (int p = 0; p < GRAD_PACKS; ++p) {
        const int at = base + p * GRAD_THREADS * N;
        if (at + N <= vocab) {
            in[p] = load_pack<T, N>(z + at);
            if constexpr (ADD) old[p] = load_pack<T, N>(out + at);
        }
    }
    between();
#pragma unroll
    for (int p = 0; p < GRAD_PACKS; ++p) {
        const int at = base + p * GRAD_THREADS * N;
        if (at + N <= vocab) {
            Pack<T, N> result;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float v = value(in[p].at(e), at + e);
                if constexpr (ADD) result.set(e, old[p].at(e) + v);
                else result.set(e, v);
            }
            store_pack(out + at, result);
        } else {
            for (int j = at; j < vocab; ++j) {
                const float v = value(static_cast<float>(z[j]), j);
                out[j] = static_cast<T>(ADD ? static_cast<float>(out[j]) + v : v);
            }
        }
    }
}

template <typename T, bool ADD>
__global__ __launch_bounds__(GRAD_THREADS) void log_probs_backward_kernel(const T* logits, T* grad, LogProbsBackward b,
                                                                          int spans) {
    const unsigned row = blockIdx.x / static_cast<unsigned>(spans);
    const long long r = row;
    const int first = static_cast<int>(blockIdx.x - row * spans) * GradSpan<T>::SIZE;
    const T* z = logits + r * b.stride;
    T* out = grad + r * b.grad_stride;
    const float m = b.stats[r], s = b.stats[b.rows + r], inv = s == 0.0f ? 0.0f : 1.0f / s;
    const long long t = b.log_prob_grad ? whole_at(b.tokens, b.tokens_wide, r) : -1;
    const float factor = b.factor ? b.factor[0] : 1.0f;
    float g = t < 0 || s == 0.0f ? 0.0f : b.scale * factor * b.log_prob_grad[r * b.log_prob_step];
    if (t >= b.vocab) g = NOT_A_NUMBER;
    const float h = b.entropy_grad && s != 0.0f ? factor * b.entropy_grad[r * b.entropy_step] : 0.0f;
    if (g == 0.0f && h == 0.0f) {
        form_span<ADD>(z, out, first, b.vocab, [](float, int) { return 0.0f; }, [] {});
    } else if (h == 0.0f) {
        const int token = static_cast<int>(t);
        const float scale = -g * inv;
        form_span<ADD>(z, out, first, b.vocab, [=](float x, int j) {
            const float v = exp2_of((x - m) * LOG2E) * scale;
            return j == token ? v + g : v;
        }, [] {});
    } else {
        const int token = static_cast<int>(t);
        // g + h (ln p + entropy) = h d + k,  d = z - m
        const float k = g + h * (b.entropy[r] - logf(s));
        form_span<ADD>(z, out, first, b.vocab, [=](float x, int j) {
            const float d = x - m;
            const float v = -(exp2_of(d * LOG2E) * inv) * (h * fmaxf(d, DIFFERENCE_FLOOR) + k);
            return j == token ? v + g : v;
        }, [] {});
    }
}

// The targets lie at a few of a row's ids: the workgroup writes coef q everywhere and then, at the ids of its
// span, coef (q - target) over it. Those logits (and, with ADD, what the gradient held) are read before the
// first write, so the gradient may take the logits' place.
template <typename T, bool ADD>
__global__ __launch_bounds__(GRAD_THREADS) void distill_backward_kernel(const T* logits, T* grad, DistillBackward b,
                                                                        int spans) {
    static_assert(DISTILL_HELD_MAX <= GRAD_THREADS, "an id a thread");
    const unsigned row = blockIdx.x / static_cast<unsigned>(spans);
    const long long r = row;
    const int first = static_cast<int>(blockIdx.x - row * spans) * GradSpan<T>::SIZE;
    const T* z = logits + r * b.stride;
    T* out = grad + r * b.grad_stride;
    const float w = b.weights[r];
    if (w == 0.0f) {
        form_span<ADD>(z, out, first, b.vocab, [](float, int) { return 0.0f; }, [] {});
        return;
    }
    const float m = b.stats[r], s = b.stats[b.rows + r], inv = s == 0.0f ? 0.0f : 1.0f / s;
    const float scale = LOG2E / b.temperature;
    const float coef = b.seed[0] * w * b.loss[1] * b.temperature;
    const auto share = [=](float x) { return exp2_of((x - m) * scale) * inv; };
    long long id = -1;
    float target = 0.0f, at_id = 0.0f, held = 0.0f;
    if (static_cast<int>(threadIdx.x) < b.held) {
        id = whole_at(b.ids, b.ids_wide, r * b.held + threadIdx.x);
        if (id >= first && id < b.vocab && id < first + GradSpan<T>::SIZE) {
            target = b.targets[r * b.held + threadIdx.x];
            at_id = static_cast<float>(z[id]);
            if constexpr (ADD) held = static_cast<float>(out[id]);
        } else {
            id = -1;
        }
    }
    form_span<ADD>(z, out, first, b.vocab, [=](float x, int) { return share(x) * coef; }, [] { __syncthreads(); });
    __syncthreads();
    if (id >= 0) out[id] = static_cast<T>(held + coef * (share(at_id) - target));
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

namespace {

// Threads of a row's workgroup: a wave while a row is at most two tiles of it (no barriers), else four.
constexpr int SMALL_ROW_BYTES = 2 * 64 * TILE_PACKS * 16, WAVE_THREADS = 64;

bool small_row(int vocab, int type) { return vocab * static_cast<std::int64_t>(type_bytes(type)) <= SMALL_ROW_BYTES; }

// Runs of a row: as many as bring the workgroups to SPLIT_GROUPS (eight a CU of the 256), of at least one tile.
// The number is fixed by the sizes, not by the device, so that results do not depend on it.
constexpr int SPLIT_GROUPS = 2048;
RowSplit row_split(std::int64_t rows, int vocab, int type) {
    if (rows == 0 || small_row(vocab, type)) return {1, vocab};
    const int unit = ROW_THREADS * 16 / type_bytes(type);  // a pack a thread
    const std::int64_t wanted = std::min<std::int64_t>(SPLIT_MAX, std::max<std::int64_t>(1, SPLIT_GROUPS / rows));
    const std::int64_t packs = (vocab + unit - 1) / unit;
    const int length = static_cast<int>(std::max<std::int64_t>(TILE_PACKS, (packs + wanted - 1) / wanted)) * unit;
    return {static_cast<int>((vocab + length - 1) / length), length};
}

RowPartials partials_in(void* workspace, std::int64_t runs, std::int64_t top) {
    auto* keys = static_cast<unsigned long long*>(workspace);
    return {reinterpret_cast<RowStats*>(keys + runs * top), keys};
}

std::int64_t partial_bytes(std::int64_t rows, const RowSplit& split, std::int64_t top) {
    if (split.chunks == 1) return 0;
    return rows * split.chunks * static_cast<std::int64_t>(sizeof(RowStats) + 8 * top);
}

}  // namespace

std::int64_t log_probs_workspace(std::int64_t rows, int vocab, int type, int top) {
    return partial_bytes(rows, row_split(rows, vocab, type), top);
}
std::int64_t distill_workspace(std::int64_t rows, int vocab, int type) {
    return partial_bytes(rows, row_split(rows, vocab, type), 0);
}

int launch_log_probs(const void* logits, int type, const LogProbsForward& f, hipStream_t stream) {
    if (f.rows == 0) return OK;
    const RowSplit split = row_split(f.rows, f.vocab, type);
    const RowPartials partials = partials_in(f.workspace, f.rows * split.chunks, f.top);
    const unsigned groups = static_cast<unsigned>(f.rows * split.chunks);
    with_type(type, [&](auto zero) {
        using T = decltype(zero);
        const T* z = static_cast<const T*>(logits);
        const auto run = [&](auto kernel, int threads) { launch(kernel, groups, threads, 0, stream, z, f, split, partials); };
        const bool small = small_row(f.vocab, type);
        if (f.top && small) run(log_probs_kernel<T, WAVE_THREADS, true>, WAVE_THREADS);
        else if (f.top) run(log_probs_kernel<T, ROW_THREADS, true>, ROW_THREADS);
        else if (small) run(log_probs_kernel<T, WAVE_THREADS, false>, WAVE_THREADS);
        else run(log_probs_kernel<T, ROW_THREADS, false>, ROW_THREADS);
    });
    MFH_TRY(MFH_CHECK_LAUNCH("log_probs", stream));
    if (split.chunks == 1) return OK;
    with_type(type, [&](auto zero) {
        using T = decltype(zero);
        launch(log_probs_join_kernel<T>, static_cast<unsigned>(f.rows), f.top ? JOIN_THREADS : 64, 0, stream,
               static_cast<const T*>(logits), f, split, partials);
    });
    return MFH_CHECK_LAUNCH("log_probs_join", stream);
}

int launch_log_probs_backward(const void* logits, void* grad, int type, const LogProbsBackward& b, hipStream_t stream) {
    if (b.rows == 0) return OK;
    with_type(type, [&](auto zero) {
        using T = decltype(zero);
        const int spans = static_cast<int>(blocks_for(b.vocab, GradSpan<T>::SIZE));
        const auto run = [&](auto kernel) {
            launch(kernel, static_cast<unsigned>(b.rows * spans), GRAD_THREADS, 0, stream, static_cast<const T*>(logits),
                   static_cast<T*>(grad), b, spans);
        };
        if (b.add) run(log_probs_backward_kernel<T, true>);
        else run(log_probs_backward_kernel<T, false>);
    });
    return MFH_CHECK_LAUNCH("log_probs_backward", stream);
}

int launch_distill(const void* logits, int type, const DistillForward& f, hipStream_t stream) {
    if (f.rows != 0) {
        const RowSplit split = row_split(f.rows, f.vocab, type);
        const RowPartials partials = partials_in(f.workspace, f.rows * split.chunks, 0);
        const unsigned groups = static_cast<unsigned>(f.rows * split.chunks);
        with_type(type, [&](auto zero) {
            using T = decltype(zero);
            const T* z = static_cast<const T*>(logits);
            if (small_row(f.vocab, type))
                launch(distill_kernel<T, WAVE_THREADS>, groups, WAVE_THREADS, 0, stream, z, f, split, partials);
            else
                launch(distill_kernel<T, ROW_THREADS>, groups, ROW_THREADS, 0, stream, z, f, split, partials);
        });
        MFH_TRY(MFH_CHECK_LAUNCH("distill", stream));
        if (split.chunks > 1) {
            with_type(type, [&](auto zero) {
                using T = decltype(zero);
                launch(distill_join_kernel<T>, static_cast<unsigned>(f.rows), 64, 0, stream, static_cast<const T*>(logits),
                       f, split, partials);
            });
            MFH_TRY(MFH_CHECK_LAUNCH("distill_join", stream));
        }
    }
    return launch_row_mean(f.row_loss, f.weights, nullptr, 0, f.rows, 1.0f, f.loss, stream);
}

int launch_distill_backward(const void* logits, void* grad, int type, const DistillBackward& b, hipStream_t stream) {
    if (b.rows == 0) return OK;
    with_type(type, [&](auto zero) {
        using T = decltype(zero);
        const int spans = static_cast<int>(blocks_for(b.vocab, GradSpan<T>::SIZE));
        const auto run = [&](auto kernel) {
            launch(kernel, static_cast<unsigned>(b.rows * spans), GRAD_THREADS, 0, stream, static_cast<const T*>(logits),
                   static_cast<T*>(grad), b, spans);
        };
        if (b.add) run(distill_backward_kernel<T, true>);
        else run(distill_backward_kernel<T, false>);
    });
    return MFH_CHECK_LAUNCH("distill_backward", stream);
}

int launch_row_mean(const float* values, const float* weights, const void* tokens, int tokens_wide, std::int64_t rows,
                    float scale, float* out, hipStream_t stream) {
    launch(row_mean_kernel, 1, MEAN_THREADS, 0, stream, values, weights, tokens, tokens_wide, rows, scale, out);
    return MFH_CHECK_LAUNCH("row_mean", stream);
}

}  // namespace mfh
