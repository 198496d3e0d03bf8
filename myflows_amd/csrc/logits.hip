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
#include <type_traits>

#include "common.h"
#include "hand_over.h"
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

using mfh::hand_over;
__device__ __forceinline__ void hand_over(RowStats* to, const RowStats& value) {
    hand_over(&to->m, value.m);
    hand_over(&to->s, value.s);
    hand_over(&to->t, value.t);
}

// A row's token and its logit, read ahead of the row's end.
struct GivenToken {
    long long token;
    float z;
    GivenToken() = default;
    template <typename T>
    __device__ __forceinline__ GivenToken(const LogProbsForward& f, const T* __restrict__ row, long long r) : token(-1), z(0.0f) {
        if (!f.log_prob) return;
        token = whole_at(f.tokens, f.tokens_wide, r * f.tokens_step);
        if (token >= 0 && token < f.vocab) z = static_cast<float>(row[token]);
    }
};

__device__ __forceinline__ void finish_log_probs(const LogProbsForward& f, long long r, const GivenToken& given,
                                                 const RowStats& row) {
    const RowEnd end(row);
    f.stats[r] = end.m;
    f.stats[f.rows + r] = end.s;
    f.log_sum[r] = end.empty ? -INFINITY : end.m + end.ln_s;
    f.entropy[r] = end.empty ? 0.0f : end.ln_s - row.t / row.s;
    if (f.log_prob) f.log_prob[r] = given.token < 0 ? 0.0f : given.token >= f.vocab ? NOT_A_NUMBER : end.log_prob(given.z);
}

__device__ __forceinline__ void write_top(const LogProbsForward& f, long long r, int k, unsigned long long key,
                                          const RowEnd& end) {
    const long long at = r * f.top + k;
    f.top_ids[at] = key ? key_index(key) : -1;
    f.top_log_probs[at] = key ? end.log_prob(key_value(key)) : NOT_A_NUMBER;
}

// The teacher's record of one row, by all threads of a workgroup: `read` loads it with the logits at its ids and
// forms the teacher's probabilities and the targets, none of which needs the row's statistics; `finish` forms
// the loss. A row that does not count (no id held, weight 0) has loss 0 and weight 0, whatever its logits hold;
// an id beyond the vocabulary makes a counting row's loss and gradient NaN.
template <int THREADS>
struct TeacherRow {
    static constexpr int EACH = DISTILL_HELD_MAX / THREADS;
    static_assert(DISTILL_HELD_MAX % THREADS == 0, "ids are shared evenly");
    float p[EACH], log_p[EACH], z[EACH];  // of the ids of this thread; p is 0 for none
    float weight;
    bool poisoned;

    // The joint result of the threads' values.
    template <typename Op>
    static __device__ __forceinline__ float joint(float v, Op op) {
        v = wave_reduce(v, op);
        if constexpr (THREADS > 64) {
            __shared__ float part[THREADS / 64];
            __syncthreads();
            if ((threadIdx.x & 63) == 0) part[threadIdx.x / 64] = v;
            __syncthreads();
            v = part[0];
#pragma unroll
            for (int w = 1; w < THREADS / 64; ++w) v = op(v, part[w]);
        }
        return v;
    }

    template <typename T>
    __device__ __forceinline__ void read(const DistillForward& f, const T* __restrict__ row, long long r, bool write) {
        __shared__ int ids[DISTILL_HELD_MAX];
        __shared__ float probs[DISTILL_HELD_MAX];
        const int tid = threadIdx.x;
        const float inv_t = 1.0f / f.temperature;
        float u[EACH], most = -INFINITY, bad = 0.0f;
        int id[EACH];
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int k = tid + i * THREADS;
            u[i] = -INFINITY;
            z[i] = 0.0f;
            id[i] = -1;
            if (k >= f.held) continue;
            const long long given = whole_at(f.ids, f.ids_wide, r * f.ids_step + k);
            if (given < 0) continue;
            u[i] = f.teacher[r * f.teacher_step + k] * inv_t;
            if (given >= f.vocab) {
                bad = 1.0f;
                continue;
            }
            id[i] = static_cast<int>(given);
            z[i] = static_cast<float>(row[given]);
        }
        const auto larger = [](float a, float b) { return b > a || b != b ? b : a; };  // a NaN wins
#pragma unroll
        for (int i = 0; i < EACH; ++i) most = larger(most, u[i]);
        most = joint(most, larger);
        bad = joint(bad, [](float a, float b) { return fmaxf(a, b); });
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            // Teacher logits of -inf alone leave no target (and -inf - -inf would not be a number).
            p[i] = most == -INFINITY ? 0.0f : exp2_of((u[i] - most) * LOG2E);
            sum += p[i];
        }
        sum = joint(sum, [](float a, float b) { return a + b; });
        weight = sum == 0.0f ? 0.0f : f.row_weights ? f.row_weights[r * f.weights_step] : 1.0f;
        poisoned = weight != 0.0f && bad != 0.0f;
        const float ln_sum = logf(sum);
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int k = tid + i * THREADS;
            p[i] = weight == 0.0f ? 0.0f : p[i] / sum;
            log_p[i] = u[i] - most - ln_sum;
            if (k < f.held) {
                ids[k] = id[i];
                probs[k] = p[i];
            }
        }
        if (!write) return;
        __syncthreads();
        // An id that the record holds twice has the sum of its probabilities as its target.
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int k = tid + i * THREADS;
            if (k >= f.held) break;
            float target = 0.0f;
            for (int other = 0; other < f.held; ++other) target += ids[other] == id[i] ? probs[other] : 0.0f;
            f.targets[r * f.held + k] = target;
        }
    }

    __device__ __forceinline__ void finish(const DistillForward& f, long long r, const RowStats& row) {
        const float inv_t = 1.0f / f.temperature, ln_s = logf(row.s);
        float loss = 0.0f;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const float log_q = row.s == 0.0f ? -INFINITY : (z[i] - row.m) * inv_t - ln_s;
            if (p[i] != 0.0f) loss += p[i] * (log_p[i] - log_q);
        }
        loss = joint(loss, [](float a, float b) { return a + b; });
        if (threadIdx.x != 0) return;
        hand_over(f.row_loss + r, weight == 0.0f ? 0.0f : poisoned ? NOT_A_NUMBER : f.temperature * f.temperature * loss);
        hand_over(f.weights + r, weight);
        f.stats[r] = row.m;
        f.stats[f.rows + r] = poisoned ? NOT_A_NUMBER : row.s;
    }
};

// ---- the pass over a row --------------------------------------------------------------------
// A workgroup takes a run of a row's logits tile by tile, in 16-byte packs, the next tile's loads in flight:
// each thread keeps the running statistics of its own logits, and the threads' are joined once, at the end of
// the run. One read of the logits, one exp a logit. Bound by HBM for float32; a bfloat16 or float16 logit
// costs about as many vector instructions as the time that its two bytes take allows (float16 compared in pairs
// and converted within the subtraction: 2048 x 32768 with 20 alternatives 38.9 us, 41.4 with conversions of its
// own). 2048 x 131072 bfloat16 with 20 alternatives 115 us (4.7 TB/s), 1000 x 50021 float32 without any 34 (5.8),
// 2048 x 32768 bfloat16 27.
//
// The top alternatives come out of the same read. The k-th largest of the threads' own maxima is at most the
// row's k-th largest logit, so only logits above that threshold can be alternatives: about k of a tile's
// thousands. Each wave keeps its own in a list in LDS, the threshold is raised as the maxima grow, and at the
// end each candidate's rank is counted. A list that overflows (all logits equal, or rising logits) is made
// again by exact_top, which needs no threshold.
constexpr int TILE_PACKS = 4;
constexpr int WAVE_CANDIDATES = 512;  // of a wave's list: a wave that holds a short run whole does not overflow

struct RowRun {
    long long row;
    int chunk, begin, end;
};

// Where a run's results go when a row is split: statistics and k keys a run.
struct RowPartials {
    RowStats* stats;
    unsigned long long* keys;
};

template <int WAVES>
struct TopState {
    unsigned long long candidates[WAVES][WAVE_CANDIDATES];
    unsigned long long best[2][TOP_MAX];
    unsigned long long wave_best[WAVES];
    int ranks[WAVES * 64];
    float kth[2][WAVES];
    int counts[WAVES];
};

template <typename T, int THREADS>
struct RowTile {
    static constexpr int N = 16 / sizeof(T), SIZE = THREADS * TILE_PACKS * N;
    Pack<T, N> packs[TILE_PACKS];

    // Index of element e of pack p of this thread in a tile that starts at base.
    static __device__ __forceinline__ int index(int base, int p, int e) {
        return base + (p * THREADS + static_cast<int>(threadIdx.x)) * N + e;
    }
    // The tile at base; -inf past a run's end that cuts it. One pack at most lies across the end.
    __device__ __forceinline__ void load(const T* __restrict__ z, int base, int end) {
        if (base + SIZE <= end) {
#pragma unroll
            for (int p = 0; p < TILE_PACKS; ++p) packs[p] = load_pack<T, N>(z + index(base, p, 0));
            return;
        }
        const Pack<T, N> none = Pack<T, N>::all(-INFINITY);
#pragma unroll
        for (int p = 0; p < TILE_PACKS; ++p) {
            const int at = index(base, p, 0);
            packs[p] = at + N <= end ? load_pack<T, N>(z + at) : none;
        }
        const int whole = end / N * N, across = (whole - base) / N, p = across / THREADS;  // N divides base
        if (across - p * THREADS == static_cast<int>(threadIdx.x) && whole < end) {
            const Pack<T, N> part = load_part<T, N>(z + whole, end - whole, -INFINITY);
#pragma unroll
            for (int i = 0; i < TILE_PACKS; ++i)
                if (i == p) packs[i] = part;
        }
    }
};

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

__device__ __forceinline__ unsigned max_of_pairs(unsigned a, unsigned b) {
    unsigned r;
    asm("v_pk_max_f16 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

// The largest of a pack; a NaN is left out, or makes it one. float16 pairs are compared as they are, two at a time.
template <typename T, int N>
__device__ __forceinline__ float largest(const Pack<T, N>& pack) {
    static_assert(N % 4 == 0, "two chains of pairs");
    if constexpr (std::is_same_v<T, _Float16>) {
        static_assert(N == 8, "four words");
        const unsigned both = max_of_pairs(max_of_pairs(pack.w[0], pack.w[1]), max_of_pairs(pack.w[2], pack.w[3]));
        const Pack<T, 2> pair{both};
        return fmaxf(pair.at(0), pair.at(1));
    }
    float a = fmaxf(pack.at(0), pack.at(1)), b = fmaxf(pack.at(2), pack.at(3));
#pragma unroll
    for (int i = 4; i < N; i += 4) {
        a = max3(a, pack.at(i), pack.at(i + 1));
        b = max3(b, pack.at(i + 2), pack.at(i + 3));
    }
    return fmaxf(a, b);
}

// Element i of a pack minus m, rounded once. The mixed multiply-add converts a float16 operand by itself.
template <typename T, int N>
__device__ __forceinline__ float less(const Pack<T, N>& pack, int i, float m) {
    if constexpr (std::is_same_v<T, _Float16>) {
        float r;
        if (i & 1) asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(pack.w[i / 2]), "v"(m));
        else asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(pack.w[i / 2]), "v"(m));
        return r;
    }
    return pack.at(i) - m;
}

// The value of lane ^ DISTANCE.
template <int DISTANCE>
__device__ __forceinline__ float lane_across(float v) {
    if constexpr (DISTANCE == 1) return lane_moved<0xB1>(v);
    else if constexpr (DISTANCE == 2) return lane_moved<0x4E>(v);
    else if constexpr (DISTANCE == 4) return lane_moved<0x1B>(lane_moved<0x141>(v));  // 7 - i, then 3 - i
    else if constexpr (DISTANCE == 8) return lane_moved<0x128>(v);  // a row of 16 lanes turned by 8
    else return __shfl_xor(v, DISTANCE);
}

// One wave's values sorted in falling order over its lanes (a bitonic network).
template <int SIZE = 2, int DISTANCE = 1>
__device__ __forceinline__ float wave_sorted(float v) {
    const int lane = threadIdx.x & 63;
    const float other = lane_across<DISTANCE>(v);
    v = ((lane & DISTANCE) == 0) == ((lane & SIZE) == 0) ? fmaxf(v, other) : fminf(v, other);
    if constexpr (DISTANCE > 1) return wave_sorted<SIZE, DISTANCE / 2>(v);
    else if constexpr (SIZE < 64) return wave_sorted<2 * SIZE, SIZE>(v);
    else return v;
}

// The next float below (of a float above -inf).
__device__ __forceinline__ float just_below(float v) {
    const unsigned bits = __float_as_uint(v);
    return __uint_as_float(v > 0.0f ? bits - 1 : v == 0.0f ? 0x80000001u : bits + 1);
}

// The k largest keys of a run in falling order (0 where there are fewer), by k rounds a tile of the largest key
// below the last, for the tiles that hold a key above the k-th best so far.
template <typename T, int THREADS>
__device__ __forceinline__ const unsigned long long* exact_top(TopState<THREADS / 64>& top, const T* __restrict__ z,
                                                               const RowRun& run, int k) {
    using Tile = RowTile<T, THREADS>;
    const int tid = threadIdx.x;
    int side = 0;
    __syncthreads();
    if (tid < k) top.best[0][tid] = 0;
    __syncthreads();
#pragma unroll 1
    for (int base = run.begin; base < run.end; base += Tile::SIZE) {
        Tile tile;
        tile.load(z, base, run.end);
        const unsigned long long least = top.best[side][k - 1];
        unsigned long long last = ~0ull;
        bool above = true;
#pragma unroll 1
        for (int i = 0; i < k && last; ++i) {
            unsigned long long mine = 0;
            int from = base;
#pragma unroll
            for (int p = 0; p < TILE_PACKS; ++p) {
                tile.packs[p].stay_packed();
                asm volatile("" : "+s"(from));  // the keys are formed anew: they would take 64 registers
#pragma unroll
                for (int e = 0; e < Tile::N; ++e) {
                    const float x = tile.packs[p].at(e);
                    const int at = Tile::index(from, p, e);
                    const unsigned long long key = key_of(x, at);
                    if (x == x && at < run.end && key < last && key > mine) mine = key;
                }
            }
            if (i == 0) {
                above = __syncthreads_or(mine > least);
                if (!above) break;
            }
            if (tid < k) {
                const unsigned long long key = top.best[side][tid];
                if (key < last && key > mine) mine = key;
            }
            for (int o = 32; o > 0; o /= 2) {
                const unsigned long long other = __shfl_xor(mine, o);
                if (other > mine) mine = other;
            }
            if constexpr (THREADS > 64) {
                __syncthreads();
                if ((tid & 63) == 0) top.wave_best[tid / 64] = mine;
                __syncthreads();
                for (int w = 0; w < THREADS / 64; ++w)
                    if (top.wave_best[w] > mine) mine = top.wave_best[w];
            }
            last = mine;
            if (tid == 0) top.best[side ^ 1][i] = last;
            if (last == 0 && tid > i && tid < k) top.best[side ^ 1][tid] = 0;
        }
        if (above) side ^= 1;
        __syncthreads();
    }
    return top.best[side];
}

// The ranks of `count` distinct keys, by all waves: emit(rank, key) for those below k. Each wave counts, for every
// key, the larger ones of its own list (of `listed` keys); 256 keys at a time, four a lane. ranks is scratch.
template <int WAVES, typename KeyAt, typename Emit>
__device__ __forceinline__ void emit_ranks(KeyAt&& key_at, int count, int k, const unsigned long long* list, int listed,
                                           int* ranks, Emit&& emit) {
    static_assert(WAVES == 1 || WAVES == 4, "a lane's four keys go to one wave or to four");
    const int tid = threadIdx.x, lane = tid & 63;
#pragma unroll 1
    for (int base = 0; base < count; base += 256) {
        unsigned long long keys[4];
        int larger[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) keys[i] = base + i * 64 + lane < count ? key_at(base + i * 64 + lane) : ~0ull;
        const int blocks = (min(count - base, 256) + 63) / 64;
        if constexpr (WAVES > 1) {
            ranks[tid] = 0;
            __syncthreads();
        }
        if (blocks <= 2) {
#pragma unroll 4
            for (int j = 0; j < listed; ++j) {
                const unsigned long long other = list[j];
                larger[0] += other > keys[0];
                larger[1] += other > keys[1];
            }
        } else {
#pragma unroll 2
            for (int j = 0; j < listed; ++j) {
                const unsigned long long other = list[j];
#pragma unroll
                for (int i = 0; i < 4; ++i) larger[i] += other > keys[i];
            }
        }
        if constexpr (WAVES > 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < blocks) atomicAdd(&ranks[i * 64 + lane], larger[i]);
            __syncthreads();
            if (base + tid < count && ranks[tid] < k) emit(ranks[tid], key_at(base + tid));
            __syncthreads();
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (keys[i] != ~0ull && larger[i] < k) emit(larger[i], keys[i]);
        }
    }
}

// Takes the run's k largest keys to emit(rank, key), and emit(rank, 0) for those that are missing. Fewer than k
// candidates mean that all logits above -inf are candidates: the first -inf of the run follow. `mine` is the
// number of the wave's candidates.
template <typename T, int THREADS, typename Emit>
__device__ __forceinline__ void emit_top(TopState<THREADS / 64>& top, const T* __restrict__ z, const RowRun& run, int k,
                                         int mine, float s, Emit&& emit) {
    constexpr int WAVES = THREADS / 64;
    if ((threadIdx.x & 63) == 0) top.counts[threadIdx.x / 64] = mine;
    __syncthreads();
    int counts[WAVES], count = 0;
    bool exact = s != s;  // a NaN among a thread's logits leaves its maximum open
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        counts[w] = __builtin_amdgcn_readfirstlane(top.counts[w]);
        count += counts[w];
        exact = exact || counts[w] > WAVE_CANDIDATES;
    }
    if (exact) {
        const unsigned long long* best = exact_top<T, THREADS>(top, z, run, k);
        if (static_cast<int>(threadIdx.x) < k) emit(static_cast<int>(threadIdx.x), best[threadIdx.x]);
        return;
    }
    const auto key_at = [&](int i) {
        int wave = 0;
#pragma unroll
        for (int w = 0; w + 1 < WAVES; ++w)
            if (wave == w && i >= counts[w]) {
                i -= counts[w];
                wave = w + 1;
            }
        return top.candidates[wave][i];
    };
    emit_ranks<WAVES>(key_at, count, k, top.candidates[threadIdx.x / 64], mine, top.ranks, emit);
    if (count >= k || threadIdx.x >= 64) return;
    int next = count;
#pragma unroll 1
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

// What a thread carries through the tiles of a run.
struct RowState {
    RowStats mine;
    float place_max[4];  // one wave: the largest at each place of a pack
    float below;         // candidates lie above this
    int count;           // of the wave's candidates
    int side;            // of the shared thresholds
    int sets, each;      // k logits reach the each-th largest of the 64 maxima of `sets` sets
    bool lanes;          // one wave: of the lanes' maxima over all places, the only set
};

// The sets of a run's logits that a threshold is formed of: what a wave holds, or, in a workgroup of one wave,
// what its threads hold at one place of their packs. The last is left out where too few of its lanes hold any.
template <int WAVES>
__device__ __forceinline__ void choose_sets(RowState& state, int logits, int k, int lane_logits) {
    const int full = 64 * lane_logits;
    int sets = min(4, (logits + full - 1) / full);
    const int last = min(64, (logits - (sets - 1) * full + lane_logits - 1) / lane_logits);
    if (sets > 1 && last < (k + sets - 1) / sets) --sets;
    state.sets = sets;
    state.each = (k + sets - 1) / sets;
    // One set of all lanes lets a third more through for 20 alternatives, and many times more for 64. One set against
    // places, 4096 rows of 1000 float32 logits: 5 alternatives 7.6 / 12.0 us, 24 9.6 / 12.8, 32 10.1 / 13.4, 48 12.0 / 14.3,
    // 64 83 / 17.4 (the lists overflow); of 2000 float16 ones 24 11.5 / 15.2, 48 14.8 / 17.2, 64 151 / 20.8. So the rule
    // stays well clear of where one set fails; between 24 and 48 it gives up 2 to 4 us.
    state.lanes = WAVES == 1 && k <= 24 && logits >= full;
    if (state.lanes) state.each = k;
}

// Raises the threshold to what the each-th largest of the 64 maxima of each set reaches: at least k logits do.
// Drops the candidates below it.
template <int WAVES>
__device__ __forceinline__ void raise_threshold(RowState& state, TopState<WAVES>& top, float to) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    float kth;
    if constexpr (WAVES > 1) {
        const float sorted = wave_sorted(to > LOWEST ? to : -INFINITY);
        const float own = lane_of(sorted, state.each - 1);
        if (lane == 0) top.kth[state.side][wave] = own;
        __syncthreads();
        kth = top.kth[state.side][0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w)
            if (w < state.sets) kth = fminf(kth, top.kth[state.side][w]);
        state.side ^= 1;  // what is written next was read before the last barrier
    } else if (state.lanes) {
        kth = lane_of(wave_sorted(to > LOWEST ? to : -INFINITY), state.each - 1);
    } else {
        kth = INFINITY;
#pragma unroll
        for (int p = 0; p < 4; ++p)
            if (p < state.sets) kth = fminf(kth, lane_of(wave_sorted(state.place_max[p]), state.each - 1));
    }
    if (!(kth > state.below)) return;
    state.below = just_below(kth);
    if (state.count > WAVE_CANDIDATES) return;  // the list is lost
    unsigned long long* list = top.candidates[wave];
    int kept = 0;
#pragma unroll 1
    for (int i = 0; i < state.count; i += 64) {
        const unsigned long long key = i + lane < state.count ? list[i + lane] : 0;
        const bool keep = key && key_value(key) > state.below;
        const unsigned long long who = __ballot(keep);
        if (keep) list[kept + __popcll(who & ((1ull << lane) - 1))] = key;  // at or before where it was read
        kept += __popcll(who);
    }
    state.count = kept;
}

// One tile into the thread's statistics and, with TOP, the wave's list of candidates. Places of packs that lie
// past the run's end are left out.
template <bool ENTROPY, bool TOP, typename T, int THREADS>
__device__ __forceinline__ void take_tile(RowTile<T, THREADS>& tile, RowState& state, float scale, int base, int end,
                                          TopState<THREADS / 64>* top, int number) {
    using Tile = RowTile<T, THREADS>;
    const auto there = [&](int p) { return p == 0 || base + p * THREADS * Tile::N < end; };
    float pack_max[TILE_PACKS], to = state.mine.m;
#pragma unroll
    for (int p = 0; p < TILE_PACKS; ++p) {
        pack_max[p] = -INFINITY;
        if (there(p)) pack_max[p] = largest(tile.packs[p]);
        to = fmaxf(to, pack_max[p]);
    }
    if constexpr (TOP) {
#pragma unroll
        for (int p = 0; p < TILE_PACKS; ++p) {
            tile.packs[p].stay_packed();
            if constexpr (THREADS == 64) state.place_max[p] = fmaxf(state.place_max[p], pack_max[p]);
        }
        // At the tiles 0, 2, 8, 32, ...: what a threshold lets through until the next is at most three times what
        // it was formed from.
        if (number == 0 || ((number & (number - 1)) == 0 && (__ffs(number) & 1) == 0))
            raise_threshold<THREADS / 64>(state, *top, to);
        unsigned long long* list = top->candidates[threadIdx.x / 64];
        const unsigned long long before = (1ull << (threadIdx.x & 63)) - 1;
#pragma unroll
        for (int p = 0; p < TILE_PACKS; ++p) {
            if (!__any(pack_max[p] > state.below)) continue;
#pragma unroll
            for (int e = 0; e < Tile::N; ++e) {
                const float x = tile.packs[p].at(e);
                const unsigned long long who = __ballot(x > state.below);
                if (!who) continue;
                const int slot = state.count + __popcll(who & before);
                if (x > state.below && slot < WAVE_CANDIDATES) list[slot] = key_of(x, Tile::index(base, p, e));
                state.count += __popcll(who);
            }
        }
    }
#pragma unroll
    for (int p = 0; p < TILE_PACKS; ++p) tile.packs[p].stay_packed();
    state.mine.rescale(to, scale);
    float s = 0.0f, t = 0.0f;  // of the tile: a chain of additions is a tile's logits and the tiles, not all logits
#pragma unroll
    for (int p = 0; p < TILE_PACKS; ++p) {
        if (!there(p)) continue;
#pragma unroll
        for (int e = 0; e < Tile::N; ++e) {
            const float d = less(tile.packs[p], e, state.mine.m);
            const float part = exp2_of(d * scale);
            s += part;
            if constexpr (ENTROPY) t += part * fmaxf(d, DIFFERENCE_FLOOR);
        }
    }
    state.mine.s += s;
    state.mine.t += t;
}

// The statistics of a run, the same in every thread, and the number of the wave's candidates. `meanwhile` runs
// while the first tile's loads are in flight.
template <bool ENTROPY, bool TOP, typename T, int THREADS, typename Meanwhile>
__device__ __forceinline__ RowStats take_run(const T* __restrict__ z, const RowRun& run, float scale,
                                             TopState<THREADS / 64>* top, int top_k, int& count, Meanwhile&& meanwhile) {
    using Tile = RowTile<T, THREADS>;
    __shared__ RowStats waves[THREADS / 64];
    __shared__ float wave_m[THREADS / 64];
    RowState state{RowStats::none(), {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, -INFINITY, 0, 0, 1, 1, false};
    if constexpr (TOP) choose_sets<THREADS / 64>(state, run.end - run.begin, top_k, Tile::N);
    Tile tile;
    tile.load(z, run.begin, run.end);
    meanwhile();
    int base = run.begin;
#pragma unroll 1
    for (int number = 0;; ++number) {
        Tile next;
        const bool last = base + Tile::SIZE >= run.end;
        if (!last) next.load(z, base + Tile::SIZE, run.end);
        take_tile<ENTROPY, TOP>(tile, state, scale, base, run.end, top, number);
        if (last) break;
        tile = next;
        base += Tile::SIZE;
    }
    count = state.count;
    RowStats mine = state.mine;
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

// Whether this workgroup is the last of `total` to get here; what the others handed over before is then there to
// read. Every wave waits until its own writes are done before the workgroup is counted. The last one leaves the
// counter at 0 for the next call. Nobody waits for another workgroup.
__device__ __forceinline__ bool last_to_come(unsigned* counter, unsigned total) {
    __shared__ bool last;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
        last = atomicAdd(counter, 1u) + 1 == total;
        if (last) hand_over(counter, 0u);
    }
    __syncthreads();
    return last;
}

constexpr int SPLIT_MAX = 64;

// The runs of a row (at most 64) joined by each wave, the same in every lane.
__device__ __forceinline__ RowStats join_runs(const RowStats* stats, int chunks, float scale) {
    const int lane = threadIdx.x & 63;
    RowStats mine = RowStats::none();
    if (lane < chunks) mine = {handed_over(&stats[lane].m), handed_over(&stats[lane].s), handed_over(&stats[lane].t)};
    mine.rescale(wave_max(mine.m), scale);
    mine.s = wave_sum(mine.s);
    mine.t = wave_sum(mine.t);
    return mine;
}

struct JoinState {
    unsigned long long kept[SPLIT_MAX * TOP_MAX], bounds[2][SPLIT_MAX];
    int ranks[ROW_THREADS], count;
};

// The first keys of a row's runs, KEPT a thread, on their way while the runs' statistics are joined.
struct JoinKeys {
    static constexpr int KEPT = 2;
    unsigned long long keys[KEPT];
    __device__ __forceinline__ JoinKeys(const unsigned long long* from, int total) {
#pragma unroll
        for (int i = 0; i < KEPT; ++i) {
            const int at = static_cast<int>(threadIdx.x) + i * ROW_THREADS;
            keys[i] = at < total ? handed_over(from + at) : 0;
        }
    }
};

// The k largest keys of a row's runs, each run's in falling order. At least k keys reach the smallest of the runs'
// keys at place ceil(k / runs), and k those of any run its k-th: keys below the larger of the two bounds are none
// of the k largest.
template <typename Emit>
__device__ __forceinline__ void join_top(JoinState& join, const JoinKeys& first, const unsigned long long* keys, int chunks,
                                         int k, Emit&& emit) {
    constexpr int WAVES = ROW_THREADS / 64;
    const int tid = threadIdx.x, total = chunks * k, place = (k + chunks - 1) / chunks - 1;
    const auto bound = [&](int at, unsigned long long key) {
        const int chunk = at / k, rank = at - chunk * k;
        if (rank == place) join.bounds[0][chunk] = key;
        if (rank == k - 1) join.bounds[1][chunk] = key;
    };
    // Calls with every key of this thread.
    const auto each = [&](auto&& take) {
#pragma unroll
        for (int i = 0; i < JoinKeys::KEPT; ++i)
            if (tid + i * ROW_THREADS < total) take(tid + i * ROW_THREADS, first.keys[i]);
        for (int at = tid + JoinKeys::KEPT * ROW_THREADS; at < total; at += ROW_THREADS) take(at, handed_over(keys + at));
    };
    __syncthreads();  // what the run's own alternatives left in LDS is read
    each(bound);
    if (tid == 0) join.count = 0;
    __syncthreads();
    unsigned long long all = ~0ull, any = 0;
    for (int i = 0; i < chunks; ++i) {
        all = min(all, join.bounds[0][i]);
        any = max(any, join.bounds[1][i]);
    }
    const unsigned long long least = max(max(all, any), 1ull);
    each([&](int, unsigned long long key) {
        if (key >= least) join.kept[atomicAdd(&join.count, 1)] = key;
    });
    __syncthreads();
    const int found = join.count, part = (found + WAVES - 1) / WAVES, from = min(found, tid / 64 * part);
    emit_ranks<WAVES>([&](int i) { return join.kept[i]; }, found, k, join.kept + from, min(part, found - from), join.ranks, emit);
    for (int i = found + tid; i < k; i += ROW_THREADS) emit(i, 0);
}

// With SPLIT a workgroup takes a run of a row and the last one of a row joins its runs.
template <typename T, int THREADS, bool TOP, bool SPLIT>
__global__ __launch_bounds__(THREADS, SPLIT ? 4 : 8) void log_probs_kernel(const T* __restrict__ logits, LogProbsForward f,
                                                                           RowSplit split, RowPartials partials) {
    union Shared {
        TopState<THREADS / 64> top;
        JoinState join;
    };
    const RowRun run = run_of(split, f.vocab);
    const T* __restrict__ z = logits + run.row * f.stride;
    const long long at = run.row * split.chunks + run.chunk;
    GivenToken given{};
    int count = 0;
    const auto meanwhile = [&] {
        if (threadIdx.x == 0) given = GivenToken(f, z, run.row);
    };
    RowStats row;
    if constexpr (TOP) {
        __shared__ std::conditional_t<SPLIT, Shared, TopState<THREADS / 64>> shared;
        auto& top = *reinterpret_cast<TopState<THREADS / 64>*>(&shared);
        row = take_run<true, true, T, THREADS>(z, run, LOG2E, &top, f.top, count, meanwhile);
        if constexpr (!SPLIT) {
            const RowEnd end(row);
            emit_top<T, THREADS>(top, z, run, f.top, count, row.s,
                                 [&](int rank, unsigned long long key) { write_top(f, run.row, rank, key, end); });
        } else {
            emit_top<T, THREADS>(top, z, run, f.top, count, row.s,
                                 [&](int rank, unsigned long long key) { hand_over(partials.keys + at * f.top + rank, key); });
        }
        if constexpr (SPLIT) {
            if (threadIdx.x == 0) hand_over(partials.stats + at, row);
            if (!last_to_come(f.counters + run.row, split.chunks)) return;
            const unsigned long long* keys = partials.keys + run.row * split.chunks * f.top;
            const JoinKeys first(keys, split.chunks * f.top);
            row = join_runs(partials.stats + run.row * split.chunks, split.chunks, LOG2E);
            const RowEnd end(row);
            join_top(reinterpret_cast<Shared*>(&shared)->join, first, keys, split.chunks, f.top,
                     [&](int rank, unsigned long long key) { write_top(f, run.row, rank, key, end); });
        }
    } else {
        row = take_run<true, false, T, THREADS>(z, run, LOG2E, nullptr, 0, count, meanwhile);
        if constexpr (SPLIT) {
            if (threadIdx.x == 0) hand_over(partials.stats + at, row);
            if (!last_to_come(f.counters + run.row, split.chunks)) return;
            row = join_runs(partials.stats + run.row * split.chunks, split.chunks, LOG2E);
        }
    }
    if (threadIdx.x == 0) finish_log_probs(f, run.row, given, row);
}

// out[0] = scale * sum w v / sum w and out[1] = 1 / sum w (both 0 when nothing counts), in FP64 by one workgroup:
// thread t adds rows t, t + threads, ... in order, a fixed tree the threads' sums. weight_of(r) is 0 for a row
// that does not count; it adds nothing, whatever its value is.
template <int THREADS, typename ValueOf, typename WeightOf>
__device__ __forceinline__ void mean_of_rows(ValueOf&& value_of, WeightOf&& weight_of, long long rows, float scale,
                                             float* __restrict__ out) {
    __shared__ double sum[THREADS], weight[THREADS];
    double a = 0.0, b = 0.0;
    for (long long r = threadIdx.x; r < rows; r += THREADS) {
        const float w = weight_of(r);
        if (w == 0.0f) continue;
        a += static_cast<double>(w) * static_cast<double>(value_of(r));
        b += static_cast<double>(w);
    }
    sum[threadIdx.x] = a;
    weight[threadIdx.x] = b;
    __syncthreads();
    for (int half = THREADS / 2; half > 0; half /= 2) {
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

// The loss of few rows comes from the last workgroup of all, that of many from a launch of its own. Last workgroup
// against launch: 16 rows of 1000 float32 logits 6.6 / 7.5 us, 64 7.0 / 7.6, 128 8.2 / 7.7, 256 10.5 / 8.1, 1024 27 / 8.2
// (its 64 threads read the rows' values one round trip after another); of 32768 bfloat16 logits, by 256 threads, 64 rows
// 8.8 / 9.6, 256 12.5 / 11.2.
constexpr int MEAN_ROWS = 128;

template <typename T, int THREADS, bool SPLIT>
__global__ __launch_bounds__(THREADS) void distill_kernel(const T* __restrict__ logits, DistillForward f, RowSplit split,
                                                          RowPartials partials) {
    const RowRun run = run_of(split, f.vocab);
    const T* __restrict__ z = logits + run.row * f.stride;
    int count;
    TeacherRow<THREADS> teacher;
    // Every run of a row reads the teacher's record while its first tile is on the way (any may be the last).
    RowStats row = take_run<false, false, T, THREADS>(z, run, LOG2E / f.temperature, nullptr, 0, count,
                                                      [&] { teacher.read(f, z, run.row, run.chunk == 0); });
    if constexpr (SPLIT) {
        if (threadIdx.x == 0) hand_over(partials.stats + run.row * split.chunks + run.chunk, row);
        if (!last_to_come(f.counters + run.row, split.chunks)) return;
        row = join_runs(partials.stats + run.row * split.chunks, split.chunks, LOG2E / f.temperature);
    }
    teacher.finish(f, run.row, row);
    if (f.rows > MEAN_ROWS || !last_to_come(f.counters + LOGIT_SPLIT_ROWS, static_cast<unsigned>(f.rows))) return;
    mean_of_rows<THREADS>([&](long long r) { return handed_over(f.row_loss + r); },
                          [&](long long r) { return handed_over(f.weights + r); }, f.rows, 1.0f, f.loss);
}

// ---- the gradients --------------------------------------------------------------------------
// A workgroup forms GRAD_PACKS packs a thread of one row's gradient: every logit is read once and every
// gradient written once, p formed again from the row's m and s. Bound by HBM: 1000 x 50021 float32 61 us (6.6
// TB/s, part of it from the cache), 2048 x 65536 bfloat16 against 64 teacher logits a row 75 behind the
// forward, which leaves part of them in the cache (7.2), and 102 alone.
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
            float result[N];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                result[e] = value(in[p].at(e), at + e);
                if constexpr (ADD) result[e] += old[p].at(e);
            }
            store_pack(out + at, Pack<T, N>::of(result));
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
    const long long t = b.log_prob_grad ? whole_at(b.tokens, b.tokens_wide, r * b.tokens_step) : -1;
    const float factor = b.factor ? b.factor[0] : 1.0f;
    float g = t < 0 ? 0.0f : b.scale * factor * b.log_prob_grad[r * b.log_prob_step];
    if (t >= b.vocab && g != 0.0f) g = NOT_A_NUMBER;  // as its log probability
    else if (s == 0.0f) g = 0.0f;
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
        id = whole_at(b.ids, b.ids_wide, r * b.ids_step + threadIdx.x);
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

// w is the row's weight, or whether its token is given, or 1.
__global__ __launch_bounds__(MEAN_THREADS) void row_mean_kernel(const float* __restrict__ values,
                                                                const float* __restrict__ weights,
                                                                const void* __restrict__ tokens, int tokens_wide,
                                                                long long tokens_step, long long rows, float scale, float* __restrict__ out) {
    mean_of_rows<MEAN_THREADS>(
        [&](long long r) { return values[r]; },
        [&](long long r) { return weights ? weights[r] : tokens && whole_at(tokens, tokens_wide, r * tokens_step) < 0 ? 0.0f : 1.0f; },
        rows, scale, out);
}

// Threads of a row's workgroup: a wave while a row is at most two tiles of it (no barriers), else four.
constexpr int SMALL_ROW_BYTES = 2 * 64 * TILE_PACKS * 16, WAVE_THREADS = 64;

bool small_row(int vocab, int type) { return vocab * static_cast<std::int64_t>(type_bytes(type)) <= SMALL_ROW_BYTES; }

// Runs of a row. Rows are split where the time that whole rows leave CUs idle is more than joining them takes:
// of 256 CUs that read ROW_RATE bytes a microsecond each (5/8 of that with one workgroup), whole rows take the most
// that one CU has of them, split ones their share and JOIN_TIME. Measured without / with 20 alternatives, float32,
// whole -> split: one row of 16384 3.8 / 8.8 -> 3.5 / 8.2 us and of 131072 17.7 / 31.2 -> 4.1 / 10.9, 250 of 16384
// 4.4 / 11.2 -> 5.9 / 11.9 and of 131072 26.2 / 44.9 -> 23.8 / 29.6. Over 260 sizes from 1 to 500 rows of 12 to
// 512 KB the rule's choice is 1% slower than the better one, always whole 18%, always split 7%. Then as many runs as
// bring the workgroups to SPLIT_GROUPS, of at least one tile; from 513 rows on that is one, whatever the estimate says.
// Whole against two runs a row there, without / with 20 alternatives: 513 x 32771 float16 11.7 / 18.7 -> 12.8 / 26.5 us,
// 777 x 32771 16.3 / 24.4 -> 17.0 / 33.1, 700 x 131072 bfloat16 37.6 / 50.3 -> 39.5 / 57.9; the best gain was 36.8 -> 32.9
// (520 x 131072 without alternatives). All of this follows from the sizes alone, so that results do not depend on the
// device.
constexpr int SPLIT_GROUPS = 1024, ROW_RATE = 20000, JOIN_TIME = 3, SPLIT_CUS = 256;
RowSplit row_split(std::int64_t rows, int vocab, int type) {
    if (rows == 0 || small_row(vocab, type)) return {1, vocab};
    const std::int64_t bytes = static_cast<std::int64_t>(vocab) * type_bytes(type);
    const std::int64_t whole = rows <= SPLIT_CUS ? bytes * 8 / 5 : (rows + SPLIT_CUS - 1) / SPLIT_CUS * bytes;
    const std::int64_t shared = rows * bytes / SPLIT_CUS;
    if (whole - shared <= JOIN_TIME * ROW_RATE) return {1, vocab};
    const int unit = ROW_THREADS * 16 / type_bytes(type);  // a pack a thread
    const std::int64_t wanted = std::min<std::int64_t>(SPLIT_MAX, std::max<std::int64_t>(1, SPLIT_GROUPS / rows));
    const std::int64_t packs = (vocab + unit - 1) / unit;
    const int length = static_cast<int>(std::max<std::int64_t>(TILE_PACKS, (packs + wanted - 1) / wanted)) * unit;
    return {static_cast<int>((vocab + length - 1) / length), length};  // several runs of at most LOGIT_SPLIT_ROWS rows
}
static_assert(SPLIT_GROUPS / 2 <= LOGIT_SPLIT_ROWS, "a counter a row that is split");

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
        if (f.top && small) run(log_probs_kernel<T, WAVE_THREADS, true, false>, WAVE_THREADS);
        else if (f.top && split.chunks > 1) run(log_probs_kernel<T, ROW_THREADS, true, true>, ROW_THREADS);
        else if (f.top) run(log_probs_kernel<T, ROW_THREADS, true, false>, ROW_THREADS);
        else if (small) run(log_probs_kernel<T, WAVE_THREADS, false, false>, WAVE_THREADS);
        else if (split.chunks > 1) run(log_probs_kernel<T, ROW_THREADS, false, true>, ROW_THREADS);
        else run(log_probs_kernel<T, ROW_THREADS, false, false>, ROW_THREADS);
    });
    return MFH_CHECK_LAUNCH("log_probs", stream);
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
            const auto run = [&](auto kernel, int threads) { launch(kernel, groups, threads, 0, stream, z, f, split, partials); };
            if (small_row(f.vocab, type)) run(distill_kernel<T, WAVE_THREADS, false>, WAVE_THREADS);
            else if (split.chunks > 1) run(distill_kernel<T, ROW_THREADS, true>, ROW_THREADS);
            else run(distill_kernel<T, ROW_THREADS, false>, ROW_THREADS);
        });
        MFH_TRY(MFH_CHECK_LAUNCH("distill", stream));
        if (f.rows <= MEAN_ROWS) return OK;
    }
    return launch_row_mean(f.row_loss, f.weights, nullptr, 0, 0, f.rows, 1.0f, f.loss, stream);
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

int launch_row_mean(const float* values, const float* weights, const void* tokens, int tokens_wide, std::int64_t tokens_step,
                    std::int64_t rows, float scale, float* out, hipStream_t stream) {
    launch(row_mean_kernel, 1, MEAN_THREADS, 0, stream, values, weights, tokens, tokens_wide, tokens_step, rows, scale, out);
    return MFH_CHECK_LAUNCH("row_mean", stream);
}

}  // namespace mfh
