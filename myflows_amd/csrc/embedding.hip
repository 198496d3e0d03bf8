// Embedding: rows of a table by token, scaled, and the table's gradient by sorted tokens.
//
//   y[p] = scale T[id[p]]            (zeros where id[p] < 0, NaN where id[p] >= vocab)
//   dT[v] = scale sum over p with id[p] = v of dy[p], in float32
//
// The gradient is dense: a row that no token names is zero (or left as it is, with add). No atomics: the positions are
// sorted by token first. The rows of a token that comes seldom are added in rising order of p; those of a frequent one
// in pieces, and in narrow rows by lanes that share a piece, whose sums are joined in a fixed order. So a gradient has
// the same bits every time, but not those of one running sum.
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "common.h"
#include "typed.h"
#include "wave.h"

namespace mfh {
namespace {

constexpr int THREADS = 256;
constexpr int SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64;
constexpr unsigned BLOCKS_MAX = 1u << 20;  // of a launch; the kernels walk on from there
constexpr float NOT_A_NUMBER = __builtin_nanf("");

// ---- lookup -----------------------------------------------------------------------------------
// Bound by HBM (each row looked up is read and written once) or, for few rows, by the two dependent loads of an
// id and its row. A workgroup takes a few neighbouring rows, whose packs its threads share whatever the rows'
// length is; four packs a thread are in flight. 65536 rows of 2048 bfloat16: 69 us (7.7 TB/s, rows of frequent tokens
// from the caches).
constexpr int LOOKUP_PACKS = 4;

template <typename T>
__global__ __launch_bounds__(THREADS) void lookup_kernel(const T* __restrict__ table, T* __restrict__ out,
                                                         EmbeddingLookup f, int block_rows, FastDiv packs) {
    constexpr int N = 16 / sizeof(T);
    for (std::int64_t first = static_cast<std::int64_t>(blockIdx.x) * block_rows; first < f.count;
         first += static_cast<std::int64_t>(gridDim.x) * block_rows) {
        const int slots = static_cast<int>(min(static_cast<std::int64_t>(block_rows), f.count - first)) * static_cast<int>(packs.d);
        for (int base = threadIdx.x; base < slots; base += LOOKUP_PACKS * THREADS) {
            long long id[LOOKUP_PACKS];
            int column[LOOKUP_PACKS];
            Pack<T, N> pack[LOOKUP_PACKS];
#pragma unroll
            for (int k = 0; k < LOOKUP_PACKS; ++k) {
                const int slot = base + k * THREADS;
                id[k] = -1, column[k] = 0;
                if (slot >= slots) continue;
                int within;
                const int row = packs.divmod(slot, within);
                column[k] = within * N;
                id[k] = whole_at(f.ids, f.ids_wide, (first + row) * f.ids_step);
            }
#pragma unroll
            for (int k = 0; k < LOOKUP_PACKS; ++k) {
                pack[k] = Pack<T, N>::all(id[k] < 0 ? 0.0f : NOT_A_NUMBER);
                if (id[k] < 0 || id[k] >= f.vocab) continue;
                const T* from = table + id[k] * f.table_stride + column[k];
                pack[k] = column[k] + N <= f.dim ? load_pack<T, N>(from) : load_part<T, N>(from, f.dim - column[k], 0.0f);
            }
#pragma unroll
            for (int k = 0; k < LOOKUP_PACKS; ++k) {
                const int slot = base + k * THREADS;
                if (slot >= slots) continue;
                float v[N];
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = pack[k].at(i) * f.scale;
                T* to = out + (first + packs.div(slot)) * f.out_stride + column[k];
                if (column[k] + N <= f.dim) {
                    store_pack(to, Pack<T, N>::of(v));
                } else {
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (column[k] + i < f.dim) to[i] = static_cast<T>(v[i]);
                }
            }
        }
    }
}

// ---- positions by token -----------------------------------------------------------------------
// Token v's slot is (v mod classes) * slice + v / classes, with a power of two of classes: neighbouring tokens,
// the frequent ones of a vocabulary, lie in different classes. order: the positions whose token lies in the table,
// by (slot, position); slots: their slots; starts[s]: where slot s's begin, and starts[classes * slice] their number.
// One launch: a workgroup owns a class and reads all ids (from the caches: the ids are few beside the gradients'
// rows). Each of its waves takes a sixteenth of the positions, counts its own of each token and lists them in
// LDS; from the sums over the tokens and waves before it, it then places those it listed in their order, lanes with
// the same token finding one another by ballots, a token at a time. A wave whose list overflows (a token of every
// fourth position, say) reads its ids again instead. Bound by the instructions of the walk: 65536 ids of 65536
// tokens, 1 / k of them the k-th, 21 us (44 with two walks, 370 with neighbouring tokens in one class). A class has at most 1024 tokens:
// beyond 262144 of them there are more classes than CUs, and their walks take turns.
struct Sorted {
    int* order;
    int* slots;
    int* starts;
    int classes_log, slice;
};

__host__ __device__ __forceinline__ int slot_of(const Sorted& s, int token) {
    return (token & ((1 << s.classes_log) - 1)) * s.slice + (token >> s.classes_log);
}

// each(whether the token is of the class, its place there, position) for the positions begin .. end - 1, a wave's
// width at a time; adds this lane's positions of lower classes to `below`.
template <typename Whole, typename F>
__device__ __forceinline__ void walk_ids(const EmbeddingGradient& g, const Sorted& s, int begin, int end, int& below, F&& each) {
    constexpr int AHEAD = 8;
    const int mask = (1 << s.classes_log) - 1, own = blockIdx.x, lane = threadIdx.x & 63;
    const Whole* ids = static_cast<const Whole*>(g.ids) + (begin + lane) * g.ids_step;
    for (int base = begin; base < end; base += 64 * AHEAD, ids += 64 * AHEAD * g.ids_step) {
        Whole id[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) id[k] = base + 64 * k + lane < end ? ids[64 * k * g.ids_step] : -1;
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            using Unsigned = std::make_unsigned_t<Whole>;
            const bool there = static_cast<Unsigned>(id[k]) < static_cast<Unsigned>(g.vocab);
            const int token = static_cast<int>(id[k]), of = token & mask;
            below += there && of < own;
            each(there && of == own, token >> s.classes_log, base + 64 * k + lane);
        }
    }
}

// The lanes below this one that a ballot holds.
__device__ __forceinline__ int lanes_before(unsigned long long ballot) {
    return __builtin_amdgcn_mbcnt_hi(static_cast<unsigned>(ballot >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<unsigned>(ballot), 0u));
}

constexpr int LISTED = 512;  // positions of a wave's list

template <typename Whole>
__global__ __launch_bounds__(SORT_THREADS) void sort_kernel(EmbeddingGradient g, Sorted s, int wave_ids) {
    extern __shared__ int counters[];  // SORT_WAVES x slice
    __shared__ int positions[SORT_WAVES][LISTED];
    __shared__ unsigned short tokens[SORT_WAVES][LISTED];
    __shared__ int below_of[SORT_WAVES], sums[SORT_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64, tid = threadIdx.x, slice = s.slice;
    const int begin = static_cast<int>(min(static_cast<std::int64_t>(wave) * wave_ids, g.count));
    const int end = static_cast<int>(min(static_cast<std::int64_t>(wave + 1) * wave_ids, g.count));
    int* const mine = counters + wave * slice;
    for (int i = lane; i < slice; i += 64) mine[i] = 0;
    wave_order();
    int below = 0, unused = 0, listed = 0;
    walk_ids<Whole>(g, s, begin, end, below, [&](bool here, int local, int position) {
        const unsigned long long all = __ballot(here);
        if (!all) return;
        const int at = listed + lanes_before(all);
        if (here) {
            atomicAdd(&mine[local], 1);
            if (at < LISTED) positions[wave][at] = position, tokens[wave][at] = static_cast<unsigned short>(local);
        }
        listed += __popcll(all);
    });
    for (int o = 32; o > 0; o /= 2) below += __shfl_xor(below, o);
    if (lane == 0) below_of[wave] = below;
    __syncthreads();
    // The sums over the tokens before, one token a thread.
    int total = 0, before = 0;
    if (tid < slice)
        for (int w = 0; w < SORT_WAVES; ++w) total += counters[w * slice + tid];
    int scan = total;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const int other = __shfl_up(scan, o);
        if (lane >= o) scan += other;
    }
    if (lane == 63) sums[wave] = scan;
    __syncthreads();
    for (int w = 0; w < SORT_WAVES; ++w) before += below_of[w] + (w < wave ? sums[w] : 0);
    int at = before + scan - total;
    const int first = static_cast<int>(blockIdx.x) * slice;
    if (tid < slice) {
        s.starts[first + tid] = at;
        if (tid == slice - 1 && blockIdx.x == gridDim.x - 1) s.starts[first + slice] = at + total;
        for (int w = 0; w < SORT_WAVES; ++w) {
            const int held = counters[w * slice + tid];
            counters[w * slice + tid] = at;
            at += held;
        }
    }
    __syncthreads();
    const auto place = [&](bool here, int local, int position) {
        for (unsigned long long left = __ballot(here); left;) {
            const int token = __builtin_amdgcn_readlane(local, __builtin_ctzll(left));
            const unsigned long long same = __ballot(here && local == token);
            const int to = mine[token];
            if (here && local == token) {
                s.order[to + lanes_before(same)] = position;
                s.slots[to + lanes_before(same)] = first + token;
            }
            wave_order();
            if (lane == 0) mine[token] = to + __popcll(same);
            wave_order();
            left &= ~same;
        }
    };
    if (listed > LISTED) {
        walk_ids<Whole>(g, s, begin, end, unused, place);
        return;
    }
    wave_order();
    for (int i = 0; i < listed; i += 64) {
        const bool here = i + lane < listed;
        const int at = here ? i + lane : 0;
        place(here, tokens[wave][at], positions[wave][at]);
    }
}

// ---- sums -------------------------------------------------------------------------------------
// A token that comes more often than SumPlan::chunk times is summed in pieces: the sorted positions lie in chunks
// of that many, and a chunk holds a piece of at most two such tokens, the one that it begins with and the one that
// it ends with. sum_kernel's first workgroups sum the pieces, the others the rows of each other token; join_kernel
// sums the pieces of a token, of which at most one begins in a chunk. Bound by HBM: each gradient row is read once,
// the table's gradient written once. 65536 rows of 2048 bfloat16 into a table of 65536: 140 us and 9 (3.6 TB/s).
struct SumPlan {
    int chunk;       // positions of a piece
    int lanes;       // lanes (a power of two) that share a row's packs
    int columns;     // groups of `lanes` packs in a row
    int part_width;  // floats of a piece's row: whole packs
    unsigned part_blocks;
};

constexpr int IN_FLIGHT = 8;

// Adds the rows begin .. end - 1 of a lane's columns, IN_FLIGHT of them loaded at a time; load(i) gives row i's pack.
template <typename P, int N, typename Load>
__device__ __forceinline__ void add_rows(float (&sum)[N], int begin, int end, Load&& load) {
    for (int i = begin; i < end; i += IN_FLIGHT) {
        P pack[IN_FLIGHT];
#pragma unroll
        for (int k = 0; k < IN_FLIGHT; ++k)
            if (i + k < end) pack[k] = load(i + k);
#pragma unroll
        for (int k = 0; k < IN_FLIGHT; ++k) {
            if (i + k >= end) break;
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] += pack[k].at(e);
        }
    }
}

// Adds the gradient's rows at the sorted positions begin .. end - 1. Where a wave is one row's, it reads 64 of the
// positions at once.
template <bool WAVE, typename T, int N>
__device__ __forceinline__ void add_positions(float (&sum)[N], const T* __restrict__ grad, const EmbeddingGradient& g,
                                              const int* __restrict__ order, int begin, int end, int column) {
    const T* at = grad + column;
    const int there = g.dim - column;
    const auto load = [&](std::int64_t position) {
        const T* row = at + position * g.grad_stride;
        return there >= N ? load_pack<T, N>(row) : load_part<T, N>(row, there, 0.0f);
    };
    if constexpr (WAVE) {
        for (int base = begin; base < end; base += 64) {
            const int here = min(64, end - base);
            const int held = order[base + min(static_cast<int>(threadIdx.x & 63), here - 1)];
            add_rows<Pack<T, N>>(sum, 0, here, [&](int i) { return load(__builtin_amdgcn_readlane(held, i)); });
        }
    } else {
        add_rows<Pack<T, N>>(sum, begin, end, [&](int i) { return load(order[i]); });
    }
}

template <typename Out, int N>
__device__ __forceinline__ void write_sum(Out* __restrict__ out, const float (&sum)[N], const EmbeddingGradient& g, int token,
                                          int column) {
    Out* to = out + token * g.out_stride + column;
    float v[N];
    if (g.add) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = column + e < g.dim ? static_cast<float>(to[e]) + sum[e] * g.scale : 0.0f;
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = sum[e] * g.scale;
    }
    if (column + N <= g.dim) {
        store_pack(to, Pack<Out, N>::of(v));
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (column + e < g.dim) to[e] = static_cast<Out>(v[e]);
    }
}

// A value that a wave's lanes share, or each lane's own.
template <bool WAVE>
__device__ __forceinline__ int shared_by(int value) {
    return WAVE ? __builtin_amdgcn_readfirstlane(value) : value;
}

// each(task, the lane's column) for the tasks of the launch's blocks from first_block on: `rows` rows by
// plan.columns, a wave's lanes sharing 64 / plan.lanes of them.
template <bool WAVE, int N, typename F>
__device__ __forceinline__ void walk_tasks(const SumPlan& plan, const EmbeddingGradient& g, unsigned first_block, unsigned blocks,
                                           std::int64_t rows, F&& each) {
    const int lanes = WAVE ? 64 : plan.lanes, groups = 64 / lanes, lane = threadIdx.x & 63;
    const std::int64_t tasks = rows * plan.columns, step = static_cast<std::int64_t>(blocks) * (THREADS / 64) * groups;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    for (std::int64_t task = (static_cast<std::int64_t>(blockIdx.x - first_block) * (THREADS / 64) + wave) * groups +
                             (WAVE ? 0 : lane / lanes);
         task < tasks; task += step) {
        const int row = shared_by<WAVE>(static_cast<int>(task / plan.columns));
        const int column = (static_cast<int>(task - static_cast<std::int64_t>(row) * plan.columns) * lanes + (WAVE ? lane : lane % lanes)) * N;
        if (WAVE || column < g.dim) each(row, min(column, g.dim - 1), column < g.dim);
    }
}

// A wave's share of the pieces: `lanes` lanes to a row, and 64 / lanes groups of them that take neighbouring ranges of the
// rows that are summed, whose sums are then added in a fixed order. each(row, the lane's column, whether it is one, group).
template <int N, typename F>
__device__ __forceinline__ void walk_waves(const SumPlan& plan, const EmbeddingGradient& g, unsigned blocks, std::int64_t rows, F&& each) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    for (std::int64_t task = static_cast<std::int64_t>(blockIdx.x) * (THREADS / 64) + wave; task < rows * plan.columns;
         task += static_cast<std::int64_t>(blocks) * (THREADS / 64)) {
        const int row = static_cast<int>(task / plan.columns);
        const int column = (static_cast<int>(task - static_cast<std::int64_t>(row) * plan.columns) * plan.lanes + lane % plan.lanes) * N;
        each(row, min(column, g.dim - 1), column < g.dim, lane / plan.lanes);
    }
}

struct Range {
    int begin, end;
    // The group's part of begin .. end - 1.
    __device__ __forceinline__ Range part(int group, int groups) const {
        const int each = (end - begin + groups - 1) / groups, from = min(begin + group * each, end);
        return {from, min(from + each, end)};
    }
};

template <int N>
__device__ __forceinline__ void add_groups(float (&sum)[N], int lanes) {
    for (int o = lanes; o < 64; o *= 2)
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] += __shfl_xor(sum[e], o);
}

template <bool WAVE, typename T, typename Out>
__global__ __launch_bounds__(THREADS) void sum_kernel(const T* __restrict__ grad, Out* __restrict__ out, EmbeddingGradient g,
                                                      SumPlan plan, Sorted s, float* __restrict__ parts) {
    constexpr int N = 16 / sizeof(T);
    if (blockIdx.x < plan.part_blocks) {
        const int given = shared_by<WAVE>(s.starts[s.slice << s.classes_log]);
        const int chunks = (given + plan.chunk - 1) / plan.chunk;
        walk_waves<N>(plan, g, plan.part_blocks, chunks, [&](int chunk, int column, bool there, int group) {
            const int begin = chunk * plan.chunk, end = min(begin + plan.chunk, given);
#pragma unroll 1
            for (int last = 0; last < 2; ++last) {
                const int slot = __builtin_amdgcn_readfirstlane(s.slots[last ? end - 1 : begin]);
                const int from = __builtin_amdgcn_readfirstlane(s.starts[slot]), to = __builtin_amdgcn_readfirstlane(s.starts[slot + 1]);
                if (to - from <= plan.chunk || (last && from <= begin)) continue;
                const Range piece{max(from, begin), min(to, end)}, mine = WAVE ? piece : piece.part(group, 64 / plan.lanes);
                float sum[N] = {};
                add_positions<WAVE, T, N>(sum, grad, g, s.order, mine.begin, mine.end, column);
                if (!WAVE) add_groups(sum, plan.lanes);
                if (!there || group) continue;
                float* to_part = parts + (2 * static_cast<std::int64_t>(chunk) + last) * plan.part_width + column;
#pragma unroll
                for (int e = 0; e < N; ++e) to_part[e] = sum[e];
            }
        });
        return;
    }
    walk_tasks<WAVE, N>(plan, g, plan.part_blocks, gridDim.x - plan.part_blocks, g.vocab, [&](int token, int column, bool there) {
        const int slot = slot_of(s, token), from = shared_by<WAVE>(s.starts[slot]), to = shared_by<WAVE>(s.starts[slot + 1]);
        if (to - from > plan.chunk || (from == to && g.add)) return;
        float sum[N] = {};
        add_positions<WAVE, T, N>(sum, grad, g, s.order, from, to, column);
        if (there) write_sum(out, sum, g, token, column);
    });
}

template <int N, typename Out>
__global__ __launch_bounds__(THREADS) void join_kernel(Out* __restrict__ out, EmbeddingGradient g, SumPlan plan, Sorted s,
                                                       const float* __restrict__ parts) {
    const int given = s.starts[s.slice << s.classes_log];
    const int chunks = (given + plan.chunk - 1) / plan.chunk;
    walk_waves<N>(plan, g, gridDim.x, chunks, [&](int chunk, int column, bool there, int group) {
        const int begin = chunk * plan.chunk, slot = __builtin_amdgcn_readfirstlane(s.slots[min(begin + plan.chunk, given) - 1]);
        const int from = __builtin_amdgcn_readfirstlane(s.starts[slot]), to = __builtin_amdgcn_readfirstlane(s.starts[slot + 1]);
        if (to - from <= plan.chunk || from < begin) return;
        // The first piece ends its chunk, unless it begins there; every further one begins its chunk.
        float sum[N] = {};
        const Range mine = Range{chunk, (to - 1) / plan.chunk + 1}.part(group, 64 / plan.lanes);
        add_rows<Pack<float, N>>(sum, mine.begin, mine.end, [&](int c) {
            const int ends = c == chunk && from != begin;
            return load_pack<float, N>(parts + (2 * static_cast<std::int64_t>(c) + ends) * plan.part_width + column / N * N);
        });
        add_groups(sum, plan.lanes);
        if (!there || group) return;
        const int token_class = slot / s.slice;
        write_sum(out, sum, g, ((slot - token_class * s.slice) << s.classes_log) + token_class, column);
    });
}

// Pieces of 64 positions, longer ones for many positions: a piece and the join of all pieces of one token take
// about as many steps.
int chunk_of(std::int64_t count) {
    int chunk = 64;
    while (static_cast<std::int64_t>(chunk) * chunk * 8 < count) chunk *= 2;
    return chunk;
}

unsigned wave_blocks(std::int64_t rows, const SumPlan& plan) {
    const std::int64_t groups = 64 / plan.lanes * (THREADS / 64);
    return static_cast<unsigned>(std::min<std::int64_t>((rows * plan.columns + groups - 1) / groups, BLOCKS_MAX));
}

std::int64_t chunks_of(const EmbeddingGradient& g, const SumPlan& plan) {
    return g.count <= plan.chunk ? 0 : (g.count + plan.chunk - 1) / plan.chunk;
}

SumPlan sum_plan(const EmbeddingGradient& g, int type) {
    const int n = 16 / type_bytes(type), packs = (g.dim + n - 1) / n;
    SumPlan plan{chunk_of(g.count), 1, 1, packs * n, 0};
    while (plan.lanes < 64 && plan.lanes < packs) plan.lanes *= 2;
    plan.columns = (packs + plan.lanes - 1) / plan.lanes;
    plan.part_blocks = static_cast<unsigned>(std::min<std::int64_t>((chunks_of(g, plan) * plan.columns + THREADS / 64 - 1) / (THREADS / 64), BLOCKS_MAX));
    return plan;
}

// A class of tokens for every workgroup that the GPU takes at once; more where a class would have over 1024.
Sorted sorted_layout(const EmbeddingGradient& g) {
    Sorted s{};
    while ((1 << s.classes_log) < device_cu_count() && (1 << s.classes_log) < g.vocab) ++s.classes_log;
    while (g.vocab > static_cast<std::int64_t>(SORT_THREADS) << s.classes_log) ++s.classes_log;
    s.slice = (g.vocab + (1 << s.classes_log) - 1) >> s.classes_log;
    return s;
}

std::int64_t aligned(std::int64_t bytes) { return (bytes + 255) / 256 * 256; }

// The bytes of order and slots, of starts, and of the pieces.
struct Workspace {
    std::int64_t positions, starts, parts;
    Workspace(const EmbeddingGradient& g, const Sorted& s, const SumPlan& plan)
        : positions(aligned(4 * g.count)), starts(aligned(4 * ((static_cast<std::int64_t>(s.slice) << s.classes_log) + 1))),
          parts(4 * 2 * chunks_of(g, plan) * plan.part_width) {}
    std::int64_t bytes() const { return 2 * positions + starts + parts; }
};

}  // namespace

int launch_embedding(const void* table, void* out, int type, const EmbeddingLookup& f, hipStream_t stream) {
    if (f.count == 0) return OK;
    const int n = 16 / type_bytes(type), packs = (f.dim + n - 1) / n;
    // Rows of a workgroup: as many as four packs a thread take, fewer where that leaves CUs idle.
    std::int64_t rows = std::max(1, LOOKUP_PACKS * THREADS / packs);
    rows = std::max<std::int64_t>(1, std::min(rows, f.count / (2 * device_cu_count())));
    const unsigned blocks = static_cast<unsigned>(std::min<std::int64_t>((f.count + rows - 1) / rows, BLOCKS_MAX));
    with_type(type, [&](auto element) {
        using T = decltype(element);
        launch(lookup_kernel<T>, dim3(blocks), dim3(THREADS), 0, stream, static_cast<const T*>(table), static_cast<T*>(out), f,
               static_cast<int>(rows), FastDiv(packs));
    });
    return MFH_CHECK_LAUNCH("embedding lookup", stream);
}

std::int64_t embedding_workspace(const EmbeddingGradient& g, int type) {
    return Workspace(g, sorted_layout(g), sum_plan(g, type)).bytes();
}

int launch_embedding_backward(const void* grad, int type, void* out, int out_type, const EmbeddingGradient& g,
                              void* workspace, hipStream_t stream) {
    const SumPlan plan = sum_plan(g, type);
    Sorted s = sorted_layout(g);
    const Workspace held(g, s, plan);
    char* at = static_cast<char*>(workspace);
    s.order = reinterpret_cast<int*>(at);
    s.slots = reinterpret_cast<int*>(at + held.positions);
    s.starts = reinterpret_cast<int*>(at + 2 * held.positions);
    float* parts = reinterpret_cast<float*>(at + 2 * held.positions + held.starts);
    const int wave_ids = static_cast<int>(((g.count + SORT_WAVES - 1) / SORT_WAVES + 63) / 64 * 64);
    launch(g.ids_wide ? sort_kernel<long long> : sort_kernel<int>, dim3(1u << s.classes_log), dim3(SORT_THREADS),
           sizeof(int) * SORT_WAVES * s.slice, stream, g, s, wave_ids);
    MFH_TRY(MFH_CHECK_LAUNCH("embedding sort", stream));
    const auto sums = [&](auto element, auto* to) {
        using T = decltype(element);
        using Out = std::remove_pointer_t<decltype(to)>;
        launch(plan.lanes == 64 ? sum_kernel<true, T, Out> : sum_kernel<false, T, Out>,
               dim3(plan.part_blocks + wave_blocks(g.vocab, plan)), dim3(THREADS), 0, stream, static_cast<const T*>(grad), to, g,
               plan, s, parts);
        MFH_TRY(MFH_CHECK_LAUNCH("embedding sums", stream));
        if (plan.part_blocks == 0) return static_cast<int>(OK);
        launch(join_kernel<16 / sizeof(T), Out>, dim3(plan.part_blocks), dim3(THREADS), 0, stream, to, g, plan, s, parts);
        return MFH_CHECK_LAUNCH("embedding join", stream);
    };
    return with_type(type, [&](auto element) {
        using T = decltype(element);
        return out_type == type ? sums(element, static_cast<T*>(out)) : sums(element, static_cast<float*>(out));
    });
}

}  // namespace mfh
