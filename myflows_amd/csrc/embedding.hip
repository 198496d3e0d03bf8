// Embedding: rows of a table by token, scaled, and the table's gradient by sorted tokens.
//
//   y[p] = scale T[id[p]]            (zeros where id[p] < 0, NaN where id[p] >= vocab)
//   dT[v] = scale sum over p with id[p] = v of dy[p], in rising order of p, in float32
//
// The gradient is dense: a row that no token names is zero (or left as it is, with add). No atomics: the
// positions are sorted by token first, then each row's are summed in their order, so a gradient has the same
// bits every time.
#include <algorithm>
#include <cstdint>

#include "common.h"
#include "typed.h"

namespace mfh {
namespace {

constexpr int THREADS = 256;
constexpr int SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64;
constexpr unsigned BLOCKS_MAX = 1u << 20;  // of a launch; the kernels walk on from there
constexpr float NOT_A_NUMBER = __builtin_nanf("");

// ---- lookup -----------------------------------------------------------------------------------
// Bound by HBM (each row looked up is read and written once) or, for few rows, by the two dependent loads of an
// id and its row. A workgroup takes a few neighbouring rows, whose packs its threads share whatever the rows'
// length is; four packs a thread are in flight.
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
// order: the positions whose token lies in the table, by (token, position); starts[v]: where token v's begin, and
// starts[vocab] their number. One launch: a workgroup owns `slice` neighbouring tokens and reads all ids twice
// (from the caches: the ids are few beside the gradients' rows). Each of its waves takes a sixteenth of the
// positions: first it counts its own of each token, then, from the sums over the tokens and waves before, it
// places them in their order. Lanes with the same token find one another by ballots.
// What one lane of a wave wrote to LDS is there for the others' next read: the wave's accesses run in order.
__device__ __forceinline__ void wave_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

template <typename F>
__device__ __forceinline__ void walk_ids(const EmbeddingGradient& g, int begin, int end, F&& each) {
    constexpr int AHEAD = 8;
    for (int at = begin + (threadIdx.x & 63); at - static_cast<int>(threadIdx.x & 63) < end; at += 64 * AHEAD) {
        int id[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int p = at + 64 * k;
            const long long v = p < end ? whole_at(g.ids, g.ids_wide, p * g.ids_step) : -1;
            id[k] = v < 0 || v >= g.vocab ? -1 : static_cast<int>(v);
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) each(id[k], at + 64 * k);
    }
}

__global__ __launch_bounds__(SORT_THREADS) void sort_kernel(EmbeddingGradient g, int slice, int wave_ids, int* __restrict__ order,
                                                            int* __restrict__ starts) {
    extern __shared__ int counters[];  // SORT_WAVES x slice
    __shared__ int below_of[SORT_WAVES], sums[SORT_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64, tid = threadIdx.x;
    const int first = static_cast<int>(blockIdx.x) * slice, tokens = min(slice, g.vocab - first);
    const int begin = static_cast<int>(min(static_cast<std::int64_t>(wave) * wave_ids, g.count));
    const int end = static_cast<int>(min(static_cast<std::int64_t>(wave + 1) * wave_ids, g.count));
    int* const mine = counters + wave * slice;
    for (int i = lane; i < slice; i += 64) mine[i] = 0;
    wave_order();
    int below = 0;
    walk_ids(g, begin, end, [&](int id, int) {
        below += __popcll(__ballot(id >= 0 && id < first));
        const int local = id - first;
        const bool here = local >= 0 && local < tokens && id >= 0;
        for (unsigned long long left = __ballot(here); left;) {
            const int token = __builtin_amdgcn_readlane(local, __builtin_ctzll(left));
            const unsigned long long same = __ballot(here && local == token);
            if (lane == 0) mine[token] += __popcll(same);
            wave_order();
            left &= ~same;
        }
    });
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
    if (tid < tokens) starts[first + tid] = at;
    if (tid == tokens - 1 && first + tokens == g.vocab) starts[g.vocab] = at + total;
    if (tid < slice)
        for (int w = 0; w < SORT_WAVES; ++w) {
            const int held = counters[w * slice + tid];
            counters[w * slice + tid] = at;
            at += held;
        }
    __syncthreads();
    walk_ids(g, begin, end, [&](int id, int position) {
        const int local = id - first;
        const bool here = local >= 0 && local < tokens && id >= 0;
        for (unsigned long long left = __ballot(here); left;) {
            const int token = __builtin_amdgcn_readlane(local, __builtin_ctzll(left));
            const unsigned long long same = __ballot(here && local == token);
            const int to = mine[token];
            if (here && local == token)
                order[to + __builtin_amdgcn_mbcnt_hi(static_cast<unsigned>(same >> 32),
                                                     __builtin_amdgcn_mbcnt_lo(static_cast<unsigned>(same), 0u))] = position;
            wave_order();
            if (lane == 0) mine[token] = to + __popcll(same);
            wave_order();
            left &= ~same;
        }
    });
}

// ---- sums -------------------------------------------------------------------------------------
// A token that comes more often than SumPlan::chunk times is summed in pieces: the sorted positions lie in chunks
// of that many, and a chunk holds a piece of at most two such tokens, the one that it begins with and the one that
// it ends with. part_kernel sums the pieces, row_kernel a token's pieces, or the rows of any other token. Bound by
// HBM: each gradient row is read once, the table's gradient written once.
struct SumPlan {
    int chunk;       // positions of a piece
    int lanes;       // lanes (a power of two) that share a row's packs
    int columns;     // groups of `lanes` packs in a row
    int part_width;  // floats of a piece's row: whole packs
};

constexpr int IN_FLIGHT = 8;

// Adds the rows row(i), i = begin .. end - 1, of which each load gives a pack at this lane's columns.
template <typename P, int N, typename Row>
__device__ __forceinline__ void add_rows(float (&sum)[N], int begin, int end, Row&& row) {
    for (int i = begin; i < end; i += IN_FLIGHT) {
        P pack[IN_FLIGHT];
#pragma unroll
        for (int k = 0; k < IN_FLIGHT; ++k) pack[k] = row(min(i + k, end - 1));
#pragma unroll
        for (int k = 0; k < IN_FLIGHT; ++k) {
            if (i + k >= end) break;
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] += pack[k].at(e);
        }
    }
}

template <typename T, int N>
__device__ __forceinline__ void add_positions(float (&sum)[N], const T* __restrict__ grad, const EmbeddingGradient& g,
                                              const int* __restrict__ order, int begin, int end, int column) {
    const T* at = grad + column;
    if (column + N <= g.dim)
        add_rows<Pack<T, N>>(sum, begin, end, [&](int i) { return load_pack<T, N>(at + order[i] * g.grad_stride); });
    else
        add_rows<Pack<T, N>>(sum, begin, end, [&](int i) { return load_part<T, N>(at + order[i] * g.grad_stride, g.dim - column, 0.0f); });
}

template <typename T>
__global__ __launch_bounds__(THREADS) void part_kernel(const T* __restrict__ grad, EmbeddingGradient g, SumPlan plan,
                                                       const int* __restrict__ order, const int* __restrict__ starts,
                                                       float* __restrict__ parts) {
    constexpr int N = 16 / sizeof(T);
    const int given = starts[g.vocab];
    const int lane = threadIdx.x & 63, groups = 64 / plan.lanes;
    const std::int64_t chunks = (static_cast<std::int64_t>(given) + plan.chunk - 1) / plan.chunk, tasks = chunks * plan.columns;
    const std::int64_t waves = static_cast<std::int64_t>(gridDim.x) * (THREADS / 64) * groups;
    for (std::int64_t task = (static_cast<std::int64_t>(blockIdx.x) * (THREADS / 64) + threadIdx.x / 64) * groups + lane / plan.lanes;
         task < tasks; task += waves) {
        const int chunk = static_cast<int>(task / plan.columns);
        const int column = (static_cast<int>(task - static_cast<std::int64_t>(chunk) * plan.columns) * plan.lanes + lane % plan.lanes) * N;
        if (column >= g.dim) continue;
        const int begin = chunk * plan.chunk, end = min(begin + plan.chunk, given);
#pragma unroll 1
        for (int last = 0; last < 2; ++last) {
            const int token = static_cast<int>(whole_at(g.ids, g.ids_wide, order[last ? end - 1 : begin] * g.ids_step));
            const int from = starts[token], to = starts[token + 1];
            if (to - from <= plan.chunk || (last && from <= begin)) continue;
            float sum[N] = {};
            add_positions<T, N>(sum, grad, g, order, max(from, begin), min(to, end), column);
            float* out = parts + (2 * static_cast<std::int64_t>(chunk) + last) * plan.part_width + column;
#pragma unroll
            for (int e = 0; e < N; ++e) out[e] = sum[e];
        }
    }
}

template <typename T, typename Out>
__global__ __launch_bounds__(THREADS) void row_kernel(const T* __restrict__ grad, Out* __restrict__ out, EmbeddingGradient g,
                                                      SumPlan plan, const int* __restrict__ order,
                                                      const int* __restrict__ starts, const float* __restrict__ parts) {
    constexpr int N = 16 / sizeof(T);
    const int lane = threadIdx.x & 63, groups = 64 / plan.lanes;
    const std::int64_t tasks = static_cast<std::int64_t>(g.vocab) * plan.columns;
    const std::int64_t waves = static_cast<std::int64_t>(gridDim.x) * (THREADS / 64) * groups;
    for (std::int64_t task = (static_cast<std::int64_t>(blockIdx.x) * (THREADS / 64) + threadIdx.x / 64) * groups + lane / plan.lanes;
         task < tasks; task += waves) {
        const int token = static_cast<int>(task / plan.columns);
        const int column = (static_cast<int>(task - static_cast<std::int64_t>(token) * plan.columns) * plan.lanes + lane % plan.lanes) * N;
        if (column >= g.dim) continue;
        const int from = starts[token], to = starts[token + 1];
        if (from == to && g.add) continue;
        float sum[N] = {};
        if (to - from <= plan.chunk) {
            add_positions<T, N>(sum, grad, g, order, from, to, column);
        } else {
            // The first piece ends its chunk, unless it begins there; every further one begins its chunk.
            const int first = from / plan.chunk, last = (to - 1) / plan.chunk;
            add_rows<Pack<float, N>>(sum, first, last + 1, [&](int c) {
                const int slot = c == first && from != first * plan.chunk;
                return load_pack<float, N>(parts + (2 * static_cast<std::int64_t>(c) + slot) * plan.part_width + column);
            });
        }
        Out* to_row = out + token * g.out_stride + column;
        float v[N];
        if (g.add) {
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = column + e < g.dim ? static_cast<float>(to_row[e]) + sum[e] * g.scale : 0.0f;
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = sum[e] * g.scale;
        }
        if (column + N <= g.dim) {
            store_pack(to_row, Pack<Out, N>::of(v));
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (column + e < g.dim) to_row[e] = static_cast<Out>(v[e]);
        }
    }
}

// Pieces of 64 positions, longer ones for many positions: a piece and the join of all pieces of one token take
// about as many steps.
int chunk_of(std::int64_t count) {
    int chunk = 64;
    while (static_cast<std::int64_t>(chunk) * chunk * 8 < count) chunk *= 2;
    return chunk;
}

SumPlan sum_plan(const EmbeddingGradient& g, int type) {
    const int n = 16 / type_bytes(type), packs = (g.dim + n - 1) / n;
    SumPlan plan{chunk_of(g.count), 1, 1, packs * n};
    while (plan.lanes < 64 && plan.lanes < packs) plan.lanes *= 2;
    plan.columns = (packs + plan.lanes - 1) / plan.lanes;
    return plan;
}

unsigned wave_blocks(std::int64_t tasks, const SumPlan& plan) {
    const std::int64_t groups = 64 / plan.lanes * (THREADS / 64);
    return static_cast<unsigned>(std::min<std::int64_t>((tasks + groups - 1) / groups, BLOCKS_MAX));
}

std::int64_t aligned(std::int64_t bytes) { return (bytes + 255) / 256 * 256; }

std::int64_t parts_of(const EmbeddingGradient& g, const SumPlan& plan) {
    return g.count <= plan.chunk ? 0 : 2 * ((g.count + plan.chunk - 1) / plan.chunk);
}

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
    const SumPlan plan = sum_plan(g, type);
    return aligned(4 * g.count) + aligned(4 * (static_cast<std::int64_t>(g.vocab) + 1)) + 4 * parts_of(g, plan) * plan.part_width;
}

int launch_embedding_backward(const void* grad, int type, void* out, int out_type, const EmbeddingGradient& g,
                              void* workspace, hipStream_t stream) {
    const SumPlan plan = sum_plan(g, type);
    char* at = static_cast<char*>(workspace);
    int* order = reinterpret_cast<int*>(at);
    int* starts = reinterpret_cast<int*>(at + aligned(4 * g.count));
    float* parts = reinterpret_cast<float*>(at + aligned(4 * g.count) + aligned(4 * (static_cast<std::int64_t>(g.vocab) + 1)));
    // A slice of tokens for every workgroup that the GPU takes at once, at least one wave's width of them.
    int slice = 64;
    while (slice < SORT_THREADS && static_cast<std::int64_t>(slice) * device_cu_count() < g.vocab) slice *= 2;
    const std::int64_t wave_ids = ((g.count + SORT_WAVES - 1) / SORT_WAVES + 63) / 64 * 64;
    launch(sort_kernel, dim3(blocks_for(g.vocab, slice)), dim3(SORT_THREADS), sizeof(int) * SORT_WAVES * slice, stream, g, slice,
           static_cast<int>(wave_ids), order, starts);
    MFH_TRY(MFH_CHECK_LAUNCH("embedding sort", stream));
    return with_type(type, [&](auto element) {
        using T = decltype(element);
        const T* from = static_cast<const T*>(grad);
        if (parts_of(g, plan)) {
            launch(part_kernel<T>, dim3(wave_blocks(parts_of(g, plan) / 2 * plan.columns, plan)), dim3(THREADS), 0, stream, from, g,
                   plan, order, starts, parts);
            MFH_TRY(MFH_CHECK_LAUNCH("embedding parts", stream));
        }
        const dim3 grid(wave_blocks(static_cast<std::int64_t>(g.vocab) * plan.columns, plan));
        if (out_type == type)
            launch(row_kernel<T, T>, grid, dim3(THREADS), 0, stream, from, static_cast<T*>(out), g, plan, order, starts, parts);
        else
            launch(row_kernel<T, float>, grid, dim3(THREADS), 0, stream, from, static_cast<float*>(out), g, plan, order, starts,
                   parts);
        return MFH_CHECK_LAUNCH("embedding rows", stream);
    });
}

}  // namespace mfh
