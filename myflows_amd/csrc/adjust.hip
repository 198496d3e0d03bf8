// Logits adjusted before they are answered with. Of a row z with a history of tokens, a prompt and behind it an
// answer, with s whether a token is in the history and n its count in the answer:
//   u = z, or where s: z / repetition for z > 0 and z repetition else
//   out = (u - frequency n) - presence [n > 0] + bias, -inf where the mask has no bit
// in float32, rounded once to the logits' type. Equal ids of a row's biases add up in their order.
#include <algorithm>
#include <cstdint>

#include "common.h"
#include "typed.h"

namespace mfh {
namespace {

// A workgroup owns a chunk of a row: PACKS packs of 16 bytes a thread, loaded first of all, and a word of LDS for each
// of its logits. Its threads read the row's whole history and count in the words what lies in the chunk; then each
// pack is adjusted (by its words, if any is not 0), masked by its own bits and stored. The logits are read and
// written once, and no store waits for another. Bound by HBM; the history costs its length a chunk, from L2.
// In place, only the packs that change are read and written.
constexpr unsigned SEEN = 1u << 31;      // in the prompt
constexpr int SLOT_SHIFT = 20;           // bits 20 to 30: 1 + the first of the row's biases of this id
constexpr unsigned COUNT = (1u << SLOT_SHIFT) - 1;  // in the answer
static_assert(ADJUST_HELD_LIMIT == static_cast<int>(COUNT) && ADJUST_BIAS_MAX < 1 << (31 - SLOT_SHIFT), "fields of a word");

constexpr int HISTORY_AHEAD = 8;

template <typename T, typename Whole, int THREADS, int PACKS>
__global__ __launch_bounds__(THREADS) void adjust_kernel(const T* __restrict__ logits, T* out, AdjustLogits a, FastDiv chunks,
                                                         int items, bool in_place) {
    constexpr int N = 16 / sizeof(T), CHUNK = THREADS * PACKS * N;
    extern __shared__ unsigned words[];  // CHUNK, where the row has tokens or biases; then the biases
    int* const bias_ids = reinterpret_cast<int*>(words + CHUNK);
    float* const bias_values = reinterpret_cast<float*>(bias_ids + a.biases);
    float* const bias_sums = bias_values + a.biases;
    const int tid = threadIdx.x;
    const bool counts = a.held > 0 || a.biases > 0;
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
        int chunk;
        const int row = chunks.divmod(item, chunk);
        const int first = chunk * CHUNK, here = min(CHUNK, a.vocab - first);
        const T* from = logits + row * a.stride + first;
        T* to = out + row * a.out_stride + first;
        // Every load that depends on no other goes out first, the history's ahead of the logits'.
        const long long prompt = a.prompt_lengths ? whole_at(a.prompt_lengths, a.prompt_wide, row * a.prompt_step) : 0;
        const float repetition = a.repetition ? a.repetition[row * a.repetition_step] : a.repetition_all;
        const float presence = a.presence ? a.presence[row * a.presence_step] : a.presence_all;
        const float frequency = a.frequency ? a.frequency[row * a.frequency_step] : a.frequency_all;
        const Whole* history = static_cast<const Whole*>(a.tokens) + row * a.tokens_step;
        Whole token[HISTORY_AHEAD];
        const auto read_history = [&](int base) {
#pragma unroll
            for (int k = 0; k < HISTORY_AHEAD; ++k) token[k] = base + k * THREADS < a.held ? history[base + k * THREADS] : -1;
        };
        read_history(tid);
        Pack<T, N> packs[PACKS];
        unsigned bits[PACKS];
        const auto load = [&](int at) {
            return at + N <= here ? load_pack<T, N>(from + at) : load_part<T, N>(from + at, here - at, 0.0f);
        };
#pragma unroll
        for (int p = 0; p < PACKS; ++p) {
            const int at = (p * THREADS + tid) * N;
            bits[p] = (1u << N) - 1;
            if (at >= here) continue;
            if (!in_place) packs[p] = load(at);
            if (a.allowed) bits[p] = a.allowed[row * a.allowed_step + (first + at) / 32] >> (first + at) % 32 & ((1u << N) - 1);
        }
        if (counts) {
            for (int i = tid * 4; i < CHUNK; i += THREADS * 4) *reinterpret_cast<uint4*>(words + i) = make_uint4(0, 0, 0, 0);
            for (int i = tid; i < a.biases; i += THREADS) {
                const long long id = whole_at(a.bias_ids, a.bias_wide, row * a.bias_step + i) - first;
                bias_ids[i] = id >= 0 && id < here ? static_cast<int>(id) : -1;
                bias_values[i] = a.bias_values[row * a.bias_values_step + i];
            }
            __syncthreads();
            for (int base = tid;;) {
#pragma unroll
                for (int k = 0; k < HISTORY_AHEAD; ++k) {
                    const Whole at = token[k] - first;
                    if (token[k] < first || at >= here) continue;
                    if (base + k * THREADS < prompt) atomicOr(&words[at], SEEN);
                    else atomicAdd(&words[at], 1u);
                }
                base += THREADS * HISTORY_AHEAD;
                if (base >= a.held) break;
                read_history(base);
            }
            // The first of a row's biases of an id sums them all.
            for (int i = tid; i < a.biases; i += THREADS) {
                const int id = bias_ids[i];
                if (id < 0) continue;
                bool leads = true;
                for (int j = 0; j < i; ++j) leads = leads && bias_ids[j] != id;
                if (!leads) continue;
                float sum = bias_values[i];
                for (int j = i + 1; j < a.biases; ++j) sum += bias_ids[j] == id ? bias_values[j] : 0.0f;
                bias_sums[i] = sum;
                atomicOr(&words[id], static_cast<unsigned>(i + 1) << SLOT_SHIFT);
            }
            __syncthreads();
        }
#pragma unroll
        for (int p = 0; p < PACKS; ++p) {
            const int at = (p * THREADS + tid) * N;
            if (at >= here) continue;
            unsigned word[N] = {}, any = 0;
            if (counts) {
#pragma unroll
                for (int i = 0; i < N; ++i) any |= word[i] = words[at + i];
            }
            const unsigned all = (1u << N) - 1;
            if (in_place) {
                if (!any && bits[p] == all) continue;
                if (bits[p]) packs[p] = load(at);
            }
            if (any || bits[p] != all) {
                float v[N];
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    float u = packs[p].at(i);
                    if (word[i]) {
#pragma clang fp contract(off)
                        const unsigned count = word[i] & COUNT, slot = word[i] >> SLOT_SHIFT & ((1u << (31 - SLOT_SHIFT)) - 1);
                        if (count || word[i] & SEEN) u = u > 0.0f ? u / repetition : u * repetition;
                        if (count) u = (u - frequency * static_cast<float>(count)) - presence;
                        if (slot) u += bias_sums[slot - 1];
                    }
                    v[i] = bits[p] >> i & 1 ? u : -INFINITY;
                }
                packs[p] = Pack<T, N>::of(v);
            }
            if (at + N <= here) {
                store_pack(to + at, packs[p]);
            } else {
                for (int i = 0; i < here - at; ++i) to[at + i] = static_cast<T>(packs[p].at(i));
            }
        }
        __syncthreads();  // the words are cleared for the next chunk
    }
}

constexpr int ITEMS_MAX = 1 << 22;  // workgroups of a launch; they walk on from there

template <typename T, int THREADS, int PACKS>
int launch_adjust_as(const T* logits, T* out, const AdjustLogits& a, hipStream_t stream) {
    constexpr int CHUNK = THREADS * PACKS * (16 / sizeof(T));
    const int chunks = (a.vocab + CHUNK - 1) / CHUNK;
    const std::int64_t items = a.rows * chunks;
    MFH_REQUIRE(items <= INDEX_LIMIT, "too many logits for one call");
    const std::size_t shared = a.held > 0 || a.biases > 0 ? 4 * static_cast<std::size_t>(CHUNK + 3 * a.biases) : 0;
    launch(a.tokens_wide ? adjust_kernel<T, long long, THREADS, PACKS> : adjust_kernel<T, int, THREADS, PACKS>, dim3(static_cast<unsigned>(std::min<std::int64_t>(items, ITEMS_MAX))), dim3(THREADS),
           shared, stream, logits, out, a, FastDiv(chunks), static_cast<int>(items), static_cast<const T*>(out) == logits);
    return MFH_CHECK_LAUNCH("adjusted logits", stream);
}

}  // namespace

int launch_adjust(const void* logits, void* out, int type, const AdjustLogits& a, hipStream_t stream) {
    if (a.rows == 0) return OK;
    return with_type(type, [&](auto element) {
        using T = decltype(element);
        const T* from = static_cast<const T*>(logits);
        T* to = static_cast<T*>(out);
        // Long chunks read the history seldom; short ones where long ones leave CUs idle.
        constexpr int LONG = 512 * 4 * (16 / sizeof(T)), SHORT = 256 * (16 / sizeof(T));
        if (a.vocab <= SHORT || a.rows * ((a.vocab + LONG - 1) / LONG) < 2 * device_cu_count())
            return launch_adjust_as<T, 256, 1>(from, to, a, stream);
        return launch_adjust_as<T, 512, 4>(from, to, a, stream);
    });
}

}  // namespace mfh
