// Logits adjusted before they are answered with. Of a row z with a history of tokens, a prompt and behind it an
// answer, with s whether a token is in the history and n its count in the answer:
//   u = z, or where s: z / repetition for z > 0 and z repetition else
//   out = (u - frequency n) - presence [n > 0] + bias, -inf where the mask has no bit
// in float32, rounded once to the logits' type. Equal ids of a row's biases add up in their order.
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "common.h"
#include "typed.h"

namespace mfh {
namespace {

// A workgroup walks some of a row's chunks, PACKS packs of 16 bytes a thread each, the next chunk's loads in flight.
// Its threads hold the row's history in registers (what is beyond HISTORY tokens a thread they read again each
// time) and count in a word of LDS for each logit of the chunk; then each pack is adjusted (by its words, if any is
// not 0), masked by its own bits and stored. The logits are read and written once, no store waits for another, and
// the history is read once a workgroup. Bound by HBM: 512 rows of 131072 float16 with 4096 tokens, 16 biases and a mask
// 72 us (3.9 TB/s; 43 us without any of them, 50 with the mask alone); the difference is the words' LDS traffic and
// the barriers around them. In place, only the packs that change are read and written.
constexpr unsigned SEEN = 1u << 31;      // in the prompt
constexpr int SLOT_SHIFT = 20;           // bits 20 to 30: 1 + the first of the row's biases of this id
constexpr unsigned COUNT = (1u << SLOT_SHIFT) - 1;  // in the answer
static_assert(ADJUST_HELD_LIMIT == static_cast<int>(COUNT) && ADJUST_BIAS_MAX < 1 << (31 - SLOT_SHIFT), "fields of a word");

constexpr unsigned SLOTS = (1u << (31 - SLOT_SHIFT)) - 1;

constexpr int HISTORY = 8;
constexpr int PROMPT = 1 << 30, TOKEN = PROMPT - 1;  // of a token held in a register; -1 is none
static_assert(LOGIT_VOCAB_LIMIT < TOKEN, "none lies beyond the vocabulary");

// The row's biases: their ids, values, and for the first of each id the id again (else -1) and the sum of its values.
struct RowBiases {
    int* ids;
    float* values;
    int* leads;
    float* sums;
};

template <int THREADS>
__device__ __forceinline__ void read_biases(const RowBiases& b, const AdjustLogits& a, int row, int padded) {
    for (int i = threadIdx.x; i < padded; i += THREADS) {
        const long long id = i < a.biases ? whole_at(a.bias_ids, a.bias_wide, row * a.bias_step + i) : -1;
        b.ids[i] = id >= 0 && id < a.vocab ? static_cast<int>(id) : -1;
        b.values[i] = i < a.biases ? a.bias_values[row * a.bias_values_step + i] : 0.0f;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.biases; i += THREADS) {
        const int id = b.ids[i];
        bool leads = id >= 0;
        float sum = 0.0f;
        for (int j = 0; leads && j < padded; j += 4) {
            const int4 other = *reinterpret_cast<const int4*>(b.ids + j);
            const int found[4] = {other.x, other.y, other.z, other.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (found[k] != id) continue;
                leads = leads && j + k >= i;
                sum += b.values[j + k];
            }
        }
        b.leads[i] = leads ? id : -1;
        b.sums[i] = sum;
    }
}

// Element i of a pack, and a value rounded into its place, for an i that each lane has of its own. The words stay in
// registers: the compiler, left to itself, indexes them in memory.
template <typename Word>
__device__ __forceinline__ Word held(Word word) {
    asm volatile("" : "+v"(word));
    return word;
}
template <typename T, int N>
__device__ __forceinline__ float element_of(const Pack<T, N>& pack, int i) {
    constexpr int SHARE = Pack<T, N>::PAIRS ? 2 : 1;
    auto w = held(pack.w[0]);
#pragma unroll
    for (int k = 1; k < Pack<T, N>::WORDS; ++k) {
        const auto other = held(pack.w[k]);
        w = i / SHARE == k ? other : w;
    }
    if constexpr (Pack<T, N>::PAIRS) return Pack<T, 2>{{i & 1 ? w >> 16 : w}}.at(0);
    else return w;
}
template <typename T, int N>
__device__ __forceinline__ void set_element(Pack<T, N>& pack, int i, float value) {
    if constexpr (Pack<T, N>::PAIRS) {
        const unsigned half = __builtin_bit_cast(unsigned short, static_cast<T>(value));
        const unsigned shifted = i & 1 ? half << 16 : half, keep = i & 1 ? 0xffffu : 0xffff0000u;
#pragma unroll
        for (int k = 0; k < Pack<T, N>::WORDS; ++k) pack.w[k] = held(i / 2 == k ? (pack.w[k] & keep) | shifted : pack.w[k]);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) pack.w[k] = held(i == k ? value : pack.w[k]);
    }
}

// -inf at the elements without their bit.
template <typename T, int N>
__device__ __forceinline__ void rule_out(Pack<T, N>& pack, unsigned bits) {
    const Pack<T, N> none = Pack<T, N>::all(-INFINITY);
#pragma unroll
    for (int k = 0; k < Pack<T, N>::WORDS; ++k) {
        if constexpr (Pack<T, N>::PAIRS) {
            const unsigned low = 0u - (bits >> 2 * k & 1), high = 0u - (bits >> (2 * k + 1) & 1);
            const unsigned keep = (low & 0xffffu) | (high & 0xffff0000u);
            pack.w[k] = (pack.w[k] & keep) | (none.w[k] & ~keep);
        } else {
            pack.w[k] = bits >> k & 1 ? pack.w[k] : none.w[k];
        }
    }
}

template <typename T, typename Whole, int THREADS, int PACKS>
__global__ __launch_bounds__(THREADS) void adjust_kernel(const T* __restrict__ logits, T* out, AdjustLogits a, FastDiv groups,
                                                         int group_chunks, int items, bool in_place) {
    constexpr int N = 16 / sizeof(T), CHUNK = THREADS * PACKS * N;
    constexpr unsigned ALL = (1u << N) - 1;
    extern __shared__ unsigned words[];  // CHUNK, where the row has tokens or biases; then the biases
    const int padded = (a.biases + 3) / 4 * 4, tid = threadIdx.x;
    const RowBiases biases{reinterpret_cast<int*>(words + CHUNK), reinterpret_cast<float*>(words + CHUNK + padded),
                           reinterpret_cast<int*>(words + CHUNK + 2 * padded), reinterpret_cast<float*>(words + CHUNK + 3 * padded)};
    const bool counts = a.held > 0 || a.biases > 0;
    if (counts)  // a thread clears its own words again when it has read them
        for (int i = tid * 4; i < CHUNK; i += THREADS * 4) *reinterpret_cast<uint4*>(words + i) = make_uint4(0, 0, 0, 0);
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
        int group;
        const int row = groups.divmod(item, group);
        const int begin = group * group_chunks * CHUNK, end = min(begin + group_chunks * CHUNK, a.vocab);
        const T* z = logits + row * a.stride;
        const unsigned* allowed = a.allowed ? a.allowed + row * a.allowed_step : nullptr;
        const long long prompt = a.prompt_lengths ? whole_at(a.prompt_lengths, a.prompt_wide, row * a.prompt_step) : 0;
        const float repetition = a.repetition ? a.repetition[row * a.repetition_step] : a.repetition_all;
        const float presence = a.presence ? a.presence[row * a.presence_step] : a.presence_all;
        const float frequency = a.frequency ? a.frequency[row * a.frequency_step] : a.frequency_all;
        const Whole* history = static_cast<const Whole*>(a.tokens) + row * a.tokens_step;
        const auto token_at = [&](int i) {
            if (i >= a.held) return -1;
            using Unsigned = std::make_unsigned_t<Whole>;
            const Whole token = history[i];
            if (static_cast<Unsigned>(token) >= static_cast<Unsigned>(a.vocab)) return -1;
            return static_cast<int>(token) | (i < prompt ? PROMPT : 0);
        };
        int tokens[HISTORY];
#pragma unroll
        for (int k = 0; k < HISTORY; ++k) tokens[k] = token_at(tid + k * THREADS);
        Pack<T, N> next[PACKS];
        unsigned next_bits[PACKS];  // whole words, so that nothing waits for them here
        const auto load = [&](int at) {
            return at + N <= end ? load_pack<T, N>(z + at) : load_part<T, N>(z + at, end - at, 0.0f);
        };
        const auto prefetch = [&](int first) {
#pragma unroll
            for (int p = 0; p < PACKS; ++p) {
                const int at = first + (p * THREADS + tid) * N;
                next_bits[p] = ~0u;
                if (at >= end) continue;
                if (!in_place) next[p] = load(at);
                if (allowed) next_bits[p] = allowed[at / 32];
            }
        };
        prefetch(begin);
        if (a.biases) read_biases<THREADS>(biases, a, row, padded);
        __syncthreads();
#pragma unroll 1
        for (int first = begin; first < end; first += CHUNK) {
            const int here = min(CHUNK, end - first);
            if (counts) {
                const auto count = [&](int token) {
                    const int at = (token & TOKEN) - first;
                    if (at < 0 || at >= here) return;
                    if (token & PROMPT) atomicOr(&words[at], SEEN);
                    else atomicAdd(&words[at], 1u);
                };
#pragma unroll
                for (int k = 0; k < HISTORY; ++k) count(tokens[k]);
                for (int i = tid + HISTORY * THREADS; i < a.held; i += HISTORY * THREADS) {
                    int more[HISTORY];
#pragma unroll
                    for (int k = 0; k < HISTORY; ++k) more[k] = token_at(i + k * THREADS);
#pragma unroll
                    for (int k = 0; k < HISTORY; ++k) count(more[k]);
                }
                for (int i = tid; i < a.biases; i += THREADS) {
                    const int at = biases.leads[i] - first;
                    if (at >= 0 && at < here) atomicOr(&words[at], static_cast<unsigned>(i + 1) << SLOT_SHIFT);
                }
                __syncthreads();
            }
            Pack<T, N> packs[PACKS];
            unsigned bits[PACKS];
#pragma unroll
            for (int p = 0; p < PACKS; ++p) packs[p] = next[p], bits[p] = next_bits[p] >> (first + (p * THREADS + tid) * N) % 32 & ALL;
            if (first + CHUNK < end) prefetch(first + CHUNK);
#pragma unroll
            for (int p = 0; p < PACKS; ++p) {
                const int within = (p * THREADS + tid) * N, at = first + within;
                if (at >= end) continue;
                unsigned named = 0;
                if (counts) {
#pragma unroll
                    for (int i = 0; i < N; i += 4) {
                        const uint4 four = *reinterpret_cast<const uint4*>(words + within + i);
                        named |= (four.x ? 1u << i : 0) | (four.y ? 2u << i : 0) | (four.z ? 4u << i : 0) | (four.w ? 8u << i : 0);
                    }
                }
                if (in_place) {
                    if (!named && bits[p] == ALL) continue;
                    if (bits[p]) packs[p] = load(at);
                }
                // A lane's few logits that the history or a bias names, one after the other.
                for (unsigned left = named; left; left &= left - 1) {
#pragma clang fp contract(off)
                    const int i = __builtin_ctz(left);
                    const unsigned word = words[within + i], n = word & COUNT, slot = word >> SLOT_SHIFT & SLOTS;
                    float u = element_of(packs[p], i);
                    if (n || word & SEEN) u = u > 0.0f ? u / repetition : u * repetition;
                    if (n) u = (u - frequency * static_cast<float>(n)) - presence;
                    if (slot) u += biases.sums[slot - 1];
                    set_element(packs[p], i, u);
                    words[within + i] = 0;
                }
                if (bits[p] != ALL) rule_out(packs[p], bits[p]);
                T* to = out + row * a.out_stride + at;
                if (at + N <= end) {
                    store_pack(to, packs[p]);
                } else {
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (at + i < end) to[i] = static_cast<T>(packs[p].at(i));
                }
            }
            if (counts) __syncthreads();
        }
    }
}

constexpr int ITEMS_MAX = 1 << 22;  // workgroups of a launch; they walk on from there

template <typename T, int THREADS, int PACKS>
int launch_adjust_as(const T* logits, T* out, const AdjustLogits& a, hipStream_t stream) {
    constexpr int CHUNK = THREADS * PACKS * (16 / sizeof(T));
    // The chunks of a workgroup: those of the fewest steps, where the GPU takes `slots` workgroups at once and one's
    // start costs about as much as a chunk (512 rows of 131072 float16: 72 us with whole rows, 79 with half ones;
    // 333 rows of 32771 float32, five chunks: 28 us with whole rows, 40 with three chunks, 31 with two).
    const int chunks = (a.vocab + CHUNK - 1) / CHUNK;
    const std::int64_t slots = static_cast<std::int64_t>(device_cu_count()) * (THREADS > 256 ? 2 : 6);
    int group_chunks = chunks;
    const auto steps = [&](int each) { return (a.rows * ((chunks + each - 1) / each) + slots - 1) / slots * (each + 1); };
    for (int each = std::min(chunks, 32); each > 0; --each)
        if (steps(each) < steps(group_chunks)) group_chunks = each;
    const int groups = (chunks + group_chunks - 1) / group_chunks;
    const std::int64_t items = a.rows * groups;
    MFH_REQUIRE(items <= INDEX_LIMIT, "too many logits for one call");
    const std::size_t shared =
        a.held > 0 || a.biases > 0 ? 4 * static_cast<std::size_t>(CHUNK + 4 * ((a.biases + 3) / 4 * 4)) : 0;
    launch(a.tokens_wide ? adjust_kernel<T, long long, THREADS, PACKS> : adjust_kernel<T, int, THREADS, PACKS>,
           dim3(static_cast<unsigned>(std::min<std::int64_t>(items, ITEMS_MAX))), dim3(THREADS), shared, stream, logits, out, a,
           FastDiv(groups), group_chunks, static_cast<int>(items), static_cast<const T*>(out) == logits);
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
