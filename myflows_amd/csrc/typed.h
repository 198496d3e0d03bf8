// Element types of the kernels that take more than float32: the type codes of the C ABI, conversion to
// and from float, and 16-byte packs of elements at any element's address.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace mfh {

constexpr int TYPE_F32 = 0, TYPE_BF16 = 1, TYPE_F16 = 2;

inline bool type_valid(int type) { return type >= TYPE_F32 && type <= TYPE_F16; }
inline int type_bytes(int type) { return type == TYPE_F32 ? 4 : 2; }

// Calls f with a value of the element type that `type` names.
template <typename F>
auto with_type(int type, F&& f) {
    if (type == TYPE_BF16) return f(__bf16{});
    if (type == TYPE_F16) return f(_Float16{});
    return f(float{});
}

// N elements that one load or store moves, half types two to a word. The address need only be aligned to one
// element: global memory takes 16-byte accesses at any address.
template <typename T, int N>
struct Pack {
    static constexpr bool PAIRS = sizeof(T) == 2 && N > 1;
    static constexpr int WORDS = PAIRS ? N / 2 : N;
    using Word = std::conditional_t<PAIRS, unsigned, T>;
    Word w[WORDS];

    __device__ __forceinline__ float at(int i) const {
        if constexpr (!PAIRS) {
            return static_cast<float>(w[i]);
        } else if constexpr (std::is_same_v<T, __bf16>) {
            return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        } else {
            return static_cast<float>(__builtin_bit_cast(T, static_cast<unsigned short>(i & 1 ? w[i / 2] >> 16 : w[i / 2])));
        }
    }
    // The floats rounded to the type.
    static __device__ __forceinline__ Pack of(const float (&x)[N]) {
        Pack pack;
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
            if constexpr (PAIRS) {
                typedef T Pair __attribute__((ext_vector_type(2)));
                pack.w[i] = __builtin_bit_cast(unsigned, Pair{static_cast<T>(x[2 * i]), static_cast<T>(x[2 * i + 1])});
            } else {
                pack.w[i] = static_cast<T>(x[i]);
            }
        }
        return pack;
    }
    static __device__ __forceinline__ Pack all(float x) {
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = x;
        return of(v);
    }
    // Between two passes over held packs: keeps the compiler from holding the first pass's floats of half types
    // for the second, at twice the registers.
    __device__ __forceinline__ void stay_packed() {
        if constexpr (PAIRS) {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) asm volatile("" : "+v"(w[i]));
        }
    }
};

template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
    Pack<T, N> pack;
    __builtin_memcpy(&pack, p, sizeof(pack));
    return pack;
}

// The pack at p of which `count` elements (fewer than N, or none) are there; `rest` beyond them.
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_part(const T* p, int count, float rest) {
    float x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = i < count ? static_cast<float>(p[i]) : rest;
    return Pack<T, N>::of(x);
}

template <typename T, int N>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& pack) {
    __builtin_memcpy(p, &pack, sizeof(pack));
}

// Element i of an array of whole numbers that holds int32 or int64.
__device__ __forceinline__ long long whole_at(const void* p, int wide, long long i) {
    return wide ? static_cast<const long long*>(p)[i] : static_cast<long long>(static_cast<const int*>(p)[i]);
}

}  // namespace mfh
