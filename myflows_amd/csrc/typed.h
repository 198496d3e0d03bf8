// Element types of the kernels that take more than float32: the type codes of the C ABI, conversion to
// and from float, and 16-byte packs of elements at any element's address.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

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

// N elements that one load or store moves. The address need only be aligned to one element: global memory
// takes 16-byte accesses at any address.
template <typename T, int N>
struct Pack {
    T v[N];
    __device__ __forceinline__ float at(int i) const { return static_cast<float>(v[i]); }
    __device__ __forceinline__ void set(int i, float x) { v[i] = static_cast<T>(x); }
};

template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
    Pack<T, N> pack;
    __builtin_memcpy(&pack, p, sizeof(pack));
    return pack;
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
