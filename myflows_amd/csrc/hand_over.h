// Values handed from workgroup to workgroup within a launch.
#pragma once

#include <hip/hip_runtime.h>

namespace mfh {

// Values that workgroups hand to one another within a launch. A fence over the whole GPU writes back and drops an
// XCD's cache, which took 200 us for a thousand workgroups; instead these values (a row's statistics, the sums of a
// split tile) are written through to the memory that all XCDs share, and read from there, as relaxed atomics of that scope. That a written-through value has
// reached that memory once s_waitcnt has counted its store is how gfx950 works; the language's memory model, which knows
// fences only, does not promise it.
template <typename V>
__device__ __forceinline__ void hand_over(V* to, V value) {
    __hip_atomic_store(to, value, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename V>
__device__ __forceinline__ V handed_over(const V* from) {
    return __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

}  // namespace mfh
