// Reductions over the 64 lanes of a wave, in a fixed order: four cross-lane steps within each row of 16 lanes
// (quad permutes and mirrors, no LDS), then the four rows through scalar registers. Every lane gets the result.
#pragma once

#include <hip/hip_runtime.h>

namespace mfh {

template <int CONTROL>
__device__ __forceinline__ float lane_moved(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CONTROL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_of(float v, int lane) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}

template <typename Op>
__device__ __forceinline__ float wave_reduce(float v, Op op) {
    v = op(v, lane_moved<0xB1>(v));   // lanes 1, 0, 3, 2 of each quad
    v = op(v, lane_moved<0x4E>(v));   // lanes 2, 3, 0, 1
    v = op(v, lane_moved<0x141>(v));  // the mirrored half row
    v = op(v, lane_moved<0x140>(v));  // the mirrored row
    return op(op(lane_of(v, 0), lane_of(v, 16)), op(lane_of(v, 32), lane_of(v, 48)));
}
__device__ __forceinline__ float wave_sum(float v) {
    return wave_reduce(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float wave_max(float v) {
    return wave_reduce(v, [](float a, float b) { return fmaxf(a, b); });
}

}  // namespace mfh
