// Sums and maxima over L neighbouring lanes of a wave (8 to 64), the same value in every one of them, by vector instructions alone: within 16
// lanes a lane reads another one's register as an operand, across them rows of 16 and halves of 32 change places.  (By LDS permutes a step costs an
// LDS round trip, about 100 cycles; here it is 4 to 12.)
#pragma once
#include "common.h"

namespace xrl {

template <int CTRL>
__device__ __forceinline__ float lane_dpp(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true)); }

template <int L, typename OP>
__device__ __forceinline__ float lane_all(float v, OP op) {
    v = op(v, lane_dpp<0xb1>(v));                                // lanes 1 0 3 2
    v = op(v, lane_dpp<0x4e>(v));                                // lanes 2 3 0 1
    v = op(v, lane_dpp<0x141>(v));                               // eight lanes backwards: the other four hold one value by now
    if (L > 8) v = op(v, lane_dpp<0x140>(v));                    // sixteen backwards
    if (L > 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    if (L > 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    return v;
}
template <int L>
__device__ __forceinline__ float lane_sum(float v) { return lane_all<L>(v, [](float a, float b) { return a + b; }); }
// a NaN reaches the result, which fmaxf would pass over
__device__ __forceinline__ float nan_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }
template <int L>
__device__ __forceinline__ float lane_max(float v) { return lane_all<L>(v, [](float a, float b) { return nan_max(a, b); }); }

}  // namespace xrl
