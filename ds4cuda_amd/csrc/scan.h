// scan.h — sums over the lanes of a wave and the waves of a workgroup by lane moves
// (DPP), for 32- and 64-bit values. Shuffles through LDS take about 60 cycles a step and word, these
// a few.
#pragma once

#include "ds4hip_common.h"

namespace ds4hip {

template <int kCtrl, int kRowMask, typename T>
__device__ __forceinline__ T dpp_or_0(T v) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), kCtrl, kRowMask, 0xF, false));
    } else {
        uint2_t x = __builtin_bit_cast(uint2_t, v);
        x[0] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x[0], kCtrl, kRowMask, 0xF, false);
        x[1] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x[1], kCtrl, kRowMask, 0xF, false);
        return __builtin_bit_cast(T, x);
    }
}

// Inclusive sum over the wave's lanes: in rows of 16, then the last lanes of the rows before.
template <typename T>
__device__ __forceinline__ T wave_scan(T x) {
    x += dpp_or_0<0x111, 0xF>(x);   // the lane 1, 2, 4, 8 before
    x += dpp_or_0<0x112, 0xF>(x);
    x += dpp_or_0<0x114, 0xF>(x);
    x += dpp_or_0<0x118, 0xF>(x);
    x += dpp_or_0<0x142, 0xA>(x);   // lane 15 of the row before, to rows 1 and 3
    x += dpp_or_0<0x143, 0xC>(x);   // lane 31, to rows 2 and 3
    return x;
}

template <typename T>
__device__ __forceinline__ T lane_of(T v, int lane) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
    } else {
        uint2_t x = __builtin_bit_cast(uint2_t, v);
        x[0] = (uint32_t)__builtin_amdgcn_readlane((int)x[0], lane);
        x[1] = (uint32_t)__builtin_amdgcn_readlane((int)x[1], lane);
        return __builtin_bit_cast(T, x);
    }
}

// Inclusive sum over the workgroup's kWaves waves, in their order; *total: of all. sums [kWaves] in LDS. (Every wave sums
// the waves' sums in its own lanes: with each thread adding up sixteen of them, a sum took half a microsecond.)
template <int kWaves, typename T>
__device__ __forceinline__ T wg_scan(T v, T *sums, T *total) {
    static_assert(kWaves <= 16 && (kWaves & (kWaves - 1)) == 0, "the waves' sums lie in a row of lanes");
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const T x = wave_scan(v);
    __syncthreads();   // (the sums before are read)
    if (lane == 63) sums[w] = x;
    __syncthreads();
    T y = sums[lane & (kWaves - 1)];
    if (kWaves > 1) y += dpp_or_0<0x111, 0xF>(y);
    if (kWaves > 2) y += dpp_or_0<0x112, 0xF>(y);
    if (kWaves > 4) y += dpp_or_0<0x114, 0xF>(y);
    if (kWaves > 8) y += dpp_or_0<0x118, 0xF>(y);
    *total = lane_of(y, kWaves - 1);
    return w ? lane_of(y, w - 1) + x : x;
}

}  // namespace ds4hip
