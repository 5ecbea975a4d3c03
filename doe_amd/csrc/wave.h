// wave.h -- small exchanges within a wave of 64 lanes.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace doe {

// v and what the lane that CTRL names holds of it (0 where there is none, and in the rows of
// sixteen lanes that ROWS leaves out).
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, ROWS, 0xf, true));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, ROWS, 0xf, true);
    return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// Inclusive sums in registers: over each sixteen lanes, and over the wave.
__device__ __forceinline__ int scan16(int v) {
    v = dpp_add<0x111, 0xf>(v);  // one lane further within sixteen, two, four, eight
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    return dpp_add<0x118, 0xf>(v);
}
__device__ __forceinline__ int wave_scan(int v) {
    v = dpp_add<0x142, 0xa>(scan16(v));  // the last lane of a sixteen to the next (rows 1 and 3)
    return dpp_add<0x143, 0xc>(v);       // lane 31 to rows 2 and 3
}

// The sum over the wave (float, double), in lane 63, and in every lane.
template <typename T>
__device__ __forceinline__ T wave_sum_last(T v) {
    v = dpp_add<0x4E, 0xf>(dpp_add<0xB1, 0xf>(v));    // the neighbour, the other pair
    v = dpp_add<0x140, 0xf>(dpp_add<0x141, 0xf>(v));  // the other four, the other eight
    return dpp_add<0x143, 0xc>(dpp_add<0x142, 0xa>(v));
}
__device__ __forceinline__ float wave_sum(float v) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(wave_sum_last(v)), 63));
}
__device__ __forceinline__ double wave_sum(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, wave_sum_last(v));
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, 63), hi = (uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), 63);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

}  // namespace doe
