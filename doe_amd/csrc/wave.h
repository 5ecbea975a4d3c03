// wave.h -- small exchanges within a wave of 64 lanes.
#pragma once

#include <hip/hip_runtime.h>

namespace doe {

// Inclusive sum over the wave's lanes, in registers.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_scan(int v) {
    v = dpp_add<0x111, 0xf>(v);  // one lane further within sixteen, two, four, eight
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);     // the last lane of a sixteen to the next (rows 1 and 3)
    return dpp_add<0x143, 0xc>(v);  // lane 31 to rows 2 and 3
}

}  // namespace doe
