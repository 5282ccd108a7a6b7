// lanes.hpp — exchanges between the lanes of a wave that stay out of LDS.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace comet {

// the value of lane ^ X
template <int X> __device__ __forceinline__ uint32_t xor_lane(uint32_t v) {
    auto dpp = [](uint32_t x, auto ctrl) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, decltype(ctrl)::value, 0xF, 0xF, true); };
    if constexpr (X == 1) return dpp(v, std::integral_constant<int, 0xB1>{});                                                            // quads: 1 0 3 2
    else if constexpr (X == 2) return dpp(v, std::integral_constant<int, 0x4E>{});                                                       // quads: 2 3 0 1
    else if constexpr (X == 4) return dpp(dpp(v, std::integral_constant<int, 0x141>{}), std::integral_constant<int, 0x1B>{});            // eights mirrored, then quads
    else if constexpr (X == 8) return dpp(v, std::integral_constant<int, 0x128>{});                                                      // sixteens turned by eight
    else {
        const auto r = X == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return (threadIdx.x & X) ? r[0] : r[1];
    }
}

}  // namespace comet
