// Exchanges between neighbouring lanes.
#ifndef VECOPS_HIP_LANE_EXCHANGE_H
#define VECOPS_HIP_LANE_EXCHANGE_H

#include "tile_gemm.h"

namespace vecops_hip {

constexpr int kNextLane = 0xb1, kNextButOne = 0x4e;   // moves within four lanes: 0 <-> 1, 2 <-> 3; 0 <-> 2, 1 <-> 3

// Of each pair of lanes that MOVE names, the first one's `b` and the second one's `a` change places.
template <int MOVE>
__device__ __forceinline__ void exchange_lanes(u32x4& a, u32x4& b, bool second) {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const uint32_t from_b = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0u, b[d], MOVE, 0xf, 0xf, true));
    const uint32_t from_a = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0u, a[d], MOVE, 0xf, 0xf, true));
    a[d] = second ? from_b : a[d];
    b[d] = second ? b[d] : from_a;
  }
#else
  (void)a; (void)b; (void)second;
#endif
}

}  // namespace vecops_hip
#endif
