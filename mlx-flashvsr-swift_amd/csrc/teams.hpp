// Sums over the lanes and waves that share a row, for the row operators (rows8.hip, rms_norm.hip).
#pragma once
#include "common.hpp"

namespace fvsr {

// the sum over a wave (every lane active), by DPP rotations within its rows of 16 lanes and a lane of each row: no LDS
// round trips
__device__ __forceinline__ float wave_sum(float x) {
  auto rot = [](float v, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  x += rot(x, std::integral_constant<int, 0x128>{});   // row_ror:8
  x += rot(x, std::integral_constant<int, 0x124>{});
  x += rot(x, std::integral_constant<int, 0x122>{});
  x += rot(x, std::integral_constant<int, 0x121>{});
  auto row = [&](int r) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 16 * r)); };
  return (row(0) + row(1)) + (row(2) + row(3));
}

// sums over the WAVES waves that share a row, in a fixed order; `sm` holds 2 * WAVES floats, which a wave may
// still read when another has left the call: successive calls alternate between two areas
template <int WAVES>
__device__ __forceinline__ void team_sum2(float& a, float& b, float* sm) {
  a = wave_sum(a);
  b = wave_sum(b);
  if constexpr (WAVES > 1) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      sm[2 * wave] = a;
      sm[2 * wave + 1] = b;
    }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      a += sm[2 * w];
      b += sm[2 * w + 1];
    }
  }
}

// one sum; a team of no wave (WAVES 0) is 16 lanes, a row of the wave's four
template <int WAVES>
__device__ __forceinline__ float team_sum(float a, float* sm) {
  if constexpr (WAVES == 0) {
    auto rot = [](float v, auto ctrl) {
      return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, false));
    };
    a += rot(a, std::integral_constant<int, 0x128>{});   // row_ror:8
    a += rot(a, std::integral_constant<int, 0x124>{});
    a += rot(a, std::integral_constant<int, 0x122>{});
    a += rot(a, std::integral_constant<int, 0x121>{});
  } else {
    a = wave_sum(a);
    if constexpr (WAVES > 1) {
      if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = a;
      __syncthreads();
      a = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) a += sm[w];
    }
  }
  return a;
}

}  // namespace fvsr
