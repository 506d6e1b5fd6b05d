// Cross-lane data movement inside one 64-wide wavefront, built from the cheapest
// CDNA4 primitive for each distance: DPP quad permutes and row mirrors (full VALU rate,
// usually folded into the consuming add), v_permlane16_swap / v_permlane32_swap.
#pragma once
#include "common.h"

namespace flh {

constexpr int kDppQuadXor1 = 0xB1;       // quad_perm:[1,0,3,2]
constexpr int kDppQuadXor2 = 0x4E;       // quad_perm:[2,3,0,1]
constexpr int kDppRowHalfMirror = 0x141; // lane i <-> 7 - i inside each group of 8
constexpr int kDppRowMirror = 0x140;     // lane i <-> 15 - i inside each row of 16
constexpr int kDppRowRor8 = 0x128;       // rotate by 8 inside each row of 16 (lane ^ 8)

template <int CTRL>
__device__ __forceinline__ float dpp_f(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
template <int CTRL>
__device__ __forceinline__ int dpp_i(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, true);
}

// value of lane (lane ^ MASK) for MASK in {1, 2, 4, 8, 16, 32}
template <int MASK>
__device__ __forceinline__ int lane_xor_i(int v) {
  if constexpr (MASK == 1) return dpp_i<kDppQuadXor1>(v);
  else if constexpr (MASK == 2) return dpp_i<kDppQuadXor2>(v);
  else if constexpr (MASK == 4) return __builtin_amdgcn_ds_swizzle(v, (4 << 10) | 0x1F);
  else if constexpr (MASK == 8) return dpp_i<kDppRowRor8>(v);
  else if constexpr (MASK == 16) return __builtin_amdgcn_ds_swizzle(v, (16 << 10) | 0x1F);
  else {
    static_assert(MASK == 32, "lane distance");
    auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    // r[0] = {v.lo, v.lo}, r[1] = {v.hi, v.hi}
    return (threadIdx.x & 32) ? r[0] : r[1];
  }
}
template <int MASK>
__device__ __forceinline__ float lane_xor_f(float v) {
  return __int_as_float(lane_xor_i<MASK>(__float_as_int(v)));
}

// max over the whole wavefront, result in every lane
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp_f<kDppQuadXor1>(v));
  v = fmaxf(v, dpp_f<kDppQuadXor2>(v));
  v = fmaxf(v, dpp_f<kDppRowHalfMirror>(v));
  v = fmaxf(v, dpp_f<kDppRowMirror>(v));
  v = fmaxf(v, lane_xor_f<16>(v));
  v = fmaxf(v, lane_xor_f<32>(v));
  return v;
}

// sum over the whole wavefront (fixed tree order), result in every lane
__device__ __forceinline__ float wave_sum(float v) {
  v += dpp_f<kDppQuadXor1>(v);
  v += dpp_f<kDppQuadXor2>(v);
  v += dpp_f<kDppRowHalfMirror>(v);
  v += dpp_f<kDppRowMirror>(v);
  v += lane_xor_f<16>(v);
  v += lane_xor_f<32>(v);
  return v;
}

// v of the lane `CTRL` names, where the rows of sixteen in ROWS have one there, added
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned add_dpp(unsigned v) {
  return v + (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
// inclusive sums over the wavefront's lanes
__device__ __forceinline__ unsigned wave_scan(unsigned v) {
  v = add_dpp<0x111, 0xF>(v);                          // row_shr:1, 2, 4, 8 inside the rows
  v = add_dpp<0x112, 0xF>(v);
  v = add_dpp<0x114, 0xF>(v);
  v = add_dpp<0x118, 0xF>(v);
  v = add_dpp<0x142, 0xA>(v);                          // row_bcast:15 into rows 1 and 3
  return add_dpp<0x143, 0xC>(v);                       // row_bcast:31 into rows 2 and 3
}

}  // namespace flh
