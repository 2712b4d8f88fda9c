// Value types of rows that may be narrower than fp32, and sums across lanes.
#pragma once
#include "cxg_common.hpp"

namespace cxg {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

inline size_t value_bytes(int type) { return type == CXG_F32 ? 4 : 2; }
inline bool value_type_ok(int type) { return type == CXG_F32 || type == CXG_BF16 || type == CXG_F16; }

// Sum over L consecutive lanes (a power of two, aligned); every lane of the group gets it.  Inside a
// row of 16 lanes by data-parallel moves, across rows by the half-swap instructions.  All 64 lanes
// of the wave have to be active.
template <int L> __device__ __forceinline__ float lanes_sum(float v) {
  typedef unsigned v2u __attribute__((ext_vector_type(2)));
  auto moved = [](float a, auto ctrl) {
    return __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(a), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  struct Xor1 { enum { value = 0xB1 }; };          // quad_perm [1,0,3,2]
  struct Xor2 { enum { value = 0x4E }; };          // quad_perm [2,3,0,1]
  struct HalfMirror { enum { value = 0x141 }; };
  struct Mirror { enum { value = 0x140 }; };
  if constexpr (L >= 2) v += moved(v, Xor1{});
  if constexpr (L >= 4) v += moved(v, Xor2{});
  if constexpr (L >= 8) v += moved(v, HalfMirror{});
  if constexpr (L >= 16) v += moved(v, Mirror{});
  if constexpr (L >= 32) {
    const v2u r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r.x) + __uint_as_float(r.y);
  }
  if constexpr (L >= 64) {
    const v2u r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r.x) + __uint_as_float(r.y);
  }
  return v;
}

// Sum over the lanes l, l + L, l + 2L, ... of the wave (same position in every group of L lanes).
template <int L> __device__ __forceinline__ float groups_sum(float v) {
  typedef unsigned v2u __attribute__((ext_vector_type(2)));
  static_assert(L >= 2, "groups of at least two lanes");
  if constexpr (L <= 2) v += __shfl_xor(v, 2, CXG_WAVE);
  if constexpr (L <= 4) v += __shfl_xor(v, 4, CXG_WAVE);
  if constexpr (L <= 8) v += __shfl_xor(v, 8, CXG_WAVE);
  if constexpr (L <= 16) {
    const v2u r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r.x) + __uint_as_float(r.y);
  }
  if constexpr (L <= 32) {
    const v2u r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r.x) + __uint_as_float(r.y);
  }
  return v;
}

// 1 / sqrt(x) by the chip's own instruction (one unit in the last place, as much as the roundings of a square
// root and a division together; those take some 25 instructions, a tenth of a narrow row's forward pass).  The
// instruction takes numbers below 2^-126 for zero, hence the scale.
__device__ __forceinline__ float inverse_sqrt(float x) {
  const bool small = x < 0x1p-96f;
  const float r = __builtin_amdgcn_rsqf(small ? x * 0x1p64f : x);
  return small ? r * 0x1p32f : r;
}

}  // namespace cxg
