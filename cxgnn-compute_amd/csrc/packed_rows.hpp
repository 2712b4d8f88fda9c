// Rows held in 8 bits (packed_rows.hip): layout, scales and decoding, shared with their readers.
#pragma once
#include "row_types.hpp"

namespace cxg {

constexpr int kPrGroup = 128;            // columns that share a scale
constexpr int kPrMinExp = 16;            // smallest exponent byte: 2^-111
constexpr int kPrNotFinite = 255;        // exponent byte of a group with an infinity or a NaN
constexpr int kPrMaxCols = 1 << 22;

inline int packed_pitch(int cols) { return (cols + 15) / 16 * 16; }
inline int packed_groups(int cols) { return (cols + kPrGroup - 1) / kPrGroup; }

#ifdef __HIPCC__
// 2^k of an exponent byte; an infinity for groups that were not finite, whose codes are 0: 0 * inf = NaN
__device__ __forceinline__ float packed_scale(unsigned byte) { return __uint_as_float(byte << 23); }

// Four codes of a register times their scale, exact.
template <int FMT> __device__ __forceinline__ void decode4(unsigned w, float scale, float* v) {
  if constexpr (FMT == CXG_PACK_INT8) {
    v[0] = (float)(int8_t)(w & 0xffu) * scale;
    v[1] = (float)(int8_t)((w >> 8) & 0xffu) * scale;
    v[2] = (float)(int8_t)((w >> 16) & 0xffu) * scale;
    v[3] = (float)(int8_t)(w >> 24) * scale;
  } else {
    typedef float v2f __attribute__((ext_vector_type(2)));
    const v2f lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = lo.x * scale; v[1] = lo.y * scale; v[2] = hi.x * scale; v[3] = hi.y * scale;
  }
}

// V values of a row from column c on; columns at or past `cols` read as 0 and are not stored.  Rows may
// start at any value: the 16-byte accesses only assume the alignment of one value, which the memory
// path of this chip takes.
template <typename T, int V> struct RowPiece {
  typedef T vec_t __attribute__((ext_vector_type(V)));
  typedef vec_t loose_t __attribute__((aligned(sizeof(T))));
  vec_t t;
  __device__ __forceinline__ void load(const T* row, int c, int cols) {
    if (c + V <= cols) {
      t = *reinterpret_cast<const loose_t*>(row + c);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) t[i] = c + i < cols ? row[c + i] : (T)0.f;
    }
  }
  __device__ __forceinline__ void widen(float (&v)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (float)t[i];
  }
  __device__ __forceinline__ void narrow(const float (&v)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = (T)v[i];
  }
  __device__ __forceinline__ void store(T* row, int c, int cols) const {
    if (c + V <= cols) {
      *reinterpret_cast<loose_t*>(row + c) = t;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (c + i < cols) row[c + i] = t[i];
    }
  }
};
#endif

}  // namespace cxg
