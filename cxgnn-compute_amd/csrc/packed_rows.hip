// Rows held in 8 bits: what a layer keeps of its input for the backward pass.
//
//   128 consecutive columns of a row share a scale 2^k;  code = x * 2^-k rounded to the nearest (ties to even)
//   int8: |code| <= 127     e4m3: |code| <= 448 (float8 e4m3fn)     k: the smallest exponent with which the
//   group's largest magnitude fits after rounding, at least -111
//
// A power of two makes both directions exact but for the one rounding: x * 2^-k and code * 2^k are
// representable, so packing what was unpacked returns the same codes, and code * 2^k is a bf16
// number (8 significant bits), which is what the matrix kernel that reads these rows needs
// (packed_wgrad.hip).  int8 keeps 7 bits below the group's largest power of two, e4m3 keeps 3 bits
// of every value down to 2^-6 * 2^k: the first for even rows, the second for rows of a wide range.
// A group with an infinity or a NaN has exponent byte 255 and codes 0: it reads back as NaN.
// A finite value is off by at most half a step of its code (2^(k-1) for int8; 1/16 of itself or 2^(k-10) for
// e4m3).  In fp16 the codes' 65536 reads back as 65504, so that finite fp16 rows stay finite; a value that rounds up
// to 2^128 has no finite fp32 or bf16 form and reads back as an infinity.
//
// Layout: codes [rows][pitch] with the columns rounded up to 16 (zeros behind the last), one
// exponent byte k + 127 per group, [rows][groups].
//
// Bound: memory, one pass.  Eight lanes own a group (two or four where a row is that short) and hold its
// values in registers between the maximum (integer maxima of the magnitudes' bits, so that a NaN is largest;
// three data-parallel moves) and the rounding; a piece of the group is 128 contiguous bytes over the eight lanes.
// Measured: 2,449,029 x 128 fp32 packed in 289 us = 5.4 TB/s (a 4 GiB copy: 4.7 TB/s).
#include <type_traits>

#include "packed_rows.hpp"

namespace cxg {
namespace {

constexpr int kPrThreads = 256;
// Lanes per group, sixteen columns each: eight, or two / four for rows of at most 32 / 64 columns (48 M bf16
// values in rows of 16: 28 us against 82 us, of 47: 34 us against 48 us).
inline int pr_lanes(int cols) { return cols <= 32 ? 2 : cols <= 64 ? 4 : 8; }

struct PackArgs {
  const void* x; int64_t ldx;
  uint8_t* codes; uint8_t* exps;
  void* out;
  int64_t rows;
  int cols, pitch, groups;
};

// Team `team` of a block that starts at group `first` of the matrix, groups counted row by row: the teams of
// a wave share the lines that groups end in, and a row's last, short group does not cost a block of its own
// (one row of blocks per group: 48 M bf16 values in rows of 200 36 us, 26 us; of 805 38 + 38 us, 33 + 25).
struct PackPlace {
  int64_t row0;                          // row of the block's first group, the same for all lanes
  int row, group;                        // row after that, group in the row
  bool live;
  __device__ __forceinline__ PackPlace(const PackArgs& a, int64_t first, int team) {
    row0 = a.groups == 1 ? first : first / a.groups;
    const unsigned n = (unsigned)(first - row0 * a.groups) + (unsigned)team, d = (unsigned)a.groups;
    // n / d: at most 1 where d > team, and n * (2^16 / d + 1) / 2^16 is exact for d < 32 and n < 2^8
    row = (int)(d >= 32 ? (n >= d ? 1u : 0u) : (n * (65536u / d + 1u)) >> 16);
    group = (int)(n - (unsigned)row * d);
    live = row0 + row < a.rows;
  }
  template <typename T> __device__ __forceinline__ T* of(T* p, int64_t ld) const { return p + row0 * ld + row * ld; }
};

template <int CTRL> __device__ __forceinline__ unsigned moved_max(unsigned m) {
  const unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, CTRL, 0xf, 0xf, false);
  return o > m ? o : m;
}

// Exponent byte of a group from the bits of its largest magnitude.
template <int FMT> __device__ __forceinline__ int exponent_byte(unsigned top) {
  const int e = (int)(top >> 23), man = (int)(top & 0x7fffffu);
  int b;
  if constexpr (FMT == CXG_PACK_INT8) b = e - 6 + (man >= 0x7f0000 ? 1 : 0);     // 127.5 / 64 and more would round to 128
  else b = e - 8 + (man > 0x600000 ? 1 : 0);                                     // 448 = 1.75 * 2^8
  b = b < kPrMinExp ? kPrMinExp : b;
  return e == 255 ? kPrNotFinite : b;
}

// Four values times 2^-k as four codes in one register.
template <int FMT> __device__ __forceinline__ unsigned encode4(const float* v, float inv) {
  if constexpr (FMT == CXG_PACK_INT8) {
    // added to 1.5 * 2^23 the product rounds to an integer, which then is the low byte of the sum
    unsigned t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = __float_as_uint(__builtin_fmaf(v[i], inv, 12582912.f));
    const unsigned lo = __builtin_amdgcn_perm(t[1], t[0], 0x0c0c0400), hi = __builtin_amdgcn_perm(t[3], t[2], 0x0c0c0400);
    return __builtin_amdgcn_perm(hi, lo, 0x05040100);
  } else {
    int t = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, t, true);
  }
}

template <typename T, int FMT, int LANES> __global__ __launch_bounds__(kPrThreads) void pack_rows_kernel(PackArgs a) {
  constexpr int V = 16 / sizeof(T), kPieces = 16 / V, kTeams = kPrThreads / LANES;
  static_assert(kTeams <= 32 || LANES < 8, "PackPlace");             // (narrow rows are one group)
  const int lit = threadIdx.x % LANES;
  const int64_t all = a.rows * a.groups;
  for (int64_t base = (int64_t)blockIdx.x * kTeams; base < all; base += (int64_t)gridDim.x * kTeams) {
    const PackPlace at(a, base, threadIdx.x / LANES);
    const int c0 = at.group * kPrGroup, cols = at.live ? a.cols : 0;   // dead teams stay: the moves need whole waves
    const T* const src = at.of(static_cast<const T*>(a.x), a.ldx);
    float v[kPieces][V];
    RowPiece<T, V> raw[kPieces];
#pragma unroll
    for (int p = 0; p < kPieces; ++p) raw[p].load(src, c0 + (p * LANES + lit) * V, cols);
    unsigned top = 0;
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      raw[p].widen(v[p]);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const unsigned m = __float_as_uint(v[p][j]) & 0x7fffffffu;
        top = m > top ? m : top;
      }
    }
    top = moved_max<0xB1>(top);                          // quad_perm [1,0,3,2]
    if constexpr (LANES >= 4) top = moved_max<0x4E>(top);            // quad_perm [2,3,0,1]
    if constexpr (LANES >= 8) top = moved_max<0x141>(top);           // row_half_mirror
    const int b = exponent_byte<FMT>(top);
    const float inv = __uint_as_float((unsigned)(254 - b) << 23);
    if (!at.live) continue;
    uint8_t* const out = at.of(a.codes, a.pitch);
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      const int c = c0 + (p * LANES + lit) * V;
      if (c >= a.pitch) continue;
      uint8_t* const dst = out + c;
      unsigned w[V / 4];
#pragma unroll
      for (int q = 0; q < V / 4; ++q) w[q] = b == kPrNotFinite ? 0u : encode4<FMT>(&v[p][4 * q], inv);
      if constexpr (V == 4) {
        *reinterpret_cast<unsigned*>(dst) = w[0];
      } else {
        *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
      }
    }
    if (lit == 0) at.of(a.exps, a.groups)[at.group] = (uint8_t)b;
  }
}

template <typename T, int FMT, int LANES> __global__ __launch_bounds__(kPrThreads) void unpack_rows_kernel(PackArgs a) {
  constexpr int V = 16 / sizeof(T), kPieces = 16 / V, kTeams = kPrThreads / LANES;
  const int lit = threadIdx.x % LANES;
  const int64_t all = a.rows * a.groups;
  for (int64_t base = (int64_t)blockIdx.x * kTeams; base < all; base += (int64_t)gridDim.x * kTeams) {
    const PackPlace at(a, base, threadIdx.x / LANES);
    if (!at.live) continue;
    const int c0 = at.group * kPrGroup;
    const uint8_t* const src = at.of<const uint8_t>(a.codes, a.pitch);
    // the piece that would pass the end of the row is moved back to end there (values of its neighbour, stored
    // twice) unless its group is shorter: 48 M bf16 values in rows of 47 30 us, value by value 62
    typedef unsigned words_t __attribute__((ext_vector_type(V / 4)));
    typedef words_t loose_t __attribute__((aligned(1)));
    words_t w[kPieces];
    int col[kPieces];
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      col[p] = c0 + (p * LANES + lit) * V;
      if (col[p] < a.cols && col[p] + V > a.cols && a.cols - V >= c0) col[p] = a.cols - V;
      w[p] = 0;
      if (col[p] < a.cols) w[p] = *reinterpret_cast<const loose_t*>(src + col[p]);      // (inside the pitch)
    }
    const float scale = packed_scale(at.of(a.exps, a.groups)[at.group]);
    T* const dst = at.of(static_cast<T*>(a.out), a.cols);
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      float v[V];
#pragma unroll
      for (int q = 0; q < V / 4; ++q) decode4<FMT>(w[p][q], scale, &v[4 * q]);
      if constexpr (std::is_same<T, f16_t>::value) {
        // fp16 values next to the largest, 65504, are held as 65536 and stay finite.  (448 * 2^7 and 127 * 2^9 are
        // below that: only groups of a large scale are looked through.)
        if (scale >= 256.f) {
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] = __builtin_fabsf(v[j]) == 65536.f ? __builtin_copysignf(65504.f, v[j]) : v[j];
        }
      }
      RowPiece<T, V> o;
      o.narrow(v);
      o.store(dst, col[p], a.cols);
    }
  }
}

int pack_check(int type, int fmt, int64_t rows, int cols) {
  CXG_REQUIRE(rows >= 0 && cols >= 1, CXG_ERR_ARG, "bad rows/cols");
  CXG_REQUIRE(value_type_ok(type), CXG_ERR_ARG, "unknown value type");
  CXG_REQUIRE(fmt == CXG_PACK_INT8 || fmt == CXG_PACK_E4M3, CXG_ERR_ARG, "unknown 8-bit format");
  CXG_REQUIRE(cols <= kPrMaxCols, CXG_ERR_UNSUPPORTED, "rows of more than %d columns", kPrMaxCols);
  return CXG_OK;
}

// (more groups per block than this fills: a loop)
dim3 pack_grid(int64_t rows, int groups, int teams) {
  const int64_t x = ceil_div(rows * groups, (int64_t)teams);
  return dim3((unsigned)(x < 16384 ? x : 16384));
}

#define CXG_PR_LAUNCH_LANES(KERNEL, T, FMT)                                                                \
  do {                                                                                                     \
    const int lanes = pr_lanes(a.cols);                                                                    \
    const dim3 grid = pack_grid(rows, a.groups, kPrThreads / lanes), block(kPrThreads);                    \
    if (lanes == 2) hipLaunchKernelGGL((KERNEL<T, FMT, 2>), grid, block, 0, st, a);                        \
    else if (lanes == 4) hipLaunchKernelGGL((KERNEL<T, FMT, 4>), grid, block, 0, st, a);                   \
    else hipLaunchKernelGGL((KERNEL<T, FMT, 8>), grid, block, 0, st, a);                                   \
  } while (0)
#define CXG_PR_LAUNCH_FMT(KERNEL, T)                                                                       \
  do {                                                                                                     \
    if (fmt == CXG_PACK_INT8) CXG_PR_LAUNCH_LANES(KERNEL, T, CXG_PACK_INT8);                               \
    else CXG_PR_LAUNCH_LANES(KERNEL, T, CXG_PACK_E4M3);                                                    \
  } while (0)
#define CXG_PR_LAUNCH(KERNEL, name)                                                                        \
  do {                                                                                                     \
    if (type == CXG_F32) CXG_PR_LAUNCH_FMT(KERNEL, float);                                                 \
    else if (type == CXG_BF16) CXG_PR_LAUNCH_FMT(KERNEL, bf16_t);                                          \
    else CXG_PR_LAUNCH_FMT(KERNEL, f16_t);                                                                 \
    CXG_LAUNCH_CHECK(name);                                                                                \
  } while (0)

}  // namespace
}  // namespace cxg

extern "C" {

int cxg_packed_pitch(int cols) { return cols < 1 ? 0 : cxg::packed_pitch(cols); }
int cxg_packed_groups(int cols) { return cols < 1 ? 0 : cxg::packed_groups(cols); }

int cxg_pack_rows(const void* x, int64_t ldx, int type, int fmt, int64_t rows, int cols, uint8_t* codes, uint8_t* exps,
                  void* stream) {
  using namespace cxg;
  const int bad = pack_check(type, fmt, rows, cols);
  if (bad) return bad;
  if (rows == 0) return CXG_OK;
  CXG_REQUIRE(x && codes && exps, CXG_ERR_ARG, "null x/codes/exps");
  CXG_REQUIRE(ldx >= 0, CXG_ERR_ARG, "negative row stride");
  CXG_REQUIRE(((uintptr_t)codes & 15) == 0, CXG_ERR_ARG, "codes must be 16-byte aligned");
  CXG_REQUIRE(((uintptr_t)x & (value_bytes(type) - 1)) == 0, CXG_ERR_ARG, "x is not aligned to its values");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  PackArgs a{x, ldx, codes, exps, nullptr, rows, cols, packed_pitch(cols), packed_groups(cols)};
  CXG_PR_LAUNCH(pack_rows_kernel, "pack_rows_kernel");
  return CXG_OK;
}

int cxg_unpack_rows(const uint8_t* codes, const uint8_t* exps, int fmt, int64_t rows, int cols, void* out, int type,
                    void* stream) {
  using namespace cxg;
  const int bad = pack_check(type, fmt, rows, cols);
  if (bad) return bad;
  if (rows == 0) return CXG_OK;
  CXG_REQUIRE(codes && exps && out, CXG_ERR_ARG, "null codes/exps/out");
  CXG_REQUIRE(((uintptr_t)codes & 15) == 0, CXG_ERR_ARG, "codes must be 16-byte aligned");
  CXG_REQUIRE(((uintptr_t)out & (value_bytes(type) - 1)) == 0, CXG_ERR_ARG, "out is not aligned to its values");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  PackArgs a{nullptr, 0, const_cast<uint8_t*>(codes), const_cast<uint8_t*>(exps), out, rows, cols, packed_pitch(cols),
             packed_groups(cols)};
  CXG_PR_LAUNCH(unpack_rows_kernel, "unpack_rows_kernel");
  return CXG_OK;
}

}  // extern "C"
