// Shared by the forward and the backward kernel of the residual norm (see residual_norm_fwd.hip).
#pragma once
#include "packed_rows.hpp"

namespace cxg {

constexpr int kRnMaxCols = 8192;
constexpr int kRnSums = 4;               // column sums of the backward pass

struct RnArgs {
  const void* x; int64_t ldx;            // stream rows
  const void* f; int64_t ldf;            // branch rows (null: y = pre(x) alone)
  const void* gate; int64_t ldg;         // channel: fp32 [cols]; row / full: branch type
  int gate_kind, post_kind, pre_kind;
  const float* post_w; const float* post_b;
  const float* pre_w; const float* pre_b;
  float res_scale, branch_scale, eps;
  int64_t rows;
  int cols;
  float* stats;                          // [rows][4]: mean, 1/std of the branch row; mean, 1/std of the stream row
  // forward
  void* r; void* y;
  // backward
  const void* dr; int64_t lddr;
  const void* dy; int64_t lddy;
  void* dx; void* df; void* dgate;
  float* partial;                        // [blocks][kRnSums][cols]
};

// How the last piece of a row ends: with the row; short, its values then come from the V last columns; or
// the whole row is shorter than one piece.
enum RnTail { kRnWhole, kRnShort, kRnTiny };

// A team of L lanes owns a row, PER columns per lane; narrow rows share a wave, wide ones take several
// waves.  Piece i of lane l starts at column (i * L + l) * V: each load of a team is one contiguous run.
template <typename TX, typename TF, int L_, int PER_, int TAIL_> struct RnTeam {
  static constexpr int L = L_, PER = PER_, V = 16 / (sizeof(TX) > sizeof(TF) ? sizeof(TX) : sizeof(TF)), ITEMS = PER / V;
  static constexpr int THREADS = L < 256 ? 256 : L, TEAMS = THREADS / L, WAVES = THREADS / CXG_WAVE;
  static constexpr int TAIL = TAIL_;
};

// V values of a row from column c on, any alignment of the row; zeros where c is past its end.  A short
// piece is read where it ends with the row, without a branch, and moved to its place by rn_widen.
template <int TAIL, typename T, int V> __device__ __forceinline__ void rn_load(RowPiece<T, V>& p, const T* row, int c, int cols) {
  if constexpr (TAIL == kRnTiny) {
    p.load(row, c, cols);
  } else {
    p.t = (T)0.f;
    if (c < cols) p.t = *reinterpret_cast<const typename RowPiece<T, V>::loose_t*>(row + (TAIL == kRnShort && c + V > cols ? cols - V : c));
  }
}
template <int TAIL, typename T, int V> __device__ __forceinline__ void rn_widen(const RowPiece<T, V>& p, int c, int cols, float (&v)[V]) {
  p.widen(v);
  if constexpr (TAIL == kRnShort) {
    if (c < cols && c + V > cols) {
      const int s = c + V - cols;                        // 1 .. V - 1 values in front of the piece
#pragma unroll
      for (int k = V / 2; k >= 1; k /= 2)
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = (s & k) ? (j + k < V ? v[j + k] : 0.f) : v[j];
    }
  }
}
template <int TAIL, typename T, int V> __device__ __forceinline__ void rn_store(const float (&v)[V], T* row, int c, int cols) {
  RowPiece<T, V> p;
  p.narrow(v);
  if constexpr (TAIL != kRnWhole) {
    p.store(row, c, cols);
  } else {
    if (c < cols) *reinterpret_cast<typename RowPiece<T, V>::loose_t*>(row + c) = p.t;
  }
}

template <int L, int V> __device__ __forceinline__ int rn_col(int item, int lane_in_team) {
  return (item * L + lane_in_team) * V;
}

// Sum over the team; every lane gets it.  Teams of several waves meet in LDS (`slot` alternates between
// two buffers, so that one barrier per sum is enough).
template <typename S, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], float (*s_red)[S::WAVES][2], int& slot) {
  static_assert(N <= 2, "two sums at most");
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lanes_sum<(S::L < CXG_WAVE ? S::L : CXG_WAVE)>(v[i]);
  if constexpr (S::L > CXG_WAVE) {
    constexpr int W = S::L / CXG_WAVE;                   // waves of a team
    const int wave = threadIdx.x >> 6, first = wave / W * W;
    if (lane_id() == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) s_red[slot][wave][i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = s_red[slot][first][i];
#pragma unroll
      for (int w = 1; w < W; ++w) v[i] += s_red[slot][first + w][i];
    }
    slot ^= 1;
  }
}

// fp32 parameter vectors: 0 where there is no column, `missing` where there is no vector
template <int L, int V, int ITEMS>
__device__ __forceinline__ void rn_params(const float* p, int cols, int lit, float missing, float (&out)[ITEMS][V]) {
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
#pragma unroll
    for (int q = 0; q < V; q += 4) {
      const int c = rn_col<L, V>(i, lit) + q;
      RowPiece<float, 4> w;
      if (p) {
        w.load(p, c, cols);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) w.t[j] = c + j < cols ? missing : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) out[i][q + j] = w.t[j];
    }
}

// F<TX, TF, L, PER, TAIL>(a, st) for the types and the width: 8 columns per lane (16 are no faster where
// they fit) up to a team of 512 lanes.
#define CXG_RN_WIDTH(F, TX, TF, TAIL)                                                      \
  do {                                                                                     \
    if (a.cols <= 32) return F<TX, TF, 4, 8, TAIL>(a, st);                                 \
    if (a.cols <= 64) return F<TX, TF, 8, 8, TAIL>(a, st);                                 \
    if (a.cols <= 128) return F<TX, TF, 16, 8, TAIL>(a, st);                               \
    if (a.cols <= 256) return F<TX, TF, 32, 8, TAIL>(a, st);                               \
    if (a.cols <= 512) return F<TX, TF, 64, 8, TAIL>(a, st);                               \
    if (a.cols <= 1024) return F<TX, TF, 128, 8, TAIL>(a, st);                             \
    if (a.cols <= 2048) return F<TX, TF, 256, 8, TAIL>(a, st);                             \
    if (a.cols <= 4096) return F<TX, TF, 512, 8, TAIL>(a, st);                             \
    return F<TX, TF, 512, 16, TAIL>(a, st);                                                \
  } while (0)
#define CXG_RN_TYPE(F, ST, TX, BT, TF)                                                     \
  if (stream_type == ST && branch_type == BT) {                                            \
    constexpr int V = 16 / (int)sizeof(TX);                                                \
    if (a.cols % V == 0) CXG_RN_WIDTH(F, TX, TF, kRnWhole);                                \
    if (a.cols > V) CXG_RN_WIDTH(F, TX, TF, kRnShort);                                     \
    return F<TX, TF, 4, 8, kRnTiny>(a, st);                                                \
  }
#define CXG_RN_TYPES(F)                                                                    \
  CXG_RN_TYPE(F, CXG_F32, float, CXG_F32, float)                                           \
  CXG_RN_TYPE(F, CXG_BF16, bf16_t, CXG_BF16, bf16_t)                                       \
  CXG_RN_TYPE(F, CXG_F16, f16_t, CXG_F16, f16_t)                                           \
  CXG_RN_TYPE(F, CXG_F32, float, CXG_BF16, bf16_t)                                         \
  CXG_RN_TYPE(F, CXG_F32, float, CXG_F16, f16_t)

int rn_check(const RnArgs& a, int stream_type, int branch_type);

}  // namespace cxg
