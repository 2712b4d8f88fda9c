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

// How the last piece of a row ends: with the row; past it, the piece is then moved back to end with the
// row; or the whole row is shorter than one piece.
enum RnTail { kRnWhole, kRnShort, kRnTiny };

// A team of L lanes owns a row, PER columns per lane; narrow rows share a wave, wide ones take several
// waves.  Piece i of lane l starts at column (i * L + l) * V: each load of a team is one contiguous run.
// A piece that was moved back holds columns that its neighbour holds too: both compute and store the same
// values for them, and sums over a row leave the second one's out.
template <typename TX, typename TF, int L_, int PER_, int TAIL_> struct RnTeam {
  static constexpr int L = L_, PER = PER_, V = 16 / (sizeof(TX) > sizeof(TF) ? sizeof(TX) : sizeof(TF)), ITEMS = PER / V;
  static constexpr int THREADS = L < 256 ? 256 : L, TEAMS = THREADS / L, WAVES = THREADS / CXG_WAVE;
  static constexpr int TAIL = TAIL_;
};

// The pieces of a lane.
template <typename S> struct RnPieces {
  int col[S::ITEMS], shared[S::ITEMS];                   // first column; leading values that the neighbour holds
  bool on[S::ITEMS];
  int cols;
  __device__ __forceinline__ RnPieces(int cols_) : cols(cols_) {
    const int lit = threadIdx.x % S::L;
#pragma unroll
    for (int i = 0; i < S::ITEMS; ++i) {
      const int c = (i * S::L + lit) * S::V;
      on[i] = c < cols;
      shared[i] = S::TAIL == kRnShort && on[i] && c + S::V > cols ? c + S::V - cols : 0;
      col[i] = c - shared[i];
    }
  }
  // whether value j of piece i counts in sums over the row
  __device__ __forceinline__ bool counts(int i, int j) const {
    return on[i] && (S::TAIL == kRnWhole || (S::TAIL == kRnShort ? j >= shared[i] : col[i] + j < cols));
  }
  // any alignment of the row; zeros where there is no column
  template <typename T> __device__ __forceinline__ void load(RowPiece<T, S::V>& p, const T* row, int i, bool live = true) const {
    p.t = (T)0.f;
    if constexpr (S::TAIL == kRnTiny) {
      if (live) p.load(row, col[i], cols);
    } else {
      if (on[i] && live) p.t = *reinterpret_cast<const typename RowPiece<T, S::V>::loose_t*>(row + col[i]);
    }
  }
  template <typename T> __device__ __forceinline__ void store(const float (&v)[S::V], T* row, int i) const {
    RowPiece<T, S::V> p;
    p.narrow(v);
    if constexpr (S::TAIL == kRnTiny) {
      p.store(row, col[i], cols);
    } else {
      if (on[i]) *reinterpret_cast<typename RowPiece<T, S::V>::loose_t*>(row + col[i]) = p.t;
    }
  }
  // fp32 parameter vectors: 0 where there is no column, `missing` where there is no vector
  __device__ __forceinline__ void params(const float* p, float missing, float (&out)[S::ITEMS][S::V]) const {
#pragma unroll
    for (int i = 0; i < S::ITEMS; ++i)
#pragma unroll
      for (int q = 0; q < S::V; q += 4) {
        RowPiece<float, 4> w;
        if (p) {
          w.load(p, col[i] + q, cols);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) w.t[j] = col[i] + q + j < cols ? missing : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) out[i][q + j] = w.t[j];
      }
  }
};

// The rows of a block's teams: the first row of this wave, the same for all its lanes, and what the lane's
// team adds to it.  (A row number per lane costs a 64-bit vector multiplication per tensor and row, a fifth
// of what the forward pass computes for a narrow row.)
template <typename S> struct RnRow {
  int wave_team, lane_team;
  int64_t first = 0;                                      // row of the wave's first team
  __device__ __forceinline__ RnRow() {
    wave_team = S::L < CXG_WAVE ? uniform_i32(threadIdx.x >> 6) * (CXG_WAVE / S::L) : uniform_i32(threadIdx.x / S::L);
    lane_team = S::L < CXG_WAVE ? (int)(threadIdx.x & (CXG_WAVE - 1)) / S::L : 0;
  }
  __device__ __forceinline__ int64_t row() const { return first + lane_team; }
  template <typename T> __device__ __forceinline__ T* of(T* p, int64_t ld) const { return p + first * ld + lane_team * ld; }
};

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

// F<TX, TF, L, PER, TAIL>(a, st) for the types and the width: 8 columns per lane (16 are no faster where
// they fit) up to a team of 512 lanes.
#define CXG_RN_WIDTH(F, TX, TF, TAIL)                                                      \
  do {                                                                                     \
    if (a.cols <= 16) return F<TX, TF, 2, 8, TAIL>(a, st);                                 \
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
    return F<TX, TF, 2, 8, kRnTiny>(a, st);                                                \
  }
#define CXG_RN_TYPES(F)                                                                    \
  CXG_RN_TYPE(F, CXG_F32, float, CXG_F32, float)                                           \
  CXG_RN_TYPE(F, CXG_BF16, bf16_t, CXG_BF16, bf16_t)                                       \
  CXG_RN_TYPE(F, CXG_F16, f16_t, CXG_F16, f16_t)                                           \
  CXG_RN_TYPE(F, CXG_F32, float, CXG_BF16, bf16_t)                                         \
  CXG_RN_TYPE(F, CXG_F32, float, CXG_F16, f16_t)

int rn_check(const RnArgs& a, int stream_type, int branch_type);

}  // namespace cxg
