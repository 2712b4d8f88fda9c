// Shared by the forward and the backward kernel of the residual norm (see residual_norm_fwd.hip).
#pragma once
#include "row_types.hpp"

namespace cxg {

constexpr int kRnThreads = 256;
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

// Team of L lanes that owns a row, ITEMS pieces of V values per lane: piece i of lane l starts at
// column (i * L + l) * V, so that each load of a team is one contiguous run.
template <int L, int V> __device__ __forceinline__ int rn_col(int item, int lane_in_team) {
  return (item * L + lane_in_team) * V;
}

// Sum over the team; every lane gets it.  L = 256: the four waves meet in LDS (`slot` alternates
// between two buffers, so that one barrier per sum is enough).
template <int L, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], float (*s_red)[kRnThreads / CXG_WAVE][2], int& slot) {
  static_assert(N <= 2, "two sums at most");
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lanes_sum<(L < CXG_WAVE ? L : CXG_WAVE)>(v[i]);
  if constexpr (L > CXG_WAVE) {
    const int wave = threadIdx.x >> 6;
    if (lane_id() == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) s_red[slot][wave][i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = (s_red[slot][0][i] + s_red[slot][1][i]) + (s_red[slot][2][i] + s_red[slot][3][i]);
    slot ^= 1;
  }
}

// fp32 parameter vectors: 0 (or `missing`) where there is no column or no vector
template <int L, int V, int ITEMS>
__device__ __forceinline__ void rn_params(const float* p, int cols, int lit, float missing, float (&out)[ITEMS][V]) {
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = rn_col<L, V>(i, lit) + j;
      out[i][j] = c < cols ? (p ? p[c] : missing) : 0.f;
    }
}

#define CXG_RN_TYPES(F)                                                                    \
  if (stream_type == CXG_F32 && branch_type == CXG_F32) return F<float, float>(a, vec, st);       \
  if (stream_type == CXG_BF16 && branch_type == CXG_BF16) return F<bf16_t, bf16_t>(a, vec, st);   \
  if (stream_type == CXG_F16 && branch_type == CXG_F16) return F<f16_t, f16_t>(a, vec, st);       \
  if (stream_type == CXG_F32 && branch_type == CXG_BF16) return F<float, bf16_t>(a, vec, st);     \
  if (stream_type == CXG_F32 && branch_type == CXG_F16) return F<float, f16_t>(a, vec, st);

int rn_check(const RnArgs& a, int stream_type, int branch_type);
bool rn_aligned(const void* p, int64_t ld, size_t bytes, int v);

}  // namespace cxg
