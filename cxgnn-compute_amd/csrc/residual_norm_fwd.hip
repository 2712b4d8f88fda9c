// Residual connection with a norm on either side of it, one pass over the rows:
//
//   r = res_scale * x + branch_scale * gate * post(f)        the residual stream after a block
//   y = pre(r)                                               what the next block reads
//
// post and pre are layer norms ((v - mean) / sqrt(var + eps) * w + b), rms norms
// (v / sqrt(mean v^2 + eps) * w + b) or nothing; the gate is one value per column, per row or per
// element, or nothing.  x and r share a type (the stream), f, the gate of rows or elements and y
// another (the branch); statistics and all arithmetic are fp32, y is formed from r before r is
// rounded to its type.
//
// Bound: memory.  A row is read once (x, f), kept in registers through both norms and written once
// (r, y); everything else are the reductions over its columns: mean first, then the sum of squared
// deviations from the registers, so a mean far from zero costs no digits.  A team of lanes owns a row,
// 8 columns per lane whatever the width: the vectors of the norms then stay in registers from row to row
// and enough waves fit a CU to keep memory busy.  (Up to 32 columns per lane left rows of 512 bf16 columns
// at 1.2 TB/s; a grid of more blocks than are resident loads the vectors more often, 3.6 against 5.1 TB/s.)  Rows
// start at any value: the 16-byte accesses assume the alignment of one value only.  Measured: 169,343 x 256 fp32, channel gate 124 us =
// 5.6 TB/s; 2,449,029 x 128 bf16, element gate 645 us = 4.9 TB/s; 187,500 x 256 fp32 beside bf16 branches 113 us = 5.1 TB/s.
#include "residual_norm.hpp"

namespace cxg {

int rn_check(const RnArgs& a, int stream_type, int branch_type) {
  CXG_REQUIRE(a.rows >= 0 && a.cols >= 1, CXG_ERR_ARG, "bad rows/cols");
  CXG_REQUIRE(value_type_ok(stream_type) && value_type_ok(branch_type), CXG_ERR_ARG, "unknown value type");
  CXG_REQUIRE(stream_type == CXG_F32 || stream_type == branch_type, CXG_ERR_UNSUPPORTED,
              "the branch has the stream's type, or the stream is fp32");
  CXG_REQUIRE(a.cols <= kRnMaxCols, CXG_ERR_UNSUPPORTED, "rows of more than %d columns", kRnMaxCols);
  CXG_REQUIRE(a.gate_kind >= CXG_GATE_NONE && a.gate_kind <= CXG_GATE_FULL, CXG_ERR_ARG, "unknown gate kind");
  CXG_REQUIRE(a.post_kind >= CXG_NORM_NONE && a.post_kind <= CXG_NORM_LAYER && a.pre_kind >= CXG_NORM_NONE &&
                  a.pre_kind <= CXG_NORM_LAYER, CXG_ERR_ARG, "unknown norm kind");
  CXG_REQUIRE(a.gate_kind == CXG_GATE_NONE || a.rows == 0 || a.gate, CXG_ERR_ARG, "null gate");
  CXG_REQUIRE(a.f || a.rows == 0 || (a.gate_kind == CXG_GATE_NONE && a.post_kind == CXG_NORM_NONE), CXG_ERR_ARG,
              "a gate or a norm of the branch needs branch rows");
  CXG_REQUIRE(a.rows == 0 || a.x, CXG_ERR_ARG, "null x");
  const uintptr_t sx = value_bytes(stream_type) - 1, sf = value_bytes(branch_type) - 1;
  CXG_REQUIRE((((uintptr_t)a.x | (uintptr_t)a.r | (uintptr_t)a.dr | (uintptr_t)a.dx) & sx) == 0 &&
                  (((uintptr_t)a.f | (uintptr_t)a.y | (uintptr_t)a.dy | (uintptr_t)a.df) & sf) == 0 &&
                  ((uintptr_t)a.gate & (a.gate_kind == CXG_GATE_CHANNEL ? 3 : sf)) == 0,
              CXG_ERR_ARG, "rows that are not aligned to their values");
  CXG_REQUIRE(a.ldx >= 0 && a.ldf >= 0 && a.ldg >= 0 && a.lddr >= 0 && a.lddy >= 0, CXG_ERR_ARG, "negative row stride");
  return CXG_OK;
}

namespace {

template <typename TX, typename TF, typename S>
__global__ __launch_bounds__(S::THREADS, S::THREADS == 256 ? 5 : S::PER == 8 ? 4 : 2) void residual_norm_fwd_kernel(RnArgs a) {
  constexpr int L = S::L, V = S::V, ITEMS = S::ITEMS, kTeams = S::TEAMS;
  __shared__ float s_red[2][S::WAVES][2];
  const int lit = threadIdx.x % L;
  const int cols = a.cols;
  const float inv_c = 1.0f / (float)cols;
  const RnPieces<S> at(cols);
  RnRow<S> of_row;
  int slot = 0;
  // what is the same for all rows, per column: branch_scale * channel gate * (post_w, post_b), pre_w, pre_b
  const bool post = a.post_kind != CXG_NORM_NONE;
  float w1[ITEMS][V], b1[ITEMS][V], w2[ITEMS][V], b2[ITEMS][V];
  at.params(post ? a.post_w : nullptr, 1.f, w1);
  at.params(post ? a.post_b : nullptr, 0.f, b1);
  at.params(a.gate_kind == CXG_GATE_CHANNEL ? static_cast<const float*>(a.gate) : nullptr, 1.f, w2);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float scale = a.branch_scale * w2[i][j];
      w1[i][j] *= scale;
      b1[i][j] *= scale;
    }
  if (a.pre_kind != CXG_NORM_NONE) {
    at.params(a.pre_w, 1.f, w2);
    at.params(a.pre_b, 0.f, b2);
  }

  // every lane stays in the loop as long as its block: the reductions need whole waves
  for (int64_t base = (int64_t)blockIdx.x * kTeams; base < a.rows; base += (int64_t)gridDim.x * kTeams) {
    of_row.first = base + of_row.wave_team;
    const bool live = of_row.row() < a.rows;
    RowPiece<TX, V> px[ITEMS];
    RowPiece<TF, V> pf[ITEMS], pg[ITEMS];
    const TX* const xrow = of_row.of(static_cast<const TX*>(a.x), a.ldx);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) at.load(px[i], xrow, i, live);
    if (a.f) {
      const TF* const frow = of_row.of(static_cast<const TF*>(a.f), a.ldf);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) at.load(pf[i], frow, i, live);
    }
    float grow = 1.f;
    if (a.gate_kind == CXG_GATE_FULL) {
      const TF* const gr = of_row.of(static_cast<const TF*>(a.gate), a.ldg);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) at.load(pg[i], gr, i, live);
    } else if (a.gate_kind == CXG_GATE_ROW && live) {
      grow = (float)*of_row.of(static_cast<const TF*>(a.gate), a.ldg);
    }

    float v[ITEMS][V];                               // the branch row, then the stream row
    float mean1 = 0.f, rstd1 = 1.f, mean2 = 0.f, rstd2 = 1.f;
    if (a.f) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) pf[i].widen(v[i]);
      if (post) {
        float s[1];
        if (a.post_kind == CXG_NORM_LAYER) {
          s[0] = 0.f;
#pragma unroll
          for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) s[0] += S::TAIL != kRnShort || at.counts(i, j) ? v[i][j] : 0.f;
          team_sum<S, 1>(s, s_red, slot);
          mean1 = s[0] * inv_c;
        }
        s[0] = 0.f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
          const float m = S::TAIL != kRnWhole || at.on[i] ? mean1 : 0.f;     // (columns that do not exist stay 0)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            v[i][j] -= m;
            s[0] += S::TAIL == kRnWhole || at.counts(i, j) ? v[i][j] * v[i][j] : 0.f;
          }
        }
        team_sum<S, 1>(s, s_red, slot);
        rstd1 = inverse_sqrt(s[0] * inv_c + a.eps);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) v[i][j] = v[i][j] * rstd1 * w1[i][j] + b1[i][j];
      }
      if (!post) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) v[i][j] *= w1[i][j];
      }
      if (a.gate_kind == CXG_GATE_FULL) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
          float g[V];
          pg[i].widen(g);
#pragma unroll
          for (int j = 0; j < V; ++j) v[i][j] *= g[j];
        }
      }
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        float x[V];
        px[i].widen(x);
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] = a.res_scale * x[j] + grow * v[i][j];
      }
    } else {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        float x[V];
        px[i].widen(x);
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] = a.res_scale * x[j];
      }
    }
    if (a.r && live) {
      TX* const out = of_row.of(static_cast<TX*>(a.r), cols);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) at.store(v[i], out, i);
    }
    if (a.pre_kind != CXG_NORM_NONE) {
      float s[1];
      if (a.pre_kind == CXG_NORM_LAYER) {
        s[0] = 0.f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) s[0] += S::TAIL != kRnShort || at.counts(i, j) ? v[i][j] : 0.f;
        team_sum<S, 1>(s, s_red, slot);
        mean2 = s[0] * inv_c;
      }
      s[0] = 0.f;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const float m = S::TAIL != kRnWhole || at.on[i] ? mean2 : 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          v[i][j] -= m;
          s[0] += S::TAIL == kRnWhole || at.counts(i, j) ? v[i][j] * v[i][j] : 0.f;
        }
      }
      team_sum<S, 1>(s, s_red, slot);
      rstd2 = inverse_sqrt(s[0] * inv_c + a.eps);
      if (live) {
        TF* const out = of_row.of(static_cast<TF*>(a.y), cols);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
          float o[V];
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] = v[i][j] * rstd2 * w2[i][j] + b2[i][j];
          at.store(o, out, i);
        }
      }
    }
    if (a.stats && live && lit == 0)
      *of_row.of(reinterpret_cast<float4*>(a.stats), 1) = make_float4(mean1, rstd1, mean2, rstd2);
  }
}

template <typename TX, typename TF, int L, int PER, int TAIL> int launch_fwd(const RnArgs& a, hipStream_t st) {
  typedef RnTeam<TX, TF, L, PER, TAIL> S;
  int64_t blocks = ceil_div(a.rows, (int64_t)S::TEAMS);
  if (blocks > 256 * 5) blocks = 256 * 5;                // what is resident: a block loads the vectors once
  hipLaunchKernelGGL((residual_norm_fwd_kernel<TX, TF, S>), dim3((unsigned)blocks), dim3(S::THREADS), 0, st, a);
  CXG_LAUNCH_CHECK("residual_norm_fwd_kernel");
  return CXG_OK;
}

}  // namespace
}  // namespace cxg

extern "C" int cxg_residual_norm_fwd(const void* x, int64_t ldx, const void* f, int64_t ldf, const void* gate,
                                     int64_t ldg, int gate_kind, int post_kind, const float* post_w,
                                     const float* post_b, int pre_kind, const float* pre_w, const float* pre_b,
                                     float res_scale, float branch_scale, float eps, int64_t rows, int cols,
                                     int stream_type, int branch_type, void* r, void* y, float* stats, void* stream) {
  using namespace cxg;
  RnArgs a{};
  a.x = x; a.ldx = ldx; a.f = f; a.ldf = ldf; a.gate = gate; a.ldg = ldg;
  a.gate_kind = gate_kind; a.post_kind = post_kind; a.pre_kind = pre_kind;
  a.post_w = post_w; a.post_b = post_b; a.pre_w = pre_w; a.pre_b = pre_b;
  a.res_scale = res_scale; a.branch_scale = branch_scale; a.eps = eps;
  a.rows = rows; a.cols = cols; a.stats = stats; a.r = r; a.y = y;
  const int bad = rn_check(a, stream_type, branch_type);
  if (bad) return bad;
  CXG_REQUIRE(rows == 0 || pre_kind == CXG_NORM_NONE || y, CXG_ERR_ARG, "null y");
  CXG_REQUIRE(rows == 0 || r || (pre_kind != CXG_NORM_NONE && !f), CXG_ERR_ARG, "null r");
  CXG_REQUIRE(((uintptr_t)stats & 15) == 0, CXG_ERR_ARG, "stats must be 16-byte aligned");
  if (rows == 0) return CXG_OK;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  CXG_RN_TYPES(launch_fwd)
  return set_error(CXG_ERR_UNSUPPORTED, "unsupported types");
}
