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
// deviations from the registers, so a mean far from zero costs no digits.  A team of L lanes owns a
// row, up to four 16-byte pieces per lane: narrow rows share a wave (8 lanes for 128 fp32 columns,
// whose reductions are three data-parallel moves each), rows beyond 64 lanes take a block.
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
  CXG_REQUIRE(a.ldx >= 0 && a.ldf >= 0 && a.ldg >= 0 && a.lddr >= 0 && a.lddy >= 0, CXG_ERR_ARG, "negative row stride");
  return CXG_OK;
}

// Whether pieces of v values can be read at every row.
bool rn_aligned(const void* p, int64_t ld, size_t bytes, int v) {
  return p == nullptr || (((uintptr_t)p & (bytes * v - 1)) == 0 && ld % v == 0);
}

namespace {

template <typename TX, typename TF, int V, int L, int ITEMS>
__global__ __launch_bounds__(kRnThreads) void residual_norm_fwd_kernel(RnArgs a) {
  __shared__ float s_red[2][kRnThreads / CXG_WAVE][2];
  constexpr int kTeams = kRnThreads / L;
  const int lit = threadIdx.x % L, team = threadIdx.x / L;
  const int cols = a.cols;
  const float inv_c = 1.0f / (float)cols;
  int slot = 0;
  float w1[ITEMS][V], b1[ITEMS][V], w2[ITEMS][V], b2[ITEMS][V], gc[ITEMS][V];
  if (a.post_kind != CXG_NORM_NONE) {
    rn_params<L, V, ITEMS>(a.post_w, cols, lit, 1.f, w1);
    rn_params<L, V, ITEMS>(a.post_b, cols, lit, 0.f, b1);
  }
  if (a.pre_kind != CXG_NORM_NONE) {
    rn_params<L, V, ITEMS>(a.pre_w, cols, lit, 1.f, w2);
    rn_params<L, V, ITEMS>(a.pre_b, cols, lit, 0.f, b2);
  }
  if (a.gate_kind == CXG_GATE_CHANNEL) rn_params<L, V, ITEMS>(static_cast<const float*>(a.gate), cols, lit, 1.f, gc);
  bool in[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) in[i] = rn_col<L, V>(i, lit) < cols;

  // every lane stays in the loop as long as its block: the reductions need whole waves
  for (int64_t base = (int64_t)blockIdx.x * kTeams; base < a.rows; base += (int64_t)gridDim.x * kTeams) {
    const int64_t row = base + team;
    const bool live = row < a.rows;
    const int64_t rr = live ? row : 0;
    Piece<TX, V> px[ITEMS];
    Piece<TF, V> pf[ITEMS], pg[ITEMS];
    const TX* const xrow = static_cast<const TX*>(a.x) + rr * a.ldx;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      px[i].clear();
      if (in[i]) px[i].load(xrow + rn_col<L, V>(i, lit));
    }
    if (a.f) {
      const TF* const frow = static_cast<const TF*>(a.f) + rr * a.ldf;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        pf[i].clear();
        if (in[i]) pf[i].load(frow + rn_col<L, V>(i, lit));
      }
    }
    float grow = 1.f;
    if (a.gate_kind == CXG_GATE_FULL) {
      const TF* const gr = static_cast<const TF*>(a.gate) + rr * a.ldg;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        pg[i].clear();
        if (in[i]) pg[i].load(gr + rn_col<L, V>(i, lit));
      }
    } else if (a.gate_kind == CXG_GATE_ROW) {
      grow = (float)static_cast<const TF*>(a.gate)[rr * a.ldg];
    }

    float v[ITEMS][V];                               // the branch row, then the stream row
    float mean1 = 0.f, rstd1 = 1.f, mean2 = 0.f, rstd2 = 1.f;
    if (a.f) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) pf[i].widen(v[i]);
      if (a.post_kind != CXG_NORM_NONE) {
        float s[1];
        if (a.post_kind == CXG_NORM_LAYER) {
          s[0] = 0.f;
#pragma unroll
          for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) s[0] += v[i][j];
          team_sum<L, 1>(s, s_red, slot);
          mean1 = s[0] * inv_c;
        }
        s[0] = 0.f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            v[i][j] = in[i] ? v[i][j] - mean1 : 0.f;
            s[0] += v[i][j] * v[i][j];
          }
        team_sum<L, 1>(s, s_red, slot);
        rstd1 = 1.0f / sqrtf(s[0] * inv_c + a.eps);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) v[i][j] = v[i][j] * rstd1 * w1[i][j] + b1[i][j];
      }
      const float bs = a.branch_scale * grow;
      if (a.gate_kind == CXG_GATE_FULL) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
          float g[V];
          pg[i].widen(g);
#pragma unroll
          for (int j = 0; j < V; ++j) v[i][j] *= g[j];
        }
      } else if (a.gate_kind == CXG_GATE_CHANNEL) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) v[i][j] *= gc[i][j];
      }
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        float x[V];
        px[i].widen(x);
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] = a.res_scale * x[j] + bs * v[i][j];
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
      TX* const out = static_cast<TX*>(a.r) + rr * cols;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        if (in[i]) {
          Piece<TX, V> p;
          p.narrow(v[i]);
          p.store(out + rn_col<L, V>(i, lit));
        }
    }
    if (a.pre_kind != CXG_NORM_NONE) {
      float s[1];
      if (a.pre_kind == CXG_NORM_LAYER) {
        s[0] = 0.f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) s[0] += v[i][j];
        team_sum<L, 1>(s, s_red, slot);
        mean2 = s[0] * inv_c;
      }
      s[0] = 0.f;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          v[i][j] = in[i] ? v[i][j] - mean2 : 0.f;
          s[0] += v[i][j] * v[i][j];
        }
      team_sum<L, 1>(s, s_red, slot);
      rstd2 = 1.0f / sqrtf(s[0] * inv_c + a.eps);
      if (live) {
        TF* const out = static_cast<TF*>(a.y) + rr * cols;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
          if (in[i]) {
            float o[V];
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = v[i][j] * rstd2 * w2[i][j] + b2[i][j];
            Piece<TF, V> p;
            p.narrow(o);
            p.store(out + rn_col<L, V>(i, lit));
          }
      }
    }
    if (a.stats && live && lit == 0)
      reinterpret_cast<float4*>(a.stats)[row] = make_float4(mean1, rstd1, mean2, rstd2);
  }
}

template <typename TX, typename TF, int V, int L, int ITEMS> int launch_fwd(const RnArgs& a, hipStream_t st) {
  constexpr int kTeams = kRnThreads / L;
  int64_t blocks = ceil_div(a.rows, (int64_t)kTeams);
  if (blocks > 256 * 16) blocks = 256 * 16;
  hipLaunchKernelGGL((residual_norm_fwd_kernel<TX, TF, V, L, ITEMS>), dim3((unsigned)blocks), dim3(kRnThreads), 0, st, a);
  CXG_LAUNCH_CHECK("residual_norm_fwd_kernel");
  return CXG_OK;
}

template <typename TX, typename TF> int dispatch_fwd(const RnArgs& a, bool vec, hipStream_t st) {
  constexpr int W = 16 / (sizeof(TX) > sizeof(TF) ? sizeof(TX) : sizeof(TF));
  const int n = vec ? a.cols / W : a.cols;                  // pieces of a row
  if (vec) {
    if (n <= 8) return launch_fwd<TX, TF, W, 8, 1>(a, st);
    if (n <= 16) return launch_fwd<TX, TF, W, 8, 2>(a, st);
    if (n <= 32) return launch_fwd<TX, TF, W, 8, 4>(a, st);
    if (n <= 64) return launch_fwd<TX, TF, W, 16, 4>(a, st);
    if (n <= 128) return launch_fwd<TX, TF, W, 32, 4>(a, st);
    if (n <= 256) return launch_fwd<TX, TF, W, 64, 4>(a, st);
    if (n <= 1024) return launch_fwd<TX, TF, W, 256, 4>(a, st);
    if constexpr (W == 4) return launch_fwd<TX, TF, W, 256, 8>(a, st);
  } else {
    if (n <= 16) return launch_fwd<TX, TF, 1, 8, 2>(a, st);
    if (n <= 64) return launch_fwd<TX, TF, 1, 16, 4>(a, st);
    if (n <= 256) return launch_fwd<TX, TF, 1, 64, 4>(a, st);
    if (n <= 1024) return launch_fwd<TX, TF, 1, 256, 4>(a, st);
    return launch_fwd<TX, TF, 1, 256, 32>(a, st);
  }
  return set_error(CXG_ERR_UNSUPPORTED, "rows of more than %d columns", kRnMaxCols);
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
  const size_t sx = value_bytes(stream_type), sf = value_bytes(branch_type);
  const int v = stream_type == CXG_F32 || branch_type == CXG_F32 ? 4 : 8;
  const bool vec = cols % v == 0 && rn_aligned(x, ldx, sx, v) && rn_aligned(f, ldf, sf, v) &&
                   (gate_kind != CXG_GATE_FULL || rn_aligned(gate, ldg, sf, v)) && rn_aligned(r, 0, sx, v) &&
                   rn_aligned(y, 0, sf, v);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  CXG_RN_TYPES(dispatch_fwd)
  return set_error(CXG_ERR_UNSUPPORTED, "unsupported types");
}
