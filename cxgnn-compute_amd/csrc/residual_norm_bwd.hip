// Backward pass of the residual norm (residual_norm_fwd.hip).  With h = post(f), fhat and rhat the
// normalised branch and stream rows, s1 and s2 their 1/std, a the residual and b the branch scale:
//
//   t  = dy * w_pre                       dw_pre = sum_rows dy * rhat        db_pre = sum_rows dy
//   g  = dr + s2 * (t - mean(t) - rhat * mean(t * rhat))                     the gradient of r
//   dx = a * g                            dgate  = b * g * h, summed over what the gate is shared by
//   d  = b * gate * g                     dw_post = sum_rows d * fhat        db_post = sum_rows d
//   u  = d * w_post                       df = s1 * (u - mean(u) - fhat * mean(u * fhat))
//
// (an rms norm has no mean(t), mean(u)).  r is formed again from x and f: what the forward pass
// normalised was r before it was rounded to its type, and x and f are read for the rest anyway.
//
// Bound: memory.  One pass reads x, f, dr, dy (and an element-wise gate) and writes dx, df (and its
// gradient).  The sums over rows stay in registers while a team walks its rows, four per column:
// sum dy * rhat, sum dy, sum c * g * fhat, sum c * g with c the gate of the row or element, 1 for a
// channel gate -- that one is the same for every row and is multiplied in at the end, and
// dgate = b * (w_post * sum g * fhat + b_post * sum g) needs no sum of its own.  Teams of a block meet
// in registers and LDS, blocks leave one partial row each, a second kernel adds the partial rows in
// block order: no atomics, and the grid depends on the shape alone, so results repeat bit for bit.
// b * channel gate * (w_post, b_post) is formed once per column: a third fewer operations per value and 16
// registers less (48 M values in rows of 8,192: bf16 181 -> 139 us, fp32 241 -> 220 us).
// Measured: 169,343 x 256 fp32, channel gate 211 us = 4.9 TB/s; 2,449,029 x 128 bf16, element gate
// 1.02 ms = 4.9 TB/s; 187,500 x 256 fp32 beside bf16 branches 179 us = 4.8 TB/s; the second kernel 9 us.  Rows of 4,097 to
// 8,191 columns that are no multiple of a piece spill 80 (two-byte types) to 146 registers per lane: 48 M fp32 values
// in rows of 8,191 624 us, of 8,192 254 us.
#include "residual_norm.hpp"

namespace cxg {
namespace {

constexpr int kRnMaxBlocks = 768;        // partial rows; three blocks of 256 threads per CU are resident

template <typename TX, typename TF, typename S>
__global__ __launch_bounds__(S::THREADS, S::THREADS == 256 ? 3 : 2) void residual_norm_bwd_kernel(RnArgs a) {
  constexpr int L = S::L, V = S::V, ITEMS = S::ITEMS, kTeams = S::TEAMS;
  __shared__ float s_red[2][S::WAVES][2];
  const int lit = threadIdx.x % L;
  const int cols = a.cols;
  const float inv_c = 1.0f / (float)cols;
  const RnPieces<S> at(cols);
  RnRow<S> of_row;
  int slot = 0;
  const bool post = a.post_kind != CXG_NORM_NONE, pre = a.pre_kind != CXG_NORM_NONE;
  const bool post_layer = a.post_kind == CXG_NORM_LAYER, pre_layer = a.pre_kind == CXG_NORM_LAYER;
  // what is the same for all rows, b * channel gate * (w_post, b_post) and w_pre, per column; columns that do
  // not exist have weight 0 and so add nothing to the sums over a row
  float w1[ITEMS][V], b1[ITEMS][V], w2[ITEMS][V];
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
  at.params(pre ? a.pre_w : nullptr, 1.f, w2);
  float sums[kRnSums][ITEMS][V];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
#pragma unroll
    for (int q = 0; q < kRnSums; ++q)
#pragma unroll
      for (int j = 0; j < V; ++j) sums[q][i][j] = 0.f;

  for (int64_t base = (int64_t)blockIdx.x * kTeams; base < a.rows; base += (int64_t)gridDim.x * kTeams) {
    of_row.first = base + of_row.wave_team;
    const bool live = of_row.row() < a.rows;
    RowPiece<TX, V> px[ITEMS], pdr[ITEMS];
    RowPiece<TF, V> pf[ITEMS], pg[ITEMS], pdy[ITEMS];
    const bool full = a.gate_kind == CXG_GATE_FULL;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {                     // a row that does not exist adds zeros everywhere
      pf[i].t = pg[i].t = pdy[i].t = (TF)0.f;
      pdr[i].t = (TX)0.f;
      at.load(px[i], of_row.of(static_cast<const TX*>(a.x), a.ldx), i, live);
      if (a.f) at.load(pf[i], of_row.of(static_cast<const TF*>(a.f), a.ldf), i, live);
      if (a.dr) at.load(pdr[i], of_row.of(static_cast<const TX*>(a.dr), a.lddr), i, live);
      if (a.dy) at.load(pdy[i], of_row.of(static_cast<const TF*>(a.dy), a.lddy), i, live);
      if (full) at.load(pg[i], of_row.of(static_cast<const TF*>(a.gate), a.ldg), i, live);
    }
    const float grow = a.gate_kind == CXG_GATE_ROW && live ? (float)*of_row.of(static_cast<const TF*>(a.gate), a.ldg) : 1.f;
    float4 st = make_float4(0.f, 1.f, 0.f, 1.f);
    if (live) st = *of_row.of(reinterpret_cast<const float4*>(a.stats), 1);

    // the normalised rows, b * channel gate * h, the gate as far as it differs between rows, t, the gradient of r
    float fh[ITEMS][V], h[ITEMS][V], gt[ITEMS][V], rh[ITEMS][V], t[ITEMS][V], g[ITEMS][V];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      float x[V], f[V], dy[V];
      px[i].widen(x);
      pf[i].widen(f);
      pdy[i].widen(dy);
      pg[i].widen(gt[i]);
      pdr[i].widen(g[i]);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        fh[i][j] = (f[j] - st.x) * st.y;                // (mean 0 and 1/std 1 without a norm)
        h[i][j] = fh[i][j] * w1[i][j] + b1[i][j];
        gt[i][j] = full ? gt[i][j] : grow;
        const float r = a.res_scale * x[j] + gt[i][j] * h[i][j];
        rh[i][j] = (r - st.z) * st.w;
        t[i][j] = dy[j] * w2[i][j];
        const float tc = S::TAIL != kRnShort || at.counts(i, j) ? t[i][j] : 0.f;
        s[0] += tc;
        s[1] += tc * rh[i][j];
        sums[0][i][j] += dy[j] * rh[i][j];
        sums[1][i][j] += dy[j];
      }
    }
    if (pre) {
      team_sum<S, 2>(s, s_red, slot);
      const float m0 = pre_layer ? s[0] * inv_c : 0.f, m1 = s[1] * inv_c;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) g[i][j] += st.w * (t[i][j] - m0 - rh[i][j] * m1);
    }
    if (a.dx && live) {
      TX* const out = of_row.of(static_cast<TX*>(a.dx), cols);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = a.res_scale * g[i][j];
        at.store(o, out, i);
      }
    }
    if (a.dgate) {
      if (full) {
        if (live) {
          TF* const out = of_row.of(static_cast<TF*>(a.dgate), cols);
#pragma unroll
          for (int i = 0; i < ITEMS; ++i) {
            float o[V];
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = g[i][j] * h[i][j];
            at.store(o, out, i);
          }
        }
      } else if (a.gate_kind == CXG_GATE_ROW) {
        float d[1] = {0.f};
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) d[0] += at.counts(i, j) ? g[i][j] * h[i][j] : 0.f;
        team_sum<S, 1>(d, s_red, slot);
        if (live && lit == 0) *of_row.of(static_cast<TF*>(a.dgate), 1) = (TF)d[0];
      }
    }
    if (a.f) {
      float q[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float cg = gt[i][j] * g[i][j];          // (0 in a row that does not exist)
          sums[2][i][j] += cg * fh[i][j];
          sums[3][i][j] += cg;
          g[i][j] = cg * w1[i][j];
          const float gc_ = S::TAIL != kRnShort || at.counts(i, j) ? g[i][j] : 0.f;
          q[0] += gc_;
          q[1] += gc_ * fh[i][j];
        }
      if (a.df) {
        float m0 = 0.f, m1 = 0.f;
        if (post) {
          team_sum<S, 2>(q, s_red, slot);
          m0 = post_layer ? q[0] * inv_c : 0.f;
          m1 = q[1] * inv_c;
        }
        if (live) {
          TF* const out = of_row.of(static_cast<TF*>(a.df), cols);
#pragma unroll
          for (int i = 0; i < ITEMS; ++i) {
            float o[V];
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = post ? st.y * (g[i][j] - m0 - fh[i][j] * m1) : g[i][j];
            at.store(o, out, i);
          }
        }
      }
    }
  }

  // the block's partial row: teams of a wave in registers, waves in LDS
  if (a.partial == nullptr) return;
  float* const out = a.partial + (size_t)blockIdx.x * kRnSums * cols;
  if constexpr (kTeams == 1) {
#pragma unroll
    for (int q = 0; q < kRnSums; ++q)
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int c = at.col[i] + j;
          if (c < cols) out[(size_t)q * cols + c] = sums[q][i][j];
        }
  } else {
    constexpr int kParts = L < CXG_WAVE ? S::WAVES : kTeams;     // waves, or teams of whole waves
    __shared__ float s_col[kParts][L * S::PER];
    const int part = L < CXG_WAVE ? (int)(threadIdx.x >> 6) : of_row.wave_team;
#pragma unroll
    for (int q = 0; q < kRnSums; ++q) {
      if (q) __syncthreads();
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float t = groups_sum<L>(sums[q][i][j]);
          if (L >= CXG_WAVE || (int)(threadIdx.x & (CXG_WAVE - 1)) < L) s_col[part][at.col[i] + j] = t;
        }
      __syncthreads();
      for (int c = threadIdx.x; c < cols; c += S::THREADS) {
        float t = s_col[0][c];
#pragma unroll
        for (int k = 1; k < kParts; ++k) t += s_col[k][c];
        out[(size_t)q * cols + c] = t;
      }
    }
  }
}

// Partial rows of all blocks -> the gradients of the vectors.  A block of 1024 threads takes
// kFinCols columns: a thread adds one of the four sums of a column over one of kFinSlices runs of
// partial rows, the runs are added across lanes.  (256 threads per 16 columns, four sums per thread
// and 16 runs: 14 us for 1024 partial rows of 256 columns, latency of 64 dependent steps.)
constexpr int kFinCols = 8, kFinSlices = 32;
constexpr int kFinThreads = kFinCols * kFinSlices * kRnSums;

struct RnFinal {
  const float* partial; int blocks, cols;
  const float* post_w; const float* post_b; const float* gate;   // gate: channel gate or null
  float branch_scale;
  bool post;
  float* dgate; float* dpost_w; float* dpost_b; float* dpre_w; float* dpre_b;
};

__global__ __launch_bounds__(kFinThreads) void residual_norm_sums_kernel(RnFinal a) {
  constexpr int kPairs = kRnSums * kFinCols;
  __shared__ float s[kFinSlices][kPairs + 1], s_out[kPairs];
  const int cl = threadIdx.x % kFinCols, q = (threadIdx.x / kFinCols) % kRnSums, slice = threadIdx.x / kPairs;
  const int c0 = blockIdx.x * kFinCols;
  float acc = 0.f;
  if (c0 + cl < a.cols) {
    const int per = (a.blocks + kFinSlices - 1) / kFinSlices;
    const int b1 = (slice + 1) * per < a.blocks ? (slice + 1) * per : a.blocks;
    const float* const p = a.partial + (size_t)q * a.cols + c0 + cl;
#pragma unroll 8
    for (int b = slice * per; b < b1; ++b) acc += p[(size_t)b * kRnSums * a.cols];
  }
  s[slice][q * kFinCols + cl] = acc;
  __syncthreads();
  static_assert(kFinSlices == 32 && kFinThreads / kFinSlices == kPairs, "half a wave per sum");
  const float total = lanes_sum<kFinSlices>(s[threadIdx.x % kFinSlices][threadIdx.x / kFinSlices]);
  if (threadIdx.x % kFinSlices == 0) s_out[threadIdx.x / kFinSlices] = total;
  __syncthreads();
  const int c = c0 + threadIdx.x;
  if (threadIdx.x >= kFinCols || c >= a.cols) return;
  const float s0 = s_out[cl], s1 = s_out[kFinCols + cl], s2 = s_out[2 * kFinCols + cl], s3 = s_out[3 * kFinCols + cl];
  const float w = a.post && a.post_w ? a.post_w[c] : 1.f, b = a.post && a.post_b ? a.post_b[c] : 0.f;
  const float scale = a.branch_scale * (a.gate ? a.gate[c] : 1.f);
  if (a.dpre_w) a.dpre_w[c] = s0;
  if (a.dpre_b) a.dpre_b[c] = s1;
  if (a.dpost_w) a.dpost_w[c] = scale * s2;
  if (a.dpost_b) a.dpost_b[c] = scale * s3;
  if (a.dgate) a.dgate[c] = a.branch_scale * (w * s2 + b * s3);
}

// Blocks of the row kernel: what is resident (one block of 512 threads per CU), each walks its rows.
int64_t bwd_blocks(int64_t rows, int teams, int threads) {
  const int64_t blocks = ceil_div(rows, (int64_t)teams), most = threads > 256 ? 256 : kRnMaxBlocks;
  return blocks > most ? most : blocks;
}

// launches the row kernel; returns the number of partial rows, or a negative status
template <typename TX, typename TF, int L, int PER, int TAIL> int launch_bwd(const RnArgs& a, hipStream_t st) {
  typedef RnTeam<TX, TF, L, PER, TAIL> S;
  const int64_t blocks = bwd_blocks(a.rows, S::TEAMS, S::THREADS);
  hipLaunchKernelGGL((residual_norm_bwd_kernel<TX, TF, S>), dim3((unsigned)blocks), dim3(S::THREADS), 0, st, a);
  CXG_LAUNCH_CHECK("residual_norm_bwd_kernel");
  return (int)blocks;
}

int dispatch_bwd(const RnArgs& a, int stream_type, int branch_type, hipStream_t st) {
  CXG_RN_TYPES(launch_bwd)
  return set_error(CXG_ERR_UNSUPPORTED, "unsupported types");
}

}  // namespace
}  // namespace cxg

extern "C" {

size_t cxg_residual_norm_workspace_bytes(int64_t rows, int cols) {
  if (rows < 0 || cols < 1) return 0;
  return (size_t)cxg::bwd_blocks(rows, 1, 256) * cxg::kRnSums * (size_t)cols * sizeof(float) + 256;
}

int cxg_residual_norm_bwd(const void* x, int64_t ldx, const void* f, int64_t ldf, const void* gate, int64_t ldg,
                          int gate_kind, int post_kind, const float* post_w, const float* post_b, int pre_kind,
                          const float* pre_w, float res_scale, float branch_scale, int64_t rows, int cols,
                          int stream_type, int branch_type, const float* stats, const void* dr, int64_t lddr,
                          const void* dy, int64_t lddy, void* dx, void* df, void* dgate, float* dpost_w,
                          float* dpost_b, float* dpre_w, float* dpre_b, void* workspace, size_t workspace_bytes,
                          void* stream) {
  using namespace cxg;
  RnArgs a{};
  a.x = x; a.ldx = ldx; a.f = f; a.ldf = ldf; a.gate = gate; a.ldg = ldg;
  a.gate_kind = gate_kind; a.post_kind = post_kind; a.pre_kind = pre_kind;
  a.post_w = post_w; a.post_b = post_b; a.pre_w = pre_w;
  a.res_scale = res_scale; a.branch_scale = branch_scale;
  a.rows = rows; a.cols = cols; a.stats = const_cast<float*>(stats);
  a.dr = dr; a.lddr = lddr; a.dy = dy; a.lddy = lddy; a.dx = dx; a.df = df;
  const int bad = rn_check(a, stream_type, branch_type);
  if (bad) return bad;
  CXG_REQUIRE(rows == 0 || (stats && ((uintptr_t)stats & 15) == 0), CXG_ERR_ARG, "stats missing or not 16-byte aligned");
  CXG_REQUIRE(rows == 0 || f || !df, CXG_ERR_ARG, "a branch gradient needs branch rows");
  CXG_REQUIRE(!dgate || gate_kind != CXG_GATE_NONE, CXG_ERR_ARG, "a gate gradient needs a gate");
  const bool channel = gate_kind == CXG_GATE_CHANNEL;
  const bool sums = dpost_w || dpost_b || dpre_w || dpre_b || (channel && dgate);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  RnFinal fin{};
  fin.cols = cols;
  fin.post_w = post_w; fin.post_b = post_b; fin.gate = channel ? static_cast<const float*>(gate) : nullptr;
  fin.branch_scale = branch_scale;
  fin.post = post_kind != CXG_NORM_NONE;
  fin.dgate = channel ? static_cast<float*>(dgate) : nullptr;
  fin.dpost_w = dpost_w; fin.dpost_b = dpost_b; fin.dpre_w = dpre_w; fin.dpre_b = dpre_b;
  if (sums) {
    const size_t need = cxg_residual_norm_workspace_bytes(rows, cols);
    CXG_REQUIRE(workspace && workspace_bytes >= need, CXG_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need,
                workspace_bytes);
    CXG_REQUIRE(((uintptr_t)workspace & 15) == 0, CXG_ERR_WORKSPACE, "workspace must be 16-byte aligned");
    a.partial = static_cast<float*>(workspace);
    fin.partial = a.partial;
  }
  if (!channel) a.dgate = dgate;
  if (rows > 0) {
    const int blocks = dispatch_bwd(a, stream_type, branch_type, st);
    if (blocks < 0) return blocks;
    fin.blocks = blocks;
  }
  if (sums) {
    hipLaunchKernelGGL(residual_norm_sums_kernel, dim3((unsigned)ceil_div(cols, kFinCols)), dim3(kFinThreads), 0,
                       st, fin);
    CXG_LAUNCH_CHECK("residual_norm_sums_kernel");
  }
  return CXG_OK;
}

}  // extern "C"
