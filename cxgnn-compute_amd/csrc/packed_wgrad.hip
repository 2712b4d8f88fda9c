// Weight gradient whose layer input is held in 8 bits (packed_rows.hip):
//
//   gW[r] (K x N)  =  sum over the rows i of segment r of  A[src(i), :]^T  (x)  G[dst(i), :]
//
// A row of A costs K bytes instead of 4 K.  Its values are code * 2^k with codes of at most 8
// significant bits, so they are bf16 numbers and multiply as they are; G goes in as bf16 parts that
// add up to it exactly -- one part for bf16, two for fp16 (11 bits), three for fp32 (24 bits), each
// the rounding of what the parts before it left -- and every part costs one product of
// v_mfma_f32_32x32x16_bf16 with fp32 accumulation.  The exponent range of bf16 is fp32's: no scaling.
//
// The reduction runs over the rows, and the matrix instruction wants eight consecutive reduction
// indices per lane, so both tiles are transposed on their way into LDS: a thread holds four columns
// of four consecutive rows and writes, per column, the four rows as one 8-byte store into
// [column][row] order (pitch 80 bytes).
//
// A block of four waves owns a 128 x 128 tile of gW over one chunk of a segment's rows, 64 x 64 per
// wave, 32 rows per step: while the waves multiply a step from LDS the rows of the next one are on
// their way into registers, and three blocks per CU cover each other's barriers.  128 columns of A
// are one scale group.  Tiles of a chunk sit side by side on one die, whose L2 then holds the
// chunk's rows for all of them.  Every block leaves its partial tile, a second kernel adds the
// chunks of a segment in order: no atomics.
//
// Row numbers that come from maps are fetched by the first wave two steps ahead into a ring in LDS
// and checked there; a row outside its matrix counts as no row.
#include "packed_rows.hpp"

namespace cxg {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));

constexpr int kPwThreads = 256;
constexpr int kPwXcds = 8;               // accelerator dies, one L2 each
constexpr int kPwRows = 32;              // rows per step
constexpr int kPwPitch = kPwRows + 8;    // LDS row pitch in bf16: 80 bytes
constexpr int kPwTile = 128;
constexpr int kPwBlocksPerCu = 3;
static_assert(kPwTile == kPrGroup, "one scale per row and tile");

struct PwArgs {
  const uint8_t* codes; const uint8_t* exps;
  int64_t a_rows;
  const void* g; int64_t ldg; int64_t g_rows;
  const int64_t* src; const int64_t* dst; const int64_t* seg;
  int64_t M;
  int K, N, R, pitch, groups;
  int64_t rows_per_chunk, chunks;
  float* partial;
};

template <typename TG> struct PwParts;
template <> struct PwParts<bf16_t> { static constexpr int value = 1; };
template <> struct PwParts<f16_t> { static constexpr int value = 2; };
template <> struct PwParts<float> { static constexpr int value = 3; };

// Rows of segment r, inside [0, M].
__device__ __forceinline__ void pw_segment(const int64_t* seg, int64_t M, int r, int64_t& b, int64_t& e) {
  b = seg ? seg[r] : 0;
  e = seg ? seg[r + 1] : M;
  b = b < 0 ? 0 : b;
  e = e > M ? M : e;
}
__device__ __forceinline__ int64_t pw_chunks(int64_t b, int64_t e, int64_t span) { return e > b ? (e - b + span - 1) / span : 0; }

// Chunk number -> first row and end of its rows; false past the last chunk.  Block-uniform.
__device__ __forceinline__ bool pw_locate(const PwArgs& a, int64_t chunk, int64_t& row0, int64_t& row_end) {
  int64_t t = chunk;
  for (int r = 0; r < a.R; ++r) {
    int64_t b, e;
    pw_segment(a.seg, a.M, r, b, e);
    const int64_t n = pw_chunks(b, e, a.rows_per_chunk);
    if (t < n) {
      row0 = b + t * a.rows_per_chunk;
      row_end = row0 + a.rows_per_chunk < e ? row0 + a.rows_per_chunk : e;
      return true;
    }
    t -= n;
  }
  return false;
}

__device__ __forceinline__ unsigned bf16_pair(float x, float y) {
  v2bf t;
  t[0] = (__bf16)x;
  t[1] = (__bf16)y;
  return __builtin_bit_cast(unsigned, t);
}

template <int FMT, typename TG, bool MAPPED>
__global__ __launch_bounds__(kPwThreads, kPwBlocksPerCu) void packed_wgrad_kernel(PwArgs a) {
  constexpr int NP = PwParts<TG>::value;
  __shared__ __attribute__((aligned(16))) uint16_t s_a[kPwTile][kPwPitch];
  __shared__ __attribute__((aligned(16))) uint16_t s_g[NP][kPwTile][kPwPitch];
  __shared__ int64_t s_ids[MAPPED ? 3 : 1][2][kPwRows];
  const int n_ct = (a.N + kPwTile - 1) / kPwTile, n_kt = (a.K + kPwTile - 1) / kPwTile, n_tile = n_ct * n_kt;
  const int64_t slot = blockIdx.x / kPwXcds;
  const int64_t chunk = (slot / n_tile) * kPwXcds + (blockIdx.x % kPwXcds);
  const int kt = (int)((slot % n_tile) / n_ct);
  const int n0 = (int)((slot % n_tile) % n_ct) * kPwTile, k0 = kt * kPwTile;
  int64_t row0 = 0, row_end = 0;
  if (chunk >= a.chunks || !pw_locate(a, chunk, row0, row_end)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform_i32(tid >> 6);
  const int steps = (int)((row_end - row0 + kPwRows - 1) / kPwRows);

  // staging: rows 4 mg .. 4 mg + 3 of a step, columns 4 c4 .. 4 c4 + 3 of the tile.  The low lane bits
  // select the rows: the lanes the LDS serves together then write different banks.
  const int mg = lane & 7, c4 = wave * 8 + (lane >> 3);
  const bool a_col = k0 + 4 * c4 < a.pitch;
  const uint8_t* const a_base = a.codes + k0 + 4 * c4;
  const uint8_t* const e_base = a.exps + kt;
  const TG* const g_base = static_cast<const TG*>(a.g);
  unsigned code[4];
  unsigned expo[4];
  RowPiece<TG, 4> gv[4];

  // MAPPED: lanes 0-31 of the first wave fetch the rows of A, lanes 32-63 those of G; a row that is
  // missing in either matrix is -1 in both
  auto fetch_ids = [&](int t) -> int64_t {
    const int64_t at = row0 + (int64_t)t * kPwRows + (lane & 31);
    int64_t id = -1;
    if (at < row_end) {
      const int64_t* const map = lane < 32 ? a.src : a.dst;
      id = map ? map[at] : at;
      if (id < 0 || id >= (lane < 32 ? a.a_rows : a.g_rows)) id = -1;
    }
    const int other = __shfl_xor(id >= 0 ? 1 : 0, 32, CXG_WAVE);
    return other ? id : -1;
  };
  auto load = [&](int t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      int64_t ia, ig;
      if constexpr (MAPPED) {
        ia = s_ids[t % 3][0][4 * mg + i];
        ig = s_ids[t % 3][1][4 * mg + i];
      } else {
        ia = row0 + (int64_t)t * kPwRows + 4 * mg + i;
        if (ia >= row_end) ia = -1;
        ig = ia;
      }
      code[i] = 0;
      expo[i] = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) gv[i].t[j] = (TG)0.f;
      if (ia >= 0) {
        if (a_col) code[i] = *reinterpret_cast<const unsigned*>(a_base + ia * a.pitch);
        expo[i] = e_base[ia * a.groups];
        gv[i].load(g_base + ig * a.ldg, n0 + 4 * c4, a.N);
      }
    }
  };
  auto stage = [&]() {
    float v[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) decode4<FMT>(code[i], packed_scale(expo[i]), v[i]);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      *reinterpret_cast<uint2*>(&s_a[4 * c4 + c][4 * mg]) = make_uint2(bf16_pair(v[0][c], v[1][c]), bf16_pair(v[2][c], v[3][c]));
#pragma unroll
    for (int i = 0; i < 4; ++i) gv[i].widen(v[i]);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float x[4] = {v[0][c], v[1][c], v[2][c], v[3][c]};
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const unsigned lo = bf16_pair(x[0], x[1]), hi = bf16_pair(x[2], x[3]);
        *reinterpret_cast<uint2*>(&s_g[p][4 * c4 + c][4 * mg]) = make_uint2(lo, hi);
        if (p + 1 < NP) {
          x[0] -= __uint_as_float(lo << 16);
          x[1] -= __uint_as_float(lo & 0xffff0000u);
          x[2] -= __uint_as_float(hi << 16);
          x[3] -= __uint_as_float(hi & 0xffff0000u);
        }
      }
    }
  };

  const int wk = (wave >> 1) * 64, wn = (wave & 1) * 64;
  v16f acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.f;

  int64_t next_ids = -1;
  if constexpr (MAPPED) {
    if (wave == 0) {
      s_ids[0][lane >> 5][lane & 31] = fetch_ids(0);
      s_ids[1][lane >> 5][lane & 31] = fetch_ids(1);
      next_ids = fetch_ids(2);
    }
    __syncthreads();
  }
  load(0);
  for (int t = 0; t < steps; ++t) {
    __syncthreads();                                     // every wave is done with the step before
    stage();
    if constexpr (MAPPED) {
      if (wave == 0) s_ids[(t + 2) % 3][lane >> 5][lane & 31] = next_ids;
    }
    __syncthreads();                                     // the step is staged, row numbers of t + 2 are there
    if (t + 1 < steps) load(t + 1);
    if constexpr (MAPPED) {
      if (wave == 0) next_ids = fetch_ids(t + 3);
    }
#pragma unroll
    for (int ms = 0; ms < kPwRows / 16; ++ms) {
      const int m = ms * 16 + (lane >> 5) * 8;
      v8bf fa[2], fg[NP][2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        fa[i] = *reinterpret_cast<const v8bf*>(&s_a[wk + 32 * i + (lane & 31)][m]);
#pragma unroll
        for (int p = 0; p < NP; ++p) fg[p][i] = *reinterpret_cast<const v8bf*>(&s_g[p][wn + 32 * i + (lane & 31)][m]);
      }
#pragma unroll
      for (int p = NP - 1; p >= 0; --p)                  // the small parts first
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (k0 + wk + 32 * i < a.K && n0 + wn + 32 * j < a.N)
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i], fg[p][j], acc[i][j], 0, 0, 0);
    }
  }
  float* const part = a.partial + (size_t)chunk * (size_t)a.K * (size_t)a.N;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int col = n0 + wn + 32 * j + (lane & 31);
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        const int k = k0 + wk + 32 * i + (q >> 2) * 8 + (lane >> 5) * 4 + (q & 3);
        if (k < a.K && col < a.N) part[(size_t)k * a.N + col] = acc[i][j][q];
      }
    }
}

// gw[r] = sum of the partial tiles of segment r's chunks: kPwSlices runs of chunks, each added by one
// thread per element, the runs in order.
constexpr int kPwElems = 16, kPwSlices = 16;

__global__ __launch_bounds__(kPwElems * kPwSlices) void packed_wgrad_sums_kernel(PwArgs a, float* __restrict__ gw, int64_t kn) {
  __shared__ float s[kPwSlices][kPwElems + 1];
  const int el = threadIdx.x % kPwElems, slice = threadIdx.x / kPwElems, r = blockIdx.y;
  const int64_t e = (int64_t)blockIdx.x * kPwElems + el;
  int64_t first = 0, b, end;
  for (int q = 0; q < r; ++q) {
    pw_segment(a.seg, a.M, q, b, end);
    first += pw_chunks(b, end, a.rows_per_chunk);
  }
  pw_segment(a.seg, a.M, r, b, end);
  int64_t last = first + pw_chunks(b, end, a.rows_per_chunk);
  last = last < a.chunks ? last : a.chunks;
  const int64_t per = last > first ? (last - first + kPwSlices - 1) / kPwSlices : 0;
  const int64_t c0 = first + slice * per, c1 = c0 + per < last ? c0 + per : last;
  float acc = 0.f;
  if (e < kn) {
    const float* const p = a.partial + e;
#pragma unroll 8
    for (int64_t c = c0; c < c1; ++c) acc += p[(size_t)c * kn];
  }
  s[slice][el] = acc;
  __syncthreads();
  if (slice == 0 && e < kn) {
    for (int q = 1; q < kPwSlices; ++q) acc += s[q][el];
    gw[(size_t)r * kn + e] = acc;
  }
}

// Rows per chunk: one round of blocks on the chip where a chunk is short (its 64 KB partial tile is
// written and read again, which a chunk should outweigh), up to four rounds where it is long (a last
// round that is not full then costs little).  A segment's last chunk is ragged: R of them per tile.
int64_t pw_chunk_rows(int64_t M, int K, int N, int R) {
  const int64_t tiles = ceil_div(K, kPwTile) * ceil_div(N, kPwTile);
  const int64_t slots = 256 * kPwBlocksPerCu;
  auto fill = [&](int64_t rounds) {                       // rows so that about `rounds` rounds are full
    int64_t chunks = ceil_div(slots * rounds, tiles) - R;
    if (chunks < 1) chunks = 1;
    return ceil_div(M, chunks);
  };
  const int64_t longest = fill(1), shortest = fill(4);
  int64_t rows = 2048;
  rows = rows > longest ? longest : rows < shortest ? shortest : rows;
  rows = ceil_div(rows, kPwRows) * kPwRows;
  return rows < 128 ? 128 : rows;
}

int64_t pw_chunk_count(int64_t M, int K, int N, int R) {
  return ceil_div(ceil_div(M, pw_chunk_rows(M, K, N, R)) + R, kPwXcds) * kPwXcds;
}

}  // namespace
}  // namespace cxg

extern "C" {

size_t cxg_packed_wgrad_workspace_bytes(int64_t M, int K, int N, int R) {
  if (M < 0 || K < 1 || N < 1 || R < 1) return 0;
  return (size_t)cxg::pw_chunk_count(M, K, N, R) * (size_t)K * (size_t)N * sizeof(float) + 256;
}

int cxg_packed_wgrad(const uint8_t* codes, const uint8_t* exps, int fmt, int64_t a_rows, const void* g, int64_t ldg,
                     int g_type, int64_t g_rows, const int64_t* src_idx, const int64_t* dst_idx, const int64_t* seg_ptr,
                     int64_t M, int K, int N, int R, float* gw, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace cxg;
  CXG_REQUIRE(M >= 0 && K >= 1 && N >= 1 && R >= 1 && a_rows >= 0 && g_rows >= 0, CXG_ERR_ARG, "bad M/K/N/R/rows");
  CXG_REQUIRE(fmt == CXG_PACK_INT8 || fmt == CXG_PACK_E4M3, CXG_ERR_ARG, "unknown 8-bit format");
  CXG_REQUIRE(value_type_ok(g_type), CXG_ERR_ARG, "unknown value type");
  CXG_REQUIRE(gw, CXG_ERR_ARG, "null gw");
  CXG_REQUIRE(seg_ptr || R == 1, CXG_ERR_ARG, "several segments need seg_ptr");
  CXG_REQUIRE(M == 0 || (codes && exps && g), CXG_ERR_ARG, "null codes/exps/g");
  CXG_REQUIRE(ldg >= 0, CXG_ERR_ARG, "negative row stride");
  CXG_REQUIRE(K <= kPrMaxCols && N <= kPrMaxCols && R <= 65535, CXG_ERR_UNSUPPORTED, "K, N or R too large");
  CXG_REQUIRE(((uintptr_t)codes & 15) == 0, CXG_ERR_ARG, "codes must be 16-byte aligned");
  CXG_REQUIRE(((uintptr_t)g & (value_bytes(g_type) - 1)) == 0, CXG_ERR_ARG, "g is not aligned to its values");
  // without a map row i is row i: the matrices have to have M of them
  CXG_REQUIRE((src_idx || a_rows >= M) && (dst_idx || g_rows >= M), CXG_ERR_ARG, "fewer rows than M");
  const size_t need = cxg_packed_wgrad_workspace_bytes(M, K, N, R);
  CXG_REQUIRE(workspace && workspace_bytes >= need, CXG_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need,
              workspace_bytes);
  CXG_REQUIRE(((uintptr_t)workspace & 255) == 0, CXG_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int64_t chunks = pw_chunk_count(M, K, N, R);
  const int64_t tiles = ceil_div(K, kPwTile) * ceil_div(N, kPwTile);
  CXG_REQUIRE(chunks * tiles < ((int64_t)1 << 31), CXG_ERR_UNSUPPORTED, "too many tiles for one launch");
  const PwArgs a{codes, exps, a_rows, g, ldg, g_rows, src_idx, dst_idx, seg_ptr, M, K, N, R, packed_pitch(K), packed_groups(K),
                 pw_chunk_rows(M, K, N, R), chunks, static_cast<float*>(workspace)};
  const bool mapped = src_idx || dst_idx;
#define CXG_PW_LAUNCH(FMT, TG)                                                                             \
  do {                                                                                                     \
    if (mapped) hipLaunchKernelGGL((packed_wgrad_kernel<FMT, TG, true>), grid, block, 0, st, a);           \
    else hipLaunchKernelGGL((packed_wgrad_kernel<FMT, TG, false>), grid, block, 0, st, a);                 \
  } while (0)
  if (M > 0) {
    const dim3 grid((unsigned)(chunks * tiles)), block(kPwThreads);
    if (fmt == CXG_PACK_INT8) {
      if (g_type == CXG_F32) CXG_PW_LAUNCH(CXG_PACK_INT8, float);
      else if (g_type == CXG_BF16) CXG_PW_LAUNCH(CXG_PACK_INT8, bf16_t);
      else CXG_PW_LAUNCH(CXG_PACK_INT8, f16_t);
    } else {
      if (g_type == CXG_F32) CXG_PW_LAUNCH(CXG_PACK_E4M3, float);
      else if (g_type == CXG_BF16) CXG_PW_LAUNCH(CXG_PACK_E4M3, bf16_t);
      else CXG_PW_LAUNCH(CXG_PACK_E4M3, f16_t);
    }
    CXG_LAUNCH_CHECK("packed_wgrad_kernel");
  }
#undef CXG_PW_LAUNCH
  const int64_t kn = (int64_t)K * N;
  CXG_REQUIRE(ceil_div(kn, kPwElems) < ((int64_t)1 << 31), CXG_ERR_UNSUPPORTED, "gw too large for one launch");
  hipLaunchKernelGGL(packed_wgrad_sums_kernel, dim3((unsigned)ceil_div(kn, kPwElems), (unsigned)R),
                     dim3(kPwElems * kPwSlices), 0, st, a, gw, kn);
  CXG_LAUNCH_CHECK("packed_wgrad_sums_kernel");
  return CXG_OK;
}

}  // extern "C"
