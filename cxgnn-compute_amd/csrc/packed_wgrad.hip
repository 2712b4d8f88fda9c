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
// indices per lane, so both tiles are transposed on their way into LDS: a thread holds some columns
// of four consecutive rows and writes, per column, the four rows as one 8-byte store into
// [column][row] order (pitch 80 or 144 bytes).
//
// A block of four waves owns a tile of gW (64 to 256 columns of A by 64 or 128 of G) over one chunk of a
// segment's rows, 64 or 32 rows per step: while the waves multiply a step from LDS the rows of the next
// one are on their way into registers, and the blocks of a CU cover each other's barriers.  128 columns of A are
// one scale group.  Tiles of a chunk sit side by side on one die, whose L2 then holds the chunk's
// rows for all of them.  Every block leaves its partial tile (and, if wanted, the sums of the rows of
// G that pass through it, the bias gradient), a second kernel adds the chunks of a segment in order:
// no atomics.
//
// Row numbers that come from maps are fetched by the first wave two steps ahead into a ring in LDS
// and checked there; a row outside its matrix counts as no row.  Exponent bytes come through LDS too,
// one load of the first wave per step.
//
// Measured, both kernels: 1 M rows x 128 x 128 of 16 types through row maps, bf16 G: 103 us, memory bound
// (0.40 GB of rows and maps, 32 MB of partial tiles written and read); 2,332,486 x 512 x 512 of 7 types,
// fp32 G: 3.6 ms = 340 useful TFLOP/s, three times that on the matrix cores, which are busy half of the time
// at the clock that the board's power allows (1.83 GHz).
#include "packed_rows.hpp"

namespace cxg {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));

constexpr int kPwThreads = 256;
constexpr int kPwXcds = 8;               // accelerator dies, one L2 each
constexpr int64_t kPwMaxBlocks = ((int64_t)1 << 32) / kPwThreads;     // a launch has fewer than 2^32 threads
constexpr int kPwFront = 8;              // columns in front of a tile of G: at least what a thread stages

// Shape of a block: KT columns of A, NT of G, ROWS rows per step, BLOCKS of them per CU.
template <int KT_, int NT_, int ROWS_, int BLOCKS_> struct PwShape {
  static constexpr int KT = KT_, NT = NT_, ROWS = ROWS_, BLOCKS = BLOCKS_;
  static constexpr int PITCH = ROWS + 8;                      // LDS pitch in bf16: 80 or 144 bytes
  static constexpr int MG = ROWS / 4;                         // groups of four rows
  static constexpr int CA = KT * ROWS / (4 * kPwThreads);     // columns of A / G that a thread stages
  static constexpr int CG = NT * ROWS / (4 * kPwThreads);
  static constexpr int MI = KT / 64, NJ = NT / 64;            // 32 x 32 blocks of a wave along K and N
};

struct PwArgs {
  const uint8_t* codes; const uint8_t* exps;
  int64_t a_rows;
  const void* g; int64_t ldg; int64_t g_rows;
  const int64_t* src; const int64_t* dst; const int64_t* seg;
  int64_t M;
  int K, N, R, pitch, groups;
  int64_t rows_per_chunk, chunks;
  float* partial;          // [chunks][K * N], then N column sums of G if they are wanted
  int64_t stride;          // floats per chunk
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

// The chunks of 64 segments from r0 on, one segment per lane: those of this lane's segment, and of the ones before
// it among the 64.  All lanes of the wave have to be active.
__device__ __forceinline__ int64_t pw_scan(const PwArgs& a, int r0, int64_t& before) {
  const int r = r0 + (int)(threadIdx.x & (CXG_WAVE - 1));
  int64_t b = 0, e = 0;
  if (r < a.R) pw_segment(a.seg, a.M, r, b, e);
  const int64_t n = pw_chunks(b, e, a.rows_per_chunk);
  int64_t sum = n;
#pragma unroll
  for (int d = 1; d < CXG_WAVE; d *= 2) {
    const int64_t o = __shfl_up(sum, d, CXG_WAVE);
    sum += (int)(threadIdx.x & (CXG_WAVE - 1)) >= d ? o : 0;
  }
  before = sum - n;
  return n;
}

// Up to this many segments are gone through one after another (30,289 x 529 x 505 of 3 types: 64 us, 66 us by the
// scan; 100,000 x 128 x 128 of 12: 25 us, 23 us by the scan), more of them 64 at a time (1 M x 128 x 128 of 600 types:
// 253 us, one after another 3.6 ms).
constexpr int kPwFewSegments = 8;

// Chunk number -> first row and end of its rows; false past the last chunk.  Block-uniform.
__device__ __forceinline__ bool pw_locate(const PwArgs& a, int64_t chunk, int64_t& row0, int64_t& row_end) {
  int64_t t = chunk, b = 0, e = 0;
  bool found = false;
  if (a.R <= kPwFewSegments) {
    for (int r = 0; r < a.R && !found; ++r) {
      pw_segment(a.seg, a.M, r, b, e);
      const int64_t n = pw_chunks(b, e, a.rows_per_chunk);
      found = t < n;
      if (!found) t -= n;
    }
  } else {
    for (int r0 = 0; r0 < a.R && !found; r0 += CXG_WAVE) {
      int64_t before;
      const int64_t n = pw_scan(a, r0, before);
      const unsigned long long here = __ballot(t >= before && t < before + n);
      found = here != 0;
      const int lane = found ? __ffsll(here) - 1 : CXG_WAVE - 1;
      t -= uniform_i64(__shfl(found ? before : before + n, lane, CXG_WAVE));
      if (found) pw_segment(a.seg, a.M, uniform_i32(r0 + lane), b, e);
    }
  }
  row0 = b + t * a.rows_per_chunk;
  row_end = row0 + a.rows_per_chunk < e ? row0 + a.rows_per_chunk : e;
  return found;
}

// Chunks of the segments before segment r.
__device__ __forceinline__ int64_t pw_first_chunk(const PwArgs& a, int r) {
  int64_t first = 0;
  if (r <= kPwFewSegments) {
    for (int q = 0; q < r; ++q) {
      int64_t b, e;
      pw_segment(a.seg, a.M, q, b, e);
      first += pw_chunks(b, e, a.rows_per_chunk);
    }
    return first;
  }
  for (int r0 = 0; r0 < r; r0 += CXG_WAVE) {
    int64_t before;
    const int64_t n = pw_scan(a, r0, before);
    const int last = r - r0 < CXG_WAVE ? r - r0 - 1 : CXG_WAVE - 1;
    first += uniform_i64(__shfl(before + n, last, CXG_WAVE));
  }
  return first;
}

__device__ __forceinline__ unsigned bf16_pair(float x, float y) {
  v2bf t;
  t[0] = (__bf16)x;
  t[1] = (__bf16)y;
  return __builtin_bit_cast(unsigned, t);
}

template <int FMT, typename TG, bool MAPPED, typename S, bool TINY>
__global__ __launch_bounds__(kPwThreads, S::BLOCKS) void packed_wgrad_kernel(PwArgs a) {
  constexpr int NP = PwParts<TG>::value;
  constexpr int ROWS = S::ROWS, MG = S::MG, CA = S::CA, CG = S::CG, MI = S::MI, NJ = S::NJ, PITCH = S::PITCH;
  constexpr int NG = (S::KT + kPrGroup - 1) / kPrGroup;                                   // scale groups of a tile
  __shared__ __attribute__((aligned(16))) uint16_t s_a[S::KT][PITCH];
  __shared__ __attribute__((aligned(16))) uint16_t s_gp[NP][kPwFront + S::NT][PITCH];   // kPwFront columns of slack in front
  __shared__ __attribute__((aligned(16))) uint8_t s_exp[2][NG][ROWS];                     // exponent bytes of a step's rows
  __shared__ int64_t s_off[MAPPED ? 3 : 1][2][MAPPED ? ROWS : 1];                         // ring: offsets of the rows of codes and g
  __shared__ unsigned long long s_live[3];                                                // and which of them are there
  const int n_ct = (a.N + S::NT - 1) / S::NT, n_kt = (a.K + S::KT - 1) / S::KT, n_tile = n_ct * n_kt;
  const int64_t slot = blockIdx.x / kPwXcds;
  const int64_t chunk = (slot / n_tile) * kPwXcds + (blockIdx.x % kPwXcds);
  const int k0 = (int)((slot % n_tile) / n_ct) * S::KT;
  const int n0 = (int)((slot % n_tile) % n_ct) * S::NT;
  int64_t row0 = 0, row_end = 0;
  if (chunk >= a.chunks || !pw_locate(a, chunk, row0, row_end)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform_i32(tid >> 6);
  const int steps = (int)((row_end - row0 + ROWS - 1) / ROWS);
  const int last_rows = (int)(row_end - row0 - (int64_t)(steps - 1) * ROWS);

  // staging: rows 4 mg .. 4 mg + 3 of a step, CA columns of A and CG of G.  The low lane bits select the
  // rows: the lanes the LDS serves together then write different banks.
  // All loads of the loop are unconditional, so that none waits for another: columns of A past the
  // pitch read column k0, a piece of G that would pass N is moved back to end there (it then writes the
  // columns it shares with its neighbour twice, the same values, and those in front of the tile into the
  // slack), rows that are not there read one that is and are cleared when they are staged.  What is staged
  // for columns of A or G that do not exist only reaches rows and columns of gW that do not exist.
  const int mg = lane % MG, cg = wave * (64 / MG) + lane / MG;
  const int ka = k0 + CA * cg;
  const uint8_t* const a_base = a.codes + (ka < a.pitch ? ka : k0);
  int ng = n0 + CG * cg;
  if (!TINY && ng + CG > a.N) ng = a.N - CG;                    // N >= CG
  const int gcol = TINY ? kPwFront + CG * cg : kPwFront + ng - n0 < 0 ? 0 : kPwFront + ng - n0;
  const TG* const g_base = static_cast<const TG*>(a.g) + (TINY ? 0 : ng);
  // exponent bytes: lane of the first wave -> row and NE groups
  constexpr int NE = (NG * ROWS + 63) / 64;
  int e_grp[NE];
#pragma unroll
  for (int j = 0; j < NE; ++j) {
    e_grp[j] = k0 / kPrGroup + lane / ROWS + j;
    e_grp[j] = e_grp[j] < a.groups ? e_grp[j] : a.groups - 1;
  }
  unsigned code[4][CA / 4];
  TG gv[4][CG];
  unsigned expo[NE] = {};
  static_assert(ROWS <= 64 && (NE == 1 || ROWS == 64), "a lane per row, or per row and group");

  auto load_row = [&](int i, int64_t oa, int64_t og) {
    typedef unsigned piece_t __attribute__((ext_vector_type(CA / 4)));
    const piece_t w = *reinterpret_cast<const piece_t*>(a_base + oa);
#pragma unroll
    for (int j = 0; j < CA / 4; ++j) code[i][j] = w[j];
    if constexpr (TINY) {
#pragma unroll
      for (int j = 0; j < CG; ++j) gv[i][j] = g_base[og + (ng + j < a.N ? ng + j : a.N - 1)];
    } else {
      constexpr int V = 16 / (int)sizeof(TG) < CG ? 16 / (int)sizeof(TG) : CG;
#pragma unroll
      for (int q = 0; q < CG / V; ++q) {
        const auto p = *reinterpret_cast<const typename RowPiece<TG, V>::loose_t*>(g_base + og + q * V);
#pragma unroll
        for (int j = 0; j < V; ++j) gv[i][q * V + j] = p[j];
      }
    }
  };
  // MAPPED: lane r of the first wave loads the map entries of row r of step t (of the last row behind the
  // end), and turns them into offsets a step later
  const int64_t* const map_a = a.src ? a.src : a.dst;
  const int64_t* const map_g = a.dst ? a.dst : a.src;
  auto clamped = [&](int t) -> int64_t {
    const int64_t at = row0 + (int64_t)t * ROWS + (lane & (ROWS - 1));
    return at < row_end ? at : row_end - 1;
  };
  // (and returns the offset of the row's exponent bytes)
  auto put = [&](int t, int64_t ia, int64_t ig) -> int64_t {
    const int64_t at = row0 + (int64_t)t * ROWS + (lane & (ROWS - 1));
    ia = a.src ? ia : at;
    ig = a.dst ? ig : at;
    const bool ok = at < row_end && ia >= 0 && ia < a.a_rows && ig >= 0 && ig < a.g_rows;
    const unsigned long long live = __ballot(ok);
    if (lane < ROWS) {
      s_off[t % 3][0][lane] = ok ? ia * a.pitch : 0;
      s_off[t % 3][1][lane] = ok ? ig * a.ldg : 0;
    }
    if (lane == 0) s_live[t % 3] = live;
    return ok ? ia * a.groups : 0;
  };
  // rows of step t into registers; behind the last step the last one again
  const int64_t a_off = (int64_t)(4 * mg) * a.pitch, g_off = (int64_t)(4 * mg) * a.ldg;
  auto load = [&](int t, int64_t off_exp) {
    t = t < steps ? t : steps - 1;
    const int64_t first = row0 + (int64_t)t * ROWS;
    const int left = t + 1 < steps ? ROWS : last_rows;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (MAPPED) {
        load_row(i, s_off[t % 3][0][4 * mg + i], s_off[t % 3][1][4 * mg + i]);
      } else {
        // row first + 4 mg + i, or first + i, or first.  (A vector multiplication per row and step, the plain
        // form of this, costs as much as decoding A.)
        const bool on = 4 * mg + i < left;
        const int64_t near = first + (i < left ? i : 0);
        load_row(i, near * a.pitch + (on ? a_off : 0), near * a.ldg + (on ? g_off : 0));
      }
    }
    if (wave == 0) {
      if constexpr (!MAPPED) {
        const int row = lane & (ROWS - 1);
        off_exp = (first + (row < left ? row : 0)) * a.groups;
      }
#pragma unroll
      for (int j = 0; j < NE; ++j) expo[j] = a.exps[off_exp + e_grp[j]];
    }
  };
  auto put_exp = [&](int t) {
    if (wave == 0 && lane < NG * ROWS) {
#pragma unroll
      for (int j = 0; j < NE; ++j) s_exp[t & 1][lane / ROWS + j][lane & (ROWS - 1)] = (uint8_t)expo[j];
    }
  };
  const bool sums = a.stride > (int64_t)a.K * a.N && k0 == 0;    // this block also adds up the rows of its columns of G
  float colsum[CG];
#pragma unroll
  for (int c = 0; c < CG; ++c) colsum[c] = 0.f;
  auto stage = [&](int t) {
    unsigned exps = *reinterpret_cast<const unsigned*>(&s_exp[t & 1][NG == 1 ? 0 : CA * cg / kPrGroup][4 * mg]);
    unsigned live;                                       // which of this thread's four rows are there
    bool whole;
    if constexpr (MAPPED) {
      const unsigned long long m = s_live[t % 3];
      live = (unsigned)(m >> (4 * mg)) & 15u;
      whole = (ROWS == 64 ? m : m | 0xffffffff00000000ull) == ~0ull;
    } else {
      const int here = t + 1 < steps ? ROWS : last_rows;
      whole = here == ROWS;
      const int n = here - 4 * mg;
      live = n >= 4 ? 15u : n <= 0 ? 0u : (1u << n) - 1u;
    }
    if (!whole) {
      // a row that is not there is a row of zeros on both sides (0 times something not finite is NaN)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool on = (live >> i) & 1u;
        exps &= on ? ~0u : ~(0xffu << (8 * i));
#pragma unroll
        for (int j = 0; j < CA / 4; ++j) code[i][j] = on ? code[i][j] : 0u;
#pragma unroll
        for (int j = 0; j < CG; ++j) gv[i][j] = on ? gv[i][j] : (TG)0.f;
      }
    }
#pragma unroll
    for (int q = 0; q < CA / 4; ++q) {
      float v[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) decode4<FMT>(code[i][q], packed_scale((exps >> (8 * i)) & 0xffu), v[i]);
#pragma unroll
      for (int c = 0; c < 4; ++c)
        *reinterpret_cast<uint2*>(&s_a[CA * cg + 4 * q + c][4 * mg]) =
            make_uint2(bf16_pair(v[0][c], v[1][c]), bf16_pair(v[2][c], v[3][c]));
    }
    if (sums) {
#pragma unroll
      for (int c = 0; c < CG; ++c) colsum[c] += ((float)gv[0][c] + (float)gv[1][c]) + ((float)gv[2][c] + (float)gv[3][c]);
    }
#pragma unroll
    for (int c = 0; c < CG; ++c) {
      if constexpr (NP == 1) {
        // bf16 values go through as they are
        uint2 o;
        o.x = (unsigned)__builtin_bit_cast(uint16_t, gv[0][c]) | ((unsigned)__builtin_bit_cast(uint16_t, gv[1][c]) << 16);
        o.y = (unsigned)__builtin_bit_cast(uint16_t, gv[2][c]) | ((unsigned)__builtin_bit_cast(uint16_t, gv[3][c]) << 16);
        *reinterpret_cast<uint2*>(&s_gp[0][gcol + c][4 * mg]) = o;
      } else {
        float x[4] = {(float)gv[0][c], (float)gv[1][c], (float)gv[2][c], (float)gv[3][c]};
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          const unsigned lo = bf16_pair(x[0], x[1]), hi = bf16_pair(x[2], x[3]);
          *reinterpret_cast<uint2*>(&s_gp[p][gcol + c][4 * mg]) = make_uint2(lo, hi);
          if (p + 1 < NP) {
            x[0] -= __uint_as_float(lo << 16);
            x[1] -= __uint_as_float(lo & 0xffff0000u);
            x[2] -= __uint_as_float(hi << 16);
            x[3] -= __uint_as_float(hi & 0xffff0000u);
          }
        }
      }
    }
  };

  const int wk = (wave >> 1) * (S::KT / 2), wn = (wave & 1) * (S::NT / 2);
  v16f acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.f;
  const bool active = k0 + wk < a.K && n0 + wn < a.N;           // else nothing of this wave's part lies inside gW

  int64_t id_a = 0, id_g = 0, off_now = 0, off_next = 0;
  if constexpr (MAPPED) {
    if (wave == 0) {
      off_now = put(0, map_a[clamped(0)], map_g[clamped(0)]);
      off_next = put(1, map_a[clamped(1)], map_g[clamped(1)]);
      id_a = map_a[clamped(2)];
      id_g = map_g[clamped(2)];
    }
    __syncthreads();
  }
  load(0, off_now);
  for (int t = 0; t < steps; ++t) {
    put_exp(t);
    __syncthreads();                                     // every wave is done with the step before
    stage(t);
    if constexpr (MAPPED) {
      off_now = off_next;
      if (wave == 0) off_next = put(t + 2, id_a, id_g);
    }
    __syncthreads();                                     // the step is staged, the rows of t + 2 are known
    load(t + 1, off_now);
    if constexpr (MAPPED) {
      if (wave == 0) {
        id_a = map_a[clamped(t + 3)];
        id_g = map_g[clamped(t + 3)];
      }
    }
    __builtin_amdgcn_s_setprio(1);                       // ahead of the other block's staging: 3.72 -> 3.65 ms at 512 x 512
#pragma unroll
    for (int ms = 0; ms < ROWS / 16; ++ms) {
      if (!active) break;
      const int m = ms * 16 + (lane >> 5) * 8;
      v8bf fa[MI], fg[NP][NJ];
#pragma unroll
      for (int i = 0; i < MI; ++i) fa[i] = *reinterpret_cast<const v8bf*>(&s_a[wk + 32 * i + (lane & 31)][m]);
#pragma unroll
      for (int p = NP - 1; p >= 0; --p)
#pragma unroll
        for (int j = 0; j < NJ; ++j) fg[p][j] = *reinterpret_cast<const v8bf*>(&s_gp[p][kPwFront + wn + 32 * j + (lane & 31)][m]);
#pragma unroll
      for (int p = NP - 1; p >= 0; --p)                  // the small parts first
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i], fg[p][j], acc[i][j], 0, 0, 0);
    }
    __builtin_amdgcn_s_setprio(0);
  }
  float* const part = a.partial + (size_t)chunk * (size_t)a.stride;
  if (sums) {
    // over the groups of four rows, through the LDS that held G (a column that two threads hold, they hold alike)
    float (*const s_sum)[kPwFront + S::NT] = reinterpret_cast<float (*)[kPwFront + S::NT]>(&s_gp[0][0][0]);
    static_assert(sizeof(float) * MG * (kPwFront + S::NT) <= sizeof(s_gp), "the sums fit");
    __syncthreads();
#pragma unroll
    for (int c = 0; c < CG; ++c) s_sum[mg][gcol + c] = colsum[c];
    __syncthreads();
    if (tid < S::NT && n0 + tid < a.N) {
      float v = 0.f;
#pragma unroll
      for (int q = 0; q < MG; ++q) v += s_sum[q][kPwFront + tid];
      part[(size_t)a.K * a.N + n0 + tid] = v;
    }
  }
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int col = n0 + wn + 32 * j + (lane & 31);
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        const int k = k0 + wk + 32 * i + (q >> 2) * 8 + (lane >> 5) * 4 + (q & 3);
        if (k < a.K && col < a.N) part[(size_t)k * a.N + col] = acc[i][j][q];
      }
    }
}

// gw[r] (and the column sums gb[r]) = sum of the partial results of segment r's chunks: SL runs of chunks,
// each added by one thread per V consecutive elements, the runs in order.
template <int V, int SL>
__global__ __launch_bounds__(256) void packed_wgrad_sums_kernel(PwArgs a, float* __restrict__ gw, float* __restrict__ gb) {
  constexpr int EL = 256 / SL;
  typedef float vec_t __attribute__((ext_vector_type(V)));
  __shared__ vec_t s[SL][EL];
  const int el = threadIdx.x % EL, slice = threadIdx.x / EL, r = blockIdx.y;
  const int64_t e = ((int64_t)blockIdx.x * EL + el) * V;
  int64_t b, end;
  const int64_t first = pw_first_chunk(a, r);
  pw_segment(a.seg, a.M, r, b, end);
  int64_t last = first + pw_chunks(b, end, a.rows_per_chunk);
  last = last < a.chunks ? last : a.chunks;
  const int64_t per = last > first ? (last - first + SL - 1) / SL : 0;
  const int64_t c0 = first + slice * per, c1 = c0 + per < last ? c0 + per : last;
  vec_t acc = 0.f;
  if (e < a.stride) {
    const float* const p = a.partial + e;
#pragma unroll 8
    for (int64_t c = c0; c < c1; ++c) acc += *reinterpret_cast<const vec_t*>(p + (size_t)c * a.stride);
  }
  s[slice][el] = acc;
  __syncthreads();
  if (slice == 0 && e < a.stride) {
#pragma unroll
    for (int q = 1; q < SL; ++q) acc += s[q][el];
    const int64_t kn = (int64_t)a.K * a.N;
    float* const dst = e < kn ? gw + (size_t)r * kn + e : gb + (size_t)r * a.N + (e - kn);
    *reinterpret_cast<vec_t*>(dst) = acc;
  }
}

// Inputs of at most 128 columns: 128 x 128 tiles, 64 rows per step, two blocks per CU (32 rows and three
// blocks: 114 against 97 us for 1 M rows x 128 x 128 of 16 types in bf16, 55 against 50 us for 169,343 x
// 128 x 256 in fp32; this kernel alone).  Wider inputs: 256 x 128 tiles, so that a step of G is staged once
// per 256 columns of A (2.33 M x 512 x 512 in fp32: 3.6 ms; 512 x 128 tiles of one block of eight waves per
// CU, staging into a second buffer while the other half multiplies: 4.1 ms).  At most 64 columns of G: tiles
// of 64, which leave room for more rows on their way (2.45 M x 256 x 47 in fp32 390 -> 290 us, 1 M x 64 x 8
// 94 -> 67 us, against 128).
typedef PwShape<64, 64, 64, 3> PwSmall;
typedef PwShape<128, 64, 64, 3> PwNarrowFew;
typedef PwShape<256, 64, 64, 2> PwWideFew;
typedef PwShape<128, 128, 64, 2> PwNarrow;
typedef PwShape<256, 128, 32, 2> PwWide;

// run(shape) with the shape for K columns of A and N of G
template <typename F> auto pw_shaped(int K, int N, F run) {
  if (N <= 64) return K <= 64 ? run(PwSmall{}) : K <= 128 ? run(PwNarrowFew{}) : run(PwWideFew{});
  return K <= 128 ? run(PwNarrow{}) : run(PwWide{});
}

// Rows per chunk: one round of blocks on the chip where a chunk is short (its partial tile is written
// and read again, which a chunk should outweigh), up to two rounds where it is long (a last round
// that is not full then costs little).  The tiles of a chunk run on one die: a round is full with as many
// chunks as fit on each die whole, the same number everywhere, the ragged last chunks of the segments among
// them (30,289 x 529 x 505 of 3 types, 12 tiles, in bf16: 42 chunks, six on two of the dies, 108 us; 40
// chunks, five on each, 76 us).  Ragged chunks have a place as long as they take at most half of it.  With more
// segments than that most chunks are short, they come on top, and a long segment is still split over the chip
// (1 M x 512 x 512 of 200 types, half of the rows in one, in fp32: 1.95 ms; with the place taken by ragged
// chunks a chunk was all rows and the long segment ran on eight blocks, 37.7 ms).  A chunk has at most kPwMaxChunk
// rows, whatever the width of gW: as many products, times the parts of G, are the longest sum in one fp32
// accumulator.  (At half as many rows 2 M x 1,024 x 1,024 in bf16 takes 5.3 ms for 5.0, partial tiles.)
constexpr int64_t kPwMaxChunk = 65536;

int64_t pw_tiles(int K, int N) {
  return pw_shaped(K, N, [&](auto s) { return ceil_div(K, s.KT) * ceil_div(N, s.NT); });
}

int64_t pw_chunk_rows(int64_t M, int K, int N, int R) {
  const int64_t tiles = pw_tiles(K, N);
  const int64_t slots = 256 / kPwXcds * pw_shaped(K, N, [](auto s) { return (int64_t)s.BLOCKS; });   // of one die
  auto fill = [&](int64_t rounds) {                       // rows so that about `rounds` rounds are full
    const int64_t each = slots * rounds / tiles;          // chunks per die
    const int64_t place = kPwXcds * (each < 1 ? 1 : each), ragged = R - 1;
    return ceil_div(M, ragged <= place / 2 ? place - ragged : place);
  };
  const int64_t longest = fill(1), shortest = fill(2);
  int64_t rows = 2048;
  rows = rows > longest ? longest : rows < shortest ? shortest : rows;
  if (rows > kPwMaxChunk) rows = ceil_div(M, kPwXcds * ceil_div(M, kPwXcds * kPwMaxChunk));   // as many on each die
  return rows < 1 ? 64 : ceil_div(rows, (int64_t)64) * 64;
}

int64_t pw_chunk_count(int64_t M, int K, int N, int R) {
  return ceil_div(ceil_div(M, pw_chunk_rows(M, K, N, R)) + R - 1, kPwXcds) * kPwXcds;
}

template <int FMT, typename TG, typename S, bool TINY> void pw_launch(const PwArgs& a, int64_t chunks, hipStream_t st) {
  const int64_t tiles = ceil_div(a.K, S::KT) * ceil_div(a.N, S::NT);
  const dim3 grid((unsigned)(chunks * tiles)), block(kPwThreads);
  static_assert(S::CG <= kPwFront, "the slack in front of a tile of G");
  if (a.src || a.dst) hipLaunchKernelGGL((packed_wgrad_kernel<FMT, TG, true, S, TINY>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((packed_wgrad_kernel<FMT, TG, false, S, TINY>), grid, block, 0, st, a);
}
template <int FMT, typename TG> void pw_launch_shape(const PwArgs& a, int64_t chunks, hipStream_t st) {
  pw_shaped(a.K, a.N, [&](auto s) {
    // 64 rows per step wherever the LDS of a CU then holds BLOCKS blocks (all but 256 x 128 in fp32): half the
    // barriers and loads twice as far apart (300,000 x 1,024 x 1,024 in bf16 1,103 -> 770 us, in fp16 1,334 -> 1,135 us
    // against 32 rows)
    using W = decltype(s);
    constexpr int NP = PwParts<TG>::value;
    constexpr int lds64 = (W::KT + NP * (kPwFront + W::NT)) * 2 * (64 + 8) + 3500;    // tiles; maps and exponent bytes
    using S = PwShape<W::KT, W::NT, lds64 * W::BLOCKS <= 160 * 1024 ? 64 : W::ROWS, W::BLOCKS>;
    if constexpr (S::NT <= 64) {
      if (a.N < S::CG) return pw_launch<FMT, TG, S, true>(a, chunks, st);
    }
    pw_launch<FMT, TG, S, false>(a, chunks, st);
  });
}
template <int FMT> void pw_launch_type(const PwArgs& a, int g_type, int64_t chunks, hipStream_t st) {
  if (g_type == CXG_F32) pw_launch_shape<FMT, float>(a, chunks, st);
  else if (g_type == CXG_BF16) pw_launch_shape<FMT, bf16_t>(a, chunks, st);
  else pw_launch_shape<FMT, f16_t>(a, chunks, st);
}

template <int V, int SL> void pw_launch_sums(const PwArgs& a, float* gw, float* gb, hipStream_t st) {
  hipLaunchKernelGGL((packed_wgrad_sums_kernel<V, SL>), dim3((unsigned)ceil_div(a.stride, V * (256 / SL)), (unsigned)a.R),
                     dim3(256), 0, st, a, gw, gb);
}

}  // namespace
}  // namespace cxg

extern "C" {

size_t cxg_packed_wgrad_workspace_bytes(int64_t M, int K, int N, int R) {
  if (M < 0 || K < 1 || N < 1 || R < 1) return 0;
  return (size_t)cxg::pw_chunk_count(M, K, N, R) * ((size_t)K + 1) * (size_t)N * sizeof(float) + 256;
}

int cxg_packed_wgrad(const uint8_t* codes, const uint8_t* exps, int fmt, int64_t a_rows, const void* g, int64_t ldg,
                     int g_type, int64_t g_rows, const int64_t* src_idx, const int64_t* dst_idx, const int64_t* seg_ptr,
                     int64_t M, int K, int N, int R, float* gw, float* gb, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace cxg;
  CXG_REQUIRE(M >= 0 && K >= 1 && N >= 1 && R >= 1 && a_rows >= 0 && g_rows >= 0, CXG_ERR_ARG, "bad M/K/N/R/rows");
  CXG_REQUIRE(fmt == CXG_PACK_INT8 || fmt == CXG_PACK_E4M3, CXG_ERR_ARG, "unknown 8-bit format");
  CXG_REQUIRE(value_type_ok(g_type), CXG_ERR_ARG, "unknown value type");
  CXG_REQUIRE(gw, CXG_ERR_ARG, "null gw");
  CXG_REQUIRE(seg_ptr || R == 1, CXG_ERR_ARG, "several segments need seg_ptr");
  const bool none = M == 0 || a_rows == 0 || g_rows == 0;       // (maps into a matrix without rows: every entry is outside)
  CXG_REQUIRE(none || (codes && exps && g), CXG_ERR_ARG, "null codes/exps/g");
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
  const int64_t tiles = pw_tiles(K, N);
  const PwArgs a{codes, exps, a_rows, g, ldg, g_rows, src_idx, dst_idx, seg_ptr, none ? 0 : M, K, N, R, packed_pitch(K), packed_groups(K),
                 pw_chunk_rows(M, K, N, R), chunks, static_cast<float*>(workspace), (int64_t)K * N + (gb ? N : 0)};
  // many chunks per segment: sixteen runs of them, else four; four elements at a time where the shapes allow
  const bool many = chunks > 64 * (int64_t)R;
  const bool vec = (int64_t)K * N % 4 == 0 && (!gb || N % 4 == 0) && (((uintptr_t)gw | (uintptr_t)gb) & 15) == 0;
  const int64_t sums = ceil_div(a.stride, (int64_t)(vec ? 4 : 1) * (many ? 16 : 64));           // blocks per segment
  CXG_REQUIRE(chunks * tiles < kPwMaxBlocks && sums < kPwMaxBlocks, CXG_ERR_UNSUPPORTED, "gw of %d x %d is too large for one launch",
              K, N);
  if (!none) {
    if (fmt == CXG_PACK_INT8) pw_launch_type<CXG_PACK_INT8>(a, g_type, chunks, st);
    else pw_launch_type<CXG_PACK_E4M3>(a, g_type, chunks, st);
    CXG_LAUNCH_CHECK("packed_wgrad_kernel");
  }
  if (vec && many) pw_launch_sums<4, 16>(a, gw, gb, st);
  else if (vec) pw_launch_sums<4, 4>(a, gw, gb, st);
  else if (many) pw_launch_sums<1, 16>(a, gw, gb, st);
  else pw_launch_sums<1, 4>(a, gw, gb, st);
  CXG_LAUNCH_CHECK("packed_wgrad_sums_kernel");
  return CXG_OK;
}

}  // extern "C"
