// Attention over 32-token tiles of the ragged store, shared by the kernels
// that read rows straight from memory into MFMA operands (a batch's own rows
// beside a shared prefix; the kept blocks of a row).
//
// A wave holds up to 16 query columns: lane l serves column l % 16 and the
// k-group l / 16.  Each column has a limit, the first token it does not see.
// State per lane: m, the reference point of its column's scaled base-2 scores
// (at most log2(Weights::kLazy) below their maximum), l, its share of the sum
// of exp2(score - m), and o[mt][j] = O^T[16 mt + 4 g + j][column].  m stays
// -inf while no score is a number above it; l then tells why: zero where there
// was no token, positive where the tokens all score -inf, NaN where one scores
// NaN.
#pragma once
#include <type_traits>

#include "hc_common.h"

namespace hc {

// The reference point moves when a lane's sum of a tile's probabilities
// exceeds kLazy, to kAbove below the maximum: they stay inside the input type's
// range, and most tiles take no maximum and rescale nothing.  fp16's range is
// used whole: with the reference at the maximum a weight below 2^-25 of it
// leaves the product with V but not the sum, and a tail of e^-17.4 a token
// behind a dominant one lost what a wave or part held of it beside that one (a
// quarter of 6000 tokens, 0.5 % of 131072).  2^10 above, weights down to 2^-24
// keep their 11 bits and those down to 2^-35 count, and the reference moves as
// seldom (16 sequences of 4 queries behind 12289 fp16 tokens of 4 heads: 31.0
// us before, 30.4, 30.7 and 31.8 with 8, 10 and 12).
template <typename T>
struct Weights {
  static constexpr float kAbove = 0.f, kLazy = 256.f;
};
template <>
struct Weights<_Float16> {
  static constexpr float kAbove = 10.f, kLazy = 65504.f;
};
// The reference point behind m, for a greatest scaled score of top.  (Beyond 2^26
// a step of fp32 is 8, and its rounding alone takes the room above.)
template <typename T>
__device__ __forceinline__ float next_reference(float m, float top) {
  if constexpr (Weights<T>::kAbove > 0.f) top = fabsf(top) < 0x1p26f ? top - Weights<T>::kAbove : top;
  return fmaxf(m, top);
}

// Floats of one partial: 128 unnormalised channels; (m, l) lie apart.
constexpr int kPartO = HC_HEAD_DIM;

template <typename T>
__device__ __forceinline__ void set8(typename Elem<T>::vec8& v, int e, float x) {
  v[e] = Elem<T>::from_f32(x);
}
template <>
__device__ __forceinline__ void set8<float>(Elem<float>::vec8& v, int e, float x) {
  if (e < 4) v.lo[e] = x; else v.hi[e - 4] = x;
}

// V operands of tokens at or beyond `end` become zero: a stale slot may hold
// NaN, which a zero probability does not silence.
template <typename T>
__device__ __forceinline__ void zero_tail(typename Elem<T>::vec8& v, int tok0, int end, int g) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (tok0 + 16 * (e >> 2) + 4 * g + (e & 3) >= end) set8<T>(v, e, 0.f);
}

// S^T of a tile's 32 tokens: element e of the pair (s[e / 4][e % 4]) is token
// 16 (e / 4) + 4 g + e % 4 against the lane's column.  In fp32, where these sums
// are the largest error, four of 32 channels each are formed apart: a rounding
// is half a step of the partial sum that it falls on.
template <typename T>
__device__ __forceinline__ void tile_scores(const typename Elem<T>::vec8 (&kr)[8],
                                            const typename Elem<T>::vec8 (&qreg)[4], f32x4 (&s)[2]) {
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f32x4 part[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) part[x] = mma_16x16x32(kr[4 * h + x], qreg[x], zero);
      s[h] = (part[0] + part[1]) + (part[2] + part[3]);
    }
  } else {
    s[0] = s[1] = zero;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      s[0] = mma_16x16x32(kr[x], qreg[x], s[0]);
      s[1] = mma_16x16x32(kr[4 + x], qreg[x], s[1]);
    }
  }
}

// Probabilities of a tile's scores (already masked; seen: the column sees one
// of its tokens) in the input type, the state m, l and, when the reference
// point moves, O following.  scale_log2 > 0.
template <typename T>
__device__ __forceinline__ typename Elem<T>::vec8 tile_probs(const f32x4 (&s)[2], bool seen, float scale_log2, float& m,
                                                             float& l, f32x4 (&o)[8]) {
  typename Elem<T>::vec8 pb;
  float ps;
  auto probs = [&](float nm) {
    float p[8];
    ps = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      p[e] = fast_exp2(fmaf(s[e >> 2][e & 3], scale_log2, nm));
      ps += p[e];
    }
    // P enters the matrix product in the input type: at most half a step per
    // probability, against sums kept in fp32 from the unrounded ones.
    pb = pack8<T>(p);
  };
  probs(-m);
  if (__any(!(ps <= Weights<T>::kLazy))) {  // also NaN, as while m = -inf
    float mx = s[0][0];
#pragma unroll
    for (int e = 1; e < 8; ++e) mx = fmaxf(mx, s[e >> 2][e & 3]);
    const float mnew = next_reference<T>(m, rows4_max(mx) * scale_log2);
    const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - mnew);
    m = mnew;
    l *= alpha;
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) o[mt] *= alpha;
    probs(mnew == -INFINITY ? 0.f : -mnew);
    if (mnew == -INFINITY && seen) ps += 1.f;
  }
  l += ps;
  return pb;
}

// O += V^T P^T over tokens tok0 + [0, 32), of which those from `end` on are
// seen by no column.
template <typename T, bool MIXED>
__device__ __forceinline__ void tile_values(typename Elem<T>::vec8 (&vr)[8], const typename Elem<T>::vec8& pb, int tok0,
                                            int end, int g, f32x4 (&o)[8]) {
  if (tok0 + HC_TILE > end) {
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) zero_tail<T>(vr[mt], tok0, end, g);
  }
  if constexpr (MIXED) {
    // Some columns do not see tokens that others see.  Their probabilities
    // are zero, but zero times an infinite or NaN value is not: with one in
    // the tile the finite values take the product, and what the others would
    // add is told by the weight that their positive and their negative ones
    // (NaN: both) have in each column.
    bool bad = false;
#pragma unroll
    for (int mt = 0; mt < 8; ++mt)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = vec8_at<T>(vr[mt], e);
        bad |= !(x - x == 0.f);
      }
    if (__any(bad)) {
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) {
        typename Elem<T>::vec8 up, down;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = vec8_at<T>(vr[mt], e);
          const bool odd = !(x - x == 0.f);
          set8<T>(up, e, odd && !(x < 0.f) ? 1.f : 0.f);
          set8<T>(down, e, odd && !(x > 0.f) ? 1.f : 0.f);
          if (odd) set8<T>(vr[mt], e, 0.f);
        }
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        const f32x4 wu = mma_16x16x32(up, pb, zero), wd = mma_16x16x32(down, pb, zero);
        o[mt] = mma_16x16x32(vr[mt], pb, o[mt]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (wu[j] > 0.f) o[mt][j] += INFINITY;
          if (wd[j] > 0.f) o[mt][j] -= INFINITY;
        }
      }
      return;
    }
  }
#pragma unroll
  for (int mt = 0; mt < 8; ++mt) o[mt] = mma_16x16x32(vr[mt], pb, o[mt]);
}

// The eight operands of a tile of K or V (8 wave loads of 1 KB in a row).
template <typename T>
__device__ __forceinline__ void load_operands(typename Elem<T>::vec8 (&r)[8], const T* p) {
#pragma unroll
  for (int x = 0; x < 8; ++x) r[x] = load8_stream<T>(p + x * 512);
}

// The weight exp2(m - M) of a state (m, l) under the reference M of several:
// one that holds no number above -inf adds nothing to one that does (but a NaN
// l, which zero does not silence).
__device__ __forceinline__ float state_weight(float m, float M) {
  return m == -INFINITY ? (M == -INFINITY ? 1.f : 0.f) : fast_exp2(m - M);
}
// An output channel of the folded state (M, L): zero without tokens, NaN where
// their scores have no softmax.
__device__ __forceinline__ float state_output(float acc, float M, float L) {
  return M == -INFINITY ? (L == 0.f ? 0.f : NAN) : acc * (1.f / L);
}

}  // namespace hc

#include "hc_internal.h"

namespace hc {

// A launch's jobs over rows of the store (rows_job).
struct RowsArgs {
  const void* q;
  int64_t q_s[3];  // element strides: batch, head, token
  const void *kstore, *vstore;
  const int64_t* row_tile_off;
  const int32_t* row_len;
  const int32_t* query_counts;  // per sequence, or null: all Q
  // Kept blocks of each (row, query): keep entries of tpb tiles, the first
  // counts of them used; null: every visible tile of the row.
  const int32_t *idx, *counts;
  int keep, tpb;
  int Hkv, G, Q, rows;
  int qpb, ncb;     // queries of a job (qpb * G <= 16 columns), jobs of a row
  int nsplit;       // workgroups of a job
  float scale_log2;
  // nsplit = 1 and no part_o: the output itself, else unnormalised partials
  // [(row * Q + query) * G + head][split][128] and (m, l) pairs.
  float *part_o, *part_ml;
  void* out;
  int64_t o_s[3];
};

// How many of the Q queries of sequence b are tokens of its rows (the others,
// behind them, are padding).
__device__ __forceinline__ int query_tokens(const int32_t* counts, int b, int Q) {
  return counts ? min(max(counts[b], 0), Q) : Q;
}

constexpr int kRowsPitch = HC_HEAD_DIM + 4;
// LDS floats of rows_job: O and (m, l) of NW waves x 64 / NW columns.
constexpr int kRowsLds = 64 * (kRowsPitch + 2);

inline int64_t rows_workgroups(const RowsArgs& a) { return ((int64_t)a.rows + 7) / 8 * 8 * a.ncb * a.nsplit; }

// Workgroup `wg` of a rows launch (NW waves): one split of one job (qpb queries
// of one row and its G heads, at most 64 / NW columns).  The waves take every
// NW-th tile of the split straight into the operand registers and are combined
// through LDS (lds: kRowsLds floats).  K's registers are refilled once the
// scores are formed, V's once the values are added, so a wave always has half a
// tile or more in flight with one tile's registers, and three waves fit a SIMD
// (a second buffer leaves two, and was slower by 2 to 10 %); a wave's last tile
// loads nothing (itself again: 7.6 against 5.9 us for 8 queries of 64 tiles).
// Bound by HBM: a token's K and V (512 bytes in 16 bits) feed 512 G operations a
// query; 1.06M tokens of 1024 rows take 92 us, 5.9 TB/s.
enum RowsMode {
  kRowsWhole,   // every visible tile of the row
  kRowsList,    // the blocks of a.idx and a.counts
  kRowsListed,  // the same in LDS: list and its count, one workgroup a job
};
template <typename T, int MODE, bool MIXED, int NW>
__device__ __forceinline__ void rows_job(const RowsArgs& a, int wg, float* lds, const int32_t* listed = nullptr,
                                         int listed_count = 0) {
  constexpr bool LIST = MODE != kRowsWhole;
  typedef typename Elem<T>::vec8 vec8;
  constexpr int kCols = 64 / NW;
  float(*s_o)[kCols][kRowsPitch] = reinterpret_cast<float(*)[kCols][kRowsPitch]>(lds);
  float(*s_m)[kCols] = reinterpret_cast<float(*)[kCols]>(lds + 64 * kRowsPitch);
  float(*s_l)[kCols] = s_m + NW;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, n = lane & 15;
  // The jobs of a row (LIST: its queries, which keep many of the same blocks)
  // go to one XCD, as workgroups are dealt to the 8 XCDs in turn.
  const int jobs = (a.rows + 7) / 8 * 8 * a.ncb;
  const int job = wg % jobs, split = wg / jobs;
  const int row = job / (8 * a.ncb) * 8 + job % 8, cb = job % (8 * a.ncb) / 8;
  if (row >= a.rows) return;
  const int b = row / a.Hkv, kv = row % a.Hkv;
  // Column n: query i0 + n / G, head n % G of the row's group.
  const int i0 = cb * a.qpb, nq = min(a.qpb, a.Q - i0), ncols = nq * a.G;
  const bool col_ok = n < ncols;
  const int qi = col_ok ? n / a.G : nq - 1, gi = col_ok ? n % a.G : 0;

  // Everything the tiles' addresses and products wait for is requested at
  // once: the length, the tile offset, the list and the queries.
  const int64_t job_q = (int64_t)row * a.Q + i0;  // LIST: one query a job
  const int32_t* const list = MODE == kRowsList ? a.idx + job_q * a.keep : listed;
  const int row_len = a.row_len[row], nqt = query_tokens(a.query_counts, b, a.Q);
  const int64_t base = a.row_tile_off[row] * (int64_t)HC_TILE_ELEMS + lane * 8;
  int kept = 0, spec = 0;
  // This wave's first 64 entries of a whole list.
  const int full = LIST ? a.keep * a.tpb : 0;
  const int f0 = (int)((int64_t)full * split / a.nsplit), f1 = (int)((int64_t)full * (split + 1) / a.nsplit);
  if constexpr (MODE == kRowsListed) kept = listed_count;
  if constexpr (MODE == kRowsList) {
    kept = a.counts[job_q];
    spec = list[min(f0 + wave + lane * NW, full - 1) / a.tpb];
  }
  vec8 qreg[4];
  {
    const T* qp = reinterpret_cast<const T*>(a.q) + b * a.q_s[0] + (int64_t)(kv * a.G + gi) * a.q_s[1] +
                  (int64_t)(i0 + qi) * a.q_s[2] + 8 * g;
#pragma unroll
    for (int s = 0; s < 4; ++s) qreg[s] = col_ok ? load8<T>(qp + 32 * s) : zero8<T>();
  }

  const int len = max(row_len, 0);
  const int lim_lo = min(max(len - nqt + 1 + i0, 0), len);
  const int lim_hi = min(max(len - nqt + i0 + nq, 0), len);
  const int lim = min(max(len - nqt + 1 + i0 + qi, 0), len);
  // Entries of the job, this workgroup's share of them and this wave's: e0 +
  // wave, e0 + wave + NW, ...
  const int vis = (lim_hi + HC_TILE - 1) / HC_TILE;
  const bool void_list = LIST && kept < 0;  // no selection was made: the output is NaN
  int entries = vis;
  if constexpr (LIST) entries = vis > 0 ? min(max(kept, 0), a.keep) * a.tpb : 0;
  const int e0 = (int)((int64_t)entries * split / a.nsplit), e1 = (int)((int64_t)entries * (split + 1) / a.nsplit);
  const int cnt = max((e1 - e0 - wave + NW - 1) / NW, 0);
  const bool whole = MODE == kRowsList && e0 == f0 && e1 == f1;

  float m = -INFINITY, l = 0.f;
  f32x4 o[8];
#pragma unroll
  for (int mt = 0; mt < 8; ++mt) o[mt] = f32x4{0.f, 0.f, 0.f, 0.f};

  const T* kb = reinterpret_cast<const T*>(a.kstore) + base;
  const T* vb = reinterpret_cast<const T*>(a.vstore) + base;
  for (int c0 = 0; c0 < cnt; c0 += 64) {
    const int nt = min(cnt - c0, 64);
    // LIST: lane x holds the tile of the wave's entry c0 + x, -1 for one that
    // is not a visible tile of the row (such an entry attends nothing).
    int mine = 0;
    if constexpr (LIST) {
      const int e = e0 + wave + (c0 + min(lane, nt - 1)) * NW;
      const int blk = whole && c0 == 0 ? spec : list[e / a.tpb];
      const int64_t t = (int64_t)blk * a.tpb + e % a.tpb;
      mine = blk >= 0 && t < vis ? (int)t : -1;
    }
    auto tile_of = [&](int i) {
      if constexpr (LIST) return __builtin_amdgcn_readlane(mine, i);
      return e0 + wave + (c0 + i) * NW;
    };
    vec8 kr[8], vr[8];
    int tile = tile_of(0);
    load_operands<T>(kr, kb + (int64_t)max(tile, 0) * HC_TILE_ELEMS);
    load_operands<T>(vr, vb + (int64_t)max(tile, 0) * HC_TILE_ELEMS);
    // One tile, and the loads of the next one (LAST: there is none), so that
    // each wait leaves the younger half tile in flight.
    auto step = [&](auto last, int next) {
      constexpr bool LAST = decltype(last)::value;
      const int64_t at = LAST ? 0 : (int64_t)max(next, 0) * HC_TILE_ELEMS;
      const bool live = !LIST || tile >= 0;
      const int tok0 = max(tile, 0) * HC_TILE;
      const int lo = live ? lim_lo : 0, hi = live ? lim_hi : 0, mylim = live ? lim : 0;
      // A tile that some columns see more of than others (a row's last one or
      // two): the next one's keys wait, which leaves it their registers.
      const bool mixed = MIXED && tok0 + HC_TILE > lo && lo < hi;
      f32x4 s[2];
      tile_scores<T>(kr, qreg, s);
      __builtin_amdgcn_sched_barrier(0);
      if (!LAST && !mixed) load_operands<T>(kr, kb + at);
      __builtin_amdgcn_sched_barrier(0);
      if (tok0 + HC_TILE > lo) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (tok0 + 16 * (e >> 2) + 4 * g + (e & 3) >= mylim) s[e >> 2][e & 3] = -INFINITY;
      }
      const vec8 pb = tile_probs<T>(s, tok0 < mylim, a.scale_log2, m, l, o);
      if (mixed) {
        tile_values<T, true>(vr, pb, tok0, hi, g, o);
        if (!LAST) load_operands<T>(kr, kb + at);
      } else {
        tile_values<T, false>(vr, pb, tok0, hi, g, o);
      }
      if (LAST) return;
      __builtin_amdgcn_sched_barrier(0);
      load_operands<T>(vr, vb + at);
      __builtin_amdgcn_sched_barrier(0);
      tile = next;
    };
    for (int i = 1; i < nt; ++i) step(std::false_type{}, tile_of(i));
    step(std::true_type{}, 0);
  }
  l = rows4_sum(l);
  if (LIST && void_list) m = 0.f, l = NAN;

  if (col_ok) {
    if (g == 0) s_m[wave][n] = m, s_l[wave][n] = l;
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) *reinterpret_cast<f32x4*>(&s_o[wave][n][16 * mt + 4 * g]) = o[mt];
  }
  __syncthreads();
  // 32 threads a column, 4 channels each.
  for (int c = threadIdx.x >> 5; c < ncols; c += NW * 2) {
    const int d0 = 4 * (threadIdx.x & 31);
    float M = s_m[0][c];
#pragma unroll
    for (int w = 1; w < NW; ++w) M = fmaxf(M, s_m[w][c]);
    float L = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = state_weight(s_m[w][c], M);
      L = fmaf(s_l[w][c], f, L);
      acc += *reinterpret_cast<const f32x4*>(&s_o[w][c][d0]) * f;
    }
    const int i = i0 + c / a.G, hd = c % a.G;
    if (a.part_o) {
      const int64_t at = (((int64_t)row * a.Q + i) * a.G + hd) * a.nsplit + split;
      *reinterpret_cast<f32x4*>(a.part_o + at * kPartO + d0) = acc;
      if (d0 == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(M, L);
    } else {
      T* op = reinterpret_cast<T*>(a.out) + b * a.o_s[0] + (int64_t)(kv * a.G + hd) * a.o_s[1] +
              (int64_t)i * a.o_s[2] + d0;
#pragma unroll
      for (int e = 0; e < 4; ++e) op[e] = Elem<T>::from_f32(state_output(acc[e], M, L));
    }
  }
}

struct MergeArgs {
  // Partials of a shared prefix: [part][column][128], column = (b * Q + i) * G
  // + g; info[2 kv] = first part, info[2 kv + 1] = parts of KV head kv.
  const float *pre_o, *pre_ml;
  const int32_t* info;
  int64_t M;  // columns of a KV head
  // Partials of the rows (RowsArgs), nsplit of each column; 0: none.
  const float *row_o, *row_ml;
  int nsplit;
  int Hkv, G, Q;
  void* out;
  int64_t o_s[3];
};

// Jobs and splits of a rows launch over at most max_tiles tiles a row.
struct RowsPlan {
  int qpb, ncb, nsplit;
};
RowsPlan rows_plan(int rows, int G, int Q, int64_t max_tiles);
int launch_block_rows(int dtype, const RowsArgs& a, int waves, hipStream_t s);
int launch_merge(int dtype, const MergeArgs& a, int64_t columns, hipStream_t s);
int device_cus();

}  // namespace hc
