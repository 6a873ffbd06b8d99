// Attention of a wave over 32-token tiles of the ragged store, shared by the
// kernels that read rows straight from memory into MFMA operands (a batch's
// own rows beside a shared prefix; the kept blocks of a row).
//
// A wave holds up to 16 query columns: lane l serves column l % 16 and the
// k-group l / 16.  Each column has a limit, the first token it does not see.
// State per lane: m, the reference point of its column's scaled base-2 scores
// (at most log2(kRowsLazy) below their maximum), l, its share of the sum of
// exp2(score - m), and o[mt][j] = O^T[16 mt + 4 g + j][column].
#pragma once
#include "hc_common.h"

namespace hc {

// The reference point moves when a lane's sum of a tile's probabilities
// exceeds this: they stay inside every input type's range, and most tiles
// take no maximum and rescale nothing.
constexpr float kRowsLazy = 256.f;

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

// Tokens tok0 + [0, 32) of a row, their K and V operands in kr and vr.  lim:
// this lane's column limit; lim_lo <= lim <= lim_hi over the wave's columns
// (both uniform), and equal unless MIXED.  scale_log2 > 0.
template <typename T, bool MIXED>
__device__ __forceinline__ void attend_rows(const typename Elem<T>::vec8 (&kr)[8], typename Elem<T>::vec8 (&vr)[8],
                                            const typename Elem<T>::vec8 (&qreg)[4], int tok0, int lim, int lim_lo,
                                            int lim_hi, int lane, float scale_log2, float& m, float& l,
                                            f32x4 (&o)[8]) {
  const int g = lane >> 4;
  f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    s[0] = mma_16x16x32(kr[x], qreg[x], s[0]);
    s[1] = mma_16x16x32(kr[4 + x], qreg[x], s[1]);
  }
  const bool edge = tok0 + HC_TILE > lim_lo;
  if (edge) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (tok0 + 16 * (e >> 2) + 4 * g + (e & 3) >= lim) s[e >> 2][e & 3] = -INFINITY;
    if (tok0 + HC_TILE > lim_hi) {
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) zero_tail<T>(vr[mt], tok0, lim_hi, g);
    }
  }
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
  if (__any(!(ps <= kRowsLazy))) {  // also NaN, as while m = -inf
    float mx = s[0][0];
#pragma unroll
    for (int e = 1; e < 8; ++e) mx = fmaxf(mx, s[e >> 2][e & 3]);
    const float mnew = fmaxf(m, rows4_max(mx) * scale_log2);
    const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - mnew);
    m = mnew;
    l *= alpha;
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) o[mt] *= alpha;
    probs(mnew == -INFINITY ? 0.f : -mnew);
  }
  l += ps;
  if (MIXED && edge && lim_lo < lim_hi) {
    // Some columns do not see tokens that others see.  Their probabilities
    // are zero, but zero times an infinite or NaN value is not: with one
    // among those tokens each limit takes its own product, over values that
    // end at it, and only its own columns keep the result.
    bool bad = false;
#pragma unroll
    for (int mt = 0; mt < 8; ++mt)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = vec8_at<T>(vr[mt], e);
        bad |= !(x - x == 0.f);
      }
    if (__any(bad)) {
      for (int end = lim_lo; end <= lim_hi; ++end) {
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) {
          typename Elem<T>::vec8 vz = vr[mt];
          zero_tail<T>(vz, tok0, end, g);
          const f32x4 r = mma_16x16x32(vz, pb, o[mt]);
          if (lim == end) o[mt] = r;
        }
      }
      return;
    }
  }
#pragma unroll
  for (int mt = 0; mt < 8; ++mt) o[mt] = mma_16x16x32(vr[mt], pb, o[mt]);
}

// K and V operands of the tile that starts at element `at` of both stores.
template <typename T>
__device__ __forceinline__ void load_rows_tile(typename Elem<T>::vec8 (&kr)[8], typename Elem<T>::vec8 (&vr)[8],
                                               const T* kb, const T* vb, int64_t at) {
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    kr[x] = load8_stream<T>(kb + at + x * 512);
    vr[x] = load8_stream<T>(vb + at + x * 512);
  }
}

// One output row's weights: the reference M of several (m, l) states and
// exp2(m - M), zero for a state without tokens.
__device__ __forceinline__ float state_weight(float m, float M) { return m == -INFINITY ? 0.f : fast_exp2(m - M); }

}  // namespace hc

#include "hc_internal.h"

namespace hc {

// Attention of a wave's query columns over rows of the store, and the fold of
// partial results; defined in hc_rows.hip.
struct RowsArgs {
  const void* q;
  int64_t q_s[3];  // element strides: batch, head, token
  const void *kstore, *vstore;
  const int64_t* row_tile_off;
  const int32_t* row_len;
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
int launch_rows_attn(int dtype, const RowsArgs& a, hipStream_t s);
int launch_merge(int dtype, const MergeArgs& a, int64_t columns, hipStream_t s);
int device_cus();

}  // namespace hc
