// Attention of a chunk of new tokens over a paged cache: more than 16 (query,
// head) columns of a row.
//
//   out[c] = sum_t softmax_t(scale q_c . k_t) v_t,   c = i * G + g,
//   t < base + i + 1
//
// A workgroup of four waves takes 128 columns, 32 a wave: the queries of all
// heads of a group lie beside each other, so a key is read once for 128 / G
// queries of every head, and the causal edge is as steep as it can be.  Keys
// advance 64 tokens at a time through LDS, copied straight from the pages
// (keys double-buffered, values once, as the next ones are requested behind
// the product that reads them); the values' operand is a transposed LDS read,
// so pages keep the order in which tokens arrive.  Scores, softmax and O stay
// in registers.
//
// Where page sizes are multiples of 16, the 16 tokens of a copy lie in one page
// and its address is scalar; other sizes pay an address a lane.
//
// Bound by the matrix cores beside the softmax's vector work: 2048 tokens over
// 63488 (32 heads over 8, bf16) in 1.94 ms, 1.12 PFLOP/s (1.10 with the append
// and the fold); few columns by the latency of an iteration's loads.  So
// probabilities enter the product with V in the input type alone: with what the
// type leaves of them, as hc_paged_rows.h has it where memory bounds, there
// would be half as much matrix work again (relative error of a bf16 output 0.0023,
// the plain form's 0.0017).
#pragma once
#include "hc_paged.h"

namespace hc {

constexpr int kWaveCols = 32;
constexpr int kCols = kPagedWaves * kWaveCols;
static_assert(kCols == kChunkCols, "columns of a workgroup");
// Tokens of an iteration: 16 KB of keys and as much of values in any type.
template <typename T>
constexpr int kKeys = sizeof(T) == 4 ? 32 : 64;
template <typename T>
constexpr int chunk_lds() {
  return 3 * kKeys<T> * Tile<T>::kRow;
}

// LDS holds an iteration's tokens of keys or values in blocks of 1 KB, 16 tokens x 64 bytes
// of channels each, block (group of 16, segment) at (group * kSegs + segment).
// A copy of a wave fills one; which 16 bytes a lane fetches sets their order in
// the block, chosen so that every operand is read at lane * (8 or 16) bytes
// plus a constant, without conflicts:
//   keys            [16-byte piece][token]
//   values, 16 bit  [pair of pieces][token][piece of the pair]: the transposed
//                   read of 16 channels takes 512 bytes in a row
//   values, fp32    [token % 4][token / 4][piece]
// (In fp32 key operands take channels 32 x + 16 half + 4 g + [0, 4), so that
// their pieces also lie together.)
constexpr int kBlock = 1024;
template <typename T>
constexpr int kSegs = Tile<T>::kRow / 64;

template <typename T>
__device__ __forceinline__ typename Elem<T>::vec8 chunk_keys(const char* set, int lane, int group, int x) {
  const char* p = set + 16 * lane;
  if constexpr (sizeof(T) == 4) {
    typename Elem<T>::vec8 r;
    r.lo = *reinterpret_cast<const f32x4*>(p + (group * kSegs<T> + 2 * x) * kBlock);
    r.hi = *reinterpret_cast<const f32x4*>(p + (group * kSegs<T> + 2 * x + 1) * kBlock);
    return r;
  } else {
    return *reinterpret_cast<const typename Elem<T>::vec8*>(p + (group * kSegs<T> + x) * kBlock);
  }
}
// Tokens 32 c + 16 (e / 4) + 4 g + e % 4 of channel 16 mt + n.
template <typename T>
__device__ __forceinline__ typename Elem<T>::vec8 chunk_values(const char* set, int lane, int c, int mt) {
  if constexpr (sizeof(T) == 4) {
    typename Elem<T>::vec8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      set8<T>(r, e, *reinterpret_cast<const float*>(set + 4 * lane + ((2 * c + (e >> 2)) * kSegs<T> + mt) * kBlock + 256 * (e & 3)));
    return r;
  } else {
    const char* p = set + 8 * lane + 2 * c * kSegs<T> * kBlock + 512 * mt;
    const short4_t lo = lds_read_transposed(p), hi = lds_read_transposed(p + kSegs<T> * kBlock);
    const short8_t both = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(typename Elem<T>::vec8, both);
  }
}

// Copies of an iteration's tokens by a workgroup: wave w takes segments w (and w + 4) of
// every group.
// MIXED: tokens from `old` on are read from the call's own tensors, which other
// workgroups of the launch store; iterations that reach them take an address a
// lane, as those over other page sizes do.
template <typename T, bool UNIFORM, bool MIXED>
struct Stage {
  static constexpr int kGroups = kKeys<T> / 16, kMine = kSegs<T> / kPagedWaves;
  typedef const __attribute__((address_space(4))) int32_t* Table;  // unchanged while the kernel runs: scalar loads
  Table tab;
  int total, old, wave, k_tok, v_tok;  // k_tok, v_tok: this lane's token of a group
  const char *k_new, *v_new;
  uint32_t k_off, v_off;               // UNIFORM: its bytes behind the group's first token; else behind its own token
  uint32_t k_piece, v_piece;           // its bytes within a token
  __device__ __forceinline__ Stage(const PagedAttn& a, int row, int total_tok, int old_tok, int lane, int wv)
      : total(total_tok), old(old_tok), wave(wv) {
    const Pool& p = a.pool;
    tab = (Table)(uintptr_t)(p.table + table_row(p, row) * p.table_stride);
    k_tok = lane & 15;
    v_tok = sizeof(T) == 4 ? 4 * (lane >> 2 & 3) + (lane >> 4) : lane >> 1 & 15;
    k_piece = 64 * wave + 16 * (lane >> 4);
    v_piece = 64 * wave + 16 * (sizeof(T) == 4 ? lane & 3 : 2 * (lane >> 5) + (lane & 1));
    k_off = k_piece + (UNIFORM ? (uint32_t)(k_tok * (int)p.k_tok) : 0u);
    v_off = v_piece + (UNIFORM ? (uint32_t)(v_tok * (int)p.v_tok) : 0u);
    if constexpr (MIXED) {
      const int b = row / p.Hkv, h = row % p.Hkv;
      k_new = a.fresh.k + b * a.fresh.k_s[0] + h * a.fresh.k_s[1];
      v_new = a.fresh.v + b * a.fresh.v_s[0] + h * a.fresh.v_s[1];
    }
  }
  __device__ __forceinline__ bool scalar(int t0) const { return UNIFORM && (!MIXED || t0 + kKeys<T> <= old); }
  // Page and place of the 16-token groups of a scalar iteration.
  struct Places {
    uint32_t page[kGroups], at[kGroups];
  };
  __device__ __forceinline__ void places(const Pool& p, int t0, Places& e, bool& bad) const {
    if (scalar(t0)) {
#pragma unroll
      for (int r = 0; r < kGroups; ++r) {
        const uint32_t t = (uint32_t)min(t0 + 16 * r, (total - 1) & ~15);
        const uint32_t pi = __umulhi(t, p.div_mul) >> (p.div_shift - 32);
        uint32_t pg = (uint32_t)__builtin_amdgcn_readfirstlane(tab[pi]);
        if (pg >= (uint32_t)p.pages) bad = true, pg = 0;
        e.page[r] = pg, e.at[r] = t - pi * (uint32_t)p.page_tokens;
      }
    }
  }
  __device__ __forceinline__ void copy(const Pool& p, int t0, const Places& e, const char* pool, int64_t s_page,
                                       int64_t s_tok, const char* fresh, int64_t s_new, int tok, uint32_t off, uint32_t piece,
                                       char* lds, bool& bad) const {
    if (scalar(t0)) {
#pragma unroll
      for (int r = 0; r < kGroups; ++r) {
        // (Strides and a page's extent lie below 2^31.)
        const char* const src = pool + ((uint64_t)e.page[r] * (uint32_t)s_page + e.at[r] * (uint32_t)s_tok);
#pragma unroll
        for (int j = 0; j < kMine; ++j) lds_dma16(src + (off + 256 * j), lds + (r * kSegs<T> + wave + kPagedWaves * j) * kBlock);
      }
      return;
    }
#pragma unroll
    for (int r = 0; r < kGroups; ++r) {
      const int t = min(t0 + 16 * r + tok, total - 1);
      const int pi = page_of(p, t);
      const bool is_new = MIXED && t >= old;
      int pg = tab[pi];
      if ((uint32_t)pg >= (uint32_t)p.pages) bad = true, pg = 0;  // (of a new token too: the append leaves it out)
      const char* src = pool + pg * s_page + (t - pi * p.page_tokens) * s_tok;
      if (is_new) src = fresh + (t - old) * s_new;
#pragma unroll
      for (int j = 0; j < kMine; ++j) lds_dma16(src + (piece + 256 * j), lds + (r * kSegs<T> + wave + kPagedWaves * j) * kBlock);
    }
  }
  __device__ __forceinline__ void keys(const PagedAttn& a, int t0, const Places& e, int hd, char* lds, bool& bad) const {
    const Pool& p = a.pool;
    copy(p, t0, e, p.k + hd * p.k_head, p.k_page, p.k_tok, k_new, a.fresh.k_s[2], k_tok, k_off, k_piece, lds, bad);
  }
  __device__ __forceinline__ void values(const PagedAttn& a, int t0, const Places& e, int hd, char* lds, bool& bad) const {
    const Pool& p = a.pool;
    copy(p, t0, e, p.v + hd * p.v_head, p.v_page, p.v_tok, v_new, a.fresh.v_s[2], v_tok, v_off, v_piece, lds, bad);
  }
};

// A query operand, channels as chunk_keys takes them.
template <typename T>
__device__ __forceinline__ typename Elem<T>::vec8 chunk_query(const T* q, int g, int x) {
  if constexpr (sizeof(T) == 4) {
    typename Elem<T>::vec8 r;
    r.lo = *reinterpret_cast<const f32x4*>(q + 32 * x + 4 * g);
    r.hi = *reinterpret_cast<const f32x4*>(q + 32 * x + 16 + 4 * g);
    return r;
  } else {
    return load8<T>(q + 32 * x + 8 * g);
  }
}

// The product of 16 channels of values with a tile's probabilities where some
// column does not see some token: what lies behind `end`, which no column sees,
// becomes zero, and an infinite or NaN value reaches the columns that give it a
// weight and no others (see tile_values in hc_rows.h).
template <typename T>
__device__ __forceinline__ void edge_values(typename Elem<T>::vec8 va, const typename Elem<T>::vec8 (&pb)[2], int tok0, int end,
                                            int g, f32x4 (&o)[2]) {
  if (tok0 + HC_TILE > end) zero_tail<T>(va, tok0, end, g);
  bool odd = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x = vec8_at<T>(va, e);
    odd |= !(x - x == 0.f);
  }
  if (__any(odd)) {
    typename Elem<T>::vec8 up, down;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = vec8_at<T>(va, e);
      const bool is = !(x - x == 0.f);
      set8<T>(up, e, is && !(x < 0.f) ? 1.f : 0.f);
      set8<T>(down, e, is && !(x > 0.f) ? 1.f : 0.f);
      if (is) set8<T>(va, e, 0.f);
    }
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const f32x4 wu = mma_16x16x32(up, pb[j], zero), wd = mma_16x16x32(down, pb[j], zero);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (wu[r] > 0.f) o[j][r] += INFINITY;
        if (wd[r] > 0.f) o[j][r] -= INFINITY;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) o[j] = mma_16x16x32(va, pb[j], o[j]);
}

// What a workgroup does: a block of 128 columns of a row, and of its keys one
// part of several.  The blocks' iterations, counted over all rows from the
// lengths on the device, are cut where the blocks alone would leave half of the
// device idle, or one row's far longer than the mean; parts of one block lie
// beside each other, and neighbours on one XCD (workgroups are dealt to the 8
// XCDs in turn), so that its L2 serves the keys that the blocks of a row share.
struct Unit {
  int row, block, part, parts, slot;
};
constexpr int kLeastIts = 8;  // iterations of a part at least

__device__ __forceinline__ float wave_sum(float v) {
  asm("" : "+v"(v));
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

__device__ __forceinline__ bool find_unit(const PagedAttn& a, const int x, int keys, int lane, Unit& u) {
  const Pool& p = a.pool;
  int enc = 0, blocks = 0, its = 0;
  auto load_rows = [&](int r0) {
    const int r = min(r0 + lane, p.rows - 1);
    const RowSpan s = row_span(p, r);
    const int cols = s.n * a.G;
    enc = s.room ? s.total : -1 - s.len;
    blocks = r0 + lane < p.rows && s.room && (cols > kFewCols || a.few == 0) ? (cols + kCols - 1) / kCols : 0;
    its = (s.total + keys - 1) / keys;
    asm("" : "+v"(enc), "+v"(blocks), "+v"(its));  // opaque: the wave's sums take every lane
  };
  int units = 0;
  float work = 0.f;
  load_rows(0);
  for (int r0 = 0;;) {
    units += __builtin_amdgcn_readlane(wave_scan_add(blocks), 63);
    work += wave_sum((float)blocks * (float)its);
    r0 += 64;
    if (r0 >= p.rows) break;
    load_rows(r0);
  }
  // At most chunk_slots workgroups belong to blocks that are cut.
  const int slots = a.chunk_slots;
  const float cut = 2 * units <= slots ? work / (float)(slots - units) : 2.f * work / (float)slots;
  const int share = __builtin_amdgcn_readfirstlane(max(kLeastIts, (int)cut + 1));
  int count = 0, split = 0;
  auto parts_of = [&]() { return blocks > 0 ? max((its + share - 1) / share, 1) : 0; };
  for (int r0 = 0; r0 < p.rows; r0 += 64) {
    if (p.rows > 64) load_rows(r0);
    const int parts = parts_of();
    const int incl = wave_scan_add(parts > 1 ? parts * blocks : 0);
    if (x == 0 && r0 + lane < p.rows) a.plan[r0 + lane] = make_int4(split + incl - (parts > 1 ? parts * blocks : 0), parts, enc, 0);
    split += __builtin_amdgcn_readlane(incl, 63);
    count += __builtin_amdgcn_readlane(wave_scan_add(parts * blocks), 63);
  }
  const int per = (count + 7) / 8, y = x % 8 * per + x / 8;
  if (x / 8 >= per || y >= count) return false;
  int before = 0, cut_before = 0;
  for (int r0 = 0; r0 < p.rows; r0 += 64) {
    if (p.rows > 64) load_rows(r0);
    const int parts = parts_of(), mine = parts * blocks;
    const int incl = wave_scan_add(mine) + before, cuts = wave_scan_add(parts > 1 ? mine : 0) + cut_before;
    const uint64_t hit = __ballot(y < incl);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      u.row = r0 + src;
      u.parts = __builtin_amdgcn_readlane(parts, src);
      const int nb = __builtin_amdgcn_readlane(blocks, src);
      const int at = y - (__builtin_amdgcn_readlane(incl, src) - u.parts * nb);
      u.block = nb - 1 - at / u.parts;  // the blocks with the most keys first
      u.part = at % u.parts;
      u.slot = u.parts > 1 ? __builtin_amdgcn_readlane(cuts, src) - u.parts * nb + at : 0;
      return true;
    }
    before = __builtin_amdgcn_readlane(incl, 63);
    cut_before = __builtin_amdgcn_readlane(cuts, 63);
  }
  return false;
}

// What paged_weigh_kernel takes of a column: the reference of its scores and the
// inverse of their sum.  No token: nothing to add; no number among the scores:
// NaN for each.
__device__ __forceinline__ float2 weigh_state(float M, float L) {
  if (M == -INFINITY) return make_float2(0.f, L == 0.f ? 0.f : NAN);
  return make_float2(M, 1.f / L);
}

// Workgroup x of a.chunk_grid.
template <typename T, bool UNIFORM, bool MIXED>
__device__ __forceinline__ void paged_chunk_job(const PagedAttn& a, const int x, char* lds) {
  typedef typename Elem<T>::vec8 vec8;
  typedef Tile<T> Tl;
  constexpr int kStep = kKeys<T>, kBlocks16 = kStep / 16, kTiles = kStep / HC_TILE;
  const Pool& p = a.pool;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g4 = lane >> 4, n16 = lane & 15;
  Unit u;
  if (!find_unit(a, x, kStep, lane, u)) return;
  const int row = u.row;
  const int b = row / p.Hkv, h = row % p.Hkv;
  const int hd = p.heads == 1 ? 0 : h;
  const RowSpan span = row_span(p, row);
  const int total = __builtin_amdgcn_readfirstlane(span.total), nq = __builtin_amdgcn_readfirstlane(span.n), ncols = nq * a.G;
  const int base = total - nq;
  const int c_first = u.block * kCols, c_wave = c_first + wave * kWaveCols;
  // The last query of the workgroup, and of the wave.
  const int i_last = (min(c_first + kCols, ncols) - 1) / a.G;
  const int its_all = (min(max(base + i_last + 1, 0), total) + kStep - 1) / kStep;
  const int share = (its_all + u.parts - 1) / u.parts;
  const int it0 = min(u.part * share, its_all), it1 = min(it0 + share, its_all);
  const bool active = c_wave < ncols;
  const int w_lo = min(max(base + c_wave / a.G + 1, 0), total);  // tokens that all columns of the wave see
  const int w_hi = active ? min(max(base + (min(c_wave + kWaveCols, ncols) - 1) / a.G + 1, 0), total) : 0;

  // Q^T operands: column c_wave + 16 j + n16, k-slots = channels 32 s + 8 g4 + [0, 8).
  vec8 qop[2][4];
  int lim[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int c = c_wave + 16 * j + n16;
    const bool ok = c < ncols;
    const int i = ok ? c / a.G : 0, gi = ok ? c % a.G : 0;
    lim[j] = ok ? min(max(base + i + 1, 0), total) : w_hi;  // (padding beside tokens sees what the last does)
    const T* qp = reinterpret_cast<const T*>(a.q) + b * a.q_s[0] + (int64_t)(h * a.G + gi) * a.q_s[1] + i * a.q_s[2];
#pragma unroll
    for (int s = 0; s < 4; ++s) qop[j][s] = ok ? chunk_query<T>(qp, g4, s) : zero8<T>();
  }

  f32x4 o[8][2];
#pragma unroll
  for (int db = 0; db < 8; ++db)
#pragma unroll
    for (int j = 0; j < 2; ++j) o[db][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  bool bad = false;

  typedef Stage<T, UNIFORM, MIXED> St;
  const St st(a, row, max(total, 1), MIXED && p.fresh ? base : total, lane, wave);
  constexpr int kSet = kStep * Tl::kRow;
  char* const sv = lds + 2 * kSet;
  typename St::Places pg;  // of the next iteration's tokens
  if (it0 < it1) {
    st.places(p, it0 * kStep, pg, bad);
    st.keys(a, it0 * kStep, pg, hd, lds, bad);
    st.values(a, it0 * kStep, pg, hd, sv, bad);
    if (it0 + 1 < it1) st.places(p, (it0 + 1) * kStep, pg, bad);
  }
  wait_lds_dma();
  __syncthreads();

  // EDGE: some column may not see all of the tokens.
  auto step = [&](auto edge_tag, int it) {
    constexpr bool EDGE = decltype(edge_tag)::value;
    const int t0 = it * kStep;
    const bool more = it + 1 < it1;
    if (more) st.keys(a, t0 + kStep, pg, hd, lds + ((it - it0 + 1) & 1) * kSet, bad);
    const bool work = active && (!EDGE || t0 < w_hi);
    const bool edge = EDGE && t0 + kStep > w_lo;
    vec8 pb[kTiles][2];
    if (work) {
      __builtin_amdgcn_s_setprio(0);
      const char* sk = lds + ((it - it0) & 1) * kSet;
      // S^T blocks: rows = tokens 16 tb + 4 g4 + r, column = c_wave + 16 j + n16.
      f32x4 sacc[kBlocks16][2];
#pragma unroll
      for (int tb = 0; tb < kBlocks16; ++tb)
#pragma unroll
        for (int j = 0; j < 2; ++j) sacc[tb][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int tb = 0; tb < kBlocks16; ++tb) {
        if constexpr (sizeof(T) == 4) {
          // Sums of 32 channels apart: a rounding is half a step of the partial
          // sum that it falls on.
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const vec8 ka = chunk_keys<T>(sk, lane, tb, s);
#pragma unroll
            for (int j = 0; j < 2; ++j) sacc[tb][j] += mma_16x16x32(ka, qop[j][s], f32x4{0.f, 0.f, 0.f, 0.f});
          }
        } else {
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const vec8 ka = chunk_keys<T>(sk, lane, tb, s);
#pragma unroll
            for (int j = 0; j < 2; ++j) sacc[tb][j] = mma_16x16x32(ka, qop[j][s], sacc[tb][j]);
          }
        }
      }
      // The softmax runs at raised wave priority: the other waves of the SIMD
      // fill the matrix pipe meanwhile.
      __builtin_amdgcn_s_setprio(1);
      if (edge) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int tb = 0; tb < kBlocks16; ++tb)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (t0 + 16 * tb + 4 * g4 + r >= lim[j]) sacc[tb][j][r] = -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float ps;
        auto probs = [&](float nm) {
          ps = 0.f;
#pragma unroll
          for (int c = 0; c < kTiles; ++c) {
            float pv[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              pv[e] = fast_exp2(fmaf(sacc[2 * c + (e >> 2)][j][e & 3], a.scale_log2, nm));
              ps += pv[e];
            }
            pb[c][j] = pack8<T>(pv);  // at most half a step of the input type per probability
          }
        };
        probs(-m[j]);
        // The reference point moves, and O with it, only when a lane's sum says
        // so (see hc_rows.h).
        if (__any(!(ps <= Weights<T>::kLazy))) {
          float mx = -INFINITY;
#pragma unroll
          for (int tb = 0; tb < kBlocks16; ++tb)
#pragma unroll
            for (int r = 0; r < 4; ++r) mx = fmaxf(mx, sacc[tb][j][r]);
          const float mnew = next_reference<T>(m[j], rows4_max(mx) * a.scale_log2);
          const float alpha = m[j] == -INFINITY ? 0.f : fast_exp2(m[j] - mnew);
          m[j] = mnew;
          l[j] *= alpha;
#pragma unroll
          for (int db = 0; db < 8; ++db) o[db][j] *= alpha;
          probs(mnew == -INFINITY ? 0.f : -mnew);
          if (mnew == -INFINITY && (!EDGE || t0 < lim[j])) ps += 1.f;
        }
        l[j] += ps;
      }
      __builtin_amdgcn_s_setprio(0);
    }
    wait_lds_dma();  // the values, and the next keys, which were requested before the scores
    __syncthreads();
    if (work) {
#pragma unroll
      for (int c = 0; c < kTiles; ++c)
#pragma unroll
        for (int db = 0; db < 8; ++db) {
          const vec8 va = chunk_values<T>(sv, lane, c, db);
          if (EDGE && edge) {
            edge_values<T>(va, pb[c], t0 + c * HC_TILE, w_hi, g4, o[db]);
          } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) o[db][j] = mma_16x16x32(va, pb[c][j], o[db][j]);
          }
        }
    }
    __syncthreads();  // the values are no longer read
    if (more) {
      st.values(a, t0 + kStep, pg, hd, sv, bad);
      if (it + 2 < it1) st.places(p, t0 + 2 * kStep, pg, bad);
    }
  };
  // Every column of the workgroup sees these iterations' tokens whole.
  const int it_whole = min(max(min(max(base + c_first / a.G + 1, 0), total) / kStep, it0), it1);
  int it = it0;
  for (; it < it_whole; ++it) step(std::false_type{}, it);
#pragma unroll 1
  for (; it < it1; ++it) step(std::true_type{}, it);

  // A page outside of the pool: NaN for all columns, and the status word.
  const bool any_bad = __syncthreads_or(bad);
  if (any_bad && tid == 0 && p.status) atomicOr(p.status, kStatusPage);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float lt = rows4_sum(l[j]);
    const int c = c_wave + 16 * j + n16;
    if (c >= ncols) continue;  // (padding: the fold writes it)
    if (any_bad) m[j] = -INFINITY, lt = NAN;
    if (u.parts > 1) {
      const int64_t at = (int64_t)u.slot * kCols + (c - c_first);
      float* pp = a.chunk_o + at * HC_HEAD_DIM + 4 * g4;
#pragma unroll
      for (int db = 0; db < 8; ++db) *reinterpret_cast<f32x4*>(pp + 16 * db) = o[db][j];
      if (g4 == 0) *reinterpret_cast<float2*>(a.chunk_ml + at * 2) = make_float2(m[j], lt);
    } else {
      if (a.ml && g4 == 0) *reinterpret_cast<float2*>(a.ml + ((int64_t)row * a.ml_stride + c) * 2) = weigh_state(m[j], lt);
      typedef T quad __attribute__((ext_vector_type(4)));
      T* op = reinterpret_cast<T*>(a.out) + b * a.o_s[0] + (int64_t)(h * a.G + c % a.G) * a.o_s[1] + (c / a.G) * a.o_s[2] + 4 * g4;
#pragma unroll
      for (int db = 0; db < 8; ++db) {
        quad r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = Elem<T>::from_f32(state_output(o[db][j][e], m[j], lt));
        *reinterpret_cast<quad*>(op + 16 * db) = r;
      }
    }
  }
}

// The cut blocks' partials folded, 32 threads a column of 4 channels each; the
// outputs of padding, of rows without room, and the new lengths.
// (Workgroup x of n.)
template <typename T>
__device__ __forceinline__ void paged_chunk_fold_job(const PagedAttn& a, const int x, const int n) {
  const Pool& p = a.pool;
  const int d0 = 4 * (threadIdx.x & 31);
  if (a.len_out) {
    const int r = x * 256 + threadIdx.x, rows = p.heads == 1 ? p.rows : p.rows / p.Hkv;
    if (r < rows) {
      const int e = a.plan[p.heads == 1 ? r : r * p.Hkv].z;
      a.len_out[r] = e >= 0 ? e : -1 - e;
    }
  }
  const int64_t columns = (int64_t)p.rows * a.cols;
  for (int64_t col = (int64_t)x * 8 + (threadIdx.x >> 5); col < columns; col += (int64_t)n * 8) {
    const int row = (int)(col / a.cols), c = (int)(col % a.cols);
    const int4 plan = a.plan[row];
    const int b = row / p.Hkv, h = row % p.Hkv;
    const int ncols = query_tokens(p.counts, b, p.Q) * a.G;
    const bool few = a.few > 0 && ncols <= kFewCols, room = plan.z >= 0;
    if (few ? c < a.few : c < ncols && room && plan.y == 1) continue;
    float M = -INFINITY, L = c < ncols && !room ? NAN : 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if (c < ncols && room) {
      const int nb = (ncols + kCols - 1) / kCols;
      const int64_t at = ((int64_t)plan.x + (nb - 1 - c / kCols) * plan.y) * kCols + c % kCols;
      const float* po = a.chunk_o + at * HC_HEAD_DIM + d0;
      const float* ml = a.chunk_ml + at * 2;
      for (int s0 = 0; s0 < plan.y; s0 += 4) {
        f32x4 o4[4];
        float2 m4[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int64_t s = min(s0 + u, plan.y - 1);
          o4[u] = *reinterpret_cast<const f32x4*>(po + s * kCols * HC_HEAD_DIM);
          m4[u] = *reinterpret_cast<const float2*>(ml + s * kCols * 2);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (s0 + u >= plan.y) continue;
          const float mn = fmaxf(M, m4[u].x), f = state_weight(M, mn), e = state_weight(m4[u].x, mn);
          L = L * f + m4[u].y * e;
          acc = acc * f + o4[u] * e;
          M = mn;
        }
      }
      if (a.ml && d0 == 0) *reinterpret_cast<float2*>(a.ml + ((int64_t)row * a.ml_stride + c) * 2) = weigh_state(M, L);
    }
    typedef T quad __attribute__((ext_vector_type(4)));
    T* op = reinterpret_cast<T*>(a.out) + b * a.o_s[0] + (int64_t)(h * a.G + c % a.G) * a.o_s[1] + (c / a.G) * a.o_s[2] + d0;
    quad r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = Elem<T>::from_f32(state_output(acc[e], M, L));
    *reinterpret_cast<quad*>(op) = r;
  }
}

// The call's new tokens into their pages: workgroups of 16 tokens of a row.  16 bytes a thread and token, K and V.
// MIXED: beside its attention, of rows of many columns (the others' store theirs).
template <bool MIXED>
__device__ __forceinline__ void paged_append_job(const PagedAttn& a, const int x, int chunks, int blocks) {
  const Pool& p = a.pool;
  const int row = x / blocks, blk = x % blocks;
  const int b = row / p.Hkv, h = row % p.Hkv;
  const int trow = table_row(p, row), hd = p.heads == 1 ? 0 : h;
  const RowSpan s = row_span(p, row);
  const bool first = p.heads == 1 || h == 0;
  if (MIXED && s.n * a.G <= kFewCols) return;
  if (blk == 0 && threadIdx.x == 0 && first) {
    if (a.len_out) a.len_out[trow] = s.total;
    if (!s.room && p.status) atomicOr(p.status, kStatusCapacity);
  }
  if (!s.room) return;
  const int32_t* const tab = p.table + trow * p.table_stride;
  const int i0 = blk * 16, n = min(s.n - i0, 16);
  for (int u = threadIdx.x; u < n * chunks; u += 256) {
    const int i = i0 + u / chunks, off = 16 * (u % chunks), t = s.len + i;
    const int pi = page_of(p, t), pg = tab[pi], at = t - pi * p.page_tokens;
    if ((uint32_t)pg >= (uint32_t)p.pages) {
      if (p.status) atomicOr(p.status, kStatusPage);
      continue;
    }
    const u32x4 k = *reinterpret_cast<const u32x4*>(a.fresh.k + b * a.fresh.k_s[0] + h * a.fresh.k_s[1] + i * a.fresh.k_s[2] + off);
    const u32x4 v = *reinterpret_cast<const u32x4*>(a.fresh.v + b * a.fresh.v_s[0] + h * a.fresh.v_s[1] + i * a.fresh.v_s[2] + off);
    *reinterpret_cast<u32x4*>(const_cast<char*>(p.k) + pg * p.k_page + hd * p.k_head + at * p.k_tok + off) = k;
    *reinterpret_cast<u32x4*>(const_cast<char*>(p.v) + pg * p.v_page + hd * p.v_head + at * p.v_tok + off) = v;
  }
  if ((int)threadIdx.x < n) {
    const int t = s.len + i0 + threadIdx.x;
    if (a.pos && first) a.pos[trow * a.pos_stride + t] = t + a.dropped[trow];
    if (a.zeroed) a.zeroed[row * a.weight_stride + t] = 0.f;
  }
}

}  // namespace hc
