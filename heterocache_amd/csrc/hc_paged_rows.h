// Attention of few queries over a paged cache: at most 16 (query, head)
// columns of a row, as in a decode step, so each key and value feeds 16 columns
// of a matrix instruction once and the kernel is bound by HBM.
//
//   out[c] = sum_t softmax_t(scale q_c . k_t) v_t
//
// The rows' tiles of 32 tokens, counted through all rows, are dealt to the
// workgroups in equal runs from the lengths on the device, so a ragged batch
// keeps every CU busy to the end; a run that crosses rows leaves a partial
// state (m, l, o) for each.  A wave copies its tiles into its own LDS buffer,
// each token's address through the table (or, for the tokens that the call
// appends, from their tensors: they are stored to the pages beside, so that
// nothing waits for a launch of its own), takes the tile's operands into
// registers and requests the next tile before it attends.  Where page sizes are
// multiples of 16, a copy's tokens lie in one page and its address is scalar;
// other sizes, and the tiles that reach behind the stored tokens, take an
// address a token.  Measured: 745 MB of a ragged fp16 batch in 122 us, 6.1 TB/s;
// 17 MB in 10.6 us, of which some 9 are the chain of cold reads (lengths, table,
// tiles), the launch and the end.
#pragma once
#include "hc_paged.h"

namespace hc {

constexpr int kFoldPitch = HC_HEAD_DIM + 4;

template <typename T>
constexpr int rows_lds() {
  const int stage = kPagedWaves * 2 * Tile<T>::kBytes;
  const int fold = kPagedWaves * 16 * (kFoldPitch + 2) * 4;
  return (stage > fold ? stage : fold) + kPagedWaves * 64 * 8;
}

__device__ __forceinline__ int tiles_of(int tokens) { return (tokens + HC_TILE - 1) / HC_TILE; }

// tile_probs of hc_rows.h with what the input type leaves of each probability
// beside it, as a second operand of the product with V: memory bounds this
// kernel, and with both a bf16 weight is exact to 2^-17 (relative error of a
// step's output, bf16: 0.0019-0.0023 without, 0.0017 with, in the same time).
template <typename T>
__device__ __forceinline__ typename Elem<T>::vec8 split_probs(const f32x4 (&s)[2], bool seen, float scale_log2, float& m, float& l,
                                                              f32x4 (&o)[8], typename Elem<T>::vec8& lo) {
  typename Elem<T>::vec8 hi;
  float ps;
  auto probs = [&](float nm) {
    float p[8];
    ps = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      p[e] = fast_exp2(fmaf(s[e >> 2][e & 3], scale_log2, nm));
      ps += p[e];
    }
    hi = pack8<T>(p);
    if constexpr (sizeof(T) == 2) {
      float rest[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) rest[e] = p[e] - vec8_at<T>(hi, e);
      lo = pack8<T>(rest);
    }
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
  return hi;
}

// tile_values of hc_rows.h for 16 channels, which leaves the loop's registers
// alone: of tokens that some column does not see, from `end` on none.
template <typename T>
__device__ __forceinline__ void edge_channels(typename Elem<T>::vec8& v, const typename Elem<T>::vec8& pb, int tok0, int end, int g,
                                              f32x4& o) {
  if (tok0 + HC_TILE > end) zero_tail<T>(v, tok0, end, g);
  bool odd = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x = vec8_at<T>(v, e);
    odd |= !(x - x == 0.f);
  }
  if (__any(odd)) {
    typename Elem<T>::vec8 up, down;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = vec8_at<T>(v, e);
      const bool is = !(x - x == 0.f);
      set8<T>(up, e, is && !(x < 0.f) ? 1.f : 0.f);
      set8<T>(down, e, is && !(x > 0.f) ? 1.f : 0.f);
      if (is) set8<T>(v, e, 0.f);
    }
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    const f32x4 wu = mma_16x16x32(up, pb, zero), wd = mma_16x16x32(down, pb, zero);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (wu[r] > 0.f) o[r] += INFINITY;
      if (wd[r] > 0.f) o[r] -= INFINITY;
    }
  }
  o = mma_16x16x32(v, pb, o);
}

// Whether a tile holds a value that is no number: the rest of a probability,
// which may be negative or zero, must not meet an infinity.
template <typename T>
__device__ __forceinline__ bool any_odd(const typename Elem<T>::vec8 (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    return false;  // (no rests)
  } else {
    typedef unsigned short __attribute__((ext_vector_type(8))) ushort8;
    constexpr unsigned short kInf = std::is_same<T, __bf16>::value ? 0x7f80 : 0x7c00;
    ushort8 top = __builtin_bit_cast(ushort8, v[0]) & (unsigned short)0x7fff;
#pragma unroll
    for (int mt = 1; mt < 8; ++mt)
      top = __builtin_elementwise_max(top, __builtin_bit_cast(ushort8, v[mt]) & (unsigned short)0x7fff);
    bool odd = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) odd |= top[e] >= kInf;
    return __any(odd);
  }
}

// Workgroup x of a.grid.
template <typename T, bool WEIGH, bool UNIFORM>
__device__ __forceinline__ void paged_rows_job(const PagedAttn& a, const int x, char* lds) {
  typedef typename Elem<T>::vec8 vec8;
  typedef Tile<T> Tl;
  const Pool& p = a.pool;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, n = lane & 15;
  char* const sk = lds + wave * 2 * Tl::kBytes;
  char* const sv = sk + Tl::kBytes;
  int64_t* const addr = reinterpret_cast<int64_t*>(lds + rows_lds<T>() - kPagedWaves * 64 * 8) + wave * 64;

  // The rows' tokens, 64 rows at a time, and the tiles of all.
  int row_e = 0, nt = 0;
  auto load_rows = [&](int r0) {
    const int r = min(r0 + lane, p.rows - 1);
    const RowSpan s = row_span(p, r);
    row_e = s.room ? s.total : -1 - s.len;
    nt = s.room && s.n > 0 && s.n * a.G <= kFewCols ? tiles_of(s.total) : 0;
    nt = r0 + lane < p.rows ? nt : 0;
    asm("" : "+v"(row_e), "+v"(nt));  // opaque: the wave's sums take every lane
  };
  int total = 0;
  load_rows(0);
  for (int r0 = 0;;) {
    total += __builtin_amdgcn_readlane(wave_scan_add(nt), 63);
    r0 += 64;
    if (r0 >= p.rows) break;
    load_rows(r0);
  }
  // Equal runs of all tiles, which may cross rows, or every row cut for itself:
  // the latter leaves workgroups idle where lengths differ, but a run that
  // crosses pays for a row's start and end again, about kCross rounds of a tile
  // a wave.  Whichever has fewer rounds (64 rows of 66 tiles with weights: 30.0
  // us in crossing runs, now 26.2).
  constexpr int kCross = 3;
  const int crossing = (total + a.grid - 1) / a.grid;
  const int apart = 2 * p.rows <= a.grid ? (total + a.grid - p.rows - 1) / (a.grid - p.rows) : 1 << 30;
  const bool cut = (apart + kPagedWaves - 1) / kPagedWaves <= (crossing + kPagedWaves - 1) / kPagedWaves + kCross;
  // (A whole number of tiles a wave.)
  const int share = cut ? max(apart, kPagedWaves) : max(crossing + kPagedWaves - 1, kPagedWaves) / kPagedWaves * kPagedWaves;
  const int64_t lo64 = (int64_t)x * share;
  const int lo = (int)min(lo64, (int64_t)total), hi = (int)min(lo64 + share, (int64_t)total);
  if (!cut && lo >= hi && x != 0) return;

  int before = 0;  // of the rows ahead of r0: tiles, or parts
  for (int r0 = 0; r0 < p.rows; r0 += 64) {
    if (p.rows > 64) load_rows(r0);
    const int parts = cut ? (nt + share - 1) / share : nt;
    const int incl = wave_scan_add(parts) + before, excl = incl - parts;
    before = __builtin_amdgcn_readlane(incl, 63);
    if (x == 0 && wave == 0 && r0 + lane < p.rows) {
      // The row's first partial, how many, its tokens.
      const int w0 = excl / share, segs = parts == 0 ? 0 : cut ? parts : (incl - 1) / share - w0 + 1;
      a.info[r0 + lane] = make_int4(cut ? excl : w0 + r0 + lane, segs, row_e, 0);
      if (row_e < 0 && p.status) atomicOr(p.status, kStatusCapacity);
    }
    uint64_t mine = __ballot(parts > 0 && (cut ? excl <= x && incl > x : excl < hi && incl > lo));
    while (mine) {
      const int src = __builtin_ctzll(mine);
      mine &= mine - 1;
      const int row = r0 + src;
      const int first = __builtin_amdgcn_readlane(excl, src), ntiles = __builtin_amdgcn_readlane(nt, src);
      const int total_tok = __builtin_amdgcn_readlane(row_e, src);
      const int np = __builtin_amdgcn_readlane(parts, src);
      const int t0 = cut ? (int)((int64_t)ntiles * (x - first) / np) : max(lo - first, 0);
      const int t1 = cut ? (int)((int64_t)ntiles * (x - first + 1) / np) : min(hi - first, ntiles);
      const int b = row / p.Hkv, h = row % p.Hkv;
      const int trow = table_row(p, row), hd = p.heads == 1 ? 0 : h;
      const int nq = __builtin_amdgcn_readfirstlane(query_tokens(p.counts, b, p.Q));
      const int base = total_tok - nq;  // query i sees tokens below base + i + 1
      const int old = p.fresh ? base : total_tok;
      const int32_t* const tab = p.table + trow * p.table_stride;
      const bool is_v = lane >= 32;
      const char* const pool = is_v ? p.v + hd * p.v_head : p.k + hd * p.k_head;
      const int64_t s_page = is_v ? p.v_page : p.k_page, s_tok = is_v ? p.v_tok : p.k_tok;
      const char* const fresh = !p.fresh ? nullptr
                                : is_v   ? a.fresh.v + b * a.fresh.v_s[0] + h * a.fresh.v_s[1]
                                         : a.fresh.k + b * a.fresh.k_s[0] + h * a.fresh.k_s[1];
      const int64_t s_fresh = is_v ? a.fresh.v_s[2] : a.fresh.k_s[2];
      bool bad = false;

      // A tile's page entries: UNIFORM, of its two groups of 16 tokens, the tile
      // being whole in the pages; else of token l % 32 in lane l.  Tokens behind
      // the last are the last.
      typedef const __attribute__((address_space(4))) int32_t* Table;  // unchanged while the kernel runs: scalar loads
      const Table stab = (Table)(uintptr_t)tab;
      struct Entries {
        int e[2];
      };
      auto whole = [&](int tile) { return UNIFORM && tile * HC_TILE + HC_TILE <= old; };
      auto entries = [&](int tile) {
        Entries r = {};
        if (whole(tile)) {
#pragma unroll
          for (int u = 0; u < 2; ++u) r.e[u] = __builtin_amdgcn_readfirstlane(stab[page_of(p, tile * HC_TILE + 16 * u)]);
        } else {
          r.e[0] = tab[page_of(p, min(tile * HC_TILE + (lane & 31), total_tok - 1))];
        }
        return r;
      };
      // (Bytes of a lane's 16 within a token, for the first tokens of a group.)
      const int tok0_lane = lane / Tl::kChunks;
      const uint32_t off_lane = 16 * ((lane % Tl::kChunks) ^ Tl::swizzle(tok0_lane));
      auto copy = [&](int tile, Entries en) {
        if (whole(tile)) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint32_t pg = (uint32_t)en.e[u];
            if (pg >= (uint32_t)p.pages) bad = true, pg = 0;
            const int t = tile * HC_TILE + 16 * u;
            const uint32_t at = (uint32_t)(t - page_of(p, t) * p.page_tokens);
            const char* const kp = p.k + hd * p.k_head + ((uint64_t)pg * (uint32_t)p.k_page + at * (uint32_t)p.k_tok);
            const char* const vp = p.v + hd * p.v_head + ((uint64_t)pg * (uint32_t)p.v_page + at * (uint32_t)p.v_tok);
#pragma unroll
            for (int j = 0; j < Tl::kLoads / 2; ++j) {
              // (The swizzle is linear in the token's bits.)
              const uint32_t off = off_lane ^ (uint32_t)(16 * Tl::swizzle(j * Tl::kTokens & 15));
              const uint32_t tok = j * Tl::kTokens + tok0_lane;
              lds_dma16_run<1, true>(kp + (off + tok * (uint32_t)p.k_tok), sk + 1024 * (u * Tl::kLoads / 2 + j));
              lds_dma16_run<1, true>(vp + (off + tok * (uint32_t)p.v_tok), sv + 1024 * (u * Tl::kLoads / 2 + j));
            }
          }
          return;
        }
        // Lane l holds the address of token l % 32: keys for the lower 32 lanes,
        // values for the upper.
        const int t = min(tile * HC_TILE + (lane & 31), total_tok - 1);
        const bool is_new = t >= old;
        int page = en.e[0];
        if (!is_new && (uint32_t)page >= (uint32_t)p.pages) bad = true, page = 0;
        const int at = t - page_of(p, t) * p.page_tokens;
        const char* src = is_new ? fresh + (t - old) * s_fresh : pool + page * s_page + at * s_tok;
        __builtin_amdgcn_wave_barrier();
        addr[lane] = reinterpret_cast<int64_t>(src);
        __builtin_amdgcn_wave_barrier();
        constexpr int kBatch = 8;  // addresses read together: each copy may write LDS, which orders the next read
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
          for (int j0 = 0; j0 < Tl::kLoads; j0 += kBatch) {
            int64_t from[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
              const int tok = (j0 + j) * Tl::kTokens + lane / Tl::kChunks;
              from[j] = addr[32 * v + tok] + 16 * ((lane % Tl::kChunks) ^ Tl::swizzle(tok));
            }
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
              lds_dma16_run<1, true>(reinterpret_cast<const char*>(from[j]), (v ? sv : sk) + 1024 * (j0 + j));
          }
      };

      const int tile0 = t0 + wave;
      // The wave's tiles, every kPagedWaves-th, from one that differs between the
      // workgroups on and round: runs of equal length begin at equal places of
      // their pages, and together they would draw on few memory channels.
      const int mine = max((t1 - tile0 + kPagedWaves - 1) / kPagedWaves, 0);
      const int end = tile0 + mine * kPagedWaves;
      auto after = [&](int tile) { return tile + kPagedWaves < end ? tile + kPagedWaves : tile0; };
      int tile = tile0 + (mine > 0 ? (int)((uint32_t)x * 5u % (uint32_t)mine) * kPagedWaves : 0);
      Entries first_e = {}, next = {};
      if (mine > 0) first_e = entries(tile);
      // Column n: query n / G, head n % G of the row's group.
      const bool col_ok = n < nq * a.G;
      const int qi = col_ok ? n / a.G : 0, gi = col_ok ? n % a.G : 0;
      vec8 qreg[4];
      {
        const T* qp = reinterpret_cast<const T*>(a.q) + b * a.q_s[0] + (int64_t)(h * a.G + gi) * a.q_s[1] + qi * a.q_s[2] + 8 * g;
#pragma unroll
        for (int s = 0; s < 4; ++s) qreg[s] = col_ok ? load8<T>(qp + 32 * s) : zero8<T>();
      }
      if (mine > 0) {
        copy(tile, first_e);
        if (mine > 1) next = entries(after(tile));
      }
      // The run that begins the row stores its new tokens.
      if (p.fresh && t0 == 0) {
        for (int u = threadIdx.x; u < nq * Tl::kChunks; u += kPagedThreads) {
          const int i = u / Tl::kChunks, off = 16 * (u % Tl::kChunks), t = old + i;
          const int pg = tab[page_of(p, t)], at = t - page_of(p, t) * p.page_tokens;
          if ((uint32_t)pg >= (uint32_t)p.pages) {
            bad = true;
            continue;
          }
          *reinterpret_cast<u32x4*>(const_cast<char*>(p.k) + pg * p.k_page + hd * p.k_head + at * p.k_tok + off) =
              *reinterpret_cast<const u32x4*>(a.fresh.k + b * a.fresh.k_s[0] + h * a.fresh.k_s[1] + i * a.fresh.k_s[2] + off);
          *reinterpret_cast<u32x4*>(const_cast<char*>(p.v) + pg * p.v_page + hd * p.v_head + at * p.v_tok + off) =
              *reinterpret_cast<const u32x4*>(a.fresh.v + b * a.fresh.v_s[0] + h * a.fresh.v_s[1] + i * a.fresh.v_s[2] + off);
        }
        if ((int)threadIdx.x < nq) {
          const int t = old + threadIdx.x;
          if (a.pos && (p.heads == 1 || h == 0)) a.pos[trow * a.pos_stride + t] = t + a.dropped[trow];
          if (a.zeroed) a.zeroed[row * a.weight_stride + t] = 0.f;
        }
      }

      const int lim_lo = min(max(base + 1, 0), total_tok);
      const int lim = col_ok ? min(max(base + 1 + qi, 0), total_tok) : total_tok;
      float m = -INFINITY, l = 0.f;
      f32x4 o[8];
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) o[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
      for (int left = mine; left > 0; --left) {
        const int tok0 = tile * HC_TILE;
        wait_lds_dma();
        __builtin_amdgcn_wave_barrier();
        vec8 kr[8], vr[8];
#pragma unroll
        for (int y = 0; y < 8; ++y) kr[y] = key_operand<T>(sk, g, n, y >> 2, y & 3);
#pragma unroll
        for (int y = 0; y < 8; ++y) vr[y] = value_operand<T>(sv, g, n, y);
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the operands are here
        __builtin_amdgcn_sched_barrier(0);
        f32x4 s[2];
        tile_scores<T>(kr, qreg, s);
        if (tok0 + HC_TILE > lim_lo) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (tok0 + 16 * (e >> 2) + 4 * g + (e & 3) >= lim) s[e >> 2][e & 3] = -INFINITY;
        }
        // (Ahead of the copies, whose wait then finds the stores done.)
        if (WEIGH && col_ok) {
          // [row][tile][column][32]
          float* sp = a.scores + row * a.score_stride + ((int64_t)tile * a.few + n) * HC_TILE + 4 * g;
          *reinterpret_cast<f32x4*>(sp) = s[0] * a.scale_log2;
          *reinterpret_cast<f32x4*>(sp + 16) = s[1] * a.scale_log2;
        }
        __builtin_amdgcn_sched_barrier(0);
        // The buffer takes the next tile.
        const int then = after(tile);
        if (left > 1) {
          copy(then, next);
          if (left > 2) next = entries(after(then));
        }
        __builtin_amdgcn_sched_barrier(0);
        vec8 lo;
        const vec8 pb = split_probs<T>(s, tok0 < lim, a.scale_log2, m, l, o, lo);
        if (tok0 + HC_TILE > lim_lo || any_odd<T>(vr)) {
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) edge_channels<T>(vr[mt], pb, tok0, total_tok, g, o[mt]);
        } else {
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) o[mt] = mma_16x16x32(vr[mt], pb, o[mt]);
        }
        if constexpr (sizeof(T) == 2) {
          // (Values that are no numbers have had their say, and are zero now.)
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) o[mt] = mma_16x16x32(vr[mt], lo, o[mt]);
        }
        tile = then;
      }
      l = rows4_sum(l);
      if (__any(bad)) {
        m = 0.f, l = NAN;
        if (p.status && lane == 0) atomicOr(p.status, kStatusPage);
      }

      // The waves' states fold into one partial.
      __syncthreads();
      float(*s_o)[16][kFoldPitch] = reinterpret_cast<float(*)[16][kFoldPitch]>(lds);
      float(*s_ml)[16][2] = reinterpret_cast<float(*)[16][2]>(lds + kPagedWaves * 16 * kFoldPitch * 4);
      if (g == 0) s_ml[wave][n][0] = m, s_ml[wave][n][1] = l;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) *reinterpret_cast<f32x4*>(&s_o[wave][n][16 * mt + 4 * g]) = o[mt];
      __syncthreads();
      const int64_t slot = (int64_t)(cut ? x : x + row) * a.few;
      for (int c = threadIdx.x >> 5; c < nq * a.G; c += kPagedThreads / 32) {
        const int d0 = 4 * (threadIdx.x & 31);
        float M = s_ml[0][c][0], L = 0.f;
#pragma unroll
        for (int w = 1; w < kPagedWaves; ++w) M = fmaxf(M, s_ml[w][c][0]);
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kPagedWaves; ++w) {
          const float f = state_weight(s_ml[w][c][0], M);
          L = fmaf(s_ml[w][c][1], f, L);
          acc += *reinterpret_cast<const f32x4*>(&s_o[w][c][d0]) * f;
        }
        *reinterpret_cast<f32x4*>(a.part_o + (slot + c) * HC_HEAD_DIM + d0) = acc;
        if (d0 == 0) *reinterpret_cast<float2*>(a.part_ml + (slot + c) * 2) = make_float2(M, L);
      }
      __syncthreads();  // the next row's copies take the buffer
    }
    if ((cut ? before > x : before >= hi) && x != 0) break;
  }
}

// The partials of a row's columns folded into outputs, the new lengths, and
// (WEIGH) every token's weight: the workgroups behind the columns' take runs of
// a row's tokens, fold the columns' (m, l) for themselves and add each token's
// probabilities.
constexpr int kWeighTokens = 1024;  // (see paged_weigh_runs)
template <typename T, bool WEIGH>
__device__ __forceinline__ void paged_fold_job(const PagedAttn& a, const int x, const int runs) {
  const Pool& p = a.pool;
  const int columns = p.rows * a.few;
  const bool weigh = WEIGH && x >= columns;
  const int row = weigh ? (x - columns) % p.rows : x / a.few;
  const int4 info = a.info[row];
  const bool room = info.z >= 0;
  const int b = row / p.Hkv, h = row % p.Hkv, total = room ? info.z : -1 - info.z;
  const int nq = query_tokens(p.counts, b, p.Q), ncols = room ? nq * a.G : 0;
  if (nq * a.G > kFewCols) return;
  const int segs = info.y;
  const float* const ml = a.part_ml + (int64_t)info.x * a.few * 2;  // [segment][column]
  if (!weigh) {
    __shared__ float s_m[8], s_l[8];
    __shared__ f32x4 s_o[8][32];
    const int c = x % a.few;
    const int grp = threadIdx.x >> 5, d0 = 4 * (threadIdx.x & 31);
    const float* const po = a.part_o + ((int64_t)info.x * a.few + c) * HC_HEAD_DIM + d0;
    float m = -INFINITY, l = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if (c < ncols) {
      for (int s0 = grp; s0 < segs; s0 += 32) {
        f32x4 o4[4];
        float2 m4[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int64_t s = min(s0 + 8 * u, segs - 1);
          o4[u] = *reinterpret_cast<const f32x4*>(po + s * a.few * HC_HEAD_DIM);
          m4[u] = *reinterpret_cast<const float2*>(ml + (s * a.few + c) * 2);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (s0 + 8 * u >= segs) continue;
          const float M = fmaxf(m, m4[u].x), f = state_weight(m, M), e = state_weight(m4[u].x, M);
          l = l * f + m4[u].y * e;
          acc = acc * f + o4[u] * e;
          m = M;
        }
      }
    }
    if (d0 == 0) s_m[grp] = m, s_l[grp] = l;
    s_o[grp][threadIdx.x & 31] = acc;
    __syncthreads();
    if (grp != 0) return;
    float M = s_m[0], L = 0.f;
#pragma unroll
    for (int w = 1; w < 8; ++w) M = fmaxf(M, s_m[w]);
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const float f = state_weight(s_m[w], M);
      L = fmaf(s_l[w], f, L);
      sum += s_o[w][threadIdx.x & 31] * f;
    }
    if (!room && c < nq * a.G) L = NAN;
    T* op = reinterpret_cast<T*>(a.out) + b * a.o_s[0] + (int64_t)(h * a.G + c % a.G) * a.o_s[1] + (c / a.G) * a.o_s[2] + d0;
#pragma unroll
    for (int e = 0; e < 4; ++e) op[e] = Elem<T>::from_f32(state_output(sum[e], M, L));
    if (c == 0 && threadIdx.x == 0 && a.len_out && (p.heads == 1 || h == 0)) a.len_out[table_row(p, row)] = total;
  } else if constexpr (WEIGH) {
    // (M, 1 / L) of the columns: 16 threads each.
    __shared__ float s_m[16][16], s_l[16][16], s_top[16], s_inv[16];
    const int c = threadIdx.x >> 4, j = threadIdx.x & 15;
    float m = -INFINITY, l = 0.f;
    if (c < ncols) {
      for (int s = j; s < segs; s += 16) {
        const float2 y = *reinterpret_cast<const float2*>(ml + ((int64_t)s * a.few + c) * 2);
        const float M = fmaxf(m, y.x);
        l = l * state_weight(m, M) + y.y * state_weight(y.x, M);
        m = M;
      }
    }
    s_m[c][j] = m, s_l[c][j] = l;
    __syncthreads();
    if (threadIdx.x < 16) {
      float M = -INFINITY, L = 0.f;
      for (int u = 0; u < 16; ++u) M = fmaxf(M, s_m[threadIdx.x][u]);
      for (int u = 0; u < 16; ++u) L = fmaf(s_l[threadIdx.x][u], state_weight(s_m[threadIdx.x][u], M), L);
      // No token: nothing to add.  No number among the scores: NaN for each.
      s_top[threadIdx.x] = M == -INFINITY ? 0.f : M;
      s_inv[threadIdx.x] = M == -INFINITY ? (L == 0.f ? 0.f : NAN) : 1.f / L;
    }
    __syncthreads();
    const int base = total - nq, old = p.fresh && room ? base : total;
    const float* const in = a.weights + row * a.weight_stride;
    float* const outw = a.weights_out + row * a.weight_stride;
    for (int t0 = (x - columns) / p.rows * kWeighTokens; t0 < total; t0 += runs * kWeighTokens) {
      const int t = t0 + 4 * threadIdx.x;
      if (t >= total) break;
      f32x4 w = {0.f, 0.f, 0.f, 0.f};
      const float* sp = a.scores + row * a.score_stride + (int64_t)(t / HC_TILE) * a.few * HC_TILE + t % HC_TILE;
#pragma unroll 4
      for (int u = 0; u < ncols; ++u) {
        const f32x4 s = *reinterpret_cast<const f32x4*>(sp + u * HC_TILE);
        const float top = s_top[u], inv = s_inv[u];
        const int lim = base + 1 + u / a.G;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (t + e < lim) w[e] = fmaf(fast_exp2(s[e] - top), inv, w[e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (t + e < total) outw[t + e] = t + e < old ? in[t + e] + w[e] : w[e];
    }
  }
}

}  // namespace hc
