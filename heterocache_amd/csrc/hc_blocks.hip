// Attention over the key blocks that a cheap score selects for each query.
//
// A row of the ragged store is cut into blocks of S tokens (S a multiple of
// the 32-token tile).  Of every complete block the index holds, per channel,
// the maximum and the minimum of its keys in 8 bits under one power of two:
//   e     = the least exponent in [-48, 48] with max_d |k_d| <= 127 * 2^e
//   hi_d  = ceil(max_t k_t,d / 2^e),  lo_d = floor(min_t k_t,d / 2^e)
// (clamped to -127..127).  A query head in 8 bits, q8 = rint(q / 2^eq) with eq
// found the same way, then scores a block by
//   s(j) = 2^(eq + e_j) * sum_d max(q8_d hi_d, q8_d lo_d),
// the largest product that any key within the block's box could form with q8:
// a block that holds one strongly matching key is not averaged away.  The sum
// is one of whole numbers below 2^21, formed on the integer matrix cores as
// q8+ . hi + q8- . lo (q8+ = max(q8, 0), q8- = min(q8, 0)), and the scales are
// powers of two, so a score is exact: the same selection comes out whatever
// the batch, the split or the order.  8 bits halve the bytes that every token
// reads of the index; rounding outwards keeps the box a bound of the keys.
//
// A query keeps its first `sink` and last `local` visible blocks and of the
// others those that the row's best query head scores highest, ties to the
// lower block, n in all, in ascending order.
#include <algorithm>
#include <cmath>

#include "hc_rows.h"

namespace hc {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMinExp = -48, kMaxExp = 48;
constexpr int kBoundBytes = 2 * HC_HEAD_DIM;  // 128 maxima, then 128 minima

__device__ __forceinline__ float power2(int e) { return __int_as_float((e + 127) << 23); }

// The least e in [-48, 48] with top <= 127 * 2^e (top >= 0).
__device__ __forceinline__ int least_exp(float top) {
  int e = (int)((__float_as_uint(top) >> 23) & 0xff) - 133;  // 64 <= top / 2^e < 128
  e = min(max(e, kMinExp), kMaxExp);
  if (top * power2(-e) > 127.f) ++e;
  return min(e, kMaxExp);
}

__device__ __forceinline__ int clamp8(float x) { return (int)fminf(fmaxf(x, -127.f), 127.f); }

// ---- bounds ------------------------------------------------------------------
struct BoundArgs {
  const void* kstore;
  const int64_t *row_tile_off, *row_blk_off;
  const int32_t* row_len;
  int8_t *bounds, *exps;
  int rows, tpb, span;  // span: blocks a row, the last complete ones
  int fresh;            // > 0: only blocks that the last `fresh` tokens completed
};

// The greater of two values, the other one where one is NaN: one instruction,
// where fmaxf first canonicalises operands it cannot prove canonical.
__device__ __forceinline__ float greater(float x, float y) { return __builtin_amdgcn_fmed3f(x, y, INFINITY); }

// Greatest values over the 16 lanes of each 16-lane row of a wave, for 16
// values a lane at once: lane l ends with its row's greatest value l % 16 (a
// reduce-scatter: the values held halve at every step).
__device__ __forceinline__ float row16_max_scatter(float (&v)[16], int lane) {
#pragma unroll
  for (int half = 8, bit = 1; half >= 1; half >>= 1, bit <<= 1) {
    const bool b = lane & bit;
#pragma unroll
    for (int j = 0; j < half; ++j) {
      const float keep = b ? v[2 * j + 1] : v[2 * j], send = b ? v[2 * j] : v[2 * j + 1];
      const float got = bit == 1   ? dpp_mov<0xB1>(send)    // quad_perm [1,0,3,2]
                        : bit == 2 ? dpp_mov<0x4E>(send)    // quad_perm [2,3,0,1]
                        : bit == 4 ? dpp_mov<0x124>(send)   // row_ror:4
                                   : dpp_mov<0x128>(send);  // row_ror:8
      v[j] = greater(keep, got);
    }
  }
  return v[0];
}

// K chunk c = ((h*4+s)*4+g)*16+m of a tile holds token 16h+m, channels
// 32s+8g+[0,8): a thread reads both halves h of its (s, g, m), so a wave's load
// is 1 KB in a row.  A thread folds the greatest values of its 8 channels and
// of their negatives, the 16 lanes m of a channel group fold theirs, and each
// rounds one of the 16 (floor(x) = -ceil(-x)).  Bound by the key stream: a
// workgroup takes every chunks-th block of a row one after another, so that
// neighbouring workgroups read neighbouring blocks (runs of blocks each: 46.4
// us against 41.6 for 258 MB), the next one's first tiles (two; ONE: blocks of
// one tile) on their way while one is folded and written.
template <typename T, bool ONE>
__global__ __launch_bounds__(256) void block_bounds_kernel(const BoundArgs a) {
  typedef typename Elem<T>::vec8 vec8;
  __shared__ float s_top[2][4];
  const int chunks = gridDim.x / a.rows;
  const int row = blockIdx.x / chunks, j0 = blockIdx.x % chunks;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row_at = a.row_tile_off[row], blk_at = a.row_blk_off[row];
  const int len = max(a.row_len[row], 0), S = a.tpb * HC_TILE;
  // Blocks counted from the last complete one back; those that were complete
  // before the last `fresh` tokens are left.
  const int have = len / S;
  const int old = a.fresh > 0 ? max(len - a.fresh, 0) / S : 0;
  const int first = have - 1 - j0, last = max(old, have - a.span);
  if (first < last) return;
  const T* kb = reinterpret_cast<const T*>(a.kstore) + tid * 8;
  constexpr int kLoads = ONE ? 2 : 4;
  vec8 x[kLoads];
  auto fetch = [&](const T* p, bool two) {  // a pair of tiles, or one twice
    x[0] = load8_stream<T>(p), x[1] = load8_stream<T>(p + 2048);
    if constexpr (!ONE) {
      const T* p1 = p + (two ? HC_TILE_ELEMS : 0);
      x[2] = load8_stream<T>(p1), x[3] = load8_stream<T>(p1 + 2048);
    }
  };
  fetch(kb + (row_at + (int64_t)first * a.tpb) * HC_TILE_ELEMS, a.tpb > 1);
  int turn = 0;
  for (int j = first; j >= last; j -= chunks) {
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = -INFINITY;
    auto fold = [&]() {
#pragma unroll
      for (int u = 0; u < kLoads; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = vec8_at<T>(x[u], e);
          v[e] = greater(v[e], y);
          v[8 + e] = greater(v[8 + e], -y);
        }
    };
    fold();
    if constexpr (!ONE)
      for (int t = 2; t < a.tpb; t += 2) {
        fetch(kb + (row_at + (int64_t)j * a.tpb + t) * HC_TILE_ELEMS, t + 1 < a.tpb);
        fold();
      }
    if (j - chunks >= last) fetch(kb + (row_at + (int64_t)(j - chunks) * a.tpb) * HC_TILE_ELEMS, a.tpb > 1);
    const float mine = row16_max_scatter(v, lane);
    // The greatest |k| is the greatest of all 16 values of all groups.
    float top = greater(mine, dpp_mov<0xB1>(mine));
    top = greater(top, dpp_mov<0x4E>(top));
    top = greater(top, dpp_mov<0x124>(top));
    top = greater(top, dpp_mov<0x128>(top));
    top = rows4_max(top);
    float* st = s_top[turn];
    turn ^= 1;
    if (lane == 0) st[wave] = top;
    // Only LDS is waited for: the next block's loads stay in flight.
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    top = fmaxf(fmaxf(st[0], st[1]), fmaxf(fmaxf(st[2], st[3]), 0.f));
    const int ex = least_exp(top);
    const int64_t blk = blk_at + j;
    // Value m of channel group tid / 16 = 4s + g: channel 8 (tid / 16) + m % 8,
    // its maximum (m < 8) or its minimum's negative.
    const int m = lane & 15, q8 = clamp8(ceilf(mine * power2(-ex)));
    a.bounds[blk * kBoundBytes + (m >> 3) * HC_HEAD_DIM + 8 * (tid >> 4) + (m & 7)] = (int8_t)(m < 8 ? q8 : -q8);
    if (tid == 0) a.exps[blk] = (int8_t)ex;
  }
}

template <typename T>
void launch_bounds(const BoundArgs& a, unsigned grid, hipStream_t s) {
  if (a.tpb == 1)
    hipLaunchKernelGGL((block_bounds_kernel<T, true>), dim3(grid), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((block_bounds_kernel<T, false>), dim3(grid), dim3(256), 0, s, a);
}

// ---- scores and selection ------------------------------------------------------
struct SelectArgs {
  const void* q;
  int64_t q_s[3];
  const int8_t *bounds, *exps;
  const int64_t* row_blk_off;
  const int32_t *row_len, *query_counts;
  float* scores;  // [row * Q + query][pitch]; unused where scores stay in LDS
  int64_t pitch;
  int32_t *idx, *counts;
  int Hkv, G, Q, rows, S, keep, sink, local;
  int chunks;      // score workgroups of a query
  int max_blocks;  // visible blocks a query has room for; one that sees more selects nothing
};

// A job is one query of one row; the queries of a row go to one XCD, whose L2
// then holds the row's bounds.
struct SelectJob {
  int row, i;
  int have;     // visible blocks
  int lo, hi;   // scored blocks: those between the first `sink` and the last `local`, if any are left out
};
__device__ __forceinline__ bool select_job(const SelectArgs& a, int x, SelectJob& j) {
  const int rest = x % (8 * a.Q);
  j.row = x / (8 * a.Q) * 8 + rest % 8;
  j.i = rest / 8;
  return j.row < a.rows;
}
// Apart from select_job: the query's loads do not wait for the row's length.
__device__ __forceinline__ void select_range(const SelectArgs& a, SelectJob& j) {
  const int len = max(a.row_len[j.row], 0), nqt = query_tokens(a.query_counts, j.row / a.Hkv, a.Q);
  j.have = (min(max(len - nqt + 1 + j.i, 0), len) + a.S - 1) / a.S;
  j.lo = a.sink;
  j.hi = j.have <= a.keep || j.have > a.max_blocks ? a.sink : j.have - a.local;
}

// A wave's 16 x 64 products: the query's heads in 8 bits are the A operand
// (lane: head l % 16, 16 bytes of the 256 a block has, steps 0 and 1 the
// positive parts against the maxima, 2 and 3 the negative ones against the
// minima), 16 blocks the B operand.
template <typename T>
struct RawQuery {
  typename Elem<T>::vec8 v[2][2];
};
struct ScoreQuery {
  i32x4 op[4];
  float unit[4];  // powers of two of heads 4g .. 4g + 3
};
// The loads and the rounding apart: the blocks' loads go out in between.
template <typename T>
__device__ __forceinline__ RawQuery<T> load_query(const SelectArgs& a, const SelectJob& j, int lane) {
  const int g = lane >> 4, n = lane & 15;
  const int b = j.row / a.Hkv, kv = j.row % a.Hkv;
  const T* p = reinterpret_cast<const T*>(a.q) + b * a.q_s[0] + (int64_t)(kv * a.G + (n < a.G ? n : 0)) * a.q_s[1] +
               (int64_t)j.i * a.q_s[2] + 16 * g;
  RawQuery<T> r;
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int u = 0; u < 2; ++u) r.v[s][u] = load8<T>(p + 64 * s + 8 * u);
  return r;
}
template <typename T>
__device__ __forceinline__ ScoreQuery score_query(const SelectArgs& a, const RawQuery<T>& raw, int lane) {
  const int g = lane >> 4;
  const bool ok = (lane & 15) < a.G;
  float x[2][16];
  float top = 0.f;
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float y = ok ? vec8_at<T>(raw.v[s][e >> 3], e & 7) : 0.f;
      x[s][e] = y;
      top = fmaxf(top, fabsf(y));
    }
  const int ex = least_exp(rows4_max(top));
  const float down = power2(-ex), up = power2(ex);
  ScoreQuery r;
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t pos = 0, neg = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int v = clamp8(rintf(x[s][4 * w + e] * down));
        pos |= (uint32_t)(max(v, 0) & 0xff) << (8 * e);
        neg |= (uint32_t)(min(v, 0) & 0xff) << (8 * e);
      }
      r.op[s][w] = (int)pos;
      r.op[2 + s][w] = (int)neg;
    }
#pragma unroll
  for (int t = 0; t < 4; ++t) r.unit[t] = __shfl(up, 4 * g + t, 64);
  return r;
}

// Bounds of U * 16 blocks from blk0 on, 4 U loads of 1 KB in flight together;
// blocks past `last` read it again.
template <int U>
struct ScoreBlocks {
  i32x4 x[U][4];
  int e[U];
};
template <int U>
__device__ __forceinline__ void load_blocks(const SelectArgs& a, int64_t blk0, int64_t last, int lane, ScoreBlocks<U>& t) {
  const int g = lane >> 4, n = lane & 15;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t blk = min(blk0 + 16 * u + n, last);
#pragma unroll
    for (int s = 0; s < 4; ++s)
      t.x[u][s] = *reinterpret_cast<const i32x4*>(a.bounds + blk * kBoundBytes + 64 * s + 16 * g);
    t.e[u] = a.exps[blk];
  }
}
// Their scores: f(u, score) with lane l's block 16 u + l % 16 (all four lanes of
// a block hold its score).
template <int U, typename F>
__device__ __forceinline__ void score_blocks(const SelectArgs& a, const ScoreQuery& q, const ScoreBlocks<U>& t, int lane,
                                             F f) {
  const int g = lane >> 4;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    i32x4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < 4; ++s) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(q.op[s], t.x[u][s], acc, 0, 0, 0);
    // Lane: heads 4g + r of block n.  Whole numbers below 2^24 and powers of
    // two: every step is exact.
    float best = -INFINITY;
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (4 * g + r < a.G) best = fmaxf(best, (float)acc[r] * q.unit[r]);
    f(u, rows4_max(best) * power2(t.e[u]));
  }
}

// Scores of long rows for few queries: many workgroups a query, through
// memory.  Bound by the index's bytes.
constexpr int kScoreWaves = 4;
template <typename T>
__global__ __launch_bounds__(kScoreWaves * 64) void block_score_kernel(const SelectArgs a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int jobs = (a.rows + 7) / 8 * 8 * a.Q;
  SelectJob j;
  if (!select_job(a, blockIdx.x % jobs, j)) return;
  const RawQuery<T> raw = load_query<T>(a, j, lane);
  const int64_t base = a.row_blk_off[j.row];
  const int chunk = blockIdx.x / jobs;
  select_range(a, j);
  const int steps = (j.hi - j.lo + 31) / 32;
  int st = chunk * kScoreWaves + wave;
  if (st >= steps) return;
  ScoreBlocks<2> t;
  load_blocks<2>(a, base + j.lo + 32 * st, base + j.hi - 1, lane, t);
  const ScoreQuery q = score_query<T>(a, raw, lane);
  float* out = a.scores + ((int64_t)j.row * a.Q + j.i) * a.pitch;
  while (true) {
    const int j0 = j.lo + 32 * st;
    score_blocks<2>(a, q, t, lane, [&](int u, float s) {
      const int blk = j0 + 16 * u + (lane & 15);
      if (lane < 16 && blk < j.hi) out[blk] = s;
    });
    st += kScoreWaves * a.chunks;
    if (st >= steps) return;
    load_blocks<2>(a, base + j.lo + 32 * st, base + j.hi - 1, lane, t);
  }
}

// The selection of one query by a workgroup of NT threads: the scores' keys (of
// score_blocks itself where SCORED is not set, by way of LDS, else from
// memory) in registers, the threshold, and one ordered pass that writes the
// kept blocks.  The threshold is found by counting the keys into equal steps
// between the least and the greatest left and going on in the step where the
// count of kept ones is reached: scores of one query lie within a few powers of
// two, where fixed digits of the key would pile up in few counters.  Bound by the latency of
// its dependent steps; a barrier each for the keys, the counts (one or two
// rounds) and the places.  128 blocks take 1 us of loads, 2 of scores and 2 of
// selection; 1000 scored ones a launch of 4.3, 4096 of 5.9.
__host__ __device__ constexpr int key_words(int blocks) { return (blocks + 15) / 16 * 16; }
constexpr int kPickKeys = 12288;  // keys in LDS, of rows scored by the same workgroup
template <int NT>
struct Pick {
  static constexpr int kWaves = NT / 64;
  static constexpr int kPer = NT / 64;  // counters that a lane reads in a row
  static constexpr int kBins = 64 * kPer;
  // Keys that a thread keeps in registers; a longer row's scores are read
  // again each time.
  static constexpr int kHeld = NT == 1024 ? 32 : 12;
  static constexpr int kBits = NT == 1024 ? 10 : NT == 512 ? 9 : 8;
  // One of padding after each row of them keeps the lanes on different banks.
  static constexpr int kSlots = 64 * (kPer + 1);
  static __device__ __forceinline__ int slot(uint32_t bin) { return (int)(bin + bin / kPer); }
  int hist[2][kSlots];
  uint32_t lo[kWaves], hi[kWaves];
  int gt[kWaves], eq[kWaves];
};

// Writes the query's counts and list to memory and, where list is not null, to
// LDS as well (a.keep entries; visible behind the next barrier); returns the
// count.  s_key: key_words(a.max_blocks) words of LDS (SCORED: none).
template <typename T, bool SCORED, int NT>
__device__ __forceinline__ int pick_blocks(const SelectArgs& a, SelectJob& j, Pick<NT>& L, uint32_t* s_key,
                                           int32_t* list) {
  typedef Pick<NT> P;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  RawQuery<T> raw;
  int64_t base = 0;
  if constexpr (!SCORED) {
    raw = load_query<T>(a, j, lane);
    base = a.row_blk_off[j.row] + a.sink;
  }
  select_range(a, j);
  const int64_t x = (int64_t)j.row * a.Q + j.i;
  int32_t* const out = a.idx + x * a.keep;
  auto put = [&](int at, int blk) {
    out[at] = blk;
    if (list) list[at] = blk;
  };
  const bool fits = j.have <= a.max_blocks;
  const int kept = fits ? min(j.have, a.keep) : -1;
  if (tid == 0) a.counts[x] = kept;
  if (!fits || j.have <= a.keep) {
    for (int k = tid; k < a.keep; k += NT) put(k, k < kept ? k : -1);
    return kept;
  }
  const int lo = j.lo, nmid = j.hi - lo;
  int need = a.keep - a.sink - a.local;  // < nmid
  for (int k = tid; k < a.sink; k += NT) put(k, k);
  for (int k = tid; k < a.local; k += NT) put(a.keep - a.local + k, j.have - a.local + k);
  if (need == 0) return kept;
  for (int k = tid; k < 2 * P::kSlots; k += NT) L.hist[0][k] = 0;
  const float* sc = SCORED ? a.scores + x * a.pitch + lo : nullptr;
  uint32_t least = 0xffffffffu, most = 0u;
  // Every thread keeps to a run of blocks, the keys of a short one in its
  // registers.  SCORED: a run starts at a multiple of four blocks of the row, for
  // 16-byte loads (what lies in front of the first scored block and behind the
  // last is not used).
  const int span = SCORED ? j.hi : nmid, skip = SCORED ? lo : 0;
  const int run = SCORED ? ((span + NT - 1) / NT + 3) / 4 * 4 : (span + NT - 1) / NT;
  const int k0 = min(tid * run, span) - skip, k1 = min(tid * run + run, span) - skip;
  const bool held = !SCORED || run <= P::kHeld;  // (launch_pick: rows scored here are short enough)
  uint32_t mine[P::kHeld];
  if constexpr (SCORED) {
    if (held) {
      const float* row = sc - lo;
#pragma unroll
      for (int e = 0; e < P::kHeld; e += 4) {
        if (e > 0 && e >= run) break;
        const f32x4 v = *reinterpret_cast<const f32x4*>(row + min((int64_t)tid * run + e, a.pitch - 4));
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          mine[e + u] = order_key(v[u]);
          if (k0 + e + u >= 0 && k0 + e + u < k1) {
            least = min(least, mine[e + u]);
            most = max(most, mine[e + u]);
          }
        }
      }
    } else {
      for (int k = tid; k < nmid; k += NT) {
        const uint32_t u = order_key(sc[k]);
        least = min(least, u);
        most = max(most, u);
      }
    }
  } else {
    // As few blocks a wave at a time as that all waves take part in.
    auto scored = [&](auto u_c) {
      constexpr int U = decltype(u_c)::value;
      if (16 * U * wave >= nmid) return;
      ScoreBlocks<U> t;
      load_blocks<U>(a, base + 16 * U * wave, base + nmid - 1, lane, t);
      const ScoreQuery q = score_query<T>(a, raw, lane);
      for (int k0 = 16 * U * wave;;) {
        score_blocks<U>(a, q, t, lane, [&](int u, float s) {
          const int k = k0 + 16 * u + (lane & 15);
          const uint32_t key = order_key(s);
          if (lane < 16 && k < nmid) s_key[k] = key;
          least = min(least, key);  // (a block past the end is the last one again)
          most = max(most, key);
        });
        k0 += 16 * U * P::kWaves;
        if (k0 >= nmid) break;
        load_blocks<U>(a, base + k0, base + nmid - 1, lane, t);
      }
    };
    if (nmid <= 16 * P::kWaves)
      scored(std::integral_constant<int, 1>{});
    else
      scored(std::integral_constant<int, 4>{});
    if (nmid <= NT / 4) {
      // Few keys: four lanes a key count the keys that go before it, a quarter
      // of them each, and no threshold is needed (with the spread of the scores
      // over the waves, 128 blocks selected and 16 attended: 12.4 to 11.9 us).
      const int words = key_words(nmid);
      for (int k = nmid + tid; k < words; k += NT) s_key[k] = 0;  // (no score's key)
      __syncthreads();
      const int kk = tid >> 2;
      const uint32_t mine = kk < nmid ? s_key[kk] : 0xffffffffu;
      int before = 0;
      for (int k = 4 * (tid & 3); k < words; k += 16) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(s_key + k);
#pragma unroll
        for (int u = 0; u < 4; ++u) before += v[u] > mine || (v[u] == mine && k + u < kk);
      }
      before += __builtin_amdgcn_mov_dpp(before, 0xB1, 0xF, 0xF, false);  // quad_perm [1,0,3,2]
      before += __builtin_amdgcn_mov_dpp(before, 0x4E, 0xF, 0xF, false);  // quad_perm [2,3,0,1]
      const bool take = (tid & 3) == 0 && kk < nmid && before < need;
      const uint64_t taken = __ballot(take);
      if (lane == 0) L.gt[wave] = __builtin_popcountll(taken);
      __syncthreads();
      int at = a.sink + __builtin_popcountll(taken & ((1ull << lane) - 1));
#pragma unroll
      for (int w = 0; w < P::kWaves; ++w)
        if (w < wave) at += L.gt[w];
      if (take) put(at, lo + kk);
      return kept;
    }
  }
  least = wave_fold(least, [](uint32_t u, uint32_t v) { return min(u, v); });
  most = wave_fold(most, [](uint32_t u, uint32_t v) { return max(u, v); });
  if (lane == 0) L.lo[wave] = least, L.hi[wave] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < P::kWaves; ++w) {
    least = min(least, L.lo[w]);
    most = max(most, L.hi[w]);
  }
  if constexpr (!SCORED) {
    if (held) {
#pragma unroll
      for (int e = 0; e < P::kHeld; ++e) {
        if (e > 0 && e >= run) break;
        mine[e] = s_key[min(k0 + e, nmid - 1)];
      }
    }
  }
  auto each = [&](auto f) {  // of the thread's run, in order: f(block, key)
    if (held) {
#pragma unroll
      for (int e = 0; e < P::kHeld; ++e) {
        if (e > 0 && e >= run) break;
        if (k0 + e >= 0 && k0 + e < k1) f(k0 + e, mine[e]);
      }
    } else {
      for (int k = max(k0, 0); k < k1; ++k) f(k, order_key(sc[k]));
    }
  };

  // Kept: the keys above T0, and the first `need` equal to it.
  uint32_t T0 = least;
  for (int round = 0; least < most; ++round) {
    const uint32_t span = most - least;
    const int shift = max(32 - __clz((int)span) - P::kBits, 0);
    int* hist = L.hist[round & 1];
    each([&](int, uint32_t u) {
      if (u >= least && u <= most) atomicAdd(&hist[P::slot((u - least) >> shift)], 1);
    });
    __syncthreads();
    // Lane y reads kPer bins in a row from the top down; keys above its first
    // one, then the bin in which the need-th highest key lies (every wave for
    // itself).
    int c[P::kPer], sum = 0;
#pragma unroll
    for (int u = 0; u < P::kPer; ++u) sum += c[u] = hist[P::kSlots - 2 - (P::kPer + 1) * lane - u];
    const int incl = wave_scan_add(sum);
    int above = incl - sum, bin = 0, in_bin = 0, before = 0;
    const bool mine = above < need && need <= incl;
#pragma unroll
    for (int u = 0; u < P::kPer; ++u) {
      if (above < need && need <= above + c[u]) bin = P::kBins - 1 - P::kPer * lane - u, in_bin = c[u], before = above;
      above += c[u];
    }
    const int src = __builtin_ctzll(__ballot(mine));
    bin = __builtin_amdgcn_readlane(bin, src);
    in_bin = __builtin_amdgcn_readlane(in_bin, src);
    need -= __builtin_amdgcn_readlane(before, src);
    least += (uint32_t)bin << shift;
    most = min(most, least + ((1u << shift) - 1u));
    T0 = least;
    if (in_bin == need) {  // the whole step is kept
      T0 = least - 1u;     // (no score's key is 0)
      need = 0;
      break;
    }
    // The counts of the round after next: their last readers are behind this
    // round's barrier, their next writers behind the one here.
    int* other = L.hist[(round + 1) & 1];
    if (round > 0) {
      for (int k = tid; k < P::kSlots; k += NT) other[k] = 0;
      __syncthreads();
    }
  }

  int gt = 0, eq = 0;
  each([&](int, uint32_t u) {
    gt += u > T0;
    eq += u == T0;
  });
  const int gt_in = wave_scan_add(gt), eq_in = wave_scan_add(eq);
  if (lane == 63) L.gt[wave] = gt_in, L.eq[wave] = eq_in;
  __syncthreads();
  int gt0 = gt_in - gt, eq0 = eq_in - eq;
#pragma unroll
  for (int w = 0; w < P::kWaves; ++w)
    if (w < wave) gt0 += L.gt[w], eq0 += L.eq[w];
  int at = a.sink + gt0 + min(eq0, need);
  int left = max(need - eq0, 0);
  each([&](int k, uint32_t u) {
    if (u > T0 || (u == T0 && left > 0)) {
      left -= u == T0;
      put(at++, lo + k);
    }
  });
  return kept;
}

template <typename T, bool SCORED, int NT>
__global__ __launch_bounds__(NT) void block_pick_kernel(const SelectArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint32_t s_key[];
  __shared__ Pick<NT> pick;
  SelectJob j;
  if (select_job(a, blockIdx.x, j)) pick_blocks<T, SCORED, NT>(a, j, pick, s_key, nullptr);
}

// Selection and attention of one query in one workgroup of eight waves, for
// few queries over short rows, where launches count: the list stays in LDS.
template <typename T>
__global__ __launch_bounds__(512, 1) void block_step_kernel(const SelectArgs a, const RowsArgs r) {
  extern __shared__ __attribute__((aligned(16))) uint32_t s_key[];  // key_words(a.max_blocks), then the list
  __shared__ __attribute__((aligned(16))) float s_rows[kRowsLds];
  __shared__ Pick<512> pick;
  SelectJob j;
  if (!select_job(a, blockIdx.x, j)) return;
  int32_t* list = reinterpret_cast<int32_t*>(s_key + key_words(a.max_blocks));
  const int kept = pick_blocks<T, false, 512>(a, j, pick, s_key, list);
  __syncthreads();
  rows_job<T, kRowsListed, false, 8>(r, blockIdx.x, s_rows, list, kept);
}

bool known(int dtype) { return dtype == HC_DTYPE_BF16 || dtype == HC_DTYPE_F16 || dtype == HC_DTYPE_F32; }

int check_shape(const char* what, int dtype, int batch, int q_heads, int kv_heads, int queries, int block) {
  if (!known(dtype)) return set_error(HC_ERR_INVALID, "%s: unknown dtype %d", what, dtype);
  if (batch < 0 || kv_heads < 1 || q_heads < 1 || q_heads % kv_heads || q_heads / kv_heads > 16 || queries < 0 ||
      (int64_t)batch * q_heads * std::max(queries, 1) > (1 << 24))
    return set_error(HC_ERR_INVALID,
                     "%s: batch=%d q_heads=%d kv_heads=%d queries=%d (q_heads a multiple of kv_heads, at most 16 of "
                     "it, at most 2^24 query rows)",
                     what, batch, q_heads, kv_heads, queries);
  if (block < HC_TILE || block % HC_TILE || block > (1 << 20))
    return set_error(HC_ERR_INVALID, "%s: block=%d (a multiple of %d)", what, block, HC_TILE);
  return HC_OK;
}

int check_q(const char* what, int dtype, const void* q, const int64_t* st) {
  const int per16 = dtype == HC_DTYPE_F32 ? 4 : 8;
  for (int i = 0; i < 3; ++i)
    if (st[i] % per16) return set_error(HC_ERR_INVALID, "%s: q strides must be multiples of 16 bytes", what);
  if (reinterpret_cast<uintptr_t>(q) & 15) return set_error(HC_ERR_INVALID, "%s: q must be 16-byte aligned", what);
  return HC_OK;
}

// Whether scores go through memory: rows whose keys LDS does not hold, and few
// queries over long rows -- one CU draws some 33 GB/s, so a workgroup that
// scores its row alone is slow where it has the device almost to itself (8
// queries of 512, 1024 and 4096 blocks: 10.3, 15.8 and 38 us against 9.4, 10.8
// and 14.5 through memory; 192 queries: 11.2, 17.4 and 42.6 against 12.3, 18.7
// and 43.3; 8 of 256 blocks: 7.7 against 8.8).
constexpr int kSoloBlocks = 256;
bool select_in_memory(int64_t jobs, int max_blocks) {
  return max_blocks > kPickKeys || (max_blocks > kSoloBlocks && jobs <= device_cus() / 2);
}
// Blocks that four waves pick from, and eight, sixteen beyond: keys that fit
// the threads' registers, by as few waves as that takes (8 queries of 1024,
// 2048, 4096 and 8192 blocks through memory, scores and all: 8.9, 10.2, 21.5
// and 29.8 us with four, 9.0, 9.7, 12.7 and 20.6 with eight, 11.4, 11.7, 14.2
// and 17.0 with sixteen; since then 8.8, 9.6, 10.7 and 15.5 as chosen).
constexpr int kFewBlocks = 1024, kMoreBlocks = 512 * Pick<512>::kHeld;

template <typename T, bool SCORED>
void launch_pick(const SelectArgs& a, dim3 grid, hipStream_t s) {
  const size_t lds = SCORED ? 0 : (size_t)std::max(key_words(a.max_blocks), 1) * sizeof(uint32_t);
  if (a.max_blocks <= kFewBlocks)
    hipLaunchKernelGGL((block_pick_kernel<T, SCORED, 256>), grid, dim3(256), lds, s, a);
  else if (a.max_blocks <= kMoreBlocks)
    hipLaunchKernelGGL((block_pick_kernel<T, SCORED, 512>), grid, dim3(512), lds, s, a);
  else
    hipLaunchKernelGGL((block_pick_kernel<T, SCORED, 1024>), grid, dim3(1024), lds, s, a);
}

int64_t score_pitch(int64_t max_blocks) { return (max_blocks + 63) / 64 * 64; }

}  // namespace
}  // namespace hc

using namespace hc;

extern "C" int hc_block_bounds(int dtype, const void* kstore, const int64_t* row_tile_off, const int32_t* row_len,
                               const int64_t* row_block_off, int rows, int block, int span, int fresh, int8_t* bounds,
                               int8_t* exps, void* stream) {
  clear_error();
  const int rc = check_shape("hc_block_bounds", dtype, rows, 1, 1, 1, block);
  if (rc) return rc;
  if (span < 0 || fresh < 0) return set_error(HC_ERR_INVALID, "hc_block_bounds: span=%d fresh=%d", span, fresh);
  if (rows == 0 || span == 0) return HC_OK;
  if (!kstore || !row_tile_off || !row_len || !row_block_off || !bounds || !exps)
    return set_error(HC_ERR_INVALID, "hc_block_bounds: null pointer argument");
  if ((reinterpret_cast<uintptr_t>(kstore) | reinterpret_cast<uintptr_t>(bounds)) & 15)
    return set_error(HC_ERR_INVALID, "hc_block_bounds: the store and the bounds must be 16-byte aligned");
  // One resident round of workgroups, each with its share of a row's blocks (16
  // rows of 1023 blocks of 64 tokens: 48.8, 47.3, 44.0 and 42.8 us with 3, 4, 8
  // and 16 workgroups a CU; 256 rows of 32: 24.0, 24.1, 28.3 and 31.1).
  const int per = (int)std::min<int64_t>(std::max<int64_t>((int64_t)rows * span / (8 * device_cus()), 1), 64);
  const int64_t grid = (int64_t)rows * ((span + (int64_t)per - 1) / per);
  if (grid > 0x7fffffffLL) return set_error(HC_ERR_INVALID, "hc_block_bounds: %d rows x %d blocks", rows, span);
  BoundArgs a = {kstore, row_tile_off, row_block_off, row_len, bounds, exps, rows, block / HC_TILE, span, fresh};
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case HC_DTYPE_BF16: launch_bounds<__bf16>(a, (unsigned)grid, s); break;
    case HC_DTYPE_F16: launch_bounds<_Float16>(a, (unsigned)grid, s); break;
    default: launch_bounds<float>(a, (unsigned)grid, s); break;
  }
  return check_launch("hc_block_bounds");
}

extern "C" size_t hc_block_select_scratch_size(int batch, int kv_heads, int queries, int max_blocks) {
  if (batch < 0 || kv_heads < 1 || queries < 0 || max_blocks < 0) return 0;
  const int64_t rows = (int64_t)batch * kv_heads;
  if (!select_in_memory((rows + 7) / 8 * 8 * queries, max_blocks)) return 0;
  return (size_t)rows * queries * score_pitch(max_blocks) * sizeof(float);
}

namespace {
// The checks and arguments of a selection.
int select_args(const char* what, int dtype, const void* q, const int64_t* q_strides, const int8_t* bounds,
                const int8_t* exps, const int64_t* row_block_off, const int32_t* row_len, const int32_t* query_counts,
                int batch, int q_heads, int kv_heads, int queries, int block, int max_blocks, int keep, int sink,
                int local, int32_t* idx, int32_t* counts, SelectArgs& a) {
  int rc = check_shape(what, dtype, batch, q_heads, kv_heads, queries, block);
  if (rc) return rc;
  if (sink < 0 || local < 1 || keep < 1 || keep > (1 << 24) || (int64_t)sink + local > keep || max_blocks < 0)
    return set_error(HC_ERR_INVALID,
                     "%s: keep=%d sink=%d local=%d max_blocks=%d (local at least 1, sink + local at most keep)", what,
                     keep, sink, local, max_blocks);
  if (batch == 0 || queries == 0) return HC_OK;
  if (!q || !q_strides || !bounds || !exps || !row_block_off || !row_len || !idx || !counts)
    return set_error(HC_ERR_INVALID, "%s: null pointer argument", what);
  if ((rc = check_q(what, dtype, q, q_strides))) return rc;
  if (reinterpret_cast<uintptr_t>(bounds) & 15)
    return set_error(HC_ERR_INVALID, "%s: the bounds must be 16-byte aligned", what);
  a = SelectArgs{};
  a.q = q, a.bounds = bounds, a.exps = exps, a.row_blk_off = row_block_off;
  a.row_len = row_len, a.query_counts = query_counts;
  for (int i = 0; i < 3; ++i) a.q_s[i] = q_strides[i];
  a.pitch = score_pitch(max_blocks), a.idx = idx, a.counts = counts;
  a.Hkv = kv_heads, a.G = q_heads / kv_heads, a.Q = queries, a.rows = batch * kv_heads, a.S = block;
  a.keep = keep, a.sink = sink, a.local = local, a.max_blocks = max_blocks;
  return HC_OK;
}

int launch_select(const char* what, int dtype, SelectArgs& a, void* scratch, hipStream_t s) {
  const int64_t jobs = ((int64_t)a.rows + 7) / 8 * 8 * a.Q;
  if (jobs > 0x7fffffffLL) return set_error(HC_ERR_INVALID, "%s: %lld queries", what, (long long)jobs);
  const dim3 grid((unsigned)jobs);
  if (!select_in_memory(jobs, a.max_blocks)) {
    switch (dtype) {
      case HC_DTYPE_BF16: launch_pick<__bf16, false>(a, grid, s); break;
      case HC_DTYPE_F16: launch_pick<_Float16, false>(a, grid, s); break;
      default: launch_pick<float, false>(a, grid, s); break;
    }
    return check_launch(what);
  }
  a.scores = reinterpret_cast<float*>(scratch);
  const int64_t most = ((int64_t)a.max_blocks + 32 * kScoreWaves - 1) / (32 * kScoreWaves);
  a.chunks = (int)std::max<int64_t>(std::min<int64_t>((8 * device_cus() + jobs - 1) / jobs, most), 1);
  if (jobs * a.chunks > 0x7fffffffLL)
    return set_error(HC_ERR_INVALID, "%s: %lld workgroups", what, (long long)(jobs * a.chunks));
  if (a.max_blocks > a.keep) {
    const dim3 g((unsigned)(jobs * a.chunks)), t(kScoreWaves * 64);
    switch (dtype) {
      case HC_DTYPE_BF16: hipLaunchKernelGGL(block_score_kernel<__bf16>, g, t, 0, s, a); break;
      case HC_DTYPE_F16: hipLaunchKernelGGL(block_score_kernel<_Float16>, g, t, 0, s, a); break;
      default: hipLaunchKernelGGL(block_score_kernel<float>, g, t, 0, s, a); break;
    }
    const int rc = check_launch(what);
    if (rc) return rc;
  }
  launch_pick<float, true>(a, grid, s);
  return check_launch(what);
}
}  // namespace

extern "C" int hc_block_select(int dtype, const void* q, const int64_t* q_strides, const int8_t* bounds,
                               const int8_t* exps, const int64_t* row_block_off, const int32_t* row_len,
                               const int32_t* query_counts, int batch, int q_heads, int kv_heads, int queries, int block,
                               int max_blocks, int keep, int sink, int local, int32_t* idx, int32_t* counts,
                               void* scratch, size_t scratch_bytes, void* stream) {
  clear_error();
  SelectArgs a;
  const int rc = select_args("hc_block_select", dtype, q, q_strides, bounds, exps, row_block_off, row_len, query_counts,
                             batch, q_heads, kv_heads, queries, block, max_blocks, keep, sink, local, idx, counts, a);
  if (rc || batch == 0 || queries == 0) return rc;
  const size_t need = hc_block_select_scratch_size(batch, kv_heads, queries, max_blocks);
  if (need > 0 && (!scratch || scratch_bytes < need || (reinterpret_cast<uintptr_t>(scratch) & 15)))
    return set_error(HC_ERR_INVALID, "hc_block_select: scratch too small (%zu < %zu bytes, 16-byte aligned)", scratch_bytes,
                     need);
  return launch_select("hc_block_select", dtype, a, scratch, (hipStream_t)stream);
}

namespace {
// The plan and workspace of hc_block_attn: one query a job, `waves` waves a
// workgroup, nsplit workgroups a job.
struct BlockPlan {
  int waves, nsplit;
  size_t part_o, bytes;
};
BlockPlan block_plan(int batch, int kv_heads, int G, int queries, int block, int keep) {
  // The least estimate in us: a wave's tiles one after another (2.4 each, the
  // latency of scattered blocks, behind 3.3 of start and end: 5.7, 8.6, 13.5,
  // 23.1 and 42.4 for 1, 2, 4, 8 and 16; more where the tiles of all waves on
  // the device take longer to stream) in as many rounds as the device needs; a
  // split adds the launch that folds it.  A CU holds three workgroups of four
  // waves or one of eight, which have at most 8 columns.  (8 to 512 queries of
  // 4 to 256 tiles: within 8 % of the best of twenty choices, but for 1.23 at 64
  // queries of 32 and 1.13 at 128 of 128.)
  BlockPlan p = {4, 1, 0, 0};
  const int64_t jobs = (int64_t)batch * kv_heads * queries, tiles = (int64_t)keep * (block / HC_TILE);
  const int64_t cus = device_cus();
  double best = 0.;
  for (int waves = 4; waves <= (G <= 8 ? 8 : 4); waves += 4)
    for (int ns : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
      if (ns > 1 && (int64_t)ns * waves > tiles) break;
      const int64_t slots = cus * (waves == 8 ? 1 : 3);
      const double rounds = (double)((jobs * ns + slots - 1) / slots);
      const double load = (double)std::min(jobs * ns, slots) * waves * HC_TILE_ELEMS * 4. / 5.5e6;
      const double own = 3.3 + std::max(2.4, load) * (double)((tiles + waves * ns - 1) / (waves * ns));
      const double t = rounds * own + (ns > 1 ? 4. : 0.);
      if (best == 0. || t < best * 0.98) best = t, p.waves = waves, p.nsplit = ns;
    }
  const size_t cols = (size_t)batch * kv_heads * queries * G * p.nsplit;
  p.part_o = cols * kPartO * sizeof(float);
  p.bytes = p.nsplit > 1 ? p.part_o + cols * 2 * sizeof(float) : 0;
  return p;
}
}  // namespace

extern "C" size_t hc_block_attn_workspace_size(int batch, int q_heads, int kv_heads, int queries, int block, int keep) {
  if (check_shape("hc_block_attn", HC_DTYPE_BF16, batch, q_heads, kv_heads, queries, block) || keep < 1 ||
      keep > (1 << 24))
    return 0;
  if (batch == 0 || queries == 0) return 0;
  return block_plan(batch, kv_heads, q_heads / kv_heads, queries, block, keep).bytes;
}

namespace {
// The checks and arguments of an attention over listed blocks.
int attn_args(const char* what, int dtype, const void* q, const int64_t* q_strides, const void* kstore,
              const void* vstore, const int64_t* row_tile_off, const int32_t* row_len, const int32_t* query_counts,
              const int32_t* idx, const int32_t* counts, int keep, int block, void* out, const int64_t* out_strides,
              int batch, int q_heads, int kv_heads, int queries, float scale, RowsArgs& r) {
  int rc = check_shape(what, dtype, batch, q_heads, kv_heads, queries, block);
  if (rc) return rc;
  if (keep < 1 || keep > (1 << 24) || (int64_t)keep * (block / HC_TILE) > (1 << 30))
    return set_error(HC_ERR_INVALID, "%s: keep=%d", what, keep);
  if (!(scale > 0.f) || std::isinf(scale)) return set_error(HC_ERR_INVALID, "%s: scale=%g", what, (double)scale);
  if (batch == 0 || queries == 0) return HC_OK;
  if (!q || !q_strides || !kstore || !vstore || !row_tile_off || !row_len || !idx || !counts || !out || !out_strides)
    return set_error(HC_ERR_INVALID, "%s: null pointer argument", what);
  if ((rc = check_q(what, dtype, q, q_strides))) return rc;
  if ((reinterpret_cast<uintptr_t>(kstore) | reinterpret_cast<uintptr_t>(vstore)) & 15)
    return set_error(HC_ERR_INVALID, "%s: tensors must be 16-byte aligned", what);
  r = RowsArgs{};
  r.q = q, r.kstore = kstore, r.vstore = vstore, r.row_tile_off = row_tile_off, r.row_len = row_len;
  r.query_counts = query_counts, r.idx = idx, r.counts = counts, r.keep = keep, r.tpb = block / HC_TILE;
  r.Hkv = kv_heads, r.G = q_heads / kv_heads, r.Q = queries, r.rows = batch * kv_heads, r.qpb = 1, r.ncb = queries;
  r.nsplit = 1, r.scale_log2 = scale * 1.4426950408889634f, r.out = out;
  for (int i = 0; i < 3; ++i) r.q_s[i] = q_strides[i], r.o_s[i] = out_strides[i];
  return HC_OK;
}

int launch_attn(int dtype, RowsArgs& r, const BlockPlan& p, void* workspace, hipStream_t s) {
  r.nsplit = p.nsplit;
  if (p.nsplit > 1) {
    r.part_o = reinterpret_cast<float*>(workspace);
    r.part_ml = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + p.part_o);
  }
  const int rc = launch_block_rows(dtype, r, p.waves, s);
  if (rc || p.nsplit == 1) return rc;
  MergeArgs mg = {};
  mg.row_o = r.part_o, mg.row_ml = r.part_ml, mg.nsplit = p.nsplit;
  mg.Hkv = r.Hkv, mg.G = r.G, mg.Q = r.Q, mg.out = r.out;
  for (int i = 0; i < 3; ++i) mg.o_s[i] = r.o_s[i];
  return launch_merge(dtype, mg, (int64_t)r.rows * r.Q * r.G, s);
}

// Whether one launch does it all: few queries, short rows and lists that eight
// waves attend unsplit.  16 of 384, 512, 640, 768 and 1024 blocks kept for 8
// queries: 13.3, 14.9, 16.5, 16.9 and 18.8 us in one launch, 15.6, 16.5, 16.3,
// 16.3 and 16.2 as selection (scores through memory) and attention; 64 queries
// 16.6 against 17.8 at 512 and 20.1 against 18.6 at 1024; with 192, which score
// their own rows either way, one launch stays 2 to 3 us ahead.  The list lies in
// LDS: 2048 entries beside the waves' states and the keys take 49 KB.
constexpr int kStepBlocks = 512;
bool one_launch(const BlockPlan& p, int64_t queries, int max_blocks, int keep) {
  return p.waves == 8 && p.nsplit == 1 && queries <= device_cus() && max_blocks <= kStepBlocks && keep <= 2048;
}

size_t align16(size_t n) { return (n + 15) / 16 * 16; }
}  // namespace

extern "C" int hc_block_attn(int dtype, const void* q, const int64_t* q_strides, const void* kstore,
                             const void* vstore, const int64_t* row_tile_off, const int32_t* row_len,
                             const int32_t* query_counts, const int32_t* idx, const int32_t* counts, int keep, int block,
                             void* out, const int64_t* out_strides, int batch, int q_heads, int kv_heads, int queries,
                             float scale, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  RowsArgs r;
  const int rc = attn_args("hc_block_attn", dtype, q, q_strides, kstore, vstore, row_tile_off, row_len, query_counts, idx,
                           counts, keep, block, out, out_strides, batch, q_heads, kv_heads, queries, scale, r);
  if (rc || batch == 0 || queries == 0) return rc;
  const BlockPlan p = block_plan(batch, kv_heads, r.G, queries, block, keep);
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return set_error(HC_ERR_INVALID, "hc_block_attn: workspace too small (%zu < %zu bytes, 16-byte aligned)",
                     workspace_bytes, p.bytes);
  return launch_attn(dtype, r, p, workspace, (hipStream_t)stream);
}

extern "C" size_t hc_block_step_workspace_size(int batch, int q_heads, int kv_heads, int queries, int block,
                                               int max_blocks, int keep) {
  if (check_shape("hc_block_step", HC_DTYPE_BF16, batch, q_heads, kv_heads, queries, block) || keep < 1 ||
      keep > (1 << 24) || max_blocks < 0 || batch == 0 || queries == 0)
    return 0;
  const BlockPlan p = block_plan(batch, kv_heads, q_heads / kv_heads, queries, block, keep);
  if (one_launch(p, (int64_t)batch * kv_heads * queries, max_blocks, keep)) return 0;
  return align16(hc_block_select_scratch_size(batch, kv_heads, queries, max_blocks)) + p.bytes;
}

extern "C" int hc_block_step(int dtype, const void* q, const int64_t* q_strides, const void* kstore,
                             const void* vstore, const int64_t* row_tile_off, const int32_t* row_len,
                             const int32_t* query_counts, const int8_t* bounds, const int8_t* exps,
                             const int64_t* row_block_off, int batch, int q_heads, int kv_heads, int queries, int block,
                             int max_blocks, int keep, int sink, int local, float scale, int32_t* idx, int32_t* counts, void* out,
                             const int64_t* out_strides, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  const char* what = "hc_block_step";
  SelectArgs a;
  RowsArgs r;
  int rc = select_args(what, dtype, q, q_strides, bounds, exps, row_block_off, row_len, query_counts, batch, q_heads,
                       kv_heads, queries, block, max_blocks, keep, sink, local, idx, counts, a);
  if (!rc)
    rc = attn_args(what, dtype, q, q_strides, kstore, vstore, row_tile_off, row_len, query_counts, idx, counts, keep,
                   block, out, out_strides, batch, q_heads, kv_heads, queries, scale, r);
  if (rc || batch == 0 || queries == 0) return rc;
  const size_t need = hc_block_step_workspace_size(batch, q_heads, kv_heads, queries, block, max_blocks, keep);
  if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return set_error(HC_ERR_INVALID, "hc_block_step: workspace too small (%zu < %zu bytes, 16-byte aligned)",
                     workspace_bytes, need);
  hipStream_t s = (hipStream_t)stream;
  const BlockPlan p = block_plan(batch, kv_heads, r.G, queries, block, keep);
  if (one_launch(p, (int64_t)a.rows * queries, max_blocks, keep)) {
    const dim3 grid((unsigned)((a.rows + 7) / 8 * 8 * queries)), t(512);
    const size_t lds = ((size_t)key_words(max_blocks) + keep) * sizeof(int32_t);
    switch (dtype) {
      case HC_DTYPE_BF16: hipLaunchKernelGGL(block_step_kernel<__bf16>, grid, t, lds, s, a, r); break;
      case HC_DTYPE_F16: hipLaunchKernelGGL(block_step_kernel<_Float16>, grid, t, lds, s, a, r); break;
      default: hipLaunchKernelGGL(block_step_kernel<float>, grid, t, lds, s, a, r); break;
    }
    return check_launch(what);
  }
  if ((rc = launch_select(what, dtype, a, workspace, s))) return rc;
  return launch_attn(dtype, r, p,
                     reinterpret_cast<char*>(workspace) +
                         align16(hc_block_select_scratch_size(batch, kv_heads, queries, max_blocks)),
                     s);
}
