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

// One workgroup a block.  K chunk c = ((h*4+s)*4+g)*16+m of a tile holds token
// 16h+m, channels 32s+8g+[0,8): a thread reads both halves h of its (s, g, m),
// so a wave's load is 1 KB in a row, and the 16 lanes m of a channel group are
// folded by row rotations.  Bound by the key stream.
template <typename T>
__global__ __launch_bounds__(256) void block_bounds_kernel(const BoundArgs a) {
  __shared__ float s_top[4];
  const int row = blockIdx.x % a.rows, j0 = blockIdx.x / a.rows;
  const int len = max(a.row_len[row], 0), S = a.tpb * HC_TILE;
  const int j = len / S - 1 - j0;
  if (j < 0) return;
  if (a.fresh > 0 && (int64_t)(j + 1) * S <= (int64_t)len - a.fresh) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* kb = reinterpret_cast<const T*>(a.kstore) + (a.row_tile_off[row] + (int64_t)j * a.tpb) * HC_TILE_ELEMS;
  float hi[8], lo[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) hi[e] = -INFINITY, lo[e] = INFINITY;
  for (int t = 0; t < a.tpb; ++t) {
    const T* kt = kb + (int64_t)t * HC_TILE_ELEMS + tid * 8;
    const typename Elem<T>::vec8 x = load8_stream<T>(kt), y = load8_stream<T>(kt + 2048);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      hi[e] = fmaxf(hi[e], fmaxf(vec8_at<T>(x, e), vec8_at<T>(y, e)));
      lo[e] = fminf(lo[e], fminf(vec8_at<T>(x, e), vec8_at<T>(y, e)));
    }
  }
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    hi[e] = fmaxf(hi[e], dpp_mov<0x128>(hi[e])), lo[e] = fminf(lo[e], dpp_mov<0x128>(lo[e]));  // row_ror:8
    hi[e] = fmaxf(hi[e], dpp_mov<0x124>(hi[e])), lo[e] = fminf(lo[e], dpp_mov<0x124>(lo[e]));  // row_ror:4
    hi[e] = fmaxf(hi[e], dpp_mov<0x4E>(hi[e])), lo[e] = fminf(lo[e], dpp_mov<0x4E>(lo[e]));    // quad_perm
    hi[e] = fmaxf(hi[e], dpp_mov<0xB1>(hi[e])), lo[e] = fminf(lo[e], dpp_mov<0xB1>(lo[e]));
    top = fmaxf(top, fmaxf(fabsf(hi[e]), fabsf(lo[e])));
  }
  top = rows4_max(top);
  if (lane == 0) s_top[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
  const int ex = least_exp(top);
  const int64_t blk = a.row_blk_off[row] + j;
  if ((lane & 15) == 0) {
    // Channel group tid / 16 = 4s + g: channels 8 * (tid / 16) + [0, 8).
    const float down = power2(-ex);
    uint32_t wh[2] = {0, 0}, wl[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      wh[e >> 2] |= (uint32_t)(clamp8(ceilf(hi[e] * down)) & 0xff) << (8 * (e & 3));
      wl[e >> 2] |= (uint32_t)(clamp8(floorf(lo[e] * down)) & 0xff) << (8 * (e & 3));
    }
    int8_t* bp = a.bounds + blk * kBoundBytes + 8 * (tid >> 4);
    *reinterpret_cast<uint2*>(bp) = make_uint2(wh[0], wh[1]);
    *reinterpret_cast<uint2*>(bp + HC_HEAD_DIM) = make_uint2(wl[0], wl[1]);
  }
  if (tid == 0) a.exps[blk] = (int8_t)ex;
}

// ---- scores ------------------------------------------------------------------
struct SelectArgs {
  const void* q;
  int64_t q_s[3];
  const int8_t *bounds, *exps;
  const int64_t* row_blk_off;
  const int32_t* row_len;
  float* scores;  // [row * Q + query][pitch]
  int64_t pitch;
  int32_t *idx, *counts;
  int Hkv, G, Q, rows, S, keep, sink, local;
  int qpb, ncb;   // queries of a 16-column block, such blocks of a row
  int chunks;     // workgroups along the blocks of a row
  int max_blocks; // visible blocks a row has room for in scores; a row of more selects nothing
};

// Visible tokens and blocks of query i of a row.
__device__ __forceinline__ int visible(int len, int Q, int i) { return min(max(len - Q + 1 + i, 0), len); }

// A wave scores 16 blocks at a time against the 16 columns (query, head):
// the blocks are the A operand (16 bytes a lane of the 256 of a block, so a
// wave's four loads read 4 KB in all), the queries' positive and negative
// parts the B operand.  Bound by the index's bytes.
constexpr int kScoreWaves = 4;
template <typename T>
__global__ __launch_bounds__(kScoreWaves * 64) void block_score_kernel(const SelectArgs a) {
  __shared__ float s_s[kScoreWaves][16][17];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, n = lane & 15;
  const int jobs = a.rows * a.ncb;
  const int job = blockIdx.x % jobs, chunk = blockIdx.x / jobs;
  const int row = job / a.ncb, cb = job % a.ncb;
  const int b = row / a.Hkv, kv = row % a.Hkv;
  const int i0 = cb * a.qpb, nq = min(a.qpb, a.Q - i0), ncols = nq * a.G;
  const int len = max(a.row_len[row], 0);
  // Blocks whose score may decide: those between the first `sink` and the
  // last `local` of some query that has more blocks than it keeps.
  const int have = (visible(len, a.Q, i0 + nq - 1) + a.S - 1) / a.S;
  const int lo = a.sink, hi = have <= a.keep || have > a.max_blocks ? a.sink : have - a.local;
  const int steps = (hi - lo + 15) / 16;
  const int st0 = chunk * kScoreWaves + wave;
  if (steps <= chunk * kScoreWaves) return;  // whole workgroups only: no barrier is missed

  const bool col_ok = n < ncols;
  i32x4 qp[4];  // B operands: steps 0, 1 the positive parts, 2, 3 the negative ones
  float unit;
  {
    const T* p = reinterpret_cast<const T*>(a.q) + b * a.q_s[0] + (int64_t)(kv * a.G + (col_ok ? n % a.G : 0)) * a.q_s[1] +
                 (int64_t)(i0 + (col_ok ? n / a.G : 0)) * a.q_s[2] + 16 * g;
    float x[2][16];
    float top = 0.f;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const typename Elem<T>::vec8 v = load8<T>(p + 64 * s + 8 * u);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = col_ok ? vec8_at<T>(v, e) : 0.f;
          x[s][8 * u + e] = y;
          top = fmaxf(top, fabsf(y));
        }
      }
    const int ex = least_exp(rows4_max(top));
    const float down = power2(-ex);
    unit = power2(ex);
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
        qp[s][w] = (int)pos;
        qp[2 + s][w] = (int)neg;
      }
  }
  const int64_t blk0 = a.row_blk_off[row];
  for (int st = st0; st < steps; st += kScoreWaves * a.chunks) {
    const int j0 = lo + 16 * st;
    const int mine = min(j0 + n, hi - 1);  // past the end: the last block again, not stored
    const int8_t* bp = a.bounds + (blk0 + mine) * kBoundBytes + 16 * g;
    i32x4 acc = {0, 0, 0, 0};
    i32x4 x[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) x[s] = *reinterpret_cast<const i32x4*>(bp + 64 * s);
    const float eu = power2(a.exps[blk0 + mine]);
#pragma unroll
    for (int s = 0; s < 4; ++s) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[s], qp[s], acc, 0, 0, 0);
    // Lane: blocks j0 + 4g + r, column n.
#pragma unroll
    for (int r = 0; r < 4; ++r) s_s[wave][4 * g + r][n] = (float)acc[r] * unit;
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    __builtin_amdgcn_wave_barrier();
    for (int y = lane; y < 16 * nq; y += 64) {
      const int jj = y & 15, i = y >> 4;
      float best = s_s[wave][jj][i * a.G];
      for (int h = 1; h < a.G; ++h) best = fmaxf(best, s_s[wave][jj][i * a.G + h]);
      best *= __shfl(eu, jj, 64);
      if (j0 + jj < hi) a.scores[((int64_t)row * a.Q + i0 + i) * a.pitch + j0 + jj] = best;
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// ---- selection ---------------------------------------------------------------
// One workgroup a query: the threshold score by four 8-bit radix passes over
// the keys of the middle blocks, then one ordered pass that writes the kept
// blocks.  The keys live in LDS where they fit (kPickKeys), else each pass
// reads the scores again.  Bound by the latency of its dependent passes.
constexpr int kPickThreads = 512;
constexpr int kPickKeys = 8192;
__global__ __launch_bounds__(kPickThreads) void block_pick_kernel(const SelectArgs a) {
  __shared__ uint32_t s_key[kPickKeys];
  __shared__ int s_hist[256];
  __shared__ int s_scan[kPickThreads / 64];
  __shared__ int s_digit, s_need;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t x = blockIdx.x;  // row * Q + query
  const int row = (int)(x / a.Q), i = (int)(x % a.Q);
  const int len = max(a.row_len[row], 0);
  const int have = (visible(len, a.Q, i) + a.S - 1) / a.S;
  int32_t* out = a.idx + x * a.keep;
  const bool fits = have <= a.max_blocks;
  if (tid == 0) a.counts[x] = fits ? min(have, a.keep) : -1;
  if (!fits) {
    for (int k = tid; k < a.keep; k += kPickThreads) out[k] = -1;
    return;
  }
  if (have <= a.keep) {
    for (int k = tid; k < a.keep; k += kPickThreads) out[k] = k < have ? k : -1;
    return;
  }
  const int lo = a.sink, nmid = have - a.local - lo;
  int need = a.keep - a.sink - a.local;  // < nmid
  for (int k = tid; k < a.sink; k += kPickThreads) out[k] = k;
  for (int k = tid; k < a.local; k += kPickThreads) out[a.keep - a.local + k] = have - a.local + k;
  if (need == 0) return;
  const float* sc = a.scores + x * a.pitch + lo;
  const bool in_lds = nmid <= kPickKeys;
  if (in_lds) {
    for (int k = tid; k < nmid; k += kPickThreads) s_key[k] = order_key(sc[k]);
  }
  auto key = [&](int k) { return in_lds ? s_key[k] : order_key(sc[k]); };
  uint32_t prefix = 0, mask = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) s_hist[tid] = 0;
    __syncthreads();
    for (int k = tid; k < nmid; k += kPickThreads) {
      const uint32_t u = key(k);
      if ((u & mask) == prefix) atomicAdd(&s_hist[(u >> shift) & 255], 1);
    }
    __syncthreads();
    if (wave == 0) {
      // Lane y: bins 255 - 4y .. 252 - 4y; keys above its first bin, then the
      // bin in which the need-th highest key lies.
      int c[4], sum = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) sum += c[u] = s_hist[255 - 4 * lane - u];
      int incl = sum;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(incl, d, 64);
        if (lane >= d) incl += v;
      }
      int above = incl - sum;
      if (above < need && need <= incl) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (above < need && need <= above + c[u]) {
            s_digit = 255 - 4 * lane - u;
            s_need = need - above;
          }
          above += c[u];
        }
      }
    }
    __syncthreads();
    prefix |= (uint32_t)s_digit << shift;
    mask |= 255u << shift;
    need = s_need;
  }
  // Keys above `prefix` are kept, and the first `need` equal to it.  Every
  // thread takes a run of blocks; two scans (equal keys, then kept ones) give
  // the places.
  const int run = (nmid + kPickThreads - 1) / kPickThreads;
  const int k0 = min(tid * run, nmid), k1 = min(k0 + run, nmid);
  int eq = 0, gt = 0;
  for (int k = k0; k < k1; ++k) {
    const uint32_t u = key(k);
    eq += u == prefix;
    gt += u > prefix;
  }
  auto scan = [&](int v) {  // exclusive, over the workgroup
    int incl = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(incl, d, 64);
      if (lane >= d) incl += u;
    }
    __syncthreads();
    if (lane == 63) s_scan[wave] = incl;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < wave; ++w) before += s_scan[w];
    return before + incl - v;
  };
  const int eq0 = scan(eq);
  const int take = min(max(need - eq0, 0), eq);
  int at = a.sink + scan(gt + take);
  int left = take;
  for (int k = k0; k < k1; ++k) {
    const uint32_t u = key(k);
    if (u > prefix || (u == prefix && left > 0)) {
      left -= u == prefix;
      out[at++] = lo + k;
    }
  }
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
  const int64_t grid = (int64_t)rows * span;
  if (grid > 0x7fffffffLL) return set_error(HC_ERR_INVALID, "hc_block_bounds: %d rows x %d blocks", rows, span);
  BoundArgs a = {kstore, row_tile_off, row_block_off, row_len, bounds, exps, rows, block / HC_TILE, span, fresh};
  hipStream_t s = (hipStream_t)stream;
  const dim3 g((unsigned)grid), t(256);
  switch (dtype) {
    case HC_DTYPE_BF16: hipLaunchKernelGGL(block_bounds_kernel<__bf16>, g, t, 0, s, a); break;
    case HC_DTYPE_F16: hipLaunchKernelGGL(block_bounds_kernel<_Float16>, g, t, 0, s, a); break;
    default: hipLaunchKernelGGL(block_bounds_kernel<float>, g, t, 0, s, a); break;
  }
  return check_launch("hc_block_bounds");
}

extern "C" size_t hc_block_select_scratch_size(int batch, int kv_heads, int queries, int max_blocks) {
  if (batch < 0 || kv_heads < 1 || queries < 0 || max_blocks < 0) return 0;
  return (size_t)batch * kv_heads * queries * score_pitch(max_blocks) * sizeof(float);
}

extern "C" int hc_block_select(int dtype, const void* q, const int64_t* q_strides, const int8_t* bounds,
                               const int8_t* exps, const int64_t* row_block_off, const int32_t* row_len, int batch,
                               int q_heads, int kv_heads, int queries, int block, int max_blocks, int keep, int sink,
                               int local, int32_t* idx, int32_t* counts, void* scratch, size_t scratch_bytes,
                               void* stream) {
  clear_error();
  int rc = check_shape("hc_block_select", dtype, batch, q_heads, kv_heads, queries, block);
  if (rc) return rc;
  if (sink < 0 || local < 1 || keep < 1 || keep > (1 << 24) || (int64_t)sink + local > keep || max_blocks < 0)
    return set_error(HC_ERR_INVALID,
                     "hc_block_select: keep=%d sink=%d local=%d max_blocks=%d (local at least 1, sink + local at most "
                     "keep)",
                     keep, sink, local, max_blocks);
  if (batch == 0 || queries == 0) return HC_OK;
  if (!q || !q_strides || !bounds || !exps || !row_block_off || !row_len || !idx || !counts)
    return set_error(HC_ERR_INVALID, "hc_block_select: null pointer argument");
  if ((rc = check_q("hc_block_select", dtype, q, q_strides))) return rc;
  if (reinterpret_cast<uintptr_t>(bounds) & 15)
    return set_error(HC_ERR_INVALID, "hc_block_select: the bounds must be 16-byte aligned");
  const size_t need = hc_block_select_scratch_size(batch, kv_heads, queries, max_blocks);
  if (need > 0 && (!scratch || scratch_bytes < need))
    return set_error(HC_ERR_INVALID, "hc_block_select: scratch too small (%zu < %zu bytes)", scratch_bytes, need);
  SelectArgs a;
  a.q = q, a.bounds = bounds, a.exps = exps, a.row_blk_off = row_block_off, a.row_len = row_len;
  for (int i = 0; i < 3; ++i) a.q_s[i] = q_strides[i];
  a.scores = reinterpret_cast<float*>(scratch), a.pitch = score_pitch(max_blocks), a.idx = idx, a.counts = counts;
  a.Hkv = kv_heads, a.G = q_heads / kv_heads, a.Q = queries, a.rows = batch * kv_heads, a.S = block;
  a.keep = keep, a.sink = sink, a.local = local, a.max_blocks = max_blocks;
  a.qpb = std::max(1, std::min(queries, 16 / a.G)), a.ncb = (queries + a.qpb - 1) / a.qpb;
  const int64_t jobs = (int64_t)a.rows * a.ncb;
  const int64_t most = (max_blocks + 16 * kScoreWaves - 1) / (16 * kScoreWaves);
  a.chunks = (int)std::max<int64_t>(std::min<int64_t>((8 * device_cus() + jobs - 1) / jobs, most), 1);
  const int64_t grid = jobs * a.chunks;
  if (grid > 0x7fffffffLL) return set_error(HC_ERR_INVALID, "hc_block_select: %lld workgroups", (long long)grid);
  hipStream_t s = (hipStream_t)stream;
  if (max_blocks > keep) {
    const dim3 g((unsigned)grid), t(kScoreWaves * 64);
    switch (dtype) {
      case HC_DTYPE_BF16: hipLaunchKernelGGL(block_score_kernel<__bf16>, g, t, 0, s, a); break;
      case HC_DTYPE_F16: hipLaunchKernelGGL(block_score_kernel<_Float16>, g, t, 0, s, a); break;
      default: hipLaunchKernelGGL(block_score_kernel<float>, g, t, 0, s, a); break;
    }
    if ((rc = check_launch("hc_block_select(scores)"))) return rc;
  }
  hipLaunchKernelGGL(block_pick_kernel, dim3((unsigned)(a.rows * a.Q)), dim3(kPickThreads), 0, s, a);
  return check_launch("hc_block_select");
}

namespace {
// The plan and workspace of hc_block_attn: one query a job.
struct BlockPlan {
  int nsplit;
  size_t part_o, bytes;
};
BlockPlan block_plan(int batch, int kv_heads, int G, int queries, int block, int keep) {
  BlockPlan p;
  p.nsplit = rows_plan(batch * kv_heads * queries, G, 1, (int64_t)keep * (block / HC_TILE)).nsplit;
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

extern "C" int hc_block_attn(int dtype, const void* q, const int64_t* q_strides, const void* kstore,
                             const void* vstore, const int64_t* row_tile_off, const int32_t* row_len,
                             const int32_t* idx, const int32_t* counts, int keep, int block, void* out,
                             const int64_t* out_strides, int batch, int q_heads, int kv_heads, int queries,
                             float scale, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  int rc = check_shape("hc_block_attn", dtype, batch, q_heads, kv_heads, queries, block);
  if (rc) return rc;
  if (keep < 1 || keep > (1 << 24) || (int64_t)keep * (block / HC_TILE) > 0x7fffffffLL)
    return set_error(HC_ERR_INVALID, "hc_block_attn: keep=%d", keep);
  if (!(scale > 0.f) || std::isinf(scale)) return set_error(HC_ERR_INVALID, "hc_block_attn: scale=%g", (double)scale);
  if (batch == 0 || queries == 0) return HC_OK;
  if (!q || !q_strides || !kstore || !vstore || !row_tile_off || !row_len || !idx || !counts || !out || !out_strides)
    return set_error(HC_ERR_INVALID, "hc_block_attn: null pointer argument");
  if ((rc = check_q("hc_block_attn", dtype, q, q_strides))) return rc;
  if ((reinterpret_cast<uintptr_t>(kstore) | reinterpret_cast<uintptr_t>(vstore) |
       reinterpret_cast<uintptr_t>(workspace)) & 15)
    return set_error(HC_ERR_INVALID, "hc_block_attn: tensors must be 16-byte aligned");
  const int G = q_heads / kv_heads;
  const BlockPlan p = block_plan(batch, kv_heads, G, queries, block, keep);
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes))
    return set_error(HC_ERR_INVALID, "hc_block_attn: workspace too small (%zu < %zu bytes)", workspace_bytes, p.bytes);
  RowsArgs r = {};
  r.q = q, r.kstore = kstore, r.vstore = vstore, r.row_tile_off = row_tile_off, r.row_len = row_len;
  r.idx = idx, r.counts = counts, r.keep = keep, r.tpb = block / HC_TILE;
  r.Hkv = kv_heads, r.G = G, r.Q = queries, r.rows = batch * kv_heads, r.qpb = 1, r.ncb = queries;
  r.nsplit = p.nsplit, r.scale_log2 = scale * 1.4426950408889634f, r.out = out;
  for (int i = 0; i < 3; ++i) r.q_s[i] = q_strides[i], r.o_s[i] = out_strides[i];
  if (p.nsplit > 1) {
    r.part_o = reinterpret_cast<float*>(workspace);
    r.part_ml = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + p.part_o);
  }
  hipStream_t s = (hipStream_t)stream;
  if ((rc = launch_block_rows(dtype, r, s)) || p.nsplit == 1) return rc;
  MergeArgs mg = {};
  mg.row_o = r.part_o, mg.row_ml = r.part_ml, mg.nsplit = p.nsplit;
  mg.Hkv = kv_heads, mg.G = G, mg.Q = queries, mg.out = out;
  for (int i = 0; i < 3; ++i) mg.o_s[i] = out_strides[i];
  return launch_merge(dtype, mg, (int64_t)batch * queries * q_heads, s);
}
