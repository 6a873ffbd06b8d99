// Attention over the rows of the ragged store for a few queries a row, and
// the fold of partial results (see hc_rows.h).
//
// Bound by HBM: a token's K and V (512 bytes in 16 bits) feed 4 * 128 * G
// operations per query.  A workgroup's four waves take every fourth tile of
// its split straight into the operand registers (two tile buffers, the next
// tile's loads in flight while one is attended) and are combined through LDS.
#include <algorithm>

#include "hc_rows.h"

namespace hc {
namespace {

constexpr int kRowsWaves = 4;
constexpr int kRowsPitch = HC_HEAD_DIM + 4;

template <typename T, bool LIST>
__global__ __launch_bounds__(kRowsWaves * 64, sizeof(T) == 4 ? 1 : 2) void rows_attn_kernel(const RowsArgs a) {
  typedef typename Elem<T>::vec8 vec8;
  __shared__ float s_o[kRowsWaves][16][kRowsPitch];
  __shared__ float s_m[kRowsWaves][16], s_l[kRowsWaves][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, n = lane & 15;
  const int jobs = a.rows * a.ncb;
  const int job = blockIdx.x % jobs, split = blockIdx.x / jobs;
  const int row = job / a.ncb, cb = job % a.ncb;
  const int b = row / a.Hkv, kv = row % a.Hkv;
  const int len = max(a.row_len[row], 0);

  // Column n: query i0 + n / G, head n % G of the row's group.
  const int i0 = cb * a.qpb, nq = min(a.qpb, a.Q - i0), ncols = nq * a.G;
  const bool col_ok = n < ncols;
  const int qi = col_ok ? n / a.G : nq - 1, gi = col_ok ? n % a.G : 0;
  const int lim_lo = min(max(len - a.Q + 1 + i0, 0), len);
  const int lim_hi = min(max(len - a.Q + i0 + nq, 0), len);
  const int lim = min(max(len - a.Q + 1 + i0 + qi, 0), len);

  vec8 qreg[4];
  {
    const T* qp = reinterpret_cast<const T*>(a.q) + b * a.q_s[0] + (int64_t)(kv * a.G + gi) * a.q_s[1] +
                  (int64_t)(i0 + qi) * a.q_s[2] + 8 * g;
#pragma unroll
    for (int s = 0; s < 4; ++s) qreg[s] = col_ok ? load8<T>(qp + 32 * s) : zero8<T>();
  }

  // Tiles of the job, this workgroup's share of them and this wave's: entries
  // e0 + wave, e0 + wave + 4, ...
  const int vis = (lim_hi + HC_TILE - 1) / HC_TILE;
  const int64_t job_q = (int64_t)row * a.Q + i0;  // LIST: one query a job
  int entries = vis;
  bool void_list = false;  // no selection was made: the output is NaN
  if constexpr (LIST) {
    const int c = a.counts[job_q];
    void_list = c < 0;
    entries = vis > 0 ? min(max(c, 0), a.keep) * a.tpb : 0;
  }
  const int e0 = (int)((int64_t)entries * split / a.nsplit), e1 = (int)((int64_t)entries * (split + 1) / a.nsplit);
  const int cnt = max((e1 - e0 - wave + kRowsWaves - 1) / kRowsWaves, 0);

  float m = -INFINITY, l = 0.f;
  f32x4 o[8];
#pragma unroll
  for (int mt = 0; mt < 8; ++mt) o[mt] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int64_t base = a.row_tile_off[row] * (int64_t)HC_TILE_ELEMS + lane * 8;
  const T* kb = reinterpret_cast<const T*>(a.kstore) + base;
  const T* vb = reinterpret_cast<const T*>(a.vstore) + base;
  vec8 kA[8], vA[8], kB[8], vB[8];
  for (int c0 = 0; c0 < cnt; c0 += 64) {
    const int nt = min(cnt - c0, 64);
    // LIST: lane x holds the tile of the wave's entry c0 + x, -1 for one that
    // is not a visible tile of the row (such an entry attends nothing).
    int mine = 0;
    if constexpr (LIST) {
      const int e = e0 + wave + (c0 + min(lane, nt - 1)) * kRowsWaves;
      const int blk = a.idx[job_q * a.keep + e / a.tpb];
      const int64_t t = (int64_t)blk * a.tpb + e % a.tpb;
      mine = blk >= 0 && t < vis ? (int)t : -1;
    }
    auto tile_of = [&](int i) {
      if constexpr (LIST) return __builtin_amdgcn_readlane(mine, i);
      return e0 + wave + (c0 + i) * kRowsWaves;
    };
    auto fetch = [&](vec8(&kr)[8], vec8(&vr)[8], int i) {
      const int t = max(tile_of(min(i, nt - 1)), 0);
      load_rows_tile<T>(kr, vr, kb, vb, (int64_t)t * HC_TILE_ELEMS);
    };
    auto attend = [&](vec8(&kr)[8], vec8(&vr)[8], int i) {
      const int t = tile_of(i);
      const bool live = !LIST || t >= 0;
      attend_rows<T, !LIST>(kr, vr, qreg, max(t, 0) * HC_TILE, live ? lim : 0, live ? lim_lo : 0, live ? lim_hi : 0, lane,
                     a.scale_log2, m, l, o);
    };
    // The loads of the pair's second tile and of the next pair's first are
    // unconditional (past the end they read the last tile again), so each
    // wait leaves the younger tile in flight.
    fetch(kA, vA, 0);
    for (int i = 0; i < nt; i += 2) {
      fetch(kB, vB, i + 1);
      __builtin_amdgcn_sched_barrier(0);
      attend(kA, vA, i);
      __builtin_amdgcn_sched_barrier(0);
      fetch(kA, vA, i + 2);
      __builtin_amdgcn_sched_barrier(0);
      if (i + 1 < nt) attend(kB, vB, i + 1);
      __builtin_amdgcn_sched_barrier(0);
    }
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
  for (int c = threadIdx.x >> 5; c < ncols; c += kRowsWaves * 2) {
    const int d0 = 4 * (threadIdx.x & 31);
    float M = s_m[0][c];
#pragma unroll
    for (int w = 1; w < kRowsWaves; ++w) M = fmaxf(M, s_m[w][c]);
    float L = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kRowsWaves; ++w) {
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
      const float inv = M == -INFINITY ? 0.f : 1.f / L;
      T* op = reinterpret_cast<T*>(a.out) + b * a.o_s[0] + (int64_t)(kv * a.G + hd) * a.o_s[1] +
              (int64_t)i * a.o_s[2] + d0;
#pragma unroll
      for (int e = 0; e < 4; ++e) op[e] = Elem<T>::from_f32(M == -INFINITY ? 0.f : acc[e] * inv);
    }
  }
}

// One workgroup an output row: 8 groups of 32 threads (4 channels each) take
// every eighth partial, kBatch of them in flight, and are combined in LDS.
constexpr int kMergeThreads = 256;
template <typename T>
__global__ __launch_bounds__(kMergeThreads) void merge_kernel(const MergeArgs a) {
  constexpr int kGroups = kMergeThreads / 32, kBatch = 4;
  __shared__ float s_m[kGroups], s_l[kGroups];
  __shared__ f32x4 s_o[kGroups][32];
  const int Hq = a.Hkv * a.G;
  const int64_t x = blockIdx.x;  // (b * Q + i) * Hq + head
  const int hq = (int)(x % Hq);
  const int64_t bi = x / Hq;
  const int64_t b = bi / a.Q;
  const int i = (int)(bi % a.Q), kv = hq / a.G, gi = hq % a.G;
  const int p0 = a.info ? a.info[2 * kv] : 0, np = a.info ? a.info[2 * kv + 1] : 0;
  const int n = np + a.nsplit;
  const int64_t col_pre = bi * a.G + gi;
  const int64_t col_row = (((b * a.Hkv + kv) * a.Q + i) * a.G + gi) * a.nsplit;
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
  float m = -INFINITY, l = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int t0 = grp; t0 < n; t0 += kGroups * kBatch) {
    f32x4 ov[kBatch];
    float2 ml[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int t = min(t0 + k * kGroups, n - 1);
      const bool pre = t < np;
      const int64_t at = pre ? (int64_t)(p0 + t) * a.M + col_pre : col_row + (t - np);
      ov[k] = *reinterpret_cast<const f32x4*>((pre ? a.pre_o : a.row_o) + at * kPartO + 4 * lane);
      ml[k] = *reinterpret_cast<const float2*>((pre ? a.pre_ml : a.row_ml) + at * 2);
    }
    float mn = m;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (t0 + k * kGroups >= n) ml[k].x = -INFINITY;
      mn = fmaxf(mn, ml[k].x);
    }
    if (mn == -INFINITY) continue;
    const float f = state_weight(m, mn);
    l *= f;
    acc *= f;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (ml[k].x == -INFINITY) continue;  // a partial without tokens: its channels add nothing
      const float e = fast_exp2(ml[k].x - mn);
      l = fmaf(ml[k].y, e, l);
      acc += ov[k] * e;
    }
    m = mn;
  }
  if (lane == 0) s_m[grp] = m, s_l[grp] = l;
  s_o[grp][lane] = acc;
  __syncthreads();
  if (grp != 0) return;
  float M = s_m[0], L = 0.f;
#pragma unroll
  for (int g = 1; g < kGroups; ++g) M = fmaxf(M, s_m[g]);
  f32x4 r = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const float e = state_weight(s_m[g], M);
    L = fmaf(s_l[g], e, L);
    r += s_o[g][lane] * e;
  }
  const float inv = M == -INFINITY ? 0.f : 1.f / L;  // no token at all: zeros
  T* op = reinterpret_cast<T*>(a.out) + b * a.o_s[0] + (int64_t)hq * a.o_s[1] + (int64_t)i * a.o_s[2] + 4 * lane;
#pragma unroll
  for (int e = 0; e < 4; ++e) op[e] = Elem<T>::from_f32(M == -INFINITY ? 0.f : r[e] * inv);
}

template <typename T>
int launch_rows_t(const RowsArgs& a, hipStream_t s) {
  const int64_t grid = (int64_t)a.rows * a.ncb * a.nsplit;
  if (grid > 0x7fffffffLL) return set_error(HC_ERR_INVALID, "row attention: %lld workgroups", (long long)grid);
  if (a.idx)
    hipLaunchKernelGGL((rows_attn_kernel<T, true>), dim3((unsigned)grid), dim3(kRowsWaves * 64), 0, s, a);
  else
    hipLaunchKernelGGL((rows_attn_kernel<T, false>), dim3((unsigned)grid), dim3(kRowsWaves * 64), 0, s, a);
  return check_launch("row attention");
}

}  // namespace

int device_cus() {
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus < 1) {
    (void)hipGetLastError();
    return 256;
  }
  return cus;
}

RowsPlan rows_plan(int rows, int G, int Q, int64_t max_tiles) {
  RowsPlan p;
  p.qpb = std::max(1, std::min(Q, 16 / G));
  p.ncb = (Q + p.qpb - 1) / p.qpb;
  // Two workgroups a CU; a split keeps a tile for each of its waves.
  const int64_t jobs = std::max<int64_t>((int64_t)rows * p.ncb, 1);
  const int64_t want = (2 * device_cus() + jobs - 1) / jobs;
  const int64_t most = std::max<int64_t>((max_tiles + kRowsWaves - 1) / kRowsWaves, 1);
  p.nsplit = (int)std::min<int64_t>(std::min(want, most), 1024);
  return p;
}

int launch_rows_attn(int dtype, const RowsArgs& a, hipStream_t s) {
  switch (dtype) {
    case HC_DTYPE_BF16: return launch_rows_t<__bf16>(a, s);
    case HC_DTYPE_F16: return launch_rows_t<_Float16>(a, s);
    default: return launch_rows_t<float>(a, s);
  }
}

int launch_merge(int dtype, const MergeArgs& a, int64_t columns, hipStream_t s) {
  if (columns > 0x7fffffffLL) return set_error(HC_ERR_INVALID, "attention merge: %lld rows", (long long)columns);
  const dim3 grid((unsigned)columns), block(kMergeThreads);
  switch (dtype) {
    case HC_DTYPE_BF16: hipLaunchKernelGGL(merge_kernel<__bf16>, grid, block, 0, s, a); break;
    case HC_DTYPE_F16: hipLaunchKernelGGL(merge_kernel<_Float16>, grid, block, 0, s, a); break;
    default: hipLaunchKernelGGL(merge_kernel<float>, grid, block, 0, s, a); break;
  }
  return check_launch("attention merge");
}

}  // namespace hc
