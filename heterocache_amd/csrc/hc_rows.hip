// Attention over the rows of the ragged store for a few queries a row, and
// the fold of partial results (see hc_rows.h).
#include <algorithm>
#include <atomic>

#include "hc_rows.h"

namespace hc {
namespace {

template <typename T, int NW>
__global__ __launch_bounds__(NW * 64, NW == 8 ? 1 : sizeof(T) == 4 ? 2 : 3) void block_rows_kernel(const RowsArgs a) {
  __shared__ __attribute__((aligned(16))) float lds[kRowsLds];
  rows_job<T, kRowsList, false, NW>(a, blockIdx.x, lds);
}

template <typename T>
void launch_block_rows_t(const RowsArgs& a, int waves, unsigned n, hipStream_t s) {
  if (waves == 8)
    hipLaunchKernelGGL((block_rows_kernel<T, 8>), dim3(n), dim3(512), 0, s, a);
  else
    hipLaunchKernelGGL((block_rows_kernel<T, 4>), dim3(n), dim3(256), 0, s, a);
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
      if (t0 + k * kGroups >= n) ml[k] = make_float2(-INFINITY, 0.f);
      mn = fmaxf(mn, ml[k].x);
    }
    const float f = state_weight(m, mn);
    l *= f;
    acc *= f;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const float e = state_weight(ml[k].x, mn);
      l = fmaf(ml[k].y, e, l);
      if (ml[k].x == -INFINITY) continue;  // no number among its scores: its channels add nothing
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
  T* op = reinterpret_cast<T*>(a.out) + b * a.o_s[0] + (int64_t)hq * a.o_s[1] + (int64_t)i * a.o_s[2] + 4 * lane;
#pragma unroll
  for (int e = 0; e < 4; ++e) op[e] = Elem<T>::from_f32(state_output(r[e], M, L));
}

}  // namespace

int device_cus() {
  // Asked for once a device: the plans of a call read it some twenty times.
  static std::atomic<int> known[64];
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) {
    (void)hipGetLastError();
    return 256;
  }
  cus = known[dev].load(std::memory_order_relaxed);
  if (cus > 0) return cus;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus < 1) {
    (void)hipGetLastError();
    return 256;
  }
  known[dev].store(cus, std::memory_order_relaxed);
  return cus;
}

RowsPlan rows_plan(int rows, int G, int Q, int64_t max_tiles) {
  RowsPlan p;
  p.qpb = std::max(1, std::min(Q, 16 / G));
  p.ncb = (Q + p.qpb - 1) / p.qpb;
  // Two workgroups a CU; a split keeps a tile for each of its four waves.
  const int64_t jobs = std::max<int64_t>((int64_t)rows * p.ncb, 1);
  const int64_t want = (2 * device_cus() + jobs - 1) / jobs;
  const int64_t most = std::max<int64_t>((max_tiles + 3) / 4, 1);
  p.nsplit = (int)std::min<int64_t>(std::min(want, most), 1024);
  return p;
}

int launch_block_rows(int dtype, const RowsArgs& a, int waves, hipStream_t s) {
  const int64_t n = rows_workgroups(a);
  if (n > 0x7fffffffLL) return set_error(HC_ERR_INVALID, "block attention: %lld workgroups", (long long)n);
  switch (dtype) {
    case HC_DTYPE_BF16: launch_block_rows_t<__bf16>(a, waves, (unsigned)n, s); break;
    case HC_DTYPE_F16: launch_block_rows_t<_Float16>(a, waves, (unsigned)n, s); break;
    default: launch_block_rows_t<float>(a, waves, (unsigned)n, s); break;
  }
  return check_launch("block attention");
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
