// Attention of few queries over a paged cache: kernels and launches (hc_paged_rows.h).
#include <algorithm>
#include <mutex>

#include "hc_paged_rows.h"

namespace hc {
namespace {

template <typename T, bool WEIGH, bool UNIFORM>
__global__ __launch_bounds__(kPagedThreads, sizeof(T) == 4 ? 1 : 2) void paged_rows_kernel(const PagedAttn a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  paged_rows_job<T, WEIGH, UNIFORM>(a, blockIdx.x, lds);
}

template <typename T, bool WEIGH>
__global__ __launch_bounds__(256) void paged_fold_kernel(const PagedAttn a, int runs, uint32_t group0) {
  paged_fold_job<T, WEIGH>(a, group0 + blockIdx.x, runs);
}

template <typename T, bool WEIGH, bool UNIFORM>
int launch_attn(const PagedAttn& a, hipStream_t s) {
  static std::once_flag once;
  static hipError_t attr = hipSuccess;
  std::call_once(once, [] {
    attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_rows_kernel<T, WEIGH, UNIFORM>),
                               hipFuncAttributeMaxDynamicSharedMemorySize, rows_lds<T>());
  });
  if (attr != hipSuccess) return set_error(HC_ERR_HIP, "hc_paged_attn: %s", hipGetErrorString(attr));
  hipLaunchKernelGGL((paged_rows_kernel<T, WEIGH, UNIFORM>), dim3(a.grid), dim3(kPagedThreads), rows_lds<T>(), s, a);
  return check_launch("hc_paged_attn(rows)");
}

template <typename T, bool WEIGH>
int launch(const PagedAttn& a, bool fold, hipStream_t s) {
  if (int rc = uniform_pages(a.pool) ? launch_attn<T, WEIGH, true>(a, s) : launch_attn<T, WEIGH, false>(a, s)) return rc;
  if (!fold) return HC_OK;
  const int runs = WEIGH ? paged_weigh_runs(a.pool) : 0;
  return in_launches(a.pool.rows * (a.few + runs), 256, [&](dim3 grid, uint32_t group0) {
    hipLaunchKernelGGL((paged_fold_kernel<T, WEIGH>), grid, dim3(256), 0, s, a, runs, group0);
    return check_launch("hc_paged_attn(fold)");
  });
}

template <typename T>
int launch(const PagedAttn& a, bool fold, hipStream_t s) {
  return a.weights_out ? launch<T, true>(a, fold, s) : launch<T, false>(a, fold, s);
}

}  // namespace

int launch_paged_rows(int dtype, const PagedAttn& a, bool fold, hipStream_t s) {
  switch (dtype) {
    case HC_DTYPE_BF16: return launch<__bf16>(a, fold, s);
    case HC_DTYPE_F16: return launch<_Float16>(a, fold, s);
    default: return launch<float>(a, fold, s);
  }
}

}  // namespace hc
