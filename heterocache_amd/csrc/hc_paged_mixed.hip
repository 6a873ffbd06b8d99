// Attention of a padded batch that brings single tokens and chunks at once, as a
// server mixes decode steps with prompts.  Where there is little to do for the
// chunks, one launch, whose workgroups attend the rows of few columns
// (hc_paged_rows.h), those of many (hc_paged_chunk.h) and store the latter's new
// tokens, which nothing in the launch reads from the pages; in its grid a chunk
// workgroup a CU comes first, then the rows', then the other chunks' (kinds in
// turn would meet on some of the XCDs and engines, to which workgroups are dealt
// in turn as well).  Otherwise a launch each: the one kernel's registers and LDS
// leave the chunks fewer waves (4 ragged sequences of up to 509 tokens: 201
// against 165 us; 5 sequences of up to 18 tokens behind 889: 36 against 50).
// Then one launch that folds both.
#include <algorithm>
#include <mutex>

#include "hc_paged_chunk.h"
#include "hc_paged_rows.h"

namespace hc {
namespace {

template <typename T>
constexpr int mixed_lds() {
  return rows_lds<T>() > chunk_lds<T>() ? rows_lds<T>() : chunk_lds<T>();
}

template <typename T, bool WEIGH, bool UNIFORM>
__global__ __launch_bounds__(kPagedThreads, sizeof(T) == 4 ? 1 : 2) void paged_mixed_kernel(const PagedAttn a, int cus, int append_blocks) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int x = blockIdx.x, first = min(cus, a.chunk_grid);
  if (x >= first && x < first + a.grid)
    paged_rows_job<T, WEIGH, UNIFORM>(a, x - first, lds);
  else if (x < a.grid + a.chunk_grid)
    paged_chunk_job<T, UNIFORM, true>(a, x < first ? x : x - a.grid, lds);
  else
    paged_append_job<true>(a, x - a.grid - a.chunk_grid, Tile<T>::kChunks, append_blocks);
}

template <typename T, bool WEIGH>
__global__ __launch_bounds__(256) void paged_mixed_fold_kernel(const PagedAttn a, int runs, int few, int many, uint32_t group0) {
  const int x = group0 + blockIdx.x;
  if (x < few)
    paged_fold_job<T, WEIGH>(a, x, runs);
  else
    paged_chunk_fold_job<T>(a, x - few, many);
}

template <typename T, bool WEIGH, bool UNIFORM>
int launch_attn(const PagedAttn& a, hipStream_t s) {
  static std::once_flag once;
  static hipError_t attr = hipSuccess;
  std::call_once(once, [] {
    attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_mixed_kernel<T, WEIGH, UNIFORM>),
                               hipFuncAttributeMaxDynamicSharedMemorySize, mixed_lds<T>());
  });
  if (attr != hipSuccess) return set_error(HC_ERR_HIP, "hc_paged_attn: %s", hipGetErrorString(attr));
  const int blocks = (a.pool.Q + 15) / 16;
  const int grid = a.grid + a.chunk_grid + (a.pool.fresh ? a.pool.rows * blocks : 0);  // (few: the work is bounded)
  hipLaunchKernelGGL((paged_mixed_kernel<T, WEIGH, UNIFORM>), dim3(grid), dim3(kPagedThreads), mixed_lds<T>(), s, a, device_cus(), blocks);
  return check_launch("hc_paged_attn(mixed)");
}

template <typename T, bool WEIGH>
int launch(int dtype, const PagedAttn& a, hipStream_t s) {
  // The lengths advance in the fold.
  PagedAttn first = a;
  first.len_out = nullptr;
  const Pool& p = a.pool;
  // Iterations of all blocks at most: some eight for each workgroup of a round.
  const int64_t work = (int64_t)p.rows * ((a.cols + kChunkCols - 1) / kChunkCols) * ((p.capacity + 63) / 64);
  int rc;
  if (work <= 8 * (int64_t)a.chunk_slots) {
    rc = uniform_pages(p) ? launch_attn<T, WEIGH, true>(first, s) : launch_attn<T, WEIGH, false>(first, s);
  } else {
    rc = p.fresh ? launch_paged_append(dtype, first, s) : HC_OK;
    if (!rc) rc = launch_paged_rows(dtype, first, false, s);
    if (!rc) rc = launch_paged_chunk(dtype, first, false, s);
  }
  if (rc) return rc;
  const int runs = WEIGH ? paged_weigh_runs(a.pool) : 0, few = a.pool.rows * (a.few + runs);
  const int many = (int)paged_chunk_fold_grid(a);
  return in_launches((int64_t)few + many, 256, [&](dim3 grid, uint32_t group0) {
    hipLaunchKernelGGL((paged_mixed_fold_kernel<T, WEIGH>), grid, dim3(256), 0, s, a, runs, few, many, group0);
    return check_launch("hc_paged_attn(fold)");
  });
}

}  // namespace

int launch_paged_mixed(int dtype, const PagedAttn& a, hipStream_t s) {
  const bool weigh = a.weights_out != nullptr;
  switch (dtype) {
    case HC_DTYPE_BF16: return weigh ? launch<__bf16, true>(dtype, a, s) : launch<__bf16, false>(dtype, a, s);
    case HC_DTYPE_F16: return weigh ? launch<_Float16, true>(dtype, a, s) : launch<_Float16, false>(dtype, a, s);
    default: return weigh ? launch<float, true>(dtype, a, s) : launch<float, false>(dtype, a, s);
  }
}

}  // namespace hc
