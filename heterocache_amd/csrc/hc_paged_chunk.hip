// Attention of a chunk of new tokens over a paged cache: kernels and launches
// (hc_paged_chunk.h), and the weights that the chunk gives every token.
#include <algorithm>
#include <mutex>

#include "hc_paged_chunk.h"

namespace hc {
namespace {

template <typename T, bool UNIFORM>
__global__ __launch_bounds__(kPagedThreads, sizeof(T) == 4 ? 2 : 3) void paged_chunk_kernel(const PagedAttn a, uint32_t group0) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  paged_chunk_job<T, UNIFORM, false>(a, group0 + blockIdx.x, lds);
}

template <typename T>
__global__ __launch_bounds__(256) void paged_chunk_fold_kernel(const PagedAttn a) {
  paged_chunk_fold_job<T>(a, blockIdx.x, gridDim.x);
}

__global__ __launch_bounds__(256) void paged_append_kernel(const PagedAttn a, int chunks, int blocks, uint32_t group0) {
  paged_append_job<false>(a, group0 + blockIdx.x, chunks, blocks);
}

// Every token's share of the chunk's attention,
//
//   weights_out[t] = weights[t] + sum_c exp2(s_ct - M_c) / L_c,
//
// from the columns' folded (M, L): the scores are formed again, tokens as the
// columns of the matrix product (their operands stay in registers), queries
// streamed through LDS 64 at a time, so a token's sum stays in its lane and no
// atomics are needed.  Per score one matrix element, a fused multiply-add, an
// exponential and an addition: bound by the vector units (4 sequences of up to 509
// tokens over 8003, 216 M scores of 4 heads: 85 us, 44 of them vector work).
template <typename T>
constexpr int weigh_lds() {
  return 2 * (64 * Tile<T>::kRow + 1024);
}

template <typename T, int NC>
__global__ __launch_bounds__(kPagedThreads, sizeof(T) == 4 ? 2 : NC == 4 ? 3 : 4) void paged_weigh_kernel(const PagedAttn a, int blocks, uint32_t group0) {
  typedef typename Elem<T>::vec8 vec8;
  typedef Tile<T> Tl;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const Pool& p = a.pool;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g4 = lane >> 4, n16 = lane & 15;
  // Rows r, r + 8, .. on one XCD, the blocks of a row behind each other: workgroups
  // are dealt in turn to the XCDs and within one to its four engines, where rows
  // of a sequence each would all meet (4 ragged sequences: 162 us, now 85).
  const uint32_t x = group0 + blockIdx.x;
  const int row = x % 8 + 8 * (x / 8 / blocks), tb = x / 8 % blocks;
  if (row >= p.rows) return;
  const int b = row / p.Hkv, h = row % p.Hkv;
  const int hd = p.heads == 1 ? 0 : h;
  // (Scalar, as what follows from them.)
  const int info = __builtin_amdgcn_readfirstlane(a.plan[row].z), nq = __builtin_amdgcn_readfirstlane(query_tokens(p.counts, b, p.Q));
  const bool room = info >= 0;
  const int total = room ? info : -1 - info, ncols = room ? nq * a.G : 0, base = total - nq;
  const int old = p.fresh && room ? base : total;
  if (a.few > 0 && nq * a.G <= kFewCols) return;  // (paged_fold_kernel's)
  const int t_block = tb * kPagedWaves * 16 * NC;
  if (t_block >= total) return;
  const int t_wave = t_block + wave * 16 * NC;
  const int32_t* const tab = p.table + table_row(p, row) * p.table_stride;

  // Key operands: token t_wave + 16 c + n16 (those behind the last repeat it and
  // are not stored), channels as the queries'.
  vec8 kop[NC][4];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int t = min(t_wave + 16 * c + n16, total - 1);
    const int pi = page_of(p, t);
    int pg = tab[pi];
    if ((uint32_t)pg >= (uint32_t)p.pages) pg = 0;  // (the columns' sums are NaN)
    const T* kp = reinterpret_cast<const T*>(p.k + hd * p.k_head + pg * p.k_page + (t - pi * p.page_tokens) * p.k_tok);
#pragma unroll
    for (int s = 0; s < 4; ++s) kop[c][s] = chunk_query<T>(kp, g4, s);
  }

  // Columns of the chunk, 64 an iteration, from the first that sees a token of
  // the workgroup on, in LDS as chunk_keys reads them.  Columns behind the last
  // repeat it, and no token is taken as seen by them.
  constexpr int kSet = 64 * Tl::kRow + 1024, kMine = kSegs<T> / kPagedWaves;
  const int c0 = max(t_block - base, 0) * a.G / 64 * 64;
  const uint32_t q_off = 64 * wave + 16 * g4;
  auto stage = [&](int set, int col) {
    char* s = lds + set * kSet;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int c = min(col + 16 * r + n16, ncols - 1);
      const int i = over_group(a, c), gi = c - i * a.G;
      const char* src = reinterpret_cast<const char*>(reinterpret_cast<const T*>(a.q) + b * a.q_s[0] +
                                                      (int64_t)(h * a.G + gi) * a.q_s[1] + i * a.q_s[2]);
#pragma unroll
      for (int j = 0; j < kMine; ++j) lds_dma16(src + (q_off + 256 * j), s + (r * kSegs<T> + wave + kPagedWaves * j) * kBlock);
    }
    // Their states, and those of as many behind, which nothing reads.
    if (wave == 0)
      lds_dma16(reinterpret_cast<const char*>(a.ml + ((int64_t)row * a.ml_stride + col) * 2) + 16 * lane, s + 64 * Tl::kRow);
  };
  float sum[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) sum[c] = 0.f;
  if (c0 < ncols) stage(0, c0);
  for (int col = c0, it = 0; col < ncols; col += 64, ++it) {
    wait_lds_dma();
    __syncthreads();
    if (col + 64 < ncols) stage((it + 1) & 1, col + 64);
    const char* s = lds + (it & 1) * kSet;
    const float* const ml = reinterpret_cast<const float*>(s + 64 * Tl::kRow);
    auto add = [&](auto edge_tag) {
      constexpr bool EDGE = decltype(edge_tag)::value;
      float part[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) part[c] = 0.f;
#pragma unroll
      for (int qb = 0; qb < 4; ++qb) {
        f32x4 acc[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const vec8 qa = chunk_keys<T>(s, lane, qb, x);
#pragma unroll
          for (int c = 0; c < NC; ++c) acc[c] = mma_16x16x32(qa, kop[c][x], acc[c]);
        }
        const f32x4 lo = *reinterpret_cast<const f32x4*>(ml + 2 * (16 * qb + 4 * g4));
        const f32x4 hi = *reinterpret_cast<const f32x4*>(ml + 2 * (16 * qb + 4 * g4) + 4);
        const float top[4] = {lo[0], lo[2], hi[0], hi[2]}, inv[4] = {lo[1], lo[3], hi[1], hi[3]};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int u = col + 16 * qb + 4 * g4 + r;
          const int lim = !EDGE ? 0 : u < ncols ? base + over_group(a, u) + 1 : 0;
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const float e = fast_exp2(fmaf(acc[c][r], a.scale_log2, -top[r])), more = fmaf(e, inv[r], part[c]);
            part[c] = !EDGE || t_wave + 16 * c + n16 < lim ? more : part[c];
          }
        }
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) sum[c] += part[c];
    };
    // Some of these columns may not see some of the wave's tokens.
    if (t_wave + 16 * NC > base + over_group(a, col) + 1 || col + 64 > ncols)
      add(std::true_type{});
    else
      add(std::false_type{});
  }
  const float* const in = a.weights + row * a.weight_stride;
  float* const outw = a.weights_out + row * a.weight_stride;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const float w = rows4_sum(sum[c]);
    const int t = t_wave + 16 * c + n16;
    if (g4 == 0 && t < total) outw[t] = t < old ? in[t] + w : w;
  }
}

template <typename T, bool UNIFORM>
int launch_attn(const PagedAttn& a, hipStream_t s) {
  static std::once_flag once;
  static hipError_t attr = hipSuccess;
  std::call_once(once, [] {
    attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_chunk_kernel<T, UNIFORM>),
                               hipFuncAttributeMaxDynamicSharedMemorySize, chunk_lds<T>());
  });
  if (attr != hipSuccess) return set_error(HC_ERR_HIP, "hc_paged_attn: %s", hipGetErrorString(attr));
  return in_launches(a.chunk_grid, kPagedThreads, [&](dim3 grid, uint32_t group0) {
    hipLaunchKernelGGL((paged_chunk_kernel<T, UNIFORM>), grid, dim3(kPagedThreads), chunk_lds<T>(), s, a, group0);
    return check_launch("hc_paged_attn(chunk)");
  });
}

template <typename T, int NC>
int launch_weigh(const PagedAttn& a, hipStream_t s) {
  static std::once_flag once;
  static hipError_t attr = hipSuccess;
  std::call_once(once, [] {
    attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_weigh_kernel<T, NC>),
                               hipFuncAttributeMaxDynamicSharedMemorySize, weigh_lds<T>());
  });
  if (attr != hipSuccess) return set_error(HC_ERR_HIP, "hc_paged_attn: %s", hipGetErrorString(attr));
  const int block = kPagedWaves * 16 * NC;
  const int blocks = (a.pool.capacity + block - 1) / block;
  return in_launches((int64_t)(a.pool.rows + 7) / 8 * 8 * blocks, kPagedThreads, [&](dim3 grid, uint32_t group0) {
    hipLaunchKernelGGL((paged_weigh_kernel<T, NC>), grid, dim3(kPagedThreads), weigh_lds<T>(), s, a, blocks, group0);
    return check_launch("hc_paged_attn(weights)");
  });
}

template <typename T>
int launch(const PagedAttn& a, bool fold, hipStream_t s) {
  if (int rc = uniform_pages(a.pool) ? launch_attn<T, true>(a, s) : launch_attn<T, false>(a, s)) return rc;
  if (!fold) return HC_OK;
  hipLaunchKernelGGL((paged_chunk_fold_kernel<T>), dim3(paged_chunk_fold_grid(a)), dim3(256), 0, s, a);
  return check_launch("hc_paged_attn(fold)");
}

template <typename T>
int launch_weights(const PagedAttn& a, hipStream_t s) {
  // More tokens a wave take fewer reads of the queries, once there are workgroups enough.
  const int64_t wide = (int64_t)a.pool.rows * ((a.pool.capacity + 255) / 256);
  if (sizeof(T) == 2 && wide >= 2048) return launch_weigh<T, 4>(a, s);
  if (sizeof(T) == 2 && wide >= 256) return launch_weigh<T, 2>(a, s);
  return launch_weigh<T, 1>(a, s);
}

// Lengths advanced in place, once an append without attention has read them.
__global__ __launch_bounds__(256) void paged_advance_kernel(const PagedAttn a, int table_rows) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r >= table_rows) return;
  const RowSpan s = row_span(a.pool, a.pool.heads == 1 ? r : r * a.pool.Hkv);
  a.len_out[r] = s.total;
}

// The weights of a call without queries, in memory of their own.
__global__ __launch_bounds__(256) void paged_carry_kernel(const PagedAttn a, int runs, uint32_t group0) {
  const int x = group0 + blockIdx.x, row = x % a.pool.rows, total = row_span(a.pool, row).total;
  const float* const in = a.weights + row * a.weight_stride;
  float* const out = a.weights_out + row * a.weight_stride;
  for (int t = x / a.pool.rows * 256 + (int)threadIdx.x; t < total; t += runs * 256) out[t] = in[t];
}

}  // namespace

int launch_paged_chunk(int dtype, const PagedAttn& a, bool fold, hipStream_t s) {
  switch (dtype) {
    case HC_DTYPE_BF16: return launch<__bf16>(a, fold, s);
    case HC_DTYPE_F16: return launch<_Float16>(a, fold, s);
    default: return launch<float>(a, fold, s);
  }
}

int launch_paged_weights(int dtype, const PagedAttn& a, hipStream_t s) {
  switch (dtype) {
    case HC_DTYPE_BF16: return launch_weights<__bf16>(a, s);
    case HC_DTYPE_F16: return launch_weights<_Float16>(a, s);
    default: return launch_weights<float>(a, s);
  }
}

int launch_paged_carry(const PagedAttn& a, hipStream_t s) {
  const int runs = paged_weigh_runs(a.pool);
  return in_launches(a.pool.rows * runs, 256, [&](dim3 grid, uint32_t group0) {
    hipLaunchKernelGGL(paged_carry_kernel, grid, dim3(256), 0, s, a, runs, group0);
    return check_launch("hc_paged_attn(weights)");
  });
}

int launch_paged_append(int dtype, const PagedAttn& a, hipStream_t s) {
  const int chunks = dtype == HC_DTYPE_F32 ? 32 : 16, blocks = std::max(1, (a.pool.Q + 15) / 16);
  PagedAttn store = a;
  const bool in_place = a.len_out && a.len_out == a.pool.row_len;
  if (in_place) store.len_out = nullptr;
  const int rc = in_launches((int64_t)a.pool.rows * blocks, 256, [&](dim3 grid, uint32_t group0) {
    hipLaunchKernelGGL(paged_append_kernel, grid, dim3(256), 0, s, store, chunks, blocks, group0);
    return check_launch("hc_paged_append");
  });
  if (rc || !in_place) return rc;
  const int table_rows = a.pool.heads == 1 ? a.pool.rows : a.pool.rows / a.pool.Hkv;
  hipLaunchKernelGGL(paged_advance_kernel, dim3((table_rows + 255) / 256), dim3(256), 0, s, a, table_rows);
  return check_launch("hc_paged_append(lengths)");
}

}  // namespace hc
