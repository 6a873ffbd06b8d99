// Eviction from a paged cache by accumulated weight.
//
// Of a table row's n tokens `keep` stay: the protected ones (the first `sink`
// and the last `recent` positions) before the others, the others by weight, of
// equals the lower slots.  A kept token in a slot below `keep` stays where
// it is; the others fill the freed slots below `keep`, both in ascending order:
// the least that can be moved (a step that drops 64 of 2112 tokens moves at
// most 64, where closing the gaps in order would move all behind the first).
// Every move reads a slot at or behind `keep` and writes one before it, so the
// moves need no order among themselves; the tokens' positions tell their order.
//
// One workgroup finds a row's least kept key by counting: digits of its keys
// (32 bits, order-preserving) into a histogram in LDS, most significant first,
// over the keys that share the digits found so far.  Keys stay in registers
// where a row's fit.  Ties at the threshold go to the lower slots, by a prefix
// count in slot order; the freed slots and the movers are ranked the same way
// and paired by rank.
#include <algorithm>

#include "hc_paged.h"

namespace hc {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kDigit = 8, kBins = 1 << kDigit;

struct EvictArgs {
  Pool pool;
  int rows;  // table rows
  const int32_t* keep;
  int keep_all, sink, recent;
  const float* weights;
  float* weights_out;
  int64_t weight_stride;
  const int32_t *pos, *dropped;
  int32_t *pos_out, *dropped_out, *len_out;
  int64_t pos_stride;
  int32_t *moves, *move_count;  // [row][capacity]: freed slots from the front, movers from the back
  int esz, move_blocks;
};

struct Found {
  uint32_t key;  // the least kept key
  int equal;     // how many of the keys equal to it are kept
};

__device__ __forceinline__ int block_scan(int v, int* s_wave, int tid) {
  // Inclusive sum over the workgroup; every thread also knows the total as s_wave[kWaves].
  const int lane = tid & 63, wave = tid >> 6;
  const int incl = wave_scan_add(v);
  if (lane == 63) s_wave[wave] = incl;
  __syncthreads();
  if (tid < 64) {
    const int w = tid < kWaves ? s_wave[tid] : 0;
    const int x = wave_scan_add(w);
    if (tid < kWaves) s_wave[tid] = x - w;
    if (tid == kWaves - 1) s_wave[kWaves] = x;
  }
  __syncthreads();
  return incl + s_wave[wave];
}

// Key of a token: ranks by weight, NaN below all, protected tokens above.
__device__ __forceinline__ uint32_t token_key(const EvictArgs& a, int row, int t, int first_recent) {
  const int heads = a.pool.heads;
  const float* w = a.weights + (int64_t)row * heads * a.weight_stride + t;
  float x;
  if (heads == 1) {
    x = *w;
  } else {
    double sum = 0.0;  // 64 bits: no order of the heads changes the rounded sum
    for (int h = 0; h < heads; ++h) sum += (double)w[h * a.weight_stride];
    x = (float)sum;
  }
  const int pos = a.pos[row * a.pos_stride + t];
  const uint32_t k = x == x ? min(max(order_key(x), 1u), 0xfffffffeu) : 1u;
  return pos < a.sink || pos >= first_recent ? 0xffffffffu : k;
}

// PER: keys a thread holds (0: read again on every pass).
template <int PER>
__global__ __launch_bounds__(kThreads) void evict_select_kernel(const EvictArgs a) {
  __shared__ int s_hist[kWaves / 4][kBins];
  __shared__ int s_wave[kWaves + 1];
  __shared__ int s_pick[3];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Pool& p = a.pool;
  const int heads = p.heads;
  const int n = min(max(p.row_len[row], 0), p.capacity);
  const int keep = max(a.keep ? a.keep[row] : a.keep_all, 0);
  const int m = min(n, keep);
  const int dropped = a.dropped[row];
  const int first_recent = n + dropped - a.recent;
  const float* const w_in = a.weights + (int64_t)row * heads * a.weight_stride;
  float* const w_out = a.weights_out + (int64_t)row * heads * a.weight_stride;
  const int32_t* const p_in = a.pos + row * a.pos_stride;
  int32_t* const p_out = a.pos_out + row * a.pos_stride;
  const bool copy_w = a.weights_out != a.weights, copy_p = a.pos_out != a.pos;
  int32_t* const list = a.moves + (int64_t)row * p.capacity;

  int moved = 0;
  if (n > keep) {
    uint32_t keys[PER > 0 ? PER : 1];
    if constexpr (PER > 0) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int t = i * kThreads + tid;
        keys[i] = t < n ? token_key(a, row, t, first_recent) : 0u;  // (no token's key is 0)
      }
    }
    auto each = [&](auto f) {
      if constexpr (PER > 0) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (i * kThreads < n) f(i * kThreads + tid, keys[i]);
      } else {
        for (int t0 = 0; t0 < n; t0 += kThreads) {
          const int t = t0 + tid;
          f(t, t < n ? token_key(a, row, t, first_recent) : 0u);
        }
      }
    };
    // The least kept key: the keep-th greatest.
    uint32_t prefix = 0, mask = 0;
    int want = keep;
    if (keep > 0) {
      for (int shift = 32 - kDigit; shift >= 0; shift -= kDigit) {
        for (int i = tid; i < (kWaves / 4) * kBins; i += kThreads) (&s_hist[0][0])[i] = 0;
        __syncthreads();
        each([&](int t, uint32_t k) {
          if (t < n && (k & mask) == prefix) atomicAdd(&s_hist[wave >> 2][k >> shift & (kBins - 1)], 1);
        });
        __syncthreads();
        // Thread b of the first 256: the keys of digit 255 - b, counted from the top.
        int count = 0;
        if (tid < kBins) {
#pragma unroll
          for (int c = 0; c < kWaves / 4; ++c) count += s_hist[c][kBins - 1 - tid];
        }
        const int incl = block_scan(tid < kBins ? count : 0, s_wave, tid);
        if (tid < kBins && incl >= want && incl - count < want) {
          s_pick[0] = kBins - 1 - tid;
          s_pick[1] = want - (incl - count);
        }
        __syncthreads();
        prefix |= (uint32_t)s_pick[0] << shift;
        mask |= (uint32_t)(kBins - 1) << shift;
        want = s_pick[1];
      }
    }
    const uint32_t least = keep > 0 ? prefix : 0xffffffffu;
    const int equal = keep > 0 ? want : 0;

    // In slot order, kThreads slots at a time: the equal keys before a slot, then
    // the freed slots (below keep) or the movers (from keep on) before it.
    int eq_before = 0, ev_before = 0;
    auto walk = [&](int t, uint32_t k) {
      const bool live = t < n;
      const bool eq = live && k == least;
      const uint64_t eqs = __ballot(eq);
      const int below = __popcll(eqs & ((1ull << lane) - 1));
      if (lane == 0) s_hist[0][wave] = __popcll(eqs);
      __syncthreads();
      int rank = eq_before + below, all = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const int c = s_hist[0][w];
        rank += w < wave ? c : 0;
        all += c;
      }
      eq_before += all;
      const bool kept = live && (k > least || (eq && rank < equal));
      const bool event = live && (t < keep ? !kept : kept);
      const uint64_t evs = __ballot(event);
      if (lane == 0) s_hist[1][wave] = __popcll(evs);
      __syncthreads();
      int at = ev_before + __popcll(evs & ((1ull << lane) - 1)), sum = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const int c = s_hist[1][w];
        at += w < wave ? c : 0;
        sum += c;
      }
      ev_before += sum;
      // Freed slots take the list from the front; the movers follow them.
      if (event) list[at] = t;
      if (kept && t < keep) {
        if (copy_w)
          for (int h = 0; h < heads; ++h) w_out[h * a.weight_stride + t] = w_in[h * a.weight_stride + t];
        if (copy_p) p_out[t] = p_in[t];
      }
      __syncthreads();
    };
    each(walk);
    moved = ev_before / 2;  // as many movers as freed slots
    __syncthreads();        // the list is whole
    for (int i = tid; i < moved; i += kThreads) {
      const int to = list[i], of = list[moved + i];
      for (int h = 0; h < heads; ++h) w_out[h * a.weight_stride + to] = w_in[h * a.weight_stride + of];
      p_out[to] = p_in[of];
    }
  } else {
    for (int t = tid; t < n; t += kThreads) {
      if (copy_w)
        for (int h = 0; h < heads; ++h) w_out[h * a.weight_stride + t] = w_in[h * a.weight_stride + t];
      if (copy_p) p_out[t] = p_in[t];
    }
  }
  if (tid == 0) {
    a.move_count[row] = moved;
    a.len_out[row] = m;
    a.dropped_out[row] = dropped + n - m;
  }
}

// The moves of all rows: 16 bytes a thread, a token's keys and values of one
// head by neighbouring threads.  Both pages of a move lie in the pool, or the
// token stays where it is and the status word says so.
__global__ __launch_bounds__(256) void evict_move_kernel(const EvictArgs a) {
  const Pool& p = a.pool;
  const int row = blockIdx.x / a.move_blocks, blk = blockIdx.x % a.move_blocks;
  const int count = a.move_count[row];
  const int chunks = HC_HEAD_DIM * a.esz / 16;  // of a token and head
  const int32_t* const list = a.moves + (int64_t)row * p.capacity;
  const int32_t* const tab = p.table + row * p.table_stride;
  const int64_t units = (int64_t)count * p.heads * chunks;
  for (int64_t u = blk * 256 + threadIdx.x; u < units; u += (int64_t)a.move_blocks * 256) {
    const int c = (int)(u % chunks), h = (int)(u / chunks % p.heads), i = (int)(u / chunks / p.heads);
    const int to = list[i], of = list[count + i];
    const int tp = page_of(p, to), op = page_of(p, of);
    const int tg = tab[tp], og = tab[op];
    if ((uint32_t)tg >= (uint32_t)p.pages || (uint32_t)og >= (uint32_t)p.pages) {
      if (p.status) atomicOr(p.status, kStatusPage);
      continue;
    }
    const int ta = to - tp * p.page_tokens, oa = of - op * p.page_tokens;
    const u32x4 k = *reinterpret_cast<const u32x4*>(p.k + og * p.k_page + oa * p.k_tok + h * p.k_head + 16 * c);
    const u32x4 v = *reinterpret_cast<const u32x4*>(p.v + og * p.v_page + oa * p.v_tok + h * p.v_head + 16 * c);
    *reinterpret_cast<u32x4*>(const_cast<char*>(p.k) + tg * p.k_page + ta * p.k_tok + h * p.k_head + 16 * c) = k;
    *reinterpret_cast<u32x4*>(const_cast<char*>(p.v) + tg * p.v_page + ta * p.v_tok + h * p.v_head + 16 * c) = v;
  }
}

}  // namespace

int fill_pool(const char* name, const hc_paged_cache* c, Pool& p, int Q, const int32_t* counts);

}  // namespace hc

using namespace hc;

extern "C" size_t hc_paged_evict_scratch_size(const hc_paged_cache* c) {
  if (!c || c->batch <= 0 || c->kv_heads <= 0 || (c->heads != 1 && c->heads != c->kv_heads) || c->table_pages <= 0 ||
      c->page_tokens <= 0)
    return 0;
  const size_t rows = (size_t)c->batch * c->kv_heads / c->heads;
  return (rows + rows * c->table_pages * c->page_tokens) * 4;
}

extern "C" int hc_paged_evict(const hc_paged_cache* c, const int32_t* keep, int keep_all, int sink, int recent,
                              int32_t* len_out, float* weights_out, int32_t* pos_out, int32_t* dropped_out, void* scratch,
                              size_t scratch_bytes, void* stream) {
  clear_error();
  EvictArgs a;
  if (int rc = fill_pool("hc_paged_evict", c, a.pool, 0, nullptr)) return rc;
  if (keep_all < 0 || sink < 0 || recent < 0)
    return set_error(HC_ERR_INVALID, "hc_paged_evict: keep=%d sink=%d recent=%d", keep_all, sink, recent);
  if (!keep && (int64_t)sink + recent > keep_all)
    return set_error(HC_ERR_INVALID, "hc_paged_evict: sink=%d and recent=%d exceed keep=%d", sink, recent, keep_all);
  if (c->batch == 0) return HC_OK;
  if (!c->weights || !c->pos || !c->dropped)
    return set_error(HC_ERR_INVALID, "hc_paged_evict: the cache has no weights, positions and dropped counts");
  if (scratch_bytes < hc_paged_evict_scratch_size(c) || !scratch || (reinterpret_cast<uintptr_t>(scratch) & 15))
    return set_error(HC_ERR_INVALID, "hc_paged_evict: scratch too small or unaligned (%zu < %zu bytes)", scratch_bytes,
                     hc_paged_evict_scratch_size(c));
  a.rows = a.pool.rows / a.pool.heads;
  a.keep = keep, a.keep_all = keep_all, a.sink = sink, a.recent = recent;
  a.weights = c->weights, a.weight_stride = c->weight_stride;
  a.weights_out = weights_out ? weights_out : c->weights;
  a.pos = c->pos, a.pos_stride = c->pos_stride, a.pos_out = pos_out ? pos_out : c->pos;
  a.dropped = c->dropped, a.dropped_out = dropped_out ? dropped_out : c->dropped;
  a.len_out = len_out ? len_out : c->row_len;
  a.move_count = reinterpret_cast<int32_t*>(scratch);
  a.moves = a.move_count + a.rows;
  a.esz = c->dtype == HC_DTYPE_F32 ? 4 : 2;
  // Workgroups of 256 chunks for the most that a row can move, at most some
  // eight a CU over all rows.
  const int64_t most = (int64_t)(a.pool.capacity / 2) * a.pool.heads * (HC_HEAD_DIM * a.esz / 16);
  a.move_blocks = (int)std::max<int64_t>(1, std::min<int64_t>((most + 255) / 256, 2048 / a.rows));
  hipStream_t s = (hipStream_t)stream;
  const int cap = a.pool.capacity;
  if (cap <= 4 * kThreads)
    hipLaunchKernelGGL((evict_select_kernel<4>), dim3(a.rows), dim3(kThreads), 0, s, a);
  else if (cap <= 16 * kThreads)
    hipLaunchKernelGGL((evict_select_kernel<16>), dim3(a.rows), dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL((evict_select_kernel<0>), dim3(a.rows), dim3(kThreads), 0, s, a);
  if (int rc = check_launch("hc_paged_evict")) return rc;
  hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)((int64_t)a.rows * a.move_blocks)), dim3(256), 0, s, a);
  return check_launch("hc_paged_evict(move)");
}
