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
// The least kept key of a row is found by counting keys (32 bits,
// order-preserving).  Short rows: one workgroup, the keys in registers, counted
// into equal steps between the least and the greatest left until a step holds
// one value (the top bits alone put most weights into a few counters, whose
// additions run one after another: 8190 tokens 48 us, so 34).  Long rows, of
// which one CU would draw some 33 GB/s: workgroups of 2048 tokens in five
// launches, counters cleared, keys counted by their top 12 bits, those that share
// the threshold's collected, the threshold found among them by every workgroup
// for itself, and the lists written from the workgroups' counts (8 rows of up to
// 131072 tokens: 37 us, one workgroup a row 346).  The candidates grow with what
// shares those bits, and every workgroup counts them all: with the inputs cached
// the whole call takes 60 us on spread weights, 146 where all lie within an eighth
// of a binade and 475 where all are equal, as a stored prompt's are.  Which way a
// row goes is decided by its table's capacity, which the host knows, not by its
// length.  Ties at the threshold go to the lower slots
// by a prefix count in slot order; freed slots and movers are ranked the same way
// and paired by rank.  Moves run at the copy rate: 134 MB in 34 us.
#include <algorithm>

#include "hc_paged.h"

namespace hc {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;

constexpr int kRun = 2048;  // tokens of a workgroup of the launches over long rows
constexpr int kRunThreads = 256;
constexpr int kRunPer = kRun / kRunThreads;
constexpr int kTopBits = 12, kTop = 1 << kTopBits;

// State of a row between the launches.
struct RowState {
  int n, keep, dropped, moved;
  uint32_t least;  // the least kept key
  int equal;       // how many of the keys equal to it are kept
  int pad[2];
};
// Keys above the threshold, and at it, of a run: in slots below keep, and from keep on.
struct RunCount {
  int above, equal, above_behind, equal_behind;
};

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
  int32_t* moves;   // [row][capacity]: freed slots, then the movers
  uint64_t* freed;  // [row][capacity / 64, rounded up]: the slots below keep that are freed, a bit each
  RowState* state;
  int esz, move_blocks;
  // Long rows.
  int runs;
  uint32_t *keys, *candidates;  // [row][capacity]
  int32_t *hist, *found;        // [row][kTop], [row]
  RunCount* counts;             // [row][run]
};

// Inclusive sum over a workgroup of NW waves; s_wave[NW] is the total.
template <int NW>
__device__ __forceinline__ int block_scan(int v, int* s_wave, int tid) {
  const int lane = tid & 63, wave = tid >> 6;
  const int incl = wave_scan_add(v);
  if (lane == 63) s_wave[wave] = incl;
  __syncthreads();
  if (tid < 64) {
    const int w = tid < NW ? s_wave[tid] : 0;
    const int x = wave_scan_add(w);
    if (tid < NW) s_wave[tid] = x - w;
    if (tid == NW - 1) s_wave[NW] = x;
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
    int h = 0;
    for (; h + 4 <= heads; h += 4) {
      float y[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) y[u] = w[(h + u) * a.weight_stride];
#pragma unroll
      for (int u = 0; u < 4; ++u) sum += (double)y[u];
    }
    for (; h < heads; ++h) sum += (double)w[h * a.weight_stride];
    x = (float)sum;
  }
  const int pos = a.pos[row * a.pos_stride + t];
  const uint32_t k = x == x ? min(max(order_key(x), 1u), 0xfffffffeu) : 1u;
  return pos < a.sink || pos >= first_recent ? 0xffffffffu : k;
}

__device__ __forceinline__ RowState row_state(const EvictArgs& a, int row) {
  RowState s;
  s.n = min(max(a.pool.row_len[row], 0), a.pool.capacity);
  s.keep = max(a.keep ? a.keep[row] : a.keep_all, 0);
  s.dropped = a.dropped[row];
  return s;
}

// Keys of rows whose weights are sums over heads, by more workgroups than rows.
__global__ __launch_bounds__(kRunThreads) void evict_keys_kernel(const EvictArgs a, uint32_t group0) {
  const uint32_t x = group0 + blockIdx.x;
  const int row = x % a.rows, t = x / a.rows * kRunThreads + threadIdx.x;
  const RowState s = row_state(a, row);
  if (s.n > s.keep && t < s.n) a.keys[(int64_t)row * a.pool.capacity + t] = token_key(a, row, t, s.n + s.dropped - a.recent);
}

// Short rows: one workgroup a row, PER keys a thread.  READY: evict_keys_kernel has formed them.
template <int PER, bool READY>
__global__ __launch_bounds__(kThreads) void evict_select_kernel(const EvictArgs a, uint32_t group0) {
  __shared__ int s_hist[kBins];
  __shared__ int s_wave[kWaves + 1];
  __shared__ int s_count[PER * kWaves];
  __shared__ uint32_t s_range[2];
  __shared__ int s_pick[2];
  const int row = group0 + blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  RowState st = row_state(a, row);
  const int n = st.n, keep = st.keep;
  int32_t* const list = a.moves + (int64_t)row * a.pool.capacity;
  uint64_t* const freed = a.freed + (int64_t)row * ((a.pool.capacity + 63) / 64);
  st.moved = 0;
  if (n > keep) {
    uint32_t keys[PER];
    uint32_t least = 0xffffffffu, most = 0u;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int t = i * kThreads + tid;
      if constexpr (READY)
        keys[i] = t < n ? a.keys[(int64_t)row * a.pool.capacity + t] : 0u;
      else
        keys[i] = t < n ? token_key(a, row, t, n + st.dropped - a.recent) : 0u;  // (no token's key is 0)
      if (t < n) least = min(least, keys[i]), most = max(most, keys[i]);
    }
    int want = keep;
    uint32_t lo = 0xffffffffu;  // keep = 0: nothing stays
    if (keep > 0) {
      least = wave_fold(least, [](uint32_t x, uint32_t y) { return min(x, y); });
      most = wave_fold(most, [](uint32_t x, uint32_t y) { return max(x, y); });
      if (lane == 0) s_hist[2 * wave] = (int)least, s_hist[2 * wave + 1] = (int)most;
      __syncthreads();
      if (tid == 0) {
        for (int w = 1; w < kWaves; ++w)
          least = min(least, (uint32_t)s_hist[2 * w]), most = max(most, (uint32_t)s_hist[2 * w + 1]);
        s_range[0] = least, s_range[1] = most;
      }
      __syncthreads();
      lo = s_range[0];
      uint32_t span = s_range[1] - lo;  // the keys left lie in [lo, lo + span]
      while (span > 0) {
        const int shift = max(32 - __clz(span) - 11, 0);
        for (int i = tid; i < kBins; i += kThreads) s_hist[i] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (keys[i] >= lo && keys[i] - lo <= span) atomicAdd(&s_hist[(keys[i] - lo) >> shift], 1);
        __syncthreads();
        // Thread b counts from the top: bins 2047 - 2 b and 2046 - 2 b.
        const int c0 = s_hist[kBins - 1 - 2 * tid], c1 = s_hist[kBins - 2 - 2 * tid];
        const int incl = block_scan<kWaves>(c0 + c1, s_wave, tid), excl = incl - c0 - c1;
        if (excl < want && incl >= want) {
          const bool upper = excl + c0 >= want;
          s_pick[0] = kBins - 1 - 2 * tid - (upper ? 0 : 1);
          s_pick[1] = want - excl - (upper ? 0 : c0);
        }
        __syncthreads();
        lo += (uint32_t)s_pick[0] << shift;
        span = min(span - ((uint32_t)s_pick[0] << shift), (1u << shift) - 1u);
        want = s_pick[1];
      }
    } else {
      want = 0;
    }

    // Rank of a flag among the workgroup's in slot order: the waves' counts of
    // every kThreads slots, then their prefix sums.
    uint64_t flags[PER];
    auto rank_all = [&]() {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (lane == 0) s_count[i * kWaves + wave] = __popcll(flags[i]);
      __syncthreads();
      const int c = tid < PER * kWaves ? s_count[tid] : 0;
      const int x = block_scan<kWaves>(c, s_wave, tid);
      if (tid < PER * kWaves) s_count[tid] = x - c;
      __syncthreads();
      return s_wave[kWaves];
    };
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll
    for (int i = 0; i < PER; ++i) flags[i] = __ballot(i * kThreads + tid < n && keys[i] == lo);
    rank_all();
    uint32_t kept = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int t = i * kThreads + tid;
      const int rank = s_count[i * kWaves + wave] + __popcll(flags[i] & below);
      if (t < n && (keys[i] > lo || (keys[i] == lo && rank < want))) kept |= 1u << i;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int t = i * kThreads + tid;
      flags[i] = __ballot(t < n && (t < keep) != ((kept >> i & 1) != 0));  // freed slots, and movers behind
    }
    st.moved = rank_all() / 2;  // as many movers as freed slots
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int t = i * kThreads + tid;
      if (flags[i] >> lane & 1) list[s_count[i * kWaves + wave] + __popcll(flags[i] & below)] = t;
      if (lane == 0 && t < keep && t < n) freed[t >> 6] = flags[i];  // (bits behind keep are not read)
    }
  }
  if (tid == 0) a.state[row] = st;
}

// Long rows, first launch: counters to zero, the rows' states.
__global__ __launch_bounds__(256) void evict_clear_kernel(const EvictArgs a) {
  const int64_t n = (int64_t)a.rows * kTop;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    a.hist[i] = 0;
    if (i < a.rows) {
      a.found[i] = 0;
      a.state[i] = row_state(a, (int)i);
    }
  }
}

// (Beyond 2^19 rows the offsets of their counters pass 2^31.)
__device__ __forceinline__ int32_t* row_hist(const EvictArgs& a, int row) { return a.hist + (int64_t)row * kTop; }

// Second: the keys, counted by their top bits.
__global__ __launch_bounds__(kRunThreads) void evict_count_kernel(const EvictArgs a, uint32_t group0) {
  __shared__ int s_hist[kTop];
  const uint32_t x = group0 + blockIdx.x;
  const int row = x % a.rows, run = x / a.rows, tid = threadIdx.x;
  const int n = a.state[row].n, keep = a.state[row].keep;
  if (n <= keep || run * kRun >= n) return;
  const int first_recent = n + a.state[row].dropped - a.recent;
  for (int i = tid; i < kTop; i += kRunThreads) s_hist[i] = 0;
  __syncthreads();
  uint32_t* const keys = a.keys + (int64_t)row * a.pool.capacity;
  uint32_t k[kRunPer];
#pragma unroll
  for (int i = 0; i < kRunPer; ++i) {
    const int t = run * kRun + i * kRunThreads + tid;
    k[i] = t < n ? token_key(a, row, t, first_recent) : 0u;
  }
#pragma unroll
  for (int i = 0; i < kRunPer; ++i) {
    const int t = run * kRun + i * kRunThreads + tid;
    if (t < n) {
      keys[t] = k[i];
      atomicAdd(&s_hist[k[i] >> (32 - kTopBits)], 1);
    }
  }
  __syncthreads();
  for (int i = tid; i < kTop; i += kRunThreads)
    if (s_hist[i]) atomicAdd(row_hist(a, row) + i, s_hist[i]);
}

// Bin, from the top, that holds the want-th of the counts (kRunThreads * PER of
// them), and which of the bin's it is.
template <int PER>
__device__ __forceinline__ int2 pick_bin(const int* hist, int want, int* s_wave, int* s_pick, int tid) {
  int c[PER], sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    c[i] = hist[kRunThreads * PER - 1 - tid * PER - i];
    sum += c[i];
  }
  const int incl = block_scan<kRunThreads / 64>(sum, s_wave, tid);
  int before = incl - sum;
  if (before < want && incl >= want) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (before < want && before + c[i] >= want) {
        s_pick[0] = kRunThreads * PER - 1 - tid * PER - i;
        s_pick[1] = want - before;
      }
      before += c[i];
    }
  }
  __syncthreads();
  return make_int2(s_pick[0], s_pick[1]);
}

// Third: the keys that share the threshold's top bits (in any order).
__global__ __launch_bounds__(kRunThreads) void evict_collect_kernel(const EvictArgs a, uint32_t group0) {
  __shared__ int s_wave[kRunThreads / 64 + 1], s_pick[2];
  __shared__ int s_base[kRunThreads / 64];
  const uint32_t x = group0 + blockIdx.x;
  const int row = x % a.rows, run = x / a.rows, tid = threadIdx.x;
  const int n = a.state[row].n, keep = a.state[row].keep;
  if (n <= keep || keep == 0 || run * kRun >= n) return;
  const uint32_t top = (uint32_t)pick_bin<kTop / kRunThreads>(row_hist(a, row), keep, s_wave, s_pick, tid).x;
  const uint32_t* const keys = a.keys + (int64_t)row * a.pool.capacity;
  uint32_t* const out = a.candidates + (int64_t)row * a.pool.capacity;
  uint32_t k[kRunPer];
  int mine = 0;
#pragma unroll
  for (int i = 0; i < kRunPer; ++i) {
    const int t = run * kRun + i * kRunThreads + tid;
    k[i] = t < n ? keys[t] : 0u;
    mine += t < n && k[i] >> (32 - kTopBits) == top;
  }
  int at = block_scan<kRunThreads / 64>(mine, s_wave, tid) - mine;
  const int all = s_wave[kRunThreads / 64];
  if (all == 0) return;
  if (tid == 0) s_base[0] = atomicAdd(a.found + row, all);
  __syncthreads();
  at += s_base[0];
#pragma unroll
  for (int i = 0; i < kRunPer; ++i) {
    const int t = run * kRun + i * kRunThreads + tid;
    if (t < n && k[i] >> (32 - kTopBits) == top) out[at++] = k[i];
  }
}

// Fourth: the threshold, and the run's keys above it and at it.
__global__ __launch_bounds__(kRunThreads) void evict_rank_kernel(const EvictArgs a, uint32_t group0) {
  __shared__ int s_hist[kRunThreads * 8];
  __shared__ int s_wave[kRunThreads / 64 + 1], s_pick[2];
  __shared__ RunCount s_count;
  const uint32_t x = group0 + blockIdx.x;
  const int row = x % a.rows, run = x / a.rows, tid = threadIdx.x;
  const int n = a.state[row].n, keep = a.state[row].keep;
  if (n <= keep || run * kRun >= n) return;
  uint32_t least = 0xffffffffu;
  int equal = 0;
  if (keep > 0) {
    const int2 top = pick_bin<kTop / kRunThreads>(row_hist(a, row), keep, s_wave, s_pick, tid);
    const int found = a.found[row];
    const uint32_t* const cand = a.candidates + (int64_t)row * a.pool.capacity;
    // The 20 bits left, 11 and 9 at a time.
    uint32_t prefix = (uint32_t)top.x << (32 - kTopBits), mask = ~0u << (32 - kTopBits);
    equal = top.y;
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
      const int shift = pass == 0 ? 9 : 0;
      const uint32_t bins = pass == 0 ? 2048 : 512;
      __syncthreads();
      for (int i = tid; i < kRunThreads * 8; i += kRunThreads) s_hist[i] = 0;
      __syncthreads();
      for (int i0 = 0; i0 < found; i0 += 4 * kRunThreads) {
        uint32_t k[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) k[u] = cand[min(i0 + u * kRunThreads + tid, found - 1)];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (i0 + u * kRunThreads + tid < found && (k[u] & mask) == prefix) atomicAdd(&s_hist[k[u] >> shift & (bins - 1)], 1);
      }
      __syncthreads();
      const int2 bin = pick_bin<8>(s_hist, equal, s_wave, s_pick, tid);
      prefix |= (uint32_t)bin.x << shift;
      mask |= (bins - 1) << shift;
      equal = bin.y;
    }
    least = prefix;
  }
  if (run == 0 && tid == 0) a.state[row].least = least, a.state[row].equal = equal;
  if (tid == 0) s_count = RunCount{0, 0, 0, 0};
  __syncthreads();
  const uint32_t* const keys = a.keys + (int64_t)row * a.pool.capacity;
  int above = 0, eq = 0, above2 = 0, eq2 = 0;
#pragma unroll
  for (int i = 0; i < kRunPer; ++i) {
    const int t = run * kRun + i * kRunThreads + tid;
    if (t >= n) continue;
    const uint32_t k = keys[t];
    const bool g = keep > 0 && k > least, e = keep > 0 && k == least;
    above += g && t < keep, eq += e && t < keep, above2 += g && t >= keep, eq2 += e && t >= keep;
  }
  above = __builtin_amdgcn_readlane(wave_scan_add(above), 63), eq = __builtin_amdgcn_readlane(wave_scan_add(eq), 63);
  above2 = __builtin_amdgcn_readlane(wave_scan_add(above2), 63), eq2 = __builtin_amdgcn_readlane(wave_scan_add(eq2), 63);
  if ((tid & 63) == 0) {
    atomicAdd(&s_count.above, above), atomicAdd(&s_count.equal, eq);
    atomicAdd(&s_count.above_behind, above2), atomicAdd(&s_count.equal_behind, eq2);
  }
  __syncthreads();
  if (tid == 0) a.counts[row * a.runs + run] = s_count;
}

// Fifth: the lists.  What the runs ahead free and move follows from their counts.
__global__ __launch_bounds__(kRunThreads) void evict_list_kernel(const EvictArgs a, uint32_t group0) {
  __shared__ int s_part[3][kRunPer * kRunThreads / 64];
  const uint32_t x = group0 + blockIdx.x;
  const int row = x % a.rows, run = x / a.rows, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const RowState st = a.state[row];
  const int n = st.n, keep = st.keep;
  if (n <= keep && run == 0 && tid == 0) a.state[row].moved = 0;
  if (n <= keep || run * kRun >= n) return;
  // Runs ahead: their equal keys, freed slots and movers; and all freed slots.
  // Every wave for itself, 64 runs at a time.
  const int runs = (n + kRun - 1) / kRun;
  int eq_before = 0, free_before = 0, move_before = 0, free_all = 0, eq_seen = 0;
  auto sum = [](int v) { return __builtin_amdgcn_readlane(wave_scan_add(v), 63); };
  for (int r0 = 0; r0 < runs; r0 += 64) {
    const int r = r0 + lane;
    const RunCount c = r < runs ? a.counts[row * a.runs + r] : RunCount{0, 0, 0, 0};
    const int eq = c.equal + c.equal_behind, eq_incl = wave_scan_add(eq) + eq_seen;
    eq_seen = __builtin_amdgcn_readlane(eq_incl, 63);
    const int left = max(st.equal - (eq_incl - eq), 0);  // equal keys that this run may still keep
    const int kept = c.above + min(c.equal, left), moved = c.above_behind + min(c.equal_behind, max(left - c.equal, 0));
    const int slots = r < runs ? min(max(keep - r * kRun, 0), kRun) : 0;  // below keep (all of them hold tokens)
    const bool ahead = r < run;
    eq_before += sum(ahead ? eq : 0);
    free_before += sum(ahead ? slots - kept : 0);
    move_before += sum(ahead ? moved : 0);
    free_all += sum(slots - kept);
  }
  if (run == 0 && tid == 0) a.state[row].moved = free_all;
  const uint32_t* const keys = a.keys + (int64_t)row * a.pool.capacity;
  int32_t* const list = a.moves + (int64_t)row * a.pool.capacity;
  uint32_t k[kRunPer];
  uint64_t eqs[kRunPer];
  constexpr int kW = kRunThreads / 64;
#pragma unroll
  for (int i = 0; i < kRunPer; ++i) {
    const int t = run * kRun + i * kRunThreads + tid;
    k[i] = t < n ? keys[t] : 0u;
    eqs[i] = __ballot(t < n && keep > 0 && k[i] == st.least);
    if (lane == 0) s_part[0][i * kW + wave] = __popcll(eqs[i]);
  }
  // (Counts of 64 slots, in slot order, to what lies before them.)
  static_assert(kRunPer * kW <= 64, "one scan");
  auto prefix = [&](int* c) {
    const int v = lane < kRunPer * kW ? c[lane] : 0;
    const int incl = wave_scan_add(v);
    if (lane < kRunPer * kW) c[lane] = incl - v;
  };
  __syncthreads();
  if (wave == 0) prefix(s_part[0]);
  __syncthreads();
  const uint64_t below = (1ull << lane) - 1;
  uint64_t freed[kRunPer], moved[kRunPer];
#pragma unroll
  for (int i = 0; i < kRunPer; ++i) {
    const int t = run * kRun + i * kRunThreads + tid;
    const int rank = eq_before + s_part[0][i * kW + wave] + __popcll(eqs[i] & below);
    const bool kept = t < n && keep > 0 && (k[i] > st.least || (k[i] == st.least && rank < st.equal));
    freed[i] = __ballot(t < keep && t < n && !kept);
    moved[i] = __ballot(t >= keep && kept);
    if (lane == 0) {
      s_part[1][i * kW + wave] = __popcll(freed[i]), s_part[2][i * kW + wave] = __popcll(moved[i]);
      if (t < keep && t < n) a.freed[(int64_t)row * ((a.pool.capacity + 63) / 64) + (t >> 6)] = freed[i];
    }
  }
  __syncthreads();
  if (wave < 2) prefix(s_part[1 + wave]);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRunPer; ++i) {
    const int t = run * kRun + i * kRunThreads + tid;
    if (freed[i] >> lane & 1) list[free_before + s_part[1][i * kW + wave] + __popcll(freed[i] & below)] = t;
    if (moved[i] >> lane & 1) list[free_all + move_before + s_part[2][i * kW + wave] + __popcll(moved[i] & below)] = t;
  }
}

// The moves of all rows, and their new lengths.  blockIdx.y: a head's keys and
// values (16 bytes a thread, neighbouring threads a token), then a head's
// weights, then the positions.  Both pages of a move lie in the pool, or the
// token's keys and values stay where they are and the status word says so.
__global__ __launch_bounds__(256) void evict_move_kernel(const EvictArgs a, uint32_t group0) {
  const Pool& p = a.pool;
  const uint32_t x = group0 + blockIdx.x;
  const int row = x / a.move_blocks, blk = x % a.move_blocks;
  const RowState st = a.state[row];
  const int count = st.moved, kept = min(st.n, st.keep);
  const int32_t* const list = a.moves + (int64_t)row * p.capacity;
  const int step = a.move_blocks * 256, first = blk * 256 + threadIdx.x;
  if ((int)blockIdx.y >= p.heads) {
    const int j = blockIdx.y - p.heads;
    const bool pos = j == p.heads;
    if (pos && first == 0) {
      a.len_out[row] = kept;
      a.dropped_out[row] = st.dropped + st.n - kept;
    }
    const int64_t at = pos ? row * a.pos_stride : ((int64_t)row * p.heads + j) * a.weight_stride;
    const uint32_t* const in = (pos ? reinterpret_cast<const uint32_t*>(a.pos) : reinterpret_cast<const uint32_t*>(a.weights)) + at;
    uint32_t* const out = (pos ? reinterpret_cast<uint32_t*>(a.pos_out) : reinterpret_cast<uint32_t*>(a.weights_out)) + at;
    for (int i = first; i < count; i += step) out[list[i]] = in[list[count + i]];
    if (in != out) {
      const uint64_t* const freed = a.freed + (int64_t)row * ((p.capacity + 63) / 64);
      for (int t = first; t < kept; t += step)
        if (count == 0 || !(freed[t >> 6] >> (t & 63) & 1)) out[t] = in[t];
    }
    return;
  }
  const int h = blockIdx.y, shift = a.esz == 4 ? 5 : 4;  // 16-byte chunks of a token
  const int32_t* const tab = p.table + row * p.table_stride;
  const char *const kh = p.k + h * p.k_head, *const vh = p.v + h * p.v_head;
  const int64_t units = (int64_t)count << shift;
  constexpr int kFlight = 2;  // chunks of a thread in flight
  for (int64_t u0 = first; u0 < units; u0 += (int64_t)kFlight * step) {
    u32x4 k[kFlight], v[kFlight];
    int64_t to_k[kFlight], to_v[kFlight];
    bool ok[kFlight];
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      const int64_t u = min(u0 + (int64_t)f * step, units - 1);
      const int i = (int)(u >> shift), off = 16 * (int)(u & ((1 << shift) - 1));
      const int to = list[i], of = list[count + i];
      const int tp = page_of(p, to), op = page_of(p, of);
      const int tg = tab[tp], og = tab[op];
      const bool live = (uint32_t)tg < (uint32_t)p.pages && (uint32_t)og < (uint32_t)p.pages;
      if (!live && p.status) atomicOr(p.status, kStatusPage);
      ok[f] = live && u0 + (int64_t)f * step < units;
      const int ta = to - tp * p.page_tokens, oa = of - op * p.page_tokens;
      const int64_t src = live ? og : 0;  // (some page of the pool)
      to_k[f] = tg * p.k_page + ta * p.k_tok + off;
      to_v[f] = tg * p.v_page + ta * p.v_tok + off;
      k[f] = *reinterpret_cast<const u32x4*>(kh + src * p.k_page + oa * p.k_tok + off);
      v[f] = *reinterpret_cast<const u32x4*>(vh + src * p.v_page + oa * p.v_tok + off);
    }
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      if (!ok[f]) continue;
      *reinterpret_cast<u32x4*>(const_cast<char*>(kh) + to_k[f]) = k[f];
      *reinterpret_cast<u32x4*>(const_cast<char*>(vh) + to_v[f]) = v[f];
    }
  }
}

// Rows of up to this many tokens go to one workgroup each.
constexpr int kShort = 16 * kThreads;

struct EvictLayout {
  size_t state, moves, freed, keys, candidates, hist, found, counts, bytes;
  int rows, runs;
  bool is_long;
};

EvictLayout evict_layout(const hc_paged_cache* c) {
  EvictLayout l = {};
  const int64_t cap = (int64_t)c->table_pages * c->page_tokens;
  l.rows = c->batch * c->kv_heads / c->heads;
  l.is_long = cap > kShort;
  l.runs = l.is_long ? (int)((cap + kRun - 1) / kRun) : 0;
  auto take = [&](size_t bytes) {
    const size_t here = l.bytes;
    l.bytes += (bytes + 255) / 256 * 256;
    return here;
  };
  l.state = take((size_t)l.rows * sizeof(RowState));
  l.moves = take((size_t)l.rows * cap * 4);
  l.freed = take((size_t)l.rows * ((cap + 63) / 64) * 8);
  if (l.is_long || c->heads > 1) l.keys = take((size_t)l.rows * cap * 4);
  if (l.is_long) {
    l.candidates = take((size_t)l.rows * cap * 4);
    l.hist = take((size_t)l.rows * kTop * 4);
    l.found = take((size_t)l.rows * 4);
    l.counts = take((size_t)l.rows * l.runs * sizeof(RunCount));
  }
  return l;
}

}  // namespace

int fill_pool(const char* name, const hc_paged_cache* c, Pool& p, int Q, const int32_t* counts);

}  // namespace hc

using namespace hc;

extern "C" size_t hc_paged_evict_scratch_size(const hc_paged_cache* c) {
  if (!c || c->batch <= 0 || c->kv_heads <= 0 || (c->heads != 1 && c->heads != c->kv_heads) || c->table_pages <= 0 ||
      c->page_tokens <= 0)
    return 0;
  return evict_layout(c).bytes;
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
  const EvictLayout l = evict_layout(c);
  if (scratch_bytes < l.bytes || !scratch || (reinterpret_cast<uintptr_t>(scratch) & 15))
    return set_error(HC_ERR_INVALID, "hc_paged_evict: scratch too small or unaligned (%zu < %zu bytes)", scratch_bytes, l.bytes);
  a.rows = l.rows;
  a.keep = keep, a.keep_all = keep_all, a.sink = sink, a.recent = recent;
  a.weights = c->weights, a.weight_stride = c->weight_stride;
  a.weights_out = weights_out ? weights_out : c->weights;
  a.pos = c->pos, a.pos_stride = c->pos_stride, a.pos_out = pos_out ? pos_out : c->pos;
  a.dropped = c->dropped, a.dropped_out = dropped_out ? dropped_out : c->dropped;
  a.len_out = len_out ? len_out : c->row_len;
  char* const ws = reinterpret_cast<char*>(scratch);
  a.state = reinterpret_cast<RowState*>(ws + l.state);
  a.moves = reinterpret_cast<int32_t*>(ws + l.moves);
  a.freed = reinterpret_cast<uint64_t*>(ws + l.freed);
  a.keys = reinterpret_cast<uint32_t*>(ws + l.keys);
  a.candidates = reinterpret_cast<uint32_t*>(ws + l.candidates);
  a.hist = reinterpret_cast<int32_t*>(ws + l.hist);
  a.found = reinterpret_cast<int32_t*>(ws + l.found);
  a.counts = reinterpret_cast<RunCount*>(ws + l.counts);
  a.runs = l.runs;
  a.esz = c->dtype == HC_DTYPE_F32 ? 4 : 2;
  // Workgroups of 256 chunks for the most that a head can move, at most some
  // eight a CU over all heads.
  const int64_t most = (int64_t)(a.pool.capacity / 2) * (HC_HEAD_DIM * a.esz / 16);
  a.move_blocks = (int)std::max<int64_t>(1, std::min<int64_t>((most + 511) / 512, 4096 / (a.rows * (2 * a.pool.heads + 1))));
  hipStream_t s = (hipStream_t)stream;
  if (a.pool.heads > 32767) return set_error(HC_ERR_INVALID, "hc_paged_evict: %d heads", a.pool.heads);
  auto launch = [&](auto kernel, int64_t n, int threads, unsigned y = 1) {
    return in_launches(n, threads, [&](dim3 grid, uint32_t group0) {
      grid.y = y;
      hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, s, a, group0);
      return check_launch("hc_paged_evict");
    });
  };
  int rc;
  if (l.is_long) {
    const int64_t runs = (int64_t)a.rows * l.runs;
    hipLaunchKernelGGL(evict_clear_kernel, dim3((unsigned)std::min<int64_t>(((int64_t)a.rows * kTop + 255) / 256, 1024)), dim3(256), 0, s, a);
    rc = check_launch("hc_paged_evict");
    if (!rc) rc = launch(evict_count_kernel, runs, kRunThreads);
    if (!rc) rc = launch(evict_collect_kernel, runs, kRunThreads);
    if (!rc) rc = launch(evict_rank_kernel, runs, kRunThreads);
    if (!rc) rc = launch(evict_list_kernel, runs, kRunThreads);
  } else {
    const bool few = a.pool.capacity <= 4 * kThreads;
    if (a.pool.heads > 1) {
      rc = launch(evict_keys_kernel, (int64_t)a.rows * ((a.pool.capacity + kRunThreads - 1) / kRunThreads), kRunThreads);
      if (!rc) rc = few ? launch(evict_select_kernel<4, true>, a.rows, kThreads) : launch(evict_select_kernel<16, true>, a.rows, kThreads);
    } else {
      rc = few ? launch(evict_select_kernel<4, false>, a.rows, kThreads) : launch(evict_select_kernel<16, false>, a.rows, kThreads);
    }
  }
  return rc ? rc : launch(evict_move_kernel, (int64_t)a.rows * a.move_blocks, 256, 2 * a.pool.heads + 1);
}
