// Attention of a batch over one shared prefix and each sequence's own rows.
//
//   out[b, i, h] = softmax over the tokens of prefix row kv(h) and the visible
//   tokens of row (b, kv(h)), times their values; query i sees the row's
//   tokens t < len - n + 1 + i, n the new tokens of the sequence (all Q
//   queries, or a count of its own behind which queries are padding).
//
// Both parts lie in ragged tiled stores; the prefix has one row per KV head,
// of its own length (a document compressed per head, or whole).  Softmax over
// the union is folded from partial states (m, l, O), so the prefix is read
// once for all sequences.  Two launches:
//  * shared_attn_kernel, two kinds of workgroups side by side.  Prefix
//    workgroups: the batch * Q * G query rows of a KV head are the columns of
//    the products S^T = K Q^T and O^T += V^T P^T over a part of the prefix,
//    whose tiles 4 waves x NC x 16 columns share through LDS.  Row
//    workgroups: each sequence's own rows (rows_job).  With many columns the
//    former are bound by the matrix cores and the latter by HBM, so they run
//    on the same CUs at once.
//  * merge_kernel (hc_rows.hip): one fold of a column's partials.
// In bf16: 32 sequences x 32 heads behind 178K prefix tokens of 8 heads, own
// rows of up to 512: 27 to 31 + 4 us, of which the bytes (128 MB) need 18 and a
// workgroup's start and end 8 to 10; 128 sequences behind 756K tokens, 1.06M of
// their own: 240 to 255 + 9 us, the prefix alone 190 (1.04 PFLOP/s, 68 % of the
// issue slots taken), the rows alone 92 (5.9 TB/s).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "hc_rows.h"

namespace hc {
namespace {

constexpr int kPreWaves = 4;
constexpr int kPreThreads = kPreWaves * 64;
// Slots of tiles in LDS, of keys and of values (one more or less changes no
// time by more than 2 %).
constexpr int kRing = 4;

struct PrefixArgs {
  const void* q;
  int64_t q_s[3];
  const void *kstore, *vstore;
  const int64_t* tile_off;
  const int32_t* len;
  int Hkv, G, Q;
  int64_t M;   // columns: batch * Q * G
  int ncg;     // column groups of 64 * NC
  int parts;   // workgroups of a column group, a multiple of 8 (0: no prefix)
  float scale_log2;
  float *part_o, *part_ml;
  int32_t* info;
};

// Tiles a part takes so that every row is covered by at most `parts` parts in
// all: each row's last part may be short, so the shares are cut from the
// parts left when every row has one.
__device__ __forceinline__ int part_tiles(uint32_t total, int rows, int parts) {
  const uint32_t n = max(parts - rows, 1);
  return (int)max((total + n - 1) / n, 1u);
}

__device__ __forceinline__ int tiles_of(int len) { return (max(len, 0) + HC_TILE - 1) / HC_TILE; }

// A barrier that waits for this wave's LDS reads and not for its loads in
// flight, as __syncthreads does.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Waits until at most `units` (0 .. U) times LOADS of this wave's loads are in
// flight.
template <int U, int LOADS>
__device__ __forceinline__ void wait_dma_units(int units) {
  if constexpr (U == 0) {
    wait_lds_dma();
  } else {
    if (units >= U)
      wait_lds_dma_but<U * LOADS>();
    else
      wait_dma_units<U - 1, LOADS>(units);
  }
}

template <typename T, int NC, bool ONCE>
__device__ __forceinline__ void prefix_job(const PrefixArgs& a, int x, T* lds) {
  typedef typename Elem<T>::vec8 vec8;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g4 = lane >> 4, n16 = lane & 15;

  // Column groups of one part go to one XCD (workgroups are dealt to the 8
  // XCDs in turn), so its L2 serves the tiles after their first read.
  const int part = (x / (8 * a.ncg)) * 8 + x % 8, cg = (x / 8) % a.ncg;

  // (row, share) of the part, from the device lengths: rows 64 at a time,
  // their tile offsets requested along with the lengths.
  int row_n = 0, nt = 0;
  int64_t row_off = 0;
  auto load_rows = [&](int r0) {
    const int r = min(r0 + lane, a.Hkv - 1);
    row_off = a.tile_off[r];
    row_n = max(a.len[r], 0);
    row_n = r0 + lane < a.Hkv ? row_n : 0;
    // Opaque: knowing which lanes hold zero, the compiler would run them apart
    // and the wave's sums over the others alone; and it would move the offsets'
    // load behind the sums.
    asm("" : "+v"(row_n), "+v"(row_off));
    nt = tiles_of(row_n);
  };
  load_rows(0);
  uint32_t total = 0;  // (2^31 tiles are 35 TB)
  for (int r0 = 0;;) {
    total += __builtin_amdgcn_readlane(wave_scan_add(nt), 63);
    r0 += 64;
    if (r0 >= a.Hkv) break;
    load_rows(r0);
  }
  const int share = part_tiles(total, a.Hkv, a.parts);
  int kv = -1, t0 = 0, t1 = 0, len = 0, first = 0;
  int64_t tile0 = 0;
  for (int r0 = 0; r0 < a.Hkv; r0 += 64) {
    if (a.Hkv > 64) load_rows(r0);
    const int np = (nt + share - 1) / share;
    const int incl = wave_scan_add(np) + first;
    if (x == 0 && wave == 0 && r0 + lane < a.Hkv) {
      a.info[2 * (r0 + lane)] = incl - np;
      a.info[2 * (r0 + lane) + 1] = np;
    }
    const uint64_t hit = __ballot(part >= incl - np && part < incl);
    if (hit && kv < 0) {
      const int src = __builtin_ctzll(hit);
      kv = r0 + src;
      t0 = (part - __builtin_amdgcn_readlane(incl - np, src)) * share;
      t1 = min(t0 + share, __builtin_amdgcn_readlane(nt, src));
      len = __builtin_amdgcn_readlane(row_n, src);
      tile0 = (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)row_off, src) |
              (int64_t)__builtin_amdgcn_readlane((int)(row_off >> 32), src) << 32;
    }
    first = __builtin_amdgcn_readlane(incl, 63);
  }
  if (kv < 0) return;

  // Q^T operands: column col0 + 16j + n16, k-slots = channels 32s + 8*g4 + [0, 8).
  const int64_t col0 = ((int64_t)cg * kPreWaves + wave) * 16 * NC;
  const int active = __builtin_amdgcn_readfirstlane(col0 < a.M);
  vec8 qop[NC][4];
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int64_t c = col0 + 16 * j + n16;
    const bool ok = c < a.M;
    const int64_t bi = ok ? c / a.G : 0;
    const T* qp = reinterpret_cast<const T*>(a.q) + (bi / a.Q) * a.q_s[0] + (kv * a.G + (ok ? c % a.G : 0)) * a.q_s[1] +
                  (bi % a.Q) * a.q_s[2] + 8 * g4;
#pragma unroll
    for (int s = 0; s < 4; ++s) qop[j][s] = ok ? load8<T>(qp + 32 * s) : zero8<T>();
  }
  __builtin_amdgcn_sched_barrier(0);

  // Staging: the tiles lie contiguous in memory and keep their layout in LDS,
  // so a tile is 16-byte units copied straight into LDS (global_load_lds).
  // Batch i holds the keys of tile i + 2 and the values of tile i.
  constexpr int kTileBytes = HC_TILE_ELEMS * (int)sizeof(T);
  constexpr int kLoads = kTileBytes / (16 * kPreThreads);  // per thread, of K and of V
  const int n = t1 - t0;
  const char* kb = reinterpret_cast<const char*>(a.kstore) + (tile0 + t0) * (int64_t)kTileBytes;
  const char* vb = reinterpret_cast<const char*>(a.vstore) + (tile0 + t0) * (int64_t)kTileBytes;
  char* const ring = reinterpret_cast<char*>(lds) + 1024 * kLoads * wave;
  const float scale_log2 = a.scale_log2;
  auto copy = [&](const char* src, int slot) {  // slots: kRing of keys, then kRing of values
    // A 32-bit offset from a scalar base, which the compiler forgets once it
    // has widened it outside of the loop.
    uint32_t own = 1024 * kLoads * wave + 16 * lane;
    asm volatile("" : "+v"(own));
    lds_dma16_run<kLoads, ONCE>(src + own, ring + slot * kTileBytes);
  };
  auto stage_k = [&](int slot) {  // the next keys, the next values
    copy(kb, slot);
    kb += kTileBytes;
  };
  auto stage_v = [&](int slot) {
    copy(vb, kRing + slot);
    vb += kTileBytes;
  };
  static_assert(kRing == 4, "slots i % 4 and their neighbours by ^ 2");
  stage_k(0);
  if (1 < n) stage_k(1);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (i + 2 < n) stage_k(i + 2);
    if (i < n) stage_v(i);
  }

  f32x4 o[8][NC], s[2][2][NC];  // s: of the tile attended, and of the next one, in turn
  vec8 pb[NC], vr[8];
  float m[NC], l[NC];
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    m[j] = -INFINITY, l[j] = 0.f;
    pb[j] = zero8<T>();
#pragma unroll
    for (int db = 0; db < 8; ++db) o[db][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < 2; ++h) s[0][h][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll
  for (int x = 0; x < 8; ++x) vr[x] = zero8<T>();
  // The queries and the first two tiles' keys are here, the batches in flight.
  if (kRing <= n)
    wait_lds_dma_but<(kRing - 2) * 2 * kLoads>();
  else
    wait_lds_dma();
  lds_barrier();
  vec8 kr[8];  // keys in the order of the products: half h = x & 1, channels 32 (x / 2) + [0, 32)
  auto key_at = [&](const T* p, int x) { return load8<T>(p + ((x & 1) * 4 + (x >> 1)) * 512 + lane * 8); };
  if (active) {
#pragma unroll
    for (int x = 0; x < 8; ++x) kr[x] = key_at(lds, x);
#pragma unroll
    for (int x = 0; x < 8; ++x) {
#pragma unroll
      for (int j = 0; j < NC; ++j) s[0][x & 1][j] = mma_16x16x32(kr[x], qop[j][x >> 1], s[0][x & 1][j]);
    }
#pragma unroll
    for (int x = 0; x < 8; ++x) kr[x] = key_at(lds + HC_TILE_ELEMS, x);
  }

  int slot = 0;  // i % kRing
  // One tile, i, with tile i + 1's scores and the product of tile i - 1's
  // values on the matrix cores while the vector unit forms the probabilities
  // between them: kr holds the keys of tile i + 1, vr and pb the values and
  // probabilities of tile i - 1, and each operand is read from LDS again, for
  // the next step, once it is used.  STEADY: four tiles or more follow.
  // (Behind the last tile: products of stale slots, which nothing reads.)
  auto step = [&](auto steady, int i, f32x4(&sc)[2][NC], f32x4(&sn)[2][NC]) {
    constexpr bool STEADY = decltype(steady)::value;
    // This wave's loads of batch i have landed, and past the barrier every
    // wave's have, while the younger ones stay in flight; every wave is also
    // done with the keys of tile i + 1 and the values of tile i - 1: batch i + 2
    // takes the slots of the keys of tile i and of the values of tile i - 2.
    if constexpr (STEADY)
      wait_lds_dma_but<2 * kLoads>();
    else  // younger values, and keys
      wait_dma_units<2, kLoads>((i + 1 < n) + (i + 3 < n));
    lds_barrier();
    if (STEADY || i + 4 < n) stage_k(slot);
    if (STEADY || i + 2 < n) stage_v(slot ^ 2);
    const T* sk = lds + (slot ^ 2) * HC_TILE_ELEMS;
    const T* sv = lds + (kRing + slot) * HC_TILE_ELEMS + lane * 8;
    slot = (slot + 1) & 3;
    if (!active) return;
    if constexpr (!STEADY) {
      const int left = len - (t0 + i) * HC_TILE;  // tokens from this tile on
      if (left < HC_TILE) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (16 * (e >> 2) + 4 * g4 + (e & 3) >= left) {
#pragma unroll
            for (int j = 0; j < NC; ++j) sc[e >> 2][j][e & 3] = -INFINITY;
          }
      }
    }
    float pv[NC][8], ps[NC];
    f32x4 upper[2][NC];  // fp32: the sums over the upper 64 channels apart (see tile_scores)
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      ps[j] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) sn[h][j] = upper[h][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int x = 0; x < 8; ++x) {
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        f32x4& acc = sizeof(T) == 4 && x >= 4 ? upper[x & 1][j] : sn[x & 1][j];
        acc = mma_16x16x32(kr[x], qop[j][x >> 1], acc);
        o[x][j] = mma_16x16x32(vr[x], pb[j], o[x][j]);
        pv[j][x] = fast_exp2(fmaf(sc[x >> 2][j][x & 3], scale_log2, -m[j]));
        ps[j] += pv[j][x];
      }
      kr[x] = key_at(sk, x);
      vr[x] = load8<T>(sv + x * 512);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) sn[h][j] += upper[h][j];
    }
    bool fine = ps[0] <= Weights<T>::kLazy;
#pragma unroll
    for (int j = 1; j < NC; ++j) fine = fine && ps[j] <= Weights<T>::kLazy;
    if (__any(!fine)) {  // also NaN, as in the first tile
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        float mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; ++e) mx = fmaxf(mx, sc[e >> 2][j][e & 3]);
        const float mnew = next_reference<T>(m[j], rows4_max(mx) * scale_log2);
        const float alpha = m[j] == -INFINITY ? 0.f : fast_exp2(m[j] - mnew);
        m[j] = mnew;
        l[j] *= alpha;
#pragma unroll
        for (int db = 0; db < 8; ++db) o[db][j] *= alpha;
        const float nm = mnew == -INFINITY ? 0.f : -mnew;
        ps[j] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          pv[j][e] = fast_exp2(fmaf(sc[e >> 2][j][e & 3], scale_log2, nm));
          ps[j] += pv[j][e];
        }
        if (mnew == -INFINITY) ps[j] += 1.f;  // tokens, but none above -inf (see hc_rows.h)
      }
    }
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      l[j] += ps[j];
      pb[j] = pack8<T>(pv[j]);  // at most half a step of the input type per probability
    }
  };
  int i = 0;
  for (; i + kRing + 1 < n; i += 2) {
    step(std::true_type{}, i, s[0], s[1]);
    step(std::true_type{}, i + 1, s[1], s[0]);
  }
  for (; i < n; ++i) {
    step(std::false_type{}, i, s[0], s[1]);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < NC; ++j) s[0][h][j] = s[1][h][j];
  }
  if (active) {
    const int left = len - (t1 - 1) * HC_TILE;
    if (left < HC_TILE) {
      // The row's last tile: its stale slots may hold NaN, which a zero
      // probability does not silence.
#pragma unroll
      for (int x = 0; x < 8; ++x) zero_tail<T>(vr[x], 0, left, g4);
    }
#pragma unroll
    for (int db = 0; db < 8; ++db) {
#pragma unroll
      for (int j = 0; j < NC; ++j) o[db][j] = mma_16x16x32(vr[db], pb[j], o[db][j]);
    }
  }

  // The partials leave through LDS: a wave stores 1 KB in a row, two columns,
  // where its registers hold 64 bytes of each of 16.
  wait_lds_dma();
  lds_barrier();
  if (!active) return;
  float(*so)[kRowsPitch] = reinterpret_cast<float(*)[kRowsPitch]>(lds) + 16 * wave;
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const float lt = rows4_sum(l[j]);
    const int64_t c0 = col0 + 16 * j;
    float* po = a.part_o + ((int64_t)part * a.M + c0) * kPartO;
#pragma unroll
    for (int db = 0; db < 8; ++db) *reinterpret_cast<f32x4*>(&so[n16][16 * db + 4 * g4]) = o[db][j];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int c = 2 * r + (lane >> 5), d = 4 * (lane & 31);
      const f32x4 v = *reinterpret_cast<const f32x4*>(&so[c][d]);
      if (c0 + c < a.M) *reinterpret_cast<f32x4*>(po + c * kPartO + d) = v;
    }
    if (g4 == 0 && c0 + n16 < a.M)
      *reinterpret_cast<float2*>(a.part_ml + ((int64_t)part * a.M + c0 + n16) * 2) = make_float2(m[j], lt);
  }
}

// LDS of a workgroup: the prefix ring, or the row waves' states.
template <typename T>
constexpr size_t shared_lds(bool prefix) {
  const size_t ring = (size_t)2 * kRing * HC_TILE_ELEMS * sizeof(T), rows = kRowsLds * sizeof(float);
  return prefix && ring > rows ? ring : rows;
}

// Prefix workgroups come first: they are the long ones.  (One round of them,
// then the rows', then the rest: 282 us against 265 for 512 columns over 756K
// tokens beside rows of 1.06M.)  Registers for three workgroups a CU serve calls
// of rows alone; beside a prefix the ring's 64 KB of LDS leave two.
template <typename T, int NC, bool MIXED>
__global__ __launch_bounds__(kPreThreads, sizeof(T) == 4 ? 1 : NC == 2 ? 2 : 3) void shared_attn_kernel(
    const PrefixArgs pre, const RowsArgs rows) {
  extern __shared__ __attribute__((aligned(16))) unsigned char shared_raw[];
  const int npre = pre.parts * pre.ncg;
  T* const lds = reinterpret_cast<T*>(shared_raw);
  // One column group reads a tile once: streamed past L2 (83 against 95 us for
  // 16 columns over 131072 tokens of 8 heads; with more column groups the
  // others' reads come from L2, and 4 of them lose 7 % by the hint).
  if ((int)blockIdx.x >= npre)
    rows_job<T, kRowsWhole, MIXED, kPreWaves>(rows, blockIdx.x - npre, reinterpret_cast<float*>(shared_raw));
  else if (pre.ncg == 1)
    prefix_job<T, NC, true>(pre, blockIdx.x, lds);
  else
    prefix_job<T, NC, false>(pre, blockIdx.x, lds);
}

// Sizes of one call: the prefix launch's column blocks and parts, the rows'
// plan, and the workspace in bytes.  Rows alone whose jobs are whole write the
// output themselves.
struct SharedPlan {
  int nc, ncg, parts;
  RowsPlan rows;
  bool direct;
  size_t info_at, pre_o, pre_ml, row_o, row_ml, bytes;
};

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Negative tile counts: no prefix, no rows.
SharedPlan shared_plan(int dtype, int batch, int Hkv, int G, int Q, int64_t prefix_tiles, int64_t row_tiles) {
  SharedPlan p = {1, 1, 0};
  const bool with_prefix = prefix_tiles >= 0, with_rows = row_tiles >= 0;
  // Sizes to cut for: beyond what a device holds they change nothing (and the
  // sums below stay in range).
  prefix_tiles = std::min<int64_t>(prefix_tiles, 1LL << 40), row_tiles = std::min<int64_t>(row_tiles, 1LL << 40);
  const int64_t M = (int64_t)batch * Q * G;
  p.rows = rows_plan(batch * Hkv, G, Q, std::max<int64_t>(row_tiles, 0));
  p.direct = !with_prefix && p.rows.nsplit == 1;
  // Column blocks a wave (nc) and prefix workgroups a CU (k): the least
  // estimate of the call's time in us, fitted to 300 timings of 15 shapes (a
  // few columns to 512, prefixes of 1K to 128K tokens, own rows of 64 to 16K)
  // and within 5 % of their best.  A part's tile of 32 tokens takes `tile` on a
  // CU of its own and 0.65 more for each further workgroup there; the prefix
  // is streamed at 6.5 TB/s at best; a column's partial costs its writing and
  // reading; the rows' stream hides a third behind the products while a CU has
  // room for a row workgroup beside them.  128 columns over 178K tokens: 36.2
  // us with nc = 1, 38.2 with 2, whose partials are twice as many; 448 over
  // 49K, bound by the products: 34.6 and 32.1.
  const int cus = device_cus();
  const bool f32 = dtype == HC_DTYPE_F32;
  const double stream = 1e6 * 2 * HC_TILE_ELEMS * (f32 ? 4. : 2.) / 6.5e12;
  // (Of rows only the longest's length is known: 0.6 of it stands for the mean.)
  const double pre_us = prefix_tiles * stream;
  const double rows_us = 0.6 * (double)batch * Hkv * std::max<int64_t>(row_tiles, 0) * stream;
  double best = 0.;
  for (int nc = 1; with_prefix && nc <= (f32 || M <= 64 ? 1 : 2); ++nc) {
    const int ncg = (int)((M + 64 * nc - 1) / (64 * nc));
    const double tile = f32 ? 1.2 : nc == 1 ? 0.35 : 0.5;
    for (const double k : {0.25, 0.5, 0.75, 1., 1.25, 1.5, 1.75, 2.}) {
      // Every KV head has four parts at least, and there are no more than tiles.
      int64_t n = std::max<int64_t>((int64_t)(k * cus) / ncg, 4 * (int64_t)Hkv);
      n = (std::min(n, prefix_tiles + Hkv + 1) + 7) / 8 * 8;  // whole rounds over the 8 XCDs
      const double kk = (double)n * ncg / cus;
      const double share = std::ceil((double)prefix_tiles / (double)std::max<int64_t>(n - Hkv / 2, 1));
      const double work = share * tile * (1. + 0.65 * (std::max(std::ceil(kk), 1.) - 1.));
      const double rows_seen = rows_us * (kk < (f32 ? 1. : 2.) ? 0.67 : 1.);
      const double t = std::max(std::max(work, pre_us) + rows_seen, pre_us + rows_us) + (double)n * M * 0.2e-3;
      if (best == 0. || t < best) best = t, p.nc = nc, p.ncg = ncg, p.parts = (int)n;
    }
  }
  const size_t pre = (size_t)p.parts * M;
  const size_t row = with_rows && !p.direct ? (size_t)batch * Hkv * Q * G * p.rows.nsplit : 0;
  p.info_at = 0;
  p.pre_o = with_prefix ? up256((size_t)Hkv * 2 * sizeof(int32_t)) : 0;
  p.pre_ml = p.pre_o + up256(pre * kPartO * sizeof(float));
  p.row_o = p.pre_ml + up256(pre * 2 * sizeof(float));
  p.row_ml = p.row_o + up256(row * kPartO * sizeof(float));
  p.bytes = p.row_ml + up256(row * 2 * sizeof(float));
  return p;
}

template <typename T>
int launch_shared(const PrefixArgs& a, const RowsArgs& r, int nc, hipStream_t s) {
  const size_t lds = shared_lds<T>(a.parts > 0);
  const bool mixed = r.qpb > 1;
  auto fn = mixed ? shared_attn_kernel<T, 1, true> : shared_attn_kernel<T, 1, false>;
  if constexpr (sizeof(T) == 2)
    if (nc == 2) fn = mixed ? shared_attn_kernel<T, 2, true> : shared_attn_kernel<T, 2, false>;
  if (lds > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)lds) != hipSuccess)
    return set_error(HC_ERR_HIP, "hc_shared_attn: %s", hipGetErrorString(hipGetLastError()));
  const int64_t grid = (int64_t)a.parts * a.ncg + rows_workgroups(r);
  if (grid > 0x7fffffffLL) return set_error(HC_ERR_INVALID, "hc_shared_attn: %lld workgroups", (long long)grid);
  hipLaunchKernelGGL(fn, dim3((unsigned)grid), dim3(kPreThreads), lds, s, a, r);
  return check_launch("hc_shared_attn");
}

bool bad_sizes(int dtype, int batch, int q_heads, int kv_heads, int queries) {
  return (dtype != HC_DTYPE_BF16 && dtype != HC_DTYPE_F16 && dtype != HC_DTYPE_F32) || batch < 0 || kv_heads < 1 ||
         q_heads < 1 || q_heads % kv_heads || q_heads / kv_heads > 16 || queries < 0 ||
         (int64_t)batch * q_heads * std::max(queries, 1) > (1 << 24);
}

}  // namespace
}  // namespace hc

using namespace hc;

extern "C" size_t hc_shared_workspace_size(int dtype, int batch, int q_heads, int kv_heads, int queries,
                                           int64_t prefix_tiles, int64_t row_tiles) {
  if (bad_sizes(dtype, batch, q_heads, kv_heads, queries)) return 0;
  if (batch == 0 || queries == 0) return 0;
  return shared_plan(dtype, batch, kv_heads, q_heads / kv_heads, queries, prefix_tiles, row_tiles).bytes;
}

extern "C" int hc_shared_attn(int dtype, const void* q, const int64_t* q_strides, const void* kprefix,
                              const void* vprefix, const int64_t* prefix_tile_off, const int32_t* prefix_len,
                              int64_t prefix_tiles, const void* kstore, const void* vstore,
                              const int64_t* row_tile_off, const int32_t* row_len, const int32_t* query_counts,
                              int64_t row_tiles, void* out, const int64_t* out_strides, int batch,
                              int q_heads, int kv_heads, int queries, float scale, void* workspace,
                              size_t workspace_bytes, void* stream) {
  clear_error();
  if (bad_sizes(dtype, batch, q_heads, kv_heads, queries))
    return set_error(HC_ERR_INVALID,
                     "hc_shared_attn: dtype=%d batch=%d q_heads=%d kv_heads=%d queries=%d (q_heads a multiple of "
                     "kv_heads, at most 16 of it, at most 2^24 query rows)",
                     dtype, batch, q_heads, kv_heads, queries);
  if ((prefix_len && prefix_tiles < 0) || (row_len && row_tiles < 0))
    return set_error(HC_ERR_INVALID, "hc_shared_attn: prefix_tiles=%lld row_tiles=%lld", (long long)prefix_tiles,
                     (long long)row_tiles);
  if (!(scale > 0.f) || std::isinf(scale)) return set_error(HC_ERR_INVALID, "hc_shared_attn: scale=%g", (double)scale);
  if (batch == 0 || queries == 0) return HC_OK;
  if (!q || !q_strides || !out || !out_strides || (prefix_len && (!kprefix || !vprefix || !prefix_tile_off)) ||
      (row_len && (!kstore || !vstore || !row_tile_off)))
    return set_error(HC_ERR_INVALID, "hc_shared_attn: null pointer argument");
  if (!prefix_len && !row_len) return set_error(HC_ERR_INVALID, "hc_shared_attn: neither a prefix nor rows");
  const int per16 = dtype == HC_DTYPE_F32 ? 4 : 8;
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] % per16) return set_error(HC_ERR_INVALID, "hc_shared_attn: q strides must be multiples of 16 bytes");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kprefix) | reinterpret_cast<uintptr_t>(vprefix) |
       reinterpret_cast<uintptr_t>(kstore) | reinterpret_cast<uintptr_t>(vstore) |
       reinterpret_cast<uintptr_t>(workspace)) & 15)
    return set_error(HC_ERR_INVALID, "hc_shared_attn: tensors must be 16-byte aligned");
  const int G = q_heads / kv_heads;
  const SharedPlan p =
      shared_plan(dtype, batch, kv_heads, G, queries, prefix_len ? prefix_tiles : -1, row_len ? row_tiles : -1);
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes))
    return set_error(HC_ERR_INVALID, "hc_shared_attn: workspace too small (%zu < %zu bytes)", workspace_bytes, p.bytes);
  char* ws = reinterpret_cast<char*>(workspace);
  const float scale_log2 = scale * 1.4426950408889634f;
  hipStream_t s = (hipStream_t)stream;
  MergeArgs mg;
  mg.pre_o = reinterpret_cast<float*>(ws + p.pre_o), mg.pre_ml = reinterpret_cast<float*>(ws + p.pre_ml);
  mg.info = prefix_len ? reinterpret_cast<int32_t*>(ws + p.info_at) : nullptr;
  mg.M = (int64_t)batch * queries * G;
  mg.row_o = reinterpret_cast<float*>(ws + p.row_o), mg.row_ml = reinterpret_cast<float*>(ws + p.row_ml);
  mg.nsplit = row_len ? p.rows.nsplit : 0;
  mg.Hkv = kv_heads, mg.G = G, mg.Q = queries, mg.out = out;
  for (int i = 0; i < 3; ++i) mg.o_s[i] = out_strides[i];
  PrefixArgs a = {};
  a.q = q, a.kstore = kprefix, a.vstore = vprefix, a.tile_off = prefix_tile_off, a.len = prefix_len;
  a.Hkv = kv_heads, a.G = G, a.Q = queries, a.M = mg.M, a.ncg = p.ncg, a.parts = prefix_len ? p.parts : 0;
  a.scale_log2 = scale_log2;
  a.part_o = reinterpret_cast<float*>(ws + p.pre_o), a.part_ml = reinterpret_cast<float*>(ws + p.pre_ml);
  a.info = reinterpret_cast<int32_t*>(ws + p.info_at);
  RowsArgs r = {};
  r.q = q, r.kstore = kstore, r.vstore = vstore, r.row_tile_off = row_tile_off, r.row_len = row_len;
  r.query_counts = query_counts;
  r.Hkv = kv_heads, r.G = G, r.Q = queries, r.rows = row_len ? batch * kv_heads : 0;
  r.qpb = p.rows.qpb, r.ncb = p.rows.ncb, r.nsplit = p.rows.nsplit, r.scale_log2 = scale_log2;
  if (!p.direct) r.part_o = reinterpret_cast<float*>(ws + p.row_o), r.part_ml = reinterpret_cast<float*>(ws + p.row_ml);
  r.out = out;
  for (int i = 0; i < 3; ++i) a.q_s[i] = r.q_s[i] = q_strides[i], r.o_s[i] = out_strides[i];
  const int rc = dtype == HC_DTYPE_BF16  ? launch_shared<__bf16>(a, r, p.nc, s)
                 : dtype == HC_DTYPE_F16 ? launch_shared<_Float16>(a, r, p.nc, s)
                                         : launch_shared<float>(a, r, p.nc, s);
  if (rc || p.direct) return rc;
  return launch_merge(dtype, mg, (int64_t)batch * queries * q_heads, s);
}
