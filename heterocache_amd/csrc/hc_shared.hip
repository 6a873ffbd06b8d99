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
#include <algorithm>
#include <cmath>

#include "hc_rows.h"

namespace hc {
namespace {

constexpr int kPreWaves = 4;
constexpr int kPreThreads = kPreWaves * 64;
constexpr int kPreRing = 3;  // tiles of K and V held in LDS: one attended, two in flight

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
__device__ __forceinline__ int part_tiles(int64_t total, int rows, int parts) {
  const int64_t n = max(parts - rows, 1);
  return (int)max((total + n - 1) / n, (int64_t)1);
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

template <typename T, int NC>
__device__ __forceinline__ void prefix_job(const PrefixArgs& a, int x, T* lds) {
  typedef typename Elem<T>::vec8 vec8;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g4 = lane >> 4, n16 = lane & 15;

  // Column groups of one part go to one XCD (workgroups are dealt to the 8
  // XCDs in turn), so its L2 serves the tiles after their first read.
  const int part = (x / (8 * a.ncg)) * 8 + x % 8, cg = (x / 8) % a.ncg;

  // (row, share) of the part, from the device lengths: rows 64 at a time.
  int64_t total = 0;
  for (int r0 = 0; r0 < a.Hkv; r0 += 64) {
    int nt = r0 + lane < a.Hkv ? tiles_of(a.len[r0 + lane]) : 0;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) nt += __shfl_xor(nt, d, 64);
    total += nt;
  }
  const int share = part_tiles(total, a.Hkv, a.parts);
  int kv = -1, t0 = 0, t1 = 0, first = 0;
  for (int r0 = 0; r0 < a.Hkv; r0 += 64) {
    const int r = r0 + lane;
    const int nt = r < a.Hkv ? tiles_of(a.len[r]) : 0;
    const int np = (nt + share - 1) / share;
    int incl = np;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(incl, d, 64);
      if (lane >= d) incl += u;
    }
    incl += first;
    if (x == 0 && wave == 0 && r < a.Hkv) {
      a.info[2 * r] = incl - np;
      a.info[2 * r + 1] = np;
    }
    const uint64_t hit = __ballot(part >= incl - np && part < incl);
    if (hit && kv < 0) {
      const int src = __builtin_ctzll(hit);
      kv = r0 + src;
      t0 = (part - __shfl(incl - np, src, 64)) * share;
      t1 = min(t0 + share, __shfl(nt, src, 64));
    }
    first = __shfl(incl, 63, 64);
  }
  kv = __builtin_amdgcn_readfirstlane(kv);
  if (kv < 0) return;
  t0 = __builtin_amdgcn_readfirstlane(t0);
  t1 = __builtin_amdgcn_readfirstlane(t1);
  const int len = a.len[kv];

  // Staging: the tiles lie contiguous in memory and keep their layout in LDS,
  // so a tile is 16-byte units copied straight into LDS (global_load_lds).
  constexpr int kTileBytes = HC_TILE_ELEMS * (int)sizeof(T);
  constexpr int kLoads = kTileBytes / (16 * kPreThreads);  // per thread, of K and of V
  const int64_t at = (a.tile_off[kv] + t0) * (int64_t)kTileBytes + 16 * tid;
  const char* kb = reinterpret_cast<const char*>(a.kstore) + at;
  const char* vb = reinterpret_cast<const char*>(a.vstore) + at;
  // One column group reads a tile once: streamed past L2 (83 against 95 us for
  // 16 columns over 131072 tokens of 8 heads; with more column groups the
  // others' reads come from L2, and 4 of them lose 7 % by the hint).
  const bool once = a.ncg == 1;
  auto stage = [&](int slot) {  // the next tile not staged yet
    char* dst = reinterpret_cast<char*>(lds + slot * 2 * HC_TILE_ELEMS) + 1024 * wave;
    if (once) {
#pragma unroll
      for (int r = 0; r < kLoads; ++r) lds_dma16_stream(kb + 16 * r * kPreThreads, dst + 16 * r * kPreThreads);
#pragma unroll
      for (int r = 0; r < kLoads; ++r)
        lds_dma16_stream(vb + 16 * r * kPreThreads, dst + kTileBytes + 16 * r * kPreThreads);
    } else {
#pragma unroll
      for (int r = 0; r < kLoads; ++r) lds_dma16(kb + 16 * r * kPreThreads, dst + 16 * r * kPreThreads);
#pragma unroll
      for (int r = 0; r < kLoads; ++r) lds_dma16(vb + 16 * r * kPreThreads, dst + kTileBytes + 16 * r * kPreThreads);
    }
    kb += kTileBytes;
    vb += kTileBytes;
  };

  stage(0);
  if (t0 + 1 < t1) stage(1);

  // Q^T operands: column col0 + 16j + n16, k-slots = channels 32s + 8*g4 + [0, 8).
  const int64_t col0 = ((int64_t)cg * kPreWaves + wave) * 16 * NC;
  const bool active = col0 < a.M;
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
  f32x4 o[8][NC];
  float m[NC], l[NC];
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    m[j] = -INFINITY, l[j] = 0.f;
#pragma unroll
    for (int db = 0; db < 8; ++db) o[db][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // The queries and the first tiles travel together; from here on the loop
  // counts its loads in flight.
  wait_lds_dma();
  asm volatile("" ::: "memory");

  int slot = 0;
  for (int t = t0; t < t1; ++t) {
    // This wave's loads of tile t have landed, and past the barrier every
    // wave's have, while tile t + 1 stays in flight; every wave is also done
    // with tile t - 1, whose slot takes tile t + 2.
    if (t + 1 < t1)
      wait_lds_dma_but<2 * kLoads>();
    else
      wait_lds_dma();
    lds_barrier();
    const T* sk = lds + slot * 2 * HC_TILE_ELEMS;
    const T* sv = sk + HC_TILE_ELEMS;
    if (t + 2 < t1) stage(slot == 0 ? 2 : slot - 1);
    slot = slot == kPreRing - 1 ? 0 : slot + 1;
    const int left = len - t * HC_TILE;  // tokens from this tile on
    if (left < HC_TILE) {
      // The row's last tile: its stale slots may hold NaN, which a zero
      // probability does not silence.  (No load is in flight any more.)
      T* z = const_cast<T*>(sv);
      for (int c = tid; c < HC_TILE_ELEMS / 8; c += kPreThreads) {
        vec8 v = load8<T>(z + 8 * c);
        zero_tail<T>(v, 0, left, (c >> 4) & 3);
        *reinterpret_cast<vec8*>(z + 8 * c) = v;
      }
      lds_barrier();
    }
    if (!active) continue;
    // All of a tile's K operands are requested before the first product, and
    // V's before the softmax that they wait behind (left to itself the
    // compiler requests two and waits for both, sixteen times a tile).
    vec8 kv8[8];
#pragma unroll
    for (int x8 = 0; x8 < 8; ++x8) kv8[x8] = load8<T>(sk + (x8 * 64 + lane) * 8);
    __builtin_amdgcn_sched_barrier(0);
    f32x4 s[2][NC];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < NC; ++j) s[h][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x4 = 0; x4 < 4; ++x4)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < NC; ++j) s[h][j] = mma_16x16x32(kv8[h * 4 + x4], qop[j][x4], s[h][j]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x8 = 0; x8 < 8; ++x8) kv8[x8] = load8<T>(sv + (x8 * 64 + lane) * 8);
    __builtin_amdgcn_sched_barrier(0);
    if (left < HC_TILE) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (16 * (e >> 2) + 4 * g4 + (e & 3) >= left) {
#pragma unroll
          for (int j = 0; j < NC; ++j) s[e >> 2][j][e & 3] = -INFINITY;
        }
    }
    vec8 pb[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      float ps;
      auto probs = [&](float nm) {
        float pv[8];
        ps = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          pv[e] = fast_exp2(fmaf(s[e >> 2][j][e & 3], a.scale_log2, nm));
          ps += pv[e];
        }
        pb[j] = pack8<T>(pv);  // at most half a step of the input type per probability
      };
      probs(-m[j]);
      if (__any(!(ps <= kRowsLazy))) {  // also NaN, as in the first tile
        float mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; ++e) mx = fmaxf(mx, s[e >> 2][j][e & 3]);
        const float mnew = fmaxf(m[j], rows4_max(mx) * a.scale_log2);
        const float alpha = m[j] == -INFINITY ? 0.f : fast_exp2(m[j] - mnew);
        m[j] = mnew;
        l[j] *= alpha;
#pragma unroll
        for (int db = 0; db < 8; ++db) o[db][j] *= alpha;
        probs(mnew == -INFINITY ? 0.f : -mnew);
      }
      l[j] += ps;
    }
#pragma unroll
    for (int db = 0; db < 8; ++db) {
#pragma unroll
      for (int j = 0; j < NC; ++j) o[db][j] = mma_16x16x32(kv8[db], pb[j], o[db][j]);
    }
  }

  if (!active) return;
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const float lt = rows4_sum(l[j]);
    const int64_t c = col0 + 16 * j + n16;
    if (c >= a.M) continue;
    const int64_t pa = part * a.M + c;
#pragma unroll
    for (int db = 0; db < 8; ++db)
      *reinterpret_cast<f32x4*>(a.part_o + pa * kPartO + 16 * db + 4 * g4) = o[db][j];
    if (g4 == 0) *reinterpret_cast<float2*>(a.part_ml + pa * 2) = make_float2(m[j], lt);
  }
}

// LDS of a workgroup: the prefix ring, or the row waves' states.
template <typename T>
constexpr size_t shared_lds() {
  const size_t ring = (size_t)kPreRing * 2 * HC_TILE_ELEMS * sizeof(T), rows = kRowsLds * sizeof(float);
  return ring > rows ? ring : rows;
}

// Prefix workgroups come first: they are the long ones.
template <typename T, int NC, bool MIXED>
__global__ __launch_bounds__(kPreThreads, sizeof(T) == 4 ? 1 : 3) void shared_attn_kernel(const PrefixArgs pre,
                                                                                         const RowsArgs rows) {
  extern __shared__ __attribute__((aligned(16))) unsigned char shared_raw[];
  const int npre = pre.parts * pre.ncg;
  if ((int)blockIdx.x < npre)
    prefix_job<T, NC>(pre, blockIdx.x, reinterpret_cast<T*>(shared_raw));
  else
    rows_job<T, kRowsWhole, MIXED, kPreWaves>(rows, blockIdx.x - npre, reinterpret_cast<float*>(shared_raw));
}

// Sizes of one call: the prefix launch's column blocks and parts, the rows'
// plan, and the workspace in bytes.
struct SharedPlan {
  int nc, ncg, parts;
  RowsPlan rows;
  size_t info_at, pre_o, pre_ml, row_o, row_ml, bytes;
};

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

SharedPlan shared_plan(int dtype, int batch, int Hkv, int G, int Q, int64_t prefix_tiles, int64_t row_tiles) {
  SharedPlan p;
  const int64_t M = (int64_t)batch * Q * G;
  p.nc = dtype != HC_DTYPE_F32 && M > 64 ? 2 : 1;
  const int64_t per = 64 * p.nc;
  p.ncg = (int)((M + per - 1) / per);
  p.rows = rows_plan(batch * Hkv, G, Q, row_tiles);
  // Prefix workgroups a CU: the least estimate of the two launches' time in
  // us.  A part's tile of 32 tokens takes 0.6 + 0.37 k with k workgroups of
  // two column blocks a wave on a CU (128, 512 and 768 workgroups over 128K
  // tokens: 330, 217 and 195 us against 327, 226 and 192), or the stream's
  // time; a column's partial costs its writing and reading; the rows' stream
  // hides behind the products while a third workgroup finds room (1024 rows
  // beside 512 columns over 128K: 260, 253 and 278 us at k = 2, 2.5 and 3).
  const int cus = device_cus();
  const bool f32 = dtype == HC_DTYPE_F32;
  const double stream = 2e6 * HC_TILE_ELEMS * (f32 ? 4. : 2.) / 5.8e12;
  const double rows_us = 0.75 * (double)batch * Hkv * row_tiles * stream;
  const double ks[] = {0.125, 0.25, 0.5, 1., 1.5, 2., 2.5, 3.};
  int64_t parts = 0;
  double best = 0.;
  for (const double k : ks) {
    if (f32 && k > 1.) break;  // LDS holds one workgroup
    // Every KV head has two parts at least, and there are no more than tiles.
    int64_t n = std::max<int64_t>((int64_t)(k * cus) / p.ncg, 2 * (int64_t)Hkv);
    n = std::min(n, prefix_tiles + Hkv + 1);
    const double kk = std::max((double)n * p.ncg / cus, 1.);
    const double tile = f32 ? 3. : p.nc == 1 ? 0.5 + 0.2 * kk : 0.6 + 0.37 * kk;
    const double share = std::ceil((double)prefix_tiles / (double)std::max<int64_t>(n - Hkv / 2, 1));
    const double t = std::max(share * tile, prefix_tiles * stream) + (double)n * M * 520. * 0.45e-6 +
                     rows_us * (f32 || kk > 2.75 ? 0.9 : kk > 2.25 ? 0.5 : 0.35);
    if (parts == 0 || t < best) best = t, parts = n;
  }
  p.parts = (int)std::min<int64_t>((parts + 7) / 8 * 8, 1 << 20);  // whole rounds over the 8 XCDs
  const size_t pre = (size_t)p.parts * M, row = (size_t)batch * Hkv * Q * G * p.rows.nsplit;
  p.info_at = 0;
  p.pre_o = up256((size_t)Hkv * 2 * sizeof(int32_t));
  p.pre_ml = p.pre_o + up256(pre * kPartO * sizeof(float));
  p.row_o = p.pre_ml + up256(pre * 2 * sizeof(float));
  p.row_ml = p.row_o + up256(row * kPartO * sizeof(float));
  p.bytes = p.row_ml + up256(row * 2 * sizeof(float));
  return p;
}

template <typename T>
int launch_shared(const PrefixArgs& a, const RowsArgs& r, int nc, hipStream_t s) {
  const size_t lds = shared_lds<T>();
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
  if (bad_sizes(dtype, batch, q_heads, kv_heads, queries) || prefix_tiles < 0 || row_tiles < 0) return 0;
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
  if (bad_sizes(dtype, batch, q_heads, kv_heads, queries) || prefix_tiles < 0 || row_tiles < 0)
    return set_error(HC_ERR_INVALID,
                     "hc_shared_attn: dtype=%d batch=%d q_heads=%d kv_heads=%d queries=%d (q_heads a multiple of "
                     "kv_heads, at most 16 of it, at most 2^24 query rows)",
                     dtype, batch, q_heads, kv_heads, queries);
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
  const SharedPlan p = shared_plan(dtype, batch, kv_heads, G, queries, prefix_tiles, row_tiles);
  if (!workspace || workspace_bytes < p.bytes)
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
  r.q = q, r.kstore = kstore, r.vstore = vstore, r.row_tile_off = row_tile_off, r.row_len = row_len, r.query_counts = query_counts;
  r.Hkv = kv_heads, r.G = G, r.Q = queries, r.rows = row_len ? batch * kv_heads : 0;
  r.qpb = p.rows.qpb, r.ncb = p.rows.ncb, r.nsplit = p.rows.nsplit, r.scale_log2 = scale_log2;
  r.part_o = reinterpret_cast<float*>(ws + p.row_o), r.part_ml = reinterpret_cast<float*>(ws + p.row_ml);
  for (int i = 0; i < 3; ++i) a.q_s[i] = r.q_s[i] = q_strides[i];
  const int rc = dtype == HC_DTYPE_BF16  ? launch_shared<__bf16>(a, r, p.nc, s)
                 : dtype == HC_DTYPE_F16 ? launch_shared<_Float16>(a, r, p.nc, s)
                                         : launch_shared<float>(a, r, p.nc, s);
  if (rc) return rc;
  return launch_merge(dtype, mg, (int64_t)batch * queries * q_heads, s);
}
