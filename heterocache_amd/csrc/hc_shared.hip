// Attention of a batch over one shared prefix and each sequence's own rows.
//
//   out[b, i, h] = softmax over the tokens of prefix row kv(h) and the visible
//   tokens of row (b, kv(h)), times their values; query i of Q sees the
//   row's tokens t < len - Q + 1 + i.
//
// Both parts lie in ragged tiled stores; the prefix has one row per KV head,
// of its own length (a document compressed per head, or whole).  Softmax over
// the union is folded from partial states (m, l, O), so the prefix is read
// once for all sequences:
//  * prefix_attn_kernel: the batch * Q * G query rows of a KV head are the
//    columns of the products S^T = K Q^T and O^T += V^T P^T over a part of
//    the prefix; a workgroup's 4 waves x NC x 16 columns share every tile
//    through LDS.
//  * rows_attn_kernel (hc_rows.hip): each sequence's own rows.
//  * merge_kernel (hc_rows.hip): one fold of a column's partials.
#include <algorithm>
#include <cmath>

#include "hc_rows.h"

namespace hc {
namespace {

constexpr int kPreWaves = 4;
constexpr int kPreThreads = kPreWaves * 64;
constexpr int kPreTiles = 2;  // tiles an iteration
constexpr int kPreKeys = kPreTiles * HC_TILE;

struct PrefixArgs {
  const void* q;
  int64_t q_s[3];
  const void *kstore, *vstore;
  const int64_t* tile_off;
  const int32_t* len;
  int Hkv, G, Q;
  int64_t M;   // columns: batch * Q * G
  int ncg;     // column groups of 64 * NC
  int parts;   // workgroups of a column group
  float scale_log2;
  float *part_o, *part_ml;
  int32_t* info;
};

// Iterations a part takes so that every row is covered by at most `parts`
// parts in all: each row's last part may be short, so the shares are cut from
// the parts left when every row has one.
__device__ __forceinline__ int part_iterations(int64_t total, int rows, int parts) {
  const int64_t n = max(parts - rows, 1);
  return (int)max((total + n - 1) / n, (int64_t)1);
}

// Lane state of one 16-column block over LDS-staged tiles; see attend_rows.
template <typename T, int NC>
__global__ __launch_bounds__(kPreThreads, sizeof(T) == 4 ? 1 : 3) void prefix_attn_kernel(const PrefixArgs a) {
  typedef typename Elem<T>::vec8 vec8;
  extern __shared__ __attribute__((aligned(16))) unsigned char pre_lds[];
  T* lds = reinterpret_cast<T*>(pre_lds);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g4 = lane >> 4, n16 = lane & 15;

  // Column groups of one part go to one XCD (workgroups are dealt to the 8
  // XCDs in turn), so its L2 serves the tiles after their first read.
  const int x = blockIdx.x;
  const int part = (x / (8 * a.ncg)) * 8 + x % 8, cg = (x / 8) % a.ncg;

  // (row, share) of the part, from the device lengths: rows 64 at a time.
  int64_t total = 0;
  for (int r0 = 0; r0 < a.Hkv; r0 += 64) {
    int it = r0 + lane < a.Hkv ? (max(a.len[r0 + lane], 0) + kPreKeys - 1) / kPreKeys : 0;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) it += __shfl_xor(it, d, 64);
    total += it;
  }
  const int share = part_iterations(total, a.Hkv, a.parts);
  int kv = -1, it0 = 0, nit = 0, first = 0;
  for (int r0 = 0; r0 < a.Hkv; r0 += 64) {
    const int r = r0 + lane;
    const int it = r < a.Hkv ? (max(a.len[r], 0) + kPreKeys - 1) / kPreKeys : 0;
    const int np = (it + share - 1) / share;
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
      it0 = (part - __shfl(incl - np, src, 64)) * share;
      nit = min(it0 + share, __shfl(it, src, 64));
    }
    first = __shfl(incl, 63, 64);
  }
  kv = __builtin_amdgcn_readfirstlane(kv);
  if (kv < 0) return;
  it0 = __builtin_amdgcn_readfirstlane(it0);
  nit = __builtin_amdgcn_readfirstlane(nit);
  const int len = a.len[kv], last_tile = (len - 1) / HC_TILE;

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

  // Staging: the tiles lie contiguous in memory and keep their layout in LDS,
  // so an iteration is 16-byte units copied straight into LDS
  // (global_load_lds): unit r * 256 + tid.  A tile past the row's last one
  // reads the last one again; its tokens are masked.
  constexpr int kUnits = (int)sizeof(T) / 2;       // 16-byte units per 8 elements
  constexpr int kPerTile = 2 * kUnits;             // units of a tile per thread
  constexpr int kTileBytes = HC_TILE_ELEMS * (int)sizeof(T);
  const int64_t row_at = a.tile_off[kv] * (int64_t)kTileBytes + 16 * tid;
  const char* kb = reinterpret_cast<const char*>(a.kstore) + row_at;
  const char* vb = reinterpret_cast<const char*>(a.vstore) + row_at;
  T* const vbuf = lds + 2 * kPreTiles * HC_TILE_ELEMS;
  auto stage = [&](const char* src, T* dst, int it) {
#pragma unroll
    for (int c = 0; c < kPreTiles; ++c) {
      const char* t = src + (int64_t)min(it * kPreTiles + c, last_tile) * kTileBytes;
#pragma unroll
      for (int r = 0; r < kPerTile; ++r)
        lds_dma16(t + 16 * r * kPreThreads,
                  reinterpret_cast<char*>(dst) + c * kTileBytes + 16 * (r * kPreThreads + wave * 64));
    }
  };

  stage(kb, lds, it0);
  stage(vb, vbuf, it0);
  wait_lds_dma();
  __syncthreads();

  // K is double-buffered; V(it + 1) is fetched behind the P.V step of it and
  // arrives while the next scores and probabilities are formed.
  for (int it = it0; it < nit; ++it) {
    const int cur = (it - it0) & 1;
    const int t0 = it * kPreKeys;
    const bool more = it + 1 < nit;
    if (more) stage(kb, lds + (cur ^ 1) * kPreTiles * HC_TILE_ELEMS, it + 1);
    vec8 pb[kPreTiles][NC];
    if (active) {
      const T* sk = lds + cur * kPreTiles * HC_TILE_ELEMS;
      f32x4 sacc[4][NC];
#pragma unroll
      for (int tb = 0; tb < 4; ++tb)
#pragma unroll
        for (int j = 0; j < NC; ++j) sacc[tb][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int tb = 0; tb < 4; ++tb) {
        const T* kt = sk + (tb >> 1) * HC_TILE_ELEMS + (tb & 1) * 4 * 64 * 8;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const vec8 ka = load8<T>(kt + (s * 64 + lane) * 8);
#pragma unroll
          for (int j = 0; j < NC; ++j) sacc[tb][j] = mma_16x16x32(ka, qop[j][s], sacc[tb][j]);
        }
      }
      if (t0 + kPreKeys > len) {
#pragma unroll
        for (int tb = 0; tb < 4; ++tb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (t0 + 16 * tb + 4 * g4 + r >= len) {
#pragma unroll
              for (int j = 0; j < NC; ++j) sacc[tb][j][r] = -INFINITY;
            }
      }
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        float ps;
        auto probs = [&](float nm) {
          ps = 0.f;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float pv[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              pv[e] = fast_exp2(fmaf(sacc[2 * c + (e >> 2)][j][e & 3], a.scale_log2, nm));
              ps += pv[e];
            }
            pb[c][j] = pack8<T>(pv);  // at most half a step of the input type per probability
          }
        };
        probs(-m[j]);
        if (__any(!(ps <= kRowsLazy))) {  // also NaN, as in the first iteration
          float mx = -INFINITY;
#pragma unroll
          for (int tb = 0; tb < 4; ++tb)
#pragma unroll
            for (int r = 0; r < 4; ++r) mx = fmaxf(mx, sacc[tb][j][r]);
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
    }
    // V(it) was fetched before K(it + 1).
    if (more)
      wait_lds_dma_but<kPreTiles * kPerTile>();
    else
      wait_lds_dma();
    __syncthreads();
    if (active) {
      const bool tail = t0 + kPreKeys > len;
#pragma unroll
      for (int c = 0; c < kPreTiles; ++c) {
        const T* vt = vbuf + c * HC_TILE_ELEMS;
#pragma unroll
        for (int db = 0; db < 8; ++db) {
          vec8 va = load8<T>(vt + (db * 64 + lane) * 8);
          // Stale slots may hold NaN, which zero probabilities do not silence.
          if (tail) zero_tail<T>(va, t0 + c * HC_TILE, len, g4);
#pragma unroll
          for (int j = 0; j < NC; ++j) o[db][j] = mma_16x16x32(va, pb[c][j], o[db][j]);
        }
      }
    }
    wait_lds_dma();   // K(it + 1) has landed
    __syncthreads();  // ... and V(it) is no longer read
    if (more) stage(vb, vbuf, it + 1);
  }

  if (!active) return;
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const float lt = rows4_sum(l[j]);
    const int64_t c = col0 + 16 * j + n16;
    if (c >= a.M) continue;
    const int64_t at = part * a.M + c;
#pragma unroll
    for (int db = 0; db < 8; ++db)
      *reinterpret_cast<f32x4*>(a.part_o + at * kPartO + 16 * db + 4 * g4) = o[db][j];
    if (g4 == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(m[j], lt);
  }
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
  // Three workgroups a CU (one in fp32), every KV head at least two parts,
  // and no more parts than iterations.
  const int64_t slots = (int64_t)device_cus() * (dtype == HC_DTYPE_F32 ? 1 : 3);
  int64_t parts = std::max<int64_t>(slots / p.ncg, 2 * (int64_t)Hkv);
  parts = std::min(parts, prefix_tiles + Hkv + 1);
  p.parts = (int)std::min<int64_t>((parts + 7) / 8 * 8, 1 << 20);  // whole rounds over the 8 XCDs
  p.rows = rows_plan(batch * Hkv, G, Q, row_tiles);
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
int launch_prefix(const PrefixArgs& a, int nc, hipStream_t s) {
  const size_t lds = (size_t)3 * kPreTiles * HC_TILE_ELEMS * sizeof(T);
  auto fn = prefix_attn_kernel<T, 1>;
  if constexpr (sizeof(T) == 2)
    if (nc == 2) fn = prefix_attn_kernel<T, 2>;
  if (lds > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)lds) != hipSuccess)
    return set_error(HC_ERR_HIP, "hc_shared_attn: %s", hipGetErrorString(hipGetLastError()));
  const int64_t grid = (int64_t)a.parts * a.ncg;
  if (grid > 0x7fffffffLL) return set_error(HC_ERR_INVALID, "hc_shared_attn: %lld workgroups", (long long)grid);
  hipLaunchKernelGGL(fn, dim3((unsigned)grid), dim3(kPreThreads), lds, s, a);
  return check_launch("hc_shared_attn(prefix)");
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
                              const int64_t* row_tile_off, const int32_t* row_len, int64_t row_tiles, void* out,
                              const int64_t* out_strides, int batch, int q_heads, int kv_heads, int queries,
                              float scale, void* workspace, size_t workspace_bytes, void* stream) {
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
  if (prefix_len) {
    PrefixArgs a;
    a.q = q, a.kstore = kprefix, a.vstore = vprefix, a.tile_off = prefix_tile_off, a.len = prefix_len;
    for (int i = 0; i < 3; ++i) a.q_s[i] = q_strides[i];
    a.Hkv = kv_heads, a.G = G, a.Q = queries, a.M = mg.M, a.ncg = p.ncg, a.parts = p.parts;
    a.scale_log2 = scale_log2;
    a.part_o = reinterpret_cast<float*>(ws + p.pre_o), a.part_ml = reinterpret_cast<float*>(ws + p.pre_ml);
    a.info = reinterpret_cast<int32_t*>(ws + p.info_at);
    const int rc = dtype == HC_DTYPE_BF16  ? launch_prefix<__bf16>(a, p.nc, s)
                   : dtype == HC_DTYPE_F16 ? launch_prefix<_Float16>(a, p.nc, s)
                                           : launch_prefix<float>(a, p.nc, s);
    if (rc) return rc;
  }
  if (row_len) {
    RowsArgs r = {};
    r.q = q, r.kstore = kstore, r.vstore = vstore, r.row_tile_off = row_tile_off, r.row_len = row_len;
    for (int i = 0; i < 3; ++i) r.q_s[i] = q_strides[i];
    r.Hkv = kv_heads, r.G = G, r.Q = queries, r.rows = batch * kv_heads;
    r.qpb = p.rows.qpb, r.ncb = p.rows.ncb, r.nsplit = p.rows.nsplit, r.scale_log2 = scale_log2;
    r.part_o = reinterpret_cast<float*>(ws + p.row_o), r.part_ml = reinterpret_cast<float*>(ws + p.row_ml);
    const int rc = launch_rows_attn(dtype, r, s);
    if (rc) return rc;
  }
  return launch_merge(dtype, mg, (int64_t)batch * queries * q_heads, s);
}
