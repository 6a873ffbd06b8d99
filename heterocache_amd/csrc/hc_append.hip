// Rotated append: new queries and keys turned by their positions, keys and
// values stored into the tiles of the ragged store, in one pass over them.
//
//   x'[d]      = x[d] cos[d] - x[d + 64] sin[d]             d < 64
//   x'[d + 64] = x[d + 64] cos[d + 64] + x[d] sin[d + 64]
//
// for every query and key (the rotate-half form of the models), formed in
// fp32 and rounded once to the tensors' type, then
//   store[b, h][len + t] = (k'[b, h, t], v[b, h, t]),  t < counts[b].
//
// Bound by HBM: each element is read once and written once, and the tables
// are read once per KV head (from L2: the workgroups of a token share them).
// A workgroup takes the new tokens of one row that fall into one 32-token
// tile, with the queries of the row's head group at the same tokens: a thread
// keeps the table values of its (token, 8 + 8 channels) over the group's heads
// and the key, four heads' loads in flight, and each 8-token x 8-channel-chunk
// store of a wave fills whole 128-byte lines of the K tile.  V's tile layout
// keeps 8 tokens of a channel together, so a whole tile goes through LDS; the
// tokens of a partly covered tile are stored one element at a time (the other
// tokens of its 16-byte chunks may be older ones, or not yet written).
// 32768 tokens of 32 + 2 x 8 heads in bf16: 151 us, 5.4 TB/s read and written.
#include "hc_common.h"
#include "hc_internal.h"

namespace hc {
namespace {

struct RotArgs {
  const void *q, *k, *v, *cos, *sin;
  void *qo, *kstore, *vstore;
  int64_t q_s[3], qo_s[3], k_s[3], v_s[3];  // element strides: batch, head, token
  int64_t t_sb, t_st;                       // tables: batch, token
  const int64_t* row_tile_off;
  const int32_t *row_len, *row_cap, *counts;
  int32_t *len_out, *status;
  int Hkv, G, T, rows, tiles;  // tiles: workgroups of a row (walk = 0)
  int walk;                    // one workgroup walks a row's tiles and writes its length
  int advance;                 // len_out is written by this launch
};


// Eight table values as fp32.
template <typename C>
__device__ __forceinline__ void load_table(const C* p, float (&x)[8]) {
  const typename Elem<C>::vec8 r = load8<C>(p);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = vec8_at<C>(r, e);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  *reinterpret_cast<typename Elem<T>::vec8*>(p) = pack8<T>(x);
}

template <typename T, typename C, int NT>
__global__ __launch_bounds__(NT, sizeof(T) == 4 ? 2 : 4) void append_rotated_kernel(const RotArgs a) {
  typedef typename Elem<T>::vec8 vec8;
  __shared__ T sv[NT == 256 ? HC_TILE : 1][HC_HEAD_DIM + 8];
  const int row = blockIdx.x % a.rows;
  const int b = row / a.Hkv, h = row % a.Hkv;
  const int tid = threadIdx.x;
  const int len = a.row_len[row];
  const int cnt = a.counts ? min(max(a.counts[b], 0), a.T) : a.T;
  // A row without room for its tokens is left as it is; its queries are turned.
  const bool room = len >= 0 && (int64_t)len + cnt <= a.row_cap[row];
  const int first = len & (HC_TILE - 1);          // slot of the first new token in its tile
  const int ntiles = (first + a.T + HC_TILE - 1) / HC_TILE;
  const T* qp = reinterpret_cast<const T*>(a.q) + b * a.q_s[0] + (int64_t)h * a.G * a.q_s[1];
  T* qo = reinterpret_cast<T*>(a.qo) + b * a.qo_s[0] + (int64_t)h * a.G * a.qo_s[1];
  const T* kp = reinterpret_cast<const T*>(a.k) + b * a.k_s[0] + h * a.k_s[1];
  const T* vp = reinterpret_cast<const T*>(a.v) + b * a.v_s[0] + h * a.v_s[1];
  const C* cp = reinterpret_cast<const C*>(a.cos) + b * a.t_sb;
  const C* sp = reinterpret_cast<const C*>(a.sin) + b * a.t_sb;
  const int64_t tile0 = a.row_tile_off[row] + len / HC_TILE;

  int j = a.walk ? 0 : blockIdx.x / a.rows;
  const int jend = a.walk ? ntiles : min(j + 1, ntiles);
  for (; j < jend; ++j) {
    // Tokens [ta, tb) of the call lie in tile j of the row's new ones;
    // [ta, ts) of them are stored.
    const int ta = max(j * HC_TILE - first, 0), tb = min((j + 1) * HC_TILE - first, a.T);
    const int n = tb - ta;
    const int ts = room ? min(tb, cnt) : ta;
    const int nst = max(ts - ta, 0);
    const int slot0 = (first + ta) & (HC_TILE - 1);
    T* kt = reinterpret_cast<T*>(a.kstore) + (tile0 + j) * (int64_t)HC_TILE_ELEMS;
    T* vt = reinterpret_cast<T*>(a.vstore) + (tile0 + j) * (int64_t)HC_TILE_ELEMS;
    const bool whole = NT == 256 && nst == HC_TILE;

    // V: chunk x = (token, 8 channels), two per thread (one token: one, of 16
    // threads).
    vec8 vr[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int x = tid + u * NT, t = x >> 4;
      if (t < nst) vr[u] = load8_stream<T>(vp + (int64_t)(ta + t) * a.v_s[2] + 8 * (x & 15));
    }

    // Q and K: eight threads a token and head; head G is the key.  A thread
    // stays with one token, so its 8 + 8 channels' table values are read once,
    // and takes every hp-th head (hp: how often the tile's tokens fit the
    // groups of 8 threads), kBatch of them in flight.
    constexpr int kBatch = 4;
    const int grp = tid >> 3, c0 = 8 * (tid & 7);
    const int hp = n > 0 ? NT / 8 / n : 0, h0 = n > 0 ? grp / n : 0;
    if (h0 < hp) {
      const int t = grp % n;
      const int64_t tok = ta + t;
      const T* const qs = qp + tok * a.q_s[2] + c0;
      const T* const ks = kp + tok * a.k_s[2] + c0;
      const C* const cs = cp + tok * a.t_st + c0;
      const C* const ss = sp + tok * a.t_st + c0;
      float cc[2][8], sn[2][8];
      load_table<C>(cs, cc[0]);
      load_table<C>(cs + 64, cc[1]);
      load_table<C>(ss, sn[0]);
      load_table<C>(ss + 64, sn[1]);
      for (int hb = 0; hb <= a.G; hb += kBatch * hp) {
        vec8 lo8[kBatch], hi8[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          if (hb + u * hp > a.G) continue;
          const int hd = hb + u * hp + h0;  // past the key: the key again, not stored
          const T* src = hd < a.G ? qs + hd * a.q_s[1] : ks;
          lo8[u] = load8_stream<T>(src), hi8[u] = load8_stream<T>(src + 64);
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          if (hb + u * hp > a.G) continue;
          const int hd = hb + u * hp + h0;
          float lo[8], hi[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x = vec8_at<T>(lo8[u], e), y = vec8_at<T>(hi8[u], e);
            lo[e] = x * cc[0][e] - y * sn[0][e];
            hi[e] = y * cc[1][e] + x * sn[1][e];
          }
          if (hd < a.G) {
            T* o = qo + hd * a.qo_s[1] + tok * a.qo_s[2] + c0;
            store8<T>(o, lo);
            store8<T>(o + 64, hi);
          } else if (hd == a.G && t < nst) {
            store8<T>(kt + k_tile_offset(slot0 + t, c0), lo);
            store8<T>(kt + k_tile_offset(slot0 + t, c0 + 64), hi);
          }
        }
      }
    }

    if (whole) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int x = tid + u * NT;
        *reinterpret_cast<vec8*>(&sv[x >> 4][8 * (x & 15)]) = vr[u];
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        // V chunk x = (mt*4+g)*16+nn: channel 16mt+nn, tokens 16*(i/4)+4g+i%4.
        const int x = tid + u * NT;
        const int nn = x & 15, g = (x >> 4) & 3, d = 16 * (x >> 6) + nn;
        float v8[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v8[i] = Elem<T>::to_f32(sv[16 * (i >> 2) + 4 * g + (i & 3)][d]);
        store8<T>(vt + 8 * x, v8);
      }
      __syncthreads();  // the next tile refills the buffer
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int x = tid + u * NT, t = x >> 4;
        if (t < nst) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            vt[v_tile_offset(slot0 + t, 8 * (x & 15) + e)] = Elem<T>::from_f32(vec8_at<T>(vr[u], e));
        }
      }
    }
  }

  if (a.walk || blockIdx.x / a.rows == 0) {
    if (a.walk) __syncthreads();  // every thread has read the length that may be overwritten
    if (tid == 0) {
      if (!room && a.status) atomicOr(a.status, 1);
      if (a.advance) a.len_out[row] = room ? len + cnt : len;
    }
  }
}

// Lengths advanced in place after a launch whose workgroups all read them.
__global__ __launch_bounds__(256) void advance_kernel(int32_t* __restrict__ row_len,
                                                      const int32_t* __restrict__ row_cap,
                                                      const int32_t* __restrict__ counts, int Hkv, int T, int rows) {
  const int row = blockIdx.x * 256 + threadIdx.x;
  if (row >= rows) return;
  const int cnt = counts ? min(max(counts[row / Hkv], 0), T) : T;
  const int len = row_len[row];
  if (len >= 0 && (int64_t)len + cnt <= row_cap[row]) row_len[row] = len + cnt;
}

template <typename T, typename C>
int launch_rotated(RotArgs& a, hipStream_t s) {
  // In place, a row's length may be written once its workgroups have read
  // it: up to 32 tokens (two tiles at most) one workgroup walks the row,
  // longer calls advance the lengths in a launch of their own.
  const bool in_place = a.len_out == a.row_len;
  a.walk = in_place && a.T <= HC_TILE;
  a.advance = a.len_out && (!in_place || a.walk);
  a.tiles = a.walk ? 1 : (a.T + 2 * HC_TILE - 2) / HC_TILE;
  const int64_t grid = (int64_t)a.tiles * a.rows;
  if (grid > 0x7fffffffLL) return set_error(HC_ERR_INVALID, "hc_append_rotated: %d rows x %d tokens", a.rows, a.T);
  // One token of many rows: a wave a row, whose eight groups of threads take the
  // heads, leaves room for all rows at once (2048 rows 6.4 against 10.2 us; 8
  // rows 4.8 against 4.4).
  if (a.T == 1 && a.rows > 512)
    hipLaunchKernelGGL((append_rotated_kernel<T, C, 64>), dim3((unsigned)grid), dim3(64), 0, s, a);
  else
    hipLaunchKernelGGL((append_rotated_kernel<T, C, 256>), dim3((unsigned)grid), dim3(256), 0, s, a);
  int rc = check_launch("hc_append_rotated");
  if (rc || !a.len_out || a.advance) return rc;
  hipLaunchKernelGGL(advance_kernel, dim3((a.rows + 255) / 256), dim3(256), 0, s, a.len_out, a.row_cap, a.counts,
                     a.Hkv, a.T, a.rows);
  return check_launch("hc_append_rotated(lengths)");
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace hc

using namespace hc;

extern "C" int hc_append_rotated(int dtype, int table_dtype, const void* q, const int64_t* q_strides, void* q_out,
                                 const int64_t* q_out_strides, const void* k, const int64_t* k_strides, const void* v,
                                 const int64_t* v_strides, const void* cos, const void* sin, int64_t table_batch_stride,
                                 int64_t table_tok_stride, void* kstore, void* vstore, const int64_t* row_tile_off,
                                 const int32_t* row_len, const int32_t* row_cap, int32_t* len_out,
                                 const int32_t* counts, int batch, int q_heads, int kv_heads, int tokens,
                                 int32_t* status, void* stream) {
  clear_error();
  if (batch < 0 || tokens < 0 || kv_heads < 1 || q_heads < 1 || q_heads % kv_heads ||
      (int64_t)batch * kv_heads > 0x7fffffffLL || tokens > 0x7fffffff - 2 * HC_TILE)
    return set_error(HC_ERR_INVALID, "hc_append_rotated: batch=%d q_heads=%d kv_heads=%d tokens=%d", batch, q_heads,
                     kv_heads, tokens);
  if (dtype != HC_DTYPE_BF16 && dtype != HC_DTYPE_F16 && dtype != HC_DTYPE_F32)
    return set_error(HC_ERR_INVALID, "hc_append_rotated: unknown dtype %d", dtype);
  if (table_dtype != dtype && table_dtype != HC_DTYPE_F32)
    return set_error(HC_ERR_INVALID, "hc_append_rotated: the tables' dtype %d is neither float32 nor %d", table_dtype,
                     dtype);
  if (batch == 0) return HC_OK;
  if (!row_len || (len_out && (!row_cap || !row_tile_off)))
    return set_error(HC_ERR_INVALID, "hc_append_rotated: null pointer argument");
  if (tokens == 0 && (!len_out || len_out == row_len)) return HC_OK;
  const int64_t gap = 4 * (int64_t)batch * kv_heads;
  const intptr_t apart = reinterpret_cast<intptr_t>(len_out) - reinterpret_cast<intptr_t>(row_len);
  if (len_out && apart != 0 && apart > -gap && apart < gap)
    return set_error(HC_ERR_INVALID, "hc_append_rotated: len_out overlaps row_len without being it");
  if (!q_strides || !q_out_strides || !k_strides || !v_strides)
    return set_error(HC_ERR_INVALID, "hc_append_rotated: null strides");
  if (tokens > 0 && (!q || !q_out || !k || !v || !cos || !sin || !kstore || !vstore || !row_tile_off || !row_cap))
    return set_error(HC_ERR_INVALID, "hc_append_rotated: null pointer argument");
  const int per16 = dtype == HC_DTYPE_F32 ? 4 : 8, tper16 = table_dtype == HC_DTYPE_F32 ? 4 : 8;
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] % per16 || q_out_strides[i] % per16 || k_strides[i] % per16 || v_strides[i] % per16)
      return set_error(HC_ERR_INVALID, "hc_append_rotated: strides must be multiples of 16 bytes");
  if (table_batch_stride % tper16 || table_tok_stride % tper16)
    return set_error(HC_ERR_INVALID, "hc_append_rotated: table strides must be multiples of 16 bytes");
  if (!aligned16(q) || !aligned16(q_out) || !aligned16(k) || !aligned16(v) || !aligned16(cos) || !aligned16(sin) ||
      !aligned16(kstore) || !aligned16(vstore))
    return set_error(HC_ERR_INVALID, "hc_append_rotated: tensors must be 16-byte aligned");
  RotArgs a;
  a.q = q, a.k = k, a.v = v, a.cos = cos, a.sin = sin, a.qo = q_out, a.kstore = kstore, a.vstore = vstore;
  for (int i = 0; i < 3; ++i)
    a.q_s[i] = q_strides[i], a.qo_s[i] = q_out_strides[i], a.k_s[i] = k_strides[i], a.v_s[i] = v_strides[i];
  a.t_sb = table_batch_stride, a.t_st = table_tok_stride;
  a.row_tile_off = row_tile_off, a.row_len = row_len, a.row_cap = row_cap, a.counts = counts;
  a.len_out = len_out, a.status = status;
  a.Hkv = kv_heads, a.G = q_heads / kv_heads, a.T = tokens, a.rows = batch * kv_heads;
  hipStream_t s = (hipStream_t)stream;
  const bool f32t = table_dtype == HC_DTYPE_F32;
  switch (dtype) {
    case HC_DTYPE_BF16: return f32t ? launch_rotated<__bf16, float>(a, s) : launch_rotated<__bf16, __bf16>(a, s);
    case HC_DTYPE_F16: return f32t ? launch_rotated<_Float16, float>(a, s) : launch_rotated<_Float16, _Float16>(a, s);
    default: return launch_rotated<float, float>(a, s);
  }
}
