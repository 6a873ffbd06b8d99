// Building blocks of the kernels over a paged cache.
//
// Pools K and V of pages [pages][page tokens][heads][128] (any strides of whole
// 16 bytes) hold the tokens of table rows: token t of table row r lies in page
// table[r][t / page tokens], at place t % page tokens.  A table row serves one
// (sequence, KV head) row, or all KV heads of a sequence.
//
// Tiles of 32 tokens are copied into LDS token by token, a token's channels in
// chunks of 16 bytes; chunk c of token t lies at place c ^ swizzle(t), so that
// the 16 keys of a matrix operand, and the 8 x 2 chunks of a transposed read of
// values, fall on different banks.
#pragma once
#include "hc_rows.h"

namespace hc {

// n workgroups in as many launches as HIP takes fewer than 2^32 threads each:
// one, but for the largest calls.  launch(grid, group0); the kernels' workgroup is
// group0 + blockIdx.x.  (Layers along z instead cost every call 0.2-0.4 us.)
constexpr int64_t kMostGroups = 0x7fffffff;
template <typename F>
inline int in_launches(int64_t n, int threads, F launch) {
  const int64_t most = ((int64_t)1 << 31) / threads;  // (whole turns of the XCDs)
  int rc = HC_OK;
  for (int64_t first = 0; first < n && rc == HC_OK; first += most)
    rc = launch(dim3((unsigned)(n - first < most ? n - first : most)), (uint32_t)first);
  return rc;
}

struct Pool {
  const char *k, *v;
  int64_t k_page, k_tok, k_head, v_page, v_tok, v_head;  // byte strides
  const int32_t* table;
  int64_t table_stride;
  const int32_t* row_len;
  const int32_t* counts;  // new tokens (queries) a sequence, or null: Q
  int32_t* status;
  uint32_t div_mul;  // t / page_tokens = (t * div_mul) >> div_shift for t < 2^31
  int div_shift;
  int page_tokens, pages, capacity;  // capacity: tokens of a table row
  int heads, Hkv, rows, Q;           // rows = batch * Hkv
  int fresh;                         // the Q tokens are appended by this call
};

__device__ __forceinline__ int page_of(const Pool& p, int t) {
  return (int)(((uint64_t)(uint32_t)t * p.div_mul) >> p.div_shift);
}

// Lengths of a row in this call: tokens before it, after it, and of the latter
// the first n queries' own, the last n.  A row without room for its new tokens
// keeps its old ones and attends nothing.
struct RowSpan {
  int len, total, n;
  bool room;
};
__device__ __forceinline__ int table_row(const Pool& p, int row) { return p.heads == 1 ? row : row / p.Hkv; }
__device__ __forceinline__ RowSpan row_span(const Pool& p, int row) {
  RowSpan s;
  const int len = p.row_len[table_row(p, row)];
  s.n = query_tokens(p.counts, row / p.Hkv, p.Q);
  s.len = min(max(len, 0), p.capacity);
  s.room = !p.fresh || (len >= 0 && (int64_t)len + s.n <= p.capacity);
  s.total = p.fresh && s.room ? s.len + s.n : s.len;
  return s;
}

// Workgroups a row that add up the weights of few columns, and a launch's that folds many.
inline int paged_weigh_runs(const Pool& p) {
  const int most = 2048 / p.rows, runs = (p.capacity + 1023) / 1024;
  return runs < most ? runs : most > 1 ? most : 1;
}

// Whether 16 tokens from a multiple of 16 lie in one page, at offsets below 2^31.
inline bool uniform_pages(const Pool& p) {
  const int64_t far = (int64_t)1 << 31;
  return p.page_tokens % 16 == 0 && p.k_page < far && p.v_page < far && p.page_tokens * p.k_tok < far &&
         p.page_tokens * p.v_tok < far;
}

constexpr int kStatusCapacity = 1, kStatusPage = 2;

template <typename T>
struct Tile {
  static constexpr int kRow = HC_HEAD_DIM * (int)sizeof(T);  // bytes of a token
  static constexpr int kBytes = HC_TILE * kRow;
  static constexpr int kLoads = kBytes / 1024;               // loads of a wave
  static constexpr int kChunks = kRow / 16;                  // chunks of a token
  static constexpr int kTokens = 1024 / kRow;                // tokens of a load
  static __device__ __forceinline__ int swizzle(int t) {
    return sizeof(T) == 4 ? t & 15 : (t & 7) << 1 | (t >> 3 & 1);
  }
};

// gfx950's transposing LDS read of 16-bit elements: lane i of a 16-lane group
// receives element i % 4 of the 8 bytes at lanes i / 4 + 4 k, k < 4.
typedef short __attribute__((ext_vector_type(4))) short4_t;
typedef short __attribute__((ext_vector_type(8))) short8_t;
__device__ __forceinline__ short4_t lds_read_transposed(const char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(p));
}

// Operand of 16 keys, tokens 16 h + n of the tile, channels 32 x + 8 g + [0, 8).
template <typename T>
__device__ __forceinline__ typename Elem<T>::vec8 key_operand(const char* tile, int g, int n, int h, int x) {
  const char* row = tile + (16 * h + n) * Tile<T>::kRow;
  const int sw = Tile<T>::swizzle(n);
  if constexpr (sizeof(T) == 4) {
    typename Elem<T>::vec8 r;
    r.lo = *reinterpret_cast<const f32x4*>(row + 16 * ((8 * x + 2 * g) ^ sw));
    r.hi = *reinterpret_cast<const f32x4*>(row + 16 * ((8 * x + 2 * g + 1) ^ sw));
    return r;
  } else {
    return *reinterpret_cast<const typename Elem<T>::vec8*>(row + 16 * ((4 * x + g) ^ sw));
  }
}

// Operand of 16 channels, 16 mt + n, of the tile's tokens 16 (e / 4) + 4 g + e % 4.
template <typename T>
__device__ __forceinline__ typename Elem<T>::vec8 value_operand(const char* tile, int g, int n, int mt) {
  if constexpr (sizeof(T) == 4) {
    typename Elem<T>::vec8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int t = 16 * (e >> 2) + 4 * g + (e & 3);
      set8<T>(r, e, *reinterpret_cast<const float*>(tile + t * Tile<T>::kRow +
                                                    16 * ((4 * mt + (n >> 2)) ^ Tile<T>::swizzle(t)) + 4 * (n & 3)));
    }
    return r;
  } else {
    const int t = 4 * g + (n >> 2);
    const char* p = tile + t * Tile<T>::kRow + 16 * ((2 * mt + (n >> 1 & 1)) ^ Tile<T>::swizzle(t)) + 8 * (n & 1);
    const short4_t lo = lds_read_transposed(p), hi = lds_read_transposed(p + 16 * Tile<T>::kRow);
    const short8_t both = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(typename Elem<T>::vec8, both);
  }
}

struct PagedNew {  // the new keys and values [batch][Hkv][Q][128]: byte strides
  const char *k, *v;
  int64_t k_s[3], v_s[3];
};

constexpr int kPagedWaves = 4, kPagedThreads = 64 * kPagedWaves;

// Rows of at most this many (query, head) columns are paged_rows_kernel's, the
// others paged_chunk_kernel's; a padded batch may hold both.
constexpr int kFewCols = 16;
constexpr int kChunkCols = 128;  // columns of a workgroup of the latter

struct PagedAttn {
  Pool pool;
  PagedNew fresh;
  const void* q;
  int64_t q_s[3];  // element strides: batch, head, token
  void* out;
  int64_t o_s[3];
  int G, cols, few;  // query heads of a KV head; columns of a row, (query, head) pairs i * G + g; and of one of few
  uint32_t g_mul;    // c / G = (c * g_mul) >> g_shift
  int g_shift;
  float scale_log2;
  int4* info;  // few columns, per row: first partial, how many, its tokens with the new ones (-1 - len: no room for them)
  float *part_o, *part_ml;  // partials: 128 channels; (m, l)
  int4* plan;               // many columns, per row: first partial, parts, tokens as above
  float *chunk_o, *chunk_ml;
  float* ml;  // a column's folded state, as weigh_state: [row][ml_stride]
  int64_t ml_stride;
  int32_t* len_out;
  // Accumulated weights of every token and the scores of few columns.
  const float* weights;
  float* weights_out;
  int64_t weight_stride;
  float* scores;
  int64_t score_stride;
  int32_t* pos;
  int64_t pos_stride;
  const int32_t* dropped;
  float* zeroed;  // weights of new tokens are set to zero here (calls that do not accumulate)
  int grid, chunk_grid, chunk_slots;
};

__device__ __forceinline__ int over_group(const PagedAttn& a, int c) {
  return (int)(((uint64_t)(uint32_t)c * a.g_mul) >> a.g_shift);
}

inline unsigned paged_chunk_fold_grid(const PagedAttn& a) {
  const int64_t work = ((int64_t)a.pool.rows * a.cols + 7) / 8, least = (a.pool.rows + 255) / 256;
  return (unsigned)(work < least ? least : work < 8192 ? work : 8192);
}

// fold: the launch that folds the partials too.
int launch_paged_rows(int dtype, const PagedAttn& a, bool fold, hipStream_t s);
int launch_paged_chunk(int dtype, const PagedAttn& a, bool fold, hipStream_t s);
int launch_paged_append(int dtype, const PagedAttn& a, hipStream_t s);
int launch_paged_carry(const PagedAttn& a, hipStream_t s);
int launch_paged_mixed(int dtype, const PagedAttn& a, hipStream_t s);
int launch_paged_weights(int dtype, const PagedAttn& a, hipStream_t s);
int paged_rows_slots(int dtype);
int paged_chunk_slots(int dtype);

}  // namespace hc
