// Entry points of the paged cache: checks, plans and launches.
#include <algorithm>
#include <cmath>

#include "hc_paged.h"

namespace hc {

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// t / d = (t * mul) >> shift for t < 2^31: mul = ceil(2^(31 + s) / d), shift = 31 + s, d <= 2^s.
static void divider(int d, uint32_t& mul, int& shift) {
  int s = 0;
  while (((int64_t)1 << s) < d) ++s;
  mul = (uint32_t)((((uint64_t)1 << (31 + s)) + d - 1) / d);
  shift = 31 + s;
}

// The cache's geometry, checked, as the kernels take it.
int fill_pool(const char* name, const hc_paged_cache* c, Pool& p, int Q, const int32_t* counts) {
  if (!c) return set_error(HC_ERR_INVALID, "%s: null cache", name);
  if (c->dtype != HC_DTYPE_BF16 && c->dtype != HC_DTYPE_F16 && c->dtype != HC_DTYPE_F32)
    return set_error(HC_ERR_INVALID, "%s: unknown dtype %d", name, c->dtype);
  if (c->batch < 0 || c->kv_heads < 1 || (c->heads != 1 && c->heads != c->kv_heads) ||
      (int64_t)c->batch * c->kv_heads > (1 << 24))
    return set_error(HC_ERR_INVALID, "%s: batch=%d kv_heads=%d heads=%d (1 or kv_heads, at most 2^24 rows)", name, c->batch,
                     c->kv_heads, c->heads);
  if (c->pages < 1 || c->page_tokens < 1 || c->table_pages < 1 ||
      (int64_t)c->table_pages * c->page_tokens > (int64_t)1 << 30)
    return set_error(HC_ERR_INVALID, "%s: pages=%d page_tokens=%d table_pages=%d (a row holds at most 2^30 tokens)", name,
                     c->pages, c->page_tokens, c->table_pages);
  if ((int64_t)c->batch * c->kv_heads * (((int64_t)c->table_pages * c->page_tokens + HC_TILE - 1) / HC_TILE) > (int64_t)1 << 30)
    return set_error(HC_ERR_INVALID, "%s: all rows' capacity exceeds 2^30 tiles of 32 tokens", name);
  if (!c->k || !c->v || !c->table || !c->row_len) return set_error(HC_ERR_INVALID, "%s: null pointer in the cache", name);
  const int esz = c->dtype == HC_DTYPE_F32 ? 4 : 2;
  for (int i = 0; i < 3; ++i)
    if (c->k_strides[i] < 0 || c->v_strides[i] < 0 || c->k_strides[i] * esz % 16 || c->v_strides[i] * esz % 16)
      return set_error(HC_ERR_INVALID, "%s: the pools' strides must be non-negative multiples of 16 bytes", name);
  if (c->k_strides[1] * esz >= 1 << 26 || c->v_strides[1] * esz >= 1 << 26)
    return set_error(HC_ERR_INVALID, "%s: a pool's token stride must be below 2^26 bytes", name);
  if (!aligned16(c->k) || !aligned16(c->v)) return set_error(HC_ERR_INVALID, "%s: the pools must be 16-byte aligned", name);
  if (c->table_stride < c->table_pages && c->batch * (int64_t)c->kv_heads / c->heads > 1)
    return set_error(HC_ERR_INVALID, "%s: table rows %lld apart hold %d entries", name, (long long)c->table_stride,
                     c->table_pages);
  const int64_t cap = (int64_t)c->table_pages * c->page_tokens;
  if (c->weights && (!c->pos || !c->dropped || c->weight_stride < cap || c->pos_stride < cap))
    return set_error(HC_ERR_INVALID, "%s: weights need positions and dropped counts, rows of each %lld entries apart or more", name,
                     (long long)cap);
  p.k = reinterpret_cast<const char*>(c->k), p.v = reinterpret_cast<const char*>(c->v);
  p.k_page = c->k_strides[0] * esz, p.k_tok = c->k_strides[1] * esz, p.k_head = c->k_strides[2] * esz;
  p.v_page = c->v_strides[0] * esz, p.v_tok = c->v_strides[1] * esz, p.v_head = c->v_strides[2] * esz;
  p.table = c->table, p.table_stride = c->table_stride, p.row_len = c->row_len, p.counts = counts, p.status = c->status;
  divider(c->page_tokens, p.div_mul, p.div_shift);
  p.page_tokens = c->page_tokens, p.pages = c->pages, p.capacity = (int)cap;
  p.heads = c->heads, p.Hkv = c->kv_heads, p.rows = c->batch * c->kv_heads, p.Q = Q;
  p.fresh = 0;
  return HC_OK;
}

namespace {

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// The parts of a call's workspace, and its grids.
struct Layout {
  bool chunk;  // rows of many columns
  int cols, few, grid, chunk_grid, chunk_slots;
  size_t info, part_o, part_ml, plan, chunk_o, chunk_ml, ml, scores, bytes;
  int64_t score_stride, ml_stride;
};

Layout layout(const hc_paged_cache* c, int q_heads, int queries, bool counts, bool weigh) {
  Layout l = {};
  const int G = q_heads / c->kv_heads, rows = c->batch * c->kv_heads;
  const int64_t cap = (int64_t)c->table_pages * c->page_tokens;
  l.cols = G * queries;
  l.chunk = l.cols > kFewCols;
  // A padded batch's short rows are attended as such.
  l.few = !l.chunk ? l.cols : counts && G <= kFewCols ? kFewCols : 0;
  auto take = [&](size_t bytes) {
    const size_t here = l.bytes;
    l.bytes += up256(bytes);
    return here;
  };
  if (l.few) {
    l.grid = paged_rows_slots(c->dtype);
    const size_t slots = (size_t)l.grid + rows;
    l.info = take((size_t)rows * sizeof(int4));
    l.part_o = take(slots * l.few * HC_HEAD_DIM * 4);
    l.part_ml = take(slots * l.few * 8);
    if (weigh) {
      l.score_stride = (cap + HC_TILE - 1) / HC_TILE * HC_TILE * l.few;
      l.scores = take((size_t)rows * l.score_stride * 4);
    }
  }
  if (l.chunk) {
    // One round of workgroups may be cut blocks' (see find_unit).
    l.chunk_slots = paged_chunk_slots(c->dtype);
    const int64_t blocks = (int64_t)rows * ((l.cols + kChunkCols - 1) / kChunkCols);
    l.chunk_grid = (int)std::min<int64_t>((l.chunk_slots + blocks + 7) / 8 * 8, 0x7ffffff8);
    l.plan = take((size_t)rows * sizeof(int4));
    l.chunk_o = take((size_t)l.chunk_slots * kChunkCols * HC_HEAD_DIM * 4);
    l.chunk_ml = take((size_t)l.chunk_slots * kChunkCols * 8);
    // (Read 128 states at a time from multiples of 64.)
    l.ml_stride = (l.cols + 63) / 64 * 64 + 64;
    if (weigh) l.ml = take((size_t)rows * l.ml_stride * 8);
  }
  return l;
}

// More than 2^26 query rows (whose product may pass 64 bits).
bool too_many(const hc_paged_cache* c, int q_heads, int queries) {
  return (int64_t)c->batch * q_heads > 1 << 26 || (int64_t)c->batch * q_heads * queries > 1 << 26;
}

bool sized(const hc_paged_cache* c, int q_heads, int queries) {
  return c && c->batch > 0 && c->kv_heads > 0 && q_heads > 0 && q_heads % c->kv_heads == 0 && queries > 0 && c->table_pages > 0 &&
         c->page_tokens > 0 && !too_many(c, q_heads, queries);
}

int check_fresh(const char* name, const hc_paged_cache* c, const void* k, const int64_t* ks, const void* v, const int64_t* vs,
                PagedNew& f) {
  const int esz = c->dtype == HC_DTYPE_F32 ? 4 : 2;
  if (!k || !v || !ks || !vs) return set_error(HC_ERR_INVALID, "%s: null pointer argument", name);
  if (!aligned16(k) || !aligned16(v)) return set_error(HC_ERR_INVALID, "%s: tensors must be 16-byte aligned", name);
  f.k = reinterpret_cast<const char*>(k), f.v = reinterpret_cast<const char*>(v);
  for (int i = 0; i < 3; ++i) {
    if (ks[i] * esz % 16 || vs[i] * esz % 16)
      return set_error(HC_ERR_INVALID, "%s: strides must be multiples of 16 bytes", name);
    f.k_s[i] = ks[i] * esz, f.v_s[i] = vs[i] * esz;
  }
  return HC_OK;
}

void take_ledger(const hc_paged_cache* c, PagedAttn& a) {
  a.weights = c->weights, a.weight_stride = c->weight_stride;
  a.pos = c->weights ? c->pos : nullptr, a.pos_stride = c->pos_stride, a.dropped = c->dropped;
  a.weights_out = nullptr, a.zeroed = c->weights;
}

}  // namespace

int paged_rows_slots(int dtype) { return device_cus() * (dtype == HC_DTYPE_F32 ? 1 : 2); }

int paged_chunk_slots(int dtype) { return device_cus() * 2; }

}  // namespace hc

using namespace hc;

extern "C" size_t hc_paged_workspace_size(const hc_paged_cache* c, int q_heads, int queries, int counts, int weigh) {
  return sized(c, q_heads, queries) ? layout(c, q_heads, queries, counts, weigh).bytes : 0;
}

extern "C" int hc_paged_append(const hc_paged_cache* c, const void* k, const int64_t* k_strides, const void* v,
                               const int64_t* v_strides, const int32_t* counts, int tokens, int32_t* len_out, void* stream) {
  clear_error();
  PagedAttn a = {};
  if (int rc = fill_pool("hc_paged_append", c, a.pool, tokens, counts)) return rc;
  if (tokens < 0) return set_error(HC_ERR_INVALID, "hc_paged_append: tokens=%d", tokens);
  if (c->batch == 0 || (tokens == 0 && !len_out)) return HC_OK;
  const intptr_t gap = 4 * (intptr_t)(a.pool.rows / c->heads);
  const intptr_t apart = reinterpret_cast<intptr_t>(len_out) - reinterpret_cast<intptr_t>(c->row_len);
  if (len_out && apart != 0 && apart > -gap && apart < gap)
    return set_error(HC_ERR_INVALID, "hc_paged_append: len_out overlaps row_len without being it");
  if (tokens > 0)
    if (int rc = check_fresh("hc_paged_append", c, k, k_strides, v, v_strides, a.fresh)) return rc;
  if ((int64_t)a.pool.rows * ((tokens + 15) / 16) > kMostGroups)
    return set_error(HC_ERR_INVALID, "hc_paged_append: %d rows x %d tokens", a.pool.rows, tokens);
  a.pool.fresh = 1;
  a.len_out = len_out ? len_out : c->row_len;
  take_ledger(c, a);
  return launch_paged_append(c->dtype, a, (hipStream_t)stream);
}

extern "C" int hc_paged_attn(const hc_paged_cache* c, const void* q, const int64_t* q_strides, int q_heads, int queries,
                             const void* k_new, const int64_t* k_strides, const void* v_new, const int64_t* v_strides,
                             const int32_t* counts, float scale, int weigh, float* weights_out, int32_t* len_out, void* out,
                             const int64_t* out_strides, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  PagedAttn a = {};
  if (int rc = fill_pool("hc_paged_attn", c, a.pool, queries, counts)) return rc;
  if (q_heads < 1 || q_heads % c->kv_heads || queries < 0 || too_many(c, q_heads, queries))
    return set_error(HC_ERR_INVALID, "hc_paged_attn: q_heads=%d kv_heads=%d queries=%d (at most 2^26 query rows)", q_heads,
                     c->kv_heads, queries);
  if (!std::isfinite(scale) || !(scale > 0.f))
    return set_error(HC_ERR_INVALID, "hc_paged_attn: scale must be finite and positive");
  if (weigh && !c->weights) return set_error(HC_ERR_INVALID, "hc_paged_attn: the cache has no weights to add to");
  if (weights_out && !weigh) return set_error(HC_ERR_INVALID, "hc_paged_attn: weights_out without weigh");
  if (c->batch == 0) return HC_OK;
  if (queries == 0) {
    // No outputs; the lengths and weights behind the call are those before it.
    if (weights_out && weights_out != c->weights) {
      take_ledger(c, a);
      a.weights_out = weights_out;
      if (int rc = launch_paged_carry(a, (hipStream_t)stream)) return rc;
    }
    return hc_paged_append(c, nullptr, nullptr, nullptr, nullptr, counts, 0, len_out, stream);
  }
  const bool fresh = k_new || v_new;
  if (len_out && !fresh) return set_error(HC_ERR_INVALID, "hc_paged_attn: len_out without new tokens");
  if (!q || !q_strides || !out || !out_strides) return set_error(HC_ERR_INVALID, "hc_paged_attn: null pointer argument");
  const int esz = c->dtype == HC_DTYPE_F32 ? 4 : 2;
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] * esz % 16 || out_strides[i] * esz % 16)
      return set_error(HC_ERR_INVALID, "hc_paged_attn: strides must be multiples of 16 bytes");
  if (!aligned16(q) || !aligned16(out)) return set_error(HC_ERR_INVALID, "hc_paged_attn: tensors must be 16-byte aligned");
  if (fresh)
    if (int rc = check_fresh("hc_paged_attn", c, k_new, k_strides, v_new, v_strides, a.fresh)) return rc;
  const Layout l = layout(c, q_heads, queries, counts != nullptr, weigh);
  if (workspace_bytes < l.bytes || !workspace || !aligned16(workspace))
    return set_error(HC_ERR_INVALID, "hc_paged_attn: workspace too small or unaligned (%zu < %zu bytes)", workspace_bytes, l.bytes);
  char* const ws = reinterpret_cast<char*>(workspace);
  a.pool.fresh = fresh;
  a.q = q, a.out = out;
  for (int i = 0; i < 3; ++i) a.q_s[i] = q_strides[i], a.o_s[i] = out_strides[i];
  a.G = q_heads / c->kv_heads, a.cols = l.cols, a.few = l.few;
  divider(a.G, a.g_mul, a.g_shift);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.info = reinterpret_cast<int4*>(ws + l.info);
  a.part_o = reinterpret_cast<float*>(ws + l.part_o);
  a.part_ml = reinterpret_cast<float*>(ws + l.part_ml);
  a.plan = reinterpret_cast<int4*>(ws + l.plan);
  a.chunk_o = reinterpret_cast<float*>(ws + l.chunk_o);
  a.chunk_ml = reinterpret_cast<float*>(ws + l.chunk_ml);
  a.grid = l.grid, a.chunk_grid = l.chunk_grid, a.chunk_slots = l.chunk_slots;
  take_ledger(c, a);
  if (!fresh) a.pos = nullptr, a.zeroed = nullptr;
  if (weigh) {
    a.weights_out = weights_out ? weights_out : c->weights;
    a.zeroed = nullptr;
    a.ml = reinterpret_cast<float*>(ws + l.ml), a.ml_stride = l.ml_stride;
    a.scores = reinterpret_cast<float*>(ws + l.scores);
    a.score_stride = l.score_stride;
  }
  hipStream_t s = (hipStream_t)stream;
  int32_t* const lens = fresh ? (len_out ? len_out : c->row_len) : nullptr;
  if (!l.chunk) {
    a.len_out = lens;
    return launch_paged_rows(c->dtype, a, true, s);
  }
  // The lengths advance in the last launch that knows the old ones.
  int rc;
  if (l.few) {
    a.len_out = lens;
    rc = launch_paged_mixed(c->dtype, a, s);
  } else {
    if (fresh && (rc = launch_paged_append(c->dtype, a, s))) return rc;
    a.len_out = lens;
    rc = launch_paged_chunk(c->dtype, a, true, s);
  }
  return rc || !weigh ? rc : launch_paged_weights(c->dtype, a, s);
}
