// Argument checks, launches and the cut of the keys that the entry points of
// the paged caches share (cache_api.cpp, cache8_api.cpp).
#pragma once

#include "../../include/xpu_cache.h"
#include "kernels/cache_types.hpp"
#include "runtime_internal.hpp"

#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

namespace xpu {
namespace checks {

constexpr double kLog2e = 1.44269504088896340736;

inline int invalid(const char *name, const std::string &what) { return set_error(XPU_ERR_INVALID, std::string(name) + ": " + what); }

inline bool aligned(const void *p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

inline bool overlap(const void *a, uint64_t a_bytes, const void *b, uint64_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + b_bytes && y < x + a_bytes;
}

// The bytes that `rows` rows of `width` elements span.
inline uint64_t span(uint64_t rows, uint64_t stride, uint64_t width) { return rows ? ((rows - 1) * stride + width) * 2 : 0; }

// Whether rows of a_width elements at a and of b_width at b share a byte. Rows
// the same stride apart may lie side by side, as columns of one buffer.
inline bool rows_overlap(uint64_t rows, uint64_t a_width, const void *a, uint64_t a_stride, uint64_t b_width,
                         const void *b, uint64_t b_stride) {
  if (!overlap(a, span(rows, a_stride, a_width), b, span(rows, b_stride, b_width))) return false;
  if (a_stride != b_stride) return true;
  const uint64_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b), stride = 2 * a_stride;
  const uint64_t apart = (x < y ? y - x : x - y) % stride;  // from the lower one's rows to the other's
  const uint64_t low = x < y ? a_width : b_width, high = x < y ? b_width : a_width;
  return apart < 2 * low || stride - apart < 2 * high;
}
inline bool rows_overlap(uint64_t rows, uint64_t width, const void *a, uint64_t a_stride, const void *b, uint64_t b_stride) {
  return rows_overlap(rows, width, a, a_stride, width, b, b_stride);
}

// A launch's threads have to fit 32 bits.
constexpr uint64_t kMostBlocks = (1ull << 24) - 1;

inline int check_runtime(const char *name, const xpu_runtime *rt) { return rt ? XPU_OK : invalid(name, "null runtime"); }

// What describes the pages, and where they lie: pages of `page` elements.
inline int check_shape(const char *name, const xpu_cache &c) {
  if (c.dtype != XPU_DTYPE_BF16 && c.dtype != XPU_DTYPE_FP16) return invalid(name, "dtype must be bf16 (0) or fp16 (1)");
  if (c.head_dim != 64 && c.head_dim != 128) return invalid(name, "head_dim must be 64 or 128");
  if (c.page_size < 16 || c.page_size > 256 || (c.page_size & (c.page_size - 1)))
    return invalid(name, "page_size must be 16, 32, 64, 128 or 256");
  if (!c.layers || !c.kv_heads || !c.n_pages) return invalid(name, "layers, kv_heads and n_pages must be positive");
  if (c.kv_heads > 4096 || c.layers > 4096) return invalid(name, "at most 4096 layers and kv_heads");
  return XPU_OK;
}
inline int check_memory(const char *name, const xpu_cache &c, uint64_t page, const char *unit) {
  if ((c.page_stride | c.layer_stride) >> 40)
    return invalid(name, std::string("strides must be below 2^40 ") + unit);
  const bool apart = (c.n_pages == 1 || c.page_stride >= page) && (c.layers == 1 || c.layer_stride >= page);
  const unsigned __int128 pages_end = static_cast<unsigned __int128>(c.n_pages - 1) * c.page_stride + page;
  const unsigned __int128 layers_end = static_cast<unsigned __int128>(c.layers - 1) * c.layer_stride + page;
  if (!apart || (c.layers > 1 && c.n_pages > 1 && c.layer_stride < pages_end && c.page_stride < layers_end))
    return invalid(name, "pages overlap at these strides");
  if (!c.k || !c.v) return invalid(name, "null cache memory");
  if (!aligned(c.k, 16) || !aligned(c.v, 16) || !aligned(c.status, 4))
    return invalid(name, "k and v must be 16-byte aligned, status 4-byte");
  return XPU_OK;
}
inline int check_cache(const char *name, const xpu_cache *c, bool memory) {
  if (!c) return invalid(name, "null cache");
  if (int rc = check_shape(name, *c)) return rc;
  if (!memory) return XPU_OK;
  if (c->page_stride % 8 || c->layer_stride % 8) return invalid(name, "strides must be multiples of 8 elements");
  return check_memory(name, *c, static_cast<uint64_t>(c->kv_heads) * c->page_size * c->head_dim, "elements");
}

// `idle`: a batch without rows has nothing to be done, so its memory may be anything.
inline int check_batch(const char *name, const xpu_batch *b, bool memory, bool idle = true) {
  if (!b) return invalid(name, "null batch");
  if (b->rows >> 31 || b->n_seqs >> 24) return invalid(name, "at most 2^31 - 1 rows and 2^24 - 1 sequences");
  if (!b->n_seqs || (idle && !b->rows)) return XPU_OK;
  if (!b->table_pitch) return invalid(name, "table_pitch must be positive");
  if (!memory) return XPU_OK;
  if (!b->tables || !b->starts || !b->context) return invalid(name, "null batch memory");
  if (!aligned(b->tables, 4) || !aligned(b->starts, 4) || !aligned(b->context, 4))
    return invalid(name, "tables, starts and context must be 4-byte aligned");
  return XPU_OK;
}

// Rows of `width` elements, `stride` apart.
inline int check_rows(const char *name, const char *what, const void *p, uint64_t stride, uint64_t width) {
  if (!p) return invalid(name, std::string("null ") + what);
  if (!aligned(p, 16)) return invalid(name, std::string(what) + " must be 16-byte aligned");
  if (stride % 8 || stride < width || stride >> 24)
    return invalid(name, std::string(what) + "_stride must be a multiple of 8, at least " + std::to_string(width) +
                             " and below 2^24 elements");
  return XPU_OK;
}

inline int check_heads(const char *name, uint32_t heads, uint32_t kv_heads, float scale) {
  if (!heads || !kv_heads || heads % kv_heads || heads > 65536)
    return invalid(name, "heads must be a positive multiple of kv_heads, at most 65536");
  if (!(scale > 0) || !std::isfinite(static_cast<float>(scale * kLog2e)))
    return invalid(name, "scale must be positive and finite, also times log2(e)");
  return XPU_OK;
}

inline PoolArgs pool_of(const xpu_cache &c) {
  PoolArgs p{};
  p.k = static_cast<uint16_t *>(c.k);
  p.v = static_cast<uint16_t *>(c.v);
  p.layer_stride = c.layer_stride;
  p.page_stride = c.page_stride;
  p.layers = c.layers;
  p.kv_heads = c.kv_heads;
  p.page_size = c.page_size;
  p.page_shift = static_cast<uint32_t>(__builtin_ctz(c.page_size));
  p.n_pages = c.n_pages;
  p.status = c.status;
  return p;
}

inline BatchArgs batch_of(const xpu_batch &b) { return {b.tables, b.starts, b.context, b.n_seqs, b.rows, b.table_pitch}; }

template <typename A>
int launch(xpu_runtime *rt, const std::string &kernel, uint64_t grid, const A &args, uint32_t grid_y = 1,
           const uint32_t *more = nullptr, uint32_t block = 256) {
  if (grid > kMostBlocks) return set_error(XPU_ERR_INVALID, kernel + ": too many rows for one launch");
  const xpu::KernelInfo *k = rt->find_exact(kernel);
  if (!k) return set_error(XPU_ERR_NOT_FOUND, "kernel is absent from module: " + kernel);
  XPU_HIP_RETURN(hipSetDevice(rt->device));
  const xpu_kernel_arg list[] = {{sizeof(A), &args}, {4, more}};
  return rt->launch(*k, static_cast<uint32_t>(grid), grid_y, block, 0, list, more ? 2 : 1);
}

// Up to n ids of pages 0 .. pool - 1: a bit for each page of a pool that is not
// large beside n, else open addressing in at least four times n places, so that
// few pairs cost what they cost whatever the pool is. The host's part of a call:
// 4 pairs in 1000000 pages 2.7 us by addressing, 13 by bits (in 64 pages 2.7);
// 8192 pairs in 1000000 pages 44 and 29, in 100000 pages 53 and 21.
class Ids {
 public:
  Ids(uint32_t n, uint32_t pool) {
    if (pool / 256 < n) {
      bits_.assign(pool / 64 + 1, 0);
      return;
    }
    while ((1ull << (64 - shift_)) < 4ull * n) --shift_;
    places_.assign(1ull << (64 - shift_), kNone);
  }
  // whether `id` was not there yet
  bool add(uint32_t id) {
    if (!bits_.empty()) {
      uint64_t &word = bits_[id / 64];
      const uint64_t bit = 1ull << id % 64;
      const bool fresh = !(word & bit);
      word |= bit;
      return fresh;
    }
    uint32_t &at = places_[find(id)];
    const bool fresh = at == kNone;
    at = id;
    return fresh;
  }
  bool has(uint32_t id) const {
    return bits_.empty() ? places_[find(id)] == id : bits_[id / 64] >> id % 64 & 1;
  }

 private:
  static constexpr uint32_t kNone = ~0u;  // no page: there are 2^32 - 1 at most
  uint64_t find(uint32_t id) const {
    uint64_t at = id * 0x9e3779b97f4a7c15ull >> shift_;  // 2^64 / the golden ratio: the top bits spread
    while (places_[at] != kNone && places_[at] != id) at = (at + 1) & (places_.size() - 1);
    return at;
  }
  int shift_ = 63;
  std::vector<uint64_t> bits_;
  std::vector<uint32_t> places_;
};

inline const char *type_name(int32_t dtype) { return dtype == XPU_DTYPE_FP16 ? "fp16" : "bf16"; }

// How a tree attention call is cut (kernels/tree_attention.hip). Every rule
// goes by what the host knows: numbers of rows and sequences, not lengths.
struct TreePlan {
  uint32_t sub_tiles = 1;  // of 32 rows per block
  uint32_t fit = 0;        // work items per kv head at most; 0: as `target` gives
  uint32_t target = 1;     // chunks aimed at per kv head
  uint32_t least = 4;      // tiles of 32 keys in a chunk, one for each wavefront
  uint64_t slots = 0;      // work items per kv head, at most
  uint64_t bytes = 0;      // of the workspace; 0: the keys are not cut
  uint64_t joins = 0;      // pairs of heads of all rows, each joined by
  uint32_t join_waves = 1; // so many wavefronts
};

// `eight`: over 8-bit pages (kernels/tree_attention8.hip).
inline TreePlan tree_plan(const xpu_runtime &rt, bool eight, uint32_t kv_heads, uint32_t page_size, uint32_t head_dim,
                          const xpu_batch &b, uint32_t heads) {
  TreePlan p;
  const uint64_t rows = static_cast<uint64_t>(b.rows) * (heads / kv_heads);
  // 16 bits: 64 rows per block where sequences have more than 22 rows on average, so
  // that the larger ones do not read their keys twice (48 ragged sequences of
  // 1 .. 26 nodes x 4 heads, 28 rows on average, 98.4 us in 32s and 90.5 in
  // 64s; 23 rows 93.8 and 90.5; 20 rows 86.8 and 88.2; 4 rows 69.5 and 72.7)
  p.sub_tiles = !eight && rows > 22ull * b.n_seqs ? 2 : 1;
  const uint64_t row_tiles = rows / (32 * p.sub_tiles) + b.n_seqs;  // at most
  const uint64_t tiles = (static_cast<uint64_t>(b.table_pitch) * page_size + 31) / 32;
  const bool cut = tiles > p.least;
  // A compute unit holds two blocks at D 128, where all of this was measured (at
  // D 64 four of one sub-tile or three of two; the rule is the same there, untimed).
  // Cut into just as many as the chip holds,
  // all run at once and end together, and none starts with nothing to do (four
  // long drafts 375 us, with 3 blocks per unit dealt as others end 420; 16
  // ragged ones of 1 .. 26 nodes 36.4 and 47.0; one token behind 32000
  // positions 28.1 and 31.5, behind 16000 19.2 and 23.6). Where more than four
  // fifths of them are row tiles, the chunks get too uneven: three per unit (48
  // single tokens 70.0 us, and 79.8 cut to fit; 32 drafts of up to 8 nodes 53.4
  // to fit and 56.0). Over 8-bit pages a unit holds three blocks of 32 rows (whole
  // calls, cut for three, two and four: the four drafts 290 us, 314 and 313; 48 of
  // up to 8 nodes 47, 45 and 49; 48 single tokens 45, 42.5 and 49; at D 64 191,
  // 233 and 172; single tokens 29.9, 27.0 and 29.0, one behind 32000 17.1, 16.1 and
  // 17.5), and two per unit do where they do not fit (48 of 1 .. 26 nodes: the
  // kernel 46.5 us, with three 51.0).
  const uint64_t fit = (eight ? 3 : 2) * rt.compute_units / kv_heads;
  if (cut && b.n_seqs <= 64 && row_tiles <= fit * 4 / 5) p.fit = static_cast<uint32_t>(fit);
  p.target = std::max(1u, (eight ? 2 : 3) * rt.compute_units / kv_heads);
  p.slots = p.fit ? fit : row_tiles + (cut ? p.target : 0);
  p.bytes = cut ? p.slots * kv_heads * (32ull * p.sub_tiles * (head_dim + 2)) * 4 : 0;
  // the fewer joins, the more wavefronts for each, which read its chunks side
  // by side: one above 6 per unit (48 sequences of 4 nodes 76.3 us, with four
  // 77.9; of 2 nodes, 6 per unit, both 73.1; of 1 node 71.2 and 70.1), four
  // above 2 per unit (48 of 1 node 70.1, with eight 71.3; one of 16 nodes at
  // 8000 positions, half per unit, 22.0 and 20.3), eight below, sixteen where
  // a row can have 128 chunks (32000 positions of 2 kv heads: 33.7 us with
  // four, 24.5 with eight, 20.6 with sixteen; of 8 kv heads, 64 chunks: 28.7,
  // 27.8, 28.6)
  p.joins = b.rows * ((heads + 1ull) / 2);
  p.join_waves = p.joins > 6ull * rt.compute_units ? 1
                 : p.joins > 2ull * rt.compute_units ? 4
                 : std::min<uint64_t>(p.fit ? p.fit : p.target, tiles / p.least) < 128 ? 8 : 16;
  return p;
}

// What tree attention takes besides the cache and the batch.
struct TreeRows {
  uint32_t heads;
  float scale;
  const void *q;
  uint64_t q_stride;
  const uint64_t *visible;
  void *out;
  uint64_t out_stride;
  void *workspace;
  uint64_t workspace_bytes;
};

inline int check_tree_rows(const char *name, const TreeRows &r, const xpu_batch &b, uint32_t head_dim) {
  const uint64_t width = static_cast<uint64_t>(r.heads) * head_dim;
  if (int rc = check_rows(name, "q", r.q, r.q_stride, width)) return rc;
  if (int rc = check_rows(name, "out", r.out, r.out_stride, width)) return rc;
  if (!aligned(r.visible, 8)) return invalid(name, "visible must be 8-byte aligned");
  if (rows_overlap(b.rows, width, r.q, r.q_stride, r.out, r.out_stride)) return invalid(name, "out must not overlap q");
  if (static_cast<uint64_t>(b.rows) * r.heads >= (1ull << 26)) return invalid(name, "too many rows");
  return XPU_OK;
}

// `pool`: the layer's pages.
inline int launch_tree(const char *name, xpu_runtime *rt, bool eight, const PoolArgs &pool, int32_t dtype,
                       uint32_t head_dim, const xpu_batch &b, const TreeRows &r) {
  const TreePlan plan = tree_plan(*rt, eight, pool.kv_heads, pool.page_size, head_dim, b, r.heads);
  if (plan.bytes && (!r.workspace || !aligned(r.workspace, 16) || r.workspace_bytes < plan.bytes))
    return invalid(name, "needs a workspace of " + std::to_string(plan.bytes) + " bytes, 16-byte aligned");
  TreeArgs a{};
  a.pool = pool;
  a.batch = batch_of(b);
  a.q = static_cast<const uint16_t *>(r.q);
  a.out = static_cast<uint16_t *>(r.out);
  a.visible = r.visible;
  a.partial = static_cast<float *>(r.workspace);
  a.q_stride = r.q_stride;
  a.out_stride = r.out_stride;
  a.heads = r.heads;
  a.fit = plan.fit;
  a.target = plan.target;
  a.least = plan.least;
  a.slots = static_cast<uint32_t>(plan.slots);
  a.scale_log2e = static_cast<float>(r.scale * kLog2e);
  const std::string form =
      std::string("_") + type_name(dtype) + "_d" + std::to_string(head_dim) + "_r" + std::to_string(plan.sub_tiles);
  if (int rc = launch(rt, (eight ? "xpu_tree_attention8" : "xpu_tree_attention") + form, plan.slots * pool.kv_heads, a))
    return rc;
  if (!plan.bytes) return XPU_OK;
  const std::string join = "xpu_tree_join" + form + "_w" + std::to_string(plan.join_waves);
  return plan.join_waves > 1 ? launch(rt, join, plan.joins, a, 1, nullptr, 64 * plan.join_waves)
                             : launch(rt, join, (plan.joins + 3) / 4, a);
}

inline int check_keep(const char *name, const xpu_batch *batch, const uint32_t *kept, const uint32_t *counts,
                      uint32_t *new_context) {
  if (int rc = check_batch(name, batch, true, false)) return rc;
  if (!batch->n_seqs) return XPU_OK;
  if ((!kept && batch->rows) || !counts) return invalid(name, "null argument");
  if (!aligned(kept, 4) || !aligned(counts, 4) || !aligned(new_context, 4))
    return invalid(name, "kept, counts and new_context must be 4-byte aligned");
  const uint64_t list = 4ull * batch->n_seqs;
  if (new_context && (overlap(new_context, list, batch->context, list) || overlap(new_context, list, counts, list) ||
                      overlap(new_context, list, batch->starts, list + 4) ||
                      (kept && overlap(new_context, list, kept, 4ull * batch->rows))))
    return invalid(name, "new_context must not overlap context, counts, starts or kept");
  return XPU_OK;
}

inline int check_copy(const char *name, uint32_t n_pages, const uint32_t *src, const uint32_t *dst, uint32_t n) {
  if (!n) return XPU_OK;
  if (!src || !dst) return invalid(name, "null argument");
  Ids to(n, n_pages);
  for (uint32_t i = 0; i < n; ++i) {
    if (src[i] >= n_pages || dst[i] >= n_pages)
      return invalid(name, "page " + std::to_string(std::max(src[i], dst[i])) + " does not exist");
    if (!to.add(dst[i])) return invalid(name, "page " + std::to_string(dst[i]) + " is copied to twice");
  }
  for (uint32_t i = 0; i < n; ++i)
    if (to.has(src[i])) return invalid(name, "page " + std::to_string(src[i]) + " is copied to and from");
  return XPU_OK;
}

// Pages of `chunks` times 16 bytes, in all layers. The pairs travel as kernel
// arguments, so many at a time.
inline int launch_copy(xpu_runtime *rt, const PoolArgs &pool, uint32_t chunks, const uint32_t *src, const uint32_t *dst,
                       uint32_t n) {
  for (uint32_t at = 0; at < n; at += kCopyPairs) {
    CopyArgs a{};
    a.pool = pool;
    a.n = std::min(n - at, kCopyPairs);
    std::copy(src + at, src + at + a.n, a.src);
    std::copy(dst + at, dst + at + a.n, a.dst);
    if (int rc = launch(rt, "xpu_cache_copy", static_cast<uint64_t>(a.n) * pool.layers * 2, a, (chunks + 2047) / 2048,
                        &chunks))
      return rc;
  }
  return XPU_OK;
}

}  // namespace checks
}  // namespace xpu
