// Entry points of the paged cache and the attention over it and over packed
// prompts (include/xpu_cache.h): argument checks, the choice of a kernel, the
// launch. Kernels: kernels/packed_attention.hip, tree_attention.hip, cache.hip.
#include "../../include/xpu_cache.h"
#include "kernels/cache_types.hpp"
#include "runtime_internal.hpp"

#include <algorithm>
#include <cmath>
#include <vector>

using xpu::guarded;
using xpu::set_error;

namespace {

constexpr double kLog2e = 1.44269504088896340736;

int invalid(const char *name, const std::string &what) { return set_error(XPU_ERR_INVALID, std::string(name) + ": " + what); }

bool aligned(const void *p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

bool overlap(const void *a, uint64_t a_bytes, const void *b, uint64_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + b_bytes && y < x + a_bytes;
}

// The bytes that `rows` rows of `width` elements span.
uint64_t span(uint64_t rows, uint64_t stride, uint64_t width) { return rows ? ((rows - 1) * stride + width) * 2 : 0; }

// Whether rows of `width` elements at a and at b share a byte. Rows the same
// stride apart may lie side by side, as columns of one buffer.
bool rows_overlap(uint64_t rows, uint64_t width, const void *a, uint64_t a_stride, const void *b, uint64_t b_stride) {
  if (!overlap(a, span(rows, a_stride, width), b, span(rows, b_stride, width))) return false;
  if (a_stride != b_stride) return true;
  const uint64_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b), stride = 2 * a_stride;
  const uint64_t apart = (x < y ? y - x : x - y) % stride;
  return apart < 2 * width || stride - apart < 2 * width;
}

// A launch's threads have to fit 32 bits.
constexpr uint64_t kMostBlocks = (1ull << 24) - 1;

int check_runtime(const char *name, const xpu_runtime *rt) { return rt ? XPU_OK : invalid(name, "null runtime"); }

int check_cache(const char *name, const xpu_cache *c, bool memory) {
  if (!c) return invalid(name, "null cache");
  if (c->dtype != XPU_DTYPE_BF16 && c->dtype != XPU_DTYPE_FP16) return invalid(name, "dtype must be bf16 (0) or fp16 (1)");
  if (c->head_dim != 64 && c->head_dim != 128) return invalid(name, "head_dim must be 64 or 128");
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
    return invalid(name, "page_size must be 16, 32, 64, 128 or 256");
  if (!c->layers || !c->kv_heads || !c->n_pages) return invalid(name, "layers, kv_heads and n_pages must be positive");
  if (c->kv_heads > 4096 || c->layers > 4096) return invalid(name, "at most 4096 layers and kv_heads");
  if (!memory) return XPU_OK;
  const uint64_t page = static_cast<uint64_t>(c->kv_heads) * c->page_size * c->head_dim;
  if (c->page_stride % 8 || c->layer_stride % 8) return invalid(name, "strides must be multiples of 8 elements");
  if ((c->page_stride | c->layer_stride) >> 40) return invalid(name, "strides must be below 2^40 elements");
  const bool apart = (c->n_pages == 1 || c->page_stride >= page) && (c->layers == 1 || c->layer_stride >= page);
  const unsigned __int128 pages_end = static_cast<unsigned __int128>(c->n_pages - 1) * c->page_stride + page;
  const unsigned __int128 layers_end = static_cast<unsigned __int128>(c->layers - 1) * c->layer_stride + page;
  if (!apart || (c->layers > 1 && c->n_pages > 1 && c->layer_stride < pages_end && c->page_stride < layers_end))
    return invalid(name, "pages overlap at these strides");
  if (!c->k || !c->v) return invalid(name, "null cache memory");
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->status, 4))
    return invalid(name, "k and v must be 16-byte aligned, status 4-byte");
  return XPU_OK;
}

// `idle`: a batch without rows has nothing to be done, so its memory may be anything.
int check_batch(const char *name, const xpu_batch *b, bool memory, bool idle = true) {
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
int check_rows(const char *name, const char *what, const void *p, uint64_t stride, uint64_t width) {
  if (!p) return invalid(name, std::string("null ") + what);
  if (!aligned(p, 16)) return invalid(name, std::string(what) + " must be 16-byte aligned");
  if (stride % 8 || stride < width || stride >> 24)
    return invalid(name, std::string(what) + "_stride must be a multiple of 8, at least " + std::to_string(width) +
                             " and below 2^24 elements");
  return XPU_OK;
}

int check_heads(const char *name, uint32_t heads, uint32_t kv_heads, float scale) {
  if (!heads || !kv_heads || heads % kv_heads || heads > 65536)
    return invalid(name, "heads must be a positive multiple of kv_heads, at most 65536");
  if (!(scale > 0) || !std::isfinite(static_cast<float>(scale * kLog2e)))
    return invalid(name, "scale must be positive and finite, also times log2(e)");
  return XPU_OK;
}

xpu::PoolArgs pool_of(const xpu_cache &c) {
  xpu::PoolArgs p{};
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

xpu::BatchArgs batch_of(const xpu_batch &b) { return {b.tables, b.starts, b.context, b.n_seqs, b.rows, b.table_pitch}; }

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

const char *type_name(int32_t dtype) { return dtype == XPU_DTYPE_FP16 ? "fp16" : "bf16"; }

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

TreePlan tree_plan(const xpu_runtime &rt, const xpu_cache &c, const xpu_batch &b, uint32_t heads) {
  TreePlan p;
  const uint64_t rows = static_cast<uint64_t>(b.rows) * (heads / c.kv_heads);
  // 64 rows per block where sequences have more than 22 rows on average, so
  // that the larger ones do not read their keys twice (48 ragged sequences of
  // 1 .. 26 nodes x 4 heads, 28 rows on average, 98.4 us in 32s and 90.5 in
  // 64s; 23 rows 93.8 and 90.5; 20 rows 86.8 and 88.2; 4 rows 69.5 and 72.7)
  p.sub_tiles = rows > 22ull * b.n_seqs ? 2 : 1;
  const uint64_t row_tiles = rows / (32 * p.sub_tiles) + b.n_seqs;  // at most
  const uint64_t tiles = (static_cast<uint64_t>(b.table_pitch) * c.page_size + 31) / 32;
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
  // to fit and 56.0).
  const uint64_t fit = 2 * rt.compute_units / c.kv_heads;
  if (cut && b.n_seqs <= 64 && row_tiles <= fit * 4 / 5) p.fit = static_cast<uint32_t>(fit);
  p.target = std::max(1u, 3 * rt.compute_units / c.kv_heads);
  p.slots = p.fit ? fit : row_tiles + (cut ? p.target : 0);
  p.bytes = cut ? p.slots * c.kv_heads * (32ull * p.sub_tiles * (c.head_dim + 2)) * 4 : 0;
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

}  // namespace

extern "C" {

int xpu_cache_append(xpu_runtime *rt, const xpu_cache *cache, const xpu_batch *batch, uint32_t layer, const void *k,
                     uint64_t k_stride, const void *v, uint64_t v_stride) {
  static constexpr char name[] = "xpu_cache_append";
  return guarded(name, [&] {
    if (int rc = check_cache(name, cache, true)) return rc;
    if (int rc = check_batch(name, batch, true)) return rc;
    if (layer >= cache->layers) return invalid(name, "no such layer");
    if (!batch->rows || !batch->n_seqs) return check_runtime(name, rt);
    const uint64_t width = static_cast<uint64_t>(cache->kv_heads) * cache->head_dim;
    if (int rc = check_rows(name, "k", k, k_stride, width)) return rc;
    if (int rc = check_rows(name, "v", v, v_stride, width)) return rc;
    if (int rc = check_runtime(name, rt)) return rc;
    xpu::AppendArgs a{pool_of(*cache), batch_of(*batch), static_cast<const uint16_t *>(k),
                      static_cast<const uint16_t *>(v), k_stride, v_stride};
    a.pool.k += layer * cache->layer_stride;
    a.pool.v += layer * cache->layer_stride;
    const uint64_t grid = std::min<uint64_t>((batch->rows + 3ull) / 4, rt->compute_units * 8ull);
    return launch(rt, cache->head_dim == 128 ? "xpu_cache_append_d128" : "xpu_cache_append_d64", grid, a);
  });
}

int xpu_tree_attention_workspace(const xpu_runtime *rt, const xpu_cache *cache, const xpu_batch *batch, uint32_t heads,
                                 uint64_t *bytes) {
  static constexpr char name[] = "xpu_tree_attention_workspace";
  return guarded(name, [&] {
    if (!bytes) return invalid(name, "null output");
    if (int rc = check_cache(name, cache, false)) return rc;
    if (int rc = check_batch(name, batch, false)) return rc;
    if (int rc = check_heads(name, heads, cache->kv_heads, 1.0f)) return rc;
    if (int rc = check_runtime(name, rt)) return rc;
    *bytes = batch->rows && batch->n_seqs ? tree_plan(*rt, *cache, *batch, heads).bytes : 0;
    return XPU_OK;
  });
}

int xpu_tree_attention(xpu_runtime *rt, const xpu_cache *cache, const xpu_batch *batch, uint32_t layer, uint32_t heads,
                       float scale, const void *q, uint64_t q_stride, const uint64_t *visible, void *out,
                       uint64_t out_stride, void *workspace, uint64_t workspace_bytes) {
  static constexpr char name[] = "xpu_tree_attention";
  return guarded(name, [&] {
    if (int rc = check_cache(name, cache, true)) return rc;
    if (int rc = check_batch(name, batch, true)) return rc;
    if (layer >= cache->layers) return invalid(name, "no such layer");
    if (int rc = check_heads(name, heads, cache->kv_heads, scale)) return rc;
    if (!batch->rows || !batch->n_seqs) return check_runtime(name, rt);
    const uint64_t width = static_cast<uint64_t>(heads) * cache->head_dim;
    if (int rc = check_rows(name, "q", q, q_stride, width)) return rc;
    if (int rc = check_rows(name, "out", out, out_stride, width)) return rc;
    if (!aligned(visible, 8)) return invalid(name, "visible must be 8-byte aligned");
    if (rows_overlap(batch->rows, width, q, q_stride, out, out_stride))
      return invalid(name, "out must not overlap q");
    if (static_cast<uint64_t>(batch->rows) * heads >= (1ull << 26)) return invalid(name, "too many rows");
    if (int rc = check_runtime(name, rt)) return rc;
    const TreePlan plan = tree_plan(*rt, *cache, *batch, heads);
    if (plan.bytes && (!workspace || !aligned(workspace, 16) || workspace_bytes < plan.bytes))
      return invalid(name, "needs a workspace of " + std::to_string(plan.bytes) + " bytes, 16-byte aligned");
    xpu::TreeArgs a{};
    a.pool = pool_of(*cache);
    a.pool.k += layer * cache->layer_stride;
    a.pool.v += layer * cache->layer_stride;
    a.batch = batch_of(*batch);
    a.q = static_cast<const uint16_t *>(q);
    a.out = static_cast<uint16_t *>(out);
    a.visible = visible;
    a.partial = static_cast<float *>(workspace);
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.heads = heads;
    a.fit = plan.fit;
    a.target = plan.target;
    a.least = plan.least;
    a.slots = static_cast<uint32_t>(plan.slots);
    a.scale_log2e = static_cast<float>(scale * kLog2e);
    const std::string form = std::string("_") + type_name(cache->dtype) + "_d" + std::to_string(cache->head_dim) +
                             "_r" + std::to_string(plan.sub_tiles);
    if (int rc = launch(rt, "xpu_tree_attention" + form, plan.slots * cache->kv_heads, a)) return rc;
    if (!plan.bytes) return XPU_OK;
    const std::string join = "xpu_tree_join" + form + "_w" + std::to_string(plan.join_waves);
    return plan.join_waves > 1 ? launch(rt, join, plan.joins, a, 1, nullptr, 64 * plan.join_waves)
                               : launch(rt, join, (plan.joins + 3) / 4, a);
  });
}

int xpu_cache_keep(xpu_runtime *rt, const xpu_cache *cache, const xpu_batch *batch, const uint32_t *kept,
                   const uint32_t *counts, uint32_t *new_context) {
  static constexpr char name[] = "xpu_cache_keep";
  return guarded(name, [&] {
    if (int rc = check_cache(name, cache, true)) return rc;
    if (int rc = check_batch(name, batch, true, false)) return rc;
    if (!batch->n_seqs) return check_runtime(name, rt);
    if ((!kept && batch->rows) || !counts) return invalid(name, "null argument");
    if (!aligned(kept, 4) || !aligned(counts, 4) || !aligned(new_context, 4))
      return invalid(name, "kept, counts and new_context must be 4-byte aligned");
    const uint64_t list = 4ull * batch->n_seqs;
    if (new_context && (overlap(new_context, list, batch->context, list) || overlap(new_context, list, counts, list) ||
                        overlap(new_context, list, batch->starts, list + 4) ||
                        (kept && overlap(new_context, list, kept, 4ull * batch->rows))))
      return invalid(name, "new_context must not overlap context, counts, starts or kept");
    if (int rc = check_runtime(name, rt)) return rc;
    const xpu::KeepArgs a{pool_of(*cache), batch_of(*batch), kept, counts, new_context};
    const uint64_t groups = (static_cast<uint64_t>(cache->layers) * cache->kv_heads * 2 + 3) / 4;
    return launch(rt, cache->head_dim == 128 ? "xpu_cache_keep_d128" : "xpu_cache_keep_d64", batch->n_seqs * groups, a);
  });
}

int xpu_cache_copy(xpu_runtime *rt, const xpu_cache *cache, const uint32_t *src, const uint32_t *dst, uint32_t n) {
  static constexpr char name[] = "xpu_cache_copy";
  return guarded(name, [&] {
    if (int rc = check_cache(name, cache, true)) return rc;
    if (!n) return check_runtime(name, rt);
    if (!src || !dst) return invalid(name, "null argument");
    Ids to(n, cache->n_pages);
    for (uint32_t i = 0; i < n; ++i) {
      if (src[i] >= cache->n_pages || dst[i] >= cache->n_pages)
        return invalid(name, "page " + std::to_string(std::max(src[i], dst[i])) + " does not exist");
      if (!to.add(dst[i])) return invalid(name, "page " + std::to_string(dst[i]) + " is copied to twice");
    }
    for (uint32_t i = 0; i < n; ++i)
      if (to.has(src[i])) return invalid(name, "page " + std::to_string(src[i]) + " is copied to and from");
    if (int rc = check_runtime(name, rt)) return rc;
    const uint32_t chunks = cache->kv_heads * cache->page_size * cache->head_dim / 8;
    // the pairs travel as kernel arguments, so many at a time
    for (uint32_t at = 0; at < n; at += xpu::kCopyPairs) {
      xpu::CopyArgs a{};
      a.pool = pool_of(*cache);
      a.n = std::min(n - at, xpu::kCopyPairs);
      std::copy(src + at, src + at + a.n, a.src);
      std::copy(dst + at, dst + at + a.n, a.dst);
      if (int rc = launch(rt, "xpu_cache_copy", static_cast<uint64_t>(a.n) * cache->layers * 2, a,
                          (chunks + 2047) / 2048, &chunks))
        return rc;
    }
    return XPU_OK;
  });
}

int xpu_prompt_attention(xpu_runtime *rt, const xpu_packed *p, const void *q, const void *k, const void *v, void *out) {
  static constexpr char name[] = "xpu_prompt_attention";
  return guarded(name, [&] {
    if (!p) return invalid(name, "null description");
    if (p->dtype != XPU_DTYPE_BF16 && p->dtype != XPU_DTYPE_FP16)
      return invalid(name, "dtype must be bf16 (0) or fp16 (1)");
    if (p->head_dim != 64 && p->head_dim != 128) return invalid(name, "head_dim must be 64 or 128");
    if (int rc = check_heads(name, p->heads, p->kv_heads, p->scale)) return rc;
    if (p->q_rows >> 31 || p->k_rows >> 31 || p->n_seqs >> 24)
      return invalid(name, "at most 2^31 - 1 rows and 2^24 - 1 sequences");
    if (!p->k_starts && p->k_rows != p->q_rows) return invalid(name, "k_rows must be q_rows without k_starts");
    if (!p->q_rows || !p->n_seqs) return check_runtime(name, rt);
    if (!p->q_starts || !aligned(p->q_starts, 4) || !aligned(p->k_starts, 4))
      return invalid(name, "q_starts must not be null, starts 4-byte aligned");
    const uint64_t q_width = static_cast<uint64_t>(p->heads) * p->head_dim,
                   k_width = static_cast<uint64_t>(p->kv_heads) * p->head_dim;
    if (int rc = check_rows(name, "q", q, p->q_stride, q_width)) return rc;
    if (int rc = check_rows(name, "out", out, p->out_stride, q_width)) return rc;
    if (p->k_rows) {  // without key rows no memory of theirs is needed
      if (int rc = check_rows(name, "k", k, p->k_stride, k_width)) return rc;
      if (int rc = check_rows(name, "v", v, p->v_stride, k_width)) return rc;
    }
    if (!(out == q && p->out_stride == p->q_stride) &&
        rows_overlap(p->q_rows, q_width, q, p->q_stride, out, p->out_stride))
      return invalid(name, "out must be q or not overlap it");
    if (int rc = check_runtime(name, rt)) return rc;
    xpu::PackedArgs a{};
    a.q = static_cast<const uint16_t *>(q);
    a.k = static_cast<const uint16_t *>(k);
    a.v = static_cast<const uint16_t *>(v);
    a.out = static_cast<uint16_t *>(out);
    a.q_starts = p->q_starts;
    a.k_starts = p->k_starts ? p->k_starts : p->q_starts;
    a.q_stride = p->q_stride;
    a.k_stride = p->k_stride;
    a.v_stride = p->v_stride;
    a.out_stride = p->out_stride;
    a.n_seqs = p->n_seqs;
    a.q_rows = p->q_rows;
    a.k_rows = p->k_rows;
    a.heads = p->heads;
    a.kv_heads = p->kv_heads;
    a.scale_log2e = static_cast<float>(p->scale * kLog2e);
    // heads of a kv head that a block takes together, one or more wavefronts each
    const uint32_t group = p->heads / p->kv_heads;
    a.pack_shift = group % 4 == 0 ? 2 : group % 2 == 0 ? 1 : 0;
    a.slots = p->q_rows / (128u >> a.pack_shift) + p->n_seqs;
    return launch(rt, std::string("xpu_packed_attention_") + type_name(p->dtype) + "_d" + std::to_string(p->head_dim),
                  static_cast<uint64_t>(a.slots) * (p->heads >> a.pack_shift), a);
  });
}

// For the tests of the kernels' checks, on host arrays: the element that
// position `pos` of a table has in a layer (2^64 - 1: none), and a sequence's
// lengths {first row, rows, context, end, bad}. Not part of the C ABI.
uint64_t xpu_internal_cache_element(uint32_t page_size, uint32_t n_pages, uint64_t page_stride, const uint32_t *table,
                                    uint32_t pitch, uint64_t pos, uint32_t head_dim) {
  xpu::PoolArgs p{};
  p.page_size = page_size;
  p.page_shift = static_cast<uint32_t>(__builtin_ctz(page_size));
  p.n_pages = n_pages;
  p.page_stride = page_stride;
  return xpu::element_of(p, table, pitch, pos, head_dim);
}

void xpu_internal_cache_lengths(uint32_t lo, uint32_t hi, uint32_t context, uint32_t rows, uint32_t pitch,
                                uint32_t page_size, uint32_t *out) {
  const xpu::Lengths s = xpu::lengths_of(lo, hi, context, rows, pitch, page_size);
  out[0] = s.first;
  out[1] = s.n;
  out[2] = s.context;
  out[3] = s.end;
  out[4] = s.bad;
}

}  // extern "C"
