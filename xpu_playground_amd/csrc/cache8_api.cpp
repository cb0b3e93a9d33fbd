// Entry points of the rotated append and of the 8-bit paged cache
// (include/xpu_cache.h, xpu_cache8.h): argument checks, the choice of a kernel,
// the launch. Kernels: kernels/rotary.hip, tree_attention8.hip, cache8.hip, and
// of cache.hip the copy.
#include "../../include/xpu_cache8.h"
#include "cache_checks.hpp"

using xpu::guarded;
using xpu::set_error;
using namespace xpu::checks;

namespace {

uint64_t page_bytes(const xpu_cache8 &c) {
  const uint64_t codes = static_cast<uint64_t>(c.kv_heads) * c.page_size * c.head_dim;
  return (codes + c.kv_heads * (c.page_size / xpu::kBlock) + 15) / 16 * 16;
}

int check_cache8(const char *name, const xpu_cache8 *c, bool memory) {
  if (!c) return invalid(name, "null cache");
  const uint64_t page = c->page_size >= 16 && c->page_size <= 256 ? page_bytes(*c) : 16;
  const xpu_cache shape{c->dtype, c->layers,  c->kv_heads, c->head_dim, c->page_size, c->n_pages,
                        c->layer_stride, c->page_stride, c->k, c->v, c->status};
  if (int rc = check_shape(name, shape)) return rc;
  if (!memory) return XPU_OK;
  if (c->page_stride % 16 || c->layer_stride % 16) return invalid(name, "strides must be multiples of 16 bytes");
  return check_memory(name, shape, page, "bytes");
}

// One layer's pages; strides in bytes.
xpu::PoolArgs pool8_of(const xpu_cache8 &c, uint32_t layer) {
  xpu::PoolArgs p{};
  p.k = reinterpret_cast<uint16_t *>(static_cast<uint8_t *>(c.k) + layer * c.layer_stride);
  p.v = reinterpret_cast<uint16_t *>(static_cast<uint8_t *>(c.v) + layer * c.layer_stride);
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

int check_rotary(const char *name, const xpu_rotary *r, uint32_t head_dim) {
  if (!r) return invalid(name, "null rotary");
  if (r->pairs != XPU_ROTARY_HALVES && r->pairs != XPU_ROTARY_ADJACENT)
    return invalid(name, "pairs must be halves (0) or adjacent (1)");
  if (!r->positions || !r->dims || r->dims % 16 || r->dims > head_dim)
    return invalid(name, "positions must be positive, dims a positive multiple of 16, at most head_dim");
  if (!(r->eps >= 0) || !std::isfinite(r->eps)) return invalid(name, "eps must be finite and not negative");
  if (!r->cos || !r->sin || !aligned(r->cos, 16) || !aligned(r->sin, 16))
    return invalid(name, "cos and sin must not be null, 16-byte aligned");
  if (!aligned(r->at, 4)) return invalid(name, "at must be 4-byte aligned");
  if (!aligned(r->q_gain, 16) || !aligned(r->k_gain, 16)) return invalid(name, "gains must be 16-byte aligned");
  return XPU_OK;
}

// What both appends take besides the cache.
struct Rows {
  const xpu_batch *batch;
  const xpu_rotary *rotary;
  uint32_t heads;
  const void *q;
  uint64_t q_stride;
  void *q_out;
  uint64_t out_stride;
  const void *k;
  uint64_t k_stride;
  const void *v;
  uint64_t v_stride;
};

int check_new_rows(const char *name, const Rows &r, uint32_t kv_heads, uint32_t head_dim) {
  const uint64_t width = static_cast<uint64_t>(kv_heads) * head_dim, q_width = static_cast<uint64_t>(r.heads) * head_dim;
  if (int rc = check_rows(name, "k", r.k, r.k_stride, width)) return rc;
  if (int rc = check_rows(name, "v", r.v, r.v_stride, width)) return rc;
  if (!r.heads) return XPU_OK;
  if (int rc = check_rows(name, "q", r.q, r.q_stride, q_width)) return rc;
  if (int rc = check_rows(name, "q_out", r.q_out, r.out_stride, q_width)) return rc;
  if (!(r.q_out == r.q && r.out_stride == r.q_stride) &&
      rows_overlap(r.batch->rows, q_width, r.q, r.q_stride, q_width, r.q_out, r.out_stride))
    return invalid(name, "q_out must be q or not overlap it");
  if (rows_overlap(r.batch->rows, width, r.k, r.k_stride, q_width, r.q_out, r.out_stride) ||
      rows_overlap(r.batch->rows, width, r.v, r.v_stride, q_width, r.q_out, r.out_stride))
    return invalid(name, "q_out must not overlap k or v");
  return XPU_OK;
}

xpu::RotateArgs rotate_args(const xpu::PoolArgs &pool, const Rows &r) {
  xpu::RotateArgs a{};
  a.pool = pool;
  a.batch = batch_of(*r.batch);
  if (const xpu_rotary *t = r.rotary)
    a.rot = {t->cos, t->sin, t->at, static_cast<const uint16_t *>(t->q_gain), static_cast<const uint16_t *>(t->k_gain),
             t->positions, t->dims / 2, t->pairs == XPU_ROTARY_ADJACENT, t->eps};
  a.q = static_cast<const uint16_t *>(r.q);
  a.k = static_cast<const uint16_t *>(r.k);
  a.v = static_cast<const uint16_t *>(r.v);
  a.q_out = static_cast<uint16_t *>(r.q_out);
  a.q_stride = r.q_stride;
  a.k_stride = r.k_stride;
  a.v_stride = r.v_stride;
  a.out_stride = r.out_stride;
  a.heads = r.heads;
  return a;
}

// Wavefronts that share a row of `heads` heads: as many as there is work for
// while there are fewer than the chip holds, else each has what it loads at a
// time (kernels/rotary.hip).
uint32_t parts_of(const xpu_runtime &rt, uint32_t rows, uint32_t heads, uint32_t head_dim) {
  const uint64_t most = (heads * (head_dim / 8ull) + 63) / 64, room = rt.compute_units * 16ull / rows;
  return static_cast<uint32_t>(std::max<uint64_t>((most + 3) / 4, std::min(most, room)));
}

std::string form_of(int32_t dtype, uint32_t head_dim) {
  return std::string("_") + type_name(dtype) + "_d" + std::to_string(head_dim);
}

}  // namespace

extern "C" {

int xpu_cache_append_rotary(xpu_runtime *rt, const xpu_cache *cache, const xpu_batch *batch, uint32_t layer,
                            const xpu_rotary *rotary, uint32_t heads, const void *q, uint64_t q_stride, void *q_out,
                            uint64_t out_stride, const void *k, uint64_t k_stride, const void *v, uint64_t v_stride) {
  static constexpr char name[] = "xpu_cache_append_rotary";
  return guarded(name, [&] {
    if (int rc = check_cache(name, cache, true)) return rc;
    if (int rc = check_batch(name, batch, true)) return rc;
    if (layer >= cache->layers) return invalid(name, "no such layer");
    if (int rc = check_rotary(name, rotary, cache->head_dim)) return rc;
    if (heads > 65536) return invalid(name, "at most 65536 heads");
    if (!batch->rows || !batch->n_seqs) return check_runtime(name, rt);
    const Rows rows{batch, rotary, heads, q, q_stride, q_out, out_stride, k, k_stride, v, v_stride};
    if (int rc = check_new_rows(name, rows, cache->kv_heads, cache->head_dim)) return rc;
    if (int rc = check_runtime(name, rt)) return rc;
    xpu::RotateArgs a = rotate_args(pool_of(*cache), rows);
    a.pool.k += layer * cache->layer_stride;
    a.pool.v += layer * cache->layer_stride;
    a.parts = parts_of(*rt, batch->rows, heads + 2 * cache->kv_heads, cache->head_dim);
    const uint64_t waves = static_cast<uint64_t>(batch->rows) * a.parts;
    return launch(rt, "xpu_cache_append_rotary" + form_of(cache->dtype, cache->head_dim),
                  std::min<uint64_t>((waves + 3) / 4, rt->compute_units * 64ull), a);
  });
}

int xpu_cache8_page_bytes(const xpu_cache8 *cache, uint64_t *bytes) {
  static constexpr char name[] = "xpu_cache8_page_bytes";
  return guarded(name, [&] {
    if (!bytes) return invalid(name, "null output");
    if (int rc = check_cache8(name, cache, false)) return rc;
    *bytes = page_bytes(*cache);
    return XPU_OK;
  });
}

int xpu_cache8_append(xpu_runtime *rt, const xpu_cache8 *cache, const xpu_batch *batch, uint32_t layer,
                      const xpu_rotary *rotary, uint32_t heads, const void *q, uint64_t q_stride, void *q_out,
                      uint64_t out_stride, const void *k, uint64_t k_stride, const void *v, uint64_t v_stride) {
  static constexpr char name[] = "xpu_cache8_append";
  return guarded(name, [&] {
    if (int rc = check_cache8(name, cache, true)) return rc;
    if (int rc = check_batch(name, batch, true)) return rc;
    if (layer >= cache->layers) return invalid(name, "no such layer");
    if (rotary)
      if (int rc = check_rotary(name, rotary, cache->head_dim)) return rc;
    if (heads > 65536) return invalid(name, "at most 65536 heads");
    if (!rotary && heads) return invalid(name, "heads must be 0 without rotary");
    if (!batch->rows || !batch->n_seqs) return check_runtime(name, rt);
    const Rows rows{batch, rotary, heads, q, q_stride, q_out, out_stride, k, k_stride, v, v_stride};
    if (int rc = check_new_rows(name, rows, cache->kv_heads, cache->head_dim)) return rc;
    if (int rc = check_runtime(name, rt)) return rc;
    xpu::RotateArgs a = rotate_args(pool8_of(*cache, layer), rows);
    a.parts = heads ? parts_of(*rt, batch->rows, heads, cache->head_dim) : 0;
    // a sequence's n rows reach n / 16 + 2 blocks at most, and n
    a.slots = static_cast<uint32_t>(std::min<uint64_t>(batch->rows, batch->rows / xpu::kBlock + 2ull * batch->n_seqs));
    const uint64_t waves =
        2ull * cache->kv_heads * a.slots + static_cast<uint64_t>(batch->rows) * a.parts;
    return launch(rt, "xpu_cache8_append" + form_of(cache->dtype, cache->head_dim),
                  std::min<uint64_t>((waves + 3) / 4, rt->compute_units * 64ull), a);
  });
}

int xpu_tree_attention8_workspace(const xpu_runtime *rt, const xpu_cache8 *cache, const xpu_batch *batch,
                                  uint32_t heads, uint64_t *bytes) {
  static constexpr char name[] = "xpu_tree_attention8_workspace";
  return guarded(name, [&] {
    if (!bytes) return invalid(name, "null output");
    if (int rc = check_cache8(name, cache, false)) return rc;
    if (int rc = check_batch(name, batch, false)) return rc;
    if (int rc = check_heads(name, heads, cache->kv_heads, 1.0f)) return rc;
    if (int rc = check_runtime(name, rt)) return rc;
    *bytes = batch->rows && batch->n_seqs
                 ? tree_plan(*rt, true, cache->kv_heads, cache->page_size, cache->head_dim, *batch, heads).bytes
                 : 0;
    return XPU_OK;
  });
}

int xpu_tree_attention8(xpu_runtime *rt, const xpu_cache8 *cache, const xpu_batch *batch, uint32_t layer,
                        uint32_t heads, float scale, const void *q, uint64_t q_stride, const uint64_t *visible,
                        void *out, uint64_t out_stride, void *workspace, uint64_t workspace_bytes) {
  static constexpr char name[] = "xpu_tree_attention8";
  return guarded(name, [&] {
    if (int rc = check_cache8(name, cache, true)) return rc;
    if (int rc = check_batch(name, batch, true)) return rc;
    if (layer >= cache->layers) return invalid(name, "no such layer");
    if (int rc = check_heads(name, heads, cache->kv_heads, scale)) return rc;
    if (!batch->rows || !batch->n_seqs) return check_runtime(name, rt);
    const TreeRows rows{heads, scale, q, q_stride, visible, out, out_stride, workspace, workspace_bytes};
    if (int rc = check_tree_rows(name, rows, *batch, cache->head_dim)) return rc;
    if (int rc = check_runtime(name, rt)) return rc;
    return launch_tree(name, rt, true, pool8_of(*cache, layer), cache->dtype, cache->head_dim, *batch,
                       rows);
  });
}

int xpu_cache8_keep(xpu_runtime *rt, const xpu_cache8 *cache, const xpu_batch *batch, const uint32_t *kept,
                    const uint32_t *counts, uint32_t *new_context) {
  static constexpr char name[] = "xpu_cache8_keep";
  return guarded(name, [&] {
    if (int rc = check_cache8(name, cache, true)) return rc;
    if (int rc = check_keep(name, batch, kept, counts, new_context)) return rc;
    if (int rc = check_runtime(name, rt)) return rc;
    if (!batch->n_seqs) return XPU_OK;
    xpu::Keep8Args a{{pool8_of(*cache, 0), batch_of(*batch), kept, counts, new_context}, 1};
    const uint64_t parts = static_cast<uint64_t>(cache->layers) * cache->kv_heads * 2, held = rt->compute_units * 8ull;
    // more blocks than run at once: each takes more, at most 64 (kernels/cache8.hip).
    // 48 drafts of 64 nodes, 8 kept: 12.6 us, with a part to a block 41.5; 16: 18 and
    // 45; 17, from which on a block's parts come one after the other: 37 and 46; 64: 39
    // and 50
    if (parts * batch->n_seqs > held)
      a.per_block = static_cast<uint32_t>(4 * std::min<uint64_t>(16, ((parts + 3) / 4 * batch->n_seqs + held - 1) / held));
    const uint64_t groups = (parts + a.per_block - 1) / a.per_block;
    return launch(rt, cache->head_dim == 128 ? "xpu_cache8_keep_d128" : "xpu_cache8_keep_d64", batch->n_seqs * groups, a);
  });
}

int xpu_cache8_copy(xpu_runtime *rt, const xpu_cache8 *cache, const uint32_t *src, const uint32_t *dst, uint32_t n) {
  static constexpr char name[] = "xpu_cache8_copy";
  return guarded(name, [&] {
    if (int rc = check_cache8(name, cache, true)) return rc;
    if (int rc = check_copy(name, cache->n_pages, src, dst, n)) return rc;
    if (int rc = check_runtime(name, rt)) return rc;
    xpu::PoolArgs pool = pool8_of(*cache, 0);
    pool.layer_stride /= 2;  // the kernel's are of 16-bit elements
    pool.page_stride /= 2;
    return launch_copy(rt, pool, static_cast<uint32_t>(page_bytes(*cache) / 16), src, dst, n);
  });
}

}  // extern "C"
