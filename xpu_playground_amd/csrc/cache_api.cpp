// Entry points of the paged cache and the attention over it and over packed
// prompts (include/xpu_cache.h): argument checks, the choice of a kernel, the
// launch. Kernels: kernels/packed_attention.hip, tree_attention.hip, cache.hip.
#include "../../include/xpu_cache.h"
#include "cache_checks.hpp"

using xpu::guarded;
using xpu::set_error;
using namespace xpu::checks;

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
    *bytes = batch->rows && batch->n_seqs ? tree_plan(*rt, false, cache->kv_heads, cache->page_size, cache->head_dim, *batch, heads).bytes : 0;
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
    const TreeRows rows{heads, scale, q, q_stride, visible, out, out_stride, workspace, workspace_bytes};
    if (int rc = check_tree_rows(name, rows, *batch, cache->head_dim)) return rc;
    if (int rc = check_runtime(name, rt)) return rc;
    xpu::PoolArgs pool = pool_of(*cache);
    pool.k += layer * cache->layer_stride;
    pool.v += layer * cache->layer_stride;
    return launch_tree(name, rt, false, pool, cache->dtype, cache->head_dim, *batch, rows);
  });
}

int xpu_cache_keep(xpu_runtime *rt, const xpu_cache *cache, const xpu_batch *batch, const uint32_t *kept,
                   const uint32_t *counts, uint32_t *new_context) {
  static constexpr char name[] = "xpu_cache_keep";
  return guarded(name, [&] {
    if (int rc = check_cache(name, cache, true)) return rc;
    if (int rc = check_keep(name, batch, kept, counts, new_context)) return rc;
    if (int rc = check_runtime(name, rt)) return rc;
    if (!batch->n_seqs) return XPU_OK;
    const xpu::KeepArgs a{pool_of(*cache), batch_of(*batch), kept, counts, new_context};
    const uint64_t groups = (static_cast<uint64_t>(cache->layers) * cache->kv_heads * 2 + 3) / 4;
    return launch(rt, cache->head_dim == 128 ? "xpu_cache_keep_d128" : "xpu_cache_keep_d64", batch->n_seqs * groups, a);
  });
}

int xpu_cache_copy(xpu_runtime *rt, const xpu_cache *cache, const uint32_t *src, const uint32_t *dst, uint32_t n) {
  static constexpr char name[] = "xpu_cache_copy";
  return guarded(name, [&] {
    if (int rc = check_cache(name, cache, true)) return rc;
    if (int rc = check_copy(name, cache->n_pages, src, dst, n)) return rc;
    if (int rc = check_runtime(name, rt)) return rc;
    return launch_copy(rt, pool_of(*cache), cache->kv_heads * cache->page_size * cache->head_dim / 8, src, dst, n);
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
