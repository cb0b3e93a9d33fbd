/*
 * xpu_cache8.h - the paged KV cache of xpu_cache.h in 8 bits (C ABI): half the
 * memory per position, and half the bytes that attention reads.
 *
 * The calls, the batch, the tables and the counting of pages (xpu_pages_*) are
 * those of xpu_cache.h, with its conventions. They have no counterpart in the
 * reference.
 *
 * A position's K and V are codes of 8 bits (e4m3: 4 significant bits, largest
 * 448) times a scale that 16 positions of a kv head share, a power of two. A
 * block of 16 positions gets the smallest scale with which all finite values of
 * the rows that come to it in one call are at most 448 codes (2^-100 at least),
 * or keeps its scale where it holds earlier positions of the sequence and that is
 * larger: a scale never falls while they stay. Where it grows, their codes are
 * rounded once more to the new one. So a block's scale is that of the largest row
 * that came to it since its first, rejected rows included, or that came to a block
 * of which xpu_cache8_keep moved a row here; that row's largest value is above 224
 * scales (or the scale 2^-100). A value is off by 2^-4 of itself and 2^-9 of its
 * block's scale at most. Infinities and NaN are stored as NaN; a value whose code
 * stands for more than the largest number of `dtype` reads as infinite.
 */
#ifndef XPU_CACHE8_H
#define XPU_CACHE8_H

#include "xpu_cache.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The pages. Of page `page` in layer `layer`, which begins at layer *
 * layer_stride + page * page_stride, the code of (head, slot, dim) is byte
 * (head * page_size + slot) * head_dim + dim, and the scale of (head, slots 16 b
 * ... 16 b + 15) is byte kv_heads * page_size * head_dim + head * (page_size /
 * 16) + b: 2^(byte - 127). Scales are only what these calls wrote. */
typedef struct {
  int32_t dtype;          /* of the rows: XPU_DTYPE_BF16 or XPU_DTYPE_FP16 */
  uint32_t layers, kv_heads;
  uint32_t head_dim;      /* 64 or 128 */
  uint32_t page_size;     /* positions per page: 16, 32, 64, 128 or 256 */
  uint32_t n_pages;       /* pages per layer; ids are 0 .. n_pages - 1 */
  uint64_t layer_stride, page_stride; /* bytes, multiples of 16 (of 128: no line of
                                         memory is in two pages) */
  void *k, *v;            /* 16-byte aligned */
  uint32_t *status;       /* as of xpu_cache */
} xpu_cache8;

/* The bytes of a page, codes and scales: the least page_stride (host only; the
 * pointers and strides of the cache are not looked at). */
int xpu_cache8_page_bytes(const xpu_cache8 *cache, uint64_t *bytes);

/* xpu_cache_append_rotary into 8 bits, K and V rounded from FP32 to codes.
 * rotary NULL: K as it is, and heads is 0. A row that is not written takes no
 * part in its block's scale. The pages of the batch's rows must be the
 * sequence's own, as for xpu_cache_append. */
int xpu_cache8_append(xpu_runtime *rt, const xpu_cache8 *cache, const xpu_batch *batch, uint32_t layer,
                      const xpu_rotary *rotary, uint32_t heads, const void *q, uint64_t q_stride, void *q_out,
                      uint64_t out_stride, const void *k, uint64_t k_stride, const void *v, uint64_t v_stride);

/* xpu_tree_attention over 8-bit pages: the same arguments and results, over
 * what the codes and scales stand for, rounded to `dtype` (exact in bf16, and in
 * fp16 from 2^-14 on). */
int xpu_tree_attention8(xpu_runtime *rt, const xpu_cache8 *cache, const xpu_batch *batch, uint32_t layer,
                        uint32_t heads, float scale, const void *q, uint64_t q_stride, const uint64_t *visible,
                        void *out, uint64_t out_stride, void *workspace, uint64_t workspace_bytes);
int xpu_tree_attention8_workspace(const xpu_runtime *rt, const xpu_cache8 *cache, const xpu_batch *batch,
                                  uint32_t heads, uint64_t *bytes);

/* xpu_cache_keep in 8 bits: the same arguments. A block that kept rows reach
 * gets the largest scale of its own and of the blocks that they come from; the
 * codes of the rows that come, of the sequence's rows before them, and of rows
 * left alone as their node does not exist, are rounded to it where it is larger
 * than theirs. The positions behind the kept ones hold nothing of use. */
int xpu_cache8_keep(xpu_runtime *rt, const xpu_cache8 *cache, const xpu_batch *batch, const uint32_t *kept,
                    const uint32_t *counts, uint32_t *new_context);

/* xpu_cache_copy in 8 bits: codes and scales of whole pages. */
int xpu_cache8_copy(xpu_runtime *rt, const xpu_cache8 *cache, const uint32_t *src, const uint32_t *dst, uint32_t n);

#ifdef __cplusplus
}
#endif
#endif
