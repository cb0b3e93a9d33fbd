/*
 * xpu_cache.h - a paged KV cache shared by many sequences on gfx950, and the
 * attention over it and over packed prompts (C ABI).
 *
 * The reference has one contiguous cache of one sequence
 * (qwen3/main.cpp:131-137), written by QwenQkvRopeCache and read by
 * QwenAttention (qwen3/kernels.hpp:128-192); these entry points are their
 * counterparts for several sequences, several query rows and shared pages.
 * They have no other counterpart in the reference.
 *
 * A step of a serving loop, layer by layer: xpu_cache_append the new rows,
 * xpu_tree_attention over all that the sequence holds (a token, a chain or a
 * tree of drafted tokens); after the last layer xpu_cache_keep moves the
 * accepted nodes to the front. A new prompt goes through
 * xpu_prompt_attention and xpu_cache_append. Which pages a sequence holds is
 * the caller's table; xpu_pages_* keeps count of them, and xpu_cache_copy
 * carries out the copies that forks and compaction ask for.
 *
 * Conventions: as xpu_kernels.h. Every launch is asynchronous on the
 * runtime's stream, allocates no device memory and reads none on the host,
 * so all of it can be captured (xpu_rt_capture_begin). Work of other streams
 * on the operands has to be ordered against the runtime's stream by the
 * caller. Operands are device pointers of the runtime's device, 16-byte
 * aligned where they hold rows, 4-byte (visible: 8-byte) aligned where they
 * hold numbers; what a call writes must not overlap what it reads, unless the
 * call says so. Row strides are in elements, multiples of 8. Host-side
 * arguments that are wrong fail with XPU_ERR_INVALID before any launch. The
 * numbers that live on the device (starts, context, tables, kept, counts)
 * are checked by the kernels: nothing outside the described buffers is read
 * or written whatever they hold, and what they make of wrong ones is said at
 * each call.
 */
#ifndef XPU_CACHE_H
#define XPU_CACHE_H

#include "xpu_kernels.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The pages. Element (layer, page, head, slot, dim) of K and of V lies at
 * layer * layer_stride + page * page_stride + (head * page_size + slot) *
 * head_dim + dim, 16-bit elements of `dtype`. */
typedef struct {
  int32_t dtype;          /* XPU_DTYPE_BF16 or XPU_DTYPE_FP16 */
  uint32_t layers, kv_heads;
  uint32_t head_dim;      /* 64 or 128 */
  uint32_t page_size;     /* positions per page: 16, 32, 64, 128 or 256 */
  uint32_t n_pages;       /* pages per layer; ids are 0 .. n_pages - 1 */
  uint64_t layer_stride, page_stride; /* elements, multiples of 8 */
  void *k, *v;
  uint32_t *status;       /* device, or NULL: set to 1 by a kernel that meets a
                             page id or a length that it cannot follow */
} xpu_cache;

/* Sequences with new rows. Sequence s has rows starts[s] .. starts[s + 1] - 1
 * of the row operands (none, one or many), at positions context[s], context[s]
 * + 1, ... of its cache; its position p lies in page tables[s * table_pitch +
 * p / page_size], slot p % page_size. starts (n_seqs + 1) ascend from any first
 * row; rows that belong to no sequence are left as they are. A sequence whose
 * starts descend or pass `rows` has no rows; rows that several sequences then
 * claim get any one's result or none. A table entry that no
 * position needs may hold anything. */
typedef struct {
  uint32_t n_seqs;
  uint32_t rows;          /* rows of the row operands */
  uint32_t table_pitch;   /* entries per sequence in tables */
  const uint32_t *tables, *starts, *context; /* device */
} xpu_batch;

/* Writes the batch's K and V rows ([kv_heads][head_dim] each, k_stride and
 * v_stride elements apart) into layer `layer` of the pages. Two rows must not
 * have the same place: a page that sequences share takes no new rows
 * (xpu_pages_own makes it one sequence's). A row whose page id is n_pages or
 * more, or whose position is past its table, is not written and sets status. */
int xpu_cache_append(xpu_runtime *rt, const xpu_cache *cache, const xpu_batch *batch, uint32_t layer,
                     const void *k, uint64_t k_stride, const void *v, uint64_t v_stride);

/* How new rows are turned on their way into a cache. Per head of Q and K,
 * in FP32 and rounded once:
 *   n = x * gain / sqrt(mean(x^2) + eps)         where there is a gain
 *   y_i = n_i cos - n_j sin,  y_j = n_j cos + n_i sin
 * for the dims / 2 pairs (i, j) of the first `dims` dims, pair by pair with the
 * entries of the row's position in the tables; the other dims stay n. */
#define XPU_ROTARY_HALVES 0   /* pair p: dims p and p + dims / 2 */
#define XPU_ROTARY_ADJACENT 1 /* pair p: dims 2 p and 2 p + 1 */
typedef struct {
  uint32_t positions;       /* rows of the tables */
  uint32_t dims;            /* a multiple of 16, at most head_dim */
  int32_t pairs;            /* XPU_ROTARY_HALVES or XPU_ROTARY_ADJACENT */
  float eps;                /* >= 0 */
  const float *cos, *sin;   /* device, [positions][dims / 2], 16-byte aligned */
  const uint32_t *at;       /* device, the position of each row of the batch (nodes of
                               a tree share depths); NULL: its position in the cache */
  const void *q_gain, *k_gain; /* device, [head_dim] of the cache's type, or NULL */
} xpu_rotary;

/* xpu_cache_append with Q and K normalised and rotated on the way. V is stored
 * as it is. heads > 0: Q ([rows][heads][head_dim], q_stride apart) is turned
 * too and goes to q_out, which may be q itself with its stride and otherwise
 * overlaps no input; heads 0: q and q_out are not looked at. A row whose
 * position is not in the tables is not written, its q_out is NaN, and sets
 * status; its q_out is written also where its place in the cache does not
 * exist. */
int xpu_cache_append_rotary(xpu_runtime *rt, const xpu_cache *cache, const xpu_batch *batch, uint32_t layer,
                            const xpu_rotary *rotary, uint32_t heads, const void *q, uint64_t q_stride, void *q_out,
                            uint64_t out_stride, const void *k, uint64_t k_stride, const void *v, uint64_t v_stride);

/* Attention of the batch's rows, which are in the cache already (appended):
 * a row sees all context[s] positions before the batch's and, of the
 * sequence's own rows ("nodes"), node j when bit j of visible[row] is set
 * (its own bit too, to see itself); at most 64 nodes per sequence then.
 * visible NULL: node i sees nodes 0 .. i, any number of nodes (a chain; with
 * one row, a decode step; with many, a further part of a prompt). A row that
 * sees nothing gives zeros. Keys that a row does not see take no part in it,
 * whatever they hold, NaN and infinities included.
 *   out[row][head] = softmax(scale * q . k) v,  head h on kv head h / (heads / kv_heads)
 * q and out: [rows][heads][head_dim] in the cache's type, rows q_stride and
 * out_stride elements apart; out must not overlap q (columns of one buffer, of
 * one stride, do not). FP32 scores, softmax and
 * sums; the probabilities are rounded to the cache's type for the product
 * with V. (The sums are of up to 2^8 times the values, so bf16 values above 2^119
 * / (keys) may become infinite.) scale > 0. A page id past n_pages, a context past
 * the table or 2^31 - 1 positions, or more than 64 nodes under `visible` makes the
 * rows of that sequence NaN and sets status. workspace: at least the size that xpu_tree_attention_workspace
 * gives for the same shapes, used from the call to its end on the stream;
 * calls on one stream may share it, graphs captured from it too. */
int xpu_tree_attention(xpu_runtime *rt, const xpu_cache *cache, const xpu_batch *batch, uint32_t layer,
                       uint32_t heads, float scale, const void *q, uint64_t q_stride, const uint64_t *visible,
                       void *out, uint64_t out_stride, void *workspace, uint64_t workspace_bytes);
/* The size, for any lengths and contexts of n_seqs sequences and `rows` rows
 * (host only; the pointers of cache and batch are not looked at). */
int xpu_tree_attention_workspace(const xpu_runtime *rt, const xpu_cache *cache, const xpu_batch *batch,
                                 uint32_t heads, uint64_t *bytes);

/* The accepted nodes of each sequence's rows move to the front, in all
 * layers: new position context[s] + j = what position context[s] + kept[
 * starts[s] + j] held before the call, for j < counts[s] (at most 64 and at
 * most the sequence's rows). kept names nodes 0 .. 63 of the sequence's rows,
 * in any order and more than once if need be. The
 * positions behind the kept ones hold what they held. kept has `rows` entries;
 * those past a sequence's count are not looked at. new_context (NULL, or
 * n_seqs entries apart from context): context[s] + counts[s]. A sequence with
 * a count that does not fit is left alone, its new_context too, and so is a row with a node or a
 * page that does not exist; both set status. The pages of the batch's rows
 * must be the sequence's own. */
int xpu_cache_keep(xpu_runtime *rt, const xpu_cache *cache, const xpu_batch *batch, const uint32_t *kept,
                   const uint32_t *counts, uint32_t *new_context);

/* Copies page src[i] to page dst[i] in all layers, i < n. src and dst are
 * HOST arrays, read before the call returns. Every id is below n_pages, no
 * page is copied to twice, and no page copied to is copied from. */
int xpu_cache_copy(xpu_runtime *rt, const xpu_cache *cache, const uint32_t *src, const uint32_t *dst, uint32_t n);

/* Packed prompts. Sequence s has query rows q_starts[s] .. q_starts[s + 1] - 1
 * and key rows k_starts[s] .. k_starts[s + 1] - 1; its last query sees all of
 * its keys, the one before one key less, and so on: with fewer queries than
 * keys the first keys are an earlier part of the prompt. k_starts NULL: the
 * same rows. A query that sees no key gives zeros. Rows that belong to no
 * sequence are left as they are; so are those of a sequence whose starts do
 * not ascend or pass the rows; rows that several sequences claim get any one's
 * result or none. */
typedef struct {
  int32_t dtype;
  uint32_t heads, kv_heads, head_dim; /* head_dim 64 or 128 */
  uint32_t n_seqs, q_rows, k_rows;
  float scale;                        /* > 0 */
  const uint32_t *q_starts, *k_starts; /* device, n_seqs + 1 entries */
  uint64_t q_stride, k_stride, v_stride, out_stride; /* elements, multiples of 8 */
} xpu_packed;

/* out[row][head] = softmax(scale * q . k) v as xpu_tree_attention, causal
 * within each sequence. q, out: [q_rows][heads][head_dim]; k, v: [k_rows][
 * kv_heads][head_dim]. out may be q itself with its stride; otherwise it must
 * not overlap an input (columns of one buffer, of one stride, do not). */
int xpu_prompt_attention(xpu_runtime *rt, const xpu_packed *packed, const void *q, const void *k, const void *v,
                         void *out);

/* ---- which pages are in use (host only, no device work) ----
 * A page has as many holders as sequences have it in their table. Ids are
 * given out lowest first. A call that fails changes nothing. Not
 * thread-safe. */
typedef struct xpu_pages xpu_pages;
int xpu_pages_create(uint32_t n_pages, xpu_pages **out);
void xpu_pages_destroy(xpu_pages *pages);
int xpu_pages_free_count(const xpu_pages *pages, uint32_t *count);
int xpu_pages_holders(const xpu_pages *pages, uint32_t id, uint32_t *count);
/* n free pages, one holder each; XPU_ERR_DEVICE when fewer are free. */
int xpu_pages_take(xpu_pages *pages, uint32_t n, uint32_t *ids);
/* One holder more for each (a fork's table holds the same pages). */
int xpu_pages_share(xpu_pages *pages, const uint32_t *ids, uint32_t n);
/* One holder less for each; a page without holders is free. */
int xpu_pages_release(xpu_pages *pages, const uint32_t *ids, uint32_t n);
/* Makes the pages the caller's alone: each id with other holders is replaced
 * in ids by a free page (it loses this holder), and src / dst (room for n
 * each) list the *copies to carry out with xpu_cache_copy. XPU_ERR_DEVICE
 * when too few are free. */
int xpu_pages_own(xpu_pages *pages, uint32_t *ids, uint32_t n, uint32_t *src, uint32_t *dst, uint32_t *copies);
/* Moves the pages in use to the ids 0 .. (pages in use) - 1: src / dst (room
 * for n_pages each) list the *moves for xpu_cache_copy, the fewest there are;
 * holders move along. xpu_pages_renumber then replaces the moved ids in a
 * table. */
int xpu_pages_compact(xpu_pages *pages, uint32_t *src, uint32_t *dst, uint32_t *moves);
int xpu_pages_renumber(const uint32_t *src, const uint32_t *dst, uint32_t moves, uint32_t *ids, uint32_t n);

#ifdef __cplusplus
}
#endif
#endif
