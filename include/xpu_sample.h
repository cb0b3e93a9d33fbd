/*
 * xpu_sample.h - the next tokens of a batch from their logits and given random
 * numbers on gfx950 (C ABI). The reference takes the largest logit
 * (QwenArgmax, qwen3/kernels.hpp:194-227); with temperature 0 so does this.
 *
 * Conventions as xpu_kernels.h: asynchronous on the runtime's stream, nothing
 * allocated and nothing read on the host, so a call can be captured.
 */
#ifndef XPU_SAMPLE_H
#define XPU_SAMPLE_H

#include "xpu_kernels.h"

#ifdef __cplusplus
extern "C" {
#endif

#define XPU_DTYPE_FP32 2

/* What is drawn of a row when the row has no answer: a logit is NaN or
 * +infinity, all are -infinity, or a number of the row is outside its range. */
#define XPU_SAMPLE_NONE 0xffffffffu

/* Row r: the tokens in order of their logits, equal ones by id, the lowest
 * first, with weights w = exp((logit - largest) / temperature). Kept is the
 * shortest of these beginnings of the order, which is one token at least:
 *   top_k  tokens (0: all);
 *   the fewest tokens that have top_p of the weight of the top_k first (1 or
 *          more: all);
 *   those with w >= min_p (0: all).
 * The token is the first of the order at which the weights up to it pass random
 * times the kept ones' sum. Temperature 0 keeps the first token alone. A logit
 * of -infinity is never drawn. The numbers of the rows are on the device, one
 * per row; NULL is temperature 1, or no filter. Weights are formed in 64 bits
 * and summed as integers, off by 2^-41 of the largest weight per token at most
 * (2^-44 up to 2^17 tokens); weights below 2^-47 of the largest may count as 0. A
 * row's token does not depend on what the rows beside it hold. How a row is summed
 * goes by the numbers of rows and tokens, so with other numbers of rows it may be
 * drawn otherwise where random times the sum is that near to a token's border. */
typedef struct {
  int32_t dtype;            /* of the logits: XPU_DTYPE_BF16, _FP16 or _FP32 */
  uint32_t rows;
  uint32_t vocab;           /* tokens of a row, at most 2^20 */
  uint64_t stride;          /* elements between rows, at least vocab; any */
  const float *temperature; /* >= 0, finite */
  const uint32_t *top_k;
  const float *top_p;       /* >= 0 */
  const float *min_p;       /* 0 .. 1 */
  const float *random;      /* >= 0 and below 1; not NULL */
} xpu_sampling;

/* tokens: `rows` entries. probability (or NULL): of each token drawn, its share
 * of the kept weight (NaN with XPU_SAMPLE_NONE). logits aligned to their
 * elements, the others to 4 bytes. workspace: at least what
 * xpu_sample_workspace gives for the same dtype, rows and vocab, 16-byte
 * aligned, used from the call to its end on the stream; calls on one stream may
 * share it, graphs captured from it too. */
int xpu_sample(xpu_runtime *rt, const xpu_sampling *sampling, const void *logits, uint32_t *tokens, float *probability,
               void *workspace, uint64_t workspace_bytes);
int xpu_sample_workspace(const xpu_runtime *rt, const xpu_sampling *sampling, uint64_t *bytes);

#ifdef __cplusplus
}
#endif
#endif
