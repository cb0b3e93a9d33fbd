// Entry points of the sampling (include/xpu_sample.h): argument checks and the
// launch. Kernel: kernels/sample.hip.
#include "../../include/xpu_sample.h"
#include "cache_checks.hpp"
#include "kernels/sample_types.hpp"

using xpu::guarded;
using xpu::set_error;
using namespace xpu::checks;

namespace {

int check_sampling(const char *name, const xpu_sampling *s, bool memory) {
  if (!s) return invalid(name, "null description");
  if (s->dtype != XPU_DTYPE_BF16 && s->dtype != XPU_DTYPE_FP16 && s->dtype != XPU_DTYPE_FP32)
    return invalid(name, "dtype must be bf16 (0), fp16 (1) or fp32 (2)");
  if (!s->vocab || s->vocab > 1u << 20) return invalid(name, "vocab must be positive, at most 2^20");
  if (s->rows > kMostBlocks / 4) return invalid(name, "at most 2^22 rows");
  if (!memory || !s->rows) return XPU_OK;
  if (s->stride < s->vocab || s->stride >> 40) return invalid(name, "stride must be at least vocab and below 2^40 elements");
  if (!s->random) return invalid(name, "null random");
  if (!aligned(s->random, 4) || !aligned(s->temperature, 4) || !aligned(s->top_k, 4) || !aligned(s->top_p, 4) ||
      !aligned(s->min_p, 4))
    return invalid(name, "the numbers of the rows must be 4-byte aligned");
  return XPU_OK;
}

}  // namespace

extern "C" {

int xpu_sample_workspace(const xpu_runtime *rt, const xpu_sampling *sampling, uint64_t *bytes) {
  static constexpr char name[] = "xpu_sample_workspace";
  return guarded(name, [&] {
    if (!bytes) return invalid(name, "null output");
    if (int rc = check_sampling(name, sampling, false)) return rc;
    if (int rc = check_runtime(name, rt)) return rc;
    *bytes = 0;
    return XPU_OK;
  });
}

int xpu_sample(xpu_runtime *rt, const xpu_sampling *sampling, const void *logits, uint32_t *tokens, float *probability,
               void *workspace, uint64_t workspace_bytes) {
  static constexpr char name[] = "xpu_sample";
  return guarded(name, [&] {
    if (int rc = check_sampling(name, sampling, true)) return rc;
    const xpu_sampling &s = *sampling;
    if (!s.rows) return check_runtime(name, rt);
    const uint32_t size = s.dtype == XPU_DTYPE_FP32 ? 4 : 2;
    if (!logits || !aligned(logits, size)) return invalid(name, "logits must not be null, aligned to their elements");
    if (!tokens || !aligned(tokens, 4) || !aligned(probability, 4))
      return invalid(name, "tokens must not be null, tokens and probability 4-byte aligned");
    const uint64_t list = 4ull * s.rows, span = ((s.rows - 1ull) * s.stride + s.vocab) * size;
    const void *const outs[] = {tokens, probability}, *const ins[] = {s.random, s.temperature, s.top_k, s.top_p, s.min_p};
    if (probability && overlap(tokens, list, probability, list)) return invalid(name, "tokens and probability overlap");
    for (const void *o : outs) {
      if (!o) continue;
      if (overlap(o, list, logits, span)) return invalid(name, "tokens and probability must not overlap the logits");
      for (const void *i : ins)
        if (i && overlap(o, list, i, list))
          return invalid(name, "tokens and probability must not overlap the numbers of the rows");
    }
    if (int rc = check_runtime(name, rt)) return rc;
    (void)workspace;
    (void)workspace_bytes;
    xpu::SampleArgs a{};
    a.logits = logits;
    a.stride = s.stride;
    a.temperature = s.temperature;
    a.top_k = s.top_k;
    a.top_p = s.top_p;
    a.min_p = s.min_p;
    a.random = s.random;
    a.tokens = tokens;
    a.probability = probability;
    a.vocab = s.vocab;
    a.bits = 62;
    while ((1ull << (62 - a.bits)) < s.vocab) --a.bits;
    const char *kernel = s.dtype == XPU_DTYPE_FP32 ? "xpu_sample_fp32" : s.dtype == XPU_DTYPE_FP16 ? "xpu_sample_fp16" : "xpu_sample_bf16";
    return launch(rt, kernel, s.rows, a, 1, nullptr, 1024);
  });
}

}  // extern "C"
