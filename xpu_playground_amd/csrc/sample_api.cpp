// Entry points of the sampling (include/xpu_sample.h): argument checks and the
// launches. Kernels: kernels/sample.hip.
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

// How a call is cut (kernels/sample.hip), by the numbers of rows and tokens
// alone: parts of a row, 0 for one launch.
struct SamplePlan {
  uint32_t parts = 0, chunk = 0;
  uint64_t firsts = 0, lists = 0, weights = 0, numbers = 0, listed = 0, groups = 0, bytes = 0;  // offsets; in all
};

SamplePlan sample_plan(const xpu_runtime &rt, const xpu_sampling &s) {
  SamplePlan p;
  if (s.vocab < 16384) return p;
  p.parts = 1;
  while (p.parts < xpu::kSampleParts && 2ull * p.parts * s.rows <= rt.compute_units &&
         s.vocab / (2 * p.parts) >= 4096)
    p.parts *= 2;
  p.chunk = (s.vocab + 8 * p.parts - 1) / (8 * p.parts) * 8;
  const uint64_t blocks = static_cast<uint64_t>(s.rows) * p.parts;
  p.lists = p.firsts + 8 * blocks;
  p.weights = p.lists + 8 * blocks * xpu::kSampleCap;
  p.numbers = p.weights + 8 * blocks * xpu::kSampleSlots;
  p.listed = p.numbers + 4 * blocks * xpu::kSampleSlots;
  p.groups = p.listed + 4 * blocks;
  p.bytes = p.groups + 4ull * s.rows * xpu::kSampleThreads;
  return p;
}

}  // namespace

extern "C" {

int xpu_sample_workspace(const xpu_runtime *rt, const xpu_sampling *sampling, uint64_t *bytes) {
  static constexpr char name[] = "xpu_sample_workspace";
  return guarded(name, [&] {
    if (!bytes) return invalid(name, "null output");
    if (int rc = check_sampling(name, sampling, false)) return rc;
    if (int rc = check_runtime(name, rt)) return rc;
    *bytes = sampling->rows ? sample_plan(*rt, *sampling).bytes : 0;
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
    const SamplePlan plan = sample_plan(*rt, s);
    if (plan.bytes && (!workspace || !aligned(workspace, 16) || workspace_bytes < plan.bytes))
      return invalid(name, "needs a workspace of " + std::to_string(plan.bytes) + " bytes, 16-byte aligned");
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
    a.fine = 44;
    while ((1ull << (61 - a.fine)) < s.vocab) --a.fine;
    const std::string form =
        s.dtype == XPU_DTYPE_FP32 ? "_fp32" : s.dtype == XPU_DTYPE_FP16 ? "_fp16" : "_bf16";
    if (plan.parts) {
      uint8_t *w = static_cast<uint8_t *>(workspace);
      a.parts = plan.parts;
      a.chunk = plan.chunk;
      a.firsts = reinterpret_cast<uint64_t *>(w + plan.firsts);
      a.lists = reinterpret_cast<uint64_t *>(w + plan.lists);
      a.weights = reinterpret_cast<uint64_t *>(w + plan.weights);
      a.numbers = reinterpret_cast<uint32_t *>(w + plan.numbers);
      a.listed = reinterpret_cast<uint32_t *>(w + plan.listed);
      a.groups = reinterpret_cast<float *>(w + plan.groups);
      const uint64_t blocks = static_cast<uint64_t>(s.rows) * plan.parts;
      if (int rc = launch(rt, "xpu_sample_look" + form, blocks, a, 1, nullptr, xpu::kSampleThreads)) return rc;
      if (int rc = launch(rt, "xpu_sample_list" + form, blocks, a, 1, nullptr, xpu::kSampleThreads)) return rc;
    }
    return launch(rt, "xpu_sample_draw" + form, s.rows, a, 1, nullptr, xpu::kSampleDraw);
  });
}

}  // extern "C"
