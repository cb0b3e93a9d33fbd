// Kernel arguments of the sampling, filled by the host (sample_api.cpp).
#pragma once

#include <stdint.h>

namespace xpu {

struct SampleArgs {
  const void *logits;
  uint64_t stride;  // elements
  const float *temperature, *top_p, *min_p, *random;
  const uint32_t *top_k;
  uint32_t *tokens;
  float *probability;
  uint32_t vocab, bits;
};

}  // namespace xpu
