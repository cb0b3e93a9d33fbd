// Kernel arguments of the sampling, filled by the host (sample_api.cpp), and
// its workspace.
#pragma once

#include <stdint.h>

namespace xpu {

// Places of a part's histogram, entries of its list, threads of a block of the
// first two launches and of the last, parts of a row at most.
constexpr uint32_t kSampleSlots = 2048, kSampleCap = 4096, kSampleThreads = 1024, kSampleDraw = 256, kSampleParts = 16;

struct SampleArgs {
  const void *logits;
  uint64_t stride;  // elements
  const float *temperature, *top_p, *min_p, *random;
  const uint32_t *top_k;
  uint32_t *tokens;
  float *probability;
  uint32_t vocab;
  uint32_t fine;  // weights are in units of 2^-fine
  // Rows are looked through by `parts` blocks each (a power of two; 0: by the
  // drawing block alone), `chunk` tokens to each. Of every row's part: the
  // place of its first token, or ~0 for a logit that is NaN or +infinity; the
  // entries of its list; the list; the weights and numbers of its tokens by
  // bins. Of every row: the largest logits of 1024 groups of threads.
  uint32_t parts, chunk;
  uint64_t *firsts, *lists, *weights;
  uint32_t *listed, *numbers;
  float *groups;
};

}  // namespace xpu
