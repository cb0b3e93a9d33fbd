// The next token of every row from its logits and a random number (xpu_sample).
//
// The tokens of a row in order of their logits, the lowest id first among
// equals, with weights w = exp((logit - largest) / T), largest = 1. Each filter
// keeps a beginning of this order, so what is kept is the shortest of them, and
// the draw is the first token at which the weights up to it pass u times those
// of all kept ones:
//   top-k  k tokens
//   top-p  as many as have p of the weight of the first k
//   min-p  those with w >= m
// So all that is ever looked for is the place in the order where a count or a
// weight is reached.
//
// The weights are formed in 64 bits and summed as integers of 2^-bits (bits +
// log2 of the tokens is 62), so sums do not depend on their order and a sum of
// 2^17 tokens is off by 2^-28 of the largest one's weight at most.
//
// A block has a row. Few tokens (top-k up to kFew): the k-th largest of the
// threads' largest values bounds the k-th largest of all from below, so a
// second pass finds little more than k candidates, which are sorted. Else: a
// histogram of the weights by (largest - logit) / T, which is in the order's
// order, gives the bin of a place, whose tokens are then sorted; a bin of too
// many (equal ones, mostly) is divided further by the bits of logit and id.
#include "device_common.hpp"
#include "sample_types.hpp"

namespace xpu {
namespace sample {

constexpr uint32_t kThreads = 1024, kWaves = kThreads / 64;
constexpr uint32_t kBins = 2048, kList = 2048, kFew = 256;
constexpr float kSpan = 31.0f;  // weights below e^-31 < 2^-44 are in the last bin

enum : int { kFp32 = 2 };

// Values are compared as these: descending logits, then ascending ids.
XPU_DEVICE uint32_t ordered(float v) {
  const uint32_t u = __float_as_uint(v);
  return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}
XPU_DEVICE float of_ordered(uint32_t k) { return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu)); }
XPU_DEVICE uint64_t place_of(float v, uint32_t id) { return static_cast<uint64_t>(ordered(v)) << 32 | ~id; }

// 2^x for x <= 0 by the series of exp around the nearest integer, to 2^-52.
XPU_DEVICE double exp2_nonpos(double x) {
  x = __builtin_fmax(x, -1000.0);
  const double n = __builtin_rint(x), r = (x - n) * 0.693147180559945309417;
  double p = 1.0 / 6227020800.0;
  p = __builtin_fma(p, r, 1.0 / 479001600.0);
  p = __builtin_fma(p, r, 1.0 / 39916800.0);
  p = __builtin_fma(p, r, 1.0 / 3628800.0);
  p = __builtin_fma(p, r, 1.0 / 362880.0);
  p = __builtin_fma(p, r, 1.0 / 40320.0);
  p = __builtin_fma(p, r, 1.0 / 5040.0);
  p = __builtin_fma(p, r, 1.0 / 720.0);
  p = __builtin_fma(p, r, 1.0 / 120.0);
  p = __builtin_fma(p, r, 1.0 / 24.0);
  p = __builtin_fma(p, r, 1.0 / 6.0);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  return __builtin_amdgcn_ldexp(p, static_cast<int>(n));
}

struct Shared {
  uint64_t hist[kBins];   // weight of the bins up to each
  uint32_t count[kBins];  // tokens of them
  uint64_t list[kList];
  uint64_t wave[kWaves];
  uint64_t found[2];
  uint32_t listed, flag;
};

// Reductions and sums over the block; every thread calls them and gets the result.
template <typename T, typename Op> XPU_DEVICE T block_reduce(Shared &sh, T v, Op op) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v = op(v, __shfl_xor(v, d));
  __syncthreads();
  if (lane_id() == 0) reinterpret_cast<T *>(sh.wave)[threadIdx.x >> 6] = v;
  __syncthreads();
  v = reinterpret_cast<T *>(sh.wave)[0];
#pragma unroll
  for (uint32_t w = 1; w < kWaves; ++w) v = op(v, reinterpret_cast<T *>(sh.wave)[w]);
  return v;
}
// Sums of threads 0 .. own - 1.
XPU_DEVICE uint64_t block_before(Shared &sh, uint64_t v) {
  const uint64_t own = v;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint64_t o = __shfl_up(v, d);
    if (lane_id() >= static_cast<uint32_t>(d)) v += o;
  }
  __syncthreads();
  if (lane_id() == 63) sh.wave[threadIdx.x >> 6] = v;
  __syncthreads();
  for (uint32_t w = 0; w < threadIdx.x >> 6; ++w) v += sh.wave[w];
  return v - own;
}

// One row.
template <int DT> struct Row {
  static constexpr uint32_t kPer = DT == kFp32 ? 4 : 8;  // tokens of 16 bytes
  const uint8_t *logits;
  uint32_t vocab;
  float largest;
  double scale;     // log2 e / T
  float by;         // bins per logit
  uint32_t bits;

  // body(value, id) for the thread's share of the tokens, ids ascending.
  template <typename Body> XPU_DEVICE void each(Body &&body) const {
    const uint32_t chunks = vocab / kPer;
#pragma unroll 2
    for (uint32_t c = threadIdx.x; c < chunks; c += kThreads) {
      const u32x4 x = *reinterpret_cast<const u32x4_any *>(logits + static_cast<uint64_t>(c) * 16u);
      if constexpr (DT == kFp32) {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) body(__uint_as_float(x[i]) + 0.0f, c * 4u + i);
      } else {
        float f[8];
        unpack8<DT>(x, f);
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) body(f[i] + 0.0f, c * 8u + i);
      }
    }
    const uint32_t id = chunks * kPer + threadIdx.x;
    if (id < vocab) {
      if constexpr (DT == kFp32) body(reinterpret_cast<const float *>(logits)[id] + 0.0f, id);
      else body(decode<DT>(reinterpret_cast<const uint16_t *>(logits)[id]) + 0.0f, id);
    }
  }
  XPU_DEVICE double weight(float v) const {
    return exp2_nonpos((static_cast<double>(v) - static_cast<double>(largest)) * scale);
  }
  XPU_DEVICE uint64_t units(double w) const {
    return static_cast<uint64_t>(__builtin_rint(__builtin_amdgcn_ldexp(w, static_cast<int>(bits))));
  }
  XPU_DEVICE uint32_t bin(float v) const {
    return static_cast<uint32_t>(__builtin_fminf((largest - v) * by, static_cast<float>(kBins - 1u)));
  }
};

// Sorts list[0 .. n - 1] descending, the rest of the power of two above filled up.
XPU_DEVICE void sort_list(Shared &sh, uint32_t n) {
  uint32_t size = 2;
  while (size < n) size *= 2;
  for (uint32_t i = n + threadIdx.x; i < size; i += kThreads) sh.list[i] = 0;
  for (uint32_t k = 2; k <= size; k *= 2)
    for (uint32_t j = k / 2; j; j /= 2) {
      __syncthreads();
      for (uint32_t t = threadIdx.x; t < size / 2; t += kThreads) {
        const uint32_t i = (t / j) * 2u * j + t % j;
        const uint64_t a = sh.list[i], b = sh.list[i + j];
        if ((a < b) == ((i & k) == 0)) {
          sh.list[i] = b;
          sh.list[i + j] = a;
        }
      }
    }
  __syncthreads();
}

// All tokens for which `is` holds, sorted, or no more than their number where
// that is over kList.
template <int DT, typename Is> XPU_DEVICE uint32_t gather(Shared &sh, const Row<DT> &row, Is &&is) {
  __syncthreads();
  if (threadIdx.x == 0) sh.listed = 0;
  __syncthreads();
  row.each([&](float v, uint32_t id) {
    if (is(v)) {
      const uint32_t at = atomicAdd(&sh.listed, 1u);
      if (at < kList) sh.list[at] = place_of(v, id);
    }
  });
  __syncthreads();
  const uint32_t n = sh.listed;
  if (n <= kList) sort_list(sh, n);
  return n;
}

// A place in the order: the token there, and the weight of the tokens up to it.
struct Found {
  uint64_t place, weight;
};
// The first of the sorted list's n tokens at which count or weight up to it
// reaches `target`, those before the list being `counted` and `weighed`.
template <int DT> XPU_DEVICE Found in_list(Shared &sh, const Row<DT> &row, uint32_t n, bool by_count, uint64_t target,
                                           uint64_t counted, uint64_t weighed) {
  uint64_t own[2], sum = 0;
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) {
    const uint32_t at = threadIdx.x * 2u + i;
    own[i] = at < n ? row.units(row.weight(of_ordered(static_cast<uint32_t>(sh.list[at] >> 32)))) : 0u;
    sum += own[i];
  }
  uint64_t upto = weighed + block_before(sh, sum);
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) {
    const uint32_t at = threadIdx.x * 2u + i;
    const uint64_t c = counted + at, before = by_count ? c : upto;
    upto += own[i];
    const uint64_t after = by_count ? c + 1u : upto;
    if (at < n && before < target && target <= after) {
      sh.found[0] = sh.list[at];
      sh.found[1] = upto;
    }
  }
  __syncthreads();
  const Found f{sh.found[0], sh.found[1]};
  __syncthreads();
  return f;
}

// The same for a bin of more tokens than a list holds: its tokens by 11, 11, 10
// bits of the logit and 10, 10 of the id.
template <int DT> XPU_DEVICE Found in_bits(Shared &sh, const Row<DT> &row, uint32_t bin, bool by_count, uint64_t target,
                                           uint64_t counted, uint64_t weighed, uint64_t *hist, uint32_t *count) {
  uint64_t prefix = 0;  // the place's bits above `shift`
  uint32_t shift = 52;
  for (uint32_t level = 0; level < 5; ++level) {
    const uint32_t width = level < 2 ? 11u : 10u;
    const uint32_t low = shift - width;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kBins; i += kThreads) {
      hist[i] = 0;
      count[i] = 0;
    }
    __syncthreads();
    row.each([&](float v, uint32_t id) {
      if (row.bin(v) != bin) return;
      // 32 bits of the logit over 20 of the id
      const uint64_t p = static_cast<uint64_t>(ordered(v)) << 20 | (0xfffffu - id);
      if (level && p >> shift != prefix) return;
      const uint32_t d = static_cast<uint32_t>(p >> low) & ((1u << width) - 1u);
      atomicAdd(&count[d], 1u);
      atomicAdd(reinterpret_cast<unsigned long long *>(&hist[d]), row.units(row.weight(v)));
    });
    __syncthreads();
    // from the highest digit down
    uint64_t c[2], w[2], csum = 0, wsum = 0;
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      const uint32_t d = kBins - 1u - (threadIdx.x * 2u + i);
      csum += c[i] = count[d];
      wsum += w[i] = hist[d];
    }
    uint64_t cb = counted + block_before(sh, csum), wb = weighed + block_before(sh, wsum);
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      const uint64_t before = by_count ? cb : wb, after = by_count ? cb + c[i] : wb + w[i];
      if (before < target && target <= after) {
        sh.flag = kBins - 1u - (threadIdx.x * 2u + i);
        sh.found[0] = cb;
        sh.found[1] = wb;
      }
      cb += c[i];
      wb += w[i];
    }
    __syncthreads();
    prefix = prefix << width | sh.flag;
    counted = sh.found[0];
    weighed = sh.found[1];
    shift = low;
  }
  __syncthreads();
  const uint32_t key = static_cast<uint32_t>(prefix >> 20), id = 0xfffffu - (static_cast<uint32_t>(prefix) & 0xfffffu);
  return {static_cast<uint64_t>(key) << 32 | ~id, weighed + row.units(row.weight(of_ordered(key)))};
}

// Where count or weight reach `target`, by the bins (hist and count hold the
// sums up to each).
template <int DT> XPU_DEVICE Found find(Shared &sh, const Row<DT> &row, bool by_count, uint64_t target,
                                        uint64_t *hist, uint32_t *count) {
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) {
    const uint32_t b = threadIdx.x * 2u + i;
    const uint64_t before = b ? by_count ? sh.count[b - 1u] : sh.hist[b - 1u] : 0u;
    const uint64_t after = by_count ? sh.count[b] : sh.hist[b];
    if (before < target && target <= after) sh.flag = b;
  }
  __syncthreads();
  const uint32_t b = sh.flag;
  const uint64_t counted = b ? sh.count[b - 1u] : 0u, weighed = b ? sh.hist[b - 1u] : 0u;
  const uint32_t n = gather(sh, row, [&](float v) { return row.bin(v) == b; });
  if (n <= kList) return in_list(sh, row, n, by_count, target, counted, weighed);
  return in_bits(sh, row, b, by_count, target, counted, weighed, hist, count);
}

template <int DT> XPU_DEVICE void sample(const SampleArgs &a) {
  __shared__ Shared sh;
  __shared__ uint64_t more_hist[kBins];
  __shared__ uint32_t more_count[kBins];
  const uint32_t r = blockIdx.x;
  const float t = a.temperature ? a.temperature[r] : 1.0f, p = a.top_p ? a.top_p[r] : 1.0f;
  const float m = a.min_p ? a.min_p[r] : 0.0f, u = a.random[r];
  const uint32_t k = a.top_k ? min(a.top_k[r], a.vocab) : 0u;
  Row<DT> row;
  row.logits = static_cast<const uint8_t *>(a.logits) + r * a.stride * (DT == kFp32 ? 4u : 2u);
  row.vocab = a.vocab;
  row.bits = a.bits;
  auto answer = [&](uint32_t token, float probability) {
    if (threadIdx.x) return;
    a.tokens[r] = token;
    if (a.probability) a.probability[r] = probability;
  };
  // (comparisons that are false for NaN)
  const bool sound = t >= 0.0f && t < __builtin_inff() && p >= 0.0f && m >= 0.0f && m <= 1.0f && u >= 0.0f && u < 1.0f;

  // the largest, the lowest id that has it, and the thread's own largest
  uint64_t own = 0;
  bool odd = false;
  row.each([&](float v, uint32_t id) {
    odd |= !(v < __builtin_inff());
    const uint64_t at = place_of(v, id);
    own = at > own ? at : own;
  });
  const uint64_t first = block_reduce(sh, own, [](uint64_t x, uint64_t y) { return x > y ? x : y; });
  const uint32_t any_odd = block_reduce(sh, odd ? 1u : 0u, [](uint32_t x, uint32_t y) { return x | y; });
  row.largest = of_ordered(static_cast<uint32_t>(first >> 32));
  if (!sound || any_odd || row.largest == -__builtin_inff()) return answer(0xffffffffu, __builtin_nanf(""));
  if (t == 0.0f || k == 1u) return answer(~static_cast<uint32_t>(first), 1.0f);
  row.scale = 1.44269504088896340736 / static_cast<double>(t);
  const bool cuts_k = k && k < a.vocab, cuts_p = p < 1.0f;

  uint64_t total = 0, min_p_weight = ~0ull;
  uint32_t n = 0;
  bool listed = false;
  if (cuts_k && k <= kFew) {
    const float top = own ? of_ordered(static_cast<uint32_t>(own >> 32)) : -__builtin_inff();
    const bool has = top > -__builtin_inff();
    const float low = block_reduce(sh, has ? top : row.largest, [](float x, float y) { return fminf(x, y); });
    row.by = low < row.largest ? kBins / fminf(row.largest - low, 0x1p100f) : 0.0f;
    for (uint32_t i = threadIdx.x; i < kBins; i += kThreads) sh.count[i] = 0;
    if (threadIdx.x == 0) sh.flag = kBins - 1u;
    __syncthreads();
    if (has) atomicAdd(&sh.count[row.bin(top)], 1u);
    __syncthreads();
    uint32_t c[2] = {sh.count[threadIdx.x * 2u], sh.count[threadIdx.x * 2u + 1u]};
    uint64_t before = block_before(sh, c[0] + c[1]);
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      if (before < k && k <= before + c[i]) sh.flag = threadIdx.x * 2u + i;
      before += c[i];
    }
    __syncthreads();
    const uint32_t last = sh.flag;
    n = gather(sh, row, [&](float v) { return row.bin(v) <= last; });
    listed = n <= kList && n >= k;
  }
  if (listed) {
    const Found kth = in_list(sh, row, n, true, k, 0, 0);
    total = kth.weight;
  } else {
    row.by = static_cast<float>(__builtin_fmin(kBins / (kSpan * static_cast<double>(t)), 0x1p100));
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kBins; i += kThreads) {
      sh.hist[i] = 0;
      sh.count[i] = 0;
    }
    __syncthreads();
    uint64_t above = 0;
    row.each([&](float v, uint32_t) {
      const double w = row.weight(v);
      const uint64_t x = row.units(w);
      const uint32_t b = row.bin(v);
      if (w >= m) above += x;
      if (x) atomicAdd(reinterpret_cast<unsigned long long *>(&sh.hist[b]), x);
      if (cuts_k) atomicAdd(&sh.count[b], 1u);
    });
    if (m > 0.0f) min_p_weight = block_reduce(sh, above, [](uint64_t x, uint64_t y) { return x + y; });
    __syncthreads();
    const uint32_t b = threadIdx.x * 2u;
    uint64_t w0 = sh.hist[b], w1 = sh.hist[b + 1u];
    const uint32_t c0 = sh.count[b], c1 = sh.count[b + 1u];
    const uint64_t wb = block_before(sh, w0 + w1);
    const uint32_t cb = static_cast<uint32_t>(block_before(sh, c0 + c1));
    sh.hist[b] = wb + w0;
    sh.hist[b + 1u] = wb + w0 + w1;
    sh.count[b] = cb + c0;
    sh.count[b + 1u] = cb + c0 + c1;
    __syncthreads();
    total = cuts_k ? find(sh, row, true, k, more_hist, more_count).weight : sh.hist[kBins - 1u];
  }
  auto reach = [&](uint64_t target) {
    return listed ? in_list(sh, row, n, false, target, 0, 0) : find(sh, row, false, target, more_hist, more_count);
  };
  // at least the first token is kept, whose weight is 2^bits
  uint64_t kept = total;
  if (cuts_p) {
    const double want = __builtin_ceil(static_cast<double>(p) * static_cast<double>(total));
    const uint64_t target = want < 1.0 ? 1u : static_cast<uint64_t>(want);
    kept = reach(target < total ? target : total).weight;
  }
  if (listed && m > 0.0f) {
    uint64_t above = 0;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
      const double w = row.weight(of_ordered(static_cast<uint32_t>(sh.list[i] >> 32)));
      if (w >= m) above += row.units(w);
    }
    min_p_weight = block_reduce(sh, above, [](uint64_t x, uint64_t y) { return x + y; });
  }
  kept = min_p_weight < kept ? min_p_weight : kept;
  const uint64_t drawn = static_cast<uint64_t>(static_cast<double>(u) * static_cast<double>(kept));
  const Found f = reach(drawn < kept ? drawn + 1u : kept);
  const double w = row.weight(of_ordered(static_cast<uint32_t>(f.place >> 32)));
  answer(~static_cast<uint32_t>(f.place),
         static_cast<float>(__builtin_amdgcn_ldexp(w, static_cast<int>(a.bits)) / static_cast<double>(kept)));
}

}  // namespace sample
}  // namespace xpu

#define XPU_SAMPLE(T, NAME)                                                                            \
  extern "C" __global__ __launch_bounds__(1024) void xpu_sample_##NAME(xpu::SampleArgs a) {            \
    xpu::sample::sample<T>(a);                                                                         \
  }
XPU_SAMPLE(xpu::kBf16, bf16)
XPU_SAMPLE(xpu::kFp16, fp16)
XPU_SAMPLE(xpu::sample::kFp32, fp32)
