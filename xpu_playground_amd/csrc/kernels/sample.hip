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
// With x = logit log2(e) / T, a token's weight is y 2^n, where n + j / 64 is
// the multiple of 1 / 64 that is nearest to x and y = 2^(x - n), formed in 64
// bits. The weights are summed as integers: y in units of 2^-fine within a bin,
// the tokens of two neighbouring multiples, which have the same n; the bins in
// units of 2^-fine of the largest's n. So sums do not depend on their order, no
// bin depends on the largest logit, and one pass over the row gives both. A sum
// is off by half a unit per token and per bin (fine + log2 of the tokens is 61
// at most), and weights below 2^-47 of the largest count as nothing.
//
// Three launches. xpu_sample_look, several blocks to a row: the histogram of
// the weights. xpu_sample_list, the same blocks: which bins the k-th token, the
// p-th part and the draw lie in (a range of them, as one depends on the other),
// and the list of their tokens. xpu_sample_draw, a block to a row: the places
// among those. With few tokens (top-k up to kFew) there are no weights to be
// summed: the k-th largest of the largest logits of 1024 groups of threads
// bounds the k-th largest of all from below, so what is at least that is little
// more than k tokens, which are listed and ranked. Short rows, and those of
// which too many tokens would be listed (equal ones, mostly), are the drawing
// block's alone.
#include "device_common.hpp"
#include "sample_types.hpp"

namespace xpu {
namespace sample {

constexpr uint32_t kThreads = kSampleThreads, kWaves = kThreads / 64, kSlots = kSampleSlots;
constexpr uint32_t kBins = 1536;  // 48 powers of two
constexpr uint32_t kList = 4096, kRanked = 1024, kFew = 256;
static_assert(kSlots == 2 * kThreads, "two bins, digits, slots to a thread");

enum : int { kFp32 = 2 };

// Values are compared as these: descending logits, then ascending ids.
XPU_DEVICE uint32_t ordered(float v) {
  const uint32_t u = __float_as_uint(v);
  return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}
XPU_DEVICE float of_ordered(uint32_t k) { return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu)); }
XPU_DEVICE uint64_t place_of(float v, uint32_t id) { return static_cast<uint64_t>(ordered(v)) << 32 | ~id; }
XPU_DEVICE float logit_of(uint64_t place) { return of_ordered(static_cast<uint32_t>(place >> 32)); }

// 2^x by the series of exp around the nearest integer, to 2^-52.
XPU_DEVICE double power(double x) {
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
  double powers[64];  // 2^(j / 64)
  uint64_t wave[kWaves];
  uint64_t found[2];
  uint32_t listed, flag, number_at;
  uint32_t tops[2];
  uint64_t weight[kSlots];  // by slots; then of the bins up to each
  uint32_t number[kSlots];  // their tokens
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
#pragma unroll
  for (uint32_t w = 0; w + 1 < kWaves; ++w) v += w < threadIdx.x >> 6 ? sh.wave[w] : 0u;
  return v - own;
}
XPU_DEVICE uint64_t larger(uint64_t x, uint64_t y) { return x > y ? x : y; }

// A row's numbers.
struct Numbers {
  float t, p, m, u;
  uint32_t k;  // 0: all
  bool sound;  // all in their ranges
  XPU_DEVICE explicit Numbers(const SampleArgs &a, uint32_t r) {
    t = a.temperature ? a.temperature[r] : 1.0f;
    p = a.top_p ? a.top_p[r] : 1.0f;
    m = a.min_p ? a.min_p[r] : 0.0f;
    u = a.random[r];
    k = a.top_k ? a.top_k[r] : 0u;
    if (k >= a.vocab && k != 1u) k = 0u;
    // (comparisons that are false for NaN)
    sound = t >= 0.0f && t < __builtin_inff() && p >= 0.0f && m >= 0.0f && m <= 1.0f && u >= 0.0f && u < 1.0f;
  }
  XPU_DEVICE bool greedy() const { return t == 0.0f || k == 1u; }
  XPU_DEVICE bool few() const { return k && k <= kFew; }
  XPU_DEVICE double scale() const { return 1.44269504088896340736 / static_cast<double>(t); }
};

// Weights. `base`: what x counts from; 0 where the blocks of a row have to
// agree, the largest logit where that is too far from 0 (apart()).
struct Weights {
  double base, scale;  // x = (logit - base) scale
  double lift;         // 2^(52 - fine): y + lift has y in units of 2^-fine in its low bits
  const double *powers;

  XPU_DEVICE Weights(const SampleArgs &a, const Numbers &n, const Shared &sh, double base_)
      : base(base_), scale(n.scale()),
        lift(__builtin_bit_cast(double, static_cast<uint64_t>(1023u + 52u - a.fine) << 52)), powers(sh.powers) {}
  // Whether x of the largest logit is too large for 32 bits of 64 x.
  static XPU_DEVICE bool apart(float largest, double scale) { return !(__builtin_fabs(largest * scale) < 0x1p23); }
  // The table, by 64 threads; the caller waits for them.
  static XPU_DEVICE void table(Shared &sh) {
    if (threadIdx.x < 64) sh.powers[threadIdx.x] = 2.0 * power((static_cast<double>(threadIdx.x) - 64.0) / 64.0);
  }
  // A token's nearest multiple k / 64, and y by the table and a series of four
  // terms for the rest |s| <= 1 / 128 (off by 2^-44 of it).
  struct Token {
    int32_t k;
    uint64_t y;
    XPU_DEVICE int32_t bin() const { return k >> 1; }
  };
  XPU_DEVICE Token token(float v) const {
    constexpr double kL = 0.693147180559945309417, kMagic = 0x1.8p46;
    const double d = static_cast<double>(v) - base;
    const double at = __builtin_fma(d, scale, kMagic), s = __builtin_fma(d, scale, kMagic - at);
    const int32_t k = static_cast<int32_t>(__builtin_bit_cast(uint64_t, at));
    double q = __builtin_fma(s, kL * kL * kL * kL / 24, kL * kL * kL / 6);
    q = __builtin_fma(q, s, kL * kL / 2);
    q = __builtin_fma(q, s, kL);
    q = __builtin_fma(q, s, 1.0);
    const double y = __builtin_fma(q, powers[k & 63], lift);
    return {k, __builtin_bit_cast(uint64_t, y) & 0xfffffffffffffull};
  }
  // A logit below all of bins from `bin` on; those from it on have bins of 32 bits.
  XPU_DEVICE float below(int32_t bin) const {
    const double d = (static_cast<double>(bin) - 64.0) / (32.0 * scale) + base;
    return static_cast<float>(__builtin_fmax(d, -0x1.fffffep127));
  }
};
// Units of n as units of a larger n.
XPU_DEVICE uint64_t rounded(uint64_t v, uint32_t shift) {
  return shift == 0 ? v : shift > 63 ? 0u : (v + (1ull << (shift - 1u))) >> shift;
}

// Tokens begin .. end - 1 of a row.
template <int DT> struct Row {
  static constexpr uint32_t kPer = DT == kFp32 ? 4 : 8;  // tokens of 16 bytes
  static constexpr uint32_t kAhead = 4;                  // loads on their way
  const uint8_t *logits;
  uint32_t begin, end;  // begin: a multiple of kPer

  XPU_DEVICE Row(const SampleArgs &a, uint32_t r, uint32_t part, bool whole) {
    logits = static_cast<const uint8_t *>(a.logits) + r * a.stride * (DT == kFp32 ? 4u : 2u);
    begin = whole ? 0u : part * a.chunk;
    end = whole ? a.vocab : min(begin + a.chunk, a.vocab);
    if (begin >= end) begin = end = 0;
  }
  XPU_DEVICE u32x4 load(uint32_t c) const {
    return *reinterpret_cast<const u32x4_any *>(logits + static_cast<uint64_t>(c) * 16u);
  }
  static XPU_DEVICE void values(const u32x4 &x, float (&f)[kPer]) {
    if constexpr (DT == kFp32) {
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) f[i] = __uint_as_float(x[i]);
    } else {
      unpack8<DT>(x, f);
    }
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) f[i] += 0.0f;  // zeros of both signs are equal
  }
  // The token behind the last whole 16 bytes that is the thread's, if any.
  XPU_DEVICE uint32_t tail() const { return end / kPer * kPer + threadIdx.x; }
  XPU_DEVICE float one(uint32_t id) const {
    if constexpr (DT == kFp32) return reinterpret_cast<const float *>(logits)[id] + 0.0f;
    else return decode<DT>(reinterpret_cast<const uint16_t *>(logits)[id]) + 0.0f;
  }

  // body(value, id) for the thread's share of the tokens, ids ascending.
  template <typename Body> XPU_DEVICE void each(Body &&body) const {
    const uint32_t last = end / kPer;
    uint32_t c = begin / kPer + threadIdx.x;
    u32x4 x[kAhead];
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i)
      if (c + i * kThreads < last) x[i] = load(c + i * kThreads);
    for (; c < last; c += kAhead * kThreads) {
#pragma unroll
      for (uint32_t i = 0; i < kAhead; ++i) {
        const uint32_t at = c + i * kThreads, next = at + kAhead * kThreads;
        if (at >= last) break;
        float f[kPer];
        values(x[i], f);
        if (next < last) x[i] = load(next);
#pragma unroll
        for (uint32_t j = 0; j < kPer; ++j) body(f[j], at * kPer + j);
      }
    }
    if (tail() < end) body(one(tail()), tail());
  }
};

// A thread's first token.
struct First {
  float top = -__builtin_inff();
  uint32_t at = 0xffffffffu;  // none above -infinity
  bool odd = false;
  XPU_DEVICE void see(float v, uint32_t id) {
    odd |= !(v < __builtin_inff());
    at = v > top ? id : at;
    top = fmaxf(top, v);
  }
  // Of the block: its place, 0 if there is none, ~0 if a logit is odd.
  XPU_DEVICE uint64_t of_block(Shared &sh) const {
    return block_reduce(sh, odd ? ~0ull : at != 0xffffffffu ? place_of(top, at) : 0u, larger);
  }
};

XPU_DEVICE void clear(Shared &sh) {
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) {
    sh.weight[i * kThreads + threadIdx.x] = 0;
    sh.number[i * kThreads + threadIdx.x] = 0;
  }
}

// Adds (v, id) to a list of `cap` entries where `is`; `count` counts all.
XPU_DEVICE void put(uint64_t *list, uint32_t *count, uint32_t cap, bool is, float v, uint32_t id) {
  if (is) {
    const uint32_t at = atomicAdd(count, 1u);
    if (at < cap) list[at] = place_of(v, id);
  }
}

// ---------------------------------------------------------------- the first launch

// The histogram of a part whose largest logit is not known: bin b is in slot b %
// kSlots, which at any time holds one of the kSlots bins up to the largest so
// far. A tile of the tokens is in registers before its largest is asked for and
// the slots of bins that it is the first to reach are cleared. Tokens kBins
// below the largest so far are left out.
template <int DT> XPU_DEVICE First histogram(Shared &sh, const Row<DT> &row, const Weights &w, bool count) {
  constexpr uint32_t kPer = Row<DT>::kPer, kAhead = Row<DT>::kAhead;
  First first;
  clear(sh);
  if (threadIdx.x < 2) sh.tops[threadIdx.x] = 0;
  __syncthreads();
  const uint32_t last = row.end / kPer;
  u32x4 x[kAhead], next[kAhead];
  auto ask = [&](uint32_t c) {
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i)
      if (c + i * kThreads < last) next[i] = row.load(c + i * kThreads);
  };
  float top = -__builtin_inff(), low = -__builtin_inff();
  int32_t most = 0, least = 0;  // bins of the largest so far, and of the last that count
  // The block's largest becomes at least the threads' `mine`; `turn` counts the calls.
  auto reach = [&](float mine, uint32_t turn) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) mine = fmaxf(mine, __shfl_xor(mine, d));
    if (lane_id() == 0) atomicMax(&sh.tops[turn & 1u], ordered(mine));
    __syncthreads();  // and all have added the tokens before
    const float now = of_ordered(sh.tops[turn & 1u]);
    if (!(now > top)) return;
    const int32_t bin = w.token(now).bin();
    if (top > -__builtin_inff()) {
      // (bins that are further apart may be no numbers of 32 bits)
      const bool far = top <= w.below(bin - static_cast<int32_t>(kSlots));
      const uint32_t grown = far ? kSlots : min(static_cast<uint32_t>(bin - most), kSlots);
      for (uint32_t i = threadIdx.x; i < grown; i += kThreads) {
        const uint32_t slot = static_cast<uint32_t>(bin - static_cast<int32_t>(i)) % kSlots;
        sh.weight[slot] = 0;
        sh.number[slot] = 0;
      }
      __syncthreads();
    }
    top = now;
    most = bin;
    least = bin - static_cast<int32_t>(kBins) + 1;
    low = w.below(least);
  };
  auto add = [&](float v) {
    if (v < low) return;
    const auto t = w.token(v);
    if (t.bin() < least) return;
    const uint32_t slot = static_cast<uint32_t>(t.bin()) % kSlots;
    atomicAdd(reinterpret_cast<unsigned long long *>(&sh.weight[slot]), t.y);
    if (count) atomicAdd(&sh.number[slot], 1u);
  };
  const uint32_t begin = row.begin / kPer;
  uint32_t turn = 0;
  ask(begin + threadIdx.x);
  for (uint32_t c0 = begin; c0 < last; c0 += kAhead * kThreads, ++turn) {
    const uint32_t c = c0 + threadIdx.x;
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i) {
      x[i] = next[i];
      const uint32_t at = c + i * kThreads;
      if (at >= last) continue;
      float f[kPer];
      row.values(x[i], f);
#pragma unroll
      for (uint32_t j = 0; j < kPer; ++j) first.see(f[j], at * kPer + j);
    }
    ask(c + kAhead * kThreads);
    reach(first.top, turn);
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i) {
      if (c + i * kThreads >= last) continue;
      float f[kPer];
      row.values(x[i], f);
#pragma unroll
      for (uint32_t j = 0; j < kPer; ++j) add(f[j]);
    }
  }
  const bool mine = row.tail() < row.end;
  const float v = mine ? row.one(row.tail()) : -__builtin_inff();
  if (mine) first.see(v, row.tail());
  reach(first.top, turn);
  if (mine) add(v);
  __syncthreads();
  return first;
}

template <int DT> XPU_DEVICE void look(const SampleArgs &a) {
  __shared__ Shared sh;
  const uint32_t r = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const Numbers n(a, r);
  const Row<DT> row(a, r, part, false);
  First first;
  if (!n.sound || n.greedy() || n.few()) {
    row.each([&](float v, uint32_t id) { first.see(v, id); });
    // groups of as many threads as the row has parts
    float top = first.top;
    for (uint32_t d = 1; d < a.parts; d *= 2) top = fmaxf(top, __shfl_xor(top, static_cast<int>(d)));
    const uint32_t groups = kThreads / a.parts;
    if (threadIdx.x % a.parts == 0) a.groups[r * kThreads + part * groups + threadIdx.x / a.parts] = top;
  } else {
    Weights::table(sh);
    first = histogram(sh, row, Weights(a, n, sh, 0.0), n.k != 0);
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      const uint32_t at = i * kThreads + threadIdx.x;
      a.weights[static_cast<uint64_t>(blockIdx.x) * kSlots + at] = sh.weight[at];
      if (n.k) a.numbers[static_cast<uint64_t>(blockIdx.x) * kSlots + at] = sh.number[at];
    }
  }
  const uint64_t place = first.of_block(sh);
  if (threadIdx.x == 0) a.firsts[blockIdx.x] = place;
}

// The first token of a row, ~0 if it has no answer.
XPU_DEVICE uint64_t first_of(const SampleArgs &a, uint32_t r) {
  uint64_t first = 0;
  for (uint32_t i = 0; i < a.parts; ++i) first = larger(first, a.firsts[r * a.parts + i]);
  return first ? first : ~0ull;
}

// ---------------------------------------------------------------- bins

// The row's bins in order: bin 0 is the largest token's. sh.weight and sh.number
// become the sums up to each.
struct Bins {
  Shared &sh;
  const Weights &w;
  int32_t most;    // the largest token's bin
  uint32_t power;  // and n

  XPU_DEVICE Bins(Shared &sh_, const Weights &w_, float largest) : sh(sh_), w(w_) {
    const int32_t k = w.token(largest).k;
    most = k >> 1;
    power = static_cast<uint32_t>(k >> 6);
  }
  XPU_DEVICE uint32_t of(float v) const {
    return v < w.below(most - static_cast<int32_t>(kBins)) ? kBins : static_cast<uint32_t>(most - w.token(v).bin());
  }
  // The shift from a bin's units to the largest's.
  XPU_DEVICE uint32_t shift(uint32_t bin) const {
    return power - static_cast<uint32_t>((most - static_cast<int32_t>(bin)) >> 5);
  }
  XPU_DEVICE uint64_t units(float v) const {
    const uint32_t bin = of(v);
    return bin < kBins ? rounded(w.token(v).y, shift(bin)) : 0u;
  }
  // From the thread's two bins.
  XPU_DEVICE void sum(const uint64_t (&weight)[2], const uint32_t (&number)[2]) {
    const uint32_t b = threadIdx.x * 2u;
    const uint64_t w0 = rounded(weight[0], shift(b)), w1 = rounded(weight[1], shift(b + 1u));
    const uint64_t wb = block_before(sh, w0 + w1), nb = block_before(sh, static_cast<uint64_t>(number[0]) + number[1]);
    __syncthreads();
    sh.weight[b] = wb + w0;
    sh.weight[b + 1u] = wb + w0 + w1;
    sh.number[b] = static_cast<uint32_t>(nb) + number[0];
    sh.number[b + 1u] = static_cast<uint32_t>(nb) + number[0] + number[1];
    __syncthreads();
  }
  // Of the parts' histograms.
  XPU_DEVICE void load(const SampleArgs &a, uint32_t r, bool count) {
    uint64_t weight[2] = {0, 0};
    uint32_t number[2] = {0, 0};
    if (threadIdx.x * 2u < kBins)
      for (uint32_t p = 0; p < a.parts; ++p) {
        const uint32_t block = r * a.parts + p;
        const uint64_t first = a.firsts[block];
        if (!first || logit_of(first) < w.below(most - static_cast<int32_t>(kBins))) continue;
        const int32_t own = w.token(logit_of(first)).bin();
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
          const int32_t bin = most - static_cast<int32_t>(threadIdx.x * 2u + i);
          if (bin > own) continue;
          const uint64_t at = static_cast<uint64_t>(block) * kSlots + static_cast<uint32_t>(bin) % kSlots;
          weight[i] += a.weights[at];
          if (count) number[i] += a.numbers[at];
        }
      }
    sum(weight, number);
  }
  // Of the block's own histogram.
  XPU_DEVICE void take() {
    uint64_t weight[2] = {0, 0};
    uint32_t number[2] = {0, 0};
    if (threadIdx.x * 2u < kBins)
#pragma unroll
      for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t slot = static_cast<uint32_t>(most - static_cast<int32_t>(threadIdx.x * 2u + i)) % kSlots;
        weight[i] = sh.weight[slot];
        number[i] = sh.number[slot];
      }
    sum(weight, number);
  }
  XPU_DEVICE uint64_t weight_to(uint32_t bin) const { return sh.weight[bin]; }
  XPU_DEVICE uint64_t weight_before(uint32_t bin) const { return bin ? sh.weight[bin - 1u] : 0u; }
  XPU_DEVICE uint32_t number_before(uint32_t bin) const { return bin ? sh.number[bin - 1u] : 0u; }
  XPU_DEVICE uint64_t total() const { return sh.weight[kBins - 1u]; }
  // Whether the k-th token is in a bin (else its weight is nothing).
  XPU_DEVICE bool counts(uint32_t k) const { return k && k <= sh.number[kBins - 1u]; }
  // The bin where the number or the weight reaches `target`, 1 .. the total.
  XPU_DEVICE uint32_t find(bool by_count, uint64_t target) {
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      const uint32_t b = threadIdx.x * 2u + i;
      const uint64_t before = by_count ? number_before(b) : weight_before(b), to = by_count ? sh.number[b] : sh.weight[b];
      if (before < target && target <= to) sh.flag = b;
    }
    __syncthreads();
    return sh.flag;
  }
  // The bins that a logit as far below the largest as w >= m allows can be in:
  // its own and, for the roundings, one on either side.
  XPU_DEVICE uint32_t floor_bin(float largest, double log_m) const {
    const double x = (static_cast<double>(largest) - w.base) * w.scale;
    const double b = static_cast<double>(most) - __builtin_floor((x + log_m) * 32.0);
    return static_cast<uint32_t>(__builtin_fmin(__builtin_fmax(b, 0.0), kBins - 2.0));
  }
};

// What top-p and the draw ask for.
XPU_DEVICE uint64_t part_of(float p, uint64_t total) {
  const double want = __builtin_ceil(static_cast<double>(p) * static_cast<double>(total));
  const uint64_t target = want < 1.0 ? 1u : static_cast<uint64_t>(want);
  return target < total ? target : total;
}
XPU_DEVICE uint64_t drawn_of(float u, uint64_t kept) {
  const uint64_t drawn = static_cast<uint64_t>(static_cast<double>(u) * static_cast<double>(kept));
  return drawn < kept ? drawn + 1u : kept;
}

// Bins for the largest logits of groups, and the last bin of which k groups are
// in it and those before: tokens whose bin is up to that are candidates.
struct Groups {
  float largest, by;
  uint32_t last;
  XPU_DEVICE uint32_t bin(float v) const {
    return static_cast<uint32_t>(__builtin_fminf((largest - v) * by, static_cast<float>(kSlots - 1u)));
  }
  XPU_DEVICE Groups(Shared &sh, float largest_, float top, uint32_t k) : largest(largest_) {
    const bool has = top > -__builtin_inff();
    const float low = block_reduce(sh, has ? top : largest, [](float x, float y) { return fminf(x, y); });
    by = low < largest ? kSlots / fminf(largest - low, 0x1p100f) : 0.0f;
    clear(sh);
    if (threadIdx.x == 0) sh.flag = kSlots - 1u;
    __syncthreads();
    if (has) atomicAdd(&sh.number[bin(top)], 1u);
    __syncthreads();
    const uint32_t c[2] = {sh.number[threadIdx.x * 2u], sh.number[threadIdx.x * 2u + 1u]};
    uint64_t before = block_before(sh, c[0] + c[1]);
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      if (before < k && k <= before + c[i]) sh.flag = threadIdx.x * 2u + i;
      before += c[i];
    }
    __syncthreads();
    last = sh.flag;
  }
};

// ---------------------------------------------------------------- the second launch

// Bins lo .. hi, and logits that include theirs.
struct Range {
  uint32_t lo, hi;
  float from, to;
  XPU_DEVICE Range() : lo(1), hi(0), from(__builtin_inff()), to(-__builtin_inff()) {}
  XPU_DEVICE Range(const Bins &b, uint32_t lo_, uint32_t hi_) : lo(lo_), hi(hi_) {
    auto edge = [&](int32_t bin, double by) {
      const double v = static_cast<double>(b.most + bin) / (32.0 * b.w.scale) + b.w.base;
      const double e = v + by * (__builtin_fabs(v) * 0x1p-20 + 0x1p-130);
      return static_cast<float>(__builtin_fmin(__builtin_fmax(e, -0x1.fffffep127), 0x1.fffffep127));
    };
    from = edge(-static_cast<int32_t>(hi) - 1, -1.0);
    to = edge(2 - static_cast<int32_t>(lo), 1.0);
  }
  XPU_DEVICE bool near(float v) const { return v >= from && v <= to; }
  XPU_DEVICE bool has(uint32_t bin) const { return bin >= lo && bin <= hi; }
};

template <int DT> XPU_DEVICE void list(const SampleArgs &a) {
  __shared__ Shared sh;
  const uint32_t r = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const Numbers n(a, r);
  const uint64_t first = first_of(a, r);
  if (!n.sound || first == ~0ull || n.greedy()) return;
  const Row<DT> row(a, r, part, false);
  const float top = logit_of(first);
  uint64_t *list = a.lists + static_cast<uint64_t>(blockIdx.x) * kSampleCap;
  if (n.few()) {
    const Groups g(sh, top, a.groups[r * kThreads + threadIdx.x], n.k);
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    row.each([&](float v, uint32_t id) { put(list, &sh.listed, kSampleCap, g.bin(v) <= g.last, v, id); });
  } else {
    const Weights w(a, n, sh, 0.0);
    if (Weights::apart(top, w.scale)) return;
    Weights::table(sh);
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    Bins bins(sh, w, top);
    bins.load(a, r, n.k != 0);
    // the weight of what is kept is between lo and hi
    Range ranges[4];
    uint64_t lo = bins.total(), hi = lo;
    if (bins.counts(n.k)) {
      const uint32_t b = bins.find(true, n.k);
      ranges[0] = Range(bins, b, b);
      lo = bins.weight_before(b) + 1u;
      hi = bins.weight_to(b);
    }
    if (n.p < 1.0f) {
      const uint32_t bl = bins.find(false, part_of(n.p, lo)), bh = bins.find(false, part_of(n.p, hi));
      ranges[1] = Range(bins, bl, bh);
      lo = bins.weight_before(bl) + 1u;
      hi = bins.weight_to(bh);
    }
    if (n.m > 0.0f) {
      const uint32_t b = bins.floor_bin(top, log2(static_cast<double>(n.m)));
      const uint32_t bl = b ? b - 1u : 0u;
      ranges[2] = Range(bins, bl, b + 1u);
      const uint64_t l = bins.weight_before(bl), h = bins.weight_to(b + 1u);
      lo = l < lo ? l : lo;
      hi = h < hi ? h : hi;
    }
    lo = lo ? lo : 1u;
    const uint32_t dl = bins.find(false, drawn_of(n.u, lo)), dh = bins.find(false, drawn_of(n.u, hi));
    ranges[3] = Range(bins, dl, dh);
    row.each([&](float v, uint32_t id) {
      if (!(ranges[0].near(v) || ranges[1].near(v) || ranges[2].near(v) || ranges[3].near(v))) return;
      const uint32_t b = bins.of(v);
      put(list, &sh.listed, kSampleCap, ranges[0].has(b) || ranges[1].has(b) || ranges[2].has(b) || ranges[3].has(b), v, id);
    });
  }
  __syncthreads();
  if (threadIdx.x == 0) a.listed[blockIdx.x] = sh.listed;
}

// ---------------------------------------------------------------- the third launch

// A place in the order: the token there, and the weight of the tokens up to it.
struct Found {
  uint64_t place, weight;
};

template <int DT> struct Draw {
  Shared &sh;
  uint64_t *list;           // kList
  uint64_t *digit_weight;   // kSlots
  uint32_t *digit_number;   // kSlots
  const SampleArgs &a;
  uint32_t r;
  const Row<DT> &row;
  bool lists;  // the parts' lists have what is asked for

  XPU_DEVICE bool complete() const {
    bool all = true;
    for (uint32_t p = 0; p < a.parts; ++p) all &= a.listed[r * a.parts + p] <= kSampleCap;
    return all;
  }
  // body(value, place) for the thread's share of the parts' lists, or of the row.
  template <typename Body> XPU_DEVICE void each(Body &&body) {
    if (lists) {
      for (uint32_t p = 0; p < a.parts; ++p)
        if (threadIdx.x < a.listed[r * a.parts + p]) {
          const uint64_t x = a.lists[static_cast<uint64_t>(r * a.parts + p) * kSampleCap + threadIdx.x];
          body(logit_of(x), x);
        }
    } else {
      row.each([&](float v, uint32_t id) { body(v, place_of(v, id)); });
    }
  }
  // The tokens for which is(value, place) into the list; their number, which
  // may be over kList.
  template <typename Is> XPU_DEVICE uint32_t gather(Is &&is) {
    __syncthreads();
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    each([&](float v, uint64_t place) {
      if (is(v, place)) {
        const uint32_t at = atomicAdd(&sh.listed, 1u);
        if (at < kList) list[at] = place;
      }
    });
    __syncthreads();
    return sh.listed;
  }

  // The first token of a bin at which the number or the weight of the bin's
  // tokens up to it, in its units, reaches `target`: the bin's places are divided
  // into kSlots pieces, the one that has the token into kSlots again, until it
  // has no more than a wavefront takes. A bin that the list does not hold is
  // looked for in the row until a piece of it is held.
  XPU_DEVICE Found within(Bins &bins, uint32_t bin, bool by_count, uint64_t target) {
    const Range range(bins, bin, bin);
    auto in_bin = [&](float v) { return range.near(v) && bins.of(v) == bin; };
    uint32_t n = gather([&](float v, uint64_t) { return in_bin(v); });
    bool held = n <= kList;
    // body(value, place) for the thread's share of the bin's tokens
    auto every = [&](auto &&body) {
      if (held) {
        for (uint32_t i = threadIdx.x; i < min(n, kList); i += kThreads) body(logit_of(list[i]), list[i]);
      } else {
        each([&](float v, uint64_t place) {
          if (in_bin(v)) body(v, place);
        });
      }
    };
    uint64_t lo = 0, hi = ~0ull, before = 0;  // the piece, and what comes before it
    uint32_t left = n;                        // its tokens
    if (left > 64) {
      uint64_t least = ~0ull, most = 0;
      every([&](float, uint64_t place) {
        least = place < least ? place : least;
        most = larger(most, place);
      });
      lo = block_reduce(sh, least, [](uint64_t x, uint64_t y) { return x < y ? x : y; });
      hi = block_reduce(sh, most, larger);
    }
    while (left > 64) {
      const uint32_t bits = 64u - static_cast<uint32_t>(__builtin_clzll(hi - lo | 1u)), by = bits > 11u ? bits - 11u : 0u;
      __syncthreads();
#pragma unroll
      for (uint32_t i = 0; i < 2; ++i) {
        digit_weight[i * kThreads + threadIdx.x] = 0;
        digit_number[i * kThreads + threadIdx.x] = 0;
      }
      __syncthreads();
      every([&](float v, uint64_t place) {
        if (place < lo || place > hi) return;
        const uint32_t d = static_cast<uint32_t>((hi - place) >> by);
        atomicAdd(&digit_number[d], 1u);
        if (!by_count) atomicAdd(reinterpret_cast<unsigned long long *>(&digit_weight[d]), bins.w.token(v).y);
      });
      __syncthreads();
      const uint32_t d0 = threadIdx.x * 2u, n0 = digit_number[d0], n1 = digit_number[d0 + 1u];
      const uint64_t v0 = by_count ? n0 : digit_weight[d0], v1 = by_count ? n1 : digit_weight[d0 + 1u];
      const uint64_t b0 = before + block_before(sh, v0 + v1), b1 = b0 + v0;
      if (b0 < target && target <= b1) {
        sh.flag = d0;
        sh.found[0] = b0;
        sh.number_at = n0;
      }
      if (b1 < target && target <= b1 + v1) {
        sh.flag = d0 + 1u;
        sh.found[0] = b1;
        sh.number_at = n1;
      }
      __syncthreads();
      const uint64_t piece = hi - (static_cast<uint64_t>(sh.flag) << by), width = (1ull << by) - 1u;
      before = sh.found[0];
      left = sh.number_at;
      lo = piece - lo > width ? piece - width : lo;
      hi = piece;
      if (!held && left <= kList) {
        n = gather([&](float v, uint64_t place) { return in_bin(v) && place >= lo && place <= hi; });
        held = true;
      }
    }
    // those of the piece, by the first wavefront
    __syncthreads();
    if (threadIdx.x == 0) sh.flag = 0;
    __syncthreads();
    every([&](float, uint64_t place) {
      if (place >= lo && place <= hi) digit_weight[atomicAdd(&sh.flag, 1u) & 63u] = place;
    });
    __syncthreads();
    if (threadIdx.x < 64) {
      const bool real = threadIdx.x < left;
      const uint64_t place = real ? digit_weight[threadIdx.x] : 0u;
      const uint64_t value = !real ? 0u : by_count ? 1u : bins.w.token(logit_of(place)).y;
      uint64_t upto = before;
      for (uint32_t j = 0; j < left; ++j) {
        const bool ahead = __shfl(place, static_cast<int>(j)) > place;
        const uint64_t v = __shfl(value, static_cast<int>(j));
        upto += ahead ? v : 0u;
      }
      if (real && upto < target && target <= upto + value) {
        sh.found[0] = place;
        sh.found[1] = upto + value;
      }
    }
    __syncthreads();
    return {sh.found[0], sh.found[1]};
  }

  // Where the weight reaches `target`, and the weight up to there.
  XPU_DEVICE Found reach(Bins &bins, uint64_t target) {
    const uint32_t b = bins.find(false, target), shift = bins.shift(b);
    const uint64_t before = bins.weight_before(b), need = target - before;
    // rounded(c, shift) >= need
    const Found f = within(bins, b, false, shift ? (need << shift) - (1ull << (shift - 1u)) : need);
    return {f.place, before + rounded(f.weight, shift)};
  }
  // The weight of the first k tokens.
  XPU_DEVICE uint64_t first_weight(Bins &bins, uint32_t k) {
    const uint32_t b = bins.find(true, k);
    const Found f = within(bins, b, true, k - bins.number_before(b));
    return bins.weight_before(b) + rounded(weight_to(bins, b, f.place), bins.shift(b));
  }
  // The weight of a bin's tokens up to a place, in its units.
  XPU_DEVICE uint64_t weight_to(Bins &bins, uint32_t bin, uint64_t to) {
    const Range range(bins, bin, bin);
    uint64_t own = 0;
    each([&](float v, uint64_t place) {
      if (place >= to && range.near(v) && bins.of(v) == bin) own += bins.w.token(v).y;
    });
    return block_reduce(sh, own, [](uint64_t x, uint64_t y) { return x + y; });
  }
  // The weight of the tokens with w >= m > 0.
  XPU_DEVICE uint64_t at_least(Bins &bins, float largest, double log_m) {
    const uint32_t b = bins.floor_bin(largest, log_m), lo = b ? b - 1u : 0u;
    const Range range(bins, lo, b + 1u);
    uint64_t own[3] = {0, 0, 0};
    each([&](float v, uint64_t) {
      if (!range.near(v) || (static_cast<double>(v) - largest) * bins.w.scale < log_m) return;
      const uint32_t bin = bins.of(v);
      if (!range.has(bin)) return;
      const uint64_t y = bins.w.token(v).y;
      own[0] += bin == lo ? y : 0u;
      own[1] += bin == lo + 1u ? y : 0u;
      own[2] += bin == lo + 2u ? y : 0u;
    });
    uint64_t sum = bins.weight_before(lo);
#pragma unroll
    for (uint32_t i = 0; i < 3; ++i)
      sum += rounded(block_reduce(sh, own[i], [](uint64_t x, uint64_t y) { return x + y; }), bins.shift(lo + i));
    return sum;
  }
};

XPU_DEVICE void answer_at(const SampleArgs &a, uint32_t r, uint32_t token, float probability) {
  a.tokens[r] = token;
  if (a.probability) a.probability[r] = probability;
}

template <int DT> XPU_DEVICE void draw(const SampleArgs &a) {
  __shared__ Shared sh;
  __shared__ uint64_t list[kList], digit_weight[kSlots];
  __shared__ uint32_t digit_number[kSlots];
  const uint32_t r = blockIdx.x;
  const Numbers n(a, r);
  auto answer = [&](uint32_t token, float probability) {
    if (threadIdx.x == 0) answer_at(a, r, token, probability);
  };
  const Row<DT> row(a, r, 0, true);
  float own_top = -__builtin_inff();
  uint64_t first;
  if (a.parts) {
    first = first_of(a, r);
  } else {
    First f;
    row.each([&](float v, uint32_t id) { f.see(v, id); });
    own_top = f.top;
    first = f.of_block(sh);
    first = first ? first : ~0ull;
  }
  if (!n.sound || first == ~0ull) return answer(0xffffffffu, __builtin_nanf(""));
  if (n.greedy()) return answer(~static_cast<uint32_t>(first), 1.0f);
  const float top = logit_of(first);
  // the row is the block's alone where there are no parts, their lists are not
  // whole, or x of the largest logit has no bins that the parts agree on
  const bool apart = Weights::apart(top, n.scale());
  bool alone = a.parts == 0 || (apart && !n.few());
  Weights::table(sh);
  Draw<DT> o{sh, list, digit_weight, digit_number, a, r, row, false};
  if (!alone) alone = !o.complete();
  o.lists = !alone;
  const Weights w(a, n, sh, alone || apart ? static_cast<double>(top) : 0.0);
  __syncthreads();
  Bins bins(sh, w, top);
  auto share = [&](uint64_t place, uint64_t kept) {
    const double rest = __builtin_fma(static_cast<double>(top) - w.base, w.scale, -static_cast<double>(static_cast<int32_t>(bins.power)));
    const double x = (static_cast<double>(logit_of(place)) - static_cast<double>(top)) * w.scale;
    return static_cast<float>(__builtin_amdgcn_ldexp(power(x) * power(rest), static_cast<int>(a.fine)) / static_cast<double>(kept));
  };
  const double log_m = n.m > 0.0f ? log2(static_cast<double>(n.m)) : 0.0;

  if (n.few()) {
    uint32_t have;
    if (!alone) {
      have = o.gather([](float, uint64_t) { return true; });
    } else {
      const Groups g(sh, top, a.parts ? a.groups[r * kThreads + threadIdx.x] : own_top, n.k);
      have = o.gather([&](float v, uint64_t) { return g.bin(v) <= g.last; });
    }
    if (have >= n.k && have <= kRanked) {
      // a token's rank is the number of those before it
      const bool real = threadIdx.x < have;
      const uint64_t place = real ? list[threadIdx.x] : 0u;
      uint32_t rank = 0;
      if ((threadIdx.x & ~63u) < have)
        for (uint32_t j = 0; j < have; ++j) rank += list[j] > place;
      __syncthreads();
      if (real) digit_weight[rank] = place;
      __syncthreads();
      const uint64_t mine = threadIdx.x < n.k ? digit_weight[threadIdx.x] : 0u;
      const float v = logit_of(mine);
      const uint64_t units = threadIdx.x < n.k ? bins.units(v) : 0u;
      const uint64_t before = block_before(sh, units), to = before + units;
      if (threadIdx.x == n.k - 1u) sh.found[0] = to;
      __syncthreads();
      uint64_t kept = sh.found[0];
      if (n.p < 1.0f) {
        const uint64_t target = part_of(n.p, kept);
        if (before < target && target <= to) sh.found[1] = to;
        __syncthreads();
        kept = sh.found[1];
      }
      if (n.m > 0.0f) {
        const bool is = threadIdx.x < n.k && (static_cast<double>(v) - top) * w.scale >= log_m;
        const uint64_t above = block_reduce(sh, is ? to : 0u, larger);
        kept = above < kept ? above : kept;
      }
      const uint64_t target = drawn_of(n.u, kept);
      if (before < target && target <= to) answer_at(a, r, ~static_cast<uint32_t>(mine), share(mine, kept));
      return;
    }
    o.lists = false;  // candidates are not all that is asked for now
    alone = true;
  }
  if (alone) {
    __syncthreads();
    histogram(sh, row, w, n.k != 0);
    bins.take();
  } else {
    bins.load(a, r, n.k != 0);
  }
  // at least the first token is kept
  uint64_t kept = bins.counts(n.k) ? o.first_weight(bins, n.k) : bins.total();
  if (n.p < 1.0f) kept = o.reach(bins, part_of(n.p, kept)).weight;
  if (n.m > 0.0f) {
    const uint64_t above = o.at_least(bins, top, log_m);
    kept = above < kept ? above : kept;
  }
  const Found f = o.reach(bins, drawn_of(n.u, kept));
  answer(~static_cast<uint32_t>(f.place), share(f.place, kept));
}

}  // namespace sample
}  // namespace xpu

#define XPU_SAMPLE(T, NAME)                                                                                  \
  extern "C" __global__ __launch_bounds__(1024) void xpu_sample_look_##NAME(xpu::SampleArgs a) {             \
    xpu::sample::look<T>(a);                                                                                 \
  }                                                                                                          \
  extern "C" __global__ __launch_bounds__(1024) void xpu_sample_list_##NAME(xpu::SampleArgs a) {             \
    xpu::sample::list<T>(a);                                                                                 \
  }                                                                                                          \
  extern "C" __global__ __launch_bounds__(1024) void xpu_sample_draw_##NAME(xpu::SampleArgs a) {             \
    xpu::sample::draw<T>(a);                                                                                 \
  }
XPU_SAMPLE(xpu::kBf16, bf16)
XPU_SAMPLE(xpu::kFp16, fp16)
XPU_SAMPLE(xpu::sample::kFp32, fp32)
