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
// With x = logit log2(e) / T, a token's weight is y 2^n, where n + j / 32 is
// the multiple of 1 / 32 that is nearest to x and y = 2^(x - n), formed in 64
// bits. The weights are summed as integers: y in units of 2^-fine within a bin,
// the tokens of one such multiple; the bins in units of 2^-fine of the
// largest's n. So sums do not depend on their order, no
// bin depends on the largest logit, and one pass over the row gives both. A sum
// is off by half a unit per token and per bin (fine + log2 of the tokens is 61
// at most), and weights below 2^-47 of the largest may count as nothing.
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
//
// 256 rows of 151936 FP32 logits with top-p: 50 us for the first launch, which
// is bound by its 31 vector instructions per token (the reading alone is 31), 33
// for the second, which reads the row again, 16 for the third, a chain of short
// steps. One bf16 row with top-k: 4.5, 6.0 and 4.8; 48 rows that ask for all
// sorts of things 14.3, 12.6 and 13 to 21 (the last by which tokens are asked for).
#include "device_common.hpp"
#include "sample_types.hpp"

#include <type_traits>

namespace xpu {
namespace sample {

// Threads of a block: many where the row is walked, few where what counts is a
// chain of short steps, of which each takes the time of all wavefronts.
constexpr uint32_t kMany = kSampleThreads, kLittle = kSampleDraw, kSlots = kSampleSlots;
constexpr uint32_t kBins = 1536;  // 48 powers of two
constexpr uint32_t kSteps = 32;   // bins of one: 8 bytes each cover the LDS banks once
constexpr uint32_t kList = 4096, kRanked = 512, kFew = 256;

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
  double powers[kSteps];  // 2^(j / kSteps)
  uint64_t wave[2][16];
  uint64_t found[2];
  uint32_t listed, flag, number_at;
  uint32_t tops[2];
  uint64_t weight[kSlots];  // by slots; then of the bins up to each
  uint32_t number[kSlots];  // their tokens
};

// Of a lane, the same for all.
XPU_DEVICE uint64_t lane_of(uint64_t v, uint32_t lane) {
  return static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane))) << 32 |
         static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}

// A lane's v and those of the lanes before it, by op (0 changes nothing): in its
// row of 16 lanes by DPP shifts, then with the last lanes of the rows before.
template <int CTRL, int ROWS, typename Op> XPU_DEVICE uint64_t shifted(uint64_t v, Op op) {
  const uint32_t lo =
      static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, false));
  const uint32_t hi =
      static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, ROWS, 0xf, false));
  return op(v, static_cast<uint64_t>(hi) << 32 | lo);
}
template <typename Op> XPU_DEVICE uint64_t row_upto(uint64_t v, Op op) {
  v = shifted<0x111, 0xf>(v, op);  // row_shr:1, 2, 4, 8
  v = shifted<0x112, 0xf>(v, op);
  v = shifted<0x114, 0xf>(v, op);
  return shifted<0x118, 0xf>(v, op);
}
template <typename Op> XPU_DEVICE uint64_t wave_upto(uint64_t v, Op op) {
  v = row_upto(v, op);
  v = shifted<0x142, 0xa>(v, op);     // row_bcast:15 to rows 1 and 3
  return shifted<0x143, 0xc>(v, op);  // row_bcast:31 to rows 2 and 3
}

// Over a block of N threads; every thread calls these, one barrier each: the
// wavefronts' results alternate between two places.
template <uint32_t N> struct Block {
  static constexpr uint32_t kWaves = N / 64, kEach = kSlots / N;  // slots, bins, digits to a thread
  Shared &sh;
  uint32_t turn = 0;
  // The wavefronts' results up to each, a lane for each.
  template <typename Op> XPU_DEVICE uint64_t meet(uint64_t v, Op op) {
    uint64_t *at = sh.wave[turn];
    turn ^= 1u;
    if (lane_id() == 63) at[threadIdx.x >> 6] = v;
    __syncthreads();
    return row_upto(at[lane_id() % kWaves], op);
  }
  template <typename Op> XPU_DEVICE uint64_t reduce(uint64_t v, Op op) {
    return lane_of(meet(wave_upto(v, op), op), kWaves - 1u);
  }
  XPU_DEVICE uint64_t sum(uint64_t v) {
    return reduce(v, [](uint64_t x, uint64_t y) { return x + y; });
  }
  XPU_DEVICE uint64_t most(uint64_t v) {
    return reduce(v, [](uint64_t x, uint64_t y) { return x > y ? x : y; });
  }
  XPU_DEVICE uint64_t least(uint64_t v) { return ~most(~v); }
  // Sums of threads 0 .. own - 1.
  XPU_DEVICE uint64_t before(uint64_t v) {
    auto add = [](uint64_t x, uint64_t y) { return x + y; };
    const uint64_t upto = wave_upto(v, add), waves = meet(upto, add);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    return upto - v + (wave ? lane_of(waves, wave - 1u) : 0u);
  }
  XPU_DEVICE void clear() {
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
      sh.weight[i * N + threadIdx.x] = 0;
      sh.number[i * N + threadIdx.x] = 0;
    }
  }
};

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
  double width;        // of a bin
  double lift;         // 2^(52 - fine): y + lift has y in units of 2^-fine in its low bits
  double series[5];    // of 2^s, from the fifth term down; in scalar registers
  const double *powers;

  XPU_DEVICE Weights(const SampleArgs &a, const Numbers &n, const Shared &sh, double base_)
      : base(base_), scale(n.scale()), width(static_cast<double>(n.t) * 0.693147180559945309417 / kSteps),
        lift(__builtin_bit_cast(double, static_cast<uint64_t>(1023u + 52u - a.fine) << 52)), powers(sh.powers) {
    constexpr double kL = 0.693147180559945309417;
    series[0] = kL * kL * kL * kL * kL / 120;
    series[1] = kL * kL * kL * kL / 24;
    series[2] = kL * kL * kL / 6;
    series[3] = kL * kL / 2;
    series[4] = kL;
#pragma unroll
    for (int i = 0; i < 5; ++i) asm("" : "+s"(series[i]));
  }
  // Whether x of the largest logit is too large for bins of 32 bits.
  static XPU_DEVICE bool apart(float largest, double scale) { return !(__builtin_fabs(largest * scale) < 0x1p23); }
  // The table; the caller waits for it.
  static XPU_DEVICE void table(Shared &sh) {
    if (threadIdx.x < kSteps) sh.powers[threadIdx.x] = 2.0 * power((static_cast<double>(threadIdx.x) - kSteps) / kSteps);
  }
  // A token's bin, the multiple of 1 / 32 nearest to x, and y by the table and a
  // series of five terms for the rest |s| <= 1 / 64 (off by 2^-48 of it).
  struct Token {
    int32_t bin;
    uint64_t y;
  };
  XPU_DEVICE Token token(float v) const {
    constexpr double kMagic = 0x1.8p52 / kSteps;
    const double d = static_cast<double>(v) - base;
    const double at = __builtin_fma(d, scale, kMagic), s = __builtin_fma(d, scale, kMagic - at);
    const int32_t bin = static_cast<int32_t>(__builtin_bit_cast(uint64_t, at));
    double q = __builtin_fma(s, series[0], series[1]);
    q = __builtin_fma(q, s, series[2]);
    q = __builtin_fma(q, s, series[3]);
    q = __builtin_fma(q, s, series[4]);
    q = __builtin_fma(q, s, 1.0);
    const double y = __builtin_fma(q, powers[static_cast<uint32_t>(bin) % kSteps], lift);
    return {bin, __builtin_bit_cast(uint64_t, y) & 0xfffffffffffffull};
  }
  // A logit below all of bins from `bin` on; those from it on have bins of 32
  // bits, and are 64 bins below `bin` at most: the first float from there up, as
  // the nearest may be any number of bins further down.
  XPU_DEVICE float below(int32_t bin) const {
    const double d = (static_cast<double>(bin) - 64.0) * width + base;
    const float f = static_cast<float>(__builtin_fmax(d, -0x1.fffffep127));
    return f < d ? of_ordered(ordered(f) + 1u) : f;
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
  XPU_DEVICE uint32_t tail() const { return end / kPer * kPer + threadIdx.x; }  // (kPer threads are enough)
  XPU_DEVICE float one(uint32_t id) const {
    if constexpr (DT == kFp32) return reinterpret_cast<const float *>(logits)[id] + 0.0f;
    else return decode<DT>(reinterpret_cast<const uint16_t *>(logits)[id]) + 0.0f;
  }

  // body(value, id) for the thread's share, of N, of the tokens, ids ascending.
  template <uint32_t N, typename Body> XPU_DEVICE void each(Body &&body) const {
    const uint32_t last = end / kPer;
    uint32_t c = begin / kPer + threadIdx.x;
    u32x4 x[kAhead];
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i)
      if (c + i * N < last) x[i] = load(c + i * N);
    for (; c < last; c += kAhead * N) {
#pragma unroll
      for (uint32_t i = 0; i < kAhead; ++i) {
        const uint32_t at = c + i * N, next = at + kAhead * N;
        if (at >= last) break;
        asm volatile("" : "+v"(x[i]));  // the tokens of one load at a time
        float f[kPer];
        values(x[i], f);
        if (next < last) x[i] = load(next);
#pragma unroll
        for (uint32_t j = 0; j < kPer; ++j) body(f[j], at * kPer + j);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (tail() < end) body(one(tail()), tail());
  }
};

// A thread's first token. Without ids its largest logit and whether there is a
// NaN, which is all that rows need of which more than one token is kept.
template <bool IDS> struct First {
  float top = -__builtin_inff();
  uint32_t at = 0;
  bool odd = false;
  XPU_DEVICE void see(float v, uint32_t id) {
    odd |= v != v;
    if (IDS) at = v > top ? id : at;
    top = fmaxf(top, v);
  }
  // Of the block: its place, 0 if there is none above -infinity, ~0 if a logit
  // is NaN or +infinity.
  template <uint32_t N> XPU_DEVICE uint64_t of_block(Block<N> &block) const {
    const bool bad = odd || top == __builtin_inff();
    return block.most(bad ? ~0ull : top > -__builtin_inff() ? place_of(top, at) : 0u);
  }
};

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
template <bool COUNT, int DT, uint32_t N>
XPU_DEVICE First<false> histogram(Block<N> &block, const Row<DT> &row, const Weights &w) {
  Shared &sh = block.sh;
  constexpr uint32_t kPer = Row<DT>::kPer, kAhead = 2;
  First<false> first;
  block.clear();
  if (threadIdx.x < 2) sh.tops[threadIdx.x] = 0;
  __syncthreads();
  const uint32_t last = row.end / kPer;
  u32x4 x[kAhead], next[kAhead];
  auto ask = [&](uint32_t c) {
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i)
      if (c + i * N < last) next[i] = row.load(c + i * N);
  };
  float top = -__builtin_inff(), low = __builtin_inff();  // nothing counts before the first finite logit
  int32_t most = 0;  // the largest's bin
  // The block's largest becomes at least the threads' `mine`; `turn` counts the calls.
  auto reach = [&](float mine, uint32_t turn) {
    mine = wave_reduce(mine, [](float p, float q) { return fmaxf(p, q); });
    if (lane_id() == 0) atomicMax(&sh.tops[turn & 1u], ordered(mine));
    __syncthreads();  // and all have added the tokens before
    const float now = of_ordered(sh.tops[turn & 1u]);
    if (!(now > top)) return;
    const int32_t bin = w.token(now).bin;
    if (top > -__builtin_inff()) {
      // (bins that are further apart may be no numbers of 32 bits)
      const bool far = top < w.below(bin - static_cast<int32_t>(kSlots));
      const uint32_t grown = far ? kSlots : min(static_cast<uint32_t>(bin - most), kSlots);
      for (uint32_t i = threadIdx.x; i < grown; i += N) {
        const uint32_t slot = static_cast<uint32_t>(bin - static_cast<int32_t>(i)) % kSlots;
        sh.weight[slot] = 0;
        sh.number[slot] = 0;
      }
      __syncthreads();
    }
    top = now;
    most = bin;
    low = w.below(bin - static_cast<int32_t>(kBins) + 1);
  };
  // (tokens that are left out are formed all the same: no branch between the others)
  auto add = [&](const float *f, auto count) {
    constexpr uint32_t kN = decltype(count)::value;
    bool any = false;
#pragma unroll
    for (uint32_t i = 0; i < kN; ++i) any |= f[i] >= low;
    if (!__builtin_amdgcn_ballot_w64(any)) return;
    typename Weights::Token t[kN];
#pragma unroll
    for (uint32_t i = 0; i < kN; ++i) t[i] = w.token(f[i]);
#pragma unroll
    for (uint32_t i = 0; i < kN; ++i) {
      const uint32_t slot = static_cast<uint32_t>(t[i].bin) % kSlots;
      if (f[i] >= low) {
        atomicAdd(reinterpret_cast<unsigned long long *>(&sh.weight[slot]), t[i].y);
        if (COUNT) atomicAdd(&sh.number[slot], 1u);
      }
    }
  };
  const uint32_t begin = row.begin / kPer;
  uint32_t turn = 0;
  ask(begin + threadIdx.x);
  for (uint32_t c0 = begin; c0 < last; c0 += kAhead * N, ++turn) {
    const uint32_t c = c0 + threadIdx.x;
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i) {
      x[i] = next[i];
      if (c + i * N >= last) continue;
      float f[kPer];
      row.values(x[i], f);
#pragma unroll
      for (uint32_t j = 0; j < kPer; ++j) first.see(f[j], 0);
    }
    ask(c + kAhead * N);
    reach(first.top, turn);
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i) {
      if (c + i * N >= last) continue;
      // the tokens of one load at a time, begun here: all of them take more
      // registers than two blocks of 1024 threads to a compute unit have
      asm volatile("" : "+v"(x[i]));
      float f[kPer];
      row.values(x[i], f);
#pragma unroll
      for (uint32_t j = 0; j < kPer; j += 4) {
        add(f + j, std::integral_constant<uint32_t, 4>{});
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  if (row.end % kPer) {  // the tokens behind the last whole 16 bytes
    const bool mine = row.tail() < row.end;
    const float v = mine ? row.one(row.tail()) : -__builtin_inff();
    first.see(v, 0);
    reach(first.top, turn);
    if (mine) add(&v, std::integral_constant<uint32_t, 1>{});
  }
  __syncthreads();
  return first;
}

template <int DT> XPU_DEVICE void look(const SampleArgs &a) {
  __shared__ Shared sh;
  Block<kMany> block{sh};
  const uint32_t r = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const Numbers n(a, r);
  const Row<DT> row(a, r, part, false);
  uint64_t place;
  if (!n.sound || n.greedy()) {
    First<true> first;
    row.template each<kMany>([&](float v, uint32_t id) { first.see(v, id); });
    place = first.of_block(block);
  } else if (n.few()) {
    First<false> first;
    row.template each<kMany>([&](float v, uint32_t) { first.see(v, 0); });
    place = first.of_block(block);
    // groups of as many threads as the row has parts
    float top = first.top;
    for (uint32_t d = 1; d < a.parts; d *= 2) top = fmaxf(top, __shfl_xor(top, static_cast<int>(d)));
    const uint32_t groups = kMany / a.parts;
    if (threadIdx.x % a.parts == 0) a.groups[r * kMany + part * groups + threadIdx.x / a.parts] = top;
  } else {
    Weights::table(sh);
    const Weights w(a, n, sh, 0.0);
    const First<false> first = n.k ? histogram<true>(block, row, w) : histogram<false>(block, row, w);
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      const uint32_t at = i * kMany + threadIdx.x;
      a.weights[static_cast<uint64_t>(blockIdx.x) * kSlots + at] = sh.weight[at];
      if (n.k) a.numbers[static_cast<uint64_t>(blockIdx.x) * kSlots + at] = sh.number[at];
    }
    place = first.of_block(block);
  }
  if (threadIdx.x == 0) a.firsts[blockIdx.x] = place;
}

// What the parts of a row said, a lane for each.
struct Parts {
  uint64_t own;    // the lane's part's first token
  uint64_t first;  // the row's, ~0 if it has no answer
  XPU_DEVICE Parts(const SampleArgs &a, uint32_t r) {
    own = lane_id() < a.parts ? a.firsts[r * a.parts + lane_id()] : 0u;
    const uint64_t most = wave_upto(own, [](uint64_t x, uint64_t y) { return x > y ? x : y; });
    first = lane_of(most, 63);
    first = first ? first : ~0ull;
  }
};

// ---------------------------------------------------------------- bins

// The row's bins in order: bin 0 is the largest token's. sh.weight and sh.number
// become the sums up to each.
template <uint32_t N> struct Bins {
  static constexpr uint32_t kEach = kSlots / N;
  Shared &sh;
  Block<N> &block;
  const Weights &w;
  int32_t most;  // the largest token's
  float low;     // below all bins

  XPU_DEVICE Bins(Block<N> &block_, const Weights &w_, float largest)
      : sh(block_.sh), block(block_), w(w_), most(w_.token(largest).bin),
        low(w_.below(most - static_cast<int32_t>(kBins))) {}
  XPU_DEVICE uint32_t of(float v) const {
    return v < low ? kBins : static_cast<uint32_t>(most - w.token(v).bin);
  }
  static XPU_DEVICE int32_t exponent(int32_t bin) { return bin >> 5; }
  // The shift from a bin's units to the largest's.
  XPU_DEVICE uint32_t shift(uint32_t bin) const {
    return static_cast<uint32_t>(exponent(most) - exponent(most - static_cast<int32_t>(bin)));
  }
  XPU_DEVICE uint64_t units(float v) const {
    const uint32_t bin = of(v);
    return bin < kBins ? rounded(w.token(v).y, shift(bin)) : 0u;
  }
  // From the thread's bins.
  XPU_DEVICE void sum(const uint64_t (&weight)[kEach], const uint32_t (&number)[kEach]) {
    const uint32_t b = threadIdx.x * kEach;
    uint64_t w[kEach], ws = 0, ns = 0;
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
      ws += w[i] = rounded(weight[i], shift(b + i));
      ns += number[i];
    }
    ws = block.before(ws);
    ns = block.before(ns);
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
      sh.weight[b + i] = ws += w[i];
      sh.number[b + i] = static_cast<uint32_t>(ns += number[i]);
    }
    __syncthreads();
  }
  // Of the parts' histograms, the loads of some parts on their way at a time.
  XPU_DEVICE void load(const SampleArgs &a, uint32_t r, const Parts &parts, bool count) {
    constexpr uint32_t kAtOnce = kEach > 2 ? 2 : 4;
    constexpr int32_t kNone = -0x7fffffff - 1;
    const float f = logit_of(parts.own);
    const int32_t own = parts.own && f >= low ? w.token(f).bin : kNone;  // the lane's part's largest bin
    uint64_t weight[kEach] = {};
    uint32_t number[kEach] = {};
    for (uint32_t p0 = 0; p0 < a.parts; p0 += kAtOnce) {
      uint64_t wt[kAtOnce][kEach];
      uint32_t nm[kAtOnce][kEach];
#pragma unroll
      for (uint32_t p = 0; p < kAtOnce; ++p)
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
          const uint64_t block = r * a.parts + min(p0 + p, a.parts - 1u);
          const uint32_t slot = static_cast<uint32_t>(most - static_cast<int32_t>(threadIdx.x * kEach + i)) % kSlots;
          wt[p][i] = a.weights[block * kSlots + slot];
          if (count) nm[p][i] = a.numbers[block * kSlots + slot];
        }
#pragma unroll
      for (uint32_t p = 0; p < kAtOnce; ++p)
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
          const int32_t largest = __builtin_amdgcn_readlane(own, p0 + p);  // kNone past the last part
          const uint32_t bin = threadIdx.x * kEach + i;
          const bool has = bin < kBins && most - static_cast<int32_t>(bin) <= largest && largest != kNone;
          weight[i] += has ? wt[p][i] : 0u;
          if (count) number[i] += has ? nm[p][i] : 0u;
        }
    }
    sum(weight, number);
  }
  // Of the block's own histogram.
  XPU_DEVICE void take() {
    uint64_t weight[kEach];
    uint32_t number[kEach];
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
      const uint32_t bin = threadIdx.x * kEach + i;
      const uint32_t slot = static_cast<uint32_t>(most - static_cast<int32_t>(bin)) % kSlots;
      weight[i] = bin < kBins ? sh.weight[slot] : 0u;
      number[i] = bin < kBins ? sh.number[slot] : 0u;
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
    for (uint32_t i = 0; i < kEach; ++i) {
      const uint32_t b = i * N + threadIdx.x;
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
    const double b = static_cast<double>(most) - __builtin_floor((x + log_m) * kSteps);
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
  // tops: the thread's groups'.
  template <uint32_t N, uint32_t G>
  XPU_DEVICE Groups(Block<N> &block, float largest_, const float (&tops)[G], uint32_t k) : largest(largest_) {
    constexpr uint32_t kEach = Block<N>::kEach;
    Shared &sh = block.sh;
    float low = largest;
#pragma unroll
    for (uint32_t i = 0; i < G; ++i) low = tops[i] > -__builtin_inff() ? fminf(low, tops[i]) : low;
    low = of_ordered(static_cast<uint32_t>(block.least(ordered(low))));
    by = low < largest ? kSlots / fminf(largest - low, 0x1p100f) : 0.0f;
    block.clear();
    if (threadIdx.x == 0) sh.flag = kSlots - 1u;
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < G; ++i)
      if (tops[i] > -__builtin_inff()) atomicAdd(&sh.number[bin(tops[i])], 1u);
    __syncthreads();
    uint32_t c[kEach], sum = 0;
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) sum += c[i] = sh.number[threadIdx.x * kEach + i];
    uint64_t before = block.before(sum);
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
      if (before < k && k <= before + c[i]) sh.flag = threadIdx.x * kEach + i;
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
  template <typename B> XPU_DEVICE Range(const B &b, uint32_t lo_, uint32_t hi_) : lo(lo_), hi(hi_) {
    auto edge = [&](int32_t bin, double by) {
      const double v = static_cast<double>(b.most + bin) * b.w.width + b.w.base;
      const double e = v + by * (__builtin_fabs(v) * 0x1p-20 + 0x1p-130);
      return static_cast<float>(__builtin_fmin(__builtin_fmax(e, -0x1.fffffep127), 0x1.fffffep127));
    };
    from = edge(-static_cast<int32_t>(hi) - 1, -1.0);
    to = edge(2 - static_cast<int32_t>(lo), 1.0);
  }
  XPU_DEVICE bool near(float v) const { return (v >= from) & (v <= to); }
  XPU_DEVICE bool has(uint32_t bin) const { return (bin >= lo) & (bin <= hi); }
};

template <int DT> XPU_DEVICE void list(const SampleArgs &a) {
  __shared__ Shared sh;
  Block<kMany> block{sh};
  const uint32_t r = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const Numbers n(a, r);
  const Parts parts(a, r);
  const uint64_t first = parts.first;
  if (!n.sound || first == ~0ull || n.greedy()) return;
  const Row<DT> row(a, r, part, false);
  const float top = logit_of(first);
  uint64_t *list = a.lists + static_cast<uint64_t>(blockIdx.x) * kSampleCap;
  if (n.few()) {
    const float tops[1] = {a.groups[r * kMany + threadIdx.x]};
    const Groups g(block, top, tops, n.k);
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    row.template each<kMany>([&](float v, uint32_t id) { put(list, &sh.listed, kSampleCap, g.bin(v) <= g.last, v, id); });
  } else {
    const Weights w(a, n, sh, 0.0);
    if (Weights::apart(top, w.scale)) return;
    Weights::table(sh);
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    Bins<kMany> bins(block, w, top);
    bins.load(a, r, parts, n.k != 0);
    // the weight of what is kept is between lo and hi
    Range ranges[4];  // the draw's, top-p's, top-k's, min-p's
    uint64_t lo = bins.total(), hi = lo;
    if (bins.counts(n.k)) {
      const uint32_t b = bins.find(true, n.k);
      ranges[2] = Range(bins, b, b);
      // (the bin's first tokens, or all of it, may round to nothing; the first bin does not)
      lo = b ? bins.weight_before(b) : 1u;
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
      ranges[3] = Range(bins, bl, b + 1u);
      const uint64_t l = bins.weight_before(bl), h = bins.weight_to(b + 1u);
      lo = l < lo ? l : lo;
      hi = h < hi ? h : hi;
    }
    lo = lo ? lo : 1u;
    const uint32_t dl = bins.find(false, drawn_of(n.u, lo)), dh = bins.find(false, drawn_of(n.u, hi));
    ranges[0] = Range(bins, dl, dh);
    // (two comparisons and no branch for each range that there may be)
    auto search = [&](auto count) {
      constexpr uint32_t kRanges = decltype(count)::value;
      row.template each<kMany>([&](float v, uint32_t id) {
        bool near = false;
#pragma unroll
        for (uint32_t i = 0; i < kRanges; ++i) near |= ranges[i].near(v);
        if (!near) return;
        const uint32_t b = bins.of(v);
        bool has = false;
#pragma unroll
        for (uint32_t i = 0; i < kRanges; ++i) has |= ranges[i].has(b);
        put(list, &sh.listed, kSampleCap, has, v, id);
      });
    };
    if (n.k == 0 && n.m == 0.0f) search(std::integral_constant<uint32_t, 2>{});
    else search(std::integral_constant<uint32_t, 4>{});
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
  static constexpr uint32_t N = kLittle, kEach = kSlots / N;
  Shared &sh;
  Block<N> &block;
  uint64_t *listed;         // kList: what the parts listed, if that is all that is asked for
  uint64_t *list;           // kList
  uint64_t *digit_weight;   // kSlots
  uint32_t *digit_number;   // kSlots
  const SampleArgs &a;
  uint32_t r;
  const Row<DT> &row;
  uint32_t entries;  // of `listed`
  bool lists;        // whether it is

  // Brings the parts' lists, of `own` entries in the lane's part; false where
  // they are not whole or too long.
  XPU_DEVICE bool fetch(uint32_t own) {
    constexpr uint32_t kAtOnce = 4;
    const uint64_t upto = wave_upto(own, [](uint64_t x, uint64_t y) { return x + y; });
    entries = static_cast<uint32_t>(lane_of(upto, 63));
    if (__builtin_amdgcn_ballot_w64(own > kSampleCap) || lane_of(upto, 63) > kList) return false;
    const uint32_t p = threadIdx.x % a.parts, each = N / a.parts;
    const uint32_t n = __shfl(own, static_cast<int>(p)), to = static_cast<uint32_t>(__shfl(upto, static_cast<int>(p))) - n;
    const uint64_t *from = a.lists + static_cast<uint64_t>(r * a.parts + p) * kSampleCap;
    for (uint32_t i = threadIdx.x / a.parts; i < n; i += kAtOnce * each) {
      uint64_t x[kAtOnce];
#pragma unroll
      for (uint32_t j = 0; j < kAtOnce; ++j) x[j] = from[min(i + j * each, n - 1u)];
#pragma unroll
      for (uint32_t j = 0; j < kAtOnce; ++j)
        if (i + j * each < n) listed[to + i + j * each] = x[j];
    }
    __syncthreads();
    return true;
  }
  // body(value, place) for the thread's share of what is listed, or of the row.
  template <typename Body> XPU_DEVICE void each(Body &&body) {
    if (lists) {
      for (uint32_t i = threadIdx.x; i < entries; i += N) body(logit_of(listed[i]), listed[i]);
    } else {
      row.template each<N>([&](float v, uint32_t id) { body(v, place_of(v, id)); });
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
  XPU_DEVICE Found within(Bins<N> &bins, uint32_t bin, bool by_count, uint64_t target) {
    const Range range(bins, bin, bin);
    auto in_bin = [&](float v) { return range.near(v) && bins.of(v) == bin; };
    uint32_t n = gather([&](float v, uint64_t) { return in_bin(v); });
    bool held = n <= kList;
    // body(value, place) for the thread's share of the bin's tokens
    auto every = [&](auto &&body) {
      if (held) {
        for (uint32_t i = threadIdx.x; i < min(n, kList); i += N) body(logit_of(list[i]), list[i]);
      } else {
        each([&](float v, uint64_t place) {
          if (in_bin(v)) body(v, place);
        });
      }
    };
    uint64_t lo = 0, hi = ~0ull, before = 0;  // the piece, and what comes before it
    uint32_t left = n;                        // its tokens
    while (left > 64) {
      // from the piece's first to its last token
      uint64_t least = ~0ull, most = 0;
      every([&](float, uint64_t place) {
        const bool is = place >= lo && place <= hi;
        least = is && place < least ? place : least;
        most = is && place > most ? place : most;
      });
      lo = block.least(least);
      hi = block.most(most);
      const uint32_t bits = 64u - static_cast<uint32_t>(__builtin_clzll(hi - lo | 1u)), by = bits > 11u ? bits - 11u : 0u;
      __syncthreads();
#pragma unroll
      for (uint32_t i = 0; i < kEach; ++i) {
        digit_weight[i * N + threadIdx.x] = 0;
        digit_number[i * N + threadIdx.x] = 0;
      }
      __syncthreads();
      every([&](float v, uint64_t place) {
        if (place < lo || place > hi) return;
        const uint32_t d = static_cast<uint32_t>((hi - place) >> by);
        atomicAdd(&digit_number[d], 1u);
        if (!by_count) atomicAdd(reinterpret_cast<unsigned long long *>(&digit_weight[d]), bins.w.token(v).y);
      });
      __syncthreads();
      uint32_t number[kEach];
      uint64_t value[kEach], sum = 0;
#pragma unroll
      for (uint32_t i = 0; i < kEach; ++i) {
        number[i] = digit_number[threadIdx.x * kEach + i];
        sum += value[i] = by_count ? number[i] : digit_weight[threadIdx.x * kEach + i];
      }
      sum = before + block.before(sum);
#pragma unroll
      for (uint32_t i = 0; i < kEach; ++i) {
        if (sum < target && target <= sum + value[i]) {
          sh.flag = threadIdx.x * kEach + i;
          sh.found[0] = sum;
          sh.number_at = number[i];
        }
        sum += value[i];
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
      for (uint32_t j = 0; j < left; ++j) upto += lane_of(place, j) > place ? lane_of(value, j) : 0u;
      if (real && upto < target && target <= upto + value) {
        sh.found[0] = place;
        sh.found[1] = upto + value;
      }
    }
    __syncthreads();
    return {sh.found[0], sh.found[1]};
  }

  // Where the weight reaches `target`, and the weight up to there.
  XPU_DEVICE Found reach(Bins<N> &bins, uint64_t target) {
    const uint32_t b = bins.find(false, target), shift = bins.shift(b);
    const uint64_t before = bins.weight_before(b), need = target - before;
    // rounded(c, shift) >= need
    const Found f = within(bins, b, false, shift ? (need << shift) - (1ull << (shift - 1u)) : need);
    return {f.place, before + rounded(f.weight, shift)};
  }
  // The weight of the first k tokens.
  XPU_DEVICE uint64_t first_weight(Bins<N> &bins, uint32_t k) {
    const uint32_t b = bins.find(true, k);
    const Found f = within(bins, b, true, k - bins.number_before(b));
    return bins.weight_before(b) + rounded(weight_to(bins, b, f.place), bins.shift(b));
  }
  // The weight of a bin's tokens up to a place, in its units.
  XPU_DEVICE uint64_t weight_to(Bins<N> &bins, uint32_t bin, uint64_t to) {
    const Range range(bins, bin, bin);
    uint64_t own = 0;
    each([&](float v, uint64_t place) {
      if (place >= to && range.near(v) && bins.of(v) == bin) own += bins.w.token(v).y;
    });
    return block.sum(own);
  }
  // The weight of the tokens with w >= m > 0.
  XPU_DEVICE uint64_t at_least(Bins<N> &bins, float largest, double log_m) {
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
      sum += rounded(block.sum(own[i]), bins.shift(lo + i));
    return sum;
  }
};

XPU_DEVICE void answer_at(const SampleArgs &a, uint32_t r, uint32_t token, float probability) {
  a.tokens[r] = token;
  if (a.probability) a.probability[r] = probability;
}

template <int DT> XPU_DEVICE void draw(const SampleArgs &a) {
  __shared__ Shared sh;
  __shared__ uint64_t listed[kList], list[kList], digit_weight[kSlots];
  __shared__ uint32_t digit_number[kSlots];
  constexpr uint32_t N = kLittle;
  Block<N> block{sh};
  const uint32_t r = blockIdx.x;
  const Numbers n(a, r);
  auto answer = [&](uint32_t token, float probability) {
    if (threadIdx.x == 0) answer_at(a, r, token, probability);
  };
  const Row<DT> row(a, r, 0, true);
  // (whatever is there, where nothing is listed)
  const uint32_t own_listed = lane_id() < a.parts ? a.listed[r * a.parts + lane_id()] : 0u;
  float tops[kMany / N];  // of the thread's groups
#pragma unroll
  for (uint32_t i = 0; i < kMany / N; ++i) tops[i] = -__builtin_inff();
  const Parts parts(a, r);
  uint64_t first = parts.first;
  if (!a.parts) {
    First<true> f;
    row.template each<N>([&](float v, uint32_t id) { f.see(v, id); });
    tops[0] = f.top;
    first = f.of_block(block);
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
  Draw<DT> o{sh, block, listed, list, digit_weight, digit_number, a, r, row, 0, false};
  if (!alone) alone = !o.fetch(own_listed);
  o.lists = !alone;
  const Weights w(a, n, sh, alone || apart ? static_cast<double>(top) : 0.0);
  __syncthreads();
  Bins<N> bins(block, w, top);
  auto share = [&](uint64_t place, uint64_t kept) {
    const double rest = __builtin_fma(static_cast<double>(top) - w.base, w.scale, -static_cast<double>(Bins<N>::exponent(bins.most)));
    const double x = (static_cast<double>(logit_of(place)) - static_cast<double>(top)) * w.scale;
    return static_cast<float>(__builtin_amdgcn_ldexp(power(x) * power(rest), static_cast<int>(a.fine)) / static_cast<double>(kept));
  };
  const double log_m = n.m > 0.0f ? log2(static_cast<double>(n.m)) : 0.0;

  if (n.few()) {
    uint32_t have = o.entries;
    const uint64_t *candidates = listed;
    if (alone) {
      if (a.parts)
#pragma unroll
        for (uint32_t i = 0; i < kMany / N; ++i) tops[i] = a.groups[r * kMany + i * N + threadIdx.x];
      const Groups g(block, top, tops, n.k);
      have = o.gather([&](float v, uint64_t) { return g.bin(v) <= g.last; });
      candidates = list;
    }
    if (have >= n.k && have <= kRanked) {
      // a token's rank is the number of those before it
      uint64_t place[kRanked / N];
      uint32_t rank[kRanked / N] = {};
#pragma unroll
      for (uint32_t i = 0; i < kRanked / N; ++i) {
        const uint32_t at = i * N + threadIdx.x;
        place[i] = at < have ? candidates[at] : 0u;
        if ((at & ~63u) < have)
          for (uint32_t j = 0; j < have; ++j) rank[i] += candidates[j] > place[i];
      }
      __syncthreads();
#pragma unroll
      for (uint32_t i = 0; i < kRanked / N; ++i)
        if (i * N + threadIdx.x < have) digit_weight[rank[i]] = place[i];
      __syncthreads();
      const uint64_t mine = threadIdx.x < n.k ? digit_weight[threadIdx.x] : 0u;
      const float v = logit_of(mine);
      const uint64_t units = threadIdx.x < n.k ? bins.units(v) : 0u;
      const uint64_t before = block.before(units), to = before + units;
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
        const uint64_t above = block.most(is ? to : 0u);
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
    histogram<true>(block, row, w);
    bins.take();
  } else {
    bins.load(a, r, parts, n.k != 0);
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
  extern "C" __global__ __launch_bounds__(1024, 8) void xpu_sample_look_##NAME(xpu::SampleArgs a) {             \
    xpu::sample::look<T>(a);                                                                                 \
  }                                                                                                          \
  extern "C" __global__ __launch_bounds__(1024, 8) void xpu_sample_list_##NAME(xpu::SampleArgs a) {             \
    xpu::sample::list<T>(a);                                                                                 \
  }                                                                                                          \
  extern "C" __global__ __launch_bounds__(256) void xpu_sample_draw_##NAME(xpu::SampleArgs a) {             \
    xpu::sample::draw<T>(a);                                                                                 \
  }
XPU_SAMPLE(xpu::kBf16, bf16)
XPU_SAMPLE(xpu::kFp16, fp16)
XPU_SAMPLE(xpu::sample::kFp32, fp32)
