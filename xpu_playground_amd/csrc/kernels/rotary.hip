// New rows into the paged cache, Q and K normalised per head and rotated on
// the way (xpu_cache_append_rotary, xpu_cache8_append).
//
//   n = x gain / sqrt(mean x^2 + eps)          per head, where there are gains
//   y_i = n_i cos - n_j sin, y_j = n_j cos + n_i sin
//
// for the pairs (i, j) = (i, i + half) or (2 i, 2 i + 1) of the first 2 half
// dims, with the row's cos and sin from FP32 tables. All of it is FP32, rounded
// once to what is stored. A lane holds 8 dims of a head (16 bytes), so a head's
// partners and its sum of squares are within a group of D / 8 lanes.
//
// In 8 bits a block of 16 positions of a head has one scale, a power of two: a
// code has a float's precision wherever it lies in the range, so the finer
// scales of other forms would not add any, and codes are rescaled exactly as
// long as they stay normal. A wavefront takes a whole block of K or of V, so
// the new rows' largest value is known before the first code is formed and no
// block is written by two.
//
// Memory bounds both where there are many rows: 24 prompts of 17 .. 1500 rows,
// 32 and 8 heads of size 128, 54 us in 16 bits with gains (220 MB, 4.05 TB/s),
// 54 in 8 bits with half of the dims turned, 65 with all and gains. A step's few
// rows are one launch and a chain of loads: 48 rows 4.4 us and 7.9, one 7.6.
#include "cache_types.hpp"
#include "device_common.hpp"

namespace xpu {
namespace cache {

// Sum over groups of D / 8 lanes; every lane of a group ends with it.
template <int D> XPU_DEVICE float group_sum(float s) {
  s += dpp_f<0xB1>(s);   // quad_perm [1,0,3,2]
  s += dpp_f<0x4E>(s);   // quad_perm [2,3,0,1]
  s += dpp_f<0x141>(s);  // row_half_mirror: the other quad of 8
  if constexpr (D == 128) s += dpp_f<0x140>(s);  // row_mirror: the other half of 16
  return s;
}

// What a lane needs of a row's table entry: cos and sin of its dims' pairs
// (halves: of 8, adjacent: of 4). Zero positions (no tables) load nothing.
struct Angles {
  float c[8], s[8];
};
template <int D> XPU_DEVICE Angles angles_of(const RotaryArgs &r, uint32_t pos) {
  Angles a;
  const uint32_t dim = lane_id() % (D / 8u) * 8u;
  const bool turns = dim < 2u * r.half && pos < r.positions;
  const uint32_t first = r.adjacent ? dim / 2u : dim < r.half ? dim : dim - r.half;
  const uint64_t at = turns ? static_cast<uint64_t>(pos) * r.half + first : 0u;
#pragma unroll
  for (uint32_t i = 0; i < 8; i += 4) {
    dma::f32x4 c{1.0f, 1.0f, 1.0f, 1.0f}, s{};
    if (turns && !(r.adjacent && i)) {
      c = *reinterpret_cast<const dma::f32x4 *>(r.cos + at + i);
      s = *reinterpret_cast<const dma::f32x4 *>(r.sin + at + i);
    }
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      a.c[i + j] = c[j];
      a.s[i + j] = s[j];
    }
  }
  return a;
}

// x normalised by the lane's gain (NULL: not) and rotated. All 64 lanes.
template <int DT, int D> XPU_DEVICE void turn(float (&x)[8], const RotaryArgs &r, const Angles &a, const uint16_t *gain) {
  const uint32_t lane = lane_id(), dim = lane % (D / 8u) * 8u;
  if (__builtin_amdgcn_ballot_w64(gain != nullptr)) {
    float ss = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) ss = __builtin_fmaf(x[i], x[i], ss);
    const float by = 1.0f / __builtin_sqrtf(group_sum<D>(ss) * (1.0f / D) + r.eps);
    if (gain) {
      float g[8];
      unpack8<DT>(*reinterpret_cast<const u32x4 *>(gain + dim), g);
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) x[i] = x[i] * by * g[i];
    }
  }
  if (r.half == 0) return;
  if (r.adjacent) {
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const float u = x[2 * i], v = x[2 * i + 1];
      if (dim < 2u * r.half) {
        x[2 * i] = u * a.c[i] - v * a.s[i];
        x[2 * i + 1] = v * a.c[i] + u * a.s[i];
      }
    }
  } else {
    const bool low = dim < r.half;
    const uint32_t step = r.half / 8u;
    const int partner = static_cast<int>(dim >= 2u * r.half ? lane : low ? lane + step : lane - step);
    const bool row = D == 128 && r.half == 64;  // the other half of a row of 16 lanes
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const float other = row ? xor8_f(x[i]) : __shfl(x[i], partner), s = low ? -a.s[i] : a.s[i];
      if (dim < 2u * r.half) x[i] = x[i] * a.c[i] + other * s;
    }
  }
}

// A wavefront's loads of rows on their way (one: the 8-bit prompts with all dims
// and gains 71 us instead of 65; no difference in 16 bits).
constexpr uint32_t kAhead = 4;

template <int DT> XPU_DEVICE u32x4 pack8(const float (&x)[8]) {
  return u32x4{dma::cvt_pack<DT>(x[0], x[1]), dma::cvt_pack<DT>(x[2], x[3]), dma::cvt_pack<DT>(x[4], x[5]),
               dma::cvt_pack<DT>(x[6], x[7])};
}

// A row's place in its sequence. turned: the position of its rotation.
struct RowAt {
  int32_t seq;
  uint64_t pos;
  uint32_t turned;
};
XPU_DEVICE RowAt row_at(const BatchArgs &b, const RotaryArgs &r, uint32_t row) {
  const Holder h = holder_of(b, row);
  if (h.seq < 0) return {-1, 0, 0};
  const uint64_t pos = static_cast<uint64_t>(b.context[h.seq]) + (row - h.first);
  const uint64_t at = r.at ? r.at[row] : pos;
  return {h.seq, pos, at < 0xffffffffull ? static_cast<uint32_t>(at) : 0xffffffffu};
}

// Q alone, of the heads of wave part `part` of a row's parts; a row whose
// position the tables do not have is NaN.
template <int DT, int D> XPU_DEVICE void turn_q(const RotateArgs &a, uint32_t row, uint32_t part) {
  constexpr uint32_t kGroup = D / 8, kPer = 64 / kGroup;
  const RowAt at = row_at(a.batch, a.rot, row);
  if (at.seq < 0) return;
  const bool known = a.rot.half == 0 || at.turned < a.rot.positions;
  if (!known) report(a.pool);
  const Angles angles = angles_of<D>(a.rot, at.turned);
  const uint32_t lane = lane_id(), dim = lane % kGroup * 8u, step = a.parts * kPer;
  for (uint32_t h0 = part * kPer; h0 < a.heads; h0 += kAhead * step) {
    auto head = [&](uint32_t j) { return h0 + j * step + lane / kGroup; };
    auto at_of = [&](uint32_t j) { return min(head(j), a.heads - 1u) * D + dim; };
    u32x4 raw[kAhead];
#pragma unroll
    for (uint32_t j = 0; j < kAhead; ++j) raw[j] = *reinterpret_cast<const u32x4 *>(a.q + row * a.q_stride + at_of(j));
#pragma unroll
    for (uint32_t j = 0; j < kAhead; ++j) {
      if (h0 + j * step >= a.heads) break;
      float x[8];
      unpack8<DT>(raw[j], x);
      turn<DT, D>(x, a.rot, angles, a.rot.q_gain);
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) x[i] = known ? x[i] : __builtin_nanf("");
      if (head(j) < a.heads) *reinterpret_cast<u32x4 *>(a.q_out + row * a.out_stride + at_of(j)) = pack8<DT>(x);
    }
  }
}

// 16 bits. A wavefront takes part of a row's Q, K and V heads, 64 / (D / 8) at
// a time.
template <int DT, int D> XPU_DEVICE void append_rotary(const RotateArgs &a) {
  constexpr uint32_t kGroup = D / 8, kPer = 64 / kGroup;
  const uint32_t lane = lane_id(), dim = lane % kGroup * 8u, kv = a.pool.kv_heads, total = a.heads + 2u * kv;
  const uint64_t waves = gridDim.x * 4ull, all = static_cast<uint64_t>(a.batch.rows) * a.parts;
  for (uint64_t w = blockIdx.x * 4u + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); w < all; w += waves) {
    const uint32_t row = static_cast<uint32_t>(w / a.parts), part = static_cast<uint32_t>(w % a.parts);
    const RowAt at = row_at(a.batch, a.rot, row);
    if (at.seq < 0) continue;
    const bool known = at.turned < a.rot.positions;
    const uint64_t place = element_of(a.pool, a.batch.tables + static_cast<uint64_t>(at.seq) * a.batch.table_pitch,
                                      a.batch.table_pitch, at.pos, D);
    if (!known || place == kNowhere) report(a.pool);
    const Angles angles = angles_of<D>(a.rot, at.turned);
    const uint32_t step = a.parts * kPer;
    for (uint32_t u0 = part * kPer; u0 < total; u0 += kAhead * step) {
      struct Unit {
        bool is_q, is_v;
        uint32_t head;
      };
      auto unit_of = [&](uint32_t j) {
        const uint32_t in = min(u0 + j * step + lane / kGroup, total - 1u);
        return Unit{in < a.heads, in >= a.heads + kv, in < a.heads ? in : (in - a.heads) % kv};
      };
      u32x4 raw[kAhead];
#pragma unroll
      for (uint32_t j = 0; j < kAhead; ++j) {
        const Unit u = unit_of(j);
        const uint16_t *from = u.is_q ? a.q + row * a.q_stride : u.is_v ? a.v + row * a.v_stride : a.k + row * a.k_stride;
        raw[j] = *reinterpret_cast<const u32x4 *>(from + u.head * D + dim);
      }
#pragma unroll
      for (uint32_t j = 0; j < kAhead; ++j) {
        if (u0 + j * step >= total) break;
        const Unit u = unit_of(j);
        float x[8];
        unpack8<DT>(raw[j], x);
        turn<DT, D>(x, a.rot, angles, u.is_q ? a.rot.q_gain : u.is_v ? nullptr : a.rot.k_gain);
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) x[i] = known ? x[i] : __builtin_nanf("");
        const u32x4 y = u.is_v ? raw[j] : pack8<DT>(x);
        if (u0 + j * step + lane / kGroup >= total || (!u.is_q && (!known || place == kNowhere))) continue;
        uint16_t *to = u.is_q ? a.q_out + row * a.out_stride + u.head * D
                              : (u.is_v ? a.pool.v : a.pool.k) + place + static_cast<uint64_t>(u.head) * a.pool.page_size * D;
        *reinterpret_cast<u32x4 *>(to + dim) = y;
      }
    }
  }
}

// Eight values times 2^(127 - scale) as codes; infinities become NaN.
XPU_DEVICE u32x2 codes8(const float (&x)[8], uint32_t scale) {
  const float by = __uint_as_float((254u - min(scale, 253u)) << 23);
  float y[8];
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i) y[i] = __builtin_fabsf(x[i]) < __builtin_inff() ? x[i] * by : __builtin_nanf("");
  u32x2 c;
#pragma unroll
  for (uint32_t w = 0; w < 2; ++w) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * w], y[4 * w + 1], 0, false);
    c[w] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * w + 2], y[4 * w + 3], v, true));
  }
  return c;
}
// Codes times 2^(from - to), from <= to.
XPU_DEVICE u32x2 rescaled(u32x2 c, uint32_t from, uint32_t to) {
  const float by = __uint_as_float((127u - min(to - from, 126u)) << 23);
  u32x2 r;
#pragma unroll
  for (uint32_t w = 0; w < 2; ++w) {
    const dma::f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(c[w]), false);
    const dma::f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(c[w]), true);
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(lo.x * by, lo.y * by, 0, false);
    r[w] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(hi.x * by, hi.y * by, v, true));
  }
  return r;
}

// Largest value of lanes 0 .. own.
XPU_DEVICE uint32_t most_upto(uint32_t v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t o = __shfl_up(v, d);
    if (lane_id() >= static_cast<uint32_t>(d)) v = max(v, o);
  }
  return v;
}

// The batch's reached blocks are numbered sequence by sequence; block `item`,
// or seq -1. One lane per sequence, 64 at a time. Rows that an earlier sequence
// has are not the later one's, so there are never more blocks than slots.
struct BlockAt {
  int32_t seq;
  uint32_t block;     // of the sequence's reached ones
  uint32_t first, n;  // the sequence's rows
  uint64_t context;   // positions before them
  uint32_t claimed;   // of these positions, the last ones that are an earlier sequence's rows
};
XPU_DEVICE BlockAt block_at(const BatchArgs &b, uint32_t item) {
  uint32_t before = 0, taken = 0;  // blocks and rows of the sequences before
  for (uint32_t at = 0; at < b.n_seqs; at += 64) {
    const uint32_t i = at + lane_id();
    uint32_t lo = 0, hi = 0, c = 0;
    if (i < b.n_seqs) {
      lo = b.starts[i];
      hi = b.starts[i + 1u];
      c = b.context[i];
      if (lo > hi || hi > b.rows) lo = hi = 0;
    }
    const uint32_t most = max(taken, most_upto(hi)), prior = __shfl_up(most, 1);
    const uint32_t first = max(lo, lane_id() ? prior : taken), n = hi > first ? hi - first : 0u;
    const uint32_t count = blocks_of(n, c + (first - lo)), upto = before + att::sum_upto(count);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(item < upto && item >= upto - count);
    if (hit) {
      const uint32_t l = __builtin_ctzll(hit);
      auto of = [&](uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(v, l)); };
      return {static_cast<int32_t>(at + l), item - of(upto - count), of(first), of(n),
              static_cast<uint64_t>(of(c)) + of(first - lo), of(first - lo)};
    }
    before = __builtin_amdgcn_readlane(upto, 63);
    taken = __builtin_amdgcn_readlane(most, 63);
  }
  return {-1, 0, 0, 0, 0, 0};
}

// 8 bits: the rows of one block of one kv head, K or V, by a wavefront.
template <int DT, int D> XPU_DEVICE void append_block(const RotateArgs &a, const BlockAt &b, uint32_t head, bool is_v) {
  constexpr uint32_t kGroup = D / 8, kPer = 64 / kGroup, kLoads = kBlock / kPer;
  const uint32_t lane = lane_id(), dim = lane % kGroup * 8u;
  const uint32_t in = static_cast<uint32_t>(b.context) & (kBlock - 1u);  // positions of the first block before the rows
  const uint64_t start = b.context - in + static_cast<uint64_t>(b.block) * kBlock;
  const uint32_t before = b.block ? 0u : in;
  const uint32_t held = before > b.claimed ? before - b.claimed : 0u;  // rows that the sequence has there
  const uint32_t done = b.block ? b.block * kBlock - in : 0u;          // rows in earlier blocks
  const uint32_t count = min(b.n - done, kBlock - before), row0 = b.first + done;
  const uint64_t place = element_of(a.pool, a.batch.tables + static_cast<uint64_t>(b.seq) * a.batch.table_pitch,
                                    a.batch.table_pitch, start, D);
  if (place == kNowhere) {
    report(a.pool);
    return;
  }
  const uint64_t slot = (start & (a.pool.page_size - 1u)), page = place - slot * D;
  uint8_t *pool = reinterpret_cast<uint8_t *>(is_v ? a.pool.v : a.pool.k) + page;
  uint8_t *codes = pool + (static_cast<uint64_t>(head) * a.pool.page_size + slot) * D + dim;
  uint8_t *scale = pool + static_cast<uint64_t>(a.pool.kv_heads) * a.pool.page_size * D +
                   head * (a.pool.page_size / kBlock) + slot / kBlock;
  const uint16_t *from = (is_v ? a.v : a.k) + head * D + dim;
  const uint64_t stride = is_v ? a.v_stride : a.k_stride;
  const uint32_t old = held ? *scale : 0u;
  float x[kLoads][8];
  bool real[kLoads];
  bool odd = false;
  uint32_t top = 0;
#pragma unroll
  for (uint32_t l = 0; l < kLoads; ++l) {
    const uint32_t j = l * kPer + lane / kGroup, row = row0 + min(j, count - 1u);
    unpack8<DT>(*reinterpret_cast<const u32x4 *>(from + row * stride), x[l]);
    real[l] = j < count;
    if (a.rot.half) {  // (a row without angles is not written, neither K nor V)
      const uint64_t at = a.rot.at ? a.rot.at[row] : start + before + j;
      const uint32_t turned = at < 0xffffffffull ? static_cast<uint32_t>(at) : 0xffffffffu;
      if (turned >= a.rot.positions) {
        odd |= real[l];
        real[l] = false;
      }
      if (!is_v) turn<DT, D>(x[l], a.rot, angles_of<D>(a.rot, turned), a.rot.k_gain);
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const uint32_t bits = __float_as_uint(x[l][i]) & 0x7fffffffu;
      if (real[l] && bits < 0x7f800000u) top = max(top, bits);
    }
  }
  if (__builtin_amdgcn_ballot_w64(odd)) report(a.pool);
  // (bits of finite positive floats are ordered as these)
  top = __float_as_uint(wave_reduce(__uint_as_float(top), [](float p, float q) { return fmaxf(p, q); }));
  const uint32_t now = max(max(scale_for(top), kLeastScale), old);
  if (held && now > old) {
#pragma unroll
    for (uint32_t l = 0; l < kLoads; ++l) {
      const uint32_t j = l * kPer + lane / kGroup;
      if (j < held) {
        u32x2 *c = reinterpret_cast<u32x2 *>(codes + j * D);
        *c = rescaled(*c, old, now);
      }
    }
  }
#pragma unroll
  for (uint32_t l = 0; l < kLoads; ++l) {
    const uint32_t j = l * kPer + lane / kGroup;
    const u32x2 c = codes8(x[l], now);
    if (real[l]) *reinterpret_cast<u32x2 *>(codes + (before + j) * D) = c;
  }
  if (lane == 0) *scale = static_cast<uint8_t>(now);
}

// The first wavefronts take the blocks (item, kv head, K or V), the others Q's
// rows (row, part).
template <int DT, int D> XPU_DEVICE void append8(const RotateArgs &a) {
  const uint32_t parts = 2u * a.pool.kv_heads;
  const uint64_t blocks = static_cast<uint64_t>(a.slots) * parts, rows = a.heads ? a.batch.rows : 0u;
  const uint64_t waves = gridDim.x * 4ull;
  for (uint64_t w = blockIdx.x * 4u + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); w < blocks + rows * a.parts;
       w += waves) {
    if (w < blocks) {
      const uint32_t part = static_cast<uint32_t>(w % parts);
      const BlockAt b = block_at(a.batch, static_cast<uint32_t>(w / parts));
      if (b.seq >= 0) append_block<DT, D>(a, b, part / 2u, part % 2u);
    } else {
      turn_q<DT, D>(a, static_cast<uint32_t>((w - blocks) / a.parts), static_cast<uint32_t>((w - blocks) % a.parts));
    }
  }
}

}  // namespace cache
}  // namespace xpu

#define XPU_APPEND_ROTARY(T, NAME, D)                                                                                 \
  extern "C" __global__ __launch_bounds__(256) void xpu_cache_append_rotary_##NAME(xpu::RotateArgs a) {               \
    xpu::cache::append_rotary<xpu::T, D>(a);                                                                          \
  }                                                                                                                   \
  extern "C" __global__ __launch_bounds__(256) void xpu_cache8_append_##NAME(xpu::RotateArgs a) {                     \
    xpu::cache::append8<xpu::T, D>(a);                                                                                \
  }
XPU_APPEND_ROTARY(kBf16, bf16_d128, 128)
XPU_APPEND_ROTARY(kFp16, fp16_d128, 128)
XPU_APPEND_ROTARY(kBf16, bf16_d64, 64)
XPU_APPEND_ROTARY(kFp16, fp16_d64, 64)
