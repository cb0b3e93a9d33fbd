// What the packed-prompt and the paged-cache attention share: one wavefront's
// R sub-tiles of 32 query rows against a tile of 32 T keys in LDS.
//
//   S^T = K Q^T      A operand: K rows from LDS, B operand: the wave's Q rows,
//                    held in registers; 32 x 32 tiles, so a lane has the
//                    scores of ONE query (lane % 32) for 16 T keys
//   online softmax   per query a reference m, p = 2^((s - m) scale log2 e),
//                    the FP32 sum of p, and the FP32 output columns; m moves
//                    (and sum and output are rescaled) only when a score
//                    passes it by more than 8 in the exponent, so p <= 256
//                    and rescales are rare after the first tiles; in fp16 all
//                    of it is 2^7 times as large (kLift)
//   O^T += V^T P^T   B operand: the lane's own p, rounded to the storage type
//                    where the MFMA reads it (the only rounding between the
//                    inputs and the result's own: with FP32 probabilities P V
//                    would take the FP32 MFMA, at a sixteenth of the rate; it
//                    puts results 1.2 to 1.4 times as far off 64 bits as FP32
//                    probabilities do), A operand: V^T by the transposing LDS
//                    read
//
// Register r of a 32 x 32 accumulator holds row 8 (r / 4) + 4 (lane / 32) +
// r % 4, so the keys of a lane's p are 4 hh .. 4 hh + 3 of every 8; the V^T
// reads take their rows in that order, and no lane exchange is needed.
//
// LDS tiles: key rows of 2 D bytes in 16-byte chunks, swizzled so that the
// K reads (32 rows, one chunk) and the V reads (4 rows, 4 chunks per half
// wave) each cover every bank once.
#pragma once
#include "device_common.hpp"

#include <type_traits>

namespace xpu {
namespace att {

using dma::f32x16;
using dma::lds_s16x4;

typedef uint32_t u32x8 __attribute__((ext_vector_type(8)));

constexpr float kLazy = 8.0f;  // rescale when the maximum grows by more, in powers of two
// p is formed 2^kLift times as large: fp16 then holds it to a full relative step
// from 2^-21 of the largest on, and to 2^-32 below (without: 2^-14 and 2^-25, and
// the many small ones of a long context came out up to 6% off), and with kLazy it
// stays below 2^15. The factor is in the sums and in the output alike, in every
// partial result, and cancels. bf16 has the exponents of FP32.
template <int DT> constexpr float kLift = DT == kFp16 ? 7.0f : 0.0f;
constexpr float kFar = 0x1p20f;  // a float holds powers of two up to here to 2^-4

// Physical chunk = chunk ^ swizzle(row).
template <int D> XPU_DEVICE uint32_t k_swz(uint32_t row) {
  if constexpr (D == 128) return row & 15u;  // 256-byte rows: 16 chunks
  else return (row >> 1) & 7u;               // 128-byte rows: two rows cover the banks
}
template <int D> XPU_DEVICE uint32_t v_swz(uint32_t row) {
  if constexpr (D == 128) return dma::b_swz(row & 3u);
  else return (row & 2u) ? 4u : 0u;
}

typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) u32x2 lds_u32x2;
typedef __attribute__((address_space(3))) uint32_t lds_u32;

// Whether a 32-bit word holds an infinity or NaN of the 16-bit type.
template <int DT> XPU_DEVICE bool nonfinite(uint32_t w) {
  constexpr uint32_t e = DT == kFp16 ? 0x7c00u : 0x7f80u;
  return (w & e) == e || (w & (e << 16)) == (e << 16);
}

// v + both 16-bit values of a word: one instruction for the two additions.
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
template <int DT> XPU_DEVICE float add_pair(uint32_t w, float v) {
  if constexpr (DT == kFp16)
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), f16x2{1.0f, 1.0f}, v, false);
  else
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), bf16x2{1.0f, 1.0f}, v, false);
}

// Sums of lanes 0 .. own, with DPP moves: shifts within rows of 16 lanes, then
// the rows' last lanes broadcast to the rows behind them.
XPU_DEVICE uint32_t sum_upto(uint32_t v) {
  auto add = [&](auto ctrl, auto rows) {
    v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), ctrl.value, rows.value, 0xf, false));
  };
  using std::integral_constant;
  constexpr integral_constant<int, 0xf> all;
  add(integral_constant<int, 0x111>{}, all);  // row_shr:1, 2, 4, 8
  add(integral_constant<int, 0x112>{}, all);
  add(integral_constant<int, 0x114>{}, all);
  add(integral_constant<int, 0x118>{}, all);
  add(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});  // row_bcast:15 to rows 1 and 3
  add(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});  // row_bcast:31 to rows 2 and 3
  return v;
}
XPU_DEVICE uint32_t wave_total(uint32_t v) { return __builtin_amdgcn_readlane(sum_upto(v), 63); }

// One wavefront's queries. R: sub-tiles of 32 rows.
template <int DT, int D, int R> struct Rows {
  static_assert(D == 64 || D == 128, "head sizes");
  static constexpr int kKs = D / 16, kDt = D / 32;
  static constexpr uint32_t kRow = 2u * D;  // bytes of a key row
  u32x4 q[R][kKs];
  f32x16 o[R][kDt];
  float m[R], sum[R], shift[R];
  float limit[R];  // wave-uniform: kLazy, or -inf where a reference is too large for its product with c (settle)
  uint32_t ka[kKs], va[kDt];  // the lane's LDS addresses in a K and a V tile at `base`

  // base: the LDS address that the tiles' offsets (kb, vb below) count from
  XPU_DEVICE void init(uint32_t base) {
    const uint32_t lane = lane_id(), hh = lane >> 5;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      m[r] = -__builtin_inff();
      sum[r] = shift[r] = 0.0f;
      limit[r] = kLazy;
#pragma unroll
      for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[r][dt][i] = 0.0f;
    }
    const uint32_t row = lane & 31u;
#pragma unroll
    for (uint32_t ks = 0; ks < kKs; ++ks) ka[ks] = base + row * kRow + 16u * ((2u * ks + hh) ^ k_swz<D>(row));
    // the transposing read: lane i of a 16-lane group gives row (i % 16) / 4
    // of the group's 4 rows, dims 16 ((lane / 16) % 2) + 4 (lane % 4)
    const uint32_t tr_row = (lane & 15u) >> 2, tr_chunk = 2u * ((lane >> 4) & 1u) + ((lane & 3u) >> 1);
#pragma unroll
    for (uint32_t dt = 0; dt < kDt; ++dt)
      va[dt] = base + (4u * hh + tr_row) * kRow + 16u * ((4u * dt + tr_chunk) ^ v_swz<D>(tr_row)) + 8u * (lane & 1u);
  }

  // The queries of sub-tile 0 from 32 rows at LDS offset `at`, laid out as a
  // tile's K rows: dims 16 ks + 8 hh .. + 7 of the lane's query in every ks.
  XPU_DEVICE void read_q(uint32_t at) {
#pragma unroll
    for (uint32_t ks = 0; ks < kKs; ++ks) q[0][ks] = *reinterpret_cast<const lds_u32x4 *>(ka[ks] + at);
  }
  // A sub-tile's queries in LDS, for wavefronts that have them in common: 16
  // bytes per lane for each ks.
  static constexpr uint32_t kQBytes = kKs * 1024u;

  // S^T of sub-tile r and a tile of 32 T keys at LDS offset kb; Q from
  // LDS at qb (QLDS) or from the registers. The reads run one step ahead of
  // the MFMAs; the barriers keep the compiler from moving all of them to the
  // front, which would take more registers than there are.
  template <int T, bool QLDS> XPU_DEVICE void scores(int r, uint32_t kb, uint32_t qb, f32x16 (&s)[T]) const {
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[t][i] = 0.0f;
    constexpr int kStep = 2;  // ks per step
    u32x4 kf[2][kStep][T], qf[2][kStep];
    auto read = [&](int step) {
#pragma unroll
      for (int j = 0; j < kStep; ++j) {
        const int ks = step * kStep + j;
#pragma unroll
        for (int t = 0; t < T; ++t)
          kf[step & 1][j][t] = *reinterpret_cast<const lds_u32x4 *>(kb + ka[ks] + 32u * t * kRow);
        if constexpr (QLDS)
          qf[step & 1][j] = *reinterpret_cast<const lds_u32x4 *>(qb + r * kQBytes + ks * 1024u + lane_id() * 16u);
        else
          qf[step & 1][j] = q[r][ks];
      }
    };
    read(0);
#pragma unroll
    for (int step = 0; step < kKs / kStep; ++step) {
      if (step + 1 < kKs / kStep) read(step + 1);
#pragma unroll
      for (int j = 0; j < kStep; ++j)
#pragma unroll
        for (int t = 0; t < T; ++t) s[t] = dma::mfma<DT>(kf[step & 1][j][t], qf[step & 1][j], s[t]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // Scores of keys that the query does not see: bit k of seen[t] is key
  // 32 t + k of the tile.
  template <int T> XPU_DEVICE static void mask(f32x16 (&s)[T], const uint32_t (&seen)[T]) {
    const uint32_t shift = 4u * (lane_id() >> 5);
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const uint32_t w = seen[t] >> shift;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (!(w >> (8 * (i / 4) + i % 4) & 1u)) s[t][i] = -__builtin_inff();
    }
  }

  // The largest score of each query.
  template <int T> XPU_DEVICE static float largest(const f32x16 (&s)[T]) {
    float top = -__builtin_inff();
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[t][i]);
    return fmaxf(top, xor32_f(top));  // the query's other half-wave
  }
  // Moves the reference where `top` passes it by more than kLazy. c = scale
  // log2 e > 0. The exponents are s c + shift in one FMA each; shift = -m c is
  // off by up to 2^-24 of itself, for all keys alike, which cancels in the
  // result as long as p stays in the storage type's range. Where a reference
  // passes kFar, the tile's scores become their differences from m, which are
  // exact enough at any size, and shift is 0: `limit` then lets every tile in
  // here, so that the others take one branch as before (8192 rows of 32 heads 490
  // us and 487 without the case, 128 rows of 16 heads 7.15 and 7.05; with a branch
  // of its own 505 and 496).
  template <int T> XPU_DEVICE void settle(int r, f32x16 (&s)[T], float top, float c) {
    const float ninf = -__builtin_inff(), by = (top - m[r]) * c;  // m = -inf: inf for any finite score
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(by >= limit[r]) != 0, 0)) {  // >=: by may be -inf
      const bool grow = by > kLazy;
      if (__builtin_amdgcn_ballot_w64(grow)) {
        const float now = grow ? top : m[r];
        const float a = m[r] == ninf ? 0.0f : __builtin_amdgcn_exp2f((m[r] - now) * c);
        sum[r] *= a;
#pragma unroll
        for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[r][dt][i] *= a;
        m[r] = now;
        if (__builtin_amdgcn_ballot_w64(now != ninf && __builtin_fabsf(now * c) > kFar)) limit[r] = ninf;
        shift[r] = limit[r] == ninf ? kLift<DT> : now == ninf ? 0.0f : kLift<DT> - now * c;
      }
      if (limit[r] == ninf) {
        const float from = m[r] == ninf ? 0.0f : m[r];
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[t][i] -= from;
      }
    }
  }
  // p of the tile packed as the MFMA takes it, word i of pk[t] for registers 2 i
  // and 2 i + 1, and their sum.
  template <int T> XPU_DEVICE void powers(int r, const f32x16 (&s)[T], float c, u32x8 (&pk)[T]) {
    float part = 0.0f;
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], c, shift[r]));
        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i + 1], c, shift[r]));
        pk[t][i / 2] = dma::cvt_pack<DT>(e0, e1);
        part = add_pair<DT>(pk[t][i / 2], part);
      }
    sum[r] += part;
  }
  template <int T> XPU_DEVICE void softmax(int r, f32x16 (&s)[T], float c, u32x8 (&pk)[T]) {
    settle<T>(r, s, largest<T>(s), c);
    powers<T>(r, s, c, pk);
  }

  // O^T += V^T P^T for the tile at LDS offset vb, the reads one step (16 keys)
  // ahead of the MFMAs.
  template <int T> XPU_DEVICE void values(uint32_t vb, const u32x8 (&pk)[R][T]) {
    u32x4 vf[2][kDt];
    auto read = [&](uint32_t ks) {
#pragma unroll
      for (uint32_t dt = 0; dt < kDt; ++dt) {
        const uint32_t at = vb + va[dt] + 16u * ks * kRow;
        const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(at)));
        const u32x2 hi =
            __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(at + 8u * kRow)));
        vf[ks & 1u][dt] = u32x4{lo.x, lo.y, hi.x, hi.y};
      }
    };
    read(0);
#pragma unroll
    for (uint32_t ks = 0; ks < 2 * T; ++ks) {
      if (ks + 1u < 2 * T) read(ks + 1u);
#pragma unroll
      for (uint32_t dt = 0; dt < kDt; ++dt)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const u32x8 &p = pk[r][ks / 2];
          const uint32_t b = 4u * (ks % 2);
          o[r][dt] = dma::mfma<DT>(vf[ks & 1u][dt], u32x4{p[b], p[b + 1], p[b + 2], p[b + 3]}, o[r][dt]);
        }
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // One wavefront's MFMAs leave its vector ALU free, so a tile's powers are
  // formed between the MFMAs of the next tile's scores, and that tile's
  // largest scores between those of P V. The order is given to the compiler
  // instruction by instruction: reads first, then an MFMA, a read and a share
  // of the vector work at a time.
  template <int DS, int VALU, int TRANS, int N, int AHEAD> XPU_DEVICE static void interleave() {
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);  // LDS reads
#pragma unroll
    for (int i = 0; i < N; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // an MFMA
      __builtin_amdgcn_sched_group_barrier(0x100, DS, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
      if (TRANS) __builtin_amdgcn_sched_group_barrier(0x400, TRANS, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  XPU_DEVICE void scores_powers(uint32_t kb, f32x16 (&next)[2], const f32x16 (&s)[2], float c, u32x8 (&pk)[2]) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) next[t][i] = 0.0f;
#pragma unroll
    for (int ks = 0; ks < kKs; ++ks)
#pragma unroll
      for (int t = 0; t < 2; ++t)
        next[t] = dma::mfma<DT>(*reinterpret_cast<const lds_u32x4 *>(kb + ka[ks] + 32u * t * kRow), q[0][ks], next[t]);
    powers<2>(0, s, c, pk);
    interleave<1, D == 128 ? 5 : 10, 0, 2 * kKs, 4>();
  }
  XPU_DEVICE float values_largest(uint32_t vb, const u32x8 (&pk)[2], const f32x16 (&next)[2]) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (uint32_t ks = 0; ks < 4; ++ks)
#pragma unroll
      for (uint32_t dt = 0; dt < kDt; ++dt) {
        const uint32_t at = va[dt] + vb + 16u * ks * kRow;
        const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(at)));
        const u32x2 hi =
            __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(at + 8u * kRow)));
        const u32x8 &p = pk[ks / 2];
        const uint32_t b = 4u * (ks % 2);
        o[0][dt] = dma::mfma<DT>(u32x4{lo.x, lo.y, hi.x, hi.y}, u32x4{p[b], p[b + 1], p[b + 2], p[b + 3]}, o[0][dt]);
      }
    const float top = largest<2>(next);
    interleave<2, 2, 0, 4 * kDt, 8>();
    return top;
  }

  // A tile with a non-finite value in a row that some query does not see: the
  // product 0 * inf of the MFMA would reach that query. So the rows that hold
  // one are added here to the queries that see them, and then cleared
  // (clear_apart) before values(). Rare; one key at a time.
  XPU_DEVICE void add_apart(uint32_t vb, int r, u32x8 pk, uint32_t seen) {
    const uint32_t hh = lane_id() >> 5;
#pragma unroll 1
    for (uint32_t key = 0; key < 32; ++key) {
      if (!row_apart(vb + key * kRow)) continue;
      const uint32_t i = 4u * (key / 8u) + key % 4u;
      const uint32_t own = pk[i / 2u] >> (16u * (i % 2u)) & 0xffffu, other = xor32_u(own);
      const bool sees = seen >> key & 1u;
      const float p = sees ? decode<DT>((key >> 2 & 1u) == hh ? own : other) : 0.0f;
      const uint32_t row = vb + key * kRow + 8u * hh;
#pragma unroll
      for (uint32_t dt = 0; dt < kDt; ++dt)
#pragma unroll
        for (uint32_t w = 0; w < 4; ++w) {
          const u32x2 v = *reinterpret_cast<const lds_u32x2 *>(row + 16u * ((4u * dt + w) ^ v_swz<D>(key)));
          const uint32_t x = sees ? v.x : 0u, y = sees ? v.y : 0u;
          o[r][dt][4u * w] = __builtin_fmaf(p, lo16<DT>(x), o[r][dt][4u * w]);
          o[r][dt][4u * w + 1u] = __builtin_fmaf(p, hi16<DT>(x), o[r][dt][4u * w + 1u]);
          o[r][dt][4u * w + 2u] = __builtin_fmaf(p, lo16<DT>(y), o[r][dt][4u * w + 2u]);
          o[r][dt][4u * w + 3u] = __builtin_fmaf(p, hi16<DT>(y), o[r][dt][4u * w + 3u]);
        }
    }
  }
  // Clears the rows with a non-finite value among `n` rows from LDS address at.
  XPU_DEVICE static void clear_apart(uint32_t at, uint32_t n) {
    asm volatile("" ::: "memory");
#pragma unroll 1
    for (uint32_t i = 0; i < n; ++i)
      if (row_apart(at + i * kRow)) *reinterpret_cast<lds_u32 *>(at + i * kRow + lane_id() * 4u % kRow) = 0u;
    asm volatile("" ::: "memory");
  }
  XPU_DEVICE static bool row_apart(uint32_t row) {
    const uint32_t w = *reinterpret_cast<const lds_u32 *>(row + lane_id() * 4u % kRow);
    return __builtin_amdgcn_ballot_w64(nonfinite<DT>(w)) != 0;
  }

  // The sum over both half-waves of each query.
  XPU_DEVICE float total(int r) const { return sum[r] + xor32_f(sum[r]); }

  // The 32 rows of sub-tile 0, each query's times its `by` and rounded to the
  // storage type, to `rows` rows of memory `stride` elements apart. Through 32
  // kRow bytes of LDS at address `at` that belong to the wavefront, so that
  // whole rows are stored (the lanes' own 8-byte pieces took twice the time of
  // all else in a short prompt's block), past the L2, which keeps the keys (24
  // sequences of 17 .. 1500 rows, 32 heads: 96.4 us with, 93.3 past it).
  XPU_DEVICE void store(uint32_t at, float by, uint16_t *to, uint64_t stride, uint32_t rows) const {
    constexpr uint32_t kCpr = D / 8, kRpi = 512u / D;
    const uint32_t lane = lane_id(), row = lane & 31u;
#pragma unroll
    for (uint32_t dt = 0; dt < kDt; ++dt)
#pragma unroll
      for (uint32_t w = 0; w < 4; ++w)
        *reinterpret_cast<lds_u32x2 *>(at + row * kRow + 16u * ((4u * dt + w) ^ k_swz<D>(row)) + 8u * (lane >> 5)) =
            u32x2{dma::cvt_pack<DT>(o[0][dt][4 * w] * by, o[0][dt][4 * w + 1] * by),
                  dma::cvt_pack<DT>(o[0][dt][4 * w + 2] * by, o[0][dt][4 * w + 3] * by)};
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (uint32_t j = 0; j < 32u / kRpi; ++j) {
      const uint32_t r = j * kRpi + lane / kCpr;
      const u32x4 v = *reinterpret_cast<const lds_u32x4 *>(at + r * kRow + 16u * ((lane % kCpr) ^ k_swz<D>(r)));
      if (r < rows) __builtin_nontemporal_store(v, reinterpret_cast<u32x4 *>(to + r * stride + lane % kCpr * 8u));
    }
  }
};

// Bits 0 .. last of a 32-key mask (last < 0: none, last >= 31: all).
XPU_DEVICE uint32_t mask_to(int32_t last) {
  return last < 0 ? 0u : last >= 31 ? 0xffffffffu : (2u << last) - 1u;
}

}  // namespace att
}  // namespace xpu
