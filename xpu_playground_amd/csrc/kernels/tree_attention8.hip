// Attention of drafted tokens over a cache of 8-bit pages (xpu_tree_attention8):
// tree_attention.hip's plan, softmax and joins; keys and values are codes (e4m3)
// times a power of two for every 16 positions of a kv head.
//
//   S^T = K Q^T, O^T += V^T P^T on the 16-bit MFMA of the queries' type: the
//   codes become 16-bit values, scale and all, in one instruction for two of
//   them on their way from LDS into the MFMA, exactly in bf16 (4 significant
//   bits, FP32's exponents; in fp16 rounded below 2^-14). So Q and the
//   probabilities keep their 16 bits; the 8-bit MFMA would take both in 4
//   significant bits.
//
// K: 16 bytes of LDS are 16 dims of a key, two steps of the MFMA's 16 with the
// other half-wave's; the queries are laid out to match. V: the transposing
// read of bytes gives a lane 8 keys of a dim, which is a whole operand; a
// lane's keys are those that the scores' registers hold, as for 16 bits.
//
// A tile of 32 keys has half the bytes of a 16-bit one, so each wavefront has
// two stages of tiles, as many bytes on their way.
#include "attention_core.hpp"
#include "cache_types.hpp"

namespace xpu {
namespace att {

typedef __attribute__((address_space(3))) i32x2 lds_i32x2;

// Two codes (the low or high pair of a word) times `scale` as 16-bit values.
template <int DT, bool HI> XPU_DEVICE uint32_t widen2(uint32_t w, float scale) {
  if constexpr (DT == kFp16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w), scale, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(w), scale, HI));
}
template <int DT> XPU_DEVICE u32x4 widen8(uint32_t lo, uint32_t hi, float scale) {
  return u32x4{widen2<DT, false>(lo, scale), widen2<DT, true>(lo, scale), widen2<DT, false>(hi, scale),
               widen2<DT, true>(hi, scale)};
}

// LDS tiles: key rows of D bytes in 16-byte chunks, physical chunk = chunk ^
// swizzle(row), so that the K reads (32 rows, one chunk) and the V reads (8
// rows, 2 chunks per half-wave) cover every bank alike.
template <int D> XPU_DEVICE uint32_t k8_swz(uint32_t row) {
  if constexpr (D == 128) return (row >> 1) & 7u;  // 128-byte rows: two cover the banks
  else return (row >> 2) & 3u;                     // 64-byte rows: four do
}
template <int D> XPU_DEVICE uint32_t v8_swz(uint32_t row) {
  if constexpr (D == 128) return (row & 2u) | (row >> 1 & 4u);
  else return row >> 2 & 2u;
}

// Whether codes times 2^(scale - 127) can be infinite in the 16-bit type.
template <int DT> XPU_DEVICE bool wide(uint32_t scale) { return scale > (DT == kFp16 ? 127u + 7u : 127u + 119u); }

template <int DT, int D, int R> struct Rows8 : Rows<DT, D, R> {
  using Base = Rows<DT, D, R>;
  using Base::kDt;
  using Base::kKs;
  static constexpr uint32_t kRow8 = D;
  uint32_t ka8[D / 32], va8[D / 32];

  XPU_DEVICE void init8(uint32_t base) {
    Base::init(base);
    const uint32_t lane = lane_id(), hh = lane >> 5, row = lane & 31u;
#pragma unroll
    for (uint32_t j = 0; j < D / 32; ++j) ka8[j] = base + row * kRow8 + 16u * ((2u * j + hh) ^ k8_swz<D>(row));
    // lane i of a 16-lane group gives 8 bytes of row (i % 16) / 2 of the group's
    // 8 rows and gets byte i % 16 of each
    const uint32_t at = (lane & 15u) >> 1, key = (at < 4u ? at : at + 4u) + 4u * hh;
#pragma unroll
    for (uint32_t dt = 0; dt < kDt; ++dt)
      va8[dt] = base + key * kRow8 + 16u * ((2u * dt + (lane >> 4 & 1u)) ^ v8_swz<D>(key)) + 8u * (lane & 1u);
  }

  // S^T of sub-tile r and 32 keys at LDS offset kb, of `scale` for the lane's
  // key; Q from LDS at qb.
  XPU_DEVICE void scores8(int r, uint32_t kb, uint32_t qb, float scale, f32x16 &s) const {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.0f;
    u32x4 kf[2], qf[2][2];
    auto read = [&](int j) {
      kf[j & 1] = *reinterpret_cast<const lds_u32x4 *>(kb + ka8[j]);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        qf[j & 1][i] =
            *reinterpret_cast<const lds_u32x4 *>(qb + r * Base::kQBytes + (2 * j + i) * 1024u + lane_id() * 16u);
    };
    read(0);
#pragma unroll
    for (int j = 0; j < kKs / 2; ++j) {
      if (j + 1 < kKs / 2) read(j + 1);
      const u32x4 &k = kf[j & 1];
      s = dma::mfma<DT>(widen8<DT>(k.x, k.y, scale), qf[j & 1][0], s);
      s = dma::mfma<DT>(widen8<DT>(k.z, k.w, scale), qf[j & 1][1], s);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // O^T += V^T P^T of the tile at LDS offset vb, of scale[ks] for keys 16 ks ...
  XPU_DEVICE void values8(uint32_t vb, const float (&scale)[2], const u32x8 (&pk)[R][1]) {
    i32x2 vf[2][kDt];
    auto read = [&](uint32_t ks) {
#pragma unroll
      for (uint32_t dt = 0; dt < kDt; ++dt)
        vf[ks][dt] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2 *)(vb + va8[dt] + 16u * ks * kRow8));
    };
    read(0);
#pragma unroll
    for (uint32_t ks = 0; ks < 2; ++ks) {
      if (ks == 0) read(1);
#pragma unroll
      for (uint32_t dt = 0; dt < kDt; ++dt) {
        const u32x4 v = widen8<DT>(static_cast<uint32_t>(vf[ks][dt].x), static_cast<uint32_t>(vf[ks][dt].y), scale[ks]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const u32x8 &p = pk[r][0];
          const uint32_t b = 4u * ks;
          this->o[r][dt] = dma::mfma<DT>(v, u32x4{p[b], p[b + 1], p[b + 2], p[b + 3]}, this->o[r][dt]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // A row with an infinite value or a NaN (wave-uniform).
  XPU_DEVICE static bool row_apart8(uint32_t row, float scale) {
    const uint32_t w = *reinterpret_cast<const lds_u32 *>(row + lane_id() * 4u % kRow8);
    return __builtin_amdgcn_ballot_w64(nonfinite<DT>(widen2<DT, false>(w, scale)) ||
                                       nonfinite<DT>(widen2<DT, true>(w, scale))) != 0;
  }
  // As add_apart and clear_apart of 16-bit tiles.
  XPU_DEVICE void add_apart8(uint32_t vb, const float (&scale)[2], int r, u32x8 pk, uint32_t seen) {
    const uint32_t hh = lane_id() >> 5;
#pragma unroll 1
    for (uint32_t key = 0; key < 32; ++key) {
      const float by = key < 16u ? scale[0] : scale[1];
      if (!row_apart8(vb + key * kRow8, by)) continue;
      const uint32_t i = 4u * (key / 8u) + key % 4u;
      const uint32_t own = pk[i / 2u] >> (16u * (i % 2u)) & 0xffffu, other = xor32_u(own);
      const bool sees = seen >> key & 1u;
      const float p = sees ? decode<DT>((key >> 2 & 1u) == hh ? own : other) : 0.0f;
      const uint32_t row = vb + key * kRow8 + 4u * hh;
#pragma unroll
      for (uint32_t dt = 0; dt < kDt; ++dt)
#pragma unroll
        for (uint32_t w = 0; w < 4; ++w) {
          const uint32_t c =
              *reinterpret_cast<const lds_u32 *>(row + 16u * ((2u * dt + w / 2u) ^ v8_swz<D>(key)) + 8u * (w % 2u));
          const uint32_t x = sees ? widen2<DT, false>(c, by) : 0u, y = sees ? widen2<DT, true>(c, by) : 0u;
          f32x16 &o = this->o[r][dt];
          o[4u * w] = __builtin_fmaf(p, lo16<DT>(x), o[4u * w]);
          o[4u * w + 1u] = __builtin_fmaf(p, hi16<DT>(x), o[4u * w + 1u]);
          o[4u * w + 2u] = __builtin_fmaf(p, lo16<DT>(y), o[4u * w + 2u]);
          o[4u * w + 3u] = __builtin_fmaf(p, hi16<DT>(y), o[4u * w + 3u]);
        }
    }
  }
  XPU_DEVICE static void clear_apart8(uint32_t at, const float (&scale)[2]) {
    asm volatile("" ::: "memory");
#pragma unroll 1
    for (uint32_t i = 0; i < 32; ++i)
      if (row_apart8(at + i * kRow8, i < 16u ? scale[0] : scale[1]))
        *reinterpret_cast<lds_u32 *>(at + i * kRow8 + lane_id() * 4u % kRow8) = 0u;
    asm volatile("" ::: "memory");
  }
};

template <int DT, int D, int R> XPU_DEVICE void tree_attention8(const TreeArgs &a) {
  constexpr uint32_t kRow = D, kTile = kTreeKeys * kRow, kStage = 2u * kTile;
  constexpr uint32_t kRpi = 1024u / D, kCpr = D / 16;
  constexpr uint32_t kDma = kTreeKeys / kRpi;  // DMA instructions per tile, K and V each
  // per wavefront two stages of a K and a V tile; then the partial results
  __shared__ __align__(1024) uint8_t lds[8u * kStage];
  static_assert(8u * kStage == 4u * 64u * (D / 2u) * 4u, "the partial results fit the tiles' memory");
  __shared__ __align__(16) uint8_t shared_q[R * Rows<DT, D, R>::kQBytes];

  const uint32_t tid = threadIdx.x, lane = tid & 63u, hh = lane >> 5;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t kvh = blockIdx.x % a.pool.kv_heads, item = blockIdx.x / a.pool.kv_heads;
  const uint32_t group = a.heads / a.pool.kv_heads;
  const Place place = find<R>(a, group, [&](uint32_t first, uint32_t count, const Sequence &) {
    return item >= first && item - first < count;
  });
  if (place.seq < 0) return;
  const uint32_t seq = static_cast<uint32_t>(place.seq);
  const Sequence &s = place.s;
  const uint32_t row_tile = (item - place.first) % s.row_tiles, chunk = (item - place.first) / s.row_tiles;
  const uint32_t c0 = static_cast<uint32_t>(static_cast<uint64_t>(s.tiles) * chunk / place.chunks);
  const uint32_t c1 = static_cast<uint32_t>(static_cast<uint64_t>(s.tiles) * (chunk + 1u) / place.chunks);
  const uint32_t t_lo = c0 + (c1 - c0) * wave / 4u, t_hi = c0 + (c1 - c0) * (wave + 1u) / 4u;

  // Page ids and scales of the wave's blocks of 16 keys, 64 at a time, a lane
  // each: the ids one window ahead of the tiles that are asked for, the scales
  // of a window once its ids are there, which is two tiles before their use.
  const uint32_t *table = a.batch.tables + static_cast<uint64_t>(seq) * a.batch.table_pitch;
  const uint8_t *k_pool = reinterpret_cast<const uint8_t *>(a.pool.k), *v_pool = reinterpret_cast<const uint8_t *>(a.pool.v);
  const uint32_t blocks = (s.end + kBlock - 1u) / kBlock, per = a.pool.page_size / kBlock;
  const uint64_t scales_at = static_cast<uint64_t>(a.pool.kv_heads) * a.pool.page_size * D + kvh * per;
  auto ids_of = [&](uint32_t from) {
    const uint32_t at = from + lane;
    return at < blocks ? table[at * kBlock >> a.pool.page_shift] : ~0u;
  };
  auto scales_of = [&](uint32_t from, uint32_t id) {  // K's, and V's in the high half
    if (id >= a.pool.n_pages) return 127u | 127u << 16;
    const uint64_t at = static_cast<uint64_t>(id) * a.pool.page_stride + scales_at + (from + lane) % per;
    return static_cast<uint32_t>(k_pool[at]) | static_cast<uint32_t>(v_pool[at]) << 16;
  };
  uint32_t w_from = 2u * t_lo, s_from = w_from;
  uint32_t ids = ids_of(w_from), ids_next = ids_of(w_from + 64u);

  const uint32_t qb = __builtin_amdgcn_readfirstlane(lds_addr(shared_q));
  Rows8<DT, D, R> rows;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(lds)) + wave * 2u * kStage;
  rows.init8(lds0);
  uint32_t node[R];
  uint64_t sees[R];  // bit j: node j
  u32x4 q_part[R][D / 64];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t row = min(32u * (row_tile * R + r) + (lane & 31u), s.n * group - 1u);
    node[r] = row / group;
    const uint16_t *q_row = a.q + (s.first + node[r]) * a.q_stride + (kvh * group + row % group) * D;
#pragma unroll
    for (uint32_t j = 0; j < D / 64; ++j) {
      const uint32_t ks = wave * (D / 64u) + j;  // dims 32 (ks / 2) + 16 hh + 8 (ks % 2) ...
      q_part[r][j] = *reinterpret_cast<const u32x4 *>(q_row + 32u * (ks / 2u) + 16u * hh + 8u * (ks % 2u));
    }
    if (a.visible) {
      sees[r] = a.visible[s.first + node[r]];
      if (s.n < 64u) sees[r] &= (1ull << s.n) - 1ull;
    }
  }
  bool bad = s.bad || (a.visible && s.n > 64u);
  uint32_t scales = scales_of(w_from, ids), scales_next = 0;

  constexpr uint32_t kHalf = kDma / 2;  // per block of 16 keys
  uint32_t k_off[kHalf], v_off[kHalf];
#pragma unroll
  for (uint32_t j = 0; j < kHalf; ++j) {
    const uint32_t row = kRpi * j + lane / kCpr;
    k_off[j] = row * kRow + 16u * ((lane % kCpr) ^ k8_swz<D>(row));
    v_off[j] = row * kRow + 16u * ((lane % kCpr) ^ v8_swz<D>(row));
  }
  const uint64_t head_at = static_cast<uint64_t>(kvh) * a.pool.page_size * D;
  // A tile is two blocks of 16 keys. The descriptor ends with the sequence; a
  // page id past the pool reads nothing.
  uint64_t from[2];
  uint32_t live[2];
  auto locate = [&](uint32_t tile) {
    if (2u * tile - w_from >= 64u) {
      w_from += 64u;
      ids = ids_next;
      ids_next = ids_of(w_from + 64u);
      scales_next = scales_of(w_from, ids);
    }
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t pos = tile * kTreeKeys + 16u * h;
      const uint32_t id = __builtin_amdgcn_readlane(ids, 2u * tile + h - w_from);
      uint32_t n = pos < s.end ? min(s.end - pos, 16u) : 0u;
      if (id >= a.pool.n_pages) {
        bad |= n != 0;
        n = 0;
      }
      from[h] = n ? static_cast<uint64_t>(id) * a.pool.page_stride + head_at +
                        static_cast<uint64_t>(pos & (a.pool.page_size - 1u)) * D
                  : 0u;
      live[h] = n * kRow;
    }
  };
  const bool once = s.row_tiles == 1;  // keys that only this block reads pass by the L2
  auto issue = [&](const uint8_t *pool, uint32_t to, const uint32_t (&off)[kHalf]) {
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const i32x4 d = rsrc(pool + from[h], static_cast<int64_t>(live[h]));
      const uint32_t at = to + h * kTile / 2u;
      if (once) {
#pragma unroll
        for (uint32_t j = 0; j < kHalf; ++j) dma16_nt(at + j * 1024u, d, off[j]);
      } else {
#pragma unroll
        for (uint32_t j = 0; j < kHalf; ++j) dma16(at + j * 1024u, d, off[j]);
      }
    }
  };
  auto stage_of = [&](uint32_t tile) { return ((tile - t_lo) & 1u) * kStage; };
  auto ask_k = [&](uint32_t tile) {
    locate(tile);
    issue(k_pool, lds0 + stage_of(tile), k_off);
  };
  auto ask_v = [&](uint32_t tile) { issue(v_pool, lds0 + stage_of(tile) + kTile, v_off); };

#pragma unroll
  for (uint32_t i = 0; i < 2; ++i)
    if (t_lo + i < t_hi) {
      ask_k(t_lo + i);
      ask_v(t_lo + i);
    }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (uint32_t j = 0; j < D / 64; ++j)
      *reinterpret_cast<lds_u32x4 *>(qb + r * Rows<DT, D, R>::kQBytes + (wave * (D / 64u) + j) * 1024u + lane * 16u) =
          q_part[r][j];
  __syncthreads();  // the queries are there
  auto reads_done = [] { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };
  auto any_nonfinite = [&](uint32_t vb) {
    bool odd = false;
#pragma unroll
    for (uint32_t j = 0; j < kDma; ++j) {
      const u32x4 w = *reinterpret_cast<const lds_u32x4 *>(vb + j * 1024u + lane * 16u);
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) odd |= (((w[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
    }
    return __builtin_amdgcn_ballot_w64(odd) != 0;
  };

  // K of the tile after the next goes out once the scores have read this one's,
  // V once P V has.
  for (uint32_t tile = t_lo; tile < t_hi; ++tile) {
    const bool next = tile + 1u < t_hi, more = tile + 2u < t_hi;
    const bool edge = (tile + 1u) * kTreeKeys > s.context;  // holds nodes, or ends the sequence
    const uint32_t at = stage_of(tile);
    if (2u * tile - s_from >= 64u) {
      s_from += 64u;
      scales = scales_next;
    }
    uint32_t both[2];
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) both[h] = __builtin_amdgcn_readlane(scales, 2u * tile + h - s_from);
    const float k_scale = __uint_as_float((lane & 16u ? both[1] : both[0]) << 23);
    const float v_scale[2] = {__uint_as_float(both[0] >> 16 << 23), __uint_as_float(both[1] >> 16 << 23)};
    u32x8 pk[R][1];
    uint32_t seen[R][1] = {};
    if (next) wait_vmcnt<3 * kDma>();
    else wait_vmcnt<kDma>();
    const int32_t base = static_cast<int32_t>(s.context - tile * kTreeKeys);  // node 0 in the tile
#pragma unroll
    for (int r = 0; r < R; ++r) {
      f32x16 sc[1];
      rows.scores8(r, at, qb, k_scale, sc[0]);
      if (r == R - 1 && more) {
        reads_done();
        ask_k(tile + 2u);
      }
      if (edge) {
        if (!a.visible) seen[r][0] = mask_to(base + static_cast<int32_t>(node[r]));
        else if (base >= 0) seen[r][0] = static_cast<uint32_t>(sees[r] << base) | ((1u << base) - 1u);
        else seen[r][0] = base > -64 ? static_cast<uint32_t>(sees[r] >> -base) : 0u;
        Rows<DT, D, R>::template mask<1>(sc, seen[r]);
      }
      rows.template softmax<1>(r, sc, a.scale_log2e, pk[r]);
    }
    if (more) wait_vmcnt<3 * kDma>();
    else if (next) wait_vmcnt<2 * kDma>();
    else wait_vmcnt<0>();
    if (edge && __builtin_expect(wide<DT>(both[0] >> 16) || wide<DT>(both[1] >> 16) || any_nonfinite(lds0 + at + kTile), 0)) {
#pragma unroll
      for (int r = 0; r < R; ++r) rows.add_apart8(lds0 + at + kTile, v_scale, r, pk[r][0], seen[r][0]);
      Rows8<DT, D, R>::clear_apart8(lds0 + at + kTile, v_scale);
    }
    rows.values8(at + kTile, v_scale, pk);
    reads_done();
    if (more) ask_v(tile + 2u);
  }

  if (bad && lane == 0 && a.pool.status) *a.pool.status = 1u;
  finish<DT, D, R>(a, rows, place, sees, item, bad, reinterpret_cast<float *>(lds), reinterpret_cast<float *>(shared_q));
}

}  // namespace att
}  // namespace xpu

#define XPU_TREE_ATTENTION8(T, NAME, D, R)                                                                \
  extern "C" __global__ __launch_bounds__(256, 2) void xpu_tree_attention8_##NAME(xpu::TreeArgs a) {      \
    xpu::att::tree_attention8<xpu::T, D, R>(a);                                                           \
  }
XPU_TREE_ATTENTION8(kBf16, bf16_d128_r1, 128, 1)
XPU_TREE_ATTENTION8(kFp16, fp16_d128_r1, 128, 1)
XPU_TREE_ATTENTION8(kBf16, bf16_d64_r1, 64, 1)
XPU_TREE_ATTENTION8(kFp16, fp16_d64_r1, 64, 1)
XPU_TREE_ATTENTION8(kBf16, bf16_d128_r2, 128, 2)
XPU_TREE_ATTENTION8(kFp16, fp16_d128_r2, 128, 2)
XPU_TREE_ATTENTION8(kBf16, bf16_d64_r2, 64, 2)
XPU_TREE_ATTENTION8(kFp16, fp16_d64_r2, 64, 2)
