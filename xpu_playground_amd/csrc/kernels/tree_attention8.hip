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
// A tile of 32 keys has half the bytes of a 16-bit one. A wavefront takes 32 rows
// and has two stages of K, one of V (its V goes out once P V has read the last),
// so three blocks share a CU where blocks of 64 rows with two stages of both
// leave room for two (this kernel alone, without the join): four drafts behind
// 90000 to 131000 positions 297 us and 313, 48 drafts of 1 .. 26 nodes behind 60 to
// 8000 46.5 and 64, 48 single tokens 39.5 and 63, and even 64 drafts of 30 .. 64
// nodes 186 and 205. What is left there: without its
// arithmetic the four drafts' kernel takes 223 us, without its loads 216, so
// neither alone bounds it; the copy's rate would be 155.
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

template <int DT, int D> struct Rows8 : Rows<DT, D, 1> {
  using Base = Rows<DT, D, 1>;
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

  // S^T of 32 keys at LDS offset kb, of `scale` for the lane's key.
  XPU_DEVICE void scores8(uint32_t kb, float scale, f32x16 &s) const {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.0f;
    u32x4 kf[2];
    auto read = [&](int j) { kf[j & 1] = *reinterpret_cast<const lds_u32x4 *>(kb + ka8[j]); };
    read(0);
#pragma unroll
    for (int j = 0; j < kKs / 2; ++j) {
      if (j + 1 < kKs / 2) read(j + 1);
      const u32x4 &k = kf[j & 1];
      s = dma::mfma<DT>(widen8<DT>(k.x, k.y, scale), this->q[0][2 * j], s);
      s = dma::mfma<DT>(widen8<DT>(k.z, k.w, scale), this->q[0][2 * j + 1], s);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // O^T += V^T P^T of the tile at LDS offset vb, of scale[ks] for keys 16 ks ...
  XPU_DEVICE void values8(uint32_t vb, const float (&scale)[2], const u32x8 &p) {
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
        const uint32_t b = 4u * ks;
        this->o[0][dt] = dma::mfma<DT>(v, u32x4{p[b], p[b + 1], p[b + 2], p[b + 3]}, this->o[0][dt]);
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
  XPU_DEVICE void add_apart8(uint32_t vb, const float (&scale)[2], u32x8 pk, uint32_t seen) {
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
          f32x16 &o = this->o[0][dt];
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

template <int DT, int D> XPU_DEVICE void tree_attention8(const TreeArgs &a) {
  constexpr uint32_t kRow = D, kTile = kTreeKeys * kRow, kHalfTile = kTile / 2;
  constexpr uint32_t kWave = 3u * kTile;  // K has two stages, V one
  constexpr uint32_t kPasses = 2;         // of the end
  constexpr uint32_t kRpi = 1024u / D, kCpr = D / 16;
  constexpr uint32_t kDma = kTreeKeys / kRpi, kHalf = kDma / 2;  // DMA instructions per tile, K and V each; per half of it
  // per wavefront the stages of its tiles; then the partial results
  __shared__ __align__(1024) uint8_t lds[4u * kWave];
  static_assert(4u * kWave >= 4u * 64u * (D / 2u) * 4u / kPasses, "the partial results fit the tiles' memory");
  __shared__ __align__(16) float meet[4 * 128];  // the (max, sum) pairs that the wavefronts exchange

  const uint32_t tid = threadIdx.x, lane = tid & 63u, hh = lane >> 5;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t kvh = blockIdx.x % a.pool.kv_heads, item = blockIdx.x / a.pool.kv_heads;
  const uint32_t group = a.heads / a.pool.kv_heads;
  const Place place = find<1>(a, group, [&](uint32_t first, uint32_t count, const Sequence &) {
    return item >= first && item - first < count;
  });
  if (place.seq < 0) return;
  const uint32_t seq = static_cast<uint32_t>(place.seq);
  const Sequence &s = place.s;
  const uint32_t row_tile = (item - place.first) % s.row_tiles, chunk = (item - place.first) / s.row_tiles;
  const uint32_t c0 = static_cast<uint32_t>(static_cast<uint64_t>(s.tiles) * chunk / place.chunks);
  const uint32_t c1 = static_cast<uint32_t>(static_cast<uint64_t>(s.tiles) * (chunk + 1u) / place.chunks);
  const uint32_t t_lo = c0 + (c1 - c0) * wave / 4u, t_hi = c0 + (c1 - c0) * (wave + 1u) / 4u;

  // The wave's blocks of 16 keys, 64 at a time, a lane each: the page's id, one
  // window ahead; where the block lies and how many bytes of it are the
  // sequence's (a block of a page past the pool has none); and the scales, once
  // the ids are there, which is two tiles before their use.
  const uint32_t *table = a.batch.tables + static_cast<uint64_t>(seq) * a.batch.table_pitch;
  const uint8_t *k_pool = reinterpret_cast<const uint8_t *>(a.pool.k), *v_pool = reinterpret_cast<const uint8_t *>(a.pool.v);
  const uint32_t blocks = (s.end + kBlock - 1u) / kBlock, per = a.pool.page_size / kBlock;
  const uint64_t head_at = static_cast<uint64_t>(kvh) * a.pool.page_size * D;
  const uint64_t scales_at = static_cast<uint64_t>(a.pool.kv_heads) * a.pool.page_size * D + kvh * per;
  bool bad = s.bad || (a.visible && s.n > 64u);
  struct Window {
    uint32_t lo, hi, live;  // the block's offset in the pools, its bytes
    uint32_t k_scale, v_scale;
  };
  auto ids_of = [&](uint32_t from) {
    const uint32_t at = from + lane;
    return at < blocks ? table[at * kBlock >> a.pool.page_shift] : ~0u;
  };
  auto window_of = [&](uint32_t from, uint32_t id) {
    const uint32_t at = from + lane, in_page = at & (per - 1u);
    const bool there = id < a.pool.n_pages;
    const uint64_t page = there ? static_cast<uint64_t>(id) * a.pool.page_stride : 0u;
    const uint64_t offset = page + (there ? head_at + in_page * kHalfTile : 0u);
    Window w;
    w.k_scale = there ? k_pool[page + scales_at + in_page] : 127u;
    w.v_scale = there ? v_pool[page + scales_at + in_page] : 127u;
    w.lo = static_cast<uint32_t>(offset);
    w.hi = static_cast<uint32_t>(offset >> 32);
    w.live = there && at < blocks ? min(s.end - at * kBlock, kBlock) * kRow : 0u;
    bad |= __builtin_amdgcn_ballot_w64(!there && at < blocks) != 0;
    return w;
  };
  uint32_t w_from = 2u * t_lo, s_from = w_from;
  uint32_t ids = ids_of(w_from), ids_next = ids_of(w_from + 64u);

  Rows8<DT, D> rows;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(lds)) + wave * kWave;
  rows.init8(lds0);
  const uint32_t in_tile = min(32u * row_tile + (lane & 31u), s.n * group - 1u), node = in_tile / group;
  const uint16_t *q_row = a.q + (s.first + node) * a.q_stride + (kvh * group + in_tile % group) * D;
#pragma unroll
  for (uint32_t ks = 0; ks < D / 16; ++ks)
    rows.q[0][ks] = *reinterpret_cast<const u32x4 *>(q_row + 32u * (ks / 2u) + 16u * hh + 8u * (ks % 2u));
  uint64_t sees[1] = {0};  // bit j: node j
  if (a.visible) {
    sees[0] = a.visible[s.first + node];
    if (s.n < 64u) sees[0] &= (1ull << s.n) - 1ull;
  }
  uint32_t k_off[kHalf], v_off[kHalf];
#pragma unroll
  for (uint32_t j = 0; j < kHalf; ++j) {
    const uint32_t row = kRpi * j + lane / kCpr;
    k_off[j] = row * kRow + 16u * ((lane % kCpr) ^ k8_swz<D>(row));
    v_off[j] = row * kRow + 16u * ((lane % kCpr) ^ v8_swz<D>(row));
  }
  Window w = window_of(w_from, ids);
  uint32_t k_scales = w.k_scale, v_scales = w.v_scale;
  // the queries are waited for here: a wait at their use would be one in the
  // loop, where it would be for every tile that is on its way
#pragma unroll
  for (uint32_t ks = 0; ks < D / 16; ++ks) asm volatile("" : "+v"(rows.q[0][ks]));

  // Where the two blocks of a tile lie.
  struct Where {
    uint64_t at[2];
    uint32_t live[2];
  };
  auto locate = [&](uint32_t tile) {
    if (2u * tile - w_from >= 64u) {
      w_from += 64u;
      ids = ids_next;
      ids_next = ids_of(w_from + 64u);
      w = window_of(w_from, ids);
    }
    Where x;
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t l = 2u * tile + h - w_from;
      x.at[h] = static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(w.hi, l))) << 32 |
                static_cast<uint32_t>(__builtin_amdgcn_readlane(w.lo, l));
      x.live[h] = __builtin_amdgcn_readlane(w.live, l);
    }
    return x;
  };
  const bool once = s.row_tiles == 1;  // keys that only this block reads pass by the L2
  auto issue = [&](const uint8_t *pool, const Where &x, uint32_t to, const uint32_t (&off)[kHalf]) {
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const uint64_t at = reinterpret_cast<uint64_t>(pool) + x.at[h];  // (below 2^48: stride 0)
      const i32x4 d{static_cast<int>(at), static_cast<int>(at >> 32), static_cast<int>(x.live[h]), 0x00020000};
#pragma unroll
      for (uint32_t j = 0; j < kHalf; ++j) {
        if (once) dma16_nt(to + h * kHalfTile + j * 1024u, d, off[j]);
        else dma16(to + h * kHalfTile + j * 1024u, d, off[j]);
      }
    }
  };
  Where v_where{};  // of the next tile's V, which goes out after the K of the tile behind it
  if (t_lo < t_hi) {
    const Where x = locate(t_lo);
    issue(k_pool, x, lds0, k_off);
    issue(v_pool, x, lds0 + 2u * kTile, v_off);
  }
  if (t_lo + 1u < t_hi) {
    v_where = locate(t_lo + 1u);
    issue(k_pool, v_where, lds0 + kTile, k_off);
  }
  auto reads_done = [] { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };
  auto any_nonfinite = [&](uint32_t vb) {
    bool odd = false;
#pragma unroll
    for (uint32_t j = 0; j < kDma; ++j) {
      const u32x4 x = *reinterpret_cast<const lds_u32x4 *>(vb + j * 1024u + lane * 16u);
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) odd |= (((x[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
    }
    return __builtin_amdgcn_ballot_w64(odd) != 0;
  };

  // K of the tile after the next goes out once the scores have read this one's, V
  // of the next once P V has.
  uint32_t kb = 0;
  for (uint32_t tile = t_lo; tile < t_hi; ++tile, kb ^= kTile) {
    const bool next = tile + 1u < t_hi, more = tile + 2u < t_hi;
    const bool edge = (tile + 1u) * kTreeKeys > s.context;  // holds nodes, or ends the sequence
    if (2u * tile - s_from >= 64u) {  // (the ids' window is this one by now, for two tiles)
      s_from += 64u;
      k_scales = w.k_scale;
      v_scales = w.v_scale;
    }
    const uint32_t l = 2u * tile - s_from;
    uint32_t ks[2], vs[2];
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      ks[h] = __builtin_amdgcn_readlane(k_scales, l + h);
      vs[h] = __builtin_amdgcn_readlane(v_scales, l + h);
    }
    const float k_scale = __uint_as_float((lane & 16u ? ks[1] : ks[0]) << 23);
    const float v_scale[2] = {__uint_as_float(vs[0] << 23), __uint_as_float(vs[1] << 23)};
    u32x8 pk[1];
    uint32_t seen[1] = {};
    f32x16 sc[1];
    // behind K of this tile: V of it and K of the next
    if (next) wait_vmcnt<2 * kDma>();
    else wait_vmcnt<kDma>();
    rows.scores8(kb, k_scale, sc[0]);
    Where k_where = v_where;
    if (more) {
      k_where = locate(tile + 2u);
      reads_done();
      issue(k_pool, k_where, lds0 + kb, k_off);
    }
    if (edge) {
      const int32_t base = static_cast<int32_t>(s.context - tile * kTreeKeys);  // node 0 in the tile
      if (!a.visible) seen[0] = mask_to(base + static_cast<int32_t>(node));
      else if (base >= 0) seen[0] = static_cast<uint32_t>(sees[0] << base) | ((1u << base) - 1u);
      else seen[0] = base > -64 ? static_cast<uint32_t>(sees[0] >> -base) : 0u;
      Rows8<DT, D>::template mask<1>(sc, seen);
    }
    rows.template softmax<1>(0, sc, a.scale_log2e, pk);
    // behind V of this tile: K of the one after the next alone
    if (more) wait_vmcnt<kDma>();
    else wait_vmcnt<0>();
    constexpr uint32_t vb = 2u * kTile;
    if (edge && __builtin_expect(wide<DT>(vs[0]) || wide<DT>(vs[1]) || any_nonfinite(lds0 + vb), 0)) {
      rows.add_apart8(lds0 + vb, v_scale, pk[0], seen[0]);
      Rows8<DT, D>::clear_apart8(lds0 + vb, v_scale);
    }
    rows.values8(vb, v_scale, pk[0]);
    reads_done();
    if (next) issue(v_pool, v_where, lds0 + vb, v_off);
    v_where = k_where;
  }

  if (bad && lane == 0 && a.pool.status) *a.pool.status = 1u;
  finish<DT, D, 1, kPasses>(a, rows, place, sees, item, bad, reinterpret_cast<float *>(lds), meet);
}

}  // namespace att
}  // namespace xpu

#define XPU_TREE_ATTENTION8(T, NAME, D)                                                                  \
  extern "C" __global__ __launch_bounds__(256, 3) void xpu_tree_attention8_##NAME(xpu::TreeArgs a) {     \
    xpu::att::tree_attention8<xpu::T, D>(a);                                                             \
  }
XPU_TREE_ATTENTION8(kBf16, bf16_d128_r1, 128)
XPU_TREE_ATTENTION8(kFp16, fp16_d128_r1, 128)
XPU_TREE_ATTENTION8(kBf16, bf16_d64_r1, 64)
XPU_TREE_ATTENTION8(kFp16, fp16_d64_r1, 64)
