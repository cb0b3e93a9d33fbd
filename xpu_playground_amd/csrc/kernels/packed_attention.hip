// Causal attention of packed prompts (xpu_prompt_attention): sequence s has
// query rows q_starts[s] .. q_starts[s + 1] - 1 and key rows k_starts[s] ..
// k_starts[s + 1] - 1; query i sees key j when j <= i + (keys - queries).
// Row layout: [row][head][D], rows `stride` elements apart.
//
// Block: 4 wavefronts of 32 queries; P = 1, 2 or 4 query heads of one kv head
// (the group's largest such divisor) x 4 / P sub-tiles of the same sequence,
// so that a sequence is cut into tiles of 128 / P queries: little is lost at
// the ends of short sequences and at the diagonal. Key tiles of 64 are staged
// by LDS-DMA, two stages of K then V, shared by the wavefronts; two blocks to
// a compute unit (220 registers; at D 64 158 and three), so one's start and end
// fall into the other's tiles. Up to 64 sequences are dealt by the place of the
// tile in its queries, the last places first, since a last heavy tile would run
// alone: that is heaviest first where the sequences have equally many keys before
// their queries, and not otherwise (a short part behind many keys comes last).
//
// Measured: 8192 rows, 32 heads on 8, D 128, 468 to 514 us from box to box, 1.07
// to 1.17 PFLOP/s of the causal half, about 90% of what a large matrix product
// reaches here (the shader clock, power-managed, is at 1.8 GHz with the MFMA
// busy in 64% of the cycles). 24 sequences of 17 .. 1500 rows, the same heads, 86
// to 99 us or 0.65 to 0.75 PFLOP/s: a block has 8 tiles on average, and its
// queries' and result's way to memory (14 us of 93 without them) and its last,
// masked tile are not hidden. 128 rows of 16 heads 7.1 us: one launch and a chain
// of loads. The keys are not cut, so few queries behind many keys leave most of
// the chip idle. D 64 has as many powers for half of the MFMAs; not measured.
#include "attention_core.hpp"
#include "cache_types.hpp"

namespace xpu {
namespace att {

struct Work {
  int32_t seq;       // -1: none
  uint32_t first_q;  // of the sequence's queries
  uint32_t q_lo, q_hi, k_lo, k_hi;
};

// Rows of sequence i, both kinds; starts that do not ascend or pass the rows
// make it one without queries, and nothing of it is touched.
XPU_DEVICE void rows_of(const PackedArgs &a, uint32_t i, Work &w) {
  w.q_lo = a.q_starts[i];
  w.q_hi = a.q_starts[i + 1];
  w.k_lo = a.k_starts[i];
  w.k_hi = a.k_starts[i + 1];
  if (w.q_lo > w.q_hi || w.q_hi > a.q_rows || w.k_lo > w.k_hi || w.k_hi > a.k_rows) w.q_hi = w.q_lo;
}

// Work item `rank` of up to 64 sequences, a lane each: the query tiles (1 <<
// shift queries) of all sequences by their place in the sequence, the last
// places first, since a tile's keys are those before it (and those before the
// sequence's queries, which are not counted here). With f(j) tiles at
// place j or behind it, the item's place is the last j with f(j) > rank, and
// its sequence the (rank - f(j + 1))-th that has a tile there.
XPU_DEVICE Work heaviest_first(const PackedArgs &a, uint32_t shift, uint32_t rank) {
  Work w{};
  if (lane_id() < a.n_seqs) rows_of(a, lane_id(), w);
  const uint32_t tiles = (w.q_hi - w.q_lo + (1u << shift) - 1u) >> shift;
  uint32_t place = 0, behind = 0;  // the place found so far; f(place + 1) once it is final
  if (wave_total(tiles) <= rank) return {-1, 0, 0, 0, 0, 0};
  for (uint32_t bit = 1u << (31u - __builtin_clz(a.q_rows >> shift | 1u)); bit; bit >>= 1) {
    const uint32_t next = place + bit;
    if (wave_total(tiles > next ? tiles - next : 0u) > rank) place = next;
  }
  behind = wave_total(tiles > place + 1u ? tiles - place - 1u : 0u);
  const uint64_t have = __builtin_amdgcn_ballot_w64(tiles > place);
  const uint32_t nth = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(have >> 32),
                                                 __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(have), 0u));
  const uint32_t l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(tiles > place && nth == rank - behind));
  auto of = [&](uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(v, l)); };
  return {static_cast<int32_t>(l), place << shift, of(w.q_lo), of(w.q_hi), of(w.k_lo), of(w.k_hi)};
}

// Work item `slot` of any number of sequences, the last first: the tiles are
// numbered sequence by sequence, 64 at a time, the next 64 on their way.
XPU_DEVICE Work by_slot(const PackedArgs &a, uint32_t shift, uint32_t slot) {
  Work w{}, next{};
  rows_of(a, min(lane_id(), a.n_seqs - 1u), w);
  uint32_t before = 0;
  for (uint32_t at = 0;;) {
    rows_of(a, min(at + 64u + lane_id(), a.n_seqs - 1u), next);
    const uint32_t tiles = at + lane_id() < a.n_seqs ? (w.q_hi - w.q_lo + (1u << shift) - 1u) >> shift : 0u;
    const uint32_t upto = sum_upto(tiles), first = before + upto - tiles;
    const uint64_t hit = __builtin_amdgcn_ballot_w64(slot >= first && slot - first < tiles);
    if (hit) {
      const uint32_t l = __builtin_ctzll(hit);
      auto of = [&](uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(v, l)); };
      return {static_cast<int32_t>(at + l), (slot - of(first)) << shift, of(w.q_lo), of(w.q_hi), of(w.k_lo), of(w.k_hi)};
    }
    if ((at += 64u) >= a.n_seqs) return {-1, 0, 0, 0, 0, 0};
    before += static_cast<uint32_t>(__builtin_amdgcn_readlane(upto, 63));
    w = next;
  }
}

template <int DT, int D> XPU_DEVICE void packed_attention(const PackedArgs &a) {
  constexpr uint32_t kKeys = 64, kTile = kKeys * 2u * D, kStage = 2u * kTile;
  constexpr uint32_t kRpi = 512u / D;          // key rows per DMA instruction
  constexpr uint32_t kCpr = D / 8;             // 16-byte chunks per key row
  constexpr uint32_t kDma = kKeys / kRpi / 4;  // DMA instructions per wave, K and V each
  __shared__ __align__(1024) uint8_t lds[2 * kStage];
  __shared__ uint32_t flags[2][4];  // per stage and wave: its V rows hold a non-finite value

  const uint32_t tid = threadIdx.x, lane = tid & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // Blocks are dealt to the 8 XCDs in turn: a kv head stays on one XCD (its K
  // and V in that L2) where the head count allows.
  const uint32_t group = a.heads / a.kv_heads, packs = group >> a.pack_shift;
  uint32_t kvh, rest;
  if (a.kv_heads % 8u == 0) {
    const uint32_t n = blockIdx.x / 8u;
    kvh = blockIdx.x % 8u + 8u * (n / (a.slots * packs));
    rest = n % (a.slots * packs);
  } else {
    kvh = blockIdx.x % a.kv_heads;
    rest = blockIdx.x / a.kv_heads;
  }
  const uint32_t qt_shift = 7u - a.pack_shift, q_tile = 1u << qt_shift;
  const uint32_t head = kvh * group + (rest % packs << a.pack_shift) + (wave & ((1u << a.pack_shift) - 1u));
  const Work work = a.n_seqs <= 64u ? heaviest_first(a, qt_shift, rest / packs)
                                    : by_slot(a, qt_shift, a.slots - 1u - rest / packs);
  if (work.seq < 0) return;
  const uint32_t first_q = work.first_q, q_lo = work.q_lo, k_lo = work.k_lo;
  const uint32_t n_q = work.q_hi - q_lo, n_k = work.k_hi - k_lo;
  const int32_t shift = static_cast<int32_t>(n_k) - static_cast<int32_t>(n_q);
  const uint32_t t0 = first_q + 32u * (wave >> a.pack_shift);  // the wave's first query
  // keys of the block and of the wave: 0 .. seen - 1
  const int32_t block_seen = static_cast<int32_t>(min(first_q + q_tile, n_q)) + shift;
  const uint32_t n_seen = block_seen < 0 ? 0u : static_cast<uint32_t>(block_seen);
  const uint32_t n_tiles = (n_seen + kKeys - 1) / kKeys;
  const int32_t wave_seen = static_cast<int32_t>(min(t0 + 32u, n_q)) + shift;
  const uint32_t wave_tiles = t0 < n_q && wave_seen > 0 ? (wave_seen + kKeys - 1) / kKeys : 0u;

  const uint32_t t = t0 + (lane & 31u);  // the lane's query
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(lds));
  Rows<DT, D, 1> rows;
  rows.init(lds0);
  // The queries come through the second stage, whole rows at a time, laid out
  // as a tile's K rows: 32 rows per wave, rows past the sequence as zeros.
  constexpr uint32_t kQDma = 32u / kRpi;
  if (t0 < n_q) {
    const i32x4 rq = rsrc(a.q + (q_lo + static_cast<uint64_t>(t0)) * a.q_stride + head * D,
                          static_cast<int64_t>((min(n_q - t0, 32u) - 1u) * a.q_stride + D) * 2);
#pragma unroll
    for (uint32_t j = 0; j < kQDma; ++j) {
      const uint32_t row = kRpi * j + lane / kCpr;
      dma16(lds0 + kStage + (wave * kQDma + j) * 1024u, rq,
            row * static_cast<uint32_t>(a.q_stride) * 2u + 16u * ((lane % kCpr) ^ k_swz<D>(row)));
    }
  }

  // DMA of the wave's share of a tile: instruction j fills LDS rows kRpi
  // (kDma wave + j) .., lane -> physical chunk lane % kCpr of row lane / kCpr.
  // The descriptor ends with the block's last key, so rows past it are zeros.
  uint32_t k_off[kDma], v_off[kDma];
#pragma unroll
  for (uint32_t j = 0; j < kDma; ++j) {
    const uint32_t row = kRpi * (kDma * wave + j) + lane / kCpr;
    k_off[j] = row * static_cast<uint32_t>(a.k_stride) * 2u + 16u * ((lane % kCpr) ^ k_swz<D>(row));
    v_off[j] = row * static_cast<uint32_t>(a.v_stride) * 2u + 16u * ((lane % kCpr) ^ v_swz<D>(row));
  }
  const uint16_t *k_head = a.k + static_cast<uint64_t>(k_lo) * a.k_stride + kvh * D;
  const uint16_t *v_head = a.v + static_cast<uint64_t>(k_lo) * a.v_stride + kvh * D;
  auto issue = [&](uint32_t tile, bool k, bool v) {
    if (tile >= n_tiles) return;
    const uint64_t first = static_cast<uint64_t>(tile) * kKeys;
    const uint32_t live = min(n_seen - tile * kKeys, kKeys);
    const uint32_t at = lds0 + (tile & 1u) * kStage + wave * kDma * 1024u;
    if (k) {
      const i32x4 r = rsrc(k_head + first * a.k_stride, static_cast<int64_t>((live - 1u) * a.k_stride + D) * 2);
#pragma unroll
      for (uint32_t j = 0; j < kDma; ++j) dma16(at + j * 1024u, r, k_off[j]);
    }
    if (v) {
      const i32x4 r = rsrc(v_head + first * a.v_stride, static_cast<int64_t>((live - 1u) * a.v_stride + D) * 2);
#pragma unroll
      for (uint32_t j = 0; j < kDma; ++j) dma16(at + kTile + j * 1024u, r, v_off[j]);
    }
  };

  // Tiles that every query of the block sees in whole: the scores of a tile are
  // formed during the softmax of the one before (scores_powers), so K runs one
  // tile ahead of V. One barrier a tile, which publishes K of the next and V of
  // this one and says that their predecessors' stages are read. The stage is
  // a constant of the two alternating halves of the loop, so the LDS reads'
  // addresses are registers and constant offsets.
  const int32_t all = static_cast<int32_t>(first_q) + shift + 1;  // keys that every query sees
  const uint32_t whole = min(all < 0 ? 0u : static_cast<uint32_t>(all) / kKeys, n_tiles);
  uint32_t tile = 0;
  issue(0, true, true);
  if (n_tiles) wait_vmcnt<2 * kDma>();
  else wait_vmcnt<0>();
  rows.read_q(kStage + wave * kQDma * 1024u);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // before the barrier that frees the stage
  if (whole) {
    wait_vmcnt<kDma>();
    __syncthreads();  // the queries are read, K of the first tile is there
    if (whole > 1) issue(1, true, false);
    f32x16 s0[2], s1[2];
    rows.template scores<2, false>(0, 0, 0, s0);
    float top = Rows<DT, D, 1>::template largest<2>(s0);
    u32x8 pk[1][2];
    auto turn = [&](auto stage_of, f32x16 (&s)[2], f32x16 (&next)[2]) {
      constexpr uint32_t kb = (stage_of ^ 1u) * kStage, vb = stage_of * kStage + kTile;
      wait_vmcnt<0>();
      __syncthreads();
      issue(tile + stage_of + 1, false, true);
      issue(tile + stage_of + 2, true, false);
      rows.template settle<2>(0, s, top, a.scale_log2e);
      rows.scores_powers(kb, next, s, a.scale_log2e, pk[0]);
      top = rows.values_largest(vb, pk[0], next);
    };
    for (; tile + 2 < whole; tile += 2) {
      turn(std::integral_constant<uint32_t, 0>{}, s0, s1);
      turn(std::integral_constant<uint32_t, 1>{}, s1, s0);
    }
    // the scores of `tile` are there, and K of the next was asked for (but not behind a single one)
    wait_vmcnt<0>();
    __syncthreads();
    issue(tile + 1, whole == 1, true);
    rows.template settle<2>(0, s0, top, a.scale_log2e);
    rows.template powers<2>(0, s0, a.scale_log2e, pk[0]);
    rows.template values<2>(kTile, pk);
    ++tile;
  }

  // The last tiles, among them those that some query does not see in whole.
  for (; tile < n_tiles; ++tile) {
    const uint32_t kb = (tile & 1u) * kStage, vb = kb + kTile;
    wait_vmcnt<0>();
    bool bad = false;  // the V rows that this wave staged, before the barrier that publishes them
#pragma unroll
    for (uint32_t j = 0; j < kDma; ++j) {
      const u32x4 w = *reinterpret_cast<const lds_u32x4 *>(lds0 + vb + (wave * kDma + j) * 1024u + lane * 16u);
      bad |= nonfinite<DT>(w.x) || nonfinite<DT>(w.y) || nonfinite<DT>(w.z) || nonfinite<DT>(w.w);
    }
    const bool any = __builtin_amdgcn_ballot_w64(bad) != 0;
    if (lane == 0) flags[tile & 1u][wave] = any;
    __syncthreads();
    issue(tile + 1, true, true);
    // a wave whose queries see the first half only forms no scores of the other
    // (32 sequences of 17 .. 200 rows, 32 heads: 16.9 us without this, 15.8)
    const bool mine = tile < wave_tiles, half = wave_seen <= static_cast<int32_t>(tile * kKeys) + 32;
    const int32_t last = static_cast<int32_t>(t) + shift - static_cast<int32_t>(tile * kKeys);
    u32x8 pk[1][2], pk_half[1][1];
    auto scored = [&](auto parts, auto &to) {
      f32x16 s[parts];
      uint32_t seen[parts];
#pragma unroll
      for (int32_t i = 0; i < parts; ++i) seen[i] = mask_to(last - 32 * i);
      rows.template scores<parts, false>(0, kb, 0, s);
      Rows<DT, D, 1>::template mask<parts>(s, seen);
      rows.template softmax<parts>(0, s, a.scale_log2e, to[0]);
    };
    if (mine && half) scored(std::integral_constant<int32_t, 1>{}, pk_half);
    if (mine && !half) scored(std::integral_constant<int32_t, 2>{}, pk);
    const uint32_t *f = flags[tile & 1u];
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(f[0] | f[1] | f[2] | f[3]), 0)) {
      // the same in every wavefront: all read the rows before any clears its own
      if (mine) {
        rows.add_apart(lds0 + vb, 0, half ? pk_half[0][0] : pk[0][0], mask_to(last));
        if (!half) rows.add_apart(lds0 + vb + kTile / 2u, 0, pk[0][1], mask_to(last - 32));
      }
      __syncthreads();
      Rows<DT, D, 1>::clear_apart(lds0 + vb + wave * kTile / 4u, kKeys / 4u);
      __syncthreads();
    }
    if (mine && half) rows.template values<1>(vb, pk_half);
    if (mine && !half) rows.template values<2>(vb, pk);
  }
  // the stage that the last tile is not in: no wavefront reads it any more
  if (t0 >= n_q) return;
  const float total = rows.total(0);
  rows.store(lds0 + (n_tiles & 1u) * kStage + wave * 32u * 2u * D,
             static_cast<int32_t>(t) + shift < 0 ? 0.0f : 1.0f / total,  // a query that sees no key: 0
             a.out + (q_lo + static_cast<uint64_t>(t0)) * a.out_stride + head * D, a.out_stride, min(n_q - t0, 32u));
}

}  // namespace att
}  // namespace xpu

#define XPU_PACKED_ATTENTION(T, NAME, D)                                                                  \
  extern "C" __global__ __launch_bounds__(256, 2) void xpu_packed_attention_##NAME(xpu::PackedArgs a) {   \
    xpu::att::packed_attention<xpu::T, D>(a);                                                             \
  }
XPU_PACKED_ATTENTION(kBf16, bf16_d128, 128)
XPU_PACKED_ATTENTION(kFp16, fp16_d128, 128)
XPU_PACKED_ATTENTION(kBf16, bf16_d64, 64)
XPU_PACKED_ATTENTION(kFp16, fp16_d64, 64)
