// Causal attention of packed prompts (xpu_prompt_attention): sequence s has
// query rows q_starts[s] .. q_starts[s + 1] - 1 and key rows k_starts[s] ..
// k_starts[s + 1] - 1; query i sees key j when j <= i + (keys - queries).
// Row layout: [row][head][D], rows `stride` elements apart.
//
// Block: 4 wavefronts of 32 queries; P = 1, 2 or 4 query heads of one kv head
// (the group's largest such divisor) x 4 / P sub-tiles of the same sequence,
// so that a sequence is cut into tiles of 128 / P queries: little is lost at
// the ends of short sequences and at the diagonal. Key tiles of 64 are staged
// by LDS-DMA, two stages of K then V, shared by the wavefronts.
#include "attention_core.hpp"
#include "cache_types.hpp"

#include <type_traits>

namespace xpu {
namespace att {

// The sequence that owns slot `slot` of the work list, where sequence s has
// the slots from starts[s] / tile + s on (tile = 1 << shift queries): at least
// as many as it has tiles, and known without a sum over the sequences. -1: none.
XPU_DEVICE int32_t sequence_of_slot(const uint32_t *starts, uint32_t n_seqs, uint32_t shift, uint32_t slot) {
  int32_t s = -1;
  for (uint32_t at = 0; at < n_seqs; at += 64) {
    const uint32_t i = at + lane_id();
    const bool before = i < n_seqs && (starts[i] >> shift) + i <= slot;
    s += __builtin_popcountll(__builtin_amdgcn_ballot_w64(before));
  }
  return __builtin_amdgcn_readfirstlane(s);
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
  // and V in that L2) where the head count allows; within it the last slots,
  // the heaviest tiles of a sequence, come first.
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
  const uint32_t slot = a.slots - 1u - rest / packs, qt_shift = 7u - a.pack_shift, q_tile = 1u << qt_shift;
  const uint32_t head = kvh * group + (rest % packs << a.pack_shift) + (wave & (1u << a.pack_shift) - 1u);

  const int32_t seq = sequence_of_slot(a.q_starts, a.n_seqs, qt_shift, slot);
  if (seq < 0) return;
  const uint32_t q_lo = __builtin_amdgcn_readfirstlane(a.q_starts[seq]);
  const uint32_t q_hi = __builtin_amdgcn_readfirstlane(a.q_starts[seq + 1]);
  const uint32_t k_lo = __builtin_amdgcn_readfirstlane(a.k_starts[seq]);
  const uint32_t k_hi = __builtin_amdgcn_readfirstlane(a.k_starts[seq + 1]);
  // starts that do not ascend or pass the rows: nothing of the sequence is touched
  if (q_lo > q_hi || q_hi > a.q_rows || k_lo > k_hi || k_hi > a.k_rows || (q_lo >> qt_shift) + seq > slot) return;
  const uint32_t first_q = (slot - ((q_lo >> qt_shift) + seq)) << qt_shift, n_q = q_hi - q_lo, n_k = k_hi - k_lo;
  if (first_q >= n_q) return;
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
  rows.load_q(0, a.q + (q_lo + min(t, n_q - 1u)) * a.q_stride + head * D);

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
  auto issue = [&](uint32_t tile, uint32_t stage) {
    const uint64_t first = static_cast<uint64_t>(tile) * kKeys;
    const uint32_t live = min(n_seen - tile * kKeys, kKeys);
    const i32x4 rk = rsrc(k_head + first * a.k_stride, static_cast<int64_t>((live - 1u) * a.k_stride + D) * 2);
    const i32x4 rv = rsrc(v_head + first * a.v_stride, static_cast<int64_t>((live - 1u) * a.v_stride + D) * 2);
    const uint32_t at = lds0 + stage * kStage + wave * kDma * 1024u;
#pragma unroll
    for (uint32_t j = 0; j < kDma; ++j) dma16(at + j * 1024u, rk, k_off[j]);
#pragma unroll
    for (uint32_t j = 0; j < kDma; ++j) dma16(at + kTile + j * 1024u, rv, v_off[j]);
  };

  // one tile of keys; the stage is a constant, so the LDS reads' addresses are
  // registers and constant offsets
  auto step = [&](uint32_t tile, auto stage_of) {
    constexpr uint32_t stage = stage_of, kb = stage * kStage, vb = kb + kTile;
    // whether some query of the block does not see some key of the tile
    const bool edge = static_cast<int32_t>(tile * kKeys + kKeys - 1u) > static_cast<int32_t>(first_q) + shift;
    wait_vmcnt<0>();
    if (edge) {  // the V rows that this wave staged, before the barrier that publishes them
      bool bad = false;
#pragma unroll
      for (uint32_t j = 0; j < kDma; ++j) {
        const u32x4 w = *reinterpret_cast<const lds_u32x4 *>(lds0 + vb + (wave * kDma + j) * 1024u + lane * 16u);
        bad |= nonfinite<DT>(w.x) || nonfinite<DT>(w.y) || nonfinite<DT>(w.z) || nonfinite<DT>(w.w);
      }
      const bool any = __builtin_amdgcn_ballot_w64(bad) != 0;
      if (lane == 0) flags[stage][wave] = any;
    }
    __syncthreads();
    if (tile + 1 < n_tiles) issue(tile + 1, stage ^ 1u);
    const bool mine = tile < wave_tiles;
    u32x8 pk[1][2];
    uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
    if (mine) {
      f32x16 s[2];
      rows.template scores<2, false>(0, kb, 0, s);
      if (static_cast<int32_t>(tile * kKeys + kKeys - 1u) > static_cast<int32_t>(t0) + shift) {  // wave-uniform
        const int32_t last = static_cast<int32_t>(t) + shift - static_cast<int32_t>(tile * kKeys);
        seen[0] = mask_to(last);
        seen[1] = mask_to(last - 32);
        Rows<DT, D, 1>::template mask<2>(s, seen);
      }
      rows.template softmax<2>(0, s, a.scale_log2e, pk[0]);
    }
    if (edge && __builtin_expect(flags[stage][0] | flags[stage][1] | flags[stage][2] | flags[stage][3], 0)) {
      // the same in every wavefront: all read the rows before any clears its own
      if (mine) {
        rows.add_apart(lds0 + vb, 0, pk[0][0], seen[0]);
        rows.add_apart(lds0 + vb + kTile / 2u, 0, pk[0][1], seen[1]);
      }
      __syncthreads();
      Rows<DT, D, 1>::clear_apart(lds0 + vb + wave * kTile / 4u, kKeys / 4u);
      __syncthreads();
    }
    if (mine) rows.template values<2>(vb, pk);
  };
  if (n_tiles) issue(0, 0);
  for (uint32_t tile = 0; tile < n_tiles; tile += 2) {
    step(tile, std::integral_constant<uint32_t, 0>{});
    if (tile + 1 < n_tiles) step(tile + 1, std::integral_constant<uint32_t, 1>{});
  }
  const float total = rows.total(0);
  if (t < n_q)  // a query that sees no key: 0
    rows.store(0, a.out + (q_lo + t) * a.out_stride + head * D, static_cast<int32_t>(t) + shift < 0 ? 0.0f : 1.0f / total);
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
