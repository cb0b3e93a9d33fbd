// Accepted drafts to the front of their draft in 8-bit pages (xpu_cache8_keep).
// A wavefront has one (sequence, layer, kv head, K or V): all its kept rows, up
// to 64 of D bytes, are in registers before the first is stored, so they may
// move in any order. They reach at most 5 blocks of 16 positions. A block's
// scale becomes the largest of its own and of the scales that rows bring, so
// codes are only ever scaled down, by powers of two; the rows before the draft
// in its first block are rescaled with it.
#include "cache_types.hpp"
#include "device_common.hpp"

namespace xpu {
namespace cache {

template <int D> XPU_DEVICE void keep8(const KeepArgs &a) {
  constexpr uint32_t kCpr = D / 16, kRpi = 64 / kCpr, kLoads = 64 / kRpi, kHeld = (kBlock + kRpi - 1) / kRpi;
  const uint32_t lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t parts = a.pool.layers * a.pool.kv_heads * 2u, groups = (parts + 3u) / 4u;
  const uint32_t seq = blockIdx.x / groups, group = blockIdx.x % groups, part = group * 4u + wave;
  const uint32_t lo = __builtin_amdgcn_readfirstlane(a.batch.starts[seq]);
  const uint32_t hi = __builtin_amdgcn_readfirstlane(a.batch.starts[seq + 1]);
  const uint32_t context = __builtin_amdgcn_readfirstlane(a.batch.context[seq]);
  const uint32_t count = __builtin_amdgcn_readfirstlane(a.counts[seq]);
  if (count > (lo <= hi && hi <= a.batch.rows ? min(hi - lo, 64u) : 0u)) {
    report(a.pool);
    return;
  }
  if (group == 0 && threadIdx.x == 0 && a.new_context) a.new_context[seq] = context + count;
  if (count == 0 || part >= parts) return;
  const uint32_t in = context & (kBlock - 1u);                    // earlier rows of the first block
  const uint32_t first_page = context >> a.pool.page_shift;
  const uint32_t within = (context & (a.pool.page_size - 1u)) - in;  // the first block in its page
  const uint64_t page = static_cast<uint64_t>(first_page) + lane;
  const uint32_t entry = a.batch.tables[static_cast<uint64_t>(seq) * a.batch.table_pitch +
                                        (page < a.batch.table_pitch ? page : a.batch.table_pitch - 1u)];
  const uint32_t id = page < a.batch.table_pitch ? entry : ~0u;  // of up to 5 pages, lanes 0 .. 4
  const uint32_t head = part / 2u % a.pool.kv_heads, layer = part / 2u / a.pool.kv_heads;
  uint8_t *pool = reinterpret_cast<uint8_t *>(part % 2u ? a.pool.v : a.pool.k) + layer * a.pool.layer_stride;
  // place `at` counts from the first block's first position
  auto page_of = [&](uint32_t at) {
    const uint32_t p = __shfl(id, static_cast<int>((within + at) >> a.pool.page_shift));
    return p < a.pool.n_pages ? p * a.pool.page_stride : kNowhere;
  };
  auto slot_of = [&](uint32_t at) { return (within + at) & (a.pool.page_size - 1u); };
  const uint64_t head_at = static_cast<uint64_t>(head) * a.pool.page_size * D;
  const uint64_t scales_at = static_cast<uint64_t>(a.pool.kv_heads) * a.pool.page_size * D +
                             head * (a.pool.page_size / kBlock);

  // the blocks' scales, lanes 0 .. 4
  const uint32_t reach = in + (hi - lo < 64u ? hi - lo : 64u);  // places with nodes
  const uint64_t block_page = page_of(min(lane, 4u) * kBlock);
  const bool has_block = lane * kBlock < reach && block_page != kNowhere;
  uint8_t *scale_at = pool + (has_block ? block_page + scales_at + slot_of(lane * kBlock) / kBlock : 0u);
  const uint32_t old = has_block ? *scale_at : 0u;

  // where each node goes: lane j is kept node j
  const uint32_t node = a.kept[lo + (lane < count ? lane : 0u)];
  const bool exists = node < hi - lo && node < 64u;
  const uint64_t from_page = page_of(in + (exists ? node : 0u)), to_page = page_of(in + lane);
  const bool real = lane < count, fine = real && exists && from_page != kNowhere && to_page != kNowhere;
  const uint32_t from_block = (in + (exists ? node : 0u)) / kBlock, to_block = (in + lane) / kBlock;
  const uint32_t brings = __shfl(old, static_cast<int>(from_block));
  uint32_t now = old;
#pragma unroll
  for (uint32_t b = 0; b < 5; ++b) {
    float s = fine && to_block == b ? static_cast<float>(brings) : 0.0f;
    s = wave_reduce(s, [](float p, float q) { return fmaxf(p, q); });
    if (lane == b) now = max(now, static_cast<uint32_t>(s));
  }
  const uint32_t gets = __shfl(now, static_cast<int>(min(to_block, 4u)));
  if (__builtin_amdgcn_ballot_w64(real && !fine)) report(a.pool);
  const bool stores = fine && (node != lane || gets != brings);

  // the rows, kRpi at a time: kCpr lanes of 16 bytes each
  const uint64_t from = from_page + head_at + static_cast<uint64_t>(slot_of(in + (exists ? node : 0u))) * D;
  const uint64_t to = to_page + head_at + static_cast<uint64_t>(slot_of(in + lane)) * D;
  u32x4 held[kLoads];
  uint64_t dst[kLoads];
  uint32_t was[kLoads], will[kLoads];
#pragma unroll
  for (uint32_t i = 0; i < kLoads; ++i) {
    const int j = static_cast<int>(i * kRpi + lane / kCpr);
    const bool goes = __shfl(stores ? 1 : 0, j);
    const uint64_t f = __shfl(from, j), t = __shfl(to, j);
    was[i] = __shfl(brings, j);
    will[i] = __shfl(gets, j);
    dst[i] = goes ? t : kNowhere;
    if (i * kRpi < count) held[i] = *reinterpret_cast<const u32x4 *>(pool + (goes ? f : 0u) + lane % kCpr * 16u);
  }
  // the rows before the draft, where their block's scale grows
  const uint32_t old0 = __builtin_amdgcn_readfirstlane(old), now0 = __builtin_amdgcn_readfirstlane(now);
  const uint64_t page0 = page_of(0);
  u32x4 before[kHeld];
  const bool grows = in && now0 > old0;  // (then page 0 is there)
  if (grows) {
#pragma unroll
    for (uint32_t i = 0; i < kHeld; ++i) {
      const uint32_t j = min(i * kRpi + lane / kCpr, in - 1u);
      before[i] = *reinterpret_cast<const u32x4 *>(pool + page0 + head_at + static_cast<uint64_t>(slot_of(j)) * D +
                                                   lane % kCpr * 16u);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  auto scaled = [](const u32x4 &c, uint32_t f, uint32_t t) {
    const u32x2 x = rescaled(u32x2{c.x, c.y}, f, t), y = rescaled(u32x2{c.z, c.w}, f, t);
    return u32x4{x.x, x.y, y.x, y.y};
  };
  if (grows) {
#pragma unroll
    for (uint32_t i = 0; i < kHeld; ++i) {
      const uint32_t j = i * kRpi + lane / kCpr;
      if (j < in)
        *reinterpret_cast<u32x4 *>(pool + page0 + head_at + static_cast<uint64_t>(slot_of(j)) * D + lane % kCpr * 16u) =
            scaled(before[i], old0, now0);
    }
  }
#pragma unroll
  for (uint32_t i = 0; i < kLoads; ++i)
    if (i * kRpi < count && dst[i] != kNowhere)
      *reinterpret_cast<u32x4 *>(pool + dst[i] + lane % kCpr * 16u) = scaled(held[i], was[i], will[i]);
  if (has_block && now != old) *scale_at = static_cast<uint8_t>(now);
}

}  // namespace cache
}  // namespace xpu

extern "C" __global__ __launch_bounds__(256) void xpu_cache8_keep_d128(xpu::KeepArgs a) { xpu::cache::keep8<128>(a); }
extern "C" __global__ __launch_bounds__(256) void xpu_cache8_keep_d64(xpu::KeepArgs a) { xpu::cache::keep8<64>(a); }
