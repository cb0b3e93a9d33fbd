// Accepted drafts to the front of their draft in 8-bit pages (xpu_cache8_keep).
// Its parts are (layer, kv head, K or V). All kept rows of a part are loaded
// before the first is stored, so they may move in any order. A wavefront has
// room for 16 rows, and a block takes one part, a wavefront 16 of its rows, or,
// where that is more blocks than the chip holds, as many parts as let it hold
// all: up to 16 rows each wavefront parts of its own, more rows one part after the
// other (one sequence of 28 layers, 8 kv heads: 4.8 us the first way, 7.3 with
// four parts a block; 48 of them 20.8 with a wavefront for up to 64 rows, which is
// twice the registers, 13.7 with four parts a block, 11.2 so). What is left is the
// chain of loads: lengths, table, scale and rows. The rows reach at most 5 blocks of 16
// positions. A block's scale becomes the largest of its own and of the scales
// that rows bring, so codes are only ever scaled down, by powers of two; the
// rows before the draft in its first block are rescaled with it.
#include "cache_types.hpp"
#include "device_common.hpp"

namespace xpu {
namespace cache {

template <int D> XPU_DEVICE void keep8(const KeepArgs &a, uint32_t per_block) {
  constexpr uint32_t kCpr = D / 16, kRpi = 64 / kCpr, kLoads = 16 / kRpi;
  const uint32_t lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t parts = a.pool.layers * a.pool.kv_heads * 2u, groups = (parts + per_block - 1u) / per_block;
  const uint32_t seq = blockIdx.x / groups, group = blockIdx.x % groups;
  const uint32_t lo = __builtin_amdgcn_readfirstlane(a.batch.starts[seq]);
  const uint32_t hi = __builtin_amdgcn_readfirstlane(a.batch.starts[seq + 1]);
  const uint32_t context = __builtin_amdgcn_readfirstlane(a.batch.context[seq]);
  const uint32_t count = __builtin_amdgcn_readfirstlane(a.counts[seq]);
  if (count > (lo <= hi && hi <= a.batch.rows ? min(hi - lo, 64u) : 0u)) {
    report(a.pool);
    return;
  }
  if (group == 0 && threadIdx.x == 0 && a.new_context) a.new_context[seq] = context + count;
  if (count == 0) return;
  const uint32_t in = context & (kBlock - 1u);                    // earlier rows of the first block
  const uint32_t first_page = context >> a.pool.page_shift;
  const uint32_t within = (context & (a.pool.page_size - 1u)) - in;  // the first block in its page
  const uint64_t page = static_cast<uint64_t>(first_page) + lane;
  const uint32_t entry = a.batch.tables[static_cast<uint64_t>(seq) * a.batch.table_pitch +
                                        (page < a.batch.table_pitch ? page : a.batch.table_pitch - 1u)];
  const uint32_t id = page < a.batch.table_pitch ? entry : ~0u;  // of up to 5 pages, lanes 0 .. 4
  // place `at` counts from the first block's first position
  auto page_of = [&](uint32_t at) {
    const uint32_t p = __shfl(id, static_cast<int>((within + at) >> a.pool.page_shift));
    return p < a.pool.n_pages ? p * a.pool.page_stride : kNowhere;
  };
  auto slot_of = [&](uint32_t at) { return (within + at) & (a.pool.page_size - 1u); };

  // where each node goes: lane j is kept node j. A place whose node does not exist
  // holds what it held: its own node, which is rescaled with its block.
  const uint32_t asked = a.kept[lo + (lane < count ? lane : 0u)];
  const bool exists = asked < hi - lo && asked < 64u;
  const uint64_t asked_page = page_of(in + (exists ? asked : 0u)), to_page = page_of(in + lane);
  const bool known = exists && asked_page != kNowhere;
  const uint32_t node = known ? asked : lane;
  const uint64_t from_page = known ? asked_page : to_page;
  const bool real = lane < count, fine = real && to_page != kNowhere;
  const uint32_t from_block = (in + node) / kBlock, to_block = (in + lane) / kBlock;
  const uint64_t from = from_page + static_cast<uint64_t>(slot_of(in + node)) * D;
  const uint64_t to = to_page + static_cast<uint64_t>(slot_of(in + lane)) * D;
  if (__builtin_amdgcn_ballot_w64(real && !(known && fine))) report(a.pool);
  // the blocks, lanes 0 .. 4
  const uint32_t reach = in + (hi - lo < 64u ? hi - lo : 64u);  // places with nodes
  const uint64_t block_page = page_of(min(lane, 4u) * kBlock), page0 = page_of(0);
  const bool has_block = lane * kBlock < reach && block_page != kNowhere;
  const uint32_t in_page = slot_of(lane * kBlock) / kBlock;

  const bool apart = per_block != 1u && count <= 16u;  // the wavefronts work on parts of their own
  for (uint32_t step = apart ? wave : 0u; step < per_block; step += apart ? 4u : 1u) {
    const uint32_t part = group * per_block + step, row = apart ? 0u : wave * 16u;
    if (part >= parts) break;
    const bool lead = apart || wave == 0;  // has the part's scales and earlier rows
    const uint32_t head = part / 2u % a.pool.kv_heads, layer = part / 2u / a.pool.kv_heads;
    uint8_t *pool = reinterpret_cast<uint8_t *>(part % 2u ? a.pool.v : a.pool.k) + layer * a.pool.layer_stride;
    uint8_t *codes = pool + static_cast<uint64_t>(head) * a.pool.page_size * D + lane % kCpr * 16u;
    uint8_t *scale_at = pool + (has_block ? block_page + static_cast<uint64_t>(a.pool.kv_heads) * a.pool.page_size * D +
                                                head * (a.pool.page_size / kBlock) + in_page
                                          : 0u);
    const uint32_t old = has_block ? *scale_at : 0u;
    // the rows, kRpi at a time: kCpr lanes of 16 bytes each (those of no page: any)
    u32x4 held[kLoads];
    uint64_t dst[kLoads];
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) {
      const int j = static_cast<int>(row + i * kRpi + lane / kCpr);
      const bool goes = __shfl(fine ? 1 : 0, j);
      const uint64_t f = __shfl(from, j), t = __shfl(to, j);
      dst[i] = goes ? t : kNowhere;
      held[i] = *reinterpret_cast<const u32x4 *>(codes + (goes ? f : 0u));
    }
    const uint32_t brings = __shfl(old, static_cast<int>(from_block));
    uint32_t now = old;
#pragma unroll
    for (uint32_t b = 0; b < 5; ++b) {
      if (b && b * kBlock >= in + count) break;  // no kept row gets there
      float s = fine && to_block == b ? static_cast<float>(brings) : 0.0f;
      s = wave_reduce(s, [](float p, float q) { return fmaxf(p, q); });
      if (lane == b) now = max(now, static_cast<uint32_t>(s));
    }
    const uint32_t gets = __shfl(now, static_cast<int>(min(to_block, 4u)));
    // the rows before the draft, where their block's scale grows (its page is there then)
    const uint32_t old0 = __builtin_amdgcn_readfirstlane(old), now0 = __builtin_amdgcn_readfirstlane(now);
    const bool grows = lead && in && now0 > old0;
    u32x4 before[kLoads];
    uint8_t *first = codes + page0 + static_cast<uint64_t>(slot_of(0)) * D;
    if (grows) {
#pragma unroll
      for (uint32_t i = 0; i < kLoads; ++i)
        before[i] = *reinterpret_cast<const u32x4 *>(first + min(i * kRpi + lane / kCpr, in - 1u) * D);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (!apart) __syncthreads();
    auto scaled = [](const u32x4 &c, uint32_t f, uint32_t t) {
      if (__builtin_amdgcn_ballot_w64(f != t) == 0) return c;
      const u32x2 x = rescaled(u32x2{c.x, c.y}, f, t), y = rescaled(u32x2{c.z, c.w}, f, t);
      return u32x4{x.x, x.y, y.x, y.y};
    };
    if (grows) {
#pragma unroll
      for (uint32_t i = 0; i < kLoads; ++i) {
        const uint32_t j = i * kRpi + lane / kCpr;
        const u32x4 c = scaled(before[i], old0, now0);
        if (j < in) *reinterpret_cast<u32x4 *>(first + j * D) = c;
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) {
      const int j = static_cast<int>(row + i * kRpi + lane / kCpr);
      const uint32_t was = __shfl(brings, j), will = __shfl(gets, j);
      const bool moves = __shfl(node, j) != static_cast<uint32_t>(j) || was != will;
      const u32x4 c = scaled(held[i], was, dst[i] != kNowhere ? will : was);
      if (dst[i] != kNowhere && moves) *reinterpret_cast<u32x4 *>(codes + dst[i]) = c;
    }
    if (lead && has_block && now != old) *scale_at = static_cast<uint8_t>(now);
  }
}

}  // namespace cache
}  // namespace xpu

extern "C" __global__ __launch_bounds__(256) void xpu_cache8_keep_d128(xpu::Keep8Args a) {
  xpu::cache::keep8<128>(a.keep, a.per_block);
}
extern "C" __global__ __launch_bounds__(256) void xpu_cache8_keep_d64(xpu::Keep8Args a) {
  xpu::cache::keep8<64>(a.keep, a.per_block);
}
