// The paged cache's row and page operations: new rows into the pages
// (append), accepted drafts to the front of their draft (keep), whole pages
// (copy). All move 16-byte chunks of rows of D 16-bit elements; a lane holds
// one chunk, so the types and head sizes are only sizes here. Bound by memory
// where they are large and by the launch and a chain of dependent loads (the
// batch's numbers, the table, the rows) where they are small. Measured with 8
// kv heads of 128: append of 48 rows 4.1 us, of the 8769 rows of 24 prompts
// 12.6 to 12.9 us or 5.6 TB/s; keep of one draft in 28 layers 6.9 us, of 48 drafts
// 11.2 to 11.4 us or 2.3 TB/s; copy of 4 pages of 16 6.0 us, of 101 pages of 64 in 28
// layers 273 to 293 us or 5.1 to 5.4 TB/s (a large copy reaches 4.8).
#include "cache_types.hpp"
#include "device_common.hpp"

namespace xpu {
namespace cache {

// The sequence that holds row `row` of the batch, and its first row; seq -1
// for a row of none. 64 sequences at a time, a lane each, the next 64 on their
// way; the first that has the row, whatever the starts of the others are.
struct Holder {
  int32_t seq;
  uint32_t first;
};
XPU_DEVICE Holder holder_of(const BatchArgs &b, uint32_t row) {
  uint32_t lo, hi, next_lo, next_hi;
  auto load = [&](uint32_t at, uint32_t &l, uint32_t &h) {  // past the last: it again, behind itself
    const uint32_t i = min(at + lane_id(), b.n_seqs - 1u);
    l = b.starts[i];
    h = b.starts[i + 1u];
  };
  load(0, lo, hi);
  for (uint32_t at = 0;;) {
    load(at + 64u, next_lo, next_hi);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(lo <= row && row < hi && hi <= b.rows);
    if (hit) {
      const uint32_t l = __builtin_ctzll(hit);
      return {static_cast<int32_t>(at + l), static_cast<uint32_t>(__builtin_amdgcn_readlane(lo, l))};
    }
    if ((at += 64u) >= b.n_seqs) return {-1, 0};
    lo = next_lo;
    hi = next_hi;
  }
}

XPU_DEVICE void report(const PoolArgs &p) {
  if (p.status && lane_id() == 0) *p.status = 1u;
}

// One wavefront per row (grid-stride): K and V, all kv heads.
template <int D> XPU_DEVICE void append(const AppendArgs &a) {
  constexpr uint32_t kCpr = D / 8;
  const uint32_t lane = lane_id(), waves = gridDim.x * 4u, chunks = a.pool.kv_heads * kCpr;
  for (uint32_t row = blockIdx.x * 4u + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); row < a.batch.rows;
       row += waves) {
    const Holder holder = holder_of(a.batch, row);
    if (holder.seq < 0) continue;
    const uint32_t seq = static_cast<uint32_t>(holder.seq);
    const uint64_t pos = static_cast<uint64_t>(a.batch.context[seq]) + (row - holder.first);
    const uint64_t at = element_of(a.pool, a.batch.tables + static_cast<uint64_t>(seq) * a.batch.table_pitch, a.batch.table_pitch, pos, D);
    if (at == kNowhere) {
      report(a.pool);
      continue;
    }
    const uint16_t *k = a.k + row * a.k_stride, *v = a.v + row * a.v_stride;
#pragma unroll 2
    for (uint32_t c = lane; c < chunks; c += 64) {
      const u32x4 x = *reinterpret_cast<const u32x4 *>(k + c * 8u), y = *reinterpret_cast<const u32x4 *>(v + c * 8u);
      const uint64_t to = at + static_cast<uint64_t>(c / kCpr) * a.pool.page_size * D + c % kCpr * 8u;
      *reinterpret_cast<u32x4 *>(a.pool.k + to) = x;
      *reinterpret_cast<u32x4 *>(a.pool.v + to) = y;
    }
  }
}

// Four (layer, kv head, K or V) parts of a sequence per block. All kept rows
// of a part are loaded before the first is stored, so they may move in any
// order: up to 16 rows a part is a wavefront's, with more the wavefronts take
// 16 rows each of one part after the other and meet in between. Branch-free up
// to the stores, so that the loads are in flight together: rows that do not
// move read the pool's first element. The pages of the up to 64 nodes lie in
// lanes 0 .. 4.
template <int D> XPU_DEVICE void keep(const KeepArgs &a) {
  constexpr uint32_t kRpi = 512u / D, kCpr = D / 8, kLoads = 16u / kRpi;
  const uint32_t lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t parts = a.pool.layers * a.pool.kv_heads * 2u, groups = (parts + 3u) / 4u;
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
  if (count == 0) return;  // no row to read the first entry of
  const uint32_t first_page = context >> a.pool.page_shift, within = context & (a.pool.page_size - 1u);
  const uint64_t page = static_cast<uint64_t>(first_page) + lane;
  const uint32_t entry = a.batch.tables[static_cast<uint64_t>(seq) * a.batch.table_pitch +
                                        (page < a.batch.table_pitch ? page : a.batch.table_pitch - 1u)];
  const uint32_t id = page < a.batch.table_pitch ? entry : ~0u;
  // the element of node `node` in a layer, kNowhere for a page that is not there
  auto element = [&](uint32_t node) {
    const uint32_t at = within + node;
    const uint32_t p = __shfl(id, static_cast<int>(at >> a.pool.page_shift));
    return p < a.pool.n_pages ? p * a.pool.page_stride + (at & (a.pool.page_size - 1u)) * D : kNowhere;
  };
  const bool apart = count <= 16u;  // the wavefronts work on parts of their own
  bool odd = false;
  for (uint32_t step = 0; step < (apart ? 1u : 4u); ++step) {
    const uint32_t part = group * 4u + (apart ? wave : step), row = apart ? 0u : wave * 16u;
    const uint32_t head = part / 2u % a.pool.kv_heads, layer = part / 2u / a.pool.kv_heads;
    uint16_t *pool = (part % 2u ? a.pool.v : a.pool.k) + static_cast<uint64_t>(head) * a.pool.page_size * D +
                     lane % kCpr * 8u + (layer < a.pool.layers ? layer * a.pool.layer_stride : 0u);
    u32x4 held[kLoads];
    uint64_t to[kLoads];
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) {
      const uint32_t j = row + i * kRpi + lane / kCpr;
      const uint32_t node = a.kept[lo + (j < count ? j : 0u)];
      const bool real = j < count, moves = real && node != j, exists = node < hi - lo && node < 64u;
      const uint64_t from = element(exists ? node : 0u), at = element(j);
      const bool fine = exists && from != kNowhere && at != kNowhere;
      to[i] = moves && fine && part < parts ? at : kNowhere;
      odd |= real && !fine;  // also a row that stays where it is
      held[i] = *reinterpret_cast<const u32x4 *>(pool + (to[i] != kNowhere ? from : 0u));
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (!apart) __syncthreads();
    // past the L2: 48 drafts in 28 layers 12.0 -> 11.2 us
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i)
      if (to[i] != kNowhere) __builtin_nontemporal_store(held[i], reinterpret_cast<u32x4 *>(pool + to[i]));
  }
  if (__builtin_amdgcn_ballot_w64(odd)) report(a.pool);
}

// Block (piece, pair, layer and K or V): 256 x 16 x 4 bytes of a page per step.
XPU_DEVICE void copy(uint32_t chunks) {
  // the pairs stay in the argument segment (the struct is the first argument)
  const auto &a = *(const __attribute__((address_space(4))) CopyArgs *)__builtin_amdgcn_kernarg_segment_ptr();
  const uint32_t pair = blockIdx.x % a.n, part = blockIdx.x / a.n;
  uint16_t *pool = (part % 2u ? a.pool.v : a.pool.k) + part / 2u * a.pool.layer_stride;
  const u32x4 *from = reinterpret_cast<const u32x4 *>(pool + a.src[pair] * a.pool.page_stride);
  u32x4 *to = reinterpret_cast<u32x4 *>(pool + a.dst[pair] * a.pool.page_stride);
  const uint32_t piece = blockIdx.y * 2048u;
  u32x4 held[8];  // chunks past the end load the last one
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i) held[i] = from[min(piece + i * 256u + threadIdx.x, chunks - 1u)];
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i) {
    const uint32_t c = piece + i * 256u + threadIdx.x;
    if (c < chunks) to[c] = held[i];
  }
}

}  // namespace cache
}  // namespace xpu

extern "C" __global__ __launch_bounds__(256) void xpu_cache_append_d128(xpu::AppendArgs a) { xpu::cache::append<128>(a); }
extern "C" __global__ __launch_bounds__(256) void xpu_cache_append_d64(xpu::AppendArgs a) { xpu::cache::append<64>(a); }
extern "C" __global__ __launch_bounds__(256) void xpu_cache_keep_d128(xpu::KeepArgs a) { xpu::cache::keep<128>(a); }
extern "C" __global__ __launch_bounds__(256) void xpu_cache_keep_d64(xpu::KeepArgs a) { xpu::cache::keep<64>(a); }
extern "C" __global__ __launch_bounds__(256) void xpu_cache_copy(xpu::CopyArgs, uint32_t chunks) {
  xpu::cache::copy(chunks);
}
