// The paged cache's row and page operations: new rows into the pages
// (append), accepted drafts to the front of their draft (keep), whole pages
// (copy). All move 16-byte chunks of rows of D 16-bit elements; a lane holds
// one chunk, so the types and head sizes are only sizes here.
#include "cache_types.hpp"
#include "device_common.hpp"

namespace xpu {
namespace cache {

// The sequence that holds row `row` of the batch, or -1 (behind the last
// one, or starts that do not ascend). The starts are counted 64 at a time.
XPU_DEVICE int32_t sequence_of_row(const BatchArgs &b, uint32_t row) {
  uint32_t s = 0;
  for (uint32_t at = 1; at <= b.n_seqs; at += 64) {
    const uint32_t i = at + lane_id();
    s += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i <= b.n_seqs && b.starts[i] <= row));
  }
  if (s >= b.n_seqs || b.starts[s] > row || b.starts[s + 1] <= row || b.starts[s + 1] > b.rows) return -1;
  return static_cast<int32_t>(__builtin_amdgcn_readfirstlane(s));
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
    const int32_t seq = sequence_of_row(a.batch, row);
    if (seq < 0) continue;
    const uint64_t pos = static_cast<uint64_t>(a.batch.context[seq]) + (row - a.batch.starts[seq]);
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

// The moves of `count` rows (at most N loads of 512 / D rows each) of one
// (layer, kv head, K or V): all are loaded before the first is stored, so they
// may overlap in any order. Branch-free up to the stores, so that the loads
// are in flight together: rows that do not move read the pool's first element.
template <int D, int N>
XPU_DEVICE void move_rows(const KeepArgs &a, uint16_t *pool, const uint32_t *table, const uint32_t *kept,
                          uint32_t context, uint32_t nodes, uint32_t count) {
  constexpr uint32_t kRpi = 512u / D, kCpr = D / 8;
  const uint32_t lane = lane_id();
  auto element = [&](uint32_t node) {
    return element_of(a.pool, table, a.batch.table_pitch, static_cast<uint64_t>(context) + node, D);
  };
  uint32_t node[N];
#pragma unroll
  for (uint32_t i = 0; i < N; ++i) {
    const uint32_t j = i * kRpi + lane / kCpr;
    node[i] = kept[j < count ? j : 0u];
  }
  u32x4 held[N];
  uint64_t to[N];
  bool odd = false;
#pragma unroll
  for (uint32_t i = 0; i < N; ++i) {
    const uint32_t j = i * kRpi + lane / kCpr;
    const bool moves = j < count && node[i] != j;
    const uint64_t from = element(node[i] < nodes ? node[i] : 0u), at = element(j);
    const bool fine = node[i] < nodes && from != kNowhere && at != kNowhere;
    to[i] = moves && fine ? at : kNowhere;
    odd |= moves && !fine;
    held[i] = *reinterpret_cast<const u32x4 *>(pool + (moves && fine ? from : 0u));
  }
  if (__builtin_amdgcn_ballot_w64(odd)) report(a.pool);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
  for (uint32_t i = 0; i < N; ++i)
    if (to[i] != kNowhere) *reinterpret_cast<u32x4 *>(pool + to[i]) = held[i];
}

// One wavefront per (layer, kv head, K or V) of a sequence.
template <int D> XPU_DEVICE void keep(const KeepArgs &a) {
  constexpr uint32_t kRpi = 512u / D;
  const uint32_t lane = lane_id();
  const uint32_t per = a.pool.layers * a.pool.kv_heads * 2u;
  const uint64_t index = static_cast<uint64_t>(blockIdx.x) * 4u + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t seq = static_cast<uint32_t>(index / per), part = static_cast<uint32_t>(index % per);
  if (seq >= a.batch.n_seqs) return;
  const uint32_t lo = __builtin_amdgcn_readfirstlane(a.batch.starts[seq]);
  const uint32_t hi = __builtin_amdgcn_readfirstlane(a.batch.starts[seq + 1]);
  const uint32_t context = __builtin_amdgcn_readfirstlane(a.batch.context[seq]);
  const uint32_t count = __builtin_amdgcn_readfirstlane(a.counts[seq]);
  const bool ok = lo <= hi && hi <= a.batch.rows && count <= hi - lo && count <= 64u;
  if (!ok) {
    report(a.pool);
    return;
  }
  if (part == 0 && lane == 0 && a.new_context) a.new_context[seq] = context + count;
  if (count == 0) return;  // no row to read the first entry of
  const uint32_t head = part / 2u % a.pool.kv_heads, layer = part / 2u / a.pool.kv_heads;
  uint16_t *pool = (part % 2u ? a.pool.v : a.pool.k) + layer * a.pool.layer_stride +
                   static_cast<uint64_t>(head) * a.pool.page_size * D + lane % (D / 8) * 8u;
  const uint32_t *table = a.batch.tables + static_cast<uint64_t>(seq) * a.batch.table_pitch, *kept = a.kept + lo;
  // accepted paths are short: few loads where few rows are kept
  if (count <= 2u * kRpi) move_rows<D, 2>(a, pool, table, kept, context, hi - lo, count);
  else if (count <= 16u) move_rows<D, 16 / kRpi>(a, pool, table, kept, context, hi - lo, count);
  else move_rows<D, 64 / kRpi>(a, pool, table, kept, context, hi - lo, count);
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
