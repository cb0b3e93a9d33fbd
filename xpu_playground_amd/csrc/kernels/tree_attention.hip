// Attention of drafted tokens over a paged cache (xpu_tree_attention).
//
// Sequence s has context[s] cached positions and then n = starts[s + 1] -
// starts[s] drafted nodes at the positions behind them, all in the pages of
// its table. A node sees every cached position and the nodes of its mask (or,
// without masks, the nodes up to itself).
//
// The G query heads of a kv head read the same keys, so the rows of a
// sequence and kv head are its n G (node, head) pairs, and a block takes up
// to 32 R of them (R sub-tiles) and a range of the keys: long contexts are cut
// into chunks so that few rows still fill the chip, and xpu_tree_join adds the
// chunks' (max, sum, output) in order. Within a block each wavefront walks
// its own keys in tiles of 32, staged by LDS-DMA into its own LDS, so there
// is no barrier in the loop: K of the next tile is fetched while the softmax
// and P V run, V of the next while the scores are formed. The four partial
// results meet in LDS at the end.
//
// The cut is worked out in the kernel from starts and context (`Cut`), so a
// call needs no lengths on the host and can be captured.
#include "attention_core.hpp"
#include "cache_types.hpp"

namespace xpu {
namespace att {

constexpr uint32_t kTreeKeys = 32;  // keys per tile

struct Sequence : Lengths {
  uint32_t row_tiles, tiles;  // tiles of rows, tiles of keys
};

// Sequence i (any lane's own i).
template <int R> XPU_DEVICE Sequence sequence(const BatchArgs &b, uint32_t page_size, uint32_t group, uint32_t i) {
  Sequence s{lengths_of(b.starts[i], b.starts[i + 1], b.context[i], b.rows, b.table_pitch, page_size), 0u, 0u};
  s.row_tiles = (s.n * group + 32u * R - 1u) / (32u * R);
  s.tiles = s.n ? (s.end + kTreeKeys - 1u) / kTreeKeys : 0u;
  return s;
}

// Sequence i, the same in every lane, in scalar registers.
template <int R>
XPU_DEVICE Sequence uniform_sequence(const BatchArgs &b, uint32_t page_size, uint32_t group, uint32_t i) {
  Sequence s = sequence<R>(b, page_size, group, i);
  for (uint32_t *v : {&s.first, &s.n, &s.context, &s.end, &s.row_tiles, &s.tiles})
    *v = __builtin_amdgcn_readfirstlane(*v);
  s.bad = __builtin_amdgcn_readfirstlane(s.bad);
  return s;
}

XPU_DEVICE uint64_t wave_sum(uint64_t v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// How the keys are cut: every chunk has at most `most` tiles, so that the
// chunks of all sequences and row tiles are at most target + the row tiles.
template <int R> XPU_DEVICE uint32_t chunk_limit(const TreeArgs &a, uint32_t group) {
  uint64_t work = 0;
  for (uint32_t i = lane_id(); i < a.batch.n_seqs; i += 64) {
    const Sequence s = sequence<R>(a.batch, a.pool.page_size, group, i);
    work += static_cast<uint64_t>(s.row_tiles) * s.tiles;
  }
  work = wave_sum(work);
  const uint64_t most = (work + a.target - 1) / a.target;
  return __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(most < a.least ? a.least : most));
}

// The work items are numbered sequence by sequence, chunk by chunk, and row
// tile by row tile within it, so that the row tiles that read the same keys
// run side by side (and, with 8 kv heads, on one XCD). find() gives the sequence for which `is(first,
// count, s)` holds, where first .. first + count - 1 are its items.
struct Place {
  int32_t seq;  // -1: none
  uint32_t first, chunks;
};
template <int R, typename Is> XPU_DEVICE Place find(const TreeArgs &a, uint32_t group, uint32_t most, Is &&is) {
  uint32_t before = 0;
  for (uint32_t at = 0; at < a.batch.n_seqs; at += 64) {
    const uint32_t i = at + lane_id();
    Sequence s{};
    uint32_t chunks = 0;
    if (i < a.batch.n_seqs) {
      s = sequence<R>(a.batch, a.pool.page_size, group, i);
      chunks = (s.tiles + most - 1) / most;
    }
    const uint32_t count = s.row_tiles * chunks;
    uint32_t upto = count;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
      const uint32_t v = __shfl_up(upto, d);
      if (lane_id() >= d) upto += v;
    }
    const uint32_t first = before + upto - count;
    const uint64_t hit = __builtin_amdgcn_ballot_w64(i < a.batch.n_seqs && is(first, count, s));
    if (hit) {
      const uint32_t l = __builtin_ctzll(hit);
      return {static_cast<int32_t>(__builtin_amdgcn_readfirstlane(at + l)),
              static_cast<uint32_t>(__builtin_amdgcn_readlane(first, l)),
              static_cast<uint32_t>(__builtin_amdgcn_readlane(chunks, l))};
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return {-1, 0, 0};
}

// Floats of one work item's partial result: 32 R rows of D sums, then their
// (max, sum) pairs.
template <int D, int R> constexpr uint32_t kPartial = 32u * R * (D + 2u);

template <int DT, int D, int R> XPU_DEVICE void tree_attention(const TreeArgs &a) {
  constexpr uint32_t kRow = 2u * D, kTile = kTreeKeys * kRow;
  constexpr uint32_t kRpi = 512u / D, kCpr = D / 8;
  constexpr uint32_t kDma = kTreeKeys / kRpi;  // DMA instructions per tile, K and V each
  constexpr uint32_t kMerge = 64u * R * (D / 2u) * 4u;  // bytes of one wave's output columns
  constexpr uint32_t kLds = 8u * kTile > 2u * kMerge ? 8u * kTile : 2u * kMerge;
  __shared__ __align__(1024) uint8_t lds[kLds];  // per wave a K and a V tile; then the partial results
  // the block's queries, then the (max, sum) pairs that its wavefronts exchange
  __shared__ __align__(16) uint8_t shared_q[R * Rows<DT, D, R>::kQBytes];

  const uint32_t tid = threadIdx.x, lane = tid & 63u, hh = lane >> 5;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t kvh = blockIdx.x % a.pool.kv_heads, item = blockIdx.x / a.pool.kv_heads;
  const uint32_t group = a.heads / a.pool.kv_heads;
  const uint32_t most = chunk_limit<R>(a, group);
  const Place place = find<R>(a, group, most, [&](uint32_t first, uint32_t count, const Sequence &) {
    return item >= first && item - first < count;
  });
  if (place.seq < 0) return;
  const uint32_t seq = static_cast<uint32_t>(place.seq);
  const Sequence s = uniform_sequence<R>(a.batch, a.pool.page_size, group, seq);
  const uint32_t row_tile = (item - place.first) % s.row_tiles, chunk = (item - place.first) / s.row_tiles;
  const uint32_t rows_in = min(s.n * group - row_tile * 32u * R, 32u * R);
  // the chunk's tiles, and the wave's share of them
  const uint32_t c0 = static_cast<uint32_t>(static_cast<uint64_t>(s.tiles) * chunk / place.chunks);
  const uint32_t c1 = static_cast<uint32_t>(static_cast<uint64_t>(s.tiles) * (chunk + 1u) / place.chunks);
  const uint32_t t_lo = c0 + (c1 - c0) * wave / 4u, t_hi = c0 + (c1 - c0) * (wave + 1u) / 4u;

  // the page ids of the wave's tiles, 64 at a time, a lane each
  const uint32_t *table = a.batch.tables + static_cast<uint64_t>(seq) * a.batch.table_pitch;
  const uint32_t pages = (s.end + a.pool.page_size - 1u) >> a.pool.page_shift;
  auto window = [&](uint32_t from) {
    const uint32_t at = from + lane;
    return at < pages ? table[at] : 0u;
  };
  uint32_t w_from = t_lo * kTreeKeys >> a.pool.page_shift;
  uint32_t ids = window(w_from), ids_next = window(w_from + 64u);

  const uint32_t qb = __builtin_amdgcn_readfirstlane(lds_addr(shared_q));
  Rows<DT, D, R> rows;
  rows.init();
  uint32_t node[R];
  uint64_t sees[R];  // bit j: node j
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t row = min(row_tile * 32u * R + 32u * r + (lane & 31u), s.n * group - 1u);
    node[r] = row / group;
    const uint16_t *q_row = a.q + (s.first + node[r]) * a.q_stride + (kvh * group + row % group) * D;
#pragma unroll
    for (uint32_t j = 0; j < D / 64; ++j)
      Rows<DT, D, R>::stage_q(qb + r * Rows<DT, D, R>::kQBytes, wave * (D / 64u) + j, q_row);
    if (a.visible) {
      sees[r] = a.visible[s.first + node[r]];
      if (s.n < 64u) sees[r] &= (1ull << s.n) - 1ull;
    }
  }
  bool bad = s.bad || (a.visible && s.n > 64u);

  uint32_t k_off[kDma / 2], v_off[kDma / 2];
#pragma unroll
  for (uint32_t j = 0; j < kDma / 2; ++j) {
    const uint32_t row = kRpi * j + lane / kCpr;
    k_off[j] = row * kRow + 16u * ((lane % kCpr) ^ k_swz<D>(row));
    v_off[j] = row * kRow + 16u * ((lane % kCpr) ^ v_swz<D>(row));
  }
  const uint32_t kb = __builtin_amdgcn_readfirstlane(lds_addr(lds)) + wave * 2u * kTile, vb = kb + kTile;
  const uint64_t head_at = static_cast<uint64_t>(kvh) * a.pool.page_size * D;
  // A tile is two halves of 16 keys, each inside one page (pages are 16 keys
  // or more). The descriptor ends with the sequence, so what older sequences
  // left in the page reads as zeros; a page id past the pool reads nothing.
  uint64_t from[2];
  uint32_t live[2];
  auto locate = [&](uint32_t tile) {
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t pos = tile * kTreeKeys + 16u * h, page = pos >> a.pool.page_shift;
      if (page - w_from >= 64u) {
        w_from += 64u;
        ids = ids_next;
        ids_next = window(w_from + 64u);
      }
      const uint32_t id = __builtin_amdgcn_readlane(ids, page - w_from);
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
  auto issue = [&](const uint16_t *pool, uint32_t to, const uint32_t (&off)[kDma / 2], const uint64_t (&at)[2],
                   const uint32_t (&bytes)[2]) {
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const i32x4 d = rsrc(pool + at[h], static_cast<int64_t>(bytes[h]));
#pragma unroll
      for (uint32_t j = 0; j < kDma / 2; ++j) dma16(to + (h * kDma / 2 + j) * 1024u, d, off[j]);
    }
  };

  if (t_lo < t_hi) {
    locate(t_lo);
    issue(a.pool.k, kb, k_off, from, live);
    issue(a.pool.v, vb, v_off, from, live);
  }
  __syncthreads();  // the queries are there
  for (uint32_t tile = t_lo; tile < t_hi; ++tile) {
    const bool more = tile + 1u < t_hi;
    wait_vmcnt<kDma>();  // K is there; V may be on its way
    const int32_t base = static_cast<int32_t>(s.context - tile * kTreeKeys);  // node 0 in the tile
    const bool edge = (tile + 1u) * kTreeKeys > s.context;  // the tile holds nodes (or ends the sequence)
    u32x8 pk[R][1];
    uint32_t seen[R][1] = {};
#pragma unroll
    for (int r = 0; r < R; ++r) {
      f32x16 sc[1];
      rows.template scores<1, true>(r, kb, qb, sc);
      if (r == R - 1 && more) {
        locate(tile + 1u);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K is read
        issue(a.pool.k, kb, k_off, from, live);
      }
      if (edge) {  // wave-uniform
        if (!a.visible) seen[r][0] = mask_to(base + static_cast<int32_t>(node[r]));
        else if (base >= 0) seen[r][0] = static_cast<uint32_t>(sees[r] << base) | ((1u << base) - 1u);
        else seen[r][0] = base > -64 ? static_cast<uint32_t>(sees[r] >> -base) : 0u;
        Rows<DT, D, R>::template mask<1>(sc, seen[r]);
      }
      rows.template softmax<1>(r, sc, a.scale_log2e, pk[r]);
    }
    if (more) wait_vmcnt<kDma>();
    else wait_vmcnt<0>();
    if (edge) {
      bool odd = false;
#pragma unroll
      for (uint32_t j = 0; j < kDma; ++j) {
        const u32x4 w = *reinterpret_cast<const lds_u32x4 *>(vb + j * 1024u + lane * 16u);
        odd |= nonfinite<DT>(w.x) || nonfinite<DT>(w.y) || nonfinite<DT>(w.z) || nonfinite<DT>(w.w);
      }
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(odd) != 0, 0)) {
#pragma unroll
        for (int r = 0; r < R; ++r) rows.add_apart(vb, r, pk[r][0], seen[r][0]);
        Rows<DT, D, R>::clear_apart(vb, kTreeKeys);
      }
    }
    rows.template values<1>(vb, pk);
    if (more) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // V is read
      issue(a.pool.v, vb, v_off, from, live);
    }
  }

  // Waves 2 and 3 hand their results to 0 and 1, and 1 to 0. Each wave's sum
  // is first that of both half-waves; `bad` makes the rows NaN.
  float sum[R];
#pragma unroll
  for (int r = 0; r < R; ++r) sum[r] = bad ? __builtin_nanf("") : rows.total(r);
  if (bad && lane == 0 && a.pool.status) *a.pool.status = 1u;
  float *po = reinterpret_cast<float *>(lds), *meet = reinterpret_cast<float *>(shared_q);
#pragma unroll
  for (uint32_t half = 2; half; half >>= 1) {
    __syncthreads();
    if (wave >= half && wave < 2u * half) {
      const uint32_t w = wave - half;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        meet[((w * R + r) * 2u) * 64u + lane] = rows.m[r];
        meet[((w * R + r) * 2u + 1u) * 64u + lane] = sum[r];
#pragma unroll
        for (uint32_t dt = 0; dt < D / 32; ++dt)
#pragma unroll
          for (uint32_t i = 0; i < 16; ++i)
            po[((w * R + r) * (D / 2u) + dt * 16u + i) * 64u + lane] = rows.o[r][dt][i];
      }
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float m2 = meet[((wave * R + r) * 2u) * 64u + lane], s2 = meet[((wave * R + r) * 2u + 1u) * 64u + lane];
        const float now = fmaxf(rows.m[r], m2), ninf = -__builtin_inff();
        const float x = rows.m[r] == ninf ? 0.0f : __builtin_amdgcn_exp2f((rows.m[r] - now) * a.scale_log2e);
        const float y = m2 == ninf ? 0.0f : __builtin_amdgcn_exp2f((m2 - now) * a.scale_log2e);
        // a side without a finite score has only zeros or NaN, which stay
        sum[r] = (rows.m[r] == ninf ? sum[r] : sum[r] * x) + (m2 == ninf ? s2 : s2 * y);
#pragma unroll
        for (uint32_t dt = 0; dt < D / 32; ++dt) {
          __builtin_amdgcn_sched_barrier(0);  // 16 reads at a time: all of them would need the registers of `o` again
#pragma unroll
          for (uint32_t i = 0; i < 16; ++i) {
            const float o2 = po[((wave * R + r) * (D / 2u) + dt * 16u + i) * 64u + lane];
            rows.o[r][dt][i] = __builtin_fmaf(rows.o[r][dt][i], x, o2 * y);
          }
        }
        rows.m[r] = now;
      }
    }
  }
  if (wave) return;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t in = 32u * r + (lane & 31u), row = row_tile * 32u * R + in;
    if (in >= rows_in) continue;
    if (place.chunks == 1) {
      const bool empty = s.context == 0 && a.visible && sees[r] == 0 && !bad;
      rows.store(r, a.out + (s.first + row / group) * a.out_stride + (kvh * group + row % group) * D,
                 empty ? 0.0f : 1.0f / sum[r]);
    } else {
      float *part = a.partial + (static_cast<uint64_t>(item) * a.pool.kv_heads + kvh) * kPartial<D, R>;
      float *to = part + in * D + 4u * hh;
#pragma unroll
      for (uint32_t dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (uint32_t w = 0; w < 4; ++w)
          *reinterpret_cast<dma::f32x4 *>(to + 32u * dt + 8u * w) = dma::f32x4{
              rows.o[r][dt][4 * w], rows.o[r][dt][4 * w + 1], rows.o[r][dt][4 * w + 2], rows.o[r][dt][4 * w + 3]};
      if (hh == 0) {
        part[32u * R * D + 2u * in] = rows.m[r];
        part[32u * R * D + 2u * in + 1u] = sum[r];
      }
    }
  }
}

// Adds the chunks of the rows whose keys were cut: one wavefront per (row,
// query head), D / 64 output dims per lane, chunks in order.
template <int DT, int D, int R> XPU_DEVICE void tree_join(const TreeArgs &a) {
  constexpr uint32_t kPer = D / 64;
  const uint32_t lane = lane_id(), index = blockIdx.x * 4u + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t row_at = index / a.heads, head = index % a.heads, group = a.heads / a.pool.kv_heads;
  if (row_at >= a.batch.rows) return;
  const uint32_t most = chunk_limit<R>(a, group);
  const Place place = find<R>(a, group, most, [&](uint32_t, uint32_t, const Sequence &s) {
    return row_at >= s.first && row_at - s.first < s.n;
  });
  if (place.seq < 0 || place.chunks < 2) return;
  const Sequence s = uniform_sequence<R>(a.batch, a.pool.page_size, group, static_cast<uint32_t>(place.seq));
  const uint32_t kvh = head / group, row = (row_at - s.first) * group + head % group;
  const uint32_t in = row % (32u * R);
  const uint64_t step = static_cast<uint64_t>(s.row_tiles) * a.pool.kv_heads * kPartial<D, R>;
  const float *part = a.partial + (static_cast<uint64_t>(place.first + row / (32u * R)) * a.pool.kv_heads + kvh) * kPartial<D, R>;
  const float *ms = part + 32u * R * D + 2u * in, *os = part + in * D + lane * kPer;
  const float ninf = -__builtin_inff();
  float top = ninf;
  for (uint32_t c = lane; c < place.chunks; c += 64) top = fmaxf(top, ms[c * step]);
  top = wave_reduce(top, [](float x, float y) { return fmaxf(x, y); });
  float sum = 0.0f, o[kPer] = {};
#pragma unroll 4
  for (uint32_t c = 0; c < place.chunks; ++c) {
    const float m = ms[c * step], l = ms[c * step + 1];
    const float x = m == ninf ? 0.0f : __builtin_amdgcn_exp2f((m - top) * a.scale_log2e);
    sum += m == ninf ? l : l * x;  // no finite score: zeros or NaN
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) o[i] = __builtin_fmaf(os[c * step + i], x, o[i]);
  }
  const float by = 1.0f / sum;  // a row that sees nothing has at most 64 positions, which are never cut
  uint16_t *to = a.out + row_at * a.out_stride + head * D + lane * kPer;
  if constexpr (kPer == 2) *reinterpret_cast<uint32_t *>(to) = dma::cvt_pack<DT>(o[0] * by, o[1] * by);
  else *to = static_cast<uint16_t>(dma::cvt_pack<DT>(o[0] * by, 0.0f));
}

}  // namespace att
}  // namespace xpu

#define XPU_TREE_ATTENTION(T, NAME, D, R)                                                                 \
  extern "C" __global__ __launch_bounds__(256, 2) void xpu_tree_attention_##NAME(xpu::TreeArgs a) {       \
    xpu::att::tree_attention<xpu::T, D, R>(a);                                                            \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(256) void xpu_tree_join_##NAME(xpu::TreeArgs a) {               \
    xpu::att::tree_join<xpu::T, D, R>(a);                                                                 \
  }
XPU_TREE_ATTENTION(kBf16, bf16_d128_r1, 128, 1)
XPU_TREE_ATTENTION(kFp16, fp16_d128_r1, 128, 1)
XPU_TREE_ATTENTION(kBf16, bf16_d64_r1, 64, 1)
XPU_TREE_ATTENTION(kFp16, fp16_d64_r1, 64, 1)
XPU_TREE_ATTENTION(kBf16, bf16_d128_r2, 128, 2)
XPU_TREE_ATTENTION(kFp16, fp16_d128_r2, 128, 2)
XPU_TREE_ATTENTION(kBf16, bf16_d64_r2, 64, 2)
XPU_TREE_ATTENTION(kFp16, fp16_d64_r2, 64, 2)
