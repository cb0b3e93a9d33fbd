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
// The cut is worked out in the kernel from starts and context (find), so a
// call needs no lengths on the host and can be captured.
//
// Without masks too every row tile walks all keys of its sequence, those behind
// its last node masked.
//
// Bound by the keys' way from memory: a variant without any of the arithmetic
// takes as long. Measured with D 128 and 8 kv heads (D 64 has not been timed): 48 single tokens behind
// up to 8000 positions 70 us, 5.65 TB/s; 48 drafts of 1 .. 26 nodes x 4 heads
// the same way 89 us, 5.0 TB/s (the counters say that no key is read twice);
// four drafts of 40 .. 64 nodes x 2 heads behind 90000 .. 131000 positions
// 375 to 396 us, 4.7 to 5.0 TB/s, each key read by two blocks of 64 rows and 25% of them
// twice from memory; of 16 nodes there, one block a key, 295 us, 6.25 TB/s;
// one token behind 2100 positions 11.5 us, two launches and their chains of
// loads, behind 32000 28.1 us, 4.6 TB/s. 128 rows to a
// block need more registers than there are (spills, 2272 us for the four
// drafts); eight wavefronts over common tiles with barriers took 432 us, a
// join in the last block to end instead of a second launch 18.4 us for the
// one token (11.8 then), for its fences.
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

// How the keys are cut: every chunk has at most `most` tiles. With `fit`, it is
// (in six halvings, so nearly) the least with which the chunks of all sequences
// (64 at most) and row tiles are at most fit: work / fit where that will do,
// else between it and work / (fit - row tiles), which always does. Without,
// work / target, which gives at most target + the row tiles.
// The work items are numbered sequence by sequence, chunk by chunk, and row
// tile by row tile within it, so that the row tiles that read the same keys
// run side by side (and, with 8 kv heads, on one XCD). find() gives the
// sequence for which `is(first, count, s)` holds, where first .. first + count
// - 1 are its items. Every wavefront works this out by itself, a lane per
// sequence, 64 sequences at a time.
struct Place {
  int32_t seq;  // -1: none
  uint32_t first, chunks;
  Sequence s;
};
template <int R, typename Is> XPU_DEVICE Place find(const TreeArgs &a, uint32_t group, Is &&is) {
  const uint32_t n = a.batch.n_seqs;
  auto of_lane = [&](uint32_t at) {
    Sequence s{};
    if (at + lane_id() < n) s = sequence<R>(a.batch, a.pool.page_size, group, at + lane_id());
    return s;
  };
  Sequence s = of_lane(0);
  uint64_t own = static_cast<uint64_t>(s.row_tiles) * s.tiles;
#pragma unroll 4
  for (uint32_t at = 64; at < n; at += 64) {
    const Sequence more = of_lane(at);
    own += static_cast<uint64_t>(more.row_tiles) * more.tiles;
  }
  // at most 2^50 in all (2^24 row tiles of 2^26 tiles of keys), in two sums of 32 bits
  const uint64_t work = wave_total(static_cast<uint32_t>(own) & 0xffffffu) +
                        (static_cast<uint64_t>(wave_total(static_cast<uint32_t>(own >> 24))) << 24);
  auto share = [&](uint32_t parts) {
    const uint64_t w = (work + parts - 1u) / parts;
    return w < a.least ? a.least : static_cast<uint32_t>(w < 0x7fffffffu ? w : 0x7fffffffu);
  };
  uint32_t most = share(a.fit ? a.fit : a.target);
  auto fits = [&](uint32_t m) { return wave_total(s.row_tiles * ((s.tiles + m - 1u) / m)) <= a.fit; };
  // (one row tile always fits; 0.3 us of a short call)
  if (a.fit && (n > 1u || a.batch.rows * group > 32u * R) && !fits(most)) {
    const uint32_t row_tiles = wave_total(s.row_tiles);
    uint32_t too_few = most;
    most = share(row_tiles < a.fit ? a.fit - row_tiles : 1u);
    for (uint32_t i = 0; i < 6 && too_few + 1u < most; ++i) {
      const uint32_t mid = too_few + (most - too_few) / 2u;
      if (fits(mid)) most = mid;
      else too_few = mid;
    }
  }
  uint32_t before = 0;
  Sequence next = of_lane(64);  // on its way (2048 single tokens with the two loops waiting for each 64: 1317 us, 1196)
  for (uint32_t at = 0;;) {
    const uint32_t chunks = (s.tiles + most - 1u) / most, count = s.row_tiles * chunks;
    const uint32_t upto = sum_upto(count), first = before + upto - count;
    const uint64_t hit = __builtin_amdgcn_ballot_w64(at + lane_id() < n && is(first, count, s));
    if (hit) {
      const uint32_t l = __builtin_ctzll(hit);
      auto of = [&](uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(v, l)); };
      Place p{static_cast<int32_t>(at + l), of(first), of(chunks), {}};
      p.s.first = of(s.first);
      p.s.n = of(s.n);
      p.s.context = of(s.context);
      p.s.end = of(s.end);
      p.s.bad = of(s.bad);
      p.s.row_tiles = of(s.row_tiles);
      p.s.tiles = of(s.tiles);
      return p;
    }
    if ((at += 64) >= n) break;
    before += __builtin_amdgcn_readlane(upto, 63);
    s = next;
    next = of_lane(at + 64);
  }
  return {-1, 0, 0, {}};
}

// Floats of one work item's partial result: 32 R rows of D sums, then their
// (max, sum) pairs.
template <int D, int R> constexpr uint32_t kPartial = 32u * R * (D + 2u);

template <int DT, int D, int R> XPU_DEVICE void tree_attention(const TreeArgs &a) {
  constexpr uint32_t kRow = 2u * D, kTile = kTreeKeys * kRow;
  constexpr uint32_t kRpi = 512u / D, kCpr = D / 8;
  constexpr uint32_t kDma = kTreeKeys / kRpi;  // DMA instructions per tile, K and V each
  // per wavefront a K and a V tile; then the partial results, D / 2 columns of
  // 64 floats each (as many bytes)
  __shared__ __align__(1024) uint8_t lds[8u * kTile];
  static_assert(8u * kTile == 4u * 64u * (D / 2u) * 4u, "the partial results fit the tiles' memory");
  // the block's queries, then the (max, sum) pairs that its wavefronts exchange
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

  // the wave's share of the queries: D / 64 of the 16-byte columns of every
  // row; on their way while the first tiles are asked for
  const uint32_t qb = __builtin_amdgcn_readfirstlane(lds_addr(shared_q));
  Rows<DT, D, R> rows;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(lds)) + wave * 2u * kTile;
  rows.init(lds0);
  uint32_t node[R];
  uint64_t sees[R];  // bit j: node j
  u32x4 q_part[R][D / 64];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t row = min(32u * (row_tile * R + r) + (lane & 31u), s.n * group - 1u);
    node[r] = row / group;
    const uint16_t *q_row = a.q + (s.first + node[r]) * a.q_stride + (kvh * group + row % group) * D;
#pragma unroll
    for (uint32_t j = 0; j < D / 64; ++j)
      q_part[r][j] = *reinterpret_cast<const u32x4 *>(q_row + (2u * (wave * (D / 64u) + j) + hh) * 8u);
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
  // Keys that only this block reads (of a kv head's rows) pass by the L2; with
  // more row tiles it serves the others.
  const bool once = s.row_tiles == 1;
  auto issue = [&](const uint16_t *pool, uint32_t to, const uint32_t (&off)[kDma / 2]) {
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const i32x4 d = rsrc(pool + from[h], static_cast<int64_t>(live[h]));
      const uint32_t at = to + h * kTile / 2u;
      if (once) {
#pragma unroll
        for (uint32_t j = 0; j < kDma / 2; ++j) dma16_nt(at + j * 1024u, d, off[j]);
      } else {
#pragma unroll
        for (uint32_t j = 0; j < kDma / 2; ++j) dma16(at + j * 1024u, d, off[j]);
      }
    }
  };

  if (t_lo < t_hi) {
    locate(t_lo);
    issue(a.pool.k, lds0, k_off);
    issue(a.pool.v, lds0 + kTile, v_off);
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (uint32_t j = 0; j < D / 64; ++j)
      *reinterpret_cast<lds_u32x4 *>(qb + r * Rows<DT, D, R>::kQBytes + (wave * (D / 64u) + j) * 1024u + lane * 16u) =
          q_part[r][j];
  __syncthreads();  // the queries are there
  // scores and softmax of a tile: p of every sub-tile, and which keys its
  // queries see where not all of them do (edge, wave-uniform)
  auto scored = [&](uint32_t tile, bool edge, u32x8 (&pk)[R][1], uint32_t (&seen)[R][1], auto &&after) {
    const int32_t base = static_cast<int32_t>(s.context - tile * kTreeKeys);  // node 0 in the tile
#pragma unroll
    for (int r = 0; r < R; ++r) {
      f32x16 sc[1];
      rows.template scores<1, true>(r, 0, qb, sc);
      if (r == R - 1) after();
      if (edge) {
        if (!a.visible) seen[r][0] = mask_to(base + static_cast<int32_t>(node[r]));
        else if (base >= 0) seen[r][0] = static_cast<uint32_t>(sees[r] << base) | ((1u << base) - 1u);
        else seen[r][0] = base > -64 ? static_cast<uint32_t>(sees[r] >> -base) : 0u;
        Rows<DT, D, R>::template mask<1>(sc, seen[r]);
      }
      rows.template softmax<1>(r, sc, a.scale_log2e, pk[r]);
    }
  };
  auto any_nonfinite = [&](uint32_t vb) {
    bool odd = false;
#pragma unroll
    for (uint32_t j = 0; j < kDma; ++j) {
      const u32x4 w = *reinterpret_cast<const lds_u32x4 *>(vb + j * 1024u + lane * 16u);
      odd |= nonfinite<DT>(w.x) || nonfinite<DT>(w.y) || nonfinite<DT>(w.z) || nonfinite<DT>(w.w);
    }
    return __builtin_amdgcn_ballot_w64(odd) != 0;
  };
  auto reads_done = [] { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };
  // whether a tile holds nodes (or ends the sequence)
  auto at_edge = [&](uint32_t tile) { return (tile + 1u) * kTreeKeys > s.context; };

  // One stage: K of the next tile goes out once the scores have read this
  // one's, V once P V has, so 8 to 16 KiB per wavefront are always on their way.
  for (uint32_t tile = t_lo; tile < t_hi; ++tile) {
    const bool more = tile + 1u < t_hi, edge = at_edge(tile);
    u32x8 pk[R][1];
    uint32_t seen[R][1] = {};
    wait_vmcnt<kDma>();  // K is there; V may be on its way
    scored(tile, edge, pk, seen, [&] {
      if (!more) return;
      locate(tile + 1u);
      reads_done();
      issue(a.pool.k, lds0, k_off);
    });
    if (more) wait_vmcnt<kDma>();
    else wait_vmcnt<0>();
    if (edge && __builtin_expect(any_nonfinite(lds0 + kTile), 0)) {
#pragma unroll
      for (int r = 0; r < R; ++r) rows.add_apart(lds0 + kTile, r, pk[r][0], seen[r][0]);
      Rows<DT, D, R>::clear_apart(lds0 + kTile, kTreeKeys);
    }
    rows.template values<1>(kTile, pk);
    reads_done();
    if (more) issue(a.pool.v, lds0 + kTile, v_off);
  }

  // The wavefronts' results meet in LDS, a sub-tile at a time; each wavefront
  // adds up a quarter of the columns (kMine registers of every lane's D / 2),
  // in the order of the keys. A side without a finite score has only zeros or
  // NaN in its sum, which stay. `bad` makes the rows NaN.
  if (bad && lane == 0 && a.pool.status) *a.pool.status = 1u;
  constexpr uint32_t kMine = D / 8;
  float *po = reinterpret_cast<float *>(lds), *meet = reinterpret_cast<float *>(shared_q);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    __syncthreads();  // the tiles, the queries, the sub-tile before are read
    meet[(wave * 2u) * 64u + lane] = rows.m[r];
    meet[(wave * 2u + 1u) * 64u + lane] = bad ? __builtin_nanf("") : rows.total(r);
#pragma unroll
    for (uint32_t dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) po[(wave * (D / 2u) + dt * 16u + i) * 64u + lane] = rows.o[r][dt][i];
    __syncthreads();
    const float ninf = -__builtin_inff();
    float m[4], x[4], top = ninf, sum = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) top = fmaxf(top, m[w] = meet[w * 128u + lane]);
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) {
      const float side = meet[w * 128u + 64u + lane];
      x[w] = m[w] == ninf ? 0.0f : __builtin_amdgcn_exp2f((m[w] - top) * a.scale_log2e);
      sum += m[w] == ninf ? side : side * x[w];
    }
    float o[kMine];
#pragma unroll
    for (uint32_t i = 0; i < kMine; ++i) {
      o[i] = 0.0f;
#pragma unroll
      for (uint32_t w = 0; w < 4; ++w)
        o[i] = __builtin_fmaf(po[(w * (D / 2u) + wave * kMine + i) * 64u + lane], x[w], o[i]);
    }
    // register wave * kMine + i: dims 32 (reg / 16) + 8 (reg % 16 / 4) + 4 hh + reg % 4
    const uint32_t in = 32u * r + (lane & 31u), row = row_tile * 32u * R + in;
    const uint32_t dim = wave * 2u * kMine + 4u * hh;
    if (in >= rows_in) continue;
    if (place.chunks == 1) {
      // (the sum has the NaN of every wavefront that met a missing page)
      const bool empty = s.context == 0 && a.visible && sees[r] == 0 && sum == 0.0f;
      const float by = empty ? 0.0f : 1.0f / sum;
      uint16_t *to = a.out + (s.first + row / group) * a.out_stride + (kvh * group + row % group) * D + dim;
#pragma unroll
      for (uint32_t w = 0; w < kMine / 4; ++w)
        *reinterpret_cast<u32x2 *>(to + 8u * w) = u32x2{dma::cvt_pack<DT>(o[4 * w] * by, o[4 * w + 1] * by),
                                                        dma::cvt_pack<DT>(o[4 * w + 2] * by, o[4 * w + 3] * by)};
    } else {
      float *slot = a.partial + (static_cast<uint64_t>(item) * a.pool.kv_heads + kvh) * kPartial<D, R>;
      float *to = slot + in * D + dim;
#pragma unroll
      for (uint32_t w = 0; w < kMine / 4; ++w)
        *reinterpret_cast<dma::f32x4 *>(to + 8u * w) = dma::f32x4{o[4 * w], o[4 * w + 1], o[4 * w + 2], o[4 * w + 3]};
      if (wave == 0 && hh == 0)
        *reinterpret_cast<dma::f32x2 *>(slot + 32u * R * D + 2u * in) = dma::f32x2{top, sum};
    }
  }
}

// Reductions over each half-wave: partners l ^ 16, 8, 4, 2, 1 of wave_reduce.
template <typename Op> XPU_DEVICE float half_reduce(float s, Op op) {
  s = op(s, xor16_f(s));
  s = op(s, xor8_f(s));
  s = op(s, dpp_f<0x124>(s));  // row_ror:4
  s = op(s, dpp_f<0x4E>(s));   // quad_perm [2,3,0,1]
  return op(s, dpp_f<0xB1>(s));  // quad_perm [1,0,3,2]
}

// Adds the chunks of the rows whose keys were cut: W wavefronts, each a W-th
// of the chunks, per row and two query heads, a half-wave each (half as many
// wavefronts, so that a batch's rows are one round of them on the chip). A lane
// takes one chunk's (max, sum) of 32, then D / 32 dims of every chunk's output,
// kAhead loads in flight, the first of which go out with the (max, sum) pairs.
template <int DT, int D, int R, int W> XPU_DEVICE void tree_join(const TreeArgs &a) {
  constexpr uint32_t kPer = D / 32, kAhead = 8;
  typedef float out_t __attribute__((ext_vector_type(kPer)));
  const uint32_t lane = lane_id(), half = lane >> 5, in_half = lane & 31u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), pairs = (a.heads + 1u) / 2u;
  const uint32_t index = W > 1 ? blockIdx.x : blockIdx.x * 4u + wave;
  const uint32_t row_at = index / pairs, head = min(index % pairs * 2u + half, a.heads - 1u);
  const bool spare = index % pairs * 2u + half >= a.heads;  // an odd number of heads
  const uint32_t group = a.heads / a.pool.kv_heads;
  if (row_at >= a.batch.rows) return;
  const Place place = find<R>(a, group, [&](uint32_t, uint32_t, const Sequence &s) {
    return row_at >= s.first && row_at - s.first < s.n;
  });
  if (place.seq < 0 || place.chunks < 2) return;
  const Sequence &s = place.s;
  // with starts that do not ascend there can be more work items than the workspace has
  if (place.first + static_cast<uint64_t>(s.row_tiles) * place.chunks > a.slots) {
    if (lane == 0 && a.pool.status) *a.pool.status = 1u;
    return;
  }
  const uint32_t kvh = head / group, row = (row_at - s.first) * group + head % group, in = row % (32u * R);
  const uint32_t begin = W > 1 ? place.chunks * wave / W : 0u;
  const uint32_t end = W > 1 ? place.chunks * (wave + 1u) / W : place.chunks;
  const uint64_t step = static_cast<uint64_t>(s.row_tiles) * a.pool.kv_heads * kPartial<D, R>;
  const float *part = a.partial + (static_cast<uint64_t>(place.first + row / (32u * R)) * a.pool.kv_heads + kvh) * kPartial<D, R>;
  const float *ms = part + 32u * R * D + 2u * in, *os = part + in * D + in_half * kPer;
  const float ninf = -__builtin_inff();
  float top = ninf, sum = 0.0f;
  out_t o = {}, v[kAhead];
  auto ask = [&](uint32_t c) {  // past the last chunk: it again, not counted
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i) v[i] = *reinterpret_cast<const out_t *>(os + min(c + i, end - 1u) * step);
  };
  for (uint32_t c0 = begin; c0 < end; c0 += 32) {
    const uint32_t mine = c0 + in_half, n = min(end - c0, 32u);
    const dma::f32x2 ml = *reinterpret_cast<const dma::f32x2 *>(ms + min(mine, end - 1u) * step);
    ask(c0);
    const float m = mine < end ? ml.x : ninf, l = mine < end ? ml.y : 0.0f;
    const float now = fmaxf(top, half_reduce(m, [](float x, float y) { return fmaxf(x, y); }));
    const float old = top == ninf ? 0.0f : __builtin_amdgcn_exp2f((top - now) * a.scale_log2e);
    const float x = m == ninf ? 0.0f : __builtin_amdgcn_exp2f((m - now) * a.scale_log2e);
    // without a finite score the sum is zeros or NaN, which stay
    sum = (top == ninf ? sum : sum * old) +
          half_reduce(m == ninf ? l : l * x, [](float x, float y) { return x + y; });
    o *= old;
    top = now;
    for (uint32_t j = 0; j < n; j += kAhead) {
      if (j) ask(c0 + j);
#pragma unroll
      for (uint32_t i = 0; i < kAhead; ++i) {
        if (j + i >= n) break;
        const float lo = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), j + i));
        const float hi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 32u + j + i));
        o += v[i] * (half ? hi : lo);
      }
    }
  }
  if constexpr (W > 1) {
    __shared__ float tops[W][64], sums[W][64];
    __shared__ __align__(16) out_t outs[W][64];
    tops[wave][lane] = top;
    sums[wave][lane] = sum;
    outs[wave][lane] = o;
    __syncthreads();
    if (wave) return;
    top = tops[0][lane];
#pragma unroll
    for (uint32_t w = 1; w < W; ++w) top = fmaxf(top, tops[w][lane]);
    sum = 0.0f;
    o = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) {
      const float t = tops[w][lane], x = t == ninf ? 0.0f : __builtin_amdgcn_exp2f((t - top) * a.scale_log2e);
      sum += t == ninf ? sums[w][lane] : sums[w][lane] * x;
      o += outs[w][lane] * x;
    }
  }
  if (spare) return;
  o *= 1.0f / sum;  // a row that sees nothing has at most 64 positions, which are never cut
  uint16_t *to = a.out + row_at * a.out_stride + head * D + in_half * kPer;
  if constexpr (kPer == 4)
    *reinterpret_cast<u32x2 *>(to) = u32x2{dma::cvt_pack<DT>(o[0], o[1]), dma::cvt_pack<DT>(o[2], o[3])};
  else
    *reinterpret_cast<uint32_t *>(to) = dma::cvt_pack<DT>(o[0], o[1]);
}

}  // namespace att
}  // namespace xpu

#define XPU_TREE_JOIN(T, NAME, D, R, W, BLOCK)                                                            \
  extern "C" __global__ __launch_bounds__(BLOCK) void xpu_tree_join_##NAME##_w##W(xpu::TreeArgs a) {      \
    xpu::att::tree_join<xpu::T, D, R, W>(a);                                                              \
  }
#define XPU_TREE_ATTENTION(T, NAME, D, R)                                                                 \
  extern "C" __global__ __launch_bounds__(256, 2) void xpu_tree_attention_##NAME(xpu::TreeArgs a) {       \
    xpu::att::tree_attention<xpu::T, D, R>(a);                                                            \
  }                                                                                                       \
  XPU_TREE_JOIN(T, NAME, D, R, 1, 256)                                                                    \
  XPU_TREE_JOIN(T, NAME, D, R, 4, 256)                                                                    \
  XPU_TREE_JOIN(T, NAME, D, R, 8, 512)                                                                    \
  XPU_TREE_JOIN(T, NAME, D, R, 16, 1024)
XPU_TREE_ATTENTION(kBf16, bf16_d128_r1, 128, 1)
XPU_TREE_ATTENTION(kFp16, fp16_d128_r1, 128, 1)
XPU_TREE_ATTENTION(kBf16, bf16_d64_r1, 64, 1)
XPU_TREE_ATTENTION(kFp16, fp16_d64_r1, 64, 1)
XPU_TREE_ATTENTION(kBf16, bf16_d128_r2, 128, 2)
XPU_TREE_ATTENTION(kFp16, fp16_d128_r2, 128, 2)
XPU_TREE_ATTENTION(kBf16, bf16_d64_r2, 64, 2)
XPU_TREE_ATTENTION(kFp16, fp16_d64_r2, 64, 2)
