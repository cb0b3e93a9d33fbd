// Kernel arguments of the paged cache and its attention, filled by the host
// (cache_api.cpp) and passed by value, and the checks of what the device-side
// numbers say (kernels, and the host's tests of them).
#pragma once

#include <stdint.h>

#ifdef __HIP__
#define XPU_BOTH __host__ __device__ __forceinline__
#else
#define XPU_BOTH inline
#endif

namespace xpu {

struct PackedArgs {
  const uint16_t *q, *k, *v;
  uint16_t *out;
  const uint32_t *q_starts, *k_starts;
  uint64_t q_stride, k_stride, v_stride, out_stride;  // elements
  uint32_t n_seqs, q_rows, k_rows, heads, kv_heads, slots, pack_shift;
  float scale_log2e;
};

// One layer of a cache: element (page, head, slot, dim) at page * page_stride
// + (head * page_size + slot) * head_dim + dim.
struct PoolArgs {
  uint16_t *k, *v;
  uint64_t layer_stride, page_stride;  // elements
  uint32_t layers, kv_heads, page_size, page_shift, n_pages;
  uint32_t *status;
};

struct BatchArgs {
  const uint32_t *tables, *starts, *context;
  uint32_t n_seqs, rows, table_pitch;
};

// Element offset of position `pos` in a layer (head 0), or kNowhere where the
// table (of pitch > 0 entries) or the pool has no such page. Without a branch:
// a load behind one would be waited for before the next is issued.
constexpr uint64_t kNowhere = ~0ull;
XPU_BOTH uint64_t element_of(const PoolArgs &p, const uint32_t *table, uint32_t pitch, uint64_t pos, uint32_t d) {
  const uint64_t page = pos >> p.page_shift;
  const uint32_t id = table[page < pitch ? page : pitch - 1u];
  return page < pitch && id < p.n_pages ? id * p.page_stride + (pos & (p.page_size - 1u)) * d : kNowhere;
}

// A sequence with rows lo .. hi - 1 behind c positions. Lengths that the batch
// or the table cannot hold are cut to them (and `bad`), so that no work and no
// access is unbounded.
struct Lengths {
  uint32_t first, n, context, end;  // first row, rows, positions before them, positions in all
  bool bad;
};
XPU_BOTH Lengths lengths_of(uint32_t lo, uint32_t hi, uint32_t c, uint32_t rows, uint32_t pitch, uint32_t page_size) {
  const bool ok = lo <= hi && hi <= rows;
  Lengths s;
  s.first = ok ? lo : 0u;
  s.n = ok ? hi - lo : 0u;
  uint64_t room = static_cast<uint64_t>(pitch) * page_size;
  if (room > 0x7fffffffull) room = 0x7fffffffull;
  const uint64_t end = static_cast<uint64_t>(c) + s.n;
  s.bad = end > room;
  s.end = static_cast<uint32_t>(s.bad ? room : end);
  s.context = c < s.end ? c : s.end;
  return s;
}

struct TreeArgs {
  PoolArgs pool;
  BatchArgs batch;
  const uint16_t *q;
  uint16_t *out;
  const uint64_t *visible;
  float *partial;
  uint64_t q_stride, out_stride;
  uint32_t heads, fit, target, least, slots;
  float scale_log2e;
};

struct AppendArgs {
  PoolArgs pool;
  BatchArgs batch;
  const uint16_t *k, *v;
  uint64_t k_stride, v_stride;
};

struct KeepArgs {
  PoolArgs pool;
  BatchArgs batch;
  const uint32_t *kept, *counts;
  uint32_t *new_context;
};

struct Keep8Args {
  KeepArgs keep;
  uint32_t per_block;  // parts (layer, kv head, K or V) that a block takes: 1, or a multiple of 4
};

// The rotation of rows on their way (half = rotated dims / 2; 0: none).
struct RotaryArgs {
  const float *cos, *sin;  // [positions][half]
  const uint32_t *at;
  const uint16_t *q_gain, *k_gain;
  uint32_t positions, half, adjacent;
  float eps;
};

// New rows, Q with them where heads > 0. Of an 8-bit cache, pool.k and pool.v
// are the codes, and strides of the pool are in bytes.
struct RotateArgs {
  PoolArgs pool;
  BatchArgs batch;
  RotaryArgs rot;
  const uint16_t *q, *k, *v;
  uint16_t *q_out;
  uint64_t q_stride, k_stride, v_stride, out_stride;  // elements
  uint32_t heads;
  uint32_t parts;  // wavefronts that share a row
  uint32_t slots;  // 8 bits: blocks of positions that the batch reaches, at most
};

// An 8-bit cache's positions share scales by blocks of 16: 2^(byte - 127).
constexpr uint32_t kBlock = 16, kLeastScale = 27;

// A sequence's blocks that rows lo .. hi - 1 behind c positions reach.
XPU_BOTH uint32_t blocks_of(uint32_t n, uint32_t c) { return n ? ((c & (kBlock - 1u)) + n + kBlock - 1u) / kBlock : 0u; }

// The scale byte with which a float of these bits (a finite one, without its
// sign) is at most 448, the largest code: 1.75 * 2^8. At most 247.
XPU_BOTH uint32_t scale_for(uint32_t bits) {
  const uint32_t e = bits >> 23, s = (bits & 0x7fffffu) > 0x600000u ? e + 1u : e;
  return s < kLeastScale + 8u ? kLeastScale : s - 8u;
}

constexpr uint32_t kCopyPairs = 400;  // per launch; the arguments stay below 4 KiB
struct CopyArgs {
  PoolArgs pool;
  uint32_t n;
  uint32_t src[kCopyPairs], dst[kCopyPairs];
};

}  // namespace xpu
