// What the plan of a ragged extension batch holds, and what its kernels share.
#pragma once

#include "gemma4_device.hpp"
#include "fast_div.hpp"

#include "gemma4_flash_attention.h"

namespace gemma4 {

// A row block is a set of consecutive rows of one sequence that one workgroup
// attends together; its keys come in tiles. A share (one workgroup's work) is a
// run of segments, each a row block's tiles [tile_lo, tile_hi).
struct ExtendGeometry {
  int32_t rows;      // rows of a row block
  int32_t wave_rows; // of a wave's columns
  int32_t tile;      // keys of a tile
  int32_t shares;    // workgroups per KV head: heads x shares fill the chip
};
constexpr ExtendGeometry kExtend256 = {64, 16, 32, 32};
constexpr ExtendGeometry kExtend512 = {8, 2, 32, 256};
constexpr int kExtendBatch = 4096;  // sequences at most

struct ExtendSegment {
  int32_t row0;        // first row of the block within its sequence
  int32_t rows;
  int32_t base;        // row of the packed batch where the sequence begins
  int32_t prior;       // keys in the cache
  int32_t sequence;
  int32_t tile_lo, tile_hi;
  int32_t partial;     // first partial row, -1: the segment holds every tile
};
static_assert(sizeof(ExtendSegment) == 32, "two 16-byte loads");

// A share: its segments [first, end), and the first of them here, so that a
// workgroup has it with one load.
struct ExtendShare {
  int32_t first, end, pad[2];
  ExtendSegment segment;
};

// Partial sums of a row block that several segments share. One segment's are
// `stride` partial rows of [16][dim] fp32. Blocks of one wave's rows at most: row,
// query head, dim. Longer ones, as they leave the registers (rows rounded up to a
// wave's): KV head, wave's columns, chunks of 32 columns x 8 dims.
__host__ __device__ inline int32_t extend_partial_rows(const ExtendGeometry &g, int32_t rows) {
  return rows <= g.wave_rows ? rows : (rows + g.wave_rows - 1) / g.wave_rows * g.wave_rows;
}
// One partial row of a split row block.
struct ExtendMerge {
  int32_t row, rows;  // the block's, of the packed batch
  int32_t partial;    // its first segment's partial rows
  int32_t parts;      // segments
  int32_t stride;     // partial rows from one segment's to the next's
  int32_t index;      // this one among them
  int32_t segment;    // the block's first
  int32_t pad;
};
static_assert(sizeof(ExtendMerge) == 32, "two 16-byte loads");

struct ExtendHeader {
  uint32_t magic;
  int32_t batch, total_rows, heads, window, sinks, page_size;
  int32_t segments;
  int32_t merges;
  int32_t most_parts;  // of a split row block
  int32_t period;      // tiles of a share, about
};
// In a (row, query head) that has to be worked out again, the first element of one of
// its quarters: a signalling NaN, which no arithmetic gives.
constexpr uint16_t kExtendOdd = 0x7FA5;
constexpr uint32_t kExtendMagic = 0x67345850;

// Sections of the plan, by byte offset; all sizes follow from what the host knows.
struct ExtendPlanLayout {
  int64_t shares, segments, merges, bytes;
  int64_t max_segments, max_merges, max_partials;
};
inline int64_t extend_round(int64_t n) { return (n + 255) & ~(int64_t)255; }
inline ExtendPlanLayout extend_layout(const ExtendGeometry &g, int32_t batch, int32_t total_rows) {
  ExtendPlanLayout l;
  const int64_t blocks = total_rows / g.rows + (batch < total_rows ? batch : total_rows);
  l.max_segments = blocks + g.shares;
  const int64_t block_rows = extend_partial_rows(g, g.rows < total_rows ? g.rows : total_rows);
  // A cut splits one row block; a block of p segments has p - 1 cuts.
  l.max_merges = (int64_t)(g.shares - 1) * block_rows;
  l.max_partials = 2 * (int64_t)(g.shares - 1) * block_rows;
  l.shares = extend_round(sizeof(ExtendHeader));
  l.segments = extend_round(l.shares + g.shares * (int64_t)sizeof(ExtendShare));
  l.merges = extend_round(l.segments + l.max_segments * (int64_t)sizeof(ExtendSegment));
  l.bytes = extend_round(l.merges + l.max_merges * (int64_t)sizeof(ExtendMerge));
  return l;
}
inline const ExtendGeometry &extend_geometry(const Gemma4KvCacheConfig &c) {
  return c.num_heads == 1 ? kExtend512 : kExtend256;
}
// Workspace: the partial rows' sums, [16][dim] fp32 each, then their {maximum, sum},
// [16] each in the same order, then the words that tell which sums are not finite: at
// [first partial row of a wave's columns][KV head] a bit per column from each of the
// four waves, which have a quarter of the dims each.
inline int64_t extend_stats_offset(const ExtendPlanLayout &l, int32_t dim) {
  return extend_round(l.max_partials * kQueryHeads * (int64_t)dim * 4);
}
inline int64_t extend_odd_offset(const ExtendPlanLayout &l, int32_t dim) {
  return extend_stats_offset(l, dim) + extend_round(l.max_partials * kQueryHeads * 8);
}

// Key tiles of a row block whose rows sit at positions [first, last]: those of
// the sinks that lie before the window's first tile, then the window's. Tile i of
// the block starts at key (i < sink_tiles ? i : i - sink_tiles + window_tile) *
// tile.
struct ExtendTiles {
  int32_t sink_tiles, window_tile, count;
};
__device__ __forceinline__ ExtendTiles extend_tiles(int32_t first, int32_t last, int32_t window,
                                                    int32_t sinks, int32_t tile) {
  ExtendTiles r;
  r.window_tile = window > 0 ? max(first - window + 1, 0) / tile : 0;
  r.sink_tiles = min((sinks > 0 ? (sinks - 1) / tile + 1 : 0), r.window_tile);
  r.count = r.sink_tiles + last / tile - r.window_tile + 1;
  return r;
}

struct ExtendParams {
  uint16_t *out;          // [total][16][D]
  const uint16_t *q;      // [total][16][D], rows q_stride apart
  const uint16_t *k;      // [total][Hk][D], rows kv_stride apart
  const uint16_t *v;
  const uint16_t *cache_k;
  const uint16_t *cache_v;
  const int32_t *page_table;
  const char *plan;
  int32_t shares, segments, merges;  // byte offsets in the plan
  int32_t max_merges, max_segments;
  Gemma4KvCacheConfig c;
  FastDiv page_div, slot_div;
  int32_t layer, batch, total_rows;
  int64_t q_stride, kv_stride;
  float q_scale;          // softmax_scale * log2(e)
  float *partial;
  float *stats;
  uint32_t *odd;
};

// The plan is the same for every workgroup and read through the scalar cache.
template <class T>
__device__ __forceinline__ T plan_read(const char *at) {
  static_assert(sizeof(T) % 4 == 0);
  constexpr int kWords = sizeof(T) / 4;
  const auto *from = (const __attribute__((address_space(4))) uint32_t *)(uintptr_t)at;
  uint32_t words[kWords];
#pragma unroll
  for (int i = 0; i < kWords; ++i) words[i] = from[i];
  T x;
  __builtin_memcpy(&x, words, sizeof(T));
  return x;
}

// Whether the plan was made for this call's sizes.
__device__ __forceinline__ bool extend_plan_fits(const ExtendParams &p, const ExtendHeader &h) {
  return h.magic == kExtendMagic && h.batch == p.batch && h.total_rows == p.total_rows &&
         h.heads == p.c.num_heads && h.page_size == p.c.page_size;
}

}  // namespace gemma4
