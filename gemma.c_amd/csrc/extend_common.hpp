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
  int32_t rows;     // rows of a row block
  int32_t tile;     // keys of a tile
  int32_t shares;   // workgroups per KV head: heads x shares fill the chip
};
constexpr ExtendGeometry kExtend256 = {64, 32, 32};
constexpr ExtendGeometry kExtend512 = {8, 32, 256};
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

// One row of a row block that several segments share.
struct ExtendMerge {
  int32_t row;      // of the packed batch
  int32_t partial;  // its row among the first segment's partial rows
  int32_t parts;
  int32_t stride;   // partial rows from one segment's to the next's
};

struct ExtendHeader {
  uint32_t magic;
  int32_t batch, total_rows, heads, window, sinks, page_size;
  int32_t segments;
  int32_t merges;
};
constexpr uint32_t kExtendMagic = 0x67345850;

// Sections of the plan, by byte offset; all sizes follow from what the host knows.
struct ExtendPlanLayout {
  int64_t share_first, segments, merges, bytes;
  int64_t max_segments, max_merges, max_partials;
};
inline int64_t extend_round(int64_t n) { return (n + 255) & ~(int64_t)255; }
inline ExtendPlanLayout extend_layout(const ExtendGeometry &g, int32_t batch, int32_t total_rows) {
  ExtendPlanLayout l;
  const int64_t blocks = total_rows / g.rows + (batch < total_rows ? batch : total_rows);
  l.max_segments = blocks + g.shares;
  const int64_t block_rows = g.rows < total_rows ? g.rows : total_rows;
  // A cut splits one row block; a block of p segments has p - 1 cuts.
  l.max_merges = (int64_t)(g.shares - 1) * block_rows;
  if (l.max_merges > total_rows) l.max_merges = total_rows;
  l.max_partials = 2 * (int64_t)(g.shares - 1) * block_rows;
  l.share_first = extend_round(sizeof(ExtendHeader));
  l.segments = extend_round(l.share_first + (g.shares + 1) * 4);
  l.merges = extend_round(l.segments + l.max_segments * (int64_t)sizeof(ExtendSegment));
  l.bytes = extend_round(l.merges + l.max_merges * (int64_t)sizeof(ExtendMerge));
  return l;
}
inline const ExtendGeometry &extend_geometry(const Gemma4KvCacheConfig &c) {
  return c.num_heads == 1 ? kExtend512 : kExtend256;
}
// Workspace: partial sums [partial row][16][dim] fp32, then {maximum, sum}
// [partial row][16].
inline int64_t extend_stats_offset(const ExtendPlanLayout &l, int32_t dim) {
  return extend_round(l.max_partials * kQueryHeads * (int64_t)dim * 4);
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
  int32_t share_first, segments, merges;  // byte offsets in the plan
  Gemma4KvCacheConfig c;
  FastDiv page_div, slot_div;
  int32_t layer, batch, total_rows;
  int64_t q_stride, kv_stride;
  float q_scale;          // softmax_scale * log2(e)
  float *partial;
  float *stats;
};

// Whether the plan was made for this call's sizes.
__device__ __forceinline__ bool extend_plan_fits(const ExtendParams &p) {
  const auto *h = reinterpret_cast<const ExtendHeader *>(p.plan);
  return h->magic == kExtendMagic && h->batch == p.batch && h->total_rows == p.total_rows &&
         h->heads == p.c.num_heads && h->page_size == p.c.page_size;
}

}  // namespace gemma4
