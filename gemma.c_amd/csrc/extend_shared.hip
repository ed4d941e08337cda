// Ragged extension of groups of sequences whose page tables begin with the same
// pages, gfx950: the plan that attends a group's shared keys once for all its rows. No
// counterpart in the reference.
//
// Softmax over a union of key sets joins from their maxima, sums and weighted values:
// m = max m_i, l = sum l_i 2^(m_i - m), o = sum o_i 2^(m_i - m) / l. So a row of a
// group is attended in two kinds of row blocks: its group's rows together over the
// prefix, and its sequence's rows over what lies behind it. To the rows' kernels both are
// ordinary segments: the group's packed rows follow each other, and a block of them
// that is said to begin behind the prefix (prior = its keys) sees all of it, by any
// member's page table. What differs is the plan, which lays prefixes' blocks and
// sequences' blocks end to end and cuts the line into equal shares, and the merge,
// which folds a row's parts of both kinds (extend_merge_kernel<.., true>).
// The prefix is cut down to whole tiles; the rest of it is read with each sequence.
//
// Of two kernels for the rows the host takes one by their number: extend_few.hip's
// blocks of a few rows, or extend_rows.hip's larger ones, which read a long prefix less
// often (few_rows).
#include "extend_few.hpp"
#include "extend_plan.hpp"

#include <algorithm>

namespace gemma4 {
namespace {

// What tells whether a group's prefix is attended together, in tiles' time: of a row
// (its sums go to memory and back twice, by way of the merge) and at all (the merge's way
// from the prefix's parts to the rows' own, while the chip would still take a tile each
// of more blocks at once).
struct SharedCosts {
  int32_t row, least;
  int32_t share;  // least cost worth a workgroup
};

struct SharedPlanParams {
  char *plan;
  int32_t shares, segments, merges;
  int64_t rows, common;
  const int32_t *row_offsets;
  const int32_t *prior_lengths;
  const int32_t *page_table;
  const int32_t *group_offsets;
  ExtendGeometry g;
  int32_t batch, groups, total_rows, heads, page_size, max_pages;
  int32_t max_prior;
  uint32_t magic;
  SharedCosts costs;
};

__device__ __forceinline__ int32_t prior_of(const SharedPlanParams &p, int32_t b) {
  return min(max(p.prior_lengths[b], 0), p.max_prior);
}

// Workgroup: a sequence; the leading pages of its table that equal those of the one
// before it, as far as both have keys. (Of a group's sequences all are equal as far as
// each equals the one before.)
constexpr int kCommonThreads = 256;
__global__ __launch_bounds__(kCommonThreads) void common_pages_kernel(SharedPlanParams p) {
  __shared__ int32_t s_first;
  const int32_t b = blockIdx.x, t = threadIdx.x;
  auto *common = reinterpret_cast<int32_t *>(p.plan + p.common);
  if (b == 0) {
    if (t == 0) common[0] = 0;
    return;
  }
  if (t == 0) s_first = 0x7fffffff;
  __syncthreads();
  const int32_t *mine = p.page_table + (int64_t)b * p.max_pages, *before = mine - p.max_pages;
  const int32_t keys = min(prior_of(p, b), prior_of(p, b - 1));
  const int32_t pages = min((int32_t)(((int64_t)keys + p.page_size - 1) / p.page_size), p.max_pages);
  int32_t first = pages;
  for (int32_t j0 = 0; j0 < pages; j0 += kCommonThreads) {
    const int32_t j = j0 + t;
    const bool differs = j < pages && mine[j] != before[j];
    if (differs) atomicMin(&s_first, j);
    __syncthreads();
    const int32_t found = s_first;
    __syncthreads();
    if (found != 0x7fffffff) {
      first = found;
      break;
    }
  }
  if (t == 0) common[b] = first;
}

// One workgroup, once a step for all layers.
template <int kPlanThreads>
__global__ __launch_bounds__(kPlanThreads) void extend_shared_plan_kernel(SharedPlanParams p) {
  constexpr int kPlanWaves = kPlanThreads / kWave;
  struct Lds {
    int32_t begin[kExtendBatch + 1];     // first row of a sequence
    int32_t prior[kExtendBatch];         // keys in the cache
    int32_t tiles0[kExtendBatch];        // tiles of its shared prefix
    int32_t group[kExtendBatch / 2 + 1]; // first sequence of a group
    int32_t blocks[kExtendBatch * 3 / 2 + 1];  // row blocks before a group's prefix, or a sequence's own
    int32_t share[kPlanShares + 1];      // first segment of a share
    int64_t waves[kPlanWaves];
    __attribute__((aligned(16))) uint32_t order[kPlanShares];
    int32_t waves32[kPlanWaves];
    int32_t parts;
    unsigned long long saved;
  };
  __shared__ Lds lds;
  const int t = threadIdx.x, lane = t & (kWave - 1), wave = t / kWave;
  auto *shares_at = reinterpret_cast<ExtendShare *>(p.plan + p.shares);
  auto *segments = reinterpret_cast<ExtendSegment *>(p.plan + p.segments);
  auto *merges = reinterpret_cast<ExtendMerge *>(p.plan + p.merges);
  auto *rows_at = reinterpret_cast<ExtendMerge *>(p.plan + p.rows);
  const auto *common = reinterpret_cast<const int32_t *>(p.plan + p.common);

  // Offsets within the batch and, by a running maximum, ascending, whatever they say.
  if (t == 0) {
    lds.parts = 0;
    lds.saved = 0;
  }
  auto ascending = [&](const int32_t *from, int32_t count, int32_t most, int32_t *to) {
    int32_t reach = 0;
    for (int32_t i0 = 0; i0 < count; i0 += kPlanThreads) {
      const int32_t i = i0 + t;
      int32_t last;
      const int32_t own = i < count ? min(max(from[i], 0), most) : 0;
      const int32_t top = max(block_prefix<kPlanWaves>(own, last, lds.waves32, Max()), reach);
      if (i < count) to[i] = top;
      reach = max(reach, last);
    }
  };
  ascending(p.row_offsets, p.batch + 1, p.total_rows, lds.begin);
  ascending(p.group_offsets, p.groups + 1, p.batch, lds.group);
  for (int32_t b = t; b < p.batch; b += kPlanThreads) {
    lds.prior[b] = prior_of(p, b);
    lds.tiles0[b] = 0;
  }
  __syncthreads();
  auto blocks_of = [&](int32_t rows) { return (rows + p.g.rows - 1) / p.g.rows; };

  // A wave a group: the whole tiles that all its sequences share, if attending them once
  // saves more than it costs. It saves the prefix's tiles in the blocks that the
  // group's rows need less when they are laid out together; it costs those blocks
  // themselves and SharedCosts. None is shared where all that is saved is less than
  // SharedCosts::least.
  for (int32_t i = wave; i < p.groups; i += kPlanWaves) {
    const int32_t from = lds.group[i], to = lds.group[i + 1];
    int32_t keys = 0x7fffffff, pages = 0x7fffffff, apart = 0;
    for (int32_t b = from + lane; b < to; b += kWave) {
      const int32_t rows = lds.begin[b + 1] - lds.begin[b];
      if (rows > 0) keys = min(keys, lds.prior[b]);
      if (b > from) pages = min(pages, common[b]);
      apart += blocks_of(rows);
    }
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      keys = min(keys, __shfl_xor(keys, d));
      pages = min(pages, __shfl_xor(pages, d));
      apart += __shfl_xor(apart, d);
    }
    const int64_t shared = min((int64_t)keys, (int64_t)pages * p.page_size);
    const int32_t tiles = to - from > 1 ? (int32_t)(min(shared, (int64_t)p.max_prior) / p.g.tile) : 0;
    const int32_t rows = to > from ? lds.begin[to] - lds.begin[from] : 0;
    const int64_t together = blocks_of(rows);
    const int64_t saved = (int64_t)tiles * (apart - together);
    const int64_t spent =
        together * block_cost(p.g, min(rows, p.g.rows)) + (int64_t)p.costs.row * rows;
    if (tiles > 0 && saved > spent) {
      for (int32_t b = from + lane; b < to; b += kWave) lds.tiles0[b] = tiles;
      if (lane == 0) atomicAdd(&lds.saved, (unsigned long long)(saved - spent));
    }
  }
  __syncthreads();
  if (lds.saved < (unsigned long long)p.costs.least)
    for (int32_t b = t; b < p.batch; b += kPlanThreads) lds.tiles0[b] = 0;
  __syncthreads();

  // Units: the groups' prefixes, then the sequences. lds.blocks: row blocks before each.
  const int32_t units = p.groups + p.batch;
  auto unit_rows = [&](int32_t u) -> int32_t {
    if (u >= p.groups) return lds.begin[u - p.groups + 1] - lds.begin[u - p.groups];
    const int32_t from = lds.group[u], to = lds.group[u + 1];
    return to > from && lds.tiles0[from] > 0 ? lds.begin[to] - lds.begin[from] : 0;
  };
  int32_t n_blocks = 0;
  for (int32_t u0 = 0; u0 < units; u0 += kPlanThreads) {
    const int32_t u = u0 + t;
    int32_t all;
    const int32_t own = u < units ? blocks_of(unit_rows(u)) : 0;
    const int32_t sum = block_prefix<kPlanWaves>(own, all, lds.waves32, Sum());
    if (u < units) lds.blocks[u] = n_blocks + sum - own;
    n_blocks += all;
  }
  if (t == 0) lds.blocks[units] = n_blocks;
  __syncthreads();

  struct Block {
    int32_t base, row0, rows, prior, sequence, tile_lo, tiles;
    bool prefix, shared;
    int64_t cost;
  };
  auto block_of = [&](int32_t j) {
    Block r{0, 0, 0, 0, 0, 0, 0, false, false, 0};
    if (j >= n_blocks) return r;
    int32_t lo = 0, hi = units;  // the last unit whose blocks begin at or before j
    while (hi - lo > 1) {
      const int32_t mid = (lo + hi) >> 1;
      if (lds.blocks[mid] <= j) lo = mid; else hi = mid;
    }
    r.prefix = lo < p.groups;
    r.sequence = r.prefix ? lds.group[lo] : lo - p.groups;
    r.base = lds.begin[r.sequence];
    const int32_t tiles0 = lds.tiles0[r.sequence];
    r.shared = tiles0 > 0;
    // A sequence's blocks first, last, second, last but one, .. (see extend_plan_kernel);
    // a prefix's all cost the same.
    const int32_t at = j - lds.blocks[lo], blocks = lds.blocks[lo + 1] - lds.blocks[lo];
    r.row0 = (at % 2 == 0 ? at / 2 : blocks - 1 - at / 2) * p.g.rows;
    r.rows = min(unit_rows(lo) - r.row0, p.g.rows);
    if (r.prefix) {
      r.prior = tiles0 * p.g.tile;
      r.tiles = tiles0;
    } else {
      r.prior = lds.prior[r.sequence];
      r.tile_lo = tiles0;
      r.tiles = (r.prior + r.row0 + r.rows - 1) / p.g.tile + 1 - tiles0;
    }
    r.cost = (int64_t)r.tiles + block_cost(p.g, r.rows);
    return r;
  };
  const Block own_block = block_of(t);
  int64_t cost = 0;
  for (int32_t j0 = 0; j0 < n_blocks; j0 += kPlanThreads) {
    int64_t all;
    block_prefix<kPlanWaves>(j0 == 0 ? own_block.cost : block_of(j0 + t).cost, all, lds.waves, Sum());
    cost += all;
  }
  const int32_t shares =
      (int32_t)min((int64_t)p.g.shares, max(cost / p.costs.share, (int64_t)1));
  const double step = (double)cost / (double)shares, per_step = 1.0 / step;
  // (One conversion to 32 bits, where that is enough, for a dozen instructions.)
  auto cut_at = [&](int32_t k) {
    const double at = (double)k * step;
    return cost <= 0x7fffffff ? (int64_t)(int32_t)at : (int64_t)at;
  };

  int64_t before = 0;                 // cost of the blocks of earlier rounds
  int64_t counts = 0, partials = 0;   // their segments and merged rows, and partial rows
  for (int32_t j0 = 0; j0 < n_blocks; j0 += kPlanThreads) {
    const Block r = j0 == 0 ? own_block : block_of(j0 + t);
    int64_t all;
    const int64_t end = before + block_prefix<kPlanWaves>(r.cost, all, lds.waves, Sum());
    const int64_t begin = end - r.cost;
    before += all;
    const int32_t ahead = block_cost(p.g, r.rows);
    // f(cut k, the tile it lies at: 0 is no cut of the block)
    auto for_cuts = [&](auto &&f) {
      if (r.rows == 0) return;
      int32_t k = max((int32_t)((double)begin * per_step), 1);  // about: put right here
      while (k > 1 && cut_at(k - 1) >= begin) --k;
      int64_t at = cut_at(k);
      while (k < shares && at < begin) at = cut_at(++k);
      for (; k < shares && at < end; at = cut_at(++k))
        f(k, (int32_t)max(at - begin - ahead, (int64_t)0));
    };
    int32_t parts = r.rows > 0 ? 1 : 0, last = 0;
    for_cuts([&](int32_t, int32_t tile) {
      if (tile > last) {
        ++parts;
        last = tile;
      }
    });
    const int32_t stride = extend_partial_rows(p.g, r.rows);
    const bool kept = r.rows > 0 && (parts > 1 || r.shared);  // as partial sums
    const bool merged = kept && (r.prefix || !r.shared);
    const int64_t own = (int64_t)parts << 32 | (merged ? stride : 0);
    const int64_t own_partial = kept ? (int64_t)parts * stride : 0;
    int64_t sums, partial_sums;
    const int64_t at = counts + block_prefix<kPlanWaves>(own, sums, lds.waves, Sum()) - own;
    const int32_t partial =
        (int32_t)(partials + block_prefix<kPlanWaves>(own_partial, partial_sums, lds.waves, Sum()) -
                  own_partial);
    counts += sums;
    partials += partial_sums;
    const int32_t segment = (int32_t)(at >> 32), merge = (int32_t)at;
    int32_t part = 0;
    last = 0;
    auto emit = [&](int32_t lo, int32_t hi) {
      segments[segment + part] = {r.row0, r.rows, r.base, r.prior, r.sequence, r.tile_lo + lo,
                                  r.tile_lo + hi, kept ? partial + part * stride : -1};
    };
    for_cuts([&](int32_t k, int32_t tile) {
      if (tile > last) {
        emit(last, tile);
        ++part;
        last = tile;
      }
      lds.share[k] = segment + part;
    });
    if (r.rows > 0) emit(last, r.tiles);
    if (merged) {
      atomicMax(&lds.parts, parts);
      for (int32_t i = 0; i < stride; ++i)
        merges[merge + i] = {r.base + r.row0, r.rows, partial, parts, stride, i, segment,
                             r.prefix ? 1 : 0};
    } else if (kept) {
      for (int32_t i = 0; i < r.rows; ++i)
        rows_at[r.base + r.row0 + i] = {r.base + r.row0, r.rows, partial, parts, stride, i, segment, 0};
    }
  }
  const int32_t n_segments = (int32_t)(counts >> 32);
  if (t == 0) lds.share[0] = 0;
  for (int32_t k = max(shares, 1) + t; k <= p.g.shares; k += kPlanThreads) lds.share[k] = n_segments;
  __threadfence_block();
  __syncthreads();
  // At 1 x 512 an XCD runs a range of the shares (see extend_rows_kernel): those of a
  // group's blocks in the order of their tiles, so that it reads an eighth of a prefix
  // once for all its rows (32 sequences, 8000 shared keys, blocks of 2 rows: 49.5 us to
  // 42.4, of 8 rows 46.6 to 44.8).
  static_assert(kPlanShares <= kPlanThreads, "a thread a share");
  static_assert(kExtend512.shares == kPlanShares && kFew512.shares == kPlanShares);
  const int32_t k = t;
  ExtendShare s = {0, 0, {}, {}};
  if (k < p.g.shares) {
    s.first = lds.share[k];
    s.end = lds.share[k + 1];
    if (s.first < s.end) s.segment = segments[s.first];
    const ExtendSegment &g = s.segment;
    const int32_t tiles0 = s.first < s.end ? lds.tiles0[g.sequence] : 0;
    // Sequence, place in the prefix in 4096ths, share: each once, prefixes' first.
    static_assert(kExtendBatch <= 1 << 12 && kPlanShares <= 1 << 8, "12, 12 and 8 bits");
    lds.order[k] = g.tile_lo < tiles0
                       ? (uint32_t)g.sequence << 20 | (uint32_t)(((int64_t)g.tile_lo << 12) / tiles0) << 8 | k
                       : 0xFFFFFF00u | k;
  }
  __syncthreads();
  if (k < p.g.shares) {
    int32_t rank = p.heads == 1 ? 0 : k;
    if (p.heads == 1) {
      const uint32_t own = lds.order[k];
#pragma unroll 16
      for (int32_t i = 0; i < kPlanShares; i += 4) {  // 1 x 512 has all of them
        const uint4 x = *reinterpret_cast<const uint4 *>(&lds.order[i]);
        rank += (x.x < own) + (x.y < own) + (x.z < own) + (x.w < own);
      }
    }
    shares_at[rank] = s;
  }
  if (t == 0) {
    *reinterpret_cast<ExtendHeader *>(p.plan) = {
        p.magic, p.batch, p.total_rows, p.heads, 0, 0, p.page_size, n_segments,
        (int32_t)counts, lds.parts, (int32_t)max(step, 1.0)};
  }
}

bool shared_sizes_ok(const Gemma4KvCacheConfig &c, int32_t batch, int32_t total_rows) {
  return extend_sizes_ok(c, batch, total_rows) && c.window_size == 0;
}
// Rows of a call up to which they go to extend_few.hip's kernel. Each of its small blocks reads
// all keys, so it depends on the keys as well, which only the device knows. Both kernels
// (us, few against large blocks) on tokens after 500, 4096, 16384 and 65536 shared keys, at
// 1 x 512 16 of them 13.4 : 17.5, 26.8 : 37.7, 38 : 43, 99 : 68, 64 of them 18.1 : 23.2,
// 40.4 : 46.0, 100 : 69, 402 : 168; at 8 x 256 14.8 : 14.5, 22.5 : 22.1, 35 : 37, 107 : 119 and
// 26.1 : 25.0, 43.8 : 32.7, 91 : 50, 307 : 132. A chunk of 64 rows after 4096, 16384 and
// 65536 keys of its own: 35.5 : 44.9, 91 : 71, 337 : 175, and 30.0 : 30.1, 74 : 44, 269 : 118.
// That is a line at about 400 000 rows x keys at 1 x 512, and at 8 x 256, beyond one block of
// 16 rows, at 200 000. A caller beyond it states more rows than there are (see the
// header).
constexpr int32_t kFewRows512 = 96, kFewRows256 = 64;
bool few_rows(const Gemma4KvCacheConfig &c, int32_t total_rows) {
  return total_rows <= (c.num_heads == 1 ? kFewRows512 : kFewRows256);
}
const ExtendGeometry &shared_geometry(const Gemma4KvCacheConfig &c, int32_t total_rows) {
  if (few_rows(c, total_rows)) return c.num_heads == 1 ? kFew512 : kFew256;
  return extend_geometry(c);
}
uint32_t shared_magic(const Gemma4KvCacheConfig &c, int32_t total_rows) {
  return few_rows(c, total_rows) ? kExtendFewMagic : kExtendSharedMagic;
}
// From where sharing took less time than not: groups of 2 to 64 sequences of a row each
// and of 5 and 300 keys behind a prefix of 64 to 16384. At 1 x 512 a few rows' line is at
// 4 sequences x 10000 keys, 8 x 5000, 16 x 4500 and 32 x 4000 (prefix blocks of two rows
// save half the reads, of which 256 workgroups make little); at 8 x 256, at 2 x 600, 10 x
// 500 and 32 x 350. In large blocks it is at 100 x 900 and at 100 x 64.
SharedCosts shared_costs(const Gemma4KvCacheConfig &c, int32_t total_rows) {
  if (few_rows(c, total_rows)) return c.num_heads == 1 ? SharedCosts{10, 256, 1} : SharedCosts{6, 0, 1};
  return c.num_heads == 1 ? SharedCosts{15, 0, kShareTiles} : SharedCosts{1, 0, kShareTiles};
}
// A larger call's buffers hold a smaller one's, also where that goes to the other kernel.
template <class Bytes>
size_t largest(const Gemma4KvCacheConfig &c, int32_t batch, int32_t total_rows, Bytes bytes) {
  if (!shared_sizes_ok(c, batch, total_rows)) return 0;
  const int32_t few = std::min(total_rows, c.num_heads == 1 ? kFewRows512 : kFewRows256);
  return std::max(
      bytes(extend_shared_layout(shared_geometry(c, total_rows), batch, total_rows).plan),
      bytes(extend_shared_layout(shared_geometry(c, few), batch, few).plan));
}
bool aligned256(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 255) == 0; }

}  // namespace
}  // namespace gemma4

using namespace gemma4;

extern "C" {

size_t gemma4_flash_attention_extend_shared_plan_bytes(Gemma4KvCacheConfig config,
                                                       int32_t batch_size, int32_t total_rows) {
  return largest(config, batch_size, total_rows,
                 [](const ExtendPlanLayout &l) { return (size_t)l.bytes; });
}

size_t gemma4_flash_attention_extend_shared_workspace_bytes(Gemma4KvCacheConfig config,
                                                            int32_t batch_size,
                                                            int32_t total_rows) {
  return largest(config, batch_size, total_rows,
                 [&](const ExtendPlanLayout &l) { return extend_workspace_bytes(l, config); });
}

hipError_t gemma4_flash_attention_extend_shared_plan(
    void *d_plan, size_t plan_bytes, const int32_t *d_row_offsets, const int32_t *d_prior_lengths,
    const int32_t *d_page_table, const int32_t *d_group_offsets, int32_t group_count,
    Gemma4KvCacheConfig config, int32_t batch_size, int32_t total_rows, hipStream_t stream) {
  if (!shared_sizes_ok(config, batch_size, total_rows) || d_plan == nullptr ||
      !aligned256(d_plan) || d_row_offsets == nullptr || d_prior_lengths == nullptr ||
      d_page_table == nullptr || d_group_offsets == nullptr || group_count < 0 ||
      group_count > kExtendBatch / 2) {
    return hipErrorInvalidValue;
  }
  const ExtendGeometry &g = shared_geometry(config, total_rows);
  const ExtendSharedLayout s = extend_shared_layout(g, batch_size, total_rows);
  if (plan_bytes < (size_t)s.plan.bytes) return hipErrorInvalidValue;
  SharedPlanParams p{};
  p.plan = static_cast<char *>(d_plan);
  p.shares = (int32_t)s.plan.shares;
  p.segments = (int32_t)s.plan.segments;
  p.merges = (int32_t)s.plan.merges;
  p.rows = s.rows;
  p.common = s.common;
  p.row_offsets = d_row_offsets;
  p.prior_lengths = d_prior_lengths;
  p.page_table = d_page_table;
  p.group_offsets = d_group_offsets;
  p.g = g;
  p.magic = shared_magic(config, total_rows);
  p.costs = shared_costs(config, total_rows);
  p.batch = batch_size;
  p.groups = group_count;
  p.total_rows = total_rows;
  p.heads = config.num_heads;
  p.page_size = config.page_size;
  p.max_pages = config.max_pages_per_seq;
  p.max_prior = (int32_t)std::min<int64_t>((int64_t)config.max_pages_per_seq * config.page_size,
                                           0x7fffffff - total_rows - 256);
  hipLaunchKernelGGL(common_pages_kernel, dim3(batch_size), dim3(kCommonThreads), 0, stream, p);
  // Where a thread of four waves has a sequence each and no more than a block of rows:
  // sixteen waves' barriers and spills take 10 us more on batches of 4 to 40 sequences
  // (17 to 23 with four); beyond, four would go round for every 256 blocks.
  if (batch_size + group_count <= 256 && total_rows / g.rows <= 256) {
    hipLaunchKernelGGL(extend_shared_plan_kernel<256>, dim3(1), dim3(256), 0, stream, p);
  } else {
    hipLaunchKernelGGL(extend_shared_plan_kernel<1024>, dim3(1), dim3(1024), 0, stream, p);
  }
  return hipGetLastError();
}

hipError_t gemma4_flash_attention_extend_shared_paged_bf16(
    gemma4_bf16 *d_out, const gemma4_bf16 *d_q, const gemma4_bf16 *d_k, const gemma4_bf16 *d_v,
    const gemma4_bf16 *d_cache_k, const gemma4_bf16 *d_cache_v, const int32_t *d_page_table,
    const void *d_plan, size_t plan_bytes, Gemma4KvCacheConfig config, int32_t layer,
    int32_t batch_size, int32_t total_rows, int64_t q_stride, int64_t kv_stride,
    float softmax_scale, void *d_workspace, size_t workspace_bytes, hipStream_t stream) {
  if (total_rows == 0) return hipSuccess;
  if (!shared_sizes_ok(config, batch_size, total_rows)) return hipErrorInvalidValue;
  const ExtendSharedLayout s =
      extend_shared_layout(shared_geometry(config, total_rows), batch_size, total_rows);
  if (plan_bytes < (size_t)s.plan.bytes) return hipErrorInvalidValue;
  return extend_attend({d_out, d_q, d_k, d_v, d_cache_k, d_cache_v, d_page_table, d_plan, config,
                        layer, batch_size, total_rows, q_stride, kv_stride, softmax_scale,
                        d_workspace, workspace_bytes},
                       s.plan, shared_magic(config, total_rows), s.rows, stream);
}

}  // extern "C"
