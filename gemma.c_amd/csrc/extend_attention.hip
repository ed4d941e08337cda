// Attention of a ragged batch of new tokens over the paged cache, gfx950: the
// plan that shares the work out, the merge of split row blocks and the entry
// points. No counterpart in the reference.
#include "extend_few.hpp"
#include "extend_plan.hpp"
#include "extend_rows.hpp"

#include <math.h>

#include <algorithm>

namespace gemma4 {
namespace {

struct PlanParams {
  char *plan;
  int32_t shares, segments, merges;
  const int32_t *row_offsets;
  const int32_t *prior_lengths;
  ExtendGeometry g;
  int32_t batch, total_rows, window, sinks, heads, page_size;
  int32_t max_prior;
};

// One workgroup, once a step for all layers: 10 to 14 us of dependent loads, barriers
// and prefix sums; up to 40 where a thread's block has most of the cuts (one token after 8192
// keys at 1 x 512). The row blocks laid end to end are cut into shares of equal cost,
// wherever the cuts fall: cuts that kept a tile or four away from a block's ends, to
// save partial sums, left shares of twice the mean where blocks are short (geometric
// mean of 32 batches of 1 to 30 sequences 38 -> 34 us without).
template <int kThreads>
__global__ __launch_bounds__(kThreads) void extend_plan_kernel(PlanParams p) {
  constexpr int kWaves = kThreads / kWave;
  __shared__ int32_t s_begin[kExtendBatch + 1];   // first row of a sequence
  __shared__ int32_t s_blocks[kExtendBatch + 1];  // row blocks before it
  __shared__ int32_t s_prior[kExtendBatch];       // keys in the cache
  __shared__ int32_t s_share[kPlanShares + 1];    // first segment of a share
  __shared__ int64_t s_waves[kWaves];
  __shared__ int32_t s_waves32[kWaves];
  __shared__ int32_t s_parts;
  const int t = threadIdx.x;
  auto *shares_at = reinterpret_cast<ExtendShare *>(p.plan + p.shares);
  auto *segments = reinterpret_cast<ExtendSegment *>(p.plan + p.segments);
  auto *merges = reinterpret_cast<ExtendMerge *>(p.plan + p.merges);

  // Offsets within the batch and, by a running maximum, ascending: whatever they
  // say, no row belongs to two sequences and the sections above hold the plan.
  if (t == 0) s_parts = 0;
  int32_t reach = 0;
  for (int32_t b0 = 0; b0 <= p.batch; b0 += kThreads) {
    const int32_t b = b0 + t;
    int32_t last;
    const int32_t own = b <= p.batch ? min(max(p.row_offsets[b], 0), p.total_rows) : 0;
    if (b < p.batch) s_prior[b] = min(max(p.prior_lengths[b], 0), p.max_prior);
    const int32_t top = max(block_prefix<kWaves>(own, last, s_waves32, Max()), reach);
    if (b <= p.batch) s_begin[b] = top;
    reach = max(reach, last);
  }
  __syncthreads();
  int32_t n_blocks = 0;
  for (int32_t b0 = 0; b0 < p.batch; b0 += kThreads) {
    const int32_t b = b0 + t;
    int32_t all;
    const int32_t own =
        b < p.batch ? (s_begin[b + 1] - s_begin[b] + p.g.rows - 1) / p.g.rows : 0;
    const int32_t sum = block_prefix<kWaves>(own, all, s_waves32, Sum());
    if (b < p.batch) s_blocks[b] = n_blocks + sum - own;
    n_blocks += all;
  }
  if (t == 0) s_blocks[p.batch] = n_blocks;
  __syncthreads();

  struct Block {
    int32_t sequence, row0, rows, prior, tiles;
    int64_t cost;
  };
  auto block_of = [&](int32_t j) {
    Block r{0, 0, 0, 0, 0, 0};
    if (j >= n_blocks) return r;
    // The last sequence whose blocks begin at or before j.
    int32_t lo = 0, hi = p.batch;
    while (hi - lo > 1) {
      const int32_t mid = (lo + hi) >> 1;
      if (s_blocks[mid] <= j) lo = mid; else hi = mid;
    }
    r.sequence = lo;
    // Causal work grows along a sequence: its blocks are laid out first, last, second,
    // last but one, .. so that every pair costs the same, and where two shares serve a
    // pair every other cut falls between blocks (2048 rows after 6144 at 1 x 512: 462 us,
    // 518 with the blocks last to first).
    const int32_t at = j - s_blocks[lo], blocks = s_blocks[lo + 1] - s_blocks[lo];
    r.row0 = (at % 2 == 0 ? at / 2 : blocks - 1 - at / 2) * p.g.rows;
    r.rows = min(s_begin[lo + 1] - s_begin[lo] - r.row0, p.g.rows);
    r.prior = s_prior[lo];
    const int32_t first = r.prior + r.row0;
    r.tiles = extend_tiles(first, first + r.rows - 1, p.window, p.sinks, p.g.tile).count;
    r.cost = (int64_t)r.tiles + block_cost(p.g, r.rows);
    return r;
  };
  const Block own_block = block_of(t);
  int64_t cost = 0;
  for (int32_t j0 = 0; j0 < n_blocks; j0 += kThreads) {
    int64_t all;
    block_prefix<kWaves>(j0 == 0 ? own_block.cost : block_of(j0 + t).cost, all, s_waves, Sum());
    cost += all;
  }
  const int32_t shares =
      (int32_t)min((int64_t)p.g.shares, max(cost / kShareTiles, (int64_t)1));
  // Cut k of 1 .. shares - 1 lies at this cost. Every thread evaluates the same
  // expression, so the blocks agree on it.
  const double step = (double)cost / (double)shares, per_step = 1.0 / step;
  auto cut_at = [&](int32_t k) { return (int64_t)((double)k * step); };

  int64_t before = 0;                        // cost of the blocks of earlier rounds
  int64_t counts = 0;                        // their segments, partial and merged rows
  for (int32_t j0 = 0; j0 < n_blocks; j0 += kThreads) {
    const Block r = j0 == 0 ? own_block : block_of(j0 + t);
    int64_t all;
    const int64_t end = before + block_prefix<kWaves>(r.cost, all, s_waves, Sum());
    const int64_t begin = end - r.cost;
    before += all;
    const int32_t ahead = block_cost(p.g, r.rows);
    // f(cut k, the tile it lies at: 0 is no cut of the block)
    auto for_cuts = [&](auto &&f) {
      if (r.rows == 0) return;
      int32_t k = max((int32_t)((double)begin * per_step), 1);  // about: put right here
      while (k > 1 && cut_at(k - 1) >= begin) --k;
      while (k < shares && cut_at(k) < begin) ++k;
      for (; k < shares && cut_at(k) < end; ++k) {
        f(k, (int32_t)max(cut_at(k) - begin - ahead, (int64_t)0));
      }
    };
    int32_t parts = r.rows > 0 ? 1 : 0, last = 0;
    for_cuts([&](int32_t, int32_t tile) {
      if (tile > last) {
        ++parts;
        last = tile;
      }
    });
    const int32_t stride = extend_partial_rows(p.g, r.rows);
    // Three counts in one word: partial rows stay below 2^16, merged ones too.
    const int64_t own = (int64_t)parts << 32 |
                        (parts > 1 ? (int64_t)(parts * stride) << 16 | stride : (int64_t)0);
    int64_t sums;
    const int64_t at = counts + block_prefix<kWaves>(own, sums, s_waves, Sum()) - own;
    counts += sums;
    const int32_t segment = (int32_t)(at >> 32);
    const int32_t partial = (int32_t)(at >> 16) & 0xFFFF, merge = (int32_t)at & 0xFFFF;
    int32_t part = 0;
    last = 0;
    auto emit = [&](int32_t lo, int32_t hi) {
      segments[segment + part] = {r.row0, r.rows, s_begin[r.sequence], r.prior, r.sequence, lo, hi,
                                  parts > 1 ? partial + part * stride : -1};
    };
    for_cuts([&](int32_t k, int32_t tile) {
      if (tile > last) {
        emit(last, tile);
        ++part;
        last = tile;
      }
      s_share[k] = segment + part;
    });
    if (r.rows > 0) emit(last, r.tiles);
    if (parts > 1) {
      atomicMax(&s_parts, parts);
      for (int32_t i = 0; i < stride; ++i)
        merges[merge + i] = {s_begin[r.sequence] + r.row0, r.rows, partial, parts, stride, i, segment, {}};
    }
  }
  const int32_t n_segments = (int32_t)(counts >> 32);
  if (t == 0) s_share[0] = 0;
  for (int32_t k = max(shares, 1) + t; k <= p.g.shares; k += kThreads) s_share[k] = n_segments;
  __threadfence_block();
  __syncthreads();
  for (int32_t k = t; k < p.g.shares; k += kThreads) {
    ExtendShare s = {s_share[k], s_share[k + 1], {}, {}};
    if (s.first < s.end) s.segment = segments[s.first];
    shares_at[k] = s;
  }
  if (t == 0) {
    *reinterpret_cast<ExtendHeader *>(p.plan) = {
        kExtendMagic, p.batch, p.total_rows, p.heads, p.window, p.sinks, p.page_size, n_segments,
        (int32_t)counts & 0xFFFF, s_parts, (int32_t)max(step, 1.0)};
  }
}

// ---- merge ----------------------------------------------------------------------
// Item: 1 KiB of partial sums (256 fp32, four to a lane) and the parts of a split row
// block that have them. A block of few parts is one wave's, kMergeBatch parts' loads
// at a time; of many, the four waves' of a workgroup, each a quarter of the parts.
// Parts are folded in a fixed order either way. Bound by the partial sums' bytes, 84 MB
// in 22 us for ten mixed sequences at 1 x 512 (3.8 TB/s), and by its launch and three
// dependent loads where there are few (4 us).
constexpr int kMergeThreads = 256;
constexpr int kMergeWaves = kMergeThreads / kWave;
constexpr int kMergeGrid = 2048;
constexpr int kMergeOwn = 4;  // parts behind a prefix whose loads are in flight together
constexpr int kMergeBatch = 4;
constexpr int kMergeFew = 16;  // parts a single wave folds

struct MergeState {
  float m = -INFINITY, l = 0.0f;
  float4 acc = {0, 0, 0, 0};
  uint32_t odd = 0;  // of the item's 32 columns, those with sums that are not finite
  __device__ __forceinline__ void fold(float mi, float li, const float4 &a) {
    const float top = fmaxf(m, mi);
    const float fa = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
    const float fb = mi == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mi - top);
    l = l * fa + li * fb;
    // A part without a visible key has nothing to add, whatever its sums are.
    acc.x = acc.x * fa + (mi == -INFINITY ? 0.0f : a.x * fb);
    acc.y = acc.y * fa + (mi == -INFINITY ? 0.0f : a.y * fb);
    acc.z = acc.z * fa + (mi == -INFINITY ? 0.0f : a.z * fb);
    acc.w = acc.w * fa + (mi == -INFINITY ? 0.0f : a.w * fb);
    m = top;
  }
};

// A (row, query head) from the keys that it sees alone, by one wave, kAgainKeys at a
// time: for columns that an infinity or NaN of V got into, which may be of a key that
// they do not see. For those only: all of 2048 rows after 6144 keys take 0.1 s.
constexpr int kAgainKeys = 4;
template <int kDim>
__device__ __forceinline__ void extend_again(int32_t segment, int32_t row, int32_t qh) {
  // The kernel's argument, read here: what only this needs takes no registers elsewhere.
  uint64_t argument = reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr());
  asm volatile("" : "+s"(argument));
  const ExtendParams p = plan_read<ExtendParams>(reinterpret_cast<const char *>(argument));
  const ExtendHeader h = plan_read<ExtendHeader>(p.plan);
  const ExtendSegment s =
      plan_read<ExtendSegment>(p.plan + p.segments + (int64_t)segment * sizeof(ExtendSegment));
  constexpr int kHeads = kDim == 256 ? 8 : 1, kPer = kDim / kWave;
  const int lane = threadIdx.x & 63, head = qh / (kQueryHeads / kHeads);
  const int32_t position = s.prior + row - s.base;
  const int64_t layer = (int64_t)p.layer * p.c.num_pages * p.c.page_size;
  typedef uint32_t Words __attribute__((ext_vector_type(kPer / 2)));  // this lane's dims
  auto load = [&](const uint16_t *row0) {
    return *reinterpret_cast<const Words *>(row0 + kPer * lane);
  };
  const Words q_words = load(p.q + row * p.q_stride + qh * kDim);
  float o[kPer] = {}, m = -INFINITY, l = 0.0f;
  const int32_t low = h.window > 0 ? max(position - h.window + 1, 0) : 0;
  const int32_t sinks = min(h.sinks, low);
  // Key i of the count = sinks + position - low + 1 that the row sees.
  const int32_t count = sinks + position - low + 1;
  for (int32_t i0 = 0; i0 < count; i0 += kAgainKeys) {
    Words k[kAgainKeys], v[kAgainKeys];
    bool ok[kAgainKeys];
#pragma unroll
    for (int j = 0; j < kAgainKeys; ++j) {
      const int32_t i = min(i0 + j, count - 1), key = i < sinks ? i : low + i - sinks;
      const uint16_t *from_k = p.k, *from_v = p.v;
      int64_t from = 0;
      ok[j] = i0 + j < count;
      if (key >= s.prior) {
        from = ((int64_t)s.base + key - s.prior) * p.kv_stride + head * kDim;
      } else {
        const uint32_t logical = fast_div((uint32_t)key, p.page_div);
        const int32_t page = p.page_table[(int64_t)s.sequence * p.c.max_pages_per_seq +
                                          fast_mod(logical, p.slot_div)];
        if (page >= 0 && page < p.c.num_pages &&
            (p.c.window_size > 0 || logical < (uint32_t)p.c.max_pages_per_seq)) {
          from = ((layer + (int64_t)page * p.c.page_size + key -
                   (int64_t)logical * p.c.page_size) * kHeads + head) * kDim;
          from_k = p.cache_k;
          from_v = p.cache_v;
        } else {
          ok[j] = false;
        }
      }
      k[j] = load(from_k + from);
      v[j] = load(from_v + from);
    }
#pragma unroll
    for (int j = 0; j < kAgainKeys; ++j) {
      if (!ok[j]) continue;
      float x = 0.0f;
#pragma unroll
      for (int e = 0; e < kPer / 2; ++e)
        x = fmaf(bf16_lo(q_words[e]), bf16_lo(k[j][e]), fmaf(bf16_hi(q_words[e]), bf16_hi(k[j][e]), x));
      for (int d = 1; d < kWave; d <<= 1) x += __shfl_xor(x, d);
      x *= p.q_scale;
      const float top = fmaxf(m, x), base = top == -INFINITY ? 0.0f : top;
      const float a = m == top ? 1.0f : __builtin_amdgcn_exp2f(m - base);
      const float w = __builtin_amdgcn_exp2f(x - base);
      l = l * a + w;
#pragma unroll
      for (int e = 0; e < kPer / 2; ++e) {
        o[2 * e] = o[2 * e] * a + w * bf16_lo(v[j][e]);
        o[2 * e + 1] = o[2 * e + 1] * a + w * bf16_hi(v[j][e]);
      }
      m = top;
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  Words words;
#pragma unroll
  for (int e = 0; e < kPer / 2; ++e) words[e] = cvt_pk_bf16(o[2 * e] * inv, o[2 * e + 1] * inv);
  *reinterpret_cast<Words *>(p.out + ((int64_t)row * kQueryHeads + qh) * kDim + kPer * lane) = words;
}

// kShared: a block of a prefix that sequences share has the prefix's parts; each of its
// rows has others, behind the prefix, in the partial sums of its own sequence's blocks,
// which are folded in when the prefix's are.
// kFew: all blocks are of a few rows (extend_few.hip).
template <int kDim, bool kShared, bool kFew = false>
__global__ __launch_bounds__(kMergeThreads, kShared ? 4 : 5) void extend_merge_kernel(ExtendParams p) {
  __shared__ float4 s_acc[kMergeWaves][kWave];
  __shared__ float2 s_stats[kMergeWaves][kWave];
  __shared__ uint32_t s_odd[kMergeWaves];
  constexpr ExtendGeometry kG = kFew ? (kDim == 256 ? kFew256 : kFew512)
                                     : (kDim == 256 ? kExtend256 : kExtend512);
  constexpr int kHeads = kDim == 256 ? 8 : 1, kGroup = kQueryHeads / kHeads;
  constexpr int kRowItems = kQueryHeads * kDim / 256;  // items of a partial row
  constexpr int kWaveDims = kDim / 4;                  // dims of a wave in the rows' kernel
  const int lane = threadIdx.x & 63, wave = wave_uniform(threadIdx.x >> 6);
  auto merge_of = [&](int32_t item) {
    return plan_read<ExtendMerge>(p.plan + p.merges + (int64_t)(item / kRowItems) * sizeof(ExtendMerge));
  };
  const int32_t first_item = wave_uniform(blockIdx.x * kMergeWaves + wave);
  // Asked for together with the header: within the plan whatever that says.
  ExtendMerge r = merge_of(min(first_item, max(p.max_merges, 1) * kRowItems - 1));
  // Marks in row blocks of one segment: a unit is a row's, four to a query head.
  auto segment_of = [&](int32_t unit) {
    return plan_read<ExtendSegment>(p.plan + p.segments +
                                    (int64_t)(unit / kG.rows) * sizeof(ExtendSegment));
  };
  auto marks_of = [&](const ExtendSegment &s, int32_t unit) -> uint16_t {
    if (s.partial >= 0 || unit % kG.rows >= s.rows) return 0;
    const int64_t row = s.base + s.row0 + unit % kG.rows;
    return p.out[(row * kQueryHeads + lane / 4) * kDim + lane % 4 * (kDim / 4)];
  };
  ExtendSegment seg = segment_of(min(first_item, p.max_segments * kG.rows - 1));
  const ExtendHeader h = plan_read<ExtendHeader>(p.plan);
  if (!extend_plan_fits(p, h)) return;
  const int32_t items = h.merges * kRowItems, units = h.segments * kG.rows;
  uint16_t mark = first_item < units ? marks_of(seg, first_item) : 0;

  // Where an item's values are: this lane's in the first part's sums and stats, and in
  // the output (out -1: a column without a row).
  struct Place {
    int64_t sum, stat, out;
    int32_t odd;   // the first part's words (all lanes' the same)
    int32_t row, head;
    uint32_t bit;  // this lane's column in them
    bool again;    // this lane's item works the column out again, if need be
  };
  auto place = [&](const ExtendMerge &m, int32_t item) {
    const int32_t chunk = m.index * kRowItems + item % kRowItems;
    Place at;
    int32_t row, head, dim;
    if (m.rows <= kG.wave_rows) {
      row = m.index;
      head = chunk % kRowItems / (kDim / 256);
      dim = chunk % (kDim / 256) * 256 + 4 * lane;
      at.stat = (int64_t)(m.partial + row) * kQueryHeads + head;
      at.odd = (m.partial * kHeads + head / kGroup) * 4;
      at.bit = 1u << (kGroup == 2 ? head % 2 * 16 + row : row * 16 + head);
      at.again = dim == 0;
    } else {
      // [KV head][group of 32 columns][wave][32 dims][8 dims][lane]
      const int32_t per_head = m.stride * kGroup * kDim / 256;
      const int32_t kv = chunk / per_head, i = chunk - kv * per_head;
      const int32_t group = i / (kDim / 8), j = i % (kDim / 8), n = lane & 31;
      row = group * kG.wave_rows + (kGroup == 2 ? n % 16 : n / 16);
      head = kv * kGroup + (kGroup == 2 ? n / 16 : n % 16);
      dim = j / (kWaveDims / 8) * kWaveDims + j % (kWaveDims / 8) * 8 + 4 * (lane >> 5);
      at.stat = (int64_t)m.partial * kQueryHeads + kv * m.stride * kGroup + group * 32 + n;
      at.odd = ((m.partial + group * kG.wave_rows) * kHeads + kv) * 4;
      at.bit = 1u << n;
      at.again = lane == j && j < 32;
    }
    at.sum = ((int64_t)m.partial * kRowItems + chunk) * 256 + 4 * lane;
    at.out = row < m.rows ? ((int64_t)(m.row + row) * kQueryHeads + head) * kDim + dim : -1;
    at.row = m.row + row;
    at.head = head;
    return at;
  };
  // The parts of this lane's column behind the prefix: one or a few, read 16 bytes a
  // lane from where the rows' kernel left them (see place).
  auto fold_own = [&](const Place &at, int32_t dim, MergeState &s, int32_t &segment) {
    if (at.out < 0) return;
    const ExtendMerge own = *reinterpret_cast<const ExtendMerge *>(
        p.plan + p.rows + (int64_t)at.row * sizeof(ExtendMerge));
    segment = own.segment;
    const int32_t row = own.index, kv = at.head / kGroup;
    int64_t sum, stat, odd;
    uint32_t bit;
    if (own.rows <= kG.wave_rows) {
      stat = (int64_t)(own.partial + row) * kQueryHeads + at.head;
      sum = stat * kDim + dim;
      odd = ((int64_t)own.partial * kHeads + kv) * 4;
      bit = 1u << (kGroup == 2 ? at.head % 2 * 16 + row : row * 16 + at.head);
    } else {
      const int32_t group = row / kG.wave_rows;
      const int32_t n = kGroup == 2 ? at.head % 2 * 16 + row % 16 : row % 2 * 16 + at.head;
      stat = (int64_t)own.partial * kQueryHeads + kv * own.stride * kGroup + group * 32 + n;
      sum = ((int64_t)own.partial * kRowItems + kv * (own.stride * kGroup * kDim / 256) +
             group * (kDim / 8) + dim / 8) * 256 + 4 * (n + dim / 4 % 2 * 32);
      odd = ((int64_t)(own.partial + group * kG.wave_rows) * kHeads + kv) * 4;
      bit = 1u << n;
    }
    const int64_t part_stats = (int64_t)own.stride * kQueryHeads;
    for (int32_t part0 = 0; part0 < own.parts; part0 += kMergeOwn) {
      float2 stats[kMergeOwn];
      float4 a[kMergeOwn];
      uint4 words[kMergeOwn];
#pragma unroll
      for (int i = 0; i < kMergeOwn; ++i) {
        if (part0 + i >= own.parts) break;
        const int64_t part = part0 + i;
        stats[i] = *reinterpret_cast<const float2 *>(p.stats + 2 * (stat + part * part_stats));
        a[i] = *reinterpret_cast<const float4 *>(p.partial + sum + part * part_stats * kDim);
        words[i] = *reinterpret_cast<const uint4 *>(p.odd + odd + part * own.stride * kHeads * 4);
      }
#pragma unroll
      for (int i = 0; i < kMergeOwn; ++i) {
        if (part0 + i >= own.parts) break;
        s.fold(stats[i].x, stats[i].y, a[i]);
        if ((words[i].x | words[i].y | words[i].z | words[i].w) & bit) s.odd |= at.bit;
      }
    }
  };
  // Parts first, first + step, .. of an item.
  auto gather = [&](const ExtendMerge &m, const Place &at, int32_t first, int32_t step) {
    MergeState s;
    // The words of the first 16 parts, asked for with the first sums.
    auto odd_of = [&](int32_t part) -> uint32_t {
      return p.odd[at.odd + min(part, m.parts - 1) * m.stride * kHeads * 4 + lane % 4];
    };
    const uint32_t odd = odd_of(first + lane / 4 * step);
    const int64_t part_stats = (int64_t)m.stride * kQueryHeads;
    for (int32_t i0 = first; i0 < m.parts; i0 += step * kMergeBatch) {
      float2 stats[kMergeBatch];
      float4 a[kMergeBatch];
#pragma unroll
      for (int i = 0; i < kMergeBatch; ++i) {
        const int32_t part = i0 + i * step;
        if (part >= m.parts) break;
        stats[i] = *reinterpret_cast<const float2 *>(p.stats + 2 * (at.stat + part * part_stats));
        a[i] = *reinterpret_cast<const float4 *>(p.partial + at.sum + part * part_stats * kDim);
      }
#pragma unroll
      for (int i = 0; i < kMergeBatch; ++i) {
        if (i0 + i * step >= m.parts) break;
        s.fold(stats[i].x, stats[i].y, a[i]);
      }
    }
    s.odd = odd;
    for (int32_t part = first + (16 + lane / 4) * step; part < m.parts; part += 16 * step)
      s.odd |= odd_of(part);
    if (__builtin_expect(__ballot(s.odd != 0) != 0, 0))
      for (int d = 1; d < kWave; d <<= 1) s.odd |= __shfl_xor(s.odd, d);
    return s;
  };
  auto store = [&](const Place &at, const ExtendMerge &m, MergeState s) {
    int32_t segment = m.segment;
    if constexpr (kShared) {
      if (m.prefix != 0) fold_own(at, (int32_t)(at.out % kDim), s, segment);
    }
    const float inv = s.l > 0.0f ? 1.0f / s.l : 0.0f;
    if (at.out >= 0 && (s.odd & at.bit) == 0)
      *reinterpret_cast<uint2 *>(p.out + at.out) = make_uint2(
          cvt_pk_bf16(s.acc.x * inv, s.acc.y * inv), cvt_pk_bf16(s.acc.z * inv, s.acc.w * inv));
    uint64_t again = __ballot((s.odd & at.bit) != 0 && at.out >= 0 && at.again);
    for (; __builtin_expect(again != 0, 0); again &= again - 1) {
      const int from = __builtin_ctzll(again);
      extend_again<kDim>(kShared ? __shfl(segment, from) : m.segment, __shfl(at.row, from),
                         __shfl(at.head, from));
    }
  };
  // Blocks of few parts.
  for (int32_t i = first_item; i < items;) {
    const int32_t ahead = i + gridDim.x * kMergeWaves;
    const ExtendMerge next = merge_of(min(ahead, items - 1));
    if (r.parts <= kMergeFew) {
      const Place at = place(r, i);
      store(at, r, gather(r, at, 0, 1));
    }
    i = ahead;
    r = next;
  }
  // Blocks of many.
  for (int32_t i = blockIdx.x; h.most_parts > kMergeFew && i < items; i += gridDim.x) {
    r = merge_of(i);
    if (r.parts <= kMergeFew) continue;
    const Place at = place(r, i);
    MergeState s = gather(r, at, wave, kMergeWaves);
    s_acc[wave][lane] = s.acc;
    s_stats[wave][lane] = make_float2(s.m, s.l);
    if (lane == 0) s_odd[wave] = s.odd;
    __syncthreads();
    if (wave == 0) {
      for (int w = 1; w < kMergeWaves; ++w) {
        s.fold(s_stats[w][lane].x, s_stats[w][lane].y, s_acc[w][lane]);
        s.odd |= s_odd[w];
      }
      store(at, r, s);
    }
    __syncthreads();
  }
  for (int32_t i = first_item; i < units;) {
    uint64_t marks = __ballot(mark == kExtendOdd);
    while (__builtin_expect(marks != 0, 0)) {
      const int qh = __builtin_ctzll(marks) / 4;
      marks &= ~(15ull << (4 * qh));
      extend_again<kDim>(i / kG.rows, seg.base + seg.row0 + i % kG.rows, qh);
    }
    i += gridDim.x * kMergeWaves;
    if (i < units) {
      seg = segment_of(i);
      mark = marks_of(seg, i);
    }
  }
}

// ---- host -------------------------------------------------------------------------
bool aligned(const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace

bool extend_sizes_ok(const Gemma4KvCacheConfig &c, int32_t batch, int32_t total_rows) {
  const bool geometry =
      (c.num_heads == 8 && c.head_dim == 256) || (c.num_heads == 1 && c.head_dim == 512);
  return geometry && batch > 0 && batch <= kExtendBatch && batch <= c.batch_size &&
         total_rows >= 0 && total_rows <= (1 << 24) && c.num_layers > 0 && c.num_pages > 0 &&
         c.page_size > 0 && c.max_pages_per_seq > 0 && c.window_size >= 0 &&
         (int64_t)c.num_pages * c.page_size <= 0x7fffffff;
}

hipError_t extend_attend(const ExtendCall &call, const ExtendPlanLayout &l, uint32_t magic,
                         int64_t shared_rows, hipStream_t stream) {
  const Gemma4KvCacheConfig &config = call.config;
  if (call.out == nullptr || call.q == nullptr || call.k == nullptr || call.v == nullptr ||
      call.cache_k == nullptr || call.cache_v == nullptr || call.page_table == nullptr ||
      call.plan == nullptr || call.workspace == nullptr || call.layer < 0 ||
      call.layer >= config.num_layers || !(call.softmax_scale > 0.0f) ||
      !isfinite(call.softmax_scale * kLog2e)) {
    return hipErrorInvalidValue;
  }
  const int64_t q_width = (int64_t)kQueryHeads * config.head_dim;
  const int64_t kv_width = (int64_t)config.num_heads * config.head_dim;
  const int64_t q_stride = call.q_stride == 0 ? q_width : call.q_stride;
  const int64_t kv_stride = call.kv_stride == 0 ? kv_width : call.kv_stride;
  const int64_t most = (int64_t)1 << 30;
  if (q_stride < q_width || kv_stride < kv_width || q_stride % kPackElems != 0 ||
      kv_stride % kPackElems != 0 || q_stride > most || kv_stride > most ||
      !aligned(call.out, 16) || !aligned(call.q, 16) || !aligned(call.k, 16) ||
      !aligned(call.v, 16) || !aligned(call.cache_k, 16) || !aligned(call.cache_v, 16) ||
      !aligned(call.plan, 256) || !aligned(call.workspace, 256) ||
      call.workspace_bytes < extend_workspace_bytes(l, config)) {
    return hipErrorInvalidValue;
  }
  ExtendParams p{};
  p.out = reinterpret_cast<uint16_t *>(call.out);
  p.q = reinterpret_cast<const uint16_t *>(call.q);
  p.k = reinterpret_cast<const uint16_t *>(call.k);
  p.v = reinterpret_cast<const uint16_t *>(call.v);
  p.cache_k = reinterpret_cast<const uint16_t *>(call.cache_k);
  p.cache_v = reinterpret_cast<const uint16_t *>(call.cache_v);
  p.page_table = call.page_table;
  p.plan = static_cast<const char *>(call.plan);
  p.shares = (int32_t)l.shares;
  p.segments = (int32_t)l.segments;
  p.merges = (int32_t)l.merges;
  p.max_merges = (int32_t)l.max_merges;
  p.max_segments = (int32_t)l.max_segments;
  p.c = config;
  p.page_div = make_fast_div(config.page_size);
  p.slot_div = make_fast_div(config.max_pages_per_seq);
  p.layer = call.layer;
  p.batch = call.batch;
  p.total_rows = call.total_rows;
  p.magic = magic;
  p.q_stride = q_stride;
  p.kv_stride = kv_stride;
  p.q_scale = call.softmax_scale * kLog2e;
  char *workspace = static_cast<char *>(call.workspace);
  p.partial = reinterpret_cast<float *>(workspace);
  p.stats = reinterpret_cast<float *>(workspace + extend_stats_offset(l, config.head_dim));
  p.odd = reinterpret_cast<uint32_t *>(workspace + extend_odd_offset(l, config.head_dim));
  p.rows = shared_rows;
  const uint32_t merge_grid = (uint32_t)std::min<int64_t>(
      kMergeGrid, std::max<int64_t>(l.max_merges, 1) * kQueryHeads * (config.head_dim / 256));
  const bool few = magic == kExtendFewMagic;
  few ? launch_extend_few(p, stream) : launch_extend_rows(p, stream);
  auto merge = [&](auto *kernel) {
    hipLaunchKernelGGL(kernel, dim3(merge_grid), dim3(kMergeThreads), 0, stream, p);
  };
  if (few) {
    config.num_heads == 1 ? merge(extend_merge_kernel<512, true, true>)
                          : merge(extend_merge_kernel<256, true, true>);
  } else if (magic == kExtendSharedMagic) {
    config.num_heads == 1 ? merge(extend_merge_kernel<512, true>)
                          : merge(extend_merge_kernel<256, true>);
  } else {
    config.num_heads == 1 ? merge(extend_merge_kernel<512, false>)
                          : merge(extend_merge_kernel<256, false>);
  }
  return hipGetLastError();
}

}  // namespace gemma4

using namespace gemma4;

extern "C" size_t gemma4_flash_attention_extend_plan_bytes(Gemma4KvCacheConfig config,
                                                           int32_t batch_size,
                                                           int32_t total_rows) {
  if (!extend_sizes_ok(config, batch_size, total_rows)) return 0;
  return (size_t)extend_layout(extend_geometry(config), batch_size, total_rows).bytes;
}

extern "C" size_t gemma4_flash_attention_extend_workspace_bytes(Gemma4KvCacheConfig config,
                                                                int32_t batch_size,
                                                                int32_t total_rows) {
  if (!extend_sizes_ok(config, batch_size, total_rows)) return 0;
  return extend_workspace_bytes(extend_layout(extend_geometry(config), batch_size, total_rows),
                                config);
}

extern "C" hipError_t gemma4_flash_attention_extend_plan(
    void *d_plan, size_t plan_bytes, const int32_t *d_row_offsets, const int32_t *d_prior_lengths,
    Gemma4KvCacheConfig config, int32_t batch_size, int32_t total_rows, int32_t window_size,
    int32_t sink_tokens, hipStream_t stream) {
  if (!extend_sizes_ok(config, batch_size, total_rows) || d_plan == nullptr || !aligned(d_plan, 256) ||
      d_row_offsets == nullptr || d_prior_lengths == nullptr || window_size < 0 ||
      sink_tokens < 0) {
    return hipErrorInvalidValue;
  }
  const int64_t capacity = (int64_t)config.max_pages_per_seq * config.page_size;
  if (config.window_size > 0 && (window_size < 1 || window_size > config.window_size ||
                                 window_size > capacity || sink_tokens > 0)) {
    return hipErrorInvalidValue;
  }
  const ExtendGeometry &g = extend_geometry(config);
  const ExtendPlanLayout l = extend_layout(g, batch_size, total_rows);
  if (plan_bytes < (size_t)l.bytes) return hipErrorInvalidValue;
  PlanParams p{};
  p.plan = static_cast<char *>(d_plan);
  p.shares = (int32_t)l.shares;
  p.segments = (int32_t)l.segments;
  p.merges = (int32_t)l.merges;
  p.row_offsets = d_row_offsets;
  p.prior_lengths = d_prior_lengths;
  p.g = g;
  p.batch = batch_size;
  p.total_rows = total_rows;
  p.window = window_size;
  p.sinks = sink_tokens;
  p.heads = config.num_heads;
  p.page_size = config.page_size;
  // A full-length cache holds no key past its table; a ring's positions only have
  // to stay below 2^31 with the new rows.
  p.max_prior = (int32_t)std::min<int64_t>(config.window_size > 0 ? 0x7fffffff : capacity,
                                           0x7fffffff - total_rows - 256);
  // A thread per row block, where that is so: barriers of four waves instead of 16 (one
  // token's plan 14.1 -> 10.4 us, 24 tokens' 17.5 -> 13.9).
  if (l.max_segments - g.shares <= 256) {
    hipLaunchKernelGGL(extend_plan_kernel<256>, dim3(1), dim3(256), 0, stream, p);
  } else {
    hipLaunchKernelGGL(extend_plan_kernel<1024>, dim3(1), dim3(1024), 0, stream, p);
  }
  return hipGetLastError();
}

extern "C" hipError_t gemma4_flash_attention_extend_paged_bf16(
    gemma4_bf16 *d_out, const gemma4_bf16 *d_q, const gemma4_bf16 *d_k, const gemma4_bf16 *d_v,
    const gemma4_bf16 *d_cache_k, const gemma4_bf16 *d_cache_v, const int32_t *d_page_table,
    const void *d_plan, size_t plan_bytes, Gemma4KvCacheConfig config, int32_t layer,
    int32_t batch_size, int32_t total_rows, int64_t q_stride, int64_t kv_stride,
    float softmax_scale, void *d_workspace, size_t workspace_bytes, hipStream_t stream) {
  if (total_rows == 0) return hipSuccess;
  if (!extend_sizes_ok(config, batch_size, total_rows)) return hipErrorInvalidValue;
  const ExtendPlanLayout l = extend_layout(extend_geometry(config), batch_size, total_rows);
  if (plan_bytes < (size_t)l.bytes) return hipErrorInvalidValue;
  return extend_attend({d_out, d_q, d_k, d_v, d_cache_k, d_cache_v, d_page_table, d_plan, config,
                        layer, batch_size, total_rows, q_stride, kv_stride, softmax_scale,
                        d_workspace, workspace_bytes},
                       l, kExtendMagic, 0, stream);
}
