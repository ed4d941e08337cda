// Pages of a pool: taking and returning them, branches of sequences (fork) and
// the closing up of kept tokens (compact), gfx950. No counterpart in the
// reference, whose page tables map a fixed page to every slot
// (src/gemma4_kv_cache.cu:108-122).
//
// State, all on the device: a page table [batch_size][max_pages_per_seq] (-1:
// unmapped) and refs[num_pages], the number of table entries that map a page (0:
// free). Free pages are given out lowest first, in table order, so the result does
// not depend on scheduling; a call that cannot be served whole changes nothing.
#include "gemma4_device.hpp"
#include "fast_div.hpp"

#include <algorithm>

namespace gemma4 {
namespace {

constexpr int kPoolThreads = 1024;
constexpr int kPoolWaves = kPoolThreads / kWave;
constexpr int kPoolUnroll = 4;                            // items per thread and round
constexpr int kPoolRound = kPoolThreads * kPoolUnroll;    // items per round
constexpr int kPoolBatch = 4096;                          // sequences at most
constexpr int kPoolList = 16384;                          // free pages held in LDS at a time

constexpr int kStatusOk = 0, kStatusPages = 1, kStatusArguments = 2, kStatusWritten = 3;

struct PoolParams {
  int32_t *page_table;
  int32_t *refs;
  Gemma4KvCacheConfig c;
  FastDiv page_div, slot_div;
};

// Logical pages [lo, hi) of one sequence as table slots: `count` of them from
// slot `first` on, around the ring's end (a full-length cache never wraps).
struct SlotRange {
  int32_t first, count;
  bool ok;
};
__device__ __forceinline__ SlotRange slot_range(const PoolParams &p, int32_t lo, int32_t hi) {
  const int32_t pages = p.c.max_pages_per_seq;
  SlotRange r{0, 0, true};
  if (hi <= lo) return r;
  if (p.c.window_size == 0) {
    r.ok = hi <= pages;
    r.first = min(lo, pages);
    r.count = min(hi, pages) - r.first;
  } else {
    r.first = (int32_t)fast_mod((uint32_t)lo, p.slot_div);
    r.count = min(hi - lo, pages);
  }
  return r;
}

// ---- release --------------------------------------------------------------
// One thread per table entry; what is read and written is a few kilobytes (64
// sequences of 512 pages: 128 KiB) and the launch is its time, 1.6 to 2.7 us.
__global__ __launch_bounds__(256) void release_pages_kernel(
    PoolParams p, const int32_t *__restrict__ first_position,
    const int32_t *__restrict__ end_position, int64_t entries) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= entries) return;
  const int32_t pages = p.c.max_pages_per_seq;
  const int32_t b = (int32_t)fast_div((uint32_t)i, p.slot_div);
  const int32_t slot = (int32_t)i - b * pages;
  const int32_t physical = p.page_table[i];
  const int32_t first = max(first_position[b], 0), end = max(end_position[b], 0);
  // Whole pages only: first rounded up, end down.
  int32_t lo = (int32_t)fast_div((uint32_t)first, p.page_div);
  if (lo * p.c.page_size != first) ++lo;
  const SlotRange r = slot_range(p, lo, (int32_t)fast_div((uint32_t)end, p.page_div));
  int32_t d = slot - r.first;
  if (d < 0) d += pages;
  if (d >= r.count || physical < 0) return;
  p.page_table[i] = -1;
  if (physical >= p.c.num_pages) return;
  // A count that is zero already stays zero.
  if (atomicSub(&p.refs[physical], 1) <= 0) atomicAdd(&p.refs[physical], 1);
}

// ---- ordered ranks over one workgroup ----------------------------------------
// Ranks of the true flags of one round in the order (u, thread): item u of
// thread t comes at u * kPoolThreads + t, so loads of a round are coalesced.
struct RankScratch {
  int32_t counts[kPoolUnroll * kPoolWaves];
};
__device__ __forceinline__ int32_t round_ranks(const bool (&flag)[kPoolUnroll],
                                               int32_t (&rank)[kPoolUnroll], RankScratch &s) {
  static_assert(kPoolUnroll * kPoolWaves == kWave, "one lane per (u, wave) count");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t votes[kPoolUnroll];
#pragma unroll
  for (int u = 0; u < kPoolUnroll; ++u) votes[u] = __ballot(flag[u]);
  if (lane == 0) {
#pragma unroll
    for (int u = 0; u < kPoolUnroll; ++u) s.counts[u * kPoolWaves + wave] = __popcll(votes[u]);
  }
  __syncthreads();
  const int32_t own = s.counts[lane];
  int32_t sum = own;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int32_t other = __shfl_up(sum, d);
    if (lane >= d) sum += other;
  }
  const int32_t total = __shfl(sum, kWave - 1);
#pragma unroll
  for (int u = 0; u < kPoolUnroll; ++u) {
    rank[u] = __shfl(sum - own, u * kPoolWaves + wave) +
              __popcll(votes[u] & ((1ull << lane) - 1));
  }
  __syncthreads();  // the counts may be written again
  return total;
}

// Counts of this thread's pages of a round; 1 behind the last page.
struct RefRound {
  int32_t refs[kPoolUnroll];
};
__device__ __forceinline__ RefRound load_refs(const PoolParams &p, uint32_t base) {
  RefRound r;
#pragma unroll
  for (int u = 0; u < kPoolUnroll; ++u) {
    const uint32_t page = base + u * kPoolThreads + threadIdx.x;
    r.refs[u] = page < (uint32_t)p.c.num_pages ? p.refs[page] : 1;
  }
  return r;
}

// Free pages with ranks [from, from + kPoolList) into `list`, in page order.
// Looks no further than to the one with rank wanted - 1; returns how many free
// pages it has seen. `next` holds the first round's counts.
__device__ __forceinline__ int32_t find_free(const PoolParams &p, int32_t from, int32_t wanted,
                                             RefRound next, int32_t *list, RankScratch &scratch) {
  int32_t seen = 0;
  for (uint32_t base = 0; base < (uint32_t)p.c.num_pages && seen < wanted; base += kPoolRound) {
    bool flag[kPoolUnroll];
    int32_t rank[kPoolUnroll];
#pragma unroll
    for (int u = 0; u < kPoolUnroll; ++u) flag[u] = next.refs[u] <= 0;
    next = load_refs(p, base + kPoolRound);
    const int32_t found = round_ranks(flag, rank, scratch);
#pragma unroll
    for (int u = 0; u < kPoolUnroll; ++u) {
      const int32_t at = seen + rank[u] - from;
      if (flag[u] && at >= 0 && at < kPoolList)
        list[at] = (int32_t)(base + u * kPoolThreads + threadIdx.x);
    }
    seen += found;
  }
  __syncthreads();
  return seen;
}

// ---- reserve ----------------------------------------------------------------
// One workgroup: the order of the pages handed out is the order of the entries.
// The entries of all ranges form one list (offsets by a prefix sum over the
// sequences), read twice: to count what is missing and shared, then to fill it. The
// chain of lengths, table, counts and table again is its time: 6.2 us for 5 sequences
// of which 2 change, 8.0 for 64 of 512 pages of which 10 do; 0.4 us of it for the
// counts of the mapped pages.
struct ReserveLds {
  int32_t offset[kPoolBatch + 1];  // of a sequence's entries in the list
  int32_t first[kPoolBatch];       // its first table slot
  bool written[kPoolBatch];        // its range begins behind position 0
  int32_t list[kPoolList];
  RankScratch scratch;
  int32_t bad;
  int32_t shared;
};
__global__ __launch_bounds__(kPoolThreads) void reserve_pages_kernel(
    PoolParams p, const int32_t *__restrict__ first_position,
    const int32_t *__restrict__ end_position, int32_t *__restrict__ status) {
  __shared__ ReserveLds lds;
  const int t = threadIdx.x, lane = t & 63;
  const int32_t batch = p.c.batch_size, pages = p.c.max_pages_per_seq;
  if (t == 0) lds.bad = lds.shared = 0;
  __syncthreads();
  for (int32_t b = t; b < batch; b += kPoolThreads) {
    const int32_t first = first_position[b], end = end_position[b];
    SlotRange r{0, 0, true};
    if (end > first) {
      if (first < 0) {
        r.ok = false;
      } else {
        const int32_t last = (int32_t)fast_div((uint32_t)(end - 1), p.page_div);
        r = slot_range(p, (int32_t)fast_div((uint32_t)first, p.page_div), last + 1);
      }
    }
    if (!r.ok) lds.bad = 1;
    lds.first[b] = r.first;
    lds.offset[b] = r.count;
    lds.written[b] = first > 0;
  }
  __syncthreads();
  if (lds.bad) {
    if (t == 0) *status = kStatusArguments;
    return;
  }
  // Exclusive prefix sum over the counts by the first wave. A table has fewer
  // than 2^31 entries (checked by the caller), so the sums fit.
  if (t < kWave) {
    int32_t carry = 0;
    for (int32_t b0 = 0; b0 < batch; b0 += kWave) {
      const int32_t own = b0 + lane < batch ? lds.offset[b0 + lane] : 0;
      int32_t sum = own;
#pragma unroll
      for (int d = 1; d < kWave; d <<= 1) {
        const int32_t other = __shfl_up(sum, d);
        if (lane >= d) sum += other;
      }
      if (b0 + lane < batch) lds.offset[b0 + lane] = carry + sum - own;
      carry += __shfl(sum, kWave - 1);
    }
    if (lane == 0) lds.offset[batch] = carry;
  }
  __syncthreads();
  const int32_t items = lds.offset[batch];
  // Table index of an item: its sequence is the last one that begins at or
  // before it.
  auto entry_of = [&](int32_t item, bool &written) -> int64_t {
    int32_t lo = 0, hi = batch;
    while (hi - lo > 1) {
      const int32_t mid = (lo + hi) >> 1;
      if (lds.offset[mid] <= item) lo = mid; else hi = mid;
    }
    int32_t slot = lds.first[lo] + (item - lds.offset[lo]);
    if (slot >= pages) slot -= pages;
    written = lds.written[lo];
    return (int64_t)lo * pages + slot;
  };
  // f(table index, rank) for every missing entry; returns how many there are. `held`
  // (page) is whether a page that a range's rows will be written to is another's too.
  auto for_missing = [&](auto &&f, auto &&held) -> int32_t {
    int32_t missing = 0;
    bool shared = false;
    for (uint32_t base = 0; base < (uint32_t)items; base += kPoolRound) {
      int64_t at[kPoolUnroll];
      int32_t page[kPoolUnroll];
      bool flag[kPoolUnroll], written[kPoolUnroll];
      int32_t rank[kPoolUnroll];
#pragma unroll
      for (int u = 0; u < kPoolUnroll; ++u) {
        const uint32_t item = base + u * kPoolThreads + t;
        written[u] = false;
        at[u] = item < (uint32_t)items ? entry_of((int32_t)item, written[u]) : -1;
        page[u] = at[u] >= 0 ? p.page_table[at[u]] : 0;
      }
#pragma unroll
      for (int u = 0; u < kPoolUnroll; ++u) {
        flag[u] = page[u] < 0;
        if (written[u] && page[u] >= 0 && page[u] < p.c.num_pages) shared |= held(page[u]);
      }
      const int32_t found = round_ranks(flag, rank, lds.scratch);
#pragma unroll
      for (int u = 0; u < kPoolUnroll; ++u)
        if (flag[u]) f(at[u], missing + rank[u]);
      missing += found;
    }
    if (shared) lds.shared = 1;
    return missing;
  };
  const int32_t wanted =
      for_missing([](int64_t, int32_t) {}, [&](int32_t page) { return p.refs[page] > 1; });
  const int32_t seen = find_free(p, 0, wanted, load_refs(p, 0), lds.list, lds.scratch);
  if (lds.shared || seen < wanted) {  // find_free ends with a barrier
    if (t == 0) *status = lds.shared ? kStatusWritten : kStatusPages;
    return;
  }
  if (t == 0) *status = kStatusOk;
  // A window of the list at a time. What an earlier window filled is no longer
  // missing: the ranks of what is left start at the window's own first.
  for (int32_t from = 0; from < wanted; from += kPoolList) {
    if (from > 0) find_free(p, 0, wanted - from, load_refs(p, 0), lds.list, lds.scratch);
    for_missing([&](int64_t at, int32_t rank) {
      if (rank >= kPoolList) return;
      const int32_t page = lds.list[rank];
      p.page_table[at] = page;
      p.refs[page] = 1;
    }, [](int32_t) { return false; });
    __threadfence_block();
    __syncthreads();
  }
}

// ---- fork -------------------------------------------------------------------
struct ForkParams {
  PoolParams pool;
  int32_t *seq_lengths;
  const int32_t *parents;
  const int32_t *children;
  int32_t count;
  int32_t *status;
};
// What a branch gets in place of a parent's page.
enum class Share { kNone, kSame, kCopy };
__device__ __forceinline__ Share fork_share(const PoolParams &p, int32_t length, int32_t slot,
                                            int32_t physical) {
  if (physical < 0 || physical >= p.c.num_pages) return Share::kNone;
  if (p.c.window_size > 0) return Share::kCopy;  // any ring page will be written again
  const int32_t whole = (int32_t)fast_div((uint32_t)length, p.page_div);
  if (slot < whole) return Share::kSame;
  return slot == whole && length > whole * p.c.page_size ? Share::kCopy : Share::kNone;
}

// Slots of a branch that may need a page of its own: all of a ring's, the begun page's
// of a full-length cache.
__device__ __forceinline__ int32_t fork_slot(const PoolParams &p, int32_t length, int32_t i) {
  return p.c.window_size > 0 ? i : (int32_t)fast_div((uint32_t)length, p.page_div);
}

// One workgroup checks the request, hands out the pages of what is copied and tells
// in `status` whether the launch behind it copies and shares: the way is a chain of
// dependent loads (requests, lengths, table, counts), which is the time. What is
// known early is asked for early and a branch's parent, child and length are kept in
// LDS (18 branches of a 1 x 512 cache, tables of 129 pages: 12.1 -> 6.0 us).
struct ForkLds {
  int32_t role[kPoolBatch];  // bit 0: a parent, bit 1: a child
  int32_t parent[kPoolBatch], child[kPoolBatch], length[kPoolBatch];  // of a branch
  int32_t list[kPoolList];
  RankScratch scratch;
  int32_t bad;
};
__global__ __launch_bounds__(kPoolThreads) void fork_tables_kernel(ForkParams f, int32_t slots,
                                                                   FastDiv by_slots) {
  __shared__ ForkLds lds;
  const PoolParams &p = f.pool;
  const int t = threadIdx.x;
  const int32_t batch = p.c.batch_size, pages = p.c.max_pages_per_seq;
  const RefRound ahead = load_refs(p, 0);
  for (int32_t b = t; b < batch; b += kPoolThreads) lds.role[b] = 0;
  if (t == 0) lds.bad = 0;
  __syncthreads();
  for (int32_t r = t; r < f.count; r += kPoolThreads) {
    const int32_t parent = f.parents[r], child = f.children[r];
    bool ok = parent >= 0 && parent < batch && child >= 0 && child < batch;
    if (ok) {
      const int32_t length = f.seq_lengths[parent];
      lds.parent[r] = parent;
      lds.child[r] = child;
      lds.length[r] = length;
      ok = length >= 0 && (p.c.window_size > 0 || length <= (int64_t)pages * p.c.page_size);
      atomicOr(&lds.role[parent], 1);
      if (atomicOr(&lds.role[child], 2) & 2) ok = false;  // a child of two
    }
    if (!ok) lds.bad = 1;
  }
  __syncthreads();
  for (int32_t b = t; b < batch; b += kPoolThreads)
    if (lds.role[b] == 3) lds.bad = 1;
  __syncthreads();
  if (lds.bad) {
    if (t == 0) *f.status = kStatusArguments;
    return;
  }
  // Entry i of branch r, of those that may be copied, at r * slots + i of a list.
  const uint32_t items = (uint32_t)(f.count * slots);
  struct Round {
    int64_t to[kPoolUnroll];      // child's table entry
    int32_t rank[kPoolUnroll];
    bool copy[kPoolUnroll];
  };
  auto load_round = [&](uint32_t base, Round &e) -> int32_t {
    int32_t physical[kPoolUnroll];
    int32_t slot[kPoolUnroll], length[kPoolUnroll];
#pragma unroll
    for (int u = 0; u < kPoolUnroll; ++u) {
      const uint32_t item = base + u * kPoolThreads + t;
      e.to[u] = -1;
      physical[u] = -1;
      if (item < items) {
        const int32_t r = (int32_t)fast_div(item, by_slots);
        length[u] = lds.length[r];
        slot[u] = fork_slot(p, length[u], (int32_t)item - r * slots);
        if (slot[u] < pages) {
          e.to[u] = (int64_t)lds.child[r] * pages + slot[u];
          physical[u] = p.page_table[(int64_t)lds.parent[r] * pages + slot[u]];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kPoolUnroll; ++u)
      e.copy[u] = e.to[u] >= 0 && fork_share(p, length[u], slot[u], physical[u]) == Share::kCopy;
    return round_ranks(e.copy, e.rank, lds.scratch);
  };
  Round first;
  int32_t wanted = load_round(0, first);
  for (uint32_t base = kPoolRound; base < items; base += kPoolRound) {
    Round e;
    wanted += load_round(base, e);
  }
  // A child holds nothing yet.
  const uint32_t entries = (uint32_t)(f.count * pages);
  bool held = false;
  for (uint32_t base = 0; base < entries; base += kPoolRound) {
#pragma unroll
    for (int u = 0; u < kPoolUnroll; ++u) {
      const uint32_t entry = base + u * kPoolThreads + t;
      if (entry >= entries) continue;
      const int32_t r = (int32_t)fast_div(entry, p.slot_div);
      held |= p.page_table[(int64_t)lds.child[r] * pages + ((int32_t)entry - r * pages)] >= 0;
    }
  }
  if (held) lds.bad = 1;
  const int32_t seen = find_free(p, 0, wanted, ahead, lds.list, lds.scratch);
  if (lds.bad || seen < wanted) {
    if (t == 0) *f.status = lds.bad ? kStatusArguments : kStatusPages;
    return;
  }
  // A page handed out is free no more, so the list of the next window starts with its
  // own first page.
  for (int32_t from = 0; from < wanted; from += kPoolList) {
    if (from > 0) find_free(p, 0, wanted - from, load_refs(p, 0), lds.list, lds.scratch);
    int32_t copies = 0;
    for (uint32_t base = 0; base < items; base += kPoolRound) {
      Round e = first;
      int32_t found = 0;
      if (items > kPoolRound) found = load_round(base, e);
#pragma unroll
      for (int u = 0; u < kPoolUnroll; ++u) {
        const int32_t rank = copies + e.rank[u] - from;
        if (!e.copy[u] || rank < 0 || rank >= kPoolList) continue;
        const int32_t page = lds.list[rank];
        p.page_table[e.to[u]] = page;
        p.refs[page] = 1;
      }
      copies += found;
    }
    __threadfence_block();
    __syncthreads();
  }
  for (int32_t r = t; r < f.count; r += kPoolThreads) f.seq_lengths[lds.child[r]] = lds.length[r];
  if (t == 0) *f.status = kStatusOk;
}

constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 8;
constexpr int kCopyPacks = kCopyThreads * kCopyUnroll;  // 16-byte packs per workgroup

// Workgroup (piece of a page, copied page of a branch, layer x {K, V}): the
// branch's table says where to, what the parent's length leaves in a begun page
// how much. All loads of a piece are in flight before its first store. In a
// full-length cache the first layer's workgroups of a branch also share its
// parent's whole pages. A ring of 1024 tokens in 40 layers of 8 x 256 (713 MB read and
// written): 139 us, 5.1 TB/s, the rate of a large copy; a branch's begun pages are
// few bytes and the launch is their time (18 of 1 x 512: 6.4 us).
__global__ __launch_bounds__(kCopyThreads) void fork_copy_kernel(ForkParams f, uint16_t *cache_k,
                                                                 uint16_t *cache_v, int32_t pieces,
                                                                 int32_t slots) {
  if (*f.status != kStatusOk) return;
  const PoolParams &p = f.pool;
  const int32_t pages = p.c.max_pages_per_seq;
  const int32_t piece = blockIdx.x % pieces, which = blockIdx.x / pieces;
  const int32_t r = which / slots;
  const int32_t parent = f.parents[r], child = f.children[r];
  const int32_t length = f.seq_lengths[parent];
  const int32_t slot = fork_slot(p, length, which - r * slots);
  int32_t rows = p.c.page_size;
  if (p.c.window_size == 0) {
    if (blockIdx.y == 0) {
      for (int32_t s = piece * kCopyThreads + threadIdx.x; s < slot; s += pieces * kCopyThreads) {
        const int32_t physical = p.page_table[(int64_t)parent * pages + s];
        if (fork_share(p, length, s, physical) != Share::kSame) continue;
        p.page_table[(int64_t)child * pages + s] = physical;
        atomicAdd(&p.refs[physical], 1);
      }
    }
    rows = length - slot * p.c.page_size;
    if (rows == 0) return;
  }
  const int32_t from = p.page_table[(int64_t)parent * pages + slot];
  const int32_t to = p.page_table[(int64_t)child * pages + slot];
  if (fork_share(p, length, slot, from) != Share::kCopy || to < 0) return;
  const int64_t row_packs = (int64_t)p.c.num_heads * p.c.head_dim / kPackElems;
  const int64_t packs = rows * row_packs, page_packs = p.c.page_size * row_packs;
  const int64_t layer = (int64_t)(blockIdx.y >> 1) * p.c.num_pages;
  uint16_t *cache = blockIdx.y & 1 ? cache_v : cache_k;
  const uint16_t *src = cache + (layer + from) * page_packs * kPackElems;
  uint16_t *dst = cache + (layer + to) * page_packs * kPackElems;
  const int64_t first = (int64_t)piece * kCopyPacks + threadIdx.x;
  uint4 x[kCopyUnroll];
#pragma unroll
  for (int u = 0; u < kCopyUnroll; ++u) {
    const int64_t i = first + u * kCopyThreads;
    if (i < packs) x[u] = load128(src + i * kPackElems);
  }
#pragma unroll
  for (int u = 0; u < kCopyUnroll; ++u) {
    const int64_t i = first + u * kCopyThreads;
    if (i < packs) store128(dst + i * kPackElems, x[u]);
  }
}

// ---- compact ------------------------------------------------------------------
struct CompactParams {
  uint16_t *cache_k;
  uint16_t *cache_v;
  Gemma4KvCacheConfig c;
  FastDiv page_div, slot_div;
  const int32_t *page_table;
  const int32_t *refs;  // null: no page is shared
  const int32_t *sequences;
  const int32_t *first;
  const int32_t *offsets;
  const int32_t *positions;
  int32_t count, total;
  int32_t slices;  // parts of a row, one workgroup each
  int32_t *status;
};
constexpr int kCompactThreads = 1024;
constexpr int kCompactList = 4096;   // rows whose places LDS holds at a time
constexpr int kCompactUnroll = 4;
constexpr int kCompactGroups = 256;  // workgroups that run at once, one per CU
// A request that breaks several rules gets the lowest of their codes.
constexpr int kStatusList = 1, kStatusUnmapped = 2, kStatusShared = 3, kStatusNone = 4;

// Workgroup (request, slice of a row, layer x {K, V}). Kept token j moves from
// position kept[j] to first + j <= kept[j], in place. Rows are taken in order,
// a batch at a time: every load of a batch has arrived before its first store,
// and a later batch's sources lie behind everything that was stored before
// (kept[j] > kept[i] >= first + i for j > i), so nothing is overwritten unread and
// the next batch's loads go out ahead of the stores. Four requests that keep 3001
// rows each in 8 layers of 1 x 512 (393 MB): 92 us, 4.3 TB/s of 4.9 for a large copy,
// the rest being the wait of a batch for its last load; 7 of 32 drafts of 8 sequences
// in 10 layers of 8 x 256: 5.9 us, the chain of list, table, row and store.
__global__ __launch_bounds__(kCompactThreads) void compact_kernel(CompactParams p) {
  __shared__ int32_t s_src[kCompactList], s_dst[kCompactList];
  __shared__ int32_t s_error;
  const int t = threadIdx.x;
  const int32_t i = blockIdx.x / p.slices, slice = blockIdx.x - i * p.slices;
  const int32_t pages = p.c.max_pages_per_seq;
  const int32_t b = p.sequences[i], first = p.first[i];
  const int32_t begin = p.offsets[i], end = p.offsets[i + 1];
  const int64_t capacity = (int64_t)pages * p.c.page_size;
  const int32_t n = end - begin;
  if (t == 0)
    s_error = b >= 0 && b < p.c.batch_size && first >= 0 && begin >= 0 && end >= begin &&
                      end <= p.total && first <= 0x7fffffff - n
                  ? kStatusNone : kStatusList;
  __syncthreads();
  int32_t error = s_error;
  const bool readable = error == kStatusNone;
  __syncthreads();  // every wave has read it before any adds what it finds
  // One request per sequence.
  if (readable) {
    for (int32_t j = t; j < p.count; j += kCompactThreads)
      if (j != i && p.sequences[j] == b) error = kStatusList;
  }
  const int32_t *table = p.page_table + (int64_t)b * pages;
  const int32_t *kept = p.positions + begin;
  // Row of the layer at a position, -1 where no page is mapped.
  auto row_of = [&](int32_t position, int32_t &page) -> int64_t {
    const uint32_t logical = fast_div((uint32_t)position, p.page_div);
    const uint32_t slot = p.c.window_size > 0 ? fast_mod(logical, p.slot_div) : logical;
    page = table[slot];
    if (page < 0 || page >= p.c.num_pages) return -1;
    return (int64_t)page * p.c.page_size + (position - (int32_t)logical * p.c.page_size);
  };
  if (readable) {
    for (int32_t j = t; j < n; j += kCompactThreads) {
      const int32_t from = kept[j], to = first + j;
      if (from < to || (j > 0 && kept[j - 1] >= from) ||
          (p.c.window_size > 0 ? from - first >= capacity : from >= capacity)) {
        error = kStatusList;
        continue;
      }
      int32_t src_page, dst_page;
      const int64_t src = row_of(from, src_page), dst = row_of(to, dst_page);
      if (src < 0 || dst < 0) {
        error = min(error, kStatusUnmapped);
      } else if (from != to && p.refs != nullptr && p.refs[dst_page] > 1) {
        error = min(error, kStatusShared);
      }
      if (j < kCompactList) {
        s_src[j] = (int32_t)src;
        s_dst[j] = from == to ? -1 : (int32_t)dst;
      }
    }
  }
  if (error != kStatusNone) atomicMin(&s_error, error);
  __syncthreads();
  error = s_error;
  if (t == 0 && slice == 0 && blockIdx.y == 0) p.status[i] = error == kStatusNone ? kStatusOk : error;
  if (error != kStatusNone) return;

  const int32_t row_packs = p.c.num_heads * p.c.head_dim / kPackElems;
  const int32_t c0 = (int32_t)((int64_t)row_packs * slice / p.slices);
  const int32_t width = (int32_t)((int64_t)row_packs * (slice + 1) / p.slices) - c0;
  uint16_t *cache = (blockIdx.y & 1 ? p.cache_v : p.cache_k) +
                    ((int64_t)(blockIdx.y >> 1) * p.c.num_pages * p.c.page_size * row_packs + c0) *
                        kPackElems;
  // Thread t: pack t % width of rows t / width + k * stride.
  const int32_t stride = kCompactThreads / width;
  const int32_t my_row = t / width, my_pack = t - my_row * width;
  const bool idle = my_row >= stride;
  for (int32_t base = 0; base < n; base += kCompactList) {
    const int32_t rows = min(n - base, kCompactList);
    if (base > 0) {
      __syncthreads();
      for (int32_t j = t; j < rows; j += kCompactThreads) {
        int32_t page;
        s_src[j] = (int32_t)row_of(kept[base + j], page);
        s_dst[j] = kept[base + j] == first + base + j ? -1 : (int32_t)row_of(first + base + j, page);
      }
      __syncthreads();
    }
    const int32_t step = stride * kCompactUnroll;
    uint4 x[kCompactUnroll], next[kCompactUnroll];
    auto load = [&](int32_t at, uint4 (&v)[kCompactUnroll]) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < kCompactUnroll; ++u) {
        const int32_t j = at + u * stride + my_row;
        if (!idle && j < rows && s_dst[j] >= 0)
          v[u] = load128(cache + ((int64_t)s_src[j] * row_packs + my_pack) * kPackElems);
      }
    };
    load(0, x);
    for (int32_t at = 0; at < rows; at += step) {
      load(at + step, next);
      // Every thread's loads of this batch (and the next) have arrived.
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
      __syncthreads();
#pragma unroll
      for (int u = 0; u < kCompactUnroll; ++u) {
        const int32_t j = at + u * stride + my_row;
        if (!idle && j < rows && s_dst[j] >= 0)
          store128(cache + ((int64_t)s_dst[j] * row_packs + my_pack) * kPackElems, x[u]);
        x[u] = next[u];
      }
    }
    // The next list's sources lie behind what was stored: no wait for the stores.
  }
}

// ---- host -------------------------------------------------------------------
bool valid_pool(const Gemma4KvCacheConfig &c) {
  return c.num_pages > 0 && c.page_size > 0 && c.max_pages_per_seq > 0 && c.batch_size > 0 &&
         c.batch_size <= kPoolBatch && c.window_size >= 0 &&
         (int64_t)c.batch_size * c.max_pages_per_seq <= 0x7fffffff &&
         (int64_t)c.num_pages * c.page_size <= 0x7fffffff;
}
bool valid_rows(const Gemma4KvCacheConfig &c) {
  return c.num_layers > 0 && c.num_layers <= 32767 && c.num_heads > 0 && c.head_dim > 0 &&
         c.head_dim % kPackElems == 0 && (int64_t)c.num_heads * c.head_dim <= (1 << 20);
}
bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
PoolParams pool_params(int32_t *page_table, int32_t *refs, const Gemma4KvCacheConfig &c) {
  return {page_table, refs, c, make_fast_div(c.page_size), make_fast_div(c.max_pages_per_seq)};
}

}  // namespace
}  // namespace gemma4

using namespace gemma4;

extern "C" {

hipError_t gemma4_kv_cache_release_pages(int32_t *d_page_table, int32_t *d_page_refs,
                                         Gemma4KvCacheConfig config,
                                         const int32_t *d_first_position,
                                         const int32_t *d_end_position, hipStream_t stream) {
  if (!valid_pool(config) || d_page_table == nullptr || d_page_refs == nullptr ||
      d_first_position == nullptr || d_end_position == nullptr) {
    return hipErrorInvalidValue;
  }
  const int64_t entries = (int64_t)config.batch_size * config.max_pages_per_seq;
  hipLaunchKernelGGL(release_pages_kernel, dim3((uint32_t)((entries + 255) / 256)), dim3(256), 0,
                     stream, pool_params(d_page_table, d_page_refs, config), d_first_position,
                     d_end_position, entries);
  return hipGetLastError();
}

hipError_t gemma4_kv_cache_reserve_pages(int32_t *d_page_table, int32_t *d_page_refs,
                                         Gemma4KvCacheConfig config,
                                         const int32_t *d_first_position,
                                         const int32_t *d_end_position, int32_t *d_status,
                                         hipStream_t stream) {
  if (!valid_pool(config) || d_page_table == nullptr || d_page_refs == nullptr ||
      d_first_position == nullptr || d_end_position == nullptr || d_status == nullptr) {
    return hipErrorInvalidValue;
  }
  hipLaunchKernelGGL(reserve_pages_kernel, dim3(1), dim3(kPoolThreads), 0, stream,
                     pool_params(d_page_table, d_page_refs, config), d_first_position,
                     d_end_position, d_status);
  return hipGetLastError();
}

hipError_t gemma4_kv_cache_fork_bf16(gemma4_bf16 *d_cache_k, gemma4_bf16 *d_cache_v,
                                     Gemma4KvCacheConfig config, int32_t *d_page_table,
                                     int32_t *d_page_refs, int32_t *d_seq_lengths,
                                     const int32_t *d_parents, const int32_t *d_children,
                                     int32_t fork_count, int32_t *d_status, hipStream_t stream) {
  if (fork_count == 0) return hipSuccess;
  if (fork_count < 0 || !valid_pool(config) || !valid_rows(config) ||
      fork_count > config.batch_size || d_cache_k == nullptr || d_cache_v == nullptr ||
      !aligned16(d_cache_k) || !aligned16(d_cache_v) || d_page_table == nullptr ||
      d_page_refs == nullptr || d_seq_lengths == nullptr || d_parents == nullptr ||
      d_children == nullptr || d_status == nullptr) {
    return hipErrorInvalidValue;
  }
  const ForkParams f = {pool_params(d_page_table, d_page_refs, config), d_seq_lengths, d_parents,
                        d_children, fork_count, d_status};
  const int64_t page_packs =
      (int64_t)config.page_size * config.num_heads * config.head_dim / kPackElems;
  const int32_t slots = config.window_size > 0 ? config.max_pages_per_seq : 1;
  const int64_t pieces = (page_packs + kCopyPacks - 1) / kCopyPacks;
  const int64_t blocks = pieces * slots * fork_count;
  // A launch holds fewer than 2^32 threads in a grid dimension. One that is refused
  // behind the tables' would leave children that map pages without their rows.
  if (blocks * kCopyThreads > 0xffffffffll) return hipErrorInvalidValue;
  hipLaunchKernelGGL(fork_tables_kernel, dim3(1), dim3(kPoolThreads), 0, stream, f, slots,
                     make_fast_div(slots));
  hipLaunchKernelGGL(fork_copy_kernel, dim3((uint32_t)blocks, 2 * config.num_layers),
                     dim3(kCopyThreads), 0, stream, f, reinterpret_cast<uint16_t *>(d_cache_k),
                     reinterpret_cast<uint16_t *>(d_cache_v), (int32_t)pieces, slots);
  return hipGetLastError();
}

hipError_t gemma4_kv_cache_compact_bf16(gemma4_bf16 *d_cache_k, gemma4_bf16 *d_cache_v,
                                        Gemma4KvCacheConfig config, const int32_t *d_page_table,
                                        const int32_t *d_page_refs, const int32_t *d_sequences,
                                        const int32_t *d_first_positions,
                                        const int32_t *d_kept_offsets,
                                        const int32_t *d_kept_positions, int32_t sequence_count,
                                        int32_t total_kept, int32_t *d_status,
                                        hipStream_t stream) {
  if (sequence_count == 0) return hipSuccess;
  if (sequence_count < 0 || total_kept < 0 || !valid_pool(config) || !valid_rows(config) ||
      sequence_count > config.batch_size || d_cache_k == nullptr || d_cache_v == nullptr ||
      !aligned16(d_cache_k) || !aligned16(d_cache_v) || d_page_table == nullptr ||
      d_sequences == nullptr || d_first_positions == nullptr || d_kept_offsets == nullptr ||
      (d_kept_positions == nullptr && total_kept > 0) || d_status == nullptr) {
    return hipErrorInvalidValue;
  }
  const int32_t row_packs = config.num_heads * (config.head_dim / kPackElems);
  // Slices of 256 bytes or more, at most a workgroup's width, as long as every
  // workgroup has a CU to itself: 1024 threads of 76 registers leave no room for a
  // second one, and a further round is the whole chain again. 8 sequences of 10 layers
  // of 8 x 256, 7 rows each: 5.9 us in 160 workgroups, 8.3 in 320, 11.1 in 640; 3001
  // rows each: 792 us, 905 and 801; 4 of 5 layers, 3001 rows each: 201 us in 160, 229
  // in 320, 220 in 640.
  const int64_t wide = (int64_t)sequence_count * 2 * config.num_layers;
  int32_t slices = (row_packs + kCompactThreads - 1) / kCompactThreads;
  while (row_packs / (2 * slices) >= 16 && wide * slices * 2 <= kCompactGroups) slices *= 2;
  const CompactParams p = {reinterpret_cast<uint16_t *>(d_cache_k),
                           reinterpret_cast<uint16_t *>(d_cache_v),
                           config,
                           make_fast_div(config.page_size),
                           make_fast_div(config.max_pages_per_seq),
                           d_page_table,
                           d_page_refs,
                           d_sequences,
                           d_first_positions,
                           d_kept_offsets,
                           d_kept_positions,
                           sequence_count,
                           total_kept,
                           slices,
                           d_status};
  hipLaunchKernelGGL(compact_kernel, dim3((uint32_t)(sequence_count * slices), 2 * config.num_layers),
                     dim3(kCompactThreads), 0, stream, p);
  return hipGetLastError();
}

}  // extern "C"
