// The rows of a ragged extension batch on bf16 MFMA, gfx950: one share of the
// plan's segments per workgroup.
//
// Formulation: S^T = K Q^T and O^T = V^T P^T with v_mfma_f32_32x32x16_bf16 on
// blocks of 32 keys. A wave owns 32 columns: (row, query head) pairs of the KV
// head, 16 rows x 2 heads at 8 x 256, 2 rows x 16 heads at 1 x 512, so that either
// geometry keeps a full MFMA and a workgroup of four waves reads every key once
// for 128 columns. In the accumulator lane l holds column l % 32 and 16 of a
// block's keys (or dims): a column's maximum needs one exchange (lane ^ 32), the
// rescale is a per-lane factor, and P^T is the second product's operand as it
// stands, its key order {4h .. 4h+3, 8+4h .. 8+4h+3} per 16 keys being the order in
// which V^T is read (ds_read_b64_tr_b16).
//
// Keys stream in tiles of 32 through LDS stages (four of 16 KiB each of K and V at
// 8 x 256, two of 32 KiB at 1 x 512), copied by the waves themselves
// (global_load_lds) from addresses their lanes resolved an iteration earlier: a
// page-table entry per key, any page size, the packed new rows behind the cached
// ones. Keys that no row of the block sees, that no page maps, or past the
// segment's tiles are copied from a row of zeros, so nothing in such a place is
// ever multiplied. Rows land swizzled by 16-byte chunks (K row k, chunk c at c ^ (k
// & 15); V at c ^ ((k & 3) << 2)), which keeps the operand reads free of bank
// conflicts.
//
// With one wave per SIMD nothing else fills the matrix cores while a wave does its
// softmax, so iteration t interleaves the softmax of tile t with the second
// product of tile t - 1. Registers: at 1 x 512 the accumulators are all 256 AGPRs
// (the second product is asm, the first one's results stay in VGPRs by a build flag
// for this file), Q^T half of the VGPRs.
#include "extend_common.hpp"
#include "extend_rows.hpp"
#include "lds_copy.hpp"

#include <math.h>

#include <type_traits>

namespace gemma4 {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr float kRescaleSlack = 8.0f;  // log2 headroom of the running maximum

// What masked places are copied from: as long as the longest row.
__device__ uint4 g_zero_row[64];

constexpr int kTile = 32;              // keys per LDS stage: one MFMA block
constexpr int kCopyKeys = kTile / kWaves;  // keys a wave copies

constexpr int kRunTiles = kWave / kCopyKeys;  // tiles whose keys a wave resolves at once

template <int kDim>
struct Shape {
  static constexpr int kHeads = kDim == 256 ? 8 : 1;
  static constexpr int kGroup = kQueryHeads / kHeads;   // query heads of a KV head
  static constexpr int kWaveRows = 32 / kGroup;         // rows of a wave's columns
  static constexpr int kRows = kWaves * kWaveRows;      // rows of a row block
  static constexpr int kRowBytes = kDim * 2;
  static constexpr int kStages = kDim == 256 ? 4 : 2;
  static constexpr int kSteps = kDim / 16;              // of S^T
  static constexpr int kDims = kDim / 32;               // 32-dim blocks of O^T
  static constexpr int kCopies = kCopyKeys * kRowBytes / 1024;  // of K, and of V
  static constexpr int kTokenBytes = kHeads * kRowBytes;        // a cached token's rows
  static constexpr int kWindow = kDim == 256 ? 16 : 8;  // K fragments read ahead
};
static_assert(Shape<256>::kRows == kExtend256.rows && kTile == kExtend256.tile);
static_assert(Shape<512>::kRows == kExtend512.rows && kTile == kExtend512.tile);

template <int kBegin, int kEnd, class F>
__device__ __forceinline__ void static_for(F &&f) {
  if constexpr (kBegin < kEnd) {
    f(std::integral_constant<int, kBegin>{});
    static_for<kBegin + 1, kEnd>(f);
  }
}

typedef unsigned u32x4v_t __attribute__((ext_vector_type(4)));

// acc += V^T P^T with the accumulators in AGPRs. The wait states cover operands
// that a VALU instruction wrote right before (the compiler does not see into asm).
__device__ __forceinline__ void mfma_pv(f32x16_t &acc, u32x4v_t v, u32x4v_t p) {
  asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(v), "v"(p));
}
// Every product above has written its accumulators (16 passes and the write).
template <int kCount>
__device__ __forceinline__ void mfma_pv_done(f32x16_t (&acc)[kCount]) {
#pragma unroll
  for (int d = 0; d < kCount; d += 8) {
    asm volatile("s_nop 15\n\ts_nop 7"
                 : "+a"(acc[d]), "+a"(acc[d + 1]), "+a"(acc[d + 2]), "+a"(acc[d + 3]),
                   "+a"(acc[d + 4]), "+a"(acc[d + 5]), "+a"(acc[d + 6]), "+a"(acc[d + 7]));
  }
}

typedef __attribute__((address_space(3))) const u32x4v_t lds_u32x4;
typedef __attribute__((address_space(3))) i16x4_t lds_i16x4;
__device__ __forceinline__ u32x4v_t lds_read128(uint32_t at) {
  return *reinterpret_cast<lds_u32x4 *>(at);
}
__device__ __forceinline__ uint2 lds_read_tr(uint32_t at) {
  return __builtin_bit_cast(
      uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_i16x4 *>(at)));
}

// By value: a ternary of captured variables would be a choice of addresses, and
// keep them in memory.
__device__ __forceinline__ uint64_t pick(bool c, uint64_t a, uint64_t b) { return c ? a : b; }

// The lane, worked out anew where it is asked for: what follows from it need not
// be held in a register from the kernel's start (at 1 x 512 none is left).
__device__ __forceinline__ int fresh_lane() {
  int lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0));
  asm volatile("" : "+v"(lane));
  return lane;
}

template <int kDim>
__global__ __launch_bounds__(kThreads, 1) void extend_rows_kernel(ExtendParams p) {
  using G = Shape<kDim>;
  constexpr int kStages = G::kStages, kStageBytes = kTile * G::kRowBytes;
  struct Lds {
    uint4 k[kStages][kStageBytes / 16];
    uint4 v[kStages][kStageBytes / 16];
    // Of the current and the next run of kRunTiles tiles, by parity: the addresses
    // of the keys that a wave copies, and which keys can be read.
    uint64_t k_rows[2][kWaves][kWave];
    uint64_t v_rows[2][kWaves][kWave];
    uint8_t valid[2][kRunTiles][kWaves];  // bit j: key kCopyKeys w + j of the tile
    int32_t pages[kWaves][kWave];         // the next run's page-table entries
  };
  __shared__ __attribute__((aligned(1024))) Lds lds;

  const int t = threadIdx.x, lane = t & 63;
  const int wave = wave_uniform(t >> 6);
  const int half = lane >> 5, n = lane & 31;
  const int head = blockIdx.x % G::kHeads, share = blockIdx.x / G::kHeads;

  const auto *header = reinterpret_cast<const ExtendHeader *>(p.plan);
  const auto *share_first = reinterpret_cast<const int32_t *>(p.plan + p.share_first);
  const auto *segments = reinterpret_cast<const ExtendSegment *>(p.plan + p.segments);
  const int32_t segment_end = share_first[share + 1];
  int32_t segment = share_first[share];
  const int32_t window = header->window, sinks = header->sinks;
  if (!extend_plan_fits(p)) return;

  const bool ring = p.c.window_size > 0;
  const int32_t max_pages = p.c.max_pages_per_seq;
  const uint64_t layer_bytes =
      (uint64_t)p.layer * p.c.num_pages * p.c.page_size * G::kTokenBytes + head * G::kRowBytes;
  const uint64_t cache_k = reinterpret_cast<uint64_t>(p.cache_k) + layer_bytes;
  const uint64_t cache_v = reinterpret_cast<uint64_t>(p.cache_v) + layer_bytes;
  const uint64_t zero_row = reinterpret_cast<uint64_t>(&g_zero_row[0]);
  const uint32_t kv_bytes = (uint32_t)(p.kv_stride * 2);

  // Row of column n among the workgroup's, and its query head.
  auto column_row = [&](int column) __attribute__((always_inline)) {
    return G::kWaveRows * wave + (G::kGroup == 2 ? column % 16 : column / 16);
  };
  auto column_head = [&](int column) __attribute__((always_inline)) {
    return head * G::kGroup + (G::kGroup == 2 ? column / 16 : column % 16);
  };

  // LDS read addresses within stage 0. K of k-step s: key n, chunk (2 s + half) ^ (n
  // & 15): bits 1 to 3 of the chunk by XOR, the rest by offset. V^T of dim block d:
  // lane i of 16-lane group vg reads keys 4 half + j (+ 8 r + 16 s2), dims 32 d + 16
  // vg + 4 q (j = (lane % 16) / 4, q = lane % 4).
  const uint32_t k_lane = lds_address(&lds.k[0][0]) + n * G::kRowBytes + ((half ^ (n & 15)) << 4);
  const int vj = (lane & 15) >> 2, vq = lane & 3, vg = (lane >> 4) & 1;
  const uint32_t v_lane = lds_address(&lds.v[0][0]) + (4 * half + vj) * G::kRowBytes +
                          (((4 * vj + 2 * vg + (vq >> 1)) << 4) | ((vq & 1) << 3));  // d = 0

  // Source byte offsets of a copying lane before the copy's own bits: key 8 w (+ 1
  // in lanes 32 .. 63 of a copy of two keys).
  static_assert(kCopyKeys == 8);
  auto k_chunk = [&](int l) __attribute__((always_inline)) -> uint32_t {
    return (G::kRowBytes == 1024 ? l ^ (8 * (wave & 1))
                                 : (l & 31) ^ (8 * (wave & 1) + (l >> 5))) << 4;
  };
  auto v_chunk = [&](int l) __attribute__((always_inline)) -> uint32_t {
    return (G::kRowBytes == 1024 ? l : (l & 31) ^ ((l >> 5) << 2)) << 4;
  };
  const uint32_t copy_row0 = kCopyKeys * wave * G::kRowBytes;
  const uint32_t k_dst = wave_uniform(lds_address(&lds.k[0][0]) + copy_row0);
  const uint32_t v_dst = wave_uniform(lds_address(&lds.v[0][0]) + copy_row0);
  const uint32_t page_dst = wave_uniform(lds_address(&lds.pages[wave][0]));

  for (; segment < segment_end; ++segment) {
    // ---- the segment ---------------------------------------------------------
    const ExtendSegment seg = segments[segment];
    const int32_t row0 = seg.row0, rows = seg.rows, base = seg.base, prior = seg.prior;
    const int32_t partial = seg.partial, tile_lo = seg.tile_lo;
    const int n_tiles = seg.tile_hi - tile_lo;
    const int32_t first = prior + row0, last = first + rows - 1;  // positions
    const ExtendTiles tiles = extend_tiles(first, last, window, sinks, kTile);
    const int32_t tile_skip = tiles.window_tile - tiles.sink_tiles;
    auto tile_key = [&](int it) __attribute__((always_inline)) -> int32_t {
      const int32_t i = tile_lo + it;
      return (i < tiles.sink_tiles ? i : i + tile_skip) * kTile;
    };

    const int32_t wave_row0 = G::kWaveRows * wave;
    const bool wave_has_rows = wave_row0 < rows;
    const bool wave_rows_full = wave_row0 + G::kWaveRows <= rows;
    const int32_t wave_qmin = first + wave_row0;
    const int32_t wave_qmax = min(wave_qmin + G::kWaveRows - 1, last);

    // ---- key rows ----------------------------------------------------------------
    // A wave resolves its keys of kRunTiles tiles at once: lane l key kCopyKeys w + l %
    // 8 of the run's tile l / 8.
    const int32_t *table = p.page_table + (int64_t)seg.sequence * max_pages;
    const uint64_t chunk_off = (uint64_t)base * kv_bytes + head * G::kRowBytes;
    const uint64_t chunk_k = reinterpret_cast<uint64_t>(p.k) + chunk_off;
    const uint64_t chunk_v = reinterpret_cast<uint64_t>(p.v) + chunk_off;
    auto run_key = [&](int run, int l) __attribute__((always_inline)) -> int32_t {
      return tile_key(run * kRunTiles + l / kCopyKeys) + kCopyKeys * wave + l % kCopyKeys;
    };
    // Table entry of this lane's key; any readable one for a new key.
    auto page_entry = [&](int run, int l) __attribute__((always_inline)) -> const int32_t * {
      const uint32_t at = (uint32_t)max(min(run_key(run, l), prior - 1), 0);
      return table + fast_mod(fast_div(at, p.page_div), p.slot_div);
    };
    auto resolve = [&](int run, int l, int32_t page) __attribute__((always_inline)) {
      const int32_t key = run_key(run, l);
      const bool fresh = key >= prior;
      const uint32_t logical = fast_div((uint32_t)key, p.page_div);
      const bool seen = (key <= last) & (run * kRunTiles + l / kCopyKeys < n_tiles) &
                        ((window == 0) | (key > first - window) | (key < sinks));
      const bool mapped = ((uint32_t)page < (uint32_t)p.c.num_pages) &
                          (ring | (logical < (uint32_t)max_pages));
      const bool ok = seen & (fresh | mapped);
      const uint32_t cached =
          (uint32_t)page * p.page_div.d + ((uint32_t)key - logical * p.page_div.d);
      const uint64_t off = pick(fresh, (uint64_t)(uint32_t)(key - prior) * kv_bytes,
                                (uint64_t)cached * G::kTokenBytes);
      lds.k_rows[run & 1][wave][l] = pick(ok, pick(fresh, chunk_k, cache_k) + off, zero_row);
      lds.v_rows[run & 1][wave][l] = pick(ok, pick(fresh, chunk_v, cache_v) + off, zero_row);
      const uint64_t valid = __builtin_amdgcn_ballot_w64(ok);
      if (l < kRunTiles) lds.valid[run & 1][l][wave] = (uint8_t)(valid >> (kCopyKeys * l));
    };
    // This lane's row address for copy a of a tile: keys kCopyKeys w + 2 a and + 1
    // (lanes 0 .. 31, 32 .. 63) at 8 x 256, key kCopyKeys w + a at 1 x 512.
    auto row_slot = [&](int tile, int a, int l) __attribute__((always_inline)) -> int {
      return tile % kRunTiles * kCopyKeys + (G::kRowBytes == 1024 ? a : 2 * a + (l >> 5));
    };
    auto k_row = [&](int tile, int a, int l) __attribute__((always_inline)) -> uint64_t {
      return lds.k_rows[tile / kRunTiles & 1][wave][row_slot(tile, a, l)];
    };
    auto v_row = [&](int tile, int a, int l) __attribute__((always_inline)) -> uint64_t {
      return lds.v_rows[tile / kRunTiles & 1][wave][row_slot(tile, a, l)];
    };
    // Lane l of a copy fills chunk l (or l % 32) of its key's row with the chunk that
    // the swizzle puts there: k_chunk and v_chunk with the key's a-dependent bits.
    auto copy_k = [&](uint64_t row, uint32_t chunk, int a, int stage)
        __attribute__((always_inline)) {
      const int key = G::kRowBytes == 1024 ? a : 2 * a;
      copy_row_pair(row + (chunk ^ ((key & 15) << 4)), k_dst + stage * kStageBytes + a * 1024);
    };
    auto copy_v = [&](uint64_t row, uint32_t chunk, int a, int stage)
        __attribute__((always_inline)) {
      const int key = G::kRowBytes == 1024 ? a : 2 * a;
      copy_row_pair(row + (chunk ^ ((key & 3) << 6)), v_dst + stage * kStageBytes + a * 1024);
    };

    // ---- before the first tile ------------------------------------------------------
    // Iteration t copies K of tile t + kStages - 1 and V of t + kStages - 2; what tile 0
    // .. kStages - 2 need goes out here. A run's table entries are copied to LDS in the
    // first iteration of the run before, and resolved in its fifth.
    int32_t page = *page_entry(0, lane);
    // Q^T operand: lane holds Q[row][16 s + 8 half .. + 8] of every k-step.
    u32x4v_t q[G::kSteps];
    {
      const int row = column_row(n);  // past the last one: any row, not stored
      const int64_t from = (int64_t)base + row0 + (row < rows ? row : 0);
      const uint16_t *q_row = p.q + from * p.q_stride + column_head(n) * kDim + 8 * half;
#pragma unroll
      for (int s = 0; s < G::kSteps; ++s)
        q[s] = *reinterpret_cast<const u32x4v_t *>(q_row + 16 * s);
    }
    // All of these are asked for before anything waits, and waited for before the
    // first copy: a later wait for them would wait for the copies too.
    asm volatile("" : "+v"(page));
#pragma unroll
    for (int s = 0; s < G::kSteps; ++s) asm volatile("" : "+v"(q[s]));
    resolve(0, lane, page);
#pragma unroll
    for (int g = 0; g < kStages - 1; ++g) {
#pragma unroll
      for (int a = 0; a < G::kCopies; ++a) {
        copy_k(k_row(g, a, lane), k_chunk(lane), a, g);
        if (g > 0) copy_v(v_row(g - 1, a, lane), v_chunk(lane), a, g - 1);
      }
    }

    float m_run = -INFINITY, l_run = 0.0f;
    f32x16_t acc[G::kDims];
#pragma unroll
    for (int d = 0; d < G::kDims; ++d) acc[d] = f32x16_t{};
    u32x4v_t weights[2];    // P^T of the tile before, 16 keys each
    bool pending = false;   // whether it still has to meet V
    bool started = false;   // whether the accumulators hold anything

    // The second product of a tile in `stage`; beside(j) rides on product j.
    auto multiply_v = [&](int stage, auto &&beside) __attribute__((always_inline)) {
      uint32_t base_at = v_lane + stage * kStageBytes;
      asm volatile("" : "+v"(base_at));  // the four offsets below are not kept either
      auto read_v = [&](int j) __attribute__((always_inline)) -> u32x4v_t {
        const int d = j % G::kDims, s2 = j / G::kDims;
        const uint32_t at = (base_at ^ ((d & 3) << 6)) + 16 * s2 * G::kRowBytes + (d >> 2) * 256;
        const uint2 lo = lds_read_tr(at), hi = lds_read_tr(at + 8 * G::kRowBytes);
        return u32x4v_t{lo.x, lo.y, hi.x, hi.y};
      };
      constexpr int kProducts = 2 * G::kDims, kAhead = 4;
      u32x4v_t v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) v[j] = read_v(j);
      static_for<0, kProducts>([&](auto jc) __attribute__((always_inline)) {
        constexpr int j = decltype(jc)::value;
        mfma_pv(acc[j % G::kDims], v[j % kAhead], weights[j / G::kDims]);
        if constexpr (j + kAhead < kProducts) v[j % kAhead] = read_v(j + kAhead);
        beside(jc);
        __builtin_amdgcn_sched_barrier(0);
      });
    };
    // One iteration more than tiles, for the last tile's second product.
    for (int it = 0; it <= n_tiles; ++it) {
      const int stage = it & (kStages - 1);
      const int k_stage = (it + kStages - 1) & (kStages - 1);  // of tile it - 1, too
      const int v_stage = (it + kStages - 2) & (kStages - 1);
      // Needed: K of tile it, V of the tile before. Of what was issued in the last
      // kStages - 2 iterations nothing is, and right after a run's first iteration its
      // entries' copy is the newest.
      constexpr int kInFlight = (kStages - 2) * 2 * G::kCopies;
      const int run = it / kRunTiles, run_tile = it % kRunTiles;
      if (run_tile == 1) {
        wait_vector<kInFlight + 1>();
      } else {
        wait_vector<kInFlight>();
      }
      lds_barrier();  // all waves' copies are there; every wave is done with iteration it - 1
      const uint32_t valid =
          wave_uniform(*reinterpret_cast<const int32_t *>(lds.valid[run & 1][run_tile]));
      const int32_t key0 = tile_key(it), key1 = key0 + kTile - 1;
      const bool live = wave_has_rows && it < n_tiles && key0 <= wave_qmax &&
                        (window == 0 || key1 > wave_qmin - window || key0 < sinks);
      const int copy_lane = fresh_lane();
      const uint32_t kc = k_chunk(copy_lane), vc = v_chunk(copy_lane);
      const int k_tile = it + kStages - 1, v_tile = it + kStages - 2;
      f32x16_t score = f32x16_t{};
      if (live) {
        const uint32_t k_at = k_lane + stage * kStageBytes;
        auto read_k = [&](int s) __attribute__((always_inline)) {
          return lds_read128((k_at ^ ((s & 7) << 5)) + (s >> 3) * 256);
        };
        u32x4v_t kf[G::kWindow];
#pragma unroll
        for (int s = 0; s < G::kWindow; ++s) kf[s] = read_k(s);
        // Copy a of K and of V ride on products 4 a + 1 and 4 a + 3, their row addresses
        // are read four products ahead.
        uint64_t kr = k_row(k_tile, 0, copy_lane), vr = v_row(v_tile, 0, copy_lane);
        uint64_t kr_next = 0, vr_next = 0;
        __builtin_amdgcn_sched_barrier(0);
        static_for<0, G::kSteps>([&](auto sc) __attribute__((always_inline)) {
          constexpr int s = decltype(sc)::value, a = s / 4;
          score = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              __builtin_bit_cast(bf16x8_t, kf[s % G::kWindow]), __builtin_bit_cast(bf16x8_t, q[s]),
              score, 0, 0, 0);
          if constexpr (s + G::kWindow < G::kSteps) kf[s % G::kWindow] = read_k(s + G::kWindow);
          if constexpr (s % 4 == 0 && a + 1 < G::kCopies) {
            kr_next = k_row(k_tile, a + 1, copy_lane);
            vr_next = v_row(v_tile, a + 1, copy_lane);
          } else if constexpr (s % 4 == 1) {
            copy_k(kr, kc, a, k_stage);
          } else if constexpr (s % 4 == 3) {
            copy_v(vr, vc, a, v_stage);
            kr = kr_next;
            vr = vr_next;
          }
          __builtin_amdgcn_sched_barrier(0);
        });
        static_assert(G::kSteps == 4 * G::kCopies);
      } else {
#pragma unroll
        for (int a = 0; a < G::kCopies; ++a) {
          copy_k(k_row(k_tile, a, copy_lane), kc, a, k_stage);
          copy_v(v_row(v_tile, a, copy_lane), vc, a, v_stage);
        }
      }
      if (run_tile == 0) {
        copy_dwords(page_entry(run + 1, copy_lane), page_dst);
      } else if (run_tile == 4) {
        resolve(run + 1, copy_lane, lds.pages[wave][copy_lane]);
      }
      if (!live && !pending) continue;
      const bool full = live && wave_rows_full && valid == 0xFFFFFFFFu && key1 <= wave_qmin &&
                        (window == 0 || key0 > wave_qmax - window || key1 < sinks);
      // Lane holds keys (i / 4) * 8 + 4 half + i % 4 of column n.
      if (!full) {
        auto below = [](int32_t count) -> uint32_t {  // keys 0 .. count - 1 of the block
          return count <= 0 ? 0u : (count >= 32 ? 0xFFFFFFFFu : (1u << count) - 1u);
        };
        const int lane2 = fresh_lane(), row = column_row(lane2 & 31);
        const int32_t qpos = first + row;
        uint32_t seen = below(qpos - key0 + 1);
        if (window > 0) seen &= ~below(qpos - window + 1 - key0) | below(sinks - key0);
        seen = (row < rows && live ? seen & valid : 0u) >> (4 * (lane2 >> 5));
#pragma unroll
        for (int i = 0; i < 16; ++i)
          score[i] = (seen >> ((i / 4) * 8 + i % 4)) & 1u ? score[i] : -INFINITY;
      }

      // ---- softmax, under the second product of the tile before ------------------------
      float top, alpha, m_use;
      bool moved;
      uint32_t pw[8];
      auto softmax = [&](auto uc) __attribute__((always_inline)) {
        constexpr int u = decltype(uc)::value;
        if constexpr (u == 0) {
          top = fmaxf(fmaxf(score[0], score[1]), score[2]);
          top = fmaxf(fmaxf(top, score[3]), score[4]);
          top = fmaxf(fmaxf(top, score[5]), score[6]);
          top = fmaxf(fmaxf(top, score[7]), score[8]);
        } else if constexpr (u == 1) {
          top = fmaxf(fmaxf(top, score[9]), score[10]);
          top = fmaxf(fmaxf(top, score[11]), score[12]);
          top = fmaxf(fmaxf(top, score[13]), score[14]);
          top = xor_max<32>(fmaxf(top, score[15])) * p.q_scale;
        } else if constexpr (u == 2) {
          // The maximum moves (and the sums are rescaled) only when a column outgrows
          // it by more than the slack: exp2's arguments stay below that.
          moved = __builtin_amdgcn_ballot_w64(top > m_run + kRescaleSlack) != 0;
          const float m_new = moved ? fmaxf(m_run, top) : m_run;
          alpha = m_run == m_new ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
          m_run = m_new;
          m_use = m_new == -INFINITY ? 0.0f : m_new;
          l_run *= alpha;
        } else if constexpr (u >= 4 && u < 12) {
          constexpr int i = 2 * (u - 4);
          const float p0 = __builtin_amdgcn_exp2f(fmaf(score[i], p.q_scale, -m_use));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(score[i + 1], p.q_scale, -m_use));
          l_run += p0 + p1;
          // P is the product's operand: bf16, half a step (2^-8) of each weight.
          pw[i / 2] = cvt_pk_bf16(p0, p1);
        }
      };
      if (pending) {
        multiply_v(k_stage, [&](auto jc) __attribute__((always_inline)) {
          constexpr int j = decltype(jc)::value, kPer = G::kDims / 8;
          if constexpr (j % kPer == 0) softmax(std::integral_constant<int, j / kPer>{});
        });
        started = true;
      } else {
        static_for<0, 12>(softmax);
      }
      if (moved && started) {
        mfma_pv_done(acc);
#pragma unroll
        for (int d = 0; d < G::kDims; ++d) acc[d] *= alpha;
      }
      weights[0] = u32x4v_t{pw[0], pw[1], pw[2], pw[3]};
      weights[1] = u32x4v_t{pw[4], pw[5], pw[6], pw[7]};
      pending = live;
    }
    wait_copies();
    mfma_pv_done(acc);

    // ---- the rows' end ---------------------------------------------------------------
    l_run = xor_sum<32>(l_run);
    const int end_lane = fresh_lane(), end_half = end_lane >> 5;
    const int row = column_row(end_lane & 31), qh = column_head(end_lane & 31);
    // Lane holds dims 32 d + 8 i + 4 half .. + 3 of its column in accumulators 4 i .. + 3.
    if (row < rows && partial < 0) {
      const float inv = l_run > 0.0f ? 1.0f / l_run : 0.0f;
      uint16_t *o = p.out + (((int64_t)base + row0 + row) * kQueryHeads + qh) * kDim + 4 * end_half;
#pragma unroll
      for (int d = 0; d < G::kDims; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<uint2 *>(o + 32 * d + 2 * i) =
              make_uint2(cvt_pk_bf16(acc[d][i] * inv, acc[d][i + 1] * inv),
                         cvt_pk_bf16(acc[d][i + 2] * inv, acc[d][i + 3] * inv));
    } else if (row < rows) {
      const int64_t at = (int64_t)(partial + row) * kQueryHeads + qh;
      float *o = p.partial + at * kDim + 4 * end_half;
#pragma unroll
      for (int d = 0; d < G::kDims; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<float4 *>(o + 32 * d + 2 * i) =
              make_float4(acc[d][i], acc[d][i + 1], acc[d][i + 2], acc[d][i + 3]);
      if (end_half == 0) *reinterpret_cast<float2 *>(p.stats + 2 * at) = make_float2(m_run, l_run);
    }
    __syncthreads();  // the next segment's copies overwrite the stages
  }
}

}  // namespace

void launch_extend_rows(const ExtendParams &p, hipStream_t stream) {
  if (p.c.num_heads == 1) {
    hipLaunchKernelGGL(extend_rows_kernel<512>, dim3(kExtend512.shares), dim3(kThreads), 0, stream,
                       p);
  } else {
    hipLaunchKernelGGL(extend_rows_kernel<256>, dim3(Shape<256>::kHeads * kExtend256.shares),
                       dim3(kThreads), 0, stream, p);
  }
}

}  // namespace gemma4
