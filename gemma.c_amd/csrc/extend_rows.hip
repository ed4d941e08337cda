// The rows of a ragged extension batch on bf16 MFMA, gfx950: one share of the
// plan's segments per workgroup.
//
// Formulation: S^T = K Q^T and O^T = V^T P^T with v_mfma_f32_32x32x16_bf16 on tiles
// of 32 keys. A workgroup of four waves has 128 columns, (row, query head) pairs of
// the KV head: 16 rows x 2 heads per wave at 8 x 256, 2 rows x 16 heads at 1 x 512.
// A wave scores its own 32 columns over all dims, with its Q^T in registers. In the
// accumulator lane l holds column l % 32 and 16 of the keys: a column's maximum
// needs one exchange (lane ^ 32), and the weights leave in the second product's
// operand order, {4h .. 4h+3, 8+4h .. 8+4h+3} per 16 keys, in which V^T is read
// (ds_read_b64_tr_b16). The second product is split by dims instead: the waves trade
// their weights through LDS (4 KiB a tile each) and each adds up a quarter of the
// dims for all 128 columns, so that V is read from LDS once per workgroup and not
// once per wave. Where a block has one wave's rows at most, the first wave scores and
// all four add up.
//
// Keys stream in tiles through LDS stages (four of 16 KiB each of K and V at 8 x 256,
// two of 32 KiB at 1 x 512), copied by the waves themselves (global_load_lds) from row
// addresses that their lanes resolve for eight tiles at once: a page-table entry per
// key, any page size, the packed new rows behind the cached ones. Keys that no row of
// the block sees, that no page maps, or past the segment's tiles are copied from a
// row of zeros, so nothing in such a place is ever multiplied. Rows land swizzled by
// 16-byte chunks (K row k, chunk c at c ^ (k & 15); V at c ^ ((k & 3) << 2)): no bank
// conflict in the operand reads (counted: 0).
//
// With one wave per SIMD nothing else fills the matrix cores while a wave does its
// softmax, so iteration t interleaves the softmax of tile t with the second
// product of tile t - 1. Registers: at 1 x 512 the accumulators are all 256 AGPRs
// (the second product is asm, the first one's results stay in VGPRs by a build flag
// for this file), Q^T half of the VGPRs.
//
// Measured, 2048 rows after 6144 keys: at 1 x 512 459 us with the merge, 1.05 PFLOP/s
// (a large library product reaches 1.30), at 8 x 256 285 us, 0.84. A tile takes 3740
// clocks at 1 x 512 and 2550 at 8 x 256, of which the matrix cores work 2048 and 1024;
// the rest is what the one wave per SIMD issues besides (some 430 and 290 instructions,
// the copies among them 340 clocks and 90) and the LDS latency behind its barrier. The
// clock itself falls to 1.95 GHz of
// 2.4 under this load, and forms with fewer or better spread instructions (scalar row
// addresses, half of the copies under each product with a barrier between) changed
// clocks and clock rate against each other and not the time. Batches of single tokens
// stream at 4.1 to 5.1 TB/s with start-up and merge (24 sequences at 1 x 512, 302 MB:
// 73 us).
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
  static constexpr int kDims = kDim / 32 / kWaves;      // 32-dim blocks of O^T per wave
  static constexpr int kCopies = kCopyKeys * kRowBytes / 1024;  // of K, and of V
  static constexpr int kTokenBytes = kHeads * kRowBytes;        // a cached token's rows
  static constexpr int kWindow = 4;  // K fragments read ahead (of all 16 at 8 x 256: 1 to 3% slower)
};
static_assert(Shape<256>::kRows == kExtend256.rows && kTile == kExtend256.tile &&
              Shape<256>::kWaveRows == kExtend256.wave_rows);
static_assert(Shape<512>::kRows == kExtend512.rows && kTile == kExtend512.tile &&
              Shape<512>::kWaveRows == kExtend512.wave_rows);

template <int kBegin, int kEnd, class F>
__device__ __forceinline__ void static_for(F &&f) {
  if constexpr (kBegin < kEnd) {
    f(std::integral_constant<int, kBegin>{});
    static_for<kBegin + 1, kEnd>(f);
  }
}

typedef unsigned u32x4v_t __attribute__((ext_vector_type(4)));

// acc += V^T P^T with the accumulators in AGPRs. No VALU instruction writes an
// operand within two issues before (both come from LDS reads): the compiler does not
// see into asm and adds no wait states.
__device__ __forceinline__ void mfma_pv(f32x16_t &acc, u32x4v_t v, u32x4v_t p) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(v), "v"(p));
}
// acc = 0 by a product of zeros: two clocks a register, where a write of each takes four
// (mixed batches 1% faster).
__device__ __forceinline__ void mfma_zero(f32x16_t &acc, u32x4v_t zero) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %1, 0" : "=a"(acc) : "v"(zero));
}
// Every product above has written its accumulators: a product is 8 passes (32 clocks,
// as the 2048 of a tile's 64 show) and the write; the waits would cover 16.
template <int kCount>
__device__ __forceinline__ void mfma_pv_done(f32x16_t (&acc)[kCount]) {
#pragma unroll
  for (int d = 0; d < kCount; d += 2)
    asm volatile("s_nop 15\n\ts_nop 7" : "+a"(acc[d]), "+a"(acc[d + 1]));
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

// Two 1 KiB LDS copies (16 bytes per lane) into consecutive KiB: the second's
// offset applies to both of its addresses and is taken back from the source.
__device__ __forceinline__ void copy_rows2(uint64_t src0, uint64_t src1, uint32_t lds_addr) {
  uint32_t m0_saved;
  src1 -= 1024;
  asm volatile(
      "s_mov_b32 %[m0s], m0\n\t"
      "s_mov_b32 m0, %[lds]\n\t"
      "s_nop 0\n\t"  // SALU write of M0 -> LDS DMA reading it: one wait state (gfx9)
      "global_load_lds_dwordx4 %[s0], off\n\t"
      "global_load_lds_dwordx4 %[s1], off offset:1024\n\t"
      "s_mov_b32 m0, %[m0s]"
      : [m0s] "=&s"(m0_saved)
      : [lds] "s"(lds_addr), [s0] "v"(src0), [s1] "v"(src1));
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
    // What the waves trade, by the parity of the tile: their columns' weights as B
    // operands, and the factor of the columns' sums where a maximum moved.
    u32x4v_t weights[2][kWaves][2][kWave];
    float alpha[2][kWaves][32];
    uint8_t moved[2][kWaves];
    float sums[kWaves][32];
  };
  __shared__ __attribute__((aligned(1024))) Lds lds;

  const int t = threadIdx.x, lane = t & 63;
  const int wave = wave_uniform(t >> 6);
  const int half = lane >> 5, n = lane & 31;
  // Workgroups go to the eight XCDs in turn. At 8 x 256 an XCD gets a KV head; at 1 x
  // 512 the shares in eight runs, so that a sequence's keys are read through the L2s
  // of few XCDs (a step of ten mixed sequences 202 -> 188 us).
  const int head = blockIdx.x % G::kHeads;
  const int share = G::kHeads == 1 ? blockIdx.x % 8 * (kExtend512.shares / 8) + blockIdx.x / 8
                                   : blockIdx.x / G::kHeads;

  const ExtendShare mine =
      plan_read<ExtendShare>(p.plan + p.shares + (int64_t)share * sizeof(ExtendShare));
  const ExtendHeader header = plan_read<ExtendHeader>(p.plan);
  if (!extend_plan_fits(p, header)) return;
  const int32_t window = header.window, sinks = header.sinks, period = header.period;

  const bool ring = p.c.window_size > 0;
  const int32_t max_pages = p.c.max_pages_per_seq;
  const uint64_t layer_bytes =
      (uint64_t)p.layer * p.c.num_pages * p.c.page_size * G::kTokenBytes + head * G::kRowBytes;
  const uint64_t cache_k = reinterpret_cast<uint64_t>(p.cache_k) + layer_bytes;
  const uint64_t cache_v = reinterpret_cast<uint64_t>(p.cache_v) + layer_bytes;
  const uint64_t zero_row = reinterpret_cast<uint64_t>(&g_zero_row[0]);
  const uint32_t kv_bytes = (uint32_t)(p.kv_stride * 2);

  // Row, among the workgroup's, of a column of wave w, and its query head.
  auto column_row = [&](int w, int column) __attribute__((always_inline)) {
    return G::kWaveRows * w + (G::kGroup == 2 ? column % 16 : column / 16);
  };
  auto column_head = [&](int column) __attribute__((always_inline)) {
    return head * G::kGroup + (G::kGroup == 2 ? column / 16 : column % 16);
  };

  // LDS read addresses of lane l within stage 0. K of k-step s: key l % 32, chunk (2 s +
  // l / 32) ^ (l & 15): bits 1 to 3 of the chunk by XOR, the rest by offset. V^T of the
  // wave's first dim block: lane i of 16-lane group vg reads keys 4 (l / 32) + j (+ 8 r +
  // 16 s2), dims 16 vg + 4 q (j = (l % 16) / 4, q = l % 4).
  auto k_address = [&](int l) __attribute__((always_inline)) -> uint32_t {
    return lds_address(&lds.k[0][0]) + (l & 31) * G::kRowBytes + (((l >> 5) ^ (l & 15)) << 4);
  };
  auto v_address = [&](int l) __attribute__((always_inline)) -> uint32_t {
    const int block = G::kDims * wave, j = (l & 15) >> 2, q = l & 3, vg = (l >> 4) & 1;
    return lds_address(&lds.v[0][0]) + (4 * (l >> 5) + j) * G::kRowBytes +
           (((4 * ((block & 3) ^ j) + 2 * vg + (q >> 1)) << 4) | ((q & 1) << 3)) +
           (block >> 2) * 256;
  };
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

  // Registers are short at 1 x 512 only.
  auto lane_now = [&]() __attribute__((always_inline)) -> int {
    if constexpr (kDim == 512) return fresh_lane();
    return lane;
  };

  int32_t elapsed = 0;  // of the share, in tiles
  for (int32_t segment = mine.first; segment < mine.end; ++segment) {
    // ---- the segment ---------------------------------------------------------
    ExtendSegment seg = mine.segment;
    if (segment != mine.first)
      seg = plan_read<ExtendSegment>(p.plan + p.segments + (int64_t)segment * sizeof(ExtendSegment));
    const int32_t row0 = seg.row0, rows = seg.rows, base = seg.base, prior = seg.prior;
    const int32_t partial = seg.partial, tile_lo = seg.tile_lo;
    const int n_tiles = seg.tile_hi - tile_lo;
    const int32_t first = prior + row0, last = first + rows - 1;  // positions
    const ExtendTiles tiles = extend_tiles(first, last, window, sinks, kTile);
    const int32_t tile_skip = tiles.window_tile - tiles.sink_tiles;
    // Shares begin at any tile of a row block, and last equally long. A share visits its
    // tiles from the one whose number is `elapsed` modulo the period on, and round to the
    // ones before: so all shares that need a tile come to it at about the same time,
    // and the later ones find it in their XCD's L2 (ten mixed sequences at 1 x 512 read 280
    // MB past L2 instead of 750, 187 -> 182 us).
    const int32_t ahead = elapsed - (tile_lo + tile_skip);
    const int32_t turn = ahead - (ahead >= 0 ? ahead : ahead - period + 1) / period * period;
    const int32_t start = turn < n_tiles ? tile_lo + turn : tile_lo;
    const int32_t before_wrap = tile_lo + n_tiles - start;
    // With a wide block's own cost. A block of one wave's rows is 3 in the plan: in
    // batches of many such blocks the shares drift apart, which costs reads past L2 only.
    elapsed += n_tiles + 6;
    auto tile_key = [&](int it) __attribute__((always_inline)) -> int32_t {
      const int32_t i = it + (it < before_wrap ? start : tile_lo - before_wrap);
      return (i < tiles.sink_tiles ? i : i + tile_skip) * kTile;
    };

    const int32_t wave_row0 = G::kWaveRows * wave;
    const bool wave_has_rows = wave_row0 < rows;
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
    // Copies a and a + 1 go out together, from rows r0 and r1.
    auto copy_k = [&](uint64_t r0, uint64_t r1, uint32_t chunk, int a, int stage)
        __attribute__((always_inline)) {
      const int key = G::kRowBytes == 1024 ? a : 2 * a, step = G::kRowBytes == 1024 ? 1 : 2;
      copy_rows2(r0 + (chunk ^ ((key & 15) << 4)), r1 + (chunk ^ (((key + step) & 15) << 4)),
                 k_dst + stage * kStageBytes + a * 1024);
    };
    auto copy_v = [&](uint64_t r0, uint64_t r1, uint32_t chunk, int a, int stage)
        __attribute__((always_inline)) {
      const int key = G::kRowBytes == 1024 ? a : 2 * a, step = G::kRowBytes == 1024 ? 1 : 2;
      copy_rows2(r0 + (chunk ^ ((key & 3) << 6)), r1 + (chunk ^ (((key + step) & 3) << 6)),
                 v_dst + stage * kStageBytes + a * 1024);
    };

    // ---- before the first tile ------------------------------------------------------
    // Iteration t copies K of tile t + kStages - 1 and V of t + kStages - 2; what tile 0
    // .. kStages - 2 need goes out here. A run's table entries are copied to LDS in the
    // first iteration of the run before, and resolved in its fifth.
    const int32_t page = *page_entry(0, lane);
    resolve(0, lane, page);
    // Iteration 0 multiplies a tile -1 of zero weights and zero rows.
    lds.weights[1][wave][0][lane] = lds.weights[1][wave][1][lane] = u32x4v_t{0, 0, 0, 0};
#pragma unroll
    for (int a = 0; a < G::kCopies; a += 2) copy_v(zero_row, zero_row, v_chunk(lane), a, kStages - 1);
#pragma unroll
    for (int a = 0; a < G::kCopies; a += 2)
      copy_k(k_row(0, a, lane), k_row(0, a + 1, lane), k_chunk(lane), a, 0);

    // Q^T operand: lane holds Q[row][16 s + 8 half .. + 8] of every k-step. Asked for
    // behind the first tile's keys, and waited for (with them) here: a wait in the loop
    // would be one for the loop's copies. The copies of further tiles go out behind: the
    // first tile is scored while they are on their way (2048 rows after 6144 at 8 x 256
    // 285 -> 281 us).
    u32x4v_t q[G::kSteps];
    if (wave_has_rows) {
      const int row = column_row(wave, n);  // past the last one: any row, not stored
      const int64_t from = (int64_t)base + row0 + (row < rows ? row : 0);
      const uint16_t *q_row = p.q + from * p.q_stride + column_head(n) * kDim + 8 * half;
#pragma unroll
      for (int s = 0; s < G::kSteps; ++s)
        q[s] = *reinterpret_cast<const u32x4v_t *>(q_row + 16 * s);
    } else {
#pragma unroll
      for (int s = 0; s < G::kSteps; ++s) q[s] = u32x4v_t{0, 0, 0, 0};
    }
#pragma unroll
    for (int s = 0; s < G::kSteps; ++s) asm volatile("" : "+v"(q[s]));
#pragma unroll
    for (int g = 1; g < kStages - 1; ++g) {
#pragma unroll
      for (int a = 0; a < G::kCopies; a += 2) {
        copy_k(k_row(g, a, lane), k_row(g, a + 1, lane), k_chunk(lane), a, g);
        copy_v(v_row(g - 1, a, lane), v_row(g - 1, a + 1, lane), v_chunk(lane), a, g - 1);
      }
    }

    // The segment with its columns in kGroups groups: all four waves' of them, or one
    // wave's where its rows are that few; then only the first wave scores, and all four
    // still share the second product by dims.
    auto attend = [&](auto groups) __attribute__((always_inline)) {
    constexpr int kGroups = decltype(groups)::value;
    float m_run = -INFINITY, l_run = 0.0f;
    bool started = false;  // whether this wave's columns have had weights
    // O^T of the wave's dims for all columns: group c, the columns of wave c.
    f32x16_t acc[kGroups * G::kDims];
    u32x4v_t zeros = {0, 0, 0, 0};
    asm volatile("s_nop 1" : "+v"(zeros));  // before a product reads what was just written
#pragma unroll
    for (int i = 0; i < kGroups * G::kDims; ++i) mfma_zero(acc[i], zeros);

    // V^T operand i = kDims s2 + d of the tile at v_at; weights of group c, 16 keys s2.
    constexpr int kOperands = 2 * G::kDims, kRing = 3;
    u32x4v_t v[kRing], w[kGroups];
    auto read_v = [&](uint32_t v_at, int i) __attribute__((always_inline)) {
      const int d = i % G::kDims, s2 = i / G::kDims;
      const uint32_t at = (v_at ^ (d << 6)) + 16 * s2 * G::kRowBytes;
      const uint2 lo = lds_read_tr(at), hi = lds_read_tr(at + 8 * G::kRowBytes);
      v[i % kRing] = u32x4v_t{lo.x, lo.y, hi.x, hi.y};
    };
    auto read_w = [&](int from, int c, int s2, int l) __attribute__((always_inline)) {
      w[c] = lds.weights[from][c][s2][l];
    };

    // Before iteration it: K of its tile, V of the tile before. Of what was issued in
    // the last kStages - 2 iterations nothing is needed, and right after a run's first
    // iteration its entries' copy is the newest.
    constexpr int kInFlight = (kStages - 2) * 2 * G::kCopies;
    wait_vector<kInFlight>();
    lds_barrier();
    // The first K fragments of a tile are asked for right behind its barrier, with
    // the word that says which of its keys can be read.
    u32x4v_t kf[G::kWindow];
    int32_t valid_word;
    auto read_k = [&](uint32_t k_at, int s) __attribute__((always_inline)) {
      kf[s % G::kWindow] = lds_read128((k_at ^ ((s & 7) << 5)) + (s >> 3) * 256);
    };
    auto read_first = [&](int tile, uint32_t k_at) __attribute__((always_inline)) {
      valid_word = *reinterpret_cast<const int32_t *>(
          lds.valid[tile / kRunTiles & 1][tile % kRunTiles]);
#pragma unroll
      for (int s = 0; s < G::kWindow; ++s) read_k(k_at, s);
    };
    uint32_t k_at = k_address(lane_now());  // of the tile's stage
    read_first(0, k_at);
    // One iteration more than tiles, for the last tile's second product.
    for (int it = 0; it <= n_tiles; ++it) {
      const int k_stage = (it + kStages - 1) & (kStages - 1);  // of tile it - 1, too
      const int v_stage = (it + kStages - 2) & (kStages - 1);
      const int run = it / kRunTiles, run_tile = it % kRunTiles;
      const int32_t key0 = tile_key(it), key1 = key0 + kTile - 1;
      const bool live = wave_has_rows && it < n_tiles && key0 <= wave_qmax &&
                        (window == 0 || key1 > wave_qmin - window || key0 < sinks);
      const int k_tile = it + kStages - 1, v_tile = it + kStages - 2;
      const int parity = it & 1;
      f32x16_t score = f32x16_t{};
      if (live) {
        // Copies a and a + 1 of K ride on product 4 a + 3, of V on 4 a + 7; their row
        // addresses are read three products ahead.
        uint64_t r0 = 0, r1 = 0;
        int l = 0;
        uint32_t kc = 0, vc = 0, v_at = 0;
        static_for<0, G::kSteps>([&](auto sc) __attribute__((always_inline)) {
          constexpr int s = decltype(sc)::value, a = s / 4;
          score = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              __builtin_bit_cast(bf16x8_t, kf[s % G::kWindow]), __builtin_bit_cast(bf16x8_t, q[s]),
              score, 0, 0, 0);
          if constexpr (s + G::kWindow < G::kSteps) read_k(k_at, s + G::kWindow);
          if constexpr (s == 0) l = lane_now();
          if constexpr (s == 1) kc = k_chunk(l);
          if constexpr (s == 5) vc = v_chunk(l);
          if constexpr (s == 6) v_at = v_address(l) + k_stage * kStageBytes;  // V of tile it - 1
          // The first operands of the second product that follows.
          constexpr int ahead = s - (G::kSteps - kGroups - kRing + 1);
          if constexpr (ahead >= 0 && ahead < kGroups) {
            read_w(parity ^ 1, ahead, 0, l);
          } else if constexpr (ahead >= kGroups) {
            read_v(v_at, ahead - kGroups);
          }
          if constexpr (s % 8 == 0) {
            r0 = k_row(k_tile, a, l);
            r1 = k_row(k_tile, a + 1, l);
          } else if constexpr (s % 8 == 3) {
            copy_k(r0, r1, kc, a, k_stage);
          } else if constexpr (s % 8 == 4) {
            r0 = v_row(v_tile, a - 1, l);
            r1 = v_row(v_tile, a, l);
          } else if constexpr (s % 8 == 7) {
            copy_v(r0, r1, vc, a - 1, v_stage);
          }
          __builtin_amdgcn_sched_barrier(0);
        });
        static_assert(G::kSteps == 4 * G::kCopies);
      } else {
        const int l = lane_now();
#pragma unroll
        for (int a = 0; a < G::kCopies; a += 2) {
          copy_k(k_row(k_tile, a, l), k_row(k_tile, a + 1, l), k_chunk(l), a, k_stage);
          copy_v(v_row(v_tile, a, l), v_row(v_tile, a + 1, l), v_chunk(l), a, v_stage);
        }
#pragma unroll
        for (int c = 0; c < kGroups; ++c) read_w(parity ^ 1, c, 0, l);
#pragma unroll
        for (int i = 0; i < kRing - 1; ++i) read_v(v_address(l) + k_stage * kStageBytes, i);
      }
      const int copy_lane = lane_now();
      const uint32_t v_at = v_address(copy_lane) + k_stage * kStageBytes;
      if (run_tile == 0) {
        copy_dwords(page_entry(run + 1, copy_lane), page_dst);
      } else if (run_tile == 4) {
        resolve(run + 1, copy_lane, lds.pages[wave][copy_lane]);
      }

      const uint32_t valid = wave_uniform(valid_word);
      // Columns without a row have some row's query; what they come to is not stored.
      const bool full = live && valid == 0xFFFFFFFFu && key1 <= wave_qmin &&
                        (window == 0 || key0 > wave_qmax - window || key1 < sinks);
      // Lane holds keys (i / 4) * 8 + 4 half + i % 4 of column n.
      if (!full) {
        auto below = [](int32_t count) -> uint32_t {  // keys 0 .. count - 1 of the block
          return count <= 0 ? 0u : (count >= 32 ? 0xFFFFFFFFu : (1u << count) - 1u);
        };
        const int lane2 = lane_now(), row = column_row(wave, lane2 & 31);
        const int32_t qpos = first + row;
        uint32_t seen = below(qpos - key0 + 1);
        if (window > 0) seen &= ~below(qpos - window + 1 - key0) | below(sinks - key0);
        seen = (row < rows && live ? seen & valid : 0u) >> (4 * (lane2 >> 5));
#pragma unroll
        for (int i = 0; i < 16; ++i)
          score[i] = (seen >> ((i / 4) * 8 + i % 4)) & 1u ? score[i] : -INFINITY;
      }

      // ---- sums of tile it - 1, and under them the softmax of tile it -------------------
      float top, alpha, m_use, even;
      bool moved = false;
      uint32_t pw[8];
      auto softmax = [&](auto uc) __attribute__((always_inline)) {
        constexpr int u = decltype(uc)::value;
        if constexpr (u == 0) {
          top = fmaxf(fmaxf(score[0], score[1]), score[2]);
          top = fmaxf(fmaxf(top, score[3]), score[4]);
        } else if constexpr (u < 4) {
          top = fmaxf(fmaxf(top, score[4 * u + 1]), score[4 * u + 2]);
          if constexpr (u < 3) {
            top = fmaxf(fmaxf(top, score[4 * u + 3]), score[4 * u + 4]);
          } else {
            top = fmaxf(top, score[15]);
          }
        } else if constexpr (u == 4) {
          top = xor_max<32>(top) * p.q_scale;
        } else if constexpr (u == 5) {
          // The maximum moves (and the sums are rescaled) only when a column outgrows
          // it by more than the slack: exp2's arguments stay below that.
          moved = __builtin_amdgcn_ballot_w64(top > m_run + kRescaleSlack) != 0;
          const float m_new = moved ? fmaxf(m_run, top) : m_run;
          alpha = m_run == m_new ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
          m_run = m_new;
          m_use = m_new == -INFINITY ? 0.0f : m_new;
          l_run *= alpha;
        } else if constexpr (u >= 7 && u < 23) {
          constexpr int i = u - 7;
          const float w = __builtin_amdgcn_exp2f(fmaf(score[i], p.q_scale, -m_use));
          // P is the product's operand in one bf16, half a step (2^-8) of each weight, as
          // in the chunk kernels: 0.0016 of the outputs' norm beside the 0.0017 of their own
          // rounding, 0.0023 together. A second bf16 for the rest would be another 1024
          // clocks of products in a tile of 3740 at 1 x 512. The sums l are of the weights
          // in 32 bits.
          if constexpr (i % 2 == 0) {
            even = w;
          } else {
            l_run += even + w;
            pw[i / 2] = cvt_pk_bf16(even, w);
          }
        } else if constexpr (u == 23) {
          if (kGroups == kWaves || wave == 0) {
            lds.weights[parity][wave][0][copy_lane] = u32x4v_t{pw[0], pw[1], pw[2], pw[3]};
            lds.weights[parity][wave][1][copy_lane] = u32x4v_t{pw[4], pw[5], pw[6], pw[7]};
            lds.alpha[parity][wave][copy_lane & 31] = alpha;
          }
          // The first weights meet sums that are zero: no factor.
          lds.moved[parity][wave] = moved && started ? 1 : 0;
          started = started || moved;
          asm volatile("" : "+v"(l_run));  // its additions stay under the products
        }
      };
      // Product j: operand i = j / kGroups, group j % kGroups.
      constexpr int kUnits = 24, kProducts = kGroups * kOperands;
      static_for<0, kProducts>([&](auto jc) __attribute__((always_inline)) {
        constexpr int j = decltype(jc)::value, i = j / kGroups, c = j % kGroups;
        mfma_pv(acc[c * G::kDims + i % G::kDims], v[i % kRing], w[c]);
        if constexpr (c == 0 && i + kRing - 1 < kOperands) read_v(v_at, i + kRing - 1);
        if constexpr (i == G::kDims - 1) read_w(parity ^ 1, c, 1, copy_lane);
        static_for<j * kUnits / kProducts, (j + 1) * kUnits / kProducts>(softmax);
        __builtin_amdgcn_sched_barrier(0);
      });

      k_at = k_address(copy_lane) + ((it + 1) & (kStages - 1)) * kStageBytes;
      if (run_tile == 0) {
        wait_vector<kInFlight + 1>();
      } else {
        wait_vector<kInFlight>();
      }
      lds_barrier();  // all waves' copies and weights are there; all are done with iteration it
      const int32_t moved_word = *reinterpret_cast<const int32_t *>(lds.moved[parity]);
      read_first(it + 1, k_at);
      const uint32_t moves = wave_uniform(moved_word);
      if (moves != 0) {
        mfma_pv_done(acc);
        static_for<0, kGroups>([&](auto cc) __attribute__((always_inline)) {
          constexpr int c = decltype(cc)::value;
          const float own = lds.alpha[parity][c][lane_now() & 31];
          const float factor = moves >> (8 * c) & 1 ? own : 1.0f;
#pragma unroll
          for (int d = 0; d < G::kDims; ++d) {
            acc[c * G::kDims + d] *= factor;
            asm volatile("" : "+a"(acc[c * G::kDims + d]));  // one at a time through VGPRs
          }
        });
        mfma_pv_done(acc);
      }
      // Pinned to AGPRs here too: the register allocator otherwise moves all sums to
      // VGPRs and back in every iteration, for the sake of the path above.
#pragma unroll
      for (int i = 0; i < kGroups * G::kDims; ++i) asm volatile("" : "+a"(acc[i]));
    }
    wait_copies();
    mfma_pv_done(acc);

    // ---- the rows' end ---------------------------------------------------------------
    const int end_lane = fresh_lane(), column = end_lane & 31, end_half = end_lane >> 5;
    l_run = xor_sum<32>(l_run);
    if (end_half == 0) lds.sums[wave][column] = l_run;
    __syncthreads();
    // Lane holds dims 32 (kDims w + d) + 8 i + 4 half .. + 3 of group c's column in
    // accumulators 4 i .. + 3. An infinity or NaN of V meets weight 0 too in the
    // products, in columns that do not see its key: a column whose sums are not all
    // finite is marked by each wave that has such sums, and the merge launch works it
    // out again from the keys that it sees.
    const int dim0 = 32 * G::kDims * wave, qh = column_head(column);
    static_for<0, kGroups>([&](auto cc) __attribute__((always_inline)) {
      constexpr int c = decltype(cc)::value;
      if (c * G::kWaveRows >= rows) return;
      const int row = column_row(c, column);
      float zero = 0.0f;  // stays that if all sums are finite
      if (partial < 0) {
        const float sum = lds.sums[c][column];
        const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
        uint16_t *o = p.out + (((int64_t)base + row0 + row) * kQueryHeads + qh) * kDim + dim0;
#pragma unroll
        for (int d = 0; d < G::kDims; ++d) {
          const f32x16_t &x = acc[c * G::kDims + d];
          uint2 words[4];
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            words[i / 4] = make_uint2(cvt_pk_bf16(x[i] * inv, x[i + 1] * inv),
                                      cvt_pk_bf16(x[i + 2] * inv, x[i + 3] * inv));
            zero = fmaf(x[i], 0.0f, fmaf(x[i + 1], 0.0f, zero));
            zero = fmaf(x[i + 2], 0.0f, fmaf(x[i + 3], 0.0f, zero));
          }
          if (row < rows) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<uint2 *>(o + 4 * end_half + 32 * d + 8 * i) = words[i];
          }
        }
        // The same lane stored this element above.
        if (xor_sum<32>(zero) != 0.0f && end_half == 0 && row < rows) *o = kExtendOdd;
      } else {
        // One wave's rows go to their places; more leave as they are, 1 KiB a store.
        const int64_t at =
            (int64_t)partial * kQueryHeads +
            (kGroups == 1 ? row * kQueryHeads + qh
                          : head * G::kGroup * ((rows + G::kWaveRows - 1) / G::kWaveRows *
                                                G::kWaveRows) + c * 32 + column);
        float *o = kGroups == 1
                       ? p.partial + at * kDim + dim0 + 4 * end_half
                       : p.partial + (at - column) * kDim + wave * (G::kDims * 1024) + 4 * end_lane;
#pragma unroll
        for (int d = 0; d < G::kDims; ++d) {
          const f32x16_t &x = acc[c * G::kDims + d];
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            if (kGroups > 1 || row < rows)
              *reinterpret_cast<float4 *>(o + (kGroups == 1 ? 32 * d + 2 * i : 1024 * d + 64 * i)) =
                  make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
            zero = fmaf(x[i], 0.0f, fmaf(x[i + 1], 0.0f, zero));
            zero = fmaf(x[i + 2], 0.0f, fmaf(x[i + 3], 0.0f, zero));
          }
        }
        if (wave == c && end_half == 0 && row < rows)
          *reinterpret_cast<float2 *>(p.stats + 2 * at) = make_float2(m_run, l_run);
        const uint64_t odd = __builtin_amdgcn_ballot_w64(zero != 0.0f);
        if (end_lane == 0)
          p.odd[((int64_t)(partial + c * G::kWaveRows) * G::kHeads + head) * kWaves + wave] =
              (uint32_t)odd | (uint32_t)(odd >> 32);
      }
    });
    };
    if (rows <= G::kWaveRows) {
      attend(std::integral_constant<int, 1>{});
    } else {
      attend(std::integral_constant<int, kWaves>{});
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
