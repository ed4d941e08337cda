// Row blocks of a few rows over the paged cache on bf16 MFMA, gfx950: tokens and drafts,
// a shared prefix under a group's tokens. Segments and partial sums are those of
// extend_rows.hip in blocks of one wave's rows; that kernel is made for long segments of
// many rows, and the start of its pipeline and the end of its 128 columns cost a short
// segment 7 to 12 us.
//
// Formulation: S^T = K Q^T and O^T = V^T P^T with v_mfma_f32_16x16x32_bf16 on 32 columns,
// (row, query head) pairs: 2 rows x 16 heads at 1 x 512, 16 rows x 2 heads at 8 x 256, in
// two blocks of 16 (one where the rows are half of that). A step is 64 keys, of which each
// of two teams of waves (4 at 512 dims, 2 at 256) has 32. A wave scores 16 of its team's
// keys, for one block of columns at 512 dims and both at 256. The team trades the weights
// through LDS, and each of its waves adds up 128 dims over the team's keys: V is read
// 256 bytes a row at a time, straight into registers, where two v_perm make the pairs of
// keys that an operand holds of two dims. K is read in whole rows and turned in LDS. The two
// teams' sums are joined at the segment's end, each team a block of columns.
//
// What bounds it: a step's 128 KB of K and V at 512 dims come out of the L2s at 14 TB/s
// in all, 2.4 us a step (0.7 of scores, 0.3 of weights, 0.7 of products with V, 0.3 of them
// of the weights' second halves, 0.6 of waiting for K and storing it); a segment's way to its first keys
// takes 3.6 us, by way of the plan, the page table and the rows, and its end 2.2. Two waves
// a SIMD because one, with all 512 registers, took 2.9 us a step: its phases, each on another
// unit, passed one after the other. The loads of the next K go out between the scores'
// products and those of V between V's: in one piece they held the waves up, 2.5 us a step.
//
// Keys that no row of the block sees, or that no page maps, are read from a row of zeros.
// An infinity or NaN of V in a key that one row sees and another does not meets weight 0
// in the products: columns whose sums are not all finite are marked, as there, and the
// merge launch works them out again.
#include "extend_few.hpp"
#include "lds_copy.hpp"

#include <math.h>

#include <type_traits>

namespace gemma4 {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x4v_t __attribute__((ext_vector_type(4)));

constexpr int kStep = 64;                      // keys of a step
constexpr int kColumns = 16;                   // of a block
constexpr float kRescaleSlack = 8.0f;          // log2 headroom of the running maximum
static_assert(kFew256.tile == kStep && kFew512.tile == kStep);

// What keys that are not there are read from: as long as the longest row.
__device__ uint4 g_zero_rows[64];

__device__ __forceinline__ uint4 load_pack(uint64_t at, uint32_t pack = 0) {
  return __builtin_bit_cast(
      uint4, reinterpret_cast<const __attribute__((address_space(1))) u32x4v_t *>(at)[pack]);
}

template <int kDim>
struct Few {
  static constexpr int kHeads = kDim == 256 ? 8 : 1;
  static constexpr int kGroup = kQueryHeads / kHeads;
  static constexpr int kBlockRows = kColumns / kGroup;  // rows of a block of columns
  static constexpr int kTeam = kDim / 128;              // waves of a team
  static constexpr int kWaves = 2 * kTeam;
  static constexpr int kThreads = kWaves * kWave;
  static constexpr int kScored = 4 / kTeam;             // blocks of columns that a wave scores
  static constexpr int kChunks = kDim / 8;              // 16-byte chunks of a row
  static constexpr int kRows = kStep / kWaves;          // rows of K that a wave reads
  static constexpr int kLoads = kRows * kChunks / kWave;
  static constexpr int kTokenBytes = kHeads * kDim * 2;
};

template <int kDim>
__global__ __launch_bounds__(Few<kDim>::kThreads) void extend_few_kernel(ExtendParams p) {
  using F = Few<kDim>;
  struct Lds {
    uint4 k[kStep * F::kChunks];              // key r's chunk c at c ^ (r % 16)
    uint4 q[2 * kColumns][F::kChunks];        // column n's chunk c at c ^ (n % 16)
    uint4 weights[2][2][2][kWave];            // operands of P^T: by team, block of columns, the
                                              // nearest bf16 of a weight and the rest
    uint64_t k_rows[F::kWaves][kStep];
    uint64_t v_rows[F::kWaves][kStep];
    float top[2][2][2 * kColumns];            // by team and half of its keys
    float l[2][2][2 * kColumns];
  };
  __shared__ __attribute__((aligned(1024))) Lds lds;

  const int thread_lane = threadIdx.x & (kWave - 1);
  const int wave = wave_uniform(threadIdx.x / kWave);
  const int team = wave / F::kTeam, slice = wave % F::kTeam;
  // The 16 of the team's 32 keys, and the blocks of columns, that the wave scores.
  const int half = slice % 2, block0 = F::kScored == 1 ? slice / 2 : 0;
  // As in extend_rows_kernel: an XCD gets a KV head, or a run of shares.
  constexpr int kShares = kDim == 256 ? kFew256.shares : kFew512.shares;
  const int head = blockIdx.x % F::kHeads;
  const int share = F::kHeads == 1 ? blockIdx.x % 8 * (kShares / 8) + blockIdx.x / 8
                                   : blockIdx.x / F::kHeads;
  const ExtendShare mine =
      plan_read<ExtendShare>(p.plan + p.shares + (int64_t)share * sizeof(ExtendShare));
  const ExtendHeader header = plan_read<ExtendHeader>(p.plan);
  if (!extend_plan_fits(p, header)) return;

  const int32_t max_pages = p.c.max_pages_per_seq;
  const uint64_t layer_bytes =
      (uint64_t)p.layer * p.c.num_pages * p.c.page_size * F::kTokenBytes + head * (kDim * 2);
  const uint64_t cache_k = reinterpret_cast<uint64_t>(p.cache_k) + layer_bytes;
  const uint64_t cache_v = reinterpret_cast<uint64_t>(p.cache_v) + layer_bytes;
  const uint64_t zero_row = reinterpret_cast<uint64_t>(&g_zero_rows[0]);
  const uint32_t kv_bytes = (uint32_t)(p.kv_stride * 2);
  for (int32_t segment = mine.first; segment < mine.end; ++segment) {
    int lane = thread_lane;
    asm volatile("" : "+v"(lane));  // what follows from it is worked out again, not spilled
    const int h = lane & 15, g = lane >> 4;
    // Lane h's chunk of V within the wave's 128 dims: the products' rows 4 g + i are chunks
    // 4 i + g, and the lanes of a column store next to each other.
    const int v_chunk = h % 4 * 4 + h / 4;
    ExtendSegment seg = mine.segment;
    if (segment != mine.first)
      seg = plan_read<ExtendSegment>(p.plan + p.segments + (int64_t)segment * sizeof(ExtendSegment));
    const int32_t rows = seg.rows, prior = seg.prior, partial = seg.partial;
    const int32_t first = prior + seg.row0, last = first + rows - 1;  // positions
    const int n_steps = seg.tile_hi - seg.tile_lo;
    const int32_t key_lo = seg.tile_lo * kStep;

    // ---- where the keys are: lane l has key l of a step --------------------------------
    const int32_t *table = p.page_table + (int64_t)seg.sequence * max_pages;
    const uint64_t chunk_off = (uint64_t)seg.base * kv_bytes + head * (kDim * 2);
    const uint64_t chunk_k = reinterpret_cast<uint64_t>(p.k) + chunk_off;
    const uint64_t chunk_v = reinterpret_cast<uint64_t>(p.v) + chunk_off;
    // Table entry of this lane's key; any readable one for a new key.
    auto page_entry = [&](int n) __attribute__((always_inline)) -> int32_t {
      const uint32_t key = (uint32_t)(key_lo + n * kStep + lane);
      const uint32_t at = (uint32_t)max(min((int32_t)key, prior - 1), 0);
      return table[fast_mod(fast_div(at, p.page_div), p.slot_div)];
    };
    uint64_t valid = 0, k_row = 0;
    auto resolve = [&](int n, int32_t page) __attribute__((always_inline)) {
      const int32_t key = key_lo + n * kStep + lane;
      const bool fresh = key >= prior;
      const uint32_t logical = fast_div((uint32_t)key, p.page_div);
      const bool mapped =
          ((uint32_t)page < (uint32_t)p.c.num_pages) & (logical < (uint32_t)max_pages);
      const bool ok = (key <= last) & (fresh | mapped);
      const uint32_t cached =
          (uint32_t)page * p.page_div.d + ((uint32_t)key - logical * p.page_div.d);
      const uint64_t off = fresh ? (uint64_t)(uint32_t)(key - prior) * kv_bytes
                                 : (uint64_t)cached * F::kTokenBytes;
      // Sums, where a choice between two captured values would become a load of one.
      const uint64_t from = fresh ? ~0ull : 0ull;
      k_row = ok ? cache_k + (from & (chunk_k - cache_k)) + off : zero_row;
      if constexpr (F::kChunks != kWave) lds.k_rows[wave][lane] = k_row;
      lds.v_rows[wave][lane] = ok ? cache_v + (from & (chunk_v - cache_v)) + off : zero_row;
      valid = __builtin_amdgcn_ballot_w64(ok);
      wave_lds_fence();
    };
    uint4 k_pack[F::kLoads], v_pack[8];
    auto load_k = [&](int from, int to) __attribute__((always_inline)) {
#pragma unroll
      for (int i = from; i < to; ++i) {
        if constexpr (F::kChunks == kWave) {  // one row: its address in scalar registers
          const uint64_t row = k_row;
          const uint32_t low = __builtin_amdgcn_readlane((uint32_t)row, F::kRows * wave + i);
          const uint32_t high = __builtin_amdgcn_readlane((uint32_t)(row >> 32), F::kRows * wave + i);
          k_pack[i] = load_pack((uint64_t)high << 32 | low, lane);
        } else {
          const int at = i * kWave + lane;  // chunk of the wave's rows
          k_pack[i] = load_pack(lds.k_rows[wave][F::kRows * wave + at / F::kChunks] +
                                16 * (at % F::kChunks));
        }
      }
    };
    auto store_k = [&]() __attribute__((always_inline)) {
      // Chunk lane % kChunks of row r = kRows wave + i rows + lane / kChunks: in bytes, so that
      // one register and an xor make the eight addresses.
      const uint32_t r0 = F::kRows * wave + lane / F::kChunks;
      const uint32_t k_at = (r0 * F::kChunks + (lane % F::kChunks ^ r0 % 16)) * 16;
#pragma unroll
      for (int i = 0; i < F::kLoads; ++i) {
        constexpr int kEach = kWave / F::kChunks;  // rows of a load
        *reinterpret_cast<uint4 *>(reinterpret_cast<char *>(&lds.k[0]) + (k_at ^ 16 * kEach * i) +
                                   i * kWave * 16) = k_pack[i];
      }
    };
    // V of the team's keys 4 g .. + 3 and 16 + 4 g .. + 3.
    auto load_v = [&](int from, int to) __attribute__((always_inline)) {
      const int key = 32 * team + 4 * g;
#pragma unroll
      for (int i = from; i < to; ++i)
        v_pack[i] = load_pack(lds.v_rows[wave][key + (i < 4 ? i : 12 + i)] + 256 * slice +
                              16 * v_chunk);
    };
    // ---- queries: column n of block c is row c * kBlockRows + .., see below --------------
    auto column_row = [&](int c, int n) __attribute__((always_inline)) -> int {
      return c * F::kBlockRows + (F::kGroup == 2 ? n % 8 : 0);
    };
    auto column_head = [&](int n) __attribute__((always_inline)) -> int {
      return F::kGroup == 2 ? n / 8 : n;
    };
    const int blocks = rows > F::kBlockRows ? 2 : 1;
    constexpr int kPerWave = 2 * kColumns * F::kChunks / kWave / F::kWaves;
    uint4 q[kPerWave];
    const int32_t page_first = page_entry(0);
    int32_t page_next = page_entry(1);
#pragma unroll
    for (int i = 0; i < kPerWave; ++i) {
      const int at = (i * F::kWaves + wave) * kWave + lane, column = at / F::kChunks;
      const int row = column_row(column / kColumns, column % kColumns);
      q[i] = load128(p.q + ((int64_t)seg.base + seg.row0 + (row < rows ? row : 0)) * p.q_stride +
                     (head * F::kGroup + column_head(column % kColumns)) * kDim +
                     at % F::kChunks * 8);
    }
    resolve(0, page_first);
    load_k(0, F::kLoads);
    load_v(0, 8);
#pragma unroll
    for (int i = 0; i < kPerWave; ++i) {
      const int at = (i * F::kWaves + wave) * kWave + lane, column = at / F::kChunks;
      lds.q[column][at % F::kChunks ^ (column % kColumns)] = q[i];
    }
    store_k();
    lds_barrier();

    auto attend = [&](auto block_count) __attribute__((always_inline)) {
      constexpr int kBlocks = decltype(block_count)::value;
      f32x4_t acc[kBlocks][8];
      constexpr int kScored = F::kScored < kBlocks ? F::kScored : kBlocks;
      float m_run[kBlocks], l_run[kScored];
      int32_t limit[kScored];  // the last key that the column sees
#pragma unroll
      for (int c = 0; c < kBlocks; ++c) {
#pragma unroll
        for (int d = 0; d < 8; ++d) acc[c][d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        m_run[c] = -INFINITY;
      }
#pragma unroll
      for (int c = 0; c < kScored; ++c) {
        l_run[c] = 0.0f;
        const int row = column_row(block0 + c, h);
        limit[c] = row < rows ? first + row : -1;
      }
      const bool scores = block0 < kBlocks;
      uint64_t valid_next = valid;
      auto step = [&](int n, auto more) __attribute__((always_inline)) {
        constexpr bool kMore = decltype(more)::value;
        const int key = 32 * team + 16 * half;  // the first of the wave's, within the step
        const uint32_t there = (uint32_t)(valid_next >> (key + 4 * g));
        const int32_t key0 = key_lo + n * kStep + key + 4 * g;
        if constexpr (kMore) {
          resolve(n + 1, page_next);
          valid_next = valid;
        }
        // ---- scores: key h of the wave's, dims 32 s + 8 g .. + 7 of step s
        float x[kScored][4];
        if (scores) {
          constexpr int kChains = kScored == 1 ? 2 : 1;
          f32x4_t score[kScored][kChains];
#pragma unroll
          for (int c = 0; c < kScored; ++c)
#pragma unroll
            for (int i = 0; i < kChains; ++i) score[c][i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
          // Operands are read a step ahead; the loads of the next K go out between the products,
          // as fast as the memory pipeline takes them.
          constexpr int kSteps = kDim / 32, kEvery = kSteps / F::kLoads;
          uint4 k_op[2], q_op[2][kScored];
          const uint4 *k_tile = &lds.k[(key + h) * F::kChunks], *q_tile = &lds.q[kColumns * block0 + h][0];
          auto operands = [&](int s) __attribute__((always_inline)) {
            const int at = s / 4 * 16 + ((s % 4 * 4 + g) ^ h);
            k_op[s % 2] = k_tile[at];
#pragma unroll
            for (int c = 0; c < kScored; ++c) q_op[s % 2][c] = q_tile[kColumns * F::kChunks * c + at];
          };
          operands(0);
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            if (s + 1 < kSteps) operands(s + 1);
            if constexpr (kMore)
              if (s % kEvery == 0) load_k(s / kEvery, s / kEvery + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int c = 0; c < kScored; ++c)
              score[c][s % kChains] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                  __builtin_bit_cast(bf16x8_t, k_op[s % 2]), __builtin_bit_cast(bf16x8_t, q_op[s % 2][c]),
                  score[c][s % kChains], 0, 0, 0);
          }
#pragma unroll
          for (int c = 0; c < kScored; ++c) {
            if constexpr (kChains == 2) score[c][0] += score[c][1];
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const bool seen = (there >> i & 1u) && key0 + i <= limit[c];
              x[c][i] = seen ? score[c][0][i] * p.q_scale : -INFINITY;
              top = fmaxf(top, x[c][i]);
            }
            top = xor_max<32>(xor_max<16>(top));
            if (g == 0) lds.top[team][half][kColumns * (block0 + c) + h] = top;
          }
        } else if constexpr (kMore) {
          load_k(0, F::kLoads);
        }
        if constexpr (kMore) page_next = page_entry(n + 2);
        lds_barrier();
        // ---- one maximum for the team's keys
#pragma unroll
        for (int c = 0; c < kBlocks; ++c) {
          const float top = fmaxf(lds.top[team][0][kColumns * c + h], lds.top[team][1][kColumns * c + h]);
          if (__builtin_amdgcn_ballot_w64(top > m_run[c] + kRescaleSlack) != 0) {
            const float m_new = fmaxf(m_run[c], top);
            const float alpha = m_run[c] == m_new ? 1.0f : __builtin_amdgcn_exp2f(m_run[c] - m_new);
            m_run[c] = m_new;
            if (c >= block0 && c < block0 + kScored) l_run[F::kScored == 1 ? 0 : c] *= alpha;
#pragma unroll
            for (int d = 0; d < 8; ++d) acc[c][d] *= alpha;
          }
        }
        if (scores) {
#pragma unroll
          for (int c = 0; c < kScored; ++c) {
            const float m = kScored < kBlocks && block0 == 1 ? m_run[kBlocks - 1] : m_run[c];
            const float m_use = m == -INFINITY ? 0.0f : m;
            // A weight is the sum of two bf16, off by 2^-17 of it, as in the decode kernels whose
            // rows may come here: one alone, off by 2^-8, left the outputs 0.0020 to 0.0023 of their
            // norm from the 64-bit result, 0.0017 so. The second product of V costs 1 to 2%
            // where few keys are shared, 7% of 32 tokens after 8000 shared keys at 1 x 512 (35.3
            // to 37.9 us), 11% of 64.
            float w[4];
            uint32_t nearest[2], rest[2];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              w[i] = __builtin_amdgcn_exp2f(x[c][i] - m_use);
              l_run[c] += w[i];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              nearest[i] = cvt_pk_bf16(w[2 * i], w[2 * i + 1]);
              rest[i] = cvt_pk_bf16(w[2 * i] - bf16_lo(nearest[i]), w[2 * i + 1] - bf16_hi(nearest[i]));
            }
            auto &to = lds.weights[team][block0 + c];
            reinterpret_cast<uint2 *>(&to[0][lane])[half] = make_uint2(nearest[0], nearest[1]);
            reinterpret_cast<uint2 *>(&to[1][lane])[half] = make_uint2(rest[0], rest[1]);
          }
        }
        lds_barrier();
        // ---- the wave's dims over the team's keys
        bf16x8_t nearest[kBlocks];
#pragma unroll
        for (int c = 0; c < kBlocks; ++c)
          nearest[c] = __builtin_bit_cast(bf16x8_t, lds.weights[team][c][0][lane]);
        auto word = [](const uint4 &x4, int w) __attribute__((always_inline)) -> uint32_t {
          return w == 0 ? x4.x : (w == 1 ? x4.y : (w == 2 ? x4.z : x4.w));
        };
        u32x4v_t low[4], high[4];  // dims 2 w and 2 w + 1 of eight keys
#pragma unroll
        for (int w = 0; w < 4; ++w) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t a = word(v_pack[2 * i], w), e = word(v_pack[2 * i + 1], w);
            low[w][i] = __builtin_amdgcn_perm(e, a, 0x05040100u);
            high[w][i] = __builtin_amdgcn_perm(e, a, 0x07060302u);
          }
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          if constexpr (kMore) load_v(2 * w, 2 * w + 2);
          bf16x8_t rest[kBlocks];  // read for every pair of dims: held all along they would be spilled
          uint32_t from = lane;
          asm volatile("" : "+v"(from));
#pragma unroll
          for (int c = 0; c < kBlocks; ++c)
            rest[c] = __builtin_bit_cast(bf16x8_t, lds.weights[team][c][1][from]);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int c = 0; c < kBlocks; ++c) {
            acc[c][2 * w] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                __builtin_bit_cast(bf16x8_t, low[w]), nearest[c], acc[c][2 * w], 0, 0, 0);
            acc[c][2 * w + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                __builtin_bit_cast(bf16x8_t, high[w]), nearest[c], acc[c][2 * w + 1], 0, 0, 0);
          }
#pragma unroll
          for (int c = 0; c < kBlocks; ++c) {
            acc[c][2 * w] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                __builtin_bit_cast(bf16x8_t, low[w]), rest[c], acc[c][2 * w], 0, 0, 0);
            acc[c][2 * w + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                __builtin_bit_cast(bf16x8_t, high[w]), rest[c], acc[c][2 * w + 1], 0, 0, 0);
          }
        }
        if constexpr (kMore) {
          store_k();
          // At 256 dims a wave reads its own rows.
          if constexpr (F::kScored == 1) lds_barrier(); else wave_lds_fence();
        }
      };
      int n = 0;
      for (; n + 1 < n_steps; ++n) step(n, std::true_type{});
      step(n, std::false_type{});

      asm volatile("" : "+v"(lane));
      const int h = lane & 15, g = lane >> 4;
      // ---- the rows' end: a team finishes a block of columns, with the other's sums of it,
      // which pass through the K tile ----------------------------------------------------
#pragma unroll
      for (int c = 0; c < kScored; ++c) {
        l_run[c] = xor_sum<32>(xor_sum<16>(l_run[c]));
        if (scores && g == 0) lds.l[team][half][kColumns * (block0 + c) + h] = l_run[c];
      }
#pragma unroll
      for (int c = 0; c < kBlocks; ++c)
        if (slice == 0 && g == 0) lds.top[team][0][kColumns * c + h] = m_run[c];
      // A wave's sums there: 16 columns of 32 chunks of four dims, chunk j of column n at j ^ n.
      f32x4_t *const mine_at = reinterpret_cast<f32x4_t *>(&lds.k[0]) + wave * (kColumns * 32);
      f32x4_t *const other_at = reinterpret_cast<f32x4_t *>(&lds.k[0]) + (wave ^ F::kTeam) * (kColumns * 32);
      static_assert(sizeof(lds.k) >= sizeof(f32x4_t) * F::kWaves * kColumns * 32, "fits");
      // Lane (g, h) holds dims 128 slice + 32 i + 8 g + d of column h in acc[..][d][i].
      auto chunk_at = [&](int i, int upper) __attribute__((always_inline)) {
        return h * 32 + ((8 * i + 2 * g + upper) ^ h);
      };
      f32x4_t o[4][2];  // dims 4 upper .. + 3 of i
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int upper = 0; upper < 2; ++upper) {
          f32x4_t give;
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const float first = acc[0][4 * upper + d][i], second = acc[kBlocks - 1][4 * upper + d][i];
            o[i][upper][d] = team == 0 ? first : second;
            give[d] = team == 0 ? second : first;
          }
          if (kBlocks == 2 || team == 1) mine_at[chunk_at(i, upper)] = give;
        }
      lds_barrier();
      if (kBlocks == 2 || team == 0) {
        const int c = kBlocks == 2 ? team : 0, n = kColumns * c + h;
        const float m_own = lds.top[team][0][n], m_other = lds.top[1 - team][0][n];
        const float m = fmaxf(m_own, m_other);
        // A team without a visible key has nothing to add, whatever its sums are. (Not one whose
        // only scores are NaN: its l is.)
        const float l_own = lds.l[team][0][n] + lds.l[team][1][n];
        const float l_other = lds.l[1 - team][0][n] + lds.l[1 - team][1][n];
        const bool adds_own = l_own != 0.0f, adds_other = l_other != 0.0f;
        float own = m_own == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_own - m);
        float other = m_other == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_other - m);
        const float l = l_own * own + l_other * other;
        if (partial < 0) {
          const float inv = l > 0.0f ? 1.0f / l : 0.0f;
          own *= inv;
          other *= inv;
        }
        f32x4_t given[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int upper = 0; upper < 2; ++upper) given[i][upper] = other_at[chunk_at(i, upper)];
        f32x4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};  // stays that if all sums are finite
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int upper = 0; upper < 2; ++upper)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
              const float x = (adds_own ? o[i][upper][d] * own : 0.0f) +
                              (adds_other ? given[i][upper][d] * other : 0.0f);
              o[i][upper][d] = x;
              zero[d] = fmaf(x, 0.0f, zero[d]);
            }
        const int row = column_row(c, h);
        const int64_t at = (int64_t)(partial + row) * kQueryHeads + head * F::kGroup + column_head(h);
        const uint64_t marks =
            __builtin_amdgcn_ballot_w64((zero[0] + zero[1]) + (zero[2] + zero[3]) != 0.0f);
        const uint32_t odd = (uint32_t)(marks | marks >> 16 | marks >> 32 | marks >> 48) & 0xFFFFu;
        if (partial < 0) {
          uint16_t *out = p.out + (((int64_t)seg.base + seg.row0 + row) * kQueryHeads +
                                   head * F::kGroup + column_head(h)) * kDim + 128 * slice + 8 * g;
          if (row < rows) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              store128(out + 32 * i, make_uint4(cvt_pk_bf16(o[i][0][0], o[i][0][1]),
                                                cvt_pk_bf16(o[i][0][2], o[i][0][3]),
                                                cvt_pk_bf16(o[i][1][0], o[i][1][1]),
                                                cvt_pk_bf16(o[i][1][2], o[i][1][3])));
            // The same lane stored this element above.
            if ((odd >> h & 1u) && g == 0) *out = kExtendOdd;
          }
        } else {
          if (row < rows && slice == 0 && g == 0)
            *reinterpret_cast<float2 *>(p.stats + 2 * at) = make_float2(m, l);
          if constexpr (kDim == 256) {
            if (row < rows) {
#pragma unroll
              for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int upper = 0; upper < 2; ++upper)
                  *reinterpret_cast<f32x4_t *>(p.partial + at * kDim + 128 * slice + 32 * i + 8 * g +
                                               4 * upper) = o[i][upper];
            }
          } else {
            // By columns, once more through LDS: 512 contiguous bytes a store, which takes
            // half the time of 16 bytes in each of 64 places (2.1 us of a share's end to
            // 1.6); at 256 dims, of half as many, it would cost 0.5 more.
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int upper = 0; upper < 2; ++upper) other_at[chunk_at(i, upper)] = o[i][upper];
            wave_lds_fence();
            f32x4_t out[kColumns / 2];
#pragma unroll
            for (int j = 0; j < kColumns / 2; ++j) {
              const int column = 2 * j + lane / 32;
              out[j] = other_at[column * 32 + (lane % 32 ^ column)];
            }
            if (c < rows) {
#pragma unroll
              for (int j = 0; j < kColumns / 2; ++j)
                *reinterpret_cast<f32x4_t *>(
                    p.partial + ((int64_t)(partial + c) * kQueryHeads + 2 * j + lane / 32) * kDim +
                    128 * slice + lane % 32 * 4) = out[j];
            }
          }
        }
        if (partial >= 0 && lane == 0) {
          uint32_t *words = p.odd + ((int64_t)partial * F::kHeads + head) * 4;
          if constexpr (F::kGroup == 2) {  // a word of the four for each slice and block
            words[2 * c + slice] = (odd & 0xFFu) << (8 * c) | (odd >> 8) << (16 + 8 * c);
            if (kBlocks == 1) words[2 + slice] = 0;
          } else if (kBlocks == 1) {
            words[slice] = odd;
          } else {
            reinterpret_cast<uint16_t *>(words)[2 * slice + c] = (uint16_t)odd;
          }
        }
      }
    };
    if (blocks == 1) {
      attend(std::integral_constant<int, 1>{});
    } else {
      attend(std::integral_constant<int, 2>{});
    }
    lds_barrier();  // the next segment's rows overwrite what this one's are read from
  }
}

}  // namespace

void launch_extend_few(const ExtendParams &p, hipStream_t stream) {
  if (p.c.num_heads == 1) {
    hipLaunchKernelGGL(extend_few_kernel<512>, dim3(kFew512.shares), dim3(Few<512>::kThreads), 0,
                       stream, p);
  } else {
    hipLaunchKernelGGL(extend_few_kernel<256>, dim3(Few<256>::kHeads * kFew256.shares),
                       dim3(Few<256>::kThreads), 0, stream, p);
  }
}

}  // namespace gemma4
