// Paged split-K decode attention over the quantised cache (e4m3 codes with a scale
// per layer and KV head), gfx950, with the optional append of the token's row. No
// counterpart in the reference, whose cache is bf16; the partials and the combine
// launch are those of the bf16 decode (decode_attention.hip).
//
//   o = s_v sum_j w_j v_j / sum_j w_j,  w_j = 2^(x_j - m),  x_j = log2(e) scale s_k q.k_j
//
// The scales of K and V are one number each for a head: they go into the scores'
// factor and the sums' end, and the loop sees codes only. A code becomes a bf16
// operand exactly (v_cvt_scalef32_pk_bf16_fp8, two a time), so both products run on
// v_mfma_f32_16x16x32_bf16 with nothing rounded but the weights, which go in as two
// bf16 numbers, the nearest and the rest (2^-17 of a weight). The matrix instructions of
// 8-bit operands would need no conversions, but add up their products to within 2^-12.8
// of sum |ab| only (measured; bf16 ones 2^-22): in the exponent of a score of 40 that is
// 0.6% of a weight.
//
// What bounds it: HBM where there are keys enough. 48 sequences of 512 to 16 384 keys at 8 x 256
// (1.5 GB) 259 us, 5.9 TB/s; 24 of 200 to 12 000 at 1 x 512 (124 MB) 33 us, 6.6 TB/s in the
// 18 that it streams, with 2 to the first loads, 3 to join the waves' sums, and the combine;
// one of 1024 at 8 x 256 8.4 as a graph, two launches' latency.
//
// Workgroup (KV head, split, sequence); a wave takes 32-key tiles of its own and
// holds all dims' sums, the waves merge once at the end.
//   K     a tile's rows are read whole (16 lanes x 16 bytes a row segment) and turned in
//         the wave's own LDS: lane (g, h) = (l / 16, l % 16) scores key 16 b + h from
//         chunks 4 j + g; chunk c of key r lies at c ^ (r % 16), no bank conflict.
//   S^T   lane (g, h) receives head h's scores of keys 4 g .. + 3 and 16 + 4 g .. + 3:
//         the eight k-slots it supplies to the second product. Nothing is exchanged.
//   V     lane (g, c) reads chunk c of just these eight keys, whole rows again. Byte d of
//         the eight is the operand row of dim 16 c + d: product d covers dims d, 16 + d,
//         .. and its operand comes from two v_perm and four conversions for each pair of
//         keys and four dims, with no trip through LDS.
// The loads of K for the next tile go out as soon as this tile's K is in LDS, those of
// V after this tile's products: one of the two is always on its way.
#include "decode_common.hpp"
#include "fast_div.hpp"
#include "fp8_common.hpp"
#include "gemma4_device.hpp"
#include "lds_copy.hpp"

#include "gemma4_flash_attention.h"

#include <math.h>
#include <stddef.h>

#include <algorithm>
#include <type_traits>

namespace gemma4 {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x4v_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x2v_t __attribute__((ext_vector_type(2)));

constexpr int kTile = 32;              // keys of a wave's tile
constexpr int kLaneKeys = 8;           // of them, a lane's
constexpr float kRescaleSlack = 8.0f;  // log2 headroom of the running maximum

// A nontemporal load from an address that was computed as a number. The address space is
// said, or the loads are flat ones: those count as LDS accesses too, and every wait for
// LDS is one for all of them (one sequence of 8193 keys at 8 x 256: 13.8 us, 13.0 so).
template <class T>
__device__ __forceinline__ T load_from(uint64_t at) {
  return __builtin_nontemporal_load(reinterpret_cast<const __attribute__((address_space(1))) T *>(at));
}
__device__ __forceinline__ uint4 load_pack(uint64_t at) {
  return __builtin_bit_cast(uint4, load_from<u32x4v_t>(at));
}

// What keys that are not there are read from: as long as the longest row.
__device__ uint4 g_zero_codes[32];

struct Fp8DecodeParams {
  uint16_t *out;
  float *partial_m;
  float *partial_l;
  float *partial_acc;
  const uint16_t *q;
  uint8_t *cache_k;  // written only by the append
  uint8_t *cache_v;
  const float *k_scales;
  const float *v_scales;
  const int32_t *page_table;
  const int32_t *seq_lengths;
  const int32_t *token_position;  // null: no append
  const uint16_t *new_k;
  const uint16_t *new_v;
  Gemma4KvCacheConfig c;
  FastDiv page_div, slot_div;
  int32_t layer;
  float q_scale;  // softmax_scale * log2(e)
  int32_t split_size;
  int32_t num_splits;
  // Nonzero: the number of KV heads, and sequences (`batch` of them, up to 64) are cut by
  // their lengths (Fp8Cut); the grid's splits are those of all of them.
  int32_t balanced;
  int32_t batch;
};
__device__ __forceinline__ int32_t window_of(const Fp8DecodeParams &p) { return p.c.window_size; }

template <int kDim>
struct Fp8Shape {
  static constexpr int kHeads = kDim == 256 ? 8 : 1;
  static constexpr int kGroup = kQueryHeads / kHeads;  // query heads of a KV head
  static constexpr int kParts = kDim / 256;            // 256-byte segments of a row
  static constexpr int kSteps = kDim / 64;             // pairs of S^T steps
  static constexpr int kChunks = kDim / 16;
};

// What a workgroup of (KV head, split, sequence) attends to, and where its keys are. A key
// is a position, or, in a ring of just the window's slots, a slot: a full ring's are
// all live, and until it is full they are the positions. So the first page-table entries
// can be asked for without the length, but in rings of more slots than the window has.
template <int kDim>
struct Fp8Split {
  const Fp8DecodeParams &p;
  int32_t head, split, b;
  int32_t split_size, seq_word, tok_word;
  bool dead = false;   // balanced: no split is left for this workgroup
  const int32_t *table;
  int32_t first, key_count, token_pos;
  int32_t token_key = -1;  // the key that is being appended, -1: not among the live ones
  bool owns = false;       // this split writes the token's row

  // What depends on the arguments alone (and, balanced, on the lengths): the words are on
  // their way.
  __device__ __forceinline__ Fp8Split(const Fp8DecodeParams &params) : p(params) {
    head = blockIdx.x;
    split = blockIdx.y;
    b = blockIdx.z;
    split_size = p.split_size;
    if (p.balanced != 0) {
      // Workgroup n serves the n-th split in sequence order.
      uint32_t upto;  // splits of sequences 0 .. lane
      const BalancedCut cut = Fp8Cut<kDim>::cut(p, lane_live_keys(p), upto);
      const int32_t n = split;
      b = __builtin_popcountll(__builtin_amdgcn_ballot_w64((int32_t)upto <= n));
      dead = b >= p.batch;
      b = dead ? 0 : b;
      split = n - (b > 0 ? __builtin_amdgcn_readlane(upto, b - 1) : 0);
      split_size = cut.size;
    }
    table = p.page_table + (int64_t)b * p.c.max_pages_per_seq;
    seq_word = p.seq_lengths[b];
    tok_word = p.token_position != nullptr ? p.token_position[b] : -1;
  }
  __device__ __forceinline__ bool early() const {
    return p.c.window_size == 0 || slots() == p.c.window_size;
  }
  __device__ __forceinline__ int64_t slots() const {
    return (int64_t)p.c.max_pages_per_seq * p.c.page_size;
  }
  __device__ __forceinline__ void finish() {
    const Gemma4KvCacheConfig &c = p.c;
    const int32_t seq_len = wave_uniform(seq_word);
    token_pos = wave_uniform(tok_word);
    const int32_t low = c.window_size > 0 ? max(seq_len - c.window_size, 0) : 0;
    // The plan's splits bound the keys, however the launch cuts them.
    const int32_t capacity =
        (int32_t)min((int64_t)p.split_size * p.num_splits, (int64_t)0x7fffffff);
    key_count = min(seq_len > low ? seq_len - low : 0, capacity);
    first = early() ? 0 : low;
    // The split that holds the token's key writes its row (split 0 where the position is
    // not among the live keys), by the skip rules of the append.
    if (p.token_position != nullptr) {
      const bool droppable =
          token_pos < 0 || (c.window_size == 0 && token_pos / c.page_size >= c.max_pages_per_seq);
      if (!droppable && token_pos >= low && token_pos < seq_len) {
        const int32_t key = early() && c.window_size > 0 ? token_pos % c.window_size : token_pos;
        if (key < first + key_count) token_key = key;
      }
      owns = !droppable && split == (token_key >= 0 ? (token_key - first) / split_size : 0);
      if (!owns) token_key = -1;
    }
  }
  __device__ __forceinline__ bool live() const {
    return split < (int32_t)(((uint32_t)key_count + (uint32_t)split_size - 1) / (uint32_t)split_size);
  }
  __device__ __forceinline__ int32_t begin() const { return first + split * split_size; }
  __device__ __forceinline__ int32_t end() const {
    return (int32_t)min((uint32_t)(first + key_count), (uint32_t)begin() + (uint32_t)split_size);
  }
  // Row of a position, -1 where no page is mapped.
  __device__ __forceinline__ int32_t row_of(int32_t key, int32_t page) const {
    const int32_t in_page = key - (int32_t)(fast_div((uint32_t)key, p.page_div) * p.page_div.d);
    return (uint32_t)page < (uint32_t)p.c.num_pages
               ? (p.layer * p.c.num_pages + page) * p.c.page_size + in_page : -1;
  }
  __device__ __forceinline__ const int32_t *entry_of(int32_t key) const {
    return table + fast_mod(fast_div((uint32_t)key, p.page_div), p.slot_div);
  }
  // Key i of the split, as far as it is known before the length: any key else.
  __device__ __forceinline__ const int32_t *early_entry(int64_t i) const {
    return entry_of((int32_t)min((int64_t)split * split_size + i, (int64_t)0x7fffffff));
  }
  // The row of a key that is the split's and that the table reaches, else -1.
  __device__ __forceinline__ int32_t live_row(int32_t key, int32_t page, int32_t end) const {
    const bool reached = p.c.window_size > 0 || fast_div((uint32_t)key, p.page_div) <
                                                    (uint32_t)p.c.max_pages_per_seq;
    return key < end && reached ? row_of(key, page) : -1;
  }
  // The token's codes, by one wave: 4 dims a lane; to LDS and its cache row.
  __device__ __forceinline__ void quantise_token(uint32_t (&codes)[2][kDim / 4], float k_scale,
                                                 float v_scale) const {
    constexpr int kHeads = Fp8Shape<kDim>::kHeads;
    const int lane = __lane_id();
    const int64_t from = ((int64_t)b * kHeads + head) * kDim;
    const int32_t row = row_of(token_pos, *entry_of(token_pos));
#pragma unroll
    for (int part = 0; part < kDim / 256; ++part) {
      const int64_t at = from + part * 256 + 4 * lane;
      const uint2 k = *reinterpret_cast<const uint2 *>(p.new_k + at);
      const uint2 v = *reinterpret_cast<const uint2 *>(p.new_v + at);
      const uint32_t kc = fp8_word(k.x, k.y, k_scale), vc = fp8_word(v.x, v.y, v_scale);
      codes[0][part * 64 + lane] = kc;
      codes[1][part * 64 + lane] = vc;
      if (row >= 0) {
        const int64_t to = ((int64_t)row * kHeads + head) * kDim + part * 256 + 4 * lane;
        *reinterpret_cast<uint32_t *>(p.cache_k + to) = kc;
        *reinterpret_cast<uint32_t *>(p.cache_v + to) = vc;
      }
    }
  }
  // No live key: zeros, by the whole workgroup of the one split.
  __device__ __forceinline__ void zero_rows(int threads) const {
    constexpr int kGroup = Fp8Shape<kDim>::kGroup;
    uint16_t *rows = p.out + ((int64_t)b * kQueryHeads + head * kGroup) * kDim;
    for (int e = threadIdx.x; e < kGroup * kDim / kPackElems; e += threads)
      store128(rows + e * kPackElems, make_uint4(0, 0, 0, 0));
  }
};

// ---- 8 x 256, and 1 x 512 in longer splits ---------------------------------------------
template <int kDim, int kWaves>
__global__ __launch_bounds__(kWaves *kWave, kDim == 256 ? 2 : 1) void decode_fp8_kernel(
    Fp8DecodeParams p) {
  using S = Fp8Shape<kDim>;
  constexpr int kParts = S::kParts;
  constexpr bool kLdsQ = kDim == 512;
  struct Lds {
    uint4 k[kWaves][kTile * S::kChunks];
    uint4 q[kLdsQ ? kQueryHeads : 1][64];  // head h's chunk c (8 dims) at c ^ h
    uint32_t rows[kWaves][kWave];
    uint32_t token[2][kDim / 4];  // the appended row's codes
    float m[kWaves][kQueryHeads];
    float l[kWaves][kQueryHeads];
  };
  __shared__ __attribute__((aligned(1024))) Lds lds;

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = wave_uniform(threadIdx.x / kWave);
  const int h = lane & 15, g = lane >> 4;
  Fp8Split<kDim> s(p);
  if (s.dead) return;
  const int32_t early_page = *s.early_entry(((lane >> 5) * kWaves + wave) * kTile + (lane & 31));
  const int32_t head = s.head, split = s.split, b = s.b;
  const int32_t q_head0 = head * S::kGroup;
  const float k_scale = fp8_scale(p.k_scales, p.c, p.layer, head);
  const float v_scale = fp8_scale(p.v_scales, p.c, p.layer, head);
  const bool direct = p.num_splits == 1;
  // Q^T operands: lane holds head h's dims 64 j + 16 g + 8 e .. + 7 of step (j, e).
  // Columns past the head's group are zero. At 512 dims they are read from LDS.
  u32x4v_t q[kLdsQ ? 1 : 2 * S::kSteps];
  uint4 q_row[kLdsQ ? kQueryHeads / kWaves : 1];
  if constexpr (kLdsQ) {
#pragma unroll
    for (int i = 0; i < kQueryHeads / kWaves; ++i)
      q_row[i] = load128(p.q + ((int64_t)b * kQueryHeads + kQueryHeads / kWaves * wave + i) * kDim + 8 * lane);
  } else {
    const uint16_t *row = p.q + ((int64_t)b * kQueryHeads + q_head0 + (h < S::kGroup ? h : 0)) * kDim;
#pragma unroll
    for (int i = 0; i < 2 * S::kSteps; ++i) {
      const uint4 x = load128(row + 64 * (i / 2) + 16 * g + 8 * (i % 2));
      q[i] = h < S::kGroup ? u32x4v_t{x.x, x.y, x.z, x.w} : u32x4v_t{0, 0, 0, 0};
    }
  }
  auto q_operand = [&](int j, int e) __attribute__((always_inline)) -> bf16x8_t {
    if constexpr (kLdsQ) return __builtin_bit_cast(bf16x8_t, lds.q[h][(8 * j + 2 * g + e) ^ h]);
    return __builtin_bit_cast(bf16x8_t, q[2 * j + e]);
  };
  s.finish();
  if (!s.live()) {
    if (s.owns && wave == 0) s.quantise_token(lds.token, k_scale, v_scale);
    if (s.key_count == 0 && split == 0 && direct) s.zero_rows(kWaves * kWave);
    return;
  }

  const int32_t begin = s.begin(), end = s.end();
  const int32_t all_tiles = (end - begin + kTile - 1) / kTile;
  const int32_t tiles = (all_tiles - wave + kWaves - 1) / kWaves;  // this wave's
  // The token's tile, by this wave's count, and its key there.
  int32_t token_tile = -1, token_key = 0;
  if (s.token_key >= 0) {
    const int32_t at = (s.token_key - begin) / kTile;
    if (at % kWaves == wave) {
      token_tile = at / kWaves;
      token_key = (s.token_key - begin) % kTile;
    }
  }
  if (s.owns && (s.token_key >= 0 ? token_tile >= 0 : wave == 0))
    s.quantise_token(lds.token, k_scale, v_scale);

  // Keys of two tiles are looked up at a time: lane l has key l % 32 of tile 2 m + l / 32.
  auto lookup_key = [&](int32_t m) __attribute__((always_inline)) -> int32_t {
    const uint32_t at = (uint32_t)begin + (uint32_t)((2 * m + (lane >> 5)) * kWaves + wave) * kTile +
                        (lane & 31);
    return (int32_t)min(at, (uint32_t)end);
  };
  auto lookup_entry = [&](int32_t m) __attribute__((always_inline)) -> int32_t {
    return *s.entry_of(min(lookup_key(m), end - 1));
  };
  uint64_t valid_pair = 0;
  auto resolve = [&](int32_t m, int32_t page) __attribute__((always_inline)) {
    const int32_t key = lookup_key(m), row = s.live_row(key, page, end);
    valid_pair = __builtin_amdgcn_ballot_w64(row >= 0);
    // The token's key is not in the cache yet.
    lds.rows[wave][lane] = (uint32_t)(key == s.token_key ? -1 : row);
    wave_lds_sync();
  };

  const uint64_t zero_row = reinterpret_cast<uint64_t>(&g_zero_codes[0]) + 16 * h;
  const uint64_t k_base = reinterpret_cast<uint64_t>(p.cache_k) + head * kDim + 16 * h;
  // Lane h's chunk of V: the products' rows 4 g + i are then chunks 4 i + g, so that the
  // lanes of a head store next to each other.
  const int v_chunk = h % 4 * 4 + h / 4;
  const uint64_t v_base = reinterpret_cast<uint64_t>(p.cache_v) + head * kDim + 16 * v_chunk;
  uint32_t rows[kLaneKeys];  // of the tile whose K was asked for last
  auto address = [&](uint64_t base, uint32_t row) __attribute__((always_inline)) -> uint64_t {
    return (int32_t)row < 0 ? zero_row : base + (uint64_t)row * (S::kHeads * kDim);
  };
  uint4 k_pack[kLaneKeys * kParts], v_pack[kLaneKeys * kParts];
  auto load_k = [&](int32_t n) __attribute__((always_inline)) {
    const uint4 lo = *reinterpret_cast<const uint4 *>(&lds.rows[wave][n % 2 * kTile + 4 * g]);
    const uint4 hi = *reinterpret_cast<const uint4 *>(&lds.rows[wave][n % 2 * kTile + 16 + 4 * g]);
    rows[0] = lo.x; rows[1] = lo.y; rows[2] = lo.z; rows[3] = lo.w;
    rows[4] = hi.x; rows[5] = hi.y; rows[6] = hi.z; rows[7] = hi.w;
#pragma unroll
    for (int i = 0; i < kLaneKeys; ++i) {
      const uint64_t at = address(k_base, rows[i]);
#pragma unroll
      for (int part = 0; part < kParts; ++part) k_pack[i * kParts + part] = load_pack(at + 256 * part);
    }
  };
  auto load_v = [&](int part) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kLaneKeys; ++i)
      v_pack[i * kParts + part] = load_pack(address(v_base, rows[i]) + 256 * part);
  };
  // Key of the tile that is a lane's i-th.
  auto key_of = [&](int i) __attribute__((always_inline)) -> int {
    return (i < 4 ? 0 : 12) + 4 * g + i;
  };
  auto put_token = [&](uint4 (&pack)[kLaneKeys * kParts], int which, int chunk) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kLaneKeys; ++i) {
      if (key_of(i) != token_key) continue;
#pragma unroll
      for (int part = 0; part < kParts; ++part)
        pack[i * kParts + part] =
            *reinterpret_cast<const uint4 *>(&lds.token[which][part * 64 + 4 * chunk]);
    }
  };

  f32x4_t acc[S::kChunks];
#pragma unroll
  for (int d = 0; d < S::kChunks; ++d) acc[d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  float m_run = -INFINITY, l_run = 0.0f;
  const float scale = p.q_scale * k_scale;
  uint4 *const k_tile = &lds.k[wave][0];

  int32_t page_next = 0;
  uint32_t valid_next = 0;
  if (tiles > 0) {
    resolve(0, s.early() ? early_page : lookup_entry(0));
    page_next = tiles > 2 ? lookup_entry(1) : 0;
    valid_next = (uint32_t)valid_pair;
    load_k(0);
#pragma unroll
    for (int part = 0; part < kParts; ++part) load_v(part);
  }
  if constexpr (kLdsQ) {
#pragma unroll
    for (int i = 0; i < kQueryHeads / kWaves; ++i) {
      const int head_row = kQueryHeads / kWaves * wave + i;
      lds.q[head_row][lane ^ head_row] = q_row[i];
    }
    lds_barrier();
  }

  auto tile = [&](int32_t n, auto more) __attribute__((always_inline)) {
    if (n == token_tile) put_token(k_pack, 0, h);
#pragma unroll
    for (int i = 0; i < kLaneKeys; ++i) {
      const int r = key_of(i);
#pragma unroll
      for (int part = 0; part < kParts; ++part)
        k_tile[r * S::kChunks + 16 * part + (h ^ (r & 15))] = k_pack[i * kParts + part];
    }
    wave_lds_sync();
    const uint32_t valid = valid_next;
    if constexpr (decltype(more)::value) {
      if ((n + 1) % 2 == 0) {
        resolve((n + 1) / 2, page_next);
        page_next = lookup_entry((n + 3) / 2);
        valid_next = (uint32_t)valid_pair;
      } else {
        valid_next = (uint32_t)(valid_pair >> 32);
      }
      load_k(n + 1);
    }

    f32x4_t score[2] = {f32x4_t{0, 0, 0, 0}, f32x4_t{0, 0, 0, 0}};
#pragma unroll
    for (int j = 0; j < S::kSteps; ++j) {
      const bf16x8_t q0 = q_operand(j, 0), q1 = q_operand(j, 1);
#pragma unroll
      for (int block = 0; block < 2; ++block) {
        const uint4 x = k_tile[(16 * block + h) * S::kChunks + ((4 * j + g) ^ h)];
        const u32x4v_t a0 = {fp8_to_bf16<false>(x.x), fp8_to_bf16<true>(x.x),
                             fp8_to_bf16<false>(x.y), fp8_to_bf16<true>(x.y)};
        const u32x4v_t a1 = {fp8_to_bf16<false>(x.z), fp8_to_bf16<true>(x.z),
                             fp8_to_bf16<false>(x.w), fp8_to_bf16<true>(x.w)};
        score[block] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a0), q0,
                                                               score[block], 0, 0, 0);
        score[block] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a1), q1,
                                                               score[block], 0, 0, 0);
      }
    }
    wave_lds_sync();  // the next tile's K goes where this one's was

    float x[kLaneKeys];
    const uint32_t seen = valid >> (4 * g);
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kLaneKeys; ++i) {
      const bool ok = (seen >> (i < 4 ? i : 12 + i)) & 1u;
      x[i] = ok ? score[i / 4][i % 4] * scale : -INFINITY;
      top = fmaxf(top, x[i]);
    }
    top = xor_max<16>(top);
    top = xor_max<32>(top);
    if (__builtin_amdgcn_ballot_w64(top > m_run + kRescaleSlack) != 0) {
      const float m_new = fmaxf(m_run, top);
      const float alpha = m_run == m_new ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < S::kChunks; ++d) acc[d] *= alpha;
    }
    const float m_use = m_run == -INFINITY ? 0.0f : m_run;
    u32x4v_t p_hi, p_lo;
#pragma unroll
    for (int i = 0; i < kLaneKeys; i += 2) {
      const float w0 = __builtin_amdgcn_exp2f(x[i] - m_use);
      const float w1 = __builtin_amdgcn_exp2f(x[i + 1] - m_use);
      l_run += w0 + w1;
      const uint32_t hi = cvt_pk_bf16(w0, w1);
      p_hi[i / 2] = hi;
      p_lo[i / 2] = cvt_pk_bf16(w0 - bf16_lo(hi), w1 - bf16_hi(hi));
    }

    if (n == token_tile) put_token(v_pack, 1, v_chunk);
    auto word = [](const uint4 &x4, int w) __attribute__((always_inline)) -> uint32_t {
      return w == 0 ? x4.x : (w == 1 ? x4.y : (w == 2 ? x4.z : x4.w));
    };
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        // Of keys 2 i and 2 i + 1: bytes 0, 0, 1, 1 and 2, 2, 3, 3.
        uint32_t low[4], high[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t a = word(v_pack[2 * i * kParts + part], w);
          const uint32_t e = word(v_pack[(2 * i + 1) * kParts + part], w);
          low[i] = __builtin_amdgcn_perm(e, a, 0x05010400u);
          high[i] = __builtin_amdgcn_perm(e, a, 0x07030602u);
        }
        auto product = [&](int d, const u32x4v_t &v) __attribute__((always_inline)) {
          f32x4_t &sum = acc[16 * part + 4 * w + d];
          sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, v),
                                                        __builtin_bit_cast(bf16x8_t, p_hi), sum, 0,
                                                        0, 0);
          sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, v),
                                                        __builtin_bit_cast(bf16x8_t, p_lo), sum, 0,
                                                        0, 0);
        };
        auto operand = [&](const uint32_t (&t)[4], auto second) __attribute__((always_inline)) {
          constexpr bool kSecond = decltype(second)::value;
          return u32x4v_t{fp8_to_bf16<kSecond>(t[0]), fp8_to_bf16<kSecond>(t[1]),
                          fp8_to_bf16<kSecond>(t[2]), fp8_to_bf16<kSecond>(t[3])};
        };
        product(0, operand(low, std::false_type{}));
        product(1, operand(low, std::true_type{}));
        product(2, operand(high, std::false_type{}));
        product(3, operand(high, std::true_type{}));
      }
      if constexpr (decltype(more)::value) load_v(part);
    }
  };
  int32_t n = 0;
  for (; n + 1 < tiles; ++n) tile(n, std::true_type{});
  if (tiles > 0) tile(n, std::false_type{});

  // ---- the waves' sums joined, and out --------------------------------------------
  l_run = xor_sum<16>(l_run);
  l_run = xor_sum<32>(l_run);
  if constexpr (kWaves > 1) {
    if (g == 0) {
      lds.m[wave][h] = m_run;
      lds.l[wave][h] = l_run;
    }
    lds_barrier();
    float m_all = -INFINITY, l_all = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m_all = fmaxf(m_all, lds.m[w][h]);
    auto factor = [&](float m) __attribute__((always_inline)) {
      return m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - m_all);
    };
#pragma unroll
    for (int w = 0; w < kWaves; ++w) l_all += lds.l[w][h] * factor(lds.m[w][h]);
    const float own = factor(m_run);
#pragma unroll
    for (int d = 0; d < S::kChunks; ++d) acc[d] *= own;
    m_run = m_all;
    l_run = l_all;
  }
  // Lane (g, h) holds dims 64 i + 16 g + d (+ 256 a part) of head h in acc[d][i].
  const float inv = l_run > 0.0f || l_run != l_run ? v_scale / l_run : 0.0f;
  const int64_t row0 = (int64_t)b * kQueryHeads + q_head0;
  auto put = [&](int of, int dim, float4 x, float f) __attribute__((always_inline)) {
    if (direct) {
      *reinterpret_cast<uint2 *>(p.out + (row0 + of) * kDim + dim) =
          make_uint2(cvt_pk_bf16(x.x * f, x.y * f), cvt_pk_bf16(x.z * f, x.w * f));
    } else {
      *reinterpret_cast<float4 *>(p.partial_acc + ((row0 + of) * p.num_splits + split) * kDim + dim) =
          make_float4(x.x * v_scale, x.y * v_scale, x.z * v_scale, x.w * v_scale);
    }
  };
  if (!direct && wave == 0 && g == 0 && h < S::kGroup) {
    // A NaN among the scores has made every sum NaN, and has to reach the output: the
    // combine leaves out parts whose l is not above zero.
    const bool odd = l_run != l_run;
    p.partial_m[(row0 + h) * p.num_splits + split] = odd && m_run == -INFINITY ? 0.0f : m_run * kLn2;
    p.partial_l[(row0 + h) * p.num_splits + split] = odd ? 1.0f : l_run;
  }
  if constexpr (kWaves == 1) {
    if (h < S::kGroup) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < S::kChunks; d += 4)
          put(h, 256 * (d / 16) + 64 * i + 16 * g + d % 16,
              make_float4(acc[d][i], acc[d + 1][i], acc[d + 2][i], acc[d + 3][i]), inv);
    }
  } else {
    // All dims at 256, half of each part's at 512, at a time: [wave][head][dim], then every
    // thread adds up its share. Over the K tiles and queries, which all waves are done with.
    constexpr int kRounds = kDim / 256, kQuarters = 4 / kRounds;
    constexpr int kHeadDims = 64 * kQuarters * kParts;  // of a head in a round
    constexpr int kRow = kHeadDims + 4;                 // padded
    float *sums = reinterpret_cast<float *>(&lds);
    static_assert(offsetof(Lds, rows) >= sizeof(float) * kWaves * S::kGroup * kRow, "fits");
    lds_barrier();
    if (wave == 0 && g == 0) lds.m[0][h] = inv;
#pragma unroll
    for (int round = 0; round < kRounds; ++round) {
      if (round > 0) lds_barrier();
      if (h < S::kGroup) {
#pragma unroll
        for (int q4 = 0; q4 < kQuarters; ++q4)
#pragma unroll
          for (int d = 0; d < S::kChunks; d += 4) {
            const int i = round * kQuarters + q4;
            *reinterpret_cast<float4 *>(sums + (wave * S::kGroup + h) * kRow +
                                        64 * (kQuarters * (d / 16) + q4) + 16 * g + d % 16) =
                make_float4(acc[d][i], acc[d + 1][i], acc[d + 2][i], acc[d + 3][i]);
          }
      }
      lds_barrier();
      for (int e = threadIdx.x; e < S::kGroup * kHeadDims / 4; e += kWaves * kWave) {
        const int of = e / (kHeadDims / 4), at = e % (kHeadDims / 4) * 4;
        float4 x = *reinterpret_cast<const float4 *>(sums + of * kRow + at);
#pragma unroll
        for (int w = 1; w < kWaves; ++w) {
          const float4 y = *reinterpret_cast<const float4 *>(sums + (w * S::kGroup + of) * kRow + at);
          x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
        }
        constexpr int kPartDims = 64 * kQuarters;
        put(of, 256 * (at / kPartDims) + kPartDims * round + at % kPartDims, x, lds.m[0][of]);
      }
    }
  }
}

// ---- 1 x 512, splits of one step ------------------------------------------------------
// A few keys under 16 heads: the work that is shared out here is the heads' 512 sums. The
// waves score 16 keys each and trade the weights through LDS, and each adds up 128 dims
// over all 64 keys: nothing is merged at the end, where four waves' sums of 32 KiB would
// be (one sequence of 1000 keys: 10.3 us with the combine, 13.6 by the kernel above; of
// 8193 11.7 and 14.5). What a lane has of the scores is half an operand of the second
// product as it stands. For longer splits the kernel above: two barriers a step and V
// in pieces of 128 bytes a row, which memory serves badly, take more than the merge saves
// (24 sequences of 140 000 keys: 47 us, 38 by the kernel above).
__global__ __launch_bounds__(256, 2) void decode_fp8_short_kernel(Fp8DecodeParams p) {
  constexpr int kDim = 512, kWaves = 4, kKeys = 64, kSteps = kDim / 64;
  struct Lds {
    uint4 k[kWaves][16 * 32];          // key r's chunk c at c ^ r
    uint4 q[kQueryHeads][64];          // head h's chunk c (8 dims) at c ^ h
    uint4 weights[2][2][kWave];        // of 32 keys each, the nearest bf16 and the rest
    uint32_t rows[kWaves][kKeys];
    uint32_t token[2][kDim / 4];
    float top[kWaves][kQueryHeads];
    float l[kWaves][kQueryHeads];
  };
  __shared__ __attribute__((aligned(1024))) Lds lds;

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = wave_uniform(threadIdx.x / kWave);
  const int h = lane & 15, g = lane >> 4;
  Fp8Split<kDim> s(p);
  const int32_t split = s.split, b = s.b;
  // Every wave looks up all keys, one a lane.
  int32_t page = *s.early_entry(lane);
  uint4 q_row[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    q_row[i] = load128(p.q + ((int64_t)b * kQueryHeads + 4 * wave + i) * kDim + 8 * lane);
  const float k_scale = fp8_scale(p.k_scales, p.c, p.layer, 0);
  const float v_scale = fp8_scale(p.v_scales, p.c, p.layer, 0);
  const bool direct = p.num_splits == 1;
  s.finish();
  if (!s.live()) {
    if (s.owns && wave == 0) s.quantise_token(lds.token, k_scale, v_scale);
    if (s.key_count == 0 && split == 0 && direct) s.zero_rows(kWaves * kWave);
    return;
  }

  const int32_t begin = s.begin(), end = s.end();
  const int32_t key = (int32_t)min((uint32_t)begin + lane, (uint32_t)end);
  if (!s.early()) page = *s.entry_of(min(key, end - 1));
  const int32_t row_word = s.live_row(key, page, end);
  const uint64_t valid = __builtin_amdgcn_ballot_w64(row_word >= 0);
  // The token's key is not in the cache yet.
  lds.rows[wave][lane] = (uint32_t)(key == s.token_key ? -1 : row_word);
  wave_lds_sync();
  const int token_at = s.token_key >= 0 ? s.token_key - begin : -1;

  const uint64_t zero_row = reinterpret_cast<uint64_t>(&g_zero_codes[0]);
  auto address = [&](const uint8_t *cache, uint32_t row, int32_t off) __attribute__((always_inline))
      -> uint64_t {
    const uint64_t at = reinterpret_cast<uint64_t>(cache) + (uint64_t)row * kDim;
    return ((int32_t)row < 0 ? zero_row : at) + off;
  };
  // Rows of keys `at` + 4 g .. + 3.
  auto rows_of = [&](int at) __attribute__((always_inline)) -> uint4 {
    return *reinterpret_cast<const uint4 *>(&lds.rows[wave][at + 4 * g]);
  };
  uint4 k_pack[4][2];
  {
    const uint4 r = rows_of(16 * wave);
    const uint32_t rows[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t at = address(p.cache_k, rows[i], 16 * h);
      k_pack[i][0] = load_pack(at);
      k_pack[i][1] = load_pack(at + 256);
    }
  }
  const int v_chunk = h % 4 * 4 + h / 4;  // of 8 dims: see above
  uint2 v_pack[2][8];
#pragma unroll
  for (int group = 0; group < 2; ++group) {
    const uint4 lo = rows_of(kTile * group), hi = rows_of(kTile * group + 16);
    const uint32_t rows[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v_pack[group][i] = __builtin_bit_cast(
          uint2, load_from<u32x2v_t>(address(p.cache_v, rows[i], 128 * wave + 8 * v_chunk)));
  }
  if (s.owns && wave == 0) s.quantise_token(lds.token, k_scale, v_scale);
#pragma unroll
  for (int i = 0; i < 4; ++i) lds.q[4 * wave + i][lane ^ (4 * wave + i)] = q_row[i];
  lds_barrier();

  // ---- scores of the wave's own 16 keys, in two chains
  uint4 *const k_tile = &lds.k[wave][0];
  if (token_at >= 0 && token_at / 16 == wave) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (4 * g + i != token_at % 16) continue;
      k_pack[i][0] = *reinterpret_cast<const uint4 *>(&lds.token[0][4 * h]);
      k_pack[i][1] = *reinterpret_cast<const uint4 *>(&lds.token[0][64 + 4 * h]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 4 * g + i;
    k_tile[r * 32 + (h ^ r)] = k_pack[i][0];
    k_tile[r * 32 + 16 + (h ^ r)] = k_pack[i][1];
  }
  wave_lds_sync();
  f32x4_t score[2] = {f32x4_t{0, 0, 0, 0}, f32x4_t{0, 0, 0, 0}};
#pragma unroll
  for (int j = 0; j < kSteps; ++j) {
    const uint4 x = k_tile[h * 32 + ((4 * j + g) ^ h)];
    const u32x4v_t a0 = {fp8_to_bf16<false>(x.x), fp8_to_bf16<true>(x.x),
                         fp8_to_bf16<false>(x.y), fp8_to_bf16<true>(x.y)};
    const u32x4v_t a1 = {fp8_to_bf16<false>(x.z), fp8_to_bf16<true>(x.z),
                         fp8_to_bf16<false>(x.w), fp8_to_bf16<true>(x.w)};
    const uint4 q0 = lds.q[h][(8 * j + 2 * g) ^ h], q1 = lds.q[h][(8 * j + 2 * g + 1) ^ h];
    score[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
        __builtin_bit_cast(bf16x8_t, a0), __builtin_bit_cast(bf16x8_t, q0), score[0], 0, 0, 0);
    score[1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
        __builtin_bit_cast(bf16x8_t, a1), __builtin_bit_cast(bf16x8_t, q1), score[1], 0, 0, 0);
  }
  // ---- one maximum for all keys
  const float scale = p.q_scale * k_scale;
  const uint32_t seen = (uint32_t)(valid >> (16 * wave + 4 * g));
  float x[4], top = -INFINITY;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = (seen >> i) & 1u ? (score[0][i] + score[1][i]) * scale : -INFINITY;
    top = fmaxf(top, x[i]);
  }
  top = xor_max<16>(top);
  top = xor_max<32>(top);
  if (g == 0) lds.top[wave][h] = top;
  lds_barrier();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, lds.top[w][h]);
  const float m_use = top == -INFINITY ? 0.0f : top;
  float l_run = 0.0f;
  uint32_t high[2], rest[2];
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const float w0 = __builtin_amdgcn_exp2f(x[i] - m_use);
    const float w1 = __builtin_amdgcn_exp2f(x[i + 1] - m_use);
    l_run += w0 + w1;
    high[i / 2] = cvt_pk_bf16(w0, w1);
    rest[i / 2] = cvt_pk_bf16(w0 - bf16_lo(high[i / 2]), w1 - bf16_hi(high[i / 2]));
  }
  reinterpret_cast<uint2 *>(&lds.weights[wave / 2][0][lane])[wave % 2] = make_uint2(high[0], high[1]);
  reinterpret_cast<uint2 *>(&lds.weights[wave / 2][1][lane])[wave % 2] = make_uint2(rest[0], rest[1]);
  l_run = xor_sum<16>(l_run);
  l_run = xor_sum<32>(l_run);
  if (g == 0) lds.l[wave][h] = l_run;
  lds_barrier();
  float l_all = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) l_all += lds.l[w][h];

  // ---- the wave's dims over all of them
  f32x4_t acc[8];
#pragma unroll
  for (int d = 0; d < 8; ++d) acc[d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int group = 0; group < 2; ++group) {
    const uint4 wh = lds.weights[group][0][lane], wl = lds.weights[group][1][lane];
    if (token_at >= 0 && token_at / kTile == group) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if ((i < 4 ? 0 : 12) + 4 * g + i == token_at % kTile)
          v_pack[group][i] = *reinterpret_cast<const uint2 *>(&lds.token[1][32 * wave + 2 * v_chunk]);
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      // Of keys 2 i and 2 i + 1: bytes 0, 0, 1, 1 and 2, 2, 3, 3.
      uint32_t low_bytes[4], high_bytes[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = w == 0 ? v_pack[group][2 * i].x : v_pack[group][2 * i].y;
        const uint32_t e = w == 0 ? v_pack[group][2 * i + 1].x : v_pack[group][2 * i + 1].y;
        low_bytes[i] = __builtin_amdgcn_perm(e, a, 0x05010400u);
        high_bytes[i] = __builtin_amdgcn_perm(e, a, 0x07030602u);
      }
      auto product = [&](int d, const uint32_t (&t)[4], auto second) __attribute__((always_inline)) {
        constexpr bool kSecond = decltype(second)::value;
        const u32x4v_t v = {fp8_to_bf16<kSecond>(t[0]), fp8_to_bf16<kSecond>(t[1]),
                            fp8_to_bf16<kSecond>(t[2]), fp8_to_bf16<kSecond>(t[3])};
        f32x4_t &sum = acc[4 * w + d];
        sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, v),
                                                      __builtin_bit_cast(bf16x8_t, wh), sum, 0, 0, 0);
        sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, v),
                                                      __builtin_bit_cast(bf16x8_t, wl), sum, 0, 0, 0);
      };
      product(0, low_bytes, std::false_type{});
      product(1, low_bytes, std::true_type{});
      product(2, high_bytes, std::false_type{});
      product(3, high_bytes, std::true_type{});
    }
  }

  // ---- out: lane (g, h) holds dims 128 wave + 32 i + 8 g + d of head h in acc[d][i]
  const int64_t row = (int64_t)b * kQueryHeads + h;
  const bool odd = l_all != l_all;  // a NaN among the scores
  if (direct) {
    const float f = l_all > 0.0f || odd ? v_scale / l_all : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      store128(p.out + row * kDim + 128 * wave + 32 * i + 8 * g,
               make_uint4(cvt_pk_bf16(acc[0][i] * f, acc[1][i] * f), cvt_pk_bf16(acc[2][i] * f, acc[3][i] * f),
                          cvt_pk_bf16(acc[4][i] * f, acc[5][i] * f), cvt_pk_bf16(acc[6][i] * f, acc[7][i] * f)));
  } else {
    const int64_t slot = row * p.num_splits + split;
    float *to = p.partial_acc + slot * kDim + 128 * wave + 8 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      *reinterpret_cast<float4 *>(to + 32 * i) = make_float4(acc[0][i] * v_scale, acc[1][i] * v_scale,
                                                            acc[2][i] * v_scale, acc[3][i] * v_scale);
      *reinterpret_cast<float4 *>(to + 32 * i + 4) = make_float4(acc[4][i] * v_scale, acc[5][i] * v_scale,
                                                                acc[6][i] * v_scale, acc[7][i] * v_scale);
    }
    if (wave == 0 && g == 0) {
      // A NaN has made every sum NaN, and has to reach the output: see above.
      p.partial_m[slot] = odd && top == -INFINITY ? 0.0f : top * kLn2;
      p.partial_l[slot] = odd ? 1.0f : l_all;
    }
  }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Waves of a split: one per tile, up to four. (At 1 x 512 up to two tiles are the four
// waves' of the short kernel.)
int split_waves(int32_t split_size) {
  return split_size <= kTile ? 1 : (split_size <= 2 * kTile ? 2 : 4);
}

void launch_split(const Fp8DecodeParams &p, int32_t splits, int32_t batch, hipStream_t stream) {
  const dim3 grid(p.c.num_heads, splits, batch);
  auto launch = [&](auto *kernel, int waves) {
    hipLaunchKernelGGL(kernel, grid, dim3(waves * kWave), 0, stream, p);
  };
  const int waves = p.balanced != 0 ? 4 : split_waves(p.split_size);
  if (p.c.head_dim == 512) {
    waves < 4 ? launch(decode_fp8_short_kernel, 4) : launch(decode_fp8_kernel<512, 4>, 4);
  } else if (waves == 1) {
    launch(decode_fp8_kernel<256, 1>, 1);
  } else if (waves == 2) {
    launch(decode_fp8_kernel<256, 2>, 2);
  } else {
    launch(decode_fp8_kernel<256, 4>, 4);
  }
}

hipError_t decode_fp8(gemma4_bf16 *out, float *pm, float *pl, float *pacc, const gemma4_bf16 *q,
                      uint8_t *cache_k, uint8_t *cache_v, const float *k_scales,
                      const float *v_scales, const int32_t *page_table,
                      const int32_t *seq_lengths, const int32_t *token_position,
                      const gemma4_bf16 *new_k, const gemma4_bf16 *new_v,
                      const Gemma4KvCacheConfig &c, int32_t layer, float softmax_scale,
                      int32_t split_size, int32_t num_splits, int32_t batch, hipStream_t stream) {
  if (batch == 0) return hipSuccess;
  if (!decode_geometry_ok(c, layer, batch, split_size, num_splits) || !(softmax_scale > 0.0f) ||
      !isfinite(softmax_scale * kLog2e) || out == nullptr || q == nullptr || cache_k == nullptr ||
      cache_v == nullptr || page_table == nullptr || seq_lengths == nullptr ||
      (num_splits > 1 && (pm == nullptr || pl == nullptr || pacc == nullptr)) ||
      !aligned16(out) || !aligned16(q) || !aligned16(cache_k) || !aligned16(cache_v) ||
      !aligned16(pacc) || !aligned16(new_k) || !aligned16(new_v)) {
    return hipErrorInvalidValue;
  }
  // No cache holds more keys, and the combine adds a length to it in 32 bits.
  split_size = std::min(split_size, 1 << 30);
  Fp8DecodeParams p{};
  p.out = reinterpret_cast<uint16_t *>(out);
  p.partial_m = pm;
  p.partial_l = pl;
  p.partial_acc = pacc;
  p.q = reinterpret_cast<const uint16_t *>(q);
  p.cache_k = cache_k;
  p.cache_v = cache_v;
  p.k_scales = k_scales;
  p.v_scales = v_scales;
  p.page_table = page_table;
  p.seq_lengths = seq_lengths;
  p.token_position = token_position;
  p.new_k = reinterpret_cast<const uint16_t *>(new_k);
  p.new_v = reinterpret_cast<const uint16_t *>(new_v);
  p.c = c;
  p.page_div = make_fast_div(c.page_size);
  p.slot_div = make_fast_div(c.max_pages_per_seq);
  p.layer = layer;
  p.q_scale = softmax_scale * kLog2e;
  p.split_size = split_size;
  p.num_splits = num_splits;
  // A batch is cut by its lengths, on the device: the plan knows only the longest. Not one
  // that the plan gives short splits.
  int64_t splits = num_splits;
  if (num_splits > 1 && batch > 1 && batch <= kBalancedBatch && split_waves(split_size) == 4) {
    p.balanced = c.num_heads;
    p.batch = batch;
    splits = std::min<int64_t>((int64_t)batch * num_splits,
                               c.head_dim == 512 ? kFp8Cus : kFp8Cus + batch);
  }
  launch_split(p, (int32_t)splits, p.balanced != 0 ? 1 : batch, stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || num_splits == 1) return e;
  if (p.balanced != 0) {
    const CombineParams cp = {p.out,         pm,         pl,         pacc,       seq_lengths, nullptr,
                              c.window_size, split_size, num_splits, p.balanced, batch};
    return launch_combine_fp8(cp, c.head_dim, batch, stream);
  }
  return gemma4_flash_attention_decode_combine_bf16(out, pm, pl, pacc, seq_lengths, c, split_size,
                                                    num_splits, batch, stream);
}

}  // namespace
}  // namespace gemma4

using namespace gemma4;

extern "C" {

hipError_t gemma4_flash_attention_decode_paged_fp8(
    gemma4_bf16 *d_out, float *d_partial_m, float *d_partial_l, float *d_partial_acc,
    const gemma4_bf16 *d_q, const uint8_t *d_cache_k, const uint8_t *d_cache_v,
    const float *d_k_scales, const float *d_v_scales, const int32_t *d_page_table,
    const int32_t *d_seq_lengths, Gemma4KvCacheConfig config, int32_t layer, float softmax_scale,
    int32_t split_size, int32_t num_splits, int32_t batch_count, hipStream_t stream) {
  return decode_fp8(d_out, d_partial_m, d_partial_l, d_partial_acc, d_q,
                    const_cast<uint8_t *>(d_cache_k), const_cast<uint8_t *>(d_cache_v), d_k_scales,
                    d_v_scales, d_page_table, d_seq_lengths, nullptr, nullptr, nullptr, config,
                    layer, softmax_scale, split_size, num_splits, batch_count, stream);
}

hipError_t gemma4_flash_attention_append_decode_paged_fp8(
    gemma4_bf16 *d_out, float *d_partial_m, float *d_partial_l, float *d_partial_acc,
    const gemma4_bf16 *d_q, uint8_t *d_cache_k, uint8_t *d_cache_v, const float *d_k_scales,
    const float *d_v_scales, const int32_t *d_page_table, const int32_t *d_seq_lengths,
    const int32_t *d_token_position, const gemma4_bf16 *d_k, const gemma4_bf16 *d_v,
    Gemma4KvCacheConfig config, int32_t layer, float softmax_scale, int32_t split_size,
    int32_t num_splits, int32_t batch_count, hipStream_t stream) {
  if (batch_count == 0) return hipSuccess;
  if (d_token_position == nullptr || d_k == nullptr || d_v == nullptr) return hipErrorInvalidValue;
  return decode_fp8(d_out, d_partial_m, d_partial_l, d_partial_acc, d_q, d_cache_k, d_cache_v,
                    d_k_scales, d_v_scales, d_page_table, d_seq_lengths, d_token_position, d_k,
                    d_v, config, layer, softmax_scale, split_size, num_splits, batch_count,
                    stream);
}

hipError_t gemma4_decode_split_plan_fp8(Gemma4KvCacheConfig config, int32_t batch_count,
                                        int32_t max_live_keys, int32_t target_workgroups,
                                        int32_t *split_size, int32_t *num_splits) {
  const bool geometry = (config.num_heads == 8 && config.head_dim == 256) ||
                        (config.num_heads == 1 && config.head_dim == 512);
  if (split_size == nullptr || num_splits == nullptr || batch_count <= 0 || max_live_keys < 0 ||
      !geometry) {
    return hipErrorInvalidValue;
  }
  const int64_t keys = std::max(max_live_keys, 1);
  const int64_t heads = config.num_heads;
  auto whole = [](int64_t n, int64_t step) { return std::max<int64_t>((n + step - 1) / step, 1) * step; };
  int64_t size;
  if (target_workgroups > 0) {
    const int64_t units = (int64_t)batch_count * heads;
    const int64_t per_unit = std::max<int64_t>((target_workgroups + units - 1) / units, 1);
    size = whole((keys + per_unit - 1) / per_unit, kTile);
  } else if (heads == 1 ? (keys + 63) / 64 * batch_count <= (batch_count > 1 ? 2 * kFp8Cus : kFp8Cus)
                        : keys <= 2 * kFp8Step) {
    // 1 x 512: the short kernel's steps, while the chip takes them in a round; 8 x 256: one
    // split, and no combine (256 keys 7.7 us, 8.6 in splits of 32).
    size = heads == 1 ? 2 * kTile : whole(keys, kFp8Step);
  } else if (batch_count == 1) {
    // A workgroup a CU, two of them from where 2048 keys are a split, in whole steps of
    // four waves where they are that long. Split + combine at 8 x 256, 2000 keys in splits
    // of 32 / 128 / 256 8.9 / 9.5 / 10.9 us, 16 000 of 128 / 256 / 512 / 1024 21.5 / 16.2 /
    // 15.8 / 20.9, 131 072 of 512 / 1024 / 2048 92.8 / 87.9 / 85.9; at 1 x 512 60 000 of
    // 64 / 128 / 256 / 512 34 / 36 / 23.4 / 25.7, 131 072 of 256 / 512 45 / 33.6.
    const int64_t even = keys * heads / kFp8Cus;
    size = even < 3 * kTile ? whole(even, kTile) : (even + kFp8Step / 2) / kFp8Step * kFp8Step;
    if (heads == 1) size = whole((keys + kFp8Cus - 1) / kFp8Cus, kFp8Step);
    if (heads != 1) size = std::min<int64_t>(size, whole(std::max<int64_t>(2048, even / 2), kFp8Step));
  } else if (batch_count <= kBalancedBatch) {
    // The lengths make the cut; here the most splits that it can come to, the longest
    // sequence being about all there is: of kFp8Long keys, and no more than kFp8Cus, where the
    // cut's grow too (Fp8Cut). Partial sums are as many as these.
    size = whole(std::max<int64_t>(std::min<int64_t>(keys * heads / kFp8Cus, kFp8Long),
                                   (keys + kFp8Cus - 1) / kFp8Cus),
                 kFp8Step);
  } else {
    size = whole(keys * heads * batch_count / 2048, kFp8Step);
  }
  // Splits are numbered in 16 bits.
  size = std::max<int64_t>(size, (keys + 65534) / 65535);
  size = std::min<int64_t>(whole(size, kTile), 0x7fffffff / kTile * kTile);
  *split_size = (int32_t)size;
  *num_splits = (int32_t)((keys + size - 1) / size);
  return hipSuccess;
}

}  // extern "C"
