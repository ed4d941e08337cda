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
// bf16 numbers, the nearest and the rest (2^-18 of a weight).
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

#include "gemma4_flash_attention.h"

#include <math.h>

#include <algorithm>
#include <type_traits>

namespace gemma4 {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x4v_t __attribute__((ext_vector_type(4)));

constexpr int kTile = 32;              // keys of a wave's tile
constexpr int kLaneKeys = 8;           // of them, a lane's
constexpr float kRescaleSlack = 8.0f;  // log2 headroom of the running maximum

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
};

template <int kDim>
struct Fp8Shape {
  static constexpr int kHeads = kDim == 256 ? 8 : 1;
  static constexpr int kGroup = kQueryHeads / kHeads;  // query heads of a KV head
  static constexpr int kParts = kDim / 256;            // 256-byte segments of a row
  static constexpr int kSteps = kDim / 64;             // pairs of S^T steps
  static constexpr int kChunks = kDim / 16;
};

template <int kDim, int kWaves>
__global__ __launch_bounds__(kWaves *kWave, kDim == 256 ? 2 : 1) void decode_fp8_kernel(
    Fp8DecodeParams p) {
  using S = Fp8Shape<kDim>;
  constexpr int kParts = S::kParts;
  struct Lds {
    uint4 k[kWaves][kTile * S::kChunks];
    uint32_t rows[kWaves][kWave];
    uint32_t token[2][kDim / 4];  // the appended row's codes
    float m[kWaves][kQueryHeads];
    float l[kWaves][kQueryHeads];
  };
  __shared__ __attribute__((aligned(1024))) Lds lds;

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = wave_uniform(threadIdx.x / kWave);
  const int h = lane & 15, g = lane >> 4;
  const Gemma4KvCacheConfig &c = p.c;
  const int32_t head = blockIdx.x, split = blockIdx.y, b = blockIdx.z;
  const int32_t q_head0 = head * S::kGroup;

  const int32_t seq_word = p.seq_lengths[b];
  const int32_t tok_word = p.token_position != nullptr ? p.token_position[b] : -1;
  const float k_scale = fp8_scale(p.k_scales, c, p.layer, head);
  const float v_scale = fp8_scale(p.v_scales, c, p.layer, head);
  // Q^T operands: lane holds head h's dims 64 j + 16 g + 8 e .. + 7 of step (j, e).
  // Columns past the head's group are zero.
  u32x4v_t q[2 * S::kSteps];
  {
    const uint16_t *row = p.q + ((int64_t)b * kQueryHeads + q_head0 + (h < S::kGroup ? h : 0)) * kDim;
#pragma unroll
    for (int s = 0; s < 2 * S::kSteps; ++s) {
      const uint4 x = load128(row + 64 * (s / 2) + 16 * g + 8 * (s % 2));
      q[s] = h < S::kGroup ? u32x4v_t{x.x, x.y, x.z, x.w} : u32x4v_t{0, 0, 0, 0};
    }
  }

  const int32_t seq_len = wave_uniform(seq_word);
  const int32_t token_pos = wave_uniform(tok_word);
  int32_t first = c.window_size > 0 ? seq_len - c.window_size : 0;
  first = first < 0 ? 0 : first;
  const int32_t capacity =
      (int32_t)min((int64_t)p.split_size * p.num_splits, (int64_t)0x7fffffff);
  const int32_t key_count = min(seq_len > first ? seq_len - first : 0, capacity);
  const int32_t live_splits =
      (int32_t)(((uint32_t)key_count + (uint32_t)p.split_size - 1) / (uint32_t)p.split_size);
  const bool direct = p.num_splits == 1;

  // The split that holds the token's key writes its row (split 0 where the position is
  // not among the live keys), by the skip rules of the append.
  bool owns = false, in_live = false;
  if (p.token_position != nullptr) {
    const bool droppable =
        token_pos < 0 || (c.window_size == 0 && token_pos / c.page_size >= c.max_pages_per_seq);
    in_live = token_pos >= first && token_pos < first + key_count;
    owns = !droppable && split == (in_live ? (token_pos - first) / p.split_size : 0);
  }
  const int32_t *table = p.page_table + (int64_t)b * c.max_pages_per_seq;
  // Row of a position, -1 where no page is mapped.
  auto row_of = [&](int32_t key, int32_t page) __attribute__((always_inline)) -> int32_t {
    const int32_t in_page = key - (int32_t)(fast_div((uint32_t)key, p.page_div) * p.page_div.d);
    return (uint32_t)page < (uint32_t)c.num_pages
               ? (p.layer * c.num_pages + page) * c.page_size + in_page : -1;
  };
  auto entry_of = [&](int32_t key) __attribute__((always_inline)) -> const int32_t * {
    return table + fast_mod(fast_div((uint32_t)key, p.page_div), p.slot_div);
  };
  // The token's codes: 4 dims a lane, as many packs as the row has.
  auto quantise_token = [&]() __attribute__((always_inline)) {
    const int64_t from = ((int64_t)b * S::kHeads + head) * kDim;
    const int32_t row = row_of(token_pos, *entry_of(token_pos));
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      const int64_t at = from + part * 256 + 4 * lane;
      const uint2 k = *reinterpret_cast<const uint2 *>(p.new_k + at);
      const uint2 v = *reinterpret_cast<const uint2 *>(p.new_v + at);
      const uint32_t kc = fp8_word(k.x, k.y, k_scale), vc = fp8_word(v.x, v.y, v_scale);
      lds.token[0][part * 64 + lane] = kc;
      lds.token[1][part * 64 + lane] = vc;
      if (row >= 0) {
        const int64_t to = ((int64_t)row * S::kHeads + head) * kDim + part * 256 + 4 * lane;
        *reinterpret_cast<uint32_t *>(p.cache_k + to) = kc;
        *reinterpret_cast<uint32_t *>(p.cache_v + to) = vc;
      }
    }
    return row >= 0;
  };

  if (split >= live_splits) {
    if (owns && wave == 0) quantise_token();
    if (key_count == 0 && split == 0 && direct) {
      // No live key: zeros.
      uint16_t *rows = p.out + ((int64_t)b * kQueryHeads + q_head0) * kDim;
      for (int e = threadIdx.x; e < S::kGroup * kDim / kPackElems; e += kWaves * kWave)
        store128(rows + e * kPackElems, make_uint4(0, 0, 0, 0));
    }
    return;
  }

  const int32_t begin = first + split * p.split_size;
  const int32_t end =
      (int32_t)min((uint32_t)(first + key_count), (uint32_t)begin + (uint32_t)p.split_size);
  const int32_t all_tiles = (end - begin + kTile - 1) / kTile;
  const int32_t tiles = (all_tiles - wave + kWaves - 1) / kWaves;  // this wave's
  // The token's tile, by this wave's count, and its key there.
  int32_t token_tile = -1, token_key = 0;
  if (owns && in_live) {
    const int32_t at = (token_pos - begin) / kTile;
    if (at % kWaves == wave) {
      token_tile = at / kWaves;
      token_key = (token_pos - begin) % kTile;
    }
  }
  bool token_there = false;
  if (owns && (in_live ? token_tile >= 0 : wave == 0)) token_there = quantise_token();

  // Keys of two tiles are looked up at a time: lane l has key l % 32 of tile 2 m + l / 32.
  auto lookup_key = [&](int32_t m) __attribute__((always_inline)) -> int32_t {
    const uint32_t at = (uint32_t)begin + (uint32_t)((2 * m + (lane >> 5)) * kWaves + wave) * kTile +
                        (lane & 31);
    return (int32_t)min(at, (uint32_t)end);
  };
  auto lookup_entry = [&](int32_t m) __attribute__((always_inline)) -> int32_t {
    return *entry_of(min(lookup_key(m), end - 1));
  };
  uint64_t valid_pair = 0;
  auto resolve = [&](int32_t m, int32_t page) __attribute__((always_inline)) {
    const int32_t key = lookup_key(m);
    const uint32_t logical = fast_div((uint32_t)key, p.page_div);
    int32_t row = row_of(key, page);
    if (key >= end || (c.window_size == 0 && logical >= (uint32_t)c.max_pages_per_seq)) row = -1;
    const bool is_token = owns && in_live && key == token_pos;
    valid_pair = __builtin_amdgcn_ballot_w64(is_token ? token_there : row >= 0);
    lds.rows[wave][lane] = (uint32_t)(is_token ? -1 : row);
    wave_lds_sync();
  };

  const uint64_t zero_row = reinterpret_cast<uint64_t>(&g_zero_codes[0]) + 16 * h;
  const uint64_t k_base = reinterpret_cast<uint64_t>(p.cache_k) + head * kDim + 16 * h;
  const uint64_t v_base = reinterpret_cast<uint64_t>(p.cache_v) + head * kDim + 16 * h;
  uint32_t rows[kLaneKeys];  // of the tile whose K was asked for last
  auto address = [&](uint64_t base, uint32_t row) __attribute__((always_inline)) -> const void * {
    const uint64_t at = base + (uint64_t)row * (S::kHeads * kDim);
    return reinterpret_cast<const void *>((int32_t)row < 0 ? zero_row : at);
  };
  uint4 k_pack[kLaneKeys * kParts], v_pack[kLaneKeys * kParts];
  auto load_k = [&](int32_t n) __attribute__((always_inline)) {
    const uint4 lo = *reinterpret_cast<const uint4 *>(&lds.rows[wave][n % 2 * kTile + 4 * g]);
    const uint4 hi = *reinterpret_cast<const uint4 *>(&lds.rows[wave][n % 2 * kTile + 16 + 4 * g]);
    rows[0] = lo.x; rows[1] = lo.y; rows[2] = lo.z; rows[3] = lo.w;
    rows[4] = hi.x; rows[5] = hi.y; rows[6] = hi.z; rows[7] = hi.w;
#pragma unroll
    for (int i = 0; i < kLaneKeys; ++i) {
      const char *at = static_cast<const char *>(address(k_base, rows[i]));
#pragma unroll
      for (int part = 0; part < kParts; ++part)
        k_pack[i * kParts + part] = load128_stream(at + 256 * part);
    }
  };
  auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kLaneKeys; ++i) {
      const char *at = static_cast<const char *>(address(v_base, rows[i]));
#pragma unroll
      for (int part = 0; part < kParts; ++part)
        v_pack[i * kParts + part] = load128_stream(at + 256 * part);
    }
  };
  // Key of the tile that is a lane's i-th.
  auto key_of = [&](int i) __attribute__((always_inline)) -> int {
    return (i < 4 ? 0 : 12) + 4 * g + i;
  };
  auto put_token = [&](uint4 (&pack)[kLaneKeys * kParts], int which) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kLaneKeys; ++i) {
      if (key_of(i) != token_key) continue;
#pragma unroll
      for (int part = 0; part < kParts; ++part)
        pack[i * kParts + part] =
            *reinterpret_cast<const uint4 *>(&lds.token[which][part * 64 + 4 * h]);
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
    resolve(0, lookup_entry(0));
    page_next = tiles > 2 ? lookup_entry(1) : 0;
    valid_next = (uint32_t)valid_pair;
    load_k(0);
    load_v();
  }

  auto tile = [&](int32_t n, auto more) __attribute__((always_inline)) {
    if (n == token_tile) put_token(k_pack, 0);
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
#pragma unroll
      for (int block = 0; block < 2; ++block) {
        const uint4 x = k_tile[(16 * block + h) * S::kChunks + ((4 * j + g) ^ h)];
        const u32x4v_t a0 = {fp8_to_bf16<false>(x.x), fp8_to_bf16<true>(x.x),
                             fp8_to_bf16<false>(x.y), fp8_to_bf16<true>(x.y)};
        const u32x4v_t a1 = {fp8_to_bf16<false>(x.z), fp8_to_bf16<true>(x.z),
                             fp8_to_bf16<false>(x.w), fp8_to_bf16<true>(x.w)};
        score[block] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            __builtin_bit_cast(bf16x8_t, a0), __builtin_bit_cast(bf16x8_t, q[2 * j]), score[block],
            0, 0, 0);
        score[block] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            __builtin_bit_cast(bf16x8_t, a1), __builtin_bit_cast(bf16x8_t, q[2 * j + 1]),
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

    if (n == token_tile) put_token(v_pack, 1);
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
    }
    if constexpr (decltype(more)::value) load_v();
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
    __syncthreads();
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
  // Lane (g, h) holds dims 16 (4 g + i) + d (+ 256 a part) of head h in acc[d][i].
  const int64_t row = (int64_t)b * kQueryHeads + q_head0 + h;
  const float l_inv = l_run > 0.0f || l_run != l_run ? 1.0f / l_run : 0.0f;
  auto put = [&](int dim, float4 x) __attribute__((always_inline)) {
    if (direct) {
      const float f = v_scale * l_inv;
      *reinterpret_cast<uint2 *>(p.out + row * kDim + dim) =
          make_uint2(cvt_pk_bf16(x.x * f, x.y * f), cvt_pk_bf16(x.z * f, x.w * f));
    } else {
      *reinterpret_cast<float4 *>(p.partial_acc + (row * p.num_splits + split) * kDim + dim) =
          make_float4(x.x * v_scale, x.y * v_scale, x.z * v_scale, x.w * v_scale);
    }
  };
  if (!direct && wave == 0 && g == 0 && h < S::kGroup) {
    // A NaN among the scores has made every sum NaN, and has to reach the output: the
    // combine leaves out parts whose l is not above zero.
    const bool odd = l_run != l_run;
    p.partial_m[row * p.num_splits + split] = odd && m_run == -INFINITY ? 0.0f : m_run * kLn2;
    p.partial_l[row * p.num_splits + split] = odd ? 1.0f : l_run;
  }
  if constexpr (kWaves == 1) {
    if (h < S::kGroup) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < S::kChunks; d += 4)
          put(256 * (d / 16) + 16 * (4 * g + i) + d % 16,
              make_float4(acc[d][i], acc[d + 1][i], acc[d + 2][i], acc[d + 3][i]));
    }
  } else {
    // Quarter i of a part's dims at a time: wave w's sums in [w][dims 64 of a part][head],
    // then every thread adds up its share. Over the K tiles, which all waves are done with.
    constexpr int kRow = 64 * kParts + 4;  // floats of a head's quarter, padded
    float *sums = reinterpret_cast<float *>(&lds.k[0][0]);
    static_assert(sizeof(lds.k) >= sizeof(float) * kWaves * S::kGroup * kRow, "fits");
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __syncthreads();
      if (h < S::kGroup) {
#pragma unroll
        for (int d = 0; d < S::kChunks; d += 4)
          *reinterpret_cast<float4 *>(sums + (wave * S::kGroup + h) * kRow + 64 * (d / 16) + 16 * g + d % 16) =
              make_float4(acc[d][i], acc[d + 1][i], acc[d + 2][i], acc[d + 3][i]);
      }
      __syncthreads();
      constexpr int kItems = S::kGroup * 16 * kParts;  // float4 of the quarter
      for (int e = threadIdx.x; e < kItems; e += kWaves * kWave) {
        const int hh = e / (16 * kParts), at = e % (16 * kParts) * 4;
        float4 x = *reinterpret_cast<const float4 *>(sums + hh * kRow + at);
#pragma unroll
        for (int w = 1; w < kWaves; ++w) {
          const float4 y = *reinterpret_cast<const float4 *>(sums + (w * S::kGroup + hh) * kRow + at);
          x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
        }
        // Element 64 part + 16 gg + d of quarter i: dim 256 part + 16 (4 gg + i) + d.
        const int part = at / 64, gg = at % 64 / 16, d = at % 16;
        const int dim = 256 * part + 16 * (4 * gg + i) + d;
        const int64_t out_row = (int64_t)b * kQueryHeads + q_head0 + hh;
        if (direct) {
          float l_row = 0.0f, m_row = -INFINITY;
#pragma unroll
          for (int w = 0; w < kWaves; ++w) m_row = fmaxf(m_row, lds.m[w][hh]);
#pragma unroll
          for (int w = 0; w < kWaves; ++w)
            l_row += lds.m[w][hh] == -INFINITY
                         ? 0.0f : lds.l[w][hh] * __builtin_amdgcn_exp2f(lds.m[w][hh] - m_row);
          const float f = l_row > 0.0f || l_row != l_row ? v_scale / l_row : 0.0f;
          *reinterpret_cast<uint2 *>(p.out + out_row * kDim + dim) =
              make_uint2(cvt_pk_bf16(x.x * f, x.y * f), cvt_pk_bf16(x.z * f, x.w * f));
        } else {
          *reinterpret_cast<float4 *>(p.partial_acc + (out_row * p.num_splits + split) * kDim + dim) =
              make_float4(x.x * v_scale, x.y * v_scale, x.z * v_scale, x.w * v_scale);
        }
      }
    }
  }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Waves of a split: one per tile, up to four.
int split_waves(int32_t split_size) {
  return split_size <= kTile ? 1 : (split_size <= 2 * kTile ? 2 : 4);
}

template <int kDim>
void launch_split(const Fp8DecodeParams &p, int32_t batch, hipStream_t stream) {
  const dim3 grid(Fp8Shape<kDim>::kHeads, p.num_splits, batch);
  switch (split_waves(p.split_size)) {
    case 1:
      hipLaunchKernelGGL((decode_fp8_kernel<kDim, 1>), grid, dim3(kWave), 0, stream, p);
      break;
    case 2:
      hipLaunchKernelGGL((decode_fp8_kernel<kDim, 2>), grid, dim3(2 * kWave), 0, stream, p);
      break;
    default:
      hipLaunchKernelGGL((decode_fp8_kernel<kDim, 4>), grid, dim3(4 * kWave), 0, stream, p);
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
  if (c.head_dim == 512) {
    launch_split<512>(p, batch, stream);
  } else {
    launch_split<256>(p, batch, stream);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || num_splits == 1) return e;
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
  if (target_workgroups <= 0) target_workgroups = batch_count > 1 ? 2048 : 256;
  const int64_t keys = std::max(max_live_keys, 1);
  const int64_t units = (int64_t)batch_count * config.num_heads;
  const int64_t per_unit = std::max<int64_t>((target_workgroups + units - 1) / units, 1);
  int64_t size = (keys + per_unit - 1) / per_unit;
  size = std::min<int64_t>(std::max<int64_t>((size + kTile - 1) / kTile * kTile, kTile),
                           0x7fffffff / kTile * kTile);
  *split_size = (int32_t)size;
  *num_splits = (int32_t)((keys + size - 1) / size);
  return hipSuccess;
}

}  // extern "C"
