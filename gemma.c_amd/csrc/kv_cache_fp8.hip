// The quantised K/V cache, gfx950: rows written as e4m3 codes and read back.
// No counterpart in the reference, whose cache is bf16 (src/gemma4_kv_cache.cu).
//
// Both move packs of 16 codes, one thread a pack of K and the same of V: 64 bytes
// of bf16 on one side, 32 of codes on the other, and nothing else per row than its
// (sequence, position) and page-table entry.
//
// What bounds them: HBM, from some thousand rows on (4 prompts at 8 x 256, 133 MB, 28 us,
// 96% of the rate of a large copy; 24 rings read back, 277 MB, 58 us, 97%). A few rows are a
// launch: 24 at 1 x 512 3.3 us.
#include "fp8_common.hpp"
#include "gemma4_device.hpp"

namespace gemma4 {
namespace {

constexpr int kRowThreads = 256;

struct Fp8RowParams {
  uint8_t *cache_k;
  uint8_t *cache_v;
  uint16_t *k;  // rows kv_stride elements apart
  uint16_t *v;
  const float *k_scales;
  const float *v_scales;
  const int32_t *page_table;
  const int32_t *token_batch;
  const int32_t *token_position;
  Gemma4KvCacheConfig c;
  int64_t kv_stride;
  int64_t packs;  // of the call
  int32_t row_packs, head_packs;
  int32_t rows, layer;
  int32_t ring_rows;  // a ring's slots where the call may bring more rows, else 0
};

// Cache row of a token by the skip rules of the bf16 append, or -1.
__device__ __forceinline__ int64_t cache_row(const Fp8RowParams &p, int32_t b, int32_t position) {
  const Gemma4KvCacheConfig &c = p.c;
  if (b < 0 || position < 0 || b >= c.batch_size) return -1;
  const int32_t logical = position / c.page_size;
  if (c.window_size == 0 && logical >= c.max_pages_per_seq) return -1;
  const int32_t page =
      p.page_table[(int64_t)b * c.max_pages_per_seq + logical % c.max_pages_per_seq];
  if (page < 0 || page >= c.num_pages) return -1;
  return ((int64_t)p.layer * c.num_pages + page) * c.page_size + (position - logical * c.page_size);
}

template <bool kWrite>
__global__ __launch_bounds__(kRowThreads) void fp8_rows_kernel(Fp8RowParams p) {
  const int64_t i = (int64_t)blockIdx.x * kRowThreads + threadIdx.x;
  if (i >= p.packs) return;
  const int32_t row = (int32_t)(i / p.row_packs);
  const int32_t pack = (int32_t)(i - (int64_t)row * p.row_packs);
  const int32_t b = p.token_batch[row], position = p.token_position[row];
  const int64_t at = cache_row(p, b, position);
  if (at < 0) return;
  if (kWrite && p.ring_rows > 0 && row + (int64_t)p.ring_rows < p.rows) {
    const int32_t newer = row + p.ring_rows;
    if (p.token_batch[newer] == b && p.token_position[newer] - (int64_t)position == p.ring_rows)
      return;
  }
  const int32_t head = pack / p.head_packs;
  const float k_scale = fp8_scale(p.k_scales, p.c, p.layer, head);
  const float v_scale = fp8_scale(p.v_scales, p.c, p.layer, head);
  const int64_t code = (at * p.row_packs + pack) * kPackCodes;
  const int64_t element = row * p.kv_stride + (int64_t)pack * kPackCodes;
  if constexpr (kWrite) {
    const uint4 k0 = load128(p.k + element), k1 = load128(p.k + element + 8);
    const uint4 v0 = load128(p.v + element), v1 = load128(p.v + element + 8);
    store128(p.cache_k + code, fp8_pack(k0, k1, k_scale));
    store128(p.cache_v + code, fp8_pack(v0, v1, v_scale));
  } else {
    auto wide = [](uint32_t w, float scale) {
      const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
      const f32x2_t hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
      return make_uint2(cvt_pk_bf16(lo[0] * scale, lo[1] * scale),
                        cvt_pk_bf16(hi[0] * scale, hi[1] * scale));
    };
    auto store = [&](uint16_t *to, const uint4 &x, float scale) {
      const uint2 a = wide(x.x, scale), b2 = wide(x.y, scale), c2 = wide(x.z, scale),
                  d = wide(x.w, scale);
      store128(to, make_uint4(a.x, a.y, b2.x, b2.y));
      store128(to + 8, make_uint4(c2.x, c2.y, d.x, d.y));
    };
    const uint4 k = load128(p.cache_k + code), v = load128(p.cache_v + code);
    store(p.k + element, k, k_scale);
    store(p.v + element, v, v_scale);
  }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <bool kWrite>
hipError_t launch_rows(uint8_t *cache_k, uint8_t *cache_v, const Gemma4KvCacheConfig &c,
                       const int32_t *page_table, const int32_t *token_batch,
                       const int32_t *token_position, int32_t token_count, int32_t layer,
                       uint16_t *k, uint16_t *v, int64_t kv_stride, const float *k_scales,
                       const float *v_scales, hipStream_t stream) {
  if (token_count == 0) return hipSuccess;
  if (token_count < 0 || layer < 0 || layer >= c.num_layers || c.num_pages <= 0 ||
      c.page_size <= 0 || c.max_pages_per_seq <= 0 || c.batch_size <= 0 || c.window_size < 0 ||
      c.num_heads <= 0 || c.head_dim <= 0 || c.head_dim % kPackCodes != 0 ||
      (int64_t)c.num_heads * c.head_dim > (1 << 20) || cache_k == nullptr || cache_v == nullptr ||
      page_table == nullptr || token_batch == nullptr || token_position == nullptr ||
      k == nullptr || v == nullptr) {
    return hipErrorInvalidValue;
  }
  const int64_t width = (int64_t)c.num_heads * c.head_dim;
  if (kv_stride == 0) kv_stride = width;
  if (kv_stride < width || kv_stride % kPackElems != 0 || kv_stride > ((int64_t)1 << 30) ||
      !aligned16(cache_k) || !aligned16(cache_v) || !aligned16(k) || !aligned16(v)) {
    return hipErrorInvalidValue;
  }
  Fp8RowParams p{};
  p.cache_k = cache_k;
  p.cache_v = cache_v;
  p.k = k;
  p.v = v;
  p.k_scales = k_scales;
  p.v_scales = v_scales;
  p.page_table = page_table;
  p.token_batch = token_batch;
  p.token_position = token_position;
  p.c = c;
  p.kv_stride = kv_stride;
  p.row_packs = (int32_t)(width / kPackCodes);
  p.head_packs = c.head_dim / kPackCodes;
  p.packs = (int64_t)token_count * p.row_packs;
  p.rows = token_count;
  p.layer = layer;
  const int64_t slots = (int64_t)c.max_pages_per_seq * c.page_size;
  p.ring_rows = kWrite && c.window_size > 0 && slots < token_count ? (int32_t)slots : 0;
  const int64_t blocks = (p.packs + kRowThreads - 1) / kRowThreads;
  // A launch holds fewer than 2^32 threads.
  if (blocks * kRowThreads > 0xffffffffll) return hipErrorInvalidValue;
  hipLaunchKernelGGL(fp8_rows_kernel<kWrite>, dim3((uint32_t)blocks), dim3(kRowThreads), 0, stream,
                     p);
  return hipGetLastError();
}

}  // namespace
}  // namespace gemma4

using namespace gemma4;

extern "C" {

hipError_t gemma4_kv_cache_write_fp8(uint8_t *d_cache_k, uint8_t *d_cache_v,
                                     Gemma4KvCacheConfig config, const int32_t *d_page_table,
                                     const int32_t *d_token_batch, const int32_t *d_token_position,
                                     int32_t token_count, int32_t layer, const gemma4_bf16 *d_k,
                                     const gemma4_bf16 *d_v, int64_t kv_stride,
                                     const float *d_k_scales, const float *d_v_scales,
                                     hipStream_t stream) {
  return launch_rows<true>(
      d_cache_k, d_cache_v, config, d_page_table, d_token_batch, d_token_position, token_count,
      layer, const_cast<uint16_t *>(reinterpret_cast<const uint16_t *>(d_k)),
      const_cast<uint16_t *>(reinterpret_cast<const uint16_t *>(d_v)), kv_stride, d_k_scales,
      d_v_scales, stream);
}

hipError_t gemma4_kv_cache_read_fp8(gemma4_bf16 *d_k, gemma4_bf16 *d_v, const uint8_t *d_cache_k,
                                    const uint8_t *d_cache_v, Gemma4KvCacheConfig config,
                                    const int32_t *d_page_table, const int32_t *d_token_batch,
                                    const int32_t *d_token_position, int32_t token_count,
                                    int32_t layer, int64_t kv_stride, const float *d_k_scales,
                                    const float *d_v_scales, hipStream_t stream) {
  return launch_rows<false>(const_cast<uint8_t *>(d_cache_k), const_cast<uint8_t *>(d_cache_v),
                            config, d_page_table, d_token_batch, d_token_position, token_count,
                            layer, reinterpret_cast<uint16_t *>(d_k),
                            reinterpret_cast<uint16_t *>(d_v), kv_stride, d_k_scales, d_v_scales,
                            stream);
}

}  // extern "C"
