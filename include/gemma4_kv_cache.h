// Paged bf16 K/V cache for gemma.c's attention layers, MI355X (gfx950) build.
//
// Drop-in for the reference header src/gemma4_kv_cache.cuh: same struct
// layout, names, argument order and error convention, with HIP types
// (hipError_t / hipStream_t / __hip_bfloat16) in place of the CUDA ones.
// Every device entry point is extern "C" and takes plain pointers and sizes.
#pragma once

#include <hip/hip_runtime_api.h>
#include <stdint.h>

#ifdef __cplusplus
struct __hip_bfloat16;  // complete in <hip/hip_bf16.h>; only pointers cross this API
typedef struct __hip_bfloat16 gemma4_bf16;
#include <vector>
#else
#include <stdbool.h>
typedef uint16_t gemma4_bf16;  // C callers pass raw bf16 bit patterns
#endif

#if defined(__HIPCC__)
#define GEMMA4_HOST_DEVICE __host__ __device__
#else
#define GEMMA4_HOST_DEVICE
#endif
#ifdef __cplusplus
#define GEMMA4_CONSTEXPR constexpr
#else
#define GEMMA4_CONSTEXPR
#endif

// Replaces src/gemma4_kv_cache.cuh:9-18 (same 8 x int32 layout, 32 bytes).
// window_size == 0 marks a full-length global cache; > 0 a sliding ring.
typedef struct Gemma4KvCacheConfig {
  int32_t num_layers;
  int32_t num_pages;
  int32_t page_size;
  int32_t max_pages_per_seq;
  int32_t batch_size;
  int32_t num_heads;
  int32_t head_dim;
  int32_t window_size;
} Gemma4KvCacheConfig;

// Replaces src/gemma4_kv_cache.cuh:27-38. Flat Layout-A element offset
// [layer][page][page_offset][head][dim]; constexpr in C++ (usable in
// constant expressions, as the reference's is).
static inline GEMMA4_CONSTEXPR GEMMA4_HOST_DEVICE int64_t gemma4_kv_cache_offset(
    const Gemma4KvCacheConfig *config, int32_t layer, int32_t page,
    int32_t page_offset, int32_t head, int32_t dim) {
  const int64_t layer_page = (int64_t)layer * config->num_pages + page;
  const int64_t token = layer_page * config->page_size + page_offset;
  return (token * config->num_heads + head) * config->head_dim + dim;
}

#ifdef __cplusplus
// Reference-style overload taking the config by reference
// (src/gemma4_kv_cache.cuh:28, __host__ __device__ constexpr).
static inline constexpr GEMMA4_HOST_DEVICE int64_t gemma4_kv_cache_offset(
    const Gemma4KvCacheConfig &config, int32_t layer, int32_t page,
    int32_t page_offset, int32_t head, int32_t dim) {
  return gemma4_kv_cache_offset(&config, layer, page, page_offset, head, dim);
}

// Replaces src/gemma4_kv_cache.cuh:42-53 (host ring-slot bookkeeping with the
// reference's std::vector arguments). Return the physical page, or -1 when
// the slot already holds a newer logical page.
int32_t gemma4_kv_cache_ensure_page(std::vector<int32_t> &page_table,
                                    std::vector<int32_t> &slot_logical_pages,
                                    const Gemma4KvCacheConfig &config,
                                    int32_t batch, int32_t position);
int32_t gemma4_kv_cache_ensure_range(std::vector<int32_t> &page_table,
                                     std::vector<int32_t> &slot_logical_pages,
                                     const Gemma4KvCacheConfig &config,
                                     int32_t batch, int32_t first_position,
                                     int32_t token_count);
extern "C" {
#endif

// Replaces src/gemma4_kv_cache.cuh:20-23 (src/gemma4_kv_cache.cu:76-91).
Gemma4KvCacheConfig gemma4_kv_cache_make_config(bool global, int32_t num_pages,
                                                int32_t page_size,
                                                int32_t max_pages_per_seq);

// Replaces src/gemma4_kv_cache.cuh:25 (src/gemma4_kv_cache.cu:94-105).
int32_t gemma4_kv_cache_layer_index(int32_t model_layer, bool global_cache);

// Plain-pointer forms of the two std::vector helpers above, for C / FFI
// callers. `entries` is the length of both arrays
// (batch_size * max_pages_per_seq); out-of-range slots return -1.
int32_t gemma4_kv_cache_ensure_page_ptr(int32_t *page_table,
                                        int32_t *slot_logical_pages,
                                        int64_t entries,
                                        const Gemma4KvCacheConfig *config,
                                        int32_t batch, int32_t position);
int32_t gemma4_kv_cache_ensure_range_ptr(int32_t *page_table,
                                         int32_t *slot_logical_pages,
                                         int64_t entries,
                                         const Gemma4KvCacheConfig *config,
                                         int32_t batch, int32_t first_position,
                                         int32_t token_count);

// Replaces src/gemma4_kv_cache.cuh:55-66 (src/gemma4_kv_cache.cu:149-180).
// Stream-ordered bit-exact copy of prepared K/V rows [token][num_heads][head_dim]
// into the paged cache. Rows whose batch/position/page is out of range are
// skipped on the device. token_count == 0 is a no-op success; bad geometry or
// null pointers return hipErrorInvalidValue before any launch.
// A sequence may bring more rows than its ring has slots (max_pages_per_seq *
// page_size) where they follow each other in the call, at consecutive positions:
// the newest of a slot stays. Other rows for one place (the same position twice, a
// lap out of order) must not come in one call.
hipError_t gemma4_kv_cache_write_bf16(
    gemma4_bf16 *d_cache_k, gemma4_bf16 *d_cache_v, Gemma4KvCacheConfig config,
    const int32_t *d_page_table, const int32_t *d_token_batch,
    const int32_t *d_token_position, int32_t token_count, int32_t layer,
    const gemma4_bf16 *d_k, const gemma4_bf16 *d_v, hipStream_t stream);

// Prefill-chunk cache write policy of src/gemma4_prefill_megakernel.cu:189-207:
// rows are batch-major [batch][seq_len]; a global cache, or a chunk of at most
// `window_size` rows, writes every row; a longer chunk into a sliding ring
// writes only the last `window_size` rows of each batch (the live ring tail).
// One launch covers all batches.
hipError_t gemma4_kv_cache_write_prefill_bf16(
    gemma4_bf16 *d_cache_k, gemma4_bf16 *d_cache_v, Gemma4KvCacheConfig config,
    const int32_t *d_page_table, const int32_t *d_token_batch,
    const int32_t *d_token_position, int32_t batch_size, int32_t seq_len,
    int32_t layer, const gemma4_bf16 *d_k, const gemma4_bf16 *d_v,
    hipStream_t stream);

// ---- a cache in 8 bits ------------------------------------------------------------
// Rows as e4m3 codes, one byte an element in the layout of the bf16 cache: half the
// bytes per token. A value is code * scale, the scale d_k_scales / d_v_scales
// [num_layers][num_heads], fixed while a cache is in use (null: 1; positive and
// finite). The codes are floating-point numbers of four significant bits from 2^-6 to 448
// and in steps of 2^-9 below, so a scale only has to keep what occurs within that range:
// prepared rows are RMS-normed, |x| <= sqrt(head_dim) * max |weight| (times the rotation's
// amplitude for K), and that bound / 448 never saturates. No counterparts in the reference.
// The page pool serves such a cache as it is, its rows are half as long: reserve, release,
// gemma4_kv_cache_fork_bf16 and gemma4_kv_cache_compact_bf16 with head_dim / 2 in the
// config and the codes as bf16.
//
// Writes prepared rows as gemma4_kv_cache_write_bf16 does (the same tokens are skipped,
// the same rows of a lap stay): code = x / scale, the quotient
// rounded to 32 bits, to the nearest code, ties to even, beyond +-448 to that; NaN stays NaN. k and v rows are kv_stride elements apart
// (a multiple of 8 up to 2^30; 0: packed). head_dim is a multiple of 16; caches, k
// and v are 16-byte aligned; token_count * num_heads * head_dim / 16 < 2^32 - 256.
hipError_t gemma4_kv_cache_write_fp8(uint8_t *d_cache_k, uint8_t *d_cache_v,
                                     Gemma4KvCacheConfig config, const int32_t *d_page_table,
                                     const int32_t *d_token_batch, const int32_t *d_token_position,
                                     int32_t token_count, int32_t layer, const gemma4_bf16 *d_k,
                                     const gemma4_bf16 *d_v, int64_t kv_stride,
                                     const float *d_k_scales, const float *d_v_scales,
                                     hipStream_t stream);

// Reads rows back: row i of k and v gets the values of (d_token_batch[i],
// d_token_position[i]), the products in 32 bits rounded to bf16; a row whose token the write would skip is
// left as it was. Over a ring a position names its slot, whichever lap it holds. Packed
// rows are a bf16 cache of their own (page tables that count up), over which a prompt's
// chunk attends. Limits as above.
hipError_t gemma4_kv_cache_read_fp8(gemma4_bf16 *d_k, gemma4_bf16 *d_v, const uint8_t *d_cache_k,
                                    const uint8_t *d_cache_v, Gemma4KvCacheConfig config,
                                    const int32_t *d_page_table, const int32_t *d_token_batch,
                                    const int32_t *d_token_position, int32_t token_count,
                                    int32_t layer, int64_t kv_stride, const float *d_k_scales,
                                    const float *d_v_scales, hipStream_t stream);

// ---- pages of a pool -------------------------------------------------------
// The operators below let page tables map any page of the cache instead of a
// fixed one per slot (no counterparts in the reference, whose
// src/gemma4_kv_cache.cu:108-122 maps physical page batch * max_pages_per_seq +
// slot). The state is the page table [batch_size][max_pages_per_seq] (-1:
// unmapped) and d_page_refs [num_pages], the number of table entries that map a
// page (0: free); both start as -1 and 0 everywhere. One table and one count
// array per cache: the layers of a cache share them, and `config` is that
// cache's. batch_size is at most 4096, batch_size * max_pages_per_seq and
// num_pages * page_size below 2^31. All are stream-ordered, allocate nothing, and
// give the same result on every run: free pages are handed out lowest first, in
// the order of the table entries. Calls that share a table, counts or a cache
// must not overlap.
//
// Positions of a sliding cache name ring slots: logical page p sits in slot
// p % max_pages_per_seq, as in gemma4_kv_cache_write_bf16, and a range of positions
// means these slots, whichever lap of the ring they hold: one that is as long as the
// ring means all of it.

// Returns pages: for every sequence b < batch_size, the pages that lie wholly in
// positions [d_first_position[b], d_end_position[b]) are unmapped and lose one
// reference each. 0 .. INT32_MAX: all of the sequence's. Over a full-length cache
// also length .. INT32_MAX: what a shortened sequence no longer needs, and sinks ..
// length - window: what no row of a windowed sequence will see again. Over a ring
// those two would reach live slots: a shortened sequence there gives back new length
// .. old length, or nothing; what the window has passed is overwritten in its place.
// An empty range changes nothing.
hipError_t gemma4_kv_cache_release_pages(int32_t *d_page_table, int32_t *d_page_refs,
                                         Gemma4KvCacheConfig config,
                                         const int32_t *d_first_position,
                                         const int32_t *d_end_position, hipStream_t stream);

// Takes pages: for every sequence b < batch_size, every unmapped page that holds
// a position of [d_first_position[b], d_end_position[b]) gets a free page with
// one reference. A range that begins behind position 0 is where a sequence goes on:
// its rows will be written, so no page of it may be shared; one from 0 on may hold
// shared pages. *d_status: 0, or with nothing changed 1 (not enough free pages), 2 (a
// negative first position of a range, or one past a full-length table's end; comes
// before the others) or 3 (a page that will be written is mapped more than once; comes
// before 1). That is a branch, or its parent, that was shortened into the pages they
// share: release what lies behind its new length, then, if it ends within a page, fork
// it to an empty sequence, which gets that page as its own, release it whole, and go
// on with the new one.
hipError_t gemma4_kv_cache_reserve_pages(int32_t *d_page_table, int32_t *d_page_refs,
                                         Gemma4KvCacheConfig config,
                                         const int32_t *d_first_position,
                                         const int32_t *d_end_position, int32_t *d_status,
                                         hipStream_t stream);

// Branches sequences: child d_children[i] becomes a copy of d_parents[i] as it
// stands at d_seq_lengths[d_parents[i]], which becomes the child's length too. A
// full-length cache's whole pages are shared (one more reference each); the begun
// page, which both will write to, is copied into a page of the child's own: its
// live rows of every layer, K and V. Pages mapped ahead of the length stay the
// parent's. A sliding ring's pages will all be written again and are all copied.
// A child must hold no page (release it first), be named once and be no parent
// in the call; fork_count <= batch_size. *d_status: 0, or with nothing changed 1
// (not enough free pages) or 2 (a sequence out of range or named against these
// rules, a length out of range). fork_count == 0 is a no-op success. Caches are
// 16-byte aligned. Copies are launched in pieces of 32 KiB of a page: fork_count *
// (a ring's max_pages_per_seq, or 1) * pieces is below 2^24.
hipError_t gemma4_kv_cache_fork_bf16(gemma4_bf16 *d_cache_k, gemma4_bf16 *d_cache_v,
                                     Gemma4KvCacheConfig config, int32_t *d_page_table,
                                     int32_t *d_page_refs, int32_t *d_seq_lengths,
                                     const int32_t *d_parents, const int32_t *d_children,
                                     int32_t fork_count, int32_t *d_status, hipStream_t stream);

// Closes up kept tokens: for request i < sequence_count, the rows of sequence
// d_sequences[i] at positions d_kept_positions[d_kept_offsets[i] ..
// d_kept_offsets[i + 1]) move to d_first_positions[i], + 1, + 2, ..., in place,
// in every layer, K and V (the accepted tokens of a verified draft; a prompt
// thinned out). Rows move as they are: a key keeps the rotation of its old
// position. (A ring has lost the keys that rejected tokens overwrote: one that
// verifies n drafts needs n slots more than its window.) A request's positions ascend strictly, none lies before its new
// place, and for a sliding cache all lie within the ring's slots of the first
// position. d_page_refs may be null where no page is shared; otherwise a request
// that would write to a page with more than one reference is refused (a way on: see
// gemma4_kv_cache_reserve_pages).
// d_status[i]: 0, or with the sequence's rows unchanged 1 (a list, sequence or
// position against these rules, two requests for one sequence), 2 (a page is
// unmapped) or 3 (a destination page is shared), the lowest where several hold.
// total_kept is the length of d_kept_positions. The table, the counts and the lengths stay as they are.
// sequence_count == 0 is a no-op success; sequence_count <= batch_size.
hipError_t gemma4_kv_cache_compact_bf16(gemma4_bf16 *d_cache_k, gemma4_bf16 *d_cache_v,
                                        Gemma4KvCacheConfig config, const int32_t *d_page_table,
                                        const int32_t *d_page_refs, const int32_t *d_sequences,
                                        const int32_t *d_first_positions,
                                        const int32_t *d_kept_offsets,
                                        const int32_t *d_kept_positions, int32_t sequence_count,
                                        int32_t total_kept, int32_t *d_status,
                                        hipStream_t stream);

#ifdef __cplusplus
}  // extern "C"
#endif
