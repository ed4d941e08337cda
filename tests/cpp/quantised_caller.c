/* A plain C caller of the 8-bit cache, the preparation of ragged rows and the extension of
 * groups: sizes, frequencies, no-op calls and refusals, which need no GPU. Built and run
 * by tests/test_quantised_and_rope_refusals.py. */
#include "gemma4_flash_attention.h"
#include "gemma4_kv_cache.h"

#include <stdio.h>

int main(void) {
  Gemma4KvCacheConfig c = gemma4_kv_cache_make_config(false, 64, 16, 65);
  c.batch_size = 4;
  c.window_size = 0;
  const size_t one = gemma4_flash_attention_extend_shared_plan_bytes(c, 1, 1);
  const size_t plan = gemma4_flash_attention_extend_shared_plan_bytes(c, 4, 300);
  const size_t ws = gemma4_flash_attention_extend_shared_workspace_bytes(c, 4, 300);
  const int sizes = one > 0 && plan >= one && ws > plan &&
                    gemma4_flash_attention_extend_shared_plan_bytes(c, 5, 300) == 0;
  double turns[64];
  float amplitude = 0.0f;
  int32_t split = 0, count = 0;
  const int host =
      gemma4_rope_frequencies(turns, &amplitude, 128, 512, 1e6, GEMMA4_ROPE_BY_PARTS, 8.0, 32768.0,
                              32.0, 1.0) == hipSuccess &&
      turns[0] > turns[63] && turns[63] > 0.0 && amplitude > 1.2f && amplitude < 1.21f &&
      gemma4_decode_split_plan_fp8(c, 2, 1000, 0, &split, &count) == hipSuccess &&
      split * count >= 1000;
  const int nothing =
      gemma4_flash_attention_extend_shared_paged_bf16(0, 0, 0, 0, 0, 0, 0, 0, 0, c, 0, 4, 0, 0, 0,
                                                      1.0f, 0, 0, 0) == hipSuccess &&
      gemma4_rope_rows_bf16(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1.0f, 128, 0, 1, 512, 0, 0, 0, 0) ==
          hipSuccess &&
      gemma4_kv_cache_write_fp8(0, 0, c, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0) == hipSuccess &&
      gemma4_kv_cache_read_fp8(0, 0, 0, 0, c, 0, 0, 0, 0, 0, 0, 0, 0, 0) == hipSuccess;
  const int refused =
      gemma4_kv_cache_write_fp8(0, 0, c, 0, 0, 0, 1, 0, 0, 0, 0, 0, 0, 0) == hipErrorInvalidValue &&
      gemma4_flash_attention_decode_paged_fp8(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, c, 0, 1.0f, 64, 1, 1,
                                              0) == hipErrorInvalidValue &&
      gemma4_flash_attention_append_decode_paged_fp8(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, c, 0,
                                                     1.0f, 64, 1, 1, 0) == hipErrorInvalidValue &&
      gemma4_flash_attention_extend_shared_plan(0, plan, 0, 0, 0, 0, 1, c, 4, 300, 0) ==
          hipErrorInvalidValue;
  printf(sizes && host && nothing && refused ? "quantised caller ok\n" : "quantised caller FAILED\n");
  return sizes && host && nothing && refused ? 0 : 1;
}
