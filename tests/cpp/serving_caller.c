/* A plain C caller of the page pool and the ragged extension: sizes, no-op calls
 * and refusals, which need no GPU. Built and run by tests/test_serving_refusals.py. */
#include "gemma4_flash_attention.h"
#include "gemma4_kv_cache.h"

#include <stdio.h>

int main(void) {
  Gemma4KvCacheConfig c = gemma4_kv_cache_make_config(false, 64, 16, 65);
  c.batch_size = 4;
  c.window_size = 0;
  const size_t one = gemma4_flash_attention_extend_plan_bytes(c, 1, 1);
  const size_t plan = gemma4_flash_attention_extend_plan_bytes(c, 4, 300);
  const size_t ws = gemma4_flash_attention_extend_workspace_bytes(c, 4, 300);
  const int sizes = one > 0 && plan >= one && ws > plan &&
                    gemma4_flash_attention_extend_plan_bytes(c, 5, 300) == 0;
  const int nothing =
      gemma4_flash_attention_extend_paged_bf16(0, 0, 0, 0, 0, 0, 0, 0, 0, c, 0, 4, 0, 0, 0, 1.0f, 0,
                                               0, 0) == hipSuccess &&
      gemma4_kv_cache_fork_bf16(0, 0, c, 0, 0, 0, 0, 0, 0, 0, 0) == hipSuccess &&
      gemma4_kv_cache_compact_bf16(0, 0, c, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0) == hipSuccess;
  const int refused =
      gemma4_kv_cache_reserve_pages(0, 0, c, 0, 0, 0, 0) == hipErrorInvalidValue &&
      gemma4_kv_cache_release_pages(0, 0, c, 0, 0, 0) == hipErrorInvalidValue &&
      gemma4_flash_attention_extend_plan(0, plan, 0, 0, c, 4, 300, 0, 0, 0) == hipErrorInvalidValue;
  printf(sizes && nothing && refused ? "serving caller ok\n" : "serving caller FAILED\n");
  return sizes && nothing && refused ? 0 : 1;
}
