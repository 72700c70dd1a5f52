// The paged cache's index arithmetic (pocketllm_amd/csrc/paged_cache.h) for tests without a GPU: built with g++.
#include "../pocketllm_amd/csrc/paged_cache.h"

extern "C" {
int idx_length(int length, int width, int shift) { return pllm::paged_length(length, width, shift); }
int idx_offset(const int32_t* cu, int s, int even, int rows) { return pllm::paged_offset(cu, s, even, rows); }
int64_t idx_first_slot(int64_t offset, int s, int unit, int spare) { return pllm::paged_first_slot(offset, s, unit, spare); }
int64_t idx_slots(int64_t rows, int seqs, int unit, int spare) { return pllm::paged_slots(rows, seqs, unit, spare); }
int idx_page(const int32_t* row, int position, int width, int shift, int pool) { return pllm::paged_page(row, position, width, shift, pool); }
int idx_blocks_seeing(int tiles, int rows, int first, int group, int block) { return pllm::paged_blocks_seeing(tiles, rows, first, group, block); }
int64_t idx_pages_touched(int64_t steps, int64_t page) { return pllm::paged_pages_touched(steps, page); }
int idx_run_keys(int length, int kv_heads) { return pllm::paged_run_keys(length, kv_heads); }
int idx_runs(int length, int kv_heads) { return pllm::paged_runs(length, kv_heads); }
int idx_runs_bound(int64_t length, int kv_heads) { return pllm::paged_runs_bound(length, kv_heads); }
}
