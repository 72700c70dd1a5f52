// The decode attention over the paged E4M3 cache as the prompt attention calls it for sequences of few rows.
#pragma once

#include "pllm_internal.h"

namespace pllm {

struct PagedDecodeArgs {
    const uint16_t* q; size_t q_stride;         // elements between tokens
    const uint8_t* key_pages; const uint8_t* value_pages;
    const float* key_scales; const float* value_scales;
    const int32_t* table; size_t table_stride;
    const int32_t* lengths; const int32_t* cu_steps;         // cu_steps null: `steps` new tokens each
    const int32_t* parents;                     // of the new tokens, which are nodes of drafted trees (at most 64 each); null: they follow one another
    float* sums; float2* stats;                 // of the runs of a row: [seqs][kv_heads][part_rows][runs_bound][D], m (base 2) and sum of weights; null: one run
    uint16_t* out;
    float scale;                                // base 2
    int seqs, steps, tokens, heads, kv_heads, page_shift, pool, width, runs_bound;
    int part_rows;                              // query rows (new tokens * heads of a key/value head) that a sequence can have; those with more are left alone
};

// bytes of `sums` and `stats` together, `sums` first (0: one run)
size_t paged_decode_parts_bytes(int64_t seqs, int64_t part_rows, int64_t kv_heads, int64_t head_dim, int64_t positions);
// sets sums, stats and runs_bound from a workspace of that many bytes, then launches
int paged_decode_launch(PagedDecodeArgs& a, void* workspace, bool bf16, int head_dim, hipStream_t stream);

constexpr int kPagedFewRows = 64;               // query rows of a sequence up to which the decode kernel may take it in a call of mixed lengths

}  // namespace pllm
