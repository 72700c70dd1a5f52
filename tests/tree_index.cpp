// The index arithmetic of drafted trees for the host.
#include "../pocketllm_amd/csrc/paged_cache.h"

extern "C" {
int idx_tree_past(int length, int n) { return pllm::tree_past(length, n); }
void idx_tree_ancestors(const int32_t* parents, int i, uint64_t* bits) {
    uint64_t b[pllm::kTreeWords];
    pllm::tree_ancestors(parents, i, b);
    for (int w = 0; w < pllm::kTreeWords; ++w) bits[w] = b[w];
}
void idx_tree_ancestors_one(const int32_t* parents, int i, uint64_t* bits) {
    uint64_t b[1];
    pllm::tree_ancestors(parents, i, b);
    bits[0] = b[0];
}
uint64_t idx_tree_window(const uint64_t* bits, int words, int64_t past, int64_t first, int64_t limit) { return pllm::tree_window(bits, words, past, first, limit); }
}
