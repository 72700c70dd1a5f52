// Index arithmetic of the paged E4M3 key/value cache: plain C++, shared by the kernels and by host programs that check it.  Tables cover fewer
// than 2^30 positions (the entries refuse others).
//
// A cache is a pool of pages: keys [pages][kv_heads][page][dim], values [pages][kv_heads][dim][page] (a page's tokens innermost, which is how
// the matrix cores want the second operand of the value product), one power-of-two float32 scale per page and head for each.  A page holds
// 16 .. 128 tokens, a power of two: any 16 neighbouring positions that begin at a multiple of 16 lie in one page.  A table row lists the pages
// of one sequence.  Lengths, offsets and page numbers are device data that no host check sees: every one is clamped or tested here, so that no
// content of these arrays leads a kernel outside its buffers.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define PLLM_HD __host__ __device__ __forceinline__
#else
#define PLLM_HD inline
#endif

namespace pllm {

constexpr int kPagedChunk = 16;                 // positions that are certain to share a page
constexpr int kPagedRunStep = 256;              // keys that a workgroup of the decode kernel takes at a time
constexpr int kPagedOneRun = 1024;              // sequences of up to so many keys are one run of it
constexpr int kPagedLeastRun = 512;             // and longer ones are cut in runs of at least so many

PLLM_HD int clamp_int(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }

// positions of a sequence that the cache can hold: never more than its table row covers
PLLM_HD int paged_length(int length, int width, int page_shift) {
    const int64_t most = static_cast<int64_t>(width) << page_shift;
    return length < 0 ? 0 : (length > most ? static_cast<int>(most) : length);
}

// row offsets of the sequences' new tokens: offset `s` of `seqs`, never outside the rows
PLLM_HD int paged_offset(const int32_t* cu_steps, int s, int even_steps, int rows) {
    if (s <= 0) return 0;
    return clamp_int(cu_steps ? cu_steps[s] : s * even_steps, 0, rows);
}

// The pages that ragged rows go to are dealt out (units of a page's tokens) without a plan made beforehand: sequence s has the slots
// from offset_s / unit + spare * s on.  Offsets that grow give every sequence at least n / unit + spare slots of its own.
PLLM_HD int64_t paged_first_slot(int64_t offset, int s, int unit, int spare) { return offset / unit + static_cast<int64_t>(spare) * s; }
PLLM_HD int64_t paged_slots(int64_t rows, int seqs, int unit, int spare) { return rows / unit + static_cast<int64_t>(spare) * seqs; }

// pages that `steps` neighbouring positions touch at most
PLLM_HD int64_t paged_pages_touched(int64_t steps, int64_t page) { return steps <= 0 ? 1 : (steps + page - 2) / page + 1; }

// Blocks of `block` query rows of one sequence that see keys of at least `tiles` tiles of 64: the last ones, since a row sees no fewer keys than those
// before it.  `rows` = new tokens * group, the first of which see `first` + 1 keys.
PLLM_HD int paged_blocks_seeing(int tiles, int rows, int first, int group, int block) {
    const int blocks = (rows + block - 1) / block;
    const int64_t need = (64 * (static_cast<int64_t>(tiles) - 1) - first) * group;           // the first row that does
    if (tiles <= 0 || need <= 0) return blocks;
    return need > rows - 1 ? 0 : blocks - static_cast<int>(need / block);
}

// page number of a position, or -1 where the table has none that lies in the pool
PLLM_HD int paged_page(const int32_t* table_row, int position, int width, int page_shift, int pool) {
    const int at = position >> page_shift;
    if (position < 0 || at >= width) return -1;
    const int page = table_row[at];
    return page >= 0 && page < pool ? page : -1;
}

// Drafted trees.  The new tokens of a sequence are nodes, parents[i] the node that i hangs from: an earlier one, or -1 (anything that is not an earlier node) where
// it follows the past.  A node sees the past, its ancestors and itself.
constexpr int kTreeNodes = 256;                 // nodes that a tree can have; of one with more no node sees anything
constexpr int kTreeWords = kTreeNodes / 64;

// position of a tree's first node, of a sequence of `length` positions whose last `n` are the tree's: below zero where the first nodes have none
PLLM_HD int tree_past(int length, int n) {
    const int64_t past = static_cast<int64_t>(length) - n;
    return past < -2 * kTreeNodes ? -2 * kTreeNodes : static_cast<int>(past);
}

// ancestors of node `i` and itself, a bit each; ends whatever parents hold, since every step goes to an earlier node
template <int WORDS, typename Parents> PLLM_HD void tree_ancestors(const Parents& parents, int i, uint64_t (&bits)[WORDS]) {
    for (int w = 0; w < WORDS; ++w) bits[w] = 0;
    while (i >= 0 && i < 64 * WORDS) {
        for (int w = 0; w < WORDS; ++w) bits[w] |= i >> 6 == w ? uint64_t{1} << (i & 63) : 0;
        const int up = parents[i];
        i = up < i ? up : -1;
    }
}

// Keys `first` .. + 63 that a node sees, a bit each, of a sequence whose tree begins at position `past`: those of the past, the ancestors' and its own; none from
// position `limit` on.  Words behind the node's are zero.
PLLM_HD uint64_t tree_window(const uint64_t* bits, int words, int64_t past, int64_t first, int64_t limit) {
    if (first >= limit) return 0;
    const uint64_t there = limit - first >= 64 ? ~uint64_t{0} : (uint64_t{1} << (limit - first)) - 1;
    const int64_t base = first - past;                                        // node of the window's first key
    if (base <= -64) return there;
    if (base >= 64 * static_cast<int64_t>(words)) return 0;
    if (base < 0) return ((bits[0] << -base) | ((uint64_t{1} << -base) - 1)) & there;
    const int word = static_cast<int>(base >> 6), shift = static_cast<int>(base & 63);
    const uint64_t low = bits[word] >> shift, high = shift > 0 && word + 1 < words ? bits[word + 1] << (64 - shift) : 0;
    return (low | high) & there;
}

// Keys of one run of the decode kernel.  By the sequence's own length and the number of heads alone, so that a sequence's sums have the
// same order in every batch: runs of at least kPagedLeastRun keys, as long as one sequence has no more of them than fill the machine.
PLLM_HD int paged_most_runs(int kv_heads) { return clamp_int(512 / kv_heads, 8, 256); }
PLLM_HD int paged_run_keys(int length, int kv_heads) {
    const int most = paged_most_runs(kv_heads), steps = (length + kPagedRunStep - 1) / kPagedRunStep;
    const int per = (steps + most - 1) / most;
    if (length <= kPagedOneRun) return kPagedOneRun;
    return (per * kPagedRunStep < kPagedLeastRun ? kPagedLeastRun : per * kPagedRunStep);
}
PLLM_HD int paged_runs(int length, int kv_heads) {
    const int keys = paged_run_keys(length, kv_heads);
    return (length + keys - 1) / keys;
}
// runs that a sequence of up to `length` positions can have
PLLM_HD int paged_runs_bound(int64_t length, int kv_heads) {
    const int64_t runs = length <= kPagedOneRun ? 1 : (length + kPagedLeastRun - 1) / kPagedLeastRun;
    const int most = paged_most_runs(kv_heads);
    return runs < 1 ? 1 : (runs < most ? static_cast<int>(runs) : most);
}

}  // namespace pllm
