// What happens to the pages of a paged E4M3 cache between two steps: the accepted path of a drafted tree moves to the places right behind the past, and the sequences
// of the next step come out of the present ones, pages shared, copied, taken and freed.  All layers of a model in one launch: they share the table.
#include "paged_device.h"
#include "pllm_internal.h"

#include <algorithm>

namespace pllm {
namespace {

constexpr int kLayers = 64;                     // layers of a launch (their addresses are among the kernel's arguments)
struct Layer { uint8_t* key_pages; uint8_t* value_pages; float* key_scales; float* value_scales; };
struct Layers { Layer layer[kLayers]; };

// ---- the accepted path ------------------------------------------------------------------------------------------------
//
// Token `first` + kept[j] of a sequence becomes token `first` + j, first = length - n.  kept rises, so every destination is at or before its source, and what a stretch
// of the path is written over is no later stretch's source.  The new scale of a page is the largest of the scales that its
// content had (its own, where it keeps older tokens or a token moves within it): codes are scaled down to it by a power of two, exact but for those that get below E4M3's
// normal values, which are rounded again.
// A workgroup has a sequence's keys, or values, of one head and layer.  Bound: a value's token is one byte in each of D rows, so whatever it is, the lines of whole pages are
// read and written for it: 32 sequences of up to 26 nodes, eight layers of 8 heads in pages of 16, 12.5 us for about 20 MB of lines (4 us), and of the chain of loads (path, table,
// scales, codes) of a workgroup 5 us.

struct CompactArgs {
    const int32_t* table; size_t table_stride;
    const int32_t* lengths; const int32_t* kept; const int32_t* counts; const int32_t* cu_steps;
    int even, most, kv_heads, pool, width, page_shift;
};

constexpr int kCompactThreads = 128, kCompactStretch = 64;                    // tokens whose codes are on their way together
template <int D>
__global__ __launch_bounds__(kCompactThreads) void paged_compact_kernel(const Layers layers, const CompactArgs a) {
    constexpr int kThreads = kCompactThreads, kWaves = kThreads / 64;
    // of token j of the path: where it comes from and goes to, from the layer's first code on, or -1; its node; the scales of the two pages; what its codes are multiplied
    // by, negative where it stays as it is.  All of them, and all codes of a stretch, at once: one page after the other each waits for its own loads
    extern __shared__ __align__(16) uint8_t smem[];
    const int room = a.most;
    int64_t* const sources = reinterpret_cast<int64_t*>(smem);
    int64_t* const targets = sources + room;
    int* const nodes = reinterpret_cast<int*>(targets + room);
    float* const ratio = reinterpret_cast<float*>(nodes + room);
    float* const target_scale = ratio + room;
    float* const factors = target_scale + room;
    uint8_t* const rows = reinterpret_cast<uint8_t*>(factors + room);         // [tokens of a stretch][D] (on 16 bytes: 32 for a token are in front of it)
    __shared__ int good;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), kind = blockIdx.x & 1, head = blockIdx.x >> 1, s = blockIdx.y;
    const Layer& layer = layers.layer[blockIdx.z];
    uint8_t* const pages = kind ? layer.value_pages : layer.key_pages;
    float* const scales = kind ? layer.value_scales : layer.key_scales;
    const int page_tokens = 1 << a.page_shift;
    // offsets as the attention takes them, without the number of rows, which nothing here is indexed by
    int64_t n = a.even;
    if (a.cu_steps) n = static_cast<int64_t>(max(a.cu_steps[s + 1], 0)) - (s > 0 ? max(a.cu_steps[s], 0) : 0);
    if (n <= 0 || n > kTreeNodes) return;
    const int count0 = min(min(max(a.counts[s], 0), a.most), static_cast<int>(n));
    const int64_t first64 = static_cast<int64_t>(a.lengths[s]) - n;
    if (count0 == 0 || first64 < -kTreeNodes || first64 >= static_cast<int64_t>(a.width) << a.page_shift) return;
    const int first = static_cast<int>(first64);
    const int32_t* table = a.table + static_cast<size_t>(s) * a.table_stride;
    if (tid == 0) good = count0;
    __syncthreads();
    for (int j = tid; j < count0; j += kThreads) {
        const int32_t* kept = a.kept + static_cast<size_t>(s) * a.most;
        const int node = kept[j], before = j ? kept[j - 1] : -1;
        if (node <= before || before < (j ? 0 : -1) || node >= n) {
            atomicMin(&good, j);                                              // from here on it is no path
            continue;
        }
        const int source = paged_page(table, first + node, a.width, a.page_shift, a.pool), target = paged_page(table, first + j, a.width, a.page_shift, a.pool);
        auto place = [&](int page, int position) {
            const int slot = position & (page_tokens - 1);
            return page < 0 ? int64_t{-1} : (static_cast<int64_t>(page) * a.kv_heads + head) * (static_cast<int64_t>(D) << a.page_shift) + (kind ? slot : slot * D);
        };
        nodes[j] = node;
        sources[j] = place(source, first + node);
        targets[j] = place(target, first + j);
        ratio[j] = source < 0 ? 0.0f : scales[static_cast<size_t>(source) * a.kv_heads + head];
        target_scale[j] = target < 0 ? 0.0f : scales[static_cast<size_t>(target) * a.kv_heads + head];
    }
    __syncthreads();
    const int count = good;
    if (count == 0) return;
    const int last_page = (first + count - 1) >> a.page_shift;
    const int page_first = max(first, 0) >> a.page_shift, held = max(first, 0) & (page_tokens - 1);           // slots of the first page that it keeps
    float held_factor = 1.0f;                                                 // what they are multiplied by
    bool moved = false;
    for (int j = tid; j < count; j += kThreads) factors[j] = -1.0f;
    __syncthreads();
    // every page's new scale
    for (int p = page_first; p <= last_page && p < a.width; ++p) {
        const int page0 = p << a.page_shift, from = max(max(first, 0), page0), to = min(first + count, page0 + page_tokens);
        const int tokens = to - from, j0 = from - first;
        if (tokens <= 0 || nodes[j0 + tokens - 1] == j0 + tokens - 1) continue;              // (all of them where they are)
        if (targets[j0] < 0) continue;
        const bool keeps = p == page_first && held > 0;
        const float own = target_scale[j0];
        bool moves = false;
        float most = keeps ? own : 0.0f;
        for (int t = tid & 63; t < tokens; t += 64) {                         // (every wave for itself)
            moves |= sources[j0 + t] >= 0;
            most = fmaxf(most, ratio[j0 + t]);
        }
        if (!__any(moves)) continue;
        moved = true;
        most = group_max<64>(most);
        if (keeps && own != most) held_factor = own / most;
        if (tid >= 64) continue;
        for (int t = tid; t < tokens; t += 64)
            if (sources[j0 + t] >= 0) factors[j0 + t] = ratio[j0 + t] == most ? 1.0f : ratio[j0 + t] / most;
        if (tid == 0) scales[static_cast<size_t>(targets[j0] >> (a.page_shift + (D == 128 ? 7 : 6)))] = most;
    }
    if (!moved) return;                                                       // (all waves alike)
    __syncthreads();
    for (int j0 = 0; j0 < count; j0 += kCompactStretch) {
        const int tokens = min(count - j0, kCompactStretch);
        // the rows, scaled, to LDS: [token][D]
        if (!kind) {
            for (int i = tid; i < tokens * (D / 16); i += kThreads) {
                const int t = i / (D / 16), piece = i % (D / 16);
                const float r = factors[j0 + t];
                if (r < 0.0f) continue;
                uint4 w = *reinterpret_cast<const uint4*>(pages + sources[j0 + t] + 16 * piece);
                if (r != 1.0f) w = make_uint4(scaled_codes(w.x, r), scaled_codes(w.y, r), scaled_codes(w.z, r), scaled_codes(w.w, r));
                *reinterpret_cast<uint4*>(rows + t * D + 16 * piece) = w;
            }
        } else {
            // a wave takes every kWaves-th token, a lane its codes of dimensions lane, lane + 64
            constexpr int kAtOnce = 4, kPer = D / 64;                         // requests on their way: of so many tokens
            for (int t0 = wave; t0 < tokens; t0 += kAtOnce * kWaves) {
                uint32_t w[kAtOnce][kPer];
#pragma unroll
                for (int u = 0; u < kAtOnce; ++u) {
                    const int t = j0 + min(t0 + u * kWaves, tokens - 1);
                    const int64_t from = factors[t] < 0.0f ? 0 : sources[t];  // (what stays: any place of the pool)
#pragma unroll
                    for (int h = 0; h < kPer; ++h) w[u][h] = pages[from + ((64 * h + lane) << a.page_shift)];
                }
#pragma unroll
                for (int u = 0; u < kAtOnce; ++u) {
                    const int t = t0 + u * kWaves;
                    if (t >= tokens) break;
                    const float r = factors[j0 + t];
#pragma unroll
                    for (int h = 0; h < kPer; ++h) rows[t * D + 64 * h + lane] = static_cast<uint8_t>(r != 1.0f ? scaled_codes(w[u][h], r) : w[u][h]);
                }
            }
        }
        __syncthreads();
        if (j0 == 0 && held_factor != 1.0f) {                                 // what the first page keeps, on the larger scale
            uint8_t* const codes = pages + (targets[0] - (kind ? held : held * D));           // (the path's first token goes behind what it keeps)
            const int across = (held + 15) / 16, pieces = kind ? D * across : held * (D / 16);
            for (int i = tid; i < pieces; i += kThreads) {
                uint4* piece = reinterpret_cast<uint4*>(kind ? codes + (static_cast<size_t>(i / across) << a.page_shift) + 16 * (i % across) : codes + 16 * i);
                const int keep = kind ? held - 16 * (i % across) : 16;
                const float r = held_factor;
                const uint4 w = *piece;
                const uint32_t m[4] = {first_bytes(keep), first_bytes(keep - 4), first_bytes(keep - 8), first_bytes(keep - 12)};
                *piece = make_uint4((scaled_codes(w.x, r) & m[0]) | (w.x & ~m[0]), (scaled_codes(w.y, r) & m[1]) | (w.y & ~m[1]), (scaled_codes(w.z, r) & m[2]) | (w.z & ~m[2]),
                                    (scaled_codes(w.w, r) & m[3]) | (w.w & ~m[3]));
            }
            __syncthreads();                                                  // (older and new values share 16 bytes)
        }
        if (!kind) {
            for (int i = tid; i < tokens * (D / 16); i += kThreads) {
                const int t = i / (D / 16);
                if (!(factors[j0 + t] < 0.0f)) *reinterpret_cast<uint4*>(pages + targets[j0 + t] + 16 * (i % (D / 16))) = *reinterpret_cast<const uint4*>(rows + 16 * i);
            }
        } else {
            // 16 values of a dimension at a time, what else is among them as it was (32 sequences of ten tokens, eight layers, pages of 16: code by code, page after page 18.6 us,
            // so 15.3)
            const int chunk0 = max(first + j0, 0) >> 4, chunks = ((first + j0 + tokens - 1) >> 4) - chunk0 + 1;
            for (int i = wave; i < chunks * (D / 64); i += kWaves) {
                const int at = 16 * (chunk0 + i / (D / 64)), d = 64 * (i % (D / 64)) + lane;
                const int from = max(at - first, j0), to = min(at + 16 - first, j0 + tokens);           // tokens that go there
                bool any = false;
                for (int t = from; t < to; ++t) any |= !(factors[t] < 0.0f);
                if (!any || targets[from] < 0) continue;
                uint4* const piece = reinterpret_cast<uint4*>(pages + (targets[from] - ((first + from) & 15)) + (static_cast<int64_t>(d) << a.page_shift));
                const uint4 old = *piece;
                uint64_t low = static_cast<uint64_t>(old.y) << 32 | old.x, high = static_cast<uint64_t>(old.w) << 32 | old.z;
                for (int t = from; t < to; ++t) {
                    if (factors[t] < 0.0f) continue;
                    const int b = (first + t) & 15, shift = 8 * (b & 7);
                    const uint64_t code = static_cast<uint64_t>(rows[(t - j0) * D + d]) << shift, keep = ~(uint64_t{0xff} << shift);
                    low = b < 8 ? (low & keep) | code : low;
                    high = b < 8 ? high : (high & keep) | code;
                }
                *piece = make_uint4(static_cast<uint32_t>(low), static_cast<uint32_t>(low >> 32), static_cast<uint32_t>(high), static_cast<uint32_t>(high >> 32));
            }
        }
        __syncthreads();
    }
}

// ---- the sequences of the next step -----------------------------------------------------------------------------------
//
// Row r of the new table goes on with the first kept[r] tokens of row sources[r] and has room for reserve[r].  Whole pages are shared.  A page that is kept in part, which
// the row goes on to fill, stays the row's if no other new row and no holder outside the table has it (of several rows that keep it in part the first); the others get a
// copy.  Then come free pages: those without a holder, lowest numbers first, to the rows in their order.  Holders are counted, free pages dealt out (by one workgroup, so
// that the order is fixed), then tables and copies made.  Integer atomics only: their order changes nothing.  What a row is to write to and has no page for is missing: what the
// pool has no more of, and a page kept in part that its source has not.  A row's room ends with the table.
// Bound: the chain of dependent loads (row, table, count) and the second launch, not the bytes: 64 sequences of up to 4000 tokens in pages of 64, four layers, 15 us, of them 8.9 and
// 6.1 in the two launches; 16 beams of 4 prompts 12.

struct ForkArgs {
    const int32_t* table; size_t table_stride;
    const int32_t* uses; const int32_t* sources; const int32_t* kept; const int32_t* reserve;
    int32_t* new_table; int32_t* new_uses; int32_t* missing;
    int32_t* first;                             // [pool] lowest new row that keeps the page in part
    int32_t* start;                             // [rows] number of the row's first free page
    int32_t* copies;                            // [rows] page to copy, -1: none
    int32_t* fresh;                             // [pool] free pages in their order
    int32_t* given;                             // [1] how many of them there are
    int seqs, rows, width, pool, page_shift, kv_heads, dim;
};
struct ForkRow { int source, kept, full, last; bool some; };                  // full pages, pages in all; one kept in part
__device__ __forceinline__ ForkRow fork_row(const ForkArgs& a, int r) {
    ForkRow f;
    const int most = a.width << a.page_shift, source = a.sources[r];
    f.source = source >= 0 && source < a.seqs ? source : -1;
    f.kept = f.source >= 0 ? clamp_int(a.kept[r], 0, most) : 0;
    f.full = f.kept >> a.page_shift;
    f.some = (f.kept & ((1 << a.page_shift) - 1)) != 0;
    f.last = static_cast<int>((static_cast<int64_t>(clamp_int(a.reserve[r], f.kept, most)) + (1 << a.page_shift) - 1) >> a.page_shift);
    return f;
}
__device__ __forceinline__ int fork_entry(const ForkArgs& a, int row, int at) {
    const int page = a.table[static_cast<size_t>(row) * a.table_stride + at];
    return page >= 0 && page < a.pool ? page : -1;
}
// (counts that other workgroups' atomics made, read past this compute unit's cache)
__device__ __forceinline__ int fork_load(const int32_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

__global__ __launch_bounds__(256) void paged_fork_begin_kernel(const ForkArgs a) {
    const int p = blockIdx.x * 256 + threadIdx.x;
    if (p >= a.pool) return;
    a.new_uses[p] = a.uses[p];
    a.first[p] = 0x7fffffff;
}

__global__ __launch_bounds__(256) void paged_fork_count_kernel(const ForkArgs a) {
    const int at = blockIdx.x * 256 + threadIdx.x, row = blockIdx.y;
    if (at >= a.width) return;
    if (row < a.seqs) {
        const int page = fork_entry(a, row, at);
        if (page >= 0) atomicSub(a.new_uses + page, 1);
        return;
    }
    const int r = row - a.seqs;
    const ForkRow f = fork_row(a, r);
    if (f.source < 0 || at > f.full || (at == f.full && !f.some)) return;
    const int page = fork_entry(a, f.source, at);
    if (page < 0) return;
    if (at < f.full) atomicAdd(a.new_uses + page, 1);
    else atomicMin(a.first + page, r);
}

// the sum over the workgroup's threads up to this one, and of all
__device__ __forceinline__ int threads_until(int v, int* parts, int& total) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 1; i < 64; i *= 2) {
        const int before = __shfl_up(v, i);
        if (lane >= i) v += before;
    }
    __syncthreads();
    if (lane == 63) parts[threadIdx.x >> 6] = v;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        if (w < static_cast<int>(threadIdx.x >> 6)) before += parts[w];
        total += parts[w];
    }
    return before + v;
}

__global__ __launch_bounds__(1024) void paged_fork_deal_kernel(const ForkArgs a) {
    __shared__ int parts[16];
    const int tid = threadIdx.x;
    int wanted = 0;
    for (int r0 = 0; r0 < a.rows; r0 += 1024) {
        const int r = r0 + tid;
        int wants = 0;
        if (r < a.rows) {
            const ForkRow f = fork_row(a, r);
            int copied = -1;
            wants = f.last - f.full - (f.some ? 1 : 0);
            if (f.some) {
                const int page = fork_entry(a, f.source, f.full);
                if (page >= 0) {
                    if (fork_load(a.first + page) == r && fork_load(a.new_uses + page) <= 0) __hip_atomic_store(a.first + page, -1 - r, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);          // stays: marked, counted below
                    else { copied = page; ++wants; }
                }
            }
            a.copies[r] = copied;
        }
        int all;
        const int until = threads_until(wants, parts, all);
        if (r < a.rows) a.start[r] = wanted + until - wants;
        wanted += all;
    }
    __threadfence();
    __syncthreads();
    int given = 0;
    constexpr int kPer = 4;
    for (int p0 = 0; p0 < a.pool; p0 += 1024 * kPer) {
        int uses[kPer], free = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int p = p0 + kPer * tid + i;
            uses[i] = 1;
            if (p < a.pool) {
                uses[i] = max(fork_load(a.new_uses + p), 0) + (fork_load(a.first + p) < 0);
                free += uses[i] == 0;
            }
        }
        int all;
        int rank = given + threads_until(free, parts, all) - free;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int p = p0 + kPer * tid + i;
            if (p >= a.pool) break;
            if (uses[i] == 0 && rank++ < wanted) {
                a.fresh[rank - 1] = p;
                uses[i] = 1;
            }
            a.new_uses[p] = uses[i];
        }
        given += all;
    }
    if (tid == 0) *a.given = min(given, wanted);
}

// The three launches above in one, for pools whose counts fit LDS, two words a page, and tables of up to 2^17 entries, old and new, which one workgroup reads about as fast as a
// launch takes (64 sequences of 63 pages 19.7 -> 15.1 us, 16 beams 18 -> 12).  Requests for four entries a thread are on their way at a time.
constexpr int kPoolInLds = 16384;
__global__ __launch_bounds__(1024) void paged_fork_small_kernel(const ForkArgs a) {
    extern __shared__ int32_t counts[];                                       // [pool] holders, [pool] lowest new row that keeps the page in part
    __shared__ int parts[16];
    constexpr int kAtOnce = 4;
    int32_t* const uses = counts;
    int32_t* const first = counts + a.pool;
    const int tid = threadIdx.x;
    for (int p0 = tid; p0 < a.pool; p0 += kAtOnce * 1024) {
        int v[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) v[i] = a.uses[min(p0 + 1024 * i, a.pool - 1)];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
            if (p0 + 1024 * i < a.pool) {
                uses[p0 + 1024 * i] = v[i];
                first[p0 + 1024 * i] = 0x7fffffff;
            }
    }
    __syncthreads();
    const int held = a.seqs * a.width, entries = (a.seqs + a.rows) * a.width; // (fit: the host's check)
    for (int at0 = tid; at0 < entries; at0 += kAtOnce * 1024) {
        int page[kAtOnce], what[kAtOnce], row[kAtOnce];                       // what: -1 a holder less, 1 a holder more, 0 kept in part, 2 nothing
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int index = at0 + 1024 * i;
            what[i] = 2;
            page[i] = -1;
            row[i] = 0;
            if (index < held) {
                what[i] = -1;
                page[i] = fork_entry(a, index / a.width, index % a.width);
            } else if (index < entries) {
                const int r = (index - held) / a.width, at = (index - held) % a.width;
                const ForkRow f = fork_row(a, r);
                if (f.source >= 0 && (at < f.full || (at == f.full && f.some))) {
                    what[i] = at < f.full ? 1 : 0;
                    page[i] = fork_entry(a, f.source, at);
                    row[i] = r;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            if (page[i] < 0) continue;
            if (what[i] == 0) atomicMin(first + page[i], row[i]);
            else if (what[i] != 2) atomicAdd(uses + page[i], what[i]);
        }
    }
    __syncthreads();
    int wanted = 0;
    for (int r0 = 0; r0 < a.rows; r0 += 1024) {
        const int r = r0 + tid;
        int wants = 0, copied = -1, stays = -1;
        if (r < a.rows) {
            const ForkRow f = fork_row(a, r);
            wants = f.last - f.full - (f.some ? 1 : 0);
            const int page = f.some ? fork_entry(a, f.source, f.full) : -1;
            if (page >= 0) {
                if (first[page] == r && uses[page] <= 0) stays = page;
                else { copied = page; ++wants; }
            }
            a.copies[r] = copied;
        }
        if (stays >= 0) first[stays] = -1;                                    // (rows of this page read either: neither is their own number)
        int all;
        const int until = threads_until(wants, parts, all);
        if (r < a.rows) a.start[r] = wanted + until - wants;
        wanted += all;
    }
    __syncthreads();
    int given = 0;
    constexpr int kPer = 4;
    for (int p0 = 0; p0 < a.pool; p0 += 1024 * kPer) {
        int holders[kPer], free = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int p = p0 + kPer * tid + i;
            holders[i] = p < a.pool ? max(uses[p], 0) + (first[p] < 0) : 1;
            free += holders[i] == 0;
        }
        int all;
        int rank = given + threads_until(free, parts, all) - free;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int p = p0 + kPer * tid + i;
            if (p >= a.pool) break;
            if (holders[i] == 0 && rank++ < wanted) {
                a.fresh[rank - 1] = p;
                holders[i] = 1;
            }
            a.new_uses[p] = holders[i];
        }
        given += all;
    }
    if (tid == 0) *a.given = min(given, wanted);
}

// Blocks of 256 entries of a row's table first, then a row's copies: blocks of 16 KB of keys or values of a layer.
__global__ __launch_bounds__(256) void paged_fork_rows_kernel(const Layers layers, const ForkArgs a, int table_blocks, int copy_blocks) {
    const int r = blockIdx.x, block = blockIdx.y, tid = threadIdx.x;
    const int start = a.start[r], given = *a.given, copied = a.copies[r];
    if (block < table_blocks) {
        const ForkRow f = fork_row(a, r);
        const int at = 256 * block + tid, fresh_from = f.full + (f.some && copied < 0 ? 1 : 0);
        if (block == 0 && tid == 0) {
            const int wants = max(f.last - fresh_from, 0);
            const bool nowhere = f.some && copied < 0 && fork_entry(a, f.source, f.full) < 0;                // (kept in part, and the source has no page there)
            a.missing[r] = wants - clamp_int(given - start, 0, wants) + nowhere;
        }
        if (at >= a.width) return;
        int page = -1;
        if (at < fresh_from) page = fork_entry(a, f.source, at);
        else if (at < f.last) {
            const int rank = start + at - fresh_from;
            page = rank < given ? a.fresh[rank] : -1;
        }
        a.new_table[static_cast<size_t>(r) * a.width + at] = page;
        return;
    }
    if (copied < 0 || start >= given) return;
    const int to = a.fresh[start], part = block - table_blocks;               // (the copy is the row's first free page)
    const int of_kind = part % copy_blocks, kind = part / copy_blocks & 1;
    const Layer& layer = layers.layer[part / copy_blocks / 2];
    const size_t bytes = static_cast<size_t>(a.kv_heads) * a.dim << a.page_shift;
    uint8_t* const pages = kind ? layer.value_pages : layer.key_pages;
    const uint4* src = reinterpret_cast<const uint4*>(pages + copied * bytes);
    uint4* dst = reinterpret_cast<uint4*>(pages + to * bytes);
    const int pieces = static_cast<int>(bytes / 16), from = 1024 * of_kind + tid;
    const uint4 w0 = src[min(from, pieces - 1)], w1 = src[min(from + 256, pieces - 1)], w2 = src[min(from + 512, pieces - 1)], w3 = src[min(from + 768, pieces - 1)];
    if (from < pieces) dst[from] = w0;
    if (from + 256 < pieces) dst[from + 256] = w1;
    if (from + 512 < pieces) dst[from + 512] = w2;
    if (from + 768 < pieces) dst[from + 768] = w3;
    if (of_kind == 0) {
        float* const scales = kind ? layer.value_scales : layer.key_scales;
        for (int h = tid; h < a.kv_heads; h += 256) scales[static_cast<size_t>(to) * a.kv_heads + h] = scales[static_cast<size_t>(copied) * a.kv_heads + h];
    }
}

bool page_ok(int64_t page_tokens, int64_t head_dim) {
    return (head_dim == 64 || head_dim == 128) && (page_tokens == 16 || page_tokens == 32 || page_tokens == 64 || page_tokens == 128);
}
int shift_of(int64_t page_tokens) { return page_tokens == 16 ? 4 : page_tokens == 32 ? 5 : page_tokens == 64 ? 6 : 7; }
// The addresses of a call's layers, [layers][4] on the host: aligned, and no two layers share any memory (one workgroup would write what another reads).
constexpr int kMostLayers = 1024;
bool layers_ok(void* const* caches, int64_t layers, size_t page_bytes, size_t scale_bytes) {
    uintptr_t some[2 * kMostLayers];
    for (int kind = 0; kind < 2; ++kind) {
        const size_t bytes = kind ? scale_bytes : page_bytes;
        for (int64_t i = 0; i < 2 * layers; ++i) {
            some[i] = reinterpret_cast<uintptr_t>(caches[4 * (i / 2) + 2 * kind + i % 2]);
            if (!some[i] || some[i] % (kind ? 4 : 16)) return false;
        }
        std::sort(some, some + 2 * layers);
        for (int64_t i = 1; i < 2 * layers; ++i)
            if (some[i] - some[i - 1] < bytes) return false;
    }
    return true;
}
Layers some_layers(void* const* caches, int64_t from, int64_t count) {
    Layers l{};
    for (int64_t i = 0; i < count; ++i) {
        void* const* c = caches + 4 * (from + i);
        l.layer[i] = Layer{static_cast<uint8_t*>(c[0]), static_cast<uint8_t*>(c[1]), static_cast<float*>(c[2]), static_cast<float*>(c[3])};
    }
    return l;
}
struct ForkLayout { size_t first, start, copies, fresh, given, bytes; };
ForkLayout fork_layout(int64_t rows, int64_t pool) {
    ForkLayout l{};
    size_t at = 0;
    auto take = [&](int64_t ints) { const size_t here = at; at += align256(ints * 4); return here; };
    l.first = take(pool);
    l.start = take(rows);
    l.copies = take(rows);
    l.fresh = take(pool);
    l.given = take(1);
    l.bytes = at;
    return l;
}

}  // namespace
}  // namespace pllm

extern "C" {

int pllm_paged_cache_compact(void* const* caches, int64_t layers, int64_t pool, int64_t page_tokens, const int32_t* block_table, int64_t table_stride, int64_t table_width,
                             const int32_t* lengths, const int32_t* kept, int64_t most, const int32_t* counts, const int32_t* cu_steps, int64_t steps, int64_t seqs, int64_t kv_heads,
                             int64_t head_dim, void* stream) {
    using namespace pllm;
    if (!caches || !block_table || !lengths || !kept || !counts || layers <= 0 || pool <= 0 || table_width <= 0 || table_stride < table_width || most <= 0 || seqs <= 0 || kv_heads <= 0 ||
        (!cu_steps && steps <= 0))
        return PLLM_ERR_INVALID_ARGUMENT;
    if (!page_ok(page_tokens, head_dim)) return PLLM_ERR_UNSUPPORTED;
    if (pool > 0x7fffffff || table_width > 0x3fffffff / page_tokens || seqs > 0xffff || kv_heads > 1024 || most > kTreeNodes || layers > kMostLayers || (!cu_steps && steps > kTreeNodes)) return PLLM_ERR_UNSUPPORTED;
    const uintptr_t words = reinterpret_cast<uintptr_t>(block_table) | reinterpret_cast<uintptr_t>(lengths) | reinterpret_cast<uintptr_t>(kept) | reinterpret_cast<uintptr_t>(counts) |
                            reinterpret_cast<uintptr_t>(cu_steps);
    if ((words & 3u) || !layers_ok(caches, layers, static_cast<size_t>(pool * kv_heads * page_tokens * head_dim), static_cast<size_t>(pool * kv_heads * 4))) return PLLM_ERR_INVALID_ARGUMENT;
    CompactArgs a{block_table, static_cast<size_t>(table_stride), lengths, kept, counts, cu_steps, static_cast<int>(steps), static_cast<int>(most), static_cast<int>(kv_heads),
                  static_cast<int>(pool), static_cast<int>(table_width), shift_of(page_tokens)};
    for (int64_t from = 0; from < layers; from += kLayers) {
        const int64_t count = std::min<int64_t>(layers - from, kLayers);
        const dim3 grid(static_cast<unsigned>(2 * kv_heads), static_cast<unsigned>(seqs), static_cast<unsigned>(count));
        // (LDS for as much of a path as there can be, so that many workgroups fit a compute unit)
        const size_t lds = static_cast<size_t>(32 * most + std::min<int64_t>(most, kCompactStretch) * head_dim);
        if (head_dim == 128) hipLaunchKernelGGL((paged_compact_kernel<128>), grid, dim3(kCompactThreads), lds, static_cast<hipStream_t>(stream), some_layers(caches, from, count), a);
        else hipLaunchKernelGGL((paged_compact_kernel<64>), grid, dim3(kCompactThreads), lds, static_cast<hipStream_t>(stream), some_layers(caches, from, count), a);
    }
    return hipGetLastError() == hipSuccess ? PLLM_OK : PLLM_ERR_LAUNCH;
}

size_t pllm_paged_cache_fork_workspace_bytes(int64_t rows, int64_t pool) {
    return rows > 0 && pool > 0 && rows <= 0xffff && pool <= 0x7fffff ? pllm::fork_layout(rows, pool).bytes : 0;
}

int pllm_paged_cache_fork(void* const* caches, int64_t layers, int64_t pool, int64_t page_tokens, const int32_t* block_table, int64_t table_stride, int64_t table_width, const int32_t* uses,
                          const int32_t* sources, const int32_t* kept, const int32_t* reserve, int64_t seqs, int64_t rows, int64_t kv_heads, int64_t head_dim, int32_t* new_table,
                          int32_t* new_uses, int32_t* missing, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace pllm;
    if (!caches || !block_table || !uses || !sources || !kept || !reserve || !new_table || !new_uses || !missing || layers <= 0 || pool <= 0 || table_width <= 0 ||
        table_stride < table_width || seqs <= 0 || rows <= 0 || kv_heads <= 0)
        return PLLM_ERR_INVALID_ARGUMENT;
    if (!page_ok(page_tokens, head_dim)) return PLLM_ERR_UNSUPPORTED;
    // grid rows, a pool that one workgroup goes through, positions and the pages of all rows together in 32 bits
    const int64_t copy_blocks = (kv_heads * page_tokens * head_dim / 16 + 1023) / 1024, table_blocks = (table_width + 255) / 256;
    if (pool > 0x7fffff || layers > kMostLayers || table_width > 0x3fffffff / page_tokens || seqs + rows > 0xffff || rows * table_width > 0x7fffffff || kv_heads > 1024 || table_blocks + 2 * kLayers * copy_blocks > 0xffff) return PLLM_ERR_UNSUPPORTED;
    const uintptr_t words = reinterpret_cast<uintptr_t>(block_table) | reinterpret_cast<uintptr_t>(uses) | reinterpret_cast<uintptr_t>(sources) | reinterpret_cast<uintptr_t>(kept) |
                            reinterpret_cast<uintptr_t>(reserve) | reinterpret_cast<uintptr_t>(new_table) | reinterpret_cast<uintptr_t>(new_uses) | reinterpret_cast<uintptr_t>(missing) |
                            reinterpret_cast<uintptr_t>(workspace);
    if ((words & 3u) || !layers_ok(caches, layers, static_cast<size_t>(pool * kv_heads * page_tokens * head_dim), static_cast<size_t>(pool * kv_heads * 4))) return PLLM_ERR_INVALID_ARGUMENT;
    const ForkLayout l = fork_layout(rows, pool);
    if (!workspace || workspace_bytes < l.bytes) return PLLM_ERR_WORKSPACE;
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    auto ints = [&](size_t at) { return reinterpret_cast<int32_t*>(ws + at); };
    ForkArgs a{block_table, static_cast<size_t>(table_stride), uses, sources, kept, reserve, new_table, new_uses, missing, ints(l.first), ints(l.start), ints(l.copies), ints(l.fresh),
               ints(l.given), static_cast<int>(seqs), static_cast<int>(rows), static_cast<int>(table_width), static_cast<int>(pool), shift_of(page_tokens), static_cast<int>(kv_heads),
               static_cast<int>(head_dim)};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    static SmemGrant granted;
    const size_t lds = 2 * sizeof(int32_t) * static_cast<size_t>(pool);
    if (pool <= kPoolInLds && (seqs + rows) * table_width <= (1 << 17)) {
        if (!grant_dynamic_smem(reinterpret_cast<const void*>(paged_fork_small_kernel), lds, granted)) return PLLM_ERR_LAUNCH;
        hipLaunchKernelGGL(paged_fork_small_kernel, dim3(1), dim3(1024), lds, st, a);
    } else {
        hipLaunchKernelGGL(paged_fork_begin_kernel, dim3(static_cast<unsigned>((pool + 255) / 256)), dim3(256), 0, st, a);
        hipLaunchKernelGGL(paged_fork_count_kernel, dim3(static_cast<unsigned>(table_blocks), static_cast<unsigned>(seqs + rows)), dim3(256), 0, st, a);
        hipLaunchKernelGGL(paged_fork_deal_kernel, dim3(1), dim3(1024), 0, st, a);
    }
    for (int64_t from = 0; from < layers; from += kLayers) {
        const int64_t count = std::min<int64_t>(layers - from, kLayers), tables = from == 0 ? table_blocks : 0;
        hipLaunchKernelGGL(paged_fork_rows_kernel, dim3(static_cast<unsigned>(rows), static_cast<unsigned>(tables + 2 * count * copy_blocks)), dim3(256), 0, st,
                           some_layers(caches, from, count), a, static_cast<int>(tables), static_cast<int>(copy_blocks));
    }
    return hipGetLastError() == hipSuccess ? PLLM_OK : PLLM_ERR_LAUNCH;
}

}  // extern "C"
