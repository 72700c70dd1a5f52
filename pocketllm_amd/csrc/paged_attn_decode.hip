// Attention of one or a few new tokens per sequence over a paged E4M3 cache, the sequences of a batch at any lengths:
//     out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - m),  k_j, v_j = code * scale of the page and head, j up to the query's position.
// Two launches: runs of keys with a running maximum each, then the runs of a row together (one launch where no sequence can have two runs).
//
// A workgroup has a run of one sequence's keys for one key/value head and 16 or 32 query rows (the heads that share it, times the new tokens).  Its
// four waves take 64 keys at a time each, with statistics of their own, and meet in LDS once, at the end.  A wave forms S^T = K Q^T
// (v_mfma_f32_16x16x32: matrix rows are keys, columns queries), whose accumulator layout, rounded to 16 bits, is what O^T = V^T P^T wants as its
// second operand if row 4 g + i of score tile t is key 16 g + 4 t + i: then a lane of group g has the 16 neighbouring keys 16 g .. + 15, and its
// values are 16 neighbouring bytes of a value page.  16 neighbouring keys share a page, so a lane needs one page number for its keys' rows, one for
// its values and two scales, whatever the page size.  Codes become 16-bit values in registers: E4M3 is exact in both types; the keys' scale goes on the
// scores, the values' scale (halved, so that fp16 holds every value that rounds up from its largest) into the conversion, both exact.
// The next 64 keys' codes are requested as soon as the registers of the last ones are free, the keys' before the softmax and the values' behind their
// product, and page numbers a step ahead of them (with all of it requested at the end of a step 64 sequences took 139 us for 122, one of 100001 positions 49 for 44).
// Bound: bytes, 2 * length * D codes per head, once for each 16 or 32 rows.  64 sequences of 1 to 8192 positions, 567 MB: 118 us, 4.8 TB/s, where a kernel
// that only reads reaches 6: runs of 512 keys, which one sequence needs to fill the machine, begin and end too often (of 1024: 3 % less,
// but 2048 positions of one sequence 13.2 for 10.4).
//
// TREE, for drafted trees of up to 64 nodes and few rows or keys: a node's ancestors are a mask of 64 bits, walked up in LDS once a workgroup beside the first requests; steps that
// hold a node's key are masked by it (one tree of 26 nodes of 48 and 8 heads behind 4000 positions 18.6 us, 8 of 32 heads of 64 behind 700 6.2).
#include "paged_attention.h"
#include "paged_device.h"

#include <algorithm>
#include <cfloat>
#include <type_traits>

namespace pllm {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kStep = 64;                       // keys that a wave takes at a time

// Softmax weights are 2^(score - m) and are rounded to 16 bits for the second product (matrix instructions on float32 have a sixteenth of the rate); their sum takes
// them unrounded: roundings to the nearest lean to no side.  In fp16 a weight below 2^-14 is rounded to a multiple of 2^-24, one below 2^-25 to nothing, so the
// largest of a wave's is 2^15 there: what is lost of a weight is 2^-40 of it at most (with 1, 1024 keys whose scores are 16.5 below another, to base e, lost an
// eighth of what they add up to).  The factor is in numerator and denominator alike; scores from 2^20 on, whose steps could make more of 15, are compared with
// themselves.  bf16 has float32's range.
template <bool BF16> __device__ __forceinline__ float weights_from(float top) {
    if constexpr (BF16) return top;
    else return fabsf(top) < 0x1p20f ? top - 15.0f : top;
}

// SETS of 16 query rows; rows of one key/value head: token * group + head in the group
// TREE: the new tokens are nodes of a tree; the steps that hold some of their keys are masked by the nodes' ancestors
template <bool BF16, int D, int SETS, bool TREE>
__global__ __launch_bounds__(kThreads, SETS == 1 ? 3 : 2) void paged_decode_kernel(const PagedDecodeArgs a, int least_rows, int most_rows) {
    constexpr int kPieces = D / 64;             // 16-byte pieces of a key row per lane
    constexpr int kTiles = D / 16;              // output tiles
    constexpr int kPitch = D + 4;
    constexpr int kRows = 16 * SETS, kStride = kStep * kWaves;
    __shared__ __align__(16) float sums[kWaves][16 * kPitch];
    __shared__ float2 stats[kWaves][16];
    __shared__ __align__(16) uint16_t queries[kRows][D + 8];                  // (in registers they cost the third workgroup of a compute unit)
    __shared__ __align__(8) uint16_t nan_keys[kWaves][D][4];                  // keys of a wave's step whose value is NaN, a bit each, per dimension
    __shared__ int parents[TREE ? 64 : 1];
    __shared__ uint64_t nodes[TREE ? 64 : 1];                                 // what the nodes see of the tree
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;
    // Neighbouring workgroups run on different XCDs: heads first, and the runs of every sequence from another one on, or the XCDs of the first runs, which
    // every sequence has, would do the most (64 sequences of 1 to 8192 positions, run numbers first / heads first 198 / 147 us).
    const int kvh = blockIdx.x % a.kv_heads, tile = blockIdx.x / a.kv_heads, s = blockIdx.z, run = (blockIdx.y + blockIdx.z) % a.runs_bound;
    const int group = a.heads / a.kv_heads;
    const int offset = a.cu_steps ? paged_offset(a.cu_steps, s, 0, a.tokens) : s * a.steps;
    const int n = a.cu_steps ? paged_offset(a.cu_steps, s + 1, 0, a.tokens) - offset : a.steps;
    const int64_t all_rows = static_cast<int64_t>(n) * group;
    if (all_rows < least_rows || all_rows > most_rows || kRows * tile >= all_rows) return;
    const int rows = static_cast<int>(all_rows);
    const int given = a.lengths[s], length = paged_length(given, a.width, a.page_shift);
    const int run_keys = paged_run_keys(length, a.kv_heads), begin = run * run_keys, end = min(begin + run_keys, length);
    if (run > 0 && begin >= length) return;
    const int32_t* table = a.table + static_cast<size_t>(s) * a.table_stride;

    const int past = tree_past(given, n);                                     // (TREE)
    if constexpr (TREE) {
        if (n > 64) return;
        if (tid < n) parents[tid] = a.parents[offset + tid];
    }
    // the columns' query rows and how many keys they see
    int limit[SETS];
#pragma unroll
    for (int c = 0; c < SETS; ++c) {
        const int r = kRows * tile + 16 * c + col;
        const int64_t sees = static_cast<int64_t>(given) - n + r / group + 1;
        limit[c] = r < rows ? static_cast<int>(sees < 0 ? 0 : (sees > length ? length : sees)) : 0x7fffffff;
    }
    const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
    v4f o[SETS][kTiles];
    float m[SETS], l[SETS], late = 1.0f;        // of the column, m as weights_from has it; l over the lane's own keys
#pragma unroll
    for (int c = 0; c < SETS; ++c) {
#pragma unroll
        for (int i = 0; i < kTiles; ++i) o[c][i] = zero;
        m[c] = -FLT_MAX;
        l[c] = 0.0f;
    }
    const size_t head_bytes = static_cast<size_t>(D) << a.page_shift, page_mask = (size_t{1} << a.page_shift) - 1;
    // page numbers of the lane's key rows (chunk col / 4 of the step) and of its values and scales (chunk g), as the table has them: checked where they are
    // used, a step later, so that nothing waits for them here
    auto pages = [&](int j0, int& key_page, int& value_page) {
        key_page = table[min(j0 + 16 * (col >> 2), length - 1) >> a.page_shift];
        value_page = table[min(j0 + 16 * g, length - 1) >> a.page_shift];
    };
    auto checked = [&](int page) { return page >= 0 && page < a.pool ? page : -1; };
    struct Step { uint4 keys[4][kPieces], values[kTiles]; float key_scale, value_scale; bool here; };
    auto request_keys = [&](Step& x, int j0, int key_page, int value_page) {
        key_page = checked(key_page);
        value_page = j0 + 16 * g < length ? checked(value_page) : -1;
        const size_t key_at = (static_cast<size_t>(max(key_page, 0)) * a.kv_heads + kvh) * head_bytes + ((j0 + 16 * (col >> 2)) & page_mask) * D;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < kPieces; ++i) x.keys[t][i] = *reinterpret_cast<const uint4*>(a.key_pages + key_at + (4 * t + (col & 3)) * D + 64 * i + 16 * g);
        const size_t scale_at = static_cast<size_t>(max(value_page, 0)) * a.kv_heads + kvh;
        x.key_scale = a.key_scales[scale_at];
        x.value_scale = a.value_scales[scale_at];
        x.here = value_page >= 0;
    };
    auto request_values = [&](Step& x, int j0, int value_page) {
        const size_t value_at = (static_cast<size_t>(max(checked(value_page), 0)) * a.kv_heads + kvh) * head_bytes + ((j0 + 16 * g) & page_mask) + (static_cast<uint32_t>(col) << a.page_shift);
#pragma unroll
        for (int i = 0; i < kTiles; ++i) x.values[i] = *reinterpret_cast<const uint4*>(a.value_pages + value_at + (static_cast<size_t>(16 * i) << a.page_shift));
    };
    // (TREE) keys `first` .. + 63 that a column's node sees
    auto window = [&](int c, int first) { return tree_window(&nodes[min((kRows * tile + 16 * c + col) / group, 63)], 1, past, first, limit[c]); };
    int key_page = 0, value_page = 0;           // of the next step to request
    // a step; with MORE the next one's keys are requested as soon as this one's are used, its values likewise
    auto work = [&](auto more, Step& x, int j0) {
        constexpr bool MORE = decltype(more)::value;
        auto& kf = x.keys;
        auto& vf = x.values;
        const float key_factor = x.key_scale * a.scale, value_scale = x.here ? 0.5f * x.value_scale : 1.0f;
        v4f sc[SETS][4];
#pragma unroll
        for (int c = 0; c < SETS; ++c)
#pragma unroll
            for (int t = 0; t < 4; ++t) sc[c][t] = zero;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            uint4 qf[SETS][2];
#pragma unroll
            for (int c = 0; c < SETS; ++c)
#pragma unroll
                for (int u = 0; u < 2; ++u) qf[c][u] = *reinterpret_cast<const uint4*>(&queries[16 * c + col][64 * i + 16 * g + 8 * u]);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const uint4 lo = half_from_codes<BF16>(kf[t][i].x, kf[t][i].y, 1.0f), hi = half_from_codes<BF16>(kf[t][i].z, kf[t][i].w, 1.0f);
#pragma unroll
                for (int c = 0; c < SETS; ++c) sc[c][t] = half_mfma16<BF16>(hi, qf[c][1], half_mfma16<BF16>(lo, qf[c][0], sc[c][t]));
            }
        }
        const float factor = fminf(key_factor * late, FLT_MAX);               // (beyond float32 a score of zero would be NaN)
#pragma unroll
        for (int c = 0; c < SETS; ++c)
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[c][t][i] *= factor;
        const int first = j0 + 16 * g;
        bool whole = true, some_nan = false;                                  // every column sees all of the lane's keys
#pragma unroll
        for (int c = 0; c < SETS; ++c) whole &= x.here && (TREE ? min(past, limit[c]) : limit[c]) - first >= 16;
        if (!__all(whole)) {
#pragma unroll
            for (int c = 0; c < SETS; ++c) {
                const int seen = x.here ? limit[c] - first : 0;
                const uint32_t bits = TREE && x.here ? static_cast<uint32_t>(window(c, first)) : 0;
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc[c][t][i] = (TREE ? (bits >> (4 * t + i) & 1) != 0 : 4 * t + i < seen) ? sc[c][t][i] : -INFINITY;
            }
            // what lies behind the last key may be anything, NaN codes too, and zero times NaN is NaN
            const int stored = x.here ? length - first : 0;
            const uint32_t keep[4] = {first_bytes(stored), first_bytes(stored - 4), first_bytes(stored - 8), first_bytes(stored - 12)};
            bool nan = false;
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
                vf[i].x &= keep[0]; vf[i].y &= keep[1]; vf[i].z &= keep[2]; vf[i].w &= keep[3];
                nan |= any_nan_code(vf[i].x) | any_nan_code(vf[i].y) | any_nan_code(vf[i].z) | any_nan_code(vf[i].w);
            }
            some_nan = __any(nan);
            if (some_nan)                                                     // of keys that not every row sees: none into the product
#pragma unroll
                for (int i = 0; i < kTiles; ++i) {
                    nan_keys[wave][16 * i + col][g] =
                        static_cast<uint16_t>(nan_codes(vf[i].x) | (nan_codes(vf[i].y) << 4) | (nan_codes(vf[i].z) << 8) | (nan_codes(vf[i].w) << 12));
                    vf[i].x = without_nan(vf[i].x); vf[i].y = without_nan(vf[i].y); vf[i].z = without_nan(vf[i].z); vf[i].w = without_nan(vf[i].w);
                }
        }
        const int next_page = value_page;
        if constexpr (MORE) {
            request_keys(x, j0 + kStride, key_page, value_page);
            pages(j0 + 2 * kStride, key_page, value_page);                    // (before the values: loads arrive in order)
        }
        uint4 p[SETS][2];
#pragma unroll
        for (int c = 0; c < SETS; ++c) {
            float top = fmaxf(fmaxf(sc[c][0][0], sc[c][0][1]), fmaxf(sc[c][0][2], sc[c][0][3]));
#pragma unroll
            for (int t = 1; t < 4; ++t) top = fmaxf(top, fmaxf(fmaxf(sc[c][t][0], sc[c][t][1]), fmaxf(sc[c][t][2], sc[c][t][3])));
            float lower, upper;
            swapped_pair<16>(top, lower, upper);
            swapped_pair<32>(fmaxf(lower, upper), lower, upper);
            const float m_new = fmaxf(m[c], weights_from<BF16>(fmaxf(lower, upper)));
            if (__any(m_new > m[c])) {
                const float back = __builtin_amdgcn_exp2f(m[c] - m_new);
                l[c] *= back;
#pragma unroll
                for (int i = 0; i < kTiles; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[c][i][j] *= back;
                m[c] = m_new;
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float e[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = __builtin_amdgcn_exp2f(sc[c][2 * u + (j >> 2)][j & 3] - m[c]);
                l[c] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
                p[c][u] = half_pack<BF16>(e);
            }
        }
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
            const uint4 lo = half_from_codes<BF16>(vf[i].x, vf[i].y, value_scale), hi = half_from_codes<BF16>(vf[i].z, vf[i].w, value_scale);
#pragma unroll
            for (int c = 0; c < SETS; ++c) o[c][i] = half_mfma16<BF16>(hi, p[c][1], half_mfma16<BF16>(lo, p[c][0], o[c][i]));
        }
        if constexpr (MORE) request_values(x, j0 + kStride, next_page);
        if (some_nan) {
            // NaN values were left out of the product: they are the end of the sums of the rows that see them
            __builtin_amdgcn_wave_barrier();                                  // (one wave's LDS operations take effect in order)
#pragma unroll
            for (int c = 0; c < SETS; ++c) {
                const int keys = limit[c] - j0;
                const uint64_t sees = TREE ? window(c, j0) : (keys >= 64 ? ~0ull : (keys <= 0 ? 0ull : (1ull << keys) - 1));
#pragma unroll
                for (int i = 0; i < kTiles; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (*reinterpret_cast<const uint64_t*>(nan_keys[wave][16 * i + 4 * g + j]) & sees) o[c][i][j] = __uint_as_float(0x7fc00000u);
            }
            __builtin_amdgcn_wave_barrier();
        }
    };
    int j0 = begin + kStep * wave;
    Step x;
    if (j0 < end) {
        pages(j0, key_page, value_page);
        const int page = value_page;
        request_keys(x, j0, key_page, page);
        pages(j0 + kStride, key_page, value_page);
        request_values(x, j0, page);
    }
    // the queries, behind the first codes; rows that the tile does not have as zeros
    {
        constexpr int kChunks = D / 8, kAtOnce = kThreads / kChunks, kPasses = (kRows + kAtOnce - 1) / kAtOnce;
        uint4 q[kPasses];
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            const int row = tid / kChunks + kAtOnce * i, at = kRows * tile + row;
            q[i] = make_uint4(0, 0, 0, 0);
            if (row < kRows && at < rows)
                q[i] = *reinterpret_cast<const uint4*>(a.q + (static_cast<size_t>(offset) + at / group) * a.q_stride + (kvh * group + at % group) * D + 8 * (tid % kChunks));
            if constexpr (BF16) {
                float v[8];
                half_eight<true>(q[i], v);
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(v[j]));
            }
        }
        // bf16 queries so large that products with codes could pass the largest float, where the scaled score need not: a power of two off, on again behind
        if (BF16 && __syncthreads_or(top >= 0x1p60f)) {
            late = 0x1p64f;
#pragma unroll
            for (int i = 0; i < kPasses; ++i) {
                float v[8];
                half_eight<true>(q[i], v);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] *= 0x1p-64f;
                q[i] = half_pack<true>(v);
            }
        }
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            const int row = tid / kChunks + kAtOnce * i;
            if (row < kRows) *reinterpret_cast<uint4*>(&queries[row][8 * (tid % kChunks)]) = q[i];
        }
    }
    if constexpr (TREE) {
        __syncthreads();
        if (tid < 64) {
            uint64_t bits[1] = {0};
            if (tid < n) tree_ancestors(parents, tid, bits);
            nodes[tid] = bits[0];
        }
    }
    __syncthreads();
    for (; j0 + kStride < end; j0 += kStride) work(std::true_type{}, x, j0);
    if (j0 < end) work(std::false_type{}, x, j0);
    // the waves together, in their order, one set of rows after the other
#pragma unroll
    for (int c = 0; c < SETS; ++c) {
        float lower, upper;
        swapped_pair<16>(l[c], lower, upper);
        swapped_pair<32>(lower + upper, lower, upper);
        if (c > 0) __syncthreads();
        if (g == 0) stats[wave][col] = make_float2(m[c], lower + upper);
#pragma unroll
        for (int i = 0; i < kTiles; ++i) *reinterpret_cast<v4f*>(&sums[wave][col * kPitch + 16 * i + 4 * g]) = o[c][i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16 * D / 4 / kThreads; ++i) {
            const int e = tid + kThreads * i, k = e / (D / 4), d = 4 * (e % (D / 4)), row = kRows * tile + 16 * c + k;
            if (row >= rows) continue;
            float top = stats[0][k].x;
#pragma unroll
            for (int w = 1; w < kWaves; ++w) top = fmaxf(top, stats[w][k].x);
            float den = 0.0f;
            v4f total = zero;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float f = __builtin_amdgcn_exp2f(stats[w][k].x - top);
                den = __builtin_fmaf(stats[w][k].y, f, den);
                const v4f part = *reinterpret_cast<const v4f*>(&sums[w][k * kPitch + d]);
#pragma unroll
                for (int j = 0; j < 4; ++j) total[j] = __builtin_fmaf(part[j], f, total[j]);
            }
            if (a.sums) {
                const size_t at = ((static_cast<size_t>(s) * a.kv_heads + kvh) * a.part_rows + row) * a.runs_bound + run;
                *reinterpret_cast<v4f*>(a.sums + at * D + d) = total;
                if (d == 0) a.stats[at] = make_float2(top, den);
            } else {
                const float inv = den == 0.0f ? 0.0f : 2.0f / den;            // (twice: the values went in halved)
                const size_t at = ((static_cast<size_t>(offset) + row / group) * a.heads + kvh * group + row % group) * D + d;
                *reinterpret_cast<uint2*>(a.out + at) = make_uint2(half_pair<BF16>(total[0] * inv, total[1] * inv), half_pair<BF16>(total[2] * inv, total[3] * inv));
            }
        }
    }
}

// The runs of one query row together, by a wave, in their order: no waits for other waves (142 sequences of one or two tokens behind up to 3000 positions, in a call
// that may hold more, 152 -> 133 us, seven of four tokens behind up to 6000 20.7 -> 18.7, 64 of one behind up to 8191 122.7 -> 117.9; twice as many runs in
// registers 23 and 133).
constexpr int kFewRuns = 16;
template <bool BF16, int D>
__device__ __forceinline__ void merge_few(const PagedDecodeArgs& a, int index0, int row, int runs, int offset, int kvh, int group) {
    constexpr int kPer = D / 64;
    const int lane = threadIdx.x & 63;
    const size_t index = (static_cast<size_t>(index0) + row) * a.runs_bound;
    const float2 mine = lane < runs ? a.stats[index + lane] : make_float2(-FLT_MAX, 0.0f);
    float v[kFewRuns][kPer];
#pragma unroll
    for (int i0 = 0; i0 < kFewRuns; i0 += 4) {
        if (i0 >= runs) break;                                                // (requests for a run again cost as much as for another)
#pragma unroll
        for (int i = i0; i < i0 + 4; ++i) {
            const float* part = a.sums + (index + min(i, runs - 1)) * D + kPer * lane;
#pragma unroll
            for (int j = 0; j < kPer; ++j) v[i][j] = part[j];
        }
    }
    const float top = group_max<64>(mine.x), factor = __builtin_amdgcn_exp2f(mine.x - top), den = group_sum<64>(mine.y * factor);
    float total[kPer] = {};
#pragma unroll
    for (int i = 0; i < kFewRuns; ++i) {
        if (i >= runs) break;
        const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(factor), i));
#pragma unroll
        for (int j = 0; j < kPer; ++j) total[j] = __builtin_fmaf(v[i][j], f, total[j]);
    }
    const float inv = den == 0.0f ? 0.0f : 2.0f / den;
    uint16_t* out = a.out + ((static_cast<size_t>(offset) + row / group) * a.heads + kvh * group + row % group) * D + kPer * lane;
    if constexpr (kPer == 2) *reinterpret_cast<uint32_t*>(out) = half_pair<BF16>(total[0] * inv, total[1] * inv);
    else *out = static_cast<uint16_t>(half_pair<BF16>(total[0] * inv, 0.0f));
}

// A workgroup per query row (where sequences have different numbers of rows, per 16th row): its runs together, an order that the number of runs fixes.
// All of up to 64 runs are requested at once.
template <bool BF16, int D>
__global__ __launch_bounds__(kThreads) void paged_merge_kernel(const PagedDecodeArgs a) {
    constexpr int kLanes = D / 4, kSlots = kThreads / kLanes, kBatch = 8;     // threads that share a run; runs side by side; of each of them at a time
    __shared__ float factors[256];
    __shared__ __align__(16) float sums[kSlots][D];
    __shared__ float red[2 * kWaves];
    const int tid = threadIdx.x, group = a.heads / a.kv_heads;
    const int index0 = blockIdx.x * a.part_rows, kvh = blockIdx.x % a.kv_heads, s = blockIdx.x / a.kv_heads;
    const int offset = a.cu_steps ? paged_offset(a.cu_steps, s, 0, a.tokens) : s * a.steps;
    const int64_t rows = static_cast<int64_t>(a.cu_steps ? paged_offset(a.cu_steps, s + 1, 0, a.tokens) - offset : a.steps) * group;
    if (rows > a.part_rows) return;
    const int runs = max(1, paged_runs(paged_length(a.lengths[s], a.width, a.page_shift), a.kv_heads));     // (256 at most)
    if (runs <= kFewRuns) {                                                   // (by the sequence, not by the table that has room for more: equal bits)
        for (int row = blockIdx.y + gridDim.y * (tid >> 6); row < rows; row += kWaves * gridDim.y) merge_few<BF16, D>(a, index0, row, runs, offset, kvh, group);
        return;
    }
    const int slot = tid / kLanes, d = 4 * (tid % kLanes);
    for (int row = blockIdx.y; row < rows; row += gridDim.y) {
        const size_t index = static_cast<size_t>(index0) + row;
        const float2* stats = a.stats + index * a.runs_bound;
        const float* part = a.sums + index * a.runs_bound * D + d;
        v4f first[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) first[i] = *reinterpret_cast<const v4f*>(part + static_cast<size_t>(min(slot + kSlots * i, runs - 1)) * D);
        const float2 mine = tid < runs ? stats[tid] : make_float2(-FLT_MAX, 0.0f);
        float top = group_max<64>(mine.x);
        if ((tid & 63) == 0) red[tid >> 6] = top;
        __syncthreads();
        top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float factor = __builtin_amdgcn_exp2f(mine.x - top);
        factors[tid] = factor;
        float den = group_sum<64>(mine.y * factor);
        if ((tid & 63) == 0) red[kWaves + (tid >> 6)] = den;
        __syncthreads();
        den = (red[kWaves] + red[kWaves + 1]) + (red[kWaves + 2] + red[kWaves + 3]);
        v4f total = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int base = slot; base < runs; base += kSlots * kBatch) {
            if (base != slot)
#pragma unroll
                for (int i = 0; i < kBatch; ++i) first[i] = *reinterpret_cast<const v4f*>(part + static_cast<size_t>(min(base + kSlots * i, runs - 1)) * D);
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const float f = base + kSlots * i < runs ? factors[base + kSlots * i] : 0.0f;
                if (base + kSlots * i < runs)
#pragma unroll
                    for (int j = 0; j < 4; ++j) total[j] = __builtin_fmaf(first[i][j], f, total[j]);
            }
        }
        *reinterpret_cast<v4f*>(&sums[slot][d]) = total;
        __syncthreads();
        if (tid < D / 2) {
            float x = 0.0f, y = 0.0f;
#pragma unroll
            for (int i = 0; i < kSlots; ++i) { x += sums[i][2 * tid]; y += sums[i][2 * tid + 1]; }
            const float inv = den == 0.0f ? 0.0f : 2.0f / den;
            *reinterpret_cast<uint32_t*>(a.out + ((static_cast<size_t>(offset) + row / group) * a.heads + kvh * group + row % group) * D + 2 * tid) = half_pair<BF16>(x * inv, y * inv);
        }
        if (row + gridDim.y < rows) __syncthreads();
    }
}

// For tables that have room for kFewRuns runs at most: a wave per query row.
template <bool BF16, int D>
__global__ __launch_bounds__(kThreads) void paged_merge_few_kernel(const PagedDecodeArgs a) {
    const int group = a.heads / a.kv_heads, kvh = blockIdx.x % a.kv_heads, s = blockIdx.x / a.kv_heads;
    const int offset = a.cu_steps ? paged_offset(a.cu_steps, s, 0, a.tokens) : s * a.steps;
    const int64_t rows = static_cast<int64_t>(a.cu_steps ? paged_offset(a.cu_steps, s + 1, 0, a.tokens) - offset : a.steps) * group;
    if (rows > a.part_rows) return;
    const int runs = max(1, paged_runs(paged_length(a.lengths[s], a.width, a.page_shift), a.kv_heads));
    for (int row = kWaves * blockIdx.y + (threadIdx.x >> 6); row < rows; row += kWaves * gridDim.y)
        merge_few<BF16, D>(a, blockIdx.x * a.part_rows, row, runs, offset, kvh, group);
}

template <bool BF16, int D, bool TREE>
int launch(const PagedDecodeArgs& a, hipStream_t stream) {
    // Two sets of rows share what is read: eight sequences behind 20718 positions, four new tokens of eight heads each, 116 -> 96 us.  They cost a compute
    // unit's third workgroup, so sequences that have one set get the other launch: 64 of one token of six heads behind up to 8000 positions, in a call
    // that may hold more, 253 -> 201 us.
    const int most = a.cu_steps ? std::min(a.part_rows, 16) : a.part_rows;
    if (most <= 16) hipLaunchKernelGGL((paged_decode_kernel<BF16, D, 1, TREE>), dim3(a.kv_heads, a.runs_bound, a.seqs), dim3(kThreads), 0, stream, a, 1, most);
    if (a.part_rows > 16)
        hipLaunchKernelGGL((paged_decode_kernel<BF16, D, 2, TREE>), dim3((a.part_rows + 31) / 32 * a.kv_heads, a.runs_bound, a.seqs), dim3(kThreads), 0, stream, a, most < a.part_rows ? 17 : 1,
                           a.part_rows);
    if (hipGetLastError() != hipSuccess) return PLLM_ERR_LAUNCH;
    if (a.sums) {
        const int rows = a.cu_steps ? std::min(a.part_rows, 16) : a.part_rows;
        if (a.runs_bound <= kFewRuns) hipLaunchKernelGGL((paged_merge_few_kernel<BF16, D>), dim3(a.seqs * a.kv_heads, (rows + kWaves - 1) / kWaves), dim3(kThreads), 0, stream, a);
        else hipLaunchKernelGGL((paged_merge_kernel<BF16, D>), dim3(a.seqs * a.kv_heads, rows), dim3(kThreads), 0, stream, a);
        if (hipGetLastError() != hipSuccess) return PLLM_ERR_LAUNCH;
    }
    return PLLM_OK;
}

}  // namespace

size_t paged_decode_parts_bytes(int64_t seqs, int64_t part_rows, int64_t kv_heads, int64_t head_dim, int64_t positions) {
    const size_t runs = static_cast<size_t>(paged_runs_bound(positions, static_cast<int>(kv_heads)));
    if (runs == 1) return 0;
    const size_t parts = static_cast<size_t>(seqs) * part_rows * kv_heads * runs;
    return align256(parts * head_dim * sizeof(float)) + align256(parts * sizeof(float2));
}

int paged_decode_launch(PagedDecodeArgs& a, void* workspace, bool bf16, int head_dim, hipStream_t stream) {
    a.runs_bound = paged_runs_bound(static_cast<int64_t>(a.width) << a.page_shift, a.kv_heads);
    a.sums = nullptr;
    a.stats = nullptr;
    if (a.runs_bound > 1) {
        a.sums = static_cast<float*>(workspace);
        a.stats = reinterpret_cast<float2*>(static_cast<unsigned char*>(workspace) +
                                            align256(static_cast<size_t>(a.seqs) * a.part_rows * a.kv_heads * a.runs_bound * head_dim * sizeof(float)));
    }
    if (a.parents) {
        if (head_dim == 128) return bf16 ? launch<true, 128, true>(a, stream) : launch<false, 128, true>(a, stream);
        return bf16 ? launch<true, 64, true>(a, stream) : launch<false, 64, true>(a, stream);
    }
    if (head_dim == 128) return bf16 ? launch<true, 128, false>(a, stream) : launch<false, 128, false>(a, stream);
    return bf16 ? launch<true, 64, false>(a, stream) : launch<false, 64, false>(a, stream);
}

}  // namespace pllm

extern "C" {

size_t pllm_paged_attention_decode_workspace_bytes(int64_t seqs, int64_t steps, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t positions) {
    if (seqs <= 0 || steps <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || positions <= 0 || seqs > 65535 || steps > 4096 || heads > 1024 || kv_heads > heads ||
        head_dim > 256)
        return 0;
    return pllm::paged_decode_parts_bytes(seqs, steps * (heads / kv_heads), kv_heads, head_dim, positions);
}

int pllm_paged_attention_decode(const void* q, int64_t q_stride, int dtype, const uint8_t* key_pages, const uint8_t* value_pages, const float* key_scales,
                                const float* value_scales, int64_t pool, int64_t page_tokens, const int32_t* block_table, int64_t table_stride,
                                int64_t table_width, const int32_t* lengths, int64_t seqs, int64_t steps, int64_t heads, int64_t kv_heads,
                                int64_t head_dim, float scale, void* out, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace pllm;
    if (!q || !key_pages || !value_pages || !key_scales || !value_scales || !block_table || !lengths || !out) return PLLM_ERR_INVALID_ARGUMENT;
    if (dtype != PLLM_F16 && dtype != PLLM_BF16) return PLLM_ERR_INVALID_ARGUMENT;
    if (seqs <= 0 || steps <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || pool <= 0 || table_width <= 0 || table_stride < table_width ||
        q_stride < heads * head_dim || !(scale >= 0.0f && scale <= 0x1p127f))
        return PLLM_ERR_INVALID_ARGUMENT;
    if ((head_dim != 64 && head_dim != 128) || (page_tokens != 16 && page_tokens != 32 && page_tokens != 64 && page_tokens != 128)) return PLLM_ERR_UNSUPPORTED;
    // pages and positions in 32 bits, one grid row per head and sequence
    if (seqs > 65535 || heads > 1024 || steps * (heads / kv_heads) > 4096 || seqs * steps * heads > 0xffffff || pool > 0x7fffffff || table_width > 0x3fffffff / page_tokens) return PLLM_ERR_UNSUPPORTED;
    const uintptr_t wide = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(key_pages) | reinterpret_cast<uintptr_t>(value_pages) |
                           reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace);
    const uintptr_t narrow = reinterpret_cast<uintptr_t>(key_scales) | reinterpret_cast<uintptr_t>(value_scales) | reinterpret_cast<uintptr_t>(block_table) |
                             reinterpret_cast<uintptr_t>(lengths);
    if ((wide & 15u) || (narrow & 3u) || q_stride % 8) return PLLM_ERR_INVALID_ARGUMENT;
    const int64_t positions = table_width * page_tokens;
    const size_t need = pllm_paged_attention_decode_workspace_bytes(seqs, steps, heads, kv_heads, head_dim, positions);
    if (need > 0 && (!workspace || workspace_bytes < need)) return PLLM_ERR_WORKSPACE;
    PagedDecodeArgs a{};
    a.q = static_cast<const uint16_t*>(q); a.q_stride = static_cast<size_t>(q_stride);
    a.key_pages = key_pages; a.value_pages = value_pages; a.key_scales = key_scales; a.value_scales = value_scales;
    a.table = block_table; a.table_stride = static_cast<size_t>(table_stride); a.lengths = lengths;
    a.out = static_cast<uint16_t*>(out);
    a.scale = scale * 1.4426950408889634f;
    a.seqs = static_cast<int>(seqs); a.steps = static_cast<int>(steps); a.heads = static_cast<int>(heads); a.kv_heads = static_cast<int>(kv_heads);
    a.page_shift = page_tokens == 16 ? 4 : page_tokens == 32 ? 5 : page_tokens == 64 ? 6 : 7;
    a.pool = static_cast<int>(pool); a.width = static_cast<int>(table_width);
    a.part_rows = static_cast<int>(steps * (heads / kv_heads));
    return paged_decode_launch(a, workspace, dtype == PLLM_BF16, static_cast<int>(head_dim), static_cast<hipStream_t>(stream));
}

}  // extern "C"
