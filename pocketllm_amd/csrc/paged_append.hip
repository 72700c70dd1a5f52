// New keys and values into a paged E4M3 cache, the rotary phases on the way, and the new queries turned beside them: one launch.
//     k' = k cos_p + swap(k) sin_p (the halves of the rotary part swapped; for keys in 64 bits), p = lengths[s] - n_s + i for token i of sequence s, or what `positions`
//     say of it (nodes of a drafted tree: the past plus their depth)
//     scale of a page and head: the least power of two with amax / scale <= 448 over what the page holds;  code = E4M3(k' / scale)
// A page that a call continues keeps its scale unless the new tokens need a larger one; then its older codes are scaled down by the ratio, a power
// of two: exact, but for codes that get below E4M3's normal values, which are rounded again.  A page that a call begins forgets what it held.
// Values that are not finite become NaN codes and do not count for the scale.
//
// A workgroup owns a page's keys, or its values, of one head: its scale needs no atomics and no second pass.  Values turn in LDS, since a page
// holds them with the tokens innermost.  The queries are rows behind these workgroups in the same grid.
// Bound: bytes for prompts (4096 tokens of 48 and 8 heads of 128: 128 MB in 24 us, 5.3 TB/s; in 32 bits 23.6), the chain of a workgroup's loads
// (offset, length, row and page, scale: 4 us) and the number of workgroups (two for every page and head) for decode steps.
#include "paged_device.h"
#include "pllm_internal.h"

#include <cfloat>

namespace pllm {
namespace {

constexpr int kHeadPasses = 4;                  // heads that a thread of a query's workgroup turns, one after the other

struct AppendArgs {
    const uint16_t* q; const uint16_t* k; const uint16_t* v;
    size_t q_stride, k_stride, v_stride;                        // elements between tokens
    uint16_t* q_out;                                            // [rows][heads][D], null: no queries
    uint8_t* key_pages; uint8_t* value_pages;
    float* key_scales; float* value_scales;
    const int32_t* table; size_t table_stride;
    const int32_t* lengths; const int32_t* cu_steps;
    const float* cos_table; const float* sin_table;             // [>= width * page][D], or [positions_end][D] where `positions` says which row
    const int32_t* positions;                                   // [rows] or null: the place in the cache
    int positions_end;
    int rows, seqs, even_steps, even_pages, heads,            // even: every sequence has that many new tokens, which touch that many pages at most
        kv_heads, pool, width, rope_half, page_blocks, head_blocks,
        row_heads;                                              // few heads: a workgroup turns so many rows of them at a time
};

struct Phases { float4 c[2], s[2]; };
// the row of the phases that a new token is turned by
__device__ __forceinline__ int turned_by(const AppendArgs& a, int row, int place) { return a.positions ? clamp_int(a.positions[row], 0, a.positions_end - 1) : place; }
__device__ __forceinline__ float of4(const float4* f, int i) {
    const float4 v = f[i >> 2];
    return (i & 3) == 0 ? v.x : (i & 3) == 1 ? v.y : (i & 3) == 2 ? v.z : v.w;
}
__device__ __forceinline__ Phases load_phases(const AppendArgs& a, int position, int dim, int d0) {
    Phases p;
    const float4* c = reinterpret_cast<const float4*>(a.cos_table + static_cast<size_t>(position) * dim + d0);
    const float4* s = reinterpret_cast<const float4*>(a.sin_table + static_cast<size_t>(position) * dim + d0);
    p.c[0] = c[0]; p.c[1] = c[1]; p.s[0] = s[0]; p.s[1] = s[1];
    return p;
}
__device__ __forceinline__ void turn(float own[8], const float other[8], const Phases& p) {
#pragma unroll
    for (int i = 0; i < 8; ++i) own[i] = __builtin_fmaf(other[i], of4(p.s, i), own[i] * of4(p.c, i));
}
// the same for what becomes codes: products and sum in 64 bits, cut so that the codes are those of the sum itself (in 32 bits one in about a million is not)
__device__ __forceinline__ void turn_for_codes(float own[8], const float other[8], const Phases& p) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
        own[i] = odd_float(__builtin_fma(static_cast<double>(other[i]), static_cast<double>(of4(p.s, i)), static_cast<double>(own[i]) * static_cast<double>(of4(p.c, i))));
}
// the least power of two that brings amax to 448 = 1.75 * 2^8 or below, at least 2^-120
__device__ __forceinline__ float page_scale(float amax) {
    const int e = static_cast<int>((__float_as_uint(amax) + 0x1fffffu) >> 23) - 8;      // (a mantissa beyond .75 carries)
    return __uint_as_float(static_cast<uint32_t>(max(e, 127 - 120)) << 23);
}
__device__ __forceinline__ float codable(float v, float inv) {
    return fabsf(v) <= FLT_MAX ? fminf(fmaxf(v * inv, -448.0f), 448.0f) : __uint_as_float(0x7fc00000u);
}
template <bool BF16, int D, int THREADS>
__device__ __forceinline__ void turn_queries(const AppendArgs& a, int block, int page_shift) {
    constexpr int kChunks = D / 8, kHeadsPerPass = THREADS / kChunks;
    const int row = block / a.head_blocks, head0 = block % a.head_blocks * (kHeadPasses * kHeadsPerPass) + threadIdx.x / kChunks;
    const int s = a.cu_steps ? paged_sequence(a.cu_steps, a.rows, a.seqs + 1, 1, 0, row) : row / a.even_steps;
    const int chunk = threadIdx.x % kChunks, d0 = 8 * chunk, half = a.rope_half;
    int64_t at = -1;
    if (s < a.seqs) at = static_cast<int64_t>(a.lengths[s]) - paged_offset(a.cu_steps, s + 1, a.even_steps, a.rows) + row;
    const bool placed = at >= 0 && at < (static_cast<int64_t>(a.width) << page_shift);
    const int position = static_cast<int>(at);
    const bool turns = placed && d0 < 2 * half;
    Phases p;
    if (turns) p = load_phases(a, turned_by(a, row, position), D, d0);
    const int partner = d0 < half ? d0 + half : d0 - half;
    const uint16_t* src = a.q + static_cast<size_t>(row) * a.q_stride;
    uint16_t* dst = a.q_out + static_cast<size_t>(row) * a.heads * D;
#pragma unroll
    for (int i = 0; i < kHeadPasses; ++i) {
        const int h = head0 + kHeadsPerPass * i;
        if (h >= a.heads) break;
        uint4 out = make_uint4(0, 0, 0, 0);                                   // rows that have no place in a sequence
        if (placed) {
            out = *reinterpret_cast<const uint4*>(src + h * D + d0);
            if (turns) {
                const uint4 across = *reinterpret_cast<const uint4*>(src + h * D + partner);
                float own[8], other[8];
                half_eight<BF16>(out, own);
                half_eight<BF16>(across, other);
                turn(own, other, p);
                out = half_pack<BF16>(own);
            }
        }
        *reinterpret_cast<uint4*>(dst + h * D + d0) = out;
    }
}

// The same where all heads of a row, or of several, are one pass of the workgroup: kHeadPasses times as many rows (27170 tokens of 4 heads of 128, with 2 heads' keys
// and values in pages of 64: 34.9 -> 23.8 us; a workgroup per row costs a nanosecond of the launch each).
template <bool BF16, int D, int THREADS>
__device__ __forceinline__ void turn_rows(const AppendArgs& a, int block, int page_shift) {
    constexpr int kChunks = D / 8;
    const int slot = threadIdx.x / kChunks, chunk = threadIdx.x % kChunks, d0 = 8 * chunk, half = a.rope_half, h = slot % a.heads;
    const int partner = d0 < half ? d0 + half : d0 - half;
    // (the first row's sequence by a search, the others' from there on: 400 sequences of up to 60 tokens 32.2 -> 23.2 us)
    int from = a.cu_steps ? paged_sequence(a.cu_steps, a.rows, a.seqs + 1, 1, 0, block * kHeadPasses * a.row_heads) : 0;
#pragma unroll
    for (int i = 0; i < kHeadPasses; ++i) {
        const int row = (block * kHeadPasses + i) * a.row_heads + slot / a.heads;
        const bool mine = slot < a.row_heads * a.heads && row < a.rows;
        int s = mine ? row / max(a.even_steps, 1) : a.seqs;
        if (a.cu_steps) {
            while (mine && from < a.seqs && paged_offset(a.cu_steps, from + 1, 0, a.rows) <= row) ++from;
            s = from;
        }
        int64_t at = -1;
        if (s < a.seqs) at = static_cast<int64_t>(a.lengths[s]) - paged_offset(a.cu_steps, s + 1, a.even_steps, a.rows) + row;
        if (!mine) continue;
        uint4 out = make_uint4(0, 0, 0, 0);                                   // rows that have no place in a sequence
        if (at >= 0 && at < (static_cast<int64_t>(a.width) << page_shift)) {
            const uint16_t* src = a.q + static_cast<size_t>(row) * a.q_stride + h * D;
            out = *reinterpret_cast<const uint4*>(src + d0);
            if (d0 < 2 * half) {
                const uint4 across = *reinterpret_cast<const uint4*>(src + partner);
                float own[8], other[8];
                half_eight<BF16>(out, own);
                half_eight<BF16>(across, other);
                turn(own, other, load_phases(a, turned_by(a, row, static_cast<int>(at)), D, d0));
                out = half_pack<BF16>(own);
            }
        }
        *reinterpret_cast<uint4*>(a.q_out + (static_cast<size_t>(row) * a.heads + h) * D + d0) = out;
    }
}

// Waves per SIMD that the rows of a page leave registers for (a thread's pass: eight for what is loaded, eight for what becomes codes).  Without the bound the 64-bit
// products take half as many again (38 prompts of 715 tokens, 4 and 2 heads of 128, pages of 64: 40.6 us, with it 35.2, in 32 bits 34.6).
constexpr int append_waves(int dim, int page) { return page * dim <= 4096 ? 8 : page * dim <= 8192 ? 6 : 4; }

// ROWS: the queries go by turn_rows (in a kernel of its own: a choice in this one cost the others 2 - 7 %).
// FEW: every sequence has the same few new tokens, no more than one pass over 64 threads takes: a workgroup of one wave (one token of each of 64 sequences
// 6.3 -> 5.3 us, of 256 14.7 -> 9.6; 48 and 8 heads of 128)
template <bool BF16, int D, int PAGE, bool FEW, bool ROWS>
__global__ __launch_bounds__(FEW ? 64 : 256, FEW ? 1 : append_waves(D, PAGE)) void paged_append_kernel(const AppendArgs a) {
    constexpr int kThreads = FEW ? 64 : 256;
    constexpr int kChunks = D / 8, kRows = kThreads / kChunks, kPasses = FEW ? 1 : (PAGE + kRows - 1) / kRows;
    constexpr int kShift = PAGE == 16 ? 4 : PAGE == 32 ? 5 : PAGE == 64 ? 6 : 7;
    __shared__ float red[4];
    __shared__ __align__(16) uint8_t turned[(FEW ? kRows : PAGE) * D];
    const int block = blockIdx.x, tid = threadIdx.x;
    if (block >= a.page_blocks) {
        if constexpr (ROWS) turn_rows<BF16, D, kThreads>(a, block - a.page_blocks, kShift);
        else turn_queries<BF16, D, kThreads>(a, block - a.page_blocks, kShift);
        return;
    }
    const bool values = block & 1;
    const int head = (block >> 1) % a.kv_heads, slot = (block >> 1) / a.kv_heads;
    const int s = a.cu_steps ? paged_sequence(a.cu_steps, a.rows, a.seqs, PAGE, 2, slot) : slot / a.even_pages;
    const int offset = paged_offset(a.cu_steps, s, a.even_steps, a.rows), n = paged_offset(a.cu_steps, s + 1, a.even_steps, a.rows) - offset;
    const int length = max(a.lengths[s], 0);
    const int first = length - n, begin = max(first, 0);                      // (a length below its new tokens: the earliest have no place)
    const int64_t mine = (begin >> kShift) + (a.cu_steps ? slot - paged_first_slot(offset, s, PAGE, 2) : slot % a.even_pages);
    if (n <= 0 || mine < 0 || mine >= a.width) return;
    const int page0 = static_cast<int>(mine) << kShift;                       // (width << kShift fits an int: the host's check)
    const int lo = max(begin, page0), hi = min(length, page0 + PAGE), count = hi - lo;
    if (count <= 0) return;

    // the new rows, eight neighbouring values of one token to a thread at a time; requested before the page that they go to is known
    const int chunk = tid % kChunks, d0 = 8 * chunk, half = a.rope_half;
    const bool turns = !values && d0 < 2 * half;
    const int partner = turns ? (d0 < half ? d0 + half : d0 - half) : d0;
    const uint16_t* src = (values ? a.v : a.k) + head * D;
    const size_t stride = values ? a.v_stride : a.k_stride;
    uint4 own[kPasses], other[kPasses];
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        const int token = min(tid / kChunks + kRows * i, count - 1);          // (threads behind the last token load it again)
        const uint16_t* row = src + static_cast<size_t>(offset + (lo + token - first)) * stride;
        own[i] = *reinterpret_cast<const uint4*>(row + d0);
        if (turns) other[i] = *reinterpret_cast<const uint4*>(row + partner);
    }
    const int page = paged_page(a.table + static_cast<size_t>(s) * a.table_stride, page0, a.width, kShift, a.pool);
    if (page < 0) return;
    const size_t at = static_cast<size_t>(page) * a.kv_heads + head;
    uint8_t* codes = (values ? a.value_pages : a.key_pages) + at * PAGE * D;
    float* scale_at = (values ? a.value_scales : a.key_scales) + at;
    const int held = lo - page0;                                              // tokens that the page keeps
    const float old = held > 0 ? *scale_at : 0.0f;
    float v[kPasses][8], amax = 0.0f;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        if (kRows * i >= count) break;
        half_eight<BF16>(own[i], v[i]);
        if (turns) {
            float across[8];
            half_eight<BF16>(other[i], across);
            const int place = lo + min(tid / kChunks + kRows * i, count - 1);
            turn_for_codes(v[i], across, load_phases(a, turned_by(a, offset + place - first, place), D, d0));
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fabsf(v[i][j]) <= FLT_MAX ? fmaxf(amax, fabsf(v[i][j])) : amax;
    }
    amax = group_max<64>(amax);
    if constexpr (!FEW) {
        if ((tid & 63) == 0) red[tid >> 6] = amax;
        __syncthreads();
        amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    }
    const float need = page_scale(amax), scale = fmaxf(old, need), inv = 1.0f / scale;
    if (tid == 0) *scale_at = scale;
    if (held > 0 && scale > old) {                                            // what the page holds, on the larger scale
        const float ratio = old / scale;
        const int pieces = values ? D * ((held + 15) / 16) : held * (D / 16);
        for (int p = tid; p < pieces; p += kThreads) {
            const int across = (held + 15) / 16;
            uint4* piece = reinterpret_cast<uint4*>(values ? codes + (p / across) * PAGE + 16 * (p % across) : codes + 16 * p);
            const int keep = values ? held - 16 * (p % across) : 16;
            const uint4 w = *piece;
            const uint32_t m[4] = {first_bytes(keep), first_bytes(keep - 4), first_bytes(keep - 8), first_bytes(keep - 12)};
            *piece = make_uint4((scaled_codes(w.x, ratio) & m[0]) | (w.x & ~m[0]), (scaled_codes(w.y, ratio) & m[1]) | (w.y & ~m[1]),
                                (scaled_codes(w.z, ratio) & m[2]) | (w.z & ~m[2]), (scaled_codes(w.w, ratio) & m[3]) | (w.w & ~m[3]));
        }
    }
    uint8_t* rows = values ? turned : codes + held * D;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        const int t = tid / kChunks + kRows * i;
        if (t >= count) break;
        float c[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = codable(v[i][j], inv);
        *reinterpret_cast<uint2*>(rows + t * D + d0) = make_uint2(four_codes(c[0], c[1], c[2], c[3]), four_codes(c[4], c[5], c[6], c[7]));
    }
    if (!values) return;
    __syncthreads();                                                          // (also between the older codes' stores and the new ones in the same 16 bytes)
    const int c0 = held / 16, pieces = D * ((held + count + 15) / 16 - c0);
    for (int p = tid; p < pieces; p += kThreads) {
        const int d = p % D, t0 = 16 * (c0 + p / D);                          // slots t0 .. t0 + 15 of dimension d
        uint8_t* dst = codes + static_cast<size_t>(d) * PAGE + t0;
        const int from = max(held, t0), to = min(held + count, t0 + 16);
        if (to - from == 16) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint8_t* c = turned + (t0 - held + 4 * j) * D + d;
                w[j] = c[0] | (c[D] << 8) | (c[2 * D] << 16) | (static_cast<uint32_t>(c[3 * D]) << 24);
            }
            *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            for (int t = from; t < to; ++t) dst[t - t0] = turned[(t - held) * D + d];
        }
    }
}

// (a kernel for every page size: small pages need few registers and little LDS, and their workgroups hide one another's waits)
template <bool BF16, int D, bool FEW, bool ROWS>
void launch(const AppendArgs& a, int64_t page_tokens, dim3 grid, hipStream_t stream) {
    const dim3 threads(FEW ? 64 : 256);
    if (page_tokens == 16) hipLaunchKernelGGL((paged_append_kernel<BF16, D, 16, FEW, ROWS>), grid, threads, 0, stream, a);
    else if (page_tokens == 32) hipLaunchKernelGGL((paged_append_kernel<BF16, D, 32, FEW, ROWS>), grid, threads, 0, stream, a);
    else if (page_tokens == 64) hipLaunchKernelGGL((paged_append_kernel<BF16, D, 64, FEW, ROWS>), grid, threads, 0, stream, a);
    else hipLaunchKernelGGL((paged_append_kernel<BF16, D, 128, FEW, ROWS>), grid, threads, 0, stream, a);
}

}  // namespace
}  // namespace pllm

extern "C" int pllm_paged_kv_append_at(const void* q, int64_t q_stride, const void* k_new, int64_t k_stride, const void* v_new, int64_t v_stride, int dtype,
                                    void* q_out, uint8_t* key_pages, uint8_t* value_pages, float* key_scales, float* value_scales, int64_t pool,
                                    int64_t page_tokens, const int32_t* block_table, int64_t table_stride, int64_t table_width, const int32_t* lengths,
                                    const int32_t* cu_steps, const float* cos_table, const float* sin_table, int64_t table_positions,
                                    const int32_t* positions, int64_t rope_dim,
                                    int64_t rows, int64_t seqs, int64_t heads, int64_t kv_heads, int64_t head_dim, void* stream) {
    using namespace pllm;
    if (!k_new || !v_new || !key_pages || !value_pages || !key_scales || !value_scales || !block_table || !lengths) return PLLM_ERR_INVALID_ARGUMENT;
    if ((q != nullptr) != (q_out != nullptr) || (dtype != PLLM_F16 && dtype != PLLM_BF16)) return PLLM_ERR_INVALID_ARGUMENT;
    if (rows <= 0 || seqs <= 0 || kv_heads <= 0 || pool <= 0 || table_width <= 0 || table_stride < table_width || (q && heads <= 0)) return PLLM_ERR_INVALID_ARGUMENT;
    if (!cu_steps && rows % seqs != 0) return PLLM_ERR_INVALID_ARGUMENT;
    if (k_stride < kv_heads * head_dim || v_stride < kv_heads * head_dim || (q && q_stride < heads * head_dim)) return PLLM_ERR_INVALID_ARGUMENT;
    if (rope_dim < 0 || rope_dim > head_dim || (rope_dim > 0 && (!cos_table || !sin_table || table_positions <= 0 || (!positions && table_positions < table_width * page_tokens))))
        return PLLM_ERR_INVALID_ARGUMENT;
    if ((head_dim != 64 && head_dim != 128) || rope_dim % 16 != 0 || (page_tokens != 16 && page_tokens != 32 && page_tokens != 64 && page_tokens != 128))
        return PLLM_ERR_UNSUPPORTED;
    // pages and positions in 32 bits, and a launch that counts its threads in 32 bits
    if (rows > 0x3fffff || seqs > 0xfffff || kv_heads > 1024 || heads > 1024 || pool > 0x7fffffff || table_width > 0x3fffffff / page_tokens) return PLLM_ERR_UNSUPPORTED;
    const int64_t even_pages = paged_pages_touched(rows / seqs, page_tokens);
    const int64_t slots = cu_steps ? paged_slots(rows, static_cast<int>(seqs), static_cast<int>(page_tokens), 2) : seqs * even_pages, page_blocks = 2 * slots * kv_heads;
    const bool few = !cu_steps && rows / seqs <= 64 * 8 / head_dim;           // a decode step
    const int64_t at_once = (few ? 64 : 256) * 8 / head_dim, head_blocks = q ? (heads + kHeadPasses * at_once - 1) / (kHeadPasses * at_once) : 0;
    const int64_t row_heads = q && !few && heads <= at_once ? at_once / heads : 0;
    const int64_t query_blocks = row_heads ? (rows + kHeadPasses * row_heads - 1) / (kHeadPasses * row_heads) : rows * head_blocks;
    if (page_blocks + query_blocks > 0xffffff) return PLLM_ERR_UNSUPPORTED;
    const uintptr_t wide = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_new) | reinterpret_cast<uintptr_t>(v_new) | reinterpret_cast<uintptr_t>(q_out) |
                           reinterpret_cast<uintptr_t>(key_pages) | reinterpret_cast<uintptr_t>(value_pages) | reinterpret_cast<uintptr_t>(cos_table) |
                           reinterpret_cast<uintptr_t>(sin_table);
    const uintptr_t narrow = reinterpret_cast<uintptr_t>(key_scales) | reinterpret_cast<uintptr_t>(value_scales) | reinterpret_cast<uintptr_t>(block_table) |
                             reinterpret_cast<uintptr_t>(lengths) | reinterpret_cast<uintptr_t>(cu_steps) | reinterpret_cast<uintptr_t>(positions);
    if ((wide & 15u) || (narrow & 3u) || (k_stride % 8) || (v_stride % 8) || (q && q_stride % 8)) return PLLM_ERR_INVALID_ARGUMENT;
    AppendArgs a{};
    a.q = static_cast<const uint16_t*>(q); a.k = static_cast<const uint16_t*>(k_new); a.v = static_cast<const uint16_t*>(v_new);
    a.q_stride = static_cast<size_t>(q_stride); a.k_stride = static_cast<size_t>(k_stride); a.v_stride = static_cast<size_t>(v_stride);
    a.q_out = static_cast<uint16_t*>(q_out);
    a.key_pages = key_pages; a.value_pages = value_pages; a.key_scales = key_scales; a.value_scales = value_scales;
    a.table = block_table; a.table_stride = static_cast<size_t>(table_stride); a.lengths = lengths; a.cu_steps = cu_steps;
    a.cos_table = cos_table; a.sin_table = sin_table; a.positions = positions; a.positions_end = static_cast<int>(table_positions < 0x7fffffff ? table_positions : 0x7fffffff);
    a.rows = static_cast<int>(rows); a.seqs = static_cast<int>(seqs); a.even_steps = static_cast<int>(rows / seqs); a.even_pages = static_cast<int>(even_pages);
    a.heads = static_cast<int>(heads); a.kv_heads = static_cast<int>(kv_heads);
    a.pool = static_cast<int>(pool); a.width = static_cast<int>(table_width); a.rope_half = static_cast<int>(rope_dim / 2);
    a.page_blocks = static_cast<int>(page_blocks);
    a.head_blocks = static_cast<int>(head_blocks);
    a.row_heads = static_cast<int>(row_heads);
    const dim3 grid(static_cast<unsigned>(page_blocks + query_blocks));
    const hipStream_t st = static_cast<hipStream_t>(stream);
#define PLLM_APPEND(BF16, D) few ? launch<BF16, D, true, false>(a, page_tokens, grid, st) : row_heads ? launch<BF16, D, false, true>(a, page_tokens, grid, st) : launch<BF16, D, false, false>(a, page_tokens, grid, st)
    if (head_dim == 128) dtype == PLLM_BF16 ? (PLLM_APPEND(true, 128)) : (PLLM_APPEND(false, 128));
    else dtype == PLLM_BF16 ? (PLLM_APPEND(true, 64)) : (PLLM_APPEND(false, 64));
#undef PLLM_APPEND
    return hipGetLastError() == hipSuccess ? PLLM_OK : PLLM_ERR_LAUNCH;
}

extern "C" int pllm_paged_kv_append(const void* q, int64_t q_stride, const void* k_new, int64_t k_stride, const void* v_new, int64_t v_stride, int dtype,
                                    void* q_out, uint8_t* key_pages, uint8_t* value_pages, float* key_scales, float* value_scales, int64_t pool,
                                    int64_t page_tokens, const int32_t* block_table, int64_t table_stride, int64_t table_width, const int32_t* lengths,
                                    const int32_t* cu_steps, const float* cos_table, const float* sin_table, int64_t table_positions, int64_t rope_dim,
                                    int64_t rows, int64_t seqs, int64_t heads, int64_t kv_heads, int64_t head_dim, void* stream) {
    return pllm_paged_kv_append_at(q, q_stride, k_new, k_stride, v_new, v_stride, dtype, q_out, key_pages, value_pages, key_scales, value_scales, pool, page_tokens, block_table, table_stride, table_width, lengths, cu_steps, cos_table, sin_table, table_positions, nullptr, rope_dim, rows, seqs, heads, kv_heads, head_dim, stream);
}
