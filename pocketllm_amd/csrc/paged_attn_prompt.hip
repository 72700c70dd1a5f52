// Causal attention of many new tokens per sequence (prompts, their continuations, any mix of lengths) over a paged E4M3 cache that holds their keys
// and values already: out = softmax(scale q K^T) V, every query up to its own position.
//
// A workgroup of four waves takes 128 query rows of one key/value head, a wave 32 of them; rows are tokens times the heads that share the
// key/value head, so short prompts fill tiles too and keys are fetched once for the whole group.  64 keys at a time: their codes are requested one
// tile ahead into registers, become 16-bit values there (exact) and go to LDS, double-buffered; every wave reads them from there as operands.  The
// wave forms S^T = K Q^T (v_mfma_f32_32x32x16: matrix rows are keys, columns queries), so a lane holds half of one query's scores and what it leaves is,
// rounded to 16 bits, the second operand of O^T = V^T P^T: within 16 keys lane half h holds keys 4 h .. + 3 and 8 + 4 h .. + 3, the words of a piece
// of 16 value codes (tokens innermost in a page) in turn.  The keys' scale, one per 16 keys, goes into the product that takes scores to exponents; the
// values' scale (halved, so that fp16 holds every value that rounds up from its largest) into the conversion.
// 16-byte pieces of a row lie permuted in LDS (key rows by row % 16, value rows by row / 2 % 8), so 16 neighbouring rows read at one piece meet no
// bank twice.  Tiles of queries are dealt out in slots (paged_cache.h), the longest of a sequence first; rows behind the last sequence get zeros.
#include "paged_device.h"
#include "pllm_internal.h"

#include <cfloat>

namespace pllm {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves, kBlockRows = 32 * kWaves;
constexpr int kTile = 64;                       // keys per step

struct PagedPromptArgs {
    const uint16_t* q; size_t q_stride;         // elements between tokens
    const uint8_t* key_pages; const uint8_t* value_pages;
    const float* key_scales; const float* value_scales;
    const int32_t* table; size_t table_stride;
    const int32_t* lengths; const int32_t* cu_steps;
    uint16_t* out;
    float scale;                                // base 2
    int tokens, seqs, heads, kv_heads, page_shift, pool, width, slots;
};

template <bool BF16, int D>
__global__ __launch_bounds__(kThreads, 2) void paged_prompt_kernel(const PagedPromptArgs a) {
    constexpr int kKeyBytes = kTile * D * 2, kTileBytes = 2 * kKeyBytes;      // keys [64][D], then values [D][64]
    constexpr int kDimTiles = D / 32;
    constexpr int kLoads = kTile * D / 16 / kThreads;                         // 16-byte pieces of codes per thread, keys and values each
    extern __shared__ __align__(1024) unsigned char smem[];                   // [2][kTileBytes]
    __shared__ __align__(16) float factors[2][4];                             // the keys' scales of a tile's chunks of 16, times `scale`
    __shared__ int notes[3];                                                  // of tile t at t % 3; bits 0 - 3: chunks whose page is missing, bit 4: a NaN value code
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.x, group = a.heads / a.kv_heads;
    const int64_t slot = a.slots - 1 - static_cast<int64_t>(blockIdx.y);
    // rows of one key/value head: token * group + head in the group; the tokens behind the last sequence are one more, without keys
    const int64_t rows_all = static_cast<int64_t>(a.tokens) * group;
    int s = 0;
    {
        int owners = 0;
        for (int base = 0; base <= a.seqs; base += 64) {
            const int c = base + lane;
            const bool begun = c <= a.seqs && paged_first_slot(static_cast<int64_t>(paged_offset(a.cu_steps, c, 0, a.tokens)) * group, c, kBlockRows, 1) <= slot;
            const int n = __popcll(__ballot(begun));
            owners += n;
            if (n < 64) break;
        }
        s = __builtin_amdgcn_readfirstlane(max(owners - 1, 0));
    }
    const bool tail = s == a.seqs;
    const int offset = paged_offset(a.cu_steps, s, 0, a.tokens), n = (tail ? a.tokens : paged_offset(a.cu_steps, s + 1, 0, a.tokens)) - offset;
    const int64_t row_first = (slot - paged_first_slot(static_cast<int64_t>(offset) * group, s, kBlockRows, 1)) * kBlockRows;
    const int64_t seq_rows = static_cast<int64_t>(n) * group;
    if (n <= 0 || row_first < 0 || row_first >= seq_rows) return;
    const int row0 = static_cast<int>(row_first), rows = static_cast<int>(min(seq_rows, rows_all));
    const int given = tail ? 0 : a.lengths[s], length = paged_length(given, a.width, a.page_shift);
    // keys that a row sees: up to its token's position
    auto visible = [&](int row) {
        const int64_t v = static_cast<int64_t>(given) - n + row / group + 1;
        return tail ? 0 : static_cast<int>(v < 0 ? 0 : (v > length ? length : v));
    };
    const int last_row = min(rows, row0 + kBlockRows) - 1;
    const int tiles = (visible(last_row) + kTile - 1) / kTile;
    const int w0 = row0 + 32 * wave, my_row = min(w0 + r, rows - 1);
    const int limit = visible(my_row);
    const int wave_end = w0 < rows ? visible(min(rows, w0 + 32) - 1) : 0, wave_full = visible(min(w0, rows - 1));   // keys that some / all rows of the wave see
    const int32_t* table = a.table + static_cast<size_t>(tail ? 0 : s) * a.table_stride;
    const size_t head_bytes = static_cast<size_t>(D) << a.page_shift;
    const int page_mask = (1 << a.page_shift) - 1;

    // staging: a thread's pieces of 16 codes of the tile's keys and values
    uint4 kraw[kLoads], vraw[kLoads];
    float vscale[kLoads], factor = 0.0f;
    bool missing = false;
    auto fetch = [&](int t) {
        const int j0 = kTile * t;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int e = tid + kThreads * i, key = e / (D / 16), piece = e % (D / 16);
            const int page = paged_page(table, min(j0 + key, length - 1), a.width, a.page_shift, a.pool);
            const uint8_t* src = a.key_pages + (static_cast<size_t>(max(page, 0)) * a.kv_heads + kvh) * head_bytes + ((j0 + key) & page_mask) * D + 16 * piece;
            kraw[i] = *reinterpret_cast<const uint4*>(src);
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int e = tid + kThreads * i, d = e >> 2, chunk = e & 3, first = j0 + 16 * chunk;
            const int page = first < length ? paged_page(table, first, a.width, a.page_shift, a.pool) : -1;
            const size_t at = static_cast<size_t>(max(page, 0)) * a.kv_heads + kvh;
            vraw[i] = *reinterpret_cast<const uint4*>(a.value_pages + at * head_bytes + (static_cast<size_t>(d) << a.page_shift) + (first & page_mask));
            vscale[i] = page >= 0 ? 0.5f * a.value_scales[at] : 1.0f;
            if (i == 0) { factor = page >= 0 ? a.key_scales[at] * a.scale : 0.0f; missing = page < 0; }
        }
    };
    auto store = [&](int t, int buf, int* noted) {
        unsigned char* kt = smem + buf * kTileBytes;
        unsigned char* vt = kt + kKeyBytes;
        const int j0 = kTile * t;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int e = tid + kThreads * i, key = e / (D / 16), piece = e % (D / 16), turn = key & (D / 8 - 1);
            unsigned char* row = kt + key * (2 * D);
            *reinterpret_cast<uint4*>(row + (((2 * piece) ^ turn) << 4)) = half_from_codes<BF16>(kraw[i].x, kraw[i].y, 1.0f);
            *reinterpret_cast<uint4*>(row + (((2 * piece + 1) ^ turn) << 4)) = half_from_codes<BF16>(kraw[i].z, kraw[i].w, 1.0f);
        }
        bool nan = false;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int e = tid + kThreads * i, d = e >> 2, chunk = e & 3, turn = (d >> 1) & 7;
            if (j0 + kTile > length || missing) {                             // what lies behind the last key may be anything, NaN codes too
                const int stored = missing ? 0 : length - j0 - 16 * chunk;
                vraw[i].x &= first_bytes(stored); vraw[i].y &= first_bytes(stored - 4); vraw[i].z &= first_bytes(stored - 8); vraw[i].w &= first_bytes(stored - 12);
            }
            nan |= any_nan_code(vraw[i].x) | any_nan_code(vraw[i].y) | any_nan_code(vraw[i].z) | any_nan_code(vraw[i].w);
            unsigned char* row = vt + d * (2 * kTile);
            *reinterpret_cast<uint4*>(row + (((2 * chunk) ^ turn) << 4)) = half_from_codes<BF16>(vraw[i].x, vraw[i].z, vscale[i]);
            *reinterpret_cast<uint4*>(row + (((2 * chunk + 1) ^ turn) << 4)) = half_from_codes<BF16>(vraw[i].y, vraw[i].w, vscale[i]);
        }
        if (tid < 4) factors[buf][tid] = factor;
        if (nan) atomicOr(noted, 16);
        if (tid < 4 && missing) atomicOr(noted, 1 << tid);
    };
    if (tid < 3) notes[tid] = 0;
    if (tiles > 0) fetch(0);
    uint4 qf[D / 16];
    float late = 1.0f;
    {
        const uint16_t* q = a.q + (static_cast<size_t>(offset) + my_row / group) * a.q_stride + (kvh * group + my_row % group) * D + 8 * h;
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            qf[i] = *reinterpret_cast<const uint4*>(q + 16 * i);
            float v[8];
            half_eight<BF16>(qf[i], v);
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(v[j]));
        }
        // bf16 queries so large that products with codes could pass the largest float, where the scaled score need not: a power of two off, on again behind
        if constexpr (BF16) {
            if (__any(top >= 0x1p60f)) {
                late = 0x1p64f;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    float v[8];
                    half_eight<true>(qf[i], v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] *= 0x1p-64f;
                    qf[i] = half_pack<true>(v);
                }
            }
        }
    }
    const v16f zero = {};
    v16f o[kDimTiles];
#pragma unroll
    for (int i = 0; i < kDimTiles; ++i) o[i] = zero;
    float m = -FLT_MAX, l = 0.0f;                                             // of the lane's query; l over its half of the keys
    __syncthreads();
    if (tiles > 0) store(0, 0, &notes[0]);
    if (tiles > 1) fetch(1);
    __syncthreads();
    for (int t = 0, now = 0; t < tiles; ++t) {
        const int buf = t & 1, j0 = kTile * t, next = now == 2 ? 0 : now + 1;
        if (tid == 0) notes[next == 2 ? 0 : next + 1] = 0;                    // read before the last barrier, written behind the next
        const unsigned char* kt = smem + buf * kTileBytes;
        const unsigned char* vt = kt + kKeyBytes;
        const bool active = j0 < wave_end;
        uint4 p[4];
        int seen = 0, note = 0;
        if (active) {
            v16f sc[2];
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint4 kf = *reinterpret_cast<const uint4*>(kt + (32 * u + r) * (2 * D) + (((2 * i + h) ^ (r & (D / 8 - 1))) << 4));
                    sc[u] = half_mfma32<BF16>(kf, qf[i], i == 0 ? zero : sc[u]);
                }
            const float4 f4 = *reinterpret_cast<const float4*>(factors[buf]);
            const float f[4] = {f4.x, f4.y, f4.z, f4.w};
            note = notes[now];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int v = 0; v < 16; ++v) sc[u][v] *= f[2 * u + (v >> 3)];
            if (BF16 && late != 1.0f)
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int v = 0; v < 16; ++v) sc[u][v] *= late;
            if (j0 + kTile > wave_full || (note & 15)) {                      // keys behind a query, or without a page
                seen = limit - j0 - 4 * h;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int v = 0; v < 16; ++v)
                        if (32 * u + 8 * (v >> 2) + (v & 3) >= seen || ((note >> (2 * u + (v >> 3))) & 1)) sc[u][v] = -INFINITY;
            } else seen = kTile;
            float top = fmaxf(sc[0][0], sc[1][0]);
#pragma unroll
            for (int v = 1; v < 16; ++v) top = fmaxf(top, fmaxf(sc[0][v], sc[1][v]));
            float x, y;
            swapped_pair<32>(top, x, y);
            const float m_new = fmaxf(m, fmaxf(x, y));
            if (__any(m_new > m)) {
                const float back = __builtin_amdgcn_exp2f(m - m_new);
                l *= back;
#pragma unroll
                for (int i = 0; i < kDimTiles; ++i)
#pragma unroll
                    for (int v = 0; v < 16; ++v) o[i][v] *= back;
                m = m_new;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float e[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = __builtin_amdgcn_exp2f(sc[i >> 1][8 * (i & 1) + j] - m);
                l += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
                p[i] = half_pack<BF16>(e);
            }
        }
        if (t + 1 < tiles) store(t + 1, buf ^ 1, &notes[next]);
        if (t + 2 < tiles) fetch(t + 2);
        if (active) {
            if ((note & 16) && j0 + kTile > wave_full) {
                // NaN values in a tile whose keys not every row sees: counted for the rows that see them, zeros for the product (zero times NaN is NaN)
                uint4 sees[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float e[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) e[j] = 16 * i + 8 * (j >> 2) + (j & 3) < seen ? 1.0f : 0.0f;
                    sees[i] = half_pack<BF16>(e);
                }
#pragma unroll
                for (int u = 0; u < kDimTiles; ++u) {
                    v16f count = zero;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint4 vf = *reinterpret_cast<const uint4*>(vt + (32 * u + r) * (2 * kTile) + (((2 * i + h) ^ ((r >> 1) & 7)) << 4));
                        float e[8], bad[8];
                        half_eight<BF16>(vf, e);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            bad[j] = e[j] != e[j] ? 1.0f : 0.0f;
                            e[j] = e[j] != e[j] ? 0.0f : e[j];
                        }
                        o[u] = half_mfma32<BF16>(half_pack<BF16>(e), p[i], o[u]);
                        count = half_mfma32<BF16>(half_pack<BF16>(bad), sees[i], count);
                    }
#pragma unroll
                    for (int v = 0; v < 16; ++v)
                        if (count[v] > 0.0f) o[u][v] = __uint_as_float(0x7fc00000u);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int u = 0; u < kDimTiles; ++u) {
                        const uint4 vf = *reinterpret_cast<const uint4*>(vt + (32 * u + r) * (2 * kTile) + (((2 * i + h) ^ ((r >> 1) & 7)) << 4));
                        o[u] = half_mfma32<BF16>(vf, p[i], o[u]);
                    }
            }
        }
        __syncthreads();                                                      // the next tile is there, this one has been read
        now = next;
    }
    float x, y;
    swapped_pair<32>(l, x, y);
    const float den = x + y, inv = den == 0.0f ? 0.0f : 2.0f / den;           // (twice: the values went in halved)
    // lane: query r, dimensions 32 u + 8 (v / 4) + 4 h + v % 4; through the wave's own part of LDS to whole rows
    __syncthreads();
    unsigned char* turn = smem + wave * (32 * 2 * D);
#pragma unroll
    for (int u = 0; u < kDimTiles; ++u)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<uint2*>(turn + r * (2 * D) + (((4 * u + g) ^ (r & (D / 8 - 1))) << 4) + 8 * h) =
                make_uint2(half_pair<BF16>(o[u][4 * g] * inv, o[u][4 * g + 1] * inv), half_pair<BF16>(o[u][4 * g + 2] * inv, o[u][4 * g + 3] * inv));
    __builtin_amdgcn_wave_barrier();                                          // (one wave's LDS operations take effect in order)
    constexpr int kRowPieces = D / 8, kRowsAtOnce = 64 / kRowPieces;
#pragma unroll
    for (int i = 0; i < 32 / kRowsAtOnce; ++i) {
        const int row = kRowsAtOnce * i + lane / kRowPieces, piece = lane % kRowPieces;
        const uint4 v = *reinterpret_cast<const uint4*>(turn + row * (2 * D) + ((piece ^ (row & (D / 8 - 1))) << 4));
        const int at = w0 + row;
        if (at < rows) *reinterpret_cast<uint4*>(a.out + ((static_cast<size_t>(offset) + at / group) * a.heads + kvh * group + at % group) * D + 8 * piece) = v;
    }
}

template <bool BF16, int D>
int launch(const PagedPromptArgs& a, hipStream_t stream) {
    static SmemGrant granted;
    const size_t smem = 2 * 2 * kTile * D * 2;
    // (with the kernel's own kilobyte beside it, 128-wide heads pass 64 KB)
    if (!grant_dynamic_smem(reinterpret_cast<const void*>(paged_prompt_kernel<BF16, D>), smem + 1024, granted)) return PLLM_ERR_LAUNCH;
    hipLaunchKernelGGL((paged_prompt_kernel<BF16, D>), dim3(a.kv_heads, a.slots), dim3(kThreads), smem, stream, a);
    return hipGetLastError() == hipSuccess ? PLLM_OK : PLLM_ERR_LAUNCH;
}

}  // namespace
}  // namespace pllm

extern "C" int pllm_paged_attention_prompt(const void* q, int64_t q_stride, int dtype, const uint8_t* key_pages, const uint8_t* value_pages,
                                           const float* key_scales, const float* value_scales, int64_t pool, int64_t page_tokens,
                                           const int32_t* block_table, int64_t table_stride, int64_t table_width, const int32_t* lengths,
                                           const int32_t* cu_steps, int64_t tokens, int64_t seqs, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                           float scale, void* out, void* stream) {
    using namespace pllm;
    if (!q || !key_pages || !value_pages || !key_scales || !value_scales || !block_table || !lengths || !cu_steps || !out) return PLLM_ERR_INVALID_ARGUMENT;
    if (dtype != PLLM_F16 && dtype != PLLM_BF16) return PLLM_ERR_INVALID_ARGUMENT;
    if (tokens <= 0 || seqs <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || pool <= 0 || table_width <= 0 || table_stride < table_width ||
        q_stride < heads * head_dim)
        return PLLM_ERR_INVALID_ARGUMENT;
    if ((head_dim != 64 && head_dim != 128) || (page_tokens != 16 && page_tokens != 32 && page_tokens != 64 && page_tokens != 128)) return PLLM_ERR_UNSUPPORTED;
    // pages, positions and rows in 32 bits
    if (tokens > 0x3fffff || seqs > 0xffff || heads > 1024 || pool > 0x7fffffff || table_width > 0x3fffffff / page_tokens) return PLLM_ERR_UNSUPPORTED;
    const int64_t rows = tokens * (heads / kv_heads), slots = paged_slots(rows, static_cast<int>(seqs) + 1, kBlockRows, 1);
    if (rows > 0x3fffffff || slots > 0xffff) return PLLM_ERR_UNSUPPORTED;
    const uintptr_t wide = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(key_pages) | reinterpret_cast<uintptr_t>(value_pages) | reinterpret_cast<uintptr_t>(out);
    const uintptr_t narrow = reinterpret_cast<uintptr_t>(key_scales) | reinterpret_cast<uintptr_t>(value_scales) | reinterpret_cast<uintptr_t>(block_table) |
                             reinterpret_cast<uintptr_t>(lengths) | reinterpret_cast<uintptr_t>(cu_steps);
    if ((wide & 15u) || (narrow & 3u) || q_stride % 8) return PLLM_ERR_INVALID_ARGUMENT;
    PagedPromptArgs a{};
    a.q = static_cast<const uint16_t*>(q); a.q_stride = static_cast<size_t>(q_stride);
    a.key_pages = key_pages; a.value_pages = value_pages; a.key_scales = key_scales; a.value_scales = value_scales;
    a.table = block_table; a.table_stride = static_cast<size_t>(table_stride); a.lengths = lengths; a.cu_steps = cu_steps;
    a.out = static_cast<uint16_t*>(out);
    a.scale = scale * 1.4426950408889634f;
    a.tokens = static_cast<int>(tokens); a.seqs = static_cast<int>(seqs); a.heads = static_cast<int>(heads); a.kv_heads = static_cast<int>(kv_heads);
    a.page_shift = page_tokens == 16 ? 4 : page_tokens == 32 ? 5 : page_tokens == 64 ? 6 : 7;
    a.pool = static_cast<int>(pool); a.width = static_cast<int>(table_width);
    a.slots = static_cast<int>(slots);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (head_dim == 128) return dtype == PLLM_BF16 ? launch<true, 128>(a, st) : launch<false, 128>(a, st);
    return dtype == PLLM_BF16 ? launch<true, 64>(a, st) : launch<false, 64>(a, st);
}
