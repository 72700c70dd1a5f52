// Causal attention of many new tokens per sequence (prompts, their continuations, any mix of lengths) over a paged E4M3 cache that holds their keys
// and values already: out = softmax(scale q K^T) V, every query up to its own position.
//
// A workgroup of eight waves takes 256 query rows of one key/value head, a wave 32 of them; rows are tokens times the heads that share the
// key/value head, so short prompts fill tiles too and keys are fetched once for the whole group.  64 keys at a time: their codes are requested one
// tile ahead into registers, become 16-bit values there (exact) and go to LDS, double-buffered; every wave reads them from there as operands.  The
// wave forms S^T = K Q^T (v_mfma_f32_32x32x16: matrix rows are keys, columns queries), so a lane holds half of one query's scores and what it leaves is,
// rounded to 16 bits, the second operand of O^T = V^T P^T: within 16 keys lane half h holds keys 4 h .. + 3 and 8 + 4 h .. + 3, the words of a piece
// of 16 value codes (tokens innermost in a page) in turn.  The keys' scale, one per 16 keys, goes into the product that takes scores to exponents; the
// values' scale (halved, so that fp16 holds every value that rounds up from its largest) into the conversion.
// 16-byte pieces of a row lie permuted in LDS (key rows by row % 16, value rows by row / 2 % 8), so 16 neighbouring rows read at one piece meet no
// bank twice.  Rows behind the last sequence get zeros.
//
// SPLIT, for calls of few blocks: 128 rows, waves 4 to 7 have those of 0 to 3 and the other 32 keys of every tile, and what they leave meets in LDS at the end.
//
// Bound: 4 D operations per row and key.  8192 tokens of 48 and 8 heads, 825 G operations: 793 us, 1040 T/s, where a large matrix product of the library
// reaches 1155; what is between is the softmax's vector instructions (48 % of the cycles, the matrix unit 47 %: the two waves of a SIMD overlap them in
// part) and the barrier of each tile.
#include "paged_attention.h"
#include "paged_device.h"

#include <algorithm>
#include <cfloat>
#include <type_traits>

namespace pllm {
namespace {

constexpr int kWaves = 8, kThreads = 64 * kWaves, kBlockRows = 32 * kWaves;
constexpr int kTile = 64;                       // keys per step

// Softmax weights are 2^(score - m), m what the row's largest score is compared with.  They are rounded to 16 bits for the second product (matrix instructions on
// float32 have a sixteenth of the rate), and in fp16 a weight below 2^-14 is rounded to a multiple of 2^-24, one below 2^-25 to nothing.  So m stays 2^11 below
// the largest score where it is set and follows when a weight would pass 2^15: what is lost of a weight is 2^-36 of the row's largest at most, of a hundred
// thousand together 2^-19.  (With m at the largest score 32768 keys whose scores are 16.5 below one, to base e, lost an eighth of what they add up to.)  The
// factor is in numerator and denominator alike.  Scores from 2^20 on, whose steps could make more of 11, are compared with themselves.  bf16 has float32's
// range: m is the largest score, and follows from 2^8 on.
template <bool BF16> constexpr float kMostWeight = BF16 ? 8.0f : 15.0f;
template <bool BF16> __device__ __forceinline__ float weights_from(float top) {
    if constexpr (BF16) return top;
    else return fabsf(top) < 0x1p20f ? top - 11.0f : top;
}

struct PagedPromptArgs {
    const uint16_t* q; size_t q_stride;         // elements between tokens
    const uint8_t* key_pages; const uint8_t* value_pages;
    const float* key_scales; const float* value_scales;
    const int32_t* table; size_t table_stride;
    const int32_t* lengths; const int32_t* cu_steps;
    uint16_t* out;
    float* sums; float2* stats;                 // of several runs of a block's keys: [runs][tokens * heads][D], m (base 2) and sum of weights; or null
    float scale;                                // base 2
    int few_rows;                               // sequences of so many query rows or fewer are another kernel's
    int runs, tokens, seqs, heads, kv_heads, page_shift, pool, width, slots;
};

// sum of the lanes up to this one
__device__ __forceinline__ int lanes_until(int x) {
#pragma unroll
    for (int i = 1; i < 64; i *= 2) {
        const int before = __shfl_up(x, i);
        if ((threadIdx.x & 63) >= i) x += before;
    }
    return x;
}

// The block of query rows that index `index` of the grid is: sequence s (a.seqs: the rows behind the last one), rows row0 .. row0 + kBlockRows - 1 of it.
// Those with the most keys come first, so that what is left at the end is short (48 and 8 heads: 30 continuations of up to 200 tokens behind up to 4000
// 267 -> 215 us, 12 of up to 300 behind up to 16000 809 -> 693; where a sequence's own order is as good already, four prompts of up to 2000 tokens, 117 -> 123); of
// more than 63 sequences only each one's own blocks are in that order.
template <int ROWS>
__device__ __forceinline__ bool find_block(const PagedPromptArgs& a, int index, int group, int& s, int& row0) {
    const int lane = threadIdx.x & 63;
    if (a.seqs == 1) {                                                        // (1024 tokens of 48 and 8 heads: 42.0 -> 40.5 us)
        const int n = paged_offset(a.cu_steps, 1, 0, a.tokens), blocks = n * group > a.few_rows ? (n * group + ROWS - 1) / ROWS : 0;
        s = index < blocks ? 0 : 1;
        row0 = (index < blocks ? blocks - 1 - index : index - blocks) * ROWS;
        return row0 < (s ? a.tokens - n : n) * group;
    }
    if (a.seqs < 64) {
        int rows = 0, first = 0, keys = 0;                                    // of the lane's sequence
        if (lane <= a.seqs) {
            const int offset = paged_offset(a.cu_steps, lane, 0, a.tokens);
            const int n = max((lane == a.seqs ? a.tokens : paged_offset(a.cu_steps, lane + 1, 0, a.tokens)) - offset, 0);
            keys = lane == a.seqs || n == 0 ? 0 : paged_length(a.lengths[lane], a.width, a.page_shift);
            rows = lane < a.seqs && n * group <= a.few_rows ? 0 : n * group;
            first = keys - n;
        }
        // (counts stay far below 2^24)
        auto seeing = [&](int tiles) { return paged_blocks_seeing(tiles, rows, first, group, ROWS); };
        auto all = [&](int count) { return static_cast<int>(group_sum<64>(static_cast<float>(count))); };
        if (index >= all(seeing(0))) return false;
        int low = 0, high = static_cast<int>(group_max<64>(static_cast<float>((keys + kTile - 1) / kTile))) + 1;
        while (low < high) {                                                  // the most tiles that more than `index` blocks see
            const int middle = (low + high + 1) / 2;
            if (all(seeing(middle)) > index) low = middle;
            else high = middle - 1;
        }
        const int mine = seeing(low) - seeing(low + 1), place = index - all(seeing(low + 1));
        const int until = lanes_until(mine);                                  // blocks of this length of the sequences up to the lane's
        const uint64_t behind = __ballot(until > place);
        s = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<unsigned long long>(behind)) - 1);
        const int block = (rows + ROWS - 1) / ROWS - seeing(low) + place - (until - mine);
        row0 = __builtin_amdgcn_readlane(block, s) * ROWS;
        return true;
    }
    int place = index;
    for (int base = 0; base <= a.seqs; base += 64) {
        const int c = base + lane;
        int rows = 0;
        if (c <= a.seqs) rows = max((c == a.seqs ? a.tokens : paged_offset(a.cu_steps, c + 1, 0, a.tokens)) - paged_offset(a.cu_steps, c, 0, a.tokens), 0) * group;
        const int blocks = c < a.seqs && rows <= a.few_rows ? 0 : (rows + ROWS - 1) / ROWS, until = lanes_until(blocks);
        const uint64_t behind = __ballot(until > place);
        if (behind) {
            const int owner = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<unsigned long long>(behind)) - 1);
            s = base + owner;
            row0 = __builtin_amdgcn_readlane(until - 1 - place, owner) * ROWS;
            return true;
        }
        place -= __builtin_amdgcn_readlane(until, 63);
    }
    return false;
}

template <bool BF16, int D, bool RUNS, bool SPLIT>
__global__ __launch_bounds__(kThreads, 2) void paged_prompt_kernel(const PagedPromptArgs a) {
    constexpr int kKeyBytes = kTile * D * 2, kTileBytes = 2 * kKeyBytes;      // keys [64][D], values [D][64]
    constexpr int kDimTiles = D / 32, kSteps = D / 16;
    constexpr int kRows = SPLIT ? kBlockRows / 2 : kBlockRows, kSets = SPLIT ? 1 : 2;         // of a workgroup; 32 keys of a tile that a wave takes
    extern __shared__ __align__(1024) unsigned char smem[];                   // [2][kTileBytes]
    __shared__ __align__(16) float factors[4][8];                             // of tile t at t % 4: per chunk the keys' scale times `scale`, and 0 or -inf
    __shared__ int nan_values[4];                                             // of tile t at t % 4 (masked tiles): some value code is NaN,
    __shared__ float unread[64 + 4 * 8];
    __shared__ float2 halves[SPLIT ? kBlockRows / 2 : 1];
    __shared__ __align__(8) uint16_t nan_keys[2][D][4];                       // which ones: a bit per key and dimension, in the tile's half
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int place = SPLIT ? wave & 3 : wave, second = SPLIT ? wave >> 2 : 0;                // the wave's rows, the half of a tile's keys
    const int kvh = blockIdx.x, group = a.heads / a.kv_heads;
    // rows of one key/value head: token * group + head in the group; the tokens behind the last sequence are one more, without keys
    int s = 0, row0 = 0;
    if (!find_block<kRows>(a, blockIdx.z, group, s, row0)) return;
    const bool tail = s == a.seqs;
    const int offset = paged_offset(a.cu_steps, s, 0, a.tokens), n = (tail ? a.tokens : paged_offset(a.cu_steps, s + 1, 0, a.tokens)) - offset;
    const int rows = n * group;                                               // (fits: the host's check)
    const int given = tail ? 0 : a.lengths[s], length = paged_length(given, a.width, a.page_shift);
    // keys that a row sees: up to its token's position
    auto visible = [&](int row) {
        const int64_t v = static_cast<int64_t>(given) - n + row / group + 1;
        return tail ? 0 : static_cast<int>(v < 0 ? 0 : (v > length ? length : v));
    };
    const int all_tiles = (visible(min(rows, row0 + kRows) - 1) + kTile - 1) / kTile;
    // this workgroup's tiles: t0 .. end - 1
    const int run = RUNS ? (all_tiles + static_cast<int>(gridDim.y) - 1) / static_cast<int>(gridDim.y) : all_tiles, t0 = RUNS ? min(static_cast<int>(blockIdx.y) * run, all_tiles) : 0;
    const int end = RUNS ? min(t0 + run, all_tiles) : all_tiles, tiles = end - t0;
    const int full = visible(row0) / kTile;                                   // tiles that every row of the workgroup sees whole
    const int w0 = row0 + 32 * place, my_row = min(w0 + r, rows - 1);
    const int limit = visible(my_row);
    const int wave_end = w0 < rows ? visible(min(rows, w0 + 32) - 1) : 0;     // keys that one of the wave's rows sees
    const int32_t* table = a.table + static_cast<size_t>(tail ? 0 : s) * a.table_stride;

    uint4 qf[kSteps];
    float late = 1.0f;
    {
        const uint16_t* q = a.q + (static_cast<size_t>(offset) + my_row / group) * a.q_stride + (kvh * group + my_row % group) * D + 8 * h;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) qf[i] = *reinterpret_cast<const uint4*>(q + 16 * i);
    }

    // Staging: a lane copies 16 codes of a tile's keys and 16 of its values, of 64-wide heads the one or the other.  All of a wave's are of one chunk of
    // 16 keys, so the page and the scales are the wave's.
    const int chunk = wave >> 1, part = wave & 1;
    const bool copies_keys = D == 128 || part == 0, copies_values = D == 128 || part == 1;
    const int piece = D == 128 ? 64 * part + lane : lane;                     // of the chunk
    const int key_row = 16 * chunk + piece / (D / 16), key_piece = piece % (D / 16), value_row = piece;
    const uint32_t key_lane = static_cast<uint32_t>((key_row & 15) * D + 16 * key_piece), value_lane = static_cast<uint32_t>(value_row) << a.page_shift;
    const int page_mask = (1 << a.page_shift) - 1;
    const size_t head_bytes = static_cast<size_t>(D) << a.page_shift;
    struct Place { size_t at; bool here; };                                   // number of a page and head in the pool; whether the table has one
    auto first_key = [&](int t) { return kTile * t + 16 * chunk; };
    auto entry = [&](int t) { return table[min(first_key(t) >> a.page_shift, a.width - 1)]; };            // the wave's page of tile t, unchecked
    auto checked = [&](int t, int page) {
        page = __builtin_amdgcn_readfirstlane(page);
        const bool here = page >= 0 && page < a.pool && first_key(t) < length;     // (no branch: the step is one block)
        return Place{static_cast<size_t>(here ? page : 0) * a.kv_heads + kvh, here};
    };
    auto load_keys = [&](int t, const Place& p) { return *reinterpret_cast<const uint4*>(a.key_pages + p.at * head_bytes + (first_key(t) & page_mask) * D + key_lane); };
    auto load_values = [&](int t, const Place& p) { return *reinterpret_cast<const uint4*>(a.value_pages + p.at * head_bytes + (first_key(t) & page_mask) + value_lane); };
    // (one lane writes the factors; the others have a place of their own to write to, which costs less than a branch)
    float* const factor_at = lane == 0 && part == 0 ? &factors[0][chunk] : &unread[lane];
    unsigned char* const key_dst = smem + key_row * (2 * D);
    unsigned char* const value_dst = smem + kKeyBytes + value_row * (2 * kTile);
    const int key_turn = key_row & (D / 8 - 1), value_turn = (value_row >> 1) & 7;
    auto blank = [](uint4 raw, bool here) {
        const uint32_t keep = here ? 0xffffffffu : 0u;
        return make_uint4(raw.x & keep, raw.y & keep, raw.z & keep, raw.w & keep);
    };
    // `half`: the tile's place in LDS, the first in the first half
    auto store_keys = [&](int t, int half, bool here, uint4 raw, float key_scale) {
        if (copies_keys) {
            raw = blank(raw, here);                                           // (NaN codes would outlive the minus infinity below)
            unsigned char* row = key_dst + half * kTileBytes;
            *reinterpret_cast<uint4*>(row + (((2 * key_piece) ^ key_turn) << 4)) = half_from_codes<BF16>(raw.x, raw.y, 1.0f);
            *reinterpret_cast<uint4*>(row + (((2 * key_piece + 1) ^ key_turn) << 4)) = half_from_codes<BF16>(raw.z, raw.w, 1.0f);
        }
        // a chunk without a page: any finite factor, and minus infinity behind it
        factor_at[8 * (t & 3)] = here ? fminf(key_scale * a.scale * late, FLT_MAX) : 1.0f;
        factor_at[8 * (t & 3) + 4] = here ? 0.0f : -INFINITY;
    };
    // PLAIN: a tile that every row sees whole
    auto store_values = [&](auto plain, int t, int half, bool here, uint4 raw, float value_scale) {
        if (!copies_values) return;
        raw = blank(raw, here);
        if constexpr (!decltype(plain)::value) {
            const int stored = length - first_key(t);                         // what lies behind the last key may be anything, NaN codes too
            raw.x &= first_bytes(stored); raw.y &= first_bytes(stored - 4); raw.z &= first_bytes(stored - 8); raw.w &= first_bytes(stored - 12);
            if (t >= full) {                                                  // a key that not every row sees: no NaN into the product, zero times NaN is NaN
                const uint32_t bits = nan_codes(raw.x) | (nan_codes(raw.y) << 4) | (nan_codes(raw.z) << 8) | (nan_codes(raw.w) << 12);
                nan_keys[half][value_row][chunk] = static_cast<uint16_t>(bits);
                if (bits) nan_values[t & 3] = 1;
                raw.x = without_nan(raw.x); raw.y = without_nan(raw.y); raw.z = without_nan(raw.z); raw.w = without_nan(raw.w);
            }
        }
        const float scale = here ? 0.5f * value_scale : 1.0f;
        unsigned char* row = value_dst + half * kTileBytes;
        *reinterpret_cast<uint4*>(row + (((2 * chunk) ^ value_turn) << 4)) = half_from_codes<BF16>(raw.x, raw.z, scale);
        *reinterpret_cast<uint4*>(row + (((2 * chunk + 1) ^ value_turn) << 4)) = half_from_codes<BF16>(raw.y, raw.w, scale);
    };

    const v16f zero = {};
    v16f o[kDimTiles], sa[kSets], sb[kSets];
#pragma unroll
    for (int i = 0; i < kDimTiles; ++i) o[i] = zero;
    float m = -FLT_MAX, l = 0.0f;                                             // of the lane's query, as weights_from has it; l over its half of the keys
    // S^T of the tile in one half of LDS
    auto scores = [&](int half, v16f (&sc)[kSets]) {
        const unsigned char* kt = smem + half * kTileBytes + 32 * second * (2 * D);
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int u = 0; u < kSets; ++u) {
                const uint4 kf = *reinterpret_cast<const uint4*>(kt + (32 * u + r) * (2 * D) + (((2 * i + h) ^ (r & (D / 8 - 1))) << 4));
                sc[u] = half_mfma32<BF16>(kf, qf[i], i == 0 ? zero : sc[u]);
            }
    };

    // the largest score of the lane's row, in the exponent's units
    auto row_top = [&](const v16f (&sc)[kSets], const float (&f)[2 * kSets], const float (&b)[2 * kSets]) {
        float most = -INFINITY;
#pragma unroll
        for (int c = 0; c < 2 * kSets; ++c) {
            // (a maximum that hands NaN on takes three operands in one instruction and needs no quieting of them; a NaN score is its row's end either way)
            float x = sc[c >> 1][8 * (c & 1)];
#pragma unroll
            for (int i = 1; i < 8; ++i) x = __builtin_elementwise_maximum(x, sc[c >> 1][8 * (c & 1) + i]);
            most = __builtin_elementwise_maximum(most, __builtin_fmaf(x, f[c], b[c]));
        }
        float lower, upper;
        swapped_pair<32>(most, lower, upper);
        return __builtin_elementwise_maximum(lower, upper);
    };
    auto load_factors = [&](int t, float (&f)[2 * kSets], float (&b)[2 * kSets]) {
        if constexpr (SPLIT) {
            const float2 f2 = *reinterpret_cast<const float2*>(factors[t & 3] + 2 * second), b2 = *reinterpret_cast<const float2*>(factors[t & 3] + 4 + 2 * second);
            f[0] = f2.x; f[1] = f2.y;
            b[0] = b2.x; b[1] = b2.y;
        } else {
            const float4 f4 = *reinterpret_cast<const float4*>(factors[t & 3]), b4 = *reinterpret_cast<const float4*>(factors[t & 3] + 4);
            f[0] = f4.x; f[1] = f4.y; f[2] = f4.z; f[3] = f4.w;
            b[0] = b4.x; b[1] = b4.y; b[2] = b4.z; b[3] = b4.w;
        }
    };
    float f[2 * kSets] = {}, b[2 * kSets] = {}, top = -INFINITY;                              // of the tile whose scores are there

    // what is on its way: codes of keys two tiles ahead of the products, of values one, page numbers and scales ahead of them
    uint4 key_raw, value_raw;
    bool values_here = false;                                                 // of value_raw's tile
    Place keys_at{0, false}, next_at{0, false};                               // of key_raw's tile, of the one behind
    int entry_next = 0;                                                       // of the one behind that
    float key_scale = 0.0f, value_scale = 0.0f, value_scale_keys = 0.0f;      // of key_raw's tile; of value_raw's; of key_raw's tile again
    const int last = end - 1;
    if (tiles > 0) {
        if (tid < 4) nan_values[tid] = 0;
        const int t1 = min(t0 + 1, last), t2 = min(t0 + 2, last), t3 = min(t0 + 3, last), t4 = min(t0 + 4, last);
        const int e0 = entry(t0), e1 = entry(t1), e2 = entry(t2), e3 = entry(t3);
        const Place p0 = checked(t0, e0), p1 = checked(t1, e1);
        keys_at = checked(t2, e2);
        next_at = checked(t3, e3);
        values_here = p1.here;
        const uint4 k0 = load_keys(t0, p0), v0 = load_values(t0, p0), k1 = load_keys(t1, p1);
        const float ks0 = a.key_scales[p0.at], vs0 = a.value_scales[p0.at], ks1 = a.key_scales[p1.at];
        value_scale = a.value_scales[p1.at];
        key_scale = a.key_scales[keys_at.at];
        value_scale_keys = a.value_scales[keys_at.at];
        key_raw = load_keys(t2, keys_at);
        value_raw = load_values(t1, p1);
        entry_next = entry(t4);
        // bf16 queries so large that products with codes could pass the largest float, where the scaled score need not: a power of two off, on again behind
        if constexpr (BF16) {
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                float v[8];
                half_eight<true>(qf[i], v);
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(v[j]));
            }
            // (all waves alike: the factors are the workgroup's)
            if (__syncthreads_or(top >= 0x1p60f)) {
                late = 0x1p64f;
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    float v[8];
                    half_eight<true>(qf[i], v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] *= 0x1p-64f;
                    qf[i] = half_pack<true>(v);
                }
            }
        } else __syncthreads();
        store_keys(t0, 0, p0.here, k0, ks0);
        store_values(std::false_type{}, t0, 0, p0.here, v0, vs0);
        store_keys(t0 + 1, 1, p1.here, k1, ks1);                                  // (one tile only: the same again, in the other half)
        __syncthreads();
        scores(0, sa);
        load_factors(t0, f, b);
        top = row_top(sa, f, b);
    }

    // One tile: its softmax weights beside the next tile's scores, its value product beside the copies of the tiles behind.
    // MASKED: some row does not see all of it; PLAIN: every row sees all of the next.
    auto step = [&](auto masked, auto plain, int t, int half, v16f (&cur)[kSets], v16f (&next)[kSets]) {
        constexpr bool MASKED = decltype(masked)::value, PLAIN = decltype(plain)::value;
        // the copies: keys two tiles ahead take the place of this tile's, values of the next tile that of the one before (behind the last tile: its
        // codes again, which nobody reads)
        auto copies = [&]() {
            if (!PLAIN && tid == 0) nan_values[(t + 2) & 3] = 0;              // read two steps ago, written in the next
            store_keys(t + 2, half, keys_at.here, key_raw, key_scale);
            store_values(plain, t + 1, half ^ 1, values_here, value_raw, value_scale);
            value_raw = load_values(min(t + 2, last), keys_at);
            key_raw = load_keys(min(t + 3, last), next_at);
            key_scale = a.key_scales[next_at.at];
            value_scale = value_scale_keys;
            value_scale_keys = a.value_scales[next_at.at];
            values_here = keys_at.here;
            keys_at = next_at;
            next_at = checked(min(t + 4, last), entry_next);
            entry_next = entry(min(t + 5, last));
        };
        const int seen = limit - kTile * t - 32 * second - 4 * h;
        auto hidden = [&](int u, int v) { return MASKED && 32 * u + 8 * (v >> 2) + (v & 3) >= seen; };
        if constexpr (MASKED) {
            top = -INFINITY;
#pragma unroll
            for (int u = 0; u < kSets; ++u)
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const float x = __builtin_fmaf(cur[u][v], f[2 * u + (v >> 3)], b[2 * u + (v >> 3)]);
                    top = __builtin_elementwise_maximum(top, hidden(u, v) ? -INFINITY : x);
                }
            float lower, upper;
            swapped_pair<32>(top, lower, upper);
            top = __builtin_elementwise_maximum(lower, upper);
        }
        // The maximum follows when a row's weights would pass their most: what it is exactly falls out of the quotient.  (By the difference, which neighbours
        // have exactly: from 2^27 on m + 8 may be the next float, m + 16, and a weight of 2^16 is fp16's infinity.)
        const bool follows = top - m > kMostWeight<BF16>;
        if (__any(follows)) {
            const float m_new = follows ? weights_from<BF16>(top) : m, back = __builtin_amdgcn_exp2f(m - m_new);
            l *= back;
#pragma unroll
            for (int i = 0; i < kDimTiles; ++i)
#pragma unroll
                for (int v = 0; v < 16; ++v) o[i][v] *= back;
            m = m_new;
        }
        // The fused product below keeps the bits that the maximum's rounding lost: up to 2^-25 of it, the same factor in every weight of a
        // row, but past the exponent's range from 2^31 on.  Scores that far out are multiplied and rounded first.
        if (__any(fabsf(m) > 0x1p20f)) {
#pragma unroll
            for (int u = 0; u < kSets; ++u)
#pragma unroll
                for (int v = 0; v < 16; ++v) cur[u][v] = __builtin_fmaf(cur[u][v], f[2 * u + (v >> 3)], b[2 * u + (v >> 3)]);
#pragma unroll
            for (int c = 0; c < 2 * kSets; ++c) { f[c] = 1.0f; b[c] = 0.0f; }
        }
        copies();
        scores(half ^ 1, next);
        uint4 p[2 * kSets];
#pragma unroll
        for (int c = 0; c < 2 * kSets; ++c) {
            float e[8];
            const float behind = b[c] - m;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int v = 8 * (c & 1) + j;
                const float x = __builtin_fmaf(cur[c >> 1][v], f[c], behind);
                e[j] = __builtin_amdgcn_exp2f(hidden(c >> 1, v) ? -INFINITY : x);
            }
            p[c] = half_pack<BF16>(e);
            l = half_pair_sum<BF16>(p[c].x, half_pair_sum<BF16>(p[c].y, half_pair_sum<BF16>(p[c].z, half_pair_sum<BF16>(p[c].w, l))));
        }
        load_factors(t + 1, f, b);
        const unsigned char* vt = smem + half * kTileBytes + kKeyBytes;
        auto value_piece = [&](int u, int c) { return *reinterpret_cast<const uint4*>(vt + (32 * u + r) * (2 * kTile) + (((4 * second + 2 * c + h) ^ ((r >> 1) & 7)) << 4)); };
        if (!MASKED || kTile * t + 32 * second < wave_end) {
#pragma unroll
            for (int c = 0; c < 2 * kSets; ++c)
#pragma unroll
                for (int u = 0; u < kDimTiles; ++u) o[u] = half_mfma32<BF16>(value_piece(u, c), p[c], o[u]);
        }
        top = row_top(next, f, b);
        if constexpr (!MASKED) {
            // the order that this stretch is issued in: operands a few instructions ahead, a share of the exponentials behind every matrix instruction
            __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
            for (int i = 0; i < kSets * kSteps; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
            }
#pragma unroll
            for (int i = 0; i < 2 * kSets * kDimTiles; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
            }
        }
        if (MASKED && nan_values[t & 3]) {
            // NaN values were left out of the product: they are the end of the sums of the rows that see them
            const int keys = limit - kTile * t;
            const uint64_t sees = keys >= 64 ? ~0ull : (keys <= 0 ? 0ull : (1ull << keys) - 1);
#pragma unroll
            for (int u = 0; u < kDimTiles; ++u)
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    if (*reinterpret_cast<const uint64_t*>(nan_keys[half][32 * u + 8 * (v >> 2) + 4 * h + (v & 3)]) & sees) o[u][v] = __uint_as_float(0x7fc00000u);
        }
        __syncthreads();
    };
    int t = t0;
    const std::true_type yes;
    const std::false_type no;
    for (; t + 3 <= min(full, end); t += 2) {                                 // (both steps copy values of tiles that every row sees whole)
        step(no, yes, t, 0, sa, sb);
        step(no, yes, t + 1, 1, sb, sa);
    }
    auto swap = [&]() {
#pragma unroll
        for (int u = 0; u < kSets; ++u) sa[u] = sb[u];
    };
    for (; t < min(full, end); ++t) {                                         // (four prompts of up to 2000 tokens, 32 and 8 heads of 64: 64.4 -> 61.5 us)
        step(no, no, t, (t - t0) & 1, sa, sb);
        swap();
    }
    for (; t < end; ++t) {
        step(yes, no, t, (t - t0) & 1, sa, sb);
        swap();
    }
    float lower, upper;
    swapped_pair<32>(l, lower, upper);
    float den = lower + upper;
    if constexpr (SPLIT) {
        // the two halves of the keys together, lane by lane
        float4* other = reinterpret_cast<float4*>(smem + place * (32 * D * 4)) + lane;
        if (second) {
            if (h == 0) halves[32 * place + r] = make_float2(m, den);
#pragma unroll
            for (int u = 0; u < kDimTiles; ++u)
#pragma unroll
                for (int g = 0; g < 4; ++g) other[64 * (4 * u + g)] = make_float4(o[u][4 * g], o[u][4 * g + 1], o[u][4 * g + 2], o[u][4 * g + 3]);
        }
        __syncthreads();
        if (second) return;
        const float2 theirs = halves[32 * place + r];
        const float most = fmaxf(m, theirs.x), mine_by = __builtin_amdgcn_exp2f(m - most), theirs_by = __builtin_amdgcn_exp2f(theirs.x - most);
        den = __builtin_fmaf(den, mine_by, theirs.y * theirs_by);
        m = most;
#pragma unroll
        for (int u = 0; u < kDimTiles; ++u)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 x = other[64 * (4 * u + g)];
                const float with[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) o[u][4 * g + i] = __builtin_fmaf(o[u][4 * g + i], mine_by, with[i] * theirs_by);
            }
    }
    if constexpr (RUNS) {
        // one of several runs of the block's keys: sums and statistics as they are, for the kernel that brings them together
        if (w0 + r < rows) {
            const size_t row = (static_cast<size_t>(blockIdx.y) * a.tokens + offset + my_row / group) * a.heads + kvh * group + my_row % group;
            if (h == 0) a.stats[row] = make_float2(m, den);
#pragma unroll
            for (int u = 0; u < kDimTiles; ++u)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *reinterpret_cast<float4*>(a.sums + row * D + 32 * u + 8 * g + 4 * h) = make_float4(o[u][4 * g], o[u][4 * g + 1], o[u][4 * g + 2], o[u][4 * g + 3]);
        }
        return;
    }
    const float inv = den == 0.0f ? 0.0f : 2.0f / den;                        // (twice: the values went in halved)
    // lane: query r, dimensions 32 u + 8 (v / 4) + 4 h + v % 4; through the wave's own part of LDS to whole rows
    unsigned char* turn = smem + place * (32 * D * (SPLIT ? 4 : 2));
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

// A wave per query row: its runs together, in their order.
template <bool BF16, int D>
__global__ __launch_bounds__(256) void paged_prompt_merge_kernel(const PagedPromptArgs a) {
    constexpr int kPer = D / 64, kBatch = 8;
    const int64_t rows = static_cast<int64_t>(a.tokens) * a.heads, row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= rows) return;
    if (a.few_rows > 0) {                                                     // rows without runs are the other kernel's
        const int s = paged_sequence(a.cu_steps, a.tokens, a.seqs + 1, 1, 0, row / a.heads);
        if (s < a.seqs && (paged_offset(a.cu_steps, s + 1, 0, a.tokens) - paged_offset(a.cu_steps, s, 0, a.tokens)) * (a.heads / a.kv_heads) <= a.few_rows) return;
    }
    const float2 mine = lane < a.runs ? a.stats[lane * rows + row] : make_float2(-FLT_MAX, 0.0f);           // (at most 64 runs)
    const float top = group_max<64>(mine.x), factor = __builtin_amdgcn_exp2f(mine.x - top), den = group_sum<64>(mine.y * factor);
    float total[kPer] = {};
    for (int i0 = 0; i0 < a.runs; i0 += kBatch) {
        float v[kBatch][kPer];
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
#pragma unroll
            for (int j = 0; j < kPer; ++j) v[i][j] = a.sums[(min(i0 + i, a.runs - 1) * rows + row) * D + kPer * lane + j];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (i0 + i >= a.runs) break;
            const float f = __shfl(factor, i0 + i);
#pragma unroll
            for (int j = 0; j < kPer; ++j) total[j] = __builtin_fmaf(v[i][j], f, total[j]);
        }
    }
    const float inv = den == 0.0f ? 0.0f : 2.0f / den;
    uint16_t* out = a.out + row * D + kPer * lane;
    if constexpr (kPer == 2) *reinterpret_cast<uint32_t*>(out) = half_pair<BF16>(total[0] * inv, total[1] * inv);
    else *out = static_cast<uint16_t>(half_pair<BF16>(total[0] * inv, 0.0f));
}

template <bool BF16, int D>
int launch(const PagedPromptArgs& a, bool split, hipStream_t stream) {
    static SmemGrant granted[4];
    const size_t smem = 2 * 2 * kTile * D * 2;
    const bool runs = a.sums != nullptr;
    const auto kernel = runs ? (split ? paged_prompt_kernel<BF16, D, true, true> : paged_prompt_kernel<BF16, D, true, false>)
                             : (split ? paged_prompt_kernel<BF16, D, false, true> : paged_prompt_kernel<BF16, D, false, false>);
    // (with the kernel's own arrays beside it, 128-wide heads pass 64 KB)
    if (!grant_dynamic_smem(reinterpret_cast<const void*>(kernel), smem + 8192, granted[2 * runs + split])) return PLLM_ERR_LAUNCH;
    // Runs before blocks: indexes without a block come last.  Workgroups go to the shader engines in turn, those that end at once too, and an engine that got more
    // of the others than it has compute units works a second round (128 tokens behind 30000 positions in blocks of half the rows 213 -> 117 us).
    hipLaunchKernelGGL(kernel, dim3(a.kv_heads, a.runs, a.slots), dim3(kThreads), smem, stream, a);
    if (hipGetLastError() != hipSuccess) return PLLM_ERR_LAUNCH;
    if (a.sums) {
        const int64_t rows = static_cast<int64_t>(a.tokens) * a.heads;
        hipLaunchKernelGGL((paged_prompt_merge_kernel<BF16, D>), dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(256), 0, stream, a);
        if (hipGetLastError() != hipSuccess) return PLLM_ERR_LAUNCH;
    }
    return PLLM_OK;
}

// Blocks of so many query rows that the sequences of a call can have: whole ones, and a last one of every sequence with more than `few` rows.
int64_t blocks_of(int64_t rows, int64_t seqs, int64_t few, int block_rows) {
    return seqs == 1 ? (rows + block_rows - 1) / block_rows : rows / block_rows + std::min(seqs, rows / (few + 1));
}

// Runs that the keys of so many blocks and heads are cut in: as many as give every compute unit a workgroup when there are few rows before a long context (one
// workgroup more than that costs a second round), none of them shorter than 4 tiles of a sequence that fills the table.
int prompt_runs(int64_t blocks, int64_t positions) {
    const int64_t runs = std::min(std::min(compute_units() / std::max(blocks, int64_t{1}), positions / (4 * kTile)), int64_t{64});
    return static_cast<int>(std::max(runs, int64_t{1}));
}

// Query rows up to which a sequence goes to the kernel of the decode steps, whose tiles have 16 or 32 rows where these have 256, and which cuts every
// sequence's keys by its own length (48 and 8 heads: 64 single tokens behind up to 8000 positions 434 -> 131 us, 142 times one or two behind up to 3000
// 377 -> 133; 64 and 8 heads, 8 times 8 tokens behind up to 8000 86 -> 52).  Its launches cost a few microseconds where no sequence is so short (30
// continuations of up to 200 tokens behind up to 4000 209 -> 215 us, six prompts 319 -> 323): 16 rows or one token's, unless most
// sequences must be short.  Of one sequence by the rows of the call, so that one kernel's launches are enough; not where what the rows would keep between
// two launches passes a gigabyte.  Where tables are no wider than one of its runs, only if most sequences have 16 rows at most and their blocks here would pass half the
// compute units (64 single tokens behind up to 900 positions 58 -> 18.6 us, behind 100 23.7 -> 9.9, 142 of one or two 115 -> 36; but eight of up to three 17.7 -> 25.8), or
// all of them together are few (four of one or two 15.7 -> 11.3).
int few_rows(int64_t tokens, int64_t seqs, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t positions) {
    const int64_t group = heads / kv_heads, all = tokens * group, least = std::max<int64_t>(group, 16);
    if (group > kPagedFewRows) return 0;
    int64_t rows;
    if (positions > kPagedOneRun) rows = seqs == 1 && all > kPagedFewRows ? 0 : (all <= 2 * kPagedFewRows * seqs ? kPagedFewRows : least);
    else if (seqs == 1) rows = 0;
    else rows = all <= kPagedFewRows ? all : (all <= least * seqs && 2 * seqs * kv_heads > compute_units() ? least : 0);
    rows = std::min(rows, all);
    while (rows > 0 && paged_decode_parts_bytes(seqs, rows, kv_heads, head_dim, positions) > (size_t{1} << 30)) rows /= 2;
    return rows < group ? 0 : static_cast<int>(rows);
}

struct Parts { int runs, few; bool split; size_t run_bytes, few_bytes; };
Parts parts_of(int64_t tokens, int64_t seqs, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t positions) {
    Parts p{};
    const int64_t rows = tokens * (heads / kv_heads);
    p.few = few_rows(tokens, seqs, heads, kv_heads, head_dim, positions);
    p.few_bytes = p.few > 0 ? paged_decode_parts_bytes(seqs, p.few, kv_heads, head_dim, positions) : 0;
    // Half the rows per workgroup while the workgroups are not more than the compute units, and of one prompt without a past, whose last rows see so much more
    // than the mean, up to twice as many (48 and 8 heads, 200 tokens 19.3 -> 14.0 us, 700 31.0 -> 24.5, 1024 42.2 -> 36.2, 1365 52 -> 46, but 1700 60 -> 71; 8 of
    // up to 300 of 32 and 8 heads 23.3 -> 26.9): every tile's codes become 16-bit values for half as many rows.  In runs too (8 and 8 heads, 128 tokens behind
    // 16000 positions 59 -> 34, 300 behind 2000 38 -> 26), but not where whole blocks' runs fill the machine and are long (48 and 8 heads, 128 behind 30000 109 / 117).
    const bool alone = seqs == 1 && positions <= 2 * tokens;
    const int64_t whole = blocks_of(rows, seqs, p.few, kBlockRows) * kv_heads, half = blocks_of(rows, seqs, p.few, kBlockRows / 2) * kv_heads;
    const int whole_runs = prompt_runs(whole, positions);
    p.split = half <= (alone ? 2 : 1) * compute_units() && (whole_runs == 1 || positions < 32 * kTile * whole_runs);
    p.runs = rows <= p.few ? 1 : (p.split ? prompt_runs(half, positions) : whole_runs);
    if (alone && p.runs == 2) p.runs = 1;                                     // (the second launch: 1024 tokens of 16 and 8 heads 32.0 -> 26.4)
    const size_t parts = static_cast<size_t>(p.runs) * tokens * heads;
    p.run_bytes = p.runs > 1 ? align256(parts * head_dim * sizeof(float)) + align256(parts * sizeof(float2)) : 0;
    return p;
}

}  // namespace
}  // namespace pllm

extern "C" {

size_t pllm_paged_attention_prompt_workspace_bytes(int64_t tokens, int64_t seqs, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t positions) {
    if (tokens <= 0 || seqs <= 0 || kv_heads <= 0 || heads < kv_heads || head_dim <= 0 || positions <= 0 || tokens > 0x3fffff || seqs > 0xffff || heads > 1024 || head_dim > 256)
        return 0;
    const pllm::Parts p = pllm::parts_of(tokens, seqs, heads, kv_heads, head_dim, positions);
    return p.run_bytes + p.few_bytes;
}

int pllm_paged_attention_prompt(const void* q, int64_t q_stride, int dtype, const uint8_t* key_pages, const uint8_t* value_pages,
                                           const float* key_scales, const float* value_scales, int64_t pool, int64_t page_tokens,
                                           const int32_t* block_table, int64_t table_stride, int64_t table_width, const int32_t* lengths,
                                           const int32_t* cu_steps, int64_t tokens, int64_t seqs, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                           float scale, void* out, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace pllm;
    if (!q || !key_pages || !value_pages || !key_scales || !value_scales || !block_table || !lengths || !cu_steps || !out) return PLLM_ERR_INVALID_ARGUMENT;
    if (dtype != PLLM_F16 && dtype != PLLM_BF16) return PLLM_ERR_INVALID_ARGUMENT;
    if (tokens <= 0 || seqs <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || pool <= 0 || table_width <= 0 || table_stride < table_width ||
        q_stride < heads * head_dim || !(scale >= 0.0f && scale <= 0x1p127f))
        return PLLM_ERR_INVALID_ARGUMENT;
    if ((head_dim != 64 && head_dim != 128) || (page_tokens != 16 && page_tokens != 32 && page_tokens != 64 && page_tokens != 128)) return PLLM_ERR_UNSUPPORTED;
    // pages, positions and rows in 32 bits
    if (tokens > 0x3fffff || seqs > 0xffff || heads > 1024 || pool > 0x7fffffff || table_width > 0x3fffffff / page_tokens) return PLLM_ERR_UNSUPPORTED;
    const Parts parts = parts_of(tokens, seqs, heads, kv_heads, head_dim, table_width * page_tokens);
    // (the rows behind the last sequence: what is left of the whole blocks, and one more)
    const int64_t rows = tokens * (heads / kv_heads), slots = blocks_of(rows, seqs, parts.few, parts.split ? kBlockRows / 2 : kBlockRows) + 1;
    if (rows > 0x3fffffff || slots > 0xffff) return PLLM_ERR_UNSUPPORTED;
    const uintptr_t wide = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(key_pages) | reinterpret_cast<uintptr_t>(value_pages) | reinterpret_cast<uintptr_t>(out) |
                           reinterpret_cast<uintptr_t>(workspace);
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
    if (parts.run_bytes + parts.few_bytes > 0 && (!workspace || workspace_bytes < parts.run_bytes + parts.few_bytes)) return PLLM_ERR_WORKSPACE;
    a.runs = parts.runs;
    a.few_rows = parts.few;
    if (a.runs > 1) {
        a.sums = static_cast<float*>(workspace);
        a.stats = reinterpret_cast<float2*>(static_cast<unsigned char*>(workspace) + align256(static_cast<size_t>(a.runs) * tokens * heads * head_dim * sizeof(float)));
    }
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool bf16 = dtype == PLLM_BF16;
    const int status = head_dim == 128 ? (bf16 ? launch<true, 128>(a, parts.split, st) : launch<false, 128>(a, parts.split, st)) : (bf16 ? launch<true, 64>(a, parts.split, st) : launch<false, 64>(a, parts.split, st));
    if (status != PLLM_OK || a.few_rows == 0) return status;
    PagedDecodeArgs d{};
    d.q = a.q; d.q_stride = a.q_stride; d.key_pages = key_pages; d.value_pages = value_pages; d.key_scales = key_scales; d.value_scales = value_scales;
    d.table = a.table; d.table_stride = a.table_stride; d.lengths = lengths; d.cu_steps = cu_steps; d.out = a.out; d.scale = a.scale;
    d.seqs = a.seqs; d.tokens = a.tokens; d.heads = a.heads; d.kv_heads = a.kv_heads; d.page_shift = a.page_shift; d.pool = a.pool; d.width = a.width;
    d.part_rows = a.few_rows;
    return paged_decode_launch(d, static_cast<unsigned char*>(workspace) + parts.run_bytes, bf16, static_cast<int>(head_dim), st);
}

}  // extern "C"
