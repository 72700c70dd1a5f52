// One token per row of logits by temperature, top-k, top-p and min-p, from a given random number:
//     w_i = exp((x_i - max x) / T);  the order: x falling, equal ones by rising index
//     kept = the first min(n_k, n_p, n_m) of it: n_k = k, n_p the least n whose first n have p of what the first n_k add up to, n_m those with w >= min_p
//     token = the least i with  sum of w over kept j <= i  >  u * sum of w over kept
// Weights are integers, w * 2^43 rounded: their sums have one value in whatever order they are formed (lanes, slices and atomics change nothing), they are exact, and what
// p, min_p and u are compared with is exact in 128 bits.  A weight is off by 2^-44 at most, so a row of 200064 logits gets the token of exact weights but for about one
// u in 10^9 (float32 weights and sums: one in a hundred).  Weights below 2^-44 are none.
//
// Nothing is sorted but a few hundred values:
//   1. the row's largest value, and about the least
//   2. a histogram over the distance from the largest, linear from it to the least value or to where weights end: values per bin and, without a small top-k, weights
//   3. in it the bins that the cuts of top-k and top-p lie in; the values of these bins to a list, of those above them only the sum of weights.  With a top-k of up
//      to kFew everything above the cut goes to the list, and no other value's weight is ever formed
//   4. the list in order, the cuts in it, the stretch of the row that the token lies in, the token
// Many rows: a workgroup each, one launch.  Few rows: four launches, the first three over slices of the rows.
// Bound: where there is no small top-k, the 64-bit exponential in two passes (about 100 instructions a value in all; the vector units are busy for 60 % of the
// time, the rest is launches, chains of loads and barriers around the cuts, and rows that do not divide among the units): 832 rows of 32000 fp16 logits, all with top-p, 99 us,
// of mixed parameters 70, 96 rows of 200064 in four launches 72, for bytes of 10 and 7.5.  With one, the bytes and, for a single row, the launches one after the other:
// 200064 fp32 logits 21 us (3.0 + 5.4 + 5.8 + 7.6 of the launches).
#include "pllm_device.h"
#include "pllm_internal.h"

#include <algorithm>
#include <cfloat>
#include <type_traits>

namespace pllm {
namespace {

constexpr int kBins = 1024, kListed = 2048;     // bins of a histogram; values of the cuts' bins that a list in LDS holds (equal logits may be more)
constexpr int kTied = 512;                      // values of one part of a bin that are ordered
constexpr int kDirect = 128;                    // listed values up to which each is compared with all
constexpr int kFew = kListed / 2;               // top-k up to which everything that is kept goes to the list
constexpr int kUnit = 43;                       // binary digits of a weight
constexpr int kThreads = 256, kRowThreads = 512, kLastThreads = 512;
constexpr int kAhead = 2;                       // chunks of a thread on their way while as many are worked on
constexpr int kStretch = 512, kMostStretches = (1 << 20) / 4 / kStretch + 1;               // chunks whose kept weights are summed up together; of a row

struct SampleArgs {
    const void* logits; size_t stride;          // elements between rows
    const float* uniform;
    const float* temperature; const int32_t* top_k; const float* top_p; const float* min_p;             // per row, or null: the values below for all
    float temperature_all; int top_k_all; float top_p_all, min_p_all;
    int64_t* tokens;
    uint64_t* best; uint32_t* least;            // [rows][slices]: order key of the largest value, then the complement of its chunk's number; order key of about the least
    uint64_t* masses;                           // [rows][stretches] of what is kept for certain
    uint64_t* mass; uint32_t* count;            // [rows][kBins]
    uint64_t* listed; uint32_t* listed_count;   // [rows][kListed], [rows]: order key and complement of the index
    int rows, vocab, slices, slice_chunks,      // chunks of 16 bytes of a slice, whole stretches
        stretches;
    bool ordered;                               // a workgroup per row, those that take longest first
};

// Logits in the order of their values as unsigned numbers; NaN and minus infinity are 0x007fffff, the least of any.
constexpr uint32_t kNone = 0x007fffffu;
__device__ __forceinline__ uint32_t order_key(float x) {
    if (!(x > -INFINITY)) return kNone;
    const uint32_t b = __float_as_uint(x + 0.0f);                             // (minus zero is zero)
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t key) { return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key); }
__device__ __forceinline__ uint64_t place_key(uint32_t key, int index) { return static_cast<uint64_t>(key) << 32 | static_cast<uint32_t>(~index); }

template <typename T> struct Chunk;             // 16 bytes of logits
template <> struct Chunk<float> {
    static constexpr int kValues = 4;
    static __device__ __forceinline__ float at(const uint4& u, int i) { return __uint_as_float(i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w); }
};
struct F16 {};
struct B16 {};
typedef _Float16 Half2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ Half2 half2_of(uint32_t w) { return __builtin_bit_cast(Half2, w); }
template <> struct Chunk<F16> {
    static constexpr int kValues = 8;
    static __device__ __forceinline__ float at(const uint4& u, int i) {
        const uint32_t w = i < 2 ? u.x : i < 4 ? u.y : i < 6 ? u.z : u.w;
        return f16_bits_to_float(i & 1 ? w >> 16 : w & 0xffffu);
    }
};
template <> struct Chunk<B16> {
    static constexpr int kValues = 8;
    static __device__ __forceinline__ float at(const uint4& u, int i) {
        const uint32_t w = i < 2 ? u.x : i < 4 ? u.y : i < 6 ? u.z : u.w;
        return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
    }
};

// A row as chunks of 16 aligned bytes: value `i` of chunk `c` is logit c * kValues + i - skew.
template <typename T> struct Row {
    static constexpr int kValues = Chunk<T>::kValues, kBytes = 16 / kValues;
    const char* base;
    int skew, vocab;
    __device__ __forceinline__ Row(const SampleArgs& a, int row) {
        base = static_cast<const char*>(a.logits) + static_cast<size_t>(row) * a.stride * kBytes;
        skew = static_cast<int>(reinterpret_cast<uintptr_t>(base) & 15) / kBytes;
        vocab = a.vocab;
    }
    __device__ __forceinline__ int chunks() const { return (vocab + skew + kValues - 1) / kValues; }
    __device__ __forceinline__ int first_of(int c) const { return c * kValues - skew; }
    // the chunk as it lies; places outside the row, and chunks from `end` on, hold NaN
    __device__ __forceinline__ uint4 load(int c, int end) const {
        const int first = first_of(c);
        if (c < end && first >= 0 && first + kValues <= vocab) return *reinterpret_cast<const uint4*>(base + static_cast<int64_t>(first) * kBytes);
        uint32_t w[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
        if (c < end) {
#pragma unroll
            for (int i = 0; i < kValues; ++i) {
                if (first + i < 0 || first + i >= vocab) continue;
                if constexpr (kBytes == 4) w[i] = reinterpret_cast<const uint32_t*>(base)[first + i];
                else {
                    const uint32_t v = reinterpret_cast<const uint16_t*>(base)[first + i];
                    w[i / 2] = i % 2 ? (w[i / 2] & 0xffffu) | v << 16 : (w[i / 2] & 0xffff0000u) | v;
                }
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    // its values, minus infinity for NaN
    static __device__ __forceinline__ void values_of(const uint4& u, float (&v)[kValues]) {
#pragma unroll
        for (int i = 0; i < kValues; ++i) v[i] = fmaxf(Chunk<T>::at(u, i), -INFINITY);
    }
    // The largest of them; the least, minus infinity among them.  (Of float32 after NaN became minus infinity: a maximum hands a signalling NaN on as a quiet one, and the
    // compiler brings two maxima together in one instruction, in which that takes the other value's place.)
    static __device__ __forceinline__ float most_of(const uint4& u) {
        if constexpr (std::is_same_v<T, F16>) {
            const Half2 m = __builtin_elementwise_max(__builtin_elementwise_max(half2_of(u.x), half2_of(u.y)), __builtin_elementwise_max(half2_of(u.z), half2_of(u.w)));
            return fmaxf(static_cast<float>(m[0]), static_cast<float>(m[1]));
        } else {
            float v[kValues];
            values_of(u, v);
            float m = v[0];
#pragma unroll
            for (int i = 1; i < kValues; ++i) m = fmaxf(m, v[i]);
            return m;
        }
    }
    static __device__ __forceinline__ float least_of(const uint4& u) {
        if constexpr (std::is_same_v<T, F16>) {
            const Half2 m = __builtin_elementwise_min(__builtin_elementwise_min(half2_of(u.x), half2_of(u.y)), __builtin_elementwise_min(half2_of(u.z), half2_of(u.w)));
            return fminf(static_cast<float>(m[0]), static_cast<float>(m[1]));
        } else {
            float v[kValues];
            values_of(u, v);
            float m = v[0];
#pragma unroll
            for (int i = 1; i < kValues; ++i) m = fminf(m, v[i]);
            return m;
        }
    }
};
// The next chunks of a thread, every STEP-th, on their way.
template <typename T, int STEP, int COUNT> struct Ahead {
    uint4 u[COUNT];
    __device__ __forceinline__ Ahead(const Row<T>& x, int c0, int end) {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) u[i] = x.load(c0 + i * STEP + static_cast<int>(threadIdx.x), end);
    }
};
// f(number, chunk) for the chunks [begin, end), every STEP-th per thread; `first` are those from `begin` on.  All threads go through all of it: behind the end, chunks of NaN.
template <typename T, int STEP, int COUNT, typename F> __device__ __forceinline__ void for_chunks(const Row<T>& x, Ahead<T, STEP, COUNT> first, int begin, int end, const F& f) {
    for (int c0 = begin; c0 < end; c0 += COUNT * STEP) {
        const Ahead<T, STEP, COUNT> next(x, c0 + COUNT * STEP, end);
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            if (c0 + i * STEP >= end) break;
            f(c0 + i * STEP + static_cast<int>(threadIdx.x), first.u[i]);
        }
        first = next;
    }
}
template <typename T, int STEP, typename F> __device__ __forceinline__ void for_chunks(const Row<T>& x, int begin, int end, const F& f) {
    for_chunks<T, STEP, 1>(x, Ahead<T, STEP, 1>(x, begin, end), begin, end, f);
}

// 2^y, y <= 0 (and above -900: below, anything), times 2^kUnit.  The nearest integer to y falls out of adding 1.5 * 2^52; 2^f for the rest, |f| <= 1/2, by the polynomial
// of degree 10 through it at Chebyshev's points (within 3e-16); the integer goes to the exponent.  Additions and fused products alone, which have four times the rate of
// the instructions that round, convert and scale, and no branches, so that a chunk's values go side by side.  The last digit is set: it stands far behind the point, and no
// weight lies in the middle between two integers, where rounding would go by the sum that it is added to.
__device__ __forceinline__ double exponential(double y) {
    const double shifted = y + 0x1.8p52, f = y - (shifted - 0x1.8p52);
    double p = 7.072585949269223e-09;
    p = __builtin_fma(p, f, 1.0208690299958306e-07);
    p = __builtin_fma(p, f, 1.321544258792169e-06);
    p = __builtin_fma(p, f, 1.5252657260200837e-05);
    p = __builtin_fma(p, f, 0.0001540353044173605);
    p = __builtin_fma(p, f, 0.0013333558230164974);
    p = __builtin_fma(p, f, 0.009618129107606888);
    p = __builtin_fma(p, f, 0.05550410866444772);
    p = __builtin_fma(p, f, 0.24022650695910097);
    p = __builtin_fma(p, f, 0.69314718055995);
    p = __builtin_fma(p, f, 1.0);
    const uint64_t bits = static_cast<uint64_t>(__double_as_longlong(p));
    const uint32_t high = static_cast<uint32_t>(bits >> 32) + ((static_cast<uint32_t>(__double_as_longlong(shifted)) + kUnit) << 20);
    return __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(high) << 32 | static_cast<uint32_t>(bits) | 1));
}
// v, or next to nothing, which adds nothing to a sum of integers.  (A mask on half a number: a choice would become a branch around what is chosen.)
__device__ __forceinline__ double only_if(bool keep, double v) {
    const uint64_t bits = static_cast<uint64_t>(__double_as_longlong(v));
    const uint32_t high = static_cast<uint32_t>(bits >> 32) & (0u - static_cast<uint32_t>(keep));
    return __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(high) << 32 | static_cast<uint32_t>(bits)));
}
// A sum of up to 256 weights begins at 2^52, where a number's last digit is 1: every addition rounds the weight that it adds to an integer, and nothing else.
constexpr double kNoWeight = 0x1p52;
__device__ __forceinline__ uint64_t whole_of(double sum) { return static_cast<uint64_t>(__double_as_longlong(sum)) & 0x000fffffffffffffull; }

// a number of [0, 1) as a 64-bit fraction
__device__ __forceinline__ uint64_t fraction(float v) { return static_cast<uint64_t>(static_cast<double>(v) * 0x1p64); }
__device__ __forceinline__ uint64_t share_up(uint64_t fraction, uint64_t of) {               // the least integer that is not below fraction * of
    return __umul64hi(fraction, of) + (fraction * of != 0);
}

struct Params {
    double factor;                              // base-2 exponent per unit of distance from the largest logit
    float most, per_bin, near;                  // the largest logit; bins per unit of distance (half of it, below); distance behind which weights are none
    uint64_t least_weight;                      // of min_p
    double least_before;                        // of a weight that rounds to no less
    float temperature, top_p;
    int top_k, index_shift;                     // index_shift: binary digits of an index behind the first ten
    bool greedy, cut, few, counts;              // the largest logit is the token; top-k or top-p leave something out; a small top-k; another one
    uint64_t best;
};
// all bits or none: a mask where a choice would be a branch around what is chosen, and a chunk's values would go one after the other
__device__ __forceinline__ uint64_t only(bool v) { return ~(static_cast<uint64_t>(v) - 1); }
// Half the distance from the largest logit, all of which may be more than the largest float.  (Plus infinity as the largest: it has no distance from itself, the others an infinite one;
// a difference that is no number is none.)
__device__ __forceinline__ float distance(const Params& p, float x) { return fmaxf(__builtin_fmaf(x, -0.5f, 0.5f * p.most), 0.0f); }
__device__ __forceinline__ bool weighs(const Params& p, float x) { return distance(p, x) <= p.near; }
__device__ __forceinline__ int bin_of(const Params& p, float x) { return static_cast<int>(fminf(distance(p, x) * p.per_bin, kBins - 1.0f)); }
__device__ __forceinline__ double weight_before(const Params& p, float x) {                   // (anything where x does not weigh)
    return exponential(fmin(static_cast<double>(x) - static_cast<double>(p.most), 0.0) * p.factor);
}
__device__ __forceinline__ uint64_t weight_of(const Params& p, float x) { return whole_of(kNoWeight + only_if(weighs(p, x), weight_before(p, x))); }
// what the caller asks of the row
struct Asked { float temperature, top_p, min_p, uniform; int top_k; };
__device__ __forceinline__ Asked asked_of(const SampleArgs& a, int row) {
    return Asked{a.temperature ? a.temperature[row] : a.temperature_all, a.top_p ? a.top_p[row] : a.top_p_all, a.min_p ? a.min_p[row] : a.min_p_all, a.uniform[row],
                 a.top_k ? a.top_k[row] : a.top_k_all};
}
// one for all lanes, in scalar registers
__device__ __forceinline__ float of_wave(float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); }
__device__ __forceinline__ uint64_t of_wave(uint64_t v) {
    const uint32_t low = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v)), high = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
    return static_cast<uint64_t>(high) << 32 | low;
}
__device__ __forceinline__ double of_wave(double v) { return __longlong_as_double(static_cast<long long>(of_wave(static_cast<uint64_t>(__double_as_longlong(v))))); }
__device__ __forceinline__ int of_wave(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ bool of_wave(bool v) { return __builtin_amdgcn_readfirstlane(v) != 0; }
__device__ __forceinline__ Params of_wave(const Params& p) {
    return Params{of_wave(p.factor), of_wave(p.most), of_wave(p.per_bin), of_wave(p.near), of_wave(p.least_weight), of_wave(p.least_before), of_wave(p.temperature), of_wave(p.top_p),
                  of_wave(p.top_k), of_wave(p.index_shift), of_wave(p.greedy), of_wave(p.cut), of_wave(p.few), of_wave(p.counts), of_wave(p.best)};
}
__device__ __forceinline__ Params params_of(const Asked& asked, int vocab, uint64_t best, uint32_t least);
// the largest and least of a wave's values, for all its lanes: shifts within 16 lanes, then the ends of 16 and of 32 lanes to those behind, then the last lane's
__device__ __forceinline__ void wave_extremes(uint64_t& best, uint32_t& least) {
#define PLLM_STEP(ctrl, rows)                                                                                                                          \
    {                                                                                                                                                  \
        const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(best), ctrl, rows, 0xf, false);                                       \
        const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(best >> 32), ctrl, rows, 0xf, false);                                 \
        const uint64_t b = static_cast<uint64_t>(hi) << 32 | lo;                                                                                       \
        best = b > best ? b : best;                                                                                                                    \
        least = min(least, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(-1, static_cast<int>(least), ctrl, rows, 0xf, false)));                   \
    }
    PLLM_STEP(0x111, 0xf)
    PLLM_STEP(0x112, 0xf)
    PLLM_STEP(0x114, 0xf)
    PLLM_STEP(0x118, 0xf)
    PLLM_STEP(0x142, 0xa)
    PLLM_STEP(0x143, 0xc)
#undef PLLM_STEP
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(best), 63), hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(best >> 32), 63);
    best = static_cast<uint64_t>(hi) << 32 | lo;
    least = __builtin_amdgcn_readlane(least, 63);
}
// the row's parameters, by a wave from what the slices left
__device__ __forceinline__ Params slices_params(const SampleArgs& a, int row, const Asked& asked) {
    const int lane = threadIdx.x & 63;
    uint64_t best = 0;
    uint32_t least = 0xffffffffu;
    for (int i = lane; i < a.slices; i += 64) {
        const uint64_t b = a.best[static_cast<size_t>(row) * a.slices + i];
        best = b > best ? b : best;
        least = min(least, a.least[static_cast<size_t>(row) * a.slices + i]);
    }
    wave_extremes(best, least);
    return params_of(asked, a.vocab, best, least);
}
__device__ __forceinline__ Params params_of(const Asked& asked, int vocab, uint64_t best, uint32_t least) {
    Params p;
    p.best = best;
    p.most = of_key(static_cast<uint32_t>(best >> 32));
    p.temperature = asked.temperature;
    p.top_k = asked.top_k;
    p.top_p = asked.top_p;
    const float min_p = asked.min_p;
    p.least_weight = min_p > 0.0f ? static_cast<uint64_t>(ceil(static_cast<double>(fminf(min_p, 1.0f)) * 0x1p43)) : 0;
    if (p.least_weight == 0) p.least_weight = 1;                              // (weights of nothing are never kept)
    p.least_before = static_cast<double>(p.least_weight) - 0.5;
    p.greedy = !(p.temperature > 0.0f) || p.top_k == 1 || static_cast<uint32_t>(best >> 32) == kNone;
    p.index_shift = max(32 - __clz(vocab) - 10, 0);
    p.few = p.top_k > 0 && p.top_k <= kFew && p.top_k < vocab;
    p.counts = p.top_k > kFew && p.top_k < vocab;
    p.cut = (p.top_k > 0 && p.top_k < vocab) || p.top_p < 1.0f;
    p.factor = 1.44269504088896340736 / static_cast<double>(p.temperature);
    // (weights below 2^-44 are none; in the last step of a float's more)
    p.near = static_cast<float>(fmin(0.5 * (kUnit + 1.5) / p.factor, static_cast<double>(FLT_MAX)));
    const float span = fmaxf(fminf(distance(p, of_key(least)), p.near), FLT_MIN);
    // (Masks can leave next to nothing between the largest value and the least.  Counted in bins of that width what is farther away would be at infinity, in none of them: no
    // bin is so narrow that `near` is not a float number of them.)
    p.per_bin = fminf(fminf(kBins / span, FLT_MAX), 0.5f * FLT_MAX / p.near);
    return of_wave(p);
}

__device__ __forceinline__ void add_to(uint64_t* at, uint64_t v) { atomicAdd(reinterpret_cast<unsigned long long*>(at), static_cast<unsigned long long>(v)); }

// The largest value of the chunks [begin, end), with the complement of its chunk's number, and about the least one: of chunks with masked values their largest, so that a mask
// here and there does not stretch the histogram (whose last bin takes all that is farther away).
template <typename T, int STEP> __device__ __forceinline__ void extremes(const Row<T>& x, int begin, int end, uint64_t& best, uint32_t& least) {
    float most = -INFINITY, low = INFINITY;
    int at = 0x7fffffff;
    for_chunks<T, STEP, kAhead>(x, Ahead<T, STEP, kAhead>(x, begin, end), begin, end, [&](int c, const uint4& u) {
        const float here = Row<T>::most_of(u), lowest = Row<T>::least_of(u);
        const bool larger = here > most;                                      // (a thread's chunks come in their order)
        most = larger ? here : most;
        at = larger ? c : at;
        low = fminf(low, lowest > -INFINITY ? lowest : (here > -INFINITY ? here : INFINITY));
    });
    if (most > -INFINITY) {
        const uint64_t k = place_key(order_key(most), at);
        best = k > best ? k : best;
        least = min(least, order_key(low));
    }
}

// Whether the histogram of a small top-k takes a chunk's largest value alone: where k of them lie, k values do at least, and should there be fewer than k chunks with any value
// that is not masked, the list holds all of them.
template <typename T> __device__ __forceinline__ bool by_chunk(const Params& p) { return p.few && p.top_k <= kListed / Row<T>::kValues; }

// the chunks' values into a histogram in LDS
template <typename T, int STEP> __device__ __forceinline__ void fill(const Row<T>& x, const Ahead<T, STEP, kAhead>& ahead, const Params& p, int begin, int end, uint64_t* mass, uint32_t* count) {
    if (by_chunk<T>(p)) {
        for_chunks<T, STEP, kAhead>(x, ahead, begin, end, [&](int, const uint4& u) {
            const float most = fmaxf(Row<T>::most_of(u), -INFINITY);
            if (weighs(p, most)) atomicAdd(count + bin_of(p, most), 1u);
        });
        return;
    }
    if (p.few) {
        for_chunks<T, STEP, kAhead>(x, ahead, begin, end, [&](int, const uint4& u) {
            float v[Row<T>::kValues];
            Row<T>::values_of(u, v);
            int bin[Row<T>::kValues];
#pragma unroll
            for (int i = 0; i < Row<T>::kValues; ++i) bin[i] = weighs(p, v[i]) ? bin_of(p, v[i]) : -1;
#pragma unroll
            for (int i = 0; i < Row<T>::kValues; ++i)
                if (bin[i] >= 0) atomicAdd(count + bin[i], 1u);
        });
        return;
    }
    for_chunks<T, STEP, kAhead>(x, ahead, begin, end, [&](int, const uint4& u) {
        float v[Row<T>::kValues];
        Row<T>::values_of(u, v);
        uint64_t w[Row<T>::kValues];
#pragma unroll
        for (int i = 0; i < Row<T>::kValues; ++i) w[i] = weight_of(p, v[i]);
#pragma unroll
        for (int i = 0; i < Row<T>::kValues; ++i) asm volatile("" : "+v"(w[i]));              // (formed side by side, not each behind the last one's addition)
#pragma unroll
        for (int i = 0; i < Row<T>::kValues; ++i)
            if (w[i]) {
                const int bin = bin_of(p, v[i]);
                add_to(mass + bin, w[i]);
                if (p.counts) atomicAdd(count + bin, 1u);
            }
    });
}

// the sum over the lanes up to this one: shifts within 16 lanes, then the ends of 16 and of 32 lanes to those behind
__device__ __forceinline__ uint64_t lanes_until(uint64_t v) {
#define PLLM_STEP(ctrl, rows)                                                                                                                          \
    {                                                                                                                                                  \
        const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(v), ctrl, rows, 0xf, false);                                          \
        const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(v >> 32), ctrl, rows, 0xf, false);                                    \
        v += static_cast<uint64_t>(hi) << 32 | lo;                                                                                                     \
    }
    PLLM_STEP(0x111, 0xf)
    PLLM_STEP(0x112, 0xf)
    PLLM_STEP(0x114, 0xf)
    PLLM_STEP(0x118, 0xf)
    PLLM_STEP(0x142, 0xa)
    PLLM_STEP(0x143, 0xc)
#undef PLLM_STEP
    return v;
}
__device__ __forceinline__ uint64_t lanes_sum(uint64_t v) {
    v = lanes_until(v);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(v), 63), hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(v >> 32), 63);
    return static_cast<uint64_t>(hi) << 32 | lo;
}
// A wave's sums of a chunk's weights (64 chunks of one stretch; all lanes take part) to one place in LDS, first together, by halves of 24 binary digits: sums of eight weights
// stay below 2^47, 64 of either half below 2^32, and half as many instructions as with 64 digits are about a sixth of what a chunk takes.
__device__ __forceinline__ void add_all(uint64_t* at, uint64_t v) {
    if (!__any(v != 0)) return;
    uint32_t low = static_cast<uint32_t>(v) & 0xffffffu, high = static_cast<uint32_t>(v >> 24);
#define PLLM_STEP(ctrl, rows)                                                                                                                          \
    low += __builtin_amdgcn_update_dpp(0, low, ctrl, rows, 0xf, false);                                                                                \
    high += __builtin_amdgcn_update_dpp(0, high, ctrl, rows, 0xf, false);
    PLLM_STEP(0x111, 0xf)
    PLLM_STEP(0x112, 0xf)
    PLLM_STEP(0x114, 0xf)
    PLLM_STEP(0x118, 0xf)
    PLLM_STEP(0x142, 0xa)
    PLLM_STEP(0x143, 0xc)
#undef PLLM_STEP
    if ((threadIdx.x & 63) == 63) add_to(at, (static_cast<uint64_t>(high) << 24) + low);
}
// the sum over the threads up to this one, and over all in `total`; `parts` [THREADS / 64]
template <int THREADS> __device__ __forceinline__ uint64_t threads_until(uint64_t v, uint64_t* parts, uint64_t& total) {
    v = lanes_until(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) parts[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        if (w < static_cast<int>(threadIdx.x >> 6)) before += parts[w];
        all += parts[w];
    }
    total = all;
    return before + v;
}
// the sum over the workgroup, for all threads
template <int THREADS> __device__ __forceinline__ uint64_t all_sum(uint64_t v, uint64_t* parts) {
    v = lanes_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) v += parts[w];
    return v;
}

// Where the cuts lie.  Bins below `low` are kept whole (as far as min_p goes), those of [low, high] hold the last one that top-p keeps, bin `last` the k-th.  A
// small top-k: low 0, high and last the k-th's bin.
struct Cuts {
    int low, high, last;                        // last: -1 without a cut by top-k; low: kBins without any cut
    uint64_t before_low, before_last, total;    // sums of weights
    uint32_t need;                              // of bin `last`
};
// A thread's part of a row's histogram.
template <int THREADS> struct Bins {
    static constexpr int kPer = kBins / THREADS;
    uint64_t mass[kPer];
    uint32_t count[kPer];
    __device__ __forceinline__ Bins(const uint64_t* masses, const uint32_t* counts) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) { mass[i] = masses[kPer * threadIdx.x + i]; count[i] = counts[kPer * threadIdx.x + i]; }
    }
};
// By a workgroup, from the row's histogram (whose weights are zero with a small top-k, and values without a top-k).
template <int THREADS>
__device__ __forceinline__ void find_cuts(const Bins<THREADS>& bins, const Params& p, Cuts& out, uint64_t* parts) {
    constexpr int kPer = Bins<THREADS>::kPer;
    const int tid = threadIdx.x;
    const auto& mass = bins.mass;
    const auto& count = bins.count;
    uint64_t masses = 0, counts = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) { masses += mass[i]; counts += count[i]; }
    uint64_t total = 0, everyone;
    const uint64_t mass0 = threads_until<THREADS>(masses, parts, total) - masses;
    const uint64_t count0 = threads_until<THREADS>(counts, parts, everyone) - counts;
    if (tid == 0) { out.low = p.few ? 0 : kBins; out.high = p.few ? kBins - 1 : kBins; out.last = p.few ? kBins - 1 : -1; out.before_low = 0; out.before_last = 0; out.total = total; out.need = 0; }
    __syncthreads();
    const uint64_t k = static_cast<uint64_t>(p.top_k);
    if (p.few ? everyone >= k : p.counts && everyone > k) {
        uint64_t c = count0, m = mass0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if (c < k && c + count[i] >= k) {                                 // (one bin of one thread)
                out.last = kPer * tid + i;
                out.before_last = m;
                out.need = static_cast<uint32_t>(k - c);
                out.total = m + mass[i];                                      // what the first k add up to, at most
                if (p.few) out.high = kPer * tid + i;
            }
            c += count[i];
            m += mass[i];
        }
        __syncthreads();
    }
    if (p.few) return;
    if (p.top_p < 1.0f) {
        const uint64_t f = p.top_p > 0.0f ? fraction(p.top_p) : 0, upper = out.total, lower = out.last >= 0 ? out.before_last + 1 : upper;
        const uint64_t first = share_up(f, lower) > 0 ? share_up(f, lower) : 1, second = share_up(f, upper) > 0 ? share_up(f, upper) : 1;
        uint64_t m = mass0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if (m < first && m + mass[i] >= first) { out.low = kPer * tid + i; out.before_low = m; }
            if (m < second && m + mass[i] >= second) out.high = kPer * tid + i;
            m += mass[i];
        }
    } else if (tid == 0 && out.last >= 0) {
        out.low = out.last;
        out.high = out.last;
        out.before_low = out.before_last;
    }
    __syncthreads();
}

// A chunk's values: those of the cuts' bins to the list in LDS, of those above them the sum of weights.
template <typename T>
__device__ __forceinline__ uint64_t sort_out(const Params& p, const uint4& u, int first, int low, int high, int last, uint64_t* list, uint32_t* listed) {
    float v[Row<T>::kValues];
    if (p.few) {
        const float most = fmaxf(Row<T>::most_of(u), -INFINITY);
        if (weighs(p, most) && bin_of(p, most) <= high) {
            Row<T>::values_of(u, v);
#pragma unroll
            for (int i = 0; i < Row<T>::kValues; ++i)
                if (weighs(p, v[i]) && bin_of(p, v[i]) <= high) {
                    const uint32_t at = atomicAdd(listed, 1u);
                    if (at < kListed) list[at] = place_key(order_key(v[i]), first + i);
                }
        }
        return 0;
    }
    Row<T>::values_of(u, v);
    // (bins as float numbers, whole ones where they are compared with `place`; the last bin has no end)
    const float from = low < kBins ? static_cast<float>(low) : INFINITY, to = high < kBins - 1 ? static_cast<float>(high + 1) : INFINITY;
    const float last_from = last >= 0 ? static_cast<float>(last) : INFINITY, last_to = last < kBins - 1 ? static_cast<float>(last + 1) : INFINITY;
    bool any = false, certain = false;
    bool above[Row<T>::kValues], inside[Row<T>::kValues];
#pragma unroll
    for (int i = 0; i < Row<T>::kValues; ++i) {
        const float d = distance(p, v[i]), place = d * p.per_bin;
        const bool here = d <= p.near;
        above[i] = here && place < from;
        inside[i] = here && ((place >= from && place < to) || (place >= last_from && place < last_to));
        certain |= above[i];
        any |= inside[i];
    }
    double sum = kNoWeight;
    if (certain) {
#pragma unroll
        for (int i = 0; i < Row<T>::kValues; ++i) {
            const double w = weight_before(p, v[i]);
            sum += only_if(above[i] && w >= p.least_before, w);
        }
    }
    if (any)
#pragma unroll
        for (int i = 0; i < Row<T>::kValues; ++i)
            if (inside[i]) {
                const uint32_t at = atomicAdd(listed, 1u);
                if (at < kListed) list[at] = place_key(order_key(v[i]), first + i);
            }
    return whole_of(sum);
}

// Values of LDS in falling order, n a power of two; up to 128 by one wave, without barriers.
template <int THREADS> __device__ __forceinline__ void sort_falling(uint64_t* list, int n) {
    auto stage = [&](int size, int step, int i) {
        const int low = 2 * i - (i & (step - 1)), high = low + step;
        const uint64_t u = list[low], v = list[high];
        if ((u < v) == ((low & size) == 0)) { list[low] = v; list[high] = u; }
    };
    if (n <= 128) {
        if (threadIdx.x < 64)
            for (int size = 2; size <= n; size *= 2)
                for (int step = size / 2; step > 0; step /= 2) {
                    if (static_cast<int>(threadIdx.x) < n / 2) stage(size, step, threadIdx.x);
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    __builtin_amdgcn_wave_barrier();                          // (one wave's LDS operations take effect in order)
                }
        __syncthreads();
        return;
    }
    for (int size = 2; size <= n; size *= 2)
        for (int step = size / 2; step > 0; step /= 2) {
            for (int i = threadIdx.x; i < n / 2; i += THREADS) stage(size, step, i);
            __syncthreads();
        }
}

template <int THREADS> struct Choice {           // LDS of the last step
    uint64_t list[kListed];
    uint64_t sums[kBins];                       // of bins, of parts of a bin, of stretches
    uint64_t few[kTied];
    uint64_t parts[THREADS / 64];
    uint64_t found[3];
    Cuts cuts;
    uint32_t fews;
};
static_assert(kMostStretches <= kBins, "stretches have a place each in sums");

// From sums [n] (n a multiple of THREADS or fewer) the first whose running sum reaches `least`: number and the sum in front of it, for all threads.
template <int THREADS> __device__ __forceinline__ int reach(Choice<THREADS>& s, int n, uint64_t least, uint64_t& before) {
    constexpr int kPer = kBins / THREADS;
    uint64_t v[kPer], mine = 0, total;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int at = kPer * static_cast<int>(threadIdx.x) + i;
        v[i] = at < n ? s.sums[at] : 0;
        mine += v[i];
    }
    uint64_t until = threads_until<THREADS>(mine, s.parts, total) - mine;
    if (until < least && until + mine >= least) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if (until < least && until + v[i] >= least) { s.found[0] = kPer * threadIdx.x + i; s.found[1] = until; }
            until += v[i];
        }
    }
    __syncthreads();
    before = s.found[1];
    return static_cast<int>(s.found[0]);
}

// a value's bin, and its part of it
__device__ __forceinline__ int part_of(const Params& p, float x, int& part) {
    const int bin = bin_of(p, x);
    // (fused by name: left to the compiler, one loop had the product rounded and the other not, and looked for a value in the neighbouring part)
    const float inside = __builtin_fmaf(distance(p, x), p.per_bin, -static_cast<float>(bin));
    part = static_cast<int>(fminf(fmaxf(inside * kBins, 0.0f), kBins - 1.0f));
    return bin;
}
// Of the listed values of a bin, in falling order of their places: the first one at which the sum (of weights, or of ones) reaches `least`.  The bin is cut in kBins parts
// once more; what is left in a part is equal values mostly.
template <int THREADS, typename Weight>
__device__ __forceinline__ uint64_t resolve(Choice<THREADS>& s, const Params& p, int listed, int bin, uint64_t least, const Weight& weight) {
    const int tid = threadIdx.x;
    auto place_of = [&](uint64_t key, int& part) { return part_of(p, of_key(static_cast<uint32_t>(key >> 32)), part); };
    __syncthreads();
    for (int i = tid; i < kBins; i += THREADS) s.sums[i] = 0;
    if (tid == 0) s.fews = 0;
    __syncthreads();
    for (int i = tid; i < listed; i += THREADS) {
        int part;
        if (place_of(s.list[i], part) == bin) add_to(&s.sums[part], weight(s.list[i]));
    }
    __syncthreads();
    uint64_t before;
    const int of = reach<THREADS>(s, kBins, least, before);
    for (int i = tid; i < listed; i += THREADS) {
        int part;
        if (place_of(s.list[i], part) == bin && part == of) {
            const uint32_t at = atomicAdd(&s.fews, 1u);
            if (at < kTied) s.few[at] = s.list[i];
        }
    }
    __syncthreads();
    int n = static_cast<int>(s.fews);
    least -= before;
    if (n > 64) {
        // many of them: of equal ones the stretch of indexes first (bf16 logits, 96 rows of 200064, mixed: the last launch 26 us
        // if they are sorted, 20 so)
        const uint32_t value = static_cast<uint32_t>(s.few[0] >> 32);
        auto in_part = [&](uint64_t key) { int part; return place_of(key, part) == bin && part == of; };
        bool others = false;
        for (int i = tid; i < listed; i += THREADS) others |= static_cast<uint32_t>(s.list[i] >> 32) != value && in_part(s.list[i]);
        if (!__syncthreads_or(others)) {
            auto span = [&](uint64_t key) { return static_cast<int>(~static_cast<uint32_t>(key)) >> p.index_shift; };           // (below kBins, rising where places fall)
            for (int i = tid; i < kBins; i += THREADS) s.sums[i] = 0;
            if (tid == 0) s.fews = 0;
            __syncthreads();
            for (int i = tid; i < listed; i += THREADS)
                if (in_part(s.list[i])) add_to(&s.sums[span(s.list[i])], weight(s.list[i]));
            __syncthreads();
            const int its = reach<THREADS>(s, kBins, least, before);
            for (int i = tid; i < listed; i += THREADS)
                if (in_part(s.list[i]) && span(s.list[i]) == its) {
                    const uint32_t at = atomicAdd(&s.fews, 1u);
                    if (at < kTied) s.few[at] = s.list[i];
                }
            __syncthreads();
            n = static_cast<int>(s.fews);
            least -= before;
        }
        if (n > kTied) return 0;                                              // (no place: the caller goes by the row)
    }
    if (n <= 64) {                                                            // each against all
        const uint64_t mine = tid < n ? s.few[tid] : 0, w = tid < n ? weight(mine) : 0;
        if (tid < 64) s.sums[tid] = w;
        __syncthreads();
        uint64_t sum = 0;
        if (tid < n) {
            for (int i = 0; i < n; ++i) sum += s.sums[i] & only(s.few[i] > mine);
            if (sum < least && sum + w >= least) s.found[2] = mine;
        }
        __syncthreads();
        return s.found[2];
    }
    int size = 128;
    while (size < n) size *= 2;
    for (int i = n + tid; i < size; i += THREADS) s.few[i] = 0;
    __syncthreads();
    sort_falling<THREADS>(s.few, size);
    for (int i = tid; i < kTied; i += THREADS) s.sums[i] = i < n ? weight(s.few[i]) : 0;
    __syncthreads();
    const int at = reach<THREADS>(s, kTied, least, before);
    return s.few[at];
}

// The last step, by a workgroup: the token.  The listed values are in s.list, unordered, `listed` of them (more than the list holds: passes over the row); certain(i) is what is
// kept for certain of stretch i (kStretch chunks).
template <typename T, int THREADS, typename Certain>
__device__ __forceinline__ int64_t choose(const Row<T>& x, const Params& p, Choice<THREADS>& s, int listed, float u, const Certain& certain) {
    constexpr int kValues = Row<T>::kValues;
    const int tid = threadIdx.x, stretches = (x.chunks() + kStretch - 1) / kStretch;
    const uint64_t u_fraction = fraction(u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f), p_fraction = p.top_p > 0.0f ? fraction(p.top_p) : 0;
    const Cuts cuts = s.cuts;
    const bool bounded = p.cut && cuts.low < kBins;
    bool ordered = bounded && listed <= kListed;
    auto weight_key = [&](uint64_t key) { return weight_of(p, of_key(static_cast<uint32_t>(key >> 32))); };
    auto bin_key = [&](uint64_t key) { return bin_of(p, of_key(static_cast<uint32_t>(key >> 32))); };
    auto one = [](uint64_t) { return uint64_t{1}; };
    uint64_t last_kept = 0;                                                   // place key of the last value that is kept
    if (ordered && p.few && listed <= kDirect) {
        // everything that is kept is in a short list: each against all, in the order of the values and in that of the indexes
        constexpr int kAtOnce = 8;                                            // (LDS reads on their way; one after the other 60 values took 4 us)
        const int padded = (listed + kAtOnce - 1) & -kAtOnce;
        uint64_t key = 0, w = 0, before = 0;
        int rank = 0;
        if (tid < padded) {
            key = tid < listed ? s.list[tid] : 0;
            w = tid < listed ? weight_key(key) : 0;
            s.few[tid] = w;
            if (tid >= listed) s.list[tid] = 0;
        }
        __syncthreads();
        for (int i0 = 0; i0 < padded; i0 += kAtOnce) {
            uint64_t other[kAtOnce], its[kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) { other[i] = s.list[i0 + i]; its[i] = s.few[i0 + i]; }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                rank += other[i] > key;
                before += its[i] & only(other[i] > key);
            }
        }
        bool stays = tid < listed && rank < p.top_k;
        const uint64_t all = all_sum<THREADS>(stays ? w : 0, s.parts), share = share_up(p_fraction, all);
        stays &= (!(p.top_p < 1.0f) || rank == 0 || before < share) && w >= p.least_weight;
        const uint64_t total = all_sum<THREADS>(stays ? w : 0, s.parts), target = __umul64hi(u_fraction, total);
        if (tid < padded) s.few[tid] = stays ? w : 0;
        __syncthreads();
        uint64_t sum = 0;
        for (int i0 = 0; i0 < padded; i0 += kAtOnce) {
            uint64_t other[kAtOnce], its[kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) { other[i] = s.list[i0 + i]; its[i] = s.few[i0 + i]; }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) sum += its[i] & only(static_cast<uint32_t>(other[i]) > static_cast<uint32_t>(key));                 // (complements)
        }
        if (stays && sum <= target && sum + w > target) s.found[2] = ~static_cast<uint32_t>(key);
        __syncthreads();
        return static_cast<int64_t>(s.found[2]);
    }
    if (ordered) {
        uint64_t all = cuts.total;                                            // what the first k add up to
        int last = cuts.last;
        uint64_t need = cuts.need;
        if (p.few) {
            // (the histogram may have had the chunks' largest values alone)
            need = 0;
            if (listed > p.top_k) {
                uint64_t before;
                __syncthreads();
                for (int i = tid; i < kBins; i += THREADS) s.sums[i] = 0;
                __syncthreads();
                for (int i = tid; i < listed; i += THREADS) add_to(&s.sums[bin_key(s.list[i])], 1);
                __syncthreads();
                last = reach<THREADS>(s, kBins, p.top_k, before);
                need = p.top_k - before;
            } else {                                                          // all of them: down to the least
                if (tid == 0) s.found[2] = ~uint64_t{0};
                __syncthreads();
                for (int i = tid; i < listed; i += THREADS) atomicMin(reinterpret_cast<unsigned long long*>(&s.found[2]), static_cast<unsigned long long>(s.list[i]));
                __syncthreads();
                last_kept = s.found[2];
            }
        }
        if (last >= 0 && need > 0) {
            last_kept = resolve<THREADS>(s, p, listed, last, need, one);
            ordered = last_kept != 0;
        }
        if (ordered && p.top_p < 1.0f) {
            if (cuts.last >= 0) {
                uint64_t sum = 0;
                for (int i = tid; i < listed; i += THREADS) sum += s.list[i] >= last_kept && (p.few || bin_key(s.list[i]) == cuts.last) ? weight_key(s.list[i]) : 0;
                all = all_sum<THREADS>(sum, s.parts) + cuts.before_last;
            }
            const uint64_t share = share_up(p_fraction, all), least = (share > 0 ? share : 1) - cuts.before_low;
            int bin = cuts.low;
            uint64_t before = 0;
            if (cuts.low != cuts.high) {
                __syncthreads();
                for (int i = tid; i < kBins; i += THREADS) s.sums[i] = 0;
                __syncthreads();
                for (int i = tid; i < listed; i += THREADS) {
                    const int b = bin_key(s.list[i]);
                    if (b <= cuts.high) add_to(&s.sums[b], weight_key(s.list[i]));
                }
                __syncthreads();
                bin = reach<THREADS>(s, kBins, least, before);
            }
            last_kept = resolve<THREADS>(s, p, listed, bin, least - before, weight_key);
            ordered = last_kept != 0;
        }
    }
    if (bounded && !ordered) {
        last_kept = 0;
        // More values at the cuts than the list holds.  Sums go to s.sums by a number per value, below zero for none: neighbours mostly have one, and theirs goes there in one addition.
        auto spread = [&](const auto& number, bool counts) {
            __syncthreads();
            for (int i = tid; i < kBins; i += THREADS) s.sums[i] = 0;
            __syncthreads();
            for_chunks<T, THREADS>(x, 0, x.chunks(), [&](int c, const uint4& u) {
                float v[kValues];
                Row<T>::values_of(u, v);
                uint64_t sum = 0;
                int at = 0;
#pragma unroll
                for (int i = 0; i < kValues; ++i) {
                    const uint64_t w = weight_of(p, v[i]);
                    const int its = w ? number(v[i], x.first_of(c) + i) : -1;
                    if (its < 0) continue;
                    if (sum && its != at) { add_to(&s.sums[at], sum); sum = 0; }
                    at = its;
                    sum += counts ? 1 : w;
                }
                const int first = __builtin_amdgcn_readfirstlane(at);
                if (__ballot(at == first) == ~0ull) {                         // (all 64 lanes)
                    sum = lanes_sum(sum);
                    if (sum && (tid & 63) == 0) add_to(&s.sums[first], sum);
                } else if (sum) add_to(&s.sums[at], sum);
            });
            __syncthreads();
        };
        if (cuts.last < 0 && !p.few) {
            // top-p alone: by the parts of its bin, the values of one of them to the list; if these are too many and equal, as they are in 16 bits, by stretches of their indexes
            // (96 rows of 200064, most values around 12 below the largest: in fp32 322 us, by digits 1320; in bf16 495, by digits 1210)
            const uint64_t share = share_up(p_fraction, cuts.total);
            uint64_t least = (share > 0 ? share : 1) - cuts.before_low, before;
            auto part_in_bin = [&](float value) { int part; return part_of(p, value, part) == cuts.low ? part : -1; };
            auto gather = [&](const auto& taken) {                            // to the list; how many there are
                if (tid == 0) s.fews = 0;
                __syncthreads();
                for_chunks<T, THREADS>(x, 0, x.chunks(), [&](int c, const uint4& u) {
                    float v[kValues];
                    Row<T>::values_of(u, v);
#pragma unroll
                    for (int i = 0; i < kValues; ++i)
                        if (weighs(p, v[i]) && taken(v[i], x.first_of(c) + i)) {
                            const uint32_t at = atomicAdd(&s.fews, 1u);
                            if (at < kListed) s.list[at] = place_key(order_key(v[i]), x.first_of(c) + i);
                        }
                });
                __syncthreads();
                return static_cast<int>(s.fews);
            };
            spread([&](float value, int) { return part_in_bin(value); }, false);
            const int of = reach<THREADS>(s, kBins, least, before);
            least -= before;
            int n = gather([&](float value, int) { return part_in_bin(value) == of; });
            if (n > kListed) {
                const uint32_t key = static_cast<uint32_t>(s.list[0] >> 32);
                bool others = false;
                spread([&](float value, int index) {
                    if (part_in_bin(value) != of) return -1;
                    others |= order_key(value) != key;
                    return index >> p.index_shift;                            // (below kBins, rising where places fall)
                }, false);
                if (!__syncthreads_or(others)) {
                    const int span = reach<THREADS>(s, kBins, least, before);
                    least -= before;
                    n = gather([&](float value, int index) { return order_key(value) == key && index >> p.index_shift == span; });
                }
            }
            if (n <= kListed) last_kept = resolve<THREADS>(s, p, n, cuts.low, least, weight_key);
        }
        // many of them equal: by the digits of their places, from the first on, a pass over the row for each of eight
        auto reached = [&](uint64_t least, bool counts) {                      // the place of the value at which the sum reaches `least`
            uint64_t place = 0;
            for (int shift = 56; shift >= 0; shift -= 8) {
                spread([&](float value, int index) {
                    const uint64_t key = place_key(order_key(value), index);
                    return shift < 56 && (key >> shift >> 8) != (place >> shift >> 8) ? -1 : 255 - static_cast<int>(key >> shift & 255);        // falling
                }, counts);
                uint64_t before;
                const int its = reach<THREADS>(s, 256, least, before);
                least -= before;
                place |= static_cast<uint64_t>(255 - its) << shift;
            }
            return place;
        };
        auto whole = [&](uint64_t from, bool counts) {
            uint64_t sum = 0;
            for_chunks<T, THREADS>(x, 0, x.chunks(), [&](int c, const uint4& u) {
                float v[kValues];
                Row<T>::values_of(u, v);
#pragma unroll
                for (int i = 0; i < kValues; ++i) {
                    const uint64_t w = place_key(order_key(v[i]), x.first_of(c) + i) < from ? 0 : weight_of(p, v[i]);
                    sum += counts ? (w != 0) : w;
                }
            });
            return all_sum<THREADS>(sum, s.parts);
        };
        const bool found = last_kept != 0;
        if (!found && p.top_k > 0 && whole(0, true) > static_cast<uint64_t>(p.top_k)) last_kept = reached(p.top_k, true);
        if (!found && p.top_p < 1.0f) {
            const uint64_t share = share_up(p_fraction, whole(last_kept, false));
            last_kept = reached(share > 0 ? share : 1, false);
        }
    }
    // what is kept of each stretch: for certain, and of the listed values
    auto kept = [&](uint64_t key, uint64_t w) { return key >= last_kept && w >= p.least_weight; };
    __syncthreads();
    for (int i = tid; i < stretches; i += THREADS) s.sums[i] = p.few ? 0 : certain(i);
    __syncthreads();
    if (ordered) {
        for (int i = tid; i < listed; i += THREADS) {
            const uint64_t key = s.list[i], w = weight_key(key);
            if (kept(key, w)) add_to(&s.sums[(static_cast<int>(~static_cast<uint32_t>(key)) + x.skew) / kValues / kStretch], w);
        }
    } else if (bounded) {
        for_chunks<T, THREADS>(x, 0, x.chunks(), [&](int c, const uint4& u) {
            float v[kValues];
            Row<T>::values_of(u, v);
            uint64_t sum = 0;
#pragma unroll
            for (int i = 0; i < kValues; ++i) {
                const uint64_t w = weight_of(p, v[i]);
                if (w && bin_of(p, v[i]) >= cuts.low && kept(place_key(order_key(v[i]), x.first_of(c) + i), w)) sum += w;
            }
            add_all(&s.sums[c / kStretch], sum);
        });
    }
    __syncthreads();
    uint64_t total = 0;
    for (int i = tid; i < stretches; i += THREADS) total += s.sums[i];
    total = all_sum<THREADS>(total, s.parts);
    const uint64_t target = __umul64hi(u_fraction, total);                    // the token's sum is the first above it
    uint64_t before;
    const int stretch = reach<THREADS>(s, stretches, target + 1, before);
    if (ordered && p.few) {
        // everything that is kept is in the list: the stretch's in rising order of their indexes, each against all (a stretch with more is looked at in the row)
        if (tid == 0) s.fews = 0;
        __syncthreads();
        for (int i = tid; i < listed; i += THREADS) {
            const uint64_t key = s.list[i];
            if ((static_cast<int>(~static_cast<uint32_t>(key)) + x.skew) / kValues / kStretch == stretch && kept(key, weight_key(key))) {
                const uint32_t at = atomicAdd(&s.fews, 1u);
                if (at < kTied) s.few[at] = key;
            }
        }
        __syncthreads();
        const int n = static_cast<int>(s.fews);
        if (n <= 64) {
            if (tid < n) {
                const uint64_t mine = s.few[tid];
                uint64_t sum = before;
                for (int i = 0; i < n; ++i) sum += static_cast<uint32_t>(s.few[i]) > static_cast<uint32_t>(mine) ? weight_key(s.few[i]) : 0;      // (complements)
                if (sum <= target && sum + weight_key(mine) > target) s.found[2] = ~static_cast<uint32_t>(mine);
            }
            __syncthreads();
            return static_cast<int64_t>(s.found[2]);
        }
    }
    const int begin = stretch * kStretch, end = min(begin + kStretch, x.chunks());
    for (int c0 = begin; c0 < end; c0 += THREADS) {
        float v[kValues];
        uint64_t w[kValues], own = 0, here;
        Row<T>::values_of(x.load(c0 + tid, end), v);
        const int first = x.first_of(c0 + tid);
#pragma unroll
        for (int i = 0; i < kValues; ++i) {
            w[i] = weight_of(p, v[i]);
            w[i] = kept(place_key(order_key(v[i]), first + i), w[i]) ? w[i] : 0;
            own += w[i];
        }
        uint64_t sum = before + threads_until<THREADS>(own, s.parts, here) - own;
        if (sum <= target && sum + own > target) {
#pragma unroll
            for (int i = 0; i < kValues; ++i) {
                if (sum <= target && sum + w[i] > target) s.found[2] = static_cast<uint64_t>(first + i);
                sum += w[i];
            }
        }
        before += here;
        if (before > target) break;                                           // (all threads alike)
    }
    __syncthreads();
    return static_cast<int64_t>(s.found[2]);
}

// the first of the largest logits, in its chunk
template <typename T> __device__ __forceinline__ int64_t greedy_token(const Row<T>& x, uint64_t best) {
    const uint32_t key = static_cast<uint32_t>(best >> 32);
    if (key == kNone) return -1;
    const int c = static_cast<int>(~static_cast<uint32_t>(best));
    float v[Row<T>::kValues];
    Row<T>::values_of(x.load(c, c + 1), v);
    int at = 0;
#pragma unroll
    for (int i = Row<T>::kValues - 1; i >= 0; --i) at = order_key(v[i]) == key ? i : at;
    return x.first_of(c) + at;
}

// ---- few rows: slices ---------------------------------------------------------------------------------------------------

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_extremes_kernel(const SampleArgs a) {
    __shared__ uint64_t bests[kThreads / 64];
    __shared__ uint32_t leasts[kThreads / 64];
    const int row = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x;
    for (int i = slice * kThreads + tid; i < kBins; i += a.slices * kThreads) {              // for the next launch
        a.mass[static_cast<size_t>(row) * kBins + i] = 0;
        a.count[static_cast<size_t>(row) * kBins + i] = 0;
    }
    if (slice == 0 && tid == 0) a.listed_count[row] = 0;
    const Row<T> x(a, row);
    uint64_t best = place_key(kNone, 0x7fffffff);
    uint32_t least = 0xffffffffu;
    extremes<T, kThreads>(x, slice * a.slice_chunks, min((slice + 1) * a.slice_chunks, x.chunks()), best, least);
    wave_extremes(best, least);
    if ((tid & 63) == 0) { bests[tid >> 6] = best; leasts[tid >> 6] = least; }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kThreads / 64; ++w) {
            best = bests[w] > best ? bests[w] : best;
            least = min(least, leasts[w]);
        }
        a.best[static_cast<size_t>(row) * a.slices + slice] = best;
        a.least[static_cast<size_t>(row) * a.slices + slice] = least;
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_histogram_kernel(const SampleArgs a) {
    __shared__ uint64_t mass[kBins];
    __shared__ uint32_t count[kBins];
    const int row = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x;
    const Row<T> x(a, row);
    const int begin = slice * a.slice_chunks, end = min(begin + a.slice_chunks, x.chunks());
    const Ahead<T, kThreads, kAhead> ahead(x, begin, end);                    // (on their way beside the parameters)
    const Params p = slices_params(a, row, asked_of(a, row));
    if (p.greedy || !p.cut) return;
    for (int i = tid; i < kBins; i += kThreads) { mass[i] = 0; count[i] = 0; }
    __syncthreads();
    fill<T, kThreads>(x, ahead, p, begin, end, mass, count);
    __syncthreads();
    for (int i = tid; i < kBins; i += kThreads) {
        if (mass[i]) add_to(a.mass + static_cast<size_t>(row) * kBins + i, mass[i]);
        if (count[i]) atomicAdd(a.count + static_cast<size_t>(row) * kBins + i, count[i]);
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_masses_kernel(const SampleArgs a) {
    __shared__ uint64_t list[kListed], parts[kThreads / 64], sums[kMostStretches];
    __shared__ Cuts cuts;
    __shared__ uint32_t listed, at;
    const int row = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x;
    const Row<T> x(a, row);
    const int begin = slice * a.slice_chunks, end = min(begin + a.slice_chunks, x.chunks());
    const Bins<kThreads> bins(a.mass + static_cast<size_t>(row) * kBins, a.count + static_cast<size_t>(row) * kBins);
    const Ahead<T, kThreads, kAhead> ahead(x, begin, end);
    const Params p = slices_params(a, row, asked_of(a, row));
    if (p.greedy) return;
    if (tid == 0) listed = 0;
    for (int i = tid; i < kMostStretches; i += kThreads) sums[i] = 0;
    int low = kBins, high = kBins, last = -1;
    if (p.cut) {
        find_cuts<kThreads>(bins, p, cuts, parts);
        low = cuts.low; high = cuts.high; last = cuts.last;
    }
    __syncthreads();
    for_chunks<T, kThreads, kAhead>(x, ahead, begin, end, [&](int c, const uint4& u) {
        const uint64_t sum = sort_out<T>(p, u, x.first_of(c), low, high, last, list, &listed);
        if (!p.few) add_all(&sums[(c - begin) / kStretch], sum);
    });
    __syncthreads();
    const int stretches = (end - begin + kStretch - 1) / kStretch;            // (slices are whole stretches)
    if (!p.few)
        for (int i = tid; i < stretches; i += kThreads) a.masses[static_cast<size_t>(row) * a.stretches + begin / kStretch + i] = sums[i];
    if (listed == 0) return;
    if (tid == 0) at = atomicAdd(a.listed_count + row, listed);               // (more than the list holds is more than that here too)
    __syncthreads();
    for (int i = tid; i < static_cast<int>(min(listed, static_cast<uint32_t>(kListed))); i += kThreads)
        if (at + i < kListed) a.listed[static_cast<size_t>(row) * kListed + at + i] = list[i];
}

template <typename T>
__global__ __launch_bounds__(kLastThreads) void sample_token_kernel(const SampleArgs a) {
    __shared__ Choice<kLastThreads> s;
    const int row = blockIdx.x, tid = threadIdx.x;
    // everything that may be asked for at once: one after the other each takes as long as all of them
    const Asked asked = asked_of(a, row);
    const Bins<kLastThreads> bins(a.mass + static_cast<size_t>(row) * kBins, a.count + static_cast<size_t>(row) * kBins);
    const int in_list = static_cast<int>(a.listed_count[row]);
    uint64_t keys[kListed / kLastThreads];
#pragma unroll
    for (int i = 0; i < kListed / kLastThreads; ++i) keys[i] = a.listed[static_cast<size_t>(row) * kListed + i * kLastThreads + tid];
    const uint64_t mass = a.masses[static_cast<size_t>(row) * a.stretches + min(tid, a.stretches - 1)];
    const Params p = slices_params(a, row, asked);
    if (p.greedy) {
        if (tid == 0) a.tokens[row] = greedy_token(Row<T>(a, row), p.best);
        return;
    }
    int listed = 0;
    if (p.cut) {
        listed = in_list;
#pragma unroll
        for (int i = 0; i < kListed / kLastThreads; ++i) s.list[i * kLastThreads + tid] = keys[i];
        // (the list of a small top-k is cut by itself)
        if (!p.few) find_cuts<kLastThreads>(bins, p, s.cuts, s.parts);
        else if (tid == 0) s.cuts = Cuts{0, kBins - 1, kBins - 1, 0, 0, 0, 0};
    }
    __syncthreads();
    const int64_t token = choose<T, kLastThreads>(Row<T>(a, row), p, s, listed, asked.uniform, [&](int i) { return i == tid ? mass : a.masses[static_cast<size_t>(row) * a.stretches + i]; });
    if (tid == 0) a.tokens[row] = token;
}

// ---- many rows: a workgroup each ----------------------------------------------------------------------------------------

// Where long rows have parameters of their own and there are more of them than compute units, those that take longest come first (no small top-k, then one, then the largest
// logit alone): left in their order a long one may begin when the others end (of 32000, mixed: 832 rows 77 -> 70 us, 1600 110 -> 99; 3000 of 8000 89 -> 90, so not for
// short ones).  Each workgroup finds the row of its place.
constexpr int kOrdered = 8 * kRowThreads;
__device__ __forceinline__ int ordered_row(const SampleArgs& a, uint64_t* parts, int& found) {
    const int tid = threadIdx.x, each = (a.rows + kRowThreads - 1) / kRowThreads, begin = min(tid * each, a.rows), end = min(begin + each, a.rows);
    auto kind = [&](int row) {
        const float temperature = a.temperature ? a.temperature[row] : a.temperature_all;
        const int top_k = a.top_k ? a.top_k[row] : a.top_k_all;
        return !(temperature > 0.0f) || top_k == 1 ? 2 : top_k > 0 && top_k <= kFew ? 1 : 0;
    };
    auto of_kind = [](uint64_t counts, int k) { return static_cast<int>(counts >> (21 * k) & 0x1fffff); };
    uint64_t counts = 0, all;
    if (tid == 0) found = blockIdx.x;                                         // (parameters that change under the call: some row)
    for (int row = begin; row < end; ++row) counts += uint64_t{1} << (21 * kind(row));
    const uint64_t before = threads_until<kRowThreads>(counts, parts, all) - counts;
    int place = blockIdx.x, k = 0;
    while (k < 2 && place >= of_kind(all, k)) place -= of_kind(all, k++);
    place -= of_kind(before, k);
    if (place >= 0 && place < of_kind(counts, k))
        for (int row = begin; row < end; ++row)
            if (kind(row) == k && place-- == 0) found = row;
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(found);
}

template <typename T>
// (three workgroups a compute unit, which costs a few registers kept in memory: 832 rows with top-p 104 -> 99 us)
__global__ __launch_bounds__(kRowThreads, 6) void sample_row_kernel(const SampleArgs a) {
    __shared__ Choice<kRowThreads> s;
    __shared__ uint32_t count[kBins], leasts[kRowThreads / 64], listed;
    __shared__ uint64_t sums[kMostStretches];
    __shared__ int found;
    const int row = a.ordered ? ordered_row(a, s.parts, found) : static_cast<int>(blockIdx.x), tid = threadIdx.x;
    const Row<T> x(a, row);
    const Asked asked = asked_of(a, row);                                     // (on its way beside the row)
    const int chunks = x.chunks();
    uint64_t best = place_key(kNone, 0x7fffffff);
    uint32_t least = 0xffffffffu;
    extremes<T, kRowThreads>(x, 0, chunks, best, least);
    wave_extremes(best, least);
    if ((tid & 63) == 0) { s.parts[tid >> 6] = best; leasts[tid >> 6] = least; }
    if (tid == 0) listed = 0;
    for (int i = tid; i < kBins; i += kRowThreads) { s.sums[i] = 0; count[i] = 0; }
    for (int i = tid; i < kMostStretches; i += kRowThreads) sums[i] = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kRowThreads / 64; ++w) {
        best = s.parts[w] > best ? s.parts[w] : best;
        least = min(least, leasts[w]);
    }
    const Params p = params_of(asked, a.vocab, best, least);
    if (p.greedy) {
        if (tid == 0) a.tokens[row] = greedy_token(x, p.best);
        return;
    }
    int low = kBins, high = kBins, last = -1;
    __syncthreads();
    if (p.cut) {
        fill<T, kRowThreads>(x, Ahead<T, kRowThreads, kAhead>(x, 0, chunks), p, 0, chunks, s.sums, count);
        __syncthreads();
        find_cuts<kRowThreads>(Bins<kRowThreads>(s.sums, count), p, s.cuts, s.parts);
        low = s.cuts.low; high = s.cuts.high; last = s.cuts.last;
    }
    for_chunks<T, kRowThreads, kAhead>(x, Ahead<T, kRowThreads, kAhead>(x, 0, chunks), 0, chunks, [&](int c, const uint4& u) {
        const uint64_t sum = sort_out<T>(p, u, x.first_of(c), low, high, last, s.list, &listed);
        if (!p.few) add_all(&sums[c / kStretch], sum);
    });
    __syncthreads();
    const int64_t token = choose<T, kRowThreads>(x, p, s, static_cast<int>(listed), asked.uniform, [&](int i) { return sums[i]; });
    if (tid == 0) a.tokens[row] = token;
}

template <typename T> int launch(const SampleArgs& a, hipStream_t stream) {
    const dim3 grid(a.slices, a.rows);
    if (a.slices == 0) {
        hipLaunchKernelGGL((sample_row_kernel<T>), dim3(a.rows), dim3(kRowThreads), 0, stream, a);
        return hipGetLastError() == hipSuccess ? PLLM_OK : PLLM_ERR_LAUNCH;
    }
    hipLaunchKernelGGL((sample_extremes_kernel<T>), grid, dim3(kThreads), 0, stream, a);
    const bool cut = a.top_k || a.top_p || (a.top_k_all > 0 && a.top_k_all < a.vocab) || a.top_p_all < 1.0f;
    const bool drawn = (a.temperature || a.temperature_all > 0.0f) && (a.top_k || a.top_k_all != 1);                  // (otherwise every row's largest)
    if (drawn && cut) hipLaunchKernelGGL((sample_histogram_kernel<T>), grid, dim3(kThreads), 0, stream, a);
    if (drawn) hipLaunchKernelGGL((sample_masses_kernel<T>), grid, dim3(kThreads), 0, stream, a);
    hipLaunchKernelGGL((sample_token_kernel<T>), dim3(a.rows), dim3(kLastThreads), 0, stream, a);
    return hipGetLastError() == hipSuccess ? PLLM_OK : PLLM_ERR_LAUNCH;
}

struct Layout { int slices, slice_chunks, stretches; size_t best, least, masses, mass, count, listed, listed_count, bytes; };
Layout layout_of(int64_t rows, int64_t vocab, int dtype) {
    const int values = dtype == PLLM_F32 ? 4 : 8;
    const int64_t chunks = (vocab + 2 * values - 2) / values;                 // (a row may begin inside a chunk)
    // A workgroup per row for rows of a few chunks per thread, and where there are more rows than compute units, if the last of them do not leave too many units idle: otherwise
    // slices, which take a little longer for the same work and 25 us more (top-p, 300 rows of 200064 in slices 199 us, by rows 279; 832 of 32000 about 107 by the same
    // figures, 99).  As many slices as give the machine about eight workgroups per compute unit (four: 96 rows of 200064, mixed, 81 -> 71 us), none of fewer
    // than two chunks per thread.
    Layout l{};
    const int64_t units = compute_units(), rounds = (rows + units - 1) / units;
    if (chunks <= 1024 || (rows >= units && 11 * rows + 10 * 12000000 / vocab > 10 * rounds * units)) {
        l.bytes = 256;
        return l;
    }
    const int64_t stretches = (chunks + kStretch - 1) / kStretch, slices = std::min(stretches, (8 * compute_units() + rows - 1) / rows), each = (stretches + slices - 1) / slices;
    l.stretches = static_cast<int>(stretches);
    l.slice_chunks = static_cast<int>(each * kStretch);
    l.slices = static_cast<int>((stretches + each - 1) / each);
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at += align256(bytes); return here; };
    l.best = take(rows * l.slices * 8);
    l.least = take(rows * l.slices * 4);
    l.masses = take(rows * l.stretches * 8);
    l.mass = take(rows * kBins * 8);
    l.count = take(rows * kBins * 4);
    l.listed = take(rows * kListed * 8);
    l.listed_count = take(rows * 4);
    l.bytes = at;
    return l;
}
bool sizes_ok(int64_t rows, int64_t vocab, int dtype) { return rows > 0 && vocab > 0 && rows <= 0xffff && vocab <= 0x100000 && dtype >= PLLM_F32 && dtype <= PLLM_BF16; }

}  // namespace
}  // namespace pllm

extern "C" {

size_t pllm_sample_tokens_workspace_bytes(int64_t rows, int64_t vocab, int dtype) {
    return pllm::sizes_ok(rows, vocab, dtype) ? pllm::layout_of(rows, vocab, dtype).bytes : 0;
}

int pllm_sample_tokens(const void* logits, int64_t stride, int dtype, const float* uniform, const float* temperature, float temperature_all, const int32_t* top_k,
                       int64_t top_k_all, const float* top_p, float top_p_all, const float* min_p, float min_p_all, int64_t rows, int64_t vocab, int64_t* tokens, void* workspace,
                       size_t workspace_bytes, void* stream) {
    using namespace pllm;
    if (!logits || !uniform || !tokens || rows <= 0 || vocab <= 0 || stride < vocab || dtype < PLLM_F32 || dtype > PLLM_BF16) return PLLM_ERR_INVALID_ARGUMENT;
    if (!sizes_ok(rows, vocab, dtype)) return PLLM_ERR_UNSUPPORTED;
    const uintptr_t words = reinterpret_cast<uintptr_t>(uniform) | reinterpret_cast<uintptr_t>(temperature) | reinterpret_cast<uintptr_t>(top_k) | reinterpret_cast<uintptr_t>(top_p) |
                            reinterpret_cast<uintptr_t>(min_p);
    const uintptr_t value = dtype == PLLM_F32 ? 4 : 2;
    if ((words & 3u) || reinterpret_cast<uintptr_t>(logits) % value || reinterpret_cast<uintptr_t>(tokens) % 8 || reinterpret_cast<uintptr_t>(workspace) % 16) return PLLM_ERR_INVALID_ARGUMENT;
    if ((!temperature && !(temperature_all >= 0.0f)) || (!top_p && !(top_p_all >= 0.0f)) || (!min_p && !(min_p_all >= 0.0f && min_p_all <= 1.0f)) || (!top_k && top_k_all < 0))
        return PLLM_ERR_INVALID_ARGUMENT;
    const Layout l = layout_of(rows, vocab, dtype);
    if (!workspace || workspace_bytes < l.bytes) return PLLM_ERR_WORKSPACE;
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    SampleArgs a{};
    a.logits = logits; a.stride = static_cast<size_t>(stride); a.uniform = uniform;
    a.temperature = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p;
    a.temperature_all = temperature_all; a.top_k_all = static_cast<int>(std::min<int64_t>(top_k_all, 0x7fffffff)); a.top_p_all = top_p_all; a.min_p_all = min_p_all;
    a.tokens = tokens;
    a.best = reinterpret_cast<uint64_t*>(ws + l.best); a.least = reinterpret_cast<uint32_t*>(ws + l.least); a.masses = reinterpret_cast<uint64_t*>(ws + l.masses);
    a.mass = reinterpret_cast<uint64_t*>(ws + l.mass); a.count = reinterpret_cast<uint32_t*>(ws + l.count);
    a.listed = reinterpret_cast<uint64_t*>(ws + l.listed); a.listed_count = reinterpret_cast<uint32_t*>(ws + l.listed_count);
    a.rows = static_cast<int>(rows); a.vocab = static_cast<int>(vocab); a.slices = l.slices; a.slice_chunks = l.slice_chunks; a.stretches = l.stretches;
    a.ordered = l.slices == 0 && (temperature || top_k) && rows > compute_units() && rows <= kOrdered && vocab * static_cast<int64_t>(value) / 16 > 2 * kRowThreads;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == PLLM_F32) return launch<float>(a, st);
    return dtype == PLLM_F16 ? launch<F16>(a, st) : launch<B16>(a, st);
}

}  // extern "C"
