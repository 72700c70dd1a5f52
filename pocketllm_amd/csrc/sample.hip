// One token per row of logits by temperature, top-k, top-p and min-p, from a given random number:
//     w_i = exp((x_i - max x) / T);  the order: x falling, equal ones by rising index
//     kept = the first min(n_k, n_p, n_m) of it: n_k = k, n_p the least n whose first n have p of what the first n_k add up to, n_m those with w >= min_p
//     token = the least i with  sum of w over kept j <= i  >  u * sum of w over kept
// Weights are integers, w * 2^43 rounded: their sums have one value in whatever order they are formed (lanes, slices and atomics change nothing), they are exact, and what
// p, min_p and u are compared with is exact in 128 bits.  A weight is off by 2^-44 at most, so a row of 200064 logits gets the token of exact weights but for about one
// u in 10^9 (float32 weights and sums: one in a hundred).  Weights below 2^-44 are none.
//
// Nothing is sorted but a few hundred values.  A row is cut in slices, a workgroup each:
//   1. the slices' largest and least values
//   2. a histogram over the distance from the largest, linear from it to the least value or to where weights end: count and sum of weights per bin
//   3. every workgroup finds in it the bins that the cuts of top-k and top-p lie in; sums of what is kept for certain per slice; the values of the cuts' bins to a list
//   4. a workgroup per row orders that list, finds the cuts, the slice and in it the token
// Bound: bytes (the row once from memory, then from the caches), the 64-bit exponential (about 20 instructions a value) and the chain of four launches.
#include "pllm_device.h"
#include "pllm_internal.h"

#include <algorithm>
#include <cfloat>

namespace pllm {
namespace {

constexpr int kBins = 2048, kListed = 4096;     // bins of a histogram; values of the cuts' bins that are ordered in LDS (equal logits may be more: by bisection)
constexpr int kUnit = 43;                       // binary digits of a weight
constexpr int kThreads = 256, kLastThreads = 1024;
constexpr uint64_t kOne = uint64_t{1} << kUnit;

struct SampleArgs {
    const void* logits; size_t stride;          // elements between rows
    const float* uniform;
    const float* temperature; const int32_t* top_k; const float* top_p; const float* min_p;             // per row, or null: the values below for all
    float temperature_all; int top_k_all; float top_p_all, min_p_all;
    int64_t* tokens;
    uint64_t* best; uint32_t* least;            // [rows][slices]: order key of the largest value, then the complement of its index; order key of the least
    uint64_t* masses;                           // [rows][slices] of what is kept for certain
    uint64_t* mass; uint32_t* count;            // [rows][kBins]
    uint64_t* listed; uint32_t* listed_count;   // [rows][kListed], [rows]: order key and complement of the index
    int rows, vocab, slices, slice_chunks;      // chunks of 16 bytes of a slice
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
    static __device__ __forceinline__ float one(const void* p, size_t i) { return static_cast<const float*>(p)[i]; }
};
struct F16 {};
struct B16 {};
template <> struct Chunk<F16> {
    static constexpr int kValues = 8;
    static __device__ __forceinline__ float at(const uint4& u, int i) {
        const uint32_t w = i < 2 ? u.x : i < 4 ? u.y : i < 6 ? u.z : u.w;
        return f16_bits_to_float(i & 1 ? w >> 16 : w & 0xffffu);
    }
    static __device__ __forceinline__ float one(const void* p, size_t i) { return f16_bits_to_float(static_cast<const uint16_t*>(p)[i]); }
};
template <> struct Chunk<B16> {
    static constexpr int kValues = 8;
    static __device__ __forceinline__ float at(const uint4& u, int i) {
        const uint32_t w = i < 2 ? u.x : i < 4 ? u.y : i < 6 ? u.z : u.w;
        return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
    }
    static __device__ __forceinline__ float one(const void* p, size_t i) { return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(p)[i]) << 16); }
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
    // the chunk's order keys and the index of its first; places outside the row hold kNone
    __device__ __forceinline__ int keys(int c, uint32_t (&key)[kValues]) const {
        const int first = c * kValues - skew;
        if (first >= 0 && first + kValues <= vocab) {
            const uint4 u = *reinterpret_cast<const uint4*>(base + static_cast<int64_t>(first) * kBytes);
#pragma unroll
            for (int i = 0; i < kValues; ++i) key[i] = order_key(Chunk<T>::at(u, i));
        } else {
#pragma unroll
            for (int i = 0; i < kValues; ++i) key[i] = first + i >= 0 && first + i < vocab ? order_key(Chunk<T>::one(base, first + i)) : kNone;
        }
        return first;
    }
};

// 2^y, y <= 0, times 2^kUnit, rounded: 2^f for |f| <= 1/2 by its series to the eleventh power (the rest is below 7e-15), the exponent added, the fraction
// rounded off by adding 2^52.
__device__ __forceinline__ uint64_t weight_of(double y) {
    if (!(y >= -(kUnit + 1.0))) return 0;
    const double n = rint(y), f = (y - n) * 0.69314718055994530942;
    double p = 1.0 / 39916800.0;
    p = __builtin_fma(p, f, 1.0 / 3628800.0);
    p = __builtin_fma(p, f, 1.0 / 362880.0);
    p = __builtin_fma(p, f, 1.0 / 40320.0);
    p = __builtin_fma(p, f, 1.0 / 5040.0);
    p = __builtin_fma(p, f, 1.0 / 720.0);
    p = __builtin_fma(p, f, 1.0 / 120.0);
    p = __builtin_fma(p, f, 1.0 / 24.0);
    p = __builtin_fma(p, f, 1.0 / 6.0);
    p = __builtin_fma(p, f, 0.5);
    p = __builtin_fma(p, f, 1.0);
    p = __builtin_fma(p, f, 1.0);
    const double scaled = __longlong_as_double(__double_as_longlong(p) + static_cast<long long>(static_cast<int>(n) + kUnit) * (1ll << 52));
    return static_cast<uint64_t>(__double_as_longlong(scaled + 0x1p52)) & 0x000fffffffffffffull;
}

// a number of [0, 1) as a 64-bit fraction
__device__ __forceinline__ uint64_t fraction(float v) { return static_cast<uint64_t>(static_cast<double>(v) * 0x1p64); }
__device__ __forceinline__ uint64_t share_up(uint64_t fraction, uint64_t of) {               // the least integer that is not below fraction * of
    return __umul64hi(fraction, of) + (fraction * of != 0);
}

struct Params {
    double most, factor, per_bin;               // the largest logit; base-2 exponent per unit of distance; bins per unit of it
    uint64_t least_weight;                      // of min_p
    float temperature, top_p;
    int top_k;
    bool greedy, cut;                           // the largest logit is the token; top-k or top-p leave something out
    uint64_t best;
};

// a value's base-2 exponent, zero or below (plus infinity as the largest: the others have minus infinity)
__device__ __forceinline__ double exponent_of(const Params& p, float x) { return x == p.most ? 0.0 : (static_cast<double>(x) - p.most) * p.factor; }
__device__ __forceinline__ int bin_of(const Params& p, double y) { return static_cast<int>(fmin(-y * p.per_bin, kBins - 1.0)); }

// the row's parameters, by a wave from what the slices left
__device__ __forceinline__ Params params_of(const SampleArgs& a, int row) {
    const int lane = threadIdx.x & 63;
    uint64_t best = 0;
    uint32_t least = 0xffffffffu;
    for (int i = lane; i < a.slices; i += 64) {
        const uint64_t b = a.best[static_cast<size_t>(row) * a.slices + i];
        best = b > best ? b : best;
        least = min(least, a.least[static_cast<size_t>(row) * a.slices + i]);
    }
#pragma unroll
    for (int i = 32; i > 0; i /= 2) {
        const uint64_t b = __shfl_xor(static_cast<unsigned long long>(best), i);
        best = b > best ? b : best;
        least = min(least, static_cast<uint32_t>(__shfl_xor(static_cast<int>(least), i)));
    }
    Params p;
    p.best = best;
    p.most = of_key(static_cast<uint32_t>(best >> 32));
    p.temperature = a.temperature ? a.temperature[row] : a.temperature_all;
    p.top_k = a.top_k ? a.top_k[row] : a.top_k_all;
    p.top_p = a.top_p ? a.top_p[row] : a.top_p_all;
    const float min_p = a.min_p ? a.min_p[row] : a.min_p_all;
    p.least_weight = min_p > 0.0f ? static_cast<uint64_t>(ceil(static_cast<double>(fminf(min_p, 1.0f)) * 0x1p43)) : 0;
    if (p.least_weight == 0) p.least_weight = 1;                              // (weights of nothing are never kept)
    p.greedy = !(p.temperature > 0.0f) || p.top_k == 1 || static_cast<uint32_t>(best >> 32) == kNone;
    p.cut = (p.top_k > 0 && p.top_k < a.vocab) || p.top_p < 1.0f;
    p.factor = 1.44269504088896340736 / static_cast<double>(p.temperature);
    const double y = exponent_of(p, of_key(least)), range = fmin(fmax(-y, 0x1p-40), kUnit + 2.0);           // (of values in a row that have weights)
    p.per_bin = kBins / range;
    return p;
}

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
    const int end = min((slice + 1) * a.slice_chunks, x.chunks());
    uint64_t best = place_key(kNone, 0x7fffffff);
    uint32_t least = 0xffffffffu;
    for (int c = slice * a.slice_chunks + tid; c < end; c += kThreads) {
        uint32_t key[Row<T>::kValues];
        const int first = x.keys(c, key);
#pragma unroll
        for (int i = 0; i < Row<T>::kValues; ++i) {
            const uint64_t k = place_key(key[i], first + i);
            if (key[i] != kNone) {
                best = k > best ? k : best;
                least = min(least, key[i]);
            }
        }
    }
#pragma unroll
    for (int i = 32; i > 0; i /= 2) {
        const uint64_t b = __shfl_xor(static_cast<unsigned long long>(best), i);
        best = b > best ? b : best;
        least = min(least, static_cast<uint32_t>(__shfl_xor(static_cast<int>(least), i)));
    }
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
    const Params p = params_of(a, row);
    if (p.greedy || !p.cut) return;
    for (int i = tid; i < kBins; i += kThreads) { mass[i] = 0; count[i] = 0; }
    __syncthreads();
    const Row<T> x(a, row);
    const int end = min((slice + 1) * a.slice_chunks, x.chunks());
    for (int c = slice * a.slice_chunks + tid; c < end; c += kThreads) {
        uint32_t key[Row<T>::kValues];
        x.keys(c, key);
#pragma unroll
        for (int i = 0; i < Row<T>::kValues; ++i) {
            if (key[i] == kNone) continue;
            const double y = exponent_of(p, of_key(key[i]));
            const uint64_t w = weight_of(y);
            if (w == 0) continue;
            const int bin = bin_of(p, y);
            atomicAdd(reinterpret_cast<unsigned long long*>(&mass[bin]), static_cast<unsigned long long>(w));
            atomicAdd(&count[bin], 1u);
        }
    }
    __syncthreads();
    for (int i = tid; i < kBins; i += kThreads)
        if (count[i]) {
            atomicAdd(reinterpret_cast<unsigned long long*>(a.mass + static_cast<size_t>(row) * kBins + i), static_cast<unsigned long long>(mass[i]));
            atomicAdd(a.count + static_cast<size_t>(row) * kBins + i, count[i]);
        }
}

__device__ __forceinline__ uint64_t lanes_until(uint64_t v) {
#pragma unroll
    for (int i = 1; i < 64; i *= 2) {
        const uint64_t before = __shfl_up(static_cast<unsigned long long>(v), i);
        if ((threadIdx.x & 63) >= i) v += before;
    }
    return v;
}
// the sum over the threads up to this one, and over all in `total`; `parts` [THREADS / 64], free again behind the next barrier
template <int THREADS> __device__ __forceinline__ uint64_t threads_until(uint64_t v, uint64_t* parts, uint64_t& total) {
    v = lanes_until(v);
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

// Where the cuts lie.  Bins below `low` are kept whole (as far as min_p goes), those of [low, high] hold the last one that top-p keeps, bin `last` the k-th.
struct Cuts {
    int low, high, last;                        // last: -1 without a cut by top-k; low: kBins without any cut
    uint64_t before_low, before_last, total;    // sums of weights
    uint32_t need;                              // of bin `last`
};
// By a workgroup, from the row's histogram.
template <int THREADS>
__device__ __forceinline__ void find_cuts(const SampleArgs& a, int row, const Params& p, Cuts& out, uint64_t* parts) {
    constexpr int kPer = kBins / THREADS;
    const int tid = threadIdx.x;
    uint64_t mass[kPer], masses = 0;
    uint32_t count[kPer], counts = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        mass[i] = a.mass[static_cast<size_t>(row) * kBins + kPer * tid + i];
        count[i] = a.count[static_cast<size_t>(row) * kBins + kPer * tid + i];
        masses += mass[i];
        counts += count[i];
    }
    uint64_t total, everyone;
    const uint64_t mass0 = threads_until<THREADS>(masses, parts, total) - masses;
    __syncthreads();
    const uint64_t count0 = threads_until<THREADS>(counts, parts, everyone) - counts;
    if (tid == 0) { out.low = kBins; out.high = kBins; out.last = -1; out.before_low = 0; out.before_last = 0; out.total = total; out.need = 0; }
    __syncthreads();
    const uint64_t k = p.top_k > 0 ? static_cast<uint64_t>(p.top_k) : ~uint64_t{0};
    if (everyone > k) {
        uint64_t c = count0, m = mass0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if (c < k && c + count[i] >= k) {                                 // (one bin of one thread)
                out.last = kPer * tid + i;
                out.before_last = m;
                out.need = static_cast<uint32_t>(k - c);
                out.total = m + mass[i];                                      // what the first k add up to, at most
            }
            c += count[i];
            m += mass[i];
        }
        __syncthreads();
    }
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

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_masses_kernel(const SampleArgs a) {
    __shared__ uint64_t parts[kThreads / 64];
    __shared__ Cuts cuts;
    const int row = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x;
    const Params p = params_of(a, row);
    if (p.greedy) return;
    int low = kBins, high = kBins, last = -1;
    if (p.cut) {
        find_cuts<kThreads>(a, row, p, cuts, parts);
        low = cuts.low; high = cuts.high; last = cuts.last;
    }
    const Row<T> x(a, row);
    const int end = min((slice + 1) * a.slice_chunks, x.chunks());
    uint64_t sum = 0;
    for (int c = slice * a.slice_chunks + tid; c < end; c += kThreads) {
        uint32_t key[Row<T>::kValues];
        const int first = x.keys(c, key);
#pragma unroll
        for (int i = 0; i < Row<T>::kValues; ++i) {
            if (key[i] == kNone) continue;
            const double y = exponent_of(p, of_key(key[i]));
            const int bin = bin_of(p, y);
            if (bin > high && bin != last) continue;
            const uint64_t w = weight_of(y);
            if (w == 0) continue;
            if (bin < low) {
                if (w >= p.least_weight) sum += w;
            } else {
                const uint32_t at = atomicAdd(a.listed_count + row, 1u);
                if (at < kListed) a.listed[static_cast<size_t>(row) * kListed + at] = place_key(key[i], first + i);
            }
        }
    }
#pragma unroll
    for (int i = 32; i > 0; i /= 2) sum += __shfl_xor(static_cast<unsigned long long>(sum), i);
    __syncthreads();
    if ((tid & 63) == 0) parts[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) a.masses[static_cast<size_t>(row) * a.slices + slice] = (parts[0] + parts[1]) + (parts[2] + parts[3]);
}

// the sum over the workgroup, for all threads
template <int THREADS> __device__ __forceinline__ void all_sum(uint64_t& v, uint64_t* parts) {
#pragma unroll
    for (int i = 32; i > 0; i /= 2) v += __shfl_xor(static_cast<unsigned long long>(v), i);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < THREADS / 64; ++w) v += parts[w];
}

template <typename T>
__global__ __launch_bounds__(kLastThreads) void sample_token_kernel(const SampleArgs a) {
    constexpr int kPer = kListed / kLastThreads, kValues = Row<T>::kValues;
    __shared__ uint64_t list[kListed];
    __shared__ uint64_t parts[kLastThreads / 64];
    __shared__ Cuts cuts;
    __shared__ uint64_t found[3];
    __shared__ int chosen;
    const int row = blockIdx.x, tid = threadIdx.x;
    const Params p = params_of(a, row);
    if (p.greedy) {
        if (tid == 0) a.tokens[row] = static_cast<uint32_t>(p.best >> 32) == kNone ? -1 : static_cast<int64_t>(~static_cast<uint32_t>(p.best));
        return;
    }
    const Row<T> x(a, row);
    uint64_t last_kept = 0;                                                   // place key of the last value that is kept
    uint32_t listed = 0;
    if (p.cut) {
        find_cuts<kLastThreads>(a, row, p, cuts, parts);
        listed = a.listed_count[row];
    }
    const bool bounded = p.cut && cuts.low < kBins;
    auto weight_key = [&](uint64_t key) { return weight_of(exponent_of(p, of_key(static_cast<uint32_t>(key >> 32)))); };
    auto bin_key = [&](uint64_t key) { return bin_of(p, exponent_of(p, of_key(static_cast<uint32_t>(key >> 32)))); };
    if (bounded && listed <= kListed) {
        // the listed values in order, falling
        int n = 64;
        while (n < static_cast<int>(listed)) n *= 2;
        for (int i = tid; i < n; i += kLastThreads) list[i] = i < static_cast<int>(listed) ? a.listed[static_cast<size_t>(row) * kListed + i] : 0;
        __syncthreads();
        for (int size = 2; size <= n; size *= 2)
            for (int step = size / 2; step > 0; step /= 2) {
                for (int i = tid; i < n / 2; i += kLastThreads) {
                    const int low = 2 * i - (i & (step - 1)), high = low + step;
                    const uint64_t u = list[low], v = list[high];
                    if ((u < v) == ((low & size) == 0)) { list[low] = v; list[high] = u; }
                }
                __syncthreads();
            }
        // sums of their weights in that order; those of bin `last` apart
        uint64_t w[kPer], mine = 0, in_last = 0;
        int at_last[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int at = kPer * tid + i;
            const bool there = at < static_cast<int>(listed);
            w[i] = there ? weight_key(list[at]) : 0;
            at_last[i] = there && cuts.last >= 0 && bin_key(list[at]) == cuts.last;
            mine += w[i];
            in_last += at_last[i];
        }
        uint64_t total, total_last;
        uint64_t until = threads_until<kLastThreads>(mine, parts, total) - mine;
        __syncthreads();
        uint64_t rank = threads_until<kLastThreads>(in_last, parts, total_last) - in_last;
        if (tid == 0) { found[0] = 0; found[1] = 0; found[2] = 0; }
        __syncthreads();
        uint64_t sums[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) { until += w[i]; sums[i] = until; }
        if (cuts.last >= 0) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                if (at_last[i] && ++rank == 1) found[0] = sums[i] - w[i];     // in front of the bin
                if (at_last[i] && rank == cuts.need) { found[1] = sums[i]; found[2] = list[kPer * tid + i]; }
            }
            __syncthreads();
        }
        last_kept = found[2];
        if (p.top_p < 1.0f) {
            const uint64_t all = cuts.last >= 0 ? cuts.before_last + found[1] - found[0] : cuts.total;
            const uint64_t share = share_up(p.top_p > 0.0f ? fraction(p.top_p) : 0, all), least = (share > 0 ? share : 1) - cuts.before_low;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (w[i] && sums[i] - w[i] < least && sums[i] >= least) found[2] = list[kPer * tid + i];
            __syncthreads();
            last_kept = found[2];
        }
    } else if (bounded) {
        // more values in the cuts' bins than the list holds, many of them equal: bisection over their places, a pass over the row each
        auto pass = [&](uint64_t from, int low, int high, bool counts) {
            uint64_t sum = 0;
            for (int c = tid; c < x.chunks(); c += kLastThreads) {
                uint32_t key[kValues];
                const int first = x.keys(c, key);
#pragma unroll
                for (int i = 0; i < kValues; ++i) {
                    if (key[i] == kNone || place_key(key[i], first + i) < from) continue;
                    const double y = exponent_of(p, of_key(key[i]));
                    const int bin = bin_of(p, y);
                    if (bin < low || bin > high) continue;
                    const uint64_t w = weight_of(y);
                    sum += counts ? (w != 0) : w;
                }
            }
            all_sum<kLastThreads>(sum, parts);
            return sum;
        };
        auto bisect = [&](uint64_t least, int low, int high, bool counts) {    // the largest place from which on there is as much
            uint64_t from = 0;
            for (uint64_t bit = uint64_t{1} << 63; bit; bit >>= 1)
                if (pass(from | bit, low, high, counts) >= least) from |= bit;
            return from;
        };
        uint64_t all = cuts.total;
        if (cuts.last >= 0) {
            last_kept = bisect(cuts.need, cuts.last, cuts.last, true);
            all = cuts.before_last + pass(last_kept, cuts.last, cuts.last, false);
        }
        if (p.top_p < 1.0f) {
            const uint64_t share = share_up(p.top_p > 0.0f ? fraction(p.top_p) : 0, all);
            last_kept = bisect((share > 0 ? share : 1) - cuts.before_low, cuts.low, cuts.high, false);
        }
    }
    // sums of the slices: what was kept for certain and the listed values that are
    auto kept = [&](uint64_t key, uint64_t w) { return key >= last_kept && w >= p.least_weight; };
    auto slice_sum = [&](int slice) { return a.masses[static_cast<size_t>(row) * a.slices + slice]; };
    __shared__ uint64_t sums[kLastThreads];                                   // (at most so many slices)
    for (int i = tid; i < a.slices; i += kLastThreads) sums[i] = slice_sum(i);
    __syncthreads();
    auto add = [&](uint64_t key, uint64_t w) {
        const int slice = (static_cast<int>(~static_cast<uint32_t>(key)) + x.skew) / kValues / a.slice_chunks;
        atomicAdd(reinterpret_cast<unsigned long long*>(&sums[slice]), static_cast<unsigned long long>(w));
    };
    if (bounded && listed <= kListed) {
        for (int i = tid; i < static_cast<int>(listed); i += kLastThreads) {
            const uint64_t w = weight_key(list[i]);
            if (kept(list[i], w)) add(list[i], w);
        }
    } else if (bounded) {
        for (int c = tid; c < x.chunks(); c += kLastThreads) {
            uint32_t key[kValues];
            const int first = x.keys(c, key);
#pragma unroll
            for (int i = 0; i < kValues; ++i) {
                if (key[i] == kNone) continue;
                const uint64_t place = place_key(key[i], first + i), w = weight_key(place);
                if (bin_key(place) >= cuts.low && kept(place, w)) add(place, w);
            }
        }
    }
    __syncthreads();
    const uint64_t mine = tid < a.slices ? sums[tid] : 0;
    uint64_t total;
    const uint64_t until = threads_until<kLastThreads>(mine, parts, total);
    const float u = a.uniform[row];
    const uint64_t target = __umul64hi(fraction(u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f), total);         // the token's sum is the first above it
    if (until - mine <= target && until > target) { chosen = tid; found[0] = until - mine; }
    __syncthreads();
    const int begin = chosen * a.slice_chunks, end = min(begin + a.slice_chunks, x.chunks());
    uint64_t before = found[0];
    for (int c0 = begin; c0 < end; c0 += kLastThreads) {
        uint32_t key[kValues];
        uint64_t w[kValues], own = 0;
        int first = 0;
#pragma unroll
        for (int i = 0; i < kValues; ++i) w[i] = 0;
        if (c0 + tid < end) {
            first = x.keys(c0 + tid, key);
#pragma unroll
            for (int i = 0; i < kValues; ++i) {
                if (key[i] == kNone) continue;
                const uint64_t place = place_key(key[i], first + i), v = weight_key(place);
                w[i] = kept(place, v) ? v : 0;
                own += w[i];
            }
        }
        uint64_t here;
        __syncthreads();
        uint64_t sum = before + threads_until<kLastThreads>(own, parts, here) - own;
        if (sum <= target && sum + own > target) {
#pragma unroll
            for (int i = 0; i < kValues; ++i) {
                if (sum <= target && sum + w[i] > target) a.tokens[row] = first + i;
                sum += w[i];
            }
        }
        before += here;
        if (before > target) break;                                           // (all threads alike)
    }
}

template <typename T> int launch(const SampleArgs& a, hipStream_t stream) {
    const dim3 grid(a.slices, a.rows);
    hipLaunchKernelGGL((sample_extremes_kernel<T>), grid, dim3(kThreads), 0, stream, a);
    const bool cut = a.top_k || a.top_p || (a.top_k_all > 0 && a.top_k_all < a.vocab) || a.top_p_all < 1.0f;
    if (cut) hipLaunchKernelGGL((sample_histogram_kernel<T>), grid, dim3(kThreads), 0, stream, a);
    hipLaunchKernelGGL((sample_masses_kernel<T>), grid, dim3(kThreads), 0, stream, a);
    hipLaunchKernelGGL((sample_token_kernel<T>), dim3(a.rows), dim3(kLastThreads), 0, stream, a);
    return hipGetLastError() == hipSuccess ? PLLM_OK : PLLM_ERR_LAUNCH;
}

struct Layout { int slices, slice_chunks; size_t best, least, masses, mass, count, listed, listed_count, bytes; };
Layout layout_of(int64_t rows, int64_t vocab, int dtype) {
    const int values = dtype == PLLM_F32 ? 4 : 8;
    const int64_t chunks = (vocab + 2 * values - 2) / values;                 // (a row may begin inside a chunk)
    // as many slices as give the machine about four workgroups per compute unit, none of fewer than two chunks per thread
    const int64_t most = std::min<int64_t>((chunks + 2 * kThreads - 1) / (2 * kThreads), kLastThreads);
    const int64_t slices = std::max<int64_t>(1, std::min(most, (1024 + rows - 1) / rows));
    Layout l{};
    l.slice_chunks = static_cast<int>((chunks + slices - 1) / slices);
    l.slices = static_cast<int>((chunks + l.slice_chunks - 1) / l.slice_chunks);
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at += align256(bytes); return here; };
    l.best = take(rows * l.slices * 8);
    l.least = take(rows * l.slices * 4);
    l.masses = take(rows * l.slices * 8);
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
    a.rows = static_cast<int>(rows); a.vocab = static_cast<int>(vocab); a.slices = l.slices; a.slice_chunks = l.slice_chunks;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == PLLM_F32) return launch<float>(a, st);
    return dtype == PLLM_F16 ? launch<F16>(a, st) : launch<B16>(a, st);
}

}  // extern "C"
