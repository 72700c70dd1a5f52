// Residual addition, RMS normalisation and E4M3 quantization of activation rows in one pass: what stands between a projection's output and the
// next FP8 projection (fp8_gemm).
//     t = round(x + residual);  n = t * rsqrt(mean(t^2) + eps) * weight;  per 128 values s = max(amax |n|, quant_eps) / 448 (a power of two
//     when asked for), code = E4M3(n / s)
// The sum leaves rounded to the stream's type, and what is normalized is that rounded value, so the operator says what the three separate ones
// say; the normalized values become codes as they are (the separate operators round them to 16 bits in between).  Squares, their sum, root, products and quotient are
// in 64 bits, and a value is cut on the way to a code so that the code is the one that the value itself rounds to: in 32 bits one in a million is its neighbour, 6 %
// away.  (Without power-of-two scales the root falls out of the codes of all blocks above quant_eps, E4M3(448 t w / max |t w|).)
// Bound: bytes for prompts (8192 rows of 5120 bf16 values: 295 MB in 55 us, 5.4 TB/s; with squares summed in 32 bits 54 - 56), the start of a launch and one round trip to
// memory for few rows (3.0 us from begin to end, 4.2 from one launch to the next).
#include "paged_device.h"
#include "pllm_internal.h"

#include <cfloat>

namespace pllm {
namespace {

struct NormArgs {
    const void* x; const void* residual; const float* weight;
    void* total; uint8_t* codes; float* scales;
    int rows, dim, pow2;
    double inv_dim, eps, quant_eps;
};

template <int DT> struct Eight { uint4 a[DT == PLLM_F32 ? 2 : 1]; };
template <int DT> __device__ __forceinline__ Eight<DT> load_eight(const void* p, size_t at) {
    Eight<DT> e;
    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(p) + at * (DT == PLLM_F32 ? 4 : 2));
#pragma unroll
    for (int i = 0; i < (DT == PLLM_F32 ? 2 : 1); ++i) e.a[i] = src[i];
    return e;
}
template <int DT> __device__ __forceinline__ float eight_value(const Eight<DT>& e, int i) {
    if constexpr (DT == PLLM_F32) {
        const uint4 w = e.a[i >> 2];
        return __uint_as_float((i & 3) == 0 ? w.x : (i & 3) == 1 ? w.y : (i & 3) == 2 ? w.z : w.w);
    } else {
        const uint32_t w = i < 2 ? e.a[0].x : i < 4 ? e.a[0].y : i < 6 ? e.a[0].z : e.a[0].w, h = (i & 1) ? w >> 16 : w & 0xffffu;
        return DT == PLLM_BF16 ? __uint_as_float(h << 16) : f16_bits_to_float(h);
    }
}
// eight sums rounded to the type, as they are stored
template <int DT> __device__ __forceinline__ Eight<DT> pack_eight(const float v[8]) {
    Eight<DT> e;
    if constexpr (DT == PLLM_F32) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            e.a[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = half_pair<DT == PLLM_BF16>(v[2 * i], v[2 * i + 1]);
        e.a[0] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return e;
}

template <int OFF> __device__ __forceinline__ double wide_peer(double v) {
    const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v));
    const uint32_t lo = __float_as_uint(butterfly_peer<OFF>(__uint_as_float(static_cast<uint32_t>(b)))), hi = __float_as_uint(butterfly_peer<OFF>(__uint_as_float(static_cast<uint32_t>(b >> 32))));
    return __longlong_as_double(static_cast<long long>((static_cast<uint64_t>(hi) << 32) | lo));
}
// 1 / v, off by a few 2^-53, for v far from the ends of the range
__device__ __forceinline__ double reciprocal(double v) {
    double r = __builtin_amdgcn_rcp(v);
#pragma unroll
    for (int i = 0; i < 2; ++i) r = __builtin_fma(__builtin_fma(-v, r, 1.0), r, r);
    return r;
}

// WAVES waves share a row (one: four rows to a workgroup), PIECES pieces of eight values per lane; the whole row stays in registers.  Sixteen
// neighbouring lanes hold the 128 values of one scale.
template <int DT, int WAVES, int PIECES>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void add_norm_fp8_kernel(const NormArgs a) {
    __shared__ double red[WAVES == 1 ? 4 : WAVES];
    const int tid = WAVES == 1 ? static_cast<int>(threadIdx.x & 63) : static_cast<int>(threadIdx.x);
    const int row = WAVES == 1 ? static_cast<int>(blockIdx.x * 4 + (threadIdx.x >> 6)) : static_cast<int>(blockIdx.x);
    if (WAVES == 1 && row >= a.rows) return;                                  // (no barrier below where a wave has a row of its own)
    const size_t base = static_cast<size_t>(row) * a.dim;
    Eight<DT> xv[PIECES], rv[PIECES];
    Eight<PLLM_F32> g[PIECES];
    int e0[PIECES];
    bool inside[PIECES];
    // What lanes beyond the row load instead, not counted: their wave's first values again, since another wave may be writing the sums over its own; a wave with none
    // (one piece: any later one lies behind a whole first) weights.  (Leaving the loads out costs more, 57.5 us for 55.7 at 8192 rows of 5120; every lane's own
    // first piece 57.3; weights for all 66 us for 63 at 2048 rows of 17408.)
    const int wave0 = WAVES == 1 ? 0 : 8 * __builtin_amdgcn_readfirstlane(tid & ~63);
    const bool none = WAVES > 1 && PIECES == 1 && wave0 >= a.dim;
    const void *const x = none ? a.weight : a.x, *const residual = none ? a.weight : a.residual;
    const size_t from = none ? 0 : base;
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
        e0[j] = 8 * (tid + 64 * WAVES * j);
        inside[j] = e0[j] < a.dim;
        const int at = inside[j] ? e0[j] : (none ? 0 : wave0);
        xv[j] = load_eight<DT>(x, from + at);
        if (a.residual) rv[j] = load_eight<DT>(residual, from + at);
        g[j] = load_eight<PLLM_F32>(a.weight, inside[j] ? e0[j] : 0);
    }
    double ss = 0.0;
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
        if (a.residual) {
            float t[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = eight_value(xv[j], i) + eight_value(rv[j], i);
            xv[j] = pack_eight<DT>(t);
            if (inside[j]) {
                uint4* dst = reinterpret_cast<uint4*>(static_cast<unsigned char*>(a.total) + (base + e0[j]) * (DT == PLLM_F32 ? 4 : 2));
#pragma unroll
                for (int i = 0; i < (DT == PLLM_F32 ? 2 : 1); ++i) dst[i] = xv[j].a[i];
            }
        }
        // squares and their sum in 64 bits: exact squares, and no row whose sum float32 would not hold
        Eight<DT> again = xv[j];                                              // (nothing of this is to be shared with what follows: 20 registers)
#pragma unroll
        for (int i = 0; i < (DT == PLLM_F32 ? 2 : 1); ++i) asm("" : "+v"(again.a[i].x), "+v"(again.a[i].y), "+v"(again.a[i].z), "+v"(again.a[i].w));
        double part = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const double v = eight_value(again, i);
            part = __builtin_fma(v, v, part);
        }
        ss += inside[j] ? part : 0.0;
    }
    ss += wide_peer<1>(ss);
    ss += wide_peer<2>(ss);
    ss += wide_peer<4>(ss);
    ss += wide_peer<8>(ss);
    ss += wide_peer<16>(ss);
    ss += wide_peer<32>(ss);
    if constexpr (WAVES > 1) {
        if ((tid & 63) == 0) red[tid >> 6] = ss;
        __syncthreads();
        ss = 0.0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) ss += red[w];
    }
    const double rstd = rsqrt(__builtin_fma(ss, a.inv_dim, a.eps));
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
        // t * weight; the root is one factor of the whole row and goes with the block's scale: one product per value behind one division per block
        double v[8], top = 0.0, none = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = static_cast<double>(eight_value(xv[j], i)) * static_cast<double>(eight_value(g[j], i));
            top = fmax(top, fabs(v[i]));
            none = __builtin_fma(v[i], 0.0, none);                            // NaN from infinities and NaN, which a maximum may drop
        }
        top = none == 0.0 ? top : HUGE_VAL;
        top = fmax(top, wide_peer<1>(top));
        top = fmax(top, wide_peer<2>(top));
        top = fmax(top, wide_peer<4>(top));
        top = fmax(top, wide_peer<8>(top));
        const double amax = top * rstd, most = fmax(amax, a.quant_eps);
        const bool usual = amax >= a.quant_eps;
        float s;
        double factor;
        if (a.pow2) {
            int e;
            const double m = frexp(most, &e);                                 // 448 = 0.875 * 2^9
            e = max(m <= 0.875 ? e - 9 : e - 8, -126);
            s = static_cast<float>(ldexp(1.0, e));
            factor = ldexp(rstd, -e);
        } else {
            s = static_cast<float>(most * (1.0 / 448.0));
            factor = (usual ? 448.0 : 448.0 * rstd) * reciprocal(usual ? top : a.quant_eps);
        }
        uint32_t lo, hi;
        if (amax <= FLT_MAX && s <= FLT_MAX) {
            float c[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) c[i] = odd_float(v[i] * factor);      // (448 and the product's own rounding at most)
            int l = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false), h = __builtin_amdgcn_cvt_pk_fp8_f32(c[4], c[5], 0, false);
            lo = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], l, true));
            hi = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c[6], c[7], h, true));
        } else {                                                              // infinities and NaN: E4M3 has only NaN for them, and so has the whole block
            s = __uint_as_float(0x7fc00000u);
            lo = hi = 0x7f7f7f7fu;
        }
        if (inside[j]) {
            *reinterpret_cast<uint2*>(a.codes + base + e0[j]) = make_uint2(lo, hi);
            if ((tid & 15) == 0) a.scales[(base + e0[j]) / 128] = s;
        }
    }
}

template <int DT, int WAVES, int PIECES>
void launch(const NormArgs& a, hipStream_t stream) {
    const unsigned blocks = WAVES == 1 ? (static_cast<unsigned>(a.rows) + 3) / 4 : static_cast<unsigned>(a.rows);
    hipLaunchKernelGGL((add_norm_fp8_kernel<DT, WAVES, PIECES>), dim3(blocks), dim3(WAVES == 1 ? 256 : 64 * WAVES), 0, stream, a);
}

template <int DT>
void launch_rows(const NormArgs& a, hipStream_t stream) {
    // Four waves to a row up to 8192 values, in as many pieces as that takes: a row in one piece of more waves is as fast where every row finds a compute unit of
    // its own (64 rows, us with eight or sixteen waves / four: 4096 bf16 values 3.8 / 3.9, 5120 4.5 / 4.4, 8192 4.8 / 5.0) and waits longer for itself where
    // not (8192 rows of 5120 78 / 55).
    if (a.dim <= 512) launch<DT, 1, 1>(a, stream);
    else if (a.dim <= 2048) launch<DT, 4, 1>(a, stream);
    else if (a.dim <= 4096) launch<DT, 4, 2>(a, stream);
    else if (a.dim <= 6144) launch<DT, 4, 3>(a, stream);
    else if (a.dim <= 8192) launch<DT, 4, 4>(a, stream);
    else if (a.dim <= 16384) launch<DT, 16, 2>(a, stream);
    else if (a.dim <= 24576) launch<DT, 16, 3>(a, stream);
    else launch<DT, 16, 4>(a, stream);
}

constexpr int64_t kWidestRow = 32768;           // four pieces of eight values for each of 1024 lanes

}  // namespace
}  // namespace pllm

extern "C" int pllm_fused_add_rms_norm_fp8(const void* x, const void* residual, int dtype, const float* weight, void* total, uint8_t* codes,
                                           float* scales, int64_t rows, int64_t dim, float eps, float quant_eps, int round_scale_pow2, void* stream) {
    using namespace pllm;
    if (!x || !weight || !codes || !scales || (residual && !total) || rows <= 0 || dim <= 0 || dim % 128 != 0 || !(quant_eps > 0.0f))
        return PLLM_ERR_INVALID_ARGUMENT;
    if (dtype != PLLM_F32 && dtype != PLLM_F16 && dtype != PLLM_BF16) return PLLM_ERR_INVALID_ARGUMENT;
    const uintptr_t wide = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(weight) |
                           reinterpret_cast<uintptr_t>(total);
    if ((wide & 15u) || (reinterpret_cast<uintptr_t>(codes) & 7u) || (reinterpret_cast<uintptr_t>(scales) & 3u)) return PLLM_ERR_INVALID_ARGUMENT;
    if (rows > 0x3fffff || dim > kWidestRow) return PLLM_ERR_UNSUPPORTED;     // (a launch counts its threads in 32 bits)
    const NormArgs a{x, residual, weight, total, codes, scales, static_cast<int>(rows), static_cast<int>(dim), round_scale_pow2 != 0, 1.0 / static_cast<double>(dim), eps, quant_eps};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == PLLM_F32) launch_rows<PLLM_F32>(a, st);
    else if (dtype == PLLM_F16) launch_rows<PLLM_F16>(a, st);
    else launch_rows<PLLM_BF16>(a, st);
    return hipGetLastError() == hipSuccess ? PLLM_OK : PLLM_ERR_LAUNCH;
}
