// Device pieces of the paged E4M3 key/value cache: 16-bit and E4M3 conversions, matrix products, the sequence that owns a unit of work.
#pragma once

#include "paged_cache.h"
#include "pllm_device.h"

namespace pllm {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

template <bool BF16> __device__ __forceinline__ float half_value(uint32_t bits) {
    if constexpr (BF16) return __uint_as_float(bits << 16);
    else return f16_bits_to_float(bits);
}
template <bool BF16> __device__ __forceinline__ uint32_t half_pair(float a, float b) {
    if constexpr (BF16) {
        const v2b p = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
        return __builtin_bit_cast(uint32_t, p);
    } else {
        const v2h p = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
        return __builtin_bit_cast(uint32_t, p);
    }
}
template <bool BF16> __device__ __forceinline__ void half_eight(const uint4& u, float v[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = half_value<BF16>(w[i] & 0xffffu);
        v[2 * i + 1] = half_value<BF16>(w[i] >> 16);
    }
}
template <bool BF16> __device__ __forceinline__ uint4 half_pack(const float v[8]) {
    return make_uint4(half_pair<BF16>(v[0], v[1]), half_pair<BF16>(v[2], v[3]), half_pair<BF16>(v[4], v[5]), half_pair<BF16>(v[6], v[7]));
}

// Eight E4M3 codes times a power of two as 16-bit values: exact wherever the type holds the value (the convert instruction takes the scale's exponent).
template <bool BF16> __device__ __forceinline__ uint4 half_from_codes(uint32_t lo, uint32_t hi, float scale) {
    if constexpr (BF16) {
        const v2b a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
        const v2b c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
        return make_uint4(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, c), __builtin_bit_cast(uint32_t, d));
    } else {
        const v2h a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, true);
        const v2h c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, true);
        return make_uint4(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, c), __builtin_bit_cast(uint32_t, d));
    }
}

template <bool BF16> __device__ __forceinline__ v4f half_mfma16(const uint4& a, const uint4& b, v4f c) {
    if constexpr (BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
template <bool BF16> __device__ __forceinline__ v16f half_mfma32(const uint4& a, const uint4& b, v16f c) {
    if constexpr (BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// v, cut to its sign, exponent and 19 bits and with the last of 20 set if anything was cut off (round to odd): what is rounded to fewer bits from here comes out
// as if rounded from v itself
__device__ __forceinline__ float odd_float(double v) {
    const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v));
    uint32_t odd;
    asm("v_min_u32 %0, 1, %1" : "=v"(odd) : "v"(static_cast<uint32_t>(b)));  // (one instruction where a comparison and a choice are two)
    return static_cast<float>(__longlong_as_double(static_cast<long long>(static_cast<uint64_t>(static_cast<uint32_t>(b >> 32) | odd) << 32)));
}

// sum + both 16-bit values of a pair
template <bool BF16> __device__ __forceinline__ float half_pair_sum(uint32_t pair, float sum) {
    if constexpr (BF16) {
        const v2b ones = {static_cast<__bf16>(1.0f), static_cast<__bf16>(1.0f)};
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2b, pair), ones, sum, false);
    } else {
        const v2h ones = {static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)};
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2h, pair), ones, sum, false);
    }
}

// four values as E4M3 codes (to the nearest, ties to even; within 448 or NaN); four codes as those of their values times a ratio of at most one
__device__ __forceinline__ uint32_t four_codes(float a, float b, float c, float d) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true));
}
__device__ __forceinline__ uint32_t scaled_codes(uint32_t w, float ratio) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    return four_codes(lo[0] * ratio, lo[1] * ratio, hi[0] * ratio, hi[1] * ratio);
}

// whether one of four E4M3 codes is NaN (0x7f or 0xff)
__device__ __forceinline__ bool any_nan_code(uint32_t w) { return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0; }
// which of them are: bit i for byte i; the codes with zeros in their place
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) {
    const uint32_t high = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    return ((high >> 7) * 0x10204080u) >> 28;
}
__device__ __forceinline__ uint32_t without_nan(uint32_t w) {
    const uint32_t high = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    return w & ~((high >> 7) * 0xffu);
}
// bytes below `count` of a word of four, as a mask
__device__ __forceinline__ uint32_t first_bytes(int count) { return count >= 4 ? 0xffffffffu : (count <= 0 ? 0u : (1u << (8 * count)) - 1u); }

// The sequence that owns a slot of work: the last of the first `count` whose first slot is not behind it.  All lanes look together.
__device__ __forceinline__ int paged_sequence(const int32_t* cu_steps, int rows, int count, int unit, int spare, int64_t slot) {
    const int lane = threadIdx.x & 63;
    int owners = 0;
    for (int base = 0; base < count; base += 64) {
        const int s = base + lane;
        const bool begun = s < count && paged_first_slot(paged_offset(cu_steps, s, 0, rows), s, unit, spare) <= slot;
        const int n = __popcll(__ballot(begun));
        owners += n;
        if (n < 64) break;
    }
    return owners > 0 ? owners - 1 : 0;
}

}  // namespace pllm
