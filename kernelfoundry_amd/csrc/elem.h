// elem.h -- the two 16-bit input types of the packed, rotary and 4-bit-cache
// kernels: fp16 (kBF = false) and bf16, their conversions and MFMAs.
#pragma once

#include "attn_kernels.h"

namespace kf {

typedef __bf16 bf16;
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <bool kBF> struct Elem;

template <> struct Elem<false> {
    typedef f16x8 x8;
    typedef f16x2 x2;
    static constexpr uint32_t kExpBits = 0x7c00u;
    static __device__ __forceinline__ f32x16 mfma32(const x8& a, const x8& b, const f32x16& c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 mfma16(const x8& a, const x8& b, const f32x4& c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    // The two 4-bit values of byte kByte of w, times a power of two: exact.
    template <int kByte>
    static __device__ __forceinline__ x2 from_fp4(uint32_t w, float scale) {
        return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, kByte);
    }
    // Two values over a power of two into byte kByte of w: nearest, ties to
    // the even code, at most 6 in magnitude.
    template <int kByte>
    static __device__ __forceinline__ uint32_t to_fp4(uint32_t w, x2 v, float scale) {
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, v, scale, kByte);
    }
};

template <> struct Elem<true> {
    typedef bf16x8 x8;
    typedef bf16x2 x2;
    static constexpr uint32_t kExpBits = 0x7f80u;
    static __device__ __forceinline__ f32x16 mfma32(const x8& a, const x8& b, const f32x16& c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 mfma16(const x8& a, const x8& b, const f32x4& c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    template <int kByte>
    static __device__ __forceinline__ x2 from_fp4(uint32_t w, float scale) {
        return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, kByte);
    }
    template <int kByte>
    static __device__ __forceinline__ uint32_t to_fp4(uint32_t w, x2 v, float scale) {
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, v, scale, kByte);
    }
};

// Eight fp32 values rounded to the 16-bit type (nearest even).
template <bool kBF>
__device__ __forceinline__ typename Elem<kBF>::x8 round8(const f32x8& v) {
    return __builtin_convertvector(v, typename Elem<kBF>::x8);
}
template <bool kBF>
__device__ __forceinline__ f32x8 widen8(const u32x4& v) {
    return __builtin_convertvector(__builtin_bit_cast(typename Elem<kBF>::x8, v), f32x8);
}
// The eight 4-bit values of a word, channel 2 i in the low half of byte i.
template <bool kBF>
__device__ __forceinline__ typename Elem<kBF>::x8 from_fp4x8(uint32_t w, float scale) {
    using E = Elem<kBF>;
    const auto a = E::template from_fp4<0>(w, scale), b = E::template from_fp4<1>(w, scale);
    const auto c = E::template from_fp4<2>(w, scale), d = E::template from_fp4<3>(w, scale);
    return __builtin_shufflevector(__builtin_shufflevector(a, b, 0, 1, 2, 3),
                                   __builtin_shufflevector(c, d, 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}

// The last sequence whose start is at or before token t of packed sequences:
// starts[0] .. starts[n] do not decrease, starts[0] <= t < starts[n] holds or
// the caller drops the token.
__device__ __forceinline__ int sequence_of(const int* starts, int n, int t) {
    int lo = 0, hi = n;  // starts[lo] <= t < starts[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= t) lo = mid; else hi = mid;
    }
    return lo;
}

}  // namespace kf
