// Device helpers of the 8-bit paged K/V cache.
#pragma once

#include "common.hpp"
#include "kernels.hpp"

namespace mslim {

// Page numbers and scales that a whole wavefront reads, through the scalar
// cache: no kernel that reads them so writes them.  (As vector loads each was
// waited for where it was issued, behind every K and V load in flight.)
__device__ __forceinline__ int32_t scalar_page(const int32_t *p) {
    return *reinterpret_cast<const __attribute__((address_space(4))) int32_t *>(reinterpret_cast<uintptr_t>(p));
}
__device__ __forceinline__ float2 scalar_scales(const float *p) {
    const uint64_t w = *reinterpret_cast<const __attribute__((address_space(4))) uint64_t *>(reinterpret_cast<uintptr_t>(p));
    return make_float2(__uint_as_float((uint32_t)w), __uint_as_float((uint32_t)(w >> 32)));
}

// The value of byte i of four.
template <int FMT>
__device__ __forceinline__ float byte_value(uint32_t w, int i) {
    if constexpr (FMT == kFormatE4m3) {
        switch (i) {
        case 0: return __builtin_amdgcn_cvt_f32_fp8((int)w, 0);
        case 1: return __builtin_amdgcn_cvt_f32_fp8((int)w, 1);
        case 2: return __builtin_amdgcn_cvt_f32_fp8((int)w, 2);
        default: return __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
        }
    } else {
        return (float)(int8_t)(w >> (8 * i));
    }
}

// Eight bytes as BF16 values of their format, exactly: both formats' values
// have at most eight significant bits.
template <int FMT>
__device__ __forceinline__ bf16x8_t widen8(uint32_t lo, uint32_t hi) {
    uint32_t w[4];
    if constexpr (FMT == kFormatE4m3) {
        w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
        w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
        w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
        w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t s = i < 2 ? lo : hi;
            const uint32_t x = __float_as_uint((float)(int8_t)(s >> (16 * (i & 1))));
            const uint32_t y = __float_as_uint((float)(int8_t)(s >> (16 * (i & 1) + 8)));
            w[i] = __builtin_amdgcn_perm(y, x, 0x07060302u);
        }
    }
    return __builtin_bit_cast(bf16x8_t, make_uint4(w[0], w[1], w[2], w[3]));
}

}  // namespace mslim
