// Microscaled 4-bit floating point on gfx950: blocks of 32 values along a row that share a scale 2^(s - 127).
//
// A value is sign, two bits of exponent and one of fraction: 0, 0.5, 1, 1.5, 2, 3, 4 or 6 times the block's scale.  The
// hardware's conversions and products take the scale's exponent as it is stored (s = 0: 2^-127, s = 255: NaN);
// conversions round to nearest even, and clamp at 6 on the way to 4 bits.
#pragma once
#include "elements.h"

namespace odie {

constexpr int kMxBlock = 32;       // values that share a scale
constexpr int kMxBytes = 16;       // of a block's codes

inline int64_t mx_blocks(int64_t width) { return (width + kMxBlock - 1) / kMxBlock; }
inline int64_t mx_code_pitch(int64_t width) { return mx_blocks(width) * kMxBytes; }
inline int64_t mx_scale_pitch(int64_t width) { return (mx_blocks(width) + 3) / 4 * 4; }

// The scale as the conversions take it.
__device__ inline float mx_scale(uint32_t s) { return __builtin_bit_cast(float, s << 23); }

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// The two values of byte kByte of `codes`.
template <int kByte> __device__ inline uint32_t mx_pair(_Float16, uint32_t codes, float scale) {
    return __builtin_bit_cast(
        uint32_t, static_cast<f16x2>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, kByte)));
}
template <int kByte> __device__ inline uint32_t mx_pair(__bf16, uint32_t codes, float scale) {
    return __builtin_bit_cast(
        uint32_t, static_cast<bf16x2>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, kByte)));
}
template <int kByte> __device__ inline f32x2 mx_pair(float, uint32_t codes, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, kByte);
}

// 16 bytes of values from `codes`: eight 16-bit ones, or the four fp32 ones of its lower or upper half.
template <class T> __device__ inline vec16 mx_values(uint32_t codes, float scale, bool upper) {
    if constexpr (sizeof(T) == 4) {
        const uint32_t half = upper ? codes >> 16 : codes;
        const f32x2 a = mx_pair<0>(T{}, half, scale), b = mx_pair<1>(T{}, half, scale);
        const float v[4] = {a[0], a[1], b[0], b[1]};
        return __builtin_bit_cast(vec16, v);
    } else {
        return vec16{mx_pair<0>(T{}, codes, scale), mx_pair<1>(T{}, codes, scale), mx_pair<2>(T{}, codes, scale),
                     mx_pair<3>(T{}, codes, scale)};
    }
}

}  // namespace odie
