// What the kernels over rows of logits (router.hip, distill.hip) share: lanes that work on one row, their
// reductions, a row's chunks, and running softmax sums.
//
// softmax(l)_e = exp(l_e - m) / s with m = max l and s = sum exp(l - m).  Parts of a row are joined by
//   m = max(m1, m2),  s = s1 exp(m1 - m) + s2 exp(m2 - m),
// so that one pass over the row gives both.  -inf is a masked logit: it adds nothing, and a row of nothing
// else has m = -inf and s = 0.  NaN and +inf make the row's softmax NaN.
#pragma once
#include <cmath>

#include "elements.h"

namespace odie {

constexpr float kNegInfinity = -INFINITY;

// op over the kLanes lanes (a power of two, aligned) that work on one row; every lane gets the result, the same
// bits.  All of these lanes are active.
template <int kLanes, class F> __device__ inline uint32_t across(uint32_t x, F&& op) {
    if constexpr (kLanes > 1) x = op(x, dpp_move<0xB1>(x));     // quad_perm: lane ^ 1
    if constexpr (kLanes > 2) x = op(x, dpp_move<0x4E>(x));     // quad_perm: lane ^ 2
    if constexpr (kLanes > 4) x = op(x, dpp_move<0x141>(x));    // row_half_mirror: lane ^ 7
    if constexpr (kLanes > 8) x = op(x, dpp_move<0x140>(x));    // row_mirror: lane ^ 15
    if constexpr (kLanes > 16) {
        const auto pair = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        x = op(pair[0], pair[1]);
    }
    if constexpr (kLanes > 32) {
        const auto pair = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        x = op(pair[0], pair[1]);
    }
    return x;
}

__device__ inline uint32_t as_bits(float x) { return __builtin_bit_cast(uint32_t, x); }
__device__ inline float as_float(uint32_t x) { return __builtin_bit_cast(float, x); }

template <int kLanes> __device__ inline float sum_across(float x) {
    return as_float(across<kLanes>(
        as_bits(x), [](uint32_t a, uint32_t b) { return as_bits(as_float(a) + as_float(b)); }));
}

// The larger one; a NaN wins.
__device__ inline float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

template <int kLanes> __device__ inline uint32_t sum_across(uint32_t x) {
    return across<kLanes>(x, [](uint32_t a, uint32_t b) { return a + b; });
}

// The same for fp64, whose halves move alike.
template <int kLanes> __device__ inline double sum_across(double x) {
    const auto move = [&](uint32_t& low, uint32_t& high, auto&& by) {
        const uint64_t bits = __builtin_bit_cast(uint64_t, x);
        low = by(static_cast<uint32_t>(bits)), high = by(static_cast<uint32_t>(bits >> 32));
        x += __builtin_bit_cast(double, static_cast<uint64_t>(high) << 32 | low);
    };
    uint32_t low, high;
    if constexpr (kLanes > 1) move(low, high, [](uint32_t v) { return dpp_move<0xB1>(v); });
    if constexpr (kLanes > 2) move(low, high, [](uint32_t v) { return dpp_move<0x4E>(v); });
    if constexpr (kLanes > 4) move(low, high, [](uint32_t v) { return dpp_move<0x141>(v); });
    if constexpr (kLanes > 8) move(low, high, [](uint32_t v) { return dpp_move<0x140>(v); });
    if constexpr (kLanes > 16)
        move(low, high, [](uint32_t v) { return static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 16)); });
    if constexpr (kLanes > 32)
        move(low, high, [](uint32_t v) { return static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 32)); });
    return x;
}

template <int kLanes> __device__ inline float max_across(float x) {
    return as_float(across<kLanes>(
        as_bits(x), [](uint32_t a, uint32_t b) { return as_bits(larger(as_float(a), as_float(b))); }));
}

// exp(x).  kExact: the library's; else the hardware's exp2, off by 2^-23 (1 + |x|) relative, for sums and for results
// that are rounded to 16 bits.
template <bool kExact> __device__ inline float exponential(float x) {
    if constexpr (kExact) return expf(x);
    return __builtin_amdgcn_exp2f(x * 1.44269504f);
}

// The value that a row's logits are taken relative to: their maximum, or 0 where all of them are masked, whose
// differences would be NaN.
__device__ inline float base_of(float m) { return m == kNegInfinity ? 0.0f : m; }

// Columns column .. column + kPerVec - 1 of a row of `width`, -inf past its end.
template <class T> __device__ inline void load_logits(const T* row, int column, int width, float v[kPerVec<T>]) {
    const int count = width - column;
    if (count >= kPerVec<T>) {
        widen<T>(load16(row + column), v);
    } else if (count > 0) {
        widen<T>(load_end(row + column, count, column), v);
#pragma unroll
        for (int i = 0; i < kPerVec<T>; ++i) v[i] = i < count ? v[i] : kNegInfinity;
    } else {
#pragma unroll
        for (int i = 0; i < kPerVec<T>; ++i) v[i] = kNegInfinity;
    }
}

// A running maximum and the sum of exponentials relative to it.
template <bool kExact> struct Running {
    float m = kNegInfinity, s = 0.0f;

    template <int kCount> __device__ void add(const float (&v)[kCount]) {
        float top = v[0];
#pragma unroll
        for (int i = 1; i < kCount; ++i) top = larger(top, v[i]);
        top = larger(m, top);
        const float base = base_of(top);
        float more = 0.0f;
#pragma unroll
        for (int i = 0; i < kCount; ++i) more += exponential<kExact>(v[i] - base);
        s = s * exponential<kExact>(m - base) + more;
        m = top;
    }
    __device__ void join(float m2, float s2) {
        const float top = larger(m, m2), base = base_of(top);
        s = s * exponential<kExact>(m - base) + s2 * exponential<kExact>(m2 - base);
        m = top;
    }
    template <int kLanes> __device__ void join_lanes() {
        const float top = max_across<kLanes>(m);
        s = sum_across<kLanes>(s * exponential<kExact>(m - base_of(top)));
        m = top;
    }
};

}  // namespace odie
