// What the operators on rows of 8-bit integers with a scale each read of their descriptors.
//   values [.., L]  int8, a row's integers
//   scales [..]     float, what a 1 in the row stands for
#pragma once

#include "cache.hpp"
#include "lanes.hpp"

namespace th {

// Where the rows of a tensor [.., L] start: its dims but the last, those that lie behind each other as one, outermost first.
struct RowsMap {
    int outer;
    uint32_t extent[TANNIC_DIMENSIONS - 1];
    FastDiv div[TANNIC_DIMENSIONS - 1];
    int64_t stride[TANNIC_DIMENSIONS - 1];
    int64_t step;      // from element to element of a row

    __device__ inline int64_t offset(uint32_t row) const {
        int64_t at = 0;
        for (int d = outer - 1; d > 0; --d) {
            uint32_t above, here;
            div[d].divmod(row, above, here);
            at += static_cast<int64_t>(here) * stride[d];
            row = above;
        }
        return at + static_cast<int64_t>(row) * stride[0];
    }
};

inline RowsMap rows_of(const tannic_tensor_t* t) {
    RowsMap m{};
    int at = TANNIC_DIMENSIONS - 1;      // (filled from the back, moved to the front below)
    for (int d = t->rank - 2; d >= 0; --d) {
        const uint32_t extent = static_cast<uint32_t>(t->shape.sizes[d]);
        if (extent == 1) continue;
        if (at < TANNIC_DIMENSIONS - 1 && t->strides.sizes[d] == m.stride[at] * static_cast<int64_t>(m.extent[at])) {
            m.extent[at] *= extent;
        } else {
            --at;
            m.extent[at] = extent;
            m.stride[at] = t->strides.sizes[d];
        }
    }
    m.outer = TANNIC_DIMENSIONS - 1 - at;
    for (int d = 0; d < m.outer; ++d) {
        m.extent[d] = m.extent[at + d];
        m.stride[d] = m.stride[at + d];
        m.div[d] = FastDiv(m.extent[d]);
    }
    m.step = stride_of(t, t->rank - 1);
    return m;
}

// The scales of values [.., L]: [..], contiguous float.
inline bool scales_of(const tannic_tensor_t* scales, const tannic_tensor_t* values) {
    if (scales->rank + 1 != values->rank) return false;
    for (int d = 0; d < scales->rank; ++d)
        if (scales->shape.sizes[d] != values->shape.sizes[d]) return false;
    return rows_contiguous(scales);
}

inline bool quantizable(int dtype) { return dtype == TANNIC_FLOAT16 || dtype == TANNIC_BFLOAT16 || dtype == TANNIC_FLOAT32; }

// A float as a number of type D.  (The empty statement keeps a product or sum before it a rounding of its own for every D: its last step and the conversion to
// float16 would become one instruction with one rounding, and float16 results other than those of the same steps one by one.)
template <class D> __device__ inline D rounded(float x) {
    if constexpr (std::is_same_v<D, f16>) asm("" : "+v"(x));
    return narrow_result<D>(x);
}
template <class D> __device__ inline D rounded(double x) { return static_cast<D>(x); }

// A row's largest magnitude as the bits of a float without its sign: they are ordered as the magnitudes are, what is not a number above infinity.
struct LargestOp {
    __device__ static inline uint32_t combine(uint32_t x, uint32_t y) { return x > y ? x : y; }
};
__device__ inline uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// A row whose largest value is smaller than this is written as if it were this: 127 times its reciprocal is finite, it divided by 127 no subnormal number.
constexpr float kLeastLargest = 0x1p-119f;

// A row's integers are the nearest ones of u * (127 * (1 / its largest magnitude)), each step rounded, ties to even, and its scale says what a 1 stands for.  A row with something
// that is not finite has the scale NaN and zeros: whatever is computed from it is NaN.
struct RowScale {
    float factor, largest;
    bool finite;
    __device__ explicit RowScale(uint32_t most) {
        finite = most < 0x7F800000u;
        largest = fmaxf(__uint_as_float(most), kLeastLargest);
        factor = 127.0f * (1.0f / largest);
    }
    __device__ inline int8_t integer(float u) const { return finite ? static_cast<int8_t>(static_cast<int>(rintf(u * factor))) : int8_t(0); }
    // (times `one`: what every element of the row is multiplied by, which cancels in the integers)
    __device__ inline float scale(float one) const { return finite ? largest * one / 127.0f : __builtin_nanf(""); }
};

}  // namespace th
