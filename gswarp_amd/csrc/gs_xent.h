// What the cross entropy's kernels share: the targets, the logits' scale, and
// what the backward keeps of a row.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gs_xent {

struct Targets {
  const void* p;
  int bits;
  int64_t ignore;
  __device__ __forceinline__ int64_t at(int64_t i) const {
    return bits == 64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
  }
};

// The order in which the rows of the features are taken: as they are (at null), or
// those that count first and the others behind, each in their order, so that the
// products are formed for `count` rows only.  A kernel works on a piece of it from `first`.
struct Order {
  const int* at;
  const int* count;
  int32_t first;
  __device__ __forceinline__ int64_t row(int i) const { return at ? at[first + i] : (int64_t)first + i; }
  // how many of the piece's n rows have to be looked at
  __device__ __forceinline__ int32_t used(int32_t n) const { return at ? max(0, min(n, *count - first)) : n; }
  Order from(int64_t i) const { return {at, count, (int32_t)i}; }
};

// What the dot products of laid-out rows are multiplied by for base-2 logits:
// scale2 times the operands' units (fp32; else null), kept a normal number so
// that minus infinity (what lies past the vocabulary) stays that under a scale
// that underflows, or is zero: the same flat distribution.
__device__ __forceinline__ float scale_of(float scale2, const float* units) {
  if (units) scale2 = scale2 * units[0] * units[1];
  return copysignf(fmaxf(fabsf(scale2), 1.17549435e-38f), scale2);
}

// A row's maximum and sum are kept as the largest dot product itself, x (turned
// upright: times the sign of the scale), and the sum of 2^((x_j - x) scale) over all
// others: x's own 1 is added in 64 bits.  A label that is all but certain then has a
// loss, and p - 1, as small as fp32 can tell, not as small as the rounding of the logits' size.
// The terms are formed with one fma as 2^(x_j scale - top), top = x scale rounded;
// this takes the sum of a set that holds x itself from there.  (1 added here would
// round once more, and up wherever the first rounding left a tie.)
constexpr float kLn2f = 0.6931471805599453f;
__device__ __forceinline__ float settled(float x, float scale, float sum) {
  const float top = x * scale, off = __builtin_fmaf(x, scale, -top);
  const float rest = sum - __builtin_amdgcn_exp2f(off);  // all but x
  return __builtin_fmaf(rest, -off * kLn2f, rest);
}

// What a sum under x weighs under x_all >= x.
__device__ __forceinline__ float weight(float x, float x_all, float scale) {
  return x == x_all ? 1.0f : __builtin_amdgcn_exp2f((x - x_all) * scale);
}

// Two sets' (x, sum over all but x) as one.  That of nothing is (-inf, -1).
__device__ __forceinline__ float2 joined(float2 a, float2 b, float scale) {
  const float2 top = b.x > a.x ? b : a, low = b.x > a.x ? a : b;
  return make_float2(fmaxf(a.x, b.x), top.y + (1.0f + low.y) * weight(low.x, top.x, scale));
}

// What the backward needs of a row, f the factor of its loss's gradient (held
// scale included): ds = share 2^(s log2 e - top) for every column but the label's, label there.
struct __attribute__((aligned(16))) RowInfo {
  float top;    // x scale, rounded
  float share;  // f / sum, and 2^(top - x scale)
  float label;  // f (p_t - 1)
  int target;   // -1: none in the vocabulary, or the row does not count
};

// fp16 (and fp32's planes) have 2^-14 as their least normal number: ds (at most 1
// in magnitude after the division by the largest g) is held times 2^15, so that
// probabilities down to 2^-29 keep all their bits.  bf16 has fp32's exponents and
// needs no scale.  Rounding ds to 16 bits adds an error of the size of the
// results' own rounding to the same type; fp32's three planes keep 22 bits of
// probabilities down to 2^-51, and an error of 2^-62.
template <typename T>
struct Held {
  static constexpr float kScale = 1.0f;
};
template <>
struct Held<_Float16> {
  static constexpr float kScale = 32768.0f;
};

// A gradient from its sum of held ds: alpha is the gradient's factor without the
// held scale, unit the other operand's (fp32; else null).  The power of two
// first, and the factors' product in 64 bits: none of them leaves fp32's range unless the gradient does.
template <typename T>
__device__ __forceinline__ float gradient_of(float sum, float factor) {
  return sum * (1.0f / Held<T>::kScale) * factor;
}
__device__ __forceinline__ float factor_of(const double* alpha, const float* unit) {
  return (float)(unit ? *alpha * (double)*unit : *alpha);
}

}  // namespace gs_xent
