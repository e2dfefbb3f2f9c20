// The activations of the feed-forward products and their derivatives, in fp32.
//
// sigmoid(z) = 1 / (1 + 2^(-z log2 e)): one ex2 and one reciprocal, each off by
// about 2 units of its last place; the product z log2 e adds |z| 2^-24, so an
// output in 16 bits is the correctly rounded one but next to ties.
//   silu      z s            s + z s (1 - s),        s = sigmoid(z)
//   gelu_tanh z s            s + z s (1 - s) p'(z),  s = sigmoid(p), p = 2 sqrt(2 / pi) (z + 0.044715 z^3),
//             which is 0.5 z (1 + tanh(p / 2))
//   softplus  max(z, 0) + log1p(e^-|z|)  (softplus.cuh's polynomial, 1/8 of fp16's half step)
// relu's derivative is 0 at 0.  A NaN stays a NaN, in values and derivatives.
#pragma once
#include <type_traits>

#include "softplus.cuh"
#include "vec.cuh"

namespace mlpk {

enum Act : int { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGeluTanh = 3, kActSoftplus = 4, kActSigmoid = 5 };

constexpr float kGeluA = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluB = 0.044715f;

__device__ __forceinline__ float sigmoid_f32(float z) { return fast_reciprocal(1.0f + ex2_approx(-kLog2e * z)); }

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == kActRelu) return z < 0.0f ? 0.0f : z;
  if constexpr (ACT == kActSilu) return z * sigmoid_f32(z);
  if constexpr (ACT == kActGeluTanh) return z * sigmoid_f32(kGeluA * fmaf(kGeluB * z, z * z, z));
  if constexpr (ACT == kActSoftplus) return softplus_f32(z);
  if constexpr (ACT == kActSigmoid) return sigmoid_f32(z);
  return z;
}
// The value, and the derivative in `slope`.
template <int ACT>
__device__ __forceinline__ float act_both(float z, float& slope) {
  if constexpr (ACT == kActRelu) {
    slope = z > 0.0f ? 1.0f : z <= 0.0f ? 0.0f : z;
    return z < 0.0f ? 0.0f : z;
  }
  if constexpr (ACT == kActSilu || ACT == kActGeluTanh) {
    const float zz = z * z;
    const float s = sigmoid_f32(ACT == kActSilu ? z : kGeluA * fmaf(kGeluB * z, zz, z));
    const float v = z * s;
    const float rest = fmaf(-v, s, v);  // z s (1 - s)
    // p' stays finite (zz does not, above |z| = 1.8e19): z s (1 - s) is 0 long before.
    slope = ACT == kActSilu ? s + rest : fmaf(rest, fmaf(3.0f * kGeluA * kGeluB, fminf(zz, 1e30f), kGeluA), s);
    return v;
  }
  if constexpr (ACT == kActSoftplus) {
    slope = sigmoid_f32(z);
    return softplus_f32(z);
  }
  if constexpr (ACT == kActSigmoid) {
    const float s = sigmoid_f32(z);
    slope = fmaf(-s, s, s);
    return s;
  }
  slope = 1.0f;
  return z;
}

// f(ACT) for the activation of a launch: one branch for a whole run of values.
template <class F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  switch (act) {
    case kActRelu: f(std::integral_constant<int, kActRelu>{}); break;
    case kActSilu: f(std::integral_constant<int, kActSilu>{}); break;
    case kActGeluTanh: f(std::integral_constant<int, kActGeluTanh>{}); break;
    case kActSoftplus: f(std::integral_constant<int, kActSoftplus>{}); break;
    case kActSigmoid: f(std::integral_constant<int, kActSigmoid>{}); break;
    default: f(std::integral_constant<int, kActNone>{}); break;
  }
}

// The scale of a checkpoint's group of 8-bit values whose largest magnitude is
// `most`: the smallest power of two with most / scale <= 448 (2^-126 at least),
// NaN where a value is not finite.  448 is 1.75 x 2^8, so it is the exponent of
// `most` less 8, and one more above 1.75.  A power of two: v / scale is exact
// before its one rounding to e4m3, and q scale is exact in fp32 and bf16, so the
// restored operand of a product has no second rounding.
__device__ __forceinline__ float checkpoint_scale(float most, float* inv) {
  const uint32_t bits = __float_as_uint(most);
  if (bits >= 0x7f800000u) {  // infinity or NaN
    *inv = 1.0f;
    return __uint_as_float(0x7fc00000u);
  }
  const int e = static_cast<int>((bits + 0x1fffffu) >> 23) - 8;
  const uint32_t biased = static_cast<uint32_t>(e < 1 ? 1 : e);
  *inv = __uint_as_float((254u - biased) << 23);
  return __uint_as_float(biased << 23);
}

// Next to fp32's largest value e4m3 rounds up to 256 x 2^120, infinity as an fp32
// product.  A kernel that computes with such values reads them as 240 x 2^120, which
// is within 1/16 of the value too.  The largest scale is 2^120, so that one test for a
// group and a rare branch, before the values are widened, is all it takes (clipped
// after that, value by value, dz of relu from 8 bits took 132 us instead of 112, 16384
// x 8192 bf16).
constexpr float kLargestScale = 1.329227995784916e+36f;  // 2^120
__device__ __forceinline__ uint32_t below_256(uint32_t w) {  // 4 values
  const uint32_t far = ((w & 0x7f7f7f7fu) + 0x08080808u) & 0x80808080u;  // the magnitude's code is 0x78 or more
  const uint32_t mask = far - (far >> 7);
  return (w & ~mask) | (0x77777777u & mask);
}

}  // namespace mlpk
