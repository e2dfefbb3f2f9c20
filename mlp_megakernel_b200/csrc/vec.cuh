// Element types and vector access of the block kernels (norm, experts,
// AdamW): fp16, bf16 and fp32 values are held as fp32 in registers, and move in
// vectors of 16 bytes (32 for AdamW's fp32 state) or, where a row of the experts
// does not allow that, of 4 bytes or one element.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>
#include <type_traits>

namespace mlpk {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Round to nearest even.
template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Elements of a 16-byte vector.
template <class T>
constexpr int kVecOf = 16 / static_cast<int>(sizeof(T));

// VEC elements as they lie in memory.  VEC is 1, or any count whose bytes are
// a multiple of 8 (the access is aligned to min(16, bytes)).
template <class T, int VEC>
struct alignas(VEC * sizeof(T) >= 16 ? 16 : VEC * sizeof(T)) Raw {
  T v[VEC];
};

template <class T, int VEC>
__device__ __forceinline__ Raw<T, VEC> load_raw(const T* p) {
  return *reinterpret_cast<const Raw<T, VEC>*>(p);
}

// Two values at a time: one instruction a value to widen, one for two to round.
__device__ __forceinline__ float2 to_float2(__half2 v) { return __half22float2(v); }
__device__ __forceinline__ float2 to_float2(__nv_bfloat162 v) { return __bfloat1622float2(v); }
template <class T>
struct Pair;
template <>
struct Pair<__half> {
  using type = __half2;
  static __device__ __forceinline__ type round(float a, float b) { return __floats2half2_rn(a, b); }
};
template <>
struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static __device__ __forceinline__ type round(float a, float b) { return __floats2bfloat162_rn(a, b); }
};

// Two values rounded for a backward pass to read, as they lie in memory: a finite
// one beyond the type's largest becomes that (rounded to infinity, it would make
// a NaN of a derivative that is 0 there); infinities and NaN stay.  Infinity less
// one, as a whole number, is the largest value of its sign.
template <class T>
constexpr float kRoundsToInfinity = std::is_same_v<T, __half> ? 65520.0f : 3.3961775292304601e+38f;  // and what is above
template <class T>
__device__ __forceinline__ uint32_t round_pair(float a, float b) {
  const typename Pair<T>::type v = Pair<T>::round(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <class T>
__device__ __forceinline__ uint32_t kept_pair(float a, float b) {
  uint32_t p = round_pair<T>(a, b);
  const float infinity = __uint_as_float(0x7f800000u);
  if (fabsf(a) >= kRoundsToInfinity<T> && fabsf(a) < infinity) p -= 1;
  if (fabsf(b) >= kRoundsToInfinity<T> && fabsf(b) < infinity) p -= 0x10000u;
  return p;
}
// Whether some of N values need that (or are infinite): one instruction for two
// values and a branch for all.  kept_pair's own tests for each of them cost the kernels
// that their epilogue bounds more (bf16, us, without any, this way, kept_pair for all:
// gated forward 20011 x 256 x 2816 84, 84, 95; linear 16384 x 512 x 4096 silu 94, 98,
// 105; 5003 x 1000 x 2056 33.8, 34.0, 34.5).
template <class T, int N>
__device__ __forceinline__ bool some_round_to_infinity(const float (&v)[N]) {
  static_assert(N % 8 == 0, "four maxima side by side, for the latency's sake");
  const auto most = [](float a, float b, float c) {  // of the magnitudes; a NaN is passed over
    float m;
    asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
    return m;
  };
  float m[4] = {};
#pragma unroll
  for (int i = 0; i < N; i += 2) m[i / 2 % 4] = i < 8 ? most(v[i], v[i], v[i + 1]) : most(m[i / 2 % 4], v[i], v[i + 1]);
  return most(most(m[0], m[1], m[2]), m[3], m[3]) >= kRoundsToInfinity<T>;
}

template <class T, int VEC>
__device__ __forceinline__ void unpack(const Raw<T, VEC>& r, float (&f)[VEC]) {
  if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {
    const typename Pair<T>::type* p = reinterpret_cast<const typename Pair<T>::type*>(r.v);
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) {
      const float2 v = to_float2(p[e]);
      f[2 * e] = v.x;
      f[2 * e + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = to_float(r.v[e]);
  }
}

template <class T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[VEC]) {
  Raw<T, VEC> r;
  if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {
    typename Pair<T>::type* q = reinterpret_cast<typename Pair<T>::type*>(r.v);
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) q[e] = Pair<T>::round(f[2 * e], f[2 * e + 1]);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) r.v[e] = from_float<T>(f[e]);
  }
  *reinterpret_cast<Raw<T, VEC>*>(p) = r;
}

// 8 fp32 values in one access (p is 32-byte aligned): two of 16 bytes each
// touch every sector of a warp's values twice.
__device__ __forceinline__ Raw<float, 8> load_32b(const float* p) {
  Raw<float, 8> r;
  asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(r.v[0]), "=f"(r.v[1]), "=f"(r.v[2]), "=f"(r.v[3]), "=f"(r.v[4]), "=f"(r.v[5]), "=f"(r.v[6]),
                 "=f"(r.v[7])
               : "l"(p)
               : "memory");
  return r;
}
__device__ __forceinline__ void store_32b(float* p, const float2 (&f)[4]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(f[0].x), "f"(f[0].y),
               "f"(f[1].x), "f"(f[1].y), "f"(f[2].x), "f"(f[2].y), "f"(f[3].x), "f"(f[3].y)
               : "memory");
}

// A 16-byte copy from global to shared memory that the thread waits for later;
// `bytes` of it are read, the rest are zeros.  A thread that reads back only
// what it copied itself needs no barrier, just cp_async_wait.
__device__ __forceinline__ uint32_t smem_address(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void cp_async16(uint32_t smem, const void* global, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(global), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t smem, const void* global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(global) : "memory");
}
template <int BYTES>  // 4 or 8
__device__ __forceinline__ void cp_async_small(uint32_t smem, const void* global) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem), "l"(global), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Until all but the N youngest groups of this thread have arrived.
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void cp_async_wait_upto(int n) {  // n from 0 to 3
  if (n >= 3) cp_async_wait<3>();
  else if (n == 2) cp_async_wait<2>();
  else if (n == 1) cp_async_wait<1>();
  else cp_async_wait<0>();
}

// Two products in one instruction, each rounded on its own.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(d)
      : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}
// Two sums, one at a time: a sum of pairs behind products of pairs came out
// contracted (a product not rounded).
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  return make_float2(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y));
}

// The values of a vector as pairs.
template <class T, int VEC>
__device__ __forceinline__ void unpack2(const Raw<T, VEC>& r, float2 (&f)[VEC / 2]) {
  float v[VEC];
  unpack(r, v);
#pragma unroll
  for (int e = 0; e < VEC / 2; ++e) f[e] = make_float2(v[2 * e], v[2 * e + 1]);
}
template <class T, int VEC>
__device__ __forceinline__ void store_vec2(T* p, const float2 (&f)[VEC / 2]) {
  float v[VEC];
#pragma unroll
  for (int e = 0; e < VEC / 2; ++e) {
    v[2 * e] = f[e].x;
    v[2 * e + 1] = f[e].y;
  }
  store_vec<T, VEC>(p, v);
}

// The 8-bit type: 4 exponent bits, 3 of mantissa (e4m3), largest value 448,
// smallest positive one 2^-9.
constexpr float kFp8Max = 448.0f;

// Rounded to e4m3 (to nearest even, NaN kept, magnitudes above 448 clipped).
__device__ __forceinline__ uint16_t to_fp8x2(float2 f) { return __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3); }

// VEC values of the 8-bit type as fp32 (exact).
template <int VEC>
__device__ __forceinline__ void unpack_fp8(const Raw<uint16_t, VEC / 2>& r, float2 (&f)[VEC / 2]) {
#pragma unroll
  for (int e = 0; e < VEC / 2; ++e)
    f[e] = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(r.v[e], __NV_E4M3)));
}

// The largest magnitude of a, b and c; a NaN stays.
__device__ __forceinline__ float max_abs(float a, float b, float c) {
  float m;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
// 1 / v to within a unit of the last place; v is 0 or a normal number.
__device__ __forceinline__ float fast_reciprocal(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Both correctly rounded by one step with a fused remainder (P. Markstein,
// "Computation of elementary functions on the IBM RISC System/6000 processor",
// 1990), in less than the compiler's division, which has to take any operands.
// 1 / v; v and 1 / v are normal numbers.
__device__ __forceinline__ float reciprocal(float v) {
  const float r = fast_reciprocal(v);
  return fmaf(r, fmaf(-v, r, 1.0f), r);
}
// a / b for a whole number b and its correctly rounded reciprocal; a may be
// infinite or NaN (the remainder is NaN then).
__device__ __forceinline__ float quotient(float a, float b, float reciprocal_b) {
  const float q = a * reciprocal_b, rest = fmaf(-q, b, a);
  return rest == rest ? fmaf(rest, reciprocal_b, q) : q;
}

// |v| as an unsigned whole number: ordered like |v|, with a NaN above
// infinity, so a maximum over it keeps a NaN.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The scale of a group of 8-bit values whose largest magnitude is `amax` (the
// product with 1 / 448 as fp32 holds it), and what to multiply by before the
// rounding: the scale's reciprocal, rounded once.  A scale below
// the smallest normal number has no finite reciprocal (and zero times infinity
// would put NaN into the group's zeros): such a group is all zeros.
__device__ __forceinline__ float fp8_scale(float amax, float* inv) {
  float scale = amax * (1.0f / kFp8Max);
  if (scale < 1.17549435e-38f) scale = 0.0f;
  *inv = scale > 0.0f && scale <= 3.402823466e+38f ? reciprocal(scale) : 0.0f;
  return scale;
}

}  // namespace mlpk
