// One AdamW step over many tensors in one launch, with the state in 32 bits
// or in 8.
//
// Per element, all in fp32, each operation rounded on its own (so that the
// 8-bit state does not depend on how a compiler contracts it):
//   m = b1 m + (1 - b1) g;   v = b2 v + (1 - b2) g g;   r = sqrt(v)
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (r / sqrt(1 - b2^t) + eps)
// 8-bit state: the elements of a tensor in blocks of 256; m and r (not v: half
// the range of exponents, and r is what the update divides by) are held as
// e4m3 times the block's scale, max / 448.  An r above zero is never rounded to
// zero: the update would divide by eps alone.  The update itself uses the m
// and r of before the rounding.
//
// The step count of a tensor is kept on the device, so that a CUDA graph of
// the step replays and a step skipped by `found_inf` does not count: every
// block adds 1 to its tensor's `ticks` after it has read them, so the steps
// taken are ticks / (blocks of the tensor), before, during and after a launch.
#pragma once
#include "pdl.cuh"
#include "vec.cuh"

namespace mlpk {

constexpr int kAdamBlock = 256;    // elements that share a scale: 8 a lane
constexpr int kAdamThreads = 256;
constexpr int kAdamChunk = 4096;   // elements of a thread block

struct AdamTensor {
  void* p;
  const void* g;
  int64_t n;
  int64_t off;     // of its state, in elements (a multiple of kAdamBlock)
  int32_t chunk0;  // the thread blocks before its first
  int32_t tick;    // its place in ticks
};

struct AdamArgs {
  float lr, b1, b1c, b2, b2c, eps, wd;  // b1c = 1 - b1, b2c = 1 - b2
  float lnb1, lnb2;                     // ln b1, ln b2
  int maximize;
  const float* lr_ptr;      // null: lr
  const float* grad_scale;  // null: 1; the gradients are divided by it
  const float* found_inf;   // null: 0; not 0 skips the step
  void* m;                  // fp32, or e4m3
  void* v;                  // fp32 v, or e4m3 r
  float* m_scale;
  float* v_scale;
  float* master;            // null: the parameters themselves
  unsigned long long* ticks;
  int count;
};

template <int CAP>
struct AdamTable {
  AdamTensor t[CAP];
};

template <class P, class G, bool BITS8, bool MASTER, int CAP>
__global__ void __launch_bounds__(kAdamThreads)
    adamw_kernel(const __grid_constant__ AdamTable<CAP> table, const __grid_constant__ AdamArgs a) {
  pdl_enter();
  if (a.found_inf && *a.found_inf != 0.0f) return;
  // The tensor of this thread block: the last one whose chunk0 is not above it.
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (table.t[mid].chunk0 <= static_cast<int>(blockIdx.x)) lo = mid;
    else hi = mid - 1;
  }
  const AdamTensor& t = table.t[lo];
  const int64_t chunk = static_cast<int64_t>(blockIdx.x) - t.chunk0;
  __shared__ float corr[2];
  if (threadIdx.x == 0) {
    const unsigned long long chunks = (t.n + kAdamChunk - 1) / kAdamChunk;
    const float step = static_cast<float>(atomicAdd(a.ticks + t.tick, 1ull) / chunks + 1);
    const float lr = a.lr_ptr ? *a.lr_ptr : a.lr;
    corr[0] = lr / -expm1f(step * a.lnb1);
    corr[1] = 1.0f / sqrtf(-expm1f(step * a.lnb2));
  }
  __syncthreads();
  const float step_size = corr[0], rcorr = corr[1];
  const float lr = a.lr_ptr ? *a.lr_ptr : a.lr;
  const float keep = 1.0f - lr * a.wd;
  const float gs = (a.maximize ? -1.0f : 1.0f) * (a.grad_scale ? 1.0f / *a.grad_scale : 1.0f);
  P* p = static_cast<P*>(t.p);
  const G* g = static_cast<const G*>(t.g);
  const bool aligned = ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g)) & 15u) == 0;

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int k = warp; k < kAdamChunk / kAdamBlock; k += kAdamThreads / 32) {
    const int64_t b0 = chunk * kAdamChunk + k * kAdamBlock;
    if (b0 >= t.n) break;
    const int64_t i = b0 + lane * 8, s = t.off + i;  // the state is padded to whole blocks
    const int left = static_cast<int>(min(static_cast<int64_t>(8), t.n - i));
    const bool whole = aligned && left == 8;
    float pf[8], gf[8], m[8], v[8], r[8];
    if (whole) {
      unpack(load_raw<G, 8>(g + i), gf);
      if constexpr (!MASTER) unpack(load_raw<P, 8>(p + i), pf);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        gf[e] = e < left ? to_float(g[i + e]) : 0.0f;
        if constexpr (!MASTER) pf[e] = e < left ? to_float(p[i + e]) : 0.0f;
      }
    }
    if constexpr (MASTER) unpack(load_raw<float, 8>(a.master + s), pf);
    if constexpr (BITS8) {
      const Raw<__nv_fp8_e4m3, 8> m8 = load_raw<__nv_fp8_e4m3, 8>(static_cast<__nv_fp8_e4m3*>(a.m) + s);
      const Raw<__nv_fp8_e4m3, 8> r8 = load_raw<__nv_fp8_e4m3, 8>(static_cast<__nv_fp8_e4m3*>(a.v) + s);
      const float ms = a.m_scale[s / kAdamBlock], rs = a.v_scale[s / kAdamBlock];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        m[e] = __fmul_rn(static_cast<float>(m8.v[e]), ms);
        v[e] = __fmul_rn(static_cast<float>(r8.v[e]), rs);
        v[e] = __fmul_rn(v[e], v[e]);
      }
    } else {
      unpack(load_raw<float, 8>(static_cast<float*>(a.m) + s), m);
      unpack(load_raw<float, 8>(static_cast<float*>(a.v) + s), v);
    }
    uint32_t mmax = 0, rmax = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = gf[e] * gs;
      m[e] = __fadd_rn(__fmul_rn(m[e], a.b1), __fmul_rn(x, a.b1c));
      v[e] = __fadd_rn(__fmul_rn(v[e], a.b2), __fmul_rn(__fmul_rn(x, x), a.b2c));
      r[e] = __fsqrt_rn(v[e]);
      pf[e] = pf[e] * keep - step_size * (m[e] / (r[e] * rcorr + a.eps));
      mmax = max(mmax, abs_bits(m[e]));
      rmax = max(rmax, abs_bits(r[e]));
    }
    if (whole) {
      store_vec<P, 8>(p + i, pf);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) p[i + e] = from_float<P>(pf[e]);
    }
    if constexpr (MASTER) store_vec<float, 8>(a.master + s, pf);
    if constexpr (BITS8) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        mmax = max(mmax, __shfl_xor_sync(0xffffffffu, mmax, o));
        rmax = max(rmax, __shfl_xor_sync(0xffffffffu, rmax, o));
      }
      float mi, ri;
      const float ms = fp8_scale(mmax, &mi), rs = fp8_scale(rmax, &ri);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        m[e] = __fmul_rn(m[e], mi);
        r[e] = r[e] > 0.0f && ri > 0.0f ? fmaxf(__fmul_rn(r[e], ri), kFp8Tiny) : __fmul_rn(r[e], ri);
      }
      store_fp8<8>(static_cast<uint8_t*>(a.m) + s, m);
      store_fp8<8>(static_cast<uint8_t*>(a.v) + s, r);
      if (lane == 0) {
        a.m_scale[s / kAdamBlock] = ms;
        a.v_scale[s / kAdamBlock] = rs;
      }
    } else {
      store_vec<float, 8>(static_cast<float*>(a.m) + s, m);
      store_vec<float, 8>(static_cast<float*>(a.v) + s, v);
    }
  }
}

}  // namespace mlpk
