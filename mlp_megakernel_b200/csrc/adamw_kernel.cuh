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
// thread block reads its tensor's `ticks` and then adds the number of its
// chunks to them, so the steps taken are ticks / (chunks of the tensor),
// before, during and after a launch.
//
// Layout: a warp steps blocks of 256 elements, 8 a lane, so a block's scales
// need shuffles alone; 8 warps have a chunk of 2048.  Products are taken two at
// a time.
//
// 32-bit state: memory bounds it.  A thread block has two chunks, one after
// the other; 4 thread blocks an SM overlap each other's loads, and fp32 values
// move 32 bytes a lane.  113 million fp16 parameters with fp32 copies: 477 us,
// 6.65 TB/s.  Measured against it: all loads of both chunks first, 3 thread
// blocks an SM, 536 us; 16-byte accesses 506; 5 thread blocks 503; 8 chunks 493.
//
// 8-bit state: 10 bytes an element and some 49 instructions (a root, a
// quotient, four conversions), so memory bounds it only while the warps hardly
// wait.  A thread block has up to 16 chunks, one after the other, and each
// thread copies its part of the next ones to its own slots of shared memory
// (cp.async): 3 under way.  233 million bf16 parameters: 419 us, 5.6 TB/s; 480
// us back to back for seconds, when the power cap takes the clock from 1.97 to
// 1.7 GHz.  Measured against it (438 us then): all loads of two chunks first 516
// us; one chunk ahead in registers 760 (the loads were put off behind the work
// they were to overlap); 4 thread blocks an SM with their registers spilling
// 516, 3 without 438; 4 copies under way 442.
#pragma once
#include <type_traits>

#include "pdl.cuh"
#include "vec.cuh"

namespace mlpk {

constexpr int kAdamBlock = 256;    // elements that share a scale: 8 a lane
constexpr int kAdamThreads = 256;
constexpr int kAdamChunk = 2048;   // 8 elements a thread
constexpr int kAdamStages8 = 3;    // chunks under way with the 8-bit state
constexpr int kAdamChunks32 = 2;   // of a thread block with the 32-bit state

struct AdamTensor {
  void* p;
  const void* g;
  int64_t n;
  int64_t off;   // of its state, in elements (a multiple of kAdamBlock)
  int32_t cta0;  // the thread blocks before its first
  int32_t tick;  // its place in ticks
};

struct AdamArgs {
  float2 b1, b1c, b2, b2c, eps;  // twice each; b1c = 1 - b1, b2c = 1 - b2
  float lr, wd, lnb1, lnb2;      // lnb1 = ln b1, lnb2 = ln b2
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
  int per;  // chunks of a thread block
};

template <int CAP>
struct AdamTable {
  AdamTensor t[CAP];
};

// The tensor of this thread block: the last one whose cta0 is not above it.
template <int CAP>
__device__ __forceinline__ const AdamTensor& adam_tensor(const AdamTable<CAP>& table, int count) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (table.t[mid].cta0 <= static_cast<int>(blockIdx.x)) lo = mid;
    else hi = mid - 1;
  }
  return table.t[lo];
}

// What a thread of the block has of its tensor: its first element and what is
// left from there to the tensor's end (at or below 0: only other lanes of its
// block of 256 have some).
struct AdamPart {
  int64_t first;  // chunk of the thread block
  int64_t chunks;
  int mine;  // chunks of the thread block
  int64_t i0;
  int left;
  bool aligned;
  __device__ AdamPart(const AdamTensor& t, int per) {
    chunks = (t.n + kAdamChunk - 1) / kAdamChunk;
    first = (static_cast<int64_t>(blockIdx.x) - t.cta0) * per;
    mine = static_cast<int>(min(static_cast<int64_t>(per), chunks - first));
    i0 = first * kAdamChunk + threadIdx.x * 8;
    left = static_cast<int>(min(t.n - i0, static_cast<int64_t>(1 << 30)));
    aligned = ((reinterpret_cast<uintptr_t>(t.p) | reinterpret_cast<uintptr_t>(t.g)) & 15u) == 0;
  }
};

__device__ __forceinline__ unsigned long long adam_ticks(const AdamArgs& a, const AdamTensor& t) {
  unsigned long long v;  // read before this thread block's addition
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(a.ticks + t.tick) : "memory");
  return v;
}

// The step's factors, twice each.
struct AdamFactors {
  float2 minus_step, rcorr, keep, gs;
  bool scaled;  // gs is not 1
};
// Thread 0 finds the factors, counts the step, and says whether to skip it.
__device__ __forceinline__ bool adam_factors(const AdamArgs& a, const AdamTensor& t, const AdamPart& part,
                                             unsigned long long ticks, AdamFactors& f) {
  __shared__ float scalars[4];
  __shared__ bool skip;
  if (threadIdx.x == 0) {
    skip = a.found_inf && *a.found_inf != 0.0f;
    if (!skip)
      asm volatile("red.relaxed.gpu.global.add.u64 [%0], %1;" ::"l"(a.ticks + t.tick),
                   "l"(static_cast<unsigned long long>(part.mine))
                   : "memory");
    const unsigned long long chunks = static_cast<unsigned long long>(part.chunks);
    const unsigned long long taken =
        (ticks | chunks) >> 32 ? ticks / chunks : static_cast<uint32_t>(ticks) / static_cast<uint32_t>(chunks);
    const float step = static_cast<float>(taken + 1);
    const float lr = a.lr_ptr ? *a.lr_ptr : a.lr;
    scalars[0] = lr / expm1f(step * a.lnb1);  // below 0
    scalars[1] = 1.0f / sqrtf(-expm1f(step * a.lnb2));
    scalars[2] = 1.0f - lr * a.wd;
    scalars[3] = (a.maximize ? -1.0f : 1.0f) * (a.grad_scale ? 1.0f / *a.grad_scale : 1.0f);
  }
  __syncthreads();
  f.minus_step = make_float2(scalars[0], scalars[0]);
  f.rcorr = make_float2(scalars[1], scalars[1]);
  f.keep = make_float2(scalars[2], scalars[2]);
  f.gs = make_float2(scalars[3], scalars[3]);
  f.scaled = scalars[3] != 1.0f;
  return skip;
}

// Two elements.
__device__ __forceinline__ void adam_update(const AdamArgs& a, const AdamFactors& f, float2& p, float2 g, float2& m,
                                            float2& v, float2& r) {
  const float2 x = f.scaled ? mul2(g, f.gs) : g;
  m = add2(mul2(m, a.b1), mul2(x, a.b1c));
  v = add2(mul2(v, a.b2), mul2(mul2(x, x), a.b2c));
  r = make_float2(__fsqrt_rn(v.x), __fsqrt_rn(v.y));
  // The quotient to within 2 units of its last place: nothing but p depends on
  // it.  r is 0 or the root of a number above 2^-150.
  const float2 d = __ffma2_rn(r, f.rcorr, a.eps);
  const float2 u = mul2(m, make_float2(fast_reciprocal(d.x), fast_reciprocal(d.y)));
  p = __ffma2_rn(u, f.minus_step, mul2(p, f.keep));
}

// 8 values from p, or element by element what is `here`.
template <class T>
__device__ __forceinline__ Raw<T, 8> adam_load(const T* p, bool whole, int here) {
  if (whole) return load_raw<T, 8>(p);
  Raw<T, 8> r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r.v[e] = e < here ? p[e] : from_float<T>(0.0f);
  return r;
}
template <class T>
__device__ __forceinline__ void adam_store(T* p, const float2 (&f)[4], bool whole, int here) {
  if (whole) {
    store_vec2<T, 8>(p, f);
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (2 * e < here) p[2 * e] = from_float<T>(f[e].x);
    if (2 * e + 1 < here) p[2 * e + 1] = from_float<T>(f[e].y);
  }
}

template <class P, class G, bool MASTER, int CAP>
__global__ void __launch_bounds__(kAdamThreads, 4)
    adamw32_kernel(const __grid_constant__ AdamTable<CAP> table, const __grid_constant__ AdamArgs a) {
  using Param = typename std::conditional<MASTER, float, P>::type;
  constexpr int N = kAdamChunks32;
  pdl_enter();
  const AdamTensor& t = adam_tensor(table, a.count);
  const unsigned long long ticks = threadIdx.x == 0 ? adam_ticks(a, t) : 0;
  const AdamPart part(t, N);
  const int lane = threadIdx.x % 32;
  P* p = static_cast<P*>(t.p) + part.i0;
  const G* g = static_cast<const G*>(t.g) + part.i0;
  float* sm = static_cast<float*>(a.m) + t.off + part.i0;
  float* sv = static_cast<float*>(a.v) + t.off + part.i0;
  float* master = MASTER ? a.master + t.off + part.i0 : nullptr;
  AdamFactors f;
  if (adam_factors(a, t, part, ticks, f)) return;
#pragma unroll 1
  for (int k = 0; k < N; ++k) {
    const int ahead = k * kAdamChunk, here = part.left - ahead;
    if (here + lane * 8 <= 0) break;  // the whole warp, at the tensor's end
    const bool whole = part.aligned && here >= 8;
    Raw<Param, 8> rp;
    const Raw<G, 8> rg = adam_load(g + ahead, whole, here);
    if constexpr (MASTER) rp = load_32b(master + ahead);
    else rp = adam_load(p + ahead, whole, here);
    const Raw<float, 8> rm = load_32b(sm + ahead), rv = load_32b(sv + ahead);
    float2 pf[4], gf[4], m[4], v[4], r;
    unpack2(rp, pf);
    unpack2(rg, gf);
    unpack2(rm, m);
    unpack2(rv, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) adam_update(a, f, pf[e], gf[e], m[e], v[e], r);
    adam_store(p + ahead, pf, whole, here);
    if constexpr (MASTER) store_32b(master + ahead, pf);
    store_32b(sm + ahead, m);
    store_32b(sv + ahead, v);
  }
}

// A thread's slot of one chunk: 16-byte pieces of the parameters and the
// gradients, one of the 8 values each of m and r, and the scale (m's in lanes 0
// to 15, r's in the others).
template <class P, class G, bool MASTER>
struct AdamSlots {
  using Param = typename std::conditional<MASTER, float, P>::type;
  static constexpr int P16 = sizeof(Param) / 2, G16 = sizeof(G) / 2, PIECES = P16 + G16 + 1;
  static constexpr int STAGE = kAdamThreads * (PIECES * 16 + 4);  // bytes
  static constexpr int BYTES = kAdamStages8 * STAGE;
};

template <class P, class G, bool MASTER, int CAP>
__global__ void __launch_bounds__(kAdamThreads, 3)
    adamw8_kernel(const __grid_constant__ AdamTable<CAP> table, const __grid_constant__ AdamArgs a) {
  using S = AdamSlots<P, G, MASTER>;
  using Param = typename S::Param;
  extern __shared__ __align__(16) uint8_t slots[];
  pdl_enter();
  const AdamTensor& t = adam_tensor(table, a.count);
  const unsigned long long ticks = threadIdx.x == 0 ? adam_ticks(a, t) : 0;
  const AdamPart part(t, a.per);
  const int lane = threadIdx.x % 32;
  const int64_t s0 = t.off + part.i0;
  P* p = static_cast<P*>(t.p) + part.i0;
  const G* g = static_cast<const G*>(t.g) + part.i0;
  uint8_t* sm = static_cast<uint8_t*>(a.m) + s0;
  uint8_t* sr = static_cast<uint8_t*>(a.v) + s0;
  float* scales = (lane < 16 ? a.m_scale : a.v_scale) + s0 / kAdamBlock;
  float* master = MASTER ? a.master + s0 : nullptr;
  const Param* pr;  // where the parameters are read
  if constexpr (MASTER) pr = master;
  else pr = p;

  // A stage's slots: the thread's 16-byte pieces, 16 * kAdamThreads apart, and
  // its scale.  `stage` is the stage's offset in bytes.
  constexpr int SCALES = S::PIECES * kAdamThreads * 16;
  const uint32_t piece0 = smem_address(slots) + threadIdx.x * 16, scale0 = smem_address(slots) + SCALES + threadIdx.x * 4;
  // Copies chunk c to its slots.  A thread at the tensor's end, or of an
  // unaligned tensor, leaves out what it will read element by element.
  auto fetch = [&](int c, int stage) {
    const int ahead = c * kAdamChunk, here = part.left - ahead;
    if (c < part.mine && here + lane * 8 > 0) {  // the whole warp
      const bool whole = part.aligned && here >= 8;
      const uint32_t to = piece0 + stage;
      if (MASTER || whole) {
#pragma unroll
        for (int k = 0; k < S::P16; ++k)
          cp_async16(to + k * kAdamThreads * 16, reinterpret_cast<const uint4*>(pr + ahead) + k);
      }
      if (whole) {
#pragma unroll
        for (int k = 0; k < S::G16; ++k)
          cp_async16(to + (S::P16 + k) * kAdamThreads * 16, reinterpret_cast<const uint4*>(g + ahead) + k);
      }
      cp_async_small<8>(to + (S::P16 + S::G16) * kAdamThreads * 16, sm + ahead);
      cp_async_small<8>(to + (S::P16 + S::G16) * kAdamThreads * 16 + 8, sr + ahead);
      cp_async_small<4>(scale0 + stage, scales + ahead / kAdamBlock);
    }
    cp_async_commit();
  };
  auto read16 = [&](auto& raw, int stage, int first) {
#pragma unroll
    for (int k = 0; k < static_cast<int>(sizeof(raw) / 16); ++k)
      reinterpret_cast<uint4*>(&raw)[k] =
          *reinterpret_cast<const uint4*>(slots + stage + ((first + k) * kAdamThreads + threadIdx.x) * 16);
  };
#pragma unroll
  for (int k = 0; k < kAdamStages8; ++k) fetch(k, k * S::STAGE);
  AdamFactors f;
  if (adam_factors(a, t, part, ticks, f)) {
    cp_async_wait<0>();
    return;
  }

  int stage = 0;
  for (int c = 0; c < part.mine; ++c) {
    cp_async_wait<kAdamStages8 - 1>();
    const int ahead = c * kAdamChunk, here = part.left - ahead;
    if (here + lane * 8 <= 0) break;  // the whole warp, at the tensor's end
    const bool whole = part.aligned && here >= 8;
    float2 pf[4], gf[4], m[4], v[4], r[4];
    Raw<Param, 8> p8;
    Raw<G, 8> g8;
    Raw<uint16_t, 8> mr;
    if (MASTER || whole) read16(p8, stage, 0);
    else p8 = adam_load(pr + ahead, false, here);
    if (whole) read16(g8, stage, S::P16);
    else g8 = adam_load(g + ahead, false, here);
    read16(mr, stage, S::P16 + S::G16);
    float scale = *reinterpret_cast<const float*>(slots + stage + SCALES + threadIdx.x * 4);
    const float ms = __shfl_sync(0xffffffffu, scale, 0), rs = __shfl_sync(0xffffffffu, scale, 16);
    unpack2(p8, pf);
    unpack2(g8, gf);
    unpack_fp8<8>(*reinterpret_cast<const Raw<uint16_t, 4>*>(mr.v), m);
    unpack_fp8<8>(*reinterpret_cast<const Raw<uint16_t, 4>*>(mr.v + 4), v);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      m[e] = mul2(m[e], make_float2(ms, ms));
      v[e] = mul2(v[e], make_float2(rs, rs));
      v[e] = mul2(v[e], v[e]);
    }
    fetch(c + kAdamStages8, stage);
    stage = stage + S::STAGE == S::BYTES ? 0 : stage + S::STAGE;
    float mmax = 0.0f, rmax = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      adam_update(a, f, pf[e], gf[e], m[e], v[e], r[e]);
      mmax = max_abs(mmax, m[e].x, m[e].y);
      rmax = max_abs(rmax, r[e].x, r[e].y);
    }
    adam_store(p + ahead, pf, whole, here);
    if constexpr (MASTER) store_vec2<float, 8>(master + ahead, pf);

    // Lanes 0 to 15 find the block's largest |m|, the others its largest r,
    // and each half that scale and its reciprocal.
    const bool low = lane < 16;
    float top = max_nan(low ? mmax : rmax, __shfl_xor_sync(0xffffffffu, low ? rmax : mmax, 16));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    float inv;
    scale = fp8_scale(top, &inv);
    const float mi = __shfl_sync(0xffffffffu, inv, 0), ri = __shfl_sync(0xffffffffu, inv, 16);
    Raw<uint16_t, 4> mq, rq;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      mq.v[e] = to_fp8x2(mul2(m[e], make_float2(mi, mi)));
      rq.v[e] = to_fp8x2(mul2(r[e], make_float2(ri, ri)));
    }
    // The smallest code for an r above 0 that was rounded to 0 (unless the
    // whole block is): only if one of the 8 codes, all below 128, is 0.
    uint32_t zero = 0;
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      const uint32_t four = rq.v[e] | static_cast<uint32_t>(rq.v[e + 1]) << 16;
      zero |= (four - 0x01010101u) & ~four & 0x80808080u;
    }
    if (zero && ri > 0.0f) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if ((rq.v[e] & 0xffu) == 0 && r[e].x > 0.0f) rq.v[e] |= 1u;
        if ((rq.v[e] >> 8) == 0 && r[e].y > 0.0f) rq.v[e] |= 0x100u;
      }
    }
    *reinterpret_cast<Raw<uint16_t, 4>*>(sm + ahead) = mq;
    *reinterpret_cast<Raw<uint16_t, 4>*>(sr + ahead) = rq;
    if (lane % 16 == 0) scales[ahead / kAdamBlock] = scale;
  }
}

}  // namespace mlpk
