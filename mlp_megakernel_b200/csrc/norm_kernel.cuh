// Root-mean-square norm with the residual's addition, its 8-bit output and
// its backward pass.
//
// Per row, all in fp32 from the loads on:
//   h = x + r;   s = rsqrt(mean_j h_j^2 + eps);   y_j = h_j s w_j
// y is computed from the unrounded h; h is rounded once, as it is stored.  The
// 8-bit output stores e4m3(y / scale) with scale = max|y| / 448 over the row
// or over each 128 columns.  Backward, from x, r and s (G = dL/dy):
//   n_j = h_j s;   c = mean_j G_j w_j n_j
//   dx_j = dr_j = s (G_j w_j - n_j c) + dL/dh_j;   dw_j = sum_rows G_j n_j
// It adds x and r again.  From the rounded h, dw's error would be half as large
// again (its own rounding and h's are of the same size); that would read 2 bytes
// less of the 18 that both passes move an element in 16 bits.
//
// What bounds it: memory; every value is read once and written once.  16,384
// rows of 4096 bf16 values with a residual: forward 96 us, 5.6 TB/s; backward
// 104 us, 6.5 TB/s, with dw's sum; 8,192 rows of 5120 to 8 bits in groups of 128:
// 56 us, 5.3 TB/s (53 with a reciprocal of the scale that is off by a unit of its
// last place in an eighth of the cases, which moves values next to a tie).
//
// Layout: TPR threads share a row, NV 16-byte vectors each (vector i of lane l
// is the row's vector i * TPR + l).  Up to 32 threads a row's sum is a warp
// shuffle and several rows share a block; above, a block has one row and sums
// through shared memory.  Blocks stay and loop over rows.  A thread copies its
// vectors of the next rows to its own slots of shared memory (cp.async) and
// reads them back itself: enough bytes are in flight whatever the registers
// hold, and no barrier guards the slots.  Rows whose slots do not fit (PIPE
// false) are read directly.  (One block a row with its loads in registers: 246
// us forward, 414 backward.)  The next row's s is loaded a row ahead (158 us
// without), and arithmetic is on pairs of values (132 us one at a time).
//
// A width that no vector divides (RAGGED): a row begins `shift` elements into
// an aligned vector of the tensor, its first and last vectors are shared with
// its neighbours, and a thread leaves out the elements that are not its row's.
// Blocks step by a multiple of VEC rows, so that `shift`, and with it each
// thread's columns, are the same in all rows of a block's row group.  (8,192
// rows of 2049 bf16 values with a residual: forward 28 us, 0.73 of the copy rate.)
#pragma once
#include "pdl.cuh"
#include "vec.cuh"

namespace mlpk {

constexpr int kNormThreads = 256;  // threads of a block of several rows
constexpr int kNormGroup = 128;    // columns that share a scale
constexpr int kNormMaxWidth = 32768;
constexpr int kNormStages = 4;     // rows that a thread has under way, at most

// Sum of v over the row's threads.  TPR > 32: `red` has two halves of 32 floats,
// one a warp (the others zero, norm_row_init), used in turn (`half`), so one
// barrier separates a write from the reads of the call before the last.
__device__ __forceinline__ void norm_row_init(float* red, int n, int tpr) {
  if (tpr <= 32) return;
  for (int k = threadIdx.x; k < n; k += blockDim.x) red[k] = 0.0f;
  __syncthreads();
}
__device__ __forceinline__ float norm_row_sum(float v, int tpr, float* red, int half) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < tpr) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (tpr <= 32) return v;
  red += half * 32;
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  // Every thread adds the warps' sums in the same order.
  v = 0.0f;
  for (int k = 0; k < tpr / 32; k += 4) {
    const float4 t = *reinterpret_cast<const float4*>(red + k);  // 32 floats a half: those of no warp stay zero
    v += (t.x + t.y) + (t.z + t.w);
  }
  return v;
}

// The largest v (not below 0) of the row's threads; a NaN stays.
__device__ __forceinline__ float norm_row_max(float v, int tpr, float* red, int half) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < tpr) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (tpr <= 32) return v;
  red += half * 32;
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  v = 0.0f;
  for (int k = 0; k < tpr / 32; k += 4) {
    const float4 t = *reinterpret_cast<const float4*>(red + k);
    v = max_abs(max_abs(v, t.x, t.y), t.z, t.w);
  }
  return v;
}

// A thread's vectors of the rows of its block's row group.  KIND: kRagged; kFull
// where a block has one row and every thread all its NV vectors (nothing to ask
// for each vector: a fifth of the instructions); else kPart.  Where it lies is
// arithmetic of no device, which tests/test_norm_copies.py goes over.
enum RowKind { kPart, kFull, kRagged };
template <class T, int NV, int KIND>
struct RowSpan {
  static constexpr bool RAGGED = KIND == kRagged;
  static constexpr int VEC = kVecOf<T>;
  int64_t total;  // elements of the tensor
  int64_t end;    // what begin() is below in the rows there are
  int width, tpr, lane, shift, nvec, step;  // step: elements from a vector to the thread's next

  // first_row: any row of the row group
  __host__ __device__ RowSpan(int64_t rows, int width_, int tpr_, int lane_, int64_t first_row)
      : total(rows * width_), width(width_), tpr(tpr_), lane(lane_) {
    shift = RAGGED ? static_cast<int>((first_row % VEC) * (width % VEC) % VEC) : 0;
    nvec = (width + shift + VEC - 1) / VEC;
    step = tpr * VEC;
    end = total + col(0);
  }
  __host__ __device__ bool has(int i) const { return KIND == kFull || i * tpr + lane < nvec; }
  __host__ __device__ int col(int i) const { return (i * tpr + lane) * VEC - shift; }  // of element 0; may be below 0
  // The thread's first element of a row, and element 0 of its vector i behind
  // it: multiples of VEC.
  __host__ __device__ int64_t begin(int64_t row) const { return row * width + col(0); }
  __host__ __device__ int64_t at(int64_t begin, int i) const { return begin + i * step; }
  __host__ __device__ bool owns(int i, int e) const {
    return !RAGGED || static_cast<unsigned>(col(i) + e) < static_cast<unsigned>(width);
  }
  __host__ __device__ bool whole(int i) const { return !RAGGED || (col(i) >= 0 && col(i) + VEC <= width); }
  // Whether there is such a row: only then do its vectors lie inside the tensor
  // (a ragged row's first one alone says nothing about the others).
  __host__ __device__ bool exists(int64_t begin) const { return begin < end; }
  // Bytes of the vector that lie inside the tensor.
  __host__ __device__ int bytes(int64_t begin, int i) const {
    if (!RAGGED) return 16;
    const int64_t left = total - at(begin, i);
    return left >= VEC ? 16 : static_cast<int>(left) * static_cast<int>(sizeof(T));
  }
  __device__ Raw<T, VEC> load(const T* p, int64_t begin, int i) const {
    if constexpr (RAGGED) {
      if (total - at(begin, i) < VEC) {
        Raw<T, VEC> r;
#pragma unroll
        for (int e = 0; e < VEC; ++e) r.v[e] = at(begin, i) + e < total ? p[at(begin, i) + e] : from_float<T>(0.0f);
        return r;
      }
    }
    return load_raw<T, VEC>(p + at(begin, i));
  }
  __device__ void store(T* p, int64_t begin, int i, const float2 (&f)[VEC / 2]) const {
    if (whole(i)) {
      store_vec2<T, VEC>(p + at(begin, i), f);
      return;
    }
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) {
      if (owns(i, 2 * e)) p[at(begin, i) + 2 * e] = from_float<T>(f[e].x);
      if (owns(i, 2 * e + 1)) p[at(begin, i) + 2 * e + 1] = from_float<T>(f[e].y);
    }
  }
  // Zeros in the place of what is not this row's.
  __device__ void mask(int i, float2 (&f)[VEC / 2]) const {
    if (whole(i)) return;
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) {
      if (!owns(i, 2 * e)) f[e].x = 0.0f;
      if (!owns(i, 2 * e + 1)) f[e].y = 0.0f;
    }
  }
  // The weight's values of the vector's columns; ones without a weight.
  template <class W>
  __device__ void weights(const W* w, int i, Raw<W, VEC>& r) const {
    if (!RAGGED && w) {
      r = load_raw<W, VEC>(w + col(i));
      return;
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) r.v[e] = w && owns(i, e) ? w[col(i) + e] : from_float<W>(1.0f);
  }
};

// A thread's weights: as floats where the registers allow it, else as they lie
// in memory.
template <class T, class W, int NV, bool FLOATS>
struct NormWeights {
  static constexpr int VEC = kVecOf<T>;
  Raw<W, VEC> raw[FLOATS ? 1 : NV];
  float2 f32[FLOATS ? NV : 1][VEC / 2];
  template <class Span>
  __device__ void load(const Span& span, const W* w) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (span.has(i)) {
        span.weights(w, i, raw[FLOATS ? 0 : i]);
        if constexpr (FLOATS) unpack2(raw[0], f32[i]);
      }
  }
  __device__ void get(int i, float2 (&f)[VEC / 2]) const {
    if constexpr (FLOATS) {
#pragma unroll
      for (int e = 0; e < VEC / 2; ++e) f[e] = f32[i][e];
    } else {
      unpack2(raw[i], f);
    }
  }
};

struct NormArgs {
  int64_t rows;
  int width;
  int tpr;  // threads of a row: a power of two up to 32, else a multiple of 32
  float eps;
  const void* x;
  const void* r;  // null: no residual
  const void* w;  // null: ones
  void* y;        // T, or e4m3 with FP8
  void* h;        // null: not stored
  float* rstd;    // null: not stored
  float* scale;   // FP8: [rows][groups]
  int group;      // FP8: columns that share a scale: 128, or 0 for the row
};

// Shared memory: 128 floats for the row sums, then with FP8, RAGGED and groups
// a maximum per group and row group, then the slots [stage][x, r][i][thread].
template <class T, class W, int NV, int KIND, bool PIPE, int MAXT, bool FP8>
__global__ void __launch_bounds__(MAXT, !FP8 ? 0 : MAXT == 256 ? (KIND == kRagged ? 3 : 4) : MAXT == 512 && NV == 2 ? 2 : 1)
    rms_norm_fwd_kernel(const NormArgs a, int stages, int slots_at) {
  using Span = RowSpan<T, NV, KIND>;
  constexpr bool RAGGED = Span::RAGGED;
  constexpr int VEC = Span::VEC, HALF = VEC / 2;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  float* red = reinterpret_cast<float*>(smem_raw);
  pdl_enter();
  const int lane = threadIdx.x % a.tpr, sub = threadIdx.x / a.tpr, subs = blockDim.x / a.tpr;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * subs + sub;
  const int64_t step = static_cast<int64_t>(gridDim.x) * subs;
  const Span span(a.rows, a.width, a.tpr, lane, first);
  const T* x = static_cast<const T*>(a.x);
  const T* r = static_cast<const T*>(a.r);
  const int streams = r ? 2 : 1;
  Raw<T, VEC>* slots = reinterpret_cast<Raw<T, VEC>*>(smem_raw + slots_at) + threadIdx.x;
  const int stage_slots = streams * NV * blockDim.x;  // `stage` counts them
  auto slot = [&](int stage, int stream, int i) { return slots + (stage + (stream * NV + i) * blockDim.x); };
  auto fetch = [&](int64_t begin, int stage) {
    if (span.exists(begin)) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (span.has(i)) {
          cp_async16(smem_address(slot(stage, 0, i)), x + span.at(begin, i), span.bytes(begin, i));
          if (r) cp_async16(smem_address(slot(stage, 1, i)), r + span.at(begin, i), span.bytes(begin, i));
        }
    }
    cp_async_commit();
  };
  const int64_t begin_step = step * a.width;
  int64_t begin = span.begin(first);
  if constexpr (PIPE)
    for (int k = 0; k < stages; ++k) fetch(begin + k * begin_step, k * stage_slots);
  NormWeights<T, W, NV, (NV <= 2 && !FP8)> w;
  w.load(span, static_cast<const W*>(a.w));
  norm_row_init(red, 128, a.tpr);

  int stage = 0, half = 0;
  const float width = static_cast<float>(a.width), inv_width = 1.0f / width;
  // Whole blocks loop together: the last rows' missing ones take part in the
  // shuffles and barriers.
  int64_t row = first;
  for (int64_t row0 = first - sub; row0 < a.rows; row0 += step, row += step, begin += begin_step, half ^= 1) {
    const bool live = KIND == kFull || row < a.rows;
    if constexpr (PIPE) cp_async_wait_upto(stages - 1);
    float2 h[NV][HALF];
    float2 sum2 = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int e = 0; e < HALF; ++e) h[i][e] = make_float2(0.0f, 0.0f);
      if (live && span.has(i)) {
        unpack2(PIPE ? *slot(stage, 0, i) : span.load(x, begin, i), h[i]);
        if (r) {
          float2 f[HALF];
          unpack2(PIPE ? *slot(stage, 1, i) : span.load(r, begin, i), f);
#pragma unroll
          for (int e = 0; e < HALF; ++e) h[i][e] = __fadd2_rn(h[i][e], f[e]);
        }
        span.mask(i, h[i]);
      }
#pragma unroll
      for (int e = 0; e < HALF; ++e) sum2 = __ffma2_rn(h[i][e], h[i][e], sum2);
    }
    if constexpr (PIPE) {
      fetch(begin + stages * begin_step, stage);
      stage = stage + stage_slots == stages * stage_slots ? 0 : stage + stage_slots;
    }
    // The mean is a quotient: as a product with a rounded 1 / width it is off by
    // a unit of its last place now and then.
    const float s = rsqrtf(quotient(norm_row_sum(sum2.x + sum2.y, a.tpr, red, half), width, inv_width) + a.eps);
    if (a.rstd && live && lane == 0) a.rstd[row] = s;
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (live && span.has(i)) {
        if (a.h) span.store(static_cast<T*>(a.h), begin, i, h[i]);
        float2 f[HALF];
        w.get(i, f);
#pragma unroll
        for (int e = 0; e < HALF; ++e) {
          h[i][e] = __fmul2_rn(__fmul2_rn(h[i][e], make_float2(s, s)), f[e]);
          if (FP8 && a.group == 0) amax = max_abs(amax, h[i][e].x, h[i][e].y);
        }
        if constexpr (!FP8) span.store(static_cast<T*>(a.y), begin, i, h[i]);
      }
    }
    if constexpr (FP8) {
      // Vector i times what its elements' groups ask for; elements from `edge`
      // on are of the next group.
      auto store = [&](int i, float inv0, float inv1, int edge) {
        uint8_t* q = static_cast<uint8_t*>(a.y) + span.at(begin, i);
        Raw<uint16_t, HALF> q8;
#pragma unroll
        for (int e = 0; e < HALF; ++e)
          q8.v[e] = to_fp8x2(__fmul2_rn(h[i][e], make_float2(2 * e < edge ? inv0 : inv1, 2 * e + 1 < edge ? inv0 : inv1)));
        if (span.whole(i)) {
          *reinterpret_cast<Raw<uint16_t, HALF>*>(q) = q8;
          return;
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (span.owns(i, e)) q[e] = static_cast<uint8_t>(q8.v[e / 2] >> (e % 2 * 8));
      };
      const int groups = (a.width + kNormGroup - 1) / kNormGroup;
      if (a.group == 0) {
        float inv;
        const float scale = fp8_scale(norm_row_max(amax, a.tpr, red + 64, half), &inv);
        if (live && lane == 0) a.scale[row] = scale;
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (live && span.has(i)) store(i, inv, inv, VEC);
      } else if constexpr (!RAGGED) {
        // The 128 / VEC lanes of a group are neighbours, or the row is narrower
        // than a group.
        constexpr int LANES = kNormGroup / VEC;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          float m = 0.0f;
#pragma unroll
          for (int e = 0; e < HALF; ++e) m = max_abs(m, h[i][e].x, h[i][e].y);
#pragma unroll
          for (int o = LANES / 2; o > 0; o >>= 1)
            if (o < a.tpr) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
          float inv;
          const float scale = fp8_scale(m, &inv);
          if (live && span.has(i)) {
            const int v = i * a.tpr + lane;
            if (v % LANES == 0) a.scale[row * groups + v / LANES] = scale;
            store(i, inv, inv, VEC);
          }
        }
      } else {
        // A vector may reach into two groups, and groups do not begin at a
        // lane: the maxima meet in shared memory (they do not depend on the
        // order; their bits are ordered as they are).
        uint32_t* gmax = reinterpret_cast<uint32_t*>(smem_raw + 512) + sub * groups;
        __syncthreads();
        for (int k = lane; k < groups; k += a.tpr) gmax[k] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (live && span.has(i)) {
            const int lo = max(span.col(i), 0) / kNormGroup, hi = (min(span.col(i) + VEC, a.width) - 1) / kNormGroup;
            const int edge = (lo + 1) * kNormGroup - span.col(i);
            float m0 = 0.0f, m1 = 0.0f;  // what is not the row's is zero
#pragma unroll
            for (int e = 0; e < HALF; ++e) {
              const float2 v = h[i][e];
              m0 = max_abs(m0, 2 * e < edge ? v.x : 0.0f, 2 * e + 1 < edge ? v.y : 0.0f);
              m1 = max_abs(m1, 2 * e < edge ? 0.0f : v.x, 2 * e + 1 < edge ? 0.0f : v.y);
            }
            atomicMax(gmax + lo, abs_bits(m0));
            if (hi != lo) atomicMax(gmax + hi, abs_bits(m1));
          }
        }
        __syncthreads();
        if (live)
          for (int k = lane; k < groups; k += a.tpr) {
            float inv;
            a.scale[row * groups + k] = fp8_scale(__uint_as_float(gmax[k]), &inv);
          }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (live && span.has(i)) {
            const int lo = max(span.col(i), 0) / kNormGroup, hi = (min(span.col(i) + VEC, a.width) - 1) / kNormGroup;
            float inv0, inv1;
            fp8_scale(__uint_as_float(gmax[lo]), &inv0);
            fp8_scale(__uint_as_float(gmax[hi]), &inv1);
            store(i, inv0, inv1, (lo + 1) * kNormGroup - span.col(i));
          }
        }
      }
    }
  }
}

struct NormBwdArgs {
  int64_t rows;
  int width;
  int tpr;
  const void* x;
  const void* r;  // null: no residual
  const float* rstd;
  const void* w;   // null: ones
  const void* gy;
  const void* gh;  // null: none
  void* dx;
  float* part;     // null: no weight gradient; else [gridDim.x][width]
};

// A block's threads keep their columns' share of dw in registers; the block's
// sum over its row groups (through shared memory, in order) is one row of
// `part`.  With 4 or more vectors a thread, a row's vectors are read from their
// slots twice (before and after the row's sum) instead of being kept in
// registers; rows without slots (PIPE false) are read from global memory, the
// second time from L2.
// Shared memory: 64 floats, then the slots [stage][x, gy, r, gh][i][thread], which
// the sum over the row groups takes over at the end.
template <class T, class W, int NV, int KIND, bool PIPE, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT == 256 ? 2 : 1) rms_norm_bwd_kernel(const NormBwdArgs a, int stages) {
  using Span = RowSpan<T, NV, KIND>;
  constexpr bool RAGGED = Span::RAGGED;
  constexpr int VEC = Span::VEC, HALF = VEC / 2;
  constexpr bool KEEP = NV <= 2;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  float* red = reinterpret_cast<float*>(smem_raw);
  pdl_enter();
  const int lane = threadIdx.x % a.tpr, sub = threadIdx.x / a.tpr, subs = blockDim.x / a.tpr;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * subs + sub;
  const int64_t step = static_cast<int64_t>(gridDim.x) * subs;
  const Span span(a.rows, a.width, a.tpr, lane, first);
  const T* in[4] = {static_cast<const T*>(a.x), static_cast<const T*>(a.gy), static_cast<const T*>(a.r),
                    static_cast<const T*>(a.gh)};
  const int streams = 2 + (a.r != nullptr) + (a.gh != nullptr);
  const int gh_slot = a.r ? 3 : 2;
  Raw<T, VEC>* slots = reinterpret_cast<Raw<T, VEC>*>(smem_raw + 256) + threadIdx.x;
  const int stage_slots = streams * NV * blockDim.x;  // `stage` counts them
  auto slot = [&](int stage, int stream, int i) { return slots + (stage + (stream * NV + i) * blockDim.x); };
  auto fetch = [&](int64_t begin, int stage) {
    if (span.exists(begin)) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (span.has(i)) {
          const int n = span.bytes(begin, i);
          cp_async16(smem_address(slot(stage, 0, i)), in[0] + span.at(begin, i), n);
          cp_async16(smem_address(slot(stage, 1, i)), in[1] + span.at(begin, i), n);
          if (in[2]) cp_async16(smem_address(slot(stage, 2, i)), in[2] + span.at(begin, i), n);
          if (in[3]) cp_async16(smem_address(slot(stage, gh_slot, i)), in[3] + span.at(begin, i), n);
        }
    }
    cp_async_commit();
  };
  const int64_t begin_step = step * a.width;
  int64_t begin = span.begin(first);
  if constexpr (PIPE)
    for (int k = 0; k < stages; ++k) fetch(begin + k * begin_step, k * stage_slots);
  float2 dw[NV][HALF];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < HALF; ++e) dw[i][e] = make_float2(0.0f, 0.0f);
  NormWeights<T, W, NV, KEEP> w;
  w.load(span, static_cast<const W*>(a.w));
  norm_row_init(red, 64, a.tpr);

  int half = 0, stage = 0;
  int64_t row = first;
  const float inv_width = 1.0f / static_cast<float>(a.width);
  float s_next = row < a.rows ? a.rstd[row] : 0.0f;
  for (int64_t row0 = first - sub; row0 < a.rows; row0 += step, row += step, begin += begin_step, half ^= 1) {
    const bool live = KIND == kFull || row < a.rows;
    const float s = s_next;  // the next row's is on its way while this one is worked on
    s_next = row + step < a.rows ? a.rstd[row + step] : 0.0f;
    if constexpr (PIPE) cp_async_wait_upto(stages - 1);
    // n and G w of vector i, and G
    auto terms = [&](int i, float2 (&n)[HALF], float2 (&gw)[HALF], float2 (&g)[HALF]) {
      unpack2(PIPE ? *slot(stage, 0, i) : span.load(in[0], begin, i), n);
      unpack2(PIPE ? *slot(stage, 1, i) : span.load(in[1], begin, i), g);
      if (in[2]) {
        float2 f[HALF];
        unpack2(PIPE ? *slot(stage, 2, i) : span.load(in[2], begin, i), f);
#pragma unroll
        for (int e = 0; e < HALF; ++e) n[e] = __fadd2_rn(n[e], f[e]);
      }
      span.mask(i, n);
      span.mask(i, g);
      float2 f[HALF];
      w.get(i, f);
#pragma unroll
      for (int e = 0; e < HALF; ++e) {
        n[e] = __fmul2_rn(n[e], make_float2(s, s));
        gw[e] = __fmul2_rn(g[e], f[e]);
      }
    };
    float2 n[KEEP ? NV : 1][HALF], gw[KEEP ? NV : 1][HALF], g[HALF];
    float2 sum2 = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (live && span.has(i)) {
        const int k = KEEP ? i : 0;
        terms(i, n[k], gw[k], g);
#pragma unroll
        for (int e = 0; e < HALF; ++e) {
          dw[i][e] = __ffma2_rn(g[e], n[k][e], dw[i][e]);
          sum2 = __ffma2_rn(gw[k][e], n[k][e], sum2);
        }
      }
    const float c = -norm_row_sum(sum2.x + sum2.y, a.tpr, red, half) * inv_width;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (live && span.has(i)) {
        const int k = KEEP ? i : 0;
        if constexpr (!KEEP) terms(i, n[k], gw[k], g);
#pragma unroll
        for (int e = 0; e < HALF; ++e) g[e] = make_float2(0.0f, 0.0f);
        if (in[3]) unpack2(PIPE ? *slot(stage, gh_slot, i) : span.load(in[3], begin, i), g);
#pragma unroll
        for (int e = 0; e < HALF; ++e)
          g[e] = __ffma2_rn(__ffma2_rn(n[k][e], make_float2(c, c), gw[k][e]), make_float2(s, s), g[e]);
        span.store(static_cast<T*>(a.dx), begin, i, g);
      }
    if constexpr (PIPE) {
      fetch(begin + stages * begin_step, stage);
      stage = stage + stage_slots == stages * stage_slots ? 0 : stage + stage_slots;
    }
  }
  if (!a.part) return;
  float* out = a.part + static_cast<int64_t>(blockIdx.x) * a.width;
  if (subs == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (span.has(i)) {
        if (!RAGGED) {
          store_vec2<float, VEC>(out + span.col(i), dw[i]);
        } else {
#pragma unroll
          for (int e = 0; e < HALF; ++e) {
            if (span.owns(i, 2 * e)) out[span.col(i) + 2 * e] = dw[i][e].x;
            if (span.owns(i, 2 * e + 1)) out[span.col(i) + 2 * e + 1] = dw[i][e].y;
          }
        }
      }
    return;
  }
  float* acc = red + 64;  // [row groups][width]
  cp_async_wait<0>();
  __syncthreads();  // the slots are free
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (span.has(i)) {
#pragma unroll
      for (int e = 0; e < HALF; ++e) {
        if (span.owns(i, 2 * e)) acc[sub * a.width + span.col(i) + 2 * e] = dw[i][e].x;
        if (span.owns(i, 2 * e + 1)) acc[sub * a.width + span.col(i) + 2 * e + 1] = dw[i][e].y;
      }
    }
  __syncthreads();
  for (int j = threadIdx.x; j < a.width; j += blockDim.x) {
    float t = 0.0f;
    for (int k = 0; k < subs; ++k) t += acc[k * a.width + j];
    out[j] = t;
  }
}

// dw[j] = sum over the blocks' rows of `part`, in a fixed order: 32 columns x
// 32 row groups a block, the groups' sums added in order.
template <class W>
__global__ void __launch_bounds__(1024) rms_norm_dw_kernel(const float* __restrict__ part, int nparts, int width,
                                                           W* __restrict__ dw) {
  __shared__ float red[32][33];
  pdl_enter();
  const int c = threadIdx.x % 32, k = threadIdx.x / 32;
  const int j = blockIdx.x * 32 + c;
  float t = 0.0f;
  if (j < width)
    for (int p = k; p < nparts; p += 32) t += part[static_cast<int64_t>(p) * width + j];
  red[k][c] = t;
  __syncthreads();
  if (k == 0 && j < width) {
    t = 0.0f;
#pragma unroll
    for (int q = 0; q < 32; ++q) t += red[q][c];
    dw[j] = from_float<W>(t);
  }
}

}  // namespace mlpk
