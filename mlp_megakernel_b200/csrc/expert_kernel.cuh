// Rows sorted by expert and back, with weights applied, and the gradients.
//
// Slot i = t * K + k holds the expert of token t's k-th choice; a slot whose
// id is outside [0, E) is dropped.  row_of[i] is the slot's place in a stable
// order by expert (a counting sort), the dropped slots last; offsets[e] is the
// first row of expert e and offsets[E] the number of rows kept.
//   dispatch:  xs[row_of[t,k]] = x[t], zeros in the dropped slots' rows
//   combine:   out[t] = sum_k w[t,k] y[row_of[t,k]] over the kept slots
//   backward of the combine, G = dL/dout:
//     dy[row_of[t,k]] = w[t,k] G[t] (zeros in the dropped slots' rows)
//     dw[t,k] = sum_j G[t,j] y[row_of[t,k],j]
//   backward of the dispatch: the combine of dL/dxs with weights of 1.
// Sums over k and over columns are fp32 in a fixed order.
#pragma once
#include "pdl.cuh"
#include "vec.cuh"

namespace mlpk {

constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kExpertMax = 1024;

template <class I>
__device__ __forceinline__ int expert_of(const I* ids, int64_t i, int64_t n, int experts) {
  if (i >= n) return -1;  // no slot
  const I e = ids[i];
  return e >= 0 && e < experts ? static_cast<int>(e) : experts;
}

// Counts per chunk: hist[chunk][e], e = E for the dropped slots.
template <class I>
__global__ void __launch_bounds__(kSortThreads) expert_count_kernel(const I* __restrict__ ids, int64_t n, int experts,
                                                                    int64_t chunk, int* __restrict__ hist) {
  extern __shared__ int cnt[];  // [E + 1]
  pdl_enter();
  for (int e = threadIdx.x; e <= experts; e += kSortThreads) cnt[e] = 0;
  __syncthreads();
  const int64_t first = blockIdx.x * chunk, last = min(n, first + chunk);
  for (int64_t i = first + threadIdx.x; i < last; i += kSortThreads)
    atomicAdd(cnt + expert_of(ids, i, n, experts), 1);
  __syncthreads();
  for (int e = threadIdx.x; e <= experts; e += kSortThreads)
    hist[static_cast<int64_t>(blockIdx.x) * (experts + 1) + e] = cnt[e];
}

// Each block places its chunk's slots: the first row of (chunk, e) is the
// number of slots of smaller experts plus those of e in earlier chunks; inside
// the chunk each warp takes a contiguous part, counts it, and places it 32
// slots at a time (equal ids among the 32 by a warp match).
template <class I>
__global__ void __launch_bounds__(kSortThreads)
    expert_place_kernel(const I* __restrict__ ids, int64_t n, int experts, int64_t chunk,
                        const int* __restrict__ hist, int* __restrict__ row_of, int* __restrict__ offsets) {
  extern __shared__ int sm[];
  int* next = sm;                                  // [warps][E + 1]: each warp's next row of e
  int* total = sm + kSortWarps * (experts + 1);    // [E + 1]: slots of e, then the first row of e
  int* before = total + (experts + 1);             // [E + 1]: slots of e in earlier chunks
  __shared__ int wsum[kSortWarps];
  pdl_enter();
  const int bins = experts + 1, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int e = threadIdx.x; e < bins; e += kSortThreads) {
    int t = 0, b = 0;
    for (int c = 0; c < gridDim.x; ++c) {
      const int v = hist[static_cast<int64_t>(c) * bins + e];
      if (c < blockIdx.x) b += v;
      t += v;
    }
    total[e] = t;
    before[e] = b;
  }
  for (int k = threadIdx.x; k < kSortWarps * bins; k += kSortThreads) next[k] = 0;
  __syncthreads();
  // Exclusive sums of total[], kSortThreads bins at a time.
  int carry = 0;
  for (int e0 = 0; e0 < bins; e0 += kSortThreads) {
    const int e = e0 + threadIdx.x;
    const int v = e < bins ? total[e] : 0;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    if (lane == 31) wsum[warp] = s;
    __syncthreads();
    int pre = carry, all = 0;
    for (int k = 0; k < kSortWarps; ++k) {
      if (k < warp) pre += wsum[k];
      all += wsum[k];
    }
    if (e < bins) {
      total[e] = pre + s - v;
      if (blockIdx.x == 0) offsets[e] = pre + s - v;
    }
    carry += all;
    __syncthreads();
  }
  // Each warp's part of the chunk: a multiple of 32 slots.
  const int64_t first = blockIdx.x * chunk, last = min(n, first + chunk);
  const int64_t part = chunk / kSortWarps;
  const int64_t w0 = first + warp * part, w1 = min(last, w0 + part);
  int* mine = next + warp * bins;
  for (int64_t i = w0 + lane; i < w1; i += 32) atomicAdd(mine + expert_of(ids, i, n, experts), 1);
  __syncthreads();
  for (int e = threadIdx.x; e < bins; e += kSortThreads) {
    int at = total[e] + before[e];
    for (int k = 0; k < kSortWarps; ++k) {
      const int c = next[k * bins + e];
      next[k * bins + e] = at;
      at += c;
    }
  }
  __syncthreads();
  for (int64_t i0 = w0; i0 < w1; i0 += 32) {
    const int64_t i = i0 + lane;
    const int e = expert_of(ids, i < w1 ? i : n, n, experts);
    const uint32_t same = __match_any_sync(0xffffffffu, e);
    const int rank = __popc(same & ((1u << lane) - 1u));
    int at = 0;
    if (e >= 0) {
      at = mine[e];
      row_of[i] = at + rank;
    }
    __syncwarp();
    if (e >= 0 && rank == 0) mine[e] = at + __popc(same);
    __syncwarp();
  }
}

// Rows are moved as words of U (16, 8, 4 or 2 bytes: the widest that divides
// a row); a thread takes one word of a token's row and stores it K times.
template <class U>
__global__ void __launch_bounds__(256) expert_dispatch_kernel(const U* __restrict__ x, int64_t tokens, int top,
                                                              int words, const int* __restrict__ row_of,
                                                              const int* __restrict__ kept, U* __restrict__ xs) {
  pdl_enter();
  const int64_t total = tokens * words;
  const int rows_kept = *kept;
  for (int64_t j = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; j < total;
       j += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t t = j / words, c = j - t * words;
    const U v = x[j];
    for (int k = 0; k < top; ++k) {
      const int row = row_of[t * top + k];
      xs[static_cast<int64_t>(row) * words + c] = row < rows_kept ? v : U{};
    }
  }
}

// out[t] = sum_k w[t,k] y[row_of[t,k]]; one vector of a token's row a thread.
template <class T, class W, int VEC>
__global__ void __launch_bounds__(256) expert_combine_kernel(const T* __restrict__ y, const W* __restrict__ w,
                                                             int64_t tokens, int top, int width,
                                                             const int* __restrict__ row_of,
                                                             const int* __restrict__ kept, T* __restrict__ out) {
  pdl_enter();
  const int nvec = width / VEC;
  const int64_t total = tokens * nvec;
  const int rows_kept = *kept;
  for (int64_t j = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; j < total;
       j += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t t = j / nvec, c = j - t * nvec;
    float acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.0f;
    for (int k = 0; k < top; ++k) {
      const int row = row_of[t * top + k];
      if (row >= rows_kept) continue;  // a dropped slot's row is not read: it may hold anything
      const float wk = w ? to_float(w[t * top + k]) : 1.0f;
      float f[VEC];
      unpack(load_raw<T, VEC>(y + static_cast<int64_t>(row) * width + c * VEC), f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] += wk * f[e];
    }
    store_vec<T, VEC>(out + j * VEC, acc);
  }
}

// dy and dw of the combine; a warp takes one slot.
template <class T, class W, int VEC>
__global__ void __launch_bounds__(256) expert_combine_bwd_kernel(const T* __restrict__ gout, const T* __restrict__ y,
                                                                 const W* __restrict__ w, int64_t tokens, int top,
                                                                 int width, const int* __restrict__ row_of,
                                                                 const int* __restrict__ kept, T* __restrict__ dy,
                                                                 W* __restrict__ dw) {
  pdl_enter();
  const int nvec = width / VEC, lane = threadIdx.x % 32;
  const int64_t slots = tokens * top;
  const int rows_kept = *kept;
  for (int64_t i = (blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x) / 32; i < slots;
       i += static_cast<int64_t>(gridDim.x) * (blockDim.x / 32)) {
    const int row = row_of[i];
    const bool on = row < rows_kept;
    const float wk = on ? (w ? to_float(w[i]) : 1.0f) : 0.0f;
    const T* g = gout + (i / top) * width;
    const int64_t base = static_cast<int64_t>(row) * width;
    float dot = 0.0f;
    for (int v = lane; v < nvec; v += 32) {
      float d[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) d[e] = 0.0f;
      if (on) {
        unpack(load_raw<T, VEC>(g + v * VEC), d);
        if (dw) {
          float f[VEC];
          unpack(load_raw<T, VEC>(y + base + v * VEC), f);
#pragma unroll
          for (int e = 0; e < VEC; ++e) dot += d[e] * f[e];
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) d[e] *= wk;
      }
      if (dy) store_vec<T, VEC>(dy + base + v * VEC, d);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (dw && lane == 0) dw[i] = from_float<W>(dot);
  }
}

}  // namespace mlpk
