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
#include <cooperative_groups.h>

#include "pdl.cuh"
#include "vec.cuh"

namespace mlpk {

// ------------------------------------------------------------------ sort
// One cluster of thread blocks does the whole sort, so it is one launch and
// reads nothing back from another: each warp has a contiguous part of the
// slots, each thread block contiguous warps.
//   1. a warp takes 32 slots at a time; equal ids among them (a warp match)
//      get consecutive ranks behind the warp's count of that id so far, kept in
//      row_of for the time being;
//   2. per id, the counts are summed over the block's warps, over the
//      cluster's lower blocks (distributed shared memory) and over lower ids;
//   3. row_of += that.
// What bounds it: the latency of step 1's chain, some 100 cycles for 32 slots
// of a warp.
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kExpertMax = 1024;
constexpr int kRowWidthMax = 1 << 24;  // columns; 65,535 parts of a row are the grid's limit
constexpr int kSortAhead = 4;  // groups of 32 slots whose ids are loaded together

template <class I>
__device__ __forceinline__ int expert_of(const I* ids, int64_t i, int64_t last, int experts) {
  if (i >= last) return -1;  // no slot
  const I e = ids[i];
  return e >= 0 && e < experts ? static_cast<int>(e) : experts;
}

// `part`: slots of a warp, a multiple of 32.
template <class I>
__global__ void __launch_bounds__(kSortThreads)
    expert_sort_kernel(const I* __restrict__ ids, int64_t n, int experts, int64_t part, int* __restrict__ row_of,
                       int* __restrict__ offsets) {
  extern __shared__ int sm[];
  const int bins = experts + 1;  // the last one for the dropped slots
  int* mine = sm + kSortWarps;                         // [bins]: this block's slots of e; then the first row of e
  int* count = mine + bins;                            // [warps][bins]
  __shared__ int carry_total;
  auto cluster = cooperative_groups::this_cluster();
  const int blocks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int k = threadIdx.x; k < kSortWarps * bins; k += kSortThreads) count[k] = 0;
  pdl_enter();
  __syncthreads();

  const int64_t first = (static_cast<int64_t>(rank) * kSortWarps + warp) * part, last = min(n, first + part);
  int* own = count + warp * bins;
  for (int64_t i0 = first; i0 < last; i0 += 32 * kSortAhead) {
    int e[kSortAhead];
#pragma unroll
    for (int k = 0; k < kSortAhead; ++k) e[k] = expert_of(ids, i0 + k * 32 + lane, last, experts);
#pragma unroll
    for (int k = 0; k < kSortAhead; ++k) {
      const uint32_t same = __match_any_sync(0xffffffffu, e[k]);
      const int before = __popc(same & ((1u << lane) - 1u));
      int at = 0;
      if (e[k] >= 0) {
        at = own[e[k]];
        row_of[i0 + k * 32 + lane] = at + before;
      }
      __syncwarp();
      if (e[k] >= 0 && before == 0) own[e[k]] = at + __popc(same);
      __syncwarp();
    }
  }
  __syncthreads();
  // Sums over the block's warps: count becomes what lies before each warp.
  for (int e = threadIdx.x; e < bins; e += kSortThreads) {
    int t = 0;
    for (int k = 0; k < kSortWarps; ++k) {
      const int c = count[k * bins + e];
      count[k * bins + e] = t;
      t += c;
    }
    mine[e] = t;
  }
  if (blocks > 1) cluster.sync();
  else __syncthreads();
  // Sums over the cluster's blocks, then over lower ids, kSortThreads ids at a
  // time; at most two rounds.
  int base[(kExpertMax + kSortThreads) / kSortThreads];
  int carry = 0;
#pragma unroll
  for (int r = 0; r < (kExpertMax + kSortThreads) / kSortThreads; ++r) {
    const int e = r * kSortThreads + threadIdx.x;
    base[r] = 0;
    if (r * kSortThreads >= bins) break;  // the whole block
    int all = 0, lower = 0;
    if (e < bins) {
      if (blocks == 1) {
        all = mine[e];
      } else {
#pragma unroll 8
        for (int b = 0; b < blocks; ++b) {
          const int c = *cluster.map_shared_rank(mine + e, b);
          if (b < rank) lower += c;
          all += c;
        }
      }
    }
    int s = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    if (lane == 31) sm[warp] = s;
    __syncthreads();
    int w = sm[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    const int pre = __shfl_sync(0xffffffffu, w, warp) - sm[warp];  // of lower warps
    const int start = carry + pre + s - all;
    if (e < bins && rank == 0) offsets[e] = start;
    base[r] = start + lower;
    if (threadIdx.x == kSortThreads - 1) carry_total = start + all;
    __syncthreads();
    carry = carry_total;
  }
  if (blocks > 1) cluster.sync();  // every block has read the others' `mine`
#pragma unroll
  for (int r = 0; r < (kExpertMax + kSortThreads) / kSortThreads; ++r) {
    const int e = r * kSortThreads + threadIdx.x;
    if (e < bins) mine[e] = base[r];
  }
  __syncthreads();
  for (int64_t i0 = first; i0 < last; i0 += 32 * kSortAhead) {
#pragma unroll
    for (int k = 0; k < kSortAhead; ++k) {
      const int64_t i = i0 + k * 32 + lane;
      const int e = expert_of(ids, i, last, experts);
      if (e >= 0) row_of[i] += mine[e] + own[e];
    }
  }
}

// ------------------------------------------------------------------ rows
// The kernels below give a token's row (or a part of it, blockIdx.y) to `tpr`
// threads, a power of two up to 256; several tokens share a block of 256.
// Memory bounds them: a token's row is read or written once, its K rows in the
// order by expert once, each access as wide as a row allows.

constexpr int kRowThreads = 256;
constexpr int kTopGroup = 4;  // rows of a token that are under way together

// Rows are moved as words of U (16, 8, 4 or 2 bytes: the widest that divides
// a row), NW a thread.
template <class U, int NW>
__global__ void __launch_bounds__(kRowThreads)
    expert_dispatch_kernel(const U* __restrict__ x, int64_t tokens, int top, int words, int tpr,
                           const int* __restrict__ row_of, const int* __restrict__ kept, U* __restrict__ xs) {
  pdl_enter();
  const int lane = threadIdx.x % tpr;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kRowThreads / tpr) + threadIdx.x / tpr;
  if (t >= tokens) return;
  const int c0 = blockIdx.y * tpr * NW + lane;
  U v[NW];
#pragma unroll
  for (int i = 0; i < NW; ++i)
    if (c0 + i * tpr < words) v[i] = x[t * words + c0 + i * tpr];
  const int rows_kept = *kept;
  for (int k = 0; k < top; ++k) {
    const int row = row_of[t * top + k];
    U* to = xs + static_cast<int64_t>(row) * words + c0;
#pragma unroll
    for (int i = 0; i < NW; ++i)
      if (c0 + i * tpr < words) to[i * tpr] = row < rows_kept ? v[i] : U{};
  }
}

// out[t] = sum_k w[t,k] y[row_of[t,k]], NW vectors of VEC elements a thread.
template <class T, class W, int VEC, int NW>
__global__ void __launch_bounds__(kRowThreads)
    expert_combine_kernel(const T* __restrict__ y, const W* __restrict__ w, int64_t tokens, int top, int width, int tpr,
                          const int* __restrict__ row_of, const int* __restrict__ kept, T* __restrict__ out) {
  pdl_enter();
  const int lane = threadIdx.x % tpr;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kRowThreads / tpr) + threadIdx.x / tpr;
  if (t >= tokens) return;
  const int nvec = width / VEC;
  const int c0 = blockIdx.y * tpr * NW + lane;
  const int rows_kept = *kept;
  float acc[NW][VEC];
#pragma unroll
  for (int i = 0; i < NW; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[i][e] = 0.0f;
  for (int k0 = 0; k0 < top; k0 += kTopGroup) {
    // A dropped slot's row is not read (it may hold anything), nor its weight.
    Raw<T, VEC> v[kTopGroup][NW];
    float wk[kTopGroup];
    bool on[kTopGroup];
#pragma unroll
    for (int k = 0; k < kTopGroup; ++k) {
      const int row = k0 + k < top ? row_of[t * top + k0 + k] : rows_kept;
      on[k] = row < rows_kept;
      wk[k] = on[k] && w ? to_float(w[t * top + k0 + k]) : 1.0f;
#pragma unroll
      for (int i = 0; i < NW; ++i)
        if (on[k] && c0 + i * tpr < nvec)
          v[k][i] = load_raw<T, VEC>(y + static_cast<int64_t>(row) * width + (c0 + i * tpr) * VEC);
    }
#pragma unroll
    for (int k = 0; k < kTopGroup; ++k) {
      if (!on[k]) continue;
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        float f[VEC];
        unpack(v[k][i], f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[i][e] += wk[k] * f[e];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NW; ++i)
    if (c0 + i * tpr < nvec) store_vec<T, VEC>(out + t * width + (c0 + i * tpr) * VEC, acc[i]);
}

// dy and dw of the combine.  The tpr threads of a token go over its columns; 4
// choices at a time, whose dot products they sum by shuffles and, above a
// warp, through shared memory.
template <class T, class W, int VEC>
__global__ void __launch_bounds__(kRowThreads)
    expert_combine_bwd_kernel(const T* __restrict__ gout, const T* __restrict__ y, const W* __restrict__ w,
                              int64_t tokens, int top, int width, int tpr, const int* __restrict__ row_of,
                              const int* __restrict__ kept, T* __restrict__ dy, W* __restrict__ dw) {
  __shared__ float red[2][kRowThreads / 32][kTopGroup];
  pdl_enter();
  const int lane = threadIdx.x % tpr;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kRowThreads / tpr) + threadIdx.x / tpr;
  const bool live = t < tokens;  // the others take part in the shuffles and barriers
  const int nvec = width / VEC;
  const int rows_kept = *kept;
  int half = 0;
  for (int k0 = 0; k0 < top; k0 += kTopGroup, half ^= 1) {
    int row[kTopGroup];  // below 0: no such choice
    float wk[kTopGroup], dot[kTopGroup];
#pragma unroll
    for (int k = 0; k < kTopGroup; ++k) {
      row[k] = live && k0 + k < top ? row_of[t * top + k0 + k] : -1;
      wk[k] = row[k] >= 0 && row[k] < rows_kept ? (w ? to_float(w[t * top + k0 + k]) : 1.0f) : 0.0f;
      dot[k] = 0.0f;
    }
    if (live)
      for (int v = lane; v < nvec; v += tpr) {
        Raw<T, VEC> yr[kTopGroup];
        if (dw) {
#pragma unroll
          for (int k = 0; k < kTopGroup; ++k)
            if (row[k] >= 0 && row[k] < rows_kept)
              yr[k] = load_raw<T, VEC>(y + static_cast<int64_t>(row[k]) * width + v * VEC);
        }
        float g[VEC];
        unpack(load_raw<T, VEC>(gout + t * width + v * VEC), g);
#pragma unroll
        for (int k = 0; k < kTopGroup; ++k) {
          if (row[k] < 0) continue;
          const bool on = row[k] < rows_kept;
          float f[VEC];
          if (dw && on) {
            unpack(yr[k], f);
#pragma unroll
            for (int e = 0; e < VEC; ++e) dot[k] += g[e] * f[e];
          }
          if (dy) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] = on ? wk[k] * g[e] : 0.0f;
            store_vec<T, VEC>(dy + static_cast<int64_t>(row[k]) * width + v * VEC, f);
          }
        }
      }
    if (!dw) continue;
#pragma unroll
    for (int k = 0; k < kTopGroup; ++k)
      for (int o = (tpr < 32 ? tpr : 32) / 2; o > 0; o >>= 1) dot[k] += __shfl_xor_sync(0xffffffffu, dot[k], o);
    if (tpr > 32) {
      const int warps = tpr / 32, warp = threadIdx.x / 32;
      if (threadIdx.x % 32 == 0) {
#pragma unroll
        for (int k = 0; k < kTopGroup; ++k) red[half][warp][k] = dot[k];
      }
      __syncthreads();
      if (lane < kTopGroup) {
        float s = 0.0f;
        for (int k = 0; k < warps; ++k) s += red[half][warp + k][lane];
        if (live && k0 + lane < top) dw[t * top + k0 + lane] = from_float<W>(s);
      }
    } else if (lane == 0 && live) {
#pragma unroll
      for (int k = 0; k < kTopGroup; ++k)
        if (k0 + k < top) dw[t * top + k0 + k] = from_float<W>(dot[k]);
    }
  }
}

}  // namespace mlpk
