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
// One cluster of thread blocks does the whole sort, so it is one launch: each
// warp has a contiguous part of the slots, each thread block contiguous warps.
//   1. a warp takes 32 slots at a time; equal ids among them (found by a ballot
//      for each bit of an id) get consecutive ranks behind the warp's count of
//      that id so far;
//   2. per id, the counts are summed over the block's warps, over the
//      cluster's lower blocks (distributed shared memory) and over lower ids;
//   3. a slot's row is its rank behind those.
// Up to 512 slots a warp (262,144 in all) ids and ranks stay in registers; above,
// the ids are read twice and row_of holds the ranks in between.
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kExpertMax = 1024;
constexpr int kSortGroups = 16;  // groups of 32 slots of a warp that registers hold

template <class I>
__device__ __forceinline__ int expert_of(const I* ids, int64_t i, int64_t last, int experts) {
  if (i >= last) return -1;  // no slot
  const I e = ids[i];
  return e >= 0 && e < experts ? static_cast<int>(e) : experts;
}

// The lanes whose e is this lane's; every e is below 2^bits.
__device__ __forceinline__ uint32_t lanes_of_same(int e, int bits) {
  uint32_t same = 0xffffffffu;
  for (int b = 0; b < bits; ++b) {
    const uint32_t set = __ballot_sync(0xffffffffu, (e >> b) & 1);
    same &= (e >> b) & 1 ? set : ~set;
  }
  return same;
}

// Rank of each lane's slot (e below 0: none) among the warp's slots of e so
// far; `own` counts them.
__device__ __forceinline__ int sort_rank(int e, int bins, int bits, int lane, int* own) {
  const uint32_t same = lanes_of_same(e < 0 ? bins : e, bits);
  const int before = __popc(same & ((1u << lane) - 1u));
  const int at = e >= 0 ? own[e] : 0;
  __syncwarp();
  if (e >= 0 && before == 0) own[e] = at + __popc(same);
  __syncwarp();
  return at + before;
}

// `part`: slots of a warp, a multiple of 32.
template <class I, bool HELD>
__global__ void __launch_bounds__(kSortThreads)
    expert_sort_kernel(const I* __restrict__ ids, int64_t n, int experts, int64_t part, int* __restrict__ row_of,
                       int* __restrict__ offsets) {
  extern __shared__ int sm[];
  const int bins = experts + 1;  // the last one for the dropped slots
  int* mine = sm + kSortWarps;   // [bins]: this block's slots of e; then the first row of its slots of e
  int* count = mine + bins;      // [warps][bins]: a warp's slots of e; then those of lower warps
  __shared__ int round_end;
  auto cluster = cooperative_groups::this_cluster();
  const int blocks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int bits = 32 - __clz(bins);  // ids are 0 to bins: bins stands for no slot
  for (int k = threadIdx.x; k < kSortWarps * bins; k += kSortThreads) count[k] = 0;
  pdl_enter();
  const int64_t first = (static_cast<int64_t>(rank) * kSortWarps + warp) * part, last = min(n, first + part);
  int* own = count + warp * bins;
  int e[kSortGroups], at[HELD ? kSortGroups : 1];
  if constexpr (HELD) {
#pragma unroll
    for (int k = 0; k < kSortGroups; ++k) e[k] = expert_of(ids, first + k * 32 + lane, last, experts);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortGroups; ++k)
      if (first + k * 32 < last) at[k] = sort_rank(e[k], bins, bits, lane, own);
  } else {
    __syncthreads();
    for (int64_t i0 = first; i0 < last; i0 += 32 * kSortGroups) {
#pragma unroll
      for (int k = 0; k < kSortGroups; ++k) e[k] = expert_of(ids, i0 + k * 32 + lane, last, experts);
#pragma unroll
      for (int k = 0; k < kSortGroups; ++k) {
        if (i0 + k * 32 >= last) break;  // the whole warp
        at[0] = sort_rank(e[k], bins, bits, lane, own);
        if (e[k] >= 0) row_of[i0 + k * 32 + lane] = at[0];
      }
    }
  }
  __syncthreads();
  // Sums over the block's warps: a warp takes an id, a lane a warp's count.
  for (int k = warp; k < bins; k += kSortWarps) {
    const int c = count[lane * bins + k];
    int s = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    count[lane * bins + k] = s - c;
    if (lane == 31) mine[k] = s;
  }
  if (blocks > 1) cluster.sync();
  else __syncthreads();
  // Sums over the cluster's blocks, then over lower ids, kSortThreads ids at a
  // time: at most two rounds.
  constexpr int ROUNDS = (kExpertMax + kSortThreads) / kSortThreads;
  int base[ROUNDS];
  int carry = 0;
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int k = r * kSortThreads + threadIdx.x;
    base[r] = 0;
    if (r * kSortThreads >= bins) break;  // the whole block
    int all = 0, lower = 0;
    if (k < bins) {
      if (blocks == 1) {
        all = mine[k];
      } else {
        int c[16];
#pragma unroll
        for (int b = 0; b < 16; ++b) c[b] = b < blocks ? *cluster.map_shared_rank(mine + k, b) : 0;
#pragma unroll
        for (int b = 0; b < 16; ++b) {
          all += c[b];
          if (b < rank) lower += c[b];
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
    if (k < bins && rank == 0) offsets[k] = start;
    base[r] = start + lower;
    if (threadIdx.x == kSortThreads - 1) round_end = start + all;
    __syncthreads();
    carry = round_end;
  }
  if (blocks > 1) cluster.sync();  // every block has read the others' `mine`
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int k = r * kSortThreads + threadIdx.x;
    if (k < bins) mine[k] = base[r];
  }
  __syncthreads();
  if constexpr (HELD) {
#pragma unroll
    for (int k = 0; k < kSortGroups; ++k)
      if (e[k] >= 0) row_of[first + k * 32 + lane] = at[k] + mine[e[k]] + own[e[k]];
  } else {
    for (int64_t i0 = first; i0 < last; i0 += 32 * kSortGroups) {
#pragma unroll
      for (int k = 0; k < kSortGroups; ++k) e[k] = expert_of(ids, i0 + k * 32 + lane, last, experts);
#pragma unroll
      for (int k = 0; k < kSortGroups; ++k)
        if (e[k] >= 0) row_of[i0 + k * 32 + lane] += mine[e[k]] + own[e[k]];
    }
  }
}

// ------------------------------------------------------------------ rows
// The kernels below give a token's row (or a part of it, blockIdx.y) to `tpr`
// threads: a power of two up to 32, or a multiple of 32 up to 256; tokens share
// a block of at most 256.  Memory bounds them: a token's row is read or written
// once, its K rows in the order by expert once, each access as wide as a row
// allows.  A row waits for its place and then for its values, so a thread has 8
// rows under way: GROUP choices of each of 8 / GROUP tokens (262,144 rows of 256
// fp16 values, 2 choices a token: the combine took 57 us with one token at a
// time).

constexpr int kRowThreads = 256;
constexpr int kRowsAhead = 8;
constexpr int kRowWidthMax = 1 << 24;  // columns; 65,535 parts of a row are the grid's limit

// Tokens of a thread: `tokens_each` of them, a block's tokens apart.
struct TokenSpan {
  int lane, sub, subs;
  int64_t first;
  __device__ TokenSpan(int tpr, int tokens_each)
      : lane(threadIdx.x % tpr), sub(threadIdx.x / tpr), subs(blockDim.x / tpr),
        first(static_cast<int64_t>(blockIdx.x) * subs * tokens_each + sub) {}
  __device__ int64_t token(int n) const { return first + static_cast<int64_t>(n) * subs; }
};

// Rows are moved as words of U (16, 8, 4 or 2 bytes: the widest that divides
// a row), NW a thread and token.
template <class U, int NT, int NW>
__global__ void __launch_bounds__(kRowThreads)
    expert_dispatch_kernel(const U* __restrict__ x, int64_t tokens, int top, int words, int tpr,
                           const int* __restrict__ row_of, const int* __restrict__ kept, U* __restrict__ xs) {
  pdl_enter();
  const TokenSpan span(tpr, NT);
  const int c0 = blockIdx.y * tpr * NW + span.lane;
  U v[NT][NW];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int64_t t = span.token(n);
#pragma unroll
    for (int i = 0; i < NW; ++i)
      if (t < tokens && c0 + i * tpr < words) v[n][i] = x[t * words + c0 + i * tpr];
  }
  const int rows_kept = *kept;
  for (int k = 0; k < top; ++k) {
    int row[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) row[n] = span.token(n) < tokens ? row_of[span.token(n) * top + k] : -1;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (row[n] < 0) continue;
      U* to = xs + static_cast<int64_t>(row[n]) * words + c0;
#pragma unroll
      for (int i = 0; i < NW; ++i)
        if (c0 + i * tpr < words) to[i * tpr] = row[n] < rows_kept ? v[n][i] : U{};
    }
  }
}

// out[t] = sum_k w[t,k] y[row_of[t,k]], NW vectors of VEC elements a thread and
// token.
template <class T, class W, int VEC, int NW, int GROUP>
__global__ void __launch_bounds__(kRowThreads)
    expert_combine_kernel(const T* __restrict__ y, const W* __restrict__ w, int64_t tokens, int top, int width, int tpr,
                          const int* __restrict__ row_of, const int* __restrict__ kept, T* __restrict__ out) {
  constexpr int NT = kRowsAhead / GROUP;
  pdl_enter();
  const TokenSpan span(tpr, NT);
  const int nvec = width / VEC;
  const int c0 = blockIdx.y * tpr * NW + span.lane;
  const int rows_kept = *kept;
  float acc[NT][NW][VEC];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < NW; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[n][i][e] = 0.0f;
  for (int k0 = 0; k0 < top; k0 += GROUP) {
    // A dropped slot's row is not read (it may hold anything), nor its weight.
    int row[NT][GROUP];
    float wk[NT][GROUP];
    Raw<T, VEC> v[NT][GROUP][NW];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < GROUP; ++k) {
        const bool slot = span.token(n) < tokens && k0 + k < top;
        row[n][k] = slot ? row_of[span.token(n) * top + k0 + k] : rows_kept;
        wk[n][k] = slot && w ? to_float(w[span.token(n) * top + k0 + k]) : 1.0f;
      }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < GROUP; ++k)
#pragma unroll
        for (int i = 0; i < NW; ++i)
          if (row[n][k] < rows_kept && c0 + i * tpr < nvec)
            v[n][k][i] = load_raw<T, VEC>(y + static_cast<int64_t>(row[n][k]) * width + (c0 + i * tpr) * VEC);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < GROUP; ++k) {
        if (row[n][k] >= rows_kept) continue;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
          float f[VEC];
          unpack(v[n][k][i], f);
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[n][i][e] += wk[n][k] * f[e];
        }
      }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < NW; ++i)
      if (span.token(n) < tokens && c0 + i * tpr < nvec)
        store_vec<T, VEC>(out + span.token(n) * width + (c0 + i * tpr) * VEC, acc[n][i]);
}

// dy and dw of the combine.  The threads of a token go over its columns, GROUP
// choices of 4 / GROUP tokens at a time; they sum the dot products by shuffles
// and, above a warp, through shared memory.
template <class T, class W, int VEC, int GROUP>
__global__ void __launch_bounds__(kRowThreads)
    expert_combine_bwd_kernel(const T* __restrict__ gout, const T* __restrict__ y, const W* __restrict__ w,
                              int64_t tokens, int top, int width, int tpr, const int* __restrict__ row_of,
                              const int* __restrict__ kept, T* __restrict__ dy, W* __restrict__ dw) {
  constexpr int NT = 4 / GROUP;
  __shared__ float red[2][kRowThreads / 32][4];
  pdl_enter();
  const TokenSpan span(tpr, NT);
  const int nvec = width / VEC;
  const int rows_kept = *kept;
  int half = 0;
  for (int k0 = 0; k0 < top; k0 += GROUP, half ^= 1) {
    int row[NT][GROUP];  // below 0: no such slot
    float wk[NT][GROUP], dot[NT * GROUP];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < GROUP; ++k) {
        const bool slot = span.token(n) < tokens && k0 + k < top;
        row[n][k] = slot ? row_of[span.token(n) * top + k0 + k] : -1;
        wk[n][k] = slot && w ? to_float(w[span.token(n) * top + k0 + k]) : 1.0f;
        dot[n * GROUP + k] = 0.0f;
      }
    for (int v = span.lane; v < nvec; v += tpr) {
      Raw<T, VEC> gr[NT], yr[NT][GROUP];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (span.token(n) < tokens) gr[n] = load_raw<T, VEC>(gout + span.token(n) * width + v * VEC);
#pragma unroll
        for (int k = 0; k < GROUP; ++k)
          if (dw && row[n][k] >= 0 && row[n][k] < rows_kept)
            yr[n][k] = load_raw<T, VEC>(y + static_cast<int64_t>(row[n][k]) * width + v * VEC);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float g[VEC];
        unpack(gr[n], g);
#pragma unroll
        for (int k = 0; k < GROUP; ++k) {
          if (row[n][k] < 0) continue;
          const bool on = row[n][k] < rows_kept;  // else its row of y is not read and its gradients are zero
          float f[VEC];
          if (dw && on) {
            unpack(yr[n][k], f);
#pragma unroll
            for (int e = 0; e < VEC; ++e) dot[n * GROUP + k] += g[e] * f[e];
          }
          if (dy) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] = on ? wk[n][k] * g[e] : 0.0f;
            store_vec<T, VEC>(dy + static_cast<int64_t>(row[n][k]) * width + v * VEC, f);
          }
        }
      }
    }
    if (!dw) continue;
#pragma unroll
    for (int j = 0; j < NT * GROUP; ++j)
      for (int o = (tpr < 32 ? tpr : 32) / 2; o > 0; o >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
    if (tpr > 32) {
      const int warp = threadIdx.x / 32;
      if (threadIdx.x % 32 == 0) {
#pragma unroll
        for (int j = 0; j < NT * GROUP; ++j) red[half][warp][j] = dot[j];
      }
      __syncthreads();
      if (span.lane < NT * GROUP) {
        const int n = span.lane / GROUP, k = k0 + span.lane % GROUP;
        float s = 0.0f;
        for (int q = 0; q < tpr / 32; ++q) s += red[half][warp + q][span.lane];
        if (span.token(n) < tokens && k < top) dw[span.token(n) * top + k] = from_float<W>(s);
      }
    } else if (span.lane == 0) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < GROUP; ++k)
          if (span.token(n) < tokens && k0 + k < top)
            dw[span.token(n) * top + k0 + k] = from_float<W>(dot[n * GROUP + k]);
    }
  }
}

}  // namespace mlpk
