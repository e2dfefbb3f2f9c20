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
// Sums over k and over columns are fp32 in a fixed order.  A place outside the
// T K rows, which no sort gives, is no row: nothing is read or written there.
#pragma once
#include <cooperative_groups.h>

#include "expert_plan.cuh"
#include "pdl.cuh"
#include "vec.cuh"

namespace mlpk {

// ------------------------------------------------------------------ sort
// Each warp has a contiguous part of the slots, each thread block contiguous
// warps.
//   1. a warp takes 32 slots at a time; equal ids among them (found by a ballot
//      for each bit of an id) get consecutive ranks behind the warp's count of
//      that id so far;
//   2. per id, the counts are summed over the block's warps, over lower blocks
//      and over lower ids;
//   3. a slot's row is its rank behind those.
// Up to 65,536 slots the blocks are one cluster, which sums its blocks' counts
// through distributed shared memory: one launch.  Above, the blocks are as many
// as have 4096 slots each, up to one an SM, in two launches: the first writes
// ranks and counts, the second adds the sums.  (262,144 slots of 64 experts: 15
// us by a cluster of 16, which are then short of issue slots, some 150
// instructions for 32 slots.)  Up to 128 slots a warp, ids and ranks stay in
// registers; 512 were held once, and the unrolled code made the smallest sorts
// slower (16 slots: 4.6 us).
constexpr int kSortRounds = (kExpertMax + kSortThreads) / kSortThreads;  // of kSortThreads ids

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

// A block's shared memory.
struct SortShared {
  int* sums;   // [warps]
  int* mine;   // [bins]: the block's slots of an id; then the first row of its slots
  int* count;  // [warps][bins]: a warp's slots of an id; then those of lower warps
  __device__ SortShared(int* sm, int bins) : sums(sm), mine(sm + kSortWarps), count(sm + kSortWarps + bins) {}
};

// Steps 1 and 2 within a block: ranks (in `at`, or in row_of unless HELD), and
// the block's counts in sh.mine.
template <class I, bool HELD>
__device__ __forceinline__ void sort_block(const I* ids, int64_t first, int64_t last, int experts,
                                           const SortShared& sh, int (&e)[kSortGroups],
                                           int (&at)[HELD ? kSortGroups : 1], int* row_of) {
  const int bins = experts + 1, bits = 32 - __clz(bins);  // ids are 0 to bins: bins stands for no slot
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int* own = sh.count + warp * bins;
  if constexpr (HELD) {
#pragma unroll
    for (int k = 0; k < kSortGroups; ++k) e[k] = expert_of(ids, first + k * 32 + lane, last, experts);
    __syncthreads();  // the counts are zero
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
        const int r = sort_rank(e[k], bins, bits, lane, own);
        if (e[k] >= 0) row_of[i0 + k * 32 + lane] = r;
      }
    }
  }
  __syncthreads();
  // Sums over the block's warps: a warp takes an id, a lane a warp's count.
  for (int k = warp; k < bins; k += kSortWarps) {
    const int c = sh.count[lane * bins + k];
    int s = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    sh.count[lane * bins + k] = s - c;
    if (lane == 31) sh.mine[k] = s;
  }
}

// Exclusive sums over the block's threads, plus `carry`, which becomes their
// end.
__device__ __forceinline__ int sort_scan(int v, int* sums, int* end, int& carry) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  if (lane == 31) sums[warp] = s;
  __syncthreads();
  int w = sums[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += u;
  }
  const int start = carry + __shfl_sync(0xffffffffu, w, warp) - sums[warp] + s - v;
  if (threadIdx.x == kSortThreads - 1) *end = start + v;
  __syncthreads();
  carry = *end;
  return start;
}

// `part`: slots of a warp, a multiple of 32 and at most 32 * kSortGroups.
template <class I>
__global__ void __launch_bounds__(kSortThreads)
    expert_sort_kernel(const I* __restrict__ ids, int64_t n, int experts, int64_t part, int* __restrict__ row_of,
                       int* __restrict__ offsets) {
  extern __shared__ int sm[];
  __shared__ int end;
  const int bins = experts + 1;  // the last one for the dropped slots
  const SortShared sh(sm, bins);
  auto cluster = cooperative_groups::this_cluster();
  const int blocks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int k = threadIdx.x; k < kSortWarps * bins; k += kSortThreads) sh.count[k] = 0;
  pdl_enter();
  const int64_t first = (static_cast<int64_t>(rank) * kSortWarps + warp) * part, last = min(n, first + part);
  int e[kSortGroups], at[kSortGroups];
  sort_block<I, true>(ids, first, last, experts, sh, e, at, row_of);
  if (blocks > 1) cluster.sync();
  else __syncthreads();
  int base[kSortRounds];
  int carry = 0;
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const int k = r * kSortThreads + threadIdx.x;
    base[r] = 0;
    if (r * kSortThreads >= bins) break;  // the whole block
    int all = 0, lower = 0;
    if (k < bins) {
      if (blocks == 1) {
        all = sh.mine[k];
      } else {
        int c[16];
#pragma unroll
        for (int b = 0; b < 16; ++b) c[b] = b < blocks ? *cluster.map_shared_rank(sh.mine + k, b) : 0;
#pragma unroll
        for (int b = 0; b < 16; ++b) {
          all += c[b];
          if (b < rank) lower += c[b];
        }
      }
    }
    const int start = sort_scan(all, sh.sums, &end, carry);
    if (k < bins && rank == 0) offsets[k] = start;
    base[r] = start + lower;
  }
  if (blocks > 1) cluster.sync();  // every block has read the others' `mine`
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const int k = r * kSortThreads + threadIdx.x;
    if (k < bins) sh.mine[k] = base[r];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSortGroups; ++k)
    if (e[k] >= 0) row_of[first + k * 32 + lane] = at[k] + sh.mine[e[k]] + sh.count[warp * bins + e[k]];
}

// The first launch of a sort of many slots: row_of[i] = the slot's rank among
// its block's slots of the same id, hist[block][id] = the block's slots.
template <class I, bool HELD>
__global__ void __launch_bounds__(kSortThreads)
    expert_rank_kernel(const I* __restrict__ ids, int64_t n, int experts, int64_t part, int* __restrict__ row_of,
                       int* __restrict__ hist) {
  extern __shared__ int sm[];
  const int bins = experts + 1;
  const SortShared sh(sm, bins);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int k = threadIdx.x; k < kSortWarps * bins; k += kSortThreads) sh.count[k] = 0;
  pdl_enter();
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * kSortWarps + warp) * part, last = min(n, first + part);
  int e[kSortGroups], at[HELD ? kSortGroups : 1];
  sort_block<I, HELD>(ids, first, last, experts, sh, e, at, row_of);
  __syncthreads();
  for (int k = threadIdx.x; k < bins; k += kSortThreads) hist[static_cast<int64_t>(blockIdx.x) * bins + k] = sh.mine[k];
  const int* own = sh.count + warp * bins;
  if constexpr (HELD) {
#pragma unroll
    for (int k = 0; k < kSortGroups; ++k)
      if (e[k] >= 0) row_of[first + k * 32 + lane] = at[k] + own[e[k]];
  } else {
    for (int64_t i = first + lane; i < last; i += 32) row_of[i] += own[expert_of(ids, i, last, experts)];
  }
}

// The second: the sums over lower blocks and lower ids.  Several threads share
// an id where there are more threads than ids; shared memory: [2][kSortThreads]
// and [bins].
template <class I>
__global__ void __launch_bounds__(kSortThreads)
    expert_place_kernel(const I* __restrict__ ids, int64_t n, int experts, int64_t part, int* __restrict__ row_of,
                        int* __restrict__ offsets, const int* __restrict__ hist) {
  extern __shared__ int sm[];
  __shared__ int end, sums[kSortWarps];
  const int bins = experts + 1;
  int *all_of = sm, *lower_of = sm + kSortThreads, *base = sm + 2 * kSortThreads;
  pdl_enter();
  const int shares = max(kSortThreads / bins, 1);
  int carry = 0;
  for (int r = 0; r * kSortThreads < bins; ++r) {  // one round unless there are 1024 experts
    const int k = r * kSortThreads + threadIdx.x % min(bins, kSortThreads), share = threadIdx.x / min(bins, kSortThreads);
    int all = 0, lower = 0;
    if (k < bins && share < shares) {
#pragma unroll 8
      for (int b = share; b < gridDim.x; b += shares) {
        const int c = hist[static_cast<int64_t>(b) * bins + k];
        all += c;
        if (b < blockIdx.x) lower += c;
      }
    }
    all_of[threadIdx.x] = all;
    lower_of[threadIdx.x] = lower;
    __syncthreads();
    all = lower = 0;
    const int id = r * kSortThreads + threadIdx.x;
    if (id < bins)
      for (int q = 0; q < shares; ++q) {
        all += all_of[q * min(bins, kSortThreads) + threadIdx.x];
        lower += lower_of[q * min(bins, kSortThreads) + threadIdx.x];
      }
    const int start = sort_scan(all, sums, &end, carry);
    if (id < bins) {
      base[id] = start + lower;
      if (blockIdx.x == 0) offsets[id] = start;
    }
    __syncthreads();
  }
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kSortWarps * part, last = min(n, first + kSortWarps * part);
  for (int64_t i0 = first; i0 < last; i0 += 4 * kSortThreads) {
    int e[4], row[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t i = i0 + q * kSortThreads + threadIdx.x;
      e[q] = expert_of(ids, i, last, experts);
      row[q] = i < last ? row_of[i] : 0;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (e[q] >= 0) row_of[i0 + q * kSortThreads + threadIdx.x] = row[q] + base[e[q]];
  }
}

// ------------------------------------------------------------------ rows
// The kernels below give a token's row (or a part of it, blockIdx.y) to `tpr`
// threads: a power of two up to 32, or a multiple of 32 up to 256; tokens share
// a block of at most 256.  Memory bounds them: a token's row is read or written
// once, its K rows in the order by expert once, each access as wide as a row
// allows.  A row waits for its place and then for its values, so what counts is
// how many rows an SM has under way: a thread has few (2 or 4 choices of one
// token) and few registers, and the SM as many threads as it can hold.  Of
// 32,768 tokens' 8 rows of 2048 bf16 values the combine takes 187 us (6.5 TB/s)
// with 48 registers a thread, 231 with 80 to 100 and twice the rows; of 131,072
// tokens' 2 rows of 256 fp16 values 36.7 with 32 registers, 45 with 100.

constexpr int kRowThreads = 256;
constexpr int kRowWidthMax = 1 << 24;  // columns; 65,535 parts of a row are the grid's limit

// A block has blockDim.x (tpr) threads a token and blockDim.y tokens at a time
// (two dimensions spare the divisions by tpr), NT times as many in all.
template <int NT>
struct TokenSpan {
  int lane;
  int64_t first;
  __device__ TokenSpan()
      : lane(threadIdx.x), first(static_cast<int64_t>(blockIdx.x) * blockDim.y * NT + threadIdx.y) {}
  __device__ int64_t token(int n) const { return first + static_cast<int64_t>(n) * blockDim.y; }
};

// The rows kept of `slots`.
__device__ __forceinline__ unsigned rows_kept_of(const int* kept, unsigned slots) {
  return min(static_cast<unsigned>(max(*kept, 0)), slots);
}

// Rows are moved as words of U (16, 8, 4 or 2 bytes: the widest that divides
// a row), NW a thread and token.
template <class U, int NT, int NW>
__global__ void __launch_bounds__(kRowThreads)
    expert_dispatch_kernel(const U* __restrict__ x, int64_t tokens, int top, int words,
                           const int* __restrict__ row_of, const int* __restrict__ kept, U* __restrict__ xs) {
  pdl_enter();
  const TokenSpan<NT> span;
  const int tpr = blockDim.x;
  const int c0 = blockIdx.y * tpr * NW + span.lane;
  U v[NT][NW];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int64_t t = span.token(n);
#pragma unroll
    for (int i = 0; i < NW; ++i)
      if (t < tokens && c0 + i * tpr < words) v[n][i] = x[t * words + c0 + i * tpr];
  }
  const unsigned slots = static_cast<unsigned>(tokens) * top, rows_kept = rows_kept_of(kept, slots);
  for (int k = 0; k < top; ++k) {
    unsigned row[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) row[n] = span.token(n) < tokens ? row_of[span.token(n) * top + k] : slots;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (row[n] >= slots) continue;
      U* to = xs + static_cast<int64_t>(row[n]) * words + c0;
#pragma unroll
      for (int i = 0; i < NW; ++i)
        if (c0 + i * tpr < words) to[i * tpr] = row[n] < rows_kept ? v[n][i] : U{};
    }
  }
}

// out[t] = sum_k w[t,k] y[row_of[t,k]], NW vectors of VEC elements a thread,
// GROUP choices at a time.
template <class T, class W, int VEC, int NW, int GROUP>
__global__ void __launch_bounds__(kRowThreads, VEC < kVecOf<T> ? 4 : GROUP == 2 ? 8 : 5)
    expert_combine_kernel(const T* __restrict__ y, const W* __restrict__ w, int64_t tokens, int top, int width,
                          const int* __restrict__ row_of, const int* __restrict__ kept, T* __restrict__ out) {
  pdl_enter();
  const TokenSpan<1> span;
  const int tpr = blockDim.x;
  const int64_t t = span.first;
  if (t >= tokens) return;
  const int nvec = width / VEC;
  const int c0 = blockIdx.y * tpr * NW + span.lane;
  const unsigned rows_kept = rows_kept_of(kept, static_cast<unsigned>(tokens) * top);
  float acc[NW][VEC];
#pragma unroll
  for (int i = 0; i < NW; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[i][e] = 0.0f;
  for (int k0 = 0; k0 < top; k0 += GROUP) {
    // A dropped slot's row is not read (it may hold anything), its weight not used.
    unsigned row[GROUP];
    float wk[GROUP];
    Raw<T, VEC> v[GROUP][NW];
#pragma unroll
    for (int k = 0; k < GROUP; ++k) {
      row[k] = k0 + k < top ? row_of[t * top + k0 + k] : rows_kept;
      wk[k] = k0 + k < top && w ? to_float(w[t * top + k0 + k]) : 1.0f;
    }
#pragma unroll
    for (int k = 0; k < GROUP; ++k)
#pragma unroll
      for (int i = 0; i < NW; ++i)
        if (row[k] < rows_kept && c0 + i * tpr < nvec)
          v[k][i] = load_raw<T, VEC>(y + static_cast<int64_t>(row[k]) * width + (c0 + i * tpr) * VEC);
#pragma unroll
    for (int k = 0; k < GROUP; ++k) {
      if (row[k] >= rows_kept) continue;
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

// dy and dw of the combine.  The threads of a token go over its columns, U
// vectors of GROUP choices at a time; they sum the dot products by shuffles and,
// above a warp, through shared memory.
template <class T, class W, int VEC, int GROUP>
__global__ void __launch_bounds__(kRowThreads, VEC < kVecOf<T> ? 4 : GROUP == 2 ? 6 : 4)
    expert_combine_bwd_kernel(const T* __restrict__ gout, const T* __restrict__ y, const W* __restrict__ w,
                              int64_t tokens, int top, int width, const int* __restrict__ row_of,
                              const int* __restrict__ kept, T* __restrict__ dy, W* __restrict__ dw) {
  constexpr int U = VEC == kVecOf<T> ? 1 : 4;
  __shared__ float red[2][kRowThreads / 32][GROUP];
  pdl_enter();
  const TokenSpan<1> span;
  const int tpr = blockDim.x;
  const int64_t t = span.first;
  const bool live = t < tokens;  // the others take part in the shuffles and barriers
  const int nvec = width / VEC;
  const unsigned slots = static_cast<unsigned>(tokens) * top, rows_kept = rows_kept_of(kept, slots);
  int half = 0;
  for (int k0 = 0; k0 < top; k0 += GROUP, half ^= 1) {
    unsigned row[GROUP];  // rows_kept and above: not kept; slots and above: no such slot
    int64_t row_at[U > 1 ? GROUP : 1];  // found once where it is used often
    float wk[GROUP], dot[GROUP];
#pragma unroll
    for (int k = 0; k < GROUP; ++k) {
      const bool slot = live && k0 + k < top;
      row[k] = slot ? row_of[t * top + k0 + k] : slots;
      wk[k] = slot && w ? to_float(w[t * top + k0 + k]) : 1.0f;
      dot[k] = 0.0f;
      if constexpr (U > 1) row_at[k] = static_cast<int64_t>(row[k]) * width;
    }
    auto on = [&](int k) { return row[k] < rows_kept; };  // else y is not read and the gradients are zero
    auto at = [&](int k) -> int64_t {
      if constexpr (U > 1) return row_at[k];
      return static_cast<int64_t>(row[k]) * width;
    };
    for (int v = live ? span.lane : nvec; v < nvec; v += tpr * U) {
      Raw<T, VEC> gr[U], yr[GROUP][U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (v + i * tpr >= nvec) break;
        gr[i] = load_raw<T, VEC>(gout + t * width + (v + i * tpr) * VEC);
#pragma unroll
        for (int k = 0; k < GROUP; ++k)
          if (dw && on(k)) yr[k][i] = load_raw<T, VEC>(y + at(k) + (v + i * tpr) * VEC);
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (v + i * tpr >= nvec) break;
        float g[VEC];
        unpack(gr[i], g);
#pragma unroll
        for (int k = 0; k < GROUP; ++k) {
          float f[VEC];
          if (dw && on(k)) {
            unpack(yr[k][i], f);
#pragma unroll
            for (int e = 0; e < VEC; ++e) dot[k] += g[e] * f[e];
          }
          if (dy && row[k] < slots) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] = on(k) ? wk[k] * g[e] : 0.0f;
            store_vec<T, VEC>(dy + at(k) + (v + i * tpr) * VEC, f);
          }
        }
      }
    }
    if (!dw) continue;
#pragma unroll
    for (int k = 0; k < GROUP; ++k)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        if (o < tpr) dot[k] += __shfl_xor_sync(0xffffffffu, dot[k], o);
    if (tpr > 32) {
      const int warp = threadIdx.y * (tpr / 32) + span.lane / 32;
      if (span.lane % 32 == 0) {
#pragma unroll
        for (int k = 0; k < GROUP; ++k) red[half][warp][k] = dot[k];
      }
      __syncthreads();
      if (span.lane < GROUP) {
        float s = 0.0f;
        for (int q = 0; q < tpr / 32; ++q) s += red[half][warp + q][span.lane];
        if (live && k0 + span.lane < top) dw[t * top + k0 + span.lane] = from_float<W>(s);
      }
    } else if (span.lane == 0 && live) {
#pragma unroll
      for (int k = 0; k < GROUP; ++k)
        if (k0 + k < top) dw[t * top + k0 + k] = from_float<W>(dot[k]);
    }
  }
}

}  // namespace mlpk
