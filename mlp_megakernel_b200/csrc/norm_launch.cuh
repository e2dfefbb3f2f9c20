// Launches of the RMS norm's kernels for one type of rows: which threads share
// a row, how many rows are under way, how many blocks loop.  norm_f16.cu,
// norm_bf16.cu and norm_f32.cu each build their type's kernels.
#pragma once
#include <algorithm>
#include <type_traits>

#include "host.cuh"
#include "norm_kernel.cuh"

namespace mlpk {
namespace norm {

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Threads a row (tpr) and vectors a thread (nv).  A row of up to 128 vectors
// belongs to a warp or a part of one: no barrier.  Wider ones take 2 vectors a
// thread while that is at most 512 threads, then 4, and 9 where 4 do not reach
// (fp32 rows above 16,384 and the widest ragged ones: 32,767 fp32 values lie in
// up to 8,193 vectors).
struct RowPlan {
  int tpr, nv, rows_per_block, threads;
  bool ragged, full;  // full: one row a block, every thread with all its vectors
};
inline RowPlan row_plan(int width, int vec) {
  RowPlan p;
  p.ragged = width % vec != 0;
  const int nvec = static_cast<int>(ceil_div(width + (p.ragged ? vec - 1 : 0), vec));  // wherever a row begins
  if (nvec <= 32) {
    p.nv = 1;
    p.tpr = 1;
    while (p.tpr < nvec) p.tpr *= 2;
  } else if (nvec <= 128) {
    p.tpr = 32;
    p.nv = nvec <= 64 ? 2 : 4;
  } else {
    p.nv = nvec <= 1024 ? 2 : nvec <= 4096 ? 4 : 9;
    p.tpr = static_cast<int>(ceil_div(ceil_div(nvec, p.nv), 32)) * 32;
  }
  p.rows_per_block = p.tpr <= 32 ? kNormThreads / p.tpr : 1;
  p.threads = p.rows_per_block * p.tpr;
  p.full = !p.ragged && p.tpr > 32 && nvec == p.tpr * p.nv;
  return p;
}
inline int vec_of(int dtype) { return dtype == MLPK_DT_F32 ? 4 : 8; }

// Rows under way a thread, of `streams` vectors each: as many as fit in
// `budget`, at least one if that fits a block at all; 0: read directly.
inline int stages_of(const RowPlan& p, int streams, size_t budget) {
  const size_t stage = static_cast<size_t>(p.nv) * p.threads * streams * 16;
  if (p.nv > 4) return 0;
  const int n = static_cast<int>(std::min<size_t>(budget / stage, kNormStages));
  return n > 0 ? n : stage + 2048 <= static_cast<size_t>(host::kMaxBlockSmem) ? 1 : 0;
}

// Blocks that loop over the rows: those the device holds at a time, or fewer
// if there are not so many rows.  Ragged rows want a step of whole vectors.
inline int64_t loop_blocks(int64_t rows, const RowPlan& p, int vec, int64_t resident) {
  const int64_t blocks = ceil_div(rows, p.rows_per_block);
  if (blocks <= resident) return blocks;
  return p.ragged ? std::max<int64_t>(resident / vec, 1) * vec : resident;
}

// Blocks of the backward pass that an SM holds: 512 threads in all (their
// registers allow no more).
inline int bwd_per_sm(const RowPlan& p) { return std::max(1, 512 / p.threads); }

// Blocks of the backward pass, each of which leaves one row of dw's partial
// sums.  (The same for every count of inputs, so that the workspace's size
// follows from rows, width and type.)
inline int64_t bwd_blocks(int64_t rows, int width, int dtype, int sm_count) {
  const RowPlan p = row_plan(width, vec_of(dtype));
  return loop_blocks(rows, p, vec_of(dtype), static_cast<int64_t>(sm_count) * bwd_per_sm(p));
}

// f(NV, KIND, PIPE, MAXT) of this call.
template <bool V>
using Bool = std::integral_constant<bool, V>;
template <int V>
using Int = std::integral_constant<int, V>;

template <class T, int KIND, class F>
int with_counts(const RowPlan& p, bool pipe, F&& f) {
  using Kind = Int<KIND>;
  switch (p.nv) {
    case 1:
      if constexpr (KIND != kFull) return f(Int<1>{}, Kind{}, Bool<true>{}, Int<256>{});
      return MLPK_ERR_UNSUPPORTED;
    case 2:
      return p.threads <= 256 ? f(Int<2>{}, Kind{}, Bool<true>{}, Int<256>{})
                              : f(Int<2>{}, Kind{}, Bool<true>{}, Int<512>{});
    case 4:
      if (p.threads <= 512) return f(Int<4>{}, Kind{}, Bool<true>{}, Int<512>{});
      return pipe ? f(Int<4>{}, Kind{}, Bool<true>{}, Int<1024>{}) : f(Int<4>{}, Kind{}, Bool<false>{}, Int<1024>{});
    default:
      if constexpr (sizeof(T) == 4 || KIND == kRagged) return f(Int<9>{}, Kind{}, Bool<false>{}, Int<1024>{});
      return MLPK_ERR_UNSUPPORTED;
  }
}
template <class T, class F>
int with_kind(const RowPlan& p, bool pipe, F&& f) {
  if (p.ragged) return with_counts<T, kRagged>(p, pipe, f);
  return p.full ? with_counts<T, kFull>(p, pipe, f) : with_counts<T, kPart>(p, pipe, f);
}

template <class T, class W, bool FP8>
int forward(NormArgs a, cudaStream_t st) {
  host::DevInfo di;
  int dev;
  int rc = host::current_device_info(&di, &dev);
  if (rc) return rc;
  const RowPlan p = row_plan(a.width, kVecOf<T>);
  const int streams = a.r ? 2 : 1;
  const int stages = stages_of(p, streams, 52 * 1024);
  a.tpr = p.tpr;
  size_t slots_at = 128 * sizeof(float);
  if (FP8 && p.ragged && a.group)
    slots_at += ceil_div(sizeof(float) * p.rows_per_block * ceil_div(a.width, kNormGroup), 16) * 16;
  const size_t smem = slots_at + static_cast<size_t>(stages) * p.nv * p.threads * streams * 16;
  return with_kind<T>(p, stages > 0, [&](auto nv, auto kind, auto pipe, auto maxt) {
    const auto kern = rms_norm_fwd_kernel<T, W, decltype(nv)::value, decltype(kind)::value, decltype(pipe)::value,
                                          decltype(maxt)::value, FP8>;
    const int per_sm = host::blocks_per_sm(reinterpret_cast<const void*>(kern), p.threads, smem, dev);
    if (per_sm == 0) return static_cast<int>(MLPK_ERR_CUDA);
    const int64_t blocks = loop_blocks(a.rows, p, kVecOf<T>, static_cast<int64_t>(di.sm_count) * per_sm);
    return host::launch_kernel_early(kern, dim3(static_cast<unsigned>(blocks)), p.threads, smem, st, a, stages,
                                     static_cast<int>(slots_at));
  });
}

// `blocks` rows of partial sums in a.part (unless it is null), then dw.
template <class T, class W>
int backward(NormBwdArgs a, int64_t blocks, W* dw, int dev, cudaStream_t st) {
  const RowPlan p = row_plan(a.width, kVecOf<T>);
  const int streams = 2 + (a.r != nullptr) + (a.gh != nullptr);
  const int stages = stages_of(p, streams, 200 * 1024 / bwd_per_sm(p));
  a.tpr = p.tpr;
  size_t smem = static_cast<size_t>(stages) * p.nv * p.threads * streams * 16;
  if (p.rows_per_block > 1) smem = std::max(smem, sizeof(float) * p.rows_per_block * static_cast<size_t>(a.width));
  smem += 64 * sizeof(float);
  const int rc = with_kind<T>(p, stages > 0, [&](auto nv, auto kind, auto pipe, auto maxt) {
    const auto kern = rms_norm_bwd_kernel<T, W, decltype(nv)::value, decltype(kind)::value, decltype(pipe)::value,
                                          decltype(maxt)::value>;
    if (host::blocks_per_sm(reinterpret_cast<const void*>(kern), p.threads, smem, dev) == 0)
      return static_cast<int>(MLPK_ERR_CUDA);
    return host::launch_kernel_early(kern, dim3(static_cast<unsigned>(blocks)), p.threads, smem, st, a, stages);
  });
  if (rc || !dw) return rc;
  return host::launch_kernel_early(rms_norm_dw_kernel<W>, dim3(static_cast<unsigned>(ceil_div(a.width, 32))), 1024, 0,
                                   st, static_cast<const float*>(a.part), static_cast<int>(blocks), a.width, dw);
}

// The entry points of one type; w32: the weight is fp32.
template <class T>
int forward_of(const NormArgs& a, bool w32, bool fp8, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (!w32) return fp8 ? forward<T, T, true>(a, st) : forward<T, T, false>(a, st);
  }
  return fp8 ? forward<T, float, true>(a, st) : forward<T, float, false>(a, st);
}
template <class T>
int backward_of(const NormBwdArgs& a, bool w32, int64_t blocks, void* dw, int dev, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (!w32) return backward<T, T>(a, blocks, static_cast<T*>(dw), dev, st);
  }
  return backward<T, float>(a, blocks, static_cast<float*>(dw), dev, st);
}

#define MLPK_NORM_TYPE(NAME)                                                                                      \
  __attribute__((visibility("hidden"))) int forward_##NAME(const NormArgs& a, bool w32, bool fp8, cudaStream_t st); \
  __attribute__((visibility("hidden"))) int backward_##NAME(const NormBwdArgs& a, bool w32, int64_t blocks,         \
                                                            void* dw, int dev, cudaStream_t st)
MLPK_NORM_TYPE(f16);
MLPK_NORM_TYPE(bf16);
MLPK_NORM_TYPE(f32);
#undef MLPK_NORM_TYPE

}  // namespace norm
}  // namespace mlpk
