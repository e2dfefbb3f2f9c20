// C-ABI entry points of the RMS norm (declared in include/mlpk.h): argument
// checks, the choice of the threads that share a row, and the launches.
#include <algorithm>
#include <type_traits>

#include "host.cuh"
#include "norm_kernel.cuh"

namespace {

using namespace mlpk;
using namespace mlpk::host;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Threads a row (tpr) and vectors a thread (nv).  A row of up to 128 vectors
// belongs to a warp or a part of one: no barrier.  Wider ones take 2 vectors a
// thread while that is at most 256 threads, then 4, and 9 where 4 do not reach
// (fp32 rows above 16,384 and the widest ragged ones: 32,767 fp32 values lie in
// up to 8,193 vectors).
struct RowPlan {
  int tpr, nv, rows_per_block, threads;
  bool ragged;
};
RowPlan row_plan(int width, int vec) {
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
    p.nv = nvec <= 512 ? 2 : nvec <= 4096 ? 4 : 9;
    p.tpr = static_cast<int>(ceil_div(ceil_div(nvec, p.nv), 32)) * 32;
  }
  p.rows_per_block = p.tpr <= 32 ? kNormThreads / p.tpr : 1;
  p.threads = p.rows_per_block * p.tpr;
  return p;
}
int vec_of(int dtype) { return dtype == MLPK_DT_F32 ? 4 : 8; }

// Rows under way a thread, of `streams` vectors each: as many as fit in
// `budget`, at least one if that fits a block at all; 0: read directly.
int stages_of(const RowPlan& p, int streams, size_t budget) {
  const size_t stage = static_cast<size_t>(p.nv) * p.threads * streams * 16;
  if (p.nv > 4) return 0;
  const int n = static_cast<int>(std::min<size_t>(budget / stage, kNormStages));
  return n > 0 ? n : stage + 2048 <= static_cast<size_t>(kMaxBlockSmem) ? 1 : 0;
}

// Blocks that loop over the rows: those the device holds at a time, or fewer
// if there are not so many rows.  Ragged rows want a step of whole vectors.
int64_t loop_blocks(int64_t rows, const RowPlan& p, int vec, int64_t resident) {
  const int64_t blocks = ceil_div(rows, p.rows_per_block);
  if (blocks <= resident) return blocks;
  return p.ragged ? std::max<int64_t>(resident / vec, 1) * vec : resident;
}

bool float_type(int dt) { return dt == MLPK_DT_F16 || dt == MLPK_DT_BF16 || dt == MLPK_DT_F32; }

int check_norm(int64_t rows, int width, int dtype, int w_dtype, bool has_w) {
  if (rows < 0 || width < 1) return MLPK_ERR_SHAPE;
  if (!float_type(dtype) || (has_w && w_dtype != dtype && w_dtype != MLPK_DT_F32)) return MLPK_ERR_UNSUPPORTED;
  if (width > kNormMaxWidth) return MLPK_ERR_UNSUPPORTED;
  return MLPK_OK;
}

// f(T, W, NV, RAGGED, PIPE, MAXT) of this call.
template <bool V>
using Bool = std::integral_constant<bool, V>;
template <int V>
using Int = std::integral_constant<int, V>;

template <class T, class W, bool RAGGED, class F>
int with_counts(const RowPlan& p, bool pipe, F&& f) {
  switch (p.nv) {
    case 1: return f(T{}, W{}, Int<1>{}, Bool<RAGGED>{}, Bool<true>{}, Int<256>{});
    case 2: return f(T{}, W{}, Int<2>{}, Bool<RAGGED>{}, Bool<true>{}, Int<256>{});
    case 4:
      if (p.threads <= 512) return f(T{}, W{}, Int<4>{}, Bool<RAGGED>{}, Bool<true>{}, Int<512>{});
      return pipe ? f(T{}, W{}, Int<4>{}, Bool<RAGGED>{}, Bool<true>{}, Int<1024>{})
                  : f(T{}, W{}, Int<4>{}, Bool<RAGGED>{}, Bool<false>{}, Int<1024>{});
    default:
      if constexpr (sizeof(T) == 4 || RAGGED) return f(T{}, W{}, Int<9>{}, Bool<RAGGED>{}, Bool<false>{}, Int<1024>{});
      return MLPK_ERR_UNSUPPORTED;
  }
}
template <class T, class W, class F>
int with_raggedness(const RowPlan& p, bool pipe, F&& f) {
  return p.ragged ? with_counts<T, W, true>(p, pipe, f) : with_counts<T, W, false>(p, pipe, f);
}
template <class F>
int with_types(int dtype, int w_dtype, const RowPlan& p, bool pipe, F&& f) {
  if (dtype == MLPK_DT_F32) return with_raggedness<float, float>(p, pipe, f);
  if (dtype == MLPK_DT_F16)
    return w_dtype == MLPK_DT_F32 ? with_raggedness<__half, float>(p, pipe, f)
                                  : with_raggedness<__half, __half>(p, pipe, f);
  return w_dtype == MLPK_DT_F32 ? with_raggedness<__nv_bfloat16, float>(p, pipe, f)
                                : with_raggedness<__nv_bfloat16, __nv_bfloat16>(p, pipe, f);
}

template <bool FP8>
int norm_forward(NormArgs a, int dtype, int w_dtype, cudaStream_t st) {
  DevInfo di;
  int dev;
  int rc = current_device_info(&di, &dev);
  if (rc) return rc;
  const RowPlan p = row_plan(a.width, vec_of(dtype));
  const int streams = a.r ? 2 : 1;
  const int stages = stages_of(p, streams, 72 * 1024);
  a.tpr = p.tpr;
  size_t slots_at = 128 * sizeof(float);
  if (FP8 && p.ragged && a.group)
    slots_at += ceil_div(sizeof(float) * p.rows_per_block * ceil_div(a.width, kNormGroup), 16) * 16;
  const size_t smem = slots_at + static_cast<size_t>(stages) * p.nv * p.threads * streams * 16;
  return with_types(dtype, w_dtype, p, stages > 0, [&](auto t, auto w, auto nv, auto ragged, auto pipe, auto maxt) {
    const auto kern = rms_norm_fwd_kernel<decltype(t), decltype(w), decltype(nv)::value, decltype(ragged)::value,
                                          decltype(pipe)::value, decltype(maxt)::value, FP8>;
    const int per_sm = blocks_per_sm(reinterpret_cast<const void*>(kern), p.threads, smem, dev);
    if (per_sm == 0) return static_cast<int>(MLPK_ERR_CUDA);
    const int64_t blocks = loop_blocks(a.rows, p, vec_of(dtype), static_cast<int64_t>(di.sm_count) * per_sm);
    return launch_kernel_early(kern, dim3(static_cast<unsigned>(blocks)), p.threads, smem, st, a, stages,
                               static_cast<int>(slots_at));
  });
}

// Blocks of the backward pass, each of which leaves one row of dw's partial
// sums.  (The same for every type and count of inputs, so that the workspace's
// size follows from rows, width and type.)
int64_t bwd_blocks(int64_t rows, int width, int dtype, int sm_count) {
  const RowPlan p = row_plan(width, vec_of(dtype));
  return loop_blocks(rows, p, vec_of(dtype), static_cast<int64_t>(sm_count) * (p.threads <= 256 ? 2 : 1));
}

template <class W>
int dw_sum(const float* part, int64_t nparts, int width, void* dw, cudaStream_t st) {
  return launch_kernel_early(rms_norm_dw_kernel<W>, dim3(static_cast<unsigned>(ceil_div(width, 32))), 1024, 0, st,
                             part, static_cast<int>(nparts), width, static_cast<W*>(dw));
}

}  // namespace

extern "C" {

int mlpk_rms_norm(int64_t rows, int width, int dtype, const void* x, const void* residual, const void* weight,
                  int w_dtype, float eps, void* y, void* h, float* rstd, mlpk_stream_t stream) {
  int rc = check_norm(rows, width, dtype, w_dtype, weight != nullptr);
  if (rc) return rc;
  if (rows == 0) return MLPK_OK;
  if (!x || !y || (residual && !h)) return MLPK_ERR_NULL;
  for (const void* p : {x, residual, weight, static_cast<const void*>(y), static_cast<const void*>(h)})
    if (!aligned16(p)) return MLPK_ERR_ALIGN;
  const NormArgs a = {rows, width, 0, eps, x, residual, weight, y, h, rstd, nullptr, 0};
  return norm_forward<false>(a, dtype, weight ? w_dtype : dtype, static_cast<cudaStream_t>(stream));
}

int mlpk_rms_norm_fp8(int64_t rows, int width, int dtype, const void* x, const void* residual, const void* weight,
                      int w_dtype, float eps, int group, void* q, float* scale, void* h, mlpk_stream_t stream) {
  int rc = check_norm(rows, width, dtype, w_dtype, weight != nullptr);
  if (rc) return rc;
  if (group != 0 && group != kNormGroup) return MLPK_ERR_UNSUPPORTED;
  if (rows == 0) return MLPK_OK;
  if (!x || !q || !scale || (residual && !h)) return MLPK_ERR_NULL;
  for (const void* p : {x, residual, weight, static_cast<const void*>(q), static_cast<const void*>(h)})
    if (!aligned16(p)) return MLPK_ERR_ALIGN;
  const NormArgs a = {rows, width, 0, eps, x, residual, weight, q, h, nullptr, scale, group};
  return norm_forward<true>(a, dtype, weight ? w_dtype : dtype, static_cast<cudaStream_t>(stream));
}

int64_t mlpk_rms_norm_bwd_workspace_size(int64_t rows, int width, int dtype) {
  if (check_norm(rows, width, dtype, dtype, false)) return -1;
  DevInfo di;
  if (current_device_info(&di, nullptr)) return -1;
  return bwd_blocks(rows, width, dtype, di.sm_count) * width * static_cast<int64_t>(sizeof(float));
}

int mlpk_rms_norm_bwd(int64_t rows, int width, int dtype, const void* x, const void* residual, const float* rstd,
                      const void* weight, int w_dtype, const void* grad_y, const void* grad_h, void* dx, void* dw,
                      void* workspace, int64_t workspace_bytes, mlpk_stream_t stream) {
  int rc = check_norm(rows, width, dtype, w_dtype, weight != nullptr);
  if (rc) return rc;
  if (dw && !weight) return MLPK_ERR_NULL;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    if (!dw) return MLPK_OK;
    return cuda_status(cudaMemsetAsync(dw, 0, static_cast<size_t>(width) * (w_dtype == MLPK_DT_F32 ? 4 : 2), st));
  }
  if (!x || !rstd || !grad_y || !dx || (dw && !workspace)) return MLPK_ERR_NULL;
  for (const void* p : {x, residual, weight, grad_y, grad_h, static_cast<const void*>(dx),
                        static_cast<const void*>(workspace)})
    if (!aligned16(p)) return MLPK_ERR_ALIGN;
  DevInfo di;
  int dev;
  if ((rc = current_device_info(&di, &dev)) != MLPK_OK) return rc;
  const RowPlan p = row_plan(width, vec_of(dtype));
  const int64_t blocks = bwd_blocks(rows, width, dtype, di.sm_count);
  if (dw && workspace_bytes < blocks * width * static_cast<int64_t>(sizeof(float))) return MLPK_ERR_SCRATCH;
  const NormBwdArgs a = {rows, width, p.tpr, x, residual, rstd, weight, grad_y, grad_h, dx,
                         dw ? static_cast<float*>(workspace) : nullptr};
  const int streams = 2 + (residual != nullptr) + (grad_h != nullptr);
  const int stages = stages_of(p, streams, 100 * 1024);
  size_t smem = static_cast<size_t>(stages) * p.nv * p.threads * streams * 16;
  if (p.rows_per_block > 1) smem = std::max(smem, sizeof(float) * p.rows_per_block * static_cast<size_t>(width));
  smem += 64 * sizeof(float);
  rc = with_types(dtype, weight ? w_dtype : dtype, p, stages > 0,
                  [&](auto t, auto w, auto nv, auto ragged, auto pipe, auto maxt) {
                    const auto kern =
                        rms_norm_bwd_kernel<decltype(t), decltype(w), decltype(nv)::value, decltype(ragged)::value,
                                            decltype(pipe)::value, decltype(maxt)::value>;
                    if (blocks_per_sm(reinterpret_cast<const void*>(kern), p.threads, smem, dev) == 0)
                      return static_cast<int>(MLPK_ERR_CUDA);
                    return launch_kernel_early(kern, dim3(static_cast<unsigned>(blocks)), p.threads, smem, st, a,
                                               stages);
                  });
  if (rc || !dw) return rc;
  if (w_dtype == MLPK_DT_F32) return dw_sum<float>(a.part, blocks, width, dw, st);
  if (w_dtype == MLPK_DT_F16) return dw_sum<__half>(a.part, blocks, width, dw, st);
  return dw_sum<__nv_bfloat16>(a.part, blocks, width, dw, st);
}

}  // extern "C"
