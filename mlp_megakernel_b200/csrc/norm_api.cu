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

// Threads a row (tpr) and vectors a thread (nv) for a row of nvec vectors.
struct RowPlan {
  int tpr, nv, rows_per_block, threads;
};
RowPlan row_plan(int nvec, bool wide) {
  RowPlan p;
  if (nvec <= 32) {
    p.nv = 1;
    p.tpr = 1;
    while (p.tpr < nvec) p.tpr *= 2;
  } else if (wide ? nvec <= 128 : nvec <= 256) {
    p.tpr = 32;
    p.nv = wide ? (nvec <= 64 ? 2 : 4) : 8;
  } else {
    p.nv = wide ? (nvec <= 4096 ? 4 : 8) : (nvec <= 8192 ? 8 : 32);
    p.tpr = static_cast<int>(ceil_div(ceil_div(nvec, p.nv), 32)) * 32;
  }
  p.rows_per_block = p.tpr <= 32 ? kNormThreads / p.tpr : 1;
  p.threads = p.rows_per_block * p.tpr;
  return p;
}

bool float_type(int dt) { return dt == MLPK_DT_F16 || dt == MLPK_DT_BF16 || dt == MLPK_DT_F32; }

int check_norm(int64_t rows, int width, int dtype, int w_dtype, bool has_w) {
  if (rows < 0 || width < 1) return MLPK_ERR_SHAPE;
  if (!float_type(dtype) || (has_w && w_dtype != dtype && w_dtype != MLPK_DT_F32)) return MLPK_ERR_UNSUPPORTED;
  if (width > kNormMaxWidth) return MLPK_ERR_UNSUPPORTED;
  return MLPK_OK;
}

// f(T, W, VEC, NV) with the types and counts of this call.
template <class T, class W, class F>
int with_counts(int width, F&& f, RowPlan* plan) {
  constexpr int V = kVecOf<T>;
  if (width % V == 0) {
    *plan = row_plan(width / V, true);
    using VT = std::integral_constant<int, V>;
    switch (plan->nv) {
      case 1: return f(T{}, W{}, VT{}, std::integral_constant<int, 1>{});
      case 2: return f(T{}, W{}, VT{}, std::integral_constant<int, 2>{});
      case 4: return f(T{}, W{}, VT{}, std::integral_constant<int, 4>{});
      default: return f(T{}, W{}, VT{}, std::integral_constant<int, 8>{});
    }
  }
  *plan = row_plan(width, false);
  using V1 = std::integral_constant<int, 1>;
  switch (plan->nv) {
    case 1: return f(T{}, W{}, V1{}, std::integral_constant<int, 1>{});
    case 8: return f(T{}, W{}, V1{}, std::integral_constant<int, 8>{});
    default: return f(T{}, W{}, V1{}, std::integral_constant<int, 32>{});
  }
}
template <class F>
int with_types(int dtype, int w_dtype, int width, RowPlan* plan, F&& f) {
  if (dtype == MLPK_DT_F32) return with_counts<float, float>(width, f, plan);
  if (dtype == MLPK_DT_F16)
    return w_dtype == MLPK_DT_F32 ? with_counts<__half, float>(width, f, plan)
                                  : with_counts<__half, __half>(width, f, plan);
  return w_dtype == MLPK_DT_F32 ? with_counts<__nv_bfloat16, float>(width, f, plan)
                                : with_counts<__nv_bfloat16, __nv_bfloat16>(width, f, plan);
}

template <bool FP8>
int norm_forward(NormArgs a, int dtype, int w_dtype, cudaStream_t st) {
  DevInfo di;
  int rc = current_device_info(&di, nullptr);
  if (rc) return rc;
  RowPlan plan;
  return with_types(dtype, w_dtype, a.width, &plan, [&](auto t, auto w, auto vec, auto nv) {
    a.tpr = plan.tpr;
    const int64_t blocks = ceil_div(a.rows, plan.rows_per_block);
    if (blocks > 0x7fffffff) return static_cast<int>(MLPK_ERR_SHAPE);
    size_t smem = 64 * sizeof(float);
    if (FP8 && decltype(vec)::value == 1 && a.group)
      smem += sizeof(float) * plan.rows_per_block * ceil_div(a.width, kNormGroup);
    return launch_kernel_early(
        rms_norm_fwd_kernel<decltype(t), decltype(w), decltype(vec)::value, decltype(nv)::value, FP8>,
        dim3(static_cast<unsigned>(blocks)), plan.threads, smem, st, a);
  });
}

// Blocks of the backward pass, each of which leaves one row of dw's partial
// sums: enough to fill the SMs, and no more than there are rows for.
int64_t bwd_blocks(int64_t rows, const RowPlan& p, int sm_count) {
  const int per_sm = std::max(1, 1024 / p.threads);
  return std::min(ceil_div(rows, p.rows_per_block), static_cast<int64_t>(sm_count) * per_sm);
}
RowPlan plan_of(int width, int dtype) {
  const int v = dtype == MLPK_DT_F32 ? 4 : 8;
  return width % v == 0 ? row_plan(width / v, true) : row_plan(width, false);
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
  return bwd_blocks(rows, plan_of(width, dtype), di.sm_count) * width * static_cast<int64_t>(sizeof(float));
}

int mlpk_rms_norm_bwd(int64_t rows, int width, int dtype, const void* h, const float* rstd, const void* weight,
                      int w_dtype, const void* grad_y, const void* grad_h, void* dx, void* dw, void* workspace,
                      int64_t workspace_bytes, mlpk_stream_t stream) {
  int rc = check_norm(rows, width, dtype, w_dtype, weight != nullptr);
  if (rc) return rc;
  if (dw && !weight) return MLPK_ERR_NULL;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  DevInfo di;
  if (rows == 0) {
    if (!dw) return MLPK_OK;
    return cuda_status(cudaMemsetAsync(dw, 0, static_cast<size_t>(width) * (w_dtype == MLPK_DT_F32 ? 4 : 2), st));
  }
  if (!h || !rstd || !grad_y || !dx || (dw && !workspace)) return MLPK_ERR_NULL;
  for (const void* p : {h, weight, grad_y, grad_h, static_cast<const void*>(dx), static_cast<const void*>(workspace)})
    if (!aligned16(p)) return MLPK_ERR_ALIGN;
  if ((rc = current_device_info(&di, nullptr)) != MLPK_OK) return rc;
  RowPlan plan;
  NormBwdArgs a = {rows, width, 0, h, rstd, weight, grad_y, grad_h, dx, dw ? static_cast<float*>(workspace) : nullptr};
  const int64_t blocks = bwd_blocks(rows, plan_of(width, dtype), di.sm_count);
  if (dw && workspace_bytes < blocks * width * static_cast<int64_t>(sizeof(float))) return MLPK_ERR_SCRATCH;
  rc = with_types(dtype, weight ? w_dtype : dtype, width, &plan, [&](auto t, auto w, auto vec, auto nv) {
    a.tpr = plan.tpr;
    const size_t smem =
        sizeof(float) * (64 + (plan.rows_per_block > 1 ? static_cast<size_t>(plan.rows_per_block) * width : 0));
    return launch_kernel_early(rms_norm_bwd_kernel<decltype(t), decltype(w), decltype(vec)::value, decltype(nv)::value>,
                               dim3(static_cast<unsigned>(blocks)), plan.threads, smem, st, a);
  });
  if (rc || !dw) return rc;
  if (w_dtype == MLPK_DT_F32) return dw_sum<float>(a.part, blocks, width, dw, st);
  if (w_dtype == MLPK_DT_F16) return dw_sum<__half>(a.part, blocks, width, dw, st);
  return dw_sum<__nv_bfloat16>(a.part, blocks, width, dw, st);
}

}  // extern "C"
