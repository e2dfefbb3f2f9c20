// C-ABI entry points of the RMS norm (declared in include/mlpk.h): argument
// checks, and the choice of the type's launches (norm_launch.cuh).
#include "norm_launch.cuh"

namespace {

using namespace mlpk;
using namespace mlpk::host;

bool float_type(int dt) { return dt == MLPK_DT_F16 || dt == MLPK_DT_BF16 || dt == MLPK_DT_F32; }

int check_norm(int64_t rows, int width, int dtype, int w_dtype, bool has_w) {
  if (rows < 0 || width < 1) return MLPK_ERR_SHAPE;
  if (!float_type(dtype) || (has_w && w_dtype != dtype && w_dtype != MLPK_DT_F32)) return MLPK_ERR_UNSUPPORTED;
  if (width > kNormMaxWidth) return MLPK_ERR_UNSUPPORTED;
  return MLPK_OK;
}

int norm_forward(const NormArgs& a, int dtype, int w_dtype, bool fp8, cudaStream_t st) {
  const bool w32 = a.w && w_dtype == MLPK_DT_F32;
  switch (dtype) {
    case MLPK_DT_F16: return norm::forward_f16(a, w32, fp8, st);
    case MLPK_DT_BF16: return norm::forward_bf16(a, w32, fp8, st);
    default: return norm::forward_f32(a, w32, fp8, st);
  }
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
  return norm_forward(a, dtype, w_dtype, false, static_cast<cudaStream_t>(stream));
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
  return norm_forward(a, dtype, w_dtype, true, static_cast<cudaStream_t>(stream));
}

int64_t mlpk_rms_norm_bwd_workspace_size(int64_t rows, int width, int dtype) {
  if (check_norm(rows, width, dtype, dtype, false)) return -1;
  DevInfo di;
  if (current_device_info(&di, nullptr)) return -1;
  return norm::bwd_blocks(rows, width, dtype, di.sm_count) * width * static_cast<int64_t>(sizeof(float));
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
  const int64_t blocks = norm::bwd_blocks(rows, width, dtype, di.sm_count);
  if (dw && workspace_bytes < blocks * width * static_cast<int64_t>(sizeof(float))) return MLPK_ERR_SCRATCH;
  const NormBwdArgs a = {rows, width, 0, x, residual, rstd, weight, grad_y, grad_h, dx,
                         dw ? static_cast<float*>(workspace) : nullptr};
  const bool w32 = weight && w_dtype == MLPK_DT_F32;
  switch (dtype) {
    case MLPK_DT_F16: return norm::backward_f16(a, w32, blocks, dw, dev, st);
    case MLPK_DT_BF16: return norm::backward_bf16(a, w32, blocks, dw, dev, st);
    default: return norm::backward_f32(a, w32, blocks, dw, dev, st);
  }
}

}  // extern "C"
