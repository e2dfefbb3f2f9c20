// C-ABI entry points of the feed-forward operators (declared in include/mlpk.h):
// argument checks, the products each call is made of, and the launches of what
// stands beside them (ff_kernel.cuh).
#define MLPK_STATUS_BY_POINTER
#include "ff_kernel.cuh"

#include <algorithm>
#include <initializer_list>

#include "host.cuh"
#include "product_epi.cuh"
#include "product_launch.cuh"

namespace {

using namespace mlpk;
using namespace mlpk::host;
using mlpk::product::Product;

constexpr int kMaxWidth = 1 << 20;  // of a feed-forward operator's rows

bool operand_type(int dt) { return dt == MLPK_DT_F16 || dt == MLPK_DT_BF16; }
bool value_type(int dt) { return operand_type(dt) || dt == MLPK_DT_F32; }
int64_t ceil_to(int64_t v, int64_t unit) { return (v + unit - 1) / unit; }

// Rows, widths (multiples of 8: 16-byte rows for TMA), types, activation, what is kept.
int check_call(int64_t rows, std::initializer_list<int> widths, int dtype, int act, int keep) {
  if (rows < 0 || rows > 0x7fffffff - 256) return MLPK_ERR_SHAPE;
  for (int w : widths)
    if (w < 1) return MLPK_ERR_SHAPE;
  if (!operand_type(dtype) || act < MLPK_ACT_NONE || act > MLPK_ACT_SIGMOID || keep < MLPK_KEEP_NONE ||
      keep > MLPK_KEEP_FP8)
    return MLPK_ERR_UNSUPPORTED;
  for (int w : widths)
    if (w % 8 || w > kMaxWidth) return MLPK_ERR_UNSUPPORTED;
  return MLPK_OK;
}
int check_layout(int layout) { return layout == MLPK_W_IN_OUT || layout == MLPK_W_OUT_IN ? MLPK_OK : MLPK_ERR_UNSUPPORTED; }
int check_ptrs(std::initializer_list<const void*> needed, std::initializer_list<const void*> maybe = {}) {
  for (const void* p : needed)
    if (!p) return MLPK_ERR_NULL;
  for (const void* p : needed)
    if (!aligned16(p)) return MLPK_ERR_ALIGN;
  for (const void* p : maybe)
    if (!aligned16(p)) return MLPK_ERR_ALIGN;
  return MLPK_OK;
}

int run(const Product& p, int dtype, mlpk_stream_t stream) {
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == MLPK_DT_F16 ? product::launch_f16(p, st) : product::launch_bf16(p, st);
}

// What a product keeps for the backward (or reads of it): g and u, or z.
void set_keep(Product* c, int keep, int width, void* const (&v)[2], float* const (&scale)[2]) {
  c->keep_kind = keep;
  if (keep != MLPK_KEEP_FP8) return;
  c->q_pitch = mlpk_fp8_pitch(width);
  c->scale_pitch = static_cast<int>(ceil_to(width, kGroupCols));
  for (int i = 0; i < 2; ++i) {
    c->q[i] = static_cast<uint8_t*>(v[i]);
    c->scale[i] = scale[i];
  }
}

// The calls as products, their operands aside.
Product linear_product(int64_t rows, int d_in, int d_out, int w_layout, int keep) {
  Product c;
  c.epi = kEpiLinear;
  c.keep_kind = keep;
  c.rows = rows;
  c.cols = d_out;
  c.k[0] = d_in;
  c.b_mn = w_layout == MLPK_W_IN_OUT;
  return c;
}
Product dx_product(int64_t rows, int d_in, int d_out, int count, int w_layout) {
  Product c;
  c.epi = kEpiPlain;
  c.rows = rows;
  c.cols = d_in;
  for (int i = 0; i < count; ++i) c.k[i] = d_out;
  c.b_mn = w_layout == MLPK_W_OUT_IN;
  return c;
}
Product dw_product(int64_t rows, int d_in, int d_out, int count, int w_layout) {
  Product c;
  c.epi = kEpiPlain;
  c.outputs = count;
  c.k[0] = rows;
  c.a_mn = c.b_mn = true;
  const bool in_out = w_layout == MLPK_W_IN_OUT;
  c.out_a = !in_out;
  c.rows = in_out ? d_in : d_out;
  c.cols = in_out ? d_out : d_in;
  return c;
}
int64_t product_workspace(const Product& c) {
  DevInfo di;
  if (c.rows == 0 || c.k[0] == 0) return 0;
  return current_device_info(&di, nullptr) ? -1 : product::workspace_bytes(c, di.sm_count);
}

template <class F>
int with_value_type(int dtype, F&& f) {
  switch (dtype) {
    case MLPK_DT_F16: return f(__half{});
    case MLPK_DT_BF16: return f(__nv_bfloat16{});
    default: return f(float{});
  }
}
// Blocks of a kernel that goes over its work in turns: as many as the SMs hold at
// a time (0: a failure).
template <class K>
unsigned stream_blocks(K kern, int64_t work, const DevInfo& di, int dev) {
  const int64_t most =
      static_cast<int64_t>(di.sm_count) * blocks_per_sm(reinterpret_cast<const void*>(kern), kStreamThreads, 0, dev);
  return static_cast<unsigned>(std::min(std::max<int64_t>(work, 1), most));
}

// Blocks of linear_dz_kernel over the rows: what the SMs hold at a time, each
// thread with 4 rows (two turns) at least.
int dz_parts(int64_t rows, int width, int sm_count) {
  const int64_t across = ceil_to(width, 8 * kDzVectors);
  const int64_t want = std::max<int64_t>(1, static_cast<int64_t>(sm_count) * kDzBlocks / across);
  return static_cast<int>(std::max<int64_t>(1, std::min(want, ceil_to(rows, 4 * kDzRows))));
}

template <class T, bool FP8>
auto dz_kernel(int act) -> void (*)(DzArgs) {
  switch (act) {
    case kActRelu: return linear_dz_kernel<T, kActRelu, FP8>;
    case kActSilu: return linear_dz_kernel<T, kActSilu, FP8>;
    case kActGeluTanh: return linear_dz_kernel<T, kActGeluTanh, FP8>;
    case kActSoftplus: return linear_dz_kernel<T, kActSoftplus, FP8>;
    case kActSigmoid: return linear_dz_kernel<T, kActSigmoid, FP8>;
    default: return linear_dz_kernel<T, kActNone, false>;
  }
}

}  // namespace

extern "C" {

int64_t mlpk_fp8_pitch(int width) { return width < 1 ? -1 : ceil_to(width, kGroupCols) * kGroupCols; }

int64_t mlpk_linear_workspace_size(int64_t rows, int d_in, int d_out, int dtype, int w_layout, int keep) {
  if (check_call(rows, {d_in, d_out}, dtype, 0, keep) || check_layout(w_layout)) return -1;
  return product_workspace(linear_product(rows, d_in, d_out, w_layout, keep));
}

int mlpk_linear(int64_t rows, int d_in, int d_out, int dtype, const void* x, const void* w, int w_layout,
                const void* bias, int bias_dtype, int act, const void* residual, void* out, int keep, void* z,
                float* z_scale, void* workspace, int64_t workspace_bytes, mlpk_stream_t stream) {
  int rc = check_call(rows, {d_in, d_out}, dtype, act, keep);
  if (rc || (rc = check_layout(w_layout))) return rc;
  if (bias && bias_dtype != dtype && bias_dtype != MLPK_DT_F32) return MLPK_ERR_UNSUPPORTED;
  if (rows == 0) return MLPK_OK;
  if ((rc = check_ptrs({x, w, out}, {bias, residual, z, workspace}))) return rc;
  if ((keep != MLPK_KEEP_NONE && !z) || (keep == MLPK_KEEP_FP8 && !z_scale)) return MLPK_ERR_NULL;
  Product c = linear_product(rows, d_in, d_out, w_layout, keep);
  c.act = act;
  c.a[0] = x;
  c.b[0] = w;
  c.workspace = workspace;
  c.workspace_bytes = workspace_bytes;
  c.bias = bias;
  c.bias32 = bias_dtype == MLPK_DT_F32;
  c.in[0] = residual;
  c.out[0] = out;
  if (keep == MLPK_KEEP_16) c.keep[0] = z;
  set_keep(&c, keep, d_out, {z, nullptr}, {z_scale, nullptr});
  return run(c, dtype, stream);
}

int64_t mlpk_linear_dz_workspace_size(int64_t rows, int width, int dtype) {
  if (check_call(rows, {width}, dtype, 0, 0)) return -1;
  DevInfo di;
  if (current_device_info(&di, nullptr)) return -1;
  return static_cast<int64_t>(dz_parts(rows, width, di.sm_count)) * width * static_cast<int64_t>(sizeof(float));
}

int mlpk_linear_dz(int64_t rows, int width, int dtype, int act, const void* grad_out, int keep, const void* z,
                   const float* z_scale, void* dz, void* db, int db_dtype, void* workspace, int64_t workspace_bytes,
                   mlpk_stream_t stream) {
  int rc = check_call(rows, {width}, dtype, act, keep);
  if (rc) return rc;
  if (db && db_dtype != dtype && db_dtype != MLPK_DT_F32) return MLPK_ERR_UNSUPPORTED;
  if (!dz && !db) return MLPK_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0)
    return db ? cuda_status(cudaMemsetAsync(db, 0, static_cast<size_t>(width) * (db_dtype == MLPK_DT_F32 ? 4 : 2), st))
              : MLPK_OK;
  if ((rc = check_ptrs({grad_out}, {z, dz, workspace}))) return rc;
  if (act != MLPK_ACT_NONE && (!z || keep == MLPK_KEEP_NONE || (keep == MLPK_KEEP_FP8 && !z_scale))) return MLPK_ERR_NULL;
  if (db && !workspace) return MLPK_ERR_NULL;
  DevInfo di;
  if ((rc = current_device_info(&di, nullptr))) return rc;
  const int parts = dz_parts(rows, width, di.sm_count);
  if (db && workspace_bytes < static_cast<int64_t>(parts) * width * static_cast<int64_t>(sizeof(float)))
    return MLPK_ERR_SCRATCH;
  DzArgs a = {rows, width, static_cast<int>(ceil_to(width, kGroupCols)), mlpk_fp8_pitch(width), grad_out, z,
              z_scale, dz, db ? static_cast<float*>(workspace) : nullptr};
  const dim3 grid(static_cast<unsigned>(ceil_to(width, 8 * kDzVectors)), parts);
  const bool fp8 = keep == MLPK_KEEP_FP8;
  const auto kern = dtype == MLPK_DT_F16 ? (fp8 ? dz_kernel<__half, true>(act) : dz_kernel<__half, false>(act))
                                         : (fp8 ? dz_kernel<__nv_bfloat16, true>(act) : dz_kernel<__nv_bfloat16, false>(act));
  rc = launch_kernel_early(kern, grid, kStreamThreads, 0, st, a);
  if (rc || !db) return rc;
  return with_value_type(db_dtype, [&](auto t) {
    using W = decltype(t);
    return launch_kernel_early(bias_grad_kernel<W>, dim3(static_cast<unsigned>(ceil_to(width, 32))), kStreamThreads, 0,
                               st, width, parts, static_cast<const float*>(workspace), static_cast<W*>(db));
  });
}

int64_t mlpk_linear_dx_workspace_size(int64_t rows, int d_in, int d_out, int dtype, int count, int w_layout) {
  if (check_call(rows, {d_in, d_out}, dtype, 0, 0) || check_layout(w_layout) || count < 1 || count > 2) return -1;
  return product_workspace(dx_product(rows, d_in, d_out, count, w_layout));
}

int mlpk_linear_dx(int64_t rows, int d_in, int d_out, int dtype, int count, const void* const* dz,
                   const void* const* w, int w_layout, void* dx, void* workspace, int64_t workspace_bytes,
                   mlpk_stream_t stream) {
  int rc = check_call(rows, {d_in, d_out}, dtype, 0, 0);
  if (rc || (rc = check_layout(w_layout))) return rc;
  if (count != 1 && count != 2) return MLPK_ERR_SHAPE;
  if (!dz || !w) return MLPK_ERR_NULL;
  if (rows == 0) return MLPK_OK;
  if ((rc = check_ptrs({dx, dz[0], w[0], dz[count - 1], w[count - 1]}, {workspace}))) return rc;
  Product c = dx_product(rows, d_in, d_out, count, w_layout);
  for (int i = 0; i < count; ++i) {
    c.a[i] = dz[i];
    c.b[i] = w[i];
  }
  c.out[0] = dx;
  c.workspace = workspace;
  c.workspace_bytes = workspace_bytes;
  return run(c, dtype, stream);
}

int64_t mlpk_linear_dw_workspace_size(int64_t rows, int d_in, int d_out, int dtype, int count, int w_layout) {
  if (check_call(rows, {d_in, d_out}, dtype, 0, 0) || check_layout(w_layout) || count < 1 || count > 2) return -1;
  return product_workspace(dw_product(rows, d_in, d_out, count, w_layout));
}

int mlpk_linear_dw(int64_t rows, int d_in, int d_out, int dtype, int count, const void* x, const void* const* dz,
                   void* const* dw, int w_layout, void* workspace, int64_t workspace_bytes, mlpk_stream_t stream) {
  int rc = check_call(rows, {d_in, d_out}, dtype, 0, 0);
  if (rc || (rc = check_layout(w_layout))) return rc;
  if (count != 1 && count != 2) return MLPK_ERR_SHAPE;
  if (!dz || !dw) return MLPK_ERR_NULL;
  if (rows == 0) {
    const size_t bytes = static_cast<size_t>(d_in) * d_out * 2;
    for (int i = 0; i < count; ++i)
      if (!dw[i]) return MLPK_ERR_NULL;
      else if ((rc = cuda_status(cudaMemsetAsync(dw[i], 0, bytes, static_cast<cudaStream_t>(stream))))) return rc;
    return MLPK_OK;
  }
  if ((rc = check_ptrs({x, dz[0], dz[count - 1], dw[0], dw[count - 1]}, {workspace}))) return rc;
  Product c = dw_product(rows, d_in, d_out, count, w_layout);
  const bool in_out = w_layout == MLPK_W_IN_OUT;
  (in_out ? c.a : c.b)[0] = x;
  for (int i = 0; i < count; ++i) {
    (in_out ? c.b : c.a)[i] = dz[i];
    c.out[i] = dw[i];
  }
  c.workspace = workspace;
  c.workspace_bytes = workspace_bytes;
  return run(c, dtype, stream);
}

int mlpk_gated(int64_t rows, int d_in, int hidden, int dtype, int act, const void* x, const void* w_gate,
               const void* w_up, int w_layout, void* h, int keep, void* g, float* g_scale, void* u, float* u_scale,
               mlpk_stream_t stream) {
  int rc = check_call(rows, {d_in, hidden}, dtype, act, keep);
  if (rc || (rc = check_layout(w_layout))) return rc;
  if (rows == 0) return MLPK_OK;
  if ((rc = check_ptrs({x, w_gate, w_up, h}, {g, u}))) return rc;
  if ((keep != MLPK_KEEP_NONE && (!g || !u)) || (keep == MLPK_KEEP_FP8 && (!g_scale || !u_scale))) return MLPK_ERR_NULL;
  Product c;
  c.epi = kEpiGated;
  c.act = act;
  c.rows = rows;
  c.cols = hidden;
  c.k[0] = d_in;
  c.a[0] = x;
  c.b[0] = w_gate;
  c.b[1] = w_up;
  c.b_mn = w_layout == MLPK_W_IN_OUT;
  c.out[0] = h;
  if (keep == MLPK_KEEP_16) {
    c.keep[0] = g;
    c.keep[1] = u;
  }
  set_keep(&c, keep, hidden, {g, u}, {g_scale, u_scale});
  return run(c, dtype, stream);
}

int mlpk_gated_bwd(int64_t rows, int hidden, int d_out, int dtype, int act, const void* grad_out, const void* w_down,
                   int w_layout, int keep, const void* g, const float* g_scale, const void* u, const float* u_scale,
                   void* dg, void* du, void* h, mlpk_stream_t stream) {
  int rc = check_call(rows, {hidden, d_out}, dtype, act, keep);
  if (rc || (rc = check_layout(w_layout))) return rc;
  if (keep == MLPK_KEEP_NONE) return MLPK_ERR_UNSUPPORTED;
  if (rows == 0) return MLPK_OK;
  if ((rc = check_ptrs({grad_out, w_down, g, u, dg, du, h}))) return rc;
  if (keep == MLPK_KEEP_FP8 && (!g_scale || !u_scale)) return MLPK_ERR_NULL;
  Product c;
  c.epi = kEpiGatedBwd;
  c.act = act;
  c.rows = rows;
  c.cols = hidden;
  c.k[0] = d_out;
  c.a[0] = grad_out;
  c.b[0] = w_down;
  c.b_mn = w_layout == MLPK_W_OUT_IN;  // dh = grad_out w_down^T
  c.out[0] = dg;
  c.out[1] = du;
  c.keep[0] = h;
  if (keep == MLPK_KEEP_16) {
    c.in[0] = g;
    c.in[1] = u;
  }
  set_keep(&c, keep, hidden, {const_cast<void*>(g), const_cast<void*>(u)},
           {const_cast<float*>(g_scale), const_cast<float*>(u_scale)});
  return run(c, dtype, stream);
}

int mlpk_fp8_checkpoint(int64_t rows, int width, int dtype, const void* x, void* q, float* scale,
                        mlpk_stream_t stream) {
  if (rows < 0 || width < 1) return MLPK_ERR_SHAPE;
  if (!value_type(dtype)) return MLPK_ERR_UNSUPPORTED;
  if (rows == 0) return MLPK_OK;
  int rc = check_ptrs({x, q, scale});
  if (rc) return rc;
  DevInfo di;
  int dev;
  if ((rc = current_device_info(&di, &dev))) return rc;
  const int groups = static_cast<int>(ceil_to(width, kGroupCols));
  if (rows > INT64_MAX / width) return MLPK_ERR_SHAPE;
  const bool vectors = width % 8 == 0;
  const int team = vectors ? 8 : 32;
  return with_value_type(dtype, [&](auto t) {
    using T = decltype(t);
    const auto kern = vectors ? checkpoint_kernel<T, true> : checkpoint_kernel<T, false>;
    const unsigned blocks = stream_blocks(kern, ceil_to(rows * groups, 2 * (kStreamThreads / team)), di, dev);
    if (!blocks) return static_cast<int>(MLPK_ERR_CUDA);
    return launch_kernel_early(kern, dim3(blocks), kStreamThreads, 0, static_cast<cudaStream_t>(stream), rows, width, groups,
                               static_cast<const T*>(x), static_cast<uint8_t*>(q), scale);
  });
}

int mlpk_fp8_restore(int64_t rows, int width, int dtype, const void* q, const float* scale, void* x,
                     mlpk_stream_t stream) {
  if (rows < 0 || width < 1) return MLPK_ERR_SHAPE;
  if (!value_type(dtype)) return MLPK_ERR_UNSUPPORTED;
  if (rows == 0) return MLPK_OK;
  int rc = check_ptrs({q, scale, x});
  if (rc) return rc;
  DevInfo di;
  int dev;
  if ((rc = current_device_info(&di, &dev))) return rc;
  if (rows > INT64_MAX / width) return MLPK_ERR_SHAPE;
  const int groups = static_cast<int>(ceil_to(width, kGroupCols));
  const int64_t total = rows * width;
  return with_value_type(dtype, [&](auto t) {
    using T = decltype(t);
    const auto kern = width % 16 == 0 ? restore_kernel<T, true> : restore_kernel<T, false>;
    const unsigned blocks = stream_blocks(kern, ceil_to(total, 16 * 2 * kStreamThreads), di, dev);
    if (!blocks) return static_cast<int>(MLPK_ERR_CUDA);
    return launch_kernel_early(kern, dim3(blocks), kStreamThreads, 0, static_cast<cudaStream_t>(stream), total, width,
                               groups, static_cast<const uint8_t*>(q), scale, static_cast<T*>(x));
  });
}

}  // extern "C"
