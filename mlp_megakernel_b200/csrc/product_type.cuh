// The launches of one operand type (included by product_f16.cu and
// product_bf16.cu alone).
#pragma once
#define MLPK_STATUS_BY_POINTER
#include <algorithm>
#include <cstring>
#include <utility>

#include "few_rows_kernel.cuh"
#include "product_kernel.cuh"
#include "product_launch.cuh"
#include "tail_kernel.cuh"

namespace mlpk {
namespace product {

using namespace mlpk::host;

// The operands' format in an instruction descriptor made for fp16.
inline uint32_t type_bits(bool bf16) { return bf16 ? (1u << 7 | 1u << 10) : 0u; }

inline int ceil_div_int(int64_t a, int64_t b) { return static_cast<int>((a + b - 1) / b); }

template <class T, int EPI, int TN>
int launch_tiles(const Product& c, const ProductPlan& plan, const DevInfo& di, int dev, cudaStream_t st) {
  using Cfg = ProductCfg<EPI, TN>;
  int rc;
  const auto kern = product_kernel<T, EPI, TN>;
  const void* entry = reinterpret_cast<const void*>(kern);
  if (!blocks_per_sm(entry, kProductThreads, Cfg::SMEM, dev)) return MLPK_ERR_CUDA;
  const int pairs = std::min(clusters_at_once(entry, kProductThreads, Cfg::SMEM, 2, dev), di.sm_count / 2);
  if (pairs < 1) return MLPK_ERR_CUDA;

  ProductArgs a;
  std::memset(&a, 0, sizeof(a));
  a.rows = static_cast<int>(c.rows);
  a.cols = c.cols;
  a.nk0 = ceil_div_int(c.k[0], kBlockK);
  a.nk = a.nk0 + ceil_div_int(c.k[1], kBlockK);
  a.tiles_m = ceil_div_int(c.rows, kPairRows);
  a.tile_cols = plan.cols;
  a.b_bytes = c.b_mn ? Cfg::B_BYTES : plan.cols / 2 * kBlockK * 2;
  a.tiles_n = ceil_div_int(c.cols, EPI == kEpiGated ? plan.cols / 2 : plan.cols);
  a.outputs = c.outputs;
  a.group = 8;
  if (plan.items() > 0x7fffffff - 256) return MLPK_ERR_SHAPE;
  a.full = static_cast<int>(plan.full);
  a.splits = plan.splits;
  a.items = static_cast<int>(plan.items());
  a.a_mn = c.a_mn;
  a.b_mn = c.b_mn;
  a.out_a = c.out_a;
  a.idesc = make_idesc_f16(kPairRows, plan.cols, c.a_mn, c.b_mn) |
            type_bits(std::is_same_v<T, __nv_bfloat16>);
  a.act = c.act;
  a.keep_kind = c.keep_kind;
  a.bias = c.bias;
  a.bias32 = c.bias32;
  a.status = device_status_word(dev);
  if (!a.status) return MLPK_ERR_CUDA;
  a.partials = static_cast<float*>(c.workspace);
  a.residual = EPI == kEpiLinear ? c.in[0] : nullptr;
  a.q_pitch = c.q_pitch;
  a.scale_pitch = c.scale_pitch;
  for (int i = 0; i < 2; ++i) {
    a.q[i] = c.q[i];
    a.scale[i] = c.scale[i];
    const uint64_t k = i == 1 && c.k[1] > 0 ? c.k[1] : c.k[0];
    const uint64_t rows = c.rows, cols = c.cols;
    if (c.a[i] && (rc = c.a_mn ? make_map_2d(&a.a[i], c.a[i], rows, k, 64, kBlockK)
                               : make_map_2d(&a.a[i], c.a[i], k, rows, kBlockK, 128)))
      return rc;
    if (c.b[i] && (rc = c.b_mn ? make_map_2d(&a.b[i], c.b[i], cols, k, 64, kBlockK)
                               : make_map_2d(&a.b[i], c.b[i], k, cols, kBlockK, plan.cols / 2)))
      return rc;
    for (const auto& [map, v] : {std::make_pair(&a.in[i], EPI == kEpiGatedBwd ? c.in[i] : nullptr),
                                 std::make_pair(&a.out[i], const_cast<const void*>(c.out[i])),
                                 std::make_pair(&a.keep[i], const_cast<const void*>(c.keep[i]))})
      if (v && (rc = make_map_2d(map, v, cols, rows, Cfg::CHUNK, 32))) return rc;
  }
  rc = launch_kernel_early(kern, dim3(2 * static_cast<unsigned>(std::min(a.items, pairs))), kProductThreads, Cfg::SMEM, st, a);
  if (rc || plan.splits == 1) return rc;
  if constexpr (EPI == kEpiPlain || EPI == kEpiLinear) {
    const TailArgs t = {a.partials, {c.out[0], c.out[1]}, a.rows, a.cols, a.tiles_m, a.tiles_n, a.outputs, a.group,
                        a.full,     a.splits,             a.act,  a.bias32, a.bias,  a.residual};
    rc = launch_kernel_early(tail_sum_kernel<T, TN>, dim3(256 * TN / 8 / kTailThreads, static_cast<unsigned>(plan.tail)),
                             kTailThreads, 0, st, t);
  }
  return rc;
}

inline int blocks_of(const Product& c) { return ceil_div_int(c.k[0], kBlockK) + ceil_div_int(c.k[1], kBlockK); }

// The tiles of a product (product_plan.cuh).  A gate's checkpoint needs the wide
// tile's 128 columns, and so does what reads it.
inline ProductPlan plan_of(const Product& c, int pairs) {
  return product_plan(c.rows, c.cols, c.outputs, c.epi == kEpiGated ? 128 : 256, blocks_of(c), pairs,
                      c.epi == kEpiPlain || (c.epi == kEpiLinear && c.keep_kind == kKeepNone),
                      c.keep_kind != kKeep8 || c.epi == kEpiLinear,
                      c.epi == kEpiPlain || (c.epi == kEpiLinear && c.keep_kind != kKeep8));
}
inline FewPlan few_plan_of(const Product& c, int sm_count) {
  return few_plan(c.rows, c.cols, blocks_of(c), c.epi == kEpiGated ? 64 : 128, sm_count);
}

template <class T, int EPI>
int launch_few(const Product& c, const DevInfo& di, int dev, cudaStream_t st) {
  int rc;
  constexpr bool GATED = EPI == kEpiGated;
  FewArgs a;
  std::memset(&a, 0, sizeof(a));
  a.rows = static_cast<int>(c.rows);
  a.cols = c.cols;
  a.nk0 = ceil_div_int(c.k[0], kBlockK);
  a.nk = a.nk0 + ceil_div_int(c.k[1], kBlockK);
  const FewPlan plan = few_plan_of(c, di.sm_count);
  a.nt = plan.nt;
  a.stages = plan.stages;
  a.w_mn = c.b_mn;
  a.idesc = make_idesc_f16(128, plan.nt, c.b_mn, 0) | type_bits(std::is_same_v<T, __nv_bfloat16>);
  a.act = c.act;
  a.keep_kind = c.keep_kind;
  a.bias = c.bias;
  a.bias32 = c.bias32;
  a.q_pitch = c.q_pitch;
  a.scale_pitch = c.scale_pitch;
  a.status = device_status_word(dev);
  if (!a.status) return MLPK_ERR_CUDA;
  for (int i = 0; i < 2; ++i) {
    a.in[i] = c.in[i];
    a.out[i] = c.out[i];
    a.keep[i] = c.keep[i];
    a.q[i] = c.q[i];
    a.scale[i] = c.scale[i];
    const uint64_t k = i == 1 && c.k[1] > 0 ? c.k[1] : c.k[0];
    if (c.a[i] && (rc = make_map_2d(&a.x[i], c.a[i], k, c.rows, kBlockK, plan.nt))) return rc;
    if (c.b[i] && (rc = c.b_mn ? make_map_2d(&a.w[i], c.b[i], c.cols, k, 64, kBlockK)
                               : make_map_2d(&a.w[i], c.b[i], k, c.cols, kBlockK, GATED ? 64 : 128)))
      return rc;
  }
  const auto kern = few_rows_kernel<T, EPI>;
  const int smem = few_smem(plan.nt, plan.stages);
  const void* entry = reinterpret_cast<const void*>(kern);
  if (!blocks_per_sm(entry, kFewThreads, smem, dev)) return MLPK_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(plan.tiles * plan.ranks, plan.row_tiles);
  cfg.blockDim = dim3(kFewThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = plan.ranks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, a));
}

// Whether a product goes to few_rows_kernel: up to 64 rows, and up to 2048 where its
// plan says that it ends earlier (a linear layer with a residual, bf16, us, there and
// in tiles of 256 rows: 128 x 4096 x 14336 31.3 and 33.1, 136 x 4096 x 8192 16.3 and
// 20.4, 320 x 8192 x 2048 16.1 and 23.0, 1024 x 8192 x 1024 22.4 and 25.3, 2000 x 4096
// x 512 17.5 and 19.7; 128 x 256 x 256 8.6 and 6.8, 256 x 4096 x 14336 49.3 and 34.2,
// 512 x 8192 x 1024 21.3 and 17.9; other epilogues were not measured for it, and
// neither estimate knows of them).  The rows must be read along the reduction, and a
// gate's checkpoint group is wider than a tile.
inline bool few_rows(const Product& c, int sm_count) {
  if (c.rows > 2048 || c.a_mn || c.outputs > 1 || (c.epi == kEpiGated && c.keep_kind == kKeep8)) return false;
  return c.rows <= 64 || few_plan_of(c, sm_count).us <= plan_of(c, sm_count / 2).us + 0.5;
}

template <class T, int EPI>
int launch_epi(const Product& c, cudaStream_t st) {
  DevInfo di;
  int dev = 0;
  const int rc = current_device_info(&di, &dev);
  if (rc) return rc;
  if (few_rows(c, di.sm_count)) return launch_few<T, EPI>(c, di, dev, st);
  const ProductPlan plan = plan_of(c, di.sm_count / 2);
  const int64_t bytes = plan.partials() * static_cast<int64_t>(sizeof(float));
  if (bytes && !c.workspace) return MLPK_ERR_NULL;
  if (c.workspace_bytes < bytes) return MLPK_ERR_SCRATCH;
  return plan.cols == 128 ? launch_tiles<T, EPI, 128>(c, plan, di, dev, st) : launch_tiles<T, EPI, 256>(c, plan, di, dev, st);
}

template <class T>
int launch_type(const Product& c, cudaStream_t st) {
  switch (c.epi) {
    case kEpiPlain: return launch_epi<T, kEpiPlain>(c, st);
    case kEpiLinear: return launch_epi<T, kEpiLinear>(c, st);
    case kEpiGated: return launch_epi<T, kEpiGated>(c, st);
    default: return launch_epi<T, kEpiGatedBwd>(c, st);
  }
}

}  // namespace product
}  // namespace mlpk
