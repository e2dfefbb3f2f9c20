// C-ABI entry points of the rows sorted by expert and back (declared in
// include/mlpk.h).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "expert_kernel.cuh"
#include "expert_plan.cuh"
#include "host.cuh"

namespace {

using namespace mlpk;
using namespace mlpk::host;

int check_rows(int64_t tokens, int top, int width, int dtype) {
  if (tokens < 0 || top < 1 || width < 1 || tokens > 0x7fffffff / top) return MLPK_ERR_SHAPE;
  if ((dtype != MLPK_DT_F16 && dtype != MLPK_DT_BF16 && dtype != MLPK_DT_F32) || width > kRowWidthMax)
    return MLPK_ERR_UNSUPPORTED;
  return MLPK_OK;
}

template <class I>
int sort_slots(int64_t slots, int experts, const void* ids_, int* row_of, int* offsets, int* hist, int dev,
               const SortPlan& p, cudaStream_t st) {
  const I* ids = static_cast<const I*>(ids_);
  const size_t smem = sizeof(int) * (kSortWarps + static_cast<size_t>(kSortWarps + 1) * (experts + 1));
  if (!p.cluster) {
    const auto rank = p.part <= 32 * kSortGroups ? expert_rank_kernel<I, true> : expert_rank_kernel<I, false>;
    if (blocks_per_sm(reinterpret_cast<const void*>(rank), kSortThreads, smem, dev) == 0) return MLPK_ERR_CUDA;
    const int rc =
        launch_kernel_early(rank, dim3(p.blocks), kSortThreads, smem, st, ids, slots, experts, p.part, row_of, hist);
    if (rc) return rc;
    return launch_kernel_early(expert_place_kernel<I>, dim3(p.blocks), kSortThreads,
                               sizeof(int) * (2 * kSortThreads + experts + 1), st, ids, slots, experts, p.part, row_of,
                               offsets, static_cast<const int*>(hist));
  }
  const auto kern = expert_sort_kernel<I>;
  if (blocks_per_sm(reinterpret_cast<const void*>(kern), kSortThreads, smem, dev) == 0) return MLPK_ERR_CUDA;
  if (p.blocks > 8) {  // more than a cluster has unasked
    static std::atomic<bool> asked[64];  // by device; asking twice does no harm
    if (dev >= 64 || !asked[dev].load(std::memory_order_relaxed)) {
      const int rc = cuda_status(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
      if (rc) return rc;
      if (dev < 64) asked[dev].store(true, std::memory_order_relaxed);
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.blocks);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.blocks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, ids, slots, experts, p.part, row_of, offsets));
}

// Threads of a token's row of `items` words or vectors, `each` a thread, and the
// blocks for the tokens, `tokens_each` a thread.
struct RowGrid {
  dim3 grid, block;
};
RowGrid row_grid(int64_t tokens, int tokens_each, int64_t items, int each, bool parts) {
  RowGrid g;
  // Parts of a row of equal size, each at most what 256 threads take.
  const int64_t n = parts ? ceil_div(items, static_cast<int64_t>(kRowThreads) * each) : 1;
  const int64_t want = std::min<int64_t>(ceil_div(ceil_div(items, n), each), kRowThreads);
  int tpr = 1;
  while (tpr < want && tpr < 32) tpr *= 2;
  if (want > 32) tpr = static_cast<int>(ceil_div(want, 32)) * 32;
  const int subs = kRowThreads / tpr;
  g.block = dim3(tpr, subs);
  g.grid = dim3(static_cast<unsigned>(ceil_div(tokens, static_cast<int64_t>(subs) * tokens_each)),
                static_cast<unsigned>(n));
  return g;
}

template <class U>
int dispatch_words(int64_t tokens, int top, int64_t words, const void* x, const int* row_of, const int* kept, void* xs,
                   cudaStream_t st) {
  constexpr int NW = sizeof(U) == 16 ? 1 : sizeof(U) == 8 ? 2 : 4, NT = 2;
  const RowGrid g = row_grid(tokens, NT, words, NW, true);
  return launch_kernel_early(expert_dispatch_kernel<U, NT, NW>, g.grid, g.block, 0, st, static_cast<const U*>(x),
                             tokens, top, static_cast<int>(words), row_of, kept, static_cast<U*>(xs));
}

// f(T, W, VEC): 16-byte vectors where the width allows them, else pairs of
// 16-bit values, else single ones.
template <class T, class W, class F>
int with_vec(int width, F&& f) {
  if (width % kVecOf<T> == 0) return f(T{}, W{}, std::integral_constant<int, kVecOf<T>>{});
  if constexpr (sizeof(T) == 2) {
    if (width % 2 == 0) return f(T{}, W{}, std::integral_constant<int, 2>{});
  }
  return f(T{}, W{}, std::integral_constant<int, 1>{});
}
template <class F>
int with_types(int dtype, int w_dtype, int width, F&& f) {
  if (dtype == MLPK_DT_F32) return with_vec<float, float>(width, f);
  if (dtype == MLPK_DT_F16)
    return w_dtype == MLPK_DT_F32 ? with_vec<__half, float>(width, f) : with_vec<__half, __half>(width, f);
  return w_dtype == MLPK_DT_F32 ? with_vec<__nv_bfloat16, float>(width, f)
                                : with_vec<__nv_bfloat16, __nv_bfloat16>(width, f);
}
// f(GROUP): choices of a token that are under way together.
template <class F>
int with_group(int top, F&& f) {
  if (top <= 2) return f(std::integral_constant<int, 2>{});
  return f(std::integral_constant<int, 4>{});
}

}  // namespace

extern "C" {

int64_t mlpk_expert_sort_workspace_size(int64_t slots, int experts) {
  if (slots < 0 || slots > 0x7fffffff || experts < 1 || experts > kExpertMax) return -1;
  if (sort_plan(slots, 1).cluster) return 0;  // on every device
  DevInfo di;
  if (current_device_info(&di, nullptr)) return -1;
  return sort_plan(slots, di.sm_count).workspace(experts);
}

int mlpk_expert_sort(int64_t slots, int experts, const void* ids, int id_bytes, int32_t* row_of, int32_t* offsets,
                     void* workspace, int64_t workspace_bytes, mlpk_stream_t stream) {
  if (slots < 0 || slots > 0x7fffffff || experts < 1) return MLPK_ERR_SHAPE;
  if (experts > kExpertMax || (id_bytes != 4 && id_bytes != 8)) return MLPK_ERR_UNSUPPORTED;
  if (!offsets || (slots > 0 && (!ids || !row_of))) return MLPK_ERR_NULL;
  if (!aligned16(ids) || !aligned16(row_of) || !aligned16(offsets) || !aligned16(workspace)) return MLPK_ERR_ALIGN;
  DevInfo di;
  int dev;
  int rc = current_device_info(&di, &dev);
  if (rc) return rc;
  const SortPlan p = sort_plan(slots, di.sm_count);
  if (!p.cluster) {
    if (!workspace) return MLPK_ERR_NULL;
    if (workspace_bytes < p.workspace(experts)) return MLPK_ERR_SCRATCH;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int* hist = static_cast<int*>(workspace);
  return id_bytes == 8 ? sort_slots<int64_t>(slots, experts, ids, row_of, offsets, hist, dev, p, st)
                       : sort_slots<int32_t>(slots, experts, ids, row_of, offsets, hist, dev, p, st);
}

int mlpk_expert_dispatch(int64_t tokens, int top, int width, int dtype, const void* x, const int32_t* row_of,
                         const int32_t* kept, void* xs, mlpk_stream_t stream) {
  int rc = check_rows(tokens, top, width, dtype);
  if (rc) return rc;
  if (tokens == 0) return MLPK_OK;
  if (!x || !row_of || !kept || !xs) return MLPK_ERR_NULL;
  if (!aligned16(x) || !aligned16(xs)) return MLPK_ERR_ALIGN;
  DevInfo di;
  if ((rc = current_device_info(&di, nullptr)) != MLPK_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t bytes = static_cast<int64_t>(width) * (dtype == MLPK_DT_F32 ? 4 : 2);
  if (bytes % 16 == 0)
    return dispatch_words<uint4>(tokens, top, bytes / 16, x, row_of, kept, xs, st);
  if (bytes % 8 == 0) return dispatch_words<uint2>(tokens, top, bytes / 8, x, row_of, kept, xs, st);
  if (bytes % 4 == 0) return dispatch_words<uint32_t>(tokens, top, bytes / 4, x, row_of, kept, xs, st);
  return dispatch_words<uint16_t>(tokens, top, bytes / 2, x, row_of, kept, xs, st);
}

int mlpk_expert_combine(int64_t tokens, int top, int width, int dtype, const void* y, const void* weights, int w_dtype,
                        const int32_t* row_of, const int32_t* kept, void* out, mlpk_stream_t stream) {
  int rc = check_rows(tokens, top, width, dtype);
  if (rc) return rc;
  if (weights && w_dtype != dtype && w_dtype != MLPK_DT_F32) return MLPK_ERR_UNSUPPORTED;
  if (tokens == 0) return MLPK_OK;
  if (!y || !row_of || !kept || !out) return MLPK_ERR_NULL;
  if (!aligned16(y) || !aligned16(out)) return MLPK_ERR_ALIGN;
  DevInfo di;
  if ((rc = current_device_info(&di, nullptr)) != MLPK_OK) return rc;
  return with_types(dtype, weights ? w_dtype : dtype, width, [&](auto t, auto w, auto vec) {
    using T = decltype(t);
    using W = decltype(w);
    constexpr int V = decltype(vec)::value, NW = V == kVecOf<T> ? 1 : 4;
    return with_group(top, [&](auto group) {
      constexpr int GROUP = decltype(group)::value;
      const RowGrid g = row_grid(tokens, 1, width / V, NW, true);
      return launch_kernel_early(expert_combine_kernel<T, W, V, NW, GROUP>, g.grid, g.block, 0,
                                 static_cast<cudaStream_t>(stream), static_cast<const T*>(y),
                                 static_cast<const W*>(weights), tokens, top, width, row_of, kept,
                                 static_cast<T*>(out));
    });
  });
}

int mlpk_expert_combine_bwd(int64_t tokens, int top, int width, int dtype, const void* grad_out, const void* y,
                            const void* weights, int w_dtype, const int32_t* row_of, const int32_t* kept, void* dy,
                            void* dw, mlpk_stream_t stream) {
  int rc = check_rows(tokens, top, width, dtype);
  if (rc) return rc;
  if ((weights || dw) && w_dtype != dtype && w_dtype != MLPK_DT_F32) return MLPK_ERR_UNSUPPORTED;
  if (tokens == 0 || (!dy && !dw)) return MLPK_OK;
  if (!grad_out || !row_of || !kept || (dw && !y)) return MLPK_ERR_NULL;
  if (!aligned16(grad_out) || !aligned16(y) || !aligned16(dy)) return MLPK_ERR_ALIGN;
  DevInfo di;
  if ((rc = current_device_info(&di, nullptr)) != MLPK_OK) return rc;
  return with_types(dtype, weights || dw ? w_dtype : dtype, width, [&](auto t, auto w, auto vec) {
    using T = decltype(t);
    using W = decltype(w);
    constexpr int V = decltype(vec)::value;
    return with_group(top, [&](auto group) {
      constexpr int GROUP = decltype(group)::value;
      const RowGrid g = row_grid(tokens, 1, width / V, V == kVecOf<T> ? 2 : 8, false);
      return launch_kernel_early(expert_combine_bwd_kernel<T, W, V, GROUP>, g.grid, g.block, 0,
                                 static_cast<cudaStream_t>(stream), static_cast<const T*>(grad_out),
                                 static_cast<const T*>(y), static_cast<const W*>(weights), tokens, top, width,
                                 row_of, kept, static_cast<T*>(dy), static_cast<W*>(dw));
    });
  });
}

}  // extern "C"
