// C-ABI entry points of the rows sorted by expert and back (declared in
// include/mlpk.h).
#include <algorithm>

#include "expert_kernel.cuh"
#include "host.cuh"

namespace {

using namespace mlpk;
using namespace mlpk::host;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int kMaxChunks = 148;

// Slots of a chunk (a multiple of 32 a warp) and the number of chunks.
void sort_chunks(int64_t slots, int64_t* chunk, int* chunks) {
  const int64_t unit = 32 * kSortWarps;
  *chunk = std::max<int64_t>(ceil_div(ceil_div(slots, kMaxChunks), unit), 1) * unit;
  *chunks = static_cast<int>(std::max<int64_t>(ceil_div(slots, *chunk), 1));
}

int check_rows(int64_t tokens, int top, int width, int dtype) {
  if (tokens < 0 || top < 1 || width < 1 || tokens > 0x7fffffff / top) return MLPK_ERR_SHAPE;
  if (dtype != MLPK_DT_F16 && dtype != MLPK_DT_BF16 && dtype != MLPK_DT_F32) return MLPK_ERR_UNSUPPORTED;
  return MLPK_OK;
}

template <class I>
int sort_slots(int64_t slots, int experts, const void* ids, int* row_of, int* offsets, int* hist, cudaStream_t st) {
  int64_t chunk;
  int chunks;
  sort_chunks(slots, &chunk, &chunks);
  const size_t bins = experts + 1;
  int rc = launch_kernel_early(expert_count_kernel<I>, dim3(chunks), kSortThreads, bins * 4, st,
                               static_cast<const I*>(ids), slots, experts, chunk, hist);
  if (rc) return rc;
  return launch_kernel_early(expert_place_kernel<I>, dim3(chunks), kSortThreads, bins * 4 * (kSortWarps + 2), st,
                             static_cast<const I*>(ids), slots, experts, chunk, static_cast<const int*>(hist), row_of,
                             offsets);
}

// Blocks for `items` pieces of work of one thread each: at most 16 blocks of
// 256 an SM, which loop.
unsigned blocks_for(int64_t items, int sm_count) {
  return static_cast<unsigned>(std::min<int64_t>(ceil_div(items, 256), static_cast<int64_t>(sm_count) * 16));
}

template <class U>
int dispatch_words(int64_t tokens, int top, int64_t words, const void* x, const int* row_of, const int* kept, void* xs,
                   int sm_count, cudaStream_t st) {
  return launch_kernel_early(expert_dispatch_kernel<U>, dim3(blocks_for(tokens * words, sm_count)), 256, 0, st,
                             static_cast<const U*>(x), tokens, top, static_cast<int>(words), row_of, kept,
                             static_cast<U*>(xs));
}

// f(T, W, VEC)
template <class T, class W, class F>
int with_vec(int width, F&& f) {
  if (width % kVecOf<T> == 0) return f(T{}, W{}, std::integral_constant<int, kVecOf<T>>{});
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

}  // namespace

extern "C" {

int64_t mlpk_expert_sort_workspace_size(int64_t slots, int experts) {
  if (slots < 0 || slots > 0x7fffffff || experts < 1) return -1;
  if (experts > kExpertMax) return -1;
  int64_t chunk;
  int chunks;
  sort_chunks(slots, &chunk, &chunks);
  return static_cast<int64_t>(chunks) * (experts + 1) * 4;
}

int mlpk_expert_sort(int64_t slots, int experts, const void* ids, int id_bytes, int32_t* row_of, int32_t* offsets,
                     void* workspace, int64_t workspace_bytes, mlpk_stream_t stream) {
  if (slots < 0 || slots > 0x7fffffff || experts < 1) return MLPK_ERR_SHAPE;
  if (experts > kExpertMax || (id_bytes != 4 && id_bytes != 8)) return MLPK_ERR_UNSUPPORTED;
  if (!offsets || !workspace || (slots > 0 && (!ids || !row_of))) return MLPK_ERR_NULL;
  if (!aligned16(ids) || !aligned16(row_of) || !aligned16(offsets) || !aligned16(workspace)) return MLPK_ERR_ALIGN;
  if (workspace_bytes < mlpk_expert_sort_workspace_size(slots, experts)) return MLPK_ERR_SCRATCH;
  DevInfo di;
  int rc = current_device_info(&di, nullptr);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int* hist = static_cast<int*>(workspace);
  return id_bytes == 8 ? sort_slots<int64_t>(slots, experts, ids, row_of, offsets, hist, st)
                       : sort_slots<int32_t>(slots, experts, ids, row_of, offsets, hist, st);
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
    return dispatch_words<uint4>(tokens, top, bytes / 16, x, row_of, kept, xs, di.sm_count, st);
  if (bytes % 8 == 0) return dispatch_words<uint2>(tokens, top, bytes / 8, x, row_of, kept, xs, di.sm_count, st);
  if (bytes % 4 == 0) return dispatch_words<uint32_t>(tokens, top, bytes / 4, x, row_of, kept, xs, di.sm_count, st);
  return dispatch_words<uint16_t>(tokens, top, bytes / 2, x, row_of, kept, xs, di.sm_count, st);
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
    constexpr int V = decltype(vec)::value;
    return launch_kernel_early(expert_combine_kernel<T, W, V>, dim3(blocks_for(tokens * (width / V), di.sm_count)), 256,
                               0, static_cast<cudaStream_t>(stream), static_cast<const T*>(y),
                               static_cast<const W*>(weights), tokens, top, width, row_of, kept, static_cast<T*>(out));
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
    return launch_kernel_early(expert_combine_bwd_kernel<T, W, decltype(vec)::value>,
                               dim3(blocks_for(tokens * top * 32, di.sm_count)), 256, 0,
                               static_cast<cudaStream_t>(stream), static_cast<const T*>(grad_out),
                               static_cast<const T*>(y), static_cast<const W*>(weights), tokens, top, width, row_of,
                               kept, static_cast<T*>(dy), static_cast<W*>(dw));
  });
}

}  // extern "C"
