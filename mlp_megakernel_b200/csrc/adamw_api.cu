// C-ABI entry point of the AdamW step (declared in include/mlpk.h).
#include <algorithm>
#include <cmath>

#include "adamw_kernel.cuh"
#include "host.cuh"

namespace {

using namespace mlpk;
using namespace mlpk::host;

// Tensors of one launch: the table travels in the kernel's parameters (32,764
// bytes at most), so nothing is copied to the device and a CUDA graph keeps
// its own.  Few tensors take the short form of it.
constexpr int kFewTensors = 32;
constexpr int kManyTensors = 768;

int64_t chunks_of(int64_t n) { return (n + kAdamChunk - 1) / kAdamChunk; }

template <class P, class G, bool BITS8, bool MASTER, int CAP>
int launch_step(int count, const int64_t* numel, void* const* p, const void* const* g, const int64_t* off,
                const int32_t* tick, AdamArgs a, cudaStream_t st) {
  DevInfo di;
  int dev;
  int rc = current_device_info(&di, &dev);
  if (rc) return rc;
  void (*kern)(AdamTable<CAP>, AdamArgs);
  size_t smem = 0;
  if constexpr (BITS8) {
    kern = adamw8_kernel<P, G, MASTER, CAP>;
    smem = AdamSlots<P, G, MASTER>::BYTES;
    if (blocks_per_sm(reinterpret_cast<const void*>(kern), kAdamThreads, smem, dev) == 0) return MLPK_ERR_CUDA;
    // 1 chunk a thread block until the step has 12 of them an SM (four waves),
    // then more, up to 16.
    int64_t all = 0;
    for (int i = 0; i < count; ++i) all += chunks_of(numel[i]);
    a.per = static_cast<int>(std::min<int64_t>(std::max<int64_t>(all / (di.sm_count * 12), 1), 16));
  } else {
    kern = adamw32_kernel<P, G, MASTER, CAP>;
    a.per = kAdamChunks32;
  }
  for (int i = 0; i < count;) {
    AdamTable<CAP> table;
    int64_t ctas = 0;
    int k = 0;
    for (; i < count && k < CAP; ++i) {
      if (numel[i] == 0) continue;
      const int64_t n = (chunks_of(numel[i]) + a.per - 1) / a.per;
      if (ctas + n > 0x7fffffff) break;
      table.t[k++] = {p[i], g[i], numel[i], off[i], static_cast<int32_t>(ctas), tick[i]};
      ctas += n;
    }
    if (k == 0) {
      if (i < count) return MLPK_ERR_SHAPE;  // a tensor of 2^43 elements
      break;
    }
    a.count = k;
    rc = launch_kernel_early(kern, dim3(static_cast<unsigned>(ctas)), kAdamThreads, smem, st, table, a);
    if (rc) return rc;
  }
  return MLPK_OK;
}

template <class P, class G, bool BITS8, bool MASTER>
int step(int count, const int64_t* numel, void* const* p, const void* const* g, const int64_t* off, const int32_t* tick,
         const AdamArgs& a, cudaStream_t st) {
  return count <= kFewTensors
             ? launch_step<P, G, BITS8, MASTER, kFewTensors>(count, numel, p, g, off, tick, a, st)
             : launch_step<P, G, BITS8, MASTER, kManyTensors>(count, numel, p, g, off, tick, a, st);
}
template <class P, class G>
int step_of(int bits, bool master, int count, const int64_t* numel, void* const* p, const void* const* g,
            const int64_t* off, const int32_t* tick, const AdamArgs& a, cudaStream_t st) {
  if constexpr (sizeof(P) == 2) {
    if (master)
      return bits == 8 ? step<P, G, true, true>(count, numel, p, g, off, tick, a, st)
                       : step<P, G, false, true>(count, numel, p, g, off, tick, a, st);
  }
  return bits == 8 ? step<P, G, true, false>(count, numel, p, g, off, tick, a, st)
                   : step<P, G, false, false>(count, numel, p, g, off, tick, a, st);
}

}  // namespace

extern "C" {

int mlpk_adamw_step(int count, const int64_t* numel, void* const* params, const void* const* grads,
                    const int64_t* state_off, const int32_t* tick, int p_dtype, int g_dtype,
                    const mlpk_adamw_state* state, const mlpk_adamw_args* args, mlpk_stream_t stream) {
  if (count < 0) return MLPK_ERR_SHAPE;
  if (!state || !args) return MLPK_ERR_NULL;
  if (state->bits != 8 && state->bits != 32) return MLPK_ERR_UNSUPPORTED;
  if (g_dtype != p_dtype && g_dtype != MLPK_DT_F32) return MLPK_ERR_UNSUPPORTED;
  if (state->master && p_dtype == MLPK_DT_F32) return MLPK_ERR_UNSUPPORTED;
  if (count == 0) return MLPK_OK;
  if (!numel || !params || !grads || !state_off || !tick || !state->exp_avg || !state->exp_avg_sq || !state->ticks)
    return MLPK_ERR_NULL;
  if (state->bits == 8 && (!state->exp_avg_scale || !state->exp_avg_sq_scale)) return MLPK_ERR_NULL;
  for (const void* p : {state->exp_avg, state->exp_avg_sq, static_cast<void*>(state->master)})
    if (reinterpret_cast<uintptr_t>(p) & 31u) return MLPK_ERR_ALIGN;
  for (int i = 0; i < count; ++i) {
    if (numel[i] < 0 || state_off[i] < 0 || tick[i] < 0) return MLPK_ERR_SHAPE;
    if (state_off[i] % kAdamBlock) return MLPK_ERR_ALIGN;
    if (numel[i] > 0 && (!params[i] || !grads[i])) return MLPK_ERR_NULL;
  }
  AdamArgs a = {};
  a.lr = static_cast<float>(args->lr);
  const auto twice = [](double v) { return make_float2(static_cast<float>(v), static_cast<float>(v)); };
  a.b1 = twice(args->beta1);
  a.b1c = twice(1.0 - args->beta1);
  a.b2 = twice(args->beta2);
  a.b2c = twice(1.0 - args->beta2);
  a.eps = twice(args->eps);
  a.lnb1 = static_cast<float>(std::log(args->beta1));
  a.lnb2 = static_cast<float>(std::log(args->beta2));
  a.wd = static_cast<float>(args->weight_decay);
  a.maximize = args->maximize;
  a.lr_ptr = args->lr_ptr;
  a.grad_scale = args->grad_scale;
  a.found_inf = args->found_inf;
  a.m = state->exp_avg;
  a.v = state->exp_avg_sq;
  a.m_scale = state->exp_avg_scale;
  a.v_scale = state->exp_avg_sq_scale;
  a.master = state->master;
  a.ticks = reinterpret_cast<unsigned long long*>(state->ticks);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool master = state->master != nullptr, same = g_dtype == p_dtype;
  switch (p_dtype) {
    case MLPK_DT_F32:
      return step_of<float, float>(state->bits, false, count, numel, params, grads, state_off, tick, a, st);
    case MLPK_DT_F16:
      return same ? step_of<__half, __half>(state->bits, master, count, numel, params, grads, state_off, tick, a, st)
                  : step_of<__half, float>(state->bits, master, count, numel, params, grads, state_off, tick, a, st);
    case MLPK_DT_BF16:
      return same ? step_of<__nv_bfloat16, __nv_bfloat16>(state->bits, master, count, numel, params, grads, state_off,
                                                          tick, a, st)
                  : step_of<__nv_bfloat16, float>(state->bits, master, count, numel, params, grads, state_off, tick, a,
                                                  st);
    default: return MLPK_ERR_UNSUPPORTED;
  }
}

}  // extern "C"
