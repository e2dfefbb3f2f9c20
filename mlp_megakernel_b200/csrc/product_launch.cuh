// Launches of the products (product_kernel.cuh), by operand type: one
// translation unit for fp16 (product_f16.cu), one for bf16 (product_bf16.cu).
#pragma once
#include "host.cuh"

namespace mlpk {
namespace product {

// One product: D[rows][cols] = sum over the ranges of A B, with an epilogue.
// An operand's matrix is stored with the reduction contiguous ([rows][k] for A,
// [cols][k] for B), or (mn) with the row / column contiguous ([k][rows], [k][cols]).
struct Product {
  int epi = 0, act = 0, keep_kind = 0;
  int64_t rows = 0;
  int cols = 0;
  int outputs = 1;           // 2: b[1] (or, with out_a, a[1]) gives the second
  bool out_a = false;
  int64_t k[2] = {0, 0};     // k[1] > 0: a second range, a[1] b[1]
  const void* a[2] = {nullptr, nullptr};
  const void* b[2] = {nullptr, nullptr};
  bool a_mn = false, b_mn = false;
  const void* in[2] = {nullptr, nullptr};
  void* out[2] = {nullptr, nullptr};
  void* keep[2] = {nullptr, nullptr};
  const void* bias = nullptr;
  bool bias32 = false;
  uint8_t* q[2] = {nullptr, nullptr};
  float* scale[2] = {nullptr, nullptr};
  int64_t q_pitch = 0;
  int scale_pitch = 0;
  void* workspace = nullptr;  // of the shares
  int64_t workspace_bytes = 0;
};

// The workspace that a product needs: from its epi, keep_kind, rows, cols, outputs, k, a_mn.
__attribute__((visibility("hidden"))) int64_t workspace_bytes(const Product& p, int sm_count);

__attribute__((visibility("hidden"))) int launch_f16(const Product& p, cudaStream_t st);
__attribute__((visibility("hidden"))) int launch_bf16(const Product& p, cudaStream_t st);

}  // namespace product
}  // namespace mlpk
