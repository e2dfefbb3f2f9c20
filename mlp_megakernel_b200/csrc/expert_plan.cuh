// How a sort by expert is launched (expert_kernel.cuh says what the kernels do).
// Host code; it needs no device.
#pragma once
#include <algorithm>
#include <cstdint>

namespace mlpk {

constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kExpertMax = 1024;
constexpr int kSortGroups = 4;       // groups of 32 slots of a warp that registers hold
constexpr int kSortBlockSlots = 4096;
constexpr int kSortCluster = 16;     // thread blocks of one cluster, at most

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Thread blocks of a sort and slots of a warp: one cluster of a power of two of
// blocks if kSortCluster of them take the slots, else two launches of at most one
// block an SM.  Which of the two follows from the slots alone, not from the
// device: the cluster's kernel takes 32 * kSortGroups slots a warp and no more.
struct SortPlan {
  bool cluster;
  int blocks;
  int64_t part;
  int64_t workspace(int experts) const {
    return cluster ? 0 : blocks * (experts + 1) * static_cast<int64_t>(sizeof(int));
  }
};
inline SortPlan sort_plan(int64_t slots, int sm_count) {
  SortPlan p;
  const int64_t want = ceil_div(slots, kSortBlockSlots);
  p.cluster = want <= kSortCluster;
  if (p.cluster) {
    p.blocks = 1;
    while (p.blocks < want) p.blocks *= 2;
  } else {
    p.blocks = static_cast<int>(std::min<int64_t>(want, sm_count));
  }
  p.part = std::max<int64_t>(ceil_div(ceil_div(slots, static_cast<int64_t>(p.blocks) * kSortWarps), 32), 1) * 32;
  return p;
}

}  // namespace mlpk
