// Kernel arguments and launch helpers of the expert selection (mx_select.hip). Host-visible; no torch types.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mx {

constexpr int kSelectLanes = 64;   // lanes of a token: groups at most
constexpr int kSelectMaxPer = 64;  // experts of a lane at most

struct SelectArgs {
  long long* topk_idx;
  float* topk_w;
  const void* logits;  // [N, E] of the launch's dtype
  const float* bias;   // [E] or null
  int N, E, top_k;
  bool softmax, top2;
  int num_groups, topk_groups;
  float scale;
  bool renormalize;
  // set by launch_select: lanes of a group (a power of two), experts of a lane, of a group; every lane of a group has
  // as many experts as the kernel holds
  int run, run_log, per, group_size;
  bool full;
  long long token0;  // first token of a launch
};
struct SelectBwdArgs {
  void* grad_logits;  // [N, E], fully written
  const long long* topk_idx;
  const float* grad_w;
  const void* logits;
  int N, E, top_k;
  bool softmax;
  float scale;
  bool renormalize;
  long long token0;  // set by launch_select_bwd: first token of a launch
};

// Experts that a lane holds for these sizes (more than kSelectMaxPer: they do not fit).
int select_per_lane(int E, int num_groups);
// dtype MXFP4_F32, _BF16 or _F16.
hipError_t launch_select(SelectArgs a, int dtype, hipStream_t s);
hipError_t launch_select_bwd(const SelectBwdArgs& a, int dtype, hipStream_t s);

}  // namespace mx
