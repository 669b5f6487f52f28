// Kernel arguments and launch helpers of the products with group-scaled 4-bit weights (mx_int4.hip).
// Host-visible; no torch types.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mx {

// One matrix [R, K], or E of them stacked: codes [R, K / 2] (low nibble = even element), scales [R, K / group]
// of the activations' type, zero points [R, K / group] bytes or null (8 everywhere).
struct Int4Matrix {
  const uint8_t* q;
  const void* s;
  const uint8_t* z;
};

// The (token, slot) pairs of a routed call; pair p is slot p % k of token p / k.
struct Int4Pairs {
  const void* idx;  // [P] expert ids of 32 or 64 bits; outside [0, E): the pair has no expert
  int idx64;
  int P, k, E;
};

struct Int4Args {
  Int4Matrix w[2];  // the second of a gate/up product
  const void* x;    // rows of K elements
  void* y;
  int M, K, R;
  // routed: x row of pair p is p / x_div, y row p
  Int4Pairs pairs;
  int x_div;
  const int4* tiles;   // {expert, first, rows, 0} into order, n_tiles of them; null: found from the ids (P <= 64)
  const int* n_tiles;
  const int* order;
  const float* row_w;  // launch_int4_token: the pairs' weights
  bool by_token;       // launch_int4_glu: each pair by itself
  int act;
  // set by the launcher: work-groups over the weight rows, the first row tile (pair, token) of this launch; of the
  // few-row form the batches of weight rows of a work-group and the waves that share a row of K
  int row_groups, tile0, batches, team;
};

// y [M, R] = x [M, K] W^T (dtype MXFP4_BF16 or _F16).
hipError_t launch_int4_gemm(const Int4Args& a, int group, int dtype, hipStream_t s);

// Rows of a routed tile for P pairs over E experts, and how many tiles there can be.
int int4_tile_rows(int P, int E);
inline int int4_max_tiles(int P, int E) { return P / int4_tile_rows(P, E) + (P < E ? P : E); }
constexpr int kInt4ScanPairs = 64;  // up to so many pairs the products find their rows themselves
hipError_t launch_int4_route(const Int4Pairs& p, int4* tiles, int* n_tiles, int* order, hipStream_t s);
// Whether a call of N tokens runs without routing, each pair by itself: launch_int4_glu with by_token, then
// launch_int4_token.
bool int4_by_token(int N, int k, int E, int D, int F);
// h [P, R] = GLU(x W1^T, x W3^T) of each pair's expert.
hipError_t launch_int4_glu(const Int4Args& a, int group, int dtype, hipStream_t s);
// y [P, R] fp32 = x W^T of each pair's expert.
hipError_t launch_int4_pairs(const Int4Args& a, int group, int dtype, hipStream_t s);
// y [N, R] of dtype = sum over each token's slots of row_w (x W^T), x's rows those of the pairs.
hipError_t launch_int4_token(const Int4Args& a, int group, int dtype, hipStream_t s);
// out [N, D] = sum over slots, in slot order, of topk_w y of the pairs that have an expert.
hipError_t launch_int4_combine(void* out, const float* y, const float* topk_w, const Int4Pairs& p, int D, int dtype,
                               hipStream_t s);

}  // namespace mx
