// Kernel argument blocks and launch helpers of the dense operators (mx_dense.hip: the gated
// feed-forward block's products; mx_rows.hip: layer / RMS norm and counter-based dropout).
// Host-visible; no torch types.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mx {

// What a dense product does with its fp32 sums.
enum DenseEpi : int {
  kDenseStore = 0,  // out[m, n] = sum
  kDenseGlu = 1,    // g, u = sums of the two weight matrices + the deltas; h = GLU(g, u); g | u kept if asked for
  kDenseDGlu = 2,   // sum = dL/dh (+ grad_h); dg | du from it and the kept g | u
};

// One product out[M, N] = A . B over one or two segments of K terms each, 16-bit elements, fp32
// sums. An operand is "K-major" when the K terms of one row (of A) or column (of the result, for B)
// are contiguous, or "row-major" when the rows / columns of one K term are.
struct DenseArgs {
  const void* a[2];  // per segment
  const void* b[2];  // per segment; kDenseGlu: the gate and the up matrix instead (one segment)
  long long lda, ldb;
  int M, N, K;  // kDenseGlu: N = columns of h
  int nseg;
  void* out;        // [M, N], rows ldo apart; rows >= split_m go to out2 (row m - split_m)
  void* out2;
  int split_m;
  long long ldo;
  const void* add0;  // kDenseGlu: gate delta [M, N] or null; kDenseDGlu: grad_h [M, N] or null
  const void* add1;  // kDenseGlu: up delta or null
  float* gu;         // [M, 2N] fp32 gate | up: kDenseGlu writes it (null: not kept), kDenseDGlu reads it
  int act;
  // set by the launcher: the tile grid, and the cut of K into `splits` runs of `run` steps, whose sums go to
  // partial [splits][M][N] (kDenseGlu: [splits][M][2N], gate | up) and meet in a second kernel (null: one run)
  int tiles_m, tiles_n;
  int splits, run;
  float* partial;
};

// The three shapes of product the block needs: A and B K-major (forward products), A K-major and B
// row-major (gradients of activations), both row-major (weight gradients).
enum DenseShape : int { kDenseForward = 0, kDenseDgrad = 1, kDenseWgrad = 2 };

// Bytes of partial sums that launch_dense may use for a product of these sizes, and the product
// (dtype MXFP4_BF16 or MXFP4_F16; partial: that many bytes).
size_t dense_partial_bytes(DenseShape shape, DenseEpi epi, int M, int N, int K, int nseg);
// What launch_dense chooses for a product: rows, tile and runs of K of its first part and of its second (0 rows:
// one part). tile: 0 .. 3 from the largest to the smallest, -1 and -2 the few-row kernel (mx_dense.hip).
void dense_choice(DenseShape shape, DenseEpi epi, int M, int N, int K, int nseg, int* choice);
hipError_t launch_dense(DenseShape shape, DenseEpi epi, const DenseArgs& a, int dtype, float* partial, hipStream_t s);

// Layer / RMS norm over rows of D elements (dtype MXFP4_F32, _BF16 or _F16), fp32 statistics
// stats[0:M] = 1 / sqrt(var + eps), stats[M:2M] = mean (layer norm). weight and bias fp32 or null.
hipError_t launch_norm_forward(void* y, float* stats, const void* x, const float* weight, const float* bias, int M,
                               int D, float eps, int layer, int dtype, hipStream_t s);
size_t norm_backward_workspace(int M, int D);
hipError_t launch_norm_backward(void* dx, float* dweight, float* dbias, const void* dy, const void* x,
                                const float* weight, const float* stats, int M, int D, int layer, int dtype,
                                float* partial, hipStream_t s);

// y[i] = keep(i) ? x[i] * scale : 0 for n elements; word(i) < threshold drops. The seed comes from
// seed_dev[0] when that is not null.
hipError_t launch_dropout(void* y, const void* x, long long n, uint64_t threshold, float scale, uint64_t seed,
                          const uint64_t* seed_dev, uint64_t stream_id, int dtype, hipStream_t s);

}  // namespace mx
