// Row-wise operators of the dense half of the latent MoE block: layer and RMS norm with their
// backward pass (RMSNormFunction, lazy_lora/streaming/trunk_streamer.py:23-34, is the RMS form), and
// the adapters' dropout (LazyLoRALinear.forward_lora_only, lazy_lora/core/lora_layer.py:104-139) with
// a mask that is recomputed from a counter wherever it is needed and stored nowhere.
#include <algorithm>

#include "../../include/lazylora_mxfp4.h"
#include "mx_dense.h"
#include "mx_device.h"

// Every fused multiply-add here is written out: left to the compiler, two forms of a kernel could round
// differently, and a gradient would depend on which others were asked for.
#pragma clang fp contract(off)

namespace mx {

namespace {

// Eight consecutive elements at element offset i, as fp32; elements at or past n read as zero. Rows of
// odd lengths start at any element, so the 16- and 32-byte accesses are declared with the element's
// alignment only (the memory pipeline takes them; whole rows stay contiguous).
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Eight {
  typedef T Vec __attribute__((ext_vector_type(8)));
  Vec v;  // a vector: an array of 16-bit elements would take a register each
};
template <typename T>
MX_DEV void load8(const T* p, int i, int n, float (&f)[8])
{
  if (i + 8 <= n) {
    const Eight<T> e = *reinterpret_cast<const Eight<T>*>(p + i);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (float)e.v[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = i + j < n ? (float)p[i + j] : 0.f;
  }
}
template <typename T>
MX_DEV Eight<T> load_raw(const T* p, int i, int n)
{
  Eight<T> e;
  if (i + 8 <= n) {
    e = *reinterpret_cast<const Eight<T>*>(p + i);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) e.v[j] = i + j < n ? p[i + j] : (T)0.f;
  }
  return e;
}
template <typename T>
MX_DEV void store8(T* p, int i, int n, const float (&f)[8])
{
  if (i + 8 <= n) {
    Eight<T> e;
#pragma unroll
    for (int j = 0; j < 8; ++j) e.v[j] = (T)f[j];
    *reinterpret_cast<Eight<T>*>(p + i) = e;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < n) p[i + j] = (T)f[j];
  }
}

MX_DEV float wave_sum(float v)
{
  v = group16_sum(v);
  v += __shfl_xor(v, 16, 64);
  v += __shfl_xor(v, 32, 64);
  return v;
}

// Sums of NS values over the G lanes of a row's team (16 or a multiple of 64 lanes), in a fixed order; every
// lane gets them. buf: NS floats per wave of the work-group; teams of several waves meet at one barrier, so
// every thread of the work-group has to come here, and the caller alternates two bufs.
template <int G, int NS>
MX_DEV void team_sum(float (&s)[NS], float* buf)
{
  if constexpr (G == 16) {
#pragma unroll
    for (int i = 0; i < NS; ++i) s[i] = group16_sum(s[i]);
  } else {
#pragma unroll
    for (int i = 0; i < NS; ++i) s[i] = wave_sum(s[i]);
    if constexpr (G > 64) {
      constexpr int W = G / 64;
      const int wave = threadIdx.x >> 6, first = wave / W * W;
      if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int i = 0; i < NS; ++i) buf[wave * NS + i] = s[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NS; ++i) s[i] = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
#pragma unroll
        for (int i = 0; i < NS; ++i) s[i] += buf[(first + w) * NS + i];
      }
    }
  }
}

// HIP takes fewer than 2^32 threads per launch: work past 2^29 of them goes in launches of its own (milliseconds
// each). launch(first, count) makes one of `count` work-groups from number `first` on.
constexpr long long kLaunchThreads = 1LL << 29;
template <typename F>
hipError_t in_launches(long long groups, int threads, const F& launch)
{
  const long long most = kLaunchThreads / threads;
  for (long long first = 0; first < groups; first += most) {
    launch(first, (unsigned)std::min(most, groups - first));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// One team of G lanes per row, the row in registers (V pieces of 8 elements per lane), so x is read once
// also where the variance needs the mean first.
template <typename T, int NT, int G, int V>
__global__ __launch_bounds__(NT) void norm_fwd_kernel(T* __restrict__ y, float* __restrict__ stats,
                                                      const T* __restrict__ x, const float* __restrict__ weight,
                                                      const float* __restrict__ bias, int M, int D, float eps, int layer,
                                                      long long first)
{
  __shared__ float buf[2][NT / 64 * 1];
  const int lane = threadIdx.x % G;
  const long long row = (first + blockIdx.x) * (NT / G) + threadIdx.x / G;
  const bool live = row < M;
  const int n = live ? D : 0;
  const T* xr = x + row * D;
  float v[V][8];
#pragma unroll
  for (int c = 0; c < V; ++c) load8(xr, 8 * (lane + G * c), n, v[c]);
  float mean = 0.f;
  if (layer) {
    float s[1] = {0.f};
#pragma unroll
    for (int c = 0; c < V; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) s[0] += v[c][j];
    team_sum<G, 1>(s, buf[0]);
    mean = s[0] / (float)D;
  }
  float q[1] = {0.f};
#pragma unroll
  for (int c = 0; c < V; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float d = v[c][j] - mean;
      if (8 * (lane + G * c) + j < n) q[0] = fmaf(d, d, q[0]);
    }
  team_sum<G, 1>(q, buf[1]);
  const float r = 1.0f / sqrtf(q[0] / (float)D + eps);
  if (!live) return;
  if (stats && lane == 0) {
    stats[row] = r;
    if (layer) stats[(long long)M + row] = mean;
  }
#pragma unroll
  for (int c = 0; c < V; ++c) {
    const int i = 8 * (lane + G * c);
    if (i >= D) continue;
    float w[8], b[8];
    if (weight) load8(weight, i, D, w);
    if (bias) load8(bias, i, D, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float o = (v[c][j] - mean) * r;
      if (weight) o *= w[j];
      if (bias) o += b[j];
      v[c][j] = o;
    }
    store8(y + row * D, i, D, v[c]);
  }
}

// Rows longer than the register form takes: a work-group per row, three passes over it.
template <typename T>
__global__ __launch_bounds__(1024) void norm_fwd_long_kernel(T* __restrict__ y, float* __restrict__ stats,
                                                             const T* __restrict__ x, const float* __restrict__ weight,
                                                             const float* __restrict__ bias, int M, int D, float eps,
                                                             int layer, long long first)
{
  __shared__ float buf[2][16];
  const long long row = first + blockIdx.x;
  const T* xr = x + row * D;
  float mean = 0.f, v[8];
  if (layer) {
    float s[1] = {0.f};
    for (int i = 8 * threadIdx.x; i < D; i += 8192) {
      load8(xr, i, D, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[0] += v[j];
    }
    team_sum<1024, 1>(s, buf[0]);
    mean = s[0] / (float)D;
  }
  float q[1] = {0.f};
  for (int i = 8 * threadIdx.x; i < D; i += 8192) {
    load8(xr, i, D, v);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < D) q[0] = fmaf(v[j] - mean, v[j] - mean, q[0]);
  }
  team_sum<1024, 1>(q, buf[1]);
  const float r = 1.0f / sqrtf(q[0] / (float)D + eps);
  if (stats && threadIdx.x == 0) {
    stats[row] = r;
    if (layer) stats[(long long)M + row] = mean;
  }
  for (int i = 8 * threadIdx.x; i < D; i += 8192) {
    float w[8], b[8];
    load8(xr, i, D, v);
    if (weight) load8(weight, i, D, w);
    if (bias) load8(bias, i, D, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = (v[j] - mean) * r;
      if (weight) v[j] *= w[j];
      if (bias) v[j] += b[j];
    }
    store8(y + row * D, i, D, v);
  }
}

// dx and, per work-group, the partial sums of dweight and dbias over the rows it takes:
//   dx = r (t - mean t [layer] - xh mean(t xh)),  t = dy w,  xh = (x - mean) r.
// A lane keeps the same columns for every row, so the column sums stay in registers to the end; the teams
// then meet in LDS. The next row's bytes are requested before this row's sums meet; rows are kept as they
// were loaded and widened twice, which costs fewer registers than the widened values. FULL: layer norm, or
// dbias wanted. partial: [gridDim.x][2][D] (dweight, dbias), added in order by norm_finish_kernel.
template <typename T, int NT, int G, int V, bool FULL>
__global__ __launch_bounds__(NT, 4) void norm_bwd_kernel(T* __restrict__ dx, float* __restrict__ partial,
                                                      const T* __restrict__ dy, const T* __restrict__ x,
                                                      const float* __restrict__ weight,
                                                      const float* __restrict__ stats, int M, int D, int layer,
                                                      int want_w, int want_b)
{
  __shared__ float buf[2][NT / 64 * 2];
  __shared__ float cols[NT * V * 8];
  constexpr int R = NT / G;
  const int lane = threadIdx.x % G, team = threadIdx.x / G;
  float w[V][8], sw[V][8], sb[V][8];
  const auto load_w = [&](int c) {
    if (weight) {
      load8(weight, 8 * (lane + G * c), D, w[c]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[c][j] = 1.f;
    }
  };
  constexpr bool kKeep = V == 1;  // the weight stays in registers; the widest form reads it (from L2) per row
#pragma unroll
  for (int c = 0; c < V; ++c) {
    if (kKeep) load_w(c);
#pragma unroll
    for (int j = 0; j < 8; ++j) sw[c][j] = sb[c][j] = 0.f;
  }
  Eight<T> nx[V], ny[V];
  float nr = 0.f, nm = 0.f;
  const auto request = [&](long long row) {
    const int n = row < M ? D : 0;
    nr = n ? stats[row] : 0.f;
    nm = FULL && n && layer ? stats[(long long)M + row] : 0.f;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      nx[c] = load_raw(x + row * D, 8 * (lane + G * c), n);
      ny[c] = load_raw(dy + row * D, 8 * (lane + G * c), n);
    }
  };
  constexpr bool kAhead = V == 1;  // the widest form has no registers for a second row
  const long long step = (long long)gridDim.x * R;
  int phase = 0;
  if (kAhead) request((long long)blockIdx.x * R + team);
  for (long long first = (long long)blockIdx.x * R; first < M; first += step) {
    const long long row = first + team;
    const bool live = row < M;
    if (!kAhead) request(row);
    const float r = nr, mean = nm;
    Eight<T> cx[V], cy[V];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const int i = 8 * (lane + G * c);
      cx[c] = nx[c];
      cy[c] = ny[c];
      if (!kKeep) load_w(c);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float g = (float)cy[c].v[j], t = g * w[c][j];
        const float xh = live && i + j < D ? ((float)cx[c].v[j] - mean) * r : 0.f;
        sw[c][j] = fmaf(g, xh, sw[c][j]);
        if (FULL) sb[c][j] += g;
        if (FULL) s[0] += t;
        s[1] = fmaf(t, xh, s[1]);
      }
    }
    if (kAhead) request(row + step);
    team_sum<G, 2>(s, buf[phase]);
    phase ^= 1;
    if (!live) continue;
    const float m0 = FULL && layer ? s[0] / (float)D : 0.f, m1 = s[1] / (float)D;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const int i = 8 * (lane + G * c);
      if (i >= D) continue;
      if (!kKeep) load_w(c);
      float o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        o[j] = r * fmaf(-((float)cx[c].v[j] - mean) * r, m1, (float)cy[c].v[j] * w[c][j] - m0);
      store8(dx + row * D, i, D, o);
    }
  }
  for (int which = 0; which < 2; ++which) {
    if (which ? !want_b : !want_w) continue;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < V; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) cols[team * (G * V * 8) + 8 * (lane + G * c) + j] = which ? sb[c][j] : sw[c][j];
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += NT) {
      float s = 0.f;
      for (int k = 0; k < R; ++k) s += cols[k * (G * V * 8) + i];
      partial[((long long)blockIdx.x * 2 + which) * D + i] = s;
    }
  }
}

// Long rows: dx alone (a work-group per row, two passes) ...
template <typename T>
__global__ __launch_bounds__(1024) void norm_bwd_long_kernel(T* __restrict__ dx, const T* __restrict__ dy,
                                                             const T* __restrict__ x,
                                                             const float* __restrict__ weight,
                                                             const float* __restrict__ stats, int M, int D, int layer,
                                                             long long first)
{
  __shared__ float buf[32];
  const long long row = first + blockIdx.x;
  const float r = stats[row], mean = layer ? stats[(long long)M + row] : 0.f;
  float s[2] = {0.f, 0.f}, a[8], b[8], w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j] = 1.f;
  for (int i = 8 * threadIdx.x; i < D; i += 8192) {
    load8(x + row * D, i, D, a);
    load8(dy + row * D, i, D, b);
    if (weight) load8(weight, i, D, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float t = b[j] * w[j];
      s[0] += t;
      if (i + j < D) s[1] = fmaf(t, (a[j] - mean) * r, s[1]);
    }
  }
  team_sum<1024, 2>(s, buf);
  const float m0 = layer ? s[0] / (float)D : 0.f, m1 = s[1] / (float)D;
  for (int i = 8 * threadIdx.x; i < D; i += 8192) {
    load8(x + row * D, i, D, a);
    load8(dy + row * D, i, D, b);
    if (weight) load8(weight, i, D, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = r * fmaf(-(a[j] - mean) * r, m1, b[j] * w[j] - m0);
    store8(dx + row * D, i, D, a);
  }
}
// ... and the column sums of a run of rows, a thread per column.
template <typename T>
__global__ __launch_bounds__(256) void norm_cols_long_kernel(float* __restrict__ partial, const T* __restrict__ dy,
                                                             const T* __restrict__ x,
                                                             const float* __restrict__ stats, int M, int D, int layer)
{
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= D) return;
  float sw = 0.f, sb = 0.f;
  for (long long row = blockIdx.y; row < M; row += gridDim.y) {
    const float t = (float)dy[row * D + i];
    const float mean = layer ? stats[(long long)M + row] : 0.f;
    sw = fmaf(t, ((float)x[row * D + i] - mean) * stats[row], sw);
    sb += t;
  }
  partial[((long long)blockIdx.y * 2) * D + i] = sw;
  partial[((long long)blockIdx.y * 2 + 1) * D + i] = sb;
}

// The partial sums of `count` work-groups, added in a fixed order: 64 columns per work-group, each of its
// sixteen waves a run of the partials.
__global__ __launch_bounds__(1024) void norm_finish_kernel(float* __restrict__ dweight, float* __restrict__ dbias,
                                                           const float* __restrict__ partial, int count, int D)
{
  __shared__ float part[16][64];
  const int which = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = blockIdx.x * 64 + lane;
  float* out = which ? dbias : dweight;
  if (!out) return;
  float s = 0.f;
  if (col < D) {
    const int per = (count + 15) / 16, end = min(count, (wave + 1) * per);
    const float* q = partial + (long long)which * D + col;
#pragma unroll 8
    for (int k = wave * per; k < end; ++k) s += q[(long long)k * 2 * D];
  }
  part[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && col < D) {
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) s += part[k][lane];
    out[col] = s;
  }
}

constexpr int kNormRegisterRow = 16384;  // longest row kept in registers
constexpr int kNormBwdGroups = 512;      // most work-groups (and partial sums) of the backward: two per CU

template <typename T, int NT, int G, int V>
hipError_t norm_fwd(void* y, float* stats, const void* x, const float* w, const float* b, int M, int D, float eps,
                    int layer, hipStream_t s)
{
  constexpr int R = NT / G;
  return in_launches((M + R - 1LL) / R, NT, [&](long long first, unsigned count) {
    hipLaunchKernelGGL((norm_fwd_kernel<T, NT, G, V>), dim3(count), dim3(NT), 0, s, (T*)y, stats, (const T*)x, w, b, M,
                       D, eps, layer, first);
  });
}
template <typename T>
hipError_t norm_fwd_any(void* y, float* stats, const void* x, const float* w, const float* b, int M, int D, float eps,
                        int layer, hipStream_t s)
{
  if (D <= 128) return norm_fwd<T, 256, 16, 1>(y, stats, x, w, b, M, D, eps, layer, s);
  if (D <= 512) return norm_fwd<T, 256, 64, 1>(y, stats, x, w, b, M, D, eps, layer, s);
  if (D <= 2048) return norm_fwd<T, 256, 256, 1>(y, stats, x, w, b, M, D, eps, layer, s);
  // longer rows: one work-group per row of sixteen waves while there are few rows, fewer
  // waves per row, which wait less for each other, where there are enough rows to fill the chip
  if (M < 2 * 256 && D <= 8192) return norm_fwd<T, 1024, 1024, 1>(y, stats, x, w, b, M, D, eps, layer, s);
  if (D <= 4096) return norm_fwd<T, 256, 256, 2>(y, stats, x, w, b, M, D, eps, layer, s);
  if (D <= 8192) return norm_fwd<T, 512, 512, 2>(y, stats, x, w, b, M, D, eps, layer, s);
  if (D <= kNormRegisterRow) return norm_fwd<T, 1024, 1024, 2>(y, stats, x, w, b, M, D, eps, layer, s);
  return in_launches(M, 1024, [&](long long first, unsigned count) {
    hipLaunchKernelGGL((norm_fwd_long_kernel<T>), dim3(count), dim3(1024), 0, s, (T*)y, stats, (const T*)x, w, b, M, D,
                       eps, layer, first);
  });
}

template <typename T, int NT, int G, int V>
hipError_t norm_bwd(void* dx, float* partial, int& groups, const void* dy, const void* x, const float* w,
                    const float* stats, int M, int D, int layer, int want_w, int want_b, hipStream_t s)
{
  constexpr int R = NT / G;
  groups = (int)std::min<long long>((M + R - 1LL) / R, NT == 1024 ? kNormBwdGroups / 2 : kNormBwdGroups);
  const auto kernel = layer || want_b ? norm_bwd_kernel<T, NT, G, V, true> : norm_bwd_kernel<T, NT, G, V, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(NT), 0, s, (T*)dx, partial, (const T*)dy, (const T*)x, w,
                     stats, M, D, layer, want_w, want_b);
  return hipGetLastError();
}
template <typename T>
hipError_t norm_bwd_any(void* dx, float* dweight, float* dbias, const void* dy, const void* x, const float* w,
                        const float* stats, int M, int D, int layer, float* partial, hipStream_t s)
{
  int groups = 0;  // M = 0: no partial sums, so the column gradients come out as zeros
  const int ww = dweight != nullptr, wb = dbias != nullptr;
  hipError_t e = hipSuccess;
  if (M <= 0) {
  } else if (D <= 128) {
    e = norm_bwd<T, 512, 16, 1>(dx, partial, groups, dy, x, w, stats, M, D, layer, ww, wb, s);
  } else if (D <= 512) {
    e = norm_bwd<T, 512, 64, 1>(dx, partial, groups, dy, x, w, stats, M, D, layer, ww, wb, s);
  } else if (D <= 2048) {
    e = norm_bwd<T, 512, 256, 1>(dx, partial, groups, dy, x, w, stats, M, D, layer, ww, wb, s);
  } else if (D <= 4096) {
    e = norm_bwd<T, 512, 512, 1>(dx, partial, groups, dy, x, w, stats, M, D, layer, ww, wb, s);
  } else if (D <= 8192) {
    e = norm_bwd<T, 1024, 1024, 1>(dx, partial, groups, dy, x, w, stats, M, D, layer, ww, wb, s);
  } else if (D <= kNormRegisterRow) {
    e = norm_bwd<T, 1024, 1024, 2>(dx, partial, groups, dy, x, w, stats, M, D, layer, ww, wb, s);
  } else {
    e = in_launches(M, 1024, [&](long long first, unsigned count) {
      hipLaunchKernelGGL((norm_bwd_long_kernel<T>), dim3(count), dim3(1024), 0, s, (T*)dx, (const T*)dy, (const T*)x, w,
                         stats, M, D, layer, first);
    });
    if (e == hipSuccess && (ww || wb)) {
      groups = std::min(M, kNormBwdGroups);
      hipLaunchKernelGGL((norm_cols_long_kernel<T>), dim3((unsigned)((D + 255) / 256), (unsigned)groups), dim3(256), 0,
                         s, partial, (const T*)dy, (const T*)x, stats, M, D, layer);
      e = hipGetLastError();
    }
  }
  if (e != hipSuccess || !(ww || wb)) return e;
  hipLaunchKernelGGL(norm_finish_kernel, dim3((unsigned)((D + 63) / 64), 2), dim3(1024), 0, s, dweight, dbias, partial,
                     groups, D);
  return hipGetLastError();
}

// ------------------------------------------------------------------ dropout
// Philox4x32 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011) with 7
// rounds, the fewest with which the paper's generator passes BigCrush: counter (c0, c1, c2, c3), key (k0, k1).
MX_DEV void philox7(uint32_t (&c)[4], uint32_t k0, uint32_t k1)
{
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c[0], p1 = (uint64_t)0xCD9E8D57u * c[2];
    c[0] = (uint32_t)(p1 >> 32) ^ c[1] ^ k0;
    c[1] = (uint32_t)p1;
    c[2] = (uint32_t)(p0 >> 32) ^ c[3] ^ k1;
    c[3] = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

// Word i of the call is word i % 4 of the block with counter (i / 4, stream) under the key `seed`, whatever the
// launch looks like, so a forward, its backward and a recomputation agree. An element is dropped when its
// word is below floor(p 2^32); a dropped element is 0 even where x is NaN or infinite.
template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(T* y, const T* x, long long n, uint64_t threshold, float scale,
                                                      uint64_t seed, const uint64_t* seed_dev, uint64_t stream,
                                                      long long first)
{
  if (seed_dev) seed = *seed_dev;
  const long long i = ((first + blockIdx.x) * 256 + threadIdx.x) * 8;
  if (i >= n) return;
  const int left = n - i < 8 ? (int)(n - i) : 8;
  float v[8];
  load8(x + i, 0, left, v);
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const uint64_t block = (uint64_t)(i >> 2) + b;
    uint32_t c[4] = {(uint32_t)block, (uint32_t)(block >> 32), (uint32_t)stream, (uint32_t)(stream >> 32)};
    philox7(c, (uint32_t)seed, (uint32_t)(seed >> 32));
#pragma unroll
    for (int j = 0; j < 4; ++j) v[4 * b + j] = c[j] >= threshold ? v[4 * b + j] * scale : 0.f;
  }
  store8(y + i, 0, left, v);
}

}  // namespace

hipError_t launch_norm_forward(void* y, float* stats, const void* x, const float* weight, const float* bias, int M,
                               int D, float eps, int layer, int dtype, hipStream_t s)
{
  if (M <= 0 || D <= 0) return hipSuccess;
  if (dtype == MXFP4_F32) return norm_fwd_any<float>(y, stats, x, weight, bias, M, D, eps, layer, s);
  if (dtype == MXFP4_BF16) return norm_fwd_any<__bf16>(y, stats, x, weight, bias, M, D, eps, layer, s);
  return norm_fwd_any<_Float16>(y, stats, x, weight, bias, M, D, eps, layer, s);
}

size_t norm_backward_workspace(int M, int D) { return sizeof(float) * 2 * (size_t)std::min(M, kNormBwdGroups) * D; }

hipError_t launch_norm_backward(void* dx, float* dweight, float* dbias, const void* dy, const void* x,
                                const float* weight, const float* stats, int M, int D, int layer, int dtype,
                                float* partial, hipStream_t s)
{
  if (D <= 0) return hipSuccess;
  if (dtype == MXFP4_F32) return norm_bwd_any<float>(dx, dweight, dbias, dy, x, weight, stats, M, D, layer, partial, s);
  if (dtype == MXFP4_BF16)
    return norm_bwd_any<__bf16>(dx, dweight, dbias, dy, x, weight, stats, M, D, layer, partial, s);
  return norm_bwd_any<_Float16>(dx, dweight, dbias, dy, x, weight, stats, M, D, layer, partial, s);
}

hipError_t launch_dropout(void* y, const void* x, long long n, uint64_t threshold, float scale, uint64_t seed,
                          const uint64_t* seed_dev, uint64_t stream_id, int dtype, hipStream_t s)
{
  if (n <= 0) return hipSuccess;
  const auto typed = [&](auto zero) {
    using T = decltype(zero);
    return in_launches((n + 2047) / 2048, 256, [&](long long first, unsigned count) {
      hipLaunchKernelGGL(dropout_kernel<T>, dim3(count), dim3(256), 0, s, (T*)y, (const T*)x, n, threshold, scale, seed,
                         seed_dev, stream_id, first);
    });
  };
  if (dtype == MXFP4_F32) return typed(0.f);
  return dtype == MXFP4_BF16 ? typed((__bf16)0.f) : typed((_Float16)0.f);
}

}  // namespace mx
