// Products with group-scaled 4-bit integer weights: y = x W^T, W[r, k] = s[r, k / G] (q[r, k] - z[r, k / G]).
//
// The codes are never scaled or rounded before the product. A nibble q shifted into the top of a 16-bit
// mantissa is the number 16 + q (two instructions for two codes), and the MFMA sums x (16 + q) and, with
// an operand of ones, x itself over a group; then
//   sum x (q - z) = sum x (16 + q) - (16 + z) sum x,
// all exact products in fp32 sums, and one multiply-add by the group's scale per result. A row of x with an
// infinity gives NaN (the difference of two infinities).
#include "mx_device.h"
#include "mx_int4.h"

namespace mx {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <typename T>
struct Num;
template <>
struct Num<__bf16> {
  static constexpr uint32_t kOnes = 0x3F803F80u, kBase = 0x41804180u, kMask = 0x00780078u;  // q << 3 in 16 + q
  static constexpr int kShift = 3;
  static MX_DEV f32x4 mfma(i32x4 a, i32x4 b, f32x4 c)
  {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  }
  static MX_DEV float widen(uint16_t v) { return bits_f((uint32_t)v << 16); }
  static MX_DEV uint16_t narrow(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
};
template <>
struct Num<_Float16> {
  static constexpr uint32_t kOnes = 0x3C003C00u, kBase = 0x4C004C00u, kMask = 0x03C003C0u;  // q << 6 in 16 + q
  static constexpr int kShift = 6;
  static MX_DEV f32x4 mfma(i32x4 a, i32x4 b, f32x4 c)
  {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  }
  static MX_DEV float widen(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
  static MX_DEV uint16_t narrow(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};

// The 8 codes of a dword as 16-bit numbers 16 + q, in pairs of codes (p, p + 4), p = 0..3.
template <typename T>
MX_DEV i32x4 decode8(uint32_t w)
{
  using N = Num<T>;
  i32x4 r;
  static_for<4>([&](auto pc) {
    constexpr int p = decltype(pc)::value, sh = 4 * p - N::kShift;
    const uint32_t v = sh < 0 ? w << (sh < 0 ? -sh : 0) : w >> (sh < 0 ? 0 : sh);
    r[p] = (int)((v & N::kMask) | N::kBase);
  });
  return r;
}
// 8 elements of x in the same pairs.
MX_DEV i32x4 pair_up(i32x4 x)
{
  return i32x4{(int)__builtin_amdgcn_perm((uint32_t)x[2], (uint32_t)x[0], 0x05040100u),
               (int)__builtin_amdgcn_perm((uint32_t)x[2], (uint32_t)x[0], 0x07060302u),
               (int)__builtin_amdgcn_perm((uint32_t)x[3], (uint32_t)x[1], 0x05040100u),
               (int)__builtin_amdgcn_perm((uint32_t)x[3], (uint32_t)x[1], 0x07060302u)};
}

// K goes in blocks of 128: lane 16 c + n of a wave loads the 16 bytes with the codes 32 c .. 32 c + 31 of
// weight row n, four dwords of 8. An MFMA sums over one dword of all four c, so its dwords must be of one
// group. Groups of 128: they are. Groups of 64 and 32: the lanes of the four c exchange dwords first (the
// 32-lane halves, then also the 16-lane rows). After that dword j of lane c holds the codes from
// block_k<G>(j, c) on.
template <int G>
MX_DEV int block_k(int j, int c)
{
  if (G == 128) return 32 * c + 8 * j;
  if (G == 64) return 32 * (2 * (j >> 1) + (c & 1)) + 8 * ((j & 1) + 2 * (c >> 1));
  return 32 * j + 8 * c;
}
template <int G>
MX_DEV void one_group(uint32_t (&d)[4])
{
  const auto swap32 = [](uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0], b = r[1];
  };
  const auto swap16 = [](uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0], b = r[1];
  };
  if (G < 128) swap32(d[0], d[2]), swap32(d[1], d[3]);
  if (G < 64) swap16(d[0], d[1]), swap16(d[2], d[3]);
}

MX_DEV int pair_expert(const Int4Pairs& p, int i)
{
  long long e;
  if (p.idx64)
    e = static_cast<const long long*>(p.idx)[i];
  else
    e = static_cast<const int*>(p.idx)[i];
  return e >= 0 && e < p.E ? (int)e : -1;
}

enum Int4Epi : int {
  kInt4Store = 0,  // y[m] = the product's row, dense
  kInt4Glu = 1,    // y[p] = GLU of the gate and the up product of pair p
  kInt4Pair = 2,   // y[p] = the product of pair p, fp32
};

// A work-group makes 16 weight rows x up to 16 MT rows of x; its waves share K, block pair by block pair (so
// that a wave reads whole 128-byte lines), and their sums meet in LDS in the waves' order.
template <typename T, int G, int MT, Int4Epi EPI, int MAXW>
__global__ __launch_bounds__(64 * MAXW) void int4_rows_kernel(Int4Args p)
{
  using N = Num<T>;
  constexpr int NMAT = EPI == kInt4Glu ? 2 : 1, NG = 128 / G, JG = 4 / NG;  // groups of a block, dwords of a group
  extern __shared__ f32x4 part[];  // [waves][NMAT][MT][64]
  __shared__ int rows[16 * MT];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int n = lane & 15, c = lane >> 4;
  const int tile = blockIdx.x / p.row_groups + p.tile0, r0 = (blockIdx.x % p.row_groups) * 16;

  int e = 0, nrows;
  if (EPI == kInt4Store) {
    nrows = min(16 * MT, p.M - tile * (16 * MT));
    if ((int)threadIdx.x < 16 * MT) rows[threadIdx.x] = tile * (16 * MT) + min((int)threadIdx.x, nrows - 1);
  } else if (p.tiles) {
    if (tile >= *p.n_tiles) return;
    const int4 t = p.tiles[tile];
    e = t.x;
    nrows = t.z;
    if ((int)threadIdx.x < 16 * MT) rows[threadIdx.x] = p.order[t.y + min((int)threadIdx.x, nrows - 1)];
  } else {
    // the pairs of this one's expert from this one on, which must be the first of their tile
    const int mine = lane < p.pairs.P ? pair_expert(p.pairs, lane) : -1;
    e = __builtin_amdgcn_readlane(mine, tile);
    if (e < 0) return;
    const uint64_t same = __builtin_amdgcn_ballot_w64(mine == e);
    const int first = __popcll(same & ((1ull << tile) - 1));
    if (first % (16 * MT)) return;
    nrows = min(16 * MT, __popcll(same) - first);
    const int at = __popcll(same & ((1ull << lane) - 1)) - first;
    if (wave == 0 && mine == e && at >= 0 && at < nrows) rows[at] = lane;
  }
  __syncthreads();

  const int wr = min(r0 + n, p.R - 1), groups = p.K / G;
  const uint8_t* wq[NMAT];
  const uint16_t* ws[NMAT];
  const uint8_t* wz[NMAT];
#pragma unroll
  for (int m = 0; m < NMAT; ++m) {
    const long long r = (long long)e * p.R + wr;
    wq[m] = p.w[m].q + r * (p.K / 2);
    ws[m] = static_cast<const uint16_t*>(p.w[m].s) + r * groups;
    wz[m] = p.w[m].z ? p.w[m].z + r * groups : nullptr;
  }
  const uint16_t* xr[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int i = rows[min(16 * t + n, nrows - 1)];
    xr[t] = static_cast<const uint16_t*>(p.x) + (long long)(EPI == kInt4Store ? i : i / p.x_div) * p.K;
  }

  f32x4 acc[NMAT][MT];
#pragma unroll
  for (int m = 0; m < NMAT; ++m)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const i32x4 ones = {(int)N::kOnes, (int)N::kOnes, (int)N::kOnes, (int)N::kOnes};
  const int blocks = (p.K + 127) / 128;

  struct Block {
    i32x4 q[NMAT], x[MT][4];
    uint16_t s[NMAT][NG];
    uint8_t z[NMAT][NG];
  };
  // past K the codes are some other of the row's and x is 0
  const auto load = [&](int b, Block& k) {
    const int kc = G == 128 ? b * 128 + 32 * c : min(b * 128 + 32 * c, p.K - 32);
#pragma unroll
    for (int m = 0; m < NMAT; ++m) {
      k.q[m] = *reinterpret_cast<const i32x4*>(wq[m] + kc / 2);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const int gi = G == 128 ? b : min(b * NG + g, groups - 1);
        k.s[m][g] = ws[m][gi];
        k.z[m][g] = wz[m] ? wz[m][gi] : (uint8_t)8;
      }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int kx = b * 128 + block_k<G>(j, c);
        k.x[t][j] = i32x4{0, 0, 0, 0};
        if (G == 128 || kx < p.K) k.x[t][j] = *reinterpret_cast<const i32x4*>(xr[t] + kx);
      }
  };
  const auto multiply = [&](const Block& k) {
    uint32_t d[NMAT][4];
#pragma unroll
    for (int m = 0; m < NMAT; ++m) {
#pragma unroll
      for (int j = 0; j < 4; ++j) d[m][j] = (uint32_t)k.q[m][j];
      one_group<G>(d[m]);
    }
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      f32x4 sum[MT], dot[NMAT][MT];
#pragma unroll
      for (int j = g * JG; j < (g + 1) * JG; ++j) {
        i32x4 w[NMAT];
#pragma unroll
        for (int m = 0; m < NMAT; ++m) w[m] = decode8<T>(d[m][j]);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const i32x4 x = pair_up(k.x[t][j]);
          sum[t] = N::mfma(x, ones, j == g * JG ? zero : sum[t]);
#pragma unroll
          for (int m = 0; m < NMAT; ++m) dot[m][t] = N::mfma(x, w[m], j == g * JG ? zero : dot[m][t]);
        }
      }
#pragma unroll
      for (int m = 0; m < NMAT; ++m) {
        const float s = N::widen(k.s[m][g]), z = -16.0f - (float)k.z[m][g];
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[m][t][i] = fmaf(s, fmaf(z, sum[t][i], dot[m][t][i]), acc[m][t][i]);
      }
    }
  };
  for (int b = 2 * wave; b < blocks; b += 2 * waves) {
    Block k0, k1;
    load(b, k0);
    if (b + 1 < blocks) load(b + 1, k1);
    multiply(k0);
    if (b + 1 < blocks) multiply(k1);
  }

#pragma unroll
  for (int m = 0; m < NMAT; ++m)
#pragma unroll
    for (int t = 0; t < MT; ++t) part[((wave * NMAT + m) * MT + t) * 64 + lane] = acc[m][t];
  __syncthreads();
  const float* sums = reinterpret_cast<const float*>(part);
  for (int i = threadIdx.x; i < MT * 256; i += blockDim.x) {
    const int row = i >> 4, col = i & 15;  // lane 16 (row % 16 / 4) + col holds it in element row % 4
    const int at = (row >> 4) * 256 + (16 * ((row & 15) >> 2) + col) * 4 + (row & 3);
    float v[NMAT];
#pragma unroll
    for (int m = 0; m < NMAT; ++m) {
      v[m] = 0.f;
      for (int w = 0; w < waves; ++w) v[m] += sums[(w * NMAT + m) * MT * 256 + at];
    }
    if (row >= nrows || r0 + col >= p.R) continue;
    const long long o = (long long)rows[row] * p.R + r0 + col;
    if (EPI == kInt4Pair)
      static_cast<float*>(p.y)[o] = v[0];
    else
      static_cast<uint16_t*>(p.y)[o] = N::narrow(EPI == kInt4Glu ? glu_fwd(v[0], v[NMAT - 1], p.act) : v[0]);
  }
}

// ------------------------------------------------------------------ routing
// The pairs in the order of their experts, and the tiles of up to tile_rows of them: one work-group, counts
// and places in LDS. The order of an expert's pairs is left to the atomics: a row's result does not depend
// on its place.
constexpr int kRouteMaxExperts = 4096;
__global__ __launch_bounds__(1024) void int4_route_kernel(Int4Pairs p, int tile_rows, int4* tiles, int* n_tiles,
                                                          int* order)
{
  __shared__ int place[kRouteMaxExperts];
  __shared__ int wave_pairs[16], wave_tiles[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int e = tid; e < p.E; e += 1024) place[e] = 0;
  __syncthreads();
  for (int i = tid; i < p.P; i += 1024) {
    const int e = pair_expert(p, i);
    if (e >= 0) atomicAdd(&place[e], 1);
  }
  __syncthreads();
  // thread t has experts t per .. t per + per - 1
  const int per = (p.E + 1023) / 1024;
  int pairs = 0, count = 0;
  for (int i = 0; i < per; ++i) {
    const int e = tid * per + i;
    if (e < p.E) {
      pairs += place[e];
      count += (place[e] + tile_rows - 1) / tile_rows;
    }
  }
  int before_p = pairs, before_t = count;  // inclusive over the wave, then exclusive over the work-group
  for (int off = 1; off < 64; off <<= 1) {
    const int a = __shfl_up(before_p, off, 64), b = __shfl_up(before_t, off, 64);
    if (lane >= off) before_p += a, before_t += b;
  }
  if (lane == 63) wave_pairs[wave] = before_p, wave_tiles[wave] = before_t;
  __syncthreads();
  before_p -= pairs;
  before_t -= count;
  for (int w = 0; w < wave; ++w) before_p += wave_pairs[w], before_t += wave_tiles[w];
  if (tid == 1023) *n_tiles = before_t + count;
  for (int i = 0; i < per; ++i) {
    const int e = tid * per + i;
    if (e >= p.E) break;
    const int rows = place[e];
    for (int r = 0; r < rows; r += tile_rows) tiles[before_t++] = int4{e, before_p + r, min(tile_rows, rows - r), 0};
    place[e] = before_p;
    before_p += rows;
  }
  __syncthreads();
  for (int i = tid; i < p.P; i += 1024) {
    const int e = pair_expert(p, i);
    if (e >= 0) order[atomicAdd(&place[e], 1)] = i;
  }
}

// out[t] = the slots' weighted rows in slot order; 4 columns per thread.
template <typename T>
__global__ __launch_bounds__(256) void int4_combine_kernel(uint16_t* out, const float* y, const float* topk_w,
                                                           Int4Pairs p, int D, long long n)
{
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const int t = (int)(i / D), d = (int)(i - (long long)t * D);
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < p.k; ++j) {
    const int q = t * p.k + j;
    if (pair_expert(p, q) < 0) continue;
    const float w = topk_w[q];
    const f32x4 v = *reinterpret_cast<const f32x4*>(y + (long long)q * D + d);
#pragma unroll
    for (int l = 0; l < 4; ++l) sum[l] = fmaf(w, v[l], sum[l]);
  }
  u32x2 r;
  r[0] = (uint32_t)Num<T>::narrow(sum[0]) | (uint32_t)Num<T>::narrow(sum[1]) << 16;
  r[1] = (uint32_t)Num<T>::narrow(sum[2]) | (uint32_t)Num<T>::narrow(sum[3]) << 16;
  *reinterpret_cast<u32x2*>(out + i) = r;
}

template <typename T, int G, int MT, Int4Epi EPI>
hipError_t launch_rows(Int4Args a, int tiles, hipStream_t s)
{
  constexpr int NMAT = EPI == kInt4Glu ? 2 : 1, MAXW = MT == 1 ? 16 : 8;
  a.row_groups = (a.R + 15) / 16;
  // waves: enough for 16 on every CU, each with a block pair at least
  const int pairs = (a.K + 255) / 256;
  const long long groups = (long long)a.row_groups * tiles;
  int waves = 4;
  while (waves < MAXW && waves * groups < 4096) waves *= 2;
  while (waves > 1 && waves / 2 >= pairs) waves /= 2;
  // a launch's threads are counted in 32 bits
  const int most = max(1, (int)(((1u << 31) / (64 * MAXW)) / a.row_groups));
  for (a.tile0 = 0; a.tile0 < tiles; a.tile0 += most) {
    const int now = min(most, tiles - a.tile0);
    int4_rows_kernel<T, G, MT, EPI, MAXW>
        <<<dim3((unsigned)now * a.row_groups), dim3(64 * waves), sizeof(f32x4) * waves * NMAT * MT * 64, s>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T, Int4Epi EPI>
hipError_t launch_group(const Int4Args& a, int group, int rows, int tiles, hipStream_t s)
{
#define MX_INT4_ROWS(G)                                                 \
  (rows == 16 ? launch_rows<T, G, 1, EPI>(a, tiles, s)                  \
              : rows == 32 ? launch_rows<T, G, 2, EPI>(a, tiles, s) : launch_rows<T, G, 4, EPI>(a, tiles, s))
  switch (group) {
    case 32: return MX_INT4_ROWS(32);
    case 64: return MX_INT4_ROWS(64);
    default: return MX_INT4_ROWS(128);
  }
#undef MX_INT4_ROWS
}

int rows_of(int m) { return m <= 16 ? 16 : m <= 32 ? 32 : 64; }

template <Int4Epi EPI>
hipError_t launch_routed(const Int4Args& a, int group, int dtype, hipStream_t s)
{
  const int rows = int4_tile_rows(a.pairs.P, a.pairs.E);
  const int tiles = a.tiles ? int4_max_tiles(a.pairs.P, a.pairs.E) : a.pairs.P;
  return dtype == 1 ? launch_group<__bf16, EPI>(a, group, rows, tiles, s)
                    : launch_group<_Float16, EPI>(a, group, rows, tiles, s);
}

}  // namespace

hipError_t launch_int4_gemm(const Int4Args& a, int group, int dtype, hipStream_t s)
{
  const int rows = rows_of(a.M), tiles = (int)(((long long)a.M + rows - 1) / rows);
  return dtype == 1 ? launch_group<__bf16, kInt4Store>(a, group, rows, tiles, s)
                    : launch_group<_Float16, kInt4Store>(a, group, rows, tiles, s);
}

int int4_tile_rows(int P, int E) { return rows_of(P / E); }

hipError_t launch_int4_route(const Int4Pairs& p, int4* tiles, int* n_tiles, int* order, hipStream_t s)
{
  int4_route_kernel<<<1, 1024, 0, s>>>(p, int4_tile_rows(p.P, p.E), tiles, n_tiles, order);
  return hipGetLastError();
}

hipError_t launch_int4_glu(const Int4Args& a, int group, int dtype, hipStream_t s)
{
  return launch_routed<kInt4Glu>(a, group, dtype, s);
}
hipError_t launch_int4_pairs(const Int4Args& a, int group, int dtype, hipStream_t s)
{
  return launch_routed<kInt4Pair>(a, group, dtype, s);
}

hipError_t launch_int4_combine(void* out, const float* y, const float* topk_w, const Int4Pairs& p, int D, int dtype,
                               hipStream_t s)
{
  const long long n = (long long)(p.P / p.k) * D;
  const long long blocks = (n / 4 + 255) / 256;
  uint16_t* o = static_cast<uint16_t*>(out);
  if (dtype == 1)
    int4_combine_kernel<__bf16><<<(unsigned)blocks, 256, 0, s>>>(o, y, topk_w, p, D, n);
  else
    int4_combine_kernel<_Float16><<<(unsigned)blocks, 256, 0, s>>>(o, y, topk_w, p, D, n);
  return hipGetLastError();
}

}  // namespace mx
