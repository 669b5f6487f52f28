// Products with group-scaled 4-bit integer weights: y = x W^T, W[r, k] = s[r, k / G] (q[r, k] - z[r, k / G]).
//
// The codes are never scaled or rounded before the product. A nibble q shifted into the top of a 16-bit
// mantissa is the number 16 + q (two instructions for two codes), and the MFMA sums x (16 + q) and, with
// an operand of ones, x itself over a group; then
//   sum x (q - z) = sum x (16 + q) - (16 + z) sum x,
// all exact products in fp32 sums, and one multiply-add by the group's scale per result. A row of x with an
// infinity gives NaN (the difference of two infinities), and so does one whose sums pass 32 bits: a group's
// sum of |x| max(31, 16 + z) has to stay below 2^127, which float16 cannot reach and bfloat16 only where |x|
// passes 2^111 in all 128 places (any zero point). An infinite or NaN scale gives such results in its weight row.
#include "mx_device.h"
#include "mx_int4.h"

namespace mx {

namespace {

constexpr int kVecRows = 8;     // weight rows of a batch of the few-row form
constexpr int kVecBatches = 16;  // batches of a work-group at most
constexpr int kStripGroups = 4;   // groups of 16 weight rows of a work-group of the form for 16 rows of x, at most
constexpr int kVecMost = 4;      // its rows of x at most
constexpr int kVecMinK = 1024;  // and the shortest rows it takes

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
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
  static MX_DEV float dot2(uint32_t a, uint32_t b, float c)
  {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, a), __builtin_bit_cast(bf16x2, b), c, false);
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
  static MX_DEV float dot2(uint32_t a, uint32_t b, float c)
  {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, a), __builtin_bit_cast(f16x2, b), c, false);
  }
  static MX_DEV float widen(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
  static MX_DEV uint16_t narrow(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};

// The decoder's constants in registers: and-or of three operands is one instruction then, which takes one
// scalar register and no literals.
struct Decoder {
  uint32_t mask, base;
};
template <typename T>
MX_DEV Decoder decoder()
{
  Decoder d;
  asm("s_mov_b32 %0, %1" : "=s"(d.mask) : "i"(Num<T>::kMask));
  asm("v_mov_b32 %0, %1" : "=v"(d.base) : "i"(Num<T>::kBase));
  return d;
}
// The 8 codes of a dword as 16-bit numbers 16 + q, in pairs of codes (p, p + 4), p = 0..3.
template <typename T>
MX_DEV i32x4 decode8(uint32_t w, Decoder k)
{
  using N = Num<T>;
  i32x4 r;
  static_for<4>([&](auto pc) {
    constexpr int p = decltype(pc)::value, sh = 4 * p - N::kShift;
    const uint32_t v = sh < 0 ? w << (sh < 0 ? -sh : 0) : w >> (sh < 0 ? 0 : sh);
    r[p] = (int)((v & k.mask) | k.base);
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

// Sum over the 16 lanes of a row, in every lane.
MX_DEV float row_sum(float v)
{
  v += dpp_lane<kDppXor1>(v);
  v += dpp_lane<kDppXor2>(v);
  v += dpp_lane<kDppHalfMirror>(v);
  return v + dpp_lane<kDppMirror>(v);
}

enum Int4Epi : int {
  kInt4Store = 0,  // y[m] = the product's row, dense
  kInt4Glu = 1,    // y[p] = GLU of the gate and the up product of pair p
  kInt4Pair = 2,   // y[p] = the product of pair p, fp32
  kInt4Token = 3,  // y[t] = the weighted sum of the products of token t's pairs
};

// Result o of a product (a gate and an up product).
template <typename T, Int4Epi EPI>
MX_DEV void store(const Int4Args& p, long long o, float a, float b)
{
  if (EPI == kInt4Pair)
    static_cast<float*>(p.y)[o] = a;
  else
    static_cast<uint16_t*>(p.y)[o] = Num<T>::narrow(EPI == kInt4Glu ? glu_fwd(a, b, p.act) : a);
}

// The rows of a work-group's tile (up to ROWS of them): their numbers into rows[] (the places behind the last
// repeat it), the expert and the count. False: there is nothing to do. The work-group synchronises after it.
template <int ROWS, Int4Epi EPI>
MX_DEV bool find_rows(const Int4Args& p, int tile, int* rows, int& e, int& nrows)
{
  const int tid = threadIdx.x, lane = tid & 63;
  if (EPI == kInt4Store) {
    e = 0;
    nrows = min(ROWS, p.M - tile * ROWS);
    if (tid < ROWS) rows[tid] = tile * ROWS + min(tid, nrows - 1);
  } else if (p.tiles) {
    if (tile >= *p.n_tiles) return false;
    const int4 t = p.tiles[tile];
    e = __builtin_amdgcn_readfirstlane(t.x);  // the same on every lane: addresses from it are scalar
    nrows = __builtin_amdgcn_readfirstlane(t.z);
    if (tid < ROWS) rows[tid] = p.order[t.y + min(tid, nrows - 1)];
  } else {
    // the pairs of this one's expert from this one on, which must be the first of their tile
    const int mine = lane < p.pairs.P ? pair_expert(p.pairs, lane) : -1;
    e = __builtin_amdgcn_readlane(mine, tile);
    if (e < 0) return false;
    const uint64_t same = __builtin_amdgcn_ballot_w64(mine == e);
    const int first = __popcll(same & ((1ull << tile) - 1));
    if (first % ROWS) return false;
    nrows = min(ROWS, __popcll(same) - first);
    const int at = __popcll(same & ((1ull << lane) - 1)) - first;
    if (tid < 64 && mine == e && at >= 0 && at < nrows) {
      rows[at] = lane;
      if (at == nrows - 1)
        for (int i = nrows; i < ROWS; ++i) rows[i] = lane;
    }
  }
  return true;
}

// A tile's rows of one matrix as buffers: codes, scales and zero points from row `first` on. A load adds a lane's
// offset (past the buffer, kOob, it gives zeros and reads nothing) and one that the wave shares.
constexpr uint32_t kOob = 0x80000000u;
struct Rows {
  __amdgpu_buffer_rsrc_t q, s, z;
};
MX_DEV __amdgpu_buffer_rsrc_t buffer(const void* base, uint32_t bytes)
{
  // scalar for certain: where the compiler does not see that it is, every load becomes a loop over the lanes
  const uint64_t b = (uint64_t)(uintptr_t)base;
  const uint64_t u = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(b >> 32)) << 32 |
                     (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)b);
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(u), 0, __builtin_amdgcn_readfirstlane(bytes),
                                           0x00020000);
}
MX_DEV Rows weight_rows(const Int4Matrix& w, long long first, int count, int K, int groups)
{
  return {buffer(w.q + first * (K / 2), (uint32_t)count * (K / 2)),
          buffer(static_cast<const uint16_t*>(w.s) + first * groups, 2u * count * groups),
          buffer(w.z + first * groups, (uint32_t)count * groups)};
}
MX_DEV i32x4 load_codes(const Rows& w, uint32_t lane, uint32_t shared)
{
  return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(w.q, (int)lane, (int)shared, 0));
}
// The byte offset of a scale, from its number: doubled without a sign, so that kOob / 2 becomes kOob (in an int that
// overflows, and what the compiler may then assume of the number is that it is smaller).
constexpr int scale_bytes(uint32_t number) { return (int)(2 * number); }
static_assert((uint32_t)scale_bytes(kOob / 2) == kOob, "past every buffer");
MX_DEV uint16_t load_scale(const Rows& w, uint32_t lane, uint32_t shared)
{
  return (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(w.s, scale_bytes(lane), scale_bytes(shared), 0);
}
MX_DEV uint8_t load_zero(const Rows& w, uint32_t lane, uint32_t shared)
{
  return (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(w.z, (int)lane, (int)shared, 0);
}

// ------------------------------------------------------------------ few rows of x
// Lane i keeps the elements 32 i .. 32 i + 31 of up to MR rows of x in registers and walks the weight rows, kVecRows
// of them loaded while those before are summed. A wave's load is 1 KiB of one row, x is loaded once for all rows of a
// work-group (with every 16 x 128 block of the codes, as the MFMA takes them, there would be as many bytes of x as of
// codes), and a product is two instructions for two codes and one dot of two for each row of x. The lanes' sums meet
// in exchanges of half-waves and quarter-waves, each of which halves how many there are, the waves' in LDS. One row
// is bound by the codes' bytes behind some 5 us of launch, first loads and last sums: rows of 8192 in groups of 64,
// us (TB/s): 4096 weight rows 6.9 (2.7), 28672 26 (4.9), 114688 89 (5.8), 229376 171 (6.0). Two rows 8.6 / 30 / 94 /
// 189; four 10.6 / 42 / 129 / 260, bound by the dots (the 4 x 4 x 4 MFMA in their place, x in its 16 registers
// whatever its rows: 8.6 / 30 / 121 / 218 with one row, 9.5 / 32 / 127 / 231 with four; not kept as a second form
// for three and four rows alone).
template <typename T, int G, bool ZP, int MR, Int4Epi EPI>
__global__ __launch_bounds__(512) void int4_vec_kernel(Int4Args p)
{
  using N = Num<T>;
  constexpr int NMAT = EPI == kInt4Glu ? 2 : 1, RB = kVecRows / NMAT, NV = kVecRows * MR;
  extern __shared__ float red[];  // [waves][batches][NV]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int item = blockIdx.x / p.row_groups + p.tile0, r0 = (blockIdx.x % p.row_groups) * (p.batches * RB);
  const int batches = min(p.batches, (p.R - r0 + RB - 1) / RB), groups = p.K / G;
  const int team = EPI == kInt4Token ? wave / p.team : 0;  // waves that share a row of K
  const int first_k = 32 * (EPI == kInt4Token ? (int)threadIdx.x - team * p.team * 64 : (int)threadIdx.x);
  const int stride_k = 32 * 64 * (EPI == kInt4Token ? p.team : waves);
  const Decoder dec = decoder<T>();
  float* mine = red + wave * p.batches * NV;
  // a lane's place of value i of a batch, i < NV / 4, after the exchanges
  const int place = (lane >> 4 & 1) * (NV / 4) + (lane >> 5) * (NV / 2);
  for (int i = lane; i < batches * NV; i += 64) mine[i] = 0.f;
  wave_lds_fence();

  // one expert's rows (of a token: one slot after another of this team's)
  const auto rows_of_expert = [&](int e, long long x_row, float weight) {
    Rows w[NMAT];
#pragma unroll
    for (int m = 0; m < NMAT; ++m)
      w[m] = weight_rows(p.w[m], (long long)e * p.R + r0, min(p.batches * RB, p.R - r0), p.K, groups);
    struct Batch {
      i32x4 q[kVecRows];
      uint16_t s[kVecRows];
      uint8_t z[kVecRows];
    };
    for (int k = first_k; k - first_k < p.K; k += stride_k) {  // the same rounds on every lane
      const bool in = k < p.K;
      const uint32_t at_q = in ? (uint32_t)k / 2 : kOob, at_s = in ? (uint32_t)k / G : kOob / 2;
      // A batch behind the last is loaded all the same, from past the buffers, so that what is in flight where the
      // one before it is summed is the same on every path: at a branch around these loads the compiler waits for all.
      const auto load = [&](int b, Batch& c) {
        const uint32_t lane_q = b < batches ? at_q : kOob, lane_s = b < batches ? at_s : kOob / 2;
#pragma unroll
        for (int r = 0; r < kVecRows; ++r) {
          const uint32_t row = min(b * RB + r % RB, p.R - 1 - r0);
          c.q[r] = load_codes(w[r / RB], lane_q, row * (p.K / 2));
          c.s[r] = load_scale(w[r / RB], lane_s, row * groups);
          c.z[r] = ZP ? load_zero(w[r / RB], lane_s, row * groups) : (uint8_t)8;
        }
      };
      Batch c0, c1;
      load(0, c0);
      uint32_t x[MR][16];
      float sum[MR];
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        const long long row = EPI == kInt4Store ? min(m, p.M - 1) : x_row;
        const i32x4* src = reinterpret_cast<const i32x4*>(static_cast<const uint16_t*>(p.x) + row * p.K + (in ? k : 0));
        sum[m] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const i32x4 t = pair_up(src[j]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[m][4 * j + i] = in ? (uint32_t)t[i] : 0u;
            sum[m] = N::dot2(x[m][4 * j + i], N::kOnes, sum[m]);
          }
        }
      }
      const auto multiply = [&](int b, const Batch& c) {
        float v[NV];
#pragma unroll
        for (int r = 0; r < kVecRows; ++r) {
          float t[MR];
#pragma unroll
          for (int m = 0; m < MR; ++m) t[m] = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const i32x4 d = decode8<T>((uint32_t)c.q[r][j], dec);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int m = 0; m < MR; ++m) t[m] = N::dot2(x[m][4 * j + i], (uint32_t)d[i], t[m]);
          }
          const float scale = N::widen(c.s[r]) * weight, zero = -16.0f - (float)c.z[r];
#pragma unroll
          for (int m = 0; m < MR; ++m) v[r * MR + m] = scale * fmaf(zero, sum[m], t[m]);
        }
        // of two values a lane keeps one, with the other lane's share
#pragma unroll
        for (int i = 0; i < NV / 2; ++i) {
          const auto r = __builtin_amdgcn_permlane32_swap(f_bits(v[i]), f_bits(v[i + NV / 2]), false, false);
          v[i] = bits_f(r[0]) + bits_f(r[1]);
        }
#pragma unroll
        for (int i = 0; i < NV / 4; ++i) {
          const auto r = __builtin_amdgcn_permlane16_swap(f_bits(v[i]), f_bits(v[i + NV / 4]), false, false);
          v[i] = row_sum(bits_f(r[0]) + bits_f(r[1]));
        }
        if ((lane & 15) == 0) {
#pragma unroll
          for (int i = 0; i < NV / 4; ++i) mine[b * NV + place + i] += v[i];
        }
      };
      for (int b = 0; b < batches; b += 2) {
        load(b + 1, c1);
        multiply(b, c0);
        if (b + 1 >= batches) break;
        load(b + 2, c0);
        multiply(b + 1, c1);
      }
    }
  };
  if (EPI == kInt4Token) {
    const int teams = waves / p.team;
    for (int j = team; j < p.pairs.k; j += teams) {
      const int q = item * p.pairs.k + j;
      const int e = __builtin_amdgcn_readfirstlane(pair_expert(p.pairs, q));
      if (e >= 0) rows_of_expert(e, q, p.row_w[q]);
    }
  } else if (EPI == kInt4Glu) {
    const int e = __builtin_amdgcn_readfirstlane(pair_expert(p.pairs, item));
    if (e < 0) return;  // the whole work-group
    rows_of_expert(e, item / p.x_div, 1.f);
  } else {
    rows_of_expert(0, 0, 1.f);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < batches * RB * MR; i += blockDim.x) {
    const int b = i / (RB * MR), j = i % (RB * MR), m = j % MR, row = r0 + b * RB + j / MR;
    float u = 0.f, v = 0.f;
    for (int w = 0; w < waves; ++w) {
      u += red[(w * p.batches + b) * NV + j];
      if (NMAT == 2) v += red[(w * p.batches + b) * NV + RB * MR + j];
    }
    const long long o = EPI == kInt4Store ? m : item;
    if ((EPI != kInt4Store || m < p.M) && row < p.R) store<T, EPI>(p, o * p.R + row, u, v);
  }
}

// ------------------------------------------------------------------ up to 16 rows of x
// A wave keeps 256 terms of up to 16 rows of x in registers, as the MFMA takes them, with their sums over each group,
// and walks groups of 16 weight rows (of a gate/up product: of both matrices), the codes of the next one in flight.
// The waves of a work-group share K; their sums meet in LDS once, in the waves' order. Bound by the codes' bytes
// where they are many (256 pairs over 128 experts, 3584 / 1536, gate/up: 0.64 GB in 121 us, 5.3 TB/s), else by the
// launch: 13 rows of [7168, 3584], groups of 32, 9.0 us, where x from L2 with every block took 17.5 and x staged in
// LDS for the whole work-group 12.9 to 17.
// Waves of a work-group at most: as many as their registers let in without spills (two matrices, or a scale loaded by
// itself for each group of 32, take more).
constexpr int strip_waves(int group, Int4Epi epi, bool wide)
{
  return epi == kInt4Glu || (group == 32 && !wide) ? 8 : 16;
}
template <typename T, int G, bool ZP, Int4Epi EPI, bool WIDE>
__global__ __launch_bounds__(64 * strip_waves(G, EPI, WIDE)) void int4_strip_kernel(Int4Args p)
{
  using N = Num<T>;
  constexpr int NMAT = EPI == kInt4Glu ? 2 : 1, NG = 128 / G, JG = 4 / NG, NB = kStripGroups;
  extern __shared__ f32x4 part[];  // [waves][p.batches][NMAT][64]
  __shared__ int rows[16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int n = lane & 15, c = lane >> 4;
  const int tile = blockIdx.x / p.row_groups + p.tile0, g0 = (blockIdx.x % p.row_groups) * p.batches;
  const int count = min(p.batches, (p.R + 15) / 16 - g0), groups = p.K / G;
  int e, nrows;
  if (!find_rows<16, EPI>(p, tile, rows, e, nrows)) return;
  __syncthreads();
  const int units = (p.K + 255) / 256, rounds = (units + waves - 1) / waves;
  const Decoder dec = decoder<T>();
  const i32x4 ones = {(int)N::kOnes, (int)N::kOnes, (int)N::kOnes, (int)N::kOnes};
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  const int x_row = rows[n];
  const uint16_t* xr =
      static_cast<const uint16_t*>(p.x) + (long long)(EPI == kInt4Store ? x_row : x_row / p.x_div) * p.K;
  Rows w[NMAT];
#pragma unroll
  for (int m = 0; m < NMAT; ++m)
    w[m] = weight_rows(p.w[m], (long long)e * p.R + 16 * g0, min(16 * count, p.R - 16 * g0), p.K, groups);

  struct Step {
    i32x4 q[NMAT][2];
    uint32_t s[NMAT][NG];            // 2 NG scales
    uint32_t z[NMAT][(NG + 1) / 2];  // 2 NG zero points
  };
  // what lies past K, past R or past the last group is loaded from past the buffers: zeros
  const uint32_t lane_q = (uint32_t)n * (p.K / 2) + 16 * c, lane_s = (uint32_t)n * groups;
  const auto load = [&](int g, int u, Step& t) {
    const bool in = (g < count) & (u < units) & (16 * (g0 + g) + n < p.R);
    const uint32_t row = 16 * g;
#pragma unroll
    for (int m = 0; m < NMAT; ++m) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const bool there = WIDE ? in : in & (256 * u + 128 * b + 32 * c < p.K);
        t.q[m][b] = load_codes(w[m], there ? lane_q : kOob, row * (p.K / 2) + 128 * u + 64 * b);
      }
      if constexpr (WIDE) {
        const uint32_t at = in ? lane_s : kOob / 2, shared = row * groups + u * (2 * NG);
        if constexpr (NG == 4) {
          const i32x4 v = __builtin_bit_cast(
              i32x4, __builtin_amdgcn_raw_buffer_load_b128(w[m].s, scale_bytes(at), scale_bytes(shared), 0));
#pragma unroll
          for (int i = 0; i < 4; ++i) t.s[m][i] = v[i];
          if (ZP) {
            const auto y = __builtin_amdgcn_raw_buffer_load_b64(w[m].z, (int)at, (int)shared, 0);
            t.z[m][0] = y[0], t.z[m][1] = y[1];
          }
        } else if constexpr (NG == 2) {
          const auto v = __builtin_amdgcn_raw_buffer_load_b64(w[m].s, scale_bytes(at), scale_bytes(shared), 0);
          t.s[m][0] = v[0], t.s[m][1] = v[1];
          if (ZP) t.z[m][0] = __builtin_amdgcn_raw_buffer_load_b32(w[m].z, (int)at, (int)shared, 0);
        } else {
          t.s[m][0] = __builtin_amdgcn_raw_buffer_load_b32(w[m].s, scale_bytes(at), scale_bytes(shared), 0);
          if (ZP) t.z[m][0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(w[m].z, (int)at, (int)shared, 0);
        }
      } else {
#pragma unroll
        for (int i = 0; i < NG; ++i) t.s[m][i] = 0;
#pragma unroll
        for (int i = 0; i < (NG + 1) / 2; ++i) t.z[m][i] = 0;
#pragma unroll
        for (int i = 0; i < 2 * NG; ++i) {
          const int group = u * (2 * NG) + i;
          const uint32_t at = in & (group < groups) ? lane_s : kOob / 2;
          t.s[m][i / 2] |= (uint32_t)load_scale(w[m], at, row * groups + group) << (16 * (i & 1));
          if (ZP) t.z[m][i / 4] |= (uint32_t)load_zero(w[m], at, row * groups + group) << (8 * (i & 3));
        }
      }
    }
  };
  f32x4 acc[NB][NMAT];
#pragma unroll
  for (int g = 0; g < NB; ++g)
#pragma unroll
    for (int m = 0; m < NMAT; ++m) acc[g][m] = zero;
  Step step[2];
  for (int r = 0; r < rounds; ++r) {
    const int u = wave + r * waves;
    load(0, u, step[0]);
    i32x4 x[2][4];
    f32x4 sum[2 * NG];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = 256 * u + 128 * b + block_k<G>(j, c);
        const bool in = k < p.K;
        const i32x4 v = *reinterpret_cast<const i32x4*>(xr + (in ? k : 0));
        x[b][j] = pair_up(in ? v : i32x4{0, 0, 0, 0});
        f32x4& s = sum[b * NG + j / JG];
        s = N::mfma(x[b][j], ones, j % JG ? s : zero);
      }
    static_for<NB>([&](auto gc) {
      constexpr int g = decltype(gc)::value;
      load(g + 1, u, step[(g + 1) & 1]);
      if (g >= count) return;
      const Step& t = step[g & 1];
      static_for<2>([&](auto bc) {
        constexpr int b = decltype(bc)::value;
        uint32_t d[NMAT][4];
#pragma unroll
        for (int m = 0; m < NMAT; ++m) {
#pragma unroll
          for (int j = 0; j < 4; ++j) d[m][j] = (uint32_t)t.q[m][b][j];
          one_group<G>(d[m]);
        }
        static_for<NG>([&](auto ic) {
          constexpr int i = b * NG + decltype(ic)::value, j0 = decltype(ic)::value * JG;
#pragma unroll
          for (int m = 0; m < NMAT; ++m) {
            f32x4 dot = zero;
#pragma unroll
            for (int j = j0; j < j0 + JG; ++j) dot = N::mfma(x[b][j], decode8<T>(d[m][j], dec), dot);
            const float s = N::widen((uint16_t)(t.s[m][i / 2] >> (16 * (i & 1))));
            const float z = ZP ? -16.0f - (float)(t.z[m][i / 4] >> (8 * (i & 3)) & 255u) : -24.0f;
#pragma unroll
            for (int l = 0; l < 4; ++l) acc[g][m][l] = fmaf(s, fmaf(z, sum[i][l], dot[l]), acc[g][m][l]);
          }
        });
      });
    });
  }
  static_for<NB>([&](auto gc) {
    constexpr int g = decltype(gc)::value;
    if (g >= count) return;
#pragma unroll
    for (int m = 0; m < NMAT; ++m) part[((wave * p.batches + g) * NMAT + m) * 64 + lane] = acc[g][m];
  });
  __syncthreads();
  const float* sums = reinterpret_cast<const float*>(part);
  for (int i = threadIdx.x; i < 16 * nrows * count; i += blockDim.x) {
    const int g = i / (16 * nrows), row = (i >> 4) - g * nrows, col = i & 15;
    const int at = (16 * (row >> 2) + col) * 4 + (row & 3);  // lane 16 (row / 4) + col holds it in element row % 4
    float v[NMAT];
#pragma unroll
    for (int m = 0; m < NMAT; ++m) {
      v[m] = 0.f;
      for (int u = 0; u < waves; ++u) v[m] += sums[((u * p.batches + g) * NMAT + m) * 256 + at];
    }
    const int r = 16 * (g0 + g) + col;
    if (r < p.R) store<T, EPI>(p, (long long)rows[row] * p.R + r, v[0], v[NMAT - 1]);
  }
}

// ------------------------------------------------------------------ many rows of x
// A team of WN waves makes 16 MT rows of x x 32 WN weight rows, 32 to each wave (of a gate/up product 16 of both
// matrices), K in blocks of 128: x of a block in LDS in the order the MFMA takes it, two buffers, the next block's x
// and codes in registers meanwhile. KS teams of a work-group take every KS-th block; their sums meet in LDS at the
// end, in the teams' order. A block's 16-byte piece (j, c) of row r lies at place r ^ (4 j + c) of 16: neither the
// writes (16 pieces of a row) nor the reads (16 rows of a piece) meet bank conflicts. Per block of 64 x 128 products
// a wave issues 32 MFMAs for the products, 16 for the sums of x, 64 instructions to decode and 64 per group for
// scales and zero points: about as long on the vector as on the matrix pipe, which is what bounds it (1000 rows of
// [2048, 7168] in groups of 64, 66 us, 446 TFLOP/s; 2000 pairs over 32 experts of 3584 / 1536, gate/up 147 us, 300
// TFLOP/s: partly filled tiles). With the accumulators in AGPRs, which the compiler chooses by itself, moves doubled
// the vector instructions (250 -> 85 us with it all).
template <typename T, int G, bool ZP, int MT, int WN, int KS, Int4Epi EPI, bool WIDE>
__global__ __launch_bounds__(64 * WN * KS) void int4_tile_kernel(Int4Args p)
{
  using N = Num<T>;
  constexpr int XR = 16 * MT, NG = 128 / G, JG = 4 / NG, NT = 2;
  constexpr int kFeatures = (EPI == kInt4Glu ? 16 : 32) * WN, kPass = 4 * WN, kPasses = XR / kPass;
  extern __shared__ i32x4 lds[];  // [KS][2][16 * XR]
  __shared__ int rows[XR];
  const int lane = threadIdx.x & 63, team = __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * WN));
  const int tid = threadIdx.x - team * (64 * WN), wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  i32x4* xs = lds + team * (2 * 16 * XR);
  const int n = lane & 15, c = lane >> 4;
  const int tile = blockIdx.x / p.row_groups + p.tile0, f0 = (blockIdx.x % p.row_groups) * kFeatures;
  int e, nrows;
  if (!find_rows<XR, EPI>(p, tile, rows, e, nrows)) return;
  __syncthreads();
  const int groups = p.K / G, blocks = (p.K + 127) / 128;
  const Decoder dec = decoder<T>();
  const i32x4 ones = {(int)N::kOnes, (int)N::kOnes, (int)N::kOnes, (int)N::kOnes};
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};

  // this wave's two groups of 16 weight rows: neighbours, or the same of both matrices
  Rows w[NT];
  int first[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    first[t] = EPI == kInt4Glu ? f0 + 16 * wave : f0 + 32 * wave + 16 * t;
    const int row = min(first[t], p.R - 1);
    w[t] = weight_rows(p.w[EPI == kInt4Glu ? t : 0], (long long)e * p.R + row, min(16, p.R - row), p.K, groups);
  }
  struct Step {
    i32x4 q[NT];
    uint32_t s[NT][(NG + 1) / 2], z[NT];
  };
  // Rows past R are loaded from past the buffer (zeros). A block behind the last is the last again: a condition on
  // b in the lanes' offsets becomes a branch around each load.
  uint32_t lane_q[NT], lane_s[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const bool in = first[t] + n < p.R;
    lane_q[t] = in ? (uint32_t)n * (p.K / 2) + 16 * c : kOob;
    lane_s[t] = in ? (uint32_t)n * groups : kOob / 2;
  }
  const auto load = [&](int block, Step& k) {
    const int b = min(block, blocks - 1);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      k.q[t] = load_codes(w[t], WIDE || 128 * b + 32 * c < p.K ? lane_q[t] : kOob, 64 * b);
      const uint32_t at = lane_s[t];
      if constexpr (WIDE && NG == 4) {
        const auto v = __builtin_amdgcn_raw_buffer_load_b64(w[t].s, scale_bytes(at), scale_bytes(NG * b), 0);
        k.s[t][0] = v[0], k.s[t][1] = v[1];
        if (ZP) k.z[t] = __builtin_amdgcn_raw_buffer_load_b32(w[t].z, (int)at, NG * b, 0);
      } else if constexpr (WIDE && NG == 2) {
        k.s[t][0] = __builtin_amdgcn_raw_buffer_load_b32(w[t].s, scale_bytes(at), scale_bytes(NG * b), 0);
        if (ZP) k.z[t] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(w[t].z, (int)at, NG * b, 0);
      } else {
#pragma unroll
        for (int i = 0; i < (NG + 1) / 2; ++i) k.s[t][i] = 0;
        k.z[t] = 0;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          const int g = min(b * NG + i, groups - 1);  // past K x is 0
          k.s[t][i / 2] |= (uint32_t)load_scale(w[t], at, g) << (16 * (i & 1));
          if (ZP) k.z[t] |= (uint32_t)load_zero(w[t], at, g) << (8 * i);
        }
      }
    }
  };
  // x: thread t of the team carries piece t % 16 of rows t / 16, + kPass, ..
  const int piece = tid & 15, xrow = tid >> 4;
  const uint16_t* xp[kPasses];
#pragma unroll
  for (int m = 0; m < kPasses; ++m) {
    const int r = rows[xrow + kPass * m];
    xp[m] = static_cast<const uint16_t*>(p.x) + (long long)(EPI == kInt4Store ? r : r / p.x_div) * p.K;
  }
  i32x4 xv[kPasses];
  const auto load_x = [&](int block) {
    const int k = 128 * min(block, blocks - 1) + 8 * piece;
#pragma unroll
    for (int m = 0; m < kPasses; ++m) {
      xv[m] = *reinterpret_cast<const i32x4*>(xp[m] + (WIDE || k < p.K ? k : 0));
      if (!WIDE && k >= p.K) xv[m] = i32x4{0, 0, 0, 0};
    }
  };
  const int a = piece >> 2, d = piece & 3;  // the place of block_k
  const int pj = G == 128 ? d : G == 64 ? 2 * (a >> 1) + (d & 1) : a;
  const int pc = G == 128 ? a : G == 64 ? (a & 1) + 2 * (d >> 1) : d;
  const int place = 4 * pj + pc;
  const auto store_x = [&](int buf) {
#pragma unroll
    for (int m = 0; m < kPasses; ++m) xs[buf * (16 * XR) + place * XR + ((xrow + kPass * m) ^ place)] = pair_up(xv[m]);
  };

  f32x4 acc[NT][MT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[t][m] = zero;
  const auto multiply = [&](int buf, const Step& k) {
    uint32_t q[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int j = 0; j < 4; ++j) q[t][j] = (uint32_t)k.q[t][j];
      one_group<G>(q[t]);
    }
    static_for<NG>([&](auto gc) {
      constexpr int g = decltype(gc)::value;
      f32x4 sum[MT], dot[NT][MT];
#pragma unroll
      for (int j = g * JG; j < (g + 1) * JG; ++j) {
        i32x4 b[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) b[t] = decode8<T>(q[t][j], dec);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const i32x4 x = xs[buf * (16 * XR) + (4 * j + c) * XR + 16 * m + (n ^ (4 * j + c))];
          sum[m] = N::mfma(x, ones, j == g * JG ? zero : sum[m]);
#pragma unroll
          for (int t = 0; t < NT; ++t) dot[t][m] = N::mfma(x, b[t], j == g * JG ? zero : dot[t][m]);
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float s = N::widen((uint16_t)(k.s[t][g / 2] >> (16 * (g & 1))));
        const float z = ZP ? -16.0f - (float)(k.z[t] >> (8 * g) & 255u) : -24.0f;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][m][i] = fmaf(s, fmaf(z, sum[m][i], dot[t][m][i]), acc[t][m][i]);
      }
    });
  };
  Step k0, k1;
  load_x(team);
  load(team, k0);
  store_x(0);
  for (int b = 0; b < blocks; b += 2 * KS) {  // of all teams; a team's is b + team
    __syncthreads();
    load_x(b + team + KS);
    load(b + team + KS, k1);
    __builtin_amdgcn_sched_barrier(0);  // the loads first, not where their registers are free at last
    if (KS == 1 || b + team < blocks) multiply(0, k0);
    store_x(1);
    if (b + KS >= blocks) break;
    __syncthreads();
    load_x(b + team + 2 * KS);
    load(b + team + 2 * KS, k0);
    __builtin_amdgcn_sched_barrier(0);
    if (KS == 1 || b + team + KS < blocks) multiply(1, k1);
    store_x(0);
  }
  if constexpr (KS > 1) {
    f32x4* part = reinterpret_cast<f32x4*>(lds) + wave * (NT * MT * 64) + lane;  // [team - 1][wave][NT][MT][64]
    __syncthreads();
    if (team > 0) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) part[((team - 1) * (WN * NT * MT) + t * MT + m) * 64] = acc[t][m];
    }
    __syncthreads();
    if (team > 0) return;
#pragma unroll
    for (int k = 0; k < KS - 1; ++k)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const f32x4 v = part[(k * (WN * NT * MT) + t * MT + m) * 64];
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][m][i] += v[i];
        }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * m + 4 * c + i;
      if (r >= nrows) continue;
      const long long o = (long long)rows[r] * p.R;
      if (EPI == kInt4Glu) {
        if (first[0] + n < p.R) store<T, EPI>(p, o + first[0] + n, acc[0][m][i], acc[1][m][i]);
      } else {
#pragma unroll
        for (int t = 0; t < NT; ++t)
          if (first[t] + n < p.R) store<T, EPI>(p, o + first[t] + n, acc[t][m][i], 0.f);
      }
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

// items: pairs (kInt4Glu) or tokens (kInt4Token)
template <typename T, int G, bool ZP, int MR, Int4Epi EPI>
hipError_t launch_vec(Int4Args a, int items, hipStream_t s)
{
  constexpr int RB = EPI == kInt4Glu ? kVecRows / 2 : kVecRows;
  int waves = min(8, (a.K + 2047) / 2048);
  if (EPI == kInt4Token) {
    a.team = waves;
    waves *= max(1, min(8 / waves, a.pairs.k));
  }
  // batches of a work-group: as many as leave the chip full once (16 waves a CU)
  const int all = (a.R + RB - 1) / RB;
  const long long full = 256 * 16 / waves;
  a.batches = (int)min((long long)kVecBatches, max(1LL, ((long long)all * items + full - 1) / full));
  a.row_groups = (all + a.batches - 1) / a.batches;
  const int most = max(1, (int)((1u << 22) / a.row_groups));  // a launch's threads are counted in 32 bits
  for (a.tile0 = 0; a.tile0 < items; a.tile0 += most) {
    int4_vec_kernel<T, G, ZP, MR, EPI><<<dim3((unsigned)min(most, items - a.tile0) * a.row_groups), 64 * waves,
                                         sizeof(float) * waves * a.batches * kVecRows * MR, s>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T, int G, bool ZP, Int4Epi EPI>
hipError_t launch_strip(Int4Args a, int tiles, hipStream_t s)
{
  constexpr int NMAT = EPI == kInt4Glu ? 2 : 1;
  const int most_waves = strip_waves(G, EPI, a.K % 256 == 0);
  const int units = (a.K + 255) / 256, rounds = (units + most_waves - 1) / most_waves;
  const int waves = (units + rounds - 1) / rounds;
  const auto kernel = a.K % 256 == 0 ? int4_strip_kernel<T, G, ZP, EPI, true> : int4_strip_kernel<T, G, ZP, EPI, false>;
  const int all = (a.R + 15) / 16;
  const long long full = 256 * 16 / waves;
  a.batches = (int)min((long long)kStripGroups, max(1LL, ((long long)all * tiles + full - 1) / full));
  a.row_groups = (all + a.batches - 1) / a.batches;
  const int most = max(1, (int)((1u << 21) / a.row_groups));
  for (a.tile0 = 0; a.tile0 < tiles; a.tile0 += most) {
    kernel<<<dim3((unsigned)min(most, tiles - a.tile0) * a.row_groups), 64 * waves,
             sizeof(f32x4) * waves * a.batches * NMAT * 64, s>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T, int G, bool ZP, int MT, int WN, int KS, Int4Epi EPI>
hipError_t launch_tile(Int4Args a, int tiles, hipStream_t s)
{
  constexpr int kFeatures = (EPI == kInt4Glu ? 16 : 32) * WN;
  const auto kernel = a.K % 128 == 0 ? int4_tile_kernel<T, G, ZP, MT, WN, KS, EPI, true>
                                     : int4_tile_kernel<T, G, ZP, MT, WN, KS, EPI, false>;
  a.row_groups = (a.R + kFeatures - 1) / kFeatures;
  const int most = max(1, (int)((1u << 21) / a.row_groups));
  for (a.tile0 = 0; a.tile0 < tiles; a.tile0 += most) {
    kernel<<<dim3((unsigned)min(most, tiles - a.tile0) * a.row_groups), 64 * WN * KS,
             sizeof(i32x4) * KS * 2 * 16 * 16 * MT, s>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// The forms by the rows of x that they take at once, and of the tile kernel by its waves. A work-group of the tile
// kernel is one or two waves per SIMD whatever its form, so while there are fewer of them than CUs, smaller ones with
// more teams on K are quicker: [2048, 7168] bf16, groups of 64, us, as 2 x 1 x 8 (MT, WN, KS) / 2 x 2 x 4 / 4 x 2 x 4
// / 4 x 4 x 2 / 4 x 4 x 1: 64 rows 18 / 27 / 36 / 64 / 72, 200 rows 36 / 28 / 37 / 64 / 77, 500 rows 71 / 49 / 40 /
// 66 / 80, 1000 rows 136 / 96 / 82 / 72 / 85, 2000 rows 267 / 187 / 157 / 146 / 128; [7168, 3584]: 32 rows 11 / 14 /
// 19 / 32 / 35, 64 rows 20 / 15 / 20 / 33 / 37, 200 rows 65 / 42 / 40 / 36 / 40, 500 rows 131 / 74 / 77 / 68 / 59.
enum Int4Form : int {
  kVec1, kVec2, kVec4,     // the few-row form
  kStrip,                  // 16 rows
  kTile218, kTile224, kTile222,  // 32 rows
  kTile424, kTile442, kTile441,  // 64 rows
};
constexpr int form_rows(Int4Form f) { return f < kStrip ? 1 << f : f == kStrip ? 16 : f < kTile424 ? 32 : 64; }
constexpr int form_waves(Int4Form f)  // of 32 weight rows side by side
{
  return f == kTile218 ? 1 : f == kTile224 || f == kTile222 || f == kTile424 ? 2 : 4;
}
constexpr int kCus = 256;
bool fills_no_round(Int4Form f, int tiles, int weight_rows)
{
  const int side = 32 * form_waves(f);
  return (long long)tiles * ((weight_rows + side - 1) / side) <= kCus;
}

// items: tiles of form_rows, or the few-row form's pairs or tokens
template <typename T, int G, bool ZP, Int4Epi EPI>
hipError_t launch_form(const Int4Args& a, Int4Form form, int items, hipStream_t s)
{
  if constexpr (EPI == kInt4Store) {
    if (form == kVec2) return launch_vec<T, G, ZP, 2, EPI>(a, items, s);
    if (form == kVec4) return launch_vec<T, G, ZP, 4, EPI>(a, items, s);
  }
  if constexpr (EPI != kInt4Pair) {
    if (form == kVec1) return launch_vec<T, G, ZP, 1, EPI>(a, items, s);
  }
  if constexpr (EPI != kInt4Token) {
    switch (form) {
      case kStrip: return launch_strip<T, G, ZP, EPI>(a, items, s);
      case kTile218: return launch_tile<T, G, ZP, 2, 1, 8, EPI>(a, items, s);
      case kTile224: return launch_tile<T, G, ZP, 2, 2, 4, EPI>(a, items, s);
      case kTile222:
        if constexpr (EPI != kInt4Store) return launch_tile<T, G, ZP, 2, 2, 2, EPI>(a, items, s);
        break;
      case kTile424: return launch_tile<T, G, ZP, 4, 2, 4, EPI>(a, items, s);
      case kTile442: return launch_tile<T, G, ZP, 4, 4, 2, EPI>(a, items, s);
      case kTile441: return launch_tile<T, G, ZP, 4, 4, 1, EPI>(a, items, s);
      default: break;
    }
  }
  return hipErrorInvalidValue;
}
template <typename T, bool ZP, Int4Epi EPI>
hipError_t launch_group(const Int4Args& a, int group, Int4Form form, int items, hipStream_t s)
{
  switch (group) {
    case 32: return launch_form<T, 32, ZP, EPI>(a, form, items, s);
    case 64: return launch_form<T, 64, ZP, EPI>(a, form, items, s);
    default: return launch_form<T, 128, ZP, EPI>(a, form, items, s);
  }
}
template <Int4Epi EPI>
hipError_t launch_typed(const Int4Args& a, int group, int dtype, Int4Form form, int items, hipStream_t s)
{
  const bool zp = a.w[0].z != nullptr;
  if (dtype == 1)
    return zp ? launch_group<__bf16, true, EPI>(a, group, form, items, s)
              : launch_group<__bf16, false, EPI>(a, group, form, items, s);
  return zp ? launch_group<_Float16, true, EPI>(a, group, form, items, s)
            : launch_group<_Float16, false, EPI>(a, group, form, items, s);
}

template <Int4Epi EPI>
hipError_t launch_routed(const Int4Args& a, int group, int dtype, hipStream_t s)
{
  const int P = a.pairs.P, rows = int4_tile_rows(P, a.pairs.E), tiles = a.tiles ? int4_max_tiles(P, a.pairs.E) : P;
  // as many tiles as there are likely to be, of weight rows as wide as a dense product's
  const int likely = P / rows + min(P, a.pairs.E) / 2, wide = EPI == kInt4Glu ? 2 * a.R : a.R;
  Int4Form form = kStrip;
  if (rows == 32) {
    form = fills_no_round(kTile224, likely, wide) ? kTile224 : kTile222;
    if (fills_no_round(kTile218, likely, wide)) form = kTile218;
  } else if (rows == 64) {
    form = fills_no_round(kTile442, likely, wide) ? kTile442 : kTile441;
    if (fills_no_round(kTile424, likely, wide)) form = kTile424;
  }
  return launch_typed<EPI>(a, group, dtype, form, tiles, s);
}

}  // namespace

hipError_t launch_int4_gemm(const Int4Args& a, int group, int dtype, hipStream_t s)
{
  const auto tiles = [&](Int4Form f) { return (a.M + form_rows(f) - 1) / form_rows(f); };
  Int4Form form = kTile441;
  if (a.M <= kVecMost && a.K >= kVecMinK) {
    form = a.M == 1 ? kVec1 : a.M == 2 ? kVec2 : kVec4;
  } else if (a.M <= 16) {
    form = kStrip;
  } else {
    for (Int4Form f : {kTile442, kTile424, kTile224, kTile218})
      if (fills_no_round(f, tiles(f), a.R)) form = f;
  }
  return launch_typed<kInt4Store>(a, group, dtype, form, tiles(form), s);
}

int int4_tile_rows(int P, int E) { return P / E <= 16 ? 16 : P / E <= 32 ? 32 : 64; }

hipError_t launch_int4_route(const Int4Pairs& p, int4* tiles, int* n_tiles, int* order, hipStream_t s)
{
  int4_route_kernel<<<1, 1024, 0, s>>>(p, int4_tile_rows(p.P, p.E), tiles, n_tiles, order);
  return hipGetLastError();
}

// A few tokens' pairs have an expert each, as a rule, and go by themselves in two launches, where one row's products
// read 1 KiB pieces; an expert that several of them name is read again, mostly from the caches. By tokens / by
// experts, us: 8 of 64 experts, 7168 / 2048, 2 tokens 72 / 112, 4 121 / 168, 8 222 / 250, 16 439 / 301; 8 of 128,
// 3584 / 1536, 2 32 / 50, 8 82 / 114, 16 161 / 156; 4 of 32, 2048 / 1024, 2 13 / 22, 8 24 / 31, 16 38 / 36; 2 of 8,
// 4096 / 1024, 2 12 / 20, 8 (two pairs for each expert) 23 / 24, 16 36 / 30.
bool int4_by_token(int N, int k, int E, int D, int F)
{
  return min(D, F) >= kVecMinK && (N == 1 || (N <= 8 && N * k <= 2 * E));
}
hipError_t launch_int4_glu(const Int4Args& a, int group, int dtype, hipStream_t s)
{
  if (a.by_token) return launch_typed<kInt4Glu>(a, group, dtype, kVec1, a.pairs.P, s);
  return launch_routed<kInt4Glu>(a, group, dtype, s);
}
hipError_t launch_int4_pairs(const Int4Args& a, int group, int dtype, hipStream_t s)
{
  return launch_routed<kInt4Pair>(a, group, dtype, s);
}
hipError_t launch_int4_token(const Int4Args& a, int group, int dtype, hipStream_t s)
{
  return launch_typed<kInt4Token>(a, group, dtype, kVec1, a.pairs.P / a.pairs.k, s);
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
