// Products of the dense gated feed-forward block (the latent MoE block's shared expert,
// lazy_lora/trainer/lazy_trainer.py:702-708) in 16-bit elements with fp32 sums:
//   forward    g | u = x Wg^T | x Wu^T (+ deltas), h = GLU(g, u);  y = h Wd^T
//   backward   dh = dy Wd (+ grad_h), dg | du = dh GLU'(g, u);  dx = dg Wg + du Wu
//              dWg = dg^T x, dWu = du^T x, dWd = dy^T h
// One tile kernel does them all: the GLU and its derivative are epilogues on the fp32 sums, so
// neither g | u (except for a backward) nor dh is ever stored for a later pass to read.
#include "../../include/lazylora_mxfp4.h"
#include "mx_dense.h"
#include "mx_device.h"

namespace mx {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <typename T>
struct Elem;
template <>
struct Elem<__bf16> {
  static MX_DEV f32x4 mfma(i32x4 a, i32x4 b, f32x4 c)
  {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  }
};
template <>
struct Elem<_Float16> {
  static MX_DEV f32x4 mfma(i32x4 a, i32x4 b, f32x4 c)
  {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  }
};

// NV consecutive 16-bit elements at element offset i of p, as fp32, and back (one rounding, to nearest even).
template <typename T, int NV>
MX_DEV void load_f(const void* p, long long i, float (&v)[NV])
{
  typedef T tv __attribute__((ext_vector_type(NV)));
  const tv t = *reinterpret_cast<const tv*>(static_cast<const T*>(p) + i);
#pragma unroll
  for (int j = 0; j < NV; ++j) v[j] = (float)t[j];
}
template <typename T, int NV>
MX_DEV void store_f(void* p, long long i, const float (&v)[NV])
{
  typedef T tv __attribute__((ext_vector_type(NV)));
  tv t;
#pragma unroll
  for (int j = 0; j < NV; ++j) t[j] = (T)v[j];
  *reinterpret_cast<tv*>(static_cast<T*>(p) + i) = t;
}

// The epilogues, on NV neighbouring columns n.. of row m.
template <typename T, int NV>
MX_DEV void epi_store(const DenseArgs& p, int m, int n, const float (&v)[NV])
{
  void* o = p.out;
  if (m >= p.split_m) {
    o = p.out2;
    m -= p.split_m;
  }
  store_f<T, NV>(o, m * p.ldo + n, v);
}
template <typename T, int NV>
MX_DEV void epi_glu(const DenseArgs& p, int m, int n, float (&g)[NV], float (&u)[NV])
{
  float t[NV];
  const long long i = (long long)m * p.N + n;
  if (p.add0) {
    load_f<T, NV>(p.add0, i, t);
#pragma unroll
    for (int j = 0; j < NV; ++j) g[j] += t[j];
  }
  if (p.add1) {
    load_f<T, NV>(p.add1, i, t);
#pragma unroll
    for (int j = 0; j < NV; ++j) u[j] += t[j];
  }
  if (p.gu) {
    float* q = p.gu + 2LL * m * p.N + n;
#pragma unroll
    for (int j = 0; j < NV; j += 4) {
      *reinterpret_cast<f32x4*>(q + j) = f32x4{g[j], g[j + 1], g[j + 2], g[j + 3]};
      *reinterpret_cast<f32x4*>(q + p.N + j) = f32x4{u[j], u[j + 1], u[j + 2], u[j + 3]};
    }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) t[j] = glu_fwd(g[j], u[j], p.act);
  store_f<T, NV>(p.out, i, t);
}
template <typename T, int NV>
MX_DEV void epi_dglu(const DenseArgs& p, int m, int n, float (&v)[NV])
{
  if (p.add0) {
    float t[NV];
    load_f<T, NV>(p.add0, (long long)m * p.N + n, t);
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] += t[j];
  }
  const float* q = p.gu + 2LL * m * p.N + n;
  float dg[NV], du[NV];
#pragma unroll
  for (int j = 0; j < NV; j += 4) {
    const f32x4 g = *reinterpret_cast<const f32x4*>(q + j), u = *reinterpret_cast<const f32x4*>(q + p.N + j);
#pragma unroll
    for (int e = 0; e < 4; ++e) glu_bwd(v[j + e], g[e], u[e], p.act, dg[j + e], du[j + e]);
  }
  const long long i = 2LL * m * p.N + n;
  store_f<T, NV>(p.out, i, dg);
  store_f<T, NV>(p.out, i + p.N, du);
}

// ------------------------------------------------------------------ the tile kernel
// A work-group of four waves (2 x 2) makes a tile of 32 FM rows x 32 FN columns, each wave FM x FN
// blocks of v_mfma_f32_16x16x32. The weights' side is the MFMA's first operand, so a lane ends up
// with 4 neighbouring columns of one row.
//
// K goes in steps of 64 through two LDS stages, filled by 16-byte buffer loads that write LDS
// directly. A lane whose element lies past a row, column or K edge gets an offset past its buffer's
// count, so it loads zeros: odd sizes cost no branches in the loop. Stage layouts, 16-byte pieces
// placed so that neither kind of read meets bank conflicts (LDS has 64 banks of 4 bytes):
//  * K-major operand: rows of 128 bytes (64 K terms); piece c of row r at place c ^ key(r). A wave
//    reads fragments of 16 rows x 32 terms with ds_read_b128, lane l row l % 16, terms 8 (l / 16)..+7;
//    key gives the 16 rows of a fragment 8 values per row parity, 256 bytes in all.
//    The columns of a B fragment pair are taken interleaved (columns 8 a + 4 f + j of 32 for fragment
//    f, a = 0..3, j = 0..3), so that a lane holds 8 neighbouring columns of the result.
//  * row-major operand: K terms of 64 FM bytes; 32-byte chunk c of term k at place c ^ g(k). The
//    fragments come from ds_read_b64_tr_b16, which hands lane t of a 16-lane group the 4 terms of
//    column t from 4 terms x 16 columns; the 8 terms that 32 lanes read at once get 8 places.
constexpr int kDenseStep = 64;
constexpr uint32_t kOob = 0x80000000u;  // at or past every buffer's count

MX_DEV int key_a(int r) { return (r >> 1) & 7; }
MX_DEV int key_b(int r) { return ((r >> 1) & 1) | ((r >> 2) & 2) | ((r >> 2) & 4); }
template <int FX>
MX_DEV int key_t(int k)
{
  return FX >= 4 ? (k & 3) + ((k >> 1) & 4) : ((k >> 1) & 1) + ((k >> 2) & 2);
}

MX_DEV i32x4 rsrc_words(const void* base, uint32_t bytes)
{
  const uint64_t b = (uint64_t)(uintptr_t)base;
  return i32x4{(int)__builtin_amdgcn_readfirstlane((uint32_t)b),
               (int)(__builtin_amdgcn_readfirstlane((uint32_t)(b >> 32)) & 0xFFFFu),
               (int)__builtin_amdgcn_readfirstlane(bytes), 0x00020000};
}
// 16 bytes per lane from buffer r at voff (range-checked) + soff to LDS byte address lds + 16 lane. The
// compiler does not know of the copy: the caller waits for it (wait_vm) before the bytes are read.
MX_DEV void dma16_buf(i32x4 r, uint32_t voff, uint32_t soff, uint32_t lds)
{
  asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(voff), "s"(r),
               "s"(soff), "s"(__builtin_amdgcn_readfirstlane(lds))
               : "memory");
}

typedef __attribute__((address_space(3))) const i32x4 lds_i32x4;
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

// One operand's side of the loop: copies into a stage and fragment reads from it. FX 16-row blocks per
// wave, TR: row-major source. ROLE 0: A, 1: B, 2: B of the gate and up matrices (columns of a wave:
// 8 FX of gate, then the same of up).
template <int FX, bool TR, int ROLE>
struct Side {
  static constexpr int kReads = TR ? 2 * FX : FX;  // LDS reads per fragment set
  uint32_t voff[FX];  // this lane's source offset of each of its wave's FX copies per step
  uint32_t raddr[TR ? FX : 2];
  const char* base[2];
  long long step_bytes;  // TR: bytes from one K term to the next
  long long col_bytes;   // TR: bytes from a term's start to this tile's first column
  int kc0;               // K-major: first K term of this lane's piece of copy 0, before the copies' key bits

  // x0: first row (column) of the tile; X: rows (columns) there are
  MX_DEV void init(const void* const* src, long long ld, int x0, int X, int wave, int lane, int wx)
  {
    const int w = wave;
    if constexpr (!TR) {
      const int m = ROLE == 2 ? (w & 1) : 0;
      base[0] = static_cast<const char*>(src[m]) + (long long)x0 * ld * 2;
      base[1] = ROLE == 2 ? base[0] : static_cast<const char*>(src[1]) + (long long)x0 * ld * 2;
#pragma unroll
      for (int j = 0; j < FX; ++j) {
        const int r = 8 * (w * FX + j) + (lane >> 3);
        const int c = (lane & 7) ^ (ROLE == 0 ? key_a(r) : key_b(r));
        const int row = ROLE == 2 ? (w >> 1) * 8 * FX + r % (8 * FX) : r;
        voff[j] = x0 + row < X ? (uint32_t)(row * ld * 2) + c * 16 : kOob;
      }
      const int i = lane & 15, b = lane >> 4;
      const int r = wx * 16 * FX + (ROLE == 0 ? i : 8 * (i >> 2) + (i & 3));
      raddr[0] = r * 128 + ((b ^ (i >> 1)) << 4);
      raddr[1] = raddr[0] ^ 64;
    } else {
      constexpr int kRow = 64 * FX, kLanes = 4 * FX, kPer = 64 / kLanes;
      col_bytes = (long long)x0 * 2;
      step_bytes = ld * 2;
      base[0] = static_cast<const char*>(src[0]) + col_bytes;
      base[1] = static_cast<const char*>(src[1]) + col_bytes;
#pragma unroll
      for (int j = 0; j < FX; ++j) {
        const int k = (w * FX + j) * kPer + lane / kLanes;
        const int pos = lane % kLanes;
        const int c = ((pos >> 1) ^ key_t<FX>(k)) * 2 + (pos & 1);
        voff[j] = x0 + c * 8 < X ? (uint32_t)(k * ld * 2) + c * 16 : kOob;
      }
      const int t = lane & 15, b = lane >> 4;
      const int k = 8 * b + (t >> 2);
#pragma unroll
      for (int f = 0; f < FX; ++f) raddr[f] = k * kRow + (((wx * FX + f) ^ key_t<FX>(k)) << 5) + (t & 3) * 8;
    }
  }

  // Copies j of the step at terms k0 of segment seg (nothing but zeros from k0 >= K) to LDS address lds.
  MX_DEV void copy(int j, int seg, int k0, int K, uint32_t lds, int wave, int lane) const
  {
    const uint32_t dst = lds + (wave * FX + j) * 1024;
    if constexpr (!TR) {
      const int r = 8 * (wave * FX + j) + (lane >> 3);
      const int c = (lane & 7) ^ (ROLE == 0 ? key_a(r) : key_b(r));
      const uint32_t v = k0 + 8 * c < K ? voff[j] : kOob;
      dma16_buf(rsrc_words(seg ? base[1] : base[0], 0x7FFFFFFFu), v, (uint32_t)k0 * 2u, dst);
    } else {
      const int left = K - k0 < kDenseStep ? K - k0 : kDenseStep;
      const uint32_t n = left > 0 ? (uint32_t)(left * step_bytes - col_bytes) : 0u;
      dma16_buf(rsrc_words((seg ? base[1] : base[0]) + (long long)k0 * step_bytes, n), voff[j], 0, dst);
    }
  }

  // Read i (0 .. kReads - 1) of the fragments of half h from the stage at lds.
  MX_DEV void read(int i, int h, uint32_t lds, i32x4 (&f)[FX]) const
  {
    if constexpr (!TR) {
      const uint32_t imm = ROLE == 0 ? i * 2048 : (i >> 1) * 4096 + (i & 1) * 512;
      f[i] = *reinterpret_cast<lds_i32x4*>(lds + raddr[h] + imm);
    } else {
      constexpr int kRow = 64 * FX;
      const int n = i >> 1, jj = i & 1;
      const i16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          reinterpret_cast<lds_i16x4*>(lds + raddr[n] + (32 * h + 4 * jj) * kRow));
      const u32x2 w = __builtin_bit_cast(u32x2, v);
      f[n][2 * jj] = (int)w[0];
      f[n][2 * jj + 1] = (int)w[1];
    }
  }
};

// Every wave's LDS reads of the finished stage and copies into the next one are done.
MX_DEV void stage_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <typename T, int FM, int FN, bool ATR, bool BTR, DenseEpi EPI>
__global__ __launch_bounds__(256) void dense_kernel(DenseArgs p)
{
  constexpr int kStage = (FM + FN) * 4096;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * kStage];
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;

  // Work-groups go to the eight XCDs in turn: each XCD gets one run of neighbouring tiles, walked in
  // columns of up to 8 tile rows, so that its own L2 holds what its tiles share.
  const int total = gridDim.x, xcd = blockIdx.x & 7;
  int id = xcd * (total >> 3) + min(xcd, total & 7) + (blockIdx.x >> 3);
  const int per_group = 8 * p.tiles_n, group = id / per_group;
  const int rows_here = min(8, p.tiles_m - group * 8);
  id -= group * per_group;
  const int m0 = (group * 8 + id % rows_here) * 32 * FM;
  constexpr int kCols = EPI == kDenseGlu ? 16 * FN : 32 * FN;
  const int n0 = id / rows_here * kCols;

  Side<FM, ATR, 0> sa;
  Side<FN, BTR, EPI == kDenseGlu ? 2 : 1> sb;
  sa.init(p.a, p.lda, m0, p.M, wave, lane, wm);
  sb.init(p.b, p.ldb, n0, p.N, wave, lane, wn);

  const int seg_steps = (p.K + kDenseStep - 1) / kDenseStep;
  const int steps = seg_steps * p.nseg;
  constexpr int kCopies = FM + FN;
  auto copy = [&](int i, int step, int stage) {
    const int seg = step >= seg_steps;
    const int k0 = (step - (seg ? seg_steps : 0)) * kDenseStep;
    const uint32_t l = lds + stage * kStage;
    if (i < FM)
      sa.copy(i, seg, k0, p.K, l, wave, lane);
    else
      sb.copy(i - FM, seg, k0, p.K, l + FM * 4096, wave, lane);
  };

  f32x4 acc[FM][FN];
#pragma unroll
  for (int m = 0; m < FM; ++m)
#pragma unroll
    for (int n = 0; n < FN; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (steps > 0) {
    static_for<kCopies>([&](auto i) { copy(i, 0, 0); });
    if (steps > 1) static_for<kCopies>([&](auto i) { copy(i, 1, 1); });
  }
  stage_barrier();
  for (int step = 0; step < steps; ++step) {
    const uint32_t l = lds + (step & 1) * kStage;
    static_for<2>([&](auto h) {
      i32x4 fa[FM], fb[FN];
      static_for<Side<FM, ATR, 0>::kReads>([&](auto i) { sa.read(i, h, l, fa); });
      static_for<decltype(sb)::kReads>([&](auto i) { sb.read(i, h, l + FM * 4096, fb); });
      static_for<FM * FN>([&](auto x) {
        constexpr int m = x % FM, n = x / FM;
        acc[m][n] = Elem<T>::mfma(fb[n], fa[m], acc[m][n]);
      });
    });
    stage_barrier();
    if (step + 2 < steps) static_for<kCopies>([&](auto i) { copy(i, step + 2, step & 1); });
  }

  const int row0 = m0 + wm * 16 * FM + (lane & 15), q = lane >> 4;
#pragma unroll
  for (int m = 0; m < FM; ++m) {
    const int row = row0 + 16 * m;
    if (row >= p.M) continue;
    if constexpr (EPI == kDenseGlu) {
#pragma unroll
      for (int n = 0; n < FN / 2; n += 2) {
        const int col = n0 + wn * 8 * FN + 16 * n + 8 * q;
        if (col >= p.N) continue;
        float g[8], u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          g[j] = acc[m][n + j / 4][j % 4];
          u[j] = acc[m][n + FN / 2 + j / 4][j % 4];
        }
        epi_glu<T, 8>(p, row, col, g, u);
      }
    } else if constexpr (!BTR) {
#pragma unroll
      for (int n = 0; n < FN; n += 2) {
        const int col = n0 + wn * 16 * FN + 16 * n + 8 * q;
        if (col >= p.N) continue;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = acc[m][n + j / 4][j % 4];
        epi_store<T, 8>(p, row, col, v);
      }
    } else {
#pragma unroll
      for (int n = 0; n < FN; ++n) {
        const int col = n0 + wn * 16 * FN + 16 * n + 4 * q;
        if (col >= p.N) continue;
        float v[4] = {acc[m][n][0], acc[m][n][1], acc[m][n][2], acc[m][n][3]};
        if constexpr (EPI == kDenseDGlu)
          epi_dglu<T, 4>(p, row, col, v);
        else
          epi_store<T, 4>(p, row, col, v);
      }
    }
  }
}

template <typename T, int FM, int FN, bool ATR, bool BTR, DenseEpi EPI>
hipError_t launch_tiles(DenseArgs a, hipStream_t s)
{
  const int cols = EPI == kDenseGlu ? 16 * FN : 32 * FN;
  a.tiles_m = (a.M + 32 * FM - 1) / (32 * FM);
  a.tiles_n = (a.N + cols - 1) / cols;
  hipLaunchKernelGGL((dense_kernel<T, FM, FN, ATR, BTR, EPI>), dim3((unsigned)(a.tiles_m * a.tiles_n)), dim3(256), 0, s,
                     a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_dense_forward(const DenseArgs& a, int dtype, DenseEpi epi, hipStream_t s)
{
  if (a.M <= 0 || a.N <= 0) return hipSuccess;
  const bool bf = dtype == MXFP4_BF16;
  if (epi == kDenseGlu)
    return bf ? launch_tiles<__bf16, 4, 4, false, false, kDenseGlu>(a, s)
              : launch_tiles<_Float16, 4, 4, false, false, kDenseGlu>(a, s);
  return bf ? launch_tiles<__bf16, 4, 4, false, false, kDenseStore>(a, s)
            : launch_tiles<_Float16, 4, 4, false, false, kDenseStore>(a, s);
}

hipError_t launch_dense_dgrad(const DenseArgs& a, int dtype, DenseEpi epi, hipStream_t s)
{
  if (a.M <= 0 || a.N <= 0) return hipSuccess;
  const bool bf = dtype == MXFP4_BF16;
  if (epi == kDenseDGlu)
    return bf ? launch_tiles<__bf16, 4, 4, false, true, kDenseDGlu>(a, s)
              : launch_tiles<_Float16, 4, 4, false, true, kDenseDGlu>(a, s);
  return bf ? launch_tiles<__bf16, 4, 4, false, true, kDenseStore>(a, s)
            : launch_tiles<_Float16, 4, 4, false, true, kDenseStore>(a, s);
}

hipError_t launch_dense_wgrad(const DenseArgs& a, int dtype, hipStream_t s)
{
  if (a.M <= 0 || a.N <= 0) return hipSuccess;
  return dtype == MXFP4_BF16 ? launch_tiles<__bf16, 4, 4, true, true, kDenseStore>(a, s)
                             : launch_tiles<_Float16, 4, 4, true, true, kDenseStore>(a, s);
}

}  // namespace mx
