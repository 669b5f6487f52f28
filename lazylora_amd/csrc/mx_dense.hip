// Products of the dense gated feed-forward block (the latent MoE block's shared expert,
// lazy_lora/trainer/lazy_trainer.py:702-708) in 16-bit elements with fp32 sums:
//   forward    g | u = x Wg^T | x Wu^T (+ deltas), h = GLU(g, u);  y = h Wd^T
//   backward   dh = dy Wd (+ grad_h), dg | du = dh GLU'(g, u);  dx = dg Wg + du Wu
//              dWg = dg^T x, dWu = du^T x, dWd = dy^T h
// One tile kernel does them all: the GLU and its derivative are epilogues on the fp32 sums, so
// neither g | u (except for a backward) nor dh is ever stored for a later pass to read.
#include <algorithm>

#include "../../include/lazylora_mxfp4.h"
#include "mx_dense.h"
#include "mx_device.h"

namespace mx {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <typename T>
struct Elem;
template <>
struct Elem<__bf16> {
  static MX_DEV f32x4 mfma16(i32x4 a, i32x4 b, f32x4 c)
  {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  }
  static MX_DEV f32x16 mfma(i32x4 a, i32x4 b, f32x16 c)
  {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  }
};
template <>
struct Elem<_Float16> {
  static MX_DEV f32x4 mfma16(i32x4 a, i32x4 b, f32x4 c)
  {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  }
  static MX_DEV f32x16 mfma(i32x4 a, i32x4 b, f32x16 c)
  {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
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

MX_DEV void store_sums(float* p, const float (&v)[8])
{
  *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
  *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
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
// A work-group of WM x WN waves makes a tile of 32 FM WM rows x 32 FN WN columns, each wave FM x FN
// blocks of v_mfma_f32_32x32x16 (twice the products per operand byte read of the 16 x 16 form: less power,
// and half the instructions between which reads and copies have to fit). The weights' side is the
// MFMA's first operand, so a lane ends up with runs of 4 neighbouring columns of one row.
//
// K goes in steps of 64 through NS LDS stages, filled by 16-byte buffer loads that write LDS
// directly. A lane whose element lies past a row, column or K edge gets an offset past its buffer's
// count, so it loads zeros: odd sizes cost no branches in the loop. Stage layouts, 16-byte pieces
// placed so that neither kind of read meets bank conflicts (LDS has 64 banks of 4 bytes):
//  * K-major operand: rows of 128 bytes (64 K terms); piece c of row r at place c ^ key_k(r). A wave
//    reads fragments of 32 rows x 16 terms with ds_read_b128, lane l row l % 32, terms 8 (l / 32)..+7;
//    the key takes 8 values over the 8 rows of each parity, so 16 rows' pieces fill 256 bytes.
//  * row-major operand: K terms of 64 bytes per block; 32-byte chunk c of term k at place c ^ key_t(k).
//    The fragments come from ds_read_b64_tr_b16, which hands lane t of a 16-lane group the 4 terms of
//    column t from 4 terms x 16 columns; 32 lanes read 4 terms x 64 bytes at once, which the key puts
//    side by side.
constexpr int kDenseStep = 64;
constexpr uint32_t kOob = 0x80000000u;  // at or past every buffer's count

MX_DEV int key_k(int r) { return (r >> 1) & 7; }
template <int BLOCKS>
MX_DEV int key_t(int k)
{
  return BLOCKS >= 4 ? (k & 3) << 1 : k & 2;
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
typedef __attribute__((address_space(3))) const f32x4 lds_f32x4;
typedef __attribute__((address_space(3))) f32x4 lds_f32x4_w;

// One operand's side of the loop: copies into a stage and fragment reads from it. WX waves of FX 32-row
// blocks each share the operand among NW waves, TR: row-major source, GLU: B of the gate and up
// matrices (columns of a wave: 16 FX of gate, then the same of up).
template <int FX, int WX, int NW, bool TR, bool GLU>
struct Side {
  static constexpr int kBlocks = FX * WX;
  static constexpr int kCopies = 4 * kBlocks / NW;     // 1 KiB copies of a wave per step
  static constexpr int kReads = (TR ? 2 : 1) * 2 * FX;  // LDS reads of a half step's fragments
  static_assert(4 * kBlocks % NW == 0 && kCopies > 0, "the waves share the copies evenly");
  uint32_t voff[kCopies];  // this lane's source offset of each of its wave's copies
  uint32_t raddr[TR ? FX : 1];
  const char* base[2];
  long long step_bytes;  // TR: bytes from one K term to the next
  long long col_bytes;   // TR: bytes from a term's start to this tile's first column

  // x0: first row (column) of the tile; X: rows (columns) there are
  MX_DEV void init(const void* const* src, long long ld, int x0, int X, int wave, int lane, int wx)
  {
    if constexpr (!TR) {
      base[0] = static_cast<const char*>(src[0]) + (long long)x0 * ld * 2;
      base[1] = static_cast<const char*>(src[1]) + (long long)x0 * ld * 2;
#pragma unroll
      for (int j = 0; j < kCopies; ++j) {
        const int r = 8 * (wave * kCopies + j) + (lane >> 3);
        const int c = (lane & 7) ^ key_k(r);
        const int row = GLU ? r / (32 * FX) * 16 * FX + r % (16 * FX) : r;
        voff[j] = x0 + row < X ? (uint32_t)(row * ld * 2) + c * 16 : kOob;
      }
      const int i = lane & 31;
      raddr[0] = (wx * 32 * FX + i) * 128 + (((lane >> 5) ^ key_k(i)) << 4);
    } else {
      constexpr int kRow = 64 * kBlocks, kLanes = 4 * kBlocks, kPer = 64 / kLanes;
      col_bytes = (long long)x0 * 2;
      step_bytes = ld * 2;
      base[0] = static_cast<const char*>(src[0]) + col_bytes;
      base[1] = static_cast<const char*>(src[1]) + col_bytes;
#pragma unroll
      for (int j = 0; j < kCopies; ++j) {
        const int k = (wave * kCopies + j) * kPer + lane / kLanes;
        const int pos = lane % kLanes;
        const int c = ((pos >> 1) ^ key_t<kBlocks>(k)) * 2 + (pos & 1);
        voff[j] = x0 + c * 8 < X ? (uint32_t)(k * ld * 2) + c * 16 : kOob;
      }
      const int t = lane & 15;
      const int k = 8 * (lane >> 5) + (t >> 2);
#pragma unroll
      for (int f = 0; f < FX; ++f)
        raddr[f] = k * kRow + (((2 * (wx * FX + f) + ((lane >> 4) & 1)) ^ key_t<kBlocks>(k)) << 5) + (t & 3) * 8;
    }
  }

  // Copies j of the step at terms k0 of segment seg (nothing but zeros from k0 >= K) to LDS address lds.
  MX_DEV void copy(int j, int seg, int k0, int K, uint32_t lds, int wave, int lane) const
  {
    const uint32_t dst = lds + (wave * kCopies + j) * 1024;
    if constexpr (!TR) {
      const int q = wave * kCopies + j;
      const int c = (lane & 7) ^ key_k(8 * q + (lane >> 3));
      const uint32_t v = k0 + 8 * c < K ? voff[j] : kOob;
      dma16_buf(rsrc_words((GLU ? (q / (2 * FX)) & 1 : seg) ? base[1] : base[0], 0x7FFFFFFFu), v, (uint32_t)k0 * 2u,
                dst);
    } else {
      const int left = K - k0 < kDenseStep ? K - k0 : kDenseStep;
      const uint32_t n = left > 0 ? (uint32_t)(left * step_bytes - col_bytes) : 0u;
      dma16_buf(rsrc_words((seg ? base[1] : base[0]) + (long long)k0 * step_bytes, n), voff[j], 0, dst);
    }
  }

  // Read i (0 .. kReads - 1) of the fragments of half h (terms 32 h..: two slices of 16) from the stage at lds.
  template <int I, int H>
  MX_DEV void read(uint32_t lds, i32x4 (&f)[2][FX]) const
  {
    constexpr int S = I / (kReads / 2), J = I % (kReads / 2);
    if constexpr (!TR) {
      f[S][J] = *reinterpret_cast<lds_i32x4*>(lds + (raddr[0] ^ (64 * H + 32 * S)) + J * 4096);
    } else {
      constexpr int kRow = 64 * kBlocks, N = J / 2, Q = J % 2;
      const i16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          reinterpret_cast<lds_i16x4*>(lds + raddr[N] + (32 * H + 16 * S + 4 * Q) * kRow));
      const u32x2 w = __builtin_bit_cast(u32x2, v);
      f[S][N][2 * Q] = (int)w[0];
      f[S][N][2 * Q + 1] = (int)w[1];
    }
  }
};

// Every wave's LDS reads so far, and all but its last N copies, are done.
template <int N>
MX_DEV void stage_barrier()
{
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

template <typename T, int WM, int WN, int FM, int FN, int NS, bool ATR, bool BTR, DenseEpi EPI>
__global__ __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(WM * WN / 4))) void dense_kernel(DenseArgs p)
{
  constexpr int NW = WM * WN;
  constexpr int kStageA = FM * WM * 4096, kStage = kStageA + FN * WN * 4096;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[NS * kStage];
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;

  // Work-groups go to the eight XCDs in turn: each XCD gets one run of neighbouring tiles of one run of K,
  // walked in columns of up to 8 tile rows, so that its own L2 holds what its tiles share.
  const int total = gridDim.x, xcd = blockIdx.x & 7;
  int id = xcd * (total >> 3) + min(xcd, total & 7) + (blockIdx.x >> 3);
  const int tiles = p.tiles_m * p.tiles_n, split = id / tiles;
  id -= split * tiles;
  const int per_group = 8 * p.tiles_n, group = id / per_group;
  const int rows_here = min(8, p.tiles_m - group * 8);
  id -= group * per_group;
  const int m0 = (group * 8 + id % rows_here) * 32 * FM * WM;
  constexpr int kCols = (EPI == kDenseGlu ? 16 : 32) * FN * WN;
  const int n0 = id / rows_here * kCols;

  Side<FM, WM, NW, ATR, false> sa;
  Side<FN, WN, NW, BTR, EPI == kDenseGlu> sb;
  sa.init(p.a, p.lda, m0, p.M, wave, lane, wm);
  sb.init(p.b, p.ldb, n0, p.N, wave, lane, wn);

  const int seg_steps = (p.K + kDenseStep - 1) / kDenseStep;
  const int first = split * p.run, steps = min(seg_steps * p.nseg, first + p.run);
  constexpr int kCopiesA = decltype(sa)::kCopies, kCopies = kCopiesA + decltype(sb)::kCopies;
  auto copy = [&](int i, int step, int stage) {
    const int seg = step >= seg_steps;
    const int k0 = step < steps ? (step - (seg ? seg_steps : 0)) * kDenseStep : p.K;  // past the last: zeros
    const uint32_t l = lds + stage * kStage;
    if (i < kCopiesA)
      sa.copy(i, seg, k0, p.K, l, wave, lane);
    else
      sb.copy(i - kCopiesA, seg, k0, p.K, l + kStageA, wave, lane);
  };

  f32x16 acc[FM][FN];
#pragma unroll
  for (int m = 0; m < FM; ++m)
#pragma unroll
    for (int n = 0; n < FN; ++n)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[m][n][j] = 0.f;

  // Fragments of the half being multiplied and of the next one, which are read while the MFMAs of a half
  // run; after the barrier in the second half of a step nobody reads its stage any more and the next step's copies have
  // landed, and the MFMAs behind it also carry the copies of step + NS into the stage. The barrier stands
  // behind the first kWait MFMAs of the second half, which run while the waves wait for each other.
  i32x4 fa[2][2][FM], fb[2][2][FN];  // [half][slice][block]
  constexpr int kMfma = 2 * FM * FN, kWait = kMfma / 4;
  constexpr int kReadsA = decltype(sa)::kReads, kReads = kReadsA + decltype(sb)::kReads;
  auto read = [&](auto i, auto h, uint32_t l) {
    if constexpr (i < kReadsA)
      sa.template read<i, h>(l, fa[h]);
    else
      sb.template read<i - kReadsA, h>(l + kStageA, fb[h]);
  };
  static_for<NS>([&](auto k) { static_for<kCopies>([&](auto i) { copy(i, first + k, k); }); });
  stage_barrier<(NS - 1) * kCopies>();
  static_for<kReads>([&](auto i) { read(i, std::integral_constant<int, 0>{}, lds); });
  int stage = 0;
  for (int step = first; step < steps; ++step) {
    const int next = stage + 1 < NS ? stage + 1 : 0;
    const uint32_t l0 = lds + stage * kStage, l1 = lds + next * kStage;
    static_for<2>([&](auto h) {
      constexpr int H = h;
      // LDS reads and copies one by one behind the MFMAs: issued in runs, they left the matrix cores idle
      static_for<kMfma>([&](auto x) {
        constexpr int sl = x / (FM * FN), m = x % FM, n = x / FM % FN;
        acc[m][n] = Elem<T>::mfma(fb[H][sl][n], fa[H][sl][m], acc[m][n]);
        constexpr int open = H == 0 ? 0 : kWait;  // reads and copies follow the MFMAs from here on
        if constexpr (H == 1 && x == kWait - 1) stage_barrier<(NS - 2) * kCopies>();
        static_for<kReads>([&](auto i) {
          if constexpr (open + i * (kMfma - open) / kReads == x)
            read(i, std::integral_constant<int, 1 - H>{}, H == 0 ? l0 : l1);
        });
        if constexpr (H == 1)
          static_for<kCopies>([&](auto i) {
            if constexpr (open + i * (kMfma - open) / kCopies == x) copy(i, step + NS, stage);
          });
        __builtin_amdgcn_sched_barrier(0);
      });
    });
    stage = next;
  }
  stage_barrier<0>();  // the stages are free for the epilogue

  // The sums go through LDS, each wave its own FMP x FN blocks at a time, so that a lane takes 8
  // neighbouring columns of a row (whole lines per row, and one short loop whatever the epilogue costs).
  // fp32 rows of 32 FN columns; 16-byte piece c of row r at place c ^ key: the rows that a write
  // instruction touches at once fall into different banks.
  constexpr int kFit = NS * kStage / (FN * 4096 * NW);  // row blocks of a wave that fit
  constexpr int FMP = kFit >= FM ? FM : kFit >= FM / 2 ? FM / 2 : FM / 4;
  static_assert(FMP > 0 && FMP * FN * 4096 * NW <= NS * kStage, "a wave's sums do not fit its part of the stages");
  const uint32_t own = lds + wave * FMP * FN * 4096;
  auto place = [&](int r, int c) {
    return own + r * 128 * FN + ((c ^ (FN >= 2 ? r & 15 : (r >> 1) & 7)) << 4);
  };
  auto eight = [&](int r, int c, float (&v)[8]) {
    const f32x4 a = *reinterpret_cast<lds_f32x4*>(place(r, c)), b = *reinterpret_cast<lds_f32x4*>(place(r, c + 1));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = a[j];
      v[4 + j] = b[j];
    }
  };
  constexpr int kCol8 = EPI == kDenseGlu ? 2 * FN : 4 * FN;  // groups of 8 result columns per wave
  const int c8 = lane % kCol8;
  const int col = n0 + wn * 8 * kCol8 + 8 * c8;
  static_for<FM / FMP>([&](auto part) {
    static_for<FMP>([&](auto m) {
      static_for<FN * 4>([&](auto v) {
        constexpr int n = v / 4, q = v % 4;
        const f32x16& a = acc[part * FMP + m][n];
        *reinterpret_cast<lds_f32x4_w*>(place(32 * m + (lane & 31), 8 * n + 2 * q + (lane >> 5))) =
            f32x4{a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
      });
    });
    wave_lds_fence();
    const int row0 = m0 + wm * 32 * FM + part * 32 * FMP;
#pragma unroll 1
    for (int r = lane / kCol8; r < 32 * FMP; r += 64 / kCol8) {
      const int row = row0 + r;
      if (row >= p.M) break;
      if (col >= p.N) continue;
      float v[8];
      eight(r, 2 * c8, v);
      if constexpr (EPI == kDenseGlu) {
        float u[8];
        eight(r, 4 * FN + 2 * c8, u);
        if (p.partial) {
          float* q = p.partial + 2 * ((long long)split * p.M + row) * p.N + col;
          store_sums(q, v);
          store_sums(q + p.N, u);
          continue;
        }
        epi_glu<T, 8>(p, row, col, v, u);
      } else if (p.partial) {
        store_sums(p.partial + ((long long)split * p.M + row) * p.N + col, v);
      } else {
        if constexpr (EPI == kDenseDGlu)
          epi_dglu<T, 8>(p, row, col, v);
        else
          epi_store<T, 8>(p, row, col, v);
      }
    }
    wave_lds_fence();
  });
}

// The runs' partial sums, added in order, and the epilogue: a thread per 8 columns of a row, one wave per
// work-group, so that the few threads of few rows spread over the CUs.
template <typename T, DenseEpi EPI>
__global__ __launch_bounds__(64) void dense_finish_kernel(DenseArgs p)
{
  const int per_row = p.N / 8;
  const long long i = (long long)blockIdx.x * 64 + threadIdx.x;
  if (i >= (long long)p.M * per_row) return;
  const int row = (int)(i / per_row), col = (int)(i % per_row) * 8;
  float v[8] = {}, u[8] = {};
  constexpr int W = EPI == kDenseGlu ? 2 : 1;
  const long long stride = (long long)p.M * p.N * W;
  const float* q = p.partial + (long long)row * p.N * W + col;
  // eight runs' loads in flight, whatever the count (the last run's again past it, not added): with few rows
  // the loop is its loads' latency and nothing else
  constexpr int kAhead = 8;
  for (int k = 0; k < p.splits; k += kAhead) {
    f32x4 in[kAhead][2 * W];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const float* r = q + min(k + j, p.splits - 1) * stride;
#pragma unroll
      for (int e = 0; e < 2 * W; ++e) in[j][e] = *reinterpret_cast<const f32x4*>(r + (e >> 1) * p.N + 4 * (e & 1));
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const bool add = k + j < p.splits;  // no branch: the loads would sink into it, one behind the other
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] += add ? in[j][0][e] : 0.f;
        v[4 + e] += add ? in[j][1][e] : 0.f;
        if constexpr (EPI == kDenseGlu) {
          u[e] += add ? in[j][2][e] : 0.f;
          u[4 + e] += add ? in[j][3][e] : 0.f;
        }
      }
    }
  }
  if constexpr (EPI == kDenseGlu)
    epi_glu<T, 8>(p, row, col, v, u);
  else if constexpr (EPI == kDenseDGlu)
    epi_dglu<T, 8>(p, row, col, v);
  else
    epi_store<T, 8>(p, row, col, v);
}

// ------------------------------------------------------------------ few rows
// The forward products of up to 64 rows: bound by reading the weights once, so a work-group takes only
// 16 WB weight rows (kDenseGlu: half of them gate, the same of up), which gives many CUs some, and its eight
// waves cut K among them: each streams its run of the rows straight into the registers of
// v_mfma_f32_16x16x32 (lane l: weight row l % 16, terms 8 (l / 16)..+7 of 32; MB blocks of 16 rows of x the
// same way, from L2; the next steps' loads in flight), and the eight sums meet in LDS in a fixed order. No
// partial sums in memory, no second launch. Rows past the last (of x or of the weights) read the last one's
// bytes and are not stored. A CU takes about 36 bytes per ns this way, its work-group's weight rows and all
// of x: two blocks of weight rows (x read half as often) pay where one would mean a second round.
// One row, D = 7168, F = 2048: gate/up 13 us (58.7 MB, 4.5 TB/s), where 64 x 128 tiles with eight runs of K
// and their join take 18. 37 rows, D = 3584, F = 1536, down: 8 us against 12; gate/up 16 against 14.
constexpr int kFewRows = 64;

template <typename T, int WB, int MB, DenseEpi EPI>
__global__ __launch_bounds__(512) void dense_few_kernel(DenseArgs p)
{
  constexpr int NW = 8, U = WB + MB <= 3 ? 8 : 4;  // waves; steps of 32 terms in flight, twice
  constexpr int kRows = 16 * MB, kWide = 16 * WB;
  __shared__ __attribute__((aligned(16))) float sums[NW][kRows][kWide];
  __shared__ __attribute__((aligned(16))) float total[kRows][kWide];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, q = lane >> 4;
  constexpr int kCols = EPI == kDenseGlu ? kWide / 2 : kWide;
  const int n0 = blockIdx.x * kCols;
  const T* wp[WB];
  const T* xp[MB];
#pragma unroll
  for (int b = 0; b < WB; ++b) {
    const int r = 16 * b + i, up = EPI == kDenseGlu && r >= kCols;
    wp[b] = static_cast<const T*>(p.b[up]) + min(n0 + (up ? r - kCols : r), p.N - 1) * p.ldb + 8 * q;
  }
#pragma unroll
  for (int b = 0; b < MB; ++b) xp[b] = static_cast<const T*>(p.a[0]) + min(16 * b + i, p.M - 1) * p.lda + 8 * q;

  f32x4 acc[MB][WB];
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int b = 0; b < WB; ++b) acc[m][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  // whole steps [s, end) of this wave; the partial step at the end of K is the last wave's extra one
  const int whole = p.K / 32, per = (whole + NW - 1) / NW;
  int s = min(wave * per, whole);
  const int end = min(s + per, whole);
  i32x4 w[2][U][WB], x[2][U][MB];
  const auto request = [&](auto h, int first) {
    static_for<U>([&](auto u) {
      const int k = min(first + u, end - 1) * 32;  // past the run: its last step again, not used
      static_for<WB>([&](auto b) { w[h][u][b] = *reinterpret_cast<const i32x4*>(wp[b] + k); });
      static_for<MB>([&](auto b) { x[h][u][b] = *reinterpret_cast<const i32x4*>(xp[b] + k); });
    });
  };
  const auto multiply = [&](auto h, int n) {
    static_for<U>([&](auto u) {
      if (u < n)
        static_for<MB>([&](auto m) {
          static_for<WB>([&](auto b) { acc[m][b] = Elem<T>::mfma16(w[h][u][b], x[h][u][m], acc[m][b]); });
        });
    });
  };
  using Zero = std::integral_constant<int, 0>;
  using One = std::integral_constant<int, 1>;
  if (s < end) {
    request(Zero{}, s);
    for (; s < end; s += 2 * U) {
      if (s + U < end) request(One{}, s + U);
      multiply(Zero{}, end - s);
      if (s + 2 * U < end) request(Zero{}, s + 2 * U);
      if (s + U < end) multiply(One{}, end - s - U);
    }
  }
  if (wave == NW - 1 && whole * 32 < p.K) {
    const bool in = whole * 32 + 8 * q < p.K;
    const int k = in ? whole * 32 : -8 * q;  // a lane past K: terms 0.., taken as zeros
    const i32x4 zero = {0, 0, 0, 0};
    i32x4 wt[WB];
    static_for<WB>([&](auto b) {
      const i32x4 v = *reinterpret_cast<const i32x4*>(wp[b] + k);
      wt[b] = in ? v : zero;
    });
    static_for<MB>([&](auto m) {
      const i32x4 v = *reinterpret_cast<const i32x4*>(xp[m] + k);
      static_for<WB>([&](auto b) { acc[m][b] = Elem<T>::mfma16(wt[b], in ? v : zero, acc[m][b]); });
    });
  }
  static_for<MB>([&](auto m) {
    static_for<WB>([&](auto b) { *reinterpret_cast<f32x4*>(&sums[wave][16 * m + i][16 * b + 4 * q]) = acc[m][b]; });
  });
  __syncthreads();
  for (int e = threadIdx.x; e < kRows * kWide; e += 512) {
    float t = 0.f;
#pragma unroll
    for (int v = 0; v < NW; ++v) t += (&sums[v][0][0])[e];
    (&total[0][0])[e] = t;
  }
  __syncthreads();
  constexpr int kGroups = kCols / 8;  // of 8 columns
  const int row = threadIdx.x / kGroups, c = threadIdx.x % kGroups * 8;
  if (row >= p.M || n0 + c >= p.N) return;
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = total[row][c + j];
  if constexpr (EPI == kDenseGlu) {
    float u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = total[row][kCols + c + j];
    epi_glu<T, 8>(p, row, n0 + c, v, u);
  } else {
    epi_store<T, 8>(p, row, n0 + c, v);
  }
}

template <typename T, int WB, DenseEpi EPI>
hipError_t launch_few(const DenseArgs& a, hipStream_t s)
{
  const int cols = 16 * WB / (EPI == kDenseGlu ? 2 : 1);
  const dim3 grid((unsigned)((a.N + cols - 1) / cols)), block(512);
  if (a.M <= 16)
    hipLaunchKernelGGL((dense_few_kernel<T, WB, 1, EPI>), grid, block, 0, s, a);
  else if (a.M <= 32)
    hipLaunchKernelGGL((dense_few_kernel<T, WB, 2, EPI>), grid, block, 0, s, a);
  else if (a.M <= 48)
    hipLaunchKernelGGL((dense_few_kernel<T, WB, 3, EPI>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((dense_few_kernel<T, WB, 4, EPI>), grid, block, 0, s, a);
  return hipGetLastError();
}

// The tiles there are (kDenseGlu: half the columns are columns of h), one work-group per CU each, and what
// they were measured to take (us; K = 7168, forward product, normally distributed operands): a step of 64
// terms while few work-groups run, the same with every CU busy (the chip then lowers its clock; between the
// two about in proportion), and a tile's start and epilogue.
struct Tile {
  int rows, cols;
  float step, busy, ends;
  float row_major;  // the same step with row-major operands: twice the LDS reads, and short runs of memory
};
constexpr Tile kTiles[] = {{256, 256, 1.13f, 1.80f, 8.f, 1.15f}, {128, 256, 0.66f, 1.02f, 7.f, 1.15f},
                           {128, 128, 0.50f, 0.57f, 6.f, 1.3f}, {64, 128, 0.42f, 0.42f, 5.f, 1.5f}};
constexpr int kNTiles = sizeof(kTiles) / sizeof(kTiles[0]);
constexpr int kCUs = 256;
constexpr int kMaxSplits = 16;

constexpr int kFewOne = -1, kFewTwo = -2;  // dense_few_kernel with one and two blocks of weight rows

struct Plan {
  int tile, splits, run;
  float us;
};

// The tile and the number of runs of K that the measurements above promise the shortest time for. Fewer tiles
// than CUs leave CUs idle, which smaller tiles or more runs mend, each at its price: smaller tiles read their
// operands more often (a step of four 128 x 128 tiles takes 1.2 x that of one 256 x 256), runs write and
// read their sums (5.3 TB/s, and 4 us for the launch). 1000 rows, D = 7168, F = 2048: gate/up 64 us with 128 x 128 tiles
// in one run, 129 with 256 x 256 in one, 73 in four.
Plan plan_dense(DenseShape shape, DenseEpi epi, int M, int N, int K, int nseg)
{
  const long long cols = epi == kDenseGlu ? 2LL * N : N;
  const int steps = (K + kDenseStep - 1) / kDenseStep * nseg;
  const float stream = ((float)cols + M) * K * nseg * 2.f / 4.5e6f;  // the operands once from HBM
  Plan best = {0, 1, steps, 1e30f};
  if (shape == kDenseForward && M <= kFewRows)
    for (int blocks = 1; blocks <= 2; ++blocks) {
      const long long groups = (cols + 16 * blocks - 1) / (16 * blocks);
      const float cu = 3.f + (float)((groups + kCUs - 1) / kCUs) * (16 * blocks + M) * K / 18e3f;
      const float us = std::max(stream + 2.f, cu) + 0.1f * cu;
      if (us < best.us) best = {blocks == 1 ? kFewOne : kFewTwo, 1, steps, us};
    }
  for (int t = 0; t < kNTiles; ++t) {
    const Tile& tile = kTiles[t];
    const float slow = shape == kDenseForward ? 1.f : tile.row_major;
    const long long tiles = ((M + tile.rows - 1LL) / tile.rows) * ((cols + tile.cols - 1) / tile.cols);
    for (int want = 1; want <= kMaxSplits && want <= std::max(steps, 1); ++want) {
      const int run = (steps + want - 1) / want, splits = run > 0 ? (steps + run - 1) / run : 1;
      if (splits != want) continue;
      const long long full = tiles * splits / kCUs, rest = tiles * splits % kCUs;
      float us = full * (run * tile.busy * slow + tile.ends);
      if (rest) us += run * (tile.step + (tile.busy - tile.step) * rest / kCUs) * slow + tile.ends;
      us = std::max(us, stream);
      if (splits > 1) us += 4.f + (float)M * cols * splits * 1.5e-6f;
      if (us < best.us) best = {t, splits, run, us};
      if (tiles * splits >= 4 * kCUs) break;
    }
  }
  return best;
}

template <typename T, int WM, int WN, int FM, int FN, int NS, DenseShape SH, DenseEpi EPI>
void launch_tiles(const DenseArgs& a, int splits, hipStream_t s)
{
  hipLaunchKernelGGL((dense_kernel<T, WM, WN, FM, FN, NS, SH == kDenseWgrad, SH != kDenseForward, EPI>),
                     dim3((unsigned)(a.tiles_m * a.tiles_n * splits)), dim3(64 * WM * WN), 0, s, a);
}

// A product whose last tile row is nearly empty takes its whole tile rows first and the rows behind them by
// themselves, where the two are expected to be quicker (4099 rows, gate/up: 4096 in one round of 256 x 256
// tiles and 3 rows, 220 us; two rounds 340).
struct Cut {
  int rows;  // of the first part; M: one part
  Plan first, rest;
};
Cut cut_dense(DenseShape shape, DenseEpi epi, int M, int N, int K, int nseg)
{
  Cut cut = {M, plan_dense(shape, epi, M, N, K, nseg), {}};
  float best = cut.first.us;
  if (shape == kDenseWgrad) return cut;  // its rows are features: no odd counts worth a launch
  for (int rows : {M / 256 * 256, M / 128 * 128}) {
    if (rows == 0 || rows == M) continue;
    const Plan a = plan_dense(shape, epi, rows, N, K, nseg), b = plan_dense(shape, epi, M - rows, N, K, nseg);
    if (a.us + b.us + 3.f < best) {
      best = a.us + b.us + 3.f;
      cut = {rows, a, b};
    }
  }
  return cut;
}
size_t plan_bytes(const Plan& p, DenseEpi epi, int M, int N)
{
  return p.splits > 1 ? sizeof(float) * p.splits * (size_t)M * N * (epi == kDenseGlu ? 2 : 1) : 0;
}

template <typename T, DenseShape SH, DenseEpi EPI>
hipError_t launch_plan(const Plan& plan, DenseArgs a, float* partial, hipStream_t s)
{
  if constexpr (SH == kDenseForward)
    if (plan.tile < 0)
      return plan.tile == kFewOne ? launch_few<T, 1, EPI>(a, s) : launch_few<T, 2, EPI>(a, s);
  const Tile& tile = kTiles[plan.tile];
  const int cols = EPI == kDenseGlu ? tile.cols / 2 : tile.cols;
  a.tiles_m = (a.M + tile.rows - 1) / tile.rows;
  a.tiles_n = (a.N + cols - 1) / cols;
  a.splits = plan.splits;
  a.run = plan.run;
  a.partial = plan.splits > 1 ? partial : nullptr;
  switch (plan.tile) {
    case 0: launch_tiles<T, 2, 4, 4, 2, 2, SH, EPI>(a, plan.splits, s); break;
    case 1: launch_tiles<T, 2, 4, 2, 2, 3, SH, EPI>(a, plan.splits, s); break;
    case 2: launch_tiles<T, 2, 2, 2, 2, 4, SH, EPI>(a, plan.splits, s); break;
    default: launch_tiles<T, 2, 2, 1, 2, 5, SH, EPI>(a, plan.splits, s); break;
  }
  if (plan.splits > 1)
    hipLaunchKernelGGL((dense_finish_kernel<T, EPI>), dim3((unsigned)(((long long)a.M * (a.N / 8) + 63) / 64)),
                       dim3(64), 0, s, a);
  return hipGetLastError();
}

template <typename T, DenseShape SH, DenseEpi EPI>
hipError_t launch_planned(DenseArgs a, float* partial, hipStream_t s)
{
  const Cut cut = cut_dense(SH, EPI, a.M, a.N, a.K, a.nseg);
  if (cut.rows == a.M) return launch_plan<T, SH, EPI>(cut.first, a, partial, s);
  const int rest = a.M - cut.rows;
  a.M = cut.rows;
  const hipError_t e = launch_plan<T, SH, EPI>(cut.first, a, partial, s);
  if (e != hipSuccess) return e;
  const auto down = [&](const void* p, long long ld) {
    return p ? static_cast<const char*>(p) + 2 * cut.rows * ld : nullptr;
  };
  a.M = rest;
  a.a[0] = down(a.a[0], a.lda);
  a.a[1] = down(a.a[1], a.lda);
  a.out = const_cast<char*>(down(a.out, EPI == kDenseStore ? a.ldo : EPI == kDenseGlu ? a.N : 2LL * a.N));
  a.add0 = down(a.add0, a.N);
  a.add1 = down(a.add1, a.N);
  if (a.gu) a.gu += 2LL * cut.rows * a.N;
  return launch_plan<T, SH, EPI>(cut.rest, a, partial, s);
}

template <typename T>
hipError_t launch_typed(DenseShape shape, DenseEpi epi, const DenseArgs& a, float* partial, hipStream_t s)
{
  if (shape == kDenseForward)
    return epi == kDenseGlu ? launch_planned<T, kDenseForward, kDenseGlu>(a, partial, s)
                            : launch_planned<T, kDenseForward, kDenseStore>(a, partial, s);
  if (shape == kDenseDgrad)
    return epi == kDenseDGlu ? launch_planned<T, kDenseDgrad, kDenseDGlu>(a, partial, s)
                             : launch_planned<T, kDenseDgrad, kDenseStore>(a, partial, s);
  return launch_planned<T, kDenseWgrad, kDenseStore>(a, partial, s);
}

}  // namespace

size_t dense_partial_bytes(DenseShape shape, DenseEpi epi, int M, int N, int K, int nseg)
{
  if (M <= 0 || N <= 0) return 0;
  const Cut cut = cut_dense(shape, epi, M, N, K, nseg);
  return std::max(plan_bytes(cut.first, epi, cut.rows, N), plan_bytes(cut.rest, epi, M - cut.rows, N));
}

void dense_choice(DenseShape shape, DenseEpi epi, int M, int N, int K, int nseg, int* choice)
{
  std::fill_n(choice, 6, 0);
  if (M <= 0 || N <= 0) return;
  const Cut cut = cut_dense(shape, epi, M, N, K, nseg);
  const Plan* part = &cut.first;
  for (int rows : {cut.rows, M - cut.rows}) {
    if (rows > 0) {
      choice[0] = rows;
      choice[1] = part->tile;
      choice[2] = part->splits;
    }
    choice += 3;
    part = &cut.rest;
  }
}

hipError_t launch_dense(DenseShape shape, DenseEpi epi, const DenseArgs& a, int dtype, float* partial, hipStream_t s)
{
  if (a.M <= 0 || a.N <= 0) return hipSuccess;
  return dtype == MXFP4_BF16 ? launch_typed<__bf16>(shape, epi, a, partial, s)
                             : launch_typed<_Float16>(shape, epi, a, partial, s);
}

}  // namespace mx
