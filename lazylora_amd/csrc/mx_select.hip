// Expert selection over scored experts, with groups (mxfp4_select_topk) and its gradient.
//
// Per token: scores s = sigmoid(l) or softmax(l) of the logits; choice c = s + bias (without a bias the
// order of s is that of l); of num_groups equal runs of experts the topk_groups best stay, by the largest
// choice of each or the sum of its two largest; the top_k largest choices of those are written in
// descending order, equal ones and equal groups by the lower number first; weights s, renormalised by
// their sum + 1e-20 and scaled.
//
// Without a bias the order is that of the logits. With one, and between groups by sums of two, it is that of
// 64-bit scores and sums on the 32-bit bias: 32-bit values that lie closer than their error are decided in 64
// bits. Without that some token in a thousand (top-16 of 896) would get its experts in another order than the
// formula gives. What 64 bits hold as equal (sigmoid(38) and sigmoid(45), say) is equal and goes by the number.
#include "mx_device.h"
#include "mx_select.h"

namespace mx {

namespace {

// Choice values as whole numbers in selection order: NaN first, then the larger value; 0 stands for "not
// selectable", below every float's key.
MX_DEV uint32_t order_key(float v)
{
  const uint32_t u = f_bits(v + 0.0f);  // -0 and 0 are one value
  return v != v ? 0xFFFFFFFFu : u & 0x80000000u ? ~u : u | 0x80000000u;
}
MX_DEV float key_value(uint32_t k) { return bits_f(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }
MX_DEV uint64_t order_key(double v)
{
  const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0);
  return v != v ? ~0ull : u >> 63 ? ~u : u | (1ull << 63);
}
MX_DEV double key_value(uint64_t k)
{
  return __builtin_bit_cast(double, k >> 63 ? k & ~(1ull << 63) : ~k);
}

template <int CTRL>
MX_DEV uint32_t dpp_u(uint32_t v)
{
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}
MX_DEV uint32_t lane_u(uint32_t v, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); }
MX_DEV float lane_f(float v, int l) { return bits_f(lane_u(f_bits(v), l)); }
// Largest key of the wave: a butterfly within each row of 16 lanes, then the four rows' lanes.
MX_DEV uint32_t wave_max(uint32_t v)
{
  v = max(v, dpp_u<kDppXor1>(v));
  v = max(v, dpp_u<kDppXor2>(v));
  v = max(v, dpp_u<kDppHalfMirror>(v));
  v = max(v, dpp_u<kDppMirror>(v));
  return max(max(lane_u(v, 0), lane_u(v, 16)), max(lane_u(v, 32), lane_u(v, 48)));
}
MX_DEV float wave_sum(float v)
{
  v += bits_f(dpp_u<kDppXor1>(f_bits(v)));
  v += bits_f(dpp_u<kDppXor2>(f_bits(v)));
  v += bits_f(dpp_u<kDppHalfMirror>(f_bits(v)));
  v += bits_f(dpp_u<kDppMirror>(f_bits(v)));
  return (lane_f(v, 0) + lane_f(v, 16)) + (lane_f(v, 32) + lane_f(v, 48));
}
MX_DEV double wave_sum(double v)
{
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

template <typename T>
MX_DEV float load_logit(const T* p);
template <>
MX_DEV float load_logit<float>(const float* p)
{
  return *p;
}
template <>
MX_DEV float load_logit<uint16_t>(const uint16_t* p)  // bfloat16
{
  return bits_f((uint32_t)*p << 16);
}
template <>
MX_DEV float load_logit<_Float16>(const _Float16* p)
{
  return (float)*p;
}

// A token's scores: what turns a logit into a score. Softmax of a row without a finite logit (every expert
// off) gives 0 everywhere, not 0 / 0; a row with +inf or NaN gives NaN.
template <typename F>
struct Score {
  bool softmax;
  F top, sum;
  MX_DEV F operator()(float l) const
  {
    if (softmax) return exp_((F)l - top) / sum;
    return (F)1 / ((F)1 + exp_(-(F)l));
  }
  static MX_DEV float exp_(float v) { return expf(v); }
  static MX_DEV double exp_(double v) { return exp(v); }
};

// Where a lane's experts lie: the 64 lanes are cut into as many runs as there are groups (up to the next
// power of two), a run's lanes hold its group's experts in order, `per` to each. So the lowest lane of a
// tie holds the lowest expert, and a group's score is a butterfly over its run.
struct Slots {
  int first, count;  // the lane's experts: first .. first + count - 1
  int group, run;    // its group, and the lanes of a run
};
MX_DEV Slots lane_slots(const SelectArgs& a, int lane)
{
  Slots s;
  s.run = a.run;
  s.group = lane >> a.run_log;
  const int at = (lane & (a.run - 1)) * a.per;
  s.first = s.group * a.group_size + at;
  s.count = s.group < a.num_groups ? max(0, min(a.per, a.group_size - at)) : 0;
  return s;
}

// The two largest keys of a run's lanes, from each lane's two.
MX_DEV void merge2(uint32_t& a, uint32_t& b, uint32_t c, uint32_t d)
{
  b = max(min(a, c), max(b, d));
  a = max(a, c);
}
MX_DEV void run_top2(uint32_t& a, uint32_t& b, int run)
{
  if (run > 1) merge2(a, b, dpp_u<kDppXor1>(a), dpp_u<kDppXor1>(b));
  if (run > 2) merge2(a, b, dpp_u<kDppXor2>(a), dpp_u<kDppXor2>(b));
  if (run > 4) merge2(a, b, dpp_u<kDppHalfMirror>(a), dpp_u<kDppHalfMirror>(b));
  if (run > 8) merge2(a, b, dpp_u<kDppMirror>(a), dpp_u<kDppMirror>(b));
  for (int off = 16; off < run; off <<= 1) merge2(a, b, __shfl_xor(a, off, 64), __shfl_xor(b, off, 64));
}
MX_DEV void run_top2(uint64_t& a, uint64_t& b, int run)
{
  for (int off = 1; off < run; off <<= 1) {
    const uint64_t c = __shfl_xor(a, off, 64), d = __shfl_xor(b, off, 64);
    b = max(min(a, c), max(b, d));
    a = max(a, c);
  }
}

// The 64-bit form of a whole token, for one whose 32-bit values leave the choice open. Rare, and written to
// be small: the values are computed again in every pass.
template <typename T>
struct Careful {
  const SelectArgs& a;
  const T* row;
  Slots at;
  Score<double> score;

  MX_DEV Careful(const SelectArgs& args, const T* r, const Slots& s, float top, int lane) : a(args), row(r), at(s)
  {
    score.softmax = a.softmax;
    score.top = top;
    score.sum = 1.0;
    if (a.softmax) {
      double sum = 0.0;
      for (int m = 0; m < at.count; ++m) sum += exp((double)load_logit<T>(row + at.first + m) - (double)top);
      sum = wave_sum(sum);
      score.sum = sum == 0.0 ? 1.0 : sum;
    }
  }
  MX_DEV double choice(int e) const
  {
    const double s = score(load_logit<T>(row + e));
    return a.bias ? s + (double)a.bias[e] : s;
  }
  // Whether the lane's group is among the kept ones.
  MX_DEV bool group_on() const
  {
    uint64_t k1 = 0, k2 = 0;
    for (int m = 0; m < at.count; ++m) {
      const uint64_t k = order_key(choice(at.first + m));
      k2 = max(k2, min(k1, k));
      k1 = max(k1, k);
    }
    run_top2(k1, k2, at.run);
    if (a.top2 && k2 != 0) k1 = order_key(key_value(k1) + key_value(k2));
    int rank = 0;
    for (int g = 0; g < a.num_groups; ++g) {
      const uint64_t other = __shfl(k1, g * at.run, 64);
      rank += other > k1 || (other == k1 && g < at.group);
    }
    return at.count > 0 && rank < a.topk_groups;
  }
  // The chosen experts in order, lane t the t-th: every round takes the first behind the last one taken.
  MX_DEV int pick(bool on, int lane) const
  {
    uint64_t last_key = ~0ull;
    int last = -1, mine = 0;
    bool first = true;
    for (int t = 0; t < a.top_k; ++t) {
      uint64_t best = 0;
      int e_best = 0x7fffffff;
      for (int m = 0; on && m < at.count; ++m) {
        const int e = at.first + m;
        const uint64_t k = order_key(choice(e));
        if (!first && (k > last_key || (k == last_key && e <= last))) continue;
        if (k > best) best = k, e_best = e;
      }
      for (int off = 32; off >= 1; off >>= 1) {
        const uint64_t k = __shfl_xor(best, off, 64);
        const int e = __shfl_xor(e_best, off, 64);
        if (k > best || (k == best && e < e_best)) best = k, e_best = e;
      }
      last_key = best;
      last = e_best;
      first = false;
      if (lane == t) mine = e_best;
    }
    return mine;
  }
};

// One wave per token, bound by instructions: a round costs some 22 of them and is a serial chain, so as many waves as
// there can be (eight per SIMD with 64 registers) run side by side. 8192 tokens, top-8 of 256 in 8 groups, sigmoid
// and bias: 11 to 12 us (9 MB of logits would take 1.8); without groups and bias 7.3; 1024 tokens, top-16 of 896 in 7
// groups, softmax and bias: 14 to 17 us; one token 3.7. A round of the selection takes the largest open key of the wave
// (four butterfly steps and four lane reads), names its holder by a ballot and retires the expert there.
template <typename T, int PER>
__global__ __launch_bounds__(256, PER <= 4 ? 8 : 1) void select_kernel(SelectArgs a)
{
  const int lane = threadIdx.x & 63;
  const long long token = a.token0 + (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (token >= a.N) return;  // whole waves leave together
  const T* row = static_cast<const T*>(a.logits) + token * a.E;
  const Slots at = lane_slots(a, lane);

  // every lane loads, from its last expert again past its own (an absent group's lanes from the first one), and with
  // one instruction where all lanes have PER
  const int base = at.count > 0 ? at.first : 0, last = max(at.count - 1, 0);
  float x[PER];
  if (a.full) {
    T raw[PER];
    __builtin_memcpy(raw, row + base, sizeof(raw));
    static_for<PER>([&](auto mc) { x[decltype(mc)::value] = load_logit<T>(raw + decltype(mc)::value); });
  } else {
    static_for<PER>([&](auto mc) { x[decltype(mc)::value] = load_logit<T>(row + base + min((int)decltype(mc)::value, last)); });
  }
  static_for<PER>([&](auto mc) {
    constexpr int m = decltype(mc)::value;
    x[m] = m < at.count ? x[m] : -__builtin_inff();
  });
  Score<float> score{a.softmax, 0.f, 1.f};
  float smax = 1.f;  // no score of the row is larger
  if (a.softmax) {
    uint32_t top = 0;
    static_for<PER>([&](auto mc) { top = max(top, order_key(x[decltype(mc)::value])); });
    score.top = key_value(wave_max(top));
    if (score.top == -__builtin_inff()) score.top = 0.f;
    float sum = 0.f;
    static_for<PER>([&](auto mc) { sum += expf(x[decltype(mc)::value] - score.top); });
    sum = wave_sum(sum);
    score.sum = sum == 0.f ? 1.f : sum;
    smax = 1.f / score.sum;
  }
  // The keys' scores take the device's exponential and reciprocal (sigmoid_f, and 2^((l - max) log2 e) / sum): off by
  // less than half of this, the rounding of the exponent (which moves a score s by s |l - max| 2^-24, at most 0.37
  // smax 2^-24), the exponential, the reciprocal and the sum behind it. The weights are computed again in full.
  const float inv = 1.f / score.sum;
  const auto quick = [&](float l) {
    return a.softmax ? __builtin_amdgcn_exp2f((l - score.top) * kLog2e) * inv : sigmoid_f(l);
  };
  const float s_err = smax * (a.softmax ? 0x1p-20f + (float)(a.per + 16) * 0x1p-23f : 0x1p-20f);

  uint32_t key[PER];  // 0: absent, in no kept group or already chosen
  if (a.bias) {
    float c[PER];
    if (a.full)
      __builtin_memcpy(c, a.bias + base, sizeof(c));
    else
      static_for<PER>([&](auto mc) { c[decltype(mc)::value] = a.bias[base + min((int)decltype(mc)::value, last)]; });
    if (a.softmax)
      static_for<PER>([&](auto mc) {
        constexpr int m = decltype(mc)::value;
        c[m] += __builtin_amdgcn_exp2f((x[m] - score.top) * kLog2e) * inv;
      });
    else
      static_for<PER>([&](auto mc) { c[decltype(mc)::value] += sigmoid_f(x[decltype(mc)::value]); });
    static_for<PER>([&](auto mc) { key[decltype(mc)::value] = order_key(c[decltype(mc)::value]); });
  } else {
    static_for<PER>([&](auto mc) { key[decltype(mc)::value] = order_key(x[decltype(mc)::value]); });
  }
  static_for<PER>([&](auto mc) {
    constexpr int m = decltype(mc)::value;
    key[m] = m < at.count ? key[m] : 0u;
  });

  bool on = at.count > 0;  // the lane's experts can be chosen
  if (a.num_groups > 1) {
    uint32_t k1 = 0, k2 = 0;
    // without a bias the keys are the logits', whose largest has the largest score; sums need the scores
    const bool scores = !a.bias && a.top2;
    static_for<PER>([&](auto mc) {
      constexpr int m = decltype(mc)::value;
      k2 = max(k2, min(k1, key[m]));
      k1 = max(k1, key[m]);
    });
    run_top2(k1, k2, at.run);
    // the group's value, its error, and whether it is infinite or NaN because a choice in it is
    const auto endless = [](float v) { return !(fabsf(v) < __builtin_inff()); };
    float c1 = key_value(k1), c2 = key_value(k2);
    if (scores) c1 = quick(c1), c2 = quick(c2);
    uint32_t gk = k1;
    bool exact = endless(c1);
    float err = s_err + 0x1p-22f * fabsf(c1);
    if (a.top2) {
      if (k2 != 0) {
        gk = order_key(c1 + c2);
        exact |= endless(c2);
        err = 2.f * s_err + 0x1p-21f * (fabsf(c1) + fabsf(c2));
      } else {
        gk = order_key(c1);
      }
    }
    int rank = 0;  // a group's
    const int place = lane & (at.run - 1), start = lane - place;
    for (int g0 = 0; g0 < a.num_groups; g0 += at.run) {  // a run's lanes compare with a group each
      const int g = g0 + place;
      const uint32_t other = (uint32_t)__shfl((int)gk, min(g, a.num_groups - 1) << a.run_log, 64);
      const bool better = (g < a.num_groups) & ((other > gk) | ((other == gk) & (g < at.group)));
      const uint64_t votes = __builtin_amdgcn_ballot_w64(better) >> start;
      rank += __popcll(at.run == 64 ? votes : votes & ((1ull << at.run) - 1));
    }
    on = on && rank < a.topk_groups;
    if ((a.top2 || a.bias) && a.topk_groups < a.num_groups) {
      // The kept groups' least possible value against the others' largest: any kept group may be the one whose error
      // (of a sum of two that cancel, say) kept it. An infinity or NaN among the choices is exact, and equal ones go
      // by their number; a sum of finite ones that 32 bits cannot hold lies past 2^127.
      const float gv = key_value(gk);
      const bool here = at.group < a.num_groups, kept = rank < a.topk_groups;
      const float below = gv == __builtin_inff() ? 0x1p127f : gv - err, above = gv == -__builtin_inff() ? -0x1p127f : gv + err;
      const uint32_t low = ~wave_max(here & kept ? ~(exact ? gk : order_key(below)) : 0u);
      const uint32_t high = wave_max(here & !kept ? exact ? gk : order_key(above) : 0u);
      if (low < high || (low == high && fabsf(key_value(low)) < __builtin_inff()))
        on = Careful<T>(a, row, at, score.top, lane).group_on();
    }
    static_for<PER>([&](auto mc) { key[decltype(mc)::value] = on ? key[decltype(mc)::value] : 0u; });
  }

  uint32_t best = 0;
  static_for<PER>([&](auto mc) { best = max(best, key[decltype(mc)::value]); });
  uint32_t mine_key = 0;  // lane t keeps the t-th chosen expert
  int mine = 0;
  const auto round = [&](int t) {
    const uint32_t win = wave_max(best);
    const int owner = __builtin_amdgcn_readfirstlane(__builtin_ctzll(__builtin_amdgcn_ballot_w64(best == win)));
    int mm = 0;
    uint32_t nb = 0;
    static_for<PER>([&](auto mc) {  // the holder's lowest expert with this key
      constexpr int m = PER - 1 - decltype(mc)::value;
      mm = key[m] == win ? m : mm;
    });
    static_for<PER>([&](auto mc) {
      constexpr int m = decltype(mc)::value;
      key[m] = lane == owner && m == mm ? 0u : key[m];
      nb = max(nb, key[m]);
    });
    best = nb;
    const int e = __builtin_amdgcn_readlane(at.first + mm, owner);
    if (lane == t) mine = e, mine_key = win;
  };
  for (int t = 0; t < a.top_k; ++t) round(t);

  if (a.bias) {
    // Neighbours of the order, and open experts behind the last, that are closer than their error.
    const float v = key_value(mine_key);
    const float err = s_err + 0x1p-22f * fabsf(v);
    const float next = key_value((uint32_t)__shfl_down((int)mine_key, 1, 64));
    const bool pair = lane < a.top_k - 1 && v - next <= err && fabsf(v) < __builtin_inff();
    const float vl = lane_f(v, a.top_k - 1), el = lane_f(err, a.top_k - 1);
    const uint32_t line = vl - el == vl - el && fabsf(vl) < __builtin_inff() ? order_key(vl - el) : 0xFFFFFFFFu;
    if (__builtin_amdgcn_ballot_w64(pair) != 0 || __builtin_amdgcn_ballot_w64(best >= line) != 0) {
      // the open experts above the line join, as many as there are lanes, and 64 bits decide the order
      int n = a.top_k;
      while (n < 64 && __builtin_amdgcn_ballot_w64(best >= line) != 0) round(n++);
      const Careful<T> careful(a, row, at, score.top, lane);
      if (__builtin_amdgcn_ballot_w64(best >= line) != 0) {
        mine = careful.pick(on, lane);
      } else {
        const uint64_t k = lane < n ? order_key(careful.choice(mine)) : 0;
        int rank = 0;
        for (int t = 0; t < n; ++t) {
          const uint64_t other = __shfl(k, t, 64);
          const int e = __builtin_amdgcn_readlane(mine, t);
          rank += other > k || (other == k && e < mine);
        }
        int sorted = mine;
        for (int t = 0; t < n; ++t) {
          const int e = __builtin_amdgcn_readlane(mine, t), r = __builtin_amdgcn_readlane(rank, t);
          if (lane == r) sorted = e;
        }
        mine = sorted;
      }
    }
  }

  float s = 0.f;
  if (lane < a.top_k) s = score(load_logit<T>(row + mine));
  float w = s;
  if (a.renormalize) w = s / (wave_sum(s) + 1e-20f);
  if (lane < a.top_k) {
    a.topk_idx[token * a.top_k + lane] = mine;
    a.topk_w[token * a.top_k + lane] = w * a.scale;
  }
}

// The gradient of the weights with respect to the logits, one wave per token. With chosen scores s_j, S =
// sum s_j + 1e-20, upstream g and the factor c:
//   ds_j = c (sum_i s_i (g_j - g_i) + 1e-20 g_j) / S^2   (renormalised),   c g_j   (otherwise);
//   sigmoid: dl_e = ds_e s_e (1 - s_e) at the chosen experts, 0 elsewhere;
//   softmax: dl_e = s_e (ds_e - d) with d = sum_j ds_j s_j, at every expert. Renormalised, d is
//   c (sum g s) 1e-20 / S^2; otherwise ds_j - d at a chosen expert is
//   c (sum_i s_i (g_j - g_i) + g_j times the scores not chosen).
// The sums go over differences of the upstream gradients: where one expert has nearly all of the score its own
// gradient is as small as the others' scores, and g_j - sum_i g_i s_i / S would leave the rounding of g_j.
// A token's ds meet its experts through a row of LDS, -0 where an expert is not chosen. 4099 tokens of 64 experts
// 4.1 us, 1024 of 896 7.0.
constexpr float kNotChosen = -0.f;
MX_DEV bool not_chosen(float v) { return f_bits(v) == 0x80000000u; }
template <typename T, int PER>
__global__ __launch_bounds__(256) void select_bwd_kernel(SelectBwdArgs a)
{
  extern __shared__ float rows[];
  const int lane = threadIdx.x & 63;
  const long long token = a.token0 + (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (token >= a.N) return;
  float* ds_row = rows + (threadIdx.x >> 6) * a.E;
  const T* row = static_cast<const T*>(a.logits) + token * a.E;
  T* out = static_cast<T*>(a.grad_logits) + token * a.E;

  float x[PER];
  static_for<PER>([&](auto mc) {
    constexpr int m = decltype(mc)::value;
    const int e = lane + 64 * m;
    x[m] = -__builtin_inff();
    if (e < a.E) {
      x[m] = load_logit<T>(row + e);
      ds_row[e] = kNotChosen;
    }
  });
  Score<float> score{a.softmax, 0.f, 1.f};
  if (a.softmax) {
    uint32_t top = 0;
    static_for<PER>([&](auto mc) { top = max(top, order_key(x[decltype(mc)::value])); });
    score.top = key_value(wave_max(top));
    if (score.top == -__builtin_inff()) score.top = 0.f;
    float sum = 0.f;
    static_for<PER>([&](auto mc) {  // from here on x is the exponentials
      constexpr int m = decltype(mc)::value;
      x[m] = expf(x[m] - score.top);
      sum += x[m];
    });
    sum = wave_sum(sum);
    score.sum = sum == 0.f ? 1.f : sum;
  }
  int e = -1;
  float s = 0.f, g = 0.f;
  if (lane < a.top_k) {
    const long long v = a.topk_idx[token * a.top_k + lane];
    if (v >= 0 && v < a.E) {
      e = (int)v;
      s = score(load_logit<T>(row + e));
      g = a.grad_w[token * a.top_k + lane] * a.scale;
    }
  }
  const float gs = wave_sum(g * s);
  float diff = 0.f;  // sum_i s_i (g - g_i)
  if (a.softmax || a.renormalize)
    for (int i = 0; i < a.top_k; ++i) diff = fmaf(lane_f(s, i), g - lane_f(g, i), diff);
  float ds = g, d = gs;  // of softmax ds - d at the chosen experts
  if (a.renormalize) {
    const float den = wave_sum(s) + 1e-20f;
    d = gs * (1e-20f / den) / den;
    ds = fmaf(1e-20f, g, diff) / den / den;
    if (a.softmax) ds -= d;
  } else if (a.softmax) {
    wave_lds_fence();
    if (e >= 0) ds_row[e] = 0.f;
    wave_lds_fence();
    float left = 0.f;
    static_for<PER>([&](auto mc) {
      constexpr int m = decltype(mc)::value;
      const int i = lane + 64 * m;
      if (i < a.E && not_chosen(ds_row[i])) left += x[m];
    });
    ds = fmaf(g, wave_sum(left) / score.sum, diff);
  }
  wave_lds_fence();
  if (e >= 0) ds_row[e] = ds + 0.f;  // never -0
  wave_lds_fence();
  static_for<PER>([&](auto mc) {
    constexpr int m = decltype(mc)::value;
    const int i = lane + 64 * m;
    if (i < a.E) {
      const float t = ds_row[i];
      float v;
      if (a.softmax) {
        v = x[m] / score.sum * (not_chosen(t) ? -d : t);
      } else {
        // 1 - s as the other side's sigmoid, without the cancellation of 1 - s
        v = t == 0.f ? 0.f : t * score(x[m]) * score(-x[m]);
      }
      if constexpr (sizeof(T) == 4)
        out[i] = v;
      else if constexpr (std::is_same_v<T, uint16_t>)
        out[i] = (uint16_t)(pack_bf16(v, 0.f) & 0xFFFFu);
      else
        out[i] = (_Float16)v;
    }
  });
}

// A launch's threads are counted in 32 bits: so many tokens take one.
constexpr long long kTokensPerLaunch = 1 << 25;
template <class Kernel, class Args>
void launch_tokens(Kernel kernel, Args a, size_t lds, hipStream_t s)
{
  for (a.token0 = 0; a.token0 < a.N; a.token0 += kTokensPerLaunch) {
    const long long now = a.N - a.token0 < kTokensPerLaunch ? a.N - a.token0 : kTokensPerLaunch;
    kernel<<<dim3((unsigned)((now + 3) / 4)), 256, lds, s>>>(a);
  }
}
template <typename T, int PER>
void launch_per(SelectArgs a, hipStream_t s)
{
  a.full = a.per == PER && a.group_size % PER == 0;
  launch_tokens(select_kernel<T, PER>, a, 0, s);
}
template <typename T>
hipError_t run_select(const SelectArgs& a, hipStream_t s)
{
  if (a.per <= 1)
    launch_per<T, 1>(a, s);
  else if (a.per <= 4)
    launch_per<T, 4>(a, s);
  else if (a.per <= 16)
    launch_per<T, 16>(a, s);
  else
    launch_per<T, 64>(a, s);
  return hipGetLastError();
}
template <typename T>
hipError_t run_select_bwd(const SelectBwdArgs& a, hipStream_t s)
{
  const size_t lds = 4 * sizeof(float) * a.E;
  if (a.E <= 4 * 64)
    launch_tokens(select_bwd_kernel<T, 4>, a, lds, s);
  else if (a.E <= 16 * 64)
    launch_tokens(select_bwd_kernel<T, 16>, a, lds, s);
  else
    launch_tokens(select_bwd_kernel<T, 64>, a, lds, s);
  return hipGetLastError();
}

}  // namespace

int select_per_lane(int E, int num_groups)
{
  int runs = 1;
  while (runs < num_groups) runs *= 2;
  const int size = E / num_groups, run = kSelectLanes / runs;
  return run > 0 ? (size + run - 1) / run : kSelectMaxPer + 1;
}

hipError_t launch_select(SelectArgs a, int dtype, hipStream_t s)
{
  int runs = 1;
  while (runs < a.num_groups) runs *= 2;
  a.run = kSelectLanes / runs;
  a.run_log = __builtin_ctz(a.run);
  a.group_size = a.E / a.num_groups;
  a.per = select_per_lane(a.E, a.num_groups);
  switch (dtype) {
    case 0: return run_select<float>(a, s);
    case 1: return run_select<uint16_t>(a, s);
    default: return run_select<_Float16>(a, s);
  }
}

hipError_t launch_select_bwd(const SelectBwdArgs& a, int dtype, hipStream_t s)
{
  switch (dtype) {
    case 0: return run_select_bwd<float>(a, s);
    case 1: return run_select_bwd<uint16_t>(a, s);
    default: return run_select_bwd<_Float16>(a, s);
  }
}

}  // namespace mx
