// Experts of every token from the router's logits, with softmax or sigmoid scores, a bias that takes part in the choice alone, and groups of
// experts of which the best are open; the gradient of the weights; and the check of a routing that a caller brings.
//
//   s = softmax(l) over the experts, or 1 / (1 + exp(-l))           key = l without a bias, s + b with one
//   a group's rank: its largest key, or the sum of its two largest s + b     the best `top_groups` groups are open
//     (masked experts have a part in such a sum with a score of zero; a group of masked ones alone is the last)
//   chosen: the k largest keys of the open groups, ties to the lower id      weight = scale s / (sum of the chosen s, or 1)
//   backward, g = scale dw, share = s / sum of the chosen s:
//     softmax, renormalised: dl = share (g - sum share g)       sigmoid: the same times 1 - s
//     softmax: dl_i = s_i (g_i - sum s g), over all experts     sigmoid: dl = s (1 - s) g
//
// Scores and keys that decide are in double: two experts whose keys differ by less than a float's step still come in their order.  An expert whose logit is -inf is
// chosen only where nothing else is left, one whose logit is no number after those; neither has a part in the others' scores.
#include <type_traits>

#include "common.hpp"

namespace mi_moe {

template <int DT>
using Logit = typename std::conditional<DT == 0, uint16_t, typename std::conditional<DT == 1, _Float16, float>::type>::type;

// keys as integers in the keys' order, the two zeros alike; 0 is for what cannot be chosen, 1 for what is no number
__device__ __forceinline__ uint32_t key_of(float f) {
  uint32_t u = __float_as_uint(f);
  if (f != f) return 1u;
  if (u == 0x80000000u) u = 0u;
  return (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(double f) {
  uint64_t u = (uint64_t)__double_as_longlong(f);
  if (f != f) return 1u;
  if (u == (uint64_t)1 << 63) u = 0u;
  return (u >> 63) ? ~u : u | (uint64_t)1 << 63;
}
__device__ __forceinline__ uint32_t wave_max_key(uint32_t k) { return wave_max_u32(k); }
__device__ __forceinline__ uint64_t wave_max_key(uint64_t k) {
  const uint32_t hi = wave_max_u32((uint32_t)(k >> 32));
  const uint32_t lo = wave_max_u32((uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
  return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t readlane_key(uint64_t k, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(k >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)k, lane);
}
__device__ __forceinline__ double sigmoid64(double l) { return 1.0 / (1.0 + exp(-l)); }

__device__ __forceinline__ void put_value(void *base, int64_t at, int dt, double v) {
  if (dt == 0) static_cast<uint16_t *>(base)[at] = f32_to_bf16((float)v);
  else if (dt == 1) static_cast<_Float16 *>(base)[at] = (_Float16)(float)v;
  else static_cast<float *>(base)[at] = (float)v;
}
__device__ __forceinline__ float get_value(const void *base, int64_t at, int dt) {
  if (dt == 0) return bf16_to_f32(static_cast<const uint16_t *>(base)[at]);
  if (dt == 1) return (float)static_cast<const _Float16 *>(base)[at];
  return static_cast<const float *>(base)[at];
}

struct SelectKernelArgs {
  SelectArgs a;
  int size, lanes_log2, slots;  // experts of a group; lanes of a group; a lane's experts
};

// A token's experts in a wave.  A group of experts goes to a run of lanes, consecutive experts to a lane, so that lanes and slots are in the order of the ids.
template <int S>
struct Slots {
  float l[S];
  bool on[S];
  int base;  // id of slot 0
};

// merges the two largest of two disjoint sets
template <class T>
__device__ __forceinline__ void merge_two(T &t1, T &t2, T o1, T o2) {
  t2 = fmax(fmin(t1, o1), fmax(t2, o2));
  t1 = fmax(t1, o1);
}
__device__ __forceinline__ float f32_of(uint32_t u) { return __uint_as_float(u); }
// whether one of the group's lanes is among `lanes` (groups > 1: of half of the lanes at most)
__device__ __forceinline__ bool group_has(uint64_t lanes, int g, int lanes_log2) { return (lanes >> (g << lanes_log2) & (((uint64_t)1 << (1 << lanes_log2)) - 1)) != 0; }

// Everything in double, u64 keys: any logits and biases.  Lane r gets the r-th expert's id.
template <int S>
__device__ __forceinline__ void select_exact(const SelectKernelArgs &p, const Slots<S> &x, int g, uint32_t &id) {
  const SelectArgs &a = p.a;
  const int lane = lane_id();
  double v[S];
  float b[S];
#pragma unroll
  for (int j = 0; j < S; ++j) b[j] = a.bias && x.on[j] ? a.bias[x.base + j] : 0.f;
  if (a.scoring == 0) {
    float most = -INFINITY;  // (fmaxf passes over what is no number)
#pragma unroll
    for (int j = 0; j < S; ++j) most = fmaxf(most, x.l[j]);
    most = wave_max_f32(most);
    double total = 0.0;
#pragma unroll
    for (int j = 0; j < S; ++j) {
      v[j] = most == -INFINITY ? 0.0 : exp((double)x.l[j] - (double)most);
      total += v[j] == v[j] || x.l[j] == x.l[j] ? v[j] : 0.0;
    }
    total = wave_sum_f64(total);
#pragma unroll
    for (int j = 0; j < S; ++j) v[j] = x.l[j] != x.l[j] ? NAN : total > 0.0 || total != total ? v[j] / total : 0.0;
  } else {
#pragma unroll
    for (int j = 0; j < S; ++j) v[j] = sigmoid64(x.l[j]);
  }
  uint64_t key[S];
#pragma unroll
  for (int j = 0; j < S; ++j) {
    v[j] += (double)b[j];
    if (x.l[j] == -INFINITY) v[j] = -INFINITY;
    key[j] = !x.on[j] ? 0 : a.bias ? key_of(v[j]) : key_of((double)x.l[j]);
  }
  if (a.groups > 1) {
    const bool two = a.group_score == 1 && p.size > 1;
    double t1 = -INFINITY, t2 = -INFINITY;  // the two largest of the group
    bool able = false;                      // this lane has an expert that is not masked
#pragma unroll
    for (int j = 0; j < S; ++j) {
      double y = a.group_score == 0 && !a.bias ? (double)x.l[j] : v[j];
      able |= x.on[j] && x.l[j] > -INFINITY && b[j] > -INFINITY;
      if (two && !(x.l[j] > -INFINITY)) y = b[j];  // (a score of zero)
      if (!x.on[j] || y != y) y = -INFINITY;
      t2 = fmax(t2, fmin(t1, y));
      t1 = fmax(t1, y);
    }
    for (int d = 0; d < p.lanes_log2; ++d) {
      const double o1 = __shfl_xor(t1, 1 << d), o2 = __shfl_xor(t2, 1 << d);
      merge_two(t1, t2, o1, o2);
    }
    const bool has = group_has(__ballot(able), g, p.lanes_log2);
    const uint64_t mine = key_of(!has ? -INFINITY : two && t2 > -INFINITY ? t1 + t2 : t1);
    int before = 0;
    for (int o = 0; o < a.groups; ++o) {
      const uint64_t other = readlane_key(mine, o << p.lanes_log2);
      before += other > mine || (other == mine && o < g);
    }
    if (before >= a.top_groups)
#pragma unroll
      for (int j = 0; j < S; ++j) key[j] = 0;
  }
  for (int r = 0; r < a.k; ++r) {
    uint64_t best = 0;
    int at = 0;
#pragma unroll
    for (int j = 0; j < S; ++j)
      if (key[j] > best) best = key[j], at = j;
    const uint64_t top = wave_max_key(best);
    const int owner = __builtin_ctzll(__ballot(best == top));
    if (lane == owner)
#pragma unroll
      for (int j = 0; j < S; ++j)
        if (j == at) key[j] = 0;
    const uint32_t chosen = (uint32_t)__builtin_amdgcn_readlane(x.base + at, owner);
    if (lane == r) id = chosen;
  }
}

// The keys and the groups' ranks in float where that decides them.  A float score is off by 2^-22 of itself for the exponential, 2^-23 for the reciprocal and, of a softmax, 14 * 2^-24 for
// the sum, which is the same factor for all of a token's; scores are at most one, so two of them differ by what doubles say to within 1.9 * 2^-20, and biased keys to within 2^-23 of their size more.
// A sigmoid is 1 / (1 + e): a quarter of the exponential's error at most, a rounding and the reciprocal, together 3.9 * 2^-24.
// Where two keys that follow each other in the choice, or two groups' ranks, are nearer than near_of and kNearOfSize of them allow, or something is an infinity above zero or no number, doubles decide
// (of random logits and small biases, 256 experts, for one token in 1700, 512 experts with 16 chosen one in 370); without a bias the logits are exact keys.  Scores of the chosen are in double, a lane each, of softmax scores that are renormalised from the chosen logits
// alone: they hold where a softmax over all would round to zero.
constexpr float kNearOfSize = 0x1p-21f;
__device__ __forceinline__ float near_of(const SelectArgs &a) { return a.scoring == 1 ? 0x1p-21f : 0x1p-19f; }

// whether floats can decide
__device__ __forceinline__ bool not_below(float l, float b) { return !(l < INFINITY && b < INFINITY); }
// what a group's rank may be off by, in kNearOfSize (a rank of minus infinity is that)
__device__ __forceinline__ float rank_size(float rank, float t1, float t2, bool two) { return rank == -INFINITY ? 0.f : two ? fabsf(t1) + fabsf(t2) : fabsf(t1); }

// score of a chosen expert but for a factor that renormalisation takes out again
__device__ __forceinline__ double score_of(const SelectArgs &a, float logit, float most, double total) {
  if (a.scoring == 1) return sigmoid64(logit);
  return logit != logit ? NAN : most == -INFINITY ? 0.0 : exp((double)logit - (double)most) / total;
}

// weights of a token's choice from its scores, in the lanes below k; `sum`: of all lanes' scores
__device__ __forceinline__ void put_choice(const SelectArgs &a, int64_t t, int lane, uint32_t id, double score, double sum) {
  const double w = !a.renormalize ? score : sum == 0.0 ? 0.0 : score / sum;
  if (lane < a.k) {
    a.idx[t * a.k + lane] = id;
    put_value(a.w, t * a.k + lane, a.w_dtype, w * (double)a.scale);
  }
}

// SUM: softmax scores that are not renormalised, whose denominator is over all experts.  KEYS: float scores decide something (a bias, or groups ranked by two scores).
template <int DT, int S, bool KEYS, bool SUM>
__global__ __launch_bounds__(256) void select_experts_kernel(SelectKernelArgs p) {
  const SelectArgs &a = p.a;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= a.T) return;
  const int lane = lane_id(), g = lane >> p.lanes_log2, from = (lane & ((1 << p.lanes_log2) - 1)) * p.slots;
  const Logit<DT> *const row = static_cast<const Logit<DT> *>(a.logits) + t * a.E;
  Slots<S> x;
  x.base = g * p.size + from;
#pragma unroll
  for (int j = 0; j < S; ++j) {
    x.on[j] = j < p.slots && from + j < p.size && g < a.groups;
    x.l[j] = x.on[j] ? as_f32(row[x.base + j]) : -INFINITY;
  }
  float b[S];
  bool odd = false;    // something that floats do not decide
  bool masks = false;  // one of the token's logits is -inf
  if constexpr (KEYS) {
    float least = INFINITY;
#pragma unroll
    for (int j = 0; j < S; ++j) {
      b[j] = a.bias && x.on[j] ? a.bias[x.base + j] : 0.f;
      odd |= x.on[j] && not_below(x.l[j], b[j]);
      if (x.on[j]) least = fminf(least, x.l[j]);
    }
    masks = __any(least == -INFINITY);
  }
  float most = -INFINITY;
  if (SUM || (KEYS && a.scoring == 0)) {
#pragma unroll
    for (int j = 0; j < S; ++j) most = fmaxf(most, x.l[j]);
    most = wave_max_f32(most);
    if constexpr (KEYS) odd |= a.scoring == 0 && most == -INFINITY;
  }
  double total = 1.0;
  if constexpr (SUM) {
    total = 0.0;
#pragma unroll
    for (int j = 0; j < S; ++j)
      if (x.l[j] == x.l[j] && most > -INFINITY) total += exp((double)x.l[j] - (double)most);
    total = wave_sum_f64(total);
  }
  uint32_t key[S];
#pragma unroll
  for (int j = 0; j < S; ++j) key[j] = x.on[j] ? key_of(x.l[j]) : 0;
  if constexpr (KEYS) {
    float s[S];
    if (a.scoring == 0) {
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < S; ++j) {
        s[j] = __expf(x.l[j] - most);
        sum[j % 4] += s[j];
      }
      const float inv = __builtin_amdgcn_rcpf((float)wave_sum_f64((double)(sum[0] + sum[1]) + (double)(sum[2] + sum[3])));
#pragma unroll
      for (int j = 0; j < S; ++j) s[j] *= inv;
    } else {
#pragma unroll
      for (int j = 0; j < S; ++j) s[j] = __builtin_amdgcn_rcpf(1.0f + __expf(-x.l[j]));
    }
#pragma unroll
    for (int j = 0; j < S; ++j) {
      s[j] += b[j];
      if (a.bias && x.on[j]) key[j] = key_of(s[j]);
    }
    const bool two = a.groups > 1 && a.group_score == 1 && p.size > 1;
    if (masks) {  // (ranked by two, they have a score of zero)
#pragma unroll
      for (int j = 0; j < S; ++j)
        if (x.on[j] && x.l[j] == -INFINITY) {
          key[j] = key_of(-INFINITY);
          if (!two) s[j] = -INFINITY;
        }
    }
    if (a.groups > 1) {
      float t1 = -INFINITY, t2 = -INFINITY;
#pragma unroll
      for (int j = 0; j < S; ++j) {
        const float y = !x.on[j] ? -INFINITY : a.group_score == 0 && !a.bias ? x.l[j] : s[j];
        t2 = fmaxf(t2, fminf(t1, y));
        t1 = fmaxf(t1, y);
      }
      const int n = p.lanes_log2;
      auto other = [&](auto ctrl) __attribute__((always_inline)) {
        constexpr int CTRL = decltype(ctrl)::value;
        merge_two(t1, t2, f32_of(dpp_u32<CTRL>(__float_as_uint(t1))), f32_of(dpp_u32<CTRL>(__float_as_uint(t2))));
      };
      if (n > 0) other(std::integral_constant<int, kDppXor1>{});
      if (n > 1) other(std::integral_constant<int, kDppXor2>{});
      if (n > 2) other(std::integral_constant<int, kDppHalfMirror>{});
      if (n > 3) other(std::integral_constant<int, kDppMirror>{});
      if (n > 4) merge_two(t1, t2, __shfl_xor(t1, 16), __shfl_xor(t2, 16));
      if (n > 5) merge_two(t1, t2, __shfl_xor(t1, 32), __shfl_xor(t2, 32));
      if (t2 == -INFINITY) t2 = 0.f;
      float mine = two ? t1 + t2 : t1;
      if (two && masks) {  // (where no logit is masked, a group of masked ones has nothing but biases of -inf)
        bool able = false;
#pragma unroll
        for (int j = 0; j < S; ++j) able |= x.on[j] && x.l[j] > -INFINITY && b[j] > -INFINITY;
        if (!group_has(__ballot(able), g, n)) mine = -INFINITY;
      }
      const float clear = 2 * near_of(a) + kNearOfSize * wave_max_f32(g >= a.groups ? 0.f : rank_size(mine, t1, t2, two));
      int before = 0, maybe = 0;  // groups that are better, and that could be
      for (int o = 0; o < a.groups; ++o) {
        const float its = f32_of((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(mine), o << n));
        before += o != g && its - mine > clear;
        maybe += o != g && !(mine - its > clear);
      }
      odd |= g < a.groups && before < a.top_groups && maybe >= a.top_groups;
      if (before >= a.top_groups)
#pragma unroll
        for (int j = 0; j < S; ++j) key[j] = 0;
    }
  } else if (a.groups > 1) {  // by their largest logits, which are exact
    uint32_t best = 0;
#pragma unroll
    for (int j = 0; j < S; ++j) best = key[j] > best ? key[j] : best;
    for (int d = 0; d < p.lanes_log2; ++d) {
      const uint32_t o = __shfl_xor(best, 1 << d);
      best = o > best ? o : best;
    }
    if (best == 1u) best = key_of(-INFINITY);  // (no numbers rank as -inf)
    int before = 0;
    for (int o = 0; o < a.groups; ++o) {
      const uint32_t its = (uint32_t)__builtin_amdgcn_readlane((int)best, o << p.lanes_log2);
      before += its > best || (its == best && o < g);
    }
    if (before >= a.top_groups)
#pragma unroll
      for (int j = 0; j < S; ++j) key[j] = 0;
  }
  uint32_t id = 0;
  bool exact = false;
  if (!KEYS || !__any(odd)) {
    float last = 0.f;
    bool near = false;
    const int rounds = KEYS && a.bias ? a.k + 1 : a.k;  // (the first that is not chosen has to be clear of the last that is)
    for (int r = 0; r < rounds; ++r) {
      uint32_t best = key[0];
#pragma unroll
      for (int j = 1; j < S; ++j) best = key[j] > best ? key[j] : best;
      const uint32_t top = wave_max_u32(best);
      if (KEYS && a.bias) {
        if (top == 0) break;  // (no more than were chosen)
        const float now = f32_of((top >> 31) ? top & 0x7fffffffu : ~top);
        near |= r > 0 && !(last - now > near_of(a) + kNearOfSize * fabsf(last));
        last = now;
      }
      const int owner = __builtin_ctzll(__ballot(best == top));
      int at = 0;
#pragma unroll
      for (int j = S - 1; j >= 0; --j)
        if (key[j] == top) at = j;
      const uint32_t chosen = (uint32_t)__builtin_amdgcn_readlane(x.base + at, owner);
#pragma unroll
      for (int j = 0; j < S; ++j)
        if (lane == owner && j == at) key[j] = 0;
      if (lane == r) id = chosen;
    }
    exact = near;
  } else {
    exact = true;
  }
  if constexpr (KEYS) {
    if (exact) select_exact<S>(p, x, g, id);
  }
  const bool mine = lane < a.k;
  const float logit = mine ? as_f32(row[id]) : -INFINITY;
  if (!SUM && a.scoring == 0) most = wave_max_f32(logit);
  const double score = mine ? score_of(a, logit, most, total) : 0.0;
  const double sum = wave_sum_f64(score);
  put_choice(a, t, lane, id, score, sum);
}

// ---------------------------------------------------------------- up to 16 groups and 16 choices: a row of 16 lanes a token
// The same choice with four tokens in a wave and up to 32 experts a lane: what a round of the choice exchanges between lanes stays in a row, and a wave's instructions serve four
// tokens.  Candidates whose order floats do not decide are ordered by their double scores; where they do not decide which those are, the whole wave goes over the token in double, a token
// after the other.  It takes over where there is a wave for each SIMD.  us, a row / a wave a token, bf16 logits but for the groups, of 2048, 4096 and 8192 tokens that floats decide:
//   128 experts, 8 chosen               4.6 / 4.5    4.7 / 5.5    5.3 / 7.5
//   512, 10                             8.7 / 6.8    8.8 / 9.7   11.0 / 15.6
//   256, 8, sigmoid, bias               9.2 / 6.9    9.4 / 8.8   10.8 / 12.7
//   256, 8, sigmoid, bias, 8 groups    10.4 / 7.7   10.7 / 10.1  12.2 / 14.6
//   512, 16, sigmoid, bias             16.5 / 12.2  16.9 / 17.8  21.6 / 27.8
// and of random ones, some of which (0.006 % to be gone over by a row's wave in the fourth line, 0.05 % to be ordered; all of those to be gone over where a wave has a token) floats do not:
//   256, 8, sigmoid, bias               9.5 / 9.0    9.5 / 10.9  10.7 / 13.3
//   256, 8, sigmoid, bias, 8 groups    10.6 / 11.0  14.0 / 11.1  13.9 / 16.5
//   512, 16, sigmoid, bias             23.7 / 18.5  23.7 / 23.7  28.4 / 33.6
// 8192 tokens of 256 float32 logits are 8.4 MB, 1.7 us of a copy's traffic.  What bounds the choice is the length of a wave's chain, not what the chip issues: four times the tokens take 1.2
// times as long (a round for each chosen, each over all of a lane's experts and then over the row; the weights' double exponentials), and a wave that goes over a token in double, 2 to 7 us longer, ends last.
constexpr int64_t kSelectWaves = 1024;
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  uint32_t o;
  o = dpp_u32<kDppXor1>(v); v = o > v ? o : v;
  o = dpp_u32<kDppXor2>(v); v = o > v ? o : v;
  o = dpp_u32<kDppHalfMirror>(v); v = o > v ? o : v;
  o = dpp_u32<kDppMirror>(v); v = o > v ? o : v;
  return v;
}
__device__ __forceinline__ uint32_t row_min(uint32_t v) { return ~row_max(~v); }
template <class F>
__device__ __forceinline__ float row_join(float v, F f) {
  v = f(v, f32_of(dpp_u32<kDppXor1>(__float_as_uint(v))));
  v = f(v, f32_of(dpp_u32<kDppXor2>(__float_as_uint(v))));
  v = f(v, f32_of(dpp_u32<kDppHalfMirror>(__float_as_uint(v))));
  return f(v, f32_of(dpp_u32<kDppMirror>(__float_as_uint(v))));
}
__device__ __forceinline__ double row_sum(double v) {
  v += dpp_f64<kDppXor1>(v);
  v += dpp_f64<kDppXor2>(v);
  v += dpp_f64<kDppHalfMirror>(v);
  return v + dpp_f64<kDppMirror>(v);
}
// f(n, v of the lane n places before in the row) for n = 1 .. 15
template <int N = 1, class F>
__device__ __forceinline__ void each_other(float v, F f) {
  if constexpr (N < 16) {
    f(N, f32_of(dpp_u32<0x120 + N>(__float_as_uint(v))));
    each_other<N + 1>(v, f);
  }
}
template <int N = 1, class F>
__device__ __forceinline__ void each_candidate(double v, uint32_t id, F f) {
  if constexpr (N < 16) {
    f(dpp_f64<0x120 + N>(v), dpp_u32<0x120 + N>(id));
    each_candidate<N + 1>(v, id, f);
  }
}

template <int DT, int S, bool KEYS, bool SUM>
__global__ __launch_bounds__(256) void select_rows_kernel(SelectKernelArgs p, SelectKernelArgs whole) {  // whole: the layout of a wave a token
  const SelectArgs &a = p.a;
  const int64_t t0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 4, t = t0 + (lane_id() >> 4);
  if (t0 >= a.T) return;
  const int lane = lane_id() & 15, g = lane >> p.lanes_log2, from = (lane & ((1 << p.lanes_log2) - 1)) * p.slots, base = g * p.size + from;
  const Logit<DT> *const row = static_cast<const Logit<DT> *>(a.logits) + (t < a.T ? t : a.T - 1) * a.E;  // (tokens outside: the last one's, not stored)
  const int n_mine = g < a.groups ? (p.size - from < p.slots ? p.size - from : p.slots) : 0;  // this lane's experts
  float l[S];
  if (p.slots == S && n_mine == S) {
    Logit<DT> v[S];
    __builtin_memcpy(v, row + base, sizeof v);
#pragma unroll
    for (int j = 0; j < S; ++j) l[j] = as_f32(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < S; ++j) l[j] = j < n_mine ? as_f32(row[base + j]) : -INFINITY;
  }
  float b[S];
  bool odd = false, masks = false;  // masks: one of the four tokens' logits is -inf
  if constexpr (KEYS) {
    if (a.bias && p.slots == S && n_mine == S) {
      __builtin_memcpy(b, a.bias + base, sizeof b);
    } else {
#pragma unroll
      for (int j = 0; j < S; ++j) b[j] = a.bias && j < n_mine ? a.bias[base + j] : 0.f;
    }
    float least = INFINITY;
    if (n_mine == S) {
#pragma unroll
      for (int j = 0; j < S; ++j) least = fminf(least, l[j]);
    } else {
#pragma unroll
      for (int j = 0; j < S; ++j)
        if (j < n_mine) least = fminf(least, l[j]);
    }
    masks = __any(least == -INFINITY);
#pragma unroll
    for (int j = 0; j < S; ++j) odd |= j < n_mine && not_below(l[j], b[j]);
  }
  auto larger = [](float x, float y) { return fmaxf(x, y); };
  float most = -INFINITY;
  if (SUM || (KEYS && a.scoring == 0)) {
#pragma unroll
    for (int j = 0; j < S; ++j) most = fmaxf(most, l[j]);
    most = row_join(most, larger);
    if constexpr (KEYS) odd |= a.scoring == 0 && most == -INFINITY;
  }
  double total = 1.0;
  if constexpr (SUM) {
    total = 0.0;
#pragma unroll
    for (int j = 0; j < S; ++j)
      if (l[j] == l[j] && most > -INFINITY) total += exp((double)l[j] - (double)most);
    total = row_sum(total);
  }
  uint32_t key[S];
  if (!KEYS || !a.bias) {
#pragma unroll
    for (int j = 0; j < S; ++j) key[j] = j < n_mine ? key_of(l[j]) : 0;
  }
  const bool two = a.groups > 1 && a.group_score == 1 && p.size > 1;
  float y[S];  // what groups are ranked by
#pragma unroll
  for (int j = 0; j < S; ++j) y[j] = l[j] == l[j] ? l[j] : -INFINITY;  // (no numbers rank as -inf)
  if constexpr (KEYS) {
    if (a.bias || a.group_score == 1) {
      if (a.scoring == 0) {
        float sum[4] = {0.f, 0.f, 0.f, 0.f};  // (of up to eight, so that no addend goes through more than 14 roundings)
#pragma unroll
        for (int j = 0; j < S; ++j) {
          y[j] = __expf(l[j] - most);
          sum[j % 4] += y[j];
        }
        const float inv = __builtin_amdgcn_rcpf(row_join((sum[0] + sum[1]) + (sum[2] + sum[3]), [](float u, float v) { return u + v; }));
#pragma unroll
        for (int j = 0; j < S; ++j) y[j] = __builtin_fmaf(y[j], inv, b[j]);
      } else {
#pragma unroll
        for (int j = 0; j < S; ++j) y[j] = __builtin_amdgcn_rcpf(1.0f + __expf(-l[j])) + b[j];
      }
      if (a.bias) {
#pragma unroll
        for (int j = 0; j < S; ++j) key[j] = j < n_mine ? key_of(y[j]) : 0;
      }
      if (masks) {  // (ranked by two, they have a score of zero)
#pragma unroll
        for (int j = 0; j < S; ++j)
          if (j < n_mine && l[j] == -INFINITY) {
            key[j] = key_of(-INFINITY);
            if (!two) y[j] = -INFINITY;
          }
      }
    }
  }
  if (a.groups > 1) {
    float t1 = -INFINITY, t2 = -INFINITY;
#pragma unroll
    for (int j = 0; j < S; ++j) {
      const float v = j < n_mine ? y[j] : -INFINITY;
      t2 = fmaxf(t2, fminf(t1, v));
      t1 = fmaxf(t1, v);
    }
    const int n = p.lanes_log2;
    auto other = [&](auto ctrl) __attribute__((always_inline)) {
      constexpr int CTRL = decltype(ctrl)::value;
      merge_two(t1, t2, f32_of(dpp_u32<CTRL>(__float_as_uint(t1))), f32_of(dpp_u32<CTRL>(__float_as_uint(t2))));
    };
    if (n > 0) other(std::integral_constant<int, kDppXor1>{});
    if (n > 1) other(std::integral_constant<int, kDppXor2>{});
    if (n > 2) other(std::integral_constant<int, kDppHalfMirror>{});
    if (t2 == -INFINITY) t2 = 0.f;
    float mine = two ? t1 + t2 : t1;
    if (two && masks) {  // (where no logit is masked, a group of masked ones has nothing but biases of -inf)
      bool able = false;
#pragma unroll
      for (int j = 0; j < S; ++j) able |= j < n_mine && l[j] > -INFINITY && b[j] > -INFINITY;
      if (!group_has(__ballot(able) >> (lane_id() & 48), g, n)) mine = -INFINITY;
    }
    float clear = 0.f;
    if constexpr (KEYS) clear = 2 * near_of(a) + kNearOfSize * row_join(g >= a.groups ? 0.f : rank_size(mine, t1, t2, two), larger);
    int before = 0, maybe = 0;  // lanes of groups that are better, and that could be
    each_other(mine, [&](int n_back, float its) __attribute__((always_inline)) {
      const int og = ((lane - n_back) & 15) >> n;
      const bool another = og != g && og < a.groups;
      if constexpr (KEYS) {
        before += another && its - mine > clear;
        maybe += another && !(mine - its > clear);
      } else {
        before += another && (its > mine || (its == mine && og < g));
      }
    });
    if constexpr (KEYS) odd |= g < a.groups && before >> n < a.top_groups && maybe >> n >= a.top_groups;
    if (before >> n >= a.top_groups)
#pragma unroll
      for (int j = 0; j < S; ++j) key[j] = 0;
  }
  // With a bias the choice goes on to one more candidate, in a lane as the others, and to the key after that one: where that is clearly below the last of the k, floats have
  // found the candidates and doubles their order.
  const int candidates = KEYS && a.bias ? (a.k < 16 ? a.k + 1 : 16) : a.k;
  uint32_t id = (uint32_t)(a.E + lane);  // (no expert)
  float last = 0.f, kth = 0.f;
  bool close = false;
#pragma unroll 1
  for (int r = 0; r < candidates + (KEYS && a.bias); ++r) {
    uint32_t best = key[0];
#pragma unroll
    for (int j = 1; j < S; ++j) best = key[j] > best ? key[j] : best;
    const uint32_t top = row_max(best);
    if (KEYS && a.bias) {
      const float now = f32_of((top >> 31) ? top & 0x7fffffffu : ~top);
      if (r == a.k - 1) kth = now;
      const float clear = near_of(a) + kNearOfSize * fabsf(r == candidates ? kth : last);
      if (r == candidates) odd |= top != 0 && !(kth - now > clear);
      else close |= r > 0 && top != 0 && !(last - now > clear);
      last = now;
    }
    uint32_t at = ~0u;
#pragma unroll
    for (int j = S - 1; j >= 0; --j)
      if (key[j] == top) at = (uint32_t)(base + j);
    const uint32_t chosen = row_min(at);
#pragma unroll
    for (int j = 0; j < S; ++j)
      if (chosen == (uint32_t)(base + j)) key[j] = 0;
    if (lane == r && top != 0) id = chosen;
  }
  const bool named = id < (uint32_t)a.E;
  const float logit = named ? as_f32(row[id]) : -INFINITY;
  if (!SUM && a.scoring == 0) most = row_join(lane < a.k ? logit : -INFINITY, larger);
  double score = named ? score_of(a, logit, most, total) : 0.0;
  if constexpr (KEYS) {
    if (__ballot(close)) {
      if (a.scoring == 0 && !SUM) {
        odd |= close;
      } else {
        const double v = named && a.bias && logit != -INFINITY ? score + (double)a.bias[id] : -INFINITY;
        int rank = 0;
        each_candidate(v, id, [&](double its, uint32_t other) __attribute__((always_inline)) { rank += its > v || (its == v && other < id); });
        if (close) {
          const int to = ((lane_id() & 48) + rank) * 4;
          id = (uint32_t)__builtin_amdgcn_ds_permute(to, (int)id);
          const uint64_t u = (uint64_t)__double_as_longlong(score);
          score = __longlong_as_double((int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_ds_permute(to, (int)(u >> 32)) << 32 | (uint32_t)__builtin_amdgcn_ds_permute(to, (int)u)));
        }
      }
    }
  }
  const double sum = row_sum(lane < a.k ? score : 0.0);
  uint64_t again = KEYS ? __ballot(odd) : 0;
  if (t < a.T && (again >> (lane_id() & 48) & 0xffff) == 0) put_choice(a, t, lane, id, score, sum);
  if constexpr (KEYS) {
    for (; again; again &= ~((uint64_t)0xffff << (__builtin_ctzll(again) & 48))) {
      const int64_t tt = t0 + (__builtin_ctzll(again) >> 4);
      if (tt >= a.T) continue;
      const Logit<DT> *const its = static_cast<const Logit<DT> *>(a.logits) + tt * a.E;
      const int wl = lane_id(), wg = wl >> whole.lanes_log2, wf = (wl & ((1 << whole.lanes_log2) - 1)) * whole.slots;
      Slots<S / 4> x;  // (a wave has four times the lanes)
      x.base = wg * whole.size + wf;
#pragma unroll
      for (int j = 0; j < S / 4; ++j) {
        x.on[j] = j < whole.slots && wf + j < whole.size && wg < a.groups;
        x.l[j] = x.on[j] ? as_f32(its[x.base + j]) : -INFINITY;
      }
      uint32_t eid = 0;
      select_exact<S / 4>(whole, x, wg, eid);
      const int from_lane = (int)(tt - t0) * 16;  // (of its row)
      const float el = wl < a.k ? as_f32(its[eid]) : -INFINITY;
      const float em = SUM ? f32_of((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(most), from_lane)) : wave_max_f32(el);
      const double es = wl < a.k ? score_of(a, el, em, SUM ? readlane_f64(total, from_lane) : 1.0) : 0.0;
      put_choice(a, tt, wl, eid, es, wave_sum_f64(es));
    }
  }
}

template <int DT, bool KEYS, bool SUM>
static hipError_t start_rows(const SelectKernelArgs &p, const SelectKernelArgs &whole, hipStream_t st) {
  const unsigned grid = (unsigned)((p.a.T + 15) / 16);
  if (p.slots <= 4) select_rows_kernel<DT, 4, KEYS, SUM><<<grid, 256, 0, st>>>(p, whole);
  else if (p.slots <= 8) select_rows_kernel<DT, 8, KEYS, SUM><<<grid, 256, 0, st>>>(p, whole);
  else if (p.slots <= 16) select_rows_kernel<DT, 16, KEYS, SUM><<<grid, 256, 0, st>>>(p, whole);
  else select_rows_kernel<DT, 32, KEYS, SUM><<<grid, 256, 0, st>>>(p, whole);
  return hipGetLastError();
}

template <int DT, bool KEYS, bool SUM>
static hipError_t start_select(const SelectKernelArgs &p, hipStream_t st) {
  const unsigned grid = (unsigned)((p.a.T + 3) / 4);
  if (p.slots <= 1) select_experts_kernel<DT, 1, KEYS, SUM><<<grid, 256, 0, st>>>(p);
  else if (p.slots <= 2) select_experts_kernel<DT, 2, KEYS, SUM><<<grid, 256, 0, st>>>(p);
  else if (p.slots <= 4) select_experts_kernel<DT, 4, KEYS, SUM><<<grid, 256, 0, st>>>(p);
  else if (p.slots <= 8) select_experts_kernel<DT, 8, KEYS, SUM><<<grid, 256, 0, st>>>(p);
  else select_experts_kernel<DT, 16, KEYS, SUM><<<grid, 256, 0, st>>>(p);
  return hipGetLastError();
}

constexpr int64_t kSelectMost = (int64_t)1 << 25;  // tokens of a launch
hipError_t launch_select_experts(const SelectArgs &a, int dt, hipStream_t st) {
  if (a.T == 0) return hipSuccess;
  if (a.T > kSelectMost) {  // (a launch has less than 2^32 threads)
    SelectArgs some = a;
    const int64_t size = dt == 2 ? 4 : 2, w_size = a.w_dtype == 2 ? 4 : 2;
    for (int64_t t = 0; t < a.T; t += kSelectMost) {
      some.logits = static_cast<const char *>(a.logits) + t * a.E * size;
      some.idx = a.idx + t * a.k;
      some.w = static_cast<char *>(a.w) + t * a.k * w_size;
      some.T = a.T - t < kSelectMost ? a.T - t : kSelectMost;
      if (hipError_t e = launch_select_experts(some, dt, st); e != hipSuccess) return e;
    }
    return hipSuccess;
  }
  auto layout = [&](int lanes_log2) {
    SelectKernelArgs p{a, a.E / a.groups, lanes_log2, 0};
    while (p.lanes_log2 > 0 && (1 << (lanes_log2 - p.lanes_log2)) < a.groups) --p.lanes_log2;  // lanes of a group
    p.slots = (p.size + (1 << p.lanes_log2) - 1) >> p.lanes_log2;
    return p;
  };
  const SelectKernelArgs p = layout(6), four = layout(4);  // p.slots: 16 at most (512 experts, and runs of lanes that leave less than half of the wave idle)
  const bool rows = a.groups <= 16 && four.slots <= 32 && a.k <= 16 && a.T >= 4 * kSelectWaves;
  const bool keys = a.bias || (a.groups > 1 && a.group_score == 1), sum = a.scoring == 0 && !a.renormalize;
  auto start = [&](auto d) {
    constexpr int DT = decltype(d)::value;
    if (rows && keys) return sum ? start_rows<DT, true, true>(four, p, st) : start_rows<DT, true, false>(four, p, st);
    if (rows) return sum ? start_rows<DT, false, true>(four, p, st) : start_rows<DT, false, false>(four, p, st);
    if (keys) return sum ? start_select<DT, true, true>(p, st) : start_select<DT, true, false>(p, st);
    return sum ? start_select<DT, false, true>(p, st) : start_select<DT, false, false>(p, st);
  };
  if (dt == 0) return start(std::integral_constant<int, 0>{});
  if (dt == 1) return start(std::integral_constant<int, 1>{});
  return start(std::integral_constant<int, 2>{});
}

// ---------------------------------------------------------------- the gradient
// A wave a token: the chosen experts' terms in a lane each, then the row of results.  An id outside the experts has no part in it.  For softmax scores that are not renormalised, in which every
// logit has a part (its exponential is computed once and kept in LDS: 8192 x 256 12.2 us, 14.8 without), and for more than 16 chosen.
template <int DT>
__global__ __launch_bounds__(256) void select_grad_kernel(SelectGradArgs a) {
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= a.T) return;
  const int lane = lane_id();
  const Logit<DT> *const row = static_cast<const Logit<DT> *>(a.logits) + t * a.E;
  const uint32_t id = lane < a.k ? a.idx[t * a.k + lane] : ~0u;
  const bool on = id < (uint32_t)a.E;
  const double l = on ? (double)as_f32(row[id]) : -INFINITY;
  const double g = on ? (double)a.scale * (double)get_value(a.dw, t * a.k + lane, a.w_dtype) : 0.0;
  const bool whole = a.scoring == 0 && !a.renormalize;  // every expert's score has a part
  __shared__ double rows[4][512];
  double *const out = rows[threadIdx.x >> 6];
  float most = -INFINITY;
  double total = 0.0;
  if (whole) {
    for (int c = lane; c < a.E; c += kWave) most = fmaxf(most, as_f32(row[c]));
    most = wave_max_f32(most);
    for (int c = lane; c < a.E; c += kWave) {
      const float x = as_f32(row[c]);
      const double e = x != x ? NAN : most == -INFINITY ? 0.0 : exp((double)x - (double)most);
      if (x == x) total += e;
      out[c] = e;
    }
    total = wave_sum_f64(total);
  } else if (a.scoring == 0) {
    most = wave_max_f32(on ? (float)l : -INFINITY);
  }
  const double s = !on ? 0.0 : a.scoring == 1 ? sigmoid64(l) : l != l ? NAN : most == -INFINITY ? 0.0 : whole ? exp(l - (double)most) / total : exp(l - (double)most);
  double inner;  // score times the gradient with respect to it
  if (a.renormalize) {
    const double sum = wave_sum_f64(s);
    const double share = sum == 0.0 ? 0.0 : s / sum;
    inner = share * (g - wave_sum_f64(share * g));
  } else {
    inner = s * g;
  }
  const double dot = whole ? wave_sum_f64(inner) : 0.0;
  if (a.scoring == 1) inner *= sigmoid64(-l);
  // the row: zeros, and a chosen expert's term (of one named twice the sum, in slot order, by the first) where it belongs
  const double factor = total > 0.0 || total != total ? -dot / total : 0.0;
  for (int c = lane; c < a.E; c += kWave) out[c] = whole ? factor * out[c] : 0.0;
  double mine = inner;
  bool first = on;
  for (int r = 0; r < a.k; ++r) {
    const uint32_t at = (uint32_t)__builtin_amdgcn_readlane((int)id, r);
    const double its = readlane_f64(inner, r);
    if (at == id && r < lane) first = false;
    if (at == id && r > lane) mine += its;
  }
  __builtin_amdgcn_wave_barrier();
  if (first) out[id] += mine;
  __builtin_amdgcn_wave_barrier();
  for (int c = lane; c < a.E; c += kWave) put_value(a.dlogits, t * a.E + c, DT, out[c]);
}

// The same where only the chosen experts' logits have a part, up to 16 of them: a row of 16 lanes a token, so that a wave's double exponentials serve four; the results of the four tokens lie
// behind each other, pass through LDS in their type, zeros but for the chosen, and leave in 16-byte stores.  us, a row / a wave a token: 32 tokens of 128 experts 4.0 / 4.5, 8192
// of 128, 256 (float32) and 512 with 16 chosen 4.4 / 7.5, 5.6 / 8.8, 5.8 / 11.9 (8.4 MB each of the last two: 1.7 of a copy's traffic).
template <int N = 15, class F>
__device__ __forceinline__ void each_chosen(double v, uint32_t tag, F f) {
  if constexpr (N > 0) {
    f(dpp_f64<0x120 + N>(v), dpp_u32<0x120 + N>(tag));
    each_chosen<N - 1>(v, tag, f);
  }
}
template <int DT>
__global__ __launch_bounds__(256) void select_grad_rows_kernel(SelectGradArgs a) {
  using Raw = Logit<DT>;
  extern __shared__ __align__(16) unsigned char grad_raw[];
  const int64_t t0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 4, t = t0 + (lane_id() >> 4);
  if (t0 >= a.T) return;
  const int lane = lane_id() & 15, share_bytes = (4 * a.E * (int)sizeof(Raw) + 15) & ~15;
  unsigned char *const out = grad_raw + (threadIdx.x >> 6) * share_bytes;
  const uint4 zeros = make_uint4(0, 0, 0, 0);  // (LDS is bytes, which the accesses of either width copy)
  for (int c = lane_id() * 16; c < share_bytes; c += kWave * 16) __builtin_memcpy(__builtin_assume_aligned(out + c, 16), &zeros, 16);
  const uint32_t id = lane < a.k && t < a.T ? a.idx[t * a.k + lane] : ~0u;
  const bool on = id < (uint32_t)a.E;
  const float l = on ? as_f32(static_cast<const Raw *>(a.logits)[t * a.E + id]) : -INFINITY;
  const double g = on ? (double)a.scale * (double)get_value(a.dw, t * a.k + lane, a.w_dtype) : 0.0;
  float most = -INFINITY;
  if (a.scoring == 0) most = row_join(l, [](float x, float y) { return fmaxf(x, y); });
  const double s = !on ? 0.0 : a.scoring == 1 ? sigmoid64(l) : l != l ? NAN : most == -INFINITY ? 0.0 : exp((double)l - (double)most);
  double inner;
  if (a.renormalize) {
    const double sum = row_sum(s), share = sum == 0.0 ? 0.0 : s / sum;
    inner = share * (g - row_sum(share * g));
  } else {
    inner = s * g;
  }
  if (a.scoring == 1) inner *= sigmoid64(-l);
  const uint32_t tag = (uint32_t)lane << 16 | (on ? id : 0xffffu);  // (ids are below 512)
  double mine = inner;
  bool first = on;
  each_chosen(inner, tag, [&](double its, uint32_t other) __attribute__((always_inline)) {
    const bool same = (other & 0xffffu) == id;
    first &= !(same && other < tag);
    if (same && other > tag) mine += its;
  });
  __builtin_amdgcn_wave_barrier();
  if (first) {
    Raw raw;
    put_value(&raw, 0, DT, mine);
    __builtin_memcpy(__builtin_assume_aligned(out + ((lane_id() >> 4) * a.E + (int)id) * (int)sizeof(Raw), sizeof(Raw)), &raw, sizeof(Raw));
  }
  __builtin_amdgcn_wave_barrier();
  const int bytes = (int)(a.T - t0 < 4 ? a.T - t0 : 4) * a.E * (int)sizeof(Raw);
  unsigned char *const to = static_cast<unsigned char *>(a.dlogits) + t0 * a.E * (int64_t)sizeof(Raw);
  for (int c = lane_id() * 16; c < bytes; c += kWave * 16) {
    if (c + 16 <= bytes) {
      uint4 v;
      __builtin_memcpy(&v, __builtin_assume_aligned(out + c, 16), 16);
      __builtin_memcpy(__builtin_assume_aligned(to + c, sizeof(Raw)), &v, 16);
    } else {
      for (int i = c; i < bytes; i += (int)sizeof(Raw))
        __builtin_memcpy(__builtin_assume_aligned(to + i, sizeof(Raw)), __builtin_assume_aligned(out + i, sizeof(Raw)), sizeof(Raw));
    }
  }
}

hipError_t launch_select_grad(const SelectGradArgs &a, int dt, hipStream_t st) {
  if (a.T == 0) return hipSuccess;
  if (a.T > kSelectMost) {
    SelectGradArgs some = a;
    const int64_t size = dt == 2 ? 4 : 2, w_size = a.w_dtype == 2 ? 4 : 2;
    for (int64_t t = 0; t < a.T; t += kSelectMost) {
      some.logits = static_cast<const char *>(a.logits) + t * a.E * size;
      some.dlogits = static_cast<char *>(a.dlogits) + t * a.E * size;
      some.idx = a.idx + t * a.k;
      some.dw = static_cast<const char *>(a.dw) + t * a.k * w_size;
      some.T = a.T - t < kSelectMost ? a.T - t : kSelectMost;
      if (hipError_t e = launch_select_grad(some, dt, st); e != hipSuccess) return e;
    }
    return hipSuccess;
  }
  if (a.k <= 16 && (a.renormalize || a.scoring == 1)) {
    const unsigned rows = (unsigned)((a.T + 15) / 16), lds = 4 * ((4 * a.E * (dt == 2 ? 4 : 2) + 15) & ~15);
    if (dt == 0) select_grad_rows_kernel<0><<<rows, 256, lds, st>>>(a);
    else if (dt == 1) select_grad_rows_kernel<1><<<rows, 256, lds, st>>>(a);
    else select_grad_rows_kernel<2><<<rows, 256, lds, st>>>(a);
    return hipGetLastError();
  }
  const unsigned grid = (unsigned)((a.T + 3) / 4);
  if (dt == 0) select_grad_kernel<0><<<grid, 256, 0, st>>>(a);
  else if (dt == 1) select_grad_kernel<1><<<grid, 256, 0, st>>>(a);
  else select_grad_kernel<2><<<grid, 256, 0, st>>>(a);
  return hipGetLastError();
}

// ---------------------------------------------------------------- a routing that the caller brings
// A wave a token copies the ids and weights into the workspace, and makes of them what the dispatch and the products rely on: k different experts.  A token's
// second mention of an expert is added to the first (in slot order, one rounding), an id outside the experts is dropped; what then stands in the slot is an expert
// that the token does not name, with a weight (kNoSlot, a zero) at which the sum over the slots passes over its result: zero times that would be no number where it is not finite.
__global__ __launch_bounds__(256) void check_routing_kernel(const uint32_t *idx, const uint16_t *w, int64_t T, int E, int k, uint32_t *idx_out, uint16_t *w_out) {
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= T) return;
  const int lane = lane_id();
  uint32_t id = lane < k ? idx[t * k + lane] : ~0u;
  float weight = lane < k ? bf16_to_f32(w[t * k + lane]) : 0.f;
  bool bad = lane < k && id >= (uint32_t)E, merged = false;
  float sum = weight;
  for (int r = 0; r < k; ++r) {
    const uint32_t other = (uint32_t)__builtin_amdgcn_readlane((int)id, r);
    const float its = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(weight), r));
    if (lane < k && other == id && id < (uint32_t)E) {
      if (r < lane) bad = true;
      else if (r > lane) sum += its, merged = true;
    }
  }
  if (merged) weight = sum;
  uint64_t left = __ballot(bad);
  if (left) {
    const uint32_t named = bad ? ~0u : id;
    for (uint32_t c = 0; left && c < (uint32_t)E; ++c) {  // (k is E at most: there is one for each)
      if (__ballot(lane < k && named == c)) continue;
      const int to = __builtin_ctzll(left);
      left &= left - 1;
      if (lane == to) id = c;
    }
  }
  if (lane < k) {
    idx_out[t * k + lane] = id;
    const uint16_t w16 = f32_to_bf16(weight);
    w_out[t * k + lane] = bad ? kNoSlot : w16 == kNoSlot ? (uint16_t)0 : w16;
  }
}

hipError_t launch_check_routing(const uint32_t *idx, const uint16_t *w, int64_t T, int E, int k, uint32_t *idx_out, uint16_t *w_out, hipStream_t st) {
  check_routing_kernel<<<(unsigned)((T + 3) / 4), 256, 0, st>>>(idx, w, T, E, k, idx_out, w_out);
  return hipGetLastError();
}

}  // namespace mi_moe
