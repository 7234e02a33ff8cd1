// Experts of every token from the router's logits, with softmax or sigmoid scores, a bias that takes part in the choice alone, and groups of
// experts of which the best are open; the gradient of the weights; and the check of a routing that a caller brings.
//
//   s = softmax(l) over the experts, or 1 / (1 + exp(-l))           key = l without a bias, s + b with one
//   a group's rank: its largest key, or the sum of its two largest s + b     the best `top_groups` groups are open
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

// A wave a token.  A group of experts goes to a run of lanes, consecutive experts to a lane, so that lanes and slots are in the order of the ids.
template <int DT, class Key, int S>
__global__ __launch_bounds__(256) void select_experts_kernel(SelectKernelArgs p) {
  const SelectArgs &a = p.a;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= a.T) return;
  const int lane = lane_id(), g = lane >> p.lanes_log2, from = (lane & ((1 << p.lanes_log2) - 1)) * p.slots;
  const Logit<DT> *const row = static_cast<const Logit<DT> *>(a.logits) + t * a.E;
  float l[S];
  double v[S];  // scores, then scores with the bias
  Key key[S];
  bool on[S];
#pragma unroll
  for (int j = 0; j < S; ++j) {
    on[j] = j < p.slots && from + j < p.size && g < a.groups;
    l[j] = on[j] ? as_f32(row[g * p.size + from + j]) : -INFINITY;
  }
  float most = -INFINITY;  // (fmaxf passes over what is no number)
  double total = 0.0;
  if (a.scoring == 0) {
#pragma unroll
    for (int j = 0; j < S; ++j) most = fmaxf(most, l[j]);
    most = wave_max_f32(most);
#pragma unroll
    for (int j = 0; j < S; ++j) {
      v[j] = most == -INFINITY ? 0.0 : exp((double)l[j] - (double)most);
      total += v[j] == v[j] || l[j] == l[j] ? v[j] : 0.0;
    }
    total = wave_sum_f64(total);
#pragma unroll
    for (int j = 0; j < S; ++j) v[j] = l[j] != l[j] ? NAN : total > 0.0 || total != total ? v[j] / total : 0.0;
  } else {
#pragma unroll
    for (int j = 0; j < S; ++j) v[j] = sigmoid64(l[j]);
  }
  double s[S];
#pragma unroll
  for (int j = 0; j < S; ++j) {
    s[j] = v[j];
    if (a.bias && on[j]) v[j] += (double)a.bias[g * p.size + from + j];
    if (l[j] == -INFINITY) v[j] = -INFINITY;
    if constexpr (sizeof(Key) == 8) key[j] = on[j] ? key_of(v[j]) : 0;
    else key[j] = on[j] ? key_of(l[j]) : 0;
  }
  if (a.groups > 1) {
    double t1 = -INFINITY, t2 = -INFINITY;  // the two largest of the group
#pragma unroll
    for (int j = 0; j < S; ++j) {
      double x = a.group_score == 0 && sizeof(Key) == 4 ? (double)l[j] : v[j];
      if (!on[j] || x != x) x = -INFINITY;
      t2 = fmax(t2, fmin(t1, x));
      t1 = fmax(t1, x);
    }
    for (int d = 0; d < p.lanes_log2; ++d) {
      const double o1 = __shfl_xor(t1, 1 << d), o2 = __shfl_xor(t2, 1 << d);
      t2 = fmax(fmin(t1, o1), fmax(t2, o2));
      t1 = fmax(t1, o1);
    }
    const uint64_t mine = key_of(a.group_score == 0 || p.size == 1 ? t1 : t1 + t2);
    int before = 0;
    for (int o = 0; o < a.groups; ++o) {
      const uint64_t other = readlane_key(mine, o << p.lanes_log2);
      before += other > mine || (other == mine && o < g);
    }
    if (before >= a.top_groups)
#pragma unroll
      for (int j = 0; j < S; ++j) key[j] = 0;
  }
  uint32_t id = 0;
  double score = 0.0;
  for (int r = 0; r < a.k; ++r) {
    Key best = 0;
    int at = 0;
    double sv = 0.0;
#pragma unroll
    for (int j = 0; j < S; ++j)
      if (key[j] > best) best = key[j], at = j, sv = s[j];
    const Key top = wave_max_key(best);
    const int owner = __builtin_ctzll(__ballot(best == top));
    if (lane == owner)
#pragma unroll
      for (int j = 0; j < S; ++j)
        if (j == at) key[j] = 0;
    const uint32_t chosen = (uint32_t)__builtin_amdgcn_readlane(g * p.size + from + at, owner);
    const double its = readlane_f64(sv, owner);
    if (lane == r) id = chosen, score = its;
  }
  double w = score;
  if (a.renormalize) {
    const double sum = wave_sum_f64(lane < a.k ? score : 0.0);
    w = sum == 0.0 ? 0.0 : score / sum;
  }
  if (lane < a.k) {
    a.idx[t * a.k + lane] = id;
    put_value(a.w, t * a.k + lane, a.w_dtype, w * (double)a.scale);
  }
}

template <int DT, class Key>
static hipError_t start_select(const SelectKernelArgs &p, hipStream_t st) {
  const unsigned grid = (unsigned)((p.a.T + 3) / 4);
  if (p.slots <= 1) select_experts_kernel<DT, Key, 1><<<grid, 256, 0, st>>>(p);
  else if (p.slots <= 2) select_experts_kernel<DT, Key, 2><<<grid, 256, 0, st>>>(p);
  else if (p.slots <= 4) select_experts_kernel<DT, Key, 4><<<grid, 256, 0, st>>>(p);
  else if (p.slots <= 8) select_experts_kernel<DT, Key, 8><<<grid, 256, 0, st>>>(p);
  else select_experts_kernel<DT, Key, 16><<<grid, 256, 0, st>>>(p);
  return hipGetLastError();
}

hipError_t launch_select_experts(const SelectArgs &a, int dt, hipStream_t st) {
  if (a.T == 0) return hipSuccess;
  SelectKernelArgs p{a, a.E / a.groups, 6, 0};
  while ((kWave >> p.lanes_log2) < a.groups) --p.lanes_log2;
  p.slots = (p.size + (1 << p.lanes_log2) - 1) >> p.lanes_log2;  // 16 at most: 512 experts, and runs of lanes that leave less than half of the wave idle
  auto start = [&](auto d) {
    constexpr int DT = decltype(d)::value;
    return a.bias ? start_select<DT, uint64_t>(p, st) : start_select<DT, uint32_t>(p, st);
  };
  if (dt == 0) return start(std::integral_constant<int, 0>{});
  if (dt == 1) return start(std::integral_constant<int, 1>{});
  return start(std::integral_constant<int, 2>{});
}

// ---------------------------------------------------------------- the gradient
// A wave a token: the chosen experts' terms in a lane each, then the row of results.  An id outside the experts has no part in it.
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
  float most = -INFINITY;
  double total = 0.0;
  if (whole) {
    for (int c = lane; c < a.E; c += kWave) most = fmaxf(most, as_f32(row[c]));
    most = wave_max_f32(most);
    for (int c = lane; c < a.E; c += kWave) {
      const float x = as_f32(row[c]);
      if (x == x && most > -INFINITY) total += exp((double)x - (double)most);
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
  for (int c0 = 0; c0 < a.E; c0 += kWave) {
    const int c = c0 + lane;
    double v = 0.0;
    if (whole && c < a.E) {
      const float x = as_f32(row[c]);
      v = x != x ? NAN : most == -INFINITY ? 0.0 : -dot * (exp((double)x - (double)most) / total);
    }
    for (int r = 0; r < a.k; ++r) {
      const uint32_t at = (uint32_t)__builtin_amdgcn_readlane((int)id, r);
      const double its = readlane_f64(inner, r);
      if (at == (uint32_t)c) v += its;
    }
    if (c < a.E) put_value(a.dlogits, t * a.E + c, DT, v);
  }
}

hipError_t launch_select_grad(const SelectGradArgs &a, int dt, hipStream_t st) {
  if (a.T == 0) return hipSuccess;
  const unsigned grid = (unsigned)((a.T + 3) / 4);
  if (dt == 0) select_grad_kernel<0><<<grid, 256, 0, st>>>(a);
  else if (dt == 1) select_grad_kernel<1><<<grid, 256, 0, st>>>(a);
  else select_grad_kernel<2><<<grid, 256, 0, st>>>(a);
  return hipGetLastError();
}

// ---------------------------------------------------------------- a routing that the caller brings
// A wave a token copies the ids and weights into the workspace, and makes of them what the dispatch and the products rely on: k different experts.  A token's
// second mention of an expert is added to the first (in slot order, one rounding), an id outside the experts is dropped; what then stands in the slot is an expert
// that the token does not name, with a weight of zero.
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
      if (lane == to) id = c, weight = 0.f;
    }
  }
  if (lane < k) {
    idx_out[t * k + lane] = id;
    w_out[t * k + lane] = f32_to_bf16(weight);
  }
}

hipError_t launch_check_routing(const uint32_t *idx, const uint16_t *w, int64_t T, int E, int k, uint32_t *idx_out, uint16_t *w_out, hipStream_t st) {
  check_routing_kernel<<<(unsigned)((T + 3) / 4), 256, 0, st>>>(idx, w, T, E, k, idx_out, w_out);
  return hipGetLastError();
}

}  // namespace mi_moe
