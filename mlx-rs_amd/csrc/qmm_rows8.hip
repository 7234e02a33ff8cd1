// Quantized linear layer on rows in eight bits: y [M, N] = (row_scale x [M, K]) . (scale code + bias)^T, each result rounded once.
//
// With x int8 and the codes centred (c' = c - 8 or c - 128, the bias with the centre's share beta = b + 8 s or b + 128 s)
//   y[m, n] = row_scale[m] * sum over groups of (s[n, g] sum_k x[m, k] c'[n, k] + beta[n, g] sum_k x[m, k]) + linear_bias[n]
// the sums over a group are integers and exact; what is in float is a term or two a group.  (The layer on 16-bit rows: mlx-rs/src/nn/quantized.rs:363-386.)
#include <type_traits>

#include "common.hpp"

namespace mi_moe {

// the four or eight codes of a word as signed bytes in their order, times 16 (4-bit codes: a nibble at the top of its byte with its first bit turned over is
// 16 (c - 8)) or as they are (8-bit)
template <int BITS>
__device__ __forceinline__ void centred_bytes(uint32_t w, int32_t (&c)[BITS == 4 ? 2 : 1]) {
  if constexpr (BITS == 4) {
    const uint32_t even = ((w << 4) & 0xf0f0f0f0u) ^ 0x80808080u, odd = (w & 0xf0f0f0f0u) ^ 0x80808080u;
    c[0] = (int32_t)__builtin_amdgcn_perm(odd, even, 0x05010400u);
    c[1] = (int32_t)__builtin_amdgcn_perm(odd, even, 0x07030602u);
  } else {
    c[0] = (int32_t)(w ^ 0x80808080u);
  }
}
template <int BITS>
struct Centre {
  static constexpr float value = BITS == 4 ? 8.f : 128.f, of_codes = BITS == 4 ? 16.f : 1.f;  // of_codes: what centred_bytes multiplies them by
};

template <int DT>
using Value = typename std::conditional<DT == 0, uint16_t, typename std::conditional<DT == 1, _Float16, float>::type>::type;
template <int DT>
__device__ __forceinline__ Value<DT> value_of(float v) {
  if constexpr (DT == 0) return f32_to_bf16(v);
  else return (Value<DT>)v;
}

// A wave a column and ROWS rows, lanes over the words of the weight row.  Any shape and alignment.
template <int DT, int BITS, int ROWS>
__global__ __launch_bounds__(256) void rows8_plain_kernel(Rows8Args a) {
  constexpr int PER = 32 / BITS;
  const int lane = lane_id();
  const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t n = wave % a.N, m0 = wave / a.N * ROWS;
  if (m0 >= a.M) return;
  const int words = a.K / PER, G = a.K / a.group;
  const uint32_t *const w = a.w + n * words;
  const Value<DT> *const s = static_cast<const Value<DT> *>(a.s) + n * G, *const b = static_cast<const Value<DT> *>(a.b) + n * G;
  float acc[ROWS] = {};
  for (int i = lane; i < words; i += kWave) {
    int32_t c[PER / 4];
    centred_bytes<BITS>(w[i], c);
    const int g = i * PER / a.group;
    const float sc = as_f32(s[g]), beta = __builtin_fmaf(Centre<BITS>::value, sc, as_f32(b[g])), sd = sc / Centre<BITS>::of_codes;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int64_t m = m0 + r < a.M ? m0 + r : a.M - 1;
      int32_t x[PER / 4], d = 0, sum = 0;
      __builtin_memcpy(x, a.x + m * a.K + i * PER, PER);
#pragma unroll
      for (int j = 0; j < PER / 4; ++j) {
        d = __builtin_amdgcn_sdot4(x[j], c[j], d, false);
        sum = __builtin_amdgcn_sdot4(x[j], 0x01010101, sum, false);
      }
      acc[r] = __builtin_fmaf(sd, (float)d, __builtin_fmaf(beta, (float)sum, acc[r]));
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    float v = acc[r];
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    if (lane == r && m0 + r < a.M) {
      v *= a.row_scales[m0 + r];
      if (a.bias) v += as_f32(static_cast<const Value<DT> *>(a.bias)[n]);
      static_cast<Value<DT> *>(a.y)[(m0 + r) * a.N + n] = value_of<DT>(v);
    }
  }
}

template <int DT, int BITS>
static hipError_t start_plain(const Rows8Args &a, hipStream_t st) {
  auto start = [&](auto rows) {
    constexpr int ROWS = decltype(rows)::value;
    const int64_t waves = (a.M + ROWS - 1) / ROWS * a.N, grid = (waves + 3) / 4;
    if (grid > INT32_MAX) return hipErrorInvalidValue;
    rows8_plain_kernel<DT, BITS, ROWS><<<(unsigned)grid, 256, 0, st>>>(a);
    return hipGetLastError();
  };
  return a.M == 1 ? start(std::integral_constant<int, 1>{}) : start(std::integral_constant<int, 8>{});
}

hipError_t launch_qmm_rows8(const Rows8Args &a, int bits, int dt, hipStream_t st) {
  if (a.M == 0) return hipSuccess;
  auto with_bits = [&](auto d) {
    constexpr int DT = decltype(d)::value;
    return bits == 4 ? start_plain<DT, 4>(a, st) : start_plain<DT, 8>(a, st);
  };
  if (dt == 0) return with_bits(std::integral_constant<int, 0>{});
  if (dt == 1) return with_bits(std::integral_constant<int, 1>{});
  return with_bits(std::integral_constant<int, 2>{});
}

}  // namespace mi_moe
