// What the kernels of the linear layer on 8-bit rows (qmm_rows8.hip, qmm_rows8_tiles.hip) share.
#pragma once
#include <type_traits>

#include "lds_copies.hpp"
#include "qmm_codes_dev.hpp"
#include "rows8_rule.hpp"

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

__device__ __forceinline__ int32_t byte_sum(uint32_t v, int32_t c) { return __builtin_amdgcn_sdot4((int32_t)v, 0x01010101, c, false); }
typedef int32_t i32x2_t __attribute__((ext_vector_type(2)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));

// Integer sums start at the bits of 1.5 * 2^23, where a float's step is one: below 2^22 (128 products of 2^14 at most are 2^21) they leave the bits of that number
// and the sum, and a subtraction takes the place of a conversion.  Measured a tile of 16 x 16 (multiply, four of either, four multiply-adds), four waves a SIMD: 36 cycles, 43 with
// conversions; the multiply alone 18, the vector instructions alone 20: the two do not overlap.
constexpr float kWhole = 12582912.f;
constexpr int kWholeBits = 0x4b400000;

// the operand of a lane's 8- or 16-byte piece of codes
template <int BITS>
__device__ __forceinline__ i32x4_t operand_of(uint2 lo, uint2 hi) {  // 8-bit: 16 codes; 4-bit: lo, two words
  if constexpr (BITS == 8) {
    return i32x4_t{(int32_t)(lo.x ^ 0x80808080u), (int32_t)(lo.y ^ 0x80808080u), (int32_t)(hi.x ^ 0x80808080u), (int32_t)(hi.y ^ 0x80808080u)};
  } else {
    auto even = [](uint32_t w) { return (int32_t)(((w << 4) & 0xf0f0f0f0u) ^ 0x80808080u); };
    auto odd = [](uint32_t w) { return (int32_t)((w & 0xf0f0f0f0u) ^ 0x80808080u); };
    return i32x4_t{even(lo.x), odd(lo.x), even(lo.y), odd(lo.y)};
  }
}

// eight bytes in their order to the even ones, then the odd ones
__device__ __forceinline__ uint2 evens_odds(uint2 v) {
  return make_uint2(__builtin_amdgcn_perm(v.y, v.x, 0x06040200u), __builtin_amdgcn_perm(v.y, v.x, 0x07050301u));
}

template <class F>
inline hipError_t rows8_with_types(int dt, int bits, int group, F f) {  // f(type, bits, group), each a compile-time constant
  auto with_group = [&](auto d, auto b) {
    if (group == 32) return f(d, b, std::integral_constant<int, 32>{});
    if (group == 64) return f(d, b, std::integral_constant<int, 64>{});
    return f(d, b, std::integral_constant<int, 128>{});
  };
  auto with_bits = [&](auto d) { return bits == 4 ? with_group(d, std::integral_constant<int, 4>{}) : with_group(d, std::integral_constant<int, 8>{}); };
  if (dt == 0) return with_bits(std::integral_constant<int, 0>{});
  if (dt == 1) return with_bits(std::integral_constant<int, 1>{});
  return with_bits(std::integral_constant<int, 2>{});
}

// Prepares the rows and multiplies them in tiles (qmm_rows8_tiles.hip); workspace: rows8_tiles_workspace_bytes.
size_t rows8_tiles_workspace_bytes(int64_t M, int K);
hipError_t launch_rows8_tiles(const Rows8Args &a, Rows8Kind kind, int bits, int dt, void *workspace, hipStream_t st);

}  // namespace mi_moe
