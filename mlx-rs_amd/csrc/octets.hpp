// Rows in eights: eight values of any of the library's types as they lie in memory (norm.hip, f8_rows.hip, sort_tokens.hip).
#pragma once
#include <type_traits>

#include "common.hpp"

namespace mi_moe {

template <int DT>
struct Octet {  // as they lie in memory; DT: mi_moe_dtype
  using Raw = typename std::conditional<DT == 0, uint16_t, typename std::conditional<DT == 1, _Float16, float>::type>::type;
  Raw v[8];
  __device__ __forceinline__ float at(int i) const { return as_f32(v[i]); }
  __device__ __forceinline__ void put2(int i, float lo, float hi) {  // i: even
    if constexpr (DT == 0) {
      const uint32_t p = cvt_pk_bf16(lo, hi);
      v[i] = (uint16_t)p, v[i + 1] = (uint16_t)(p >> 16);
    } else {
      v[i] = (Raw)lo, v[i + 1] = (Raw)hi;
    }
  }
  __device__ __forceinline__ void put(int i, float f) {
    if constexpr (DT == 0) v[i] = f32_to_bf16(f);
    else v[i] = (Raw)f;
  }
};
// `n` values at p (8, or fewer at a row's end), in 16-byte accesses that assume no more than the elements' own alignment: a row of an odd number
// of values starts anywhere.  What is missing is zeros.
template <int DT>
__device__ __forceinline__ Octet<DT> load_octet(const void *base, int64_t at, int n) {
  using Raw = typename Octet<DT>::Raw;
  const Raw *p = static_cast<const Raw *>(base) + at;
  Octet<DT> o;
  if (n >= 8) {
    __builtin_memcpy(o.v, p, sizeof o.v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o.v[i] = i < n ? p[i] : Raw(0);
  }
  return o;
}
template <int DT>
__device__ __forceinline__ void store_octet(void *base, int64_t at, int n, const Octet<DT> &o) {
  using Raw = typename Octet<DT>::Raw;
  Raw *p = static_cast<Raw *>(base) + at;
  if (n >= 8) {
    __builtin_memcpy(p, o.v, sizeof o.v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = o.v[i];
    asm volatile("");  // (else the compiler makes one short store of the first value and of the last ones of both branches, and three of the other)
  }
}

}  // namespace mi_moe
