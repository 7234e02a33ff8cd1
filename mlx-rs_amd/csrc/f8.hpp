// Linear layers and experts on e4m3 weights with a scale for each block of 128 x 128, and rows in e4m3 with a scale for each run of 128 values:
// launchers, and what their kernels share.
//
//   W[n][k] = scale[n / 128][k / 128] * code[n][k]        x[r][k] = scale[r][k / 128] * code[r][k]
//   y[r][n] = sum over runs j of  sx[r][j] * sw[n / 128][j] * (sum over the run's 128 products of codes)
//
// A run's products are summed by the matrix instructions on codes; scales come in once a run, in float32.
//
// The f8 matrix instructions add eight products along the summed axis at a time, each cut towards zero at 2^-13 of the largest power of two that the exponents of two codes of the eight make (measured,
// on 32x32x64 and 16x16x128, with codes of all sizes, one large product among small ones, and two products alone; the eights are then added in float32): an eight's sum is off by less than seven times
// 2^-13 of its largest product, 1.4e-5 of the results' length with normally distributed rows and weights, several percent of a result where large products cancel.  Results of float16 and float32
// are computed with the bf16 instructions instead, on codes taken to bf16, where every product is exact and sums are float32; so are those of a few rows (f8_few.hip).  Those of bfloat16 in tiles are
// not: a value's own rounding to e4m3 is off by up to 2^-4 of it, which a large product brings into the sum 70 times over what an eight loses beside it, and the f8 instructions are what makes the
// tiles fast (4096 x 4096 x 4096 89 us, 157 on the bf16 ones; 4096 tokens through 8 of 128 experts of 2048 x 768 377 and 519).
#pragma once
#include "common.hpp"
#include "f8_rule.hpp"

namespace mi_moe {

// rows in e4m3 as the products read them: codes [rows][whole runs], scales [runs][rows]
struct F8Rows {
  const uint8_t *codes;
  const float *scales;
  int64_t rows;
};
struct F8Mat {
  const uint8_t *w;
  const float *s;
};
struct F8Product {
  F8Rows x;
  // instead of codes, for a few rows (f8_in_blocks), rows that every block of the product rounds for itself: of element type raw_dt, or silu(raw) * raw_up in float32
  const void *raw, *raw_up;
  int raw_dt;
  const uint32_t *order;    // sorted row r reads x row order[r] / k_div; nullptr: r
  int k_div;
  const uint32_t *ids;      // instead of order and list, for a few rows: row r is of x row r / k_div and matrix ids[r] (none, if there is no such one), a piece of its own
  const uint4 *list;        // the pieces of at most f8_tile_rows rows that the matrices' rows are cut into, and rows of no matrix, which are zeros of y (f8_list).  nullptr: one
  int n_mats;               // matrix, all rows
  int few;                  // with a list, how many rows a matrix on average the kernel for a few rows takes; 0: what is best for this product alone (f8_tile_rows)
  int64_t rows;             // of y
  F8Mat m[2];               // the second one: of a gate/up pair (y1 or h), or of a second half of the summed axis (pair_sum)
  bool transpose;           // matrices [N][K], else [K][N]
  bool pair_sum;
  int N, K;
  int n_first, n_count;     // tiles: the columns of y that are computed, from a multiple of kF8TileN on, and as many values a row of y has; n_count 0: all N
  const void *bias;
  void *y, *y1;
  int dt;
  float *y_scales;  // tiles, bfloat16: y is float16, a row's values of 64 columns times a power of two of their own, [rows][columns / 64] (the other way round
                    // the sum over the slots of 4096 tokens read a line for every scale and took 40 us, not 37).  Rows that are summed over
                    // slots afterwards: rounded to bfloat16 here and once more behind the sum, the experts' results were 1.5 times as far off as with one rounding.  (Those to be summed to float16
                    // would be 1.4 times as far off with these: they are float32, some columns at a time.)
  float *parts;  // room for the sums of blocks that share a tile's summed axis (f8_parts_bytes), or nullptr: none do
  uint8_t *h;  // gate/up pairs: silu(gate) * up in e4m3, as F8Rows
  float *hs;
};
// Whether tiles sum on the bf16 instructions: for results (or, of gate/up pairs, tokens) of float16 and float32.  Us, to float16, so and on the f8 instructions, rounding of the rows and all:
// 4096^3 143 and 87, 1000 x 4096 x 4096 47 and 39, its gradient 53 and 46; 4096 tokens through 8 of 128 experts of 2048 x 768 540 and 478.
inline bool f8_exact(const F8Product &p) { return p.dt != 0; }
inline F8Sizes f8_sizes(const F8Product &p) {
  const bool by_matrix = p.list || p.ids;
  return {p.rows, p.N, p.K, by_matrix ? p.n_mats : 1, by_matrix, p.list != nullptr, p.transpose, p.h != nullptr, p.pair_sum, f8_exact(p), p.parts != nullptr, p.few};
}
inline int f8_tile_rows(const F8Product &p) { return f8_tile_rows(f8_sizes(p)); }
inline F8Plan f8_plan(const F8Product &p) { return f8_plan(f8_sizes(p)); }
inline bool f8_few_rows(const F8Product &p) { return f8_tile_rows(p) < 64; }
// Whether the blocks of a product for a few rows round them by themselves, where a matrix has `most` rows as a rule.  (A piece may hold as many as its kernel takes, of tokens that
// name an expert more than once: there is room for them.)
inline size_t f8_own_bytes(const F8Product &p) {
  const int tile = p.ids ? 1 : f8_tile_rows(p);
  return (size_t)(p.rows < tile ? p.rows : tile) * (size_t)(f8_row_bytes(p.K) + 16 + 4 * f8_runs(p.K));
}
inline bool f8_in_blocks(const F8Product &p, int64_t most) { return f8_few_rows(p) && most * f8_runs(p.K) <= 64 && f8_own_bytes(p) <= 48 * 1024; }
inline int64_t f8_most_pieces(int64_t rows, int n_mats, int tile) { return rows / tile + (n_mats + 1 < rows ? n_mats + 1 : rows); }
inline int64_t f8_list_places(int64_t rows, int n_mats) { return f8_most_pieces(rows, n_mats, 16); }
// What is to be listed, beside the rounding of rows (launch_quantize_f8_rows): up to two lists.
struct F8Lists {
  const uint32_t *offsets = nullptr;  // [n_mats + 1]
  int n_mats = 0;
  int64_t rows = 0;
  uint4 *list[2] = {nullptr, nullptr};
  int tile[2] = {0, 0};
  int places[2] = {0, 0};
};
hipError_t launch_f8_few(const F8Product &p, hipStream_t st);    // a few rows a matrix (f8_few.hip); transposed only
hipError_t launch_f8_tiles(const F8Product &p, hipStream_t st);  // tiles (f8_tiles.hip)
// Rows of a token or two (ids; k_div of each): down's product on raw and raw_up, and the sum over the slots, into out [tokens][N] of type dt.
size_t f8_token_bytes(const F8Product &p);
hipError_t launch_f8_token(const F8Product &p, const void *weights, int w_dtype, void *out, int dt, hipStream_t st);
inline hipError_t launch_f8_product(const F8Product &p, hipStream_t st) { return f8_few_rows(p) ? launch_f8_few(p, st) : launch_f8_tiles(p, st); }

// f8_rows.hip.  Codes go to `codes` + row * code_stride, the scale of a row's run j to scales[row * row_stride + j * run_stride].
struct F8Out {
  uint8_t *codes;
  int64_t code_stride;
  float *scales;
  int64_t row_stride, run_stride;
  bool pad;  // zeros up to the end of the last run
};
inline F8Out f8_workspace_rows(uint8_t *codes, float *scales, int64_t rows, int cols) { return {codes, f8_row_bytes(cols), scales, 1, rows, true}; }
hipError_t launch_quantize_f8_rows(const void *x, int dt, int64_t rows, int cols, const F8Out &to, hipStream_t st, const F8Lists &lists = F8Lists());
hipError_t launch_quantize_f8_blocks(const void *x, int dt, int64_t rows, int cols, uint8_t *codes, float *scales, hipStream_t st);
hipError_t launch_dequantize_f8(const uint8_t *codes, const float *scales, int64_t rows, int cols, int block_rows, int dt, void *out, hipStream_t st);
// h = silu(gate) * up of float32 rows, in e4m3
hipError_t launch_swiglu_f8(const float *g, const float *u, int64_t rows, int cols, const F8Out &to, hipStream_t st);
// Its gradient for sorted rows: dh (but for the slot's weight) float32; dg and du in e4m3, one row of both (dg's runs first), and the weights' gradient
struct F8SwigluGrad {
  const float *g, *u, *dh;
  const void *weights;
  int w_dtype;
  const uint32_t *order, *offsets;  // offsets[n_experts]: where the named rows end
  int n_experts;
  int64_t rows;
  int cols;
  uint8_t *codes;
  float *scales;
  void *dweights;
};
hipError_t launch_swiglu_f8_grad(const F8SwigluGrad &a, hipStream_t st);

// Tokens sorted by expert (sort_tokens.hip).  inverse: a slot's row, or -1 - row where it names no expert (those rows lie behind the others').
struct SortTokens {
  const uint32_t *ids;
  int64_t T;
  int k, E;
  uint32_t *order;
  int32_t *inverse;
  uint32_t *offsets;  // [E + 1]
};
size_t sort_tokens_bytes(int64_t T, int k, int E);
constexpr int64_t kSortSmall = 2048;  // pairs up to which one launch sorts, and lists
// rows != nullptr: the sorted rows of x, those that no slot names zeros
// lists (up to kSortSmall pairs): made beside it
hipError_t launch_sort_tokens(const SortTokens &a, const void *x, int dt, int H, void *rows, void *scratch, hipStream_t st, const F8Lists &lists = F8Lists());
// weights nullptr: sums without weights (the sorting's gradient).  out of type dt, its rows out_stride values from each other; rows of type dt, or scaled float16 (y_scales), or float32 for fewer bits of dt
hipError_t launch_unsort_made(const void *rows, const float *y_scales, const void *weights, int w_dtype, const int32_t *inverse, int64_t T, int k, int H, int dt, void *out,
                              int out_stride, hipStream_t st);
hipError_t launch_unsort_tokens(const void *rows, const void *weights, int w_dtype, const int32_t *inverse, int64_t T, int k, int H, int dt, void *out,
                                hipStream_t st);
hipError_t launch_unsort_tokens_grad(const void *dout, const void *rows, const void *weights, int w_dtype, const int32_t *inverse, int64_t T, int k, int H, int dt,
                                     void *drows, void *dweights, hipStream_t st);

#ifdef __HIPCC__
// ---------------------------------------------------------------- codes
constexpr float kF8Most = 448.f;

// scale = largest / 448, what it makes of the values (quotient and code as the definition rounds them), and whether they have codes at all: a run of zeros has a scale and
// codes of zero, one that holds an infinity or a NaN codes of zero and a scale that is NaN, so that what is made of it is, too.
struct F8Scale {
  float scale, inv;
  bool coded, plain;
  __device__ __forceinline__ explicit F8Scale(uint32_t largest_bits) {
    const float most = __uint_as_float(largest_bits);
    coded = largest_bits < 0x7f800000u;
    scale = coded ? most / kF8Most : NAN;
    coded = coded && scale > 0.f;
    // reciprocal and residual: with inv = round(1 / scale), q0 = round(v inv) is off by at most an ulp, and round(q0 + (v - q0 scale) inv) is the correctly rounded
    // quotient, if the residual is exact: with scale above 2^-93 it is no smaller than the least float for every quotient that has a code (2^-10 and more).
    plain = largest_bits < 0x17800000u;  // 2^-80
    inv = coded ? 1.f / scale : 0.f;
  }
  __device__ __forceinline__ float quotient(float v) const {
    float q;
    if (plain) {
      q = coded ? v / scale : 0.f;
    } else {
      const float q0 = v * inv;
      q = __builtin_fmaf(__builtin_fmaf(-q0, scale, v), inv, q0);
    }
    return __builtin_amdgcn_fmed3f(q, -kF8Most, kF8Most);  // (beyond it where the scale itself is a few of the least floats)
  }
  // four codes, the first value's in the low byte
  __device__ __forceinline__ uint32_t codes(float a, float b, float c, float d) const {
    if (!coded) return 0u;
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(quotient(a), quotient(b), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(quotient(c), quotient(d), w, true);
  }
};
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }  // ordered as the magnitudes, NaN behind infinity
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t max_of_16_lanes(uint32_t m) {
  m = umax(m, dpp_u32<kDppXor1>(m));
  m = umax(m, dpp_u32<kDppXor2>(m));
  m = umax(m, dpp_u32<kDppHalfMirror>(m));
  return umax(m, dpp_u32<kDppMirror>(m));
}
// (v_rcp_f32 is within an ulp; where exp(-g) is infinite it gives zero, and g times it the limit's own)
__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.f + __expf(-g)); }
__device__ __forceinline__ float silu(float g) { return g * sigmoid(g); }

// ---------------------------------------------------------------- segments
// A piece of at most `tile` rows of one matrix (n_mats: of none); rows 0: nothing.
struct F8Piece {
  int mat;
  uint32_t row, rows;
};
__device__ __forceinline__ F8Piece f8_piece(const F8Product &p, uint32_t tile, uint32_t m) {
  if (p.ids) {
    const uint32_t e = p.ids[m];
    return {__builtin_amdgcn_readfirstlane((int)(e < (uint32_t)p.n_mats ? e : (uint32_t)p.n_mats)), m, 1u};
  }
  if (!p.list) {
    const uint32_t row = m * tile, total = (uint32_t)p.rows;
    return {0, row, row >= total ? 0u : total - row < tile ? total - row : tile};
  }
  const uint4 v = p.list[m];
  return {__builtin_amdgcn_readfirstlane((int)v.x), (uint32_t)__builtin_amdgcn_readfirstlane((int)v.y), (uint32_t)__builtin_amdgcn_readfirstlane((int)v.z)};
}
// The list of pieces of the segments that offsets[n_mats + 1] cut the rows into, by one wave.  A segment is cut into as few pieces of at most `tile` rows as it can be, of about one
// size (multiples of 32 rows).  Behind the segments' pieces come those of the rows that belong to none, then empty ones.  Offsets out of order or range only make pieces
// that overlap or are missing.
// In the experts' order: with whole pieces first and the rest of the segments behind them, the longest first, the launch ends more evenly, but its first half multiplies and its
// second one waits for weights (4096 tokens, skewed routing over 128 experts of 2048 x 768: down 138 us, 156 so).
__device__ __forceinline__ void f8_list(const uint32_t *__restrict__ offsets, int n_mats, uint32_t total, uint32_t tile, uint4 *__restrict__ list, uint32_t places) {
  const int lane = lane_id();
  uint32_t before = 0;
  for (int e0 = 0; e0 <= n_mats; e0 += kWave) {
    const int e = e0 + lane;
    uint32_t lo = 0, hi = 0;
    if (e <= n_mats) {
      lo = offsets[e];
      hi = e < n_mats ? offsets[e + 1] : total;
      lo = lo < total ? lo : total;
      hi = hi < lo ? lo : hi < total ? hi : total;
    }
    const uint32_t pieces = (hi - lo + tile - 1) / tile;
    uint32_t upto = pieces;
    for (int d = 1; d < kWave; d <<= 1) {
      const uint32_t up = __shfl_up(upto, d, kWave);
      if (lane >= d) upto += up;
    }
    const uint32_t even = pieces <= 1 ? tile : ((hi - lo + pieces - 1) / pieces + 31) / 32 * 32, size = even < tile ? even : tile, first = before + upto - pieces;
    for (uint32_t i = 0; i < pieces && first + i < places; ++i) {
      const uint32_t row = lo + i * size;
      list[first + i] = make_uint4((uint32_t)e, row, hi - row < size ? hi - row : size, 0u);
    }
    before += (uint32_t)__builtin_amdgcn_readlane((int)upto, kWave - 1);
  }
  for (uint32_t i = before + lane; i < places; i += kWave) list[i] = make_uint4(0, 0, 0, 0);
}

// ---------------------------------------------------------------- products
typedef int32_t i32x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_f8 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x16_t mfma_f8_32(i32x8_t a, i32x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
}
// eight codes as bf16 (exact)
__device__ __forceinline__ bf16x8_t codes_to_bf16(uint32_t lo, uint32_t hi) {
  typedef __bf16 pair_t __attribute__((ext_vector_type(2)));
  struct { pair_t p[4]; } v = {{__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true),
                                __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true)}};
  return __builtin_bit_cast(bf16x8_t, v);
}
__device__ __forceinline__ void store4(void *base, int64_t at, int n, int dt, const float v[4]) {  // n of four values, rounded
  if (dt == 2) {
    float *p = static_cast<float *>(base) + at;
    if (n >= 4) __builtin_memcpy(p, v, 16);
    else
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < n) p[i] = v[i];
    return;
  }
  uint16_t *p = static_cast<uint16_t *>(base) + at;
  uint16_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = dt == 0 ? f32_to_bf16(v[i]) : __builtin_bit_cast(uint16_t, (_Float16)v[i]);
  if (n >= 4) __builtin_memcpy(p, o, 8);
  else
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = o[i];
}
__device__ __forceinline__ float value_of(const void *base, int64_t at, int dt) {
  return dt == 0 ? bf16_to_f32(static_cast<const uint16_t *>(base)[at]) : dt == 1 ? (float)static_cast<const _Float16 *>(base)[at] : static_cast<const float *>(base)[at];
}
__device__ __forceinline__ void put_value(void *base, int64_t at, int dt, float v) {
  if (dt == 0) static_cast<uint16_t *>(base)[at] = f32_to_bf16(v);
  else if (dt == 1) static_cast<_Float16 *>(base)[at] = (_Float16)v;
  else static_cast<float *>(base)[at] = v;
}
#endif

}  // namespace mi_moe
