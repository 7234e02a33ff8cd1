// Quantized linear layer on rows in eight bits: y [M, N] = (row_scale x [M, K]) . (scale code + bias)^T, each result rounded once.
//
// With x int8 and the codes centred (c' = c - 8 or c - 128, the bias with the centre's share beta = b + 8 s or b + 128 s)
//   y[m, n] = row_scale[m] * sum over groups of (s[n, g] sum_k x[m, k] c'[n, k] + beta[n, g] sum_k x[m, k]) + linear_bias[n]
// the sums over a group are integers and exact; what is in float is a term or two a group.  (The layer on 16-bit rows: mlx-rs/src/nn/quantized.rs:363-386.)
#include <type_traits>

#include "lds_copies.hpp"
#include "qmm_codes_dev.hpp"

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

constexpr int kRows8Few = 16;  // rows up to which the kernel without preparation runs

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

// ---------------------------------------------------------------- many rows: tiles on the int8 matrix cores
// Rows as the matrix instructions take them: for every 16 rows and 64 K values a tile of 1024 bytes, 16 a lane (row l % 16, part kb = l / 16 of the values), in the
// order in which the lane that holds the same values of a weight row has them after unpacking:
//   8-bit codes                16 consecutive values
//   4-bit codes                the words 2 kb and 2 kb + 1 of the eight, of each the even nibbles, then the odd ones
//   groups of 32 (two a tile)  8 values of each, 8 kb .. 8 kb + 7 of the group, in that order within a word
// and the group sums, four groups of 16 rows a tile of 64 floats (lane: row l % 16, group 4 q + kb; zeros past the last group).
__host__ __device__ constexpr int64_t row_tiles(int64_t M) { return (M + 15) / 16; }
constexpr size_t rows8_tiles_bytes(int64_t M, int K) { return (size_t)row_tiles(M) * 16 * K; }
constexpr size_t rows8_sums_bytes(int64_t M, int K, int group) { return (size_t)row_tiles(M) * ((K / group + 3) / 4) * 256; }

__device__ __forceinline__ int32_t byte_sum(uint32_t v, int32_t c) { return __builtin_amdgcn_sdot4((int32_t)v, 0x01010101, c, false); }
// eight bytes in their order to the even ones, then the odd ones
__device__ __forceinline__ uint2 evens_odds(uint2 v) {
  return make_uint2(__builtin_amdgcn_perm(v.y, v.x, 0x06040200u), __builtin_amdgcn_perm(v.y, v.x, 0x07050301u));
}

// A wave makes the tiles of 16 rows and four groups.
template <int BITS, int GROUP>
__global__ __launch_bounds__(256) void rows8_prepare_kernel(const signed char *x, int64_t M, int K, uint4 *tiles, float *sums) {
  constexpr int NT = GROUP * 4 / 64;  // tiles of four groups
  const int lane = lane_id(), kb = lane >> 4, quads = (K / GROUP + 3) / 4, n_tiles = K / 64;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), mt = unit / quads;
  const int q = (int)(unit % quads);
  if (mt >= row_tiles(M)) return;
  const int64_t row = mt * 16 + (lane & 15);
  int32_t sum[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int kt = q * NT + i;
    uint2 a = make_uint2(0, 0), b = a;
    if (kt < n_tiles && row < M) {
      const signed char *const p = x + row * K + kt * 64;
      a = *reinterpret_cast<const uint2 *>(p + (GROUP == 32 ? 8 * kb : 16 * kb));
      b = *reinterpret_cast<const uint2 *>(p + (GROUP == 32 ? 32 + 8 * kb : 16 * kb + 8));
    }
    if constexpr (GROUP == 32) {
      sum[2 * i] = byte_sum(a.y, byte_sum(a.x, 0));
      sum[2 * i + 1] = byte_sum(b.y, byte_sum(b.x, 0));
    } else {
      sum[i * 64 / GROUP] = byte_sum(b.y, byte_sum(b.x, byte_sum(a.y, byte_sum(a.x, sum[i * 64 / GROUP]))));
    }
    if constexpr (BITS == 4) a = evens_odds(a), b = evens_odds(b);
    if (kt < n_tiles) tiles[(mt * n_tiles + kt) * 64 + lane] = make_uint4(a.x, a.y, b.x, b.y);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    sum[i] += __shfl_xor(sum[i], 16);
    sum[i] += __shfl_xor(sum[i], 32);
  }
  sums[(mt * quads + q) * 64 + lane] = (float)(kb == 0 ? sum[0] : kb == 1 ? sum[1] : kb == 2 ? sum[2] : sum[3]);
}

typedef int32_t i32x2_t __attribute__((ext_vector_type(2)));

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

// y = rows x weights in tiles of 16 MI WM rows and 16 NI WN columns, a wave 16 MI x 16 NI of them.  A stage is 128 K values: the rows' tiles and the codes are copied straight
// into LDS, one stage ahead.  Codes: 64 or 128 bytes of a weight row a stage, its 16-byte pieces in an order turned by the row, so that the lanes' reads meet all banks.
// A group is one matrix instruction a 16 x 16 tile (two for 128 values, one of half the depth for 32), whose integer sums are exact; then a conversion and a
// multiply-add a result.  That vector work, 32 cycles a tile and 64 values, is what bounds it: twice the instruction's own 16.  The biases' terms are a product over
// the groups by the float32 matrix instructions, four groups a time.
template <int DT, int BITS, int GROUP, int MI, int NI, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2) void rows8_tiles_kernel(Rows8Args a, const uint4 *tiles, const float *sums, int n_mtiles, int n_ntiles) {
  constexpr int kWaves = WM * WN, ROWS = 16 * MI * WM, COLS = 16 * NI * WN;
  constexpr int CODES = 128 * BITS / 8, PIECES = CODES / 16;  // bytes and 16-byte pieces of a weight row's stage
  constexpr int A_BYTES = ROWS * 128, STAGE = A_BYTES + COLS * CODES;
  constexpr int GS = 128 / GROUP, PERIOD = GROUP / 32;  // groups of a stage; stages of four groups
  extern __shared__ __align__(16) unsigned char lds_raw[];
  const int xcd = blockIdx.x & 7, j = blockIdx.x >> 3, nt = j / n_mtiles * 8 + xcd;  // an XCD takes every eighth column tile and all row tiles of it
  if (nt >= n_ntiles) return;
  const int64_t mt0 = (int64_t)(j % n_mtiles) * (MI * WM);
  const int n0 = nt * COLS;
  const int lane = lane_id(), ln = lane & 15, kb = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
  const int K = a.K, n_stages = K / 128, G = K / GROUP, quads = (G + 3) / 4, row_bytes = K * BITS / 8;
  const int64_t x_bytes = (row_tiles(a.M) - mt0) * K * 16, w_bytes = (int64_t)(a.N - n0) * row_bytes;
  const i32x4_t xr = words_of(reinterpret_cast<const char *>(tiles) + mt0 * K * 16, (uint32_t)(x_bytes < INT32_MAX ? x_bytes : INT32_MAX));
  const i32x4_t wr = words_of(reinterpret_cast<const char *>(a.w) + (int64_t)n0 * row_bytes, (uint32_t)(w_bytes < INT32_MAX ? w_bytes : INT32_MAX));
  // copies: 1024 bytes an instruction; of the rows tile (i / 2) of 16 and half i % 2 of the stage, of the codes 1024 / CODES weight rows
  constexpr int A_COPIES = MI * WM * 2, B_ROWS = 1024 / CODES, B_COPIES = COLS / B_ROWS;
  static_assert(A_COPIES % kWaves == 0 && B_COPIES % kWaves == 0);
  const int brow = lane / PIECES;
  auto turn = [](int row) { return PIECES == 4 ? (row >> 2) & 3 : (row >> 1) & 7; };
  auto copy_stage = [&](int t) __attribute__((always_inline)) {
    const uint32_t to = (uint32_t)(t & 1) * STAGE;
#pragma unroll
    for (int u = 0; u < A_COPIES / kWaves; ++u) {
      const int i = u * kWaves + wave;
      copy_to_lds(xr, lane * 16, (i >> 1) * (K * 16) + t * 2048 + (i & 1) * 1024, to + i * 1024);
    }
#pragma unroll
    for (int u = 0; u < B_COPIES / kWaves; ++u) {
      const int i = u * kWaves + wave, row = i * B_ROWS + brow;
      copy_to_lds(wr, row * row_bytes + ((lane % PIECES) ^ turn(row)) * 16, t * CODES, to + A_BYTES + i * 1024);
    }
  };
  using T = Value<DT>;
  // Scales and biases, a window of 16 bytes a column (8 groups, or 4 of float32) at a time: a piece a thread, loaded a window ahead and laid into LDS in the window's last
  // stage but one.  (Each lane loading its own, a few bytes a stage: 16 lines of 128 bytes a load, 83 KB a stage through an L1 of 32, and 205 us for 4096 x 4096 x 4096.)
  constexpr int WINDOW = 16 / sizeof(T), WSTAGES = WINDOW / GS;
  static_assert(2 * COLS == 64 * kWaves);
  unsigned char *const scales_at = lds_raw + 2 * STAGE;
  const T *piece_row;
  {
    const int64_t col = n0 + (int)threadIdx.x % COLS;  // (columns outside: the last one's, not stored)
    piece_row = static_cast<const T *>(threadIdx.x < COLS ? a.s : a.b) + (col < a.N ? col : a.N - 1) * G;
  }
  struct __align__(16) Window { T v[WINDOW]; };
  Window window;
  auto load_window = [&](int w) __attribute__((always_inline)) {
    const int g = w * WINDOW;
    if (g + WINDOW <= G) {
      __builtin_memcpy(window.v, piece_row + g, 16);  // (rows of scales start anywhere)
    } else {
#pragma unroll
      for (int i = 0; i < WINDOW; ++i) window.v[i] = piece_row[g + i < G ? g + i : G - 1];
    }
  };
  auto put_window = [&](int w) __attribute__((always_inline)) {
    *reinterpret_cast<Window *>(scales_at + (w & 1) * (COLS * 32) + threadIdx.x * 16) = window;
  };
  const float *sump[MI];
#pragma unroll
  for (int m = 0; m < MI; ++m) {
    const int64_t mt = mt0 + wm * MI + m;
    sump[m] = sums + (mt < row_tiles(a.M) ? mt : row_tiles(a.M) - 1) * quads * 64 + lane;
  }
  float qx[MI];
  auto load_sums = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < MI; ++m) qx[m] = sump[m][t / PERIOD * 64];
  };
  f32x4_t acc[MI][NI];
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int n = 0; n < NI; ++n) acc[m][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // Integer sums start at the bits of 1.5 * 2^23, where a float's step is one: below 2^22 (128 products of 2^14 at most are 2^21) they leave the bits of that number
  // and the sum, and a subtraction in place of a conversion, which is a quarter as fast.
  constexpr float kWhole = 12582912.f;
  constexpr int kWholeBits = 0x4b400000;
  i32x4_t whole = {kWholeBits, kWholeBits, kWholeBits, kWholeBits};
  asm("" : "+v"(whole));  // (a literal is not among the instruction's operands)
  copy_stage(0);
  load_sums(0);
  load_window(0);
  put_window(0);
  load_window(1);
#pragma unroll 1
  for (int t = 0; t < n_stages; ++t) {
    wait_copies<0>();
    block_barrier();
    const int w = t / WSTAGES;
    const unsigned char *const mine = scales_at + (w & 1) * (COLS * 32) + (wn * NI * 16 + ln) * 16;  // this lane's columns: every 16th
    float s[NI][GS];
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      T v[GS];
      __builtin_memcpy(v, __builtin_assume_aligned(mine + n * 256 + t % WSTAGES * (int)sizeof v, sizeof v), sizeof v);
#pragma unroll
      for (int g = 0; g < GS; ++g) s[n][g] = as_f32(v[g]);
    }
    if (t % PERIOD == 0) {
      const int g = (t / PERIOD * 4 + kb) % WINDOW * (int)sizeof(T);
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        constexpr float k = Centre<BITS>::of_codes;
        const float beta = __builtin_fmaf(k * Centre<BITS>::value, as_f32(*reinterpret_cast<const T *>(mine + n * 256 + g)),
                                          k * as_f32(*reinterpret_cast<const T *>(mine + COLS * 16 + n * 256 + g)));
#pragma unroll
        for (int m = 0; m < MI; ++m) acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(qx[m], beta, acc[m][n], 0, 0, 0);
      }
    }
    if ((t + 1) % WSTAGES == 0) {  // (what was loaded a window ago is there: every stage waits for all loads before it)
      put_window(w + 1);
      load_window(w + 2);
    }
    if (t + 1 < n_stages) {
      if ((t + 1) % PERIOD == 0) load_sums(t + 1);
      copy_stage(t + 1);
    }
    const unsigned char *const at = lds_raw + (t & 1) * STAGE;
    struct Half {  // the operands of 64 values
      i32x4_t x[MI], w[NI];
      uint2 lo[NI], hi[NI];
    };
    Half half[2];
    auto read_x = [&](int h, int m) __attribute__((always_inline)) {
      half[h].x[m] = *reinterpret_cast<const i32x4_t *>(at + ((wm * MI + m) * 2 + h) * 1024 + lane * 16);
    };
    auto read_w = [&](int h, int n) __attribute__((always_inline)) {
      const int row = (wn * NI + n) * 16 + ln;
      const unsigned char *const r = at + A_BYTES + row * CODES;
      auto piece = [&](int byte) { return r + (((byte >> 4) ^ turn(row)) << 4) + (byte & 15); };
      uint2 &lo = half[h].lo[n], &hi = half[h].hi[n];
      hi = make_uint2(0, 0);
      if constexpr (BITS == 8 && GROUP != 32) {
        const uint4 v = *reinterpret_cast<const uint4 *>(piece(h * 64 + 16 * kb));
        lo = make_uint2(v.x, v.y), hi = make_uint2(v.z, v.w);
      } else if constexpr (BITS == 8) {
        lo = *reinterpret_cast<const uint2 *>(piece(h * 64 + 8 * kb));
        hi = *reinterpret_cast<const uint2 *>(piece(h * 64 + 32 + 8 * kb));
      } else if constexpr (GROUP != 32) {
        lo = *reinterpret_cast<const uint2 *>(piece(h * 32 + 8 * kb));
      } else {
        lo = make_uint2(*reinterpret_cast<const uint32_t *>(piece(h * 32 + 4 * kb)), *reinterpret_cast<const uint32_t *>(piece(h * 32 + 16 + 4 * kb)));
      }
    };
    auto unpack = [&](int h, int n) __attribute__((always_inline)) { half[h].w[n] = operand_of<BITS>(half[h].lo[n], half[h].hi[n]); };
    // The tiles one after the other, each multiplied LEAD steps before its sums are converted and scaled: written out in the order in which it is to run (the compiler's own
    // order has a multiply's results used right behind it: 195.7 us for 4096 x 4096 x 4096, 4-bit, groups of 64).
    constexpr int PER = GROUP == 32 ? 2 : 1, HALVES = GROUP == 128 ? 1 : 2, TILES = MI * NI, STEPS = HALVES * TILES * PER, LEAD = 3;
    i32x4_t d[LEAD + 1];
    auto multiply = [&](int k) __attribute__((always_inline)) {
      const int h = k / (TILES * PER), m = k / PER % TILES / NI, n = k / PER % NI, g = k % PER;
      if constexpr (GROUP == 32) {
        const i32x2_t x2 = {half[h].x[m][2 * g], half[h].x[m][2 * g + 1]}, w2 = {half[h].w[n][2 * g], half[h].w[n][2 * g + 1]};
        d[k % (LEAD + 1)] = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, x2), __builtin_bit_cast(long, w2), whole, 0, 0, 0);
      } else {
        d[k % (LEAD + 1)] = __builtin_amdgcn_mfma_i32_16x16x64_i8(half[h].x[m], half[h].w[n], whole, 0, 0, 0);
        if constexpr (GROUP == 128) d[k % (LEAD + 1)] = __builtin_amdgcn_mfma_i32_16x16x64_i8(half[1].x[m], half[1].w[n], d[k % (LEAD + 1)], 0, 0, 0);
      }
    };
    auto scale = [&](int k) __attribute__((always_inline)) {
      const int h = k / (TILES * PER), m = k / PER % TILES / NI, n = k / PER % NI, g = k % PER;
      const i32x4_t v = d[k % (LEAD + 1)];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][n][i] = __builtin_fmaf(s[n][h * PER + g], __int_as_float(v[i]) - kWhole, acc[m][n][i]);
    };
#pragma unroll
    for (int h = 0; h < (GROUP == 128 ? 2 : 1); ++h) {
#pragma unroll
      for (int n = 0; n < NI; ++n) read_w(h, n);
#pragma unroll
      for (int m = 0; m < MI; ++m) read_x(h, m);
#pragma unroll
      for (int n = 0; n < NI; ++n) unpack(h, n);
    }
#pragma unroll
    for (int k = 0; k < STEPS + LEAD; ++k) {
      if constexpr (HALVES == 2) {  // the second half's operands: read during the first steps, unpacked ahead of their own
        if (k < NI) read_w(1, k);
        if (k < MI) read_x(1, k);
        if (k >= TILES * PER - NI && k < TILES * PER) unpack(1, k - (TILES * PER - NI));
      }
      if (k < STEPS) multiply(k);
      if (k >= LEAD) scale(k - LEAD);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = (mt0 + wm * MI + m) * 16 + 4 * kb + i;
      if (row >= a.M) continue;
      const float scale = a.row_scales[row] / Centre<BITS>::of_codes;
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        const int col = n0 + (wn * NI + n) * 16 + ln;
        if (col >= a.N) continue;
        float v = acc[m][n][i] * scale;
        if (a.bias) v += as_f32(static_cast<const T *>(a.bias)[col]);
        static_cast<T *>(a.y)[row * a.N + col] = value_of<DT>(v);
      }
    }
}

template <int DT, int BITS, int GROUP>
static hipError_t start_tiles(const Rows8Args &a, void *workspace, hipStream_t st) {
  uint4 *const tiles = static_cast<uint4 *>(workspace);
  float *const sums = reinterpret_cast<float *>(static_cast<char *>(workspace) + rows8_tiles_bytes(a.M, a.K));
  const int64_t units = row_tiles(a.M) * ((a.K / GROUP + 3) / 4);
  if (units > (int64_t)4 * INT32_MAX) return hipErrorInvalidValue;
  rows8_prepare_kernel<BITS, GROUP><<<(unsigned)((units + 3) / 4), 256, 0, st>>>(a.x, a.M, a.K, tiles, sums);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  constexpr int MI = 4, NI = 4, WM = 2, WN = 2, ROWS = 16 * MI * WM, COLS = 16 * NI * WN, lds = 2 * (ROWS * 128 + COLS * 128 * BITS / 8) + 2 * COLS * 32;
  const int64_t n_mtiles = (a.M + ROWS - 1) / ROWS, n_ntiles = (a.N + COLS - 1) / COLS, grid = (n_ntiles + 7) / 8 * 8 * n_mtiles;
  if (grid > INT32_MAX) return hipErrorInvalidValue;
  const auto kernel = &rows8_tiles_kernel<DT, BITS, GROUP, MI, NI, WM, WN>;
  static std::atomic<uint64_t> allowed{0};
  if (hipError_t e = allow_lds(reinterpret_cast<const void *>(kernel), lds, allowed); e != hipSuccess) return e;
  kernel<<<(unsigned)grid, 64 * WM * WN, lds, st>>>(a, tiles, sums, (int)n_mtiles, (int)n_ntiles);
  return hipGetLastError();
}

size_t rows8_workspace_bytes(int64_t M, int K) { return M <= kRows8Few || K % 128 ? 0 : rows8_tiles_bytes(M, K) + rows8_sums_bytes(M, K, 32); }

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

hipError_t launch_qmm_rows8(const Rows8Args &a, int bits, int dt, void *workspace, size_t workspace_bytes, hipStream_t st) {
  if (a.M == 0) return hipSuccess;
  auto even = [](const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  const size_t need = rows8_workspace_bytes(a.M, a.K);
  const bool tiles = need && workspace && even(workspace) && workspace_bytes >= need && a.K <= 1 << 20 && even(a.x) && even(a.w) && even(a.s) && even(a.b);
  auto with_bits = [&](auto d, auto b) {
    constexpr int DT = decltype(d)::value, BITS = decltype(b)::value;
    if (!tiles) return start_plain<DT, BITS>(a, st);
    if (a.group == 32) return start_tiles<DT, BITS, 32>(a, workspace, st);
    if (a.group == 64) return start_tiles<DT, BITS, 64>(a, workspace, st);
    return start_tiles<DT, BITS, 128>(a, workspace, st);
  };
  auto with_dtype = [&](auto d) { return bits == 4 ? with_bits(d, std::integral_constant<int, 4>{}) : with_bits(d, std::integral_constant<int, 8>{}); };
  if (dt == 0) return with_dtype(std::integral_constant<int, 0>{});
  if (dt == 1) return with_dtype(std::integral_constant<int, 1>{});
  return with_dtype(std::integral_constant<int, 2>{});
}

}  // namespace mi_moe
