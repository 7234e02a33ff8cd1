// Quantized linear layer on rows in eight bits: y [M, N] = (row_scale x [M, K]) . (scale code + bias)^T, each result rounded once.
//
// With x int8 and the codes centred (c' = c - 8 or c - 128, the bias with the centre's share beta = b + 8 s or b + 128 s)
//   y[m, n] = row_scale[m] * sum over groups of (s[n, g] sum_k x[m, k] c'[n, k] + beta[n, g] sum_k x[m, k]) + linear_bias[n]
// the sums over a group are integers and exact; what is in float is a term or two a group.  (The layer on 16-bit rows: mlx-rs/src/nn/quantized.rs:363-386.)
#include "qmm_rows8_dev.hpp"

namespace mi_moe {

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
    const int64_t most = ((int64_t)1 << 25) / a.N * ROWS, step = most ? most : ROWS;  // rows of a launch, which has less than 2^32 threads
    for (int64_t m = 0; m < a.M; m += step) {
      Rows8Args some = a;
      some.x = a.x + m * a.K;
      some.row_scales = a.row_scales + m;
      some.y = static_cast<Value<DT> *>(a.y) + m * a.N;
      some.M = a.M - m < step ? a.M - m : step;
      const int64_t grid = ((some.M + ROWS - 1) / ROWS * a.N + 3) / 4;
      if (grid >= (int64_t)1 << 24) return hipErrorInvalidValue;
      rows8_plain_kernel<DT, BITS, ROWS><<<(unsigned)grid, 256, 0, st>>>(some);
      if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
  };
  return a.M == 1 ? start(std::integral_constant<int, 1>{}) : start(std::integral_constant<int, 8>{});
}

// ---------------------------------------------------------------- one row, two rows
__device__ __forceinline__ float wave_sum_in_order(float v) {
  v += __uint_as_float(dpp_u32<kDppXor1>(__float_as_uint(v)));
  v += __uint_as_float(dpp_u32<kDppXor2>(__float_as_uint(v)));
  v += __uint_as_float(dpp_u32<kDppHalfMirror>(__float_as_uint(v)));
  v += __uint_as_float(dpp_u32<kDppMirror>(__float_as_uint(v)));
  auto row = [&](int lane) { return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), lane)); };
  return (row(0) + row(16)) + (row(32) + row(48));
}

// A wave has two columns; a lane 16 bytes of each column's codes at a time, of one group, which it multiplies four at a time (v_dot4) and scales once; whole lines are loaded and nothing
// is loaded twice.  What bounds it is memory, for a few thousand columns the latency of a wave's loads.  us, 4-bit, groups of 64, K = 4096 (the matrix instructions below for five rows: 5.4, 11.6):
//   1 x 4096 3.9, 1 x 14336 6.7 (4.9 TB/s), 2 rows 4.7 and 8.7; four would be 5.9 and 12.2; one column a wave 4.0 and 7.7 (one row), four 3.9 and 6.8 and more registers.
template <int DT, int BITS, int GROUP, int ROWS>
__global__ __launch_bounds__(256) void rows8_dot_kernel(Rows8Args a) {
  using T = Value<DT>;
  constexpr int COLS = 2, CODES = 128 / BITS, WORDS = CODES / 4;  // a lane's codes of a step, and the words of as many rows' values
  const int lane = lane_id(), pieces = a.K / CODES, G = a.K / GROUP;
  const int64_t n0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * COLS;
  if (n0 >= a.N) return;
  const uint4 *wp[COLS];
  const T *sp[COLS], *bp[COLS];
#pragma unroll
  for (int c = 0; c < COLS; ++c) {  // columns outside: the last one again, not stored
    const int64_t n = n0 + c < a.N ? n0 + c : a.N - 1;
    wp[c] = reinterpret_cast<const uint4 *>(a.w) + n * pieces;
    sp[c] = static_cast<const T *>(a.s) + n * G;
    bp[c] = static_cast<const T *>(a.b) + n * G;
  }
  struct Step {
    uint4 w[COLS];
    T s[COLS], b[COLS];
    uint4 x[ROWS][WORDS / 4];
  };
  auto load = [&](int p, Step &S) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      S.w[c] = wp[c][p];
      S.s[c] = sp[c][p * CODES / GROUP];
      S.b[c] = bp[c][p * CODES / GROUP];
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int i = 0; i < WORDS / 4; ++i) S.x[r][i] = reinterpret_cast<const uint4 *>(a.x + (r < a.M ? r : a.M - 1) * a.K)[p * (WORDS / 4) + i];
  };
  float acc[ROWS][COLS] = {};
  Step next;
  if (lane < pieces) load(lane, next);
#pragma unroll 1
  for (int p = lane; p < pieces; p += kWave) {
    const Step S = next;
    if (p + kWave < pieces) load(p + kWave, next);
    int32_t x[ROWS][WORDS], sum[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      sum[r] = 0;
#pragma unroll
      for (int i = 0; i < WORDS / 4; ++i) {
        const uint4 v = S.x[r][i];
        const uint2 lo = BITS == 4 ? evens_odds(make_uint2(v.x, v.y)) : make_uint2(v.x, v.y), hi = BITS == 4 ? evens_odds(make_uint2(v.z, v.w)) : make_uint2(v.z, v.w);
        x[r][4 * i] = (int32_t)lo.x, x[r][4 * i + 1] = (int32_t)lo.y, x[r][4 * i + 2] = (int32_t)hi.x, x[r][4 * i + 3] = (int32_t)hi.y;
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[r] = byte_sum((uint32_t)x[r][4 * i + k], sum[r]);
      }
    }
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      constexpr float k = Centre<BITS>::of_codes;
      const float s = as_f32(S.s[c]), beta = __builtin_fmaf(k * Centre<BITS>::value, s, k * as_f32(S.b[c]));
      int32_t w[WORDS];
      if constexpr (BITS == 4) {
        const i32x4_t lo = operand_of<4>(make_uint2(S.w[c].x, S.w[c].y), make_uint2(0, 0)), hi = operand_of<4>(make_uint2(S.w[c].z, S.w[c].w), make_uint2(0, 0));
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = lo[j], w[4 + j] = hi[j];
      } else {
        const i32x4_t v = operand_of<8>(make_uint2(S.w[c].x, S.w[c].y), make_uint2(S.w[c].z, S.w[c].w));
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = v[j];
      }
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        int32_t d = 0;
#pragma unroll
        for (int j = 0; j < WORDS; ++j) d = __builtin_amdgcn_sdot4(x[r][j], w[j], d, false);
        acc[r][c] = __builtin_fmaf(s, (float)d, __builtin_fmaf(beta, (float)sum[r], acc[r][c]));
      }
    }
  }
  float mine = 0.f;  // lane r COLS + c: that result
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      const float v = wave_sum_in_order(acc[r][c]);
      if (lane == r * COLS + c) mine = v;
    }
  const int r = lane / COLS;
  const int64_t col = n0 + lane % COLS;
  if (r >= ROWS || r >= a.M || col >= a.N) return;
  mine *= a.row_scales[r] / Centre<BITS>::of_codes;
  if (a.bias) mine += as_f32(static_cast<const T *>(a.bias)[col]);
  static_cast<T *>(a.y)[r * a.N + col] = value_of<DT>(mine);
}

template <int DT, int BITS, int GROUP, int ROWS>
static hipError_t start_dot(const Rows8Args &a, hipStream_t st) {
  const int64_t grid = ((int64_t)a.N + 7) / 8;
  if (grid >= (int64_t)1 << 24) return hipErrorInvalidValue;  // (a launch has less than 2^32 threads)
  rows8_dot_kernel<DT, BITS, GROUP, ROWS><<<(unsigned)grid, 256, 0, st>>>(a);
  return hipGetLastError();
}

// ---------------------------------------------------------------- few rows
// A block multiplies 16 MI rows by 16 NI columns; its eight waves share K, a run of stages of 128 values each, and meet in LDS in a fixed order.  Nothing is prepared: a wave
// loads its codes, scales and rows straight into registers (a stage ahead), unpacks the codes in the rows' own order, and forms the group sums beside the products
// (a lane's part of them is an operand of the biases' product as it is).
// What bounds it is the L1 cache's tags: an operand's 16 rows are 16 lanes that follow each other, so a load is 64 accesses whatever its width (counted, 0.76 lookups a
// cycle at 16 x 14336, 0.72 at 64 x 4096).  So every load is 16 bytes a lane, also where a lane's
// values are then not those that one product of a group wants of it, and scales come for several stages at once.  us, 4-bit, groups of 64, before (8 bytes of codes and a stage's scales a load) / so:
//   8 x 4096, 4096 values 7.5 / 5.4   16 x 14336 21.9 / 12.7   32 x 4096 10.2 / 7.7   64 x 4096 14.3 / 11.0   128 x 4096 19.4 / 16.6   16 x 14336, groups of 32 35 / 16.3
// (Whole lines through LDS, passed to the lanes there: 10.1 for 16 x 4096, 32 for 16 x 14336.)
template <int DT, int BITS, int GROUP, int MI, int NI>
__global__ __launch_bounds__(512, MI * NI < 4 && !(DT == 2 && NI == 2) ? 4 : 2) void rows8_few_kernel(Rows8Args a, int wide) {
  using T = Value<DT>;
  constexpr int kWaves = 8, GS = 128 / GROUP, ROWS = 16 * MI, COLS = 16 * NI;
  constexpr int WSTAGES = GROUP == 32 ? 2 : 4, WINDOW = WSTAGES * GS;  // stages and groups whose scales are loaded at once
  __shared__ float parts[kWaves][ROWS][COLS];
  const int n0 = (int)(blockIdx.x % (uint32_t)wide) * COLS;
  const int64_t m0 = (int64_t)(blockIdx.x / (uint32_t)wide) * ROWS;
  const int lane = lane_id(), ln = lane & 15, kb = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // A lane loads 16 bytes: of 4-bit codes 32 values that follow each other (and 32 of a row), both products' of a stage; of 8-bit codes 16, one product's.  They are of one group; where the other
  // lanes' are of other groups (APART), a group's product takes zeros for the rows' values there.
  constexpr bool PAIR = BITS == 4;
  auto group_of = [&](int h) { return (PAIR ? kb * 32 : h * 64 + kb * 16) / GROUP; };
  constexpr bool APART = PAIR ? GROUP < 128 : GROUP < 64;
  const int K = a.K, n_stages = K / 128, G = K / GROUP, each = (n_stages + kWaves - 1) / kWaves;
  const int first = wave * each, last = first + each < n_stages ? first + each : n_stages;
  const signed char *xp[MI];
#pragma unroll
  for (int m = 0; m < MI; ++m) {  // rows and columns outside: the last ones again, not stored
    const int64_t row = m0 + 16 * m + ln;
    xp[m] = a.x + (row < a.M ? row : a.M - 1) * K + (PAIR ? 32 : 16) * kb;
  }
  const unsigned char *wp[NI];
  const T *sp[NI], *bp[NI];
#pragma unroll
  for (int n = 0; n < NI; ++n) {
    const int64_t col = n0 + 16 * n + ln < a.N ? n0 + 16 * n + ln : a.N - 1;
    wp[n] = reinterpret_cast<const unsigned char *>(a.w) + col * (K / 8 * BITS) + 16 * kb;
    sp[n] = static_cast<const T *>(a.s) + col * G;
    bp[n] = static_cast<const T *>(a.b) + col * G;
  }
  struct Stage {
    uint4 x[2][MI], w[PAIR ? 1 : 2][NI];
  };
  constexpr int STEP = GS * (int)sizeof(T), DWORDS = WINDOW * (int)sizeof(T) / 4;  // bytes of a stage, words of a window
  struct Window {
    uint32_t s[NI][DWORDS], b[NI][DWORDS];
  };
  auto pass = [](uint32_t (&v)[DWORDS]) __attribute__((always_inline)) {  // the next stage's to the front
#pragma unroll
    for (int i = 0; i < DWORDS; ++i) {
      if constexpr (STEP == 2) v[i] = v[i] >> 16 | (i + 1 < DWORDS ? v[i + 1] << 16 : 0u);
      else if (i + STEP / 4 < DWORDS) v[i] = v[i + STEP / 4];
    }
  };
  auto load = [&](int t, Stage &S) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < (PAIR ? 1 : 2); ++h)
#pragma unroll
      for (int n = 0; n < NI; ++n) S.w[h][n] = *reinterpret_cast<const uint4 *>(wp[n] + (t * 128 + h * 64) * BITS / 8);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int m = 0; m < MI; ++m) S.x[h][m] = *reinterpret_cast<const uint4 *>(xp[m] + t * 128 + h * (PAIR ? 16 : 64));
  };
  auto load_window = [&](int t, Window &V) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      if (t + WSTAGES <= n_stages) {
        __builtin_memcpy(V.s[n], sp[n] + t * GS, sizeof V.s[n]);
        __builtin_memcpy(V.b[n], bp[n] + t * GS, sizeof V.b[n]);
      } else {  // what is left of the columns, a stage at a time
#pragma unroll
        for (int i = 0; i < WSTAGES; ++i)
          if (t + i < n_stages) {
            __builtin_memcpy(reinterpret_cast<char *>(V.s[n]) + i * STEP, sp[n] + (t + i) * GS, STEP);
            __builtin_memcpy(reinterpret_cast<char *>(V.b[n]) + i * STEP, bp[n] + (t + i) * GS, STEP);
          }
      }
    }
  };
  i32x4_t whole = {kWholeBits, kWholeBits, kWholeBits, kWholeBits};
  asm("" : "+v"(whole));
  f32x4_t acc[MI][NI];
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int n = 0; n < NI; ++n) acc[m][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  Stage next;
  Window scales;
  if (first < last) {
    load_window(first, scales);
    load(first, next);
  }
#pragma unroll 1
  for (int t = first; t < last; ++t) {
    const Stage S = next;
    if (t + 1 < last) load(t + 1, next);
    float s[NI][GS], beta[NI][GS];
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      T sv[GS], bv[GS];
      __builtin_memcpy(sv, scales.s[n], sizeof sv);
      __builtin_memcpy(bv, scales.b[n], sizeof bv);
#pragma unroll
      for (int g = 0; g < GS; ++g) {
        constexpr float k = Centre<BITS>::of_codes;
        s[n][g] = as_f32(sv[g]);
        beta[n][g] = __builtin_fmaf(k * Centre<BITS>::value, s[n][g], k * as_f32(bv[g]));
      }
      pass(scales.s[n]);
      pass(scales.b[n]);
    }
    if ((t - first) % WSTAGES == WSTAGES - 1 && t + 1 < last) load_window(t + 1, scales);
    i32x4_t w[2][NI];
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      if constexpr (BITS == 4) {
        auto codes = [](uint32_t u, uint32_t v) {
          int32_t lo[2], hi[2];
          centred_bytes<4>(u, lo);
          centred_bytes<4>(v, hi);
          return i32x4_t{lo[0], lo[1], hi[0], hi[1]};
        };
        w[0][n] = codes(S.w[0][n].x, S.w[0][n].y);
        w[1][n] = codes(S.w[0][n].z, S.w[0][n].w);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) w[h][n] = operand_of<8>(make_uint2(S.w[h][n].x, S.w[h][n].y), make_uint2(S.w[h][n].z, S.w[h][n].w));
      }
    }
#pragma unroll
    for (int m = 0; m < MI; ++m) {
      i32x4_t x[2];
      int32_t sum[2];  // of a lane's values
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        x[h] = __builtin_bit_cast(i32x4_t, S.x[h][m]);
        sum[h] = 0;
#pragma unroll
        for (int p = 0; p < 4; ++p) sum[h] = byte_sum((uint32_t)x[h][p], sum[h]);
      }
      constexpr int SUMS = PAIR || GROUP == 128 ? 1 : 2;  // products of sums and biases: one takes what a lane has of one group
      if constexpr (SUMS == 1) sum[0] += sum[1];
#pragma unroll
      for (int n = 0; n < NI; ++n)
#pragma unroll
        for (int h = 0; h < SUMS; ++h) {
          float mine = beta[n][0];
#pragma unroll
          for (int g = 1; g < GS; ++g) mine = group_of(h) == g ? beta[n][g] : mine;
          acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)sum[h], mine, acc[m][n], 0, 0, 0);
        }
#pragma unroll
      for (int g = 0; g < GS; ++g) {
        constexpr int PER = PAIR || GROUP == 128 ? 2 : 1;  // products of a group
        i32x4_t rows[PER];
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const int h = PER == 2 ? k : g * GROUP / 64;
          rows[k] = !APART || group_of(h) == g ? x[h] : i32x4_t{0, 0, 0, 0};
        }
#pragma unroll
        for (int n = 0; n < NI; ++n) {
          i32x4_t d = whole;
#pragma unroll
          for (int k = 0; k < PER; ++k) d = __builtin_amdgcn_mfma_i32_16x16x64_i8(rows[k], w[PER == 2 ? k : g * GROUP / 64][n], d, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[m][n][i] = __builtin_fmaf(s[n][g], __int_as_float(d[i]) - kWhole, acc[m][n][i]);
        }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int n = 0; n < NI; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) parts[wave][16 * m + 4 * kb + i][16 * n + ln] = acc[m][n][i];
  __syncthreads();
#pragma unroll
  for (int c = 0; c < (ROWS * COLS + 511) / 512; ++c) {
    const int cell = c * 512 + (int)threadIdx.x, r = cell / COLS, col = n0 + cell % COLS;
    const int64_t row = m0 + r;
    if (cell >= ROWS * COLS || row >= a.M || col >= a.N) continue;
    float p[kWaves];
#pragma unroll
    for (int u = 0; u < kWaves; ++u) p[u] = parts[u][r][cell % COLS];
    float v = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    v *= a.row_scales[row] / Centre<BITS>::of_codes;
    if (a.bias) v += as_f32(static_cast<const T *>(a.bias)[col]);
    static_cast<T *>(a.y)[row * a.N + col] = value_of<DT>(v);
  }
}

template <int DT, int BITS, int GROUP, int MI, int NI>
static hipError_t start_few(const Rows8Args &a, hipStream_t st) {
  const int64_t wide = (a.N + 16 * NI - 1) / (16 * NI), grid = (a.M + 16 * MI - 1) / (16 * MI) * wide;
  if (grid > kRows8Blocks) return hipErrorInvalidValue;
  rows8_few_kernel<DT, BITS, GROUP, MI, NI><<<(unsigned)grid, 512, 0, st>>>(a, (int)wide);
  return hipGetLastError();
}

static hipError_t launch_few(const Rows8Args &a, Rows8Kind kind, int bits, int dt, hipStream_t st) {
  return rows8_with_types(dt, bits, a.group, [&](auto d, auto b, auto g) {
    constexpr int DT = decltype(d)::value, BITS = decltype(b)::value, GROUP = decltype(g)::value;
    switch (kind) {
      case Rows8Kind::kFew16x16: return start_few<DT, BITS, GROUP, 1, 1>(a, st);
      case Rows8Kind::kFew16x32: return start_few<DT, BITS, GROUP, 1, 2>(a, st);
      case Rows8Kind::kFew32x16: return start_few<DT, BITS, GROUP, 2, 1>(a, st);
      case Rows8Kind::kFew32x32: return start_few<DT, BITS, GROUP, 2, 2>(a, st);
      default: return start_few<DT, BITS, GROUP, 4, 2>(a, st);
    }
  });
}

// Operands that the fast kernels take: rows, codes and scales in pieces of up to 16 bytes, whole stages of 128 values.
static bool rows8_even(const Rows8Args &a) {
  auto even = [](const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  return a.K % 128 == 0 && a.K <= 1 << 20 && even(a.x) && even(a.w) && even(a.s) && even(a.b);
}

size_t rows8_workspace_bytes(int64_t M, int K) { return M <= kRows8NoTiles || K % 128 ? 0 : rows8_tiles_workspace_bytes(M, K); }

hipError_t launch_qmm_rows8(const Rows8Args &a, int bits, int dt, void *workspace, size_t workspace_bytes, hipStream_t st) {
  if (a.M == 0) return hipSuccess;
  if (!rows8_even(a)) {
    return rows8_with_types(dt, bits, a.group, [&](auto d, auto b, auto) { return start_plain<decltype(d)::value, decltype(b)::value>(a, st); });
  }
  if (a.M <= kRows8Dot) {
    return rows8_with_types(dt, bits, a.group, [&](auto d, auto b, auto g) {
      constexpr int DT = decltype(d)::value, BITS = decltype(b)::value, GROUP = decltype(g)::value;
      return a.M == 1 ? start_dot<DT, BITS, GROUP, 1>(a, st) : start_dot<DT, BITS, GROUP, 2>(a, st);
    });
  }
  const bool words = a.K / a.group * (dt == 2 ? 4 : 2) % 4 == 0;  // (groups of 128, 16-bit scales: an odd number of them starts half of the columns off a word)
  const bool tiles = words && workspace && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0 && workspace_bytes >= rows8_workspace_bytes(a.M, a.K);
  const Rows8Kind kind = rows8_kind(a.M, a.N, a.K, tiles);
  const int64_t step = rows8_step(kind, a.N, a.K, a.group);
  if (step == 0) return hipErrorInvalidValue;
  for (int64_t m = 0; m < a.M; m += step) {
    Rows8Args some = a;
    some.x = a.x + m * a.K;
    some.row_scales = a.row_scales + m;
    some.y = static_cast<char *>(a.y) + m * a.N * (dt == 2 ? 4 : 2);
    some.M = a.M - m < step ? a.M - m : step;
    const hipError_t e = kRows8Costs[(int)kind].tiles ? launch_rows8_tiles(some, kind, bits, dt, workspace, st) : launch_few(some, kind, bits, dt, st);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace mi_moe
