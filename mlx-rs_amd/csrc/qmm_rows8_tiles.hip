// The linear layer on 8-bit rows for many rows: tiles on the int8 matrix cores, rows prepared for them (arithmetic: qmm_rows8.hip).
#include "qmm_rows8_dev.hpp"

namespace mi_moe {

// Rows as the matrix instructions take them: for every 16 rows and 64 K values a tile of 1024 bytes, 16 a lane (row l % 16, part kb = l / 16 of the values), in the
// order in which the lane that holds the same values of a weight row has them after unpacking:
//   8-bit codes                16 consecutive values
//   4-bit codes                the words 2 kb and 2 kb + 1 of the eight, of each the even nibbles, then the odd ones
//   groups of 32 (two a tile)  8 values of each, 8 kb .. 8 kb + 7 of the group, in that order within a word
// and the group sums of 16 rows, zeros past the last group:
//   16-bit scales   eight groups a tile of 512 bytes, a lane's (row l % 16) of the groups 2 kb and 2 kb + 1: the sums' multiples of 128 as two bf16 values, then the rests, -64 .. 64 (both are
//                   exact: a sum is 2^14 at most)
//   float32 scales  four groups a tile of 64 floats (lane: row l % 16, group 4 q + kb)
__host__ __device__ constexpr int64_t row_tiles(int64_t M) { return (M + 15) / 16; }
constexpr size_t rows8_tiles_bytes(int64_t M, int K) { return (size_t)row_tiles(M) * 16 * K; }
constexpr size_t rows8_sums_bytes(int64_t M, int K, int group) { return (size_t)row_tiles(M) * ((K / group + 7) / 8) * 512; }

// A wave makes the tiles of 16 rows and four groups.
template <int BITS, int GROUP, bool WIDE>
__global__ __launch_bounds__(256) void rows8_prepare_kernel(const signed char *x, int64_t M, int K, uint4 *tiles, void *sums) {  // WIDE: float32 scales
  constexpr int NT = GROUP * 4 / 64;  // tiles of four groups
  const int lane = lane_id(), kb = lane >> 4, quads = rows8_quads(K / GROUP), n_tiles = K / 64;
  const uint32_t unit = (uint32_t)__builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));  // (fewer than 2^25)
  const int64_t mt = unit / (uint32_t)quads;
  const int q = (int)(unit % (uint32_t)quads);
  if (mt >= row_tiles(M)) return;
  const int64_t row = mt * 16 + (lane & 15);
  uint4 v[NT];  // all under way before the first is stored; outside: the last ones again
  const signed char *const at = x + (row < M ? row : M - 1) * K;
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const signed char *const p = at + (q * NT + i < n_tiles ? q * NT + i : n_tiles - 1) * 64;
    if constexpr (GROUP == 32) {
      const uint2 a = *reinterpret_cast<const uint2 *>(p + 8 * kb), b = *reinterpret_cast<const uint2 *>(p + 32 + 8 * kb);
      v[i] = make_uint4(a.x, a.y, b.x, b.y);
    } else {
      v[i] = *reinterpret_cast<const uint4 *>(p + 16 * kb);
    }
  }
  int32_t sum[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int kt = q * NT + i;
    const bool there = kt < n_tiles && row < M;
    uint2 a = there ? make_uint2(v[i].x, v[i].y) : make_uint2(0, 0), b = there ? make_uint2(v[i].z, v[i].w) : make_uint2(0, 0);
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
  if constexpr (WIDE) {
    static_cast<float *>(sums)[(mt * quads + q) * 64 + lane] = (float)(kb == 0 ? sum[0] : kb == 1 ? sum[1] : kb == 2 ? sum[2] : sum[3]);
  } else if (kb < 2) {
    const int32_t v0 = kb == 0 ? sum[0] : sum[2], v1 = kb == 0 ? sum[1] : sum[3], h0 = (v0 + 64) & ~127, h1 = (v1 + 64) & ~127;
    static_cast<uint2 *>(sums)[(mt * quads + q) * 32 + lane] = make_uint2(cvt_pk_bf16((float)h0, (float)h1), cvt_pk_bf16((float)(v0 - h0), (float)(v1 - h1)));
  }
}

// copy_to_lds with scalars that are the whole wave's, taken back out of the vector registers where the compiler holds them there
__device__ __forceinline__ void copy_scalars_to_lds(i32x4_t rsrc, uint32_t voff, uint32_t soff, uint32_t to) {
  copy_to_lds(rsrc, voff, (uint32_t)__builtin_amdgcn_readfirstlane((int)soff), (uint32_t)__builtin_amdgcn_readfirstlane((int)to));
}

// y = rows x weights in tiles of 16 MI WM rows and 16 NI WN columns, a wave 16 MI x 16 NI of them; KS groups of such waves share K, every KS-th stage each, and meet in LDS.
// A stage is 128 K values.  Everything comes in copies straight into LDS, NB - 1 stages ahead: the rows' tiles, the codes, the group sums, and the scales and biases, 16 bytes
// of a column (a window of 8 groups, or 4 of float32) at a time: a few bytes of each column a stage would be 128 lines of 128 bytes (205 us for 4096 x 4096 x 4096, 4-bit, groups of 64;
// 149 in windows).  Codes: 64 or 128 bytes of a weight row a stage, its 16-byte pieces in an order turned by the row, so that the lanes' reads meet all banks.
// A group is one matrix instruction a 16 x 16 tile (two for 128 values, one of half the depth for 32), whose integer sums are exact; then a subtraction and a
// multiply-add a result.  What bounds it is those, a matrix unit and a vector unit that do not run at once (kWhole): 4096 x 4096 x 4096, 4-bit, groups of 64, 144 us with the rows' preparation
// (956 TFLOP/s), groups of 128 1320 TFLOP/s, 32 710; counted, vector instructions are 0.86 of a SIMD's cycles and matrix units at work in 0.29.  The biases' terms are a product over the groups as well, eight of them a bf16 instruction: the sums in two exact values, their factors
// b + 8 s (b + 128 s) in as many as hold all of it.  Of bf16 scales those are two: where the smaller of b and 8 s is below half a step of the larger, it is what the first piece leaves, and has
// eight bits; where it is not, its last bit is 2^-15 or more of the larger's power of two, and what a piece of eight bits leaves, 2^-7 of that at most, has eight again.  Of f16 scales, of eleven bits, they are
// three, the last in an instruction of half the depth (with two, a factor's error would be up to 2^-17 of it; 77 and 45 us for 75 and 44 with 2048 and 777 rows, 4096 x 4096, 8-bit).  (Four groups of
// float32 a float32 instruction are 32 cycles for 16: 149, 1290 and 670; with float32 scales they remain.)
template <int DT, int BITS, int GROUP, int MI, int NI, int WM, int WN, int KS, int NB>
struct Rows8Tile {
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves * KS, ROWS = 16 * MI * WM, COLS = 16 * NI * WN;
  static constexpr int CODES = 128 * BITS / 8, PIECES = CODES / 16;                     // bytes and 16-byte pieces of a weight row's stage
  static constexpr int GS = 128 / GROUP;                                                // groups of a stage
  static constexpr int WINDOW = 16 / (DT == 2 ? 4 : 2), WSTAGES = WINDOW / GS;          // groups and stages of a window
  static constexpr int LW = WSTAGES > KS ? WSTAGES / KS : 1, NW = (NB - 2) / LW + 2;    // a group of waves' own stages in a window; windows in LDS
  static constexpr int A = ROWS * 128, B = COLS * CODES, STAGE = A + B, SCALES = COLS * 32, SUMS = ROWS * WINDOW * 4;
  static constexpr int SHARE = NB * STAGE + NW * (SCALES + SUMS);                       // of LDS, a group of waves'
  static constexpr int MEET = (KS - 1) * ROWS * COLS * 4;                               // where the groups meet, in the same place
  static constexpr int LDS = KS * SHARE > MEET ? KS * SHARE : MEET;
  static constexpr int A_COPIES = ROWS / 8, B_COPIES = B / 1024, W_COPIES = COLS / 32, S_COPIES = SUMS / 1024;
  static constexpr int COPIES = (A_COPIES + B_COPIES) / kWaves;                         // of a wave and stage, but for windows
  static_assert(A_COPIES % kWaves == 0 && B_COPIES % kWaves == 0 && W_COPIES + S_COPIES <= kWaves && ROWS % 64 == 0);
  static_assert(NB >= 2 && (NW - 1) * LW >= NB - 1 && LDS <= 160 * 1024);
};

template <int DT, int BITS, int GROUP, int MI, int NI, int WM, int WN, int KS, int NB, int OCC>
__global__ __launch_bounds__(64 * WM * WN * KS, OCC) void rows8_tiles_kernel(Rows8Args a, const uint4 *tiles, const char *sums, int n_mtiles, int n_ntiles) {
  using L = Rows8Tile<DT, BITS, GROUP, MI, NI, WM, WN, KS, NB>;
  using T = Value<DT>;
  constexpr int kWaves = L::kWaves, COLS = L::COLS, CODES = L::CODES, PIECES = L::PIECES, GS = L::GS, STAGE = L::STAGE;
  extern __shared__ __align__(16) unsigned char lds_raw[];
  const int xcd = blockIdx.x & 7, j = blockIdx.x >> 3, nt = j / n_mtiles * 8 + xcd;  // an XCD takes every eighth column tile and all row tiles of it
  if (nt >= n_ntiles) return;
  const int64_t mt0 = (int64_t)(j % n_mtiles) * (MI * WM), mt_all = row_tiles(a.M);
  const int n0 = nt * COLS;
  const int lane = lane_id(), ln = lane & 15, kb = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), share = wave / kWaves, wv = wave % kWaves, wm = wv / WN, wn = wv % WN;
  const int K = a.K, n_stages = K / 128, G = K / GROUP, sums_row = rows8_quads(G) * 256, row_bytes = K * BITS / 8, s_row = G * (int)sizeof(T);
  const uint32_t my_lds = share * L::SHARE, my_scales = my_lds + NB * STAGE;
  auto clip = [](int64_t v) { return (uint32_t)(v < INT32_MAX ? v : INT32_MAX); };
  const int64_t cols_left = a.N - n0, tiles_left = mt_all - mt0;  // (what a descriptor ends behind is zeros)
  const i32x4_t xr = words_of(reinterpret_cast<const char *>(tiles) + mt0 * K * 16, clip(tiles_left * K * 16));
  const i32x4_t qr = words_of(sums + mt0 * sums_row, clip(tiles_left * sums_row));
  const i32x4_t wr = words_of(reinterpret_cast<const char *>(a.w) + (int64_t)n0 * row_bytes, clip(cols_left * row_bytes));
  const i32x4_t sr = words_of(static_cast<const char *>(a.s) + (int64_t)n0 * s_row, clip(cols_left * s_row));
  const i32x4_t br = words_of(static_cast<const char *>(a.b) + (int64_t)n0 * s_row, clip(cols_left * s_row));
  auto turn = [](int row) { return PIECES == 4 ? (row >> 2) & 3 : (row >> 1) & 7; };
  // the stage at which the groups of the window q are multiplied with the biases: each of the groups of waves has its turn
  auto owner = [&](int q) {
    const int t = q * L::WSTAGES + q % (L::WSTAGES < KS ? L::WSTAGES : KS);
    return t < n_stages ? t : n_stages - 1;
  };
  auto copy_stage = [&](int u) __attribute__((always_inline)) {  // this share's u-th
    const int t = u * KS + share;
    const uint32_t to = my_lds + (uint32_t)(u % NB) * STAGE;
#pragma unroll
    for (int c = 0; c < L::A_COPIES / kWaves; ++c) {
      const int i = c * kWaves + wv;  // half i % 2 of tile i / 2
      copy_scalars_to_lds(xr, lane * 16, (i >> 1) * (K * 16) + t * 2048 + (i & 1) * 1024, to + i * 1024);
    }
#pragma unroll
    for (int c = 0; c < L::B_COPIES / kWaves; ++c) {
      const int i = c * kWaves + wv, row = i * (64 / PIECES) + lane / PIECES;
      copy_scalars_to_lds(wr, row * row_bytes + ((lane % PIECES) ^ turn(row)) * 16, t * CODES, to + L::A + i * 1024);
    }
    if (u % L::LW == 0) {
      const int q = t / L::WSTAGES;
      const uint32_t place = my_scales + (uint32_t)(u / L::LW % L::NW) * (L::SCALES + L::SUMS);
      if (wv < L::W_COPIES) {
        const bool second = wv >= L::W_COPIES / 2;
        const int i = second ? wv - L::W_COPIES / 2 : wv;
        if (second) copy_scalars_to_lds(br, (i * 64 + lane) * s_row, q * 16, place + wv * 1024);
        else copy_scalars_to_lds(sr, (i * 64 + lane) * s_row, q * 16, place + wv * 1024);
      }
      if (const int i = kWaves - 1 - wv; i < L::S_COPIES && (KS == 1 || owner(q) % KS == share)) {
        constexpr int LANES = L::WINDOW * 4;  // of a tile of sums
        copy_scalars_to_lds(qr, (i * (64 / LANES) + lane / LANES) * sums_row + lane % LANES * 16, q * L::WINDOW * 64, place + L::SCALES + i * 1024);
      }
    }
  };
  f32x4_t acc[MI][NI];
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int n = 0; n < NI; ++n) acc[m][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  i32x4_t whole = {kWholeBits, kWholeBits, kWholeBits, kWholeBits};
  asm("" : "+v"(whole));  // (a literal is not among the instruction's operands)
  const int mine = (n_stages - share + KS - 1) / KS, most = (n_stages + KS - 1) / KS;
#pragma unroll
  for (int u = 0; u < NB - 1; ++u)
    if (u < mine) copy_stage(u);
#pragma unroll 1
  for (int u = 0; u < most; ++u) {
    // this stage's copies are older than those of the NB - 2 behind it
    if (u + NB - 2 < mine) wait_copies<(NB - 2) * L::COPIES>();
    else wait_copies<0>();
    block_barrier();
    if (u + NB - 1 < mine) copy_stage(u + NB - 1);
    if (KS > 1 && u >= mine) break;  // (the last stage, for some of the shares)
    const int t = u * KS + share;
    const unsigned char *const at = lds_raw + my_lds + u % NB * STAGE;
    const unsigned char *const scales = lds_raw + my_scales + u / L::LW % L::NW * (L::SCALES + L::SUMS) + (wn * NI * 16 + ln) * 16;  // this lane's columns: every 16th
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
      const unsigned char *const r = at + L::A + row * CODES;
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
#pragma unroll
    for (int h = 0; h < (GROUP == 128 ? 2 : 1); ++h) {
#pragma unroll
      for (int n = 0; n < NI; ++n) read_w(h, n);
#pragma unroll
      for (int m = 0; m < MI; ++m) read_x(h, m);
    }
    float s[NI][GS];
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      T v[GS];
      __builtin_memcpy(v, __builtin_assume_aligned(scales + n * 256 + t % L::WSTAGES * (int)sizeof v, sizeof v), sizeof v);
#pragma unroll
      for (int g = 0; g < GS; ++g) s[n][g] = as_f32(v[g]);
    }
    if (const int q = t / L::WSTAGES; t == owner(q)) {
      constexpr float k = Centre<BITS>::of_codes;
      const unsigned char *const my_sums = lds_raw + my_scales + u / L::LW % L::NW * (L::SCALES + L::SUMS) + L::SCALES + wm * MI * L::WINDOW * 64;
      if constexpr (DT == 2) {
        const int g = (q * 4 + kb < G ? kb : G - 1 - q * 4) * 4;  // (past the last group the sums are zeros)
#pragma unroll
        for (int n = 0; n < NI; ++n) {
          const float beta = __builtin_fmaf(k * Centre<BITS>::value, *reinterpret_cast<const float *>(scales + n * 256 + g),
                                            k * *reinterpret_cast<const float *>(scales + COLS * 16 + n * 256 + g));
#pragma unroll
          for (int m = 0; m < MI; ++m)
            acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(*reinterpret_cast<const float *>(my_sums + m * 256 + lane * 4), beta, acc[m][n], 0, 0, 0);
        }
      } else {
        const bool there = q * 8 + 2 * kb < G;  // (an even number of groups)
        i32x4_t sum[MI];
#pragma unroll
        for (int m = 0; m < MI; ++m) {
          const uint2 v = *reinterpret_cast<const uint2 *>(my_sums + m * 512 + lane * 8);
          sum[m] = i32x4_t{(int32_t)v.x, (int32_t)v.y, (int32_t)v.x, (int32_t)v.y};
        }
#pragma unroll
        for (int n = 0; n < NI; ++n) {
          T sv[2], bv[2];
          __builtin_memcpy(sv, __builtin_assume_aligned(scales + n * 256 + 4 * kb, 4), 4);
          __builtin_memcpy(bv, __builtin_assume_aligned(scales + COLS * 16 + n * 256 + 4 * kb, 4), 4);
          float beta[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) beta[i] = there ? __builtin_fmaf(k * Centre<BITS>::value, as_f32(sv[i]), k * as_f32(bv[i])) : 0.f;
          auto pieces = [&] {  // as bf16, and what they leave
            const uint32_t p = cvt_pk_bf16(beta[0], beta[1]);
            beta[0] -= __uint_as_float(p << 16), beta[1] -= __uint_as_float(p & 0xffff0000u);
            return p;
          };
          const uint32_t first = pieces(), rest = pieces(), last = DT == 1 ? pieces() : 0;
          const i32x4_t b4 = {(int32_t)first, (int32_t)first, (int32_t)rest, (int32_t)rest};
#pragma unroll
          for (int m = 0; m < MI; ++m) {
            acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, sum[m]), __builtin_bit_cast(bf16x8_t, b4), acc[m][n], 0, 0, 0);
            if constexpr (DT == 1)
              acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(i16x4_t, i32x2_t{sum[m][0], sum[m][1]}), __builtin_bit_cast(i16x4_t, i32x2_t{(int32_t)last, (int32_t)last}),
                                                                    acc[m][n], 0, 0, 0);
          }
        }
      }
    }
    // The tiles one after the other, each multiplied LEAD steps before its sums are scaled: written out in the order in which it is to run (the compiler's own
    // order has a multiply's results used right behind it).
    constexpr int PER = GROUP == 32 ? 2 : 1, HALVES = GROUP == 128 ? 1 : 2, TILES = MI * NI, STEPS = HALVES * TILES * PER, LEAD = 2;
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
    for (int h = 0; h < (GROUP == 128 ? 2 : 1); ++h)
#pragma unroll
      for (int n = 0; n < NI; ++n) unpack(h, n);
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
  if constexpr (KS > 1) {  // the shares' results, added in their order
    f32x4_t *const meet = reinterpret_cast<f32x4_t *>(lds_raw) + wv * (MI * NI * 64) + lane;
    constexpr int EACH = kWaves * MI * NI * 64;
    wait_copies<0>();
    block_barrier();
    if (share > 0) {
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int n = 0; n < NI; ++n) meet[(share - 1) * EACH + (m * NI + n) * 64] = acc[m][n];
    }
    wait_reads();
    block_barrier();
    if (share > 0) return;
#pragma unroll
    for (int m = 0; m < MI; ++m)
#pragma unroll
      for (int n = 0; n < NI; ++n)
#pragma unroll
        for (int o = 0; o < KS - 1; ++o) acc[m][n] += meet[o * EACH + (m * NI + n) * 64];
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

template <int DT, int BITS, int GROUP, int MI, int NI, int WM, int WN, int KS, int NB, int OCC>
static hipError_t start_tile(const Rows8Args &a, const uint4 *tiles, const char *sums, hipStream_t st) {
  using L = Rows8Tile<DT, BITS, GROUP, MI, NI, WM, WN, KS, NB>;
  const int64_t n_mtiles = (a.M + L::ROWS - 1) / L::ROWS, n_ntiles = (a.N + L::COLS - 1) / L::COLS, grid = (n_ntiles + 7) / 8 * 8 * n_mtiles;
  if (grid * L::kThreads >= (int64_t)1 << 32) return hipErrorInvalidValue;
  const auto kernel = &rows8_tiles_kernel<DT, BITS, GROUP, MI, NI, WM, WN, KS, NB, OCC>;
  static std::atomic<uint64_t> allowed{0};
  if (hipError_t e = allow_lds(reinterpret_cast<const void *>(kernel), L::LDS, allowed); e != hipSuccess) return e;
  kernel<<<(unsigned)grid, L::kThreads, L::LDS, st>>>(a, tiles, sums, (int)n_mtiles, (int)n_ntiles);
  return hipGetLastError();
}

size_t rows8_tiles_workspace_bytes(int64_t M, int K) { return rows8_tiles_bytes(M, K) + rows8_sums_bytes(M, K, 32); }

hipError_t launch_rows8_tiles(const Rows8Args &a, Rows8Kind kind, int bits, int dt, void *workspace, hipStream_t st) {
  uint4 *const tiles = static_cast<uint4 *>(workspace);
  char *const sums = static_cast<char *>(workspace) + rows8_tiles_bytes(a.M, a.K);
  const int64_t units = row_tiles(a.M) * rows8_quads(a.K / a.group);
  if (units > kRows8Units) return hipErrorInvalidValue;
  return rows8_with_types(dt, bits, a.group, [&](auto d, auto b, auto g) {
    constexpr int DT = decltype(d)::value, BITS = decltype(b)::value, GROUP = decltype(g)::value;
    rows8_prepare_kernel<BITS, GROUP, DT == 2><<<(unsigned)((units + 3) / 4), 256, 0, st>>>(a.x, a.M, a.K, tiles, sums);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    if (kind == Rows8Kind::kTiles64x64) return start_tile<DT, BITS, GROUP, 2, 2, 2, 2, 2, 2, 4>(a, tiles, sums, st);
    if (kind == Rows8Kind::kTiles64x128) return start_tile<DT, BITS, GROUP, 2, 2, 2, 4, 1, 2, 4>(a, tiles, sums, st);
    return start_tile<DT, BITS, GROUP, 4, 2, 2, 4, 1, 2, 4>(a, tiles, sums, st);
  });
}

}  // namespace mi_moe
