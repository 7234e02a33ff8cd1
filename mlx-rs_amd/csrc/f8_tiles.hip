// Products with e4m3 weights in tiles: prompts, training batches, and gradients with respect to the input (weights summed along their rows).
//
// A block of eight waves, two along the token rows and four along the weight rows, computes TM token rows x 256 weight rows (kPair: 128 gate and the matching 128 up
// rows).  Its stage is one run of 128 values: the weight rows are the 32x32x64 instruction's rows and token rows its columns, so that a lane has one token row's scale
// and sixteen sums of it.  A run's two instructions start from zero, their sums are scaled and added in float32 while the next ones run.
#include <atomic>
#include <type_traits>

#include "f8.hpp"
#include "lds_copies.hpp"

namespace mi_moe {

enum F8Mode { kRowsOfWeights, kPair, kColsOfWeights };  // matrices [N][K]; two such, into h; matrices [K][N]
constexpr int kF8Threads = 512, kF8FewPieces = 32;
constexpr uint32_t kF8Outside = 0xfffffff0u;  // an offset past every descriptor's end: zeros

// 4 bytes a lane into LDS, at `to` + 4 lane
__device__ __forceinline__ void copy4_to_lds(i32x4_t rsrc, uint32_t voff, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(to), "v"(voff), "s"(rsrc) : "m0", "memory");
}
__device__ __forceinline__ i32x4_t uniform(i32x4_t v) {
  return i32x4_t{__builtin_amdgcn_readfirstlane(v.x), __builtin_amdgcn_readfirstlane(v.y), __builtin_amdgcn_readfirstlane(v.z), __builtin_amdgcn_readfirstlane(v.w)};
}
__device__ __forceinline__ uint32_t at_most_4g(int64_t bytes) { return bytes > 0xffffff00ll ? 0xffffff00u : (uint32_t)bytes; }

// The sixteen-byte pieces of a tile's row of 128 lie turned by the row's number, so that sixteen rows one after the other, which a read takes at once, have a piece in
// different banks.
__device__ __forceinline__ constexpr int f8_turn(int row) { return row >> 1 & 7; }

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)lo) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)hi) << 16;
}

template <int TM>
struct F8Stage {
  // token rows, weight rows, a scale a token row, and 256 bytes each of the scale of the tile's first and second 128 weight rows
  static constexpr int X = TM * 128, W = kF8TileN * 128, S = TM * 4, BYTES = X + W + S + 512;
};

constexpr size_t f8_tiles_lds(int tm) {  // two stages, and what a thread copies
  return 2 * (size_t)(tm * 128 + kF8TileN * 128 + tm * 4 + 512) + kF8Threads * 4 * (tm / 64) + tm * 4;
}

struct F8Grid {
  int m_tiles, n_tiles, xcds_m, m_each, n_each;  // one matrix: xcds_m XCDs along the token rows, rectangles of m_each x n_each tiles
  int part_steps;                                // stages of a block: fewer than all where blocks share a tile, whose sums then go to a.parts
  int n_first, n_end;                            // columns of y (F8Product)
  uint32_t first;                                // block, where a product takes more than one launch
};

// Sums of parts, in their order, a bias added, rounded.
__global__ __launch_bounds__(256) void f8_parts_kernel(const float *__restrict__ parts, int n_parts, int64_t rows, int N, const void *__restrict__ bias, int dt, void *__restrict__ y) {
  const int n = ((int)blockIdx.x * 256 + (int)threadIdx.x) * 4;
  const int64_t row = blockIdx.y;
  if (n >= N) return;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int p = 0; p < n_parts; ++p) {
    const float *const from = parts + ((int64_t)p * rows + row) * N + n;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (n + 4 <= N) __builtin_memcpy(v, from, 16);
    else
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = n + i < N ? from[i] : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] += v[i];
  }
  if (bias)
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] += n + i < N ? value_of(bias, n + i, dt) : 0.f;
  store4(y, row * N + n, N - n, dt, sum);
}

// EXACT: on the bf16 instructions (f8_exact).  WIDE: results are float32.
template <int TM, F8Mode MODE, bool EXACT, bool WIDE>
__global__ __launch_bounds__(kF8Threads) void f8_tiles_kernel(F8Product a, F8Grid g) {
  typedef F8Stage<TM> L;
  constexpr int XC = TM / 64, MT = TM / 64;  // copies of token rows a wave; sub-tiles of 32 token rows a wave
  extern __shared__ __align__(16) unsigned char lds[];
  const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)lds;
  const int N = a.N, K = a.K, runs = f8_runs(K), n_blocks = f8_runs(N), steps = a.pair_sum ? 2 * runs : runs;
  const int begin = (int)blockIdx.y * g.part_steps, end = begin + g.part_steps < steps ? begin + g.part_steps : steps;
  // Blocks go round the eight XCDs, each of which has an L2 of its own.  One matrix: an XCD takes a rectangle of tiles.  Several: all tiles of a piece go to one XCD.  (A matrix's
  // pieces beside each other on one XCD, and blocks that take tile after tile, were tried: fewer misses of L2, and no faster, or slower by what the shares differ in time.)
  const uint32_t block = g.first + blockIdx.x, xcd = block & 7, q = block >> 3;
  uint32_t mt, nt;
  if (!a.list) {
    mt = (xcd % (uint32_t)g.xcds_m) * (uint32_t)g.m_each + q % (uint32_t)g.m_each;
    nt = (xcd / (uint32_t)g.xcds_m) * (uint32_t)g.n_each + q / (uint32_t)g.m_each;
  } else if (g.m_tiles < kF8FewPieces) {  // (too few pieces to give each XCD as many: 26 rows at one matrix of 2128 x 1792 took 23 us, all on one, not 16)
    mt = block % (uint32_t)g.m_tiles;
    nt = block / (uint32_t)g.m_tiles;
  } else {
    mt = q / (uint32_t)g.n_tiles * 8 + xcd;
    nt = q % (uint32_t)g.n_tiles;
  }
  if (mt >= (uint32_t)g.m_tiles || nt >= (uint32_t)g.n_tiles) return;
  const F8Piece piece = f8_piece(a, TM, mt);
  const int rows = (int)piece.rows, mat = piece.mat;
  const uint32_t row0 = piece.row;
  if (rows == 0) return;
  const int lane = threadIdx.x & 63, ln = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 2, wn = wave & 3;
  // (column n of y's row r: r y_stride + n - n_first; only float32 rows come in parts of the columns, and the others' ends are 2 % faster without this)
  const int n_first = WIDE ? g.n_first : 0, n_end = WIDE ? g.n_end : N;
  const int64_t y_stride = n_end - n_first;
  const int n0 = MODE == kPair ? nt * 128 : n_first + nt * kF8TileN;
  const int product = MODE == kRowsOfWeights ? (int)blockIdx.z : 0;  // (two at most, of the same rows)
  void *const y = product ? a.y1 : a.y;
  if (mat == a.n_mats) {  // rows of no matrix (scaled ones are read by nobody)
    if constexpr (MODE != kPair) {
      const float none[4] = {0.f, 0.f, 0.f, 0.f};
      const bool part = g.part_steps < steps;
      void *const to = part ? a.parts + (int64_t)blockIdx.y * a.rows * N : y;  // (parts: of all columns)
      for (int i = threadIdx.x; i < rows * (kF8TileN / 4); i += kF8Threads) {
        const int n = n0 + i % (kF8TileN / 4) * 4;
        if (n < n_end) store4(to, (row0 + i / (kF8TileN / 4)) * y_stride + n - n_first, n_end - n, part ? 2 : a.dt, none);
      }
    }
    return;
  }
  // ---- what a lane copies of a stage
  const int64_t wide = (int64_t)steps * kF8Run;
  auto source = [&](int r) __attribute__((always_inline)) {  // x row of the piece's row r, as the descriptors below count (rows past the end are zeros)
    if (!a.order) return (uint32_t)r;
    const uint32_t at = a.order[row0 + r] / (uint32_t)a.k_div;
    return at < (uint32_t)a.x.rows ? at : 0u;
  };
  const int64_t x_first = a.order ? 0 : row0, x_rows = a.order ? a.x.rows : rows;
  const i32x4_t xr = uniform(words_of(a.x.codes + x_first * wide, at_most_4g(x_rows * wide)));
  // (in LDS between a stage and the next: the registers are for the sums)
  uint32_t *const x_offs = reinterpret_cast<uint32_t *>(lds + 2 * L::BYTES), *const s_offs = reinterpret_cast<uint32_t *>(lds + 2 * L::BYTES) + kF8Threads * XC;
#pragma unroll
  for (int c = 0; c < XC; ++c) {
    const int r = (wave * XC + c) * 8 + lane / 8;
    x_offs[threadIdx.x * XC + c] = r < rows ? source(r) * (uint32_t)wide + (uint32_t)((lane % 8) ^ f8_turn(r)) * 16 : kF8Outside;
  }
  if (threadIdx.x < TM) s_offs[threadIdx.x] = (int)threadIdx.x < rows ? source(threadIdx.x) * 4 : kF8Outside;
  const int64_t matrix = (int64_t)mat * N * K;
  i32x4_t wr{};
  if constexpr (MODE != kColsOfWeights) {
    const int which = MODE == kPair ? wave >> 2 : product;  // waves 4 to 7 copy the up rows
    wr = uniform(words_of(a.m[which].w + matrix + (int64_t)n0 * K, at_most_4g((int64_t)(N - n0) * K)));
  }
  // where the scales of the wave's half of the weight rows are (past the last block its own again, of rows that are never stored)
  const float *w_scale[2];
  {
    const int second = wave & 1, block = MODE == kPair ? nt : n0 / kF8Run + second < n_blocks ? n0 / kF8Run + second : n_blocks - 1;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      w_scale[i] = MODE == kPair ? a.m[second].s + ((int64_t)mat * n_blocks + block) * runs : MODE == kRowsOfWeights ? a.m[product].s + ((int64_t)mat * n_blocks + block) * runs
                                                                                                                     : a.m[i].s + (int64_t)mat * runs * n_blocks + block;
  }
  // Token rows and all scales, XC + 2 copies.  (Every wave copies scales, several the same: with a branch around them the compiler puts the sums' arithmetic off past it.)
  struct Offsets {
    uint32_t x[XC], s;
  };
  auto offsets = [&]() __attribute__((always_inline)) {
    Offsets o;
    uint32_t own = threadIdx.x;
    asm volatile("" : "+v"(own));  // (addresses are made where they are used: there are no registers to keep them)
#pragma unroll
    for (int c = 0; c < XC; ++c) o.x[c] = x_offs[own * XC + c];
    o.s = s_offs[wave % (TM / 64) * 64 + own % 64];
    return o;
  };
  auto fetch_rows = [&](int j, const Offsets &o) __attribute__((always_inline)) {
    const uint32_t at = lds_at + (j & 1) * L::BYTES;
#pragma unroll
    for (int c = 0; c < XC; ++c) copy_to_lds(xr, o.x[c], (uint32_t)(j * kF8Run), at + (wave * XC + c) * 1024);
    copy4_to_lds(uniform(words_of(a.x.scales + (int64_t)j * a.x.rows + x_first, at_most_4g(x_rows * 4))), o.s, at + L::X + L::W + wave % (TM / 64) * 256);
    const float *const from = MODE != kColsOfWeights ? w_scale[0] + j : j < runs ? w_scale[0] + (int64_t)j * n_blocks : w_scale[1] + (int64_t)(j - runs) * n_blocks;
    copy4_to_lds(uniform(words_of(from, 4)), 0, at + L::X + L::W + L::S + (wave & 1) * 256);
  };
  auto fetch_weights = [&](int j) __attribute__((always_inline)) {  // four copies
    const uint32_t at = lds_at + (j & 1) * L::BYTES;
    uint32_t l = threadIdx.x & 63;
    asm volatile("" : "+v"(l));
    if constexpr (MODE != kColsOfWeights) {
      // rows c * 8 + l / 8 of the wave's 32, whose pieces are turned by half the row's number
      const bool whole = (j + 1) * kF8Run <= K;
      const uint32_t row = (uint32_t)((MODE == kPair ? wave & 3 : wave) * 32 + l / 8) * (uint32_t)K, piece = ((l % 8) ^ (l / 16)) * 16;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        // (the scalar offset stays within a row: past the descriptor's end it would not be checked)
        const uint32_t k = piece ^ ((c & 1) * 64), off = row + (uint32_t)(c * 8 * K) + k;
        copy_to_lds(wr, whole || j * kF8Run + (int)k < K ? off : kF8Outside, (uint32_t)(j * kF8Run), at + L::X + (wave * 4 + c) * 1024);
      }
    } else {
      // matrices [K][N]: rows c * 4 + l / 16 of the wave's sixteen, 256 columns each, whose pieces of sixteen are turned by twice the row's number (mod 8)
      const bool second = j >= runs;
      const int k0 = (second ? j - runs : j) * kF8Run;
      // (rows past the matrix's last one are past the descriptor's end)
      const i32x4_t from = uniform(words_of(a.m[second].w + matrix + (int64_t)k0 * N + n0, at_most_4g(((int64_t)K - k0) * N - n0)));
      const uint32_t row = (uint32_t)(wave * 16 + l / 16) * (uint32_t)N, piece = ((l % 16) ^ (l / 16 * 2)) * 16;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t col = piece ^ ((c & 1) * 128);
        copy_to_lds(from, n0 + (int)col < N ? row + (uint32_t)(c * 4 * N) + col : kF8Outside, 0, at + L::X + (wave * 4 + c) * 1024);
      }
    }
  };

  f32x16_t acc[MT][2];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[t][i][v] = 0.f;
  const int x_at = (wm * 32 + ln) * 128, w_at0 = (MODE == kPair ? wn * 32 + ln : wn * 64 + ln) * 128, w_at1 = w_at0 + (MODE == kPair ? 128 : 32) * 128;
  // matrices [K][N]: a lane's place for the transposing reads, which give each of sixteen lanes eight values of its column out of eight rows of sixteen columns
  const int c_k = (lane & 15) >> 1, c_at = (half * 32 + c_k) * 256 + (((wn * 4 + (lane >> 4 & 1)) ^ (2 * c_k)) * 16) + (lane & 1) * 8;
  const int turn = f8_turn(ln);  // (rows 32 apart are turned alike)
  auto operand = [&](const unsigned char *row, int q) __attribute__((always_inline)) {  // values 64 q + 32 half to 64 q + 32 half + 31
    const u32x4_f8 lo = *reinterpret_cast<const u32x4_f8 *>(row + ((4 * q + 2 * half) ^ turn) * 16), hi = *reinterpret_cast<const u32x4_f8 *>(row + ((4 * q + 2 * half + 1) ^ turn) * 16);
    return i32x8_t{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
  };
  auto weights = [&](const unsigned char *tile, int i, int q) __attribute__((always_inline)) {
    if constexpr (MODE != kColsOfWeights) return operand(tile + (i ? w_at1 : w_at0), q);
    typedef int pair_t __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) pair_t lds_pair_t;
    i32x8_t v;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const pair_t r = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_pair_t *)(tile + (c_at ^ (i * 32)) + (64 * q + 8 * p) * 256));
      v[2 * p] = r.x, v[2 * p + 1] = r.y;
    }
    return v;
  };
  auto multiply = [&](const i32x8_t &w, const i32x8_t &x, f32x16_t sum) __attribute__((always_inline)) {
    if constexpr (EXACT) {
#pragma unroll
      for (int p = 0; p < 4; ++p)
        sum = __builtin_amdgcn_mfma_f32_32x32x16_bf16(codes_to_bf16((uint32_t)w[2 * p], (uint32_t)w[2 * p + 1]), codes_to_bf16((uint32_t)x[2 * p], (uint32_t)x[2 * p + 1]), sum, 0, 0, 0);
      return sum;
    } else {
      return mfma_f8_32(w, x, sum);
    }
  };

  // The stages of a wave with LIVE sub-tiles of token rows.  An operand's registers take the next one's values as soon as its last multiply has been issued: those of the
  // next sub-tile, and in the last sub-tile's time those of the next stage.  So a stage has one barrier, amid its multiplies, ahead of the last sub-tile: all waves have read what
  // they read of the stage by then, whose place the copies of the stage after the next may take, and the next stage's copies have arrived.
  auto add = [&](f32x16_t &to, const f32x16_t &sum, float f) __attribute__((always_inline)) {
#pragma unroll
    for (int v = 0; v < 16; ++v) to[v] = __builtin_fmaf(sum[v], f, to[v]);
  };
  auto all_stages = [&](auto live_of) __attribute__((always_inline)) {
    constexpr int LIVE = decltype(live_of)::value, LAST = LIVE - 1;
    i32x8_t w[2][2], x[2];  // [weight sub-tile][half of the run]
    auto stage = [&](int j, bool more) __attribute__((always_inline)) {
      if constexpr (LIVE == 0) {
        wait_copies<0>();
        block_barrier();
        if (more) {
          fetch_rows(j + 2, offsets());
          fetch_weights(j + 2);
        }
      } else {
        const unsigned char *const at = lds + (j & 1) * L::BYTES, *const next = lds + ((j + 1) & 1) * L::BYTES;  // (behind the last stage: a place that nothing waits for)
        const float *const sx = reinterpret_cast<const float *>(at + L::X + L::W) + wm * 32 + ln, *const sw = reinterpret_cast<const float *>(at + L::X + L::W + L::S);
        const float s0 = sw[MODE == kPair ? 0 : (wn >> 1) * 64], s1 = MODE == kPair ? sw[64] : s0;
        float s = sx[0];
#pragma unroll
        for (int t = 0; t < LIVE; ++t) {
          Offsets o{};
          if (t == LAST) {
            wait_copies<0>();
            block_barrier();
            if (more) o = offsets();
          }
          f32x16_t sum[2] = {};
          const float now = s;
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            sum[0] = multiply(w[0][q], x[q], sum[0]);
            sum[1] = multiply(w[1][q], x[q], sum[1]);
            __builtin_amdgcn_sched_barrier(0);  // (no operand earlier: there are no registers for more)
            if (t == LAST) {
              if (more && q == 0) fetch_rows(j + 2, o);
              if (more && q == 1) fetch_weights(j + 2);
              w[0][q] = weights(next + L::X, 0, q);
              w[1][q] = weights(next + L::X, 1, q);
              x[q] = operand(next + x_at, q);
            } else {
              x[q] = operand(at + x_at + (t + 1) * 64 * 128, q);
              if (q == 0) s = sx[(t + 1) * 64];
            }
          }
          add(acc[t][0], sum[0], now * s0);
          add(acc[t][1], sum[1], now * s1);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    if constexpr (LIVE > 0) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const unsigned char *const at = lds + (begin & 1) * L::BYTES;
        w[0][q] = weights(at + L::X, 0, q);
        w[1][q] = weights(at + L::X, 1, q);
        x[q] = operand(at + x_at, q);
      }
    }
    int j = begin;
    for (; j + 2 < end; ++j) stage(j, true);
    for (; j < end; ++j) stage(j, false);
  };
  __syncthreads();  // (offsets of scales come from other threads)
  fetch_rows(begin, offsets());
  fetch_weights(begin);
  if (begin + 1 < end) {
    fetch_rows(begin + 1, offsets());
    fetch_weights(begin + 1);
    wait_copies<XC + 6>();
  } else {
    wait_copies<0>();
  }
  block_barrier();
  const int live = (rows - wm * 32 + 63) / 64;  // sub-tiles of this wave's (every other one of the block's) that hold rows
  if (live >= MT) all_stages(std::integral_constant<int, MT>());
  else if (MT > 3 && live == 3) all_stages(std::integral_constant<int, (MT > 3 ? 3 : 0)>());
  else if (MT > 2 && live == 2) all_stages(std::integral_constant<int, (MT > 2 ? 2 : 0)>());
  else if (MT > 1 && live == 1) all_stages(std::integral_constant<int, (MT > 1 ? 1 : 0)>());
  else all_stages(std::integral_constant<int, 0>());

  // Results: a lane has token row ln of each sub-tile, and of weight rows 8 g + 4 half + 0..3 the sums 4 g + 0..3.  They go through LDS, rows of 128 bytes whose pieces of
  // sixteen are turned as the operands', and out of it in whole lines: stored as they lie, 8 bytes a lane and 32 rows an instruction, a 4096 x 4096 bf16 result took 16 us.
  __syncthreads();  // (all waves have read their last operands)
  if constexpr (MODE == kPair) {
    float *const most = reinterpret_cast<float *>(lds + TM * 128);  // [4][TM]
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      if (t < live) {
        uint32_t m = 0;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          acc[t][0][v] = silu(acc[t][0][v]) * acc[t][1][v];
          m = umax(m, abs_bits(acc[t][0][v]));
        }
        m = umax(m, (uint32_t)__shfl_xor((int)m, 32, kWave));
        if (half == 0) most[wn * TM + (2 * t + wm) * 32 + ln] = __uint_as_float(m);
      }
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      if (t < live) {
        const int r = (2 * t + wm) * 32 + ln;
        uint32_t all = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) all = umax(all, __float_as_uint(most[i * TM + r]));
        const F8Scale s(all);
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<uint32_t *>(lds + r * 128 + ((wn * 2 + (g >> 1)) ^ f8_turn(r)) * 16 + (g & 1) * 8 + half * 4) =
              s.codes(acc[t][0][4 * g], acc[t][0][4 * g + 1], acc[t][0][4 * g + 2], acc[t][0][4 * g + 3]);
        if (wn == 0 && half == 0 && r < rows) a.hs[(int64_t)nt * a.rows + row0 + r] = s.scale;
      }
    }
    __syncthreads();
    const int64_t h_wide = (int64_t)n_blocks * kF8Run;
    for (int r = threadIdx.x / 8; r < rows; r += kF8Threads / 8)
      *reinterpret_cast<u32x4_f8 *>(a.h + (int64_t)(row0 + r) * h_wide + n0 + ((threadIdx.x % 8) ^ f8_turn(r)) * 16) =
          *reinterpret_cast<const u32x4_f8 *>(lds + r * 128 + threadIdx.x % 8 * 16);
  } else if (g.part_steps < steps) {
    float *const to = a.parts + (int64_t)blockIdx.y * a.rows * N;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int r = (2 * t + wm) * 32 + ln;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int n = n0 + wn * 64 + i * 32 + 8 * v + 4 * half;
          const float o[4] = {acc[t][i][4 * v], acc[t][i][4 * v + 1], acc[t][i][4 * v + 2], acc[t][i][4 * v + 3]};
          if (r < rows && n < N) store4(to, (int64_t)(row0 + r) * N + n, N - n, 2, o);
        }
    }
  } else {
    constexpr int SIZE = WIDE ? 4 : 2, EACH = 16 / SIZE, PASSES = WIDE ? 2 : 1;  // bytes of a value, values of a piece; 64 weight rows at once, or 32
    unsigned char *const own = lds + wave * (32 * MT * 128);
    float down[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) down[t] = 1.f;
    if constexpr (!WIDE) {
      if (a.y_scales) {
        // to within 2^15, by the exponent of the largest of a row's 64 values
        const int column = n0 / 64 + wn;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          if (t >= live) continue;
          float most = 0.f;  // (of the numbers among them)
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int v = 0; v < 16; ++v) most = fmaxf(most, fabsf(acc[t][i][v]));
          most = fmaxf(most, __shfl_xor(most, 32, kWave));
          if (most == __builtin_inff()) {  // (rare: the scale is that of the finite ones)
            most = 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int v = 0; v < 16; ++v)
                if (const float one = fabsf(acc[t][i][v]); one < __builtin_inff()) most = fmaxf(most, one);
            most = fmaxf(most, __shfl_xor(most, 32, kWave));
          }
          const int r = (2 * t + wm) * 32 + ln, exponent = (int)(__float_as_uint(most) >> 23);
          const int by = exponent < 27 ? -114 : exponent - 141;  // (the least values a little less exactly)
          down[t] = __uint_as_float((uint32_t)(127 - by) << 23);
          if (half == 0 && r < rows && column * 64 < N) a.y_scales[(int64_t)(row0 + r) * ((N + 63) / 64) + column] = __uint_as_float((uint32_t)(127 + by) << 23);
        }
      }
    }
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
#pragma unroll
      for (int i = pass; i < (WIDE ? pass + 1 : 2); ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float bias[4] = {0.f, 0.f, 0.f, 0.f};
          if (a.bias)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              const int n = n0 + wn * 64 + i * 32 + 8 * g + 4 * half + v;
              bias[v] = n < N ? value_of(a.bias, n, a.dt) : 0.f;
            }
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            if (t >= live) continue;
            const int r = t * 32 + ln;
            float o[4];
#pragma unroll
            for (int v = 0; v < 4; ++v) o[v] = __builtin_fmaf(acc[t][i][4 * g + v], down[t], bias[v]);
            const int piece = WIDE ? 2 * g + half : i * 4 + g;
            unsigned char *const to = own + r * 128 + (piece ^ f8_turn(r)) * 16 + (WIDE ? 0 : half * 8);
            if constexpr (WIDE) *reinterpret_cast<f32x4_t *>(to) = f32x4_t{o[0], o[1], o[2], o[3]};
            else if (a.dt == 0 && !a.y_scales) *reinterpret_cast<uint2 *>(to) = make_uint2(cvt_pk_bf16(o[0], o[1]), cvt_pk_bf16(o[2], o[3]));
            else *reinterpret_cast<uint2 *>(to) = make_uint2(pack_f16(o[0], o[1]), pack_f16(o[2], o[3]));
          }
        }
#pragma unroll
      for (int r0 = 0; r0 < 32 * MT; r0 += 8) {
        if (r0 >= 32 * live) continue;
        const int r = r0 + lane / 8, n = n0 + wn * 64 + pass * 32 + ((lane % 8) ^ f8_turn(r)) * EACH;
        const u32x4_f8 v = *reinterpret_cast<const u32x4_f8 *>(own + r * 128 + lane % 8 * 16);
        const int row = (r0 / 32 * 2 + wm) * 32 + r % 32;
        if (row < rows && n < n_end) {
          unsigned char *const to = static_cast<unsigned char *>(y) + ((row0 + row) * y_stride + n - n_first) * SIZE;
          if (n + EACH <= n_end) {
            __builtin_memcpy(to, &v, 16);
          } else {
#pragma unroll
            for (int e = 0; e < EACH; ++e)
              if (n + e < n_end) __builtin_memcpy(to + e * SIZE, reinterpret_cast<const unsigned char *>(&v) + e * SIZE, SIZE);
          }
        }
      }
    }
  }
}

template <int TM, F8Mode MODE, bool EXACT, bool WIDE>
static hipError_t launch_tiles(const F8Product &p, hipStream_t st) {
  constexpr size_t lds = f8_tiles_lds(TM);
  constexpr int kMaxDevices = 64;
  static std::atomic<bool> raised[kMaxDevices];  // more LDS than a kernel gets without asking
  int dev = 0;
  if (hipError_t e = hipGetDevice(&dev); e != hipSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices || !raised[dev].load(std::memory_order_acquire)) {
    if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&f8_tiles_kernel<TM, MODE, EXACT, WIDE>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds); e != hipSuccess) return e;
    if (dev >= 0 && dev < kMaxDevices) raised[dev].store(true, std::memory_order_release);
  }
  const int n_end = p.n_count ? p.n_first + p.n_count : p.N;
  const int64_t n_tiles = (n_end - p.n_first + (MODE == kPair ? 127 : kF8TileN - 1)) / (MODE == kPair ? 128 : kF8TileN), m_tiles = p.list ? f8_most_pieces(p.rows, p.n_mats, TM) : (p.rows + TM - 1) / TM;
  const int steps = f8_runs(p.K) * (p.pair_sum ? 2 : 1), parts = f8_plan(p).parts;
  F8Grid g{(int)m_tiles, (int)n_tiles, 1, (int)m_tiles, (int)((n_tiles + 7) / 8), (steps + parts - 1) / parts, p.n_first, n_end, 0};
  int64_t each;  // blocks of an XCD
  if (p.list) {
    each = m_tiles < kF8FewPieces ? (m_tiles * n_tiles + 7) / 8 : (m_tiles + 7) / 8 * n_tiles;
  } else {
    for (int xm = 2; xm <= 8; xm *= 2) {
      const int m_each = (int)((m_tiles + xm - 1) / xm), n_each = (int)((n_tiles + 8 / xm - 1) / (8 / xm));
      const int64_t now = (int64_t)g.m_each * g.n_each, then = (int64_t)m_each * n_each;
      if (then < now || (then == now && m_each * TM + n_each * kF8TileN < g.m_each * TM + g.n_each * kF8TileN)) g.xcds_m = xm, g.m_each = m_each, g.n_each = n_each;
    }
    each = (int64_t)g.m_each * g.n_each;
  }
  const unsigned used = (unsigned)((steps + g.part_steps - 1) / g.part_steps);
  constexpr int64_t most = (int64_t)1 << 22;  // blocks of a launch, which has less than 2^32 threads
  for (int64_t first = 0; first < each * 8; first += most) {
    g.first = (uint32_t)first;
    f8_tiles_kernel<TM, MODE, EXACT, WIDE><<<dim3((unsigned)(each * 8 - first < most ? each * 8 - first : most), used, p.y1 ? 2 : 1), kF8Threads, lds, st>>>(p, g);
  }
  if (used > 1) f8_parts_kernel<<<dim3((unsigned)((p.N + 1023) / 1024), (unsigned)p.rows), 256, 0, st>>>(p.parts, (int)used, p.rows, p.N, p.bias, p.dt, p.y);
  return hipGetLastError();
}

template <F8Mode MODE>
static hipError_t launch_mode(const F8Product &p, hipStream_t st) {
  const int tile = f8_plan(p).tile;
  if (!f8_exact(p))
    return tile == 256 ? launch_tiles<256, MODE, false, false>(p, st) : tile == 128 ? launch_tiles<128, MODE, false, false>(p, st) : launch_tiles<64, MODE, false, false>(p, st);
  if constexpr (MODE != kPair)
    if (p.dt == 2) return tile == 128 ? launch_tiles<128, MODE, true, true>(p, st) : launch_tiles<64, MODE, true, true>(p, st);
  return tile == 128 ? launch_tiles<128, MODE, true, false>(p, st) : launch_tiles<64, MODE, true, false>(p, st);
}

hipError_t launch_f8_tiles(const F8Product &p, hipStream_t st) {
  if (p.rows == 0) return hipSuccess;
  if (p.h) return launch_mode<kPair>(p, st);
  if (!p.transpose) return launch_mode<kColsOfWeights>(p, st);
  return launch_mode<kRowsOfWeights>(p, st);
}

}  // namespace mi_moe
