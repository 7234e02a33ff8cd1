// Products with e4m3 weights in tiles: prompts, training batches, and gradients with respect to the input (weights summed along their rows).
//
// A block of eight waves, two along the token rows and four along the weight rows, computes TM token rows x 256 weight rows (kPair: 128 gate and the matching 128 up
// rows).  Its stage is one run of 128 values: the weight rows are the 32x32x64 instruction's rows and token rows its columns, so that a lane has one token row's scale
// and sixteen sums of it.  A run's two instructions start from zero, their sums are scaled and added in float32 while the next ones run.
#include <atomic>

#include "f8.hpp"
#include "lds_copies.hpp"

namespace mi_moe {

enum F8Mode { kRowsOfWeights, kPair, kColsOfWeights };  // matrices [N][K]; two such, into h; matrices [K][N]
constexpr int kF8TileN = 256, kF8Threads = 512;
constexpr uint32_t kF8Outside = 0xfffffff0u;  // an offset past every descriptor's end: zeros

// 4 bytes a lane into LDS, at `to` + 4 lane
__device__ __forceinline__ void copy4_to_lds(i32x4_t rsrc, uint32_t voff, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(to), "v"(voff), "s"(rsrc) : "m0", "memory");
}
__device__ __forceinline__ i32x4_t uniform(i32x4_t v) {
  return i32x4_t{__builtin_amdgcn_readfirstlane(v.x), __builtin_amdgcn_readfirstlane(v.y), __builtin_amdgcn_readfirstlane(v.z), __builtin_amdgcn_readfirstlane(v.w)};
}
__device__ __forceinline__ uint32_t at_most_4g(int64_t bytes) { return bytes > 0xffffff00ll ? 0xffffff00u : (uint32_t)bytes; }

// The sixteen-byte pieces of a tile's row of 128 lie turned by a number of the row's: eight rows one after the other, and eight rows four apart, have a piece in different banks
// (the reads of eight lanes; the writes of eight lanes whose columns are four apart).
__device__ __forceinline__ constexpr int f8_turn(int row) { return (row & 7) ^ (row >> 3 & 3); }

template <int TM>
struct F8Stage {
  static constexpr int X = TM * 128, W = kF8TileN * 128, S = TM * 4, BYTES = X + W + S;
};

template <int TM, F8Mode MODE, bool F32>
__global__ __launch_bounds__(kF8Threads) void f8_tiles_kernel(F8Product a, int n_tiles, int m_tiles) {
  typedef F8Stage<TM> L;
  constexpr int XC = TM / 64, MT = TM / 64;  // copies of token rows a wave; sub-tiles of 32 token rows a wave
  extern __shared__ __align__(16) unsigned char lds[];
  const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)lds;
  const int lane = threadIdx.x & 63, ln = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 2, wn = wave & 3;
  // blocks go round the eight XCDs: with many pieces all tiles of a piece go to one, whose L2 then serves its rows
  int mt, nt;
  if (m_tiles >= 16) {
    const int q = (int)blockIdx.x >> 3;
    mt = q / n_tiles * 8 + ((int)blockIdx.x & 7);
    nt = q % n_tiles;
  } else {
    mt = (int)blockIdx.x / n_tiles;
    nt = (int)blockIdx.x % n_tiles;
  }
  if (mt >= m_tiles) return;
  const F8Piece piece = f8_piece(a.offsets, a.n_mats, (uint32_t)a.rows, TM, (uint32_t)mt);
  const int rows = __builtin_amdgcn_readfirstlane((int)piece.rows), mat = __builtin_amdgcn_readfirstlane(piece.mat);
  const uint32_t row0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)piece.row);
  if (rows == 0) return;
  const int N = a.N, K = a.K, runs = f8_runs(K), n_blocks = f8_runs(N), steps = a.pair_sum ? 2 * runs : runs;
  const int n0 = nt * (MODE == kPair ? 128 : kF8TileN);
  if (mat == a.n_mats) {  // rows of no matrix
    if constexpr (MODE != kPair) {
      const float none[4] = {0.f, 0.f, 0.f, 0.f};
      for (int i = threadIdx.x; i < rows * (kF8TileN / 4); i += kF8Threads) {
        const int n = n0 + i % (kF8TileN / 4) * 4;
        if (n < N) store4(a.y, (int64_t)(row0 + i / (kF8TileN / 4)) * N + n, N - n, a.dt, none);
      }
    }
    return;
  }
  // ---- what a lane copies of a stage
  const int64_t wide = (int64_t)steps * kF8Run;
  auto source = [&](int r) __attribute__((always_inline)) {  // x row of the piece's row r, as the descriptors below count; rows past the end repeat the last one (never stored)
    const uint32_t tr = (uint32_t)(r < rows ? r : rows - 1);
    if (!a.order) return tr;
    const uint32_t at = a.order[row0 + tr] / (uint32_t)a.k_div;
    return at < (uint32_t)a.x.rows ? at : 0u;
  };
  const int64_t x_first = a.order ? 0 : row0, x_rows = a.order ? a.x.rows : rows;
  const i32x4_t xr = uniform(words_of(a.x.codes + x_first * wide, at_most_4g(x_rows * wide)));
  uint32_t x_off[XC];
#pragma unroll
  for (int c = 0; c < XC; ++c) {
    const int r = (wave * XC + c) * 8 + lane / 8;
    x_off[c] = source(r) * (uint32_t)wide + (uint32_t)((lane % 8) ^ f8_turn(r)) * 16;
  }
  const uint32_t s_off = wave < TM / 64 ? source(wave * 64 + lane) * 4 : 0;
  const int64_t matrix = (int64_t)mat * N * K;
  uint32_t w_off[4], w_k[4];
  i32x4_t wr{};
  uint32_t w_reg[16];
  if constexpr (MODE != kColsOfWeights) {
    const int which = MODE == kPair ? wave >> 2 : 0;  // waves 4 to 7 copy the up rows
    wr = uniform(words_of(a.m[which].w + matrix + (int64_t)n0 * K, at_most_4g((int64_t)(N - n0) * K)));
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int r = (wave * 4 + c) * 8 + lane / 8;
      w_k[c] = (uint32_t)((lane % 8) ^ f8_turn(r)) * 16;
      w_off[c] = (uint32_t)(MODE == kPair ? r & 127 : r) * (uint32_t)K + w_k[c];
    }
  }
  const bool w_inside = n0 + 4 * lane < N;
  auto fetch = [&](int j, int place) __attribute__((always_inline)) {
    const uint32_t at = lds_at + place * L::BYTES;
#pragma unroll
    for (int c = 0; c < XC; ++c) copy_to_lds(xr, x_off[c], (uint32_t)(j * kF8Run), at + (wave * XC + c) * 1024);
    if (wave < TM / 64) copy4_to_lds(uniform(words_of(a.x.scales + (int64_t)j * a.x.rows + x_first, at_most_4g(x_rows * 4))), s_off, at + L::X + L::W + wave * 256);
    if constexpr (MODE != kColsOfWeights) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        copy_to_lds(wr, (uint32_t)(j * kF8Run) + w_k[c] < (uint32_t)K ? w_off[c] : kF8Outside, (uint32_t)(j * kF8Run), at + L::X + (wave * 4 + c) * 1024);
    } else {
      const bool second = j >= runs;
      const int k0 = (second ? j - runs : j) * kF8Run + wave * 16;
      // (what lies past the matrix's last row is past the descriptor's end)
      const int64_t left = ((int64_t)K - k0) * N - n0;
      const __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(a.m[second].w + matrix + (int64_t)k0 * N + n0), 0,
                                                                             (int)(left > 0 ? at_most_4g(left) : 0u), 0x00020000);
#pragma unroll
      for (int i = 0; i < 16; ++i) w_reg[i] = __builtin_amdgcn_raw_buffer_load_b32(from, w_inside ? lane * 4 : (int)kF8Outside, i * N, 0);
    }
  };
  auto put_columns = [&](int place) __attribute__((always_inline)) {  // sixteen weight rows of four columns: 16 bytes of each column
    if constexpr (MODE == kColsOfWeights) {
      uint32_t o[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t *const d = w_reg + 4 * i;
        const uint32_t t0 = __builtin_amdgcn_perm(d[1], d[0], 0x05010400u), t1 = __builtin_amdgcn_perm(d[1], d[0], 0x07030602u);
        const uint32_t t2 = __builtin_amdgcn_perm(d[3], d[2], 0x05010400u), t3 = __builtin_amdgcn_perm(d[3], d[2], 0x07030602u);
        o[0][i] = __builtin_amdgcn_perm(t2, t0, 0x05040100u), o[1][i] = __builtin_amdgcn_perm(t2, t0, 0x07060302u);
        o[2][i] = __builtin_amdgcn_perm(t3, t1, 0x05040100u), o[3][i] = __builtin_amdgcn_perm(t3, t1, 0x07060302u);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int r = 4 * lane + c;
        *reinterpret_cast<u32x4_f8 *>(lds + place * L::BYTES + L::X + r * 128 + (wave ^ f8_turn(r)) * 16) = u32x4_f8{o[c][0], o[c][1], o[c][2], o[c][3]};
      }
    }
  };
  const float *ws[2];
  if constexpr (MODE == kPair) {
#pragma unroll
    for (int i = 0; i < 2; ++i) ws[i] = a.m[i].s + ((int64_t)mat * n_blocks + nt) * runs;
  } else {
    const int block = (n0 + wn * 64) / kF8Run < n_blocks ? (n0 + wn * 64) / kF8Run : n_blocks - 1;
#pragma unroll
    for (int i = 0; i < 2; ++i) ws[i] = MODE == kRowsOfWeights ? a.m[0].s + ((int64_t)mat * n_blocks + block) * runs : a.m[i].s + (int64_t)mat * runs * n_blocks + block;
  }
  auto weight_scale = [&](int j, int i) __attribute__((always_inline)) {
    if constexpr (MODE == kColsOfWeights) return j < runs ? ws[0][(int64_t)j * n_blocks] : ws[1][(int64_t)(j - runs) * n_blocks];
    return ws[i][j];
  };

  f32x16_t acc[MT][2];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[t][i][v] = 0.f;
  const int x_at = (wm * 32 * MT + ln) * 128, w_at0 = (MODE == kPair ? wn * 32 + ln : wn * 64 + ln) * 128, w_at1 = w_at0 + (MODE == kPair ? 128 : 32) * 128;
  const int turn = f8_turn(ln);  // (rows 32 apart are turned alike)
  auto operand = [&](const unsigned char *row, int q) __attribute__((always_inline)) {  // values 64 q + 32 half to 64 q + 32 half + 31
    const u32x4_f8 lo = *reinterpret_cast<const u32x4_f8 *>(row + ((4 * q + 2 * half) ^ turn) * 16), hi = *reinterpret_cast<const u32x4_f8 *>(row + ((4 * q + 2 * half + 1) ^ turn) * 16);
    return i32x8_t{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
  };
  auto multiply = [&](const i32x8_t *w, const i32x8_t *x) __attribute__((always_inline)) {
    f32x16_t sum{};
    if constexpr (F32) {
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int p = 0; p < 4; ++p)
          sum = __builtin_amdgcn_mfma_f32_32x32x16_bf16(codes_to_bf16((uint32_t)w[q][2 * p], (uint32_t)w[q][2 * p + 1]), codes_to_bf16((uint32_t)x[q][2 * p], (uint32_t)x[q][2 * p + 1]),
                                                        sum, 0, 0, 0);
    } else {
      sum = mfma_f8_32(w[0], x[0], sum);
      sum = mfma_f8_32(w[1], x[1], sum);
    }
    return sum;
  };

  fetch(0, 0);
  wait_copies<0>();
  put_columns(0);
  wait_reads();
  block_barrier();
  for (int j = 0; j < steps; ++j) {
    const int place = j & 1;
    if (j + 1 < steps) fetch(j + 1, place ^ 1);
    const unsigned char *const at = lds + place * L::BYTES;
    const float *const sx = reinterpret_cast<const float *>(at + L::X + L::W) + wm * 32 * MT + ln;
    const float s0 = weight_scale(j, 0), s1 = MODE == kPair ? weight_scale(j, 1) : s0;
    i32x8_t w[2][2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      w[0][q] = operand(at + L::X + w_at0, q);
      w[1][q] = operand(at + L::X + w_at1, q);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      if (wm * 32 * MT + t * 32 < rows) {
        i32x8_t x[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) x[q] = operand(at + x_at + t * 32 * 128, q);
        const float s = sx[t * 32];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const f32x16_t sum = multiply(w[i], x);
          const float f = s * (i ? s1 : s0);
#pragma unroll
          for (int v = 0; v < 16; ++v) acc[t][i][v] = __builtin_fmaf(sum[v], f, acc[t][i][v]);
        }
      }
    }
    wait_copies<0>();
    if (j + 1 < steps) put_columns(place ^ 1);
    wait_reads();
    block_barrier();
  }

  // lane: token row ln of each sub-tile; of weight rows 8 g + 4 half + 0..3 the sums 4 g + 0..3
  if constexpr (MODE == kPair) {
    float *const most = reinterpret_cast<float *>(lds);  // [4][TM]
    uint32_t m[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      m[t] = 0;
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        acc[t][0][v] = silu(acc[t][0][v]) * acc[t][1][v];
        m[t] = umax(m[t], abs_bits(acc[t][0][v]));
      }
      m[t] = umax(m[t], (uint32_t)__shfl_xor((int)m[t], 32, kWave));
      if (half == 0) most[wn * TM + wm * 32 * MT + t * 32 + ln] = __uint_as_float(m[t]);
    }
    __syncthreads();
    const int64_t h_wide = (int64_t)n_blocks * kF8Run;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int r = wm * 32 * MT + t * 32 + ln;
      uint32_t all = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) all = umax(all, __float_as_uint(most[i * TM + r]));
      const F8Scale s(all);
      if (r < rows) {
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<uint32_t *>(a.h + (int64_t)(row0 + r) * h_wide + n0 + wn * 32 + 8 * g + 4 * half) =
              s.codes(acc[t][0][4 * g], acc[t][0][4 * g + 1], acc[t][0][4 * g + 2], acc[t][0][4 * g + 3]);
        if (wn == 0 && half == 0) a.hs[(int64_t)nt * a.rows + row0 + r] = s.scale;
      }
    }
  } else {
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int r = wm * 32 * MT + t * 32 + ln;
      if (r < rows) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int n = n0 + wn * 64 + i * 32 + 8 * g + 4 * half;
            if (n < N) {
              float o[4];
#pragma unroll
              for (int v = 0; v < 4; ++v) o[v] = acc[t][i][4 * g + v] + (a.bias && n + v < N ? value_of(a.bias, n + v, a.dt) : 0.f);
              store4(a.y, (int64_t)(row0 + r) * N + n, N - n, a.dt, o);
            }
          }
      }
    }
  }
}

template <int TM, F8Mode MODE, bool F32>
static hipError_t launch_tiles(const F8Product &p, hipStream_t st) {
  constexpr size_t lds = 2 * F8Stage<TM>::BYTES;
  constexpr int kMaxDevices = 64;
  static std::atomic<bool> raised[kMaxDevices];  // more LDS than a kernel gets without asking
  int dev = 0;
  if (hipError_t e = hipGetDevice(&dev); e != hipSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices || !raised[dev].load(std::memory_order_acquire)) {
    if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&f8_tiles_kernel<TM, MODE, F32>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds); e != hipSuccess) return e;
    if (dev >= 0 && dev < kMaxDevices) raised[dev].store(true, std::memory_order_release);
  }
  const int64_t n_tiles = (p.N + (MODE == kPair ? 127 : kF8TileN - 1)) / (MODE == kPair ? 128 : kF8TileN), m_tiles = f8_most_pieces(p, TM);
  const int64_t grid = n_tiles * (m_tiles >= 16 ? (m_tiles + 7) / 8 * 8 : m_tiles);
  if (grid > (int64_t)1 << 22) return hipErrorInvalidValue;  // (a launch has less than 2^32 threads)
  f8_tiles_kernel<TM, MODE, F32><<<(unsigned)grid, kF8Threads, lds, st>>>(p, (int)n_tiles, (int)m_tiles);
  return hipGetLastError();
}

template <F8Mode MODE>
static hipError_t launch_mode(const F8Product &p, hipStream_t st) {
  const int64_t avg = p.rows / (p.offsets ? p.n_mats : 1);
  if (p.dt == 2) return avg > 128 ? launch_tiles<128, MODE, true>(p, st) : launch_tiles<64, MODE, true>(p, st);
  return avg > 192 ? launch_tiles<256, MODE, false>(p, st) : avg > 64 ? launch_tiles<128, MODE, false>(p, st) : launch_tiles<64, MODE, false>(p, st);
}

hipError_t launch_f8_tiles(const F8Product &p, hipStream_t st) {
  if (p.rows == 0) return hipSuccess;
  if (p.h) return launch_mode<kPair>(p, st);
  if (!p.transpose) return launch_mode<kColsOfWeights>(p, st);
  if (p.y1) {  // two products: one after the other
    F8Product q = p;
    q.y1 = nullptr;
    if (hipError_t e = launch_mode<kRowsOfWeights>(q, st); e != hipSuccess) return e;
    q.m[0] = p.m[1];
    q.y = p.y1;
    return launch_mode<kRowsOfWeights>(q, st);
  }
  return launch_mode<kRowsOfWeights>(p, st);
}

}  // namespace mi_moe
