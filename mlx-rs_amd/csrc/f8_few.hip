// Product of a few rows a matrix with e4m3 weights: one token's or a decode batch's linear layers and experts.  Memory bound: a matrix's codes are read once for up to
// 16 TG rows.
//
// A block of four waves computes 16 weight rows (the rows of 16x16x32 matrix instructions) for up to 16 TG token rows (their columns).  The waves share the summed
// axis, every fourth run of 128 values each; a lane's 32 bytes of a run are two pieces of 16, at 16 (l / 16) and 64 bytes on, for codes and rows alike (which values a lane
// multiplies is free as long as both sides agree), so that one load takes 64 consecutive bytes of a weight row.  Codes go from memory into registers and there to bf16, where their
// products are exact and sums float32 (f8.hpp; on the f8 instructions, which take the codes as they are, a launch waits for the same bytes: 300 rows at 128 matrices of 768 x 2048
// 37.4 us, 38.4 so; 16 rows of 4096 x 4096 11.7, 11.6; one 6.9, 7.3); token rows come the same way out of L2.  A run's sums are scaled in float32; the waves' sums meet in LDS in a fixed order.
#include "f8.hpp"
#include "octets.hpp"

namespace mi_moe {

constexpr int kFewWaves = 4;

// IN: rows as codes; as they are, or a gate and an up product of them, both rounded to e4m3 by the block itself, into LDS, while its first weights are on their way.  A launch
// less (2 us) for a few microseconds of work.
enum F8In { kCodes, kRaw, kGateUp };
// A run of row `from`, by sixteen lanes: its codes to a row in LDS, its scale to the row's.
template <F8In IN>
__device__ __forceinline__ void round_run(const F8Product &a, int64_t from_row, int run, uint8_t *codes, float *scales) {
  const int k = run * kF8Run + (threadIdx.x % 16) * 8, n = a.K - k;
  const int64_t from = from_row * a.K + (n > 0 ? k : 0);
  float v[8];
  auto load = [&](auto dt_of) __attribute__((always_inline)) {
    constexpr int DT = decltype(dt_of)::value;
    const Octet<DT> o = load_octet<DT>(a.raw, from, n > 0 ? n : 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = o.at(i);
  };
  if constexpr (IN == kGateUp) {
    load(std::integral_constant<int, 2>());
    const Octet<2> up = load_octet<2>(a.raw_up, from, n > 0 ? n : 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = silu(v[i]) * up.v[i];
  } else if (a.raw_dt == 0) {
    load(std::integral_constant<int, 0>());
  } else if (a.raw_dt == 1) {
    load(std::integral_constant<int, 1>());
  } else {
    load(std::integral_constant<int, 2>());
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = umax(m, abs_bits(v[i]));
  const F8Scale q(max_of_16_lanes(m));
  *reinterpret_cast<uint2 *>(codes + k) = make_uint2(q.codes(v[0], v[1], v[2], v[3]), q.codes(v[4], v[5], v[6], v[7]));
  if (threadIdx.x % 16 == 0) scales[run] = q.scale;
}
// the sums of a run, of 16 weight rows and 16 token rows
struct FewRow {
  u32x4_f8 v[2];
};
__device__ __forceinline__ f32x4_t few_run(const u32x4_f8 (&w)[2], const FewRow &x) {
  f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int p = 0; p < 2; ++p)
      sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes_to_bf16(w[h][2 * p], w[h][2 * p + 1]), codes_to_bf16(x.v[h][2 * p], x.v[h][2 * p + 1]), sum, 0, 0, 0);
  return sum;
}
template <int TG, F8In IN>
__global__ __launch_bounds__(kFewWaves *kWave, 5) void f8_few_kernel(F8Product a) {
  constexpr int AHEAD = TG == 1 ? 4 : 2;  // runs whose loads are in flight at once
  extern __shared__ __align__(16) uint8_t own_rows[];  // [rows][whole runs + 16], then scales [rows][runs]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ln = lane & 15, part = lane >> 4;
  const int tiles = (a.N + 15) / 16, which = (int)blockIdx.x / tiles, n0 = ((int)blockIdx.x - which * tiles) * 16;
  const F8Piece piece = f8_piece(a, 16 * TG, blockIdx.y);
  if (piece.rows == 0) return;
  void *const y = which ? a.y1 : a.y;
  if (piece.mat == a.n_mats) {  // rows of no matrix
    const float none[4] = {0.f, 0.f, 0.f, 0.f};
    for (int r = threadIdx.x / 4; r < (int)piece.rows; r += kFewWaves * kWave / 4) {
      const int n = n0 + (threadIdx.x % 4) * 4;
      store4(y, (int64_t)(piece.row + r) * a.N + n, a.N - n, a.dt, none);
    }
    return;
  }
  const int runs = f8_runs(a.K), wide = f8_runs(a.K) * kF8Run;
  const F8Mat m = which ? a.m[1] : a.m[0];
  const uint8_t *const w = m.w + (int64_t)piece.mat * a.N * a.K + (int64_t)(n0 + ln < a.N ? n0 + ln : a.N - 1) * a.K;
  const float *const ws = m.s + ((int64_t)piece.mat * f8_runs(a.N) + n0 / kF8Run) * runs;
  auto source = [&](uint32_t r) __attribute__((always_inline)) {
    const int64_t at = a.order ? a.order[r] / (uint32_t)a.k_div : a.ids ? r / (uint32_t)a.k_div : r;
    return at < a.x.rows ? at : 0;  // (never followed out of the rows)
  };
  u32x4_f8 wv[AHEAD][2];
  float s[AHEAD];
  auto fetch = [&](int j0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int j = j0 + i * kFewWaves < runs ? j0 + i * kFewWaves : runs - 1;  // (past the end the last run again, with a scale of zero)
      s[i] = j0 + i * kFewWaves < runs ? ws[j] : 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = j * kF8Run + h * 64 + part * 16;
        wv[i][h] = *reinterpret_cast<const u32x4_f8 *>(w + (k < a.K ? k : 0));
        if (k >= a.K) wv[i][h] = u32x4_f8{0, 0, 0, 0};
      }
    }
  };
  fetch(wave);
  const uint8_t *x[TG];
  const float *xs[TG];
  if constexpr (IN == kCodes) {
#pragma unroll
    for (int t = 0; t < TG; ++t) {
      const int64_t at = source(t * 16 + ln < (int)piece.rows ? piece.row + t * 16 + ln : piece.row);
      x[t] = a.x.codes + at * wide;
      xs[t] = a.x.scales + at;
    }
  } else {
    float *const own_scales = reinterpret_cast<float *>(own_rows + piece.rows * (wide + 16));
    for (int at = threadIdx.x / 16; at < (int)piece.rows * runs; at += kFewWaves * kWave / 16) {
      const int r = at / runs, run = at - r * runs;
      round_run<IN>(a, IN == kGateUp ? (int64_t)(piece.row + r) : source(piece.row + r), run, own_rows + r * (wide + 16), own_scales + r * runs);
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TG; ++t) {
      const int r = t * 16 + ln < (int)piece.rows ? t * 16 + ln : 0;
      x[t] = own_rows + r * (wide + 16);
      xs[t] = own_scales + r * runs;
    }
  }
  f32x4_t acc[TG] = {};
  for (int j0 = wave; j0 < runs; j0 += kFewWaves * AHEAD) {
    if (j0 != wave) fetch(j0);
    FewRow xv[AHEAD][TG];
    float sx[AHEAD][TG];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int j = j0 + i * kFewWaves < runs ? j0 + i * kFewWaves : runs - 1;
#pragma unroll
      for (int t = 0; t < TG; ++t) {
#pragma unroll
        for (int h = 0; h < 2; ++h) xv[i][t].v[h] = *reinterpret_cast<const u32x4_f8 *>(x[t] + j * kF8Run + h * 64 + part * 16);
        sx[i][t] = IN == kCodes ? xs[t][(int64_t)j * a.x.rows] : xs[t][j];
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // (all loads ahead of the products: in between, and with one wave a SIMD less, 16 rows of 4096 x 4096 took 12.4 us, not 11.6)
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
#pragma unroll
      for (int t = 0; t < TG; ++t) {
        const f32x4_t sum = few_run(wv[i], xv[i][t]);
        const float f = s[i] * sx[i][t];
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[t][v] = __builtin_fmaf(sum[v], f, acc[t][v]);
      }
  }
  __shared__ f32x4_t sums[kFewWaves][TG][kWave];
#pragma unroll
  for (int t = 0; t < TG; ++t) sums[wave][t][lane] = acc[t];
  __syncthreads();
  for (int t = wave; t < TG; t += kFewWaves) {
    const f32x4_t v = (sums[0][t][lane] + sums[1][t][lane]) + (sums[2][t][lane] + sums[3][t][lane]);
    const int r = t * 16 + ln, n = n0 + part * 4;  // lane: token row ln of the group, four weight rows
    if (r >= (int)piece.rows || n >= a.N) continue;
    float o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = v[i] + (a.bias && n + i < a.N ? value_of(a.bias, n + i, a.dt) : 0.f);
    store4(y, (int64_t)(piece.row + r) * a.N + n, a.N - n, a.dt, o);
  }
}

// A token or two: down, and the sum over a token's k_div slots.  A block has 16 columns of a token's result, its sixteen waves share the slots and, of a slot's summed axis, every `each`th run; rows are
// rounded as above.  The slots' rows are summed over the waves, then weighted and summed in the slots' order, all in float32.  A launch less than with rows in memory.
constexpr int kTokenWaves = 16, kTokenSlots = 32;
__global__ __launch_bounds__(kTokenWaves *kWave) void f8_token_kernel(F8Product a, const void *__restrict__ weights, int w_dtype, void *__restrict__ out, int out_dt) {
  constexpr int AHEAD = 4;
  const uint32_t first = blockIdx.y * (uint32_t)a.k_div;  // the token's first pair
  const uint32_t *const ids = a.ids + first;
  extern __shared__ __align__(16) uint8_t own_rows[];  // [slots][whole runs + 16], then scales [slots][runs]
  __shared__ float sums[kTokenSlots][16];  // [slot][wave of the slot's]: no more than sixteen of both, or one wave a slot
  __shared__ float slot_weight[kTokenSlots];
  __shared__ bool slot_named[kTokenSlots];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ln = lane & 15, part = lane >> 4, n0 = (int)blockIdx.x * 16;
  const int slots = a.k_div, runs = f8_runs(a.K), wide = runs * kF8Run;
  const int at_once = slots < kTokenWaves ? slots : kTokenWaves, each = kTokenWaves / at_once;  // slots at once, waves of a slot
  const int mine = wave % each, turns = (runs + each - 1) / each, all = wave / each < at_once ? (slots - wave / each + at_once - 1) / at_once * turns : 0;
  float *const own_scales = reinterpret_cast<float *>(own_rows + slots * (wide + 16));
  struct Item {
    int slot, run;
    bool there;
  };
  auto item = [&](int i) __attribute__((always_inline)) {  // the wave's i-th: a run of a slot, some of them past the end
    const int slot = wave / each + i / turns * at_once, run = i % turns * each + mine;
    return Item{i < all ? slot : 0, run < runs ? run : 0, i < all && run < runs};
  };
  u32x4_f8 wv[AHEAD][2];
  float s[AHEAD];
  auto fetch = [&](int i0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const Item it = item(i0 + i);
      const uint32_t e = ids[it.slot];
      const bool named = it.there && e < (uint32_t)a.n_mats;
      const int64_t mat = named ? e : 0;
      const uint8_t *const w = a.m[0].w + (mat * a.N + (n0 + ln < a.N ? n0 + ln : a.N - 1)) * a.K;
      s[i] = named ? a.m[0].s[(mat * f8_runs(a.N) + n0 / kF8Run) * runs + it.run] : 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = it.run * kF8Run + h * 64 + part * 16;
        wv[i][h] = *reinterpret_cast<const u32x4_f8 *>(w + (k < a.K ? k : 0));
        if (k >= a.K || !named) wv[i][h] = u32x4_f8{0, 0, 0, 0};
      }
    }
  };
  fetch(0);
  if ((int)threadIdx.x < slots) {  // (loaded where they are used, one after the other, they took 0.7 us)
    slot_named[threadIdx.x] = ids[threadIdx.x] < (uint32_t)a.n_mats;
    slot_weight[threadIdx.x] = value_of(weights, first + threadIdx.x, w_dtype);
  }
  for (int at = threadIdx.x / 16; at < slots * runs; at += kTokenWaves * kWave / 16) {
    const int r = at / runs, run = at - r * runs;
    round_run<kGateUp>(a, first + r, run, own_rows + r * (wide + 16), own_scales + r * runs);
  }
  __syncthreads();
  f32x4_t acc = {};
  for (int i0 = 0; i0 < all; i0 += AHEAD) {
    if (i0) fetch(i0);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const Item it = item(i0 + i);
      const uint8_t *const x = own_rows + it.slot * (wide + 16) + it.run * kF8Run + part * 16;
      const f32x4_t sum = few_run(wv[i], {*reinterpret_cast<const u32x4_f8 *>(x), *reinterpret_cast<const u32x4_f8 *>(x + 64)});
      const float f = it.there ? s[i] * own_scales[it.slot * runs + it.run] : 0.f;
#pragma unroll
      for (int v = 0; v < 4; ++v) acc[v] = __builtin_fmaf(sum[v], f, acc[v]);
      if ((i0 + i) % turns == turns - 1 && i0 + i < all) {  // a slot's last
        if (ln == 0)
#pragma unroll
          for (int v = 0; v < 4; ++v) sums[it.slot * each + mine][part * 4 + v] = acc[v];
        acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
      }
    }
  }
  __syncthreads();
  const int n = n0 + (int)threadIdx.x;
  if (threadIdx.x >= 16 || n >= a.N) return;
  float y = 0.f;
  for (int slot = 0; slot < slots; ++slot) {
    if (!slot_named[slot]) continue;
    float row = 0.f;
    for (int w = 0; w < each; ++w) row += sums[slot * each + w][threadIdx.x];
    y = __builtin_fmaf(slot_weight[slot], row, y);
  }
  put_value(out, (int64_t)blockIdx.y * a.N + n, out_dt, y);
}
size_t f8_token_bytes(const F8Product &p) { return (size_t)p.k_div * (size_t)(f8_row_bytes(p.K) + 16 + 4 * f8_runs(p.K)); }
hipError_t launch_f8_token(const F8Product &p, const void *weights, int w_dtype, void *out, int dt, hipStream_t st) {
  f8_token_kernel<<<dim3((unsigned)((p.N + 15) / 16), (unsigned)(p.rows / p.k_div)), kTokenWaves * kWave, f8_token_bytes(p), st>>>(p, weights, w_dtype, out, dt);
  return hipGetLastError();
}

hipError_t launch_f8_few(const F8Product &p, hipStream_t st) {
  if (p.rows == 0) return hipSuccess;
  const unsigned tiles = (unsigned)((p.N + 15) / 16) * (p.y1 ? 2 : 1);
  const int tile = f8_tile_rows(p);
  const int64_t pieces = p.ids ? p.rows : p.list ? f8_most_pieces(p.rows, p.n_mats, tile) : (p.rows + tile - 1) / tile;
  const size_t own = p.raw ? f8_own_bytes(p) : 0;
  auto launch = [&](auto *kernel) {
    kernel<<<dim3(tiles, (unsigned)pieces), kFewWaves * kWave, own, st>>>(p);
    return hipGetLastError();
  };
  auto kind = [&](auto in_of) {
    constexpr F8In IN = decltype(in_of)::value;
    return tile == 32 ? launch(&f8_few_kernel<2, IN>) : launch(&f8_few_kernel<1, IN>);
  };
  return !p.raw ? kind(std::integral_constant<F8In, kCodes>()) : !p.raw_up ? kind(std::integral_constant<F8In, kRaw>()) : kind(std::integral_constant<F8In, kGateUp>());
}

}  // namespace mi_moe
