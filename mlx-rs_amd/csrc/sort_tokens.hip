// Tokens to rows sorted by expert and back, with the weights applied, and the gradients of both.
//
//   sort      row[place(t, s)] = x[t]                       its gradient  dx[t] = sum over s of drow[place(t, s)]
//   unsort    out[t] = sum over s of w[t][s] row[place(t, s)]             drow[place(t, s)] = w[t][s] dout[t],  dw[t][s] = dout[t] . row[place(t, s)]
//
// place: the stable sort of the (token, slot) pairs by expert (dispatch.hip).  Slots that name no expert have the places behind all others: their rows are zeros and have
// no part in any sum.  Sums are float32, over the slots in their order, over a row's values in a fixed tree.  All four move bytes: a token's row is read (or written) once
// and its k rows written (or read) once.
#include "dispatch_dev.hpp"
#include "f8.hpp"
#include "octets.hpp"

namespace mi_moe {

constexpr int kSortThreads = 256, kSortMostSlots = 32;

// a token's row to its places: 16 bytes a thread and step, with no more alignment than the elements' own
__device__ __forceinline__ void spread_row(const char *from, char *rows, int64_t bytes, const int32_t *at, int k) {
  for (int64_t b = (int64_t)threadIdx.x * 16; b < bytes; b += kSortThreads * 16) {
    const int n = bytes - b < 16 ? (int)(bytes - b) / 2 : 8;
    uint16_t v[8] = {};
    if (n == 8) __builtin_memcpy(v, from + b, 16);
    else
      for (int i = 0; i < n; ++i) __builtin_memcpy(&v[i], from + b + 2 * i, 2);
    for (int s = 0; s < k; ++s) {
      const int32_t to = at[s];
      const bool named = to >= 0;
      char *const p = rows + (int64_t)(named ? to : ~to) * bytes + b;
      uint16_t o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = named ? v[i] : 0;
      if (n == 8) __builtin_memcpy(p, o, 16);
      else
        for (int i = 0; i < n; ++i) __builtin_memcpy(p + 2 * i, &o[i], 2);
    }
  }
}

// Few pairs: block t finds the places of token t's pairs by counting the pairs before each (a smaller expert, or the same and an earlier pair), and writes its rows; the last block
// counts the experts' rows.  One launch, no block waits for another.
__global__ __launch_bounds__(kSortThreads) void sort_few_kernel(SortTokens a, const char *__restrict__ x, int64_t row_bytes, char *__restrict__ rows,
                                                                F8Lists lists) {
  __shared__ uint32_t ids[kSortSmall];
  __shared__ int32_t at[kSortMostSlots];
  __shared__ uint32_t count[513];
  const int P = (int)a.T * a.k, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t E = (uint32_t)a.E;
  for (int i = threadIdx.x; i < P; i += kSortThreads) ids[i] = a.ids[i] < E ? a.ids[i] : E;
  if ((int64_t)blockIdx.x == a.T) {
    for (int e = threadIdx.x; e <= a.E; e += kSortThreads) count[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < P; i += kSortThreads) atomicAdd(&count[ids[i]], 1u);
    __syncthreads();
    if (wave == 0) {
      uint32_t before = 0;
      for (int e0 = 0; e0 <= a.E; e0 += kWave) {
        const uint32_t own = e0 + lane <= a.E ? count[e0 + lane] : 0u;
        uint32_t upto = own;
        for (int d = 1; d < kWave; d <<= 1) {
          const uint32_t v = __shfl_up(upto, d, kWave);
          if (lane >= d) upto += v;
        }
        if (e0 + lane <= a.E) {
          a.offsets[e0 + lane] = before + upto - own;
          count[e0 + lane] = before + upto - own;
        }
        before += __shfl(upto, kWave - 1, kWave);
      }
    }
    __syncthreads();
    if (wave < 2 && lists.list[wave]) f8_list(count, a.E, (uint32_t)P, (uint32_t)lists.tile[wave], lists.list[wave], (uint32_t)lists.places[wave]);
    return;
  }
  __syncthreads();
  const int first = (int)blockIdx.x * a.k;
  for (int s = wave; s < a.k; s += kSortThreads / kWave) {
    const int p = first + s;
    const uint32_t e = ids[p];
    int n = 0;
    for (int q = lane; q < P; q += kWave) n += ids[q] < e || (ids[q] == e && q < p);
    for (int d = 1; d < kWave; d <<= 1) n += __shfl_xor(n, d, kWave);
    if (lane == 0) {
      at[s] = e < E ? n : ~n;
      a.order[n] = (uint32_t)p;
      a.inverse[p] = e < E ? n : ~n;
    }
  }
  if (!rows) return;
  __syncthreads();
  spread_row(x + blockIdx.x * row_bytes, rows, row_bytes, at, a.k);
}

// Behind the dispatch of more pairs, with one expert more for those that name none: `inverse` gets its form (a place that has it already stays what it is), rows are written.
__global__ __launch_bounds__(kSortThreads) void sort_rows_kernel(SortTokens a, const uint32_t *__restrict__ offsets, const char *__restrict__ x, int64_t row_bytes,
                                                                 char *__restrict__ rows) {
  __shared__ int32_t at[kSortMostSlots];
  const int64_t first = (int64_t)blockIdx.x * a.k;
  if ((int)threadIdx.x < a.k) {
    const int32_t n = a.inverse[first + threadIdx.x];
    at[threadIdx.x] = a.ids[first + threadIdx.x] < (uint32_t)a.E ? n : ~n;
    a.inverse[first + threadIdx.x] = at[threadIdx.x];
  }
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e <= a.E; e += kSortThreads) a.offsets[e] = offsets[e];
  __syncthreads();
  spread_row(x + blockIdx.x * row_bytes, rows, row_bytes, at, a.k);
}

__global__ __launch_bounds__(kSortThreads) void sort_places_kernel(SortTokens a, const uint32_t *__restrict__ offsets, int64_t P) {
  const int64_t p = (int64_t)blockIdx.x * kSortThreads + threadIdx.x;
  if (p < P && a.ids[p] >= (uint32_t)a.E) a.inverse[p] = ~a.inverse[p];
  if (p <= a.E) a.offsets[p] = offsets[p];
}

size_t sort_tokens_bytes(int64_t T, int k, int E) {
  return T * k <= kSortSmall ? 0 : ((size_t)(E + 2) * 4 + 255) / 256 * 256 + dispatch_workspace_bytes(E + 1, T * k);
}

hipError_t launch_sort_tokens(const SortTokens &a, const void *x, int dt, int H, void *rows, void *scratch, hipStream_t st, const F8Lists &lists) {
  const int64_t P = a.T * a.k, row_bytes = (int64_t)H * (dt == 2 ? 4 : 2);
  if (P <= kSortSmall) {  // (no tokens: the offsets alone)
    sort_few_kernel<<<(unsigned)a.T + 1, kSortThreads, 0, st>>>(a, static_cast<const char *>(x), row_bytes, static_cast<char *>(rows), lists);
    return hipGetLastError();
  }
  uint32_t *const offsets = static_cast<uint32_t *>(scratch);
  if (hipError_t e = launch_dispatch(a.ids, P, a.E + 1, a.k, nullptr, offsets, a.order, reinterpret_cast<uint32_t *>(a.inverse), nullptr, Records(), nullptr, 0, 0, ShortTiles(),
                                     PrepareArgs(), static_cast<char *>(scratch) + ((size_t)(a.E + 2) * 4 + 255) / 256 * 256, st);
      e != hipSuccess)
    return e;
  if (!rows) {
    sort_places_kernel<<<(unsigned)((P + kSortThreads - 1) / kSortThreads), kSortThreads, 0, st>>>(a, offsets, P);
    return hipGetLastError();
  }
  sort_rows_kernel<<<(unsigned)a.T, kSortThreads, 0, st>>>(a, offsets, static_cast<const char *>(x), row_bytes, static_cast<char *>(rows));
  return hipGetLastError();
}

// How a block's threads lie over tokens and columns of eight: whole tokens a block where rows are short.
struct TokenGrid {
  int lanes, tokens, columns;  // threads of a token (a power of two), tokens of a block, blocks of a token
  TokenGrid(int H, int most) {
    const int octets = (H + 7) / 8;
    lanes = most;
    while (lanes > 16 && lanes / 2 >= octets) lanes /= 2;
    tokens = most / lanes;
    columns = (octets + lanes - 1) / lanes;
  }
};

// Eight columns from h on of several rows (-1: of the first, for nobody).  The whole octets' loads stand together: with a condition around each, they were waited for one by one.
template <int DT, int N>
__device__ __forceinline__ void load_octets(Octet<DT> (&v)[N], const void *rows, const int64_t (&row)[N], int H, int h, int n) {
  if (n >= 8) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = load_octet<DT>(rows, (row[j] < 0 ? 0 : row[j]) * H + h, 8);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = load_octet<DT>(rows, (row[j] < 0 ? 0 : row[j]) * H + (n > 0 ? h : 0), n > 0 ? n : 0);
  }
}

// A thread eight columns of a token; its slots' rows N at a time, all their loads in flight together.  Blocks of 256 threads: of 64, the launch of blocks is what it waits
// for (8192 tokens of 2048 bf16 and eight slots: 80 us).
// N: eight, or of fewer slots two or four, where the loads for slots past the last one took as long as those for the slots (4096 tokens of 2048 bf16, one and four slots: 20 and 22 us, 10 and 15 so).
// IN, DT: types of the rows and of the result.  SCALED: the rows' values are times scales[row][column / 64].
template <int IN, int DT, bool SCALED, int N>
__global__ __launch_bounds__(kSortThreads) void unsort_kernel(const void *__restrict__ rows, const float *__restrict__ scales, const void *__restrict__ weights, int w_dtype, const int32_t *__restrict__ inverse,
                                                              int64_t T, int k, int H, int lanes_log2, void *__restrict__ out, int out_stride) {
  const int lanes = 1 << lanes_log2;
  const int64_t t = (int64_t)blockIdx.x * (kSortThreads >> lanes_log2) + (threadIdx.x >> lanes_log2);
  const int h = (int)(blockIdx.y * lanes + (threadIdx.x & (lanes - 1))) * 8, n = H - h;
  if (n <= 0 || t >= T) return;
  float acc[8] = {};
  for (int s0 = 0; s0 < k; s0 += N) {
    Octet<IN> v[N];
    float w[N];
    int64_t row[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int64_t s = t * k + (s0 + j < k ? s0 + j : k - 1);
      const int32_t at = inverse[s];
      row[j] = s0 + j < k && at >= 0 && at < T * k ? at : -1;
      w[j] = weights ? value_of(weights, s, w_dtype) : 1.f;
    }
    load_octets(v, rows, row, H, h, n);
    float scale[N];  // (of the values, which are what they were with it; with the weight it may leave float32's range where their products do not)
    if constexpr (SCALED)
#pragma unroll
      for (int j = 0; j < N; ++j) scale[j] = scales[(row[j] < 0 ? 0 : row[j]) * ((H + 63) / 64) + h / 64];
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        acc[i] = row[j] >= 0 ? __builtin_fmaf(w[j], SCALED ? v[j].at(i) * scale[j] : v[j].at(i), acc[i]) : acc[i];  // (not multiplied by zero: row or weight may be infinite)
  }
  Octet<DT> o;
#pragma unroll
  for (int i = 0; i < 8; i += 2) o.put2(i, acc[i], acc[i + 1]);
  store_octet<DT>(out, t * out_stride + h, n, o);
}

template <int IN, int DT, bool SCALED = false>
static hipError_t launch_unsort(const void *rows, const float *scales, const void *weights, int w_dtype, const int32_t *inverse, int64_t T, int k, int H, void *out, int out_stride,
                                hipStream_t st) {
  if (T == 0) return hipSuccess;
  const TokenGrid g(H, kSortThreads);
  auto *const kernel = k > 4 ? &unsort_kernel<IN, DT, SCALED, 8> : k > 2 ? &unsort_kernel<IN, DT, SCALED, 4> : &unsort_kernel<IN, DT, SCALED, 2>;
  kernel<<<dim3((unsigned)((T + g.tokens - 1) / g.tokens), (unsigned)g.columns), kSortThreads, 0, st>>>(rows, scales, weights, w_dtype, inverse, T, k, H,
                                                                                                         __builtin_ctz((unsigned)g.lanes), out, out_stride);
  return hipGetLastError();
}
hipError_t launch_unsort_tokens(const void *rows, const void *weights, int w_dtype, const int32_t *inverse, int64_t T, int k, int H, int dt, void *out, hipStream_t st) {
  auto *const launch = dt == 0 ? &launch_unsort<0, 0> : dt == 1 ? &launch_unsort<1, 1> : &launch_unsort<2, 2>;
  return launch(rows, nullptr, weights, w_dtype, inverse, T, k, H, out, H, st);
}
hipError_t launch_unsort_made(const void *rows, const float *y_scales, const void *weights, int w_dtype, const int32_t *inverse, int64_t T, int k, int H, int dt, void *out,
                              int out_stride, hipStream_t st) {
  auto *const launch = y_scales ? (dt == 0 ? &launch_unsort<1, 0, true> : &launch_unsort<1, 1, true>) : dt == 0 ? &launch_unsort<2, 0> : &launch_unsort<2, 1>;
  return launch(rows, y_scales, weights, w_dtype, inverse, T, k, H, out, out_stride, st);
}

__device__ __forceinline__ float wave_sum_f32(float v) {  // in a fixed order
  auto moved = [](float u, auto ctrl) __attribute__((always_inline)) { return __uint_as_float(dpp_u32<decltype(ctrl)::value>(__float_as_uint(u))); };
  v += moved(v, std::integral_constant<int, kDppXor1>());
  v += moved(v, std::integral_constant<int, kDppXor2>());
  v += moved(v, std::integral_constant<int, kDppHalfMirror>());
  v += moved(v, std::integral_constant<int, kDppMirror>());
  auto lane = [&](int l) __attribute__((always_inline)) { return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), l)); };
  return (lane(0) + lane(16)) + (lane(32) + lane(48));
}

// A block a token; N slots' rows in flight at once: four, or two or three where that leaves out none (4096 tokens of 2048 bf16, one slot: 16 us, 13 so; 1000 of 2045 f16, six: 16.5, 15.5).  A wave's share of a slot's dot product is kept in LDS from one pass over the columns to the next.
template <int DT, int N>
__global__ __launch_bounds__(kSortThreads) void unsort_grad_kernel(const void *__restrict__ dout, const void *__restrict__ rows, const void *__restrict__ weights, int w_dtype,
                                                                   const int32_t *__restrict__ inverse, int64_t T, int k, int H, void *__restrict__ drows,
                                                                   void *__restrict__ dweights) {
  __shared__ float sums[kSortMostSlots][kSortThreads / kWave];
  const int64_t t = blockIdx.x;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  for (int h0 = 0; h0 < H; h0 += kSortThreads * 8) {
    const int h = h0 + (int)threadIdx.x * 8, n = H - h;
    const Octet<DT> g = load_octet<DT>(dout, t * H + (n > 0 ? h : 0), n > 0 ? n : 0);
    for (int s0 = 0; s0 < k; s0 += N) {
      Octet<DT> v[N];
      int64_t row[N], read[N];
      float w[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int s = s0 + j < k ? s0 + j : k - 1;
        const int32_t at = inverse[t * k + s];
        row[j] = at >= 0 ? at : ~at;
        if (s0 + j >= k || row[j] >= T * k) row[j] = -1;  // (no place at all: nothing is written)
        read[j] = at >= 0 ? row[j] : -1;
        w[j] = value_of(weights, t * k + s, w_dtype);
      }
      load_octets(v, rows, read, H, h, n);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        Octet<DT> o{};
        float dot = 0.f;
        if (read[j] >= 0) {
#pragma unroll
          for (int i = 0; i < 8; i += 2) o.put2(i, w[j] * g.at(i), w[j] * g.at(i + 1));
#pragma unroll
          for (int i = 0; i < 8; ++i) dot = __builtin_fmaf(g.at(i), v[j].at(i), dot);
        }
        if (n > 0 && row[j] >= 0) store_octet<DT>(drows, row[j] * H + h, n, o);
        dot = wave_sum_f32(dot);
        if (lane == 0 && s0 + j < k) sums[s0 + j][wave] = h0 ? sums[s0 + j][wave] + dot : dot;
      }
    }
  }
  __syncthreads();
  if ((int)threadIdx.x < k) {
    const float *const p = sums[threadIdx.x];
    put_value(dweights, t * k + threadIdx.x, w_dtype, (p[0] + p[1]) + (p[2] + p[3]));
  }
}

hipError_t launch_unsort_tokens_grad(const void *dout, const void *rows, const void *weights, int w_dtype, const int32_t *inverse, int64_t T, int k, int H, int dt,
                                     void *drows, void *dweights, hipStream_t st) {
  if (T == 0) return hipSuccess;
  auto of = [&](auto dt_of) {
    constexpr int DT = decltype(dt_of)::value;
    return k <= 2 ? &unsort_grad_kernel<DT, 2> : k % 3 == 0 && k < 12 ? &unsort_grad_kernel<DT, 3> : &unsort_grad_kernel<DT, 4>;
  };
  auto *const kernel = dt == 0 ? of(std::integral_constant<int, 0>()) : dt == 1 ? of(std::integral_constant<int, 1>()) : of(std::integral_constant<int, 2>());
  kernel<<<(unsigned)T, kSortThreads, 0, st>>>(dout, rows, weights, w_dtype, inverse, T, k, H, drows, dweights);
  return hipGetLastError();
}

}  // namespace mi_moe
