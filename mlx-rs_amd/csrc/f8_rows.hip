// Rows and matrices to e4m3 with their scales and back, silu(gate) * up on the way, and its gradient.
//
//   scale = round(max |v| / 448), code = the e4m3 value nearest to round(v / scale) (ties to even); both roundings to float32.
//
// One pass: a lane holds eight values of a run, sixteen lanes the run, whose largest magnitude they find by four exchanges inside a row of lanes.
#include "f8.hpp"
#include "octets.hpp"

namespace mi_moe {

constexpr int kRowThreads = 256, kRowRuns = kRowThreads / 16;  // runs of a block

// `n` codes (8, or fewer at a row's end)
__device__ __forceinline__ void put_f8(uint8_t *to, int n, uint32_t lo, uint32_t hi) {
  const uint32_t q[2] = {lo, hi};
  if (n >= 8) __builtin_memcpy(to, q, 8);
  else
    for (int i = 0; i < n; ++i) to[i] = (uint8_t)(q[i / 4] >> (8 * (i % 4)));
}

// the run of which this lane holds eight values, v[i] = 0 beyond the row's end; n: how many values the row has from this lane's first one on
__device__ __forceinline__ void write_run(const float v[8], const F8Out &to, int64_t row, int run, int n) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = umax(m, abs_bits(v[i]));
  const F8Scale s(max_of_16_lanes(m));
  const int l = threadIdx.x % 16;
  put_f8(to.codes + row * to.code_stride + run * kF8Run + l * 8, to.pad ? 8 : n, s.codes(v[0], v[1], v[2], v[3]), s.codes(v[4], v[5], v[6], v[7]));
  if (l == 0) to.scales[row * to.row_stride + run * to.run_stride] = s.scale;
}

// lists: blocks of their own, ahead of the rows', list the pieces of the product that follows, which else were a launch or a search at the start of every block of it.
template <int DT>
__global__ __launch_bounds__(kRowThreads) void quantize_rows_kernel(const void *__restrict__ x, int64_t rows, int cols, F8Out to, F8Lists lists, int n_lists) {
  if ((int)blockIdx.x < n_lists) {
    if (threadIdx.x < kWave) f8_list(lists.offsets, lists.n_mats, (uint32_t)lists.rows, (uint32_t)lists.tile[blockIdx.x], lists.list[blockIdx.x], (uint32_t)lists.places[blockIdx.x]);
    return;
  }
  const int runs = f8_runs(cols);
  const uint32_t first = (blockIdx.x - n_lists) * (2 * kRowRuns) + threadIdx.x / 16, all = (uint32_t)rows * (uint32_t)runs;  // (in 32 bits: in_launches)
  Octet<DT> o[2];
  int64_t row[2];
  int run[2], n[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {  // (two loads in flight: one took 14 us for 4096 x 4096 bf16)
    const uint32_t at = first + i * kRowRuns < all ? first + i * kRowRuns : all - 1, r = at / (uint32_t)runs;
    row[i] = r;
    run[i] = (int)(at - r * (uint32_t)runs);
    const int k = run[i] * kF8Run + (threadIdx.x % 16) * 8;
    n[i] = cols - k;
    o[i] = load_octet<DT>(x, row[i] * cols + (n[i] > 0 ? k : 0), n[i] > 0 ? n[i] : 0);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = o[i].at(j);
    if (first + i * kRowRuns < all) write_run(v, to, row[i], run[i], n[i]);  // (whole rows of lanes)
  }
}

static unsigned quantize_blocks(int64_t rows, int cols) { return (unsigned)((rows * f8_runs(cols) + 2 * kRowRuns - 1) / (2 * kRowRuns)); }
static unsigned run_blocks(int64_t rows, int cols) { return (unsigned)((rows * f8_runs(cols) + kRowRuns - 1) / kRowRuns); }
// f(first row, rows) for parts of the rows that a launch holds: less than 2^32 threads
template <class F>
static hipError_t in_launches(int64_t rows, int cols, F f) {
  const int64_t most = (((int64_t)1 << 27) / f8_runs(cols) + kF8Run - 1) / kF8Run * kF8Run;  // (whole blocks)
  for (int64_t r = 0; r < rows; r += most) {
    f(r, rows - r < most ? rows - r : most);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}
static F8Out rows_from(F8Out to, int64_t row) {
  to.codes += row * to.code_stride;
  to.scales += row * to.row_stride;
  return to;
}
static const char *value_at(const void *x, int dt, int64_t at) { return static_cast<const char *>(x) + at * (dt == 2 ? 4 : 2); }

hipError_t launch_quantize_f8_rows(const void *x, int dt, int64_t rows, int cols, const F8Out &to, hipStream_t st, const F8Lists &lists) {
  if (rows == 0 || cols == 0) return hipSuccess;
  const int n_lists = lists.list[1] ? 2 : lists.list[0] ? 1 : 0;
  auto *const kernel = dt == 0 ? &quantize_rows_kernel<0> : dt == 1 ? &quantize_rows_kernel<1> : &quantize_rows_kernel<2>;
  return in_launches(rows, cols, [&](int64_t r, int64_t n) {
    const int also = r == 0 ? n_lists : 0;
    kernel<<<quantize_blocks(n, cols) + also, kRowThreads, 0, st>>>(value_at(x, dt, r * cols), n, cols, rows_from(to, r), lists, also);
  });
}

// A block of 128 x 128 values, a thread eight columns of eight rows sixteen apart.
template <int DT>
__global__ __launch_bounds__(256) void quantize_blocks_kernel(const void *__restrict__ x, int64_t rows, int cols, uint8_t *__restrict__ codes, float *__restrict__ scales) {
  __shared__ uint32_t most[4];
  const int l = threadIdx.x % 16, k = blockIdx.x * kF8Run + l * 8, n = cols - k;
  const int64_t row0 = (int64_t)blockIdx.y * kF8Run + threadIdx.x / 16;
  Octet<DT> o[8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = row0 + 16 * i;
    o[i] = load_octet<DT>(x, (row < rows ? row : 0) * cols + (n > 0 ? k : 0), row < rows && n > 0 ? n : 0);
#pragma unroll
    for (int j = 0; j < 8; ++j) m = umax(m, abs_bits(o[i].at(j)));
  }
  m = wave_max_u32(m);
  if (threadIdx.x % kWave == 0) most[threadIdx.x / kWave] = m;
  __syncthreads();
  const F8Scale s(umax(umax(most[0], most[1]), umax(most[2], most[3])));
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = row0 + 16 * i;
    if (row < rows && n > 0)
      put_f8(codes + row * cols + k, n, s.codes(o[i].at(0), o[i].at(1), o[i].at(2), o[i].at(3)), s.codes(o[i].at(4), o[i].at(5), o[i].at(6), o[i].at(7)));
  }
  if (threadIdx.x == 0) scales[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = s.scale;
}

hipError_t launch_quantize_f8_blocks(const void *x, int dt, int64_t rows, int cols, uint8_t *codes, float *scales, hipStream_t st) {
  if (rows == 0 || cols == 0) return hipSuccess;
  auto *const kernel = dt == 0 ? &quantize_blocks_kernel<0> : dt == 1 ? &quantize_blocks_kernel<1> : &quantize_blocks_kernel<2>;
  const int64_t down = (rows + kF8Run - 1) / kF8Run, most = 65535;  // (a launch's y extent)
  for (int64_t y = 0; y < down; y += most) {
    const int64_t row = y * kF8Run, n = down - y < most ? down - y : most;
    kernel<<<dim3(f8_runs(cols), (unsigned)n), 256, 0, st>>>(value_at(x, dt, row * cols), rows - row, cols, codes + row * cols, scales + y * f8_runs(cols));
  }
  return hipGetLastError();
}

template <int DT>
__global__ __launch_bounds__(kRowThreads) void dequantize_f8_kernel(const uint8_t *__restrict__ codes, const float *__restrict__ scales, int64_t rows, int cols, int block_rows,
                                                                    void *__restrict__ out) {
  const int runs = f8_runs(cols);
  const uint32_t at = blockIdx.x * kRowRuns + threadIdx.x / 16;
  if (at >= (uint32_t)rows * (uint32_t)runs) return;
  const int64_t row = at / (uint32_t)runs;
  const int run = (int)(at - row * runs), k = run * kF8Run + (threadIdx.x % 16) * 8, n = cols - k;
  if (n <= 0) return;
  const float s = scales[row / block_rows * runs + run];
  uint32_t q[2] = {0, 0};
  const uint8_t *const from = codes + row * cols + k;
  if (n >= 8) __builtin_memcpy(q, from, 8);
  else
    for (int i = 0; i < n; ++i) q[i / 4] |= (uint32_t)from[i] << (8 * (i % 4));
  Octet<DT> o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[i / 2], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[i / 2], true);
    o.put(2 * i, (i % 2 ? hi[0] : lo[0]) * s);
    o.put(2 * i + 1, (i % 2 ? hi[1] : lo[1]) * s);
  }
  store_octet<DT>(out, row * cols + k, n, o);
}

hipError_t launch_dequantize_f8(const uint8_t *codes, const float *scales, int64_t rows, int cols, int block_rows, int dt, void *out, hipStream_t st) {
  if (rows == 0 || cols == 0) return hipSuccess;
  auto *const kernel = dt == 0 ? &dequantize_f8_kernel<0> : dt == 1 ? &dequantize_f8_kernel<1> : &dequantize_f8_kernel<2>;
  return in_launches(rows, cols, [&](int64_t r, int64_t n) {
    kernel<<<run_blocks(n, cols), kRowThreads, 0, st>>>(codes + r * cols, scales + r / block_rows * f8_runs(cols), n, cols, block_rows,
                                                        const_cast<char *>(value_at(out, dt, r * cols)));
  });
}

// ---------------------------------------------------------------- silu(gate) * up
__global__ __launch_bounds__(kRowThreads) void swiglu_f8_kernel(const float *__restrict__ g, const float *__restrict__ u, int64_t rows, int cols, F8Out to) {
  const int runs = f8_runs(cols);
  const uint32_t at = blockIdx.x * kRowRuns + threadIdx.x / 16;
  if (at >= (uint32_t)rows * (uint32_t)runs) return;
  const int64_t row = at / (uint32_t)runs;
  const int run = (int)(at - row * runs), k = run * kF8Run + (threadIdx.x % 16) * 8, n = cols - k;
  float v[8] = {};
  if (n > 0) {
    const Octet<2> a = load_octet<2>(g, row * cols + k, n), b = load_octet<2>(u, row * cols + k, n);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = silu(a.v[i]) * b.v[i];
  }
  write_run(v, to, row, run, n);
}

hipError_t launch_swiglu_f8(const float *g, const float *u, int64_t rows, int cols, const F8Out &to, hipStream_t st) {
  if (rows == 0 || cols == 0) return hipSuccess;
  return in_launches(rows, cols, [&](int64_t r, int64_t n) {
    swiglu_f8_kernel<<<run_blocks(n, cols), kRowThreads, 0, st>>>(g + r * cols, u + r * cols, n, cols, rows_from(to, r));
  });
}

// With s = sigmoid(g) and the slot's weight w:  dg = w dh u s (1 + g (1 - s)),  du = w dh g s,  dw = sum over the row of dh (g s u).
// (dw of g s u itself, not of the codes that the forward call makes of it: the rounding is passed through as in dg and du.)
// A block a row, its threads over the runs of both gradients; the weight's sum in float32, a thread's values in order, then the threads' in a fixed tree.
__global__ __launch_bounds__(kRowThreads) void swiglu_f8_grad_kernel(F8SwigluGrad a) {
  __shared__ float sums[kRowThreads / kWave];
  const int64_t row = blockIdx.x;
  const uint32_t pair = a.order[row];
  const bool named = row < (int64_t)a.offsets[a.n_experts];
  if (!named) {  // (its codes are read by no product)
    if (threadIdx.x == 0) put_value(a.dweights, pair, a.w_dtype, 0.f);
    return;
  }
  const float w = value_of(a.weights, pair, a.w_dtype);
  const int runs = f8_runs(a.cols);
  const F8Out to{a.codes, 2 * f8_row_bytes(a.cols), a.scales, 1, a.rows, true};
  float dw = 0.f;
  for (int run = threadIdx.x / 16; run < runs; run += kRowRuns) {
    const int k = run * kF8Run + (threadIdx.x % 16) * 8, n = a.cols - k;
    float dg[8] = {}, du[8] = {};
    if (n > 0) {
      const Octet<2> g = load_octet<2>(a.g, row * a.cols + k, n), u = load_octet<2>(a.u, row * a.cols + k, n), dh = load_octet<2>(a.dh, row * a.cols + k, n);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float s = sigmoid(g.v[i]), gs = g.v[i] * s, d = w * dh.v[i];
        dw += dh.v[i] * (gs * u.v[i]);
        dg[i] = d * u.v[i] * s * (1.f + g.v[i] * (1.f - s));
        du[i] = d * gs;
      }
    }
    write_run(dg, to, row, run, n);
    write_run(du, to, row, runs + run, n);
  }
  for (int d = 1; d < kWave; d <<= 1) dw += __shfl_xor(dw, d, kWave);
  if (threadIdx.x % kWave == 0) sums[threadIdx.x / kWave] = dw;
  __syncthreads();
  if (threadIdx.x == 0) put_value(a.dweights, pair, a.w_dtype, (sums[0] + sums[1]) + (sums[2] + sums[3]));
}

hipError_t launch_swiglu_f8_grad(const F8SwigluGrad &a, hipStream_t st) {
  if (a.rows == 0) return hipSuccess;
  swiglu_f8_grad_kernel<<<(unsigned)a.rows, kRowThreads, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace mi_moe
