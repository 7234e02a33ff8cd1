// The residual's addition and the RMS norm behind it in one pass over the rows, with the normalised rows in the input's type or in
// eight bits, and the backward pass.
//
//   h = round(x + r)   rstd = 1 / sqrt(mean(h^2) + eps)   y = round(w (h rstd))
//   rows in 8 bits: with z = w h rstd, s = max |z| / 127 and q the integer nearest to z / s (ties to even).  rstd has no part in q:
//     z / s = 127 w h / max |w h|
//   backward, hat = h rstd: dx = dh + rstd (w dy - hat mean(w dy hat)),  dw = sum over rows of dy hat
//
// Contract of the norm: mlx_fast_rms_norm (mlx-rs/src/fast.rs:190-207; nn::RmsNorm, nn/normalization.rs:233-275) on the rounded sum: in bfloat16
// the bits of mi_moe_rms_norm on x + r.  The square sums are in double (exact products; any order gives the same float).
#include <type_traits>

#include "common.hpp"

namespace mi_moe {

__device__ __forceinline__ double wave_max_f64(double v) {
  v = fmax(v, dpp_f64<kDppXor1>(v));
  v = fmax(v, dpp_f64<kDppXor2>(v));
  v = fmax(v, dpp_f64<kDppHalfMirror>(v));
  v = fmax(v, dpp_f64<kDppMirror>(v));
  return fmax(fmax(readlane_f64(v, 0), readlane_f64(v, 16)), fmax(readlane_f64(v, 32), readlane_f64(v, 48)));
}

// ---------------------------------------------------------------- eight values of a row
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
  }
}

// 1 / sqrt(mean + eps) from the double square sum: mi_moe_rms_norm's float operations, and double ones where the mean leaves the floats' range
__device__ __forceinline__ float rstd_of(double ss, int H, float eps) {
  const double m = ss / (double)H;
  if (m > 1e-30 && m < 1e37) return 1.0f / sqrtf((float)m + eps);
  return (float)(1.0 / sqrt(m + (double)eps));
}

// the codes of an octet in eight bits; most: the row's largest |w h|, inv = 127 / most
template <int DT>
__device__ __forceinline__ void put_codes(unsigned char *to, int n, const Octet<DT> &h, const Octet<DT> &w, double most) {
  // rows of zeros have a scale and codes of zero; rows that hold an infinity or no number a scale that is none, so that what is made of them is none either
  const bool none = !(most > 0.0 && most < INFINITY), wide = !(most > 1e-30 && most < 1e30);
  const float inv = none ? 0.f : (float)(127.0 / most);
  uint32_t q[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = h.at(i) * w.at(i) * inv;
    float k = rintf(v);
    // the float quotient is up to 2^-15 off (three roundings of a value below 128): where that could change the integer, or the products leave
    // the floats' range, the exact products decide
    if (none) k = 0.f;
    else if (wide || fabsf(v - k) > 0.4999f) k = (float)rint(127.0 * ((double)h.at(i) * (double)w.at(i)) / most);
    q[i / 4] |= ((uint32_t)(int)k & 0xffu) << (8 * (i % 4));
  }
  if (n >= 8) __builtin_memcpy(to, q, 8);
  else
    for (int i = 0; i < n; ++i) to[i] = (unsigned char)(q[i / 4] >> (8 * (i % 4)));
}
__device__ __forceinline__ float scale_of(double most, float rstd) {
  return most > 0.0 && most < INFINITY ? (float)(most * (double)rstd / 127.0) : most > 0.0 ? NAN : 0.f;
}
// the largest |w h| of an octet and `most`, infinite where one is infinite or no number
template <int DT>
__device__ __forceinline__ double largest(double most, const Octet<DT> &h, const Octet<DT> &w) {
  bool finite = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const double p = fabs((double)h.at(i) * (double)w.at(i));
    finite &= p < INFINITY;
    most = p > most ? p : most;
  }
  return finite ? most : INFINITY;
}
// a block's sums and largest values, in the order of its waves
template <int WAVES>
__device__ __forceinline__ void meet(double (&part)[WAVES][2], double &sum, double &other, bool is_sum) {
  if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x / kWave % WAVES][0] = sum, part[threadIdx.x / kWave % WAVES][1] = other;
  __syncthreads();
  sum = 0.0;
  other = 0.0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) sum += part[i][0], other = is_sum ? other + part[i][1] : fmax(other, part[i][1]);
}

struct NormArgs {
  const void *x, *r, *w;  // r: or nullptr, then the sum is x
  float eps;
  int64_t T;
  int H;
  void *sum, *y;  // sum: or nullptr; y: rows in the input's type, or in eight bits
  float *scales;
};

// A row goes to TPR threads (a wave and more), CH octets each, and stays in their registers between its sums and its results: memory is passed once.
template <int DT, int TPR, int CH, bool ROWS8>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void add_rms_norm_kernel(NormArgs a) {
  constexpr int kRows = TPR < 256 ? 256 / TPR : 1, kWaves = TPR / kWave;
  __shared__ double part[kWaves][2];
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
  if (kWaves == 1 && row >= a.T) return;  // (rows of several waves have a block each: none is outside)
  const int64_t at = row * a.H;
  Octet<DT> h[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) h[c] = load_octet<DT>(a.x, at + (c * TPR + t) * 8, a.H - (c * TPR + t) * 8);
  if (a.r) {
    Octet<DT> r[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) r[c] = load_octet<DT>(a.r, at + (c * TPR + t) * 8, a.H - (c * TPR + t) * 8);
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < 8; i += 2) h[c].put2(i, h[c].at(i) + r[c].at(i), h[c].at(i + 1) + r[c].at(i + 1));
  }
  double ss = 0.0, most = 0.0;  // most: the largest |w h|; infinite where one of them is infinite or no number
  if (a.sum) {
#pragma unroll
    for (int c = 0; c < CH; ++c) store_octet<DT>(a.sum, at + (c * TPR + t) * 8, a.H - (c * TPR + t) * 8, h[c]);
  }
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __builtin_fma((double)h[c].at(i), (double)h[c].at(i), ss);
  Octet<DT> w[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) w[c] = load_octet<DT>(a.w, (c * TPR + t) * 8, a.H - (c * TPR + t) * 8);
  if constexpr (ROWS8) {
#pragma unroll
    for (int c = 0; c < CH; ++c) most = largest<DT>(most, h[c], w[c]);
  }
  ss = wave_sum_f64(ss);
  if constexpr (ROWS8) most = wave_max_f64(most);
  if constexpr (kWaves > 1) meet<kWaves>(part, ss, most, false);
  const float rstd = rstd_of(ss, a.H, a.eps);
  if constexpr (!ROWS8) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
      for (int i = 0; i < 8; i += 2) h[c].put2(i, w[c].at(i) * (h[c].at(i) * rstd), w[c].at(i + 1) * (h[c].at(i + 1) * rstd));
      store_octet<DT>(a.y, at + (c * TPR + t) * 8, a.H - (c * TPR + t) * 8, h[c]);
    }
  } else {
    if (t == 0) a.scales[row] = scale_of(most, rstd);
#pragma unroll
    for (int c = 0; c < CH; ++c)
      put_codes<DT>(static_cast<unsigned char *>(a.y) + at + (c * TPR + t) * 8, a.H - (c * TPR + t) * 8, h[c], w[c], most);
  }
}

// Rows of more values than 1024 threads hold octets: passed twice, the second time through the caches.
constexpr int kLong = 1024;
template <int DT, bool ROWS8>
__global__ __launch_bounds__(kLong) void add_rms_norm_long_kernel(NormArgs a) {
  __shared__ double part[kLong / kWave][2];
  const int64_t at = (int64_t)blockIdx.x * a.H;
  double ss = 0.0, most = 0.0;
#pragma unroll 1
  for (int j = threadIdx.x * 8; j < a.H; j += kLong * 8) {
    Octet<DT> h = load_octet<DT>(a.x, at + j, a.H - j);
    if (a.r) {
      const Octet<DT> r = load_octet<DT>(a.r, at + j, a.H - j);
#pragma unroll
      for (int i = 0; i < 8; i += 2) h.put2(i, h.at(i) + r.at(i), h.at(i + 1) + r.at(i + 1));
    }
    if (a.sum) store_octet<DT>(a.sum, at + j, a.H - j, h);
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __builtin_fma((double)h.at(i), (double)h.at(i), ss);
    if constexpr (ROWS8) most = largest<DT>(most, h, load_octet<DT>(a.w, j, a.H - j));
  }
  ss = wave_sum_f64(ss);
  if constexpr (ROWS8) most = wave_max_f64(most);
  meet<kLong / kWave>(part, ss, most, false);
  const float rstd = rstd_of(ss, a.H, a.eps);
  if (ROWS8 && threadIdx.x == 0) a.scales[blockIdx.x] = scale_of(most, rstd);
  const void *const from = a.r ? a.sum : a.x;  // (a thread's own octets)
#pragma unroll 1
  for (int j = threadIdx.x * 8; j < a.H; j += kLong * 8) {
    Octet<DT> h = load_octet<DT>(from, at + j, a.H - j);
    const Octet<DT> w = load_octet<DT>(a.w, j, a.H - j);
    if constexpr (ROWS8) {
      put_codes<DT>(static_cast<unsigned char *>(a.y) + at + j, a.H - j, h, w, most);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i += 2) h.put2(i, w.at(i) * (h.at(i) * rstd), w.at(i + 1) * (h.at(i + 1) * rstd));
      store_octet<DT>(a.y, at + j, a.H - j, h);
    }
  }
}

template <int DT>
static hipError_t start_norm_long(const NormArgs &a, bool rows8, hipStream_t st) {
  if (rows8) add_rms_norm_long_kernel<DT, true><<<(unsigned)a.T, kLong, 0, st>>>(a);
  else add_rms_norm_long_kernel<DT, false><<<(unsigned)a.T, kLong, 0, st>>>(a);
  return hipGetLastError();
}

template <int DT, int TPR, int CH>
static hipError_t start_norm(const NormArgs &a, bool rows8, hipStream_t st) {
  constexpr int block = TPR < 256 ? 256 : TPR, rows = block / TPR;
  const unsigned grid = (unsigned)((a.T + rows - 1) / rows);
  if (rows8) add_rms_norm_kernel<DT, TPR, CH, true><<<grid, block, 0, st>>>(a);
  else add_rms_norm_kernel<DT, TPR, CH, false><<<grid, block, 0, st>>>(a);
  return hipGetLastError();
}

template <class F>
static hipError_t with_dtype(int dt, F f) {
  if (dt == 0) return f(std::integral_constant<int, 0>{});
  if (dt == 1) return f(std::integral_constant<int, 1>{});
  return f(std::integral_constant<int, 2>{});
}

hipError_t launch_add_rms_norm(const void *x, const void *r, const void *w, float eps, int64_t T, int H, int dt, void *sum, void *y, float *scales,
                               hipStream_t st) {
  if (T == 0) return hipSuccess;
  const bool rows8 = scales != nullptr;
  constexpr int64_t kMost = (int64_t)1 << 21;  // rows of a launch, which has less than 2^32 threads
  if (T > kMost) {
    const int64_t size = dt == 2 ? 4 : 2;
    auto in = [&](const void *base, int64_t at) { return base ? static_cast<const char *>(base) + at : nullptr; };
    auto out = [&](void *base, int64_t at) { return base ? static_cast<char *>(base) + at : nullptr; };
    for (int64_t t = 0; t < T; t += kMost) {
      const int64_t at = t * H * size;
      const hipError_t e = launch_add_rms_norm(in(x, at), in(r, at), w, eps, T - t < kMost ? T - t : kMost, H, dt, out(sum, at), out(y, rows8 ? t * H : at), rows8 ? scales + t : nullptr, st);
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  }
  const NormArgs a{x, r, w, eps, T, H, sum, y, scales};
  return with_dtype(dt, [&](auto d) {
    constexpr int DT = decltype(d)::value;
    if (H <= 512) return start_norm<DT, 64, 1>(a, rows8, st);
    if (H <= 1024) return start_norm<DT, 64, 2>(a, rows8, st);
    if (H <= 2048) return start_norm<DT, 256, 1>(a, rows8, st);
    if (H <= 4096) return start_norm<DT, 256, 2>(a, rows8, st);
    if (H <= 8192) return start_norm<DT, 256, 4>(a, rows8, st);
    return start_norm_long<DT>(a, rows8, st);
  });
}

// ---------------------------------------------------------------- backward
struct NormGradArgs {
  const void *dy, *h, *dh, *w;  // dh: or nullptr
  float eps;
  int64_t T;
  int H;
  void *dx;
  float *parts;  // [blocks, H]: every block's sums over its rows
};

// A block has every blocks-th row (rows of up to 1024 values: a wave each, four at a time), the next one's loads under way while it works on one, and its columns' sums for dw in
// registers; the sums of the blocks meet in a second launch, in a fixed order.  Bound by memory: what the forward pass reads and writes, and the blocks' sums twice.
template <int DT, int TPR, int CH>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR, 4) void norm_grad_kernel(NormGradArgs a) {
  constexpr int kRows = TPR < 256 ? 256 / TPR : 1, kWaves = TPR / kWave;
  __shared__ double part[2][kWaves][2];
  const int t = threadIdx.x % TPR, which = threadIdx.x / TPR;
  const int64_t step = (int64_t)gridDim.x * kRows;
  Octet<DT> w[CH];
  float dw[CH][8];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    w[c] = load_octet<DT>(a.w, (c * TPR + t) * 8, a.H - (c * TPR + t) * 8);
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[c][i] = 0.f;
  }
  int64_t row = (int64_t)blockIdx.x * kRows + which;
  for (int turn = 0; row < a.T; row += step, turn ^= 1) {  // (rows of several waves: the same for all of the block's)
    struct { Octet<DT> h[CH], dy[CH], dh[CH]; } R;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int j = (c * TPR + t) * 8;
      R.h[c] = load_octet<DT>(a.h, row * a.H + j, a.H - j);
      R.dy[c] = load_octet<DT>(a.dy, row * a.H + j, a.H - j);
      if (a.dh) R.dh[c] = load_octet<DT>(a.dh, row * a.H + j, a.H - j);
    }
    double ss = 0.0, dot = 0.0;  // sums of h^2 and of w dy h
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double v = R.h[c].at(i);
        ss = __builtin_fma(v, v, ss);
        const double g = DT == 2 ? (double)w[c].at(i) * (double)R.dy[c].at(i) : (double)(w[c].at(i) * R.dy[c].at(i));  // (exact either way)
        dot = __builtin_fma(g, v, dot);
      }
    ss = wave_sum_f64(ss);
    dot = wave_sum_f64(dot);
    if constexpr (kWaves > 1) meet<kWaves>(part[turn], ss, dot, true);  // (one barrier a row: the next row's sums go to the other half)
    const float rstd = rstd_of(ss, a.H, a.eps);
    const float mean = (float)(dot * (double)rstd / (double)a.H);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int j = (c * TPR + t) * 8;
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        float d[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float hat = R.h[c].at(i + k) * rstd, g = R.dy[c].at(i + k);
          dw[c][i + k] = __builtin_fmaf(g, hat, dw[c][i + k]);
          d[k] = rstd * __builtin_fmaf(-hat, mean, w[c].at(i + k) * g);
          if (a.dh) d[k] += R.dh[c].at(i + k);
        }
        R.h[c].put2(i, d[0], d[1]);
      }
      store_octet<DT>(a.dx, row * a.H + j, a.H - j, R.h[c]);
    }
  }
  float *const to = a.parts + (int64_t)blockIdx.x * a.H;
  if constexpr (kRows > 1) {  // the block's rows' sums, one after the other
    __shared__ float meet[kRows - 1][CH * TPR * 8];
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (which > 0) meet[which - 1][(c * 8 + i) * TPR + t] = dw[c][i];
    __syncthreads();
    if (which > 0) return;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int r = 0; r < kRows - 1; ++r) dw[c][i] += meet[r][(c * 8 + i) * TPR + t];
  }
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int j = (c * TPR + t) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (j + i < a.H) to[j + i] = dw[c][i];
  }
}

// Rows of more values than 1024 threads hold octets: passed twice, and the sums for dw kept where they go.
template <int DT>
__global__ __launch_bounds__(kLong) void norm_grad_long_kernel(NormGradArgs a) {
  __shared__ double part[2][kLong / kWave][2];
  float *const to = a.parts + (int64_t)blockIdx.x * a.H;
  int turn = 0;
#pragma unroll 1
  for (int64_t row = blockIdx.x; row < a.T; row += gridDim.x, turn ^= 1) {
    const int64_t at = row * a.H;
    double ss = 0.0, dot = 0.0;
#pragma unroll 1
    for (int j = threadIdx.x * 8; j < a.H; j += kLong * 8) {
      const Octet<DT> h = load_octet<DT>(a.h, at + j, a.H - j), dy = load_octet<DT>(a.dy, at + j, a.H - j), w = load_octet<DT>(a.w, j, a.H - j);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double v = h.at(i);
        ss = __builtin_fma(v, v, ss);
        dot = __builtin_fma((double)w.at(i) * (double)dy.at(i), v, dot);
      }
    }
    ss = wave_sum_f64(ss);
    dot = wave_sum_f64(dot);
    meet<kLong / kWave>(part[turn], ss, dot, true);
    const float rstd = rstd_of(ss, a.H, a.eps);
    const float mean = (float)(dot * (double)rstd / (double)a.H);
#pragma unroll 1
    for (int j = threadIdx.x * 8; j < a.H; j += kLong * 8) {
      Octet<DT> h = load_octet<DT>(a.h, at + j, a.H - j), dh;
      const Octet<DT> dy = load_octet<DT>(a.dy, at + j, a.H - j), w = load_octet<DT>(a.w, j, a.H - j);
      if (a.dh) dh = load_octet<DT>(a.dh, at + j, a.H - j);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float hat = h.at(i) * rstd, g = dy.at(i);
        if (j + i < a.H) to[j + i] = row == blockIdx.x ? g * hat : __builtin_fmaf(g, hat, to[j + i]);
        float d = rstd * __builtin_fmaf(-hat, mean, w.at(i) * g);
        if (a.dh) d += dh.at(i);
        h.put(i, d);
      }
      store_octet<DT>(a.dx, at + j, a.H - j, h);
    }
  }
}

// dw = the blocks' sums: 16 columns a block, every 64th block's sums a thread
template <int DT>
__global__ __launch_bounds__(1024) void norm_grad_weight_kernel(const float *parts, int blocks, int H, void *dw) {
  __shared__ float sums[64][17];
  const int c = threadIdx.x & 15, col = blockIdx.x * 16 + c, slice = threadIdx.x >> 4;
  float s = 0.f;
  if (col < H) {
#pragma unroll 4
    for (int g = slice; g < blocks; g += 64) s += parts[(int64_t)g * H + col];
  }
  sums[slice][c] = s;
  __syncthreads();
  if (threadIdx.x < 256) {  // 16 threads a column, four sums each, then a tree
    const int cc = threadIdx.x >> 4, q = threadIdx.x & 15;
    float v = (sums[q][cc] + sums[q + 16][cc]) + (sums[q + 32][cc] + sums[q + 48][cc]);
    v += __uint_as_float(dpp_u32<kDppXor1>(__float_as_uint(v)));
    v += __uint_as_float(dpp_u32<kDppXor2>(__float_as_uint(v)));
    v += __uint_as_float(dpp_u32<kDppHalfMirror>(__float_as_uint(v)));
    v += __uint_as_float(dpp_u32<kDppMirror>(__float_as_uint(v)));
    if (q == 0 && blockIdx.x * 16 + cc < H) {
      Octet<DT> o;
      o.put(0, v);
      static_cast<typename Octet<DT>::Raw *>(dw)[blockIdx.x * 16 + cc] = o.v[0];
    }
  }
}

// Blocks of the backward pass: what the chip holds at once (of 1024 threads one a CU), and rows enough for each that its sums for dw are little beside them.  us, bf16, 256 / 512 / 768 / 1024
// blocks: 1000 x 2048 12.0, 12.8, 15.0, 18.0; 4096 x 4096 42.8, 37.5, 41.0, 41.8; 16384 x 1024 51.3, 36.0, 29.8, 32.1; float32 2048 x 8192 51.5, 62.8, 72.3, 82.7.  (The next row's loads
// ahead of a row's sums cost registers, and with them waves: 46.3, 39.1, 44.0, 45.7 for 4096 x 4096.)
static int norm_grad_blocks(int64_t T, int H) {
  const int64_t rows = H <= 1024 ? (T + 3) / 4 : T, most = H <= 1024 ? 768 : H <= 4096 ? 512 : 256;
  const int64_t few = rows / 5 > 256 ? rows / 5 : 256, blocks = few < most ? few : most;
  return (int)(rows < blocks ? rows : blocks);
}
size_t norm_grad_bytes(int64_t T, int H) { return (size_t)norm_grad_blocks(T, H) * H * sizeof(float); }

template <int DT, int TPR, int CH>
static hipError_t start_norm_grad(const NormGradArgs &a, int blocks, hipStream_t st) {
  norm_grad_kernel<DT, TPR, CH><<<(unsigned)blocks, TPR < 256 ? 256 : TPR, 0, st>>>(a);
  return hipGetLastError();
}

template <int DT>
static hipError_t start_norm_grad_long(const NormGradArgs &a, int blocks, hipStream_t st) {
  norm_grad_long_kernel<DT><<<(unsigned)blocks, kLong, 0, st>>>(a);
  return hipGetLastError();
}

hipError_t launch_norm_grad(const void *dy, const void *h, const void *dh, const void *w, float eps, int64_t T, int H, int dt, void *dx, void *dw,
                            float *parts, hipStream_t st) {
  const NormGradArgs a{dy, h, dh, w, eps, T, H, dx, parts};
  const int blocks = norm_grad_blocks(T, H);
  return with_dtype(dt, [&](auto d) {
    constexpr int DT = decltype(d)::value;
    hipError_t e = hipSuccess;
    if (T > 0)
      e = H <= 512     ? start_norm_grad<DT, 64, 1>(a, blocks, st)
          : H <= 1024  ? start_norm_grad<DT, 64, 2>(a, blocks, st)
          : H <= 2048  ? start_norm_grad<DT, 256, 1>(a, blocks, st)
          : H <= 4096  ? start_norm_grad<DT, 512, 1>(a, blocks, st)
          : H <= 8192  ? start_norm_grad<DT, 1024, 1>(a, blocks, st)
                       : start_norm_grad_long<DT>(a, blocks, st);
    if (e != hipSuccess) return e;
    norm_grad_weight_kernel<DT><<<(unsigned)((H + 15) / 16), 1024, 0, st>>>(parts, blocks, H, dw);  // (no rows: zeros)
    return hipGetLastError();
  });
}

}  // namespace mi_moe
