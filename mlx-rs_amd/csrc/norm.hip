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

template <int CTRL>
__device__ __forceinline__ double dpp_of(double v) { return dpp_f64<CTRL>(v); }
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_of(uint32_t v) { return dpp_u32<CTRL>(v); }

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
    asm volatile("");  // (else the compiler makes one short store of the first value and of the last ones of both branches, and three of the other)
  }
}

// 1 / sqrt(mean + eps) from the double square sum: mi_moe_rms_norm's float operations, and double ones where the mean leaves the floats' range
__device__ __forceinline__ float rstd_of(double ss, int H, float eps) {
  const double m = ss / (double)H;
  if (m > 1e-30 && m < 1e37) return 1.0f / sqrtf((float)m + eps);
  return (float)(1.0 / sqrt(m + (double)eps));
}

// the integer nearest to 127 p / most, ties to even, of a quotient that is within 2^-13 of the half m: by the sign of 127 p - m most, whose products are taken with their rounding errors
__device__ __forceinline__ float beside_half(float m, double p, double most) {
  const double a = 127.0 * p, b = (double)m * most, d = (a - b) + (__builtin_fma(127.0, p, -a) - __builtin_fma((double)m, most, -b));
  return d > 0.0 ? m + 0.5f : d < 0.0 ? m - 0.5f : rintf(m);
}
// the codes of an octet in eight bits; most: the row's largest |w h|
template <int DT>
__device__ __forceinline__ void put_codes(unsigned char *to, int n, const Octet<DT> &h, const Octet<DT> &w, double most) {
  // rows of zeros have a scale and codes of zero; rows that hold an infinity or no number a scale that is none, so that what is made of them is none either
  uint32_t q[2] = {0, 0};
  if (most > 0.0 && most < INFINITY) {
    constexpr float kWhole = 12582912.f;  // 1.5 * 2^23: added to a small float, its low bits are the nearest integer, ties to even
    float v[8], off = 0.f;
    if (most > 1e-30 && most < 1e30) {
      const float inv = 127.f * __builtin_amdgcn_rcpf((float)most);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = h.at(i) * w.at(i) * inv;
    } else {  // products outside the floats' range
      const double inv = 127.0 / most;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (float)((double)h.at(i) * (double)w.at(i) * inv);
    }
    uint32_t k[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float t = v[i] + kWhole;
      off = fmaxf(off, fabsf(v[i] - (t - kWhole)));
      k[i] = __float_as_uint(t);
    }
    // the float quotient is up to 2^-14 off (2^-21.4 of a value below 128: a reciprocal to 2^-23 and five roundings): where that could change an integer, the exact products decide
    if (off > 0.4999f) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (fabsf(v[i] - rintf(v[i])) > 0.4999f) k[i] = __float_as_uint(kWhole + beside_half(rintf(2.f * v[i]) * 0.5f, (double)h.at(i) * (double)w.at(i), most));
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
      q[j] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(k[4 * j + 3], k[4 * j + 2], 0x0c0c0400u), __builtin_amdgcn_perm(k[4 * j + 1], k[4 * j], 0x0c0c0400u), 0x05040100u);
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
// The same as the bits of a float where the products are exact floats or nearly so (16-bit types): what is infinite or no number comes out above everything.  Good for a row
// whose result is a normal float well above the smallest; others (products beyond the floats' range, or below) are gone over in double.
template <int DT>
__device__ __forceinline__ uint32_t largest_bits(uint32_t most, const Octet<DT> &h, const Octet<DT> &w) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t p = __float_as_uint(h.at(i) * w.at(i)) & 0x7fffffffu;
    most = p > most ? p : most;
  }
  return most;
}
__device__ __forceinline__ bool in_floats(uint32_t bits) { return bits - 0x12800000u < 0x7f800000u - 0x12800000u; }  // 2^-90 and more

// f over the values of WAVES (up to 16) lanes that follow each other, in all of them and in one order
template <int WAVES, class T, class F>
__device__ __forceinline__ T join_waves(T v, F f) {
  if constexpr (WAVES > 1) v = f(v, dpp_of<kDppXor1>(v));
  if constexpr (WAVES > 2) v = f(v, dpp_of<kDppXor2>(v));
  if constexpr (WAVES > 4) v = f(v, dpp_of<kDppHalfMirror>(v));
  if constexpr (WAVES > 8) v = f(v, dpp_of<kDppMirror>(v));
  return v;
}
// a block's sums and largest values from its waves': a lane reads one wave's (all of them in each lane are 64 registers for 16 waves, and what was in those in scratch memory)
template <int WAVES, bool BOTH = true>
__device__ __forceinline__ void meet(double (&part)[WAVES][2], double &sum, double &other, bool is_sum) {  // BOTH: `other` too
  static_assert((WAVES & (WAVES - 1)) == 0 && WAVES <= 16);
  if ((threadIdx.x & (kWave - 1)) == 0) {
    part[threadIdx.x / kWave % WAVES][0] = sum;
    if constexpr (BOTH) part[threadIdx.x / kWave % WAVES][1] = other;
  }
  __syncthreads();
  const int i = threadIdx.x & (WAVES - 1);
  sum = join_waves<WAVES>(part[i][0], [](double u, double v) { return u + v; });
  if constexpr (BOTH) other = join_waves<WAVES>(part[i][1], [&](double u, double v) { return is_sum ? u + v : fmax(u, v); });
}

struct NormArgs {
  const void *x, *r, *w;  // r: or nullptr, then the sum is x
  float eps;
  int64_t T;
  int H;
  void *sum, *y;  // sum: or nullptr; y: rows in the input's type, or in eight bits
  float *scales;
};

// A row goes to TPR threads, an octet each, and stays in their registers between its sums and its results: memory is passed once, which is what bounds it.  One octet rather than two or
// four: fewer registers, more waves with loads under way.  us, one octet a thread / two (of 8192 values: four), with a residual, values that are read and written each once:
//   300 x 1024 3.5 / 4.2   16384 x 1024 23.0 / 27.7   777 x 4096 6.8 / 7.9   8192 x 4096 40.5 / 46.0 (6.6 TB/s)   2048 x 8192 22.9 / 30.1   8192 x 8192 93.7 / 119   (bf16)
//   rows in eight bits: 16384 x 1024 25.6 / 26.5   8192 x 4096 43.5 / 43.8   2048 x 8192 25.5 / 33.8   8192 x 8192 91.7 / 138
template <int DT, int TPR, bool ROWS8>
__global__ __launch_bounds__(TPR == kWave ? 256 : TPR, ROWS8 && DT == 1 ? 4 : 8) void add_rms_norm_kernel(NormArgs a) {
  constexpr int kRows = TPR == kWave ? 4 : 1, kWaves = TPR / kWave;
  constexpr bool BITS = ROWS8 && DT != 2;  // the largest |w h| as a float's bits
  __shared__ double part[kWaves][2];
  __shared__ uint32_t part_bits[BITS ? kWaves : 1];
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
  if (kWaves == 1 && row >= a.T) return;  // (rows of several waves have a block each: none is outside)
  const int64_t at = row * a.H + t * 8;
  const int n = a.H - t * 8;
  Octet<DT> h, r, w;
  if (n >= 8) {  // (all loads under way at once: one branch around them)
    h = load_octet<DT>(a.x, at, 8);
    w = load_octet<DT>(a.w, t * 8, 8);
    if (a.r) r = load_octet<DT>(a.r, at, 8);
  } else {
    h = load_octet<DT>(a.x, at, n);
    w = load_octet<DT>(a.w, t * 8, n);
    if (a.r) r = load_octet<DT>(a.r, at, n);
  }
  if (a.r) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) h.put2(i, h.at(i) + r.at(i), h.at(i + 1) + r.at(i + 1));
  }
  if (a.sum) store_octet<DT>(a.sum, at, n, h);
  double ss = 0.0, most = 0.0;  // most: the largest |w h|; infinite where one of them is infinite or no number
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = __builtin_fma((double)h.at(i), (double)h.at(i), ss);
  uint32_t bits = 0;
  if constexpr (BITS) {
    bits = wave_max_u32(largest_bits<DT>(0, h, w));
    if (kWaves > 1 && (threadIdx.x & (kWave - 1)) == 0) part_bits[threadIdx.x / kWave] = bits;
  } else if constexpr (ROWS8) {
    most = wave_max_f64(largest<DT>(0.0, h, w));
  }
  ss = wave_sum_f64(ss);
  if constexpr (kWaves > 1) meet<kWaves, ROWS8 && !BITS>(part, ss, most, false);
  if constexpr (BITS) {
    if constexpr (kWaves > 1) bits = join_waves<kWaves>(part_bits[threadIdx.x & (kWaves - 1)], [](uint32_t u, uint32_t v) { return u > v ? u : v; });
    most = (double)__uint_as_float(bits);
    if (!in_floats(bits)) {  // (the same in all of the row's threads)
      most = wave_max_f64(largest<DT>(0.0, h, w));
      double none = 0.0;
      if constexpr (kWaves > 1) {
        __syncthreads();
        meet<kWaves>(part, none, most, false);
      }
    }
  }
  const float rstd = rstd_of(ss, a.H, a.eps);
  if constexpr (!ROWS8) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) h.put2(i, w.at(i) * (h.at(i) * rstd), w.at(i + 1) * (h.at(i + 1) * rstd));
    store_octet<DT>(a.y, at, n, h);
  } else {
    if (t == 0) a.scales[row] = scale_of(most, rstd);
    put_codes<DT>(static_cast<unsigned char *>(a.y) + at, n, h, w, most);
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

template <int DT, int TPR>
static hipError_t start_norm(const NormArgs &a, bool rows8, hipStream_t st) {
  constexpr int block = TPR == kWave ? 256 : TPR, rows = block / TPR;
  const unsigned grid = (unsigned)((a.T + rows - 1) / rows);
  if (rows8) add_rms_norm_kernel<DT, TPR, true><<<grid, block, 0, st>>>(a);
  else add_rms_norm_kernel<DT, TPR, false><<<grid, block, 0, st>>>(a);
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
    if (H <= 512) return start_norm<DT, 64>(a, rows8, st);
    if (H <= 1024) return start_norm<DT, 128>(a, rows8, st);
    if (H <= 2048) return start_norm<DT, 256>(a, rows8, st);
    if (H <= 4096) return start_norm<DT, 512>(a, rows8, st);
    if (H <= 8192) return start_norm<DT, 1024>(a, rows8, st);
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

constexpr int norm_grad_threads(int tpr, bool together) { return tpr == kWave ? 256 : together ? 1024 : tpr; }

// A block has every blocks-th run of kRows rows (of up to 1024 values: a wave each) and their columns' sums for dw in registers; the sums of the blocks meet in a second launch, in a
// fixed order.  4096 x 4096, bf16, with the gradient along the residual: 32.4 us, 134 MB at 4.1 TB/s; bound by memory (those, and the blocks' sums written and read, 8 MB) and by the latency of
// a row, whose loads, sums and barrier follow each other.
template <int DT, int TPR, int CH, bool TOGETHER>
__global__ __launch_bounds__(norm_grad_threads(TPR, TOGETHER), 4) void norm_grad_kernel(NormGradArgs a) {
  constexpr int kRows = norm_grad_threads(TPR, TOGETHER) / TPR, kWaves = TPR / kWave;
  __shared__ double part[2][kRows][kWaves][2];
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
  int turn = 0;
  for (int64_t base = (int64_t)blockIdx.x * kRows; base < a.T; base += step, turn ^= 1) {  // (the same turns for all of a block's)
    const int64_t row = base + which < a.T ? base + which : a.T - 1;
    const bool mine = base + which < a.T;  // (else the last row again, without a result)
    struct { Octet<DT> h[CH], dy[CH], dh[CH]; } R;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int j = (c * TPR + t) * 8, n = a.H - j;
      if (n >= 8) {
        R.h[c] = load_octet<DT>(a.h, row * a.H + j, 8);
        R.dy[c] = load_octet<DT>(a.dy, row * a.H + j, 8);
        if (a.dh) R.dh[c] = load_octet<DT>(a.dh, row * a.H + j, 8);
      } else {
        R.h[c] = load_octet<DT>(a.h, row * a.H + j, n);
        R.dy[c] = load_octet<DT>(a.dy, row * a.H + j, n);
        if (a.dh) R.dh[c] = load_octet<DT>(a.dh, row * a.H + j, n);
      }
    }
    double ss = 0.0, dot = 0.0;  // sums of h^2 and of w dy h
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double v = R.h[c].at(i);
        ss = __builtin_fma(v, v, ss);
        const double g = DT == 2 ? (double)w[c].at(i) * (double)R.dy[c].at(i) : (double)(w[c].at(i) * R.dy[c].at(i));  // (exact of float16; of bfloat16 within the floats' range)
        dot = __builtin_fma(g, v, dot);
      }
    ss = wave_sum_f64(ss);
    dot = wave_sum_f64(dot);
    if constexpr (kWaves > 1) meet<kWaves>(part[turn][which], ss, dot, true);  // (one barrier a row: the next row's sums go to the other half)
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
          if (mine) dw[c][i + k] = __builtin_fmaf(g, hat, dw[c][i + k]);
          d[k] = rstd * __builtin_fmaf(-hat, mean, w[c].at(i + k) * g);
          if (a.dh) d[k] += R.dh[c].at(i + k);
        }
        R.h[c].put2(i, d[0], d[1]);
      }
      if (mine) store_octet<DT>(a.dx, row * a.H + j, a.H - j, R.h[c]);
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

// Rows of a block of 1024 threads are worked on at once, as many as it holds, where there are more rows than CUs: their sums for dw meet in LDS, and half or a quarter as many blocks' sums go through
// memory.  us, together / a block a row and more blocks: 1000 x 2048 10.9 / 11.3, 1000 x 2045 12.0 / 13.1, 300 x 4096 10.9 / 12.1, 8192 x 4096 53.2 / 53.1; 32 x 2048 7.7 / 6.4.
static bool norm_grad_together(int64_t T) { return T > 256; }
// Blocks of the backward pass: one a CU, of rows up to 1024 values what the chip holds at once and rows enough for each that its sums for dw are little beside them.  us, bf16, 256 / 512 / 768 / 1024
// blocks of 256 threads: 16384 x 1024 34.0, 27.9, 28.4, 28.5.  (The next row's loads ahead of a row's sums cost registers, and with them waves: 39.1 where 4096 x 4096 took 37.5; so does holding
// 64 registers, for twice the waves: 48 for 32.)
static int norm_grad_blocks(int64_t T, int H) {
  const int64_t each = H <= 1024 ? 4 : !norm_grad_together(T) ? 1 : H <= 2048 ? 4 : H <= 4096 ? 2 : 1, rows = (T + each - 1) / each;  // (turns of a block)
  const int64_t few = rows / 5 > 256 ? rows / 5 : 256, most = H <= 1024 ? 768 : 256, blocks = few < most ? few : most;
  return (int)(rows < blocks ? rows : blocks);
}
// (of no fewer rows less: what a batch has reserved is enough for every smaller one)
size_t norm_grad_bytes(int64_t T, int H) { return (size_t)(H > 1024 ? (T < 256 ? T : 256) : norm_grad_blocks(T, H)) * H * sizeof(float); }

template <int DT, int TPR, int CH>
static hipError_t start_norm_grad(const NormGradArgs &a, int blocks, hipStream_t st) {
  constexpr bool able = TPR > kWave && TPR < 1024;
  if (able && norm_grad_together(a.T)) norm_grad_kernel<DT, TPR, CH, able><<<(unsigned)blocks, norm_grad_threads(TPR, able), 0, st>>>(a);
  else norm_grad_kernel<DT, TPR, CH, false><<<(unsigned)blocks, norm_grad_threads(TPR, false), 0, st>>>(a);
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
