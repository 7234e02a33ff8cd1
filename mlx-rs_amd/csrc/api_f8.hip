// C ABI of the experts and linear layers on e4m3 weights (include/mi_moe_f8.h): validation, workspaces and the launch sequences.
#include "../../include/mi_moe_f8.h"

#include <algorithm>

#include "entries.hpp"
#include "f8.hpp"

using namespace mi_moe;

namespace {

constexpr int64_t kMostPairs = ((int64_t)1 << 24) - 1;  // a block a token or row, in launches of less than 2^32 threads
constexpr int32_t kMostExtent = 1 << 22, kMostExperts = 512;

int check_types(const char *who, int32_t dtype, int32_t w_dtype = MI_MOE_DTYPE_BF16) {
  for (int32_t d : {dtype, w_dtype})
    if (d != MI_MOE_DTYPE_BF16 && d != MI_MOE_DTYPE_F16 && d != MI_MOE_DTYPE_F32) return fail("%s: dtype must be MI_MOE_DTYPE_BF16, _F16 or _F32, got %d", who, d);
  return 0;
}
int check_slots(const char *who, int64_t T, int32_t top_k, int32_t hidden) {
  if (top_k < 1 || top_k > 32) return fail("%s: top_k must be in [1, 32], got %d", who, top_k);
  if (T < 0 || T > kMostPairs / top_k) return fail("%s: token count out of range (tokens times top_k up to 2^24 - 1)", who);
  if (hidden < 1 || hidden > kMostExtent) return fail("%s: hidden must be in [1, 2^22], got %d", who, hidden);
  return 0;
}
int check_experts(const char *who, int32_t n) {
  return n < 1 || n > 512 ? fail("%s: n_experts must be in [1, 512], got %d", who, n) : 0;
}
int check_workspace(const char *who, const void *p, size_t bytes, size_t need) {
  if (need && (!p || !aligned16(p) || bytes < need)) return fail("%s: workspace must be 16-byte aligned and hold %zu bytes, got %zu", who, need, bytes);
  return 0;
}

// rows in e4m3 in a workspace
struct RowsIn {
  uint8_t *codes;
  float *scales;
  RowsIn(Carver &c, int64_t rows, int cols, int halves = 1)
      : codes(c.take<uint8_t>((size_t)(rows * f8_row_bytes(cols) * halves))), scales(c.take<float>((size_t)(rows * f8_runs(cols) * halves))) {}
  F8Rows as(int64_t rows) const { return {codes, scales, rows}; }
  F8Out out(int64_t rows, int cols) const { return f8_workspace_rows(codes, scales, rows, cols); }
};

int check_linear(const char *who, const void *x, const void *w, const float *scales, int64_t M, int32_t N, int32_t K, int32_t transpose, int32_t dtype, const void *y) {
  if (check_types(who, dtype)) return 1;
  if (N < 1 || K < 1 || N > kMostExtent || K > kMostExtent) return fail("%s: N and K must be in [1, 2^22], got N = %d, K = %d", who, N, K);
  if (transpose ? K % 16 : N % 16) return fail("%s: a matrix's rows (%s = %d) must be a multiple of 16 values", who, transpose ? "K" : "N", transpose ? K : N);
  if (M < 0 || M > ((int64_t)1 << 35) / N || M > ((int64_t)1 << 35) / K || M > (int64_t)1 << 30) return fail("%s: row count out of range (rows times columns up to 2^35)", who);
  if (M == 0) return 0;
  if (!x || !w || !scales || !y) return fail("%s: x, w, scales and y must be non-NULL", who);
  if (!aligned16(w)) return fail("%s: w must be 16-byte aligned", who);
  return 0;
}
// What linear() keeps in its workspace; parts only where the rows are few enough for them.
struct LinearWs {
  RowsIn x;
  uint4 *list;
  float *parts;
  size_t bytes;
  LinearWs(void *at, int64_t M, int N, int K) : LinearWs(Carver(at), M, N, K) {}

 private:
  LinearWs(Carver c, int64_t M, int N, int K)
      : x(c, M, K), list(c.take<uint4>((size_t)f8_list_places(M, kMostExperts))),
        parts(M <= f8_parts_rows(N, f8_runs(K)) ? reinterpret_cast<float *>(c.take<char>(f8_parts_bytes(M, N, f8_runs(K)))) : nullptr), bytes(c.off + 256) {}
};
size_t linear_bytes(int64_t M, int N, int K) {  // (never less for more rows: parts may be room that a larger product's rows take)
  return std::max(LinearWs(nullptr, M, N, K).bytes, LinearWs(nullptr, std::min(M, f8_parts_rows(N, f8_runs(K))), N, K).bytes);
}
// A list for a product, or none for one matrix.
void list_for(F8Product &p, F8Lists &lists, int i, uint4 *at) {
  p.list = at;
  lists.list[i] = at;
  lists.tile[i] = f8_tile_rows(p);
  lists.places[i] = (int)f8_most_pieces(p.rows, p.n_mats, lists.tile[i]);
}

int linear(const char *who, const void *x, const void *w, const float *scales, const void *bias, const uint32_t *offsets, int64_t M, int E, int32_t N, int32_t K, int32_t transpose,
           int32_t dtype, void *y, void *workspace, size_t workspace_bytes, hipStream_t st) {
  if (check_workspace(who, workspace, workspace_bytes, linear_bytes(M, N, K))) return 1;
  if (y == x) return fail("%s: y must not be x", who);
  const LinearWs ws(workspace, M, N, K);
  F8Product p{};
  p.x = ws.x.as(M);
  p.n_mats = E;
  p.rows = M;
  p.m[0] = p.m[1] = {static_cast<const uint8_t *>(w), scales};
  p.transpose = transpose != 0;
  p.N = N;
  p.K = K;
  p.bias = bias;
  p.y = y;
  p.dt = dtype;
  F8Lists lists;
  lists.offsets = offsets;
  lists.n_mats = E;
  lists.rows = M;
  if (offsets) list_for(p, lists, 0, ws.list);
  p.parts = ws.parts;
  if (!offsets && f8_in_blocks(p, M)) {
    p.raw = x;
    p.raw_dt = dtype;
    MI_HIP(launch_f8_product(p, st));
    return 0;
  }
  MI_HIP(launch_quantize_f8_rows(x, dtype, M, K, ws.x.out(M, K), st, lists));
  MI_HIP(launch_f8_product(p, st));
  return 0;
}

// What the experts keep in their workspace.
struct ExpertsWs {
  uint32_t *order, *offsets;
  int32_t *inverse;
  uint4 *list[3];
  void *sort;
  RowsIn x, dout;   // rows of tokens
  float *g, *u, *dh;  // float32 rows of pairs: gradients, and batches of a few rows an expert
  RowsIn h;         // rows of pairs: h, or dg and du side by side
  void *y;          // of pairs, for the sum over slots: float32, or scaled float16
  float *y_scales;
  float *parts;     // gradients: of a few rows an expert
  size_t bytes;
  ExpertsWs(void *at, int64_t T, int H, int I, int E, int k, bool grad) : ExpertsWs(Carver(at), T, T * k, H, I, E, k, grad) {}

 private:
  ExpertsWs(Carver c, int64_t T, int64_t P, int H, int I, int E, int k, bool grad)
      : order(c.take<uint32_t>((size_t)P)), offsets(c.take<uint32_t>((size_t)E + 1)), inverse(c.take<int32_t>((size_t)P)),
        list{c.take<uint4>((size_t)f8_list_places(P, E)), c.take<uint4>((size_t)f8_list_places(P, E)), c.take<uint4>((size_t)f8_list_places(P, E))}, sort(c.take<char>(sort_tokens_bytes(T, k, E))),
        x(c, T, H), dout(c, grad ? T : 0, H), g(c.take<float>(float_rows(P, E, grad) * I)), u(c.take<float>(float_rows(P, E, grad) * I)), dh(c.take<float>(grad ? (size_t)P * I : 0)),
        h(c, P, I, grad ? 2 : 1), y(c.take<char>(y_bytes(P, H, E))), y_scales(c.take<float>((size_t)P * ((H + 63) / 64))),
        parts(reinterpret_cast<float *>(c.take<char>(grad ? parts_bytes(std::min(P, (int64_t)16 * E), H, I) : 0))), bytes(c.off + 256) {}
  static size_t parts_bytes(int64_t rows, int H, int I) {  // the gradient at h, of H stages' values by I columns, and that at x
    return std::max(f8_parts_bytes(rows, I, f8_stages(H, false)), f8_parts_bytes(rows, H, f8_stages(I, true)));
  }
  static size_t y_bytes(int64_t P, int H, int E) {  // halves, or floats: of few rows an expert (all columns), or of some columns at a time
    return std::max({(size_t)P * H * 2, (size_t)std::min(P, (int64_t)16 * E) * H * 4, (size_t)P * half_columns(H) * 4});
  }
  static int half_columns(int H) { return std::min(H, ((H + kF8TileN - 1) / kF8TileN + 1) / 2 * kF8TileN); }  // whole tiles

 public:
  static int float_columns(int64_t P, int H, int E) { return P <= (int64_t)16 * E ? H : half_columns(H); }  // columns of float32 rows that y holds

 private:
  static size_t float_rows(int64_t P, int E, bool grad) { return (size_t)(grad || P <= (int64_t)16 * E ? P : (int64_t)16 * E); }  // (never less for more tokens)
};

int check_switch(const char *who, const mi_moe_f8_experts *e, const void *x, const uint32_t *idx, const void *w, int32_t w_dtype, int64_t T, int32_t hidden, int32_t intermediate,
                 int32_t n_experts, int32_t top_k, int32_t dtype) {
  if (check_types(who, dtype, w_dtype) || check_slots(who, T, top_k, hidden) || check_experts(who, n_experts)) return 1;
  if (dtype == MI_MOE_DTYPE_F32) return fail("%s: dtype must be MI_MOE_DTYPE_BF16 or _F16", who);
  if (hidden % 16 || intermediate < 1 || intermediate > kMostExtent || intermediate % 16)
    return fail("%s: hidden and intermediate must be multiples of 16 up to 2^22, got %d, %d", who, hidden, intermediate);
  if (T * f8_row_bytes(hidden) >= (int64_t)0xffffff00) return fail("%s: tokens times hidden must be below 2^32", who);
  if (T * top_k * (int64_t)hidden > (int64_t)1 << 35 || T * top_k * (int64_t)intermediate > (int64_t)1 << 35) return fail("%s: rows times columns up to 2^35", who);
  if (T == 0) return 0;
  if (!e || !e->gate || !e->up || !e->down || !e->gate_scales || !e->up_scales || !e->down_scales) return fail("%s: the experts' weights and scales must be non-NULL", who);
  if (!aligned16(e->gate) || !aligned16(e->up) || !aligned16(e->down)) return fail("%s: weights must be 16-byte aligned", who);
  if (!x || !idx || !w) return fail("%s: x, topk_idx and topk_w must be non-NULL", who);
  return 0;
}

// A product of sorted rows, and the sums of tokens' rows over the slots, `columns` at a time.
hipError_t product_to_tokens(F8Product p, int columns, const void *weights, int w_dtype, const int32_t *inverse, int64_t T, int k, int dt, void *out, hipStream_t st) {
  const int H = p.N;
  for (int n = 0; n < H; n += columns) {
    const int count = std::min(columns, H - n);
    if (count < H) p.n_first = n, p.n_count = count;
    if (hipError_t e = launch_f8_product(p, st); e != hipSuccess) return e;
    if (hipError_t e = launch_unsort_made(p.y, p.y_scales, weights, w_dtype, inverse, T, k, count, dt, static_cast<uint16_t *>(out) + n, H, st); e != hipSuccess) return e;
  }
  return hipSuccess;
}

F8Mat mat(const void *w, const float *s) { return {static_cast<const uint8_t *>(w), s}; }

}  // namespace

extern "C" {

int mi_moe_sort_tokens_workspace_size(int64_t T, int32_t top_k, int32_t n_experts, size_t *bytes) try {
  if (!bytes) return fail("sort_tokens_workspace_size: bytes is NULL");
  if (check_slots("sort_tokens_workspace_size", T, top_k, 1) || check_experts("sort_tokens_workspace_size", n_experts)) return 1;
  *bytes = sort_tokens_bytes(T, top_k, n_experts);
  return 0;
} MI_CATCH("sort_tokens_workspace_size")

int mi_moe_sort_tokens(const void *x, const uint32_t *topk_idx, int64_t T, int32_t top_k, int32_t n_experts, int32_t hidden, int32_t dtype, void *rows, uint32_t *order,
                       int32_t *inverse, uint32_t *offsets, void *workspace, size_t workspace_bytes, void *stream) try {
  if (check_types("sort_tokens", dtype) || check_slots("sort_tokens", T, top_k, hidden) || check_experts("sort_tokens", n_experts)) return 1;
  if (!offsets || (T > 0 && (!topk_idx || !order || !inverse || (rows && !x)))) return fail("sort_tokens: topk_idx, order, inverse, offsets, and x with rows, must be non-NULL");
  if (check_workspace("sort_tokens", workspace, workspace_bytes, sort_tokens_bytes(T, top_k, n_experts))) return 1;
  if (rows && rows == x && T > 0) return fail("sort_tokens: rows must not be x");
  MI_HIP(launch_sort_tokens({topk_idx, T, top_k, n_experts, order, inverse, offsets}, x, dtype, hidden, rows, workspace, static_cast<hipStream_t>(stream)));
  return 0;
} MI_CATCH("sort_tokens")

int mi_moe_sort_tokens_grad(const void *drows, const int32_t *inverse, int64_t T, int32_t top_k, int32_t hidden, int32_t dtype, void *dx, void *stream) try {
  if (check_types("sort_tokens_grad", dtype) || check_slots("sort_tokens_grad", T, top_k, hidden)) return 1;
  if (T == 0) return 0;
  if (!drows || !inverse || !dx) return fail("sort_tokens_grad: drows, inverse and dx must be non-NULL");
  if (dx == drows) return fail("sort_tokens_grad: dx must not be drows");
  MI_HIP(launch_unsort_tokens(drows, nullptr, 0, inverse, T, top_k, hidden, dtype, dx, static_cast<hipStream_t>(stream)));
  return 0;
} MI_CATCH("sort_tokens_grad")

int mi_moe_unsort_tokens(const void *rows, const void *topk_w, int32_t w_dtype, const int32_t *inverse, int64_t T, int32_t top_k, int32_t hidden, int32_t dtype, void *out,
                         void *stream) try {
  if (check_types("unsort_tokens", dtype, w_dtype) || check_slots("unsort_tokens", T, top_k, hidden)) return 1;
  if (T == 0) return 0;
  if (!rows || !topk_w || !inverse || !out) return fail("unsort_tokens: rows, topk_w, inverse and out must be non-NULL");
  if (out == rows) return fail("unsort_tokens: out must not be rows");
  MI_HIP(launch_unsort_tokens(rows, topk_w, w_dtype, inverse, T, top_k, hidden, dtype, out, static_cast<hipStream_t>(stream)));
  return 0;
} MI_CATCH("unsort_tokens")

int mi_moe_unsort_tokens_grad(const void *dout, const void *rows, const void *topk_w, int32_t w_dtype, const int32_t *inverse, int64_t T, int32_t top_k, int32_t hidden,
                              int32_t dtype, void *drows, void *dweights, void *stream) try {
  if (check_types("unsort_tokens_grad", dtype, w_dtype) || check_slots("unsort_tokens_grad", T, top_k, hidden)) return 1;
  if (T == 0) return 0;
  if (!dout || !rows || !topk_w || !inverse || !drows || !dweights) return fail("unsort_tokens_grad: dout, rows, topk_w, inverse, drows and dweights must be non-NULL");
  if (drows == rows || drows == dout) return fail("unsort_tokens_grad: drows must not be %s", drows == rows ? "rows" : "dout");
  MI_HIP(launch_unsort_tokens_grad(dout, rows, topk_w, w_dtype, inverse, T, top_k, hidden, dtype, drows, dweights, static_cast<hipStream_t>(stream)));
  return 0;
} MI_CATCH("unsort_tokens_grad")

static int check_f8(const char *who, int32_t dtype, int64_t rows, int64_t cols, int32_t block_rows) {
  if (check_types(who, dtype)) return 1;
  if (block_rows != 1 && block_rows != kF8Run) return fail("%s: block_rows must be 1 or 128, got %d", who, block_rows);
  if (cols < 1 || cols > kMostExtent) return fail("%s: cols must be in [1, 2^22]", who);
  if (rows < 0 || rows > ((int64_t)1 << 40) / cols) return fail("%s: row count out of range", who);
  return 0;
}

int mi_moe_quantize_f8(const void *x, int32_t dtype, int64_t rows, int64_t cols, int32_t block_rows, void *codes, float *scales, void *stream) try {
  if (check_f8("quantize_f8", dtype, rows, cols, block_rows)) return 1;
  if (rows == 0) return 0;
  if (!x || !codes || !scales) return fail("quantize_f8: x, codes and scales must be non-NULL");
  uint8_t *const q = static_cast<uint8_t *>(codes);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (block_rows == 1) MI_HIP(launch_quantize_f8_rows(x, dtype, rows, (int)cols, {q, cols, scales, f8_runs((int)cols), 1, false}, st));
  else MI_HIP(launch_quantize_f8_blocks(x, dtype, rows, (int)cols, q, scales, st));
  return 0;
} MI_CATCH("quantize_f8")

int mi_moe_dequantize_f8(const void *codes, const float *scales, int64_t rows, int64_t cols, int32_t block_rows, int32_t dtype, void *out, void *stream) try {
  if (check_f8("dequantize_f8", dtype, rows, cols, block_rows)) return 1;
  if (rows == 0) return 0;
  if (!codes || !scales || !out) return fail("dequantize_f8: codes, scales and out must be non-NULL");
  MI_HIP(launch_dequantize_f8(static_cast<const uint8_t *>(codes), scales, rows, (int)cols, block_rows, dtype, out, static_cast<hipStream_t>(stream)));
  return 0;
} MI_CATCH("dequantize_f8")

int mi_moe_linear_f8_workspace_size(int64_t M, int32_t N, int32_t K, size_t *bytes) try {
  if (!bytes) return fail("linear_f8_workspace_size: bytes is NULL");
  if (M < 0 || M > (int64_t)1 << 30 || N < 1 || N > kMostExtent || K < 1 || K > kMostExtent || M > ((int64_t)1 << 35) / K || M > ((int64_t)1 << 35) / N) return fail("linear_f8_workspace_size: bad sizes");
  *bytes = linear_bytes(M, N, K);
  return 0;
} MI_CATCH("linear_f8_workspace_size")

int mi_moe_linear_f8(const void *x, const void *w, const float *scales, const void *linear_bias, int64_t M, int32_t N, int32_t K, int32_t transpose, int32_t dtype, void *y,
                     void *workspace, size_t workspace_bytes, void *stream) try {
  if (check_linear("linear_f8", x, w, scales, M, N, K, transpose, dtype, y)) return 1;
  if (linear_bias && !transpose) return fail("linear_f8: a linear bias goes with transpose");
  if (M == 0) return 0;
  return linear("linear_f8", x, w, scales, linear_bias, nullptr, M, 1, N, K, transpose, dtype, y, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
} MI_CATCH("linear_f8")

int mi_moe_grouped_linear_f8(const void *x, const void *w, const float *scales, const uint32_t *offsets, int64_t rows, int32_t n_experts, int32_t N, int32_t K, int32_t transpose,
                             int32_t dtype, void *y, void *workspace, size_t workspace_bytes, void *stream) try {
  if (check_linear("grouped_linear_f8", x, w, scales, rows, N, K, transpose, dtype, y) || check_experts("grouped_linear_f8", n_experts)) return 1;
  if (rows == 0) return 0;
  if (!offsets) return fail("grouped_linear_f8: offsets must be non-NULL");
  return linear("grouped_linear_f8", x, w, scales, nullptr, offsets, rows, n_experts, N, K, transpose, dtype, y, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
} MI_CATCH("grouped_linear_f8")

int mi_moe_switch_glu_f8_workspace_size(int64_t T, int32_t hidden, int32_t intermediate, int32_t n_experts, int32_t top_k, int32_t grad, size_t *bytes) try {
  if (!bytes) return fail("switch_glu_f8_workspace_size: bytes is NULL");
  if (check_slots("switch_glu_f8_workspace_size", T, top_k, hidden) || check_experts("switch_glu_f8_workspace_size", n_experts)) return 1;
  if (intermediate < 1 || intermediate > kMostExtent) return fail("switch_glu_f8_workspace_size: intermediate must be in [1, 2^22], got %d", intermediate);
  *bytes = ExpertsWs(nullptr, T, hidden, intermediate, n_experts, top_k, grad != 0).bytes;
  return 0;
} MI_CATCH("switch_glu_f8_workspace_size")

int mi_moe_switch_glu_f8(const void *x, const uint32_t *topk_idx, const void *topk_w, int32_t w_dtype, const mi_moe_f8_experts *experts, int64_t T, int32_t hidden,
                         int32_t intermediate, int32_t n_experts, int32_t top_k, int32_t dtype, void *out, void *workspace, size_t workspace_bytes, void *stream) try {
  if (check_switch("switch_glu_f8", experts, x, topk_idx, topk_w, w_dtype, T, hidden, intermediate, n_experts, top_k, dtype)) return 1;
  if (T == 0) return 0;
  if (!out) return fail("switch_glu_f8: out must be non-NULL");
  const ExpertsWs ws(workspace, T, hidden, intermediate, n_experts, top_k, false);
  if (check_workspace("switch_glu_f8", workspace, workspace_bytes, ws.bytes)) return 1;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t P = T * top_k;
  F8Product p{};
  p.x = ws.x.as(T);
  p.order = ws.order;
  p.k_div = top_k;
  p.n_mats = n_experts;
  p.rows = P;
  p.list = ws.list[0];
  p.m[0] = mat(experts->gate, experts->gate_scales);
  p.m[1] = mat(experts->up, experts->up_scales);
  p.transpose = true;
  p.N = intermediate;
  p.K = hidden;
  p.dt = MI_MOE_DTYPE_F32;
  F8Product d{};
  d.x = ws.h.as(P);
  d.k_div = top_k;
  d.n_mats = n_experts;
  d.rows = P;
  d.m[0] = d.m[1] = mat(experts->down, experts->down_scales);
  d.transpose = true;
  d.N = hidden;
  d.K = intermediate;
  d.y = ws.y;
  d.list = ws.list[1];
  d.dt = dtype;
  // A few tokens: the lists come beside the sorting, rows are rounded where they are multiplied.  More of them go to the tiles, where silu(gate) * up is made in a block's registers,
  // from two rows an expert on (32 / 64 / 256 tokens, 8 of 128 experts of 2048 x 768: 113 / 150 / 232 us on the kernels for a few rows, 99 / 126 / 148 on tiles).
  // Slots of one or two tokens, and of four among many experts, as a rule name an expert each: they are not sorted, each has a piece and the sum over them comes with down (1, 2, 4 tokens as
  // above: 24, 34, 46 us sorted, 19, 22, 37 so; 4 tokens, 2 of 16 experts of 4096 x 1536: 45, 49.  An expert that is named twice is read as often).
  const bool unsorted = T <= 4 && (T <= 2 ? P : 4 * P) <= n_experts && f8_few_rows(p) && f8_few_rows(d) && f8_runs(hidden) <= 64 && f8_token_bytes(d) <= 32 * 1024;
  const bool in_blocks = unsorted || (P <= kSortSmall && f8_in_blocks(p, T) && f8_in_blocks(d, T));
  if (!in_blocks) p.few = d.few = 1;
  const bool few = f8_few_rows(p);
  if (few) {
    p.y = ws.g;
    p.y1 = ws.u;
  } else {
    p.dt = dtype;  // (which instructions)
    p.h = ws.h.codes;
    p.hs = ws.h.scales;
  }
  if (f8_few_rows(d) || dtype == MI_MOE_DTYPE_F16) d.dt = MI_MOE_DTYPE_F32;
  else d.y_scales = ws.y_scales;
  F8Lists lists;
  lists.offsets = ws.offsets;
  lists.n_mats = n_experts;
  lists.rows = P;
  list_for(p, lists, 0, ws.list[0]);
  list_for(d, lists, 1, ws.list[1]);
  if (unsorted) {
    p.ids = d.ids = topk_idx;
    p.order = nullptr;
    p.list = d.list = nullptr;
  } else MI_HIP(launch_sort_tokens({topk_idx, T, top_k, n_experts, ws.order, ws.inverse, ws.offsets}, nullptr, dtype, hidden, nullptr, ws.sort, st, in_blocks ? lists : F8Lists()));
  if (in_blocks) {
    p.raw = x;
    p.raw_dt = dtype;
    d.raw = ws.g;
    d.raw_up = ws.u;
  } else {
    MI_HIP(launch_quantize_f8_rows(x, dtype, T, hidden, ws.x.out(T, hidden), st, lists));
  }
  MI_HIP(launch_f8_product(p, st));
  if (unsorted) {
    MI_HIP(launch_f8_token(d, topk_w, w_dtype, out, dtype, st));
    return 0;
  }
  if (few && !in_blocks) MI_HIP(launch_swiglu_f8(ws.g, ws.u, P, intermediate, ws.h.out(P, intermediate), st));
  MI_HIP(product_to_tokens(d, d.y_scales ? hidden : ExpertsWs::float_columns(P, hidden, n_experts), topk_w, w_dtype, ws.inverse, T, top_k, dtype, out, st));
  return 0;
} MI_CATCH("switch_glu_f8")

int mi_moe_switch_glu_f8_grad(const void *dout, const void *x, const uint32_t *topk_idx, const void *topk_w, int32_t w_dtype, const mi_moe_f8_experts *experts, int64_t T,
                              int32_t hidden, int32_t intermediate, int32_t n_experts, int32_t top_k, int32_t dtype, void *dx, void *dweights, void *workspace,
                              size_t workspace_bytes, void *stream) try {
  if (check_switch("switch_glu_f8_grad", experts, x, topk_idx, topk_w, w_dtype, T, hidden, intermediate, n_experts, top_k, dtype)) return 1;
  if (T == 0) return 0;
  if (!dout || !dx || !dweights) return fail("switch_glu_f8_grad: dout, dx and dweights must be non-NULL");
  const ExpertsWs ws(workspace, T, hidden, intermediate, n_experts, top_k, true);
  if (check_workspace("switch_glu_f8_grad", workspace, workspace_bytes, ws.bytes)) return 1;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t P = T * top_k;
  MI_HIP(launch_sort_tokens({topk_idx, T, top_k, n_experts, ws.order, ws.inverse, ws.offsets}, nullptr, dtype, hidden, nullptr, ws.sort, st));
  // gate, up and the gradient at h (but for the slot's weight), in float32: the weights' gradient is made of them
  F8Product p{};
  p.x = ws.x.as(T);
  p.order = ws.order;
  p.k_div = top_k;
  p.n_mats = n_experts;
  p.rows = P;
  p.list = ws.list[0];
  p.m[0] = mat(experts->gate, experts->gate_scales);
  p.m[1] = mat(experts->up, experts->up_scales);
  p.transpose = true;
  p.N = intermediate;
  p.K = hidden;
  p.y = ws.g;
  p.y1 = ws.u;
  p.dt = MI_MOE_DTYPE_F32;
  F8Product b = p;
  b.x = ws.dout.as(T);
  b.m[0] = b.m[1] = mat(experts->down, experts->down_scales);
  b.transpose = false;
  b.y = ws.dh;
  b.y1 = nullptr;
  F8Product d{};
  d.x = ws.h.as(P);
  d.n_mats = n_experts;
  d.rows = P;
  d.list = ws.list[1];
  d.m[0] = mat(experts->gate, experts->gate_scales);
  d.m[1] = mat(experts->up, experts->up_scales);
  d.pair_sum = true;
  d.N = hidden;
  d.K = intermediate;
  d.y = ws.y;
  int columns = hidden;
  if (dtype == MI_MOE_DTYPE_F16) {
    d.dt = MI_MOE_DTYPE_F32;
    if (hidden <= 3 * (int64_t)intermediate) d.y = ws.g;  // (to dh: read by then.  1000 tokens through 2 of 16 experts of 2048 x 1792: 183 us, with half of the columns at a time 231)
    else columns = ExpertsWs::float_columns(P, hidden, n_experts);
  } else {
    d.dt = dtype;
    d.y_scales = ws.y_scales;
  }
  if (P <= (int64_t)16 * n_experts) {  // (room for float32 rows, and for parts)
    b.parts = d.parts = ws.parts;
    d.list = ws.list[1];
    if (f8_plan(d).parts > 1) {
      d.dt = MI_MOE_DTYPE_F32;
      d.y_scales = nullptr;
    } else {
      d.parts = nullptr;
    }
  }
  // three lists, the forward products' beside the rounding of x, the others' beside that of dout
  F8Lists lists, back;
  lists.offsets = back.offsets = ws.offsets;
  lists.n_mats = back.n_mats = n_experts;
  lists.rows = back.rows = P;
  list_for(p, lists, 0, ws.list[0]);
  list_for(b, back, 0, ws.list[2]);
  list_for(d, back, 1, ws.list[1]);
  MI_HIP(launch_quantize_f8_rows(x, dtype, T, hidden, ws.x.out(T, hidden), st, lists));
  MI_HIP(launch_quantize_f8_rows(dout, dtype, T, hidden, ws.dout.out(T, hidden), st, back));
  MI_HIP(launch_f8_product(p, st));
  MI_HIP(launch_f8_product(b, st));
  MI_HIP(launch_swiglu_f8_grad({ws.g, ws.u, ws.dh, topk_w, w_dtype, ws.order, ws.offsets, n_experts, P, intermediate, ws.h.codes, ws.h.scales, dweights}, st));
  MI_HIP(product_to_tokens(d, columns, nullptr, 0, ws.inverse, T, top_k, dtype, dx, st));
  return 0;
} MI_CATCH("switch_glu_f8_grad")

}  // extern "C"
