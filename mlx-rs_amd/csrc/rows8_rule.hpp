// Which kernel a linear layer on 8-bit rows takes: arithmetic alone, for host and device code.
#pragma once
#include <cstdint>

namespace mi_moe {

// rows x columns of a block
enum class Rows8Kind {
  kFew16x16, kFew16x32, kFew32x16, kFew32x32, kFew64x32,  // nothing prepared, eight waves share K (qmm_rows8.hip)
  kTiles64x64, kTiles64x128, kTiles128x128,    // prepared rows (qmm_rows8_tiles.hip)
};
struct Rows8Cost {
  int rows, cols;
  bool tiles;
  // us = start + first K / 4096 + (x - 1) (more K / 4096 + more0), x: blocks of the fullest XCD a CU, at least one
  float start, first, more, more0;
};
// Fitted to 110 products (16 to 2048 rows, 1024 to 14336 columns, K = 1024, 2048 and 4096; groups of 64 with 4- and 8-bit codes, of 32 and 128 with 4-bit ones): what the rule takes is 0.5 %
// slower than the fastest kind on average, 22 % at most.  The times, us, 4-bit, groups of 64, K = 4096, in the order of the kinds:
//   16 x 4096     6.2, 7.6, 6.8, 8.6, 12.2
//   16 x 14336    16.3, 12.9, 18.9, 16.2, 23.6
//   32 x 4096     9.4, 7.9, 8.3, 10.2, 13.3, 19.8, 29.9, 39.5
//   64 x 4096     16.4, 12.6, 13.3, 10.5, 16.8, 20.6, 30.2, 41.8
//   64 x 14336    47.0, 35.2, 38.4, 34.6, 31.4, 22.3, 31.6, 43.6
//   128 x 4096    28.2, 21.4, 23.0, 18.2, 17.4, 21.3, 30.9, 42.3
//   256 x 4096    52.7, 38.4, 42.0, 33.5, 31.2, 23.1, 32.3, 43.4
//   512 x 4096    101, 73.0, 80.2, 64.1, 57.0, 31.8, 35.6, 46.2
//   1024 x 4096   198, 143, 157, 127, 111, 54.8, 48.6, 49.6
//   2048 x 4096   393, 281, 309, 250, 217, 106, 88.6, 79.5
constexpr Rows8Cost kRows8Costs[] = {
    {16, 16, false, 3.8f, 2.9f, 3.0f, 0.5f},   {16, 32, false, 4.1f, 4.7f, 4.0f, 1.3f},    {32, 16, false, 3.7f, 4.2f, 4.5f, 0.8f},   {32, 32, false, 4.6f, 6.0f, 6.6f, 2.4f},
    {64, 32, false, 4.6f, 10.4f, 12.3f, 3.0f},
    {64, 64, true, 8.7f, 14.5f, 10.3f, 1.7f},  {64, 128, true, 8.5f, 27.5f, 15.0f, 2.0f},  {128, 128, true, 10.5f, 43.0f, 28.0f, 2.0f},
};
constexpr float rows8_time(const Rows8Cost &c, int64_t M, int N, int K) {
  const int64_t tall = (M + c.rows - 1) / c.rows, wide = ((int64_t)N + c.cols - 1) / c.cols;
  const float blocks = c.tiles ? 8.f * (float)((wide + 7) / 8 * tall) : (float)(wide * tall), k = (float)K / 4096.f;
  const float x = blocks > 256.f ? blocks / 256.f : 1.f;
  return c.start + c.first * k + (x - 1.f) * (c.more * k + c.more0);
}
constexpr int kRows8Dot = 2;       // rows that take no matrix instructions at all
constexpr int kRows8NoTiles = 16;   // rows that no number of columns brings to the tiles
// tiles: there is a workspace, and the columns' scales start where copies can
constexpr Rows8Kind rows8_kind(int64_t M, int N, int K, bool tiles) {
  int best = 0;
  for (int i = 1; i < 8; ++i)
    if (((tiles && M > kRows8NoTiles) || !kRows8Costs[i].tiles) && rows8_time(kRows8Costs[i], M, N, K) < rows8_time(kRows8Costs[best], M, N, K)) best = i;
  return static_cast<Rows8Kind>(best);
}

// A launch has less than 2^32 threads: blocks of 512 for every kind, and waves of the rows' preparation, in blocks of 256, that take 16 rows and four groups each.
constexpr int64_t kRows8Blocks = ((int64_t)1 << 23) - 1, kRows8Units = ((int64_t)1 << 25) - 1;
constexpr int rows8_quads(int G) { return (G + 7) / 8 * 2; }  // fours of groups, in whole eights
constexpr int64_t rows8_blocks(Rows8Kind kind, int64_t M, int N) {
  const Rows8Cost &c = kRows8Costs[(int)kind];
  const int64_t tall = (M + c.rows - 1) / c.rows, wide = ((int64_t)N + c.cols - 1) / c.cols;
  return tall * (c.tiles ? (wide + 7) / 8 * 8 : wide);
}
// rows of a launch, in whole blocks; 0: one block of rows already has too many columns
constexpr int64_t rows8_step(Rows8Kind kind, int N, int K, int group) {
  const Rows8Cost &c = kRows8Costs[(int)kind];
  const int64_t rows = kRows8Blocks / rows8_blocks(kind, 1, N) * c.rows, prepared = kRows8Units / rows8_quads(K / group) * 16 / c.rows * c.rows;
  return c.tiles && prepared < rows ? prepared : rows;
}

}  // namespace mi_moe
