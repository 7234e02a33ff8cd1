// Which kernel a linear layer on 8-bit rows takes: arithmetic alone, for host and device code.
#pragma once
#include <cstdint>

namespace mi_moe {

// rows x columns of a block
enum class Rows8Kind {
  kFew16x16, kFew32x16, kFew32x32, kFew64x32,  // nothing prepared, eight waves share K (qmm_rows8.hip)
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
//   16 x 4096     8.4, 9.0, 12.4, 14.6                      64 x 14336    76, 53, 47, 37, 22.3, 31.6, 43.6
//   32 x 4096     13.8, 10.6, 14.1, 16.4, 19.8, 30, 40      256 x 4096    87, 59, 46, 36.6, 23.1, 32.3, 43
//   64 x 4096     24.4, 17.6, 14.5, 19.3, 20.6, 30, 42      512 x 4096    170, 115, 87, 68, 31.8, 35.6, 46.3
//   128 x 4096    45.4, 31.6, 25.4, 19.9, 21.3, 31, 42      1024 x 4096   337, 226, 171, 134, 54.8, 48.6, 49.6
//   16 x 14336    25.0, 27.2, 23.0, 28.1                    2048 x 4096   671, 447, 338, 264, 106, 88.6, 79.5
constexpr Rows8Cost kRows8Costs[] = {
    {16, 16, false, 3.3f, 5.1f, 6.2f, 0.1f},   {32, 16, false, 3.4f, 6.6f, 7.0f, 0.3f},    {32, 32, false, 3.5f, 10.5f, 11.5f, 1.5f}, {64, 32, false, 4.1f, 15.2f, 15.0f, 2.6f},
    {64, 64, true, 8.7f, 14.5f, 10.3f, 1.7f},  {64, 128, true, 8.5f, 27.5f, 15.0f, 2.0f},  {128, 128, true, 10.5f, 43.0f, 28.0f, 2.0f},
};
constexpr float rows8_time(const Rows8Cost &c, int64_t M, int N, int K) {
  const int64_t tall = (M + c.rows - 1) / c.rows, wide = (N + c.cols - 1) / c.cols;
  const float blocks = c.tiles ? 8.f * (float)((wide + 7) / 8 * tall) : (float)(wide * tall), k = (float)K / 4096.f;
  const float x = blocks > 256.f ? blocks / 256.f : 1.f;
  return c.start + c.first * k + (x - 1.f) * (c.more * k + c.more0);
}
constexpr int kRows8Dot = 4;       // rows that take no matrix instructions at all
constexpr int kRows8NoTiles = 16;   // rows that no number of columns brings to the tiles
// tiles: there is a workspace, and the columns' scales start where copies can
constexpr Rows8Kind rows8_kind(int64_t M, int N, int K, bool tiles) {
  int best = 0;
  for (int i = 1; i < 7; ++i)
    if (((tiles && M > kRows8NoTiles) || !kRows8Costs[i].tiles) && rows8_time(kRows8Costs[i], M, N, K) < rows8_time(kRows8Costs[best], M, N, K)) best = i;
  return static_cast<Rows8Kind>(best);
}

}  // namespace mi_moe
