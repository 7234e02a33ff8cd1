// Which kernel a product with e4m3 weights takes, and in which pieces: arithmetic alone, for host and device code.
#pragma once
#include <cstddef>
#include <cstdint>

namespace mi_moe {

constexpr int kF8Run = 128;
constexpr int f8_runs(int n) { return (n + kF8Run - 1) / kF8Run; }
constexpr int64_t f8_row_bytes(int k) { return (int64_t)f8_runs(k) * kF8Run; }  // of a row of codes in a workspace: whole runs, zeros behind the last value
constexpr int kF8TileN = 256;  // columns of a tile

// What the rules go by.
struct F8Sizes {
  int64_t rows;
  int N, K;
  int n_mats;      // 1 for one matrix
  bool by_matrix;  // rows by matrix, in listed pieces or a piece each
  bool pieces;     // (listed ones)
  bool transpose;  // matrices [N][K]
  bool pair;       // gate and up, into h
  bool pair_sum;   // two halves of the summed axis
  bool exact;      // sums on the bf16 instructions
  bool parts;      // there is room for parts
  int few;         // F8Product
};

// Rows of a piece: what the product's kernel takes at once (16 or 32: the one for a few rows).
inline int f8_tile_rows(const F8Sizes &p) {
  const int64_t mats = p.n_mats, avg = p.rows / mats;
  // One matrix: 4096 x 4096, 16 / 32 / 48 / 64 rows in pieces of 32 take 10 / 12 / 16 / 17 us.  By expert, this kernel / tiles, us: 128 matrices of 768 x 2048 at 2, 4, 6, 16 rows each
  // 34 / 40, 39 / 41, 49 / 41, 62 / 43; 16 of 1792 x 2048, whose tiles are half as many as the CUs, at 4, 8, 12, 16 rows 18 / 20, 21 / 21, 22 / 22, 24 / 22.
  const int64_t tiles = (p.N + (p.pair ? 127 : 255)) / (p.pair ? 128 : 256) * mats;
  const int64_t few = !p.by_matrix ? 48 : p.few ? p.few : tiles >= 256 ? 4 : 12;
  if (p.transpose && !p.pair && !p.pair_sum && p.rows <= few * mats) return avg > 4 ? 32 : 16;
  // Tiles of 64 / 128 rows to float32, us: 16 matrices of 1792 x 2048 at 56, 72, 100, 160 rows each 29 / 31, 31 / 37, 45 / 39, 51 / 42; 128 of 768 x 2048 72 / 77, 94 / 87, 127 / 99,
  // 171 / 142.  To bfloat16, of 64 / 128 / 256 rows: the 128 at 40, 72, 100, 128, 200 rows 50 / 51 / 53, 81 / 63 / 67, 105 / 73 / 79, 117 / 96 / 90, 168 / 133 / 107; the 16, which have
  // fewer tiles than there are CUs, at 56, 100, 200, 260 rows 24 / 24 / 26, 41 / 26 / 29, 48 / 32 / 41, 54 / 50 / 43.
  if (p.exact) return avg > 64 ? 128 : 64;
  return avg > (tiles >= 256 ? 112 : 208) ? 256 : avg > 48 ? 128 : 64;
}

// Parts are made where tiles of 64 x 256 and more are fewer than the chip's CUs: kF8MostParts of a product at most, 256 tiles of all of them, two stages or more each.  A join costs by the parts' values
// and saves by the stages: beyond 2^11 values for each value of the summed axis it does not pay.
constexpr int kF8MostParts = 16;
constexpr int f8_stages(int K, bool pair_sum) { return f8_runs(K) * (pair_sum ? 2 : 1); }
constexpr int64_t f8_most_parts_values(int stages) {
  const int64_t most = (int64_t)stages * kF8Run << 11, tiles = (int64_t)256 * 256 * 256;
  return stages < 4 ? 0 : most < tiles ? most : tiles;
}
// the most rows of which parts are made, and room for them; with more rows never less
constexpr int64_t f8_parts_rows(int N, int stages) { return f8_most_parts_values(stages) / (2 * (int64_t)N); }
inline size_t f8_parts_bytes(int64_t M, int N, int stages) {
  const int64_t all = M * N * kF8MostParts, most = f8_most_parts_values(stages);
  return (size_t)(all < most ? all : most) * 4;
}
struct F8Plan {
  int tile, parts;
};
// How many blocks share a tile's summed axis where the tiles alone leave CUs idle, and for one matrix the tile, by the time they take.  Us, measured: a launch 6; a stage 0.65 with a few
// blocks and 1.1 with one on every CU (64 token rows), 1.0 and 1.45 (128), 1.7 and 2.2 (256); a join of parts 3, their bytes out and back 2.5 MB each.
// By expert weights come from memory and not out of L2: a stage with a block on every CU 1.6 (64 token rows), a join 5.
inline F8Plan f8_plan_of(const F8Sizes &p, int tile, int64_t tiles, F8Plan best, double &least) {
  const int steps = f8_stages(p.K, p.pair_sum);
  for (int parts = 1; parts <= (p.parts ? kF8MostParts : 1); parts *= 2) {
    if (parts > 1 && (steps < 2 * parts || tiles * parts > 256 || (int64_t)parts * p.rows * p.N > f8_most_parts_values(steps))) break;
    const double full = (double)(tiles * parts < 256 ? tiles * parts : 256) / 256, few = tile == 64 ? 0.65 : tile == 128 ? 1.0 : 1.7;
    const double t = (double)((tiles * parts + 255) / 256) * ((steps + parts - 1) / parts) * (few + (p.pieces ? 0.95 : 0.45) * full) + (parts > 1 ? (p.pieces ? 5.0 : 3.0) + (double)parts * p.rows * p.N * 8 / 2.5e6 : 0.0);
    if (t < least) least = t, best = {tile, parts};
  }
  return best;
}
inline F8Plan f8_plan(const F8Sizes &p) {
  F8Plan best{64, 1};
  double least = 1e30;
  const int64_t columns = (p.N + kF8TileN - 1) / kF8TileN;
  if (p.pieces) {  // (as many pieces as there are matrices with rows, if each has a few)
    best.tile = f8_tile_rows(p);
    return p.parts ? f8_plan_of(p, best.tile, (p.rows / best.tile + (p.n_mats < p.rows ? p.n_mats : p.rows)) * columns, best, least) : best;
  }
  for (int tile = 64; tile <= 256; tile *= 2)
    if (tile != 256 || !p.exact) best = f8_plan_of(p, tile, (p.rows + tile - 1) / tile * columns, best, least);
  return best;
}

}  // namespace mi_moe
