// project_work.h -- how a projection's work is cut, and its workspace (host and
// device; the CPU tests compile it on its own).
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <algorithm>

namespace fdm {

constexpr int kStepBytes = 128;        // of a row of x or of the matrix that a step of the products takes
constexpr int kProjectMaxSeqs = 4096;  // FDM_PROJECT_MAX_SEQS
constexpr int kMaxAdapters = 1024;     // FDM_MAX_ADAPTERS
constexpr int kMaxRank = 128;          // FDM_MAX_RANK
constexpr int kMaxUSplits = 8;
constexpr int kRankPart = 64;          // of a rank, that a workgroup of the adapters' first product takes

// Rows of x and of the matrix in a workgroup's tile.
enum ProjectTile { kTile32, kTile64, kTile128, kTile256 };
struct TileSize {
  int rows, cols;
};
constexpr TileSize kTiles[] = {{32, 128}, {64, 128}, {128, 128}, {256, 256}};

struct ProjectPlan {
  int tile;
  int full;        // tiles that a workgroup does whole
  int splits;      // parts of the inner dimension of every other tile
  int u_splits;    // the same of the adapters' first product
};

inline int steps_of(int64_t row_bytes) { return (int)((row_bytes + kStepBytes - 1) / kStepBytes); }
inline int64_t tiles_of(int tile, int T, int out) {
  return ((int64_t)T + kTiles[tile].rows - 1) / kTiles[tile].rows * (((int64_t)out + kTiles[tile].cols - 1) / kTiles[tile].cols);
}
// Tiles of 32 rows of one adapter, at most, and parts of the rank.
inline int adapter_tiles(int T, int B, int n_adapters) { return (T + 31) / 32 + std::min(B, n_adapters); }
inline int rank_parts(int rank) { return (rank + kRankPart - 1) / kRankPart; }

// Rounds of tiles over the CUs (a workgroup has one to itself) leave some of them idle in the
// last; its tiles are cut into parts of the inner dimension where that is worth what parts
// cost, their sums being written and read again.  What a cut takes, in us, from what was
// measured over 1 to 8192 rows of 1536 to 16384 values:
//   a step of 128 bytes in a workgroup  0.3, 0.42, 0.53, 1.6 by tile; 3 a round for its two ends
//   a part                              0.015, 0.02, 0.03, 0.13; 5 for the joining launch
// (500 rows of 16384 BF16 values by 7168: tiles of 128 rows 137 us, of 256 in four parts 138;
// 1000 rows 276 and, in two parts, 238; 256 rows 79 and 93; 128 rows of 1536 by 24576 in tiles
// of 64 rows 23.7, of 128 17.2.)
// It takes tiles of 128 rows too soon where 128 to 256 rows meet few columns: 128 rows of 7168
// BF16 values by 576 and 2112 19 and 14 parts of them (at their best 15.1 and 18.0 us) where 20 and
// 7 of 64 rows take 11.9 and 15.9; 256 rows by 576 16.4 and 13.8, of codes by 2112 21.8 and 18.9;
// and leaves 1000 rows by 2112 whole, 59.7, in three parts 54.8.
constexpr double kStepUs[] = {0.3, 0.42, 0.53, 1.6}, kPartUs[] = {0.015, 0.02, 0.03, 0.13};
// Parts at most: two for every CU, one of the largest tiles (64 MB of sums).
inline int most_parts(int tile, int cus) { return tile == kTile256 ? cus : 2 * cus; }
// Tiles that are mostly rows past the end are not considered.
inline bool tile_fits(int tile, int T) { return tile == kTile32 ? T <= 32 : T > kTiles[tile].rows / 2; }

// The adapters of a call: workgroups that their first product takes at least (0: none), rank,
// how many there are, and requests.
struct ProjectU {
  int tiles, rank, n, B;
};
struct ProjectCut {
  int64_t full;
  int splits, u_splits;
  double us;
};
// The best number of splits of the adapters' first product, and what the launches up to the
// join take with it: beside the `parts` of a cut where there is room for both (a few too many
// do not matter), else before them.  Before whole tiles (parts 0) it has a launch of its own
// and one split.
// 4.5 us and, for a step of its eight waves, 0.3 and 0.035 a value of the rank: 512 rows of
// 7168 values of rank 64 43, 25, 16.4 and 12.3 in 1, 2, 4 and 8 splits, 256 rows of 16384 of
// rank 16 30.6, 18.0, 11.7 and 8.4.
inline double with_u(ProjectU u, int steps, int64_t parts, double main, int cus, int* splits) {
  *splits = 0;
  if (!u.tiles) return main;
  // two workgroups a CU at most
  const int most = parts ? std::max(std::min(2 * cus / u.tiles, std::min(kMaxUSplits, steps)), 1) : 1;
  const int64_t room = parts ? cus + cus / 20 - parts % cus : 0;
  double least = 0;
  for (int s = 1, each = 0; s <= most; ++s) {
    if ((steps + 8 * s - 1) / (8 * s) == each) continue;  // more splits, no fewer steps
    each = (steps + 8 * s - 1) / (8 * s);
    const double us = 4.5 + (double)each * (0.3 + 0.035 * std::min(u.rank, kRankPart));
    const int64_t groups = (int64_t)u.tiles * s;
    const double t = groups <= room ? std::max(us, main) + 0.1 * us : us * ((groups + cus - 1) / cus) + main;
    if (s == 1 || t < least) least = t, *splits = s;
  }
  return least;
}
inline ProjectCut project_cut(int tile, int T, int out, int steps, ProjectU u, int cus) {
  const int rows = kTiles[tile].rows;
  const int64_t tiles = tiles_of(tile, T, out), rest = tiles % cus;
  auto round = [&](int n) { return n * kStepUs[tile] + 3; };
  const double rounds = (double)(tiles / cus) * round(steps);
  // a tile's second products: 2 us, and 2 an adapter among its rows
  const double second = u.tiles ? 2 + 2 * std::min<double>(std::min(u.n, rows), 1 + (double)u.B * std::min(rows, T) / T) : 0;
  ProjectCut c{tiles, 1, 0, 0.0};
  c.us = with_u(u, steps, 0, rounds + (rest ? round(steps) : 0) + (double)((tiles + cus - 1) / cus) * second, cus, &c.u_splits);
  // (uncut tiles may be joined too, for the adapters' products in two launches of few rows)
  for (int s = u.tiles && tiles < cus ? 1 : 2; s <= steps && rest * s <= most_parts(tile, cus) && rest; ++s) {
    const double main = rounds + (double)(tiles / cus) * second + (double)((rest * s + cus - 1) / cus) * round((steps + s - 1) / s);
    const double join = rest * s * kPartUs[tile] * std::min(1.0, (double)T / rows) + 5;
    if (main + join >= c.us) continue;  // (the adapters take nothing away)
    int u_splits;
    const double us = with_u(u, steps, tiles < cus ? rest * s : 0, main, cus, &u_splits) + join;
    if (us < c.us) c = {tiles - rest, s, u_splits, us};
  }
  return c;
}
// B requests of n adapters; rank 0: none.
inline ProjectPlan project_plan(int T, int64_t row_bytes, int out, int B, int n, int rank, int cus) {
  const ProjectU u{rank ? adapter_tiles(T, B, n) * rank_parts(rank) : 0, rank, n, B};
  ProjectPlan p{};
  ProjectCut c{};
  bool any = false;
  for (int tile = kTile32; tile <= kTile256; ++tile) {
    if (!tile_fits(tile, T)) continue;
    const ProjectCut t = project_cut(tile, T, out, steps_of(row_bytes), u, cus);
    if (!any || t.us < c.us) c = t, p.tile = tile, any = true;
  }
  p.full = (int)c.full;
  p.splits = c.splits;
  p.u_splits = c.u_splits;
  return p;
}

// How the parts are joined (kJoinNone: every tile is whole).  One chunk of 256 values a workgroup, so
// that rows with adapters of their own do not wait for each other, or where there are many,
// four: 64 rows by 2112 15.4 us a call against 19.2, 24 by 24576 20.3 and 21.6, 500 by 2111
// with two adapters 75 and 60, 256 by 7168 with 32 109 and 104.5.
// Many chunks on the matrix cores instead where 16 rows have two adapters at most, or B's rows
// are more than 64 bytes, so that a row a lane takes them apart.  650 rows by 2112 of 3, 80 and
// 650 requests with adapters of their own, rank 16: 7.1, 9.5 and 25 us on the matrix cores, 7.7,
// 8.5 and 12.7 without; rank 64: 12.5, 15.7 and 46, and 15.2, 27 and 124.  (256 rows by 7168
// with 32 adapters of rank 64 in turn are slower, 79 and 64.)
enum ProjectJoin { kJoinNone, kJoinOne, kJoinFour, kJoinRows };
inline int join_chunks(int tile, int T) { return (std::min(kTiles[tile].rows, T) * kTiles[tile].cols + 255) / 256; }
inline ProjectJoin project_join(const ProjectPlan& p, int T, int out, int B, int rank, int cus) {
  const int64_t rest = tiles_of(p.tile, T, out) - p.full;
  if (!rest) return kJoinNone;
  if (rest * join_chunks(p.tile, T) <= 16 * cus) return kJoinOne;
  return rank && (rank > 32 || (int64_t)16 * B <= T) ? kJoinRows : kJoinFour;
}

// fp32 values of the parts [splits][tiles][rows][cols] and of the adapters' first product
// [u_splits][T][rank]
inline size_t project_part_floats(const ProjectPlan& p, int T, int out) {
  return (size_t)p.splits * (tiles_of(p.tile, T, out) - p.full) * kTiles[p.tile].rows * kTiles[p.tile].cols;
}
inline size_t project_u_floats(const ProjectPlan& p, int T, int rank) { return (size_t)p.u_splits * T * rank; }
inline size_t project_bytes(const ProjectPlan& p, int T, int out, int rank) {
  return (project_u_floats(p, T, rank) * 4 + 255) / 256 * 256 + project_part_floats(p, T, out) * 4;
}

// What any call of up to T rows needs, whatever its format and its requests.
inline size_t project_most_bytes(int T, int in, int out, int rank, int cus) {
  size_t most = 0;
  for (int tile = kTile32; tile <= kTile256; ++tile) {
    const int rows = tile == kTile32 ? std::min(T, 32) : T;
    if (tile != kTile32 && !tile_fits(tile, T)) continue;
    const int64_t parts = std::min<int64_t>(most_parts(tile, cus), tiles_of(tile, rows, out) * steps_of((int64_t)in * 2));
    most = std::max(most, (size_t)parts * kTiles[tile].rows * kTiles[tile].cols * 4);
  }
  // (the splits of u are as many as leave two workgroups a CU, and there is one for 32 rows)
  const int64_t u_rows = std::max<int64_t>(T, std::min<int64_t>((int64_t)kMaxUSplits * T, (int64_t)64 * cus));
  return std::max<size_t>(((size_t)u_rows * rank * 4 + 255) / 256 * 256 + most, 256);
}

}  // namespace fdm
