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
// cost, their sums being written and read again.
//   us a step of 128 bytes in a workgroup: 1.7 of the largest tiles, 0.8 of the others
//   us a part: 0.1 (256 KB) and 0.03; 8 us for the joining launch
// u_tiles: workgroups that the adapters' first product takes at least, 0: no adapters.
inline ProjectPlan project_plan(int T, int64_t row_bytes, int out, int u_tiles, int cus) {
  ProjectPlan p{};
  const int steps = steps_of(row_bytes);
  p.tile = T <= 32 ? kTile32 : T <= 64 ? kTile64 : kTile128;
  if (T > 128 && tiles_of(kTile256, T, out) * 4 >= cus * 3) p.tile = kTile256;
  const int64_t tiles = tiles_of(p.tile, T, out), rest = tiles % cus;
  const double step = p.tile == kTile256 ? 1.7 : 0.8, part = p.tile == kTile256 ? 0.1 : 0.03;
  p.full = (int)(tiles - rest);
  p.splits = 1;
  // few rows: the adapters' first product runs beside the matrix's, the joining launch has the second
  const bool join = u_tiles && T <= 64;
  double least = step * steps + (join ? rest * part : 0);
  for (int s = 2; s <= steps && rest * s <= 2 * cus; ++s) {
    const double t = (double)((rest * s + cus - 1) / cus) * ((steps + s - 1) / s) * step + rest * s * part + (join ? 0 : 8);
    if (t < least) least = t, p.splits = s;
  }
  if (p.splits == 1 && !join) p.full = (int)tiles;
  // what it takes to fill the CUs: twice by itself, and what the parts leave beside them
  const int64_t room = p.full ? 2 * cus : cus - rest * p.splits;
  p.u_splits = u_tiles ? (int)std::min<int64_t>(std::max<int64_t>(room / u_tiles, 1), std::min(kMaxUSplits, steps)) : 0;
  return p;
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
  auto see = [&](int t) {
    for (int size : {1, 2})
      for (int u_tiles : {0, rank ? 1 : 0})
        most = std::max(most, project_part_floats(project_plan(t, (int64_t)in * size, out, u_tiles, cus), t, out) * 4);
  };
  see(std::min(T, 32));
  see(std::min(T, 64));
  // the cut is the same from one multiple of 128 rows to the next
  for (int64_t t = 128; t < T; t += 128) see((int)t);
  see(T);
  return std::max<size_t>(((size_t)kMaxUSplits * T * rank * 4 + 255) / 256 * 256 + most, 256);
}

}  // namespace fdm
