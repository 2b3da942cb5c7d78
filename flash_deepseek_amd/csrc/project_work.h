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

// Rows of x and of the matrix in a workgroup's tile.
enum ProjectTile { kTile32, kTile64, kTile128, kTile256 };
struct TileSize {
  int rows, cols;
};
constexpr TileSize kTiles[] = {{32, 128}, {64, 128}, {128, 128}, {256, 256}};

struct ProjectPlan {
  int tile;
  int splits;      // parts of the inner dimension, each with its own fp32 part
  int u_splits;    // the same of the adapters' first product
  bool join;       // parts (and the adapters' second product) are added by a launch of their own
};

inline int steps_of(int64_t row_bytes) { return (int)((row_bytes + kStepBytes - 1) / kStepBytes); }

inline ProjectPlan project_plan(int T, int64_t row_bytes, int out, bool adapters, int cus) {
  ProjectPlan p{};
  auto tiles = [&](int t) { return ((int64_t)T + kTiles[t].rows - 1) / kTiles[t].rows * ((out + kTiles[t].cols - 1) / kTiles[t].cols); };
  p.tile = T <= 32 ? kTile32 : T <= 64 ? kTile64 : kTile128;
  if (T > 128 && tiles(kTile256) * 4 >= cus * 3) p.tile = kTile256;
  const int steps = steps_of(row_bytes);
  p.splits = 1;
  const int64_t n = tiles(p.tile);
  if (n < cus) p.splits = (int)std::max<int64_t>(std::min<int64_t>(cus / n, (steps + 3) / 4), 1);
  // few rows: the adapters' first product runs beside the matrix's, and a joining launch has the second
  p.join = p.splits > 1 || (adapters && T <= 64);
  p.u_splits = p.join ? std::min(8, std::max(1, steps / 8)) : 1;
  return p;
}

// fp32 values of the parts [splits][T][out] and of the adapters' first product [u_splits][T][rank]
inline size_t project_part_floats(const ProjectPlan& p, int T, int out) { return p.join ? (size_t)p.splits * T * out : 0; }
inline size_t project_u_floats(const ProjectPlan& p, int T, int rank) { return (size_t)p.u_splits * T * rank; }
inline size_t project_bytes(const ProjectPlan& p, int T, int out, int rank) {
  return (project_u_floats(p, T, rank) * 4 + 255) / 256 * 256 + project_part_floats(p, T, out) * 4;
}
// What any call of up to T rows needs.  The cut is the same from one multiple of 128 rows
// to the next but for the tiles of 32 and 64, and from 128 x the CUs on nothing is cut.
inline size_t project_most_bytes(int T, int in, int out, int rank, int cus) {
  size_t most = 256;
  auto see = [&](int t) {
    for (int size : {1, 2})
      for (int r : {0, rank})
        most = std::max(most, project_bytes(project_plan(t, (int64_t)in * size, out, r > 0, cus), t, out, r));
  };
  see(std::min(T, 32));
  see(std::min(T, 64));
  for (int64_t t = 128; t < T && t <= (int64_t)128 * cus; t += 128) see((int)t);
  see(T);
  return most;
}

}  // namespace fdm
