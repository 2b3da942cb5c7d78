// mla_work.h -- how the latent attention's work is counted and cut (host and
// device; the CPU tests compile it on its own).
//
// The (token, head) rows of a sequence, heads fastest, are cut into tiles of R.
// A tile has a step for every S positions that its last token may see (one at
// least, so that rows that see nothing are written) and counts kTileCost units
// more, what beginning and ending it costs a workgroup (queries, first steps,
// results: about 12 us against 2 us a step; 64 sequences of one token over 4095
// FP8 positions 94.5 us without, 90.9 with four, 86.3 with six).  The units of all tiles
// in order (sequence, tile, unit) are cut into equal ranges, one a workgroup.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fdm {

#define FDM_HD __host__ __device__ __forceinline__

constexpr int kMlaMaxSeqs = 512;  // FDM_MLA_MAX_SEQS
constexpr int kTileRows = 128;    // (token, head) rows of a workgroup
constexpr int kTilePos = 32;      // positions of a step
constexpr int kTileCost = 6;
// A call's units are below 2^40 (the host refuses calls whose tables could make
// them more); starts that pass it all the same (sequences that share tokens) are cut.
constexpr uint64_t kMaxUnits = (1ull << 40) - 1;

struct SeqWork {
  int n, len, t0;  // tokens, positions, first token
};

template <int R>
FDM_HD int tiles_of(const SeqWork& s, int H) { return (s.n * H + R - 1) / R; }
template <int R, int S>
FDM_HD int tile_steps(const SeqWork& s, int tile, int H, bool in_order) {
  const int upto = (R * (tile + 1) - 1) / H + 1;  // tokens up to the tile's last
  const int last = upto < s.n ? upto : s.n;
  const int64_t seen = in_order ? (int64_t)s.len - s.n + last : s.len;
  const int steps = (int)((seen + S - 1) / S);
  return steps > 1 ? steps : 1;
}
template <int R, int S>
FDM_HD int tile_units(const SeqWork& s, int tile, int H, bool in_order) {
  return tile_steps<R, S>(s, tile, H, in_order) + kTileCost;
}
// ceil(1 / 2^k) + .. + ceil(x / 2^k)
FDM_HD int64_t step_sum(int64_t x, int k) {
  const int64_t q = x >> k, r = x & ((1 << k) - 1);
  return ((q * (q + 1) / 2) << k) + r * (q + 1);
}
// sum over i < n of floor((a i + b) / m), the lattice points under a line, by the
// known reduction along Euclid's algorithm: whole parts of a and b are taken out, and
// the points under what is left of the line are counted along the other axis.
FDM_HD uint64_t floor_sum(uint64_t n, uint64_t m, uint64_t a, uint64_t b) {
  uint64_t sum = 0;
  for (;;) {
    sum += n * (n - 1) / 2 * (a / m) + n * (b / m);
    a %= m;
    b %= m;
    const uint64_t end = a * n + b;
    if (end < m) return sum;
    n = end / m;
    b = end % m;
    const uint64_t t = m;
    m = a;
    a = t;
  }
}
// units of the sequence's tiles 0 .. tiles - 1
template <int R, int S>
FDM_HD int64_t units_before(const SeqWork& s, int tiles, int H, bool in_order) {
  if (!in_order || s.n <= 1) return (int64_t)tiles * tile_units<R, S>(s, 0, H, in_order);
  int64_t sum = 0;
  // ceil((before + last) / S) each, before the positions in front of the tokens
  // and last the tile's last token (from 1): k (i + 1) with k = R / H whole tokens a
  // tile, else floor((R (i + 1) - 1) / H) + 1; the sequence's last tile may have fewer
  // than R rows.  Tokens before the first position (before < 0): the tiles that see
  // nothing, those of the first -before H rows, have one step.
  const int64_t before = (int64_t)s.len - s.n;
  const int whole = tiles == tiles_of<R>(s, H) ? tiles - 1 : tiles, k = R / H;
  if (whole < tiles) sum = s.len > S ? ((int64_t)s.len + S - 1) / S : 1;
  if (whole > 0) {
    if (before >= 0 && R % H == 0 && S % k == 0) {  // with before in whole k, rounded up, ceil((before / k + i) / (S / k))
      const int kb = __builtin_ctz(k), per = __builtin_ctz(S) - kb;
      const int64_t p = (before + k - 1) >> kb;
      sum += step_sum(p + whole, per) - step_sum(p, per);
    } else {
      const int dark = before < 0 ? (int)(-before * H) / R : 0, none = dark < whole ? dark : whole;
      sum += none;
      if (none < whole)
        sum += (int64_t)floor_sum(whole - none, (uint64_t)H * S, R, (uint64_t)(R - 1 + (int64_t)R * none + H * (before + S)));
    }
  }
  return sum + (int64_t)tiles * kTileCost;
}

// The most units that a call can have whose tables cover max_len positions of a sequence.
FDM_HD uint64_t most_units(int N, int H, int B, int max_len) {
  const uint64_t tiles = ((uint64_t)N * H + kTileRows - 1) / kTileRows + B;
  return tiles * (((uint64_t)max_len + kTilePos - 1) / kTilePos + 1 + kTileCost);
}

// The units before each sequence, 40 bits each (LDS is short).
struct UnitMarks {
  uint32_t lo[kMlaMaxSeqs + 1];
  uint8_t hi[kMlaMaxSeqs + 1];
  FDM_HD void put(int b, uint64_t u) { lo[b] = (uint32_t)u, hi[b] = (uint8_t)(u >> 32); }
  FDM_HD uint64_t at(int b) const { return (uint64_t)hi[b] << 32 | lo[b]; }
};

// T units in G ranges, at most 256: range g is [g T / G, (g + 1) T / G), with T =
// q G + r as g q + g r / G.  The quotient in two divisions of 32 bits: the ones of
// 64 bits are long subroutines, 3 % of 64 sequences of one token.
struct Ranges {
  uint64_t q, total;
  uint32_t r, groups;
  FDM_HD Ranges(uint64_t total, uint32_t groups) : total(total), groups(groups) {
    const uint32_t high = (uint32_t)(total >> 16), qh = high / groups;
    const uint32_t low = (high - qh * groups) << 16 | (uint32_t)(total & 0xFFFF), ql = low / groups;
    q = ((uint64_t)qh << 16) + ql;
    r = low - ql * groups;
  }
  FDM_HD uint64_t start(uint32_t g) const { return g * q + g * r / groups; }
  // the range that has unit u: about u G / T, and the neighbours looked at
  FDM_HD int at(uint64_t u) const {
    uint32_t g = (uint32_t)((float)u * ((float)groups / (float)total));
    if (g >= groups) g = groups - 1;
    while (start(g) > u) --g;
    while (start(g + 1) <= u) ++g;
    return (int)g;
  }
};

}  // namespace fdm
