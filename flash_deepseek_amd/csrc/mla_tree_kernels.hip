// mla_tree_kernels.hip -- latent attention of several sequences' query tokens
// over the paged cache (fdm_mla_attend).
//   s_ij = scale (q_lat_i . c_j + q_rope_i . r_j) over the positions j that
//   token i sees, p = softmax(s), o_i = sum_j p_ij c_j, lse_i = log sum exp.
// Position j of a sequence of len positions with n tokens is seen if it
// stands before the tokens (j < len - n), or if bit j - (len - n) of the
// token's mask is set; without a mask, if it does not stand behind token i's
// own place len - n + i.
//
// The heads of a token share its sequence's rows, so (token, head) pairs are
// the rows of two matrix products with the cached rows, 1088 products a pair
// and position: 242 flops a byte of a BF16 cache with 128 heads, about what
// separates the matrix cores from HBM.  A workgroup takes 128 such rows (one
// token of 128 heads, eight of 16), four waves that each have a SIMD and its 512
// registers to themselves: 256 of them hold 64 rows x 256 of the result's dims,
// 144 the queries of 32 rows, so that of each step of 32 positions only the cached
// rows move, once into LDS and from there as either product's operand.
// The bound is what a single wave issues around its products (a step takes 4150
// cycles, 2176 of them products) and, as soon as that is better, the power: the
// clock falls from 2.4 to 1.9 GHz.  512 tokens of 128 heads over 4608 positions
// 560 to 580 us with the card, 1.07 to 1.1 PFLOP/s, where a library product of
// 8192^3 reaches 1.21.
#include "latent_device.h"
#include "mla_work.h"

namespace fdm {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kLatBytes = kTilePos * kLatDim * 2, kRotBytes = kTilePos * kRotDim * 2;
constexpr int kPBytes = kTileRows * kTilePos * 2;
// LDS: four steps' latent rows (one's values, one's keys, one landed, one landing),
// three steps' rotary parts, the weights of two steps
constexpr int kRotAt = 4 * kLatBytes, kPAt = kRotAt + 3 * kRotBytes, kStepLds = kPAt + 2 * kPBytes;
constexpr size_t kPartFloats = (size_t)kTileRows * kLatDim;
constexpr int kMaxGroups = 256;  // workgroups that share the work
// Weights are 2^(s - m), s in log2.  A row's m is kAbove under its maximum when it is
// moved, which is when the maximum grew by more than kGrow since: a weight is at
// most 2^(kAbove + kGrow).  That uses F16's numbers above 1: rounded to it, a weight
// is off by 2^-32 of the row's largest at most, where with m the maximum itself
// weights of 2^-25 were none, and 32768 of them 9e-4 of the values.  BF16 reaches as
// far down as the fp32 sums.
constexpr float kGrow = 8.0f;
template <int FMT>
constexpr float kAbove = FMT == kKvF16 ? 7.0f : 0.0f;

// A tile that several workgroups share is put together from their parts; the
// workgroup that has its first part says so.
struct JoinDesc {
  int t0, tile, parts, rows;  // its sequence's first token; rows of the tile
};

// workspace: JoinDesc [groups], row statistics [2 groups][128] (max, sum),
// parts [2 groups][128][512]
struct Space {
  JoinDesc* desc;
  float2* stat;
  float* part;
};
__host__ __device__ size_t space_stat_at(int groups) { return ((size_t)groups * sizeof(JoinDesc) + 255) / 256 * 256; }
__host__ __device__ size_t space_part_at(int groups) { return space_stat_at(groups) + (size_t)2 * groups * kTileRows * sizeof(float2); }
__device__ Space space_of(void* p, int groups) {
  char* c = static_cast<char*>(p);
  return {reinterpret_cast<JoinDesc*>(c), reinterpret_cast<float2*>(c + space_stat_at(groups)),
          reinterpret_cast<float*>(c + space_part_at(groups))};
}

template <int FMT>
struct Half {
  typedef std::conditional_t<FMT == kKvF16, _Float16, __bf16> T;
  typedef std::conditional_t<FMT == kKvF16, f16x4, bf16x4> x4;
  typedef std::conditional_t<FMT == kKvF16, f16x8, bf16x8> x8;
};
// The matrix products in assembly: the 256 accumulation registers hold the
// output all along and the scores' sums are in VGPRs, which the compiler does
// not do by itself (it moves the output between the two files in every turn,
// and spills).  It knows nothing of a product in assembly and inserts no waits
// for one, so the source sees to them:
//  - an operand that an ALU instruction wrote needs two states before the
//    product: every operand here was loaded, from LDS or memory;
//  - a result needs 12 states before an ALU instruction reads it (what this
//    compiler keeps behind its own such products on gfx950): products_done()
//    stands before such reads;
//  - products that add to one sum need none between them.
#define FDM_MFMA_OF(FMT, form, ...)                               \
  if constexpr (FMT == kKvF16) {                                  \
    asm("v_mfma_f32_32x32x16_f16 " form : __VA_ARGS__); \
  } else {                                                        \
    asm("v_mfma_f32_32x32x16_bf16 " form : __VA_ARGS__); \
  }
template <int FMT, bool FIRST>
__device__ __forceinline__ void mfma_score(f32x16& c, i32x4 a, i32x4 b) {
  if constexpr (FIRST) {
    FDM_MFMA_OF(FMT, "%0, %1, %2, 0", "=&v"(c) : "v"(a), "v"(b))
  } else {
    FDM_MFMA_OF(FMT, "%0, %1, %2, %0", "+v"(c) : "v"(a), "v"(b))
  }
}
template <int FMT>
__device__ __forceinline__ void mfma_out(f32x16& o, i32x4 a, i32x4 b) {
  FDM_MFMA_OF(FMT, "%0, %1, %2, %0", "+a"(o) : "v"(a), "v"(b))
}
#undef FDM_MFMA_OF
// Between the two files, one register at a time, so that no sum is ever a
// tuple of VGPRs to the compiler.
__device__ __forceinline__ float acc_get(float a) {
  float v;
  asm("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(a));
  return v;
}
__device__ __forceinline__ float acc_put(float v) {
  float a;
  asm("v_accvgpr_write_b32 %0, %1" : "=a"(a) : "v"(v));
  return a;
}
__device__ __forceinline__ float acc_zero() {
  float a;
  asm volatile("v_accvgpr_write_b32 %0, 0" : "=a"(a));  // one each, not copies of one
  return a;
}
// Before an ALU instruction reads what products have written, the compiler's
// own copies where control flow meets among them.
__device__ __forceinline__ void products_done() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 11" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
#define FDM_LDS __attribute__((address_space(3)))
// 16 bytes a lane from memory straight into LDS: lane i's land at `to` + 16 i.
// In assembly, because the compiler lets no LDS read start while a direct load
// that it knows of is in flight, whichever part of LDS that fills; there is no
// result register, and landed() waits for these loads.  With a scalar base
// that v_readlane wrote, five states must lie between that and this.
__device__ __forceinline__ void lds_load16(const char* from, char* to) {
  const int at = (int)(uintptr_t)(FDM_LDS char*)to;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(from) : "memory");
}
__device__ __forceinline__ void lds_load16(uint64_t base, int off, char* to) {
  const int at = (int)(uintptr_t)(FDM_LDS char*)to;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(off), "s"(base) : "memory");
}
// Two rows of a base's next four: the loads' offset moves both of their ends.
template <int ROW>
__device__ __forceinline__ void lds_load_rows(uint64_t base, int off0, int off1, char* to) {
  const int at = (int)(uintptr_t)(FDM_LDS char*)to;
  asm volatile(
      "s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3 offset:%4\n\t"
      "global_load_lds_dwordx4 %2, %3 offset:%5" ::"s"(at), "v"(off0), "v"(off1), "s"(base), "n"(ROW * 1024), "n"(ROW * 1024 + 1024)
      : "memory");
}
// four rows x 16 columns of 16-bit values, lane i of 16 pointing at four
// columns of row i / 4: lane i gets column i of the four rows
__device__ __forceinline__ f16x4 read_turned(const char* p, f16x4) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((FDM_LDS s16x4*)p));
}
__device__ __forceinline__ bf16x4 read_turned(const char* p, bf16x4) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((FDM_LDS bf16x4*)p);
}

// the row's place of its 16-byte piece g is g ^ row_swap(row): 16 rows' same
// piece lie in 16 bank groups, and four rows' same four pieces in four
__device__ __forceinline__ int row_swap(int row) { return ((row & 3) << 2) | ((row >> 2) & 3); }

// a value that is the same in every lane, in scalar registers
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return (int64_t)(((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32) | (uint32_t)uniform((int)v));
}

// A value that the compiler computes where it stands: it would otherwise
// keep dozens of addresses that differ by constants over the whole loop.
__device__ __forceinline__ int here(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// A condition whose code stands out of the way: a taken branch costs a wave
// that has its SIMD alone some 60 cycles.
__device__ __forceinline__ bool rare(bool v) { return __builtin_expect(v, 0); }

// f with the constants 0 .. N - 1
template <typename F, int... I>
__device__ __forceinline__ void unrolled(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void unrolled(F f) {
  unrolled(f, std::make_integer_sequence<int, N>{});
}

// the value of lane ^ 32, combined
template <typename F>
__device__ __forceinline__ float across_halves(float v, F f) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return f(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

__device__ __attribute__((aligned(16))) uint32_t zero_row[8 * kLatDim * 2 / 4];  // stands for eight rows that are none

}  // namespace

// ---- the work: tiles of rows, steps of positions (mla_work.h) ---------------------------
__device__ __forceinline__ SeqWork seq_work(const MlaTreeArgs& a, int b) {
  SeqWork s;
  s.t0 = min(max(a.q_start[b], 0), a.N);
  s.n = max(min(a.q_start[b + 1], a.N) - s.t0, 0);
  s.len = min(max(a.kv_len[b], 0), a.max_len);
  return s;
}
// The last tile that starts at or before unit u of the sequence; every lane of a
// wave looks at one of 64 at a time.
template <int R, int S>
__device__ __forceinline__ int tile_at(const SeqWork& s, int64_t u, int H, bool in_order) {
  int lo = 0, n = tiles_of<R>(s, H);  // it is among lo .. lo + n - 1
  while (n > 1) {
    const int every = (n + 63) / 64, at = (int)(threadIdx.x & 63) * every;
    const bool starts = at < n && units_before<R, S>(s, lo + at, H, in_order) <= u;
    const int last = 63 - __builtin_clzll(__ballot(starts) | 1);
    lo += last * every;
    n = min(every, n - last * every);
  }
  return uniform(lo);
}

// Units before each sequence into before[0 .. B], two sequences a thread of 256.
// U: of 32 bits unless the call can have more.
template <int R, int S, typename U>
__device__ __forceinline__ void count_units(const MlaTreeArgs& a, UnitMarks& before, uint64_t* wave_total) {
  constexpr U kMost = sizeof(U) == 8 ? (U)kMaxUnits : (U)0x7FFFFFFF;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool in_order = a.mask == nullptr;
  U mine[2], sum = 0;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    mine[k] = sum;
    const int b = 2 * tid + k;
    if (b < a.B) {
      const SeqWork s = seq_work(a, b);
      sum = (U)min((uint64_t)sum + (uint64_t)units_before<R, S>(s, tiles_of<R>(s, a.H), a.H, in_order), (uint64_t)kMost);
    }
  }
  U upto = sum;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const U v = __shfl_up(upto, d);
    if (lane >= d) upto = min(upto + v, kMost);
  }
  if (lane == 63) wave_total[wave] = upto;
  const U inside = __shfl_up(upto, 1);
  __syncthreads();
  U base = 0;
  for (int w = 0; w < wave; ++w) base = min(base + (U)wave_total[w], kMost);
  base = min(base + (lane ? inside : 0), kMost);
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (2 * tid + k <= a.B) before.put(2 * tid + k, min(base + mine[k], kMost));
  if (tid == 255 && a.B == kMlaMaxSeqs) before.put(kMlaMaxSeqs, min(base + sum, kMost));
  __syncthreads();
}
__device__ __forceinline__ uint64_t units_at(const UnitMarks& before, int b) { return uniform((int64_t)before.at(b)); }

// A workgroup's range of units, and the part of a tile that it is at.
struct Range {
  uint64_t u, end;      // next unit, end
  int group;            // number of the range
  int b, tile;          // sequence and tile of the part (tile -1: to be looked for)
  int from, to;         // steps of the part; it ends before unit u
  SeqWork s;
};
// A range that is cut out of a tile costs a part, 256 KB written and read again,
// so few units are not spread over all workgroups: U units over G take 2 U / G us
// of steps and about 0.13 G us of parts, least at G = sqrt(15 U); but no fewer than
// there are tiles, and two units at least.  One token of 128 heads over 1024
// positions in ranges of two 20.3 us, of one 21.4; over 32768 in ranges of eight 47,
// of four 60; eight sequences of one token over 4096 44 and 52.
__device__ __forceinline__ uint32_t range_count(const MlaTreeArgs& a, uint64_t total) {
  const uint32_t tiles = (uint32_t)(((int64_t)a.N * a.H + kTileRows - 1) / kTileRows) + a.B;  // at most
  const uint32_t few = max((uint32_t)__builtin_amdgcn_sqrtf(15.0f * (float)total), tiles);
  return (uint32_t)uniform((int)min((uint64_t)min((uint32_t)gridDim.x, few), total / 2));
}
__device__ __forceinline__ Range range_of(const MlaTreeArgs& a, const UnitMarks& before) {
  Range r;
  const uint64_t total = units_at(before, a.B);
  const uint32_t groups = range_count(a, total);
  // Neighbours in the list on one XCD (workgroups go round the eight in turn),
  // where they share rows; fewer ranges than workgroups are spread over all.
  const bool full = groups == gridDim.x && gridDim.x % 8 == 0;
  r.group = full ? (blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8 : blockIdx.x;
  r.u = r.end = 0;
  r.b = 0;
  r.tile = -1;
  if ((uint32_t)r.group >= groups) return r;
  const Ranges ranges(total, groups);
  r.u = uniform((int64_t)ranges.start(r.group));
  r.end = uniform((int64_t)ranges.start(r.group + 1));
  int hi = a.B - 1;  // the last sequence that starts at or before u
  while (r.b < hi) {
    const int mid = (r.b + hi + 1) / 2;
    if (units_at(before, mid) <= r.u) r.b = mid;
    else hi = mid - 1;
  }
  return r;
}
// The next part that has steps; false at the end of the range.
template <int R, int S>
__device__ __forceinline__ bool next_part(const MlaTreeArgs& a, const UnitMarks& before, Range& r) {
  const bool in_order = a.mask == nullptr;
  while (r.u < r.end) {
    while (units_at(before, r.b + 1) <= r.u) ++r.b, r.tile = -1;
    const int64_t seq_u = units_at(before, r.b);
    int64_t start = r.u;  // the tile behind the one before starts here
    if (r.tile >= 0) {
      ++r.tile;
    } else {
      r.s = seq_work(a, r.b);
      r.s = {uniform(r.s.n), uniform(r.s.len), uniform(r.s.t0)};
      r.tile = (int64_t)r.u == seq_u ? 0 : tile_at<R, S>(r.s, r.u - seq_u, a.H, in_order);
      start = uniform(seq_u + units_before<R, S>(r.s, r.tile, a.H, in_order));
    }
    const int64_t tile_u = start + kTileCost;  // its first step
    r.from = (int)max((int64_t)r.u - tile_u, (int64_t)0);
    r.to = (int)min((int64_t)tile_steps<R, S>(r.s, r.tile, a.H, in_order), (int64_t)r.end - tile_u);
    if (r.to <= 0) break;  // the range ends before the tile's first step
    r.u = tile_u + r.to;
    if (r.to > r.from) return true;
  }
  return false;
}
// Workgroups that have steps of the part's tile of so many steps.
__device__ __forceinline__ int parts_of(const MlaTreeArgs& a, const UnitMarks& before, const Range& r, int steps) {
  const uint64_t total = units_at(before, a.B), first = r.u - r.to;
  const Ranges ranges(total, range_count(a, total));
  return ranges.at(first + steps - 1) - ranges.at(first) + 1;
}

// Which of the positions j0 .. j0 + 31 the sequence's token `place` sees (bits).
__device__ __forceinline__ uint32_t sees(const MlaTreeArgs& a, const SeqWork& s, int place, int64_t j0) {
  const int64_t d0 = j0 - (s.len - s.n);  // the token place of the first position
  uint32_t see = d0 >= 0 ? 0u : d0 <= -32 ? ~0u : (1u << -d0) - 1;
  if (d0 > -32) {
    if (!a.mask) {
      const int64_t last = place - d0;  // of the 32
      see = last >= 31 ? ~0u : last < 0 ? see : (see | ((2u << last) - 1));
    } else {
      // bits d0 .. d0 + 31 of the mask
      const uint64_t* mask = a.mask + (size_t)(s.t0 + place) * a.mask_words;
      const int64_t at = d0 >= 0 ? d0 : 0;
      const int64_t w = at >> 6;
      uint64_t bits = w < a.mask_words ? mask[w] >> (at & 63) : 0;
      if ((at & 63) && w + 1 < a.mask_words) bits |= mask[w + 1] << (64 - (at & 63));
      see |= d0 >= 0 ? (uint32_t)bits : (uint32_t)bits << -d0;
    }
    // positions behind the sequence's end
    const int64_t in = s.len - j0;
    see &= in >= 32 ? ~0u : in <= 0 ? 0u : (1u << in) - 1;
  }
  return see;
}

template <int FMT, bool WHOLE>
__global__ __launch_bounds__(256, 1) void k_mla_tree(MlaTreeArgs a) {
  typedef typename Half<FMT>::T T;
  typedef typename Half<FMT>::x4 x4;
  typedef typename Half<FMT>::x8 x8;
  __shared__ __attribute__((aligned(256))) char lds[kStepLds];
  __shared__ float scale_by[2][kTileRows];   // what the rows' sums so far are scaled by
  __shared__ int moved[2][4];                // the step at which a wave's rows last were
  __shared__ int live[4];                    // bytes: which rows of a step exist
  __shared__ UnitMarks before;               // units before each sequence
  __shared__ uint64_t wave_total[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, h = lane >> 5;

  if (a.wide_units) count_units<kTileRows, kTilePos, uint64_t>(a, before, wave_total);
  else count_units<kTileRows, kTilePos, uint32_t>(a, before, wave_total);
  Range range = range_of(a, before);
  const int group = range.group;
  const Space space = space_of(a.workspace, gridDim.x);
  if (tid == 0) space.desc[group] = {0, 0, 0, 0};  // unless it begins a tile that others go on with

  while (next_part<kTileRows, kTilePos>(a, before, range)) {
    const SeqWork s = range.s;
    const int from = range.from, to = range.to, len = s.len;
    const int row0 = kTileRows * range.tile, rows = min(kTileRows, s.n * a.H - row0);
    // from this step on not all of the tile's tokens see all positions
    const int first_edge = max(len - s.n + (a.mask ? 0 : row0 / a.H + 1), 0) / kTilePos;

    // The lane's scores are those of row 32 wave + l32.  What is needed of it is
    // computed where it is needed: registers are short in the loop.
    auto token_of = [&](int r) { return (row0 + min(r, rows - 1)) / a.H; };
    // ---- a step's rows into LDS: wave w brings rows 8 w .. 8 w + 7, in kBring
    // pieces of work.  16-bit rows go straight into LDS.  FP8 codes go into
    // registers, eight lanes a row, and from there in the same turn as 16-bit
    // values (exact) into LDS.  A row that is none reads zeros.
    // WHOLE: a wave's eight rows lie in one page (pages of 8 and more).  Where
    // they are is known to all its lanes, and a piece is two rows; positions behind
    // the sequence's end are read as they are, and hidden.  Otherwise a lane
    // looks after the row that it is one of eight of, and a piece is one row: 85
    // instructions more a step, 81 us against 77 for 128 sequences of three tokens
    // of 16 heads over 2048 positions, 577 against 562 for 512 tokens of 128 over 4608.
    constexpr bool kCodes = FMT == kKvFp8;
    constexpr int kBring = kCodes || WHOLE ? 8 : 12;
    const int my_row = 8 * wave + (lane >> 3);
    const int* pages = a.pages + (size_t)range.b * a.pages_stride;
    const char* none = reinterpret_cast<const char*>(zero_row);
    int page;                // of the next step to be placed (this lane's row)
    int slot = 0;            // the step placed last: this lane's row (WHOLE: the wave's first); -1: none
    const char* mine;        // 16 bits: that row
    uint64_t base;           //   the row that the next piece brings
    u32x4 code[4];           // FP8: that row's codes (16 of each group) and scales
    uint32_t code_scale = 0;
    auto page_of = [&](int step) {
      return pages[min(step * kTilePos + (WHOLE ? 8 * wave : my_row), max(len - 1, 0)) >> a.page_shift];
    };
    auto place = [&](int step) {
      const int j = step * kTilePos + (WHOLE ? 8 * wave : my_row);
      const int at = WHOLE ? uniform(page) : page;
      const bool is = (unsigned)at < (unsigned)a.n_pages & j < len & step < to;
      slot = is ? (at << a.page_shift) + (j & ((1 << a.page_shift) - 1)) : -1;
    };
    auto announce = [&](int step, int rot_at) {  // which rows exist, and their rotary parts
      const int swap = 16 * ((lane & 7) ^ ((my_row >> 1) & 7));
      if constexpr (WHOLE) {
        reinterpret_cast<uint8_t*>(&live[step & 3])[wave] = (uint8_t)(slot >= 0 ? 0xFF : 0);
        const char* rp = slot >= 0 ? static_cast<const char*>(a.rope) + (size_t)slot * (kRotDim * 2) : none;
        lds_load16((uint64_t)rp, here((lane >> 3) * (kRotDim * 2) + swap), lds + rot_at + wave * 1024);
      } else {
        const uint64_t all = __ballot(slot >= 0);
        uint32_t byte = 0xFF;
        if (all != ~0ull) {
          byte = 0;
#pragma unroll
          for (int k = 0; k < 8; ++k) byte |= (uint32_t)((all >> (8 * k)) & 1) << k;
        }
        reinterpret_cast<uint8_t*>(&live[step & 3])[wave] = (uint8_t)byte;
        const char* rp = static_cast<const char*>(a.rope) + (size_t)max(slot, 0) * (kRotDim * 2) + here(swap);
        lds_load16(slot >= 0 ? rp : none, lds + rot_at + wave * 1024);
      }
    };
    auto base_of = [&](int k) {
      return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uintptr_t)mine, 8 * k) |
             (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)((uintptr_t)mine >> 32), 8 * k) << 32;
    };
    auto load_scales = [&] {
      const char* sc = slot >= 0 ? reinterpret_cast<const char*>(a.scale) + (size_t)slot * 4 : none;
      code_scale = *reinterpret_cast<const uint32_t*>(WHOLE ? sc + (uint32_t)here((lane >> 3) * 4) : sc);
    };
    auto load_codes = [&](int k) {
      const char* p = slot >= 0 ? static_cast<const char*>(a.latent) + (size_t)slot * kLatDim : none;
      const int at = here(WHOLE ? (lane >> 3) * kLatDim + 16 * (lane & 7) : 16 * (lane & 7));
      code[k] = *reinterpret_cast<const u32x4*>(p + (uint32_t)at + 128 * k);
    };
    auto widen = [&](int step, int piece) {  // in eight pieces
      if constexpr (kCodes) {
        const int k = piece >> 1, half = piece & 1;
        const int at = here((step & 3) * kLatBytes + my_row * 1024 + (((2 * (lane & 7)) ^ row_swap(my_row)) << 4));
        const float sc = scale_value((int)((code_scale >> (8 * k)) & 0xFF));
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          v[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(code[k][2 * half + i], sc, false));
          v[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(code[k][2 * half + i], sc, true));
        }
        *reinterpret_cast<u32x4*>(lds + (at ^ (16 * half)) + 256 * k) = v;
      }
    };
    auto bring = [&](int step, auto piece, int rot_at) {
      constexpr int P = decltype(piece)::value;
      if constexpr (P == 0) {
        place(step);
      } else if constexpr (P == 1) {
        page = page_of(step + 1);
      } else if constexpr (P == 2) {
        announce(step, rot_at);
      } else if constexpr (P == 3 && kCodes) {
        load_scales();
      } else if constexpr (P == 3) {
        const char* at = slot >= 0 ? static_cast<const char*>(a.latent) + (size_t)slot * (kLatDim * 2) : none;
        if constexpr (WHOLE) base = (uint64_t)at;
        else mine = at, base = base_of(0);
      } else if constexpr (kCodes) {
        load_codes(P - 4);
      } else {
        constexpr int K = WHOLE ? 2 * P - 8 : P - 4;  // first row
        const int swap = here((lane ^ ((2 * wave) & 3)) << 4) ^ ((K >> 2) << 4);
        char* to = lds + (step & 3) * kLatBytes + (8 * wave + (WHOLE ? K & 4 : K)) * 1024;
        if constexpr (WHOLE) {
          lds_load_rows<(K & 3)>(base, swap ^ ((K & 3) << 6), swap ^ (((K + 1) & 3) << 6), to);
          if (K == 2) base += 4 * kLatDim * 2;
        } else {
          lds_load16(base, swap ^ ((K & 3) << 6), to);
          if (K < 7) base = base_of(K + 1);
        }
      }
    };

    // ---- the products
    f32x16 o[8][2];  // [32 dims][32 rows]: dims 256 (wave & 1) + 32 i, rows 64 (wave >> 1) + 32 k
    x8 q[36];        // the queries of the lane's row: the products' B operand
    float m = -__builtin_inff(), l = 0.0f;
    const int rh = wave >> 1, dh = wave & 1;
    const bool works = 64 * rh < rows;  // otherwise the wave only brings

    // Operands come out of LDS kAhead reads before the product that wants them:
    // 36 of keys (position = l32, 8 dims at 16 k + 8 h), then 16 of values (dim =
    // l32 of a block of 32; positions 16 s + 4 h + {0 .. 3, 8 .. 11}, the ones
    // whose weights the lane has).
    constexpr int kKeys = 36, kVals = 16, kAhead = 4;
    static_assert(kKeys % kAhead == 0, "keys and values take the registers in turn");
    i32x4 f[kAhead];
    int key_at, rot_at, v0_at, v1_at;  // this lane's addresses
    auto key_place = [&](int step, int rot) {
      key_at = here((step & 3) * kLatBytes + l32 * 1024 + ((row_swap(l32) ^ h) << 4));
      rot_at = here(rot + l32 * 128 + ((((l32 >> 1) & 7) ^ h) << 4));
    };
    auto val_place = [&](int step) {
      const int i16 = lane & 15, u4 = 2 * ((lane >> 4) & 1) + ((i16 >> 1) & 1);
      v0_at = here((step & 3) * kLatBytes + (4 * h + (i16 >> 2)) * 1024 + (((i16 >> 2) << 6) | ((u4 ^ h) << 4)) +
                   8 * (i16 & 1) + 512 * dh);
      v1_at = here((v0_at + 8 * 1024) ^ 32);
    };
    auto fetch_key = [&](int k) {
      f[k % kAhead] = k < 32 ? *reinterpret_cast<const i32x4*>(lds + (key_at ^ ((k & 7) << 5)) + (k >> 3) * 256)
                             : *reinterpret_cast<const i32x4*>(lds + (rot_at ^ ((k & 3) << 5)));
    };
    auto fetch_val = [&](int i, int place) {  // block i & 7 of 32 dims, positions 16 (i >> 3) ..
      const int off = (i >> 3) * 16384 + ((i >> 2) & 1) * 256;
      const x4 lo = read_turned(lds + (v0_at ^ ((i & 3) << 6)) + off, x4{});
      const x4 hi = read_turned(lds + (v1_at ^ ((i & 3) << 6)) + off, x4{});
      const u32x2 x = __builtin_bit_cast(u32x2, lo), y = __builtin_bit_cast(u32x2, hi);
      f[place % kAhead] = i32x4{(int)x[0], (int)x[1], (int)y[0], (int)y[1]};
    };
    i32x4 w[2][2];  // the weights of step j - 1: [16 positions][32 rows]
    auto fetch_weights = [&](int step, int s) {
      const int at = here((step & 1) * kPBytes + 2 * rh * 1024 + lane * 16);
#pragma unroll
      for (int i = 0; i < 2; ++i) w[s][i] = *reinterpret_cast<const i32x4*>(lds + kPAt + at + s * 4096 + i * 1024);
    };
    f32x16 c;  // scores of 32 positions x this wave's 32 rows: D row = position, column = query row
    auto key_product = [&](int k) {
      const i32x4 b = __builtin_bit_cast(i32x4, q[k]);
      if (k == 0) mfma_score<FMT, true>(c, f[0], b);
      else mfma_score<FMT, false>(c, f[k % kAhead], b);
    };
    auto val_product = [&](int i, int place, int k) { mfma_out<FMT>(o[i & 7][k], f[place % kAhead], w[i >> 3][k]); };

    // The step's weights from its scores, in kWeigh pieces.  A wave issues in
    // order and has its SIMD alone, so a piece is what is issued while one product
    // is worked on, and nothing stands next to what it needs: one piece has a
    // pair's exponents, one the sum and rounding of the pair before and the
    // products of the pair after the next.  Weights round to the cache's 16-bit type,
    // the only one that the second product takes beside its values (in two 16-bit
    // halves they would double its 32 of a step's 68 matrix instructions); their sum is
    // that of the unrounded ones, in fp32.
    constexpr int kWeigh = 23;
    float top = 0.0f, off = 0.0f;
    auto hide = [&](uint32_t see) {
      const uint32_t mine = see >> (4 * h);
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (!((mine >> (8 * (e >> 2) + (e & 3))) & 1)) c[e] = -__builtin_inff();
    };
    i32x4 p8[2];
    auto weigh = [&](int step, int piece) {
      if (piece == 0) {
        float t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = fmaxf(c[i], c[4 + i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = fmaxf(fmaxf(t[i], c[8 + i]), c[12 + i]);
        top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
      } else if (piece == 1) {
        // s - m rounded as a weight's is, so that none passes its limit however coarse s is
        top = across_halves(top, [](float x, float y) { return fmaxf(x, y); });
        const bool need = fmaf(top, a.scale_log2, -m) > kGrow + kAbove<FMT>;
        if (rare(__any(need))) {
          const float to_m = fmaf(top, a.scale_log2, -kAbove<FMT>);
          const float keep = need ? __builtin_amdgcn_exp2f(m - to_m) : 1.0f;
          m = need ? to_m : m;
          l *= keep;
          scale_by[step & 1][here(32 * wave + l32)] = keep;  // both halves of the wave have it
          moved[step & 1][wave] = step;
        }
        off = m == -__builtin_inff() ? 0.0f : m;
      }
      auto scaled = [&](int i) {
        c[2 * i] = fmaf(c[2 * i], a.scale_log2, -off);
        c[2 * i + 1] = fmaf(c[2 * i + 1], a.scale_log2, -off);
      };
      if (piece == 3) scaled(0), scaled(1);
      const int p = (piece - 4) >> 1;  // a pair
      if (piece >= 4 && piece % 2 == 0 && p < 8) {
        c[2 * p] = __builtin_amdgcn_exp2f(c[2 * p]);
        c[2 * p + 1] = __builtin_amdgcn_exp2f(c[2 * p + 1]);
      }
      if (piece >= 5 && piece % 2 == 1) {
        if (p + 2 < 8) scaled(p + 2);
        if (p >= 1 && p < 9) {
          const int i = p - 1;
          typedef T x2 __attribute__((ext_vector_type(2)));
          p8[i >> 2][i & 3] = __builtin_bit_cast(int, x2{(T)c[2 * i], (T)c[2 * i + 1]});
          l += c[2 * i] + c[2 * i + 1];
        }
      }
      if (piece == 14 || piece == 22)
        *reinterpret_cast<i32x4*>(lds + kPAt + (step & 1) * kPBytes + here((wave * 64 + lane) * 16) + (piece == 22) * 4096) =
            p8[piece == 22];
    };
    // the rows' sums so far follow a moved maximum
    auto follow = [&](int step, int mv0, int mv1) {
      products_done();
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float f = (k ? mv1 : mv0) == step ? scale_by[step & 1][64 * rh + 32 * k + l32] : 1.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
          for (int e = 0; e < 16; ++e) o[i][k][e] = acc_put(acc_get(o[i][k][e]) * f);
          __builtin_amdgcn_sched_barrier(0);  // 16 of them in VGPRs at a time
        }
      }
    };
    // values that are no numbers count for the tokens that see them through
    // their score; a weight of 0 must not meet them
    auto clean = [&](int step) {
      char* at = lds + (step & 3) * kLatBytes + 8 * wave * 1024 + 16 * lane;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        x8 v = *reinterpret_cast<x8*>(at + r * 1024);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (!(__builtin_fabsf((float)v[e]) < __builtin_inff())) v[e] = (T)0.0f;
        *reinterpret_cast<x8*>(at + r * 1024) = v;
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // In one turn step j's keys and then step j - 1's values are multiplied.
    // Step j + 1 is in LDS already, so its first keys are requested before the
    // turn ends, and the barrier stands among the keys' products: behind it the
    // weights of step j - 1 are whole, step j + 2 may be brought where step j - 2
    // was, and what was brought in the turn before has landed.  Beside the values
    // step j's weights are computed.  The order of issue is the source's: behind
    // each product about as much of that work as is issued in its 32 cycles.
    // A step takes some 4150 cycles for 2176 of products, at 1.9 to 2.1 GHz: with
    // fewer cycles (4270 before the work was cut so finely) the clock falls.
    constexpr int kBarrier = 6;             // after so many of the keys' products
    constexpr int kClear = kBarrier + 14;   // marks of moved maxima read by then, values not yet
    constexpr int kApart = 3;               // products between two pieces of what is brought
    constexpr int kBesideKeys = 8;          // so many pieces, the others beside the values
    static_assert(kBarrier + 2 + (kBesideKeys - 1) * kApart < kKeys, "the pieces have a place beside the keys");
    int rot_now = kRotAt, rot_next = kRotAt + kRotBytes, rot_then = kRotAt + 2 * kRotBytes;
    auto landed = [&] {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __syncthreads();
    };
    auto edge = [&](int j) { return j >= first_edge; };
    int mv0 = -1, mv1 = -1;
    auto moves = [&](int j) {
      mv0 = moved[j & 1][2 * rh];
      mv1 = moved[j & 1][2 * rh + 1];
    };
    auto clear_of = [&](int j) {  // step j's values and the sums made ready for its weights
      mv0 = uniform(mv0);
      mv1 = uniform(mv1);
      if (rare(edge(j) | (mv0 == j) | (mv1 == j))) {
        if (edge(j)) {
          clean(j);
          __syncthreads();
        }
        if ((mv0 == j || mv1 == j) && j > from) follow(j, mv0, mv1);  // the first step's sums are zeros
      }
    };
    auto apart = [&] {  // v_readlane's scalar and the load that it is the address of
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_nop 4" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    };
    auto next_rot = [&] {
      const int r = rot_now;
      rot_now = rot_next;
      rot_next = rot_then;
      rot_then = r;
    };
    auto turn = [&](int j, auto with_values) {
      constexpr bool VALUES = decltype(with_values)::value;
      const int exists = live[j & 3];
      unrolled<kKeys>([&](auto at) {
        constexpr int k = decltype(at)::value;
        key_product(k);
        if (k + kAhead < kKeys) fetch_key(k + kAhead);
        else if (VALUES) fetch_val(k + kAhead - kKeys, k + kAhead);
        if (k == kBarrier - 1) {
          landed();
          if (VALUES) moves(j - 1);
        }
        if (VALUES && k == kClear) clear_of(j - 1);
        if (VALUES && k == kClear + 1) val_place(j - 1);
        if (VALUES && k == kKeys - 4) fetch_weights(j - 1, 0);
        constexpr int from_barrier = k - kBarrier - 2;
        if constexpr (from_barrier >= 0 && from_barrier % kApart == 0 && from_barrier / kApart < kBesideKeys)
          bring(j + 2, std::integral_constant<int, from_barrier / kApart>{}, rot_then);
        __builtin_amdgcn_sched_barrier(0);
      });
      uint32_t see = (uint32_t)uniform(exists);
      if (rare(edge(j))) see &= sees(a, s, token_of(here(32 * wave + l32)), (int64_t)j * kTilePos);
      if constexpr (VALUES) val_product(0, kKeys, 0), val_product(0, kKeys, 1);
      products_done();
      if (rare(__any(see != ~0u))) hide(see);
      key_place(j + 1, rot_next);
      if constexpr (VALUES) {
        unrolled<kVals>([&](auto at) {
          constexpr int i = decltype(at)::value;
          if (i) val_product(i, kKeys + i, 0);
          weigh(j, 2 * i);
          if (i >= kVals - 4) widen(j + 2, 2 * (i - (kVals - 4)));
          __builtin_amdgcn_sched_barrier(0);
          if (i) val_product(i, kKeys + i, 1);
          if (i + kAhead < kVals) fetch_val(i + kAhead, kKeys + i + kAhead);
          else fetch_key((kKeys + i) % kAhead);  // the register that this product has left
          if (i == 4) fetch_weights(j - 1, 1);
          weigh(j, 2 * i + 1);
          if (i >= kVals - 4) widen(j + 2, 2 * (i - (kVals - 4)) + 1);
          if constexpr (i % 4 == 1 && kBesideKeys + i / 4 < kBring)
            bring(j + 2, std::integral_constant<int, kBesideKeys + i / 4>{}, rot_then);
          __builtin_amdgcn_sched_barrier(0);
        });
        static_assert(kWeigh <= 2 * kVals, "all pieces have a place");
      } else {
#pragma unroll
        for (int i = 0; i < kWeigh; ++i) weigh(j, i);
#pragma unroll
        for (int i = 0; i < 8; ++i) widen(j + 2, i);
        unrolled<kBring - kBesideKeys>([&](auto i) {
          bring(j + 2, std::integral_constant<int, kBesideKeys + decltype(i)::value>{}, rot_then);
          apart();
        });
#pragma unroll
        for (int k = 0; k < kAhead; ++k) fetch_key(k);
      }
      next_rot();
    };
    page = page_of(from);
    __syncthreads();  // the tile before has left LDS
    if (tid < 8) moved[tid >> 2][tid & 3] = -1;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      unrolled<kBring>([&](auto k) {
        bring(from + t, k, t ? rot_next : rot_now);
        if constexpr (!kCodes) apart();
      });
#pragma unroll
      for (int k = 0; k < 8; ++k) widen(from + t, k);
    }
    // the queries are requested behind the first rows, which take longer
    {
      const int tok = token_of(32 * wave + l32), head = row0 + min(32 * wave + l32, rows - 1) - tok * a.H;
      const T* ql = static_cast<const T*>(a.q_lat) + (int64_t)(s.t0 + tok) * a.ql_token + head * a.ql_head + 8 * h;
      const T* qr = static_cast<const T*>(a.q_rope) + (int64_t)(s.t0 + tok) * a.qr_token + head * a.qr_head + 8 * h;
#pragma unroll
      for (int k = 0; k < 32; ++k) q[k] = *reinterpret_cast<const x8*>(ql + 16 * k);
#pragma unroll
      for (int k = 0; k < 4; ++k) q[32 + k] = *reinterpret_cast<const x8*>(qr + 16 * k);
    }
    if (works) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[i][k][e] = acc_zero();
    }
    landed();
    if (works) {
      key_place(from, rot_now);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) fetch_key(k);
      turn(from, std::false_type{});
#pragma nounroll
      for (int j = from + 1; j < to; ++j) turn(j, std::true_type{});
      landed();
      moves(to - 1);
      clear_of(to - 1);
      val_place(to - 1);
      fetch_weights(to - 1, 0);
      fetch_weights(to - 1, 1);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) fetch_val(i, i);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kVals; ++i) {
        val_product(i, i, 0), val_product(i, i, 1);
        if (i + kAhead < kVals) fetch_val(i + kAhead, i + kAhead);
        __builtin_amdgcn_sched_barrier(0);
      }
      products_done();

      // ---- the tile's results, or a part of them
      l = across_halves(l, [](float x, float y) { return x + y; });
      __syncthreads();
      float* stat = reinterpret_cast<float*>(lds + kPAt);  // [128] m, [128] sum
      if (lane < 32) {
        stat[32 * wave + l32] = m;
        stat[kTileRows + 32 * wave + l32] = l;
      }
      __syncthreads();
      const int steps = tile_steps<kTileRows, kTilePos>(s, range.tile, a.H, a.mask == nullptr);
      if (from == 0 && to == steps) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int r = 64 * rh + 32 * k + l32;
          if (r < rows) {
            const int t = (row0 + r) / a.H, hd = row0 + r - t * a.H;
            const float sum = stat[kTileRows + r], inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            T* out = static_cast<T*>(a.out) + (int64_t)(s.t0 + t) * a.out_token + hd * a.out_head + 256 * dh + 8 * h;
            // The lane has dims 4 h .. of every eight; with what lane ^ 32 has, the
            // eight of one block of two, stored at once: a prompt of 2048 tokens 682 us,
            // 807 with 8-byte stores, 738 with whole rows put together in LDS.
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
              for (int e = 0; e < 4; e += 2) {
                x4 u, v;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                  u[c] = (T)(acc_get(o[i][k][4 * e + c]) * inv);
                  v[c] = (T)(acc_get(o[i][k][4 * e + 4 + c]) * inv);
                }
                const u32x2 x = __builtin_bit_cast(u32x2, u), y = __builtin_bit_cast(u32x2, v);
                const uint32_t x0 = x[0], x1 = x[1], y0 = y[0], y1 = y[1];
                const auto lo = __builtin_amdgcn_permlane32_swap(x0, y0, false, false);
                const auto hi = __builtin_amdgcn_permlane32_swap(x1, y1, false, false);
                *reinterpret_cast<u32x4*>(out + 32 * i + 8 * e) = u32x4{(uint32_t)lo[0], (uint32_t)hi[0], (uint32_t)lo[1], (uint32_t)hi[1]};
                __builtin_amdgcn_sched_barrier(0);
              }
          }
        }
        const int r = here(32 * wave + l32);
        if (a.lse && lane < 32 && r < rows) {
          const int tok = token_of(r);
          a.lse[(size_t)(s.t0 + tok) * a.H + row0 + r - tok * a.H] =
              l == 0.0f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
        }
      } else {
        // the range's first tile may have begun in the workgroup before; its last goes on in the next
        const int part = 2 * group + (from == 0 ? 1 : 0);
        if (from == 0 && tid == 0) space.desc[group] = {s.t0, range.tile, parts_of(a, before, range, steps), rows};
        if (tid < kTileRows) space.stat[(size_t)part * kTileRows + tid] = make_float2(stat[tid], stat[kTileRows + tid]);
        f32x4* to_part = reinterpret_cast<f32x4*>(space.part + (size_t)part * kPartFloats) + (2 * rh * 16 + 8 * dh) * 256 + lane;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (64 * rh + 32 * k >= rows) break;
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              to_part[(k * 16 + i) * 256 + e * 64] =
                  f32x4{acc_get(o[i][k][4 * e]), acc_get(o[i][k][4 * e + 1]), acc_get(o[i][k][4 * e + 2]),
                        acc_get(o[i][k][4 * e + 3])};
              __builtin_amdgcn_sched_barrier(0);
            }
        }
      }
    } else {  // the same barriers
#pragma nounroll
      for (int j = from; j <= to; ++j) {
        landed();
        if (j > from && edge(j - 1)) {
          clean(j - 1);
          __syncthreads();
        }
        if (j == to) break;
        unrolled<kBring>([&](auto k) {
          bring(j + 2, k, rot_then);
          apart();
        });
#pragma unroll
        for (int k = 0; k < 8; ++k) widen(j + 2, k);
        next_rot();
      }
      __syncthreads();  // and those of the results
      __syncthreads();
    }
  }
}

// A tile's parts put together: M = max m (not the maximum, but near it), out = sum 2^(m - M) part / sum 2^(m - M) l.
// Workgroup (x, y): of the x-th tile that has parts, 32 rows and I blocks of 32
// dims; 256 threads of four dims each, S times over for every S-th part.  A thread
// reads its row's statistics itself, twice, from the caches, and requests the first
// parts before them.  Few tiles of many parts are bound by latency (I = 1, S = 4:
// one token over 1024 positions, 16 parts, 4.6 us; I = 8, S = 1 would have 8
// workgroups there), many of few by memory (I = 8, S = 1: 64 sequences of one token
// over 4095 positions, 82 MB of parts, 17.5 us; blocks of four at a time 1 % more of
// the whole).
template <int FMT, int R, int S, int I>
__global__ __launch_bounds__(256 * S) void k_mla_tree_join(MlaTreeArgs a, int groups) {
  typedef typename Half<FMT>::T T;
  typedef typename Half<FMT>::x4 x4;
  constexpr int kFlight = S > 1 ? 8 : 4;  // parts requested at a time
  __shared__ int first[4];                // tiles that begin in the groups before a wave's 64
  __shared__ int owner;
  __shared__ JoinDesc found;
  __shared__ float4 red[S > 1 ? S - 1 : 1][256];
  __shared__ float red_l[S > 1 ? S - 1 : 1][32];
  __shared__ float red_top[S][32];
  const Space space = space_of(a.workspace, groups);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // the x-th group that has the first part of a tile
  if (tid == 0) owner = -1;
  const JoinDesc mine = space.desc[min(tid, groups - 1)];
  const uint64_t has = __ballot(tid < groups && mine.parts != 0);
  if (wave < 4 && lane == 0) first[wave] = __popcll(has);
  __syncthreads();
  if (wave < 4) {
    int before = 0;
    for (int w = 0; w < wave; ++w) before += first[w];
    if (((has >> lane) & 1) && before + __popcll(has & ((1ull << lane) - 1)) == (int)blockIdx.x) {
      owner = tid;
      found = mine;
    }
  }
  __syncthreads();
  const int group = owner;
  if (group < 0) return;
  const int parts = min(found.parts, groups - group), rows = found.rows, tile0 = R * found.tile, t0 = found.t0;
  constexpr int kBlocks = R / 32;  // of rows
  const int dim0 = (int)blockIdx.y / kBlocks * I, rb = (int)blockIdx.y % kBlocks;  // first block of 32 dims, of 16
  if (32 * rb >= rows) return;
  const int id = tid & 255, ps = tid >> 8, e = id >> 6, l32 = lane & 31, h = lane >> 5;
  const int r = 32 * rb + l32;
  auto part_of = [&](int p) { return (size_t)(p ? 2 * (group + p) : 2 * group + 1); };
  const float2* stat = space.stat + r;
  const f32x4* part = reinterpret_cast<const f32x4*>(space.part) + (rb * 16 + dim0) * 256 + e * 64 + lane;
  f32x4 v[I][kFlight];
  auto request = [&](int p0) {
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int t = 0; t < kFlight; ++t)
        if (p0 + t * S < parts) v[i][t] = __builtin_nontemporal_load(part + part_of(p0 + t * S) * (R * kLatDim / 4) + i * 256);
  };
  request(ps);  // ahead of the statistics that they wait for
  // the largest m of the row
  float top = -__builtin_inff();
  for (int p0 = ps; p0 < parts; p0 += kFlight * S) {
    float m[kFlight];
#pragma unroll
    for (int t = 0; t < kFlight; ++t) m[t] = p0 + t * S < parts ? stat[part_of(p0 + t * S) * R].x : -__builtin_inff();
#pragma unroll
    for (int t = 0; t < kFlight; ++t) top = fmaxf(top, m[t]);
  }
  if constexpr (S > 1) {
    if (e == 0 && h == 0) red_top[ps][l32] = top;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < S; ++t) top = fmaxf(top, red_top[t][l32]);
  }
  const float off = top == -__builtin_inff() ? 0.0f : top;
  float l = 0.0f;
  f32x4 sum[I];
#pragma unroll
  for (int i = 0; i < I; ++i) sum[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int p0 = ps; p0 < parts; p0 += kFlight * S) {
    if (p0 != ps) request(p0);
#pragma unroll
    for (int t = 0; t < kFlight; ++t)
      if (p0 + t * S < parts) {
        const float2 st = stat[part_of(p0 + t * S) * R];
        const float f = __builtin_amdgcn_exp2f(st.x - off);
        l = fmaf(f, st.y, l);
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) sum[i][c] = fmaf(f, v[i][t][c], sum[i][c]);
      }
  }
  if constexpr (S > 1) {
    static_assert(I == 1, "one block of dims where parts are shared out");
    if (ps) {
      red[ps - 1][id] = make_float4(sum[0][0], sum[0][1], sum[0][2], sum[0][3]);
      if (e == 0 && h == 0) red_l[ps - 1][l32] = l;
    }
    __syncthreads();
    if (ps) return;
#pragma unroll
    for (int t = 0; t < S - 1; ++t) {
      const float4 other = red[t][id];
      sum[0] += f32x4{other.x, other.y, other.z, other.w};
      l += red_l[t][l32];
    }
  }
  if (r >= rows) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int t = (tile0 + r) / a.H, hd = tile0 + r - t * a.H;
  T* out = static_cast<T*>(a.out) + (int64_t)(t0 + t) * a.out_token + hd * a.out_head + 32 * dim0 + 8 * e + 4 * h;
#pragma unroll
  for (int i = 0; i < I; ++i) {
    x4 y;
#pragma unroll
    for (int c = 0; c < 4; ++c) y[c] = (T)(sum[i][c] * inv);
    *reinterpret_cast<x4*>(out + 32 * i) = y;
  }
  if (a.lse && dim0 == 0 && e == 0 && h == 0)
    a.lse[(size_t)(t0 + t) * a.H + hd] =
        l == 0.0f ? -__builtin_inff() : (top + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

static int mla_tree_groups() { return min(max(1, g_num_cus), kMaxGroups); }

size_t mla_tree_workspace(int, int) {
  const int groups = mla_tree_groups();
  return space_part_at(groups) + (size_t)2 * groups * kPartFloats * sizeof(float);
}

namespace {
template <int FMT, int R>
void join_parts(const MlaTreeArgs& a, int groups, hipStream_t s) {
  // no more tiles than these, whatever the sequences' sizes
  const int64_t most = ((int64_t)a.N * a.H + R - 1) / R + a.B;
  const int tiles = (int)min((int64_t)groups, most);
  if (tiles * 16 <= groups)  // 16 parts a tile, if all workgroups have work
    k_mla_tree_join<FMT, R, 4, 1><<<dim3(tiles, R / 32 * 16), 1024, 0, s>>>(a, groups);
  else
    k_mla_tree_join<FMT, R, 1, 8><<<dim3(tiles, R / 32 * 2), 256, 0, s>>>(a, groups);
}
template <int FMT>
void launch_fmt(const MlaTreeArgs& a, hipStream_t s) {
  const int groups = mla_tree_groups();
  if (a.page_shift >= 3) k_mla_tree<FMT, true><<<groups, 256, 0, s>>>(a);
  else k_mla_tree<FMT, false><<<groups, 256, 0, s>>>(a);
  join_parts<FMT, kTileRows>(a, groups, s);
}
}  // namespace

hipError_t launch_mla_tree(const MlaTreeArgs& a, int fmt, hipStream_t s) {
  switch (fmt) {
    case kKvF16: launch_fmt<kKvF16>(a, s); break;
    case kKvBf16: launch_fmt<kKvBf16>(a, s); break;
    default: launch_fmt<kKvFp8>(a, s);
  }
  return hipGetLastError();
}

}  // namespace fdm
