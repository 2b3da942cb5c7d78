// project_kernels.hip -- a shared projection and the low-rank adapters of many
// requests beside it (fdm_project):
//   y_t = W x_t + c_a B_a (A_a x_t),   a the adapter of row t's request, or none.
// x and W in F16, BF16, or e4m3 with power-of-two scales (128 values of a row of x,
// 128 x 128 of W); A, B in F16 beside F16, else in BF16; sums in fp32.
#include "latent_device.h"
#include "project_work.h"

namespace fdm {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// How rows and matrix are read: as they are, or e4m3 as one product of 64 codes (kRowFp8) or
// widened to BF16 (kRowFp8Wide).  The fp8 products of gfx950 add eight neighbours in steps
// of 2^-13 of the largest one's power of two before they go into the fp32 sum (measured; 2^-23
// in BF16 and F16).  Of a row of 7168 normal values that is 1.5e-5 of the result, a
// hundredth of a BF16 result's own rounding and a fourteenth of an F16 one's, but 130 times
// what an fp32 one is off by: fp32 results take the BF16 products, in which codes and scales
// are exact.
constexpr int kRowF16 = 0, kRowBf16 = 1, kRowFp8 = 2, kRowFp8Wide = 3;

template <int FMT>
struct Half {
  typedef std::conditional_t<FMT == kRowF16, _Float16, __bf16> T;
  typedef std::conditional_t<FMT == kRowF16, f16x8, bf16x8> x8;
};
__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

__device__ __attribute__((aligned(16))) uint32_t zeros16[4];  // stands for 16 bytes behind a row's end

#define FDM_LDS __attribute__((address_space(3)))
// 16 bytes a lane from memory straight into LDS: lane i's land at `to` + 16 i.  In
// assembly, because the compiler lets no LDS read start while a direct load that it
// knows of is in flight; there is no result register, and wait_loads() is the wait.
__device__ __forceinline__ void lds_load16(const char* from, char* to) {
  const int at = (int)(uintptr_t)(FDM_LDS char*)to;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(from) : "memory");
}
// The same from a scalar base (not one that v_readlane wrote within the last five states)
// and a byte offset a lane.
__device__ __forceinline__ void lds_load16(const char* base, uint32_t off, char* to) {
  const int at = (int)(uintptr_t)(FDM_LDS char*)to;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(off), "s"(base) : "memory");
}
// A byte a lane, widened to four: lane i's land at `to` + 4 i.
__device__ __forceinline__ void lds_load_byte(const uint8_t* from, char* to) {
  const int at = (int)(uintptr_t)(FDM_LDS char*)to;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, off" ::"s"(at), "v"(from) : "memory");
}
// Sixteen e4m3 codes times a power of two, in BF16: exact, four bits of significand.
__device__ __forceinline__ void widen16(i32x4 c, float scale, bf16x8* v) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const auto lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[k], scale, false);
    const auto hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[k], scale, true);
    v[k / 2][4 * (k % 2)] = lo[0];
    v[k / 2][4 * (k % 2) + 1] = lo[1];
    v[k / 2][4 * (k % 2) + 2] = hi[0];
    v[k / 2][4 * (k % 2) + 3] = hi[1];
  }
}
// Eight codes.
__device__ __forceinline__ bf16x8 widen8(uint2 c, float scale) {
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.x, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.x, scale, true);
  const auto d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.y, scale, false), e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.y, scale, true);
  return bf16x8{a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
}
// at most N of the wave's loads are still in flight, and none of its LDS reads
template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The request whose tokens row t is among, its adapter; -1: none.
__device__ __forceinline__ int adapter_of(const ProjectArgs& a, int t) {
  if (t >= a.T) return -1;
  int lo = 0, hi = a.B + 1;  // the first b with q_start[b] > t, B + 1 if none
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (a.q_start[mid] <= t) lo = mid + 1;
    else hi = mid;
  }
  if (lo < 1 || lo > a.B) return -1;
  const int k = a.adapter[lo - 1];
  return k < a.n_adapters ? k : -1;
}

// ---- a wave's sums -----------------------------------------------------------------------
// The matrix's rows are the products' first operand and x's the second, so that a lane
// holds one row of the result a block.  Products of 16-bit values are 16 x 16 x 32: 32 x 32 x 16
// ones have the same rate but draw more, 1.80 against 2.11 PFLOP/s where the power
// limits them (random values, nothing beside the products).  fp8 ones are 32 x 32 x 64.
// Which row of the matrix stands in which place of the first operand is chosen such that
// a lane's columns, over its NB blocks, are neighbours.
template <int FMT>
struct Block {
  static constexpr bool k32 = FMT == kRowFp8;
  static constexpr int kRows = k32 ? 32 : 16;  // of x, and columns
  static constexpr int kOf = k32 ? 16 : 4;     // a lane's columns
  typedef std::conditional_t<k32, f32x16, f32x4> sum_t;
};
// The matrix's row (of a wave's) in place i of block j's operand.
template <int FMT, int NB>
__device__ __forceinline__ int matrix_row(int i, int j) {
  return Block<FMT>::k32 ? (i >> 2 & 1) * 16 * NB + 16 * j + (i >> 3) * 4 + (i & 3) : (i >> 2) * 4 * NB + 4 * j + (i & 3);
}
// Where a row's 16-byte piece c of a step lies: at c ^ swap8(row).  A read of 16 bytes a lane
// is served sixteen lanes at a time, 0-3, 12-15, 20-23 and 24-27 of each 32 and then the
// others; the swap is such that these, four rows each from four places of an operand above
// (and with 16 x 16 blocks two pieces), find sixteen bank groups.
template <int FMT>
__device__ __forceinline__ int swap8(int row) {
  const int q = row >> 2 & 3, upper = Block<FMT>::k32 ? q : q ^ (row >> 4 & 3);
  return upper << 1 | (row >> 1 & 1);
}

// The adapters' second product on a wave's sums: for every adapter among the rows of a
// block, B_a u on the matrix cores, u as sums of 16-bit numbers (a.planes of 8 bits each in
// BF16, two of 11 in F16), kept by the rows that are the adapter's own.  A row that
// has another keeps its sum untouched, whatever B_a holds.
template <int FMT, int NB>
__device__ __forceinline__ void add_adapters(const ProjectArgs& a, int u_splits, int m, int id, int n0, typename Block<FMT>::sum_t* acc) {
  typedef typename Half<FMT>::T T16;
  typedef typename Half<FMT>::x8 x8;
  constexpr int kRows = Block<FMT>::kRows, kK = 8 * 64 / kRows;  // values of the rank that a product takes
  const int lane = threadIdx.x & 63, i0 = lane % kRows, g = lane / kRows;
  uint64_t left = __ballot(id >= 0);
  const float* u = a.u + (int64_t)m * a.rank;
  while (left) {
    const int k = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    const bool mine = id == k;
    left &= ~__ballot(mine);
    const T16* B = static_cast<const T16*>(a.b) + (int64_t)k * a.out * a.rank;
    for (int j0 = 0; j0 < a.rank; j0 += kK) {
      const int j = j0 + 8 * g;
      float v[8];
      x8 bv[NB];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.0f;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 8; ++i) bv[nb][i] = (T16)0.0f;
      if (j < a.rank) {
        if (mine) load8(u + j, true, v);
        for (int p = 1; p < u_splits; ++p) {
          float more[8];
          if (mine) {
            load8(u + (int64_t)p * a.T * a.rank + j, true, more);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += more[i];
          }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const int n = min(n0 + matrix_row<FMT, NB>(i0, nb), a.out - 1);
          bv[nb] = *reinterpret_cast<const x8*>(B + (int64_t)n * a.rank + j);
        }
      }
      // F16 numbers: the largest of these brought to [1, 2) (below 4 where 2^-127 would be its
      // factor), so that none overflows and few are lost
      float down = 1.0f;
      if constexpr (FMT == kRowF16) {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const int e = min(max((int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127, -126), 126);
        const float up = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
        down = __builtin_bit_cast(float, (uint32_t)(127 + e) << 23);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= up;
      }
      typename Block<FMT>::sum_t sum[NB];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < Block<FMT>::kOf; ++i) sum[nb][i] = 0.0f;
      // v as 16-bit numbers, each the rest of those before it (an infinity has none)
      auto next = [&]() {
        x8 w;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          w[i] = (T16)v[i];
          const float rest = v[i] - (float)w[i];
          v[i] = fabsf(rest) < __builtin_inff() ? rest : 0.0f;
        }
        return w;
      };
      if constexpr (FMT == kRowF16) {
        // The rest, at most 2^-10, times 2^24 and its product first: beside values near 1 it
        // would lie below F16's steps of 2^-24 from 2^-14 on.  So a value is off by 2^-22 of itself,
        // or 2^-36 of the largest.
        const x8 first = next();
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= 0x1p24f;
        const x8 second = next();
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          sum[nb] = mfma(bv[nb], second, sum[nb]);
          sum[nb] = mfma(bv[nb], first, sum[nb] * 0x1p-24f);
        }
      } else {
        for (int p = 0; p < a.planes; ++p) {
          const x8 w = next();
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) sum[nb] = mfma(bv[nb], w, sum[nb]);
        }
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < Block<FMT>::kOf; ++i) acc[nb][i] = mine ? fmaf(sum[nb][i], down, acc[nb][i]) : acc[nb][i];
    }
  }
}

// A lane's columns n .. n + COUNT - 1 of a row.
template <int COUNT, typename TY, typename S>
__device__ __forceinline__ void store_columns(TY* y, int n, int out, bool vec, const S* c) {
  constexpr int kOf = sizeof(S) / 4;
#pragma unroll
  for (int p = 0; p < COUNT; p += 8) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c[(p + i) / kOf][(p + i) % kOf];
    if (vec && n + p + 8 <= out) {
      store8(y + n + p, true, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n + p + i < out) y[n + p + i] = (TY)v[i];
    }
  }
}

// A wave's sums, MB blocks of rows by NB of columns, that begin at row m0 and column n0 of the
// result: into y with the adapters' part, or (part not null) into the part's tile of `width`
// columns, where they begin at `part`.  ids: the rows' adapters.
template <int FMT, int MB, int NB>
__device__ __forceinline__ void store_tile(const ProjectArgs& a, typename Block<FMT>::sum_t (*acc)[NB], float* part, int width, int m0, int n0,
                                           const int* ids) {
  constexpr int kRows = Block<FMT>::kRows, kCount = NB * Block<FMT>::kOf;
  const int lane = threadIdx.x & 63, i0 = lane % kRows, col = lane / kRows * kCount;
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int m = m0 + kRows * i + i0;
    if (part) {
      if (m < a.T) store_columns<kCount>(part + (kRows * i + i0) * width, col, width, true, acc[i]);
      continue;
    }
    if (a.n_adapters) add_adapters<FMT, NB>(a, 1, m, ids[kRows * i + i0], n0, acc[i]);
    if (m >= a.T) continue;
    char* y = static_cast<char*>(a.y) + (int64_t)m * a.y_bytes;
    if (a.y_type == ElemType::f32) store_columns<kCount>(reinterpret_cast<float*>(y), n0 + col, a.out, a.vec_y, acc[i]);
    else if (a.y_type == ElemType::f16) store_columns<kCount>(reinterpret_cast<_Float16*>(y), n0 + col, a.out, a.vec_y, acc[i]);
    else store_columns<kCount>(reinterpret_cast<__bf16*>(y), n0 + col, a.out, a.vec_y, acc[i]);
  }
}

// ---- the adapters' first product: u_t = c_a A_a x_t ----------------------------------
// A workgroup takes up to 32 rows of one adapter, wherever they stand: all count the
// requests' rows by adapter in LDS, and tile `mine` of the list (adapters in order,
// their rows in order) is found from that; tiles <= rows / 32 + adapters in use.  The waves
// share the values of part `split` of `splits` of the inner dimension, 128 bytes of a
// row of x at a time, the next ones on their way; their sums meet in LDS.  Ranks above 64
// are two halves, tiles of their own (more sums and operands do not fit the registers).
// Bound by what a CU brings of x from beyond its L2, some 25 bytes a ns: 5050 rows of 16384 BF16
// values of rank 32 83 us on 162 CUs whatever is under way (one step a wave or four, eight waves or
// sixteen, rows a power of two apart or not).  In three parts, on all CUs, 59, but then every
// tile of the second product adds them up, which takes as much again.
struct AdapterLds {
  int count[kMaxAdapters];
  int list[32], chosen[2], of_wave[8];
  float sums[8][32][20];
};
template <int FMT, int RB, int WAVES>
__device__ __forceinline__ void adapter_in(const ProjectArgs& a, int split, int splits, int mine, int rank0, AdapterLds& l) {
  constexpr int kThreads = 64 * WAVES, kEach = kMaxAdapters / kThreads;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i < a.n_adapters; i += kThreads) l.count[i] = 0;
  if (tid == 0) l.chosen[0] = -1;
  if (tid < 32) l.list[tid] = -1;
  __syncthreads();
  for (int b = tid; b < a.B; b += kThreads) {
    const int k = a.adapter[b], t0 = min(max(a.q_start[b], 0), a.T), n = min(max(a.q_start[b + 1], 0), a.T) - t0;
    if (k >= 0 && k < a.n_adapters && n > 0) atomicAdd(&l.count[k], n);
  }
  __syncthreads();
  // tiles before each adapter, kEach consecutive ones a thread
  int tiles = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (tid * kEach + i < a.n_adapters) tiles += (l.count[tid * kEach + i] + 31) / 32;
  int upto = tiles;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int v = __shfl_up(upto, d);
    if (lane >= d) upto += v;
  }
  if (lane == 63) l.of_wave[wave] = upto;
  __syncthreads();
  int before = upto - tiles;
  for (int w = 0; w < wave; ++w) before += l.of_wave[w];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int k = tid * kEach + i;
    if (k >= a.n_adapters) break;
    const int n = (l.count[k] + 31) / 32;
    if (mine >= before && mine < before + n) {
      l.chosen[0] = k;
      l.chosen[1] = 32 * (mine - before);
    }
    before += n;
  }
  __syncthreads();
  const int k = __builtin_amdgcn_readfirstlane(l.chosen[0]), row0 = l.chosen[1];
  if (k < 0) return;  // no such tile
  // the adapter's rows row0 .. row0 + 31
  int seen = 0;
  for (int b0 = 0; b0 < a.B && seen < row0 + 32; b0 += kThreads) {
    const int b = b0 + tid;
    int t0 = 0, n = 0;
    if (b < a.B && a.adapter[b] == k) {
      t0 = min(max(a.q_start[b], 0), a.T);
      n = max(min(max(a.q_start[b + 1], 0), a.T) - t0, 0);
    }
    int sum = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(sum, d);
      if (lane >= d) sum += v;
    }
    __syncthreads();
    if (lane == 63) l.of_wave[wave] = sum;
    __syncthreads();
    int at = seen + sum - n;
    for (int w = 0; w < WAVES; ++w) {
      if (w < wave) at += l.of_wave[w];
      seen += l.of_wave[w];
    }
    for (int i = max(at, row0); i < min(at + n, row0 + 32); ++i) l.list[i - row0] = t0 + (i - at);
  }
  __syncthreads();

  typedef typename Half<FMT>::T T16;
  typedef typename Half<FMT>::x8 x8;
  constexpr bool kCodes = FMT == kRowFp8 || FMT == kRowFp8Wide;
  typedef std::conditional_t<kCodes, uint2, x8> piece_t;  // eight values of x
  constexpr int kUnits = kCodes ? 4 : 2;                  // products of 32 values in 128 bytes of x
  const int r = lane & 15, g = lane >> 4;
  const int steps = a.steps, parts = splits * WAVES, part = split * WAVES + wave;
  const int s0 = (int)((int64_t)steps * part / parts), s1 = (int)((int64_t)steps * (part + 1) / parts);
  const char* x[2];
  const uint8_t* scale[2] = {};
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const int t = max(l.list[16 * m + r], 0);
    x[m] = static_cast<const char*>(a.x) + (int64_t)t * a.x_bytes;
    if (kCodes) scale[m] = a.x_scale + (int64_t)t * a.x_scale_bytes;
  }
  const int rank = min(a.rank - rank0, kRankPart);
  const T16* A = static_cast<const T16*>(a.a) + ((int64_t)k * a.rank + rank0) * a.in;
  f32x4 acc[2][RB];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int j = 0; j < RB; ++j) acc[m][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  struct Step {
    piece_t x[2][kUnits];
    x8 a[RB][kUnits];
    int scale[2];
  };
  auto load = [&](int s, Step& v) {
#pragma unroll
    for (int q = 0; q < kUnits; ++q) {
      const int at = (s * kUnits + q) * 32 + 8 * g;
      const bool in = at < a.in;
#pragma unroll
      for (int m = 0; m < 2; ++m) v.x[m][q] = in ? *reinterpret_cast<const piece_t*>(x[m] + at * (kCodes ? 1 : 2)) : piece_t{};
#pragma unroll
      for (int j = 0; j < RB; ++j) v.a[j][q] = in && 16 * j + r < rank ? *reinterpret_cast<const x8*>(A + (int64_t)(16 * j + r) * a.in + at) : x8{};
    }
    if constexpr (kCodes)
#pragma unroll
      for (int m = 0; m < 2; ++m) v.scale[m] = scale[m][s];
  };
  auto use = [&](const Step& v) {
#pragma unroll
    for (int q = 0; q < kUnits; ++q)
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        x8 xv;
        if constexpr (kCodes) xv = widen8(v.x[m][q], scale_value(v.scale[m]));
        else xv = v.x[m][q];
#pragma unroll
        for (int j = 0; j < RB; ++j) acc[m][j] = mfma(v.a[j][q], xv, acc[m][j]);
      }
  };
  Step v[2];
  if (s0 < s1) load(s0, v[0]);
  for (int s = s0; s < s1; s += 2) {
    if (s + 1 < s1) load(s + 1, v[1]);
    use(v[0]);
    if (s + 2 < s1) load(s + 2, v[0]);
    if (s + 1 < s1) use(v[1]);
  }
  const float c = a.times ? a.times[k] : 1.0f;
#pragma unroll
  for (int j = 0; j < RB; ++j) {
    // lane: rows r and 16 + r, columns 4 g + 0 .. 3 of the block
    if (j) __syncthreads();
#pragma unroll
    for (int m = 0; m < 2; ++m) *reinterpret_cast<f32x4*>(&l.sums[wave][16 * m + r][4 * g]) = acc[m][j];
    __syncthreads();
    for (int i = tid; i < 32 * 16; i += kThreads) {
      const int m = i / 16, col = i % 16;
      if (l.list[m] < 0 || 16 * j + col >= rank) continue;
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) s += l.sums[w][m][col];
      a.u[((int64_t)split * a.T + l.list[m]) * a.rank + rank0 + 16 * j + col] = s * c;
    }
  }
}
template <int FMT, int WAVES>
__device__ __forceinline__ void adapter_in(const ProjectArgs& a, int split, int splits, int mine, int rank0, AdapterLds& l) {
  if (a.rank <= 16) adapter_in<FMT, 1, WAVES>(a, split, splits, mine, rank0, l);
  else if (a.rank <= 32) adapter_in<FMT, 2, WAVES>(a, split, splits, mine, rank0, l);
  else adapter_in<FMT, 4, WAVES>(a, split, splits, mine, rank0, l);
}

}  // namespace

template <int FMT, int RB>
__global__ __launch_bounds__(512) void k_adapter_in(ProjectArgs a) {
  __shared__ AdapterLds l;
  adapter_in<FMT, RB, 8>(a, blockIdx.x, gridDim.x, blockIdx.y, blockIdx.z * kRankPart, l);
}

// ---- the tiles -----------------------------------------------------------------------------
// Tiles of a projection in the order in which workgroups take them.  Neighbours in the list
// run on one XCD (workgroups go round the eight in turn) and share what they read: bands of
// four tiles of rows, down and then along.
struct Place {
  int part, m, n;
};
__device__ __forceinline__ int on_xcd(int i, int count) {
  const int xcd = i % 8;
  return xcd * (count / 8) + min(xcd, count % 8) + i / 8;
}
__device__ __forceinline__ Place place_of(int tile, int m_tiles, int n_tiles) {
  const int band = tile / (4 * n_tiles), high = min(4, m_tiles - 4 * band), in_band = tile - band * 4 * n_tiles;
  return {0, 4 * band + in_band % high, in_band / high};
}

// A tile of BM rows of x by BN of the matrix, WM x WN waves, over the steps (128 bytes of
// every row) of its part of the inner dimension.  Steps go straight into LDS, into a ring of
// RING, RING - 1 of them under way, and from there as operands.  Whole lines of 128 bytes,
// because half a line costs a CU's loads as much as a whole one (32 against 53 bytes a cycle).
// TURN (eight waves, two a SIMD; 0: without): a wave's turn is TURN bytes of the rows and has
// two parts, its operands' LDS reads, in a step's first turn with the requests for a step to
// come, and the products; the two waves of a SIMD take opposite parts, with a barrier
// between, so that the products of one run while the other reads:
//   interval   2 j         2 j + 1       2 j + 2
//   waves 0-3  read j      products j    read j + 1
//   waves 4-7  products    read j        products j
// The requests for step s + RING - 1 fill the place of s - 1, which both have read an interval
// before.  Without turns all read, then multiply.
// The first a.u_groups workgroups do the adapters' first product, the next a.full a tile
// each, the others a part of one.
// Measured (a launch; the library's BF16 product of 8192^3 reaches 1.38 PFLOP/s, its e4m3 one
// 2.65): 5050 rows of 16384 BF16 values by 7168 in tiles of 256 x 256 1020 us with the adapters' second
// product, 1.16 PFLOP/s, 10276 of 7168 codes by 18432 1200 us, 2.26: the matrix cores are busy 61 and
// 56 % of the cycles, at 1.7 GHz of 2.4, which the products' power leaves (the library reaches 1.34 on
// the first matrix and 3.20 on 8192 rows by the second, with one scale an operand).  256 rows of 16384 by 7168 91 us, 2.9 TB/s; 24 of 1536 F16 by
// 24576 14.5, 5.5 TB/s; one row of 7168 by 1536 7.1, two launches' latencies with the join.
template <int FMT, int BM, int BN, int WM, int WN, int RING, int TURN>
__global__ __launch_bounds__(64 * WM * WN) void k_project(ProjectArgs a) {
  constexpr bool kCodes = FMT == kRowFp8 || FMT == kRowFp8Wide;
  constexpr int kWaves = WM * WN, kThreads = 64 * kWaves, kStage = (BM + BN) * kStepBytes;
  constexpr int kLoadsX = BM / 8 / kWaves, kLoads = (BM + BN) / 8 / kWaves;  // of a wave and step, eight rows each
  constexpr int kBlock = Block<FMT>::kRows, MB = BM / WM / kBlock, NB = BN / WN / kBlock;
  constexpr int kPieces = kBlock / 16;         // 16-byte pieces of a lane's operand
  constexpr int kHalves = TURN == 64 ? 1 : 2;  // of a step (a product each) that are read at a time
  constexpr int kGroups = BN / 128, kScales = (BM + kGroups + 63) / 64 * 64;
  static_assert(BM % (8 * kWaves) == 0 && BN % (8 * kWaves) == 0 && BN % 128 == 0, "whole loads and groups");
  static_assert(MB * WM * kBlock == BM && NB * WN * kBlock == BN && kScales <= kThreads && (!TURN || kWaves == 8), "whole blocks");
  static_assert(sizeof(AdapterLds) <= RING * kStage, "LDS");
  typedef std::conditional_t<kCodes, i32x4, typename Half<FMT>::x8> piece_t;
  __shared__ __attribute__((aligned(16))) char lds[RING * kStage];
  __shared__ __attribute__((aligned(16))) int scales[kCodes ? RING : 1][kScales];  // rows of x, then the matrix's groups
  __shared__ int ids[BM];
  if ((int)blockIdx.x < a.u_groups) {
    const int halves = (a.rank + kRankPart - 1) / kRankPart, tile = blockIdx.x / a.u_splits;
    adapter_in<FMT, kWaves>(a, blockIdx.x % a.u_splits, a.u_splits, tile / halves, tile % halves * kRankPart, *reinterpret_cast<AdapterLds*>(lds));
    return;
  }
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane % kBlock, h = lane / kBlock;
  const bool second = wave >= 4;
  const int m_tiles = (a.T + BM - 1) / BM, n_tiles = (a.out + BN - 1) / BN, tiles = m_tiles * n_tiles;
  const int group = (int)blockIdx.x - a.u_groups;
  int tile, part = 0, parts = 1;
  if (group < a.full) {
    tile = on_xcd(group, a.full);
  } else {
    const int rest = tiles - a.full, at = on_xcd(group - a.full, rest * a.splits);
    part = at / rest;
    parts = a.splits;
    tile = a.full + at - part * rest;
  }
  const Place place = place_of(tile, m_tiles, n_tiles);
  const int m0 = BM * place.m, n0 = BN * place.n;
  const int step0 = (int)((int64_t)a.steps * part / parts), step1 = (int)((int64_t)a.steps * (part + 1) / parts);
  const int whole = a.row_bytes / kStepBytes;  // steps

  // this wave's loads: offsets of their rows, those past the end being the last one again
  const char* base_x = static_cast<const char*>(a.x) + (int64_t)m0 * a.x_bytes;
  const char* base_w = static_cast<const char*>(a.w) + (int64_t)n0 * a.w_bytes;
  uint32_t off[kLoads];
  int piece[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const bool of_x = i < kLoadsX;
    const int row = (kWaves * (of_x ? i : i - kLoadsX) + wave) * 8 + lane / 8;
    piece[i] = ((lane & 7) ^ swap8<FMT>(row)) * 16;
    off[i] = (of_x ? (uint32_t)(min(row, a.T - 1 - m0) * a.x_bytes) : (uint32_t)(min(row, a.out - 1 - n0) * a.w_bytes)) + piece[i];
  }
  auto bring = [&](int step) {
    if (step >= step1) return;
    char* to = lds + (unsigned)step % RING * kStage + wave * 1024;
    auto at = [&](int i) { return to + (i < kLoadsX ? i * kWaves * 1024 : BM * kStepBytes + (i - kLoadsX) * kWaves * 1024); };
    if (step < whole) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) lds_load16((i < kLoadsX ? base_x : base_w) + (int64_t)step * kStepBytes, off[i], at(i));
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int b = step * kStepBytes + piece[i];
        lds_load16(b < a.row_bytes ? (i < kLoadsX ? base_x : base_w) + off[i] + step * kStepBytes : reinterpret_cast<const char*>(zeros16), at(i));
      }
    }
  };
  // the scales of a step: a byte a thread, by the waves that have some
  const bool scaler = kCodes && wave * 64 < kScales;
  const uint8_t* scale_at = nullptr;
  if constexpr (kCodes)
    scale_at = tid < BM ? a.x_scale + (int64_t)min(m0 + tid, a.T - 1) * a.x_scale_bytes
                        : a.w_scale + (int64_t)min(n0 / 128 + (tid - BM) % kGroups, (a.out - 1) / 128) * a.w_scale_bytes;
  auto bring_scales = [&](int step) {
    if (scaler && step < step1) lds_load_byte(scale_at + step, reinterpret_cast<char*>(&scales[(unsigned)step % RING][64 * wave]));
  };

  typename Block<FMT>::sum_t acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int e = 0; e < Block<FMT>::kOf; ++e) acc[i][j][e] = 0.0f;

  // where a lane's pieces of a step's first half lie, for the first block of x's rows and for
  // each of the matrix's: the pieces kPieces h + 0 .. kPieces - 1; of the second half 64 bytes apart
  const int wm = wave / WN, wn = wave % WN;
  int at_x[kPieces], at_w[NB][kPieces];
  auto place_in = [&](int row, int c) { return row * kStepBytes + (c ^ swap8<FMT>(row)) * 16; };
#pragma unroll
  for (int p = 0; p < kPieces; ++p) {
    at_x[p] = place_in(BM / WM * wm + r, kPieces * h + p);
#pragma unroll
    for (int j = 0; j < NB; ++j) at_w[j][p] = BM * kStepBytes + place_in(BN / WN * wn + matrix_row<FMT, NB>(r, j), kPieces * h + p);
  }

  piece_t xv[MB][kHalves][kPieces], wv[NB][kHalves][kPieces];
  int xs[MB] = {}, ws = 0;
  auto read = [&](int step, int half0) {
    const char* s = lds + (unsigned)step % RING * kStage;
#pragma unroll
    for (int k = 0; k < kHalves; ++k)
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
#pragma unroll
        for (int i = 0; i < NB; ++i) wv[i][k][p] = *reinterpret_cast<const piece_t*>(s + (at_w[i][p] ^ (half0 + k) << 6));
#pragma unroll
        for (int i = 0; i < MB; ++i)  // (row kBlock i + r's swap is that of kBlock i and of r)
          xv[i][k][p] = *reinterpret_cast<const piece_t*>(s + (at_x[p] ^ ((half0 + k) << 6 ^ swap8<FMT>(kBlock * i) << 4)) + kBlock * kStepBytes * i);
      }
    if constexpr (kCodes) {
      if (half0 == 0) {
        const int* c = scales[(unsigned)step % RING];
#pragma unroll
        for (int i = 0; i < MB; ++i) xs[i] = c[BM / WM * wm + r + kBlock * i];
        ws = c[BM + BN / WN * wn / 128];
      }
    }
  };
  auto products = [&]() {
#pragma unroll
    for (int k = 0; k < kHalves; ++k) {
      if constexpr (FMT == kRowFp8) {
        auto eight = [](const piece_t* v) { return i32x8{v[0][0], v[0][1], v[0][2], v[0][3], v[1][0], v[1][1], v[1][2], v[1][3]}; };
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int j = 0; j < NB; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(eight(wv[j][k]), eight(xv[i][k]), acc[i][j], 0, 0, 0, ws, 0, xs[i]);
      } else if constexpr (FMT == kRowFp8Wide) {
        bf16x8 w[NB][2];
#pragma unroll
        for (int j = 0; j < NB; ++j) widen16(wv[j][k][0], scale_value(ws), w[j]);
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          bf16x8 x[2];
          widen16(xv[i][k][0], scale_value(xs[i]), x);
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] = mfma(w[j][e], x[e], acc[i][j]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int j = 0; j < NB; ++j) acc[i][j] = mfma(wv[j][k][0], xv[i][k][0], acc[i][j]);
      }
    }
  };
  // Step s + 1 has landed when no more are under way than the requests behind its own: those
  // of RING - 2 steps, with a scales' one each; near the end, when none follow, all have.
  auto landed = [&](int step) {
    if (step + RING - 1 >= step1) wait_loads<0>();
    else if (scaler) wait_loads<(RING - 2) * (kLoads + 1)>();
    else wait_loads<(RING - 2) * kLoads>();
  };

#pragma unroll
  for (int s = 0; s < RING - 1; ++s) {
    bring(step0 + s);
    if constexpr (kCodes) bring_scales(step0 + s);
  }
  if (a.n_adapters && group < a.full)
    for (int i = tid; i < BM; i += kThreads) ids[i] = adapter_of(a, m0 + i);
  landed(step0 - 1);
  if constexpr (TURN) {
    barrier();
    if (second) barrier();
  }
  for (int step = step0; step < step1; ++step) {
    if constexpr (!TURN) {
      if (step > step0) landed(step - 1);
      barrier();
      read(step, 0);
      bring(step + RING - 1);
      if constexpr (kCodes) bring_scales(step + RING - 1);
      products();
    } else {
#pragma unroll
      for (int turn = 0; turn < 2 / kHalves; ++turn) {
        const bool last = turn == 2 / kHalves - 1;
        read(step, turn);
        if (turn == 0) {
          bring(step + RING - 1);
          if constexpr (kCodes) bring_scales(step + RING - 1);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (last && second) landed(step);
        else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        barrier();
        __builtin_amdgcn_s_setprio(1);
        __builtin_amdgcn_sched_barrier(0);
        products();
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int e = 0; e < NB; ++e) asm volatile("" : "+v"(acc[i][e]));  // here, not where the sums are next used
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(0);
        if (last && !second) landed(step);
        barrier();
      }
    }
  }
  if constexpr (TURN)
    if (!second) barrier();

  float* to = nullptr;
  if (group >= a.full)
    to = a.part + ((int64_t)part * (tiles - a.full) + tile - a.full) * (BM * BN) + BM / WM * wm * BN + BN / WN * wn;
  store_tile<FMT, MB, NB>(a, acc, to, BN, m0 + BM / WM * wm, n0 + BN / WN * wn, ids + BM / WM * wm);
}

// ---- parts and the adapters' second product, added -------------------------------------
// CHUNKS times 256 neighbouring values of a tile's parts a workgroup, 256 / BN rows each, a
// value a thread and chunk.  All of a thread's parts are requested before the rows' adapters
// are looked up; where there is one chunk the four waves share them, four values a lane.  B's row
// of an adapter is read once for the neighbouring rows that have it.  Bound by latency: 64 rows by
// 2112 in eight parts, rank 16, 4.9 us; 256 by 7168 in two 5.1, with an adapter a row 11.7.
template <int FMT, int BM, int BN, int CHUNKS>
__global__ __launch_bounds__(256) void k_project_join(ProjectArgs a) {
  typedef typename Half<FMT>::T T16;
  typedef typename Half<FMT>::x8 x8;
  constexpr int kSub = 256 / BN, kRows = CHUNKS * kSub;
  __shared__ __attribute__((aligned(16))) float sums[4][256];
  __shared__ __attribute__((aligned(16))) float u[kRows][kMaxRank];
  __shared__ int ids[kRows];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int m_tiles = (a.T + BM - 1) / BM, n_tiles = (a.out + BN - 1) / BN, rest = m_tiles * n_tiles - a.full;
  const Place place = place_of(a.full + blockIdx.x, m_tiles, n_tiles);
  const int t0 = BM * place.m + kRows * (int)blockIdx.y, rows = min(kRows, a.T - t0);
  if (rows <= 0) return;
  const int sub = tid / BN, n = BN * place.n + tid % BN;
  const float* part = a.part + (int64_t)blockIdx.x * (BM * BN) + kRows * (int)blockIdx.y * BN;
  const int64_t next = (int64_t)rest * (BM * BN);
  float y[CHUNKS];
  if constexpr (CHUNKS == 1) {
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int p = wave; p < a.splits; p += 4) s += *reinterpret_cast<const f32x4*>(part + p * next + 4 * lane);
    *reinterpret_cast<f32x4*>(&sums[wave][4 * lane]) = s;
  } else {
#pragma unroll
    for (int m = 0; m < CHUNKS; ++m) y[m] = part[256 * m + tid];
    for (int p = 1; p < a.splits; ++p) {
#pragma unroll
      for (int m = 0; m < CHUNKS; ++m) y[m] += part[p * next + 256 * m + tid];
    }
  }
  if (a.n_adapters) {
    if (tid < kRows) ids[tid] = -1;
    __syncthreads();
    for (int b = tid; b < a.B; b += 256) {
      const int k = a.adapter[b], from = max(a.q_start[b], t0), to = min(a.q_start[b + 1], t0 + rows);
      if (k >= 0 && k < a.n_adapters)
        for (int t = from; t < to; ++t) ids[t - t0] = k;
    }
    __syncthreads();
    const int quads = a.rank / 4;
    for (int i = tid; i < rows * quads; i += 256) {
      const int m = i / quads, j = 4 * (i - m * quads);
      if (ids[m] < 0) continue;
      f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
      for (int p = 0; p < a.u_splits; ++p) s += *reinterpret_cast<const f32x4*>(a.u + ((int64_t)p * a.T + t0 + m) * a.rank + j);
      *reinterpret_cast<f32x4*>(&u[m][j]) = s;
    }
  }
  __syncthreads();
  if constexpr (CHUNKS == 1) y[0] = (sums[0][tid] + sums[1][tid]) + (sums[2][tid] + sums[3][tid]);
  if (n >= a.out) return;
  if (a.n_adapters) {
    const int own = (rows - sub + kSub - 1) / kSub;  // chunks that hold a row of this thread's
    for (int m = 0; m < own;) {
      const int k = ids[m * kSub + sub];
      int end = m + 1;
      while (end < own && ids[end * kSub + sub] == k) ++end;
      if (k >= 0) {
        const T16* B = static_cast<const T16*>(a.b) + ((int64_t)k * a.out + n) * a.rank;
#pragma unroll 4
        for (int j = 0; j < a.rank; j += 8) {
          const x8 v = *reinterpret_cast<const x8*>(B + j);
#pragma unroll
          for (int i = 0; i < CHUNKS; ++i)
            if (i >= m && i < end) {
              const f32x4 lo = *reinterpret_cast<const f32x4*>(&u[i * kSub + sub][j]), hi = *reinterpret_cast<const f32x4*>(&u[i * kSub + sub][j + 4]);
#pragma unroll
              for (int e = 0; e < 4; ++e) y[i] = fmaf(lo[e], (float)v[e], y[i]);
#pragma unroll
              for (int e = 0; e < 4; ++e) y[i] = fmaf(hi[e], (float)v[4 + e], y[i]);
            }
        }
      }
      m = end;
    }
  }
#pragma unroll
  for (int m = 0; m < CHUNKS; ++m) {
    const int row = m * kSub + sub;
    if (row >= rows) break;
    char* to = static_cast<char*>(a.y) + (int64_t)(t0 + row) * a.y_bytes;
    if (a.y_type == ElemType::f32) reinterpret_cast<float*>(to)[n] = y[m];
    else if (a.y_type == ElemType::f16) reinterpret_cast<_Float16*>(to)[n] = (_Float16)y[m];
    else reinterpret_cast<__bf16*>(to)[n] = (__bf16)y[m];
  }
}

// The same on the matrix cores: a wave adds the parts of 16 rows by 32 columns and then B u of every
// adapter among the rows.
constexpr int kJoinCols = 128;  // of a workgroup
template <int FMT, int BM, int BN>
__global__ __launch_bounds__(256) void k_project_join_rows(ProjectArgs a) {
  constexpr int NB = kJoinCols / 64;
  __shared__ __attribute__((aligned(16))) float sums[16][kJoinCols + 4];
  __shared__ int ids[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int m_tiles = (a.T + BM - 1) / BM, n_tiles = (a.out + BN - 1) / BN, rest = m_tiles * n_tiles - a.full;
  const Place place = place_of(a.full + blockIdx.x, m_tiles, n_tiles);
  const int row = 16 * ((int)blockIdx.y / (BN / kJoinCols)), col = kJoinCols * ((int)blockIdx.y % (BN / kJoinCols)) + 16 * NB * wave;
  const int t0 = BM * place.m + row, n0 = BN * place.n + col, m = t0 + lane % 16;
  if (t0 >= a.T) return;
  const float* part = a.part + (int64_t)blockIdx.x * (BM * BN) + (row + lane % 16) * BN + col + lane / 16 * 4 * NB;
  const int64_t next = (int64_t)rest * (BM * BN);
  f32x4 acc[1][NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) acc[0][i] = *reinterpret_cast<const f32x4*>(part + 4 * i);
  for (int p = 1; p < a.splits; ++p)
#pragma unroll
    for (int i = 0; i < NB; ++i) acc[0][i] += *reinterpret_cast<const f32x4*>(part + p * next + 4 * i);
  if (tid < 16) ids[tid] = -1;
  __syncthreads();
  for (int b = tid; b < a.B; b += 256) {
    const int k = a.adapter[b], from = max(a.q_start[b], t0), to = min(a.q_start[b + 1], min(t0 + 16, a.T));
    if (k >= 0 && k < a.n_adapters)
      for (int t = from; t < to; ++t) ids[t - t0] = k;
  }
  __syncthreads();
  if (n0 < a.out) add_adapters<FMT, NB>(a, a.u_splits, m, ids[lane % 16], n0, acc[0]);
  if (a.vec_y) {
    if (m >= a.T) return;
    char* y = static_cast<char*>(a.y) + (int64_t)m * a.y_bytes;
    const int n = n0 + lane / 16 * 4 * NB;
    if (a.y_type == ElemType::f32) store_columns<4 * NB>(reinterpret_cast<float*>(y), n, a.out, true, acc[0]);
    else if (a.y_type == ElemType::f16) store_columns<4 * NB>(reinterpret_cast<_Float16*>(y), n, a.out, true, acc[0]);
    else store_columns<4 * NB>(reinterpret_cast<__bf16*>(y), n, a.out, true, acc[0]);
    return;
  }
  // value by value, in whole rows: 650 rows by 2111 of rank 64 in fp32 12.5 us, from the lanes 14.4
#pragma unroll
  for (int i = 0; i < NB; ++i) *reinterpret_cast<f32x4*>(&sums[lane % 16][16 * NB * wave + lane / 16 * 4 * NB + 4 * i]) = acc[0][i];
  __syncthreads();
  const int n = n0 - 16 * NB * wave + tid % kJoinCols;
  if (n >= a.out) return;
#pragma unroll
  for (int i = tid / kJoinCols; i < 16; i += 256 / kJoinCols) {
    if (t0 + i >= a.T) break;
    const float v = sums[i][tid % kJoinCols];
    char* to = static_cast<char*>(a.y) + (int64_t)(t0 + i) * a.y_bytes;
    if (a.y_type == ElemType::f32) reinterpret_cast<float*>(to)[n] = v;
    else if (a.y_type == ElemType::f16) reinterpret_cast<_Float16*>(to)[n] = (_Float16)v;
    else reinterpret_cast<__bf16*>(to)[n] = (__bf16)v;
  }
}

namespace {

template <int FMT>
hipError_t launch_adapter_in(const ProjectArgs& a, hipStream_t s) {
  const dim3 grid(a.u_splits, adapter_tiles(a.T, a.B, a.n_adapters), rank_parts(a.rank));
  if (a.rank <= 16) k_adapter_in<FMT, 1><<<grid, 512, 0, s>>>(a);
  else if (a.rank <= 32) k_adapter_in<FMT, 2><<<grid, 512, 0, s>>>(a);
  else k_adapter_in<FMT, 4><<<grid, 512, 0, s>>>(a);
  return hipGetLastError();
}

template <int FMT, int BM, int BN, int WM, int WN, int RING, int TURN>
hipError_t launch_tiles(ProjectArgs a, const ProjectPlan& p, hipStream_t s) {
  const int m_tiles = (a.T + BM - 1) / BM, tiles = m_tiles * ((a.out + BN - 1) / BN), rest = tiles - a.full;
  a.u_groups = 0;
  if (a.n_adapters && a.full) {
    const hipError_t e = launch_adapter_in<FMT>(a, s);
    if (e != hipSuccess) return e;
  } else if (a.n_adapters) {
    a.u_groups = adapter_tiles(a.T, a.B, a.n_adapters) * rank_parts(a.rank) * a.u_splits;
  }
  k_project<FMT, BM, BN, WM, WN, RING, TURN><<<a.u_groups + a.full + rest * a.splits, 64 * WM * WN, 0, s>>>(a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !rest) return e;
  constexpr int kHalf = FMT == kRowF16 ? kRowF16 : kRowBf16;
  const int rows = std::min(BM, a.T), chunks = join_chunks(p.tile, a.T);
  switch (project_join(p, a.T, a.out, a.B, a.rank, g_num_cus)) {
    case kJoinOne: k_project_join<FMT, BM, BN, 1><<<dim3(rest, chunks), 256, 0, s>>>(a); break;
    case kJoinRows: k_project_join_rows<kHalf, BM, BN><<<dim3(rest, (rows + 15) / 16 * (BN / kJoinCols)), 256, 0, s>>>(a); break;
    default: k_project_join<FMT, BM, BN, 4><<<dim3(rest, (chunks + 3) / 4), 256, 0, s>>>(a); break;
  }
  return hipGetLastError();
}

template <int FMT>
hipError_t launch_fmt(const ProjectArgs& a, const ProjectPlan& p, hipStream_t s) {
  switch (p.tile) {
    case kTile32: return launch_tiles<FMT, 32, 128, 1, 4, 6, 0>(a, p, s);
    case kTile64: return launch_tiles<FMT, 64, 128, 2, 4, 5, 0>(a, p, s);
    case kTile128: return launch_tiles<FMT, 128, 128, 2, 4, 4, 0>(a, p, s);
    default: return launch_tiles<FMT, 256, 256, 2, 4, 2, 64>(a, p, s);
  }
}

}  // namespace

hipError_t launch_project(const ProjectArgs& a, const ProjectPlan& p, int fmt, hipStream_t s) {
  switch (fmt) {
    case kRowF16: return launch_fmt<kRowF16>(a, p, s);
    case kRowBf16: return launch_fmt<kRowBf16>(a, p, s);
    case kRowFp8Wide: return launch_fmt<kRowFp8Wide>(a, p, s);
    default: return launch_fmt<kRowFp8>(a, p, s);
  }
}

}  // namespace fdm
