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
// widened to BF16 (kRowFp8Wide).  The fp8 products of gfx950 add eight neighbours before
// they go into the fp32 sum, and what lies 2^-14 and more under the largest of the eight is
// cut off there (measured; 2^-24 in BF16 and F16).  Of a row of 7168 normal values that
// is 1e-4 of the result, a tenth of a 16-bit result's own rounding, but a thousand times an
// fp32 one's: fp32 results take the BF16 products, in which codes and scales are exact.
constexpr int kRowF16 = 0, kRowBf16 = 1, kRowFp8 = 2, kRowFp8Wide = 3;

template <int FMT>
struct Half {
  typedef std::conditional_t<FMT == kRowF16, _Float16, __bf16> T;
  typedef std::conditional_t<FMT == kRowF16, f16x8, bf16x8> x8;
};
__device__ __forceinline__ f32x16 mfma16(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma16(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

__device__ __attribute__((aligned(16))) uint32_t zeros16[4];  // stands for 16 bytes behind a row's end

#define FDM_LDS __attribute__((address_space(3)))
// 16 bytes a lane from memory straight into LDS: lane i's land at `to` + 16 i.  In
// assembly, because the compiler lets no LDS read start while a direct load that it
// knows of is in flight; there is no result register, and wait_loads() is the wait.
__device__ __forceinline__ void lds_load16(const char* from, char* to) {
  const int at = (int)(uintptr_t)(FDM_LDS char*)to;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(from) : "memory");
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
// at most N of the wave's loads are still in flight, and none of its LDS reads
template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A row's 16-byte piece c lies at c ^ piece_swap(row): sixteen rows' same piece
// lie in sixteen bank groups.
__device__ __forceinline__ int piece_swap(int row) { return (row >> 1) & 7; }

// The request whose tokens row t is among; -1: none.
__device__ __forceinline__ int request_of(const int* q_start, int B, int t) {
  int lo = 0, hi = B + 1;  // the first b with q_start[b] > t, B + 1 if none
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (q_start[mid] <= t) lo = mid + 1;
    else hi = mid;
  }
  return lo <= B ? lo - 1 : -1;
}
__device__ __forceinline__ int adapter_of(const ProjectArgs& a, int t) {
  if (!a.n_adapters || t >= a.T) return -1;
  const int b = request_of(a.q_start, a.B, t);
  const int k = b < 0 ? -1 : a.adapter[b];
  return k < a.n_adapters ? k : -1;
}

}  // namespace

// ---- the adapters' first product: u_t = c_a A_a x_t ----------------------------------
// A workgroup takes up to 32 rows of one adapter, wherever they stand: all count the
// requests' rows by adapter in LDS, and the grid's y-th tile of the list (adapters in
// order, their rows in order) is found from that; tiles <= rows / 32 + adapters in use.
// Four waves share the part of the inner dimension; their sums meet in LDS.
template <int FMT, int RB>
__global__ __launch_bounds__(256) void k_adapter_in(ProjectArgs a) {
  __shared__ int count[kMaxAdapters];
  __shared__ int list[32];
  __shared__ int chosen[3];  // adapter, its first row of the tile, rows of the adapter
  __shared__ int of_wave[4];
  __shared__ float sums[4][32][36];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i < a.n_adapters; i += 256) count[i] = 0;
  if (tid == 0) chosen[0] = -1;
  if (tid < 32) list[tid] = -1;
  __syncthreads();
  for (int b = tid; b < a.B; b += 256) {
    const int k = a.adapter[b], t0 = min(max(a.q_start[b], 0), a.T), n = min(a.q_start[b + 1], a.T) - t0;
    if (k >= 0 && k < a.n_adapters && n > 0) atomicAdd(&count[k], n);
  }
  __syncthreads();
  // tiles before each adapter, four consecutive ones a thread
  int tiles = 0;
#pragma unroll
  for (int i = 0; i < kMaxAdapters / 256; ++i) {
    const int k = tid * (kMaxAdapters / 256) + i;
    if (k < a.n_adapters) tiles += (count[k] + 31) / 32;
  }
  int upto = tiles;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int v = __shfl_up(upto, d);
    if (lane >= d) upto += v;
  }
  if (lane == 63) of_wave[wave] = upto;
  __syncthreads();
  int before = upto - tiles;
  for (int w = 0; w < wave; ++w) before += of_wave[w];
  const int mine = blockIdx.y;
#pragma unroll
  for (int i = 0; i < kMaxAdapters / 256; ++i) {
    const int k = tid * (kMaxAdapters / 256) + i;
    if (k >= a.n_adapters) break;
    const int n = (count[k] + 31) / 32;
    if (mine >= before && mine < before + n) {
      chosen[0] = k;
      chosen[1] = 32 * (mine - before);
      chosen[2] = count[k];
    }
    before += n;
  }
  __syncthreads();
  const int k = chosen[0], row0 = chosen[1];
  if (k < 0) return;  // no such tile
  // the adapter's rows row0 .. row0 + 31
  int seen = 0;
  for (int b0 = 0; b0 < a.B && seen < row0 + 32; b0 += 256) {
    const int b = b0 + tid;
    int t0 = 0, n = 0;
    if (b < a.B && a.adapter[b] == k) {
      t0 = min(max(a.q_start[b], 0), a.T);
      n = max(min(a.q_start[b + 1], a.T) - t0, 0);
    }
    int sum = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(sum, d);
      if (lane >= d) sum += v;
    }
    __syncthreads();
    if (lane == 63) of_wave[wave] = sum;
    __syncthreads();
    int at = seen + sum - n;
    for (int w = 0; w < 4; ++w) {
      if (w < wave) at += of_wave[w];
      seen += of_wave[w];
    }
    for (int i = max(at, row0); i < min(at + n, row0 + 32); ++i) list[i - row0] = t0 + (i - at);
  }
  __syncthreads();

  typedef typename Half<FMT>::T T16;
  typedef typename Half<FMT>::x8 x8;
  const int r = lane & 31, h = lane >> 5;
  const int t = max(list[r], 0);
  const int units = (a.in + 15) / 16;  // of sixteen values; each lane has eight
  const int parts = gridDim.x * 4, part = blockIdx.x * 4 + wave;
  const int u0 = (int)((int64_t)units * part / parts), u1 = (int)((int64_t)units * (part + 1) / parts);
  const char* x = static_cast<const char*>(a.x) + (int64_t)t * a.x_bytes;
  const T16* A = static_cast<const T16*>(a.a) + (int64_t)k * a.rank * a.in;
  f32x16 acc[RB];
#pragma unroll
  for (int j = 0; j < RB; ++j)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[j][i] = 0.0f;
  for (int u = u0; u < u1; ++u) {
    const int at = 16 * u + 8 * h;
    x8 xv, av[RB];
#pragma unroll
    for (int i = 0; i < 8; ++i) xv[i] = (T16)0.0f;
#pragma unroll
    for (int j = 0; j < RB; ++j) av[j] = xv;
    if (at < a.in) {
      if constexpr (FMT == kRowFp8 || FMT == kRowFp8Wide) {
        const uint2 c = *reinterpret_cast<const uint2*>(x + at);
        const float s = scale_value(a.x_scale[(int64_t)t * a.x_scale_bytes + at / 128]);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint32_t word = w ? c.y : c.x;
          const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(word, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(word, true);
          xv[4 * w] = (T16)(lo[0] * s);  // exact: four bits of significand
          xv[4 * w + 1] = (T16)(lo[1] * s);
          xv[4 * w + 2] = (T16)(hi[0] * s);
          xv[4 * w + 3] = (T16)(hi[1] * s);
        }
      } else {
        xv = *reinterpret_cast<const x8*>(x + 2 * at);
      }
#pragma unroll
      for (int j = 0; j < RB; ++j) {
        const int row = 32 * j + r;
        if (row < a.rank) av[j] = *reinterpret_cast<const x8*>(A + (int64_t)row * a.in + at);
      }
    }
#pragma unroll
    for (int j = 0; j < RB; ++j) acc[j] = mfma16(av[j], xv, acc[j]);
  }
  const float c = a.times ? a.times[k] : 1.0f;
#pragma unroll
  for (int j = 0; j < RB; ++j) {
    // lane: row r, columns 8 q + 4 h + 0 .. 3 of the block
    if (j) __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<f32x4*>(&sums[wave][r][8 * q + 4 * h]) =
          f32x4{acc[j][4 * q], acc[j][4 * q + 1], acc[j][4 * q + 2], acc[j][4 * q + 3]};
    __syncthreads();
    for (int i = tid; i < 32 * 32; i += 256) {
      const int m = i / 32, col = i % 32;
      if (list[m] < 0 || 32 * j + col >= a.rank) continue;
      const float s = (sums[0][m][col] + sums[1][m][col]) + (sums[2][m][col] + sums[3][m][col]);
      a.u[((int64_t)blockIdx.x * a.T + list[m]) * a.rank + 32 * j + col] = s * c;
    }
  }
}

// ---- the projection --------------------------------------------------------------------
// The adapters' second product on a wave's sums: for every adapter among the 32 rows of
// a block, B_a u on the matrix cores, u as sums of 16-bit numbers (PLANES of them: 8 bits
// each in BF16, 11 in F16), kept by the rows that are the adapter's own.  A row that
// has another keeps its sum untouched, whatever B_a holds.
template <int FMT, int NB>
__device__ __forceinline__ void add_adapters(const ProjectArgs& a, int m, int id, int n0, f32x16* acc, int planes) {
  typedef typename Half<FMT>::T T16;
  typedef typename Half<FMT>::x8 x8;
  const int lane = threadIdx.x & 63, h = lane >> 5;
  uint64_t left = __ballot(id >= 0);
  const float* u = a.u + (int64_t)m * a.rank;
  // F16 planes: the row's largest brought to [1, 2), so that none overflows and few are lost
  float up = 1.0f, down = 1.0f;
  if constexpr (FMT == kRowF16) {
    float top = 0.0f;
    if (id >= 0)
      for (int j = 0; j < a.rank; ++j) top = fmaxf(top, fabsf(u[j]));
    const int e = min(max((int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127, -100), 100);
    up = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
    down = __builtin_bit_cast(float, (uint32_t)(127 + e) << 23);
  }
  while (left) {
    const int k = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    const bool mine = id == k;
    left &= ~__ballot(mine);
    const T16* B = static_cast<const T16*>(a.b) + (int64_t)k * a.out * a.rank;
    f32x16 sum[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int i = 0; i < 16; ++i) sum[nb][i] = 0.0f;
    for (int j0 = 0; j0 < a.rank; j0 += 16) {
      const int j = j0 + 8 * h;
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.0f;
      x8 bv[NB];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 8; ++i) bv[nb][i] = (T16)0.0f;
      if (j < a.rank) {
        if (mine) load8(u + j, true, v);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const int n = min(n0 + 32 * nb + (lane & 31), a.out - 1);
          bv[nb] = *reinterpret_cast<const x8*>(B + (int64_t)n * a.rank + j);
        }
      }
      for (int p = 0; p < planes; ++p) {
        x8 w;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (p == 0) v[i] *= up;
          w[i] = (T16)v[i];
          const float rest = v[i] - (float)w[i];
          v[i] = fabsf(rest) < __builtin_inff() ? rest : 0.0f;  // an infinity has no rest
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) sum[nb] = mfma16(bv[nb], w, sum[nb]);
      }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[nb][i] = mine ? fmaf(sum[nb][i], down, acc[nb][i]) : acc[nb][i];
  }
}

__device__ __forceinline__ float swap_halves(float lo, float hi, float* other) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi), false, false);
  *other = __builtin_bit_cast(float, (uint32_t)r[1]);
  return __builtin_bit_cast(float, (uint32_t)r[0]);
}

// Row m's columns n0 .. n0 + 31 of a block's sums: lane (m, h) has the columns
// 8 q + 4 h + 0 .. 3; the halves exchange so that each has eight neighbours twice.
template <typename TY>
__device__ __forceinline__ void store_block(TY* y, bool live, int n0, int out, bool vec, const f32x16& c) {
  const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = swap_halves(c[8 * p + i], c[8 * p + 4 + i], &v[4 + i]);
    const int n = n0 + 16 * p + 8 * h;
    if (!live) continue;
    if (vec && n + 8 <= out) {
      store8(y + n, true, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n + i < out) y[n + i] = (TY)v[i];
    }
  }
}

// A tile of 32 MB WM rows of x by 32 NB WN rows of the matrix, WM x WN waves, over the
// steps of its part.  Each step's 128 bytes of every row go straight into LDS (STAGES
// steps there at a time, so that STAGES - 1 are under way), and from there as operands:
// the matrix's rows first, so that a lane holds one row of the result.
template <int FMT, int MB, int NB, int WM, int WN, int STAGES>
__global__ __launch_bounds__(64 * WM * WN) void k_project(ProjectArgs a) {
  constexpr int kWaves = WM * WN, BM = 32 * MB * WM, BN = 32 * NB * WN, kRows = BM + BN;
  constexpr int kStage = kRows * kStepBytes;
  constexpr int kLoads = kRows / 8 / kWaves;  // of a wave and step, eight rows each
  static_assert(kRows % (8 * kWaves) == 0 && BM % 8 == 0, "whole loads");
  __shared__ __attribute__((aligned(16))) char lds[STAGES * kStage];
  __shared__ int ids[BM];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, h = lane >> 5;
  const int m_tiles = (a.T + BM - 1) / BM;
  const int tile = blockIdx.x;
  const int m0 = tile % m_tiles * BM, n0 = tile / m_tiles * BN;
  const int part = blockIdx.y;
  const int step0 = (int)((int64_t)a.steps * part / gridDim.y), step1 = (int)((int64_t)a.steps * (part + 1) / gridDim.y);

  // this wave's loads: their rows' addresses; rows past the end are the last one's again
  const char* from[kLoads];
  int piece[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int row = 8 * (wave * kLoads + i) + lane / 8;
    piece[i] = ((lane & 7) ^ piece_swap(row)) * 16;
    from[i] = row < BM ? static_cast<const char*>(a.x) + (int64_t)min(m0 + row, a.T - 1) * a.x_bytes
                       : static_cast<const char*>(a.w) + (int64_t)min(n0 + row - BM, a.out - 1) * a.w_bytes;
  }
  auto bring = [&](int step) {
    char* to = lds + (step % STAGES) * kStage + wave * kLoads * 1024;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = step * kStepBytes + piece[i];
      lds_load16(at < a.row_bytes ? from[i] + at : reinterpret_cast<const char*>(zeros16), to + 1024 * i);
    }
  };

  f32x16 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

  const int wm = wave / WN, wn = wave % WN;
  const int row_m = 32 * MB * wm + r, row_n = BM + 32 * NB * wn + r;  // in a stage
  const int swap = piece_swap(r);
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s)
    if (step0 + s < step1) bring(step0 + s);
  for (int step = step0; step < step1; ++step) {
    // (the last steps wait for everything: nothing is under way behind them)
    if (step + STAGES - 1 <= step1) wait_loads<(STAGES - 2) * kLoads>();
    else wait_loads<0>();
    barrier();
    if (step + STAGES - 1 < step1) bring(step + STAGES - 1);
    const char* stage = lds + (step % STAGES) * kStage;
    int xs[MB], ws[NB];
    if constexpr (FMT == kRowFp8 || FMT == kRowFp8Wide) {
#pragma unroll
      for (int i = 0; i < MB; ++i) xs[i] = a.x_scale[(int64_t)min(m0 + row_m + 32 * i, a.T - 1) * a.x_scale_bytes + step];
#pragma unroll
      for (int j = 0; j < NB; ++j) ws[j] = a.w_scale[(int64_t)(min(n0 + row_n - BM + 32 * j, a.out - 1) / 128) * a.w_scale_bytes + step];
    }
    if constexpr (FMT == kRowFp8Wide) {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int at = ((2 * s + h) ^ swap) << 4;
        bf16x8 xv[MB][2], wv[NB][2];
#pragma unroll
        for (int i = 0; i < MB; ++i) widen16(*reinterpret_cast<const i32x4*>(stage + (row_m + 32 * i) * kStepBytes + at), scale_value(xs[i]), xv[i]);
#pragma unroll
        for (int j = 0; j < NB; ++j) widen16(*reinterpret_cast<const i32x4*>(stage + (row_n + 32 * j) * kStepBytes + at), scale_value(ws[j]), wv[j]);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] = mfma16(wv[j][k], xv[i][k], acc[i][j]);
      }
    } else if constexpr (FMT == kRowFp8) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        auto operand = [&](int row) {
          const char* p = stage + row * kStepBytes;
          const i32x4 lo = *reinterpret_cast<const i32x4*>(p + (((4 * s + 2 * h) ^ swap) << 4));
          const i32x4 hi = *reinterpret_cast<const i32x4*>(p + (((4 * s + 2 * h + 1) ^ swap) << 4));
          return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        };
        i32x8 xv[MB], wv[NB];
#pragma unroll
        for (int i = 0; i < MB; ++i) xv[i] = operand(row_m + 32 * i);
#pragma unroll
        for (int j = 0; j < NB; ++j) wv[j] = operand(row_n + 32 * j);
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int j = 0; j < NB; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv[j], xv[i], acc[i][j], 0, 0, 0, ws[j], 0, xs[i]);
      }
    } else {
      typedef typename Half<FMT>::x8 x8;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int at = ((2 * s + h) ^ swap) << 4;
        x8 xv[MB], wv[NB];
#pragma unroll
        for (int i = 0; i < MB; ++i) xv[i] = *reinterpret_cast<const x8*>(stage + (row_m + 32 * i) * kStepBytes + at);
#pragma unroll
        for (int j = 0; j < NB; ++j) wv[j] = *reinterpret_cast<const x8*>(stage + (row_n + 32 * j) * kStepBytes + at);
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int j = 0; j < NB; ++j) acc[i][j] = mfma16(wv[j], xv[i], acc[i][j]);
      }
    }
  }

  const bool direct = a.part == nullptr;
  if (direct && a.n_adapters) {
    for (int i = tid; i < BM; i += 64 * kWaves) ids[i] = adapter_of(a, m0 + i);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int m = m0 + row_m + 32 * i, nb0 = n0 + row_n - BM - r;
    if (direct && a.n_adapters) add_adapters<FMT, NB>(a, m, ids[row_m + 32 * i], nb0, acc[i], a.planes);
    const bool live = m < a.T;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int n = nb0 + 32 * j;
      if (!direct) {
        store_block(a.part + ((int64_t)part * a.T + m) * a.out, live, n, a.out, a.vec_part, acc[i][j]);
      } else {
        char* y = static_cast<char*>(a.y) + (int64_t)m * a.y_bytes;
        if (a.y_type == ElemType::f32) store_block(reinterpret_cast<float*>(y), live, n, a.out, a.vec_y, acc[i][j]);
        else if (a.y_type == ElemType::f16) store_block(reinterpret_cast<_Float16*>(y), live, n, a.out, a.vec_y, acc[i][j]);
        else store_block(reinterpret_cast<__bf16*>(y), live, n, a.out, a.vec_y, acc[i][j]);
      }
    }
  }
}

// ---- parts and the adapters' second product, added -------------------------------------
// One row a workgroup of 256 columns; u in LDS.
template <int FMT>
__global__ __launch_bounds__(256) void k_project_join(ProjectArgs a) {
  typedef typename Half<FMT>::T T16;
  typedef typename Half<FMT>::x8 x8;
  __shared__ float u[kMaxRank];
  const int t = blockIdx.y, n = blockIdx.x * 256 + threadIdx.x;
  const int k = adapter_of(a, t);
  if (k >= 0)
    for (int j = threadIdx.x; j < a.rank; j += 256) {
      float s = 0.0f;
      for (int p = 0; p < a.u_splits; ++p) s += a.u[((int64_t)p * a.T + t) * a.rank + j];
      u[j] = s;
    }
  __syncthreads();
  if (n >= a.out) return;
  float y = 0.0f;
  for (int p = 0; p < a.splits; ++p) y += a.part[((int64_t)p * a.T + t) * a.out + n];
  if (k >= 0) {
    const T16* B = static_cast<const T16*>(a.b) + ((int64_t)k * a.out + n) * a.rank;
    float d = 0.0f;
    for (int j = 0; j < a.rank; j += 8) {
      const x8 v = *reinterpret_cast<const x8*>(B + j);
#pragma unroll
      for (int i = 0; i < 8; ++i) d = fmaf(u[j + i], (float)v[i], d);
    }
    y += d;
  }
  char* to = static_cast<char*>(a.y) + (int64_t)t * a.y_bytes;
  if (a.y_type == ElemType::f32) reinterpret_cast<float*>(to)[n] = y;
  else if (a.y_type == ElemType::f16) reinterpret_cast<_Float16*>(to)[n] = (_Float16)y;
  else reinterpret_cast<__bf16*>(to)[n] = (__bf16)y;
}

namespace {

template <int FMT>
hipError_t launch_adapter_in(const ProjectArgs& a, hipStream_t s) {
  const dim3 grid(a.u_splits, (a.T + 31) / 32 + std::min(a.B, a.n_adapters));
  if (a.rank <= 32) k_adapter_in<FMT, 1><<<grid, 256, 0, s>>>(a);
  else if (a.rank <= 64) k_adapter_in<FMT, 2><<<grid, 256, 0, s>>>(a);
  else k_adapter_in<FMT, 4><<<grid, 256, 0, s>>>(a);
  return hipGetLastError();
}

template <int FMT, int MB, int NB, int WM, int WN, int STAGES>
hipError_t launch_tiles(const ProjectArgs& a, hipStream_t s) {
  constexpr int BM = 32 * MB * WM, BN = 32 * NB * WN;
  const dim3 grid(((a.T + BM - 1) / BM) * ((a.out + BN - 1) / BN), a.splits);
  k_project<FMT, MB, NB, WM, WN, STAGES><<<grid, 64 * WM * WN, 0, s>>>(a);
  return hipGetLastError();
}

template <int FMT>
hipError_t launch_fmt(const ProjectArgs& a, const ProjectPlan& p, hipStream_t s) {
  hipError_t e = hipSuccess;
  if (a.n_adapters) e = launch_adapter_in<FMT>(a, s);
  if (e != hipSuccess) return e;
  switch (p.tile) {
    case kTile32: e = launch_tiles<FMT, 1, 1, 1, 4, 6>(a, s); break;
    case kTile64: e = launch_tiles<FMT, 2, 1, 1, 4, 5>(a, s); break;
    case kTile128: e = launch_tiles<FMT, 2, 2, 2, 2, 4>(a, s); break;
    default: e = launch_tiles<FMT, 4, 2, 2, 4, 2>(a, s);
  }
  if (e != hipSuccess || !p.join) return e;
  k_project_join<FMT><<<dim3((a.out + 255) / 256, a.T), 256, 0, s>>>(a);
  return hipGetLastError();
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
