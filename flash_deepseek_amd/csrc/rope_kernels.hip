// rope_kernels.hip -- rotary positions: of each head's D values the R from
// `offset` on are turned in pairs, (u, v) -> mul (u cos a - v sin a,
// u sin a + v cos a) with a = position x frequency of the pair; pairs are
// (2 i, 2 i + 1) or (i, i + R / 2).  The others pass through.  Every head of
// a token turns by the same angles.
#include "latent_device.h"

namespace fdm {

// A workgroup takes `tpw` tokens.  Their R / 2 sines and cosines are computed
// once into LDS; then a thread walks (token, head, item), an item being eight
// consecutive values (two runs of eight, R / 2 apart, for rotated ones in the
// half layout), so a 16-bit head moves by 16-byte accesses.  Values that pass
// through are items too, unless the call is in place.
// Bound by memory: 4097 tokens of 64 x 128 BF16 values 27.5 us a call, 134 MB
// at 4.9 TB/s, where a large copy reaches 5.1.  A step of 16 tokens is 3 us of
// kernel and the host's 6 us a call.
template <typename TX, typename TY, bool HALF, int N>
__global__ __launch_bounds__(256) void k_rope(RopeArgs a, RopeTurns<N> table) {
  extern __shared__ float2 sc[];  // [tpw][R / 2] (sine, cosine)
  const int t0 = blockIdx.x * a.tpw, nt = min(a.tpw, a.T - t0);
  const int half = table.dim / 2;
  for (int i = threadIdx.x; i < nt * half; i += 256) {
    const int t = i / half, p = i - t * half;
    const uint64_t turns = (uint64_t)(int64_t)a.pos[t0 + t] * table.turns[p];
    float s, c;
    turn_sincos(turns, &s, &c);
    sc[i] = make_float2(s * table.mul, c * table.mul);
  }
  __syncthreads();
  const bool vx = a.vec_x, vy = a.vec_y;
  const int rot_items = HALF ? half / 8 : half / 4;  // whole items; a tail of pairs follows
  const int rot_done = rot_items * (HALF ? 8 : 4);   // pairs they cover
  const int tail = half - rot_done;                  // pairs one by one
  const int before = a.offset, behind = a.D - a.offset - table.dim;
  const int pass0 = a.pass ? (before + 7) / 8 : 0, pass1 = a.pass ? (behind + 7) / 8 : 0;
  const int items = rot_items + tail + pass0 + pass1;
  const int total = nt * a.H * items;
  const int h0 = blockIdx.y;
  for (int i = h0 * 256 + threadIdx.x; i < total; i += 256 * gridDim.y) {
    const int row = i / items;
    int it = i - row * items;
    const int t = row / a.H, h = row - t * a.H;
    const TX* x = static_cast<const TX*>(a.x) + (int64_t)(t0 + t) * a.x_token + (int64_t)h * a.x_head;
    TY* y = static_cast<TY*>(a.y) + (int64_t)(t0 + t) * a.y_token + (int64_t)h * a.y_head;
    if (it < rot_items) {
      float u[8], v[8];
      if constexpr (HALF) {
        const int at = a.offset + 8 * it;
        load8(x + at, vx, u);
        load8(x + at + half, vx, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float2 w = sc[t * half + 8 * it + k];
          const float p = u[k], q = v[k];
          u[k] = p * w.y - q * w.x;
          v[k] = p * w.x + q * w.y;
        }
        store8(y + at, vy, u);
        store8(y + at + half, vy, v);
      } else {
        const int at = a.offset + 8 * it;
        load8(x + at, vx, u);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 w = sc[t * half + 4 * it + k];
          const float p = u[2 * k], q = u[2 * k + 1];
          u[2 * k] = p * w.y - q * w.x;
          u[2 * k + 1] = p * w.x + q * w.y;
        }
        store8(y + at, vy, u);
      }
      continue;
    }
    it -= rot_items;
    if (it < tail) {
      const int p = rot_done + it;
      const int iu = a.offset + (HALF ? p : 2 * p), iv = HALF ? iu + half : iu + 1;
      const float2 w = sc[t * half + p];
      const float u = (float)x[iu], v = (float)x[iv];
      y[iu] = (TY)(u * w.y - v * w.x);
      y[iv] = (TY)(u * w.x + v * w.y);
      continue;
    }
    it -= tail;
    const bool first = it < pass0;
    const int at = first ? 8 * it : a.offset + table.dim + 8 * (it - pass0);
    const int n = min(8, (first ? a.offset : a.D) - at);
    // behind the rotated part the run starts where that ends: aligned if R is
    if (n == 8 && (first || a.vec_behind)) {
      float u[8];
      load8(x + at, vx, u);
      store8(y + at, vy, u);
    } else {
      for (int k = 0; k < n; ++k) y[at + k] = (TY)(float)x[at + k];
    }
  }
}

namespace {
template <typename TX, typename TY, int N>
void launch_layout(const RopeArgs& a, const RopeTable& table, dim3 grid, size_t lds, hipStream_t s) {
  RopeTurns<N> t;
  t.dim = table.dim;
  t.layout = table.layout;
  t.mul = table.mul;
  for (int i = 0; i < N; ++i) t.turns[i] = table.turns[i];
  if (table.layout)
    k_rope<TX, TY, true, N><<<grid, 256, lds, s>>>(a, t);
  else
    k_rope<TX, TY, false, N><<<grid, 256, lds, s>>>(a, t);
}
template <typename TX, int N>
void launch_to(const RopeArgs& a, const RopeTable& table, dim3 grid, size_t lds, hipStream_t s) {
  switch (a.y_type) {
    case ElemType::f32: return launch_layout<TX, float, N>(a, table, grid, lds, s);
    case ElemType::f16: return launch_layout<TX, _Float16, N>(a, table, grid, lds, s);
    case ElemType::bf16: return launch_layout<TX, __bf16, N>(a, table, grid, lds, s);
  }
}
template <int N>
void launch_from(const RopeArgs& a, const RopeTable& table, dim3 grid, size_t lds, hipStream_t s) {
  switch (a.x_type) {
    case ElemType::f32: return launch_to<float, N>(a, table, grid, lds, s);
    case ElemType::f16: return launch_to<_Float16, N>(a, table, grid, lds, s);
    case ElemType::bf16: return launch_to<__bf16, N>(a, table, grid, lds, s);
  }
}
}  // namespace

hipError_t launch_rope(RopeArgs a, const RopeTable& table, hipStream_t s) {
  const int half = table.dim / 2;
  const int per_token = a.H * ((a.D + 7) / 8);  // items of a token, about
  a.tpw = max(1, min(1024 / per_token, 2048 / half));
  const int wgs = (a.T + a.tpw - 1) / a.tpw;
  // few tokens: several workgroups share one token's heads
  const int split = max(1, min((a.tpw * per_token + 255) / 256, 2 * g_num_cus / wgs));
  const dim3 grid(wgs, split);
  const size_t lds = (size_t)a.tpw * half * sizeof(float2);
  if (half <= 32)
    launch_from<32>(a, table, grid, lds, s);
  else
    launch_from<kRopeMaxDim / 2>(a, table, grid, lds, s);
  return hipGetLastError();
}

}  // namespace fdm
