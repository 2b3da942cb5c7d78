// norm_kernels.hip -- the residual's addition and its norm in one pass
// (fdm_add_rms_norm):
//   s = x + add,   y = s / sqrt(mean(s^2) + eps) * w,
// y in a wide type, or in e4m3 with a power-of-two scale for every 128 values.
#include "latent_device.h"

namespace fdm {

namespace {

constexpr int kNormGroup = 128;  // values of a row that share a scale: 16 threads' eight

// Eight values from `at` on of a row of d, zeros behind it.  `plain`: the row's type
// and alignment are what the kernel was made for; else value by value, of any type.
template <typename T>
__device__ __forceinline__ void load_row(const void* row, ElemType type, int at, int d, float* v) {
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = 0.0f;
  if constexpr (!std::is_void_v<T>) {
    if (at < d) load8(static_cast<const T*>(row) + at, true, v);
  } else {
    for (int k = 0; k < 8; ++k)
      if (at + k < d)
        v[k] = type == ElemType::f32 ? static_cast<const float*>(row)[at + k]
               : type == ElemType::f16 ? (float)static_cast<const _Float16*>(row)[at + k]
                                       : (float)static_cast<const __bf16*>(row)[at + k];
  }
}
__device__ __forceinline__ void store_row(void* row, ElemType type, bool vec, int at, int d, const float* v) {
  if (vec) {
    if (at >= d) return;
    if (type == ElemType::f32) store8(static_cast<float*>(row) + at, true, v);
    else if (type == ElemType::f16) store8(static_cast<_Float16*>(row) + at, true, v);
    else store8(static_cast<__bf16*>(row) + at, true, v);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (at + k < d) {
        if (type == ElemType::f32) static_cast<float*>(row)[at + k] = v[k];
        else if (type == ElemType::f16) static_cast<_Float16*>(row)[at + k] = (_Float16)v[k];
        else static_cast<__bf16*>(row)[at + k] = (__bf16)v[k];
      }
  }
}

// One row a workgroup of NT threads, eight consecutive values a thread and chunk,
// C chunks held in registers between the sum and the result, so that every value is
// read once.  TX, TA: the types of x and add where every row is 16-byte aligned and
// whole eights, void for any other call.
// Sums, the mean and the root are fp32; s is rounded where it is kept and where it is given,
// not between.  A scale's 128 values are sixteen lanes' of one chunk, whose maximum they exchange.
// Bound by memory: 16384 rows of 7168 BF16 values with an addition into codes 157 us, 5.24 TB/s (a
// copy of 1 GiB: 5.09).  16 rows of 7168 fp32 values 4.4 us of kernel: one chain of load, sum and
// store.
template <typename TX, typename TA, int NT, int C>
__global__ __launch_bounds__(NT) void k_add_rms_norm(NormArgs a) {
  constexpr bool kVec = !std::is_void_v<TX>;
  __shared__ float of_wave[NT / 64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t row = blockIdx.x;
  const char* x = static_cast<const char*>(a.x) + row * a.x_bytes;
  const char* add = static_cast<const char*>(a.add) + row * a.add_bytes;
  float v[C][8];
#pragma unroll
  for (int c = 0; c < C; ++c) load_row<TX>(x, a.x_type, 8 * (c * NT + tid), a.d, v[c]);
  if (a.add) {
    float u[C][8];
#pragma unroll
    for (int c = 0; c < C; ++c) load_row<TA>(add, a.add_type, 8 * (c * NT + tid), a.d, u[c]);
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int k = 0; k < 8; ++k) v[c][k] += u[c][k];
  }
  float s = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int k = 0; k < 8; ++k) s = fmaf(v[c][k], v[c][k], s);
  if (a.sum) {
    char* sum = static_cast<char*>(a.sum) + row * a.sum_bytes;
#pragma unroll
    for (int c = 0; c < C; ++c) store_row(sum, a.x_type, kVec, 8 * (c * NT + tid), a.d, v[c]);
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) s += __shfl_xor(s, m);
  if (NT > 64) {
    if (lane == 0) of_wave[tid >> 6] = s;
    __syncthreads();
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) s += of_wave[w];
  }
  const float inv = 1.0f / sqrtf(s / (float)a.d + a.eps);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int at = 8 * (c * NT + tid);
    if (a.w) {
      float w[8];
      if (kVec) load_row<float>(a.w, ElemType::f32, at, a.d, w);
      else load_row<void>(a.w, ElemType::f32, at, a.d, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[c][k] = (v[c][k] * inv) * w[k];
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[c][k] *= inv;
    }
    char* y = static_cast<char*>(a.y) + row * a.y_bytes;
    if (!a.scale) {
      store_row(y, a.y_type, kVec, at, a.d, v[c]);
      continue;
    }
    float m = 0.0f;  // places behind the row change no maximum
#pragma unroll
    for (int k = 0; k < 8; ++k) m = at + k < a.d ? amax_bits(m, v[c][k]) : m;
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) m = amax_bits(m, __shfl_xor(m, d));
    if (at >= a.d) continue;
    const int byte = fp8_scale_byte(m);
    uint32_t code[2];
    fp8_codes8(v[c], byte, code);
    if (kVec) {
      *reinterpret_cast<uint2*>(y + at) = make_uint2(code[0], code[1]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (at + k < a.d) reinterpret_cast<uint8_t*>(y)[at + k] = (uint8_t)(code[k / 4] >> (8 * (k % 4)));
    }
    if ((lane & 15) == 0) a.scale[row * a.scale_bytes + at / kNormGroup] = (uint8_t)byte;
  }
}

template <typename TX, typename TA>
hipError_t launch_of(const NormArgs& a, hipStream_t s) {
  const int chunks = (a.d + 7) / 8;
#define FDM_NORM(NT, C) k_add_rms_norm<TX, TA, NT, C><<<a.T, NT, 0, s>>>(a)
  // few rows: a chunk a thread, the shortest chain (16 rows of 7168: 4.4 us, with four chunks 6.2);
  // many: four a thread, more in flight where the workgroups fill the card anyway
  if (chunks <= 64) FDM_NORM(64, 1);
  else if (chunks <= 256) FDM_NORM(256, 1);
  else if (a.T <= g_num_cus && chunks <= 1024) FDM_NORM(1024, 1);
  else if (chunks <= 512) FDM_NORM(256, 2);
  else if (chunks <= 1024) FDM_NORM(256, 4);
  else if (chunks <= 2048) FDM_NORM(512, 4);
  else FDM_NORM(1024, 4);  // kNormMaxDim
#undef FDM_NORM
  return hipGetLastError();
}

}  // namespace

// An update in the residual's type or in BF16 moves by 16-byte accesses; any other
// pair of types, and rows that are not aligned, value by value: 16384 rows of 7168 fp32 values
// and F16 ones into codes 808 us (with BF16 ones 245), of 7167 BF16 values 687 (7168: 178).
hipError_t launch_add_rms_norm(const NormArgs& a, hipStream_t s) {
  const ElemType add = a.add ? a.add_type : a.x_type;
  if (a.vec && (add == a.x_type || add == ElemType::bf16)) {
    switch (a.x_type) {
      case ElemType::f32: return add == ElemType::f32 ? launch_of<float, float>(a, s) : launch_of<float, __bf16>(a, s);
      case ElemType::f16: return add == ElemType::f16 ? launch_of<_Float16, _Float16>(a, s) : launch_of<_Float16, __bf16>(a, s);
      default: return launch_of<__bf16, __bf16>(a, s);
    }
  }
  return launch_of<void, void>(a, s);
}

}  // namespace fdm
