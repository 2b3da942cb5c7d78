// kvcache_kernels.hip -- rows of the paged latent cache, written and read
// back.  A row is 512 latent values (keys and values at once) and 64 rotary
// ones (keys).  Three planes, each [n_pages][page_size][..]: latent, rotary
// part, and for FP8 rows four scale bytes.
#include "latent_device.h"

namespace fdm {

namespace {

// One wave a row, eight consecutive latent values a lane: a group of 128 is
// 16 lanes.
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m);
  return v;
}

}  // namespace

// x[576] -> n = x[:512] / sqrt(mean(x[:512]^2) + 1e-6) * w (or x[:512] as it
// is), r = x[512:] turned by the row's position (or as it is), into the row's
// slot.  F16 / BF16: rounded to nearest even.  FP8: per 128 latent values the
// power-of-two scale of fp8_scale_byte, n 2^-e rounded to e4m3; r in bf16.
// Power-of-two scales make n 2^-e and what is read back exact: the code is
// the only rounding.
// One wave a row, so that the norm's sum and a group's maximum stay in registers
// and need no barrier, four rows a workgroup.  Bound by memory: 32768 fp32 rows
// into BF16 23.9 us a call, 113 MB at 4.75 TB/s; 64 rows are 4 us of kernel (load,
// sum, rotation, store one after the other) and the host's 6 us a call.
template <typename TX, int FMT>
__global__ __launch_bounds__(256) void k_kv_write(KvWriteArgs a) {
  const int lane = threadIdx.x & 63;
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.T) return;
  const int slot = a.slots[row];
  if (slot < 0 || slot >= a.rows) return;  // a padding row, or no row of this cache
  const TX* x = static_cast<const TX*>(a.x) + (int64_t)row * a.x_stride;
  float v[8], rot[2] = {0.0f, 0.0f};
  load8(x + 8 * lane, a.vec_x, v);
  const int layout = a.table.layout;
  const int iu = kLatDim + (layout ? (lane & 31) : 2 * (lane & 31)), iv = layout ? iu + 32 : iu + 1;
  if (lane < 32) {
    rot[0] = (float)x[iu];
    rot[1] = (float)x[iv];
  }
  if (a.norm_w) {
    float w[8], s = 0.0f;
    load8(a.norm_w + 8 * lane, a.vec_w, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) s = fmaf(v[k], v[k], s);
    s = wave_sum(s);
    const float inv = 1.0f / sqrtf(s / (float)kLatDim + 1e-6f);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = (v[k] * inv) * w[k];
  }
  if (a.rotate && lane < 32) {
    float s, c;
    turn_sincos((uint64_t)(int64_t)a.pos[row] * a.table.turns[lane], &s, &c);
    s *= a.table.mul;
    c *= a.table.mul;
    const float p = rot[0], q = rot[1];
    rot[0] = p * c - q * s;
    rot[1] = p * s + q * c;
  }
  const size_t at = (size_t)slot;
  if constexpr (FMT == kKvFp8) {
    float m = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = amax_bits(m, v[k]);
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) m = amax_bits(m, __shfl_xor(m, d));
    const int byte = fp8_scale_byte(m);
    const float inv = scale_value(byte == kScaleNan ? 127 : 254 - byte);  // 2^-e
    uint32_t code[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float q[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j] = fminf(fmaxf(v[4 * k + j] * inv, -448.0f), 448.0f);
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
      code[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
    }
    if (byte == kScaleNan) code[0] = code[1] = 0x7F7F7F7Fu;  // e4m3's NaN
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.latent) + at * kLatDim + 8 * lane) = make_uint2(code[0], code[1]);
    if ((lane & 15) == 0) a.scale[at * 4 + (lane >> 4)] = (uint8_t)byte;
    if (lane < 32) {
      __bf16* r = static_cast<__bf16*>(a.rope) + at * kRotDim - kLatDim;
      r[iu] = (__bf16)rot[0];
      r[iv] = (__bf16)rot[1];
    }
  } else {
    typedef std::conditional_t<FMT == kKvF16, _Float16, __bf16> T;
    store8(static_cast<T*>(a.latent) + at * kLatDim + 8 * lane, true, v);
    if (lane < 32) {
      T* r = static_cast<T*>(a.rope) + at * kRotDim - kLatDim;
      r[iu] = (T)rot[0];
      r[iv] = (T)rot[1];
    }
  }
}

// The row's values, widened: code 2^e and the rotary part, rounded once to
// the output's type.  Rows whose slot is none of the cache's are left as they
// were.  Bound by memory: 16384 FP8 rows into BF16 6.6 us, 29.5 MB at 4.4 TB/s;
// 1000 rows are 2.9 us of kernel and the host's 5.5 us a call.
template <typename TY, int FMT>
__global__ __launch_bounds__(256) void k_kv_read(KvReadArgs a) {
  const int lane = threadIdx.x & 63;
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.T) return;
  const int slot = a.slots[row];
  if (slot < 0 || slot >= a.rows) return;
  const size_t at = (size_t)slot;
  TY* y = static_cast<TY*>(a.y) + (int64_t)row * a.y_stride;
  float v[8], r[8];
  if constexpr (FMT == kKvFp8) {
    const uint2 c = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.latent) + at * kLatDim + 8 * lane);
    const float s = scale_value(a.scale[at * 4 + (lane >> 4)]);
    if (lane < 8) load8(static_cast<const __bf16*>(a.rope) + at * kRotDim + 8 * lane, true, r);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t w = k ? c.y : c.x;
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
      v[4 * k] = lo[0] * s;
      v[4 * k + 1] = lo[1] * s;
      v[4 * k + 2] = hi[0] * s;
      v[4 * k + 3] = hi[1] * s;
    }
  } else {
    typedef std::conditional_t<FMT == kKvF16, _Float16, __bf16> T;
    load8(static_cast<const T*>(a.latent) + at * kLatDim + 8 * lane, true, v);
    if (lane < 8) load8(static_cast<const T*>(a.rope) + at * kRotDim + 8 * lane, true, r);
  }
  store8(y + 8 * lane, a.vec_y, v);
  if (lane < 8) store8(y + kLatDim + 8 * lane, a.vec_y, r);
}

hipError_t launch_kv_write(const KvWriteArgs& a, int fmt, ElemType x, hipStream_t s) {
  const int wgs = (a.T + 3) / 4;
#define FDM_KV_WRITE(TX)                                                        \
  switch (fmt) {                                                                \
    case kKvF16: k_kv_write<TX, kKvF16><<<wgs, 256, 0, s>>>(a); break;          \
    case kKvBf16: k_kv_write<TX, kKvBf16><<<wgs, 256, 0, s>>>(a); break;        \
    default: k_kv_write<TX, kKvFp8><<<wgs, 256, 0, s>>>(a);                     \
  }
  switch (x) {
    case ElemType::f32: FDM_KV_WRITE(float) break;
    case ElemType::f16: FDM_KV_WRITE(_Float16) break;
    case ElemType::bf16: FDM_KV_WRITE(__bf16) break;
  }
#undef FDM_KV_WRITE
  return hipGetLastError();
}

hipError_t launch_kv_read(const KvReadArgs& a, int fmt, ElemType y, hipStream_t s) {
  const int wgs = (a.T + 3) / 4;
#define FDM_KV_READ(TY)                                                         \
  switch (fmt) {                                                                \
    case kKvF16: k_kv_read<TY, kKvF16><<<wgs, 256, 0, s>>>(a); break;           \
    case kKvBf16: k_kv_read<TY, kKvBf16><<<wgs, 256, 0, s>>>(a); break;         \
    default: k_kv_read<TY, kKvFp8><<<wgs, 256, 0, s>>>(a);                      \
  }
  switch (y) {
    case ElemType::f32: FDM_KV_READ(float) break;
    case ElemType::f16: FDM_KV_READ(_Float16) break;
    case ElemType::bf16: FDM_KV_READ(__bf16) break;
  }
#undef FDM_KV_READ
  return hipGetLastError();
}

}  // namespace fdm
