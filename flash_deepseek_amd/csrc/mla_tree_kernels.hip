// mla_tree_kernels.hip -- latent attention of several sequences' query tokens
// over the paged cache (fdm_mla_attend).
//   s_ij = scale (q_lat_i . c_j + q_rope_i . r_j) over the positions j that
//   token i sees, p = softmax(s), o_i = sum_j p_ij c_j, lse_i = log sum exp.
// Position j of a sequence of len positions with n tokens is seen if it
// stands before the tokens (j < len - n), or if bit j - (len - n) of the
// token's mask is set; without a mask, if it does not stand behind token i's
// own place len - n + i.
#include "latent_device.h"

namespace fdm {

namespace {

__device__ __forceinline__ bool tree_sees(const MlaTreeArgs& a, int token, int place, int64_t prefix, int64_t j) {
  const int64_t d = j - prefix;
  if (d < 0) return true;
  if (!a.mask) return d <= place;
  if (d >= 64 * (int64_t)a.mask_words) return false;
  return (a.mask[(size_t)token * a.mask_words + (d >> 6)] >> (d & 63)) & 1;
}

template <int FMT>
__device__ __forceinline__ float cache_value(const MlaTreeArgs& a, int64_t slot, int d) {
  if constexpr (FMT == kKvFp8) {
    const float s = scale_value(a.scale[slot * 4 + d / kLatGroup]);
    return __builtin_amdgcn_cvt_f32_fp8(static_cast<const uint8_t*>(a.latent)[slot * kLatDim + d], 0) * s;
  } else if constexpr (FMT == kKvF16) {
    return (float)static_cast<const _Float16*>(a.latent)[slot * kLatDim + d];
  } else {
    return (float)static_cast<const __bf16*>(a.latent)[slot * kLatDim + d];
  }
}

}  // namespace

// One workgroup a (token, head): 256 positions at a time, a score a thread,
// then two latent dims a thread over the chunk's positions.
template <int FMT>
__global__ __launch_bounds__(256) void k_mla_tree_plain(MlaTreeArgs a) {
  typedef std::conditional_t<FMT == kKvF16, _Float16, __bf16> T;
  __shared__ float q[kLatDim + kRotDim], red[4], ps[256];
  __shared__ int slots[256];
  const int token = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  int b = -1;
  for (int k = 0; k < a.B; ++k)
    if (token >= a.q_start[k] && token < a.q_start[k + 1]) {
      b = k;
      break;
    }
  if (b < 0) return;
  const int place = token - a.q_start[b];
  const int64_t len = min(max(a.kv_len[b], 0), a.max_len);
  const int64_t prefix = len - (a.q_start[b + 1] - a.q_start[b]);
  const T* ql = static_cast<const T*>(a.q_lat) + token * a.ql_token + h * a.ql_head;
  const T* qr = static_cast<const T*>(a.q_rope) + token * a.qr_token + h * a.qr_head;
  for (int d = tid; d < kLatDim; d += 256) q[d] = (float)ql[d];
  if (tid < kRotDim) q[kLatDim + tid] = (float)qr[tid];
  float m = -__builtin_inff(), was = m, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
  for (int64_t j0 = 0; j0 < len; j0 += 256) {
    __syncthreads();
    const int64_t j = j0 + tid;
    int slot = -1;
    if (j < len && tree_sees(a, token, place, prefix, j)) {
      const int page = a.pages[(size_t)b * a.pages_stride + (j >> a.page_shift)];
      if (page >= 0 && page < a.n_pages) slot = (page << a.page_shift) + (int)(j & ((1 << a.page_shift) - 1));
    }
    float s = -__builtin_inff();
    if (slot >= 0) {
      s = 0.0f;
      for (int d = 0; d < kLatDim; ++d) s = fmaf(q[d], cache_value<FMT>(a, slot, d), s);
      const T* r = static_cast<const T*>(a.rope) + (size_t)slot * kRotDim;
      for (int d = 0; d < kRotDim; ++d) s = fmaf(q[kLatDim + d], (float)r[d], s);
      s *= a.scale_log2;
    }
    slots[tid] = slot;
    float c = s;
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) c = fmaxf(c, __shfl_xor(c, k));
    if ((tid & 63) == 0) red[tid >> 6] = c;
    __syncthreads();
    c = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    m = fmaxf(m, c);
    const float top = m == -__builtin_inff() ? 0.0f : m;  // nothing but -infinity or NaN so far
    const float keep = exp2f(was - top);
    ps[tid] = slot >= 0 ? exp2f(s - top) : 0.0f;
    __syncthreads();
    was = m;
    l *= keep;
    o0 *= keep;
    o1 *= keep;
    for (int k = 0; k < 256; ++k) {
      if (slots[k] < 0) continue;
      const float p = ps[k];
      l += p;
      o0 = fmaf(p, cache_value<FMT>(a, slots[k], tid), o0);
      o1 = fmaf(p, cache_value<FMT>(a, slots[k], tid + 256), o1);
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  T* out = static_cast<T*>(a.out) + token * a.out_token + h * a.out_head;
  out[tid] = (T)(o0 * inv);
  out[tid + 256] = (T)(o1 * inv);
  if (a.lse && tid == 0)
    a.lse[(size_t)token * a.H + h] = l == 0.0f ? -__builtin_inff() : (m + log2f(l)) * 0.6931471805599453f;
}

size_t mla_tree_workspace(int N, int H) {
  (void)N;
  (void)H;
  return 256;
}

hipError_t launch_mla_tree(const MlaTreeArgs& a, int fmt, hipStream_t s) {
  const dim3 grid(a.N, a.H);
  switch (fmt) {
    case kKvF16: k_mla_tree_plain<kKvF16><<<grid, 256, 0, s>>>(a); break;
    case kKvBf16: k_mla_tree_plain<kKvBf16><<<grid, 256, 0, s>>>(a); break;
    default: k_mla_tree_plain<kKvFp8><<<grid, 256, 0, s>>>(a);
  }
  return hipGetLastError();
}

}  // namespace fdm
