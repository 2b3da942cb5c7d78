// kvpages_kernels.hip -- the books of the paged latent cache: which pages a
// sequence has, which are free, and where a step's tokens go.
//   free[0 .. n_free - 1] is a stack.  Sequence b holds the pages
//   pages[b][0 .. ceil(kv_len[b] / page) - 1].
// Pages are taken from the stack's top in the order of (sequence, page) and given
// back in the opposite one, so that what a call took and another gives back leaves
// the stack as it was, and the same calls give the same pages.
#include "fdm_internal.h"

namespace fdm {

namespace {

// Exclusive sums over the workgroup's threads, N of them at a time; total gets the sums of all.
template <int NT, int N, typename T>
struct Scan {
  T of_wave[NT / 64][N];
  __device__ __forceinline__ void operator()(T (&v)[N], T (&total)[N]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T upto[N];
#pragma unroll
    for (int n = 0; n < N; ++n) upto[n] = v[n];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1)
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const T below = __shfl_up(upto[n], d);
        if (lane >= d) upto[n] += below;
      }
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (lane == 63) of_wave[wave][n] = upto[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n] = upto[n] - v[n];
      total[n] = 0;
#pragma unroll
      for (int w = 0; w < NT / 64; ++w) {
        if (w < wave) v[n] += of_wave[w][n];
        total[n] += of_wave[w][n];
      }
    }
  }
};

// The last b of start[0 .. B] (not falling) with start[b] <= i.
__device__ __forceinline__ int owner(const int* start, int B, int i) {
  int lo = 0, hi = B;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (start[mid] <= i) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ int pages_for(int len, int shift) { return (int)(((int64_t)len + (1 << shift) - 1) >> shift); }

// Whether this workgroup is the last of the launch to come here: the others have
// read the state that it may now change.  The word counts up to the workgroups
// and starts again.
__device__ __forceinline__ bool is_last(unsigned* turn, int* said) {
  if (gridDim.x == 1) {
    __syncthreads();
    return true;
  }
  __syncthreads();
  if (threadIdx.x == 0) *said = atomicInc(turn, gridDim.x - 1) == gridDim.x - 1;
  __syncthreads();
  return *said;
}

}  // namespace

// Every workgroup counts all sequences itself (B <= 4096, four a thread at most), so that one
// launch needs no second one behind it; the last one to come to its end changes the
// state that the others read.  A thread gives four places at a time: the first's sequence is
// searched for in LDS and its page read, the others mostly share them; the first token of a
// new page names the page in the table.
// Bound by latency, a chain of loads and scans: 64 sequences of up to four tokens 5.0 us of
// kernel, 786,000 tokens of 512 sequences on pages of 16 10.2 (their 6.3 MB take 1.2).
template <int NT>
__global__ __launch_bounds__(NT) void k_kv_grow(KvPagesArgs a, KvGrowArgs g) {
  __shared__ int start[kKvMaxSeqs + 1], first[kKvMaxSeqs], len[kKvMaxSeqs];
  __shared__ Scan<NT, 2, int64_t> wide;
  __shared__ Scan<NT, 3, int> narrow;
  __shared__ int said;
  const int tid = threadIdx.x, per = (a.B + NT - 1) / NT, b0 = tid * per, b1 = min(b0 + per, a.B);
  const int n_free = min(max(*a.n_free, 0), a.n_pages);
  // what the sequences that have room ask for, up to each: pages, tokens
  int64_t asked[2] = {0, 0}, all64[2];
  for (int b = b0; b < b1; ++b) {
    const int l = min(max(a.kv_len[b], 0), a.max_len), n = max(g.more[b], 0);
    const bool room = n <= a.max_len - l;
    len[b] = l;
    start[b] = room ? n : -1;
    first[b] = room ? pages_for(l + n, a.shift) - pages_for(l, a.shift) : 0;
    asked[0] += first[b];
    asked[1] += room ? n : 0;
  }
  wide(asked, all64);
  // who is served: tokens, pages, and those who are not
  int got[3] = {0, 0, 0}, all[3];
  for (int b = b0; b < b1; ++b) {
    const int n = start[b], need = first[b];
    asked[0] += need;
    asked[1] += max(n, 0);
    const bool served = n >= 0 && (need == 0 || asked[0] <= n_free) && asked[1] <= g.N;
    got[2] += !served && n != 0;
    start[b] = served ? n : 0;
    first[b] = served ? need : 0;
    got[0] += start[b];
    got[1] += first[b];
  }
  narrow(got, all);
  const int total = all[0];
  for (int b = b0; b < b1; ++b) {
    const int n = start[b], need = first[b];
    start[b] = got[0];
    first[b] = got[1];
    got[0] += n;
    got[1] += need;
  }
  if (tid == 0) start[a.B] = total;
  __syncthreads();
  const int inside = (1 << a.shift) - 1;
  for (int64_t t0 = 4 * ((int64_t)blockIdx.x * NT + tid); t0 < g.N; t0 += (int64_t)4 * NT * gridDim.x) {
    int pos[4], slot[4];
    int b = t0 < total ? owner(start, a.B, (int)t0) : 0, page = -1;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t t = t0 + k;
      pos[k] = 0;
      slot[k] = -1;
      if (t < total) {
        bool same = k > 0;
        while (start[b + 1] <= t) ++b, same = false;
        pos[k] = len[b] + (int)(t - start[b]);
        const int at = pos[k] & inside;
        if (!same || at == 0) {
          const int p = pos[k] >> a.shift, have = pages_for(len[b], a.shift);
          int* entry = a.pages + (int64_t)b * a.P + p;
          page = p < have ? *entry : a.free[n_free - 1 - (first[b] + p - have)];
          if (p >= have && at == 0) *entry = page;
        }
        if (page >= 0 && page < a.n_pages) slot[k] = (page << a.shift) | at;
      }
    }
    if (g.vec && t0 + 4 <= g.N) {
      *reinterpret_cast<int4*>(g.pos + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      *reinterpret_cast<int4*>(g.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (t0 + k < g.N) {
          g.pos[t0 + k] = pos[k];
          g.slots[t0 + k] = slot[k];
        }
    }
  }
  if (!is_last(a.turn, &said)) return;
  for (int b = b0; b < b1; ++b) {
    g.q_start[b] = start[b];
    a.kv_len[b] = len[b] + start[b + 1] - start[b];
  }
  if (tid == 0) {
    g.q_start[a.B] = total;
    *a.n_free = n_free - all[1];
    if (g.refused) *g.refused = all[2];
  }
}

// The pages behind what each sequence keeps, onto the stack; one launch as above.
template <int NT>
__global__ __launch_bounds__(NT) void k_kv_trim(KvPagesArgs a, const int* keep) {
  __shared__ int before[kKvMaxSeqs + 1], stay[kKvMaxSeqs], len[kKvMaxSeqs];
  __shared__ Scan<NT, 1, int> scan;
  __shared__ int said;
  const int tid = threadIdx.x, per = (a.B + NT - 1) / NT, b0 = tid * per, b1 = min(b0 + per, a.B);
  const int n_free = min(max(*a.n_free, 0), a.n_pages);
  int at[1] = {0}, all[1];
  for (int b = b0; b < b1; ++b) {
    const int l = min(max(a.kv_len[b], 0), a.max_len), k = keep[b] < 0 ? l : min(keep[b], l);
    len[b] = k;
    stay[b] = pages_for(k, a.shift);
    before[b] = pages_for(l, a.shift) - stay[b];
    at[0] += before[b];
  }
  scan(at, all);
  const int total = all[0];
  for (int b = b0; b < b1; ++b) {
    const int n = before[b];
    before[b] = at[0];
    at[0] += n;
  }
  if (tid == 0) before[a.B] = total;
  __syncthreads();
  for (int64_t i = (int64_t)blockIdx.x * NT + tid; i < total; i += (int64_t)NT * gridDim.x) {
    const int b = owner(before, a.B, (int)i);
    const int64_t to = (int64_t)n_free + total - 1 - i;
    if (to < a.n_pages) a.free[to] = a.pages[(int64_t)b * a.P + stay[b] + (i - before[b])];
  }
  if (!is_last(a.turn, &said)) return;
  for (int b = b0; b < b1; ++b) a.kv_len[b] = len[b];
  if (tid == 0) *a.n_free = (int)min((int64_t)n_free + total, (int64_t)a.n_pages);
}

// Few sequences and places: workgroups of four waves, whose scans are the shorter (64 sequences of
// up to four tokens: grow 5.0 us, with sixteen waves 6.4; trim 3.2 and 3.4); else of sixteen,
// of which fewer follow each other at the last word (512 sequences, 786,000 tokens: 13.5 us and
// 10.2; 140,000 pages of 16 given back 7.0 and 5.2).  A workgroup for every four places a thread (of the table, of
// which a call seldom gives back much, four entries), one a CU at most.
hipError_t launch_kv_grow(const KvPagesArgs& a, const KvGrowArgs& g, hipStream_t s) {
  const auto wgs = [&](int threads) {
    return (int)std::min<int64_t>(std::max<int64_t>(((int64_t)g.N + 4 * threads - 1) / (4 * threads), 1), g_num_cus);
  };
  if (a.B <= 1024 && g.N <= 4096) k_kv_grow<256><<<wgs(256), 256, 0, s>>>(a, g);
  else k_kv_grow<1024><<<wgs(1024), 1024, 0, s>>>(a, g);
  return hipGetLastError();
}
hipError_t launch_kv_trim(const KvPagesArgs& a, const int* keep, hipStream_t s) {
  const int64_t entries = (int64_t)a.B * a.P;
  const auto wgs = [&](int per) { return (int)std::min<int64_t>((entries + per - 1) / per, g_num_cus); };
  if (a.B <= 1024 && entries <= 16384) k_kv_trim<256><<<wgs(4096), 256, 0, s>>>(a, keep);
  else k_kv_trim<1024><<<wgs(4096), 1024, 0, s>>>(a, keep);
  return hipGetLastError();
}

}  // namespace fdm
