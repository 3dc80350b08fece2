// Attention of each sequence's new tokens over its paged key/value cache.
//
// Sequence s has n = q_start[s+1] - q_start[s] new tokens (rows of q) and L = kv_lens[s]
// cached tokens, the new ones included: new token i sits at position L - n + i and sees
// keys (position - window, position] (window 0: all of [0, position]).
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - max);  lse2 = log2 sum exp
// A row that sees no key (L < n, or an unused batch slot) gives o = 0, lse2 = -inf.
//
// One warp per (token, head): the lanes hold the head dimension, 4 keys at a time.
#include <math_constants.h>

#include "common.cuh"
#include "kernels.h"
#include "serving.h"

namespace rt {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct Params {
  PagedAttnArgs a;
  int64_t n_rows;  // cache rows: pages x kv_heads x page_size
  int page_shift;
  float scale_log2;
};

// Keys [lo, hi) of one head for one row, one warp: running max m (log2 domain), sum l
// and the lane's HD / 32 entries of the unnormalised output.
template <int HD, bool I8>
__device__ void row_attend(const PagedAttnArgs& a, int page_shift, const int32_t* table, int kvh, const float (&q)[HD / 32],
                           int lo, int hi, float scale_log2, float& m, float& l, float (&o)[HD / 32]) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31;
  for (int j = lo; j < hi; ++j) {
    int64_t page = table[j >> page_shift];
    if (page < 0 || page >= a.cache.num_pages) {
      if (lane == 0) set_error(a.err, kDevBadIndex);
      page = 0;
    }
    const int64_t at = (((page * a.cache.kv_heads + kvh) << page_shift) + (j & ((1 << page_shift) - 1)));
    float k[E], v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int64_t i = at * HD + lane * E + e;
      if (I8) {
        k[e] = static_cast<float>(static_cast<const int8_t*>(a.cache.k)[i]);
        v[e] = static_cast<float>(static_cast<const int8_t*>(a.cache.v)[i]);
      } else {
        k[e] = __bfloat162float(static_cast<const __nv_bfloat16*>(a.cache.k)[i]);
        v[e] = __bfloat162float(static_cast<const __nv_bfloat16*>(a.cache.v)[i]);
      }
    }
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s += q[e] * k[e];
#pragma unroll
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    if (I8) s *= a.cache.k_scale[at];
    s *= scale_log2;
    const float m2 = fmaxf(m, s);
    // a score of -inf under a running maximum of -inf adds nothing
    const float f = m == m2 ? 1.f : exp2f(m - m2);
    const float p = s == -CUDART_INF_F ? 0.f : exp2f(s - m2);
    l = l * f + p;
    const float pv = I8 ? p * a.cache.v_scale[at] : p;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * f + pv * v[e];
    m = m2;
  }
}

template <int HD, bool I8>
__global__ void __launch_bounds__(256) attn_paged_row_kernel(const Params p) {
  constexpr int E = HD / 32;
  const PagedAttnArgs& a = p.a;
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int tok = static_cast<int>(item / a.heads), h = static_cast<int>(item % a.heads);
  if (tok >= a.T) return;
  int s = 0;
  while (s + 1 < a.nseq && a.q_start[s + 1] <= tok) ++s;
  const int t0 = a.q_start[s], t1 = a.q_start[s + 1];
  const int kvh = h / (a.heads / a.cache.kv_heads);
  float q[E], o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = __bfloat162float(a.q[tok * a.ldq + h * HD + lane * E + e]);
    o[e] = 0.f;
  }
  int len = a.kv_lens[s];
  if (len < 0 || len > a.table_ld << p.page_shift) {
    if (lane == 0) set_error(a.err, kDevBadIndex);
    len = 0;
  }
  const int hi = len - (t1 - t0) + (tok - t0) + 1;
  const int lo = a.window > 0 ? max(0, hi - a.window) : 0;
  float m = -CUDART_INF_F, l = 0.f;
  if (tok >= t0 && tok < t1)
    row_attend<HD, I8>(a, p.page_shift, a.table + s * a.table_ld, kvh, q, lo, hi, p.scale_log2, m, l, o);
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e)
    a.out[tok * a.ldo + h * HD + lane * E + e] = __float2bfloat16(l == 0.f ? 0.f : o[e] * inv);
  if (a.lse2 && lane == 0)
    a.lse2[static_cast<int64_t>(tok) * a.heads + h] = l == 0.f ? -CUDART_INF_F : m + log2f(l);
}

}  // namespace

int64_t attn_paged_workspace_bytes(int) { return 4096; }

int attn_paged(const PagedAttnArgs& a, cudaStream_t s) {
  if (!kv_pages_ok(a.cache) || a.nseq < 0 || a.T < 0 || a.heads <= 0 || a.heads % a.cache.kv_heads) return -1;
  const int64_t cols = static_cast<int64_t>(a.heads) * a.cache.hd;
  if (a.ldq % 8 || a.ldo % 8 || a.ldq < cols || a.ldo < cols || a.table_ld < 0 || a.window < 0) return -1;
  if ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out)) & 15) return -1;
  if (a.workspace_bytes < attn_paged_workspace_bytes(a.cache.hd)) return -1;
  if (a.T == 0 || a.nseq == 0) return 0;
  Params p;
  p.a = a;
  p.n_rows = a.cache.num_pages * a.cache.kv_heads * a.cache.page_size;
  p.page_shift = 31 - __builtin_clz(a.cache.page_size);
  p.scale_log2 = a.scale * kLog2e;
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(a.T) * a.heads + 7) / 8);
  if (a.cache.hd == 128) {
    if (a.cache.int8) attn_paged_row_kernel<128, true><<<grid, 256, 0, s>>>(p);
    else attn_paged_row_kernel<128, false><<<grid, 256, 0, s>>>(p);
  } else {
    if (a.cache.int8) attn_paged_row_kernel<64, true><<<grid, 256, 0, s>>>(p);
    else attn_paged_row_kernel<64, false><<<grid, 256, 0, s>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace rt
