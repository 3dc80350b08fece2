// From logits to a choice: penalties for tokens that the row's history holds, biases, a
// grammar mask and the greedy token, in one pass over the logits.
//
// Row b, token v with logit l, from the row's history (prompt tokens, then the answer's
// own): seen = v occurs anywhere, n = its count in the answer.
//   seen:  l = l > 0 ? l / repetition : l * repetition
//   n > 0: l = l - frequency * n - presence
//   bias:  l = l + value, for each list entry of v in list order
//   mask bit v clear: l = -inf (whatever l was, NaN included)
// token = the first index of the largest value; NaN never wins, and a row with nothing
// above -inf gives -1.  All fp32.
//
// HBM-bound: 4 bytes read and 4 written per logit.  A cluster of 1 to 8 CTAs owns a row,
// each CTA one slice of the vocabulary; counts live in shared memory for at most kSub
// tokens at a time and every CTA reads the row's whole history (4 bytes a token, from L2
// after the first CTA) into them with integer atomics, whose order does not change the
// counts.  The CTAs' best tokens meet in the first CTA's shared memory.
#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels.h"
#include "serving.h"

namespace rt {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kSub = 16384;                // tokens counted at a time: 64 KB, three CTAs an SM
constexpr uint32_t kSeen = 0x80000000u;    // occurs in the prompt part
constexpr uint32_t kBiased = 0x40000000u;  // has a bias entry
constexpr uint32_t kCount = 0x3fffffffu;

struct Best {
  float v;
  int i;
};
__device__ __forceinline__ Best better(Best a, Best b) {
  // index -1 is "nothing"; equal values: the lower index
  if (b.i < 0) return a;
  if (a.i < 0 || b.v > a.v || (b.v == a.v && b.i < a.i)) return b;
  return a;
}

struct Params {
  LogitsArgs a;
  int slice;  // tokens per CTA, a multiple of 128
};

template <bool VEC>
__global__ void __launch_bounds__(kThreads) logits_adjust_kernel(const Params p) {
  extern __shared__ uint32_t cnt[];
  __shared__ Best warp_best[kThreads / 32];
  __shared__ Best cta_best;
  const LogitsArgs& a = p.a;
  const int b = blockIdx.y, rank = blockIdx.x, tid = threadIdx.x;
  const int lo_all = min(a.V, rank * p.slice), hi_all = min(a.V, lo_all + p.slice);
  const float* in = a.logits + b * a.ldl;
  float* out = a.out + b * a.ldo;
  auto clamp_to = [](int64_t v, int64_t n) { return v < 0 ? int64_t(0) : v > n ? n : v; };
  int64_t h0 = 0, h1 = 0, b0 = 0, b1 = 0;
  if (a.hist) {
    h0 = clamp_to(a.hist_start[b], a.n_hist);
    h1 = clamp_to(a.hist_start[b + 1], a.n_hist);
  }
  if (a.bias_ids) {
    b0 = clamp_to(a.bias_start[b], a.n_bias);
    b1 = clamp_to(a.bias_start[b + 1], a.n_bias);
  }
  const int64_t made0 = a.n_prompt ? h0 + max(0, a.n_prompt[b]) : h0;  // the answer's first token
  const float rep = a.repetition ? a.repetition[b] : 1.f;
  const float pres = a.presence ? a.presence[b] : 0.f;
  const float freq = a.frequency ? a.frequency[b] : 0.f;
  const uint32_t* mask = a.mask ? a.mask + b * a.mask_ld : nullptr;
  const bool counted = h1 > h0 || b1 > b0;
  Best best{-INFINITY, -1};

  auto adjust = [&](float l, uint32_t c) {
    if (c & (kSeen | kCount)) l = l > 0.f ? l / rep : l * rep;
    const uint32_t n = c & kCount;
    if (n) l = l - freq * static_cast<float>(n) - pres;
    return l;
  };
  auto allowed = [&](int v) { return !mask || ((mask[v >> 5] >> (v & 31)) & 1u); };
  auto consider = [&](float l, int v) {
    if (l > best.v) best = {l, v};  // ascending v per thread within a pass: ties keep the first
    else if (l == best.v && best.i > v) best.i = v;
  };

  for (int lo = lo_all; lo < hi_all; lo += kSub) {
    const int hi = min(hi_all, lo + kSub), n = hi - lo;
    if (counted) {
      for (int i = tid; i < n; i += kThreads) cnt[i] = 0;
      __syncthreads();
#pragma unroll 4
      for (int64_t j = h0 + tid; j < h1; j += kThreads) {
        const int id = a.hist[j];
        if (id < 0 || id >= a.V) set_error(a.err, kDevBadToken);
        else if (id >= lo && id < hi) {
          if (j < made0) atomicOr(&cnt[id - lo], kSeen);
          else atomicAdd(&cnt[id - lo], 1u);
        }
      }
      for (int64_t j = b0 + tid; j < b1; j += kThreads) {
        const int id = a.bias_ids[j];
        if (id < 0 || id >= a.V) set_error(a.err, kDevBadToken);
        else if (id >= lo && id < hi) atomicOr(&cnt[id - lo], kBiased);
      }
      __syncthreads();
    }
    // A biased token's penalised logit waits in its count's place for the list below.
    if (VEC) {
#pragma unroll 2
      for (int v = lo + 4 * tid; v < hi; v += 4 * kThreads) {
        if (v + 4 <= hi) {
          const float4 l4 = __ldcs(reinterpret_cast<const float4*>(in + v));
          uint4 c4 = make_uint4(0, 0, 0, 0);
          if (counted) c4 = *reinterpret_cast<const uint4*>(cnt + (v - lo));
          const uint32_t bits = mask ? mask[v >> 5] >> (v & 31) : 0xfu;
          float l[4] = {l4.x, l4.y, l4.z, l4.w};
          const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            l[e] = adjust(l[e], c[e]);
            if (c[e] & kBiased) {
              cnt[v - lo + e] = __float_as_uint(l[e]);
            } else {
              if (!((bits >> e) & 1u)) l[e] = -INFINITY;
              consider(l[e], v + e);
            }
          }
          __stcs(reinterpret_cast<float4*>(out + v), make_float4(l[0], l[1], l[2], l[3]));
        } else {
          for (int w = v; w < hi; ++w) {
            const uint32_t c = counted ? cnt[w - lo] : 0u;
            float l = adjust(in[w], c);
            if (c & kBiased) {
              cnt[w - lo] = __float_as_uint(l);
              continue;
            }
            if (!allowed(w)) l = -INFINITY;
            consider(l, w);
            out[w] = l;
          }
        }
      }
    } else {
#pragma unroll 8
      for (int v = lo + tid; v < hi; v += kThreads) {
        const uint32_t c = counted ? cnt[v - lo] : 0u;
        float l = adjust(__ldcs(in + v), c);
        if (c & kBiased) {
          cnt[v - lo] = __float_as_uint(l);
        } else {
          if (!allowed(v)) l = -INFINITY;
          consider(l, v);
          __stcs(out + v, l);
        }
      }
    }
    if (b1 > b0) {
      __syncthreads();
      if (tid < 32) {
        // 32 entries at a time in list order; lanes with the same token add up one after another
        for (int64_t base = b0; base < b1; base += 32) {
          const int64_t j = base + tid;
          int id = -1;
          float val = 0.f;
          if (j < b1) {
            id = a.bias_ids[j];
            val = a.bias_vals[j];
            if (id < lo || id >= hi) id = -1;
          }
          const uint32_t same = __match_any_sync(0xffffffffu, id);
          const bool leader = id >= 0 && (same & ((1u << tid) - 1)) == 0;
          float sum = leader ? __uint_as_float(cnt[id - lo]) : 0.f;
          for (int k = 0; k < 32; ++k) {
            const float other = __shfl_sync(0xffffffffu, val, k);
            if (leader && ((same >> k) & 1u)) sum += other;
          }
          if (leader) cnt[id - lo] = __float_as_uint(sum);
          __syncwarp();
        }
      }
      __syncthreads();
      for (int64_t j = b0 + tid; j < b1; j += kThreads) {  // entries of one token write the same value
        const int id = a.bias_ids[j];
        if (id < lo || id >= hi) continue;
        float l = __uint_as_float(cnt[id - lo]);
        if (!allowed(id)) l = -INFINITY;
        consider(l, id);
        out[id] = l;
      }
    }
    __syncthreads();
  }

  if (!a.token) return;
#pragma unroll
  for (int o = 16; o; o >>= 1)
    best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.i, o)});
  if ((tid & 31) == 0) warp_best[tid >> 5] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kThreads / 32; ++w) best = better(best, warp_best[w]);
    cta_best = best;
  }
  cg::cluster_group cl = cg::this_cluster();
  cl.sync();
  if (rank == 0 && tid == 0) {
    for (int r = 1; r < static_cast<int>(gridDim.x); ++r) best = better(best, *cl.map_shared_rank(&cta_best, r));
    a.token[b] = best.i;
  }
  cl.sync();  // no CTA leaves while its shared memory may be read
}

}  // namespace

int logits_adjust(const LogitsArgs& a, cudaStream_t s) {
  if (a.B < 0 || a.V <= 0 || a.V > (1 << 30) || a.B > 65535 || a.ldl < a.V || a.ldo < a.V) return -1;
  if (a.mask && a.mask_ld < (a.V + 31) / 32) return -1;
  if (a.B == 0) return 0;
  // CTAs per row: enough for two an SM over all rows, or for a slice to fit the counts at
  // once, but slices of 1024 tokens at least.
  const int sms = num_sms();
  int c = 1;
  while (c < 8 && a.V / (2 * c) >= 1024 && (static_cast<int64_t>(a.B) * c < 2 * sms || a.V > c * kSub)) c *= 2;
  Params p;
  p.a = a;
  p.slice = ((a.V + c - 1) / c + 127) / 128 * 128;
  // in and out rows on 16-byte boundaries take 16-byte accesses
  const bool vec = a.ldl % 4 == 0 && a.ldo % 4 == 0 &&
                   ((reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.out)) & 15) == 0;
  const void* fn = vec ? reinterpret_cast<const void*>(logits_adjust_kernel<true>)
                       : reinterpret_cast<const void*>(logits_adjust_kernel<false>);
  const bool counted = a.hist || a.bias_ids;
  const int words = p.slice < kSub ? p.slice : kSub;
  const cudaError_t attr = smem_limit_once(fn, kSub * 4);
  if (attr != cudaSuccess) return attr;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(c, a.B);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = counted ? words * 4 : 0;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = c;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return vec ? cudaLaunchKernelEx(&cfg, logits_adjust_kernel<true>, p)
             : cudaLaunchKernelEx(&cfg, logits_adjust_kernel<false>, p);
}

}  // namespace rt
