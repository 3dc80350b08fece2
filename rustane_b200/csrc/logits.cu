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
// 192 rows of 128003 with 2000 history tokens and 40 biases each: 83 us, 2.4 TB/s of the 8 bytes a
// logit (76 us without the biases, 61 without the history, 48 with neither): parts of 8192 tokens alternate counting,
// streaming and biases between barriers, and half of all issue slots go to the penalties of
// vectors that hold a listed token.  Biases and the first history tokens are fetched ahead (89 us
// without; 8 tokens a thread instead of 4: 87).  A list of the touched tokens that does the
// penalties after the streaming took 97 us, whole waves of 3 CTAs a row 121, 128 threads a CTA 89
// to 119, branch-free penalties 93.
#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels.h"
#include "serving.h"

namespace rt {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kSub = 8192;                 // tokens counted at a time: 32 KB, four CTAs an SM
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
  int slice;  // places per CTA, a multiple of 128
};

constexpr int kHist = 4;   // history tokens in flight per thread
constexpr int kBatch = 4;  // 16-byte loads (or 4-byte ones, VEC false) in flight per thread

// VEC: the rows of in and out are equally far from a 16-byte boundary, so both take 16-byte
// accesses from there on; place x = v + (that distance in floats) counts tokens from the
// boundary before the row.  Otherwise x = v, 4 bytes at a time.
template <bool VEC>
__global__ void __launch_bounds__(kThreads, 4) logits_adjust_kernel(const Params p) {
  extern __shared__ uint32_t cnt[];
  __shared__ int32_t held_ids[kThreads];
  __shared__ float held_vals[kThreads];
  __shared__ Best warp_best[kThreads / 32];
  __shared__ Best cta_best[8];  // of the cluster's CTAs, in the first one
  const LogitsArgs& a = p.a;
  const int b = blockIdx.y, rank = blockIdx.x, tid = threadIdx.x;
  const float* in = a.logits + b * a.ldl;
  float* out = a.out + b * a.ldo;
  const int shift = VEC ? static_cast<int>((reinterpret_cast<uintptr_t>(in) >> 2) & 3) : 0;
  const int x_end = a.V + shift;
  const int lo_all = min(x_end, rank * p.slice), hi_all = min(x_end, lo_all + p.slice);
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
  asm volatile("barrier.cluster.arrive.relaxed;");  // this CTA runs: its shared memory may be written

  auto adjust = [&](float l, uint32_t c) {
    if (c & (kSeen | kCount)) l = l > 0.f ? l / rep : l * rep;
    const uint32_t n = c & kCount;
    if (n) l = l - freq * static_cast<float>(n) - pres;
    return l;
  };
  auto allowed = [&](int v) { return !mask || ((mask[v >> 5] >> (v & 31)) & 1u); };
  auto consider = [&](float l, int v) {
    if (l > best.v) best = {l, v};
    else if (l == best.v && best.i > v) best.i = v;
  };

  // VEC: the thread's next kBatch vectors, one round ahead (the first are on their way while the
  // history is counted); edge vectors of the row are read where they are used
  constexpr int kRound = 4 * kThreads * kBatch;
  float4 ahead[kBatch];
  auto load = [&](int x0) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int x = x0 + u * 4 * kThreads;
      if (x >= shift && x + 4 <= x_end && x < hi_all) ahead[u] = __ldcs(reinterpret_cast<const float4*>(in + (x - shift)));
    }
  };
  if (VEC) load(lo_all + 4 * tid);

  // The thread's first history tokens (every part starts with them) and the row's biases, fetched
  // before anything waits.
  int id0[kHist];
  auto fetch = [&](int64_t j0, int (&id)[kHist]) {  // -1: no token
#pragma unroll
    for (int u = 0; u < kHist; ++u) id[u] = j0 + u * kThreads < h1 ? a.hist[j0 + u * kThreads] : -1;
  };
  fetch(h0 + tid, id0);
  const int32_t* bias_ids = a.bias_ids + b0;
  const float* bias_vals = a.bias_vals + b0;
  const int64_t nb = b1 - b0;
  if (nb > 0 && nb <= kThreads) {
    if (tid < nb) {
      held_ids[tid] = bias_ids[tid];
      held_vals[tid] = bias_vals[tid];
    }
    bias_ids = held_ids;
    bias_vals = held_vals;
  }

  for (int lo = lo_all; lo < hi_all; lo += kSub) {
    const int hi = min(hi_all, lo + kSub), n = hi - lo;
    const int id_lo = lo - shift, id_hi = hi - shift;  // tokens of these places
    if (counted) {
      for (int i = 4 * tid; i < n; i += 4 * kThreads) *reinterpret_cast<uint4*>(cnt + i) = make_uint4(0, 0, 0, 0);
      __syncthreads();
      auto count = [&](int64_t j0, const int (&id)[kHist]) {
#pragma unroll
        for (int u = 0; u < kHist; ++u) {
          if (static_cast<unsigned>(id[u]) >= static_cast<unsigned>(a.V)) {
            if (id[u] != -1) set_error(a.err, kDevBadToken);
          } else if (static_cast<unsigned>(id[u] - id_lo) < static_cast<unsigned>(n)) {
            if (j0 + u * kThreads < made0) atomicOr(&cnt[id[u] - id_lo], kSeen);
            else atomicAdd(&cnt[id[u] - id_lo], 1u);
          }
        }
      };
      if (h0 + tid < h1) count(h0 + tid, id0);
      for (int64_t j0 = h0 + tid + kHist * kThreads; j0 < h1; j0 += kHist * kThreads) {
        int id[kHist];
        fetch(j0, id);
        count(j0, id);
      }
      for (int64_t j = tid; j < nb; j += kThreads) {
        const int id = bias_ids[j];
        if (id < -1 || id >= a.V) set_error(a.err, kDevBadToken);
        else if (id >= max(id_lo, 0) && id < id_hi) atomicOr(&cnt[id - id_lo], kBiased);
      }
      __syncthreads();
    }
    // A biased token's penalised logit waits in its count's place for the list below.
    auto one = [&](int x, float raw) {
      const int v = x - shift;
      const uint32_t c = counted ? cnt[x - lo] : 0u;
      float l = adjust(raw, c);
      if (c & kBiased) {
        cnt[x - lo] = __float_as_uint(l);
        return;
      }
      if (!allowed(v)) l = -INFINITY;
      consider(l, v);
      __stcs(out + v, l);
    };
    if (VEC) {
      for (int x0 = lo + 4 * tid; x0 < hi; x0 += kRound) {
        float4 raw[kBatch];
        uint32_t w0[kBatch], w1[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int x = x0 + u * 4 * kThreads, v = x - shift;
          raw[u] = ahead[u];
          w0[u] = w1[u] = ~0u;
          if (mask && v >= 0 && x + 4 <= hi) {
            w0[u] = mask[v >> 5];
            w1[u] = mask[(v + 3) >> 5];
          }
        }
        load(x0 + kRound < hi ? x0 + kRound : hi + 4 * tid);  // the next round, of this part or the next
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int x = x0 + u * 4 * kThreads, v = x - shift;
          if (x >= hi) break;
          if (v < 0 || x + 4 > x_end) {  // the row's first or last places
            for (int y = max(x, shift); y < min(x + 4, hi); ++y) one(y, in[y - shift]);
            continue;
          }
          float l[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
          uint4 c4 = make_uint4(0, 0, 0, 0);
          if (counted) c4 = *reinterpret_cast<const uint4*>(cnt + (x - lo));
          const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
          uint32_t bits = __funnelshift_r(w0[u], w1[u], v & 31);
          if (c4.x | c4.y | c4.z | c4.w) {
#pragma unroll
            for (int e = 0; e < 4; ++e) l[e] = adjust(l[e], c[e]);
            if ((c4.x | c4.y | c4.z | c4.w) & kBiased) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (c[e] & kBiased) {
                  cnt[x - lo + e] = __float_as_uint(l[e]);
                  bits &= ~(1u << e);  // not a candidate yet; the list writes it
                }
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!((bits >> e) & 1u)) l[e] = -INFINITY;
          // ascending order within a thread: only a larger value replaces the best
          const float top = fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3]));
          if (top > best.v) {
            best.v = top;
            best.i = v + (l[0] == top ? 0 : l[1] == top ? 1 : l[2] == top ? 2 : 3);
          }
          __stcs(reinterpret_cast<float4*>(out + v), make_float4(l[0], l[1], l[2], l[3]));
        }
      }
    } else {
      for (int x0 = lo + tid; x0 < hi; x0 += 2 * kBatch * kThreads) {
        float raw[2 * kBatch];
#pragma unroll
        for (int u = 0; u < 2 * kBatch; ++u) raw[u] = x0 + u * kThreads < hi ? __ldcs(in + x0 + u * kThreads) : 0.f;
#pragma unroll
        for (int u = 0; u < 2 * kBatch; ++u)
          if (x0 + u * kThreads < hi) one(x0 + u * kThreads, raw[u]);
      }
    }
    if (nb > 0) {
      __syncthreads();
      if (tid < 32) {
        // 32 entries at a time in list order; lanes with the same token add up one after another
        for (int64_t base = 0; base < nb; base += 32) {
          const int64_t j = base + tid;
          int id = -1;
          float val = 0.f;
          if (j < nb) {
            id = bias_ids[j];
            val = bias_vals[j];
            if (id < max(id_lo, 0) || id >= id_hi) id = -1;
          }
          const uint32_t same = __match_any_sync(0xffffffffu, id);
          const bool leader = id >= 0 && (same & ((1u << tid) - 1)) == 0;
          float sum = leader ? __uint_as_float(cnt[id - id_lo]) + val : 0.f;
          if (__any_sync(0xffffffffu, id >= 0 && !leader)) {
            for (int k = 0; k < 32; ++k) {
              const float other = __shfl_sync(0xffffffffu, val, k);
              if (leader && k != tid && ((same >> k) & 1u)) sum += other;
            }
          }
          if (leader) cnt[id - id_lo] = __float_as_uint(sum);
          __syncwarp();
        }
      }
      __syncthreads();
      for (int64_t j = tid; j < nb; j += kThreads) {  // entries of one token write the same value
        const int id = bias_ids[j];
        if (id < max(id_lo, 0) || id >= id_hi) continue;
        float l = __uint_as_float(cnt[id - id_lo]);
        if (!allowed(id)) l = -INFINITY;
        consider(l, id);
        out[id] = l;
      }
    }
    __syncthreads();
  }

  asm volatile("barrier.cluster.wait;" ::: "memory");
  if (!a.token) return;
#pragma unroll
  for (int o = 16; o; o >>= 1)
    best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.i, o)});
  if ((tid & 31) == 0) warp_best[tid >> 5] = best;
  __syncthreads();
  cg::cluster_group cl = cg::this_cluster();
  if (tid < 32) {
    best = tid < kThreads / 32 ? warp_best[tid] : Best{-INFINITY, -1};
#pragma unroll
    for (int o = kThreads / 64; o; o >>= 1)
      best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.i, o)});
    if (tid == 0) *cl.map_shared_rank(&cta_best[rank], 0) = best;
  }
  cl.sync();
  if (rank == 0 && tid == 0) {
    best = cta_best[0];
    for (int r = 1; r < static_cast<int>(gridDim.x); ++r) best = better(best, cta_best[r]);
    a.token[b] = best.i;
  }
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
  while (c < 8 && a.V / (2 * c) >= 1024 && (static_cast<int64_t>(a.B) * c < 2 * sms || a.V > 2 * c * kSub)) c *= 2;
  // VEC: equal distances from a 16-byte boundary in every row
  const bool vec = (a.ldl - a.ldo) % 4 == 0 &&
                   ((reinterpret_cast<uintptr_t>(a.logits) ^ reinterpret_cast<uintptr_t>(a.out)) & 15) == 0;
  Params p;
  p.a = a;
  p.slice = ((a.V + 3 + c - 1) / c + 127) / 128 * 128;
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
