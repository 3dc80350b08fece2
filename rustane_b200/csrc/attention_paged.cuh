// Shared by the two kernels of attention over the paged cache (attention_paged.cu: few
// rows per key head; attention_paged_tc.cu: many): the split of the work over CTAs, the
// join of an item that several CTAs worked on, and the one-row fallback.
//
// Rows.  Of sequence s and key head h, row r = i * G + g is new token i of query head h * G +
// g (G = heads / kv_heads); a tile is bm consecutive rows, an item (s, h, tile).  Keys come
// in blocks of BK; an item costs the blocks that any of its rows sees, one if none.
//
// Split.  All items' blocks, in order (s, h, tile, block), are cut into P equal ranges, one
// per CTA: every CTA has the same number of blocks whatever the lengths, which only the
// device knows.  A CTA's range begins inside at most one item and ends inside at most one,
// so it leaves at most two partial results (slots 0 and 1 of the workspace); of an item's
// CTAs the last to arrive (a counter, named by the item's first CTA) adds the partials in
// ascending order and sets the counter back to 0.  No CTA waits for another.
#pragma once

#include <math_constants.h>

#include "common.cuh"
#include "serving.h"

namespace rt {
namespace paged {

constexpr int kMaxCtas = 1024;                 // counters
constexpr int64_t kCounterBytes = kMaxCtas * 4;
constexpr float kRescale = 8.0f;  // keep a running maximum that is at most 2^8 too low: P stays <= 256

struct Params {
  PagedAttnArgs a;
  int G;           // query heads per key head
  int bm;          // rows per tile
  int tile_tokens; // bm / G where that is whole, else 0
  int page_shift;
  int max_len;     // tokens the entries of a row of the page table hold
  float scale_log2;
};

// Partial results: [CTA][2] x (o [BM][HD], m [BM], l [BM]) behind the counters.
template <int BM, int HD>
__device__ __forceinline__ float* partial_slot(const Params& p, int cta, int which) {
  return reinterpret_cast<float*>(static_cast<uint8_t*>(p.a.workspace) + kCounterBytes) +
         (static_cast<int64_t>(cta) * 2 + which) * (BM * (HD + 2));
}

// Walks one CTA's range of blocks, item by item.
template <int BK>
struct Walk {
  const Params* p;
  int s, h, t;            // item
  int q0, n, len, tiles;  // of the sequence: first row of q, new tokens, cached tokens, tiles per head
  int lo, hi;             // keys that any row of the tile sees
  int blk0, nb;           // its blocks
  int off;                // of which the ones before this CTA's part
  int64_t g, g1;          // the CTA's next block and end, in the order of all blocks

  __device__ __forceinline__ void seq(int ss) {
    const PagedAttnArgs& a = p->a;
    q0 = min(max(a.q_start[ss], 0), a.T);
    n = min(max(a.q_start[ss + 1], q0), a.T) - q0;
    len = a.kv_lens[ss];
    if (len < 0 || len > p->max_len) {
      set_error(a.err, kDevBadIndex);
      len = 0;
    }
    tiles = (n * p->G + p->bm - 1) / p->bm;
  }
  __device__ __forceinline__ void tile(int tt) {
    const int tok = p->tile_tokens;  // a division less
    const int i0 = tok ? tt * tok : tt * p->bm / p->G;
    const int i1 = min(n - 1, tok ? i0 + tok - 1 : (tt * p->bm + p->bm - 1) / p->G);
    hi = max(0, len - n + i1 + 1);
    lo = p->a.window > 0 ? max(0, len - n + i0 + 1 - p->a.window) : 0;
    blk0 = lo / BK;
    nb = hi > lo ? (hi + BK - 1) / BK - blk0 : 1;
  }
  __device__ __forceinline__ int64_t head_blocks() {  // of one key head of the sequence
    int64_t b = 0;
    for (int tt = 0; tt < tiles; ++tt) {
      tile(tt);
      b += nb;
    }
    return b;
  }
  __device__ __forceinline__ bool more() const { return g < g1; }
  __device__ __forceinline__ bool empty() const { return hi <= lo; }
  // blocks of the item in this CTA's range: [off, off + count())
  __device__ __forceinline__ int count() const {
    const int64_t left = g1 - g;
    return left < nb - off ? static_cast<int>(left) : nb - off;
  }
  __device__ __forceinline__ void next() {
    g += count();
    off = 0;
    if (++t == tiles) {
      t = 0;
      if (++h == p->a.cache.kv_heads) {
        h = 0;
        if (!more()) return;
        do {
          seq(++s);
        } while (tiles == 0);  // more blocks to come: a sequence with rows follows
      }
    }
    if (more()) tile(t);
  }
  // keys [first, last) that row r of the tile sees
  __device__ __forceinline__ int row_hi(int r) const { return len - n + (t * p->bm + r) / p->G + 1; }
  __device__ __forceinline__ int row_lo(int r) const {
    return p->a.window > 0 ? max(0, row_hi(r) - p->a.window) : 0;
  }
  __device__ __forceinline__ int rows() const { return min(p->bm, n * p->G - t * p->bm); }
};

// All NT threads of the CTA: the CTA's range of all blocks and its first item.  `total` and
// `P` (CTAs that share the work) are the same in every CTA.
template <int BK, int NT>
__device__ __forceinline__ Walk<BK> start_walk(const Params& p, int64_t& total, int& P) {
  __shared__ int64_t warp_sum[NT / 32];
  __shared__ int64_t first_rem, first_head;  // of the CTA's first block in its sequence; the sequence's blocks a head
  __shared__ int first_seq;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Walk<BK> w;
  w.p = &p;
  const int heads = p.a.cache.kv_heads;
  const int per = (p.a.nseq + NT - 1) / NT;
  const int s0 = min(tid * per, p.a.nseq), s1 = min(s0 + per, p.a.nseq);
  int64_t mine = 0, last = 0;
  for (int s = s0; s < s1; ++s) {
    w.seq(s);
    last = w.head_blocks();
    mine += last * heads;
  }
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) {
    if (i < warp) before += warp_sum[i];
    total += warp_sum[i];
  }
  P = total < gridDim.x ? static_cast<int>(total) : static_cast<int>(gridDim.x);
  const int c = blockIdx.x;
  w.g = w.g1 = 0;
  if (c < P) {
    if (total < (1 << 20)) {  // P <= 1024: 32-bit divisions
      w.g = static_cast<unsigned>(total) * c / P;
      w.g1 = static_cast<unsigned>(total) * (c + 1) / P;
    } else {
      w.g = total * c / P;
      w.g1 = total * (c + 1) / P;
    }
  }
  int64_t at = before + incl - mine;  // blocks before this thread's sequences
  if (c < P && w.g >= at && w.g < at + mine) {
    for (int s = s0; s < s1; ++s) {
      if (s1 - s0 > 1) {
        w.seq(s);
        last = w.head_blocks();
      }
      if (w.g < at + last * heads) {
        first_seq = s;
        first_rem = w.g - at;
        first_head = last;
        break;
      }
      at += last * heads;
    }
  }
  __syncthreads();
  if (!w.more()) return w;
  w.s = first_seq;
  w.seq(w.s);
  int64_t rem = first_rem;
  w.h = 0;
  if (rem >= first_head) {
    w.h = first_head < (1 << 30) && rem < (int64_t(1) << 31) ? static_cast<unsigned>(rem) / static_cast<unsigned>(first_head)
                                                            : static_cast<int>(rem / first_head);
    rem -= w.h * first_head;
  }
  for (w.t = 0;; ++w.t) {
    w.tile(w.t);
    if (rem < w.nb) break;
    rem -= w.nb;
  }
  w.off = static_cast<int>(rem);
  return w;
}

// First and last CTA of the current item: CTA c owns blocks [total c / P, total (c + 1) / P).
__device__ __forceinline__ int block_owner(int64_t x, int64_t total, int P) {
  if (total < (1 << 20)) return (static_cast<unsigned>(x + 1) * P - 1) / static_cast<unsigned>(total);
  return static_cast<int>(((x + 1) * P - 1) / total);
}

__device__ __forceinline__ int checked_page(const Params& p, int page) {
  if (page >= 0 && page < p.a.cache.num_pages) return page;
  set_error(p.a.err, kDevBadIndex);
  return 0;
}
__device__ __forceinline__ int page_of(const Params& p, const int32_t* table, int key) {
  return checked_page(p, table[key >> p.page_shift]);
}

// Keys [lo, hi) of head h for one row, one warp, fp32 throughout: running maximum m (log2
// domain), sum l and the lane's HD / 32 entries of the unnormalised output.  Only keys of
// the range are touched.  The tile kernels weigh keys that a row does not see by 0, which
// a NaN or infinite v turns into NaN; rows that came out NaN take this instead (of the few-row kernel, a
// warp of which has 4 at most; it needs few registers, which the main loop would miss).
template <int HD>
__device__ __noinline__ void row_attend(const Params& p, const int32_t* table, int h, const __nv_bfloat16* qrow, int lo,
                                        int hi, float& m, float& l, float (&o)[HD / 32]) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31;
  const __nv_bfloat16 *kc = static_cast<const __nv_bfloat16*>(p.a.cache.k),
                      *vc = static_cast<const __nv_bfloat16*>(p.a.cache.v);
  float q[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = __bfloat162float(qrow[lane * E + e]);
    o[e] = 0.f;
  }
  m = -CUDART_INF_F;
  l = 0.f;
  for (int j = lo; j < hi; ++j) {
    const int64_t page = page_of(p, table, j);
    const int64_t at = ((page * p.a.cache.kv_heads + h) << p.page_shift) + (j & ((1 << p.page_shift) - 1));
    float v[E], s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      s += q[e] * __bfloat162float(kc[at * HD + lane * E + e]);
      v[e] = __bfloat162float(vc[at * HD + lane * E + e]);
    }
#pragma unroll
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= p.scale_log2;
    const float m2 = fmaxf(m, s);
    const float f = m == m2 ? 1.f : exp2f(m - m2);
    const float pj = s == -CUDART_INF_F ? 0.f : exp2f(s - m2);
    l = l * f + pj;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * f + pj * v[e];
    m = m2;
  }
}

}  // namespace paged

int attn_paged_few(const paged::Params& p, cudaStream_t s);
int attn_paged_many(const paged::Params& p, cudaStream_t s);
int64_t attn_paged_many_ctas();

}  // namespace rt
