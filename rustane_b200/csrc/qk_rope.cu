// Per-head RMSNorm of q and k with the rotary position in the same pass,
// forward and backward, and the two ends of the paged cache: the same forward
// pass writing k and v into pages (bf16, or int8 with a scale per token and
// head), and reading tokens back.
//
// Math, per token and head vector x[hd] (gamma optional):
//   n = x * r * gamma, r = 1 / sqrt(mean(x^2) + eps);   y = R(pos) n
// with R the rotation of the first `rot` entries by the tables' (cos, sin); the
// tables may carry a factor, so the backward uses R's transpose, not its inverse:
//   dn = R^T dy;  dgamma += dn * x * r;  dx = r (dn gamma - x r mean(dn gamma x r)).
// int8 rows: s = amax|y| / 127, code = rint(y / s) (a true division: the code is
// the nearest one), read back as code * s.  A row with a NaN or infinity gets a
// NaN scale and reads back as NaN.  All arithmetic in fp32, rounded once.
//
// All are HBM-bound.  hd / 8 lanes own one head vector, 16 bytes a lane, so a
// warp holds 32 / (hd / 8) vectors; a warp takes kU such groups of one token
// at a time, loads first, so kU 512-byte loads are in flight, and the token's
// tables and the gammas are read once per kU groups.
#include "common.cuh"
#include "kernels.h"
#include "serving.h"

namespace rt {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kU = 4;

__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8]) {
  v[0] = bf16lo(u.x); v[1] = bf16hi(u.x); v[2] = bf16lo(u.y); v[3] = bf16hi(u.y);
  v[4] = bf16lo(u.z); v[5] = bf16hi(u.z); v[6] = bf16lo(u.w); v[7] = bf16hi(u.w);
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                    pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void load8f(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

// Sum / max over the LPH lanes that share a head vector.
template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = LPH / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int LPH>
__device__ __forceinline__ float head_max(float v) {
#pragma unroll
  for (int o = LPH / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

struct RopeDev {
  const float* cos;
  const float* sin;
  const int32_t* pos;
  int n_pos, rot, half;
};

// One lane's part of a token's tables: interleaved pairs need 4 angles, halves 8.
struct Angles {
  float c[8], s[8];
};
__device__ __forceinline__ void load_angles(Angles& a, const RopeDev& r, int pos, int sub) {
  const int d0 = sub * 8;
  if (d0 >= r.rot) return;
  const int64_t base = static_cast<int64_t>(pos) * (r.rot / 2);
  if (r.half) {
    const int i = d0 < r.rot / 2 ? d0 : d0 - r.rot / 2;
    load8f(r.cos + base + i, a.c);
    load8f(r.sin + base + i, a.s);
  } else {
    const float4 c = *reinterpret_cast<const float4*>(r.cos + base + d0 / 2);
    const float4 s = *reinterpret_cast<const float4*>(r.sin + base + d0 / 2);
    a.c[0] = c.x; a.c[1] = c.y; a.c[2] = c.z; a.c[3] = c.w;
    a.s[0] = s.x; a.s[1] = s.y; a.s[2] = s.z; a.s[3] = s.w;
  }
}
// v <- R v (BACK: R^T v).  Every lane of the warp calls it (the halves exchange by shuffles).
template <int LPH, bool BACK>
__device__ __forceinline__ void rotate(float (&v)[8], const Angles& a, const RopeDev& r, int sub) {
  const int d0 = sub * 8;
  if (r.half) {
    const int step = r.rot / 16;  // lanes between the two halves of a pair
    const bool first = d0 < r.rot / 2;
    const int lane = threadIdx.x & 31;
    const int src = d0 >= r.rot ? lane : first ? lane + step : lane - step;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float p = __shfl_sync(0xffffffffu, v[i], src);
      const float s = first != BACK ? -a.s[i] : a.s[i];
      if (d0 < r.rot) v[i] = v[i] * a.c[i] + p * s;
    }
  } else if (d0 < r.rot) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = v[2 * i], y = v[2 * i + 1], s = BACK ? -a.s[i] : a.s[i];
      v[2 * i] = x * a.c[i] - y * s;
      v[2 * i + 1] = y * a.c[i] + x * s;
    }
  }
}

struct FwdParams {
  const __nv_bfloat16* x;
  int64_t ldx;
  __nv_bfloat16* out;
  int64_t ldo;
  RopeDev rope;
  const float* gq;
  const float* gk;
  float eps;
  int T, heads, kv_heads, total_heads, chunks;
  const int32_t* slots;
  void* ck;
  void* cv;
  float* sk;
  float* sv;
  int64_t n_slots;
  int page_shift;
  int* err;
};

enum Dest : int { kToRows, kToBf16Pages, kToInt8Pages };

template <int HD, int DEST>
__global__ void __launch_bounds__(kThreads) qk_rope_fwd_kernel(const FwdParams p) {
  constexpr int LPH = HD / 8, HPW = 32 / LPH;  // lanes per head vector, vectors per warp
  const int lane = threadIdx.x & 31, sub = lane % LPH, hw = lane / LPH;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int64_t tok64 = item / p.chunks;
  if (tok64 >= p.T) return;  // the whole warp
  const int tok = static_cast<int>(tok64);
  const int h0 = static_cast<int>(item - tok64 * p.chunks) * (HPW * kU) + hw;

  uint4 raw[kU];
  const __nv_bfloat16* row = p.x + tok * p.ldx + sub * 8;
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    const int h = h0 + u * HPW;
    raw[u] = h < p.total_heads ? *reinterpret_cast<const uint4*>(row + static_cast<int64_t>(h) * HD)
                               : make_uint4(0, 0, 0, 0);
  }
  int pos = p.rope.pos[tok];
  if (pos < 0 || pos >= p.rope.n_pos) {
    if (lane == 0) set_error(p.err, kDevBadIndex);
    pos = 0;
  }
  int64_t slot = -1;
  if (DEST != kToRows) {
    slot = p.slots[tok];
    if (slot < -1 || slot >= p.n_slots) {
      if (lane == 0) set_error(p.err, kDevBadIndex);
      slot = -1;
    }
  }
  Angles ang;
  load_angles(ang, p.rope, pos, sub);

#pragma unroll
  for (int u = 0; u < kU; ++u) {
    const int h = h0 + u * HPW;
    const bool is_q = h < p.heads, is_v = h >= p.heads + p.kv_heads;
    float v[8];
    unpack8(raw[u], v);
    if (p.gq) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += v[i] * v[i];
      const float r = rsqrtf(head_sum<LPH>(ss) * (1.0f / HD) + p.eps);
      if (!is_v) {
        float g[8];
        load8f((is_q ? p.gq : p.gk) + sub * 8, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] * r * g[i];
      }
    }
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = v[i];
    rotate<LPH, false>(w, ang, p.rope, sub);
    if (!is_v) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = w[i];
    }
    float amax = 0.f;
    bool finite = true;
    if (DEST == kToInt8Pages) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        amax = fmaxf(amax, fabsf(v[i]));
        finite = finite && isfinite(v[i]);
      }
      amax = head_max<LPH>(finite ? amax : INFINITY);
    }
    if (h >= p.total_heads) continue;
    if (DEST == kToRows || is_q) {
      *reinterpret_cast<uint4*>(p.out + tok * p.ldo + static_cast<int64_t>(h) * HD + sub * 8) = pack8(v);
    } else if (slot >= 0) {
      const int kh = is_v ? h - p.heads - p.kv_heads : h - p.heads;
      const int64_t page = slot >> p.page_shift, off = slot & ((1 << p.page_shift) - 1);
      const int64_t at = (((page * p.kv_heads + kh) << p.page_shift) + off);
      if (DEST == kToBf16Pages) {
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(is_v ? p.cv : p.ck) + at * HD + sub * 8) = pack8(v);
      } else {
        const float s = isinf(amax) ? NAN : amax / 127.0f;
        uint32_t b[2] = {0, 0};
        if (s > 0.f) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            // |y / s| <= 127 but for the rounding of a denormal scale
            const int c = max(-127, min(127, __float2int_rn(v[i] / s)));
            b[i >> 2] |= static_cast<uint32_t>(c & 0xff) << (8 * (i & 3));
          }
        }
        *reinterpret_cast<uint2*>(static_cast<int8_t*>(is_v ? p.cv : p.ck) + at * HD + sub * 8) =
            make_uint2(b[0], b[1]);
        if (sub == 0) (is_v ? p.sv : p.sk)[at] = s;
      }
    }
  }
}

// Backward.  A fixed grid walks the items (token, kU groups of heads) in strides, so
// every warp keeps its dgamma sums in registers; each CTA adds its warps' sums in a
// fixed order and writes one partial row per gamma.
struct BwdParams {
  const __nv_bfloat16* dy;
  int64_t lddy;
  const __nv_bfloat16* x;
  int64_t ldx;
  __nv_bfloat16* dx;
  int64_t lddx;
  RopeDev rope;
  const float* gq;
  const float* gk;
  float eps;
  int T, heads, kv_heads, total_heads, chunks;
  float* part;  // [2][gridDim.x][HD]
  int* err;
};

template <int HD>
__global__ void __launch_bounds__(kThreads) qk_rope_bwd_kernel(const BwdParams p) {
  constexpr int LPH = HD / 8, HPW = 32 / LPH;
  __shared__ float red[2][kWarps * HPW][HD];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % LPH, hw = lane / LPH;
  const int64_t items = static_cast<int64_t>(p.T) * p.chunks;
  float gq[8], gk[8], dgq[8], dgk[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) gq[i] = gk[i] = dgq[i] = dgk[i] = 0.f;
  if (p.gq) {
    load8f(p.gq + sub * 8, gq);
    load8f(p.gk + sub * 8, gk);
  }
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * kWarps + warp; item < items;
       item += static_cast<int64_t>(gridDim.x) * kWarps) {
    const int64_t tok = item / p.chunks;
    const int h0 = static_cast<int>(item - tok * p.chunks) * (HPW * kU) + hw;
    uint4 rd[kU], rx[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int h = h0 + u * HPW;
      rd[u] = rx[u] = make_uint4(0, 0, 0, 0);
      if (h < p.total_heads)
        rd[u] = *reinterpret_cast<const uint4*>(p.dy + tok * p.lddy + static_cast<int64_t>(h) * HD + sub * 8);
      if (p.gq && h < p.heads + p.kv_heads)
        rx[u] = *reinterpret_cast<const uint4*>(p.x + tok * p.ldx + static_cast<int64_t>(h) * HD + sub * 8);
    }
    int pos = p.rope.pos[tok];
    if (pos < 0 || pos >= p.rope.n_pos) {
      if (lane == 0) set_error(p.err, kDevBadIndex);
      pos = 0;
    }
    Angles ang;
    load_angles(ang, p.rope, pos, sub);
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int h = h0 + u * HPW;
      const bool is_q = h < p.heads, is_v = h >= p.heads + p.kv_heads;
      float d[8];
      unpack8(rd[u], d);
      rotate<LPH, true>(d, ang, p.rope, sub);
      if (p.gq) {
        float x[8], xh[8];
        unpack8(rx[u], x);
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
        const float r = rsqrtf(head_sum<LPH>(ss) * (1.0f / HD) + p.eps);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          xh[i] = x[i] * r;
          const float t = d[i] * xh[i];
          if (is_q) dgq[i] += t;
          else if (!is_v) dgk[i] += t;
          d[i] *= is_q ? gq[i] : gk[i];
          dot += d[i] * xh[i];
        }
        dot = head_sum<LPH>(dot) * (1.0f / HD);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = r * (d[i] - xh[i] * dot);
      }
      if (h < p.total_heads)
        *reinterpret_cast<uint4*>(p.dx + tok * p.lddx + static_cast<int64_t>(h) * HD + sub * 8) =
            is_v ? rd[u] : pack8(d);
    }
  }
  if (!p.gq) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    red[0][warp * HPW + hw][sub * 8 + i] = dgq[i];
    red[1][warp * HPW + hw][sub * 8 + i] = dgk[i];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * HD; i += kThreads) {
    const int which = i / HD, d = i % HD;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps * HPW; ++w) s += red[which][w][d];
    p.part[(static_cast<int64_t>(which) * gridDim.x + blockIdx.x) * HD + d] = s;
  }
}

// dgamma[d] = (accumulate ? dgamma[d] : 0) + sum of its partial rows, in a fixed order;
// blockIdx.y: q, k.  One launch for both.
__global__ void __launch_bounds__(1024) qk_dgamma_kernel(const float* part, int nblk, float* dgq, float* dgk, int hd,
                                                         int accumulate) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = blockIdx.x * 32 + lane;
  const float* src = part + static_cast<int64_t>(blockIdx.y) * nblk * hd;
  float s = 0.f;
  for (int b = warp; b < nblk; b += 32) s += src[static_cast<int64_t>(b) * hd + d];
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 32; ++w) t += red[w][lane];
    float* out = blockIdx.y ? dgk : dgq;
    out[d] = accumulate ? out[d] + t : t;
  }
}

struct GatherParams {
  const void* ck;
  const void* cv;
  const float* sk;
  const float* sv;
  const int32_t* slots;
  __nv_bfloat16* k_out;
  __nv_bfloat16* v_out;
  int64_t ldo, n_slots;
  int T, kv_heads, chunks, page_shift;
  int* err;
};

template <int HD, bool I8>
__global__ void __launch_bounds__(kThreads) kv_gather_kernel(const GatherParams p) {
  constexpr int LPH = HD / 8, HPW = 32 / LPH;
  const int lane = threadIdx.x & 31, sub = lane % LPH, hw = lane / LPH;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int64_t tok = item / p.chunks;
  if (tok >= p.T) return;
  const int h0 = static_cast<int>(item - tok * p.chunks) * (HPW * kU) + hw;
  int64_t slot = p.slots[tok];
  if (slot < -1 || slot >= p.n_slots) {
    if (lane == 0) set_error(p.err, kDevBadIndex);
    slot = -1;
  }
  const int64_t page = slot >> p.page_shift, off = slot & ((1 << p.page_shift) - 1);
  uint4 raw[2][kU];  // [k, v]
  float sc[2][kU];
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    const int h = h0 + u * HPW;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      raw[w][u] = make_uint4(0, 0, 0, 0);
      sc[w][u] = 0.f;
      if (h >= p.kv_heads || slot < 0) continue;
      const int64_t at = ((page * p.kv_heads + h) << p.page_shift) + off;
      const void* src = w ? p.cv : p.ck;
      if (I8) {
        const uint2 c = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(src) + at * HD + sub * 8);
        raw[w][u].x = c.x;
        raw[w][u].y = c.y;
        sc[w][u] = (w ? p.sv : p.sk)[at];
      } else {
        raw[w][u] = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(src) + at * HD + sub * 8);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    const int h = h0 + u * HPW;
    if (h >= p.kv_heads) continue;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      uint4 o = raw[w][u];
      if (I8) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          v[i] = static_cast<float>(static_cast<int8_t>((i < 4 ? raw[w][u].x : raw[w][u].y) >> (8 * (i & 3)))) *
                 sc[w][u];
        o = pack8(v);
      }
      *reinterpret_cast<uint4*>((w ? p.v_out : p.k_out) + tok * p.ldo + static_cast<int64_t>(h) * HD + sub * 8) = o;
    }
  }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

inline int chunks_of(int total_heads, int hd) {
  const int per = (32 / (hd / 8)) * kU;
  return (total_heads + per - 1) / per;
}
inline int log2_exact(int v) {
  for (int i = 0; i < 31; ++i)
    if (v == 1 << i) return i;
  return -1;
}
// Blocks of kWarps items, or -1 when the grid would not hold them.
inline int64_t blocks_of(int64_t items) {
  const int64_t b = (items + kWarps - 1) / kWarps;
  return b < (int64_t(1) << 31) ? b : -1;
}

bool rope_ok(const QkRopeArgs& a) {
  if (a.hd != 64 && a.hd != 128) return false;
  if (a.T < 0 || a.heads <= 0 || a.kv_heads <= 0 || a.v_heads < 0) return false;
  if (a.rope.n_pos <= 0 || a.rope.rot <= 0 || a.rope.rot > a.hd || a.rope.rot % 16) return false;
  if (!aligned16(a.rope.cos) || !aligned16(a.rope.sin)) return false;
  if ((a.gamma_q == nullptr) != (a.gamma_k == nullptr) || !aligned16(a.gamma_q) || !aligned16(a.gamma_k)) return false;
  return true;
}
bool rows_ok(const void* p, int64_t ld, int64_t cols) { return aligned16(p) && ld % 8 == 0 && ld >= cols; }

RopeDev rope_dev(const QkRopeArgs& a) {
  return {a.rope.cos, a.rope.sin, a.pos, a.rope.n_pos, a.rope.rot, a.rope.half ? 1 : 0};
}

int launch_fwd(const QkRopeArgs& a, int dest, cudaStream_t s) {
  FwdParams p{};
  p.x = a.x; p.ldx = a.ldx; p.out = a.out; p.ldo = a.ldo;
  p.rope = rope_dev(a);
  p.gq = a.gamma_q; p.gk = a.gamma_k; p.eps = a.eps;
  p.T = a.T; p.heads = a.heads; p.kv_heads = a.kv_heads;
  p.total_heads = a.heads + a.kv_heads + a.v_heads;
  p.chunks = chunks_of(p.total_heads, a.hd);
  p.slots = a.slots;
  p.ck = a.cache.k; p.cv = a.cache.v; p.sk = a.cache.k_scale; p.sv = a.cache.v_scale;
  p.n_slots = a.cache.num_pages * a.cache.page_size;
  p.page_shift = dest == kToRows ? 0 : log2_exact(a.cache.page_size);
  p.err = a.err;
  const int64_t nb = blocks_of(static_cast<int64_t>(a.T) * p.chunks);
  if (nb < 0) return -1;
  if (nb == 0) return 0;
  const dim3 grid(static_cast<unsigned>(nb));
#define RT_FWD(HD, DEST) qk_rope_fwd_kernel<HD, DEST><<<grid, kThreads, 0, s>>>(p)
  if (a.hd == 128) {
    if (dest == kToRows) RT_FWD(128, kToRows);
    else if (dest == kToBf16Pages) RT_FWD(128, kToBf16Pages);
    else RT_FWD(128, kToInt8Pages);
  } else {
    if (dest == kToRows) RT_FWD(64, kToRows);
    else if (dest == kToBf16Pages) RT_FWD(64, kToBf16Pages);
    else RT_FWD(64, kToInt8Pages);
  }
#undef RT_FWD
  return cudaGetLastError();
}

}  // namespace

bool kv_pages_ok(const KvPages& c) {
  if (c.hd != 64 && c.hd != 128) return false;
  if (c.num_pages <= 0 || c.kv_heads <= 0) return false;
  if (c.page_size < 16 || c.page_size > 128 || log2_exact(c.page_size) < 0) return false;
  // rows (page, head, token) are TMA coordinates and slots are int32
  if (c.num_pages > (int64_t(1) << 31) / (static_cast<int64_t>(c.kv_heads) * c.page_size) - 1) return false;
  if (!aligned16(c.k) || !aligned16(c.v) || !aligned16(c.k_scale) || !aligned16(c.v_scale)) return false;
  return true;
}

int qk_rope_fwd(const QkRopeArgs& a, cudaStream_t s) {
  const int64_t cols = static_cast<int64_t>(a.heads + a.kv_heads + a.v_heads) * a.hd;
  if (!rope_ok(a) || !rows_ok(a.x, a.ldx, cols) || !rows_ok(a.out, a.ldo, cols)) return -1;
  return launch_fwd(a, kToRows, s);
}

int kv_append(const QkRopeArgs& in, cudaStream_t s) {
  QkRopeArgs a = in;
  a.kv_heads = a.v_heads = a.cache.kv_heads;
  a.hd = a.cache.hd;
  const int64_t cols = static_cast<int64_t>(a.heads + 2 * a.kv_heads) * a.hd;
  if (!kv_pages_ok(a.cache) || !rope_ok(a) || !rows_ok(a.x, a.ldx, cols) ||
      !rows_ok(a.out, a.ldo, static_cast<int64_t>(a.heads) * a.hd))
    return -1;
  return launch_fwd(a, a.cache.int8 ? kToInt8Pages : kToBf16Pages, s);
}

// One CTA holds up to 8 warps of items; 4 CTAs an SM.
int qk_rope_bwd_blocks(int T, int heads, int kv_heads) {
  if (T <= 0 || heads <= 0 || kv_heads <= 0) return 1;
  const int64_t groups = static_cast<int64_t>(T) * ((heads + 2 * kv_heads + 2 * kU - 1) / (2 * kU));
  const int64_t b = (groups + kWarps - 1) / kWarps;
  return static_cast<int>(b < 148 * 4 ? b : 148 * 4);
}

int qk_rope_bwd(const QkRopeArgs& a, cudaStream_t s) {
  const int64_t qk = static_cast<int64_t>(a.heads + a.kv_heads) * a.hd;
  const int64_t cols = qk + static_cast<int64_t>(a.v_heads) * a.hd;
  if (!rope_ok(a) || !rows_ok(a.dy, a.lddy, cols) || !rows_ok(a.out, a.ldo, cols)) return -1;
  if (a.gamma_q && !rows_ok(a.x, a.ldx, qk)) return -1;
  BwdParams p{};
  p.dy = a.dy; p.lddy = a.lddy; p.x = a.x; p.ldx = a.ldx; p.dx = a.out; p.lddx = a.ldo;
  p.rope = rope_dev(a);
  p.gq = a.gamma_q; p.gk = a.gamma_k; p.eps = a.eps;
  p.T = a.T; p.heads = a.heads; p.kv_heads = a.kv_heads;
  p.total_heads = a.heads + a.kv_heads + a.v_heads;
  p.chunks = chunks_of(p.total_heads, a.hd);
  p.part = a.partials;
  p.err = a.err;
  const int blocks = qk_rope_bwd_blocks(a.T, a.heads, a.kv_heads);
  if (a.hd == 128) qk_rope_bwd_kernel<128><<<blocks, kThreads, 0, s>>>(p);
  else qk_rope_bwd_kernel<64><<<blocks, kThreads, 0, s>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || !a.gamma_q) return e;
  qk_dgamma_kernel<<<dim3(a.hd / 32, 2), 1024, 0, s>>>(a.partials, blocks, a.dgamma_q, a.dgamma_k, a.hd, a.accumulate);
  return cudaGetLastError();
}

int kv_gather(const KvPages& c, const int32_t* slots, __nv_bfloat16* k_out, __nv_bfloat16* v_out, int64_t ldo, int T,
              int* err, cudaStream_t s) {
  const int64_t cols = static_cast<int64_t>(c.kv_heads) * c.hd;
  if (!kv_pages_ok(c) || T < 0 || !rows_ok(k_out, ldo, cols) || !rows_ok(v_out, ldo, cols)) return -1;
  GatherParams p{};
  p.ck = c.k; p.cv = c.v; p.sk = c.k_scale; p.sv = c.v_scale;
  p.slots = slots; p.k_out = k_out; p.v_out = v_out; p.ldo = ldo;
  p.n_slots = c.num_pages * c.page_size;
  p.T = T; p.kv_heads = c.kv_heads;
  p.chunks = chunks_of(c.kv_heads, c.hd);
  p.page_shift = log2_exact(c.page_size);
  p.err = err;
  const int64_t nb = blocks_of(static_cast<int64_t>(T) * p.chunks);
  if (nb < 0) return -1;
  if (nb == 0) return 0;
  const dim3 grid(static_cast<unsigned>(nb));
  if (c.hd == 128) {
    if (c.int8) kv_gather_kernel<128, true><<<grid, kThreads, 0, s>>>(p);
    else kv_gather_kernel<128, false><<<grid, kThreads, 0, s>>>(p);
  } else {
    if (c.int8) kv_gather_kernel<64, true><<<grid, kThreads, 0, s>>>(p);
    else kv_gather_kernel<64, false><<<grid, kThreads, 0, s>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace rt
