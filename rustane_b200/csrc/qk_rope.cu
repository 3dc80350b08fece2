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
// All are HBM-bound.  hd / 8 lanes own one head vector: a lane holds 4 first entries of
// rotated pairs and their 4 second ones (interleaved: 16 contiguous bytes; halves: 8 bytes each
// of two places), so pairs never cross lanes, and all arithmetic runs in packed fp32x2.  A
// warp holds 32 / (hd / 8) vectors; kU (backward kUb) of these are a group, loaded at once.
// The groups of all tokens are cut into equal runs, one per warp of a grid that fits the
// GPU: a warp has the next group's loads in flight while it works on one, and reads a token's
// position and tables once per run.  (Pairs exchanged by shuffles and scalar arithmetic: 17
// instructions an entry, half of all issue slots, 4.2 TB/s on 8209 tokens of 96 heads.)
// Measured: forward + backward of 16389 tokens of 32 + 8 + 8 heads of 128 215 us, 4.5 TB/s; append
// of 8209 tokens of 96 heads into bf16 pages 77 us, 5.3 TB/s; gather from int8 pages 116 us, 6.4
// TB/s, the copy rate.  16 warps an SM with one group in flight each are short of the copy rate:
// 24 warps with the groups as they are spill (378 us), with half the group 242 us.
#include "common.cuh"
#include "kernels.h"
#include "serving.h"

namespace rt {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kCtasPerSm = 2;
constexpr int kU = 4;   // vectors per lane group and group of heads: forward, gather
constexpr int kUb = 2;  // backward, which holds two inputs and two running sums

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }

// Sum / max over the LPH lanes that share a head vector (`mask`: at least those lanes).
template <int LPH>
__device__ __forceinline__ float head_sum(float v, uint32_t mask) {
#pragma unroll
  for (int o = LPH / 2; o; o >>= 1) v += __shfl_xor_sync(mask, v, o);
  return v;
}
template <int LPH>
__device__ __forceinline__ float head_max(float v, uint32_t mask) {
#pragma unroll
  for (int o = LPH / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(mask, v, o));
  return v;
}

struct RopeDev {
  const float* cos;
  const float* sin;
  const int32_t* pos;
  int n_pos, rot;
};

// Where lane `sub` of a vector finds its entries: 4 at a, 4 at b (interleaved: a's 8 entries
// alternate between the two).  Lanes past the rotated columns take 8 contiguous ones.
template <bool HALF>
struct Place {
  int a, b;
  bool turns;
  __device__ __forceinline__ Place(int sub, int rot) {
    turns = sub * 8 < rot;
    a = HALF && turns ? sub * 4 : sub * 8;
    b = HALF && turns ? sub * 4 + rot / 2 : sub * 8 + 4;
  }
  // the 8 entries as packed pairs of first entries f[2] and of second ones s[2]
  __device__ __forceinline__ void unpack(const uint4& u, uint64_t (&f)[2], uint64_t (&s)[2]) const {
    if (HALF) {
      f[0] = f2_pack(bf16lo(u.x), bf16hi(u.x));
      f[1] = f2_pack(bf16lo(u.y), bf16hi(u.y));
      s[0] = f2_pack(bf16lo(u.z), bf16hi(u.z));
      s[1] = f2_pack(bf16lo(u.w), bf16hi(u.w));
    } else {
      f[0] = f2_pack(bf16lo(u.x), bf16lo(u.y));
      f[1] = f2_pack(bf16lo(u.z), bf16lo(u.w));
      s[0] = f2_pack(bf16hi(u.x), bf16hi(u.y));
      s[1] = f2_pack(bf16hi(u.z), bf16hi(u.w));
    }
  }
  // v[8] in the order of the entries at a, then at b
  __device__ __forceinline__ void spread(const uint64_t (&f)[2], const uint64_t (&s)[2], float (&v)[8]) const {
    if (HALF) {
      f2_unpack(f[0], v[0], v[1]);
      f2_unpack(f[1], v[2], v[3]);
      f2_unpack(s[0], v[4], v[5]);
      f2_unpack(s[1], v[6], v[7]);
    } else {
      f2_unpack(f[0], v[0], v[2]);
      f2_unpack(f[1], v[4], v[6]);
      f2_unpack(s[0], v[1], v[3]);
      f2_unpack(s[1], v[5], v[7]);
    }
  }
  __device__ __forceinline__ uint4 load(const __nv_bfloat16* row) const {
    if (!HALF) return *reinterpret_cast<const uint4*>(row + a);
    const uint2 x = *reinterpret_cast<const uint2*>(row + a), y = *reinterpret_cast<const uint2*>(row + b);
    return make_uint4(x.x, x.y, y.x, y.y);
  }
  __device__ __forceinline__ void store(__nv_bfloat16* row, const uint4& u) const {
    if (HALF) {
      *reinterpret_cast<uint2*>(row + a) = make_uint2(u.x, u.y);
      *reinterpret_cast<uint2*>(row + b) = make_uint2(u.z, u.w);
    } else {
      *reinterpret_cast<uint4*>(row + a) = u;
    }
  }
  __device__ __forceinline__ uint4 pack(const uint64_t (&f)[2], const uint64_t (&s)[2]) const {
    float v[8];
    spread(f, s, v);
    return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                      pack_bf16x2(v[6], v[7]));
  }
  // the lane's entries of an fp32 vector, in the same packing
  __device__ __forceinline__ void gather(const float* g, uint64_t (&f)[2], uint64_t (&s)[2]) const {
    const float4 x = load4(g + a), y = load4(g + b);
    if (HALF) {
      f[0] = f2_pack(x.x, x.y);
      f[1] = f2_pack(x.z, x.w);
      s[0] = f2_pack(y.x, y.y);
      s[1] = f2_pack(y.z, y.w);
    } else {
      f[0] = f2_pack(x.x, x.z);
      f[1] = f2_pack(y.x, y.z);
      s[0] = f2_pack(x.y, x.w);
      s[1] = f2_pack(y.y, y.w);
    }
  }
};

// One lane's 4 angles of a token (either layout: pairs 4 sub .. 4 sub + 3).
struct Angles {
  uint64_t c[2], s[2];
};
__device__ __forceinline__ void load_angles(Angles& a, const RopeDev& r, int pos, int sub) {
  const int64_t at = static_cast<int64_t>(pos) * (r.rot / 2) + sub * 4;
  const float4 c = load4(r.cos + at), s = load4(r.sin + at);
  a.c[0] = f2_pack(c.x, c.y);
  a.c[1] = f2_pack(c.z, c.w);
  a.s[0] = f2_pack(s.x, s.y);
  a.s[1] = f2_pack(s.z, s.w);
}
__device__ __forceinline__ uint64_t f2_neg(uint64_t x) { return x ^ 0x8000000080000000ull; }
// (f, s) <- R (f, s) (BACK: R^T)
template <bool BACK>
__device__ __forceinline__ void rotate(uint64_t (&f)[2], uint64_t (&s)[2], const Angles& a) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint64_t up = BACK ? a.s[i] : f2_neg(a.s[i]), dn = BACK ? f2_neg(a.s[i]) : a.s[i];
    const uint64_t x = f2_fma(s[i], up, f2_mul(f[i], a.c[i]));
    s[i] = f2_fma(f[i], dn, f2_mul(s[i], a.c[i]));
    f[i] = x;
  }
}
// (f, s) <- (f, s) * r * (g, h)
__device__ __forceinline__ void scale(uint64_t (&f)[2], uint64_t (&s)[2], float r, const uint64_t (&g)[2],
                                      const uint64_t (&h)[2]) {
  const uint64_t r2 = f2_pack(r, r);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f[i] = f2_mul(f2_mul(f[i], r2), g[i]);
    s[i] = f2_mul(f2_mul(s[i], r2), h[i]);
  }
}
__device__ __forceinline__ float dot8(const uint64_t (&f)[2], const uint64_t (&s)[2], const uint64_t (&g)[2],
                                      const uint64_t (&h)[2]) {
  float x, y;
  f2_unpack(f2_fma(s[1], h[1], f2_fma(s[0], h[0], f2_fma(f[1], g[1], f2_mul(f[0], g[0])))), x, y);
  return x + y;
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

// A warp's run [g, g1) of the groups (token, chunk of heads), and the position at hand.
struct Run {
  int64_t g, g1;
  int tok, chunk;
  __device__ __forceinline__ Run(int64_t groups, int chunks) {
    const int64_t w = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    const int64_t n = static_cast<int64_t>(gridDim.x) * kWarps;
    g = groups * w / n;
    g1 = groups * (w + 1) / n;
    tok = static_cast<int>(g / chunks);
    chunk = static_cast<int>(g - static_cast<int64_t>(tok) * chunks);
  }
  __device__ __forceinline__ void next(int chunks) {
    ++g;
    if (++chunk == chunks) {
      chunk = 0;
      ++tok;
    }
  }
};

__device__ __forceinline__ int position(const RopeDev& r, int tok, int* err) {
  const int pos = r.pos[tok];
  if (pos >= 0 && pos < r.n_pos) return pos;
  set_error(err, kDevBadIndex);
  return 0;
}

template <int HD, int DEST, bool HALF>
__global__ void __launch_bounds__(kThreads, 2) qk_rope_fwd_kernel(const FwdParams p) {
  constexpr int LPH = HD / 8, HPW = 32 / LPH;  // lanes per head vector, vectors per warp
  __shared__ __align__(16) float gam[2][HD];
  const int lane = threadIdx.x & 31, sub = lane % LPH, hw = lane / LPH;
  const uint32_t mates = ((1u << LPH) - 1u) << (hw * LPH);  // the vector's lanes
  const Place<HALF> at(sub, p.rope.rot);
  if (p.gq) {
    for (int i = threadIdx.x; i < 2 * HD; i += kThreads) gam[i / HD][i % HD] = (i < HD ? p.gq : p.gk)[i % HD];
    __syncthreads();
  }
  Run run(static_cast<int64_t>(p.T) * p.chunks, p.chunks);
  uint4 ahead[kU];
  auto load = [&](const Run& r) {
    const __nv_bfloat16* row = p.x + r.tok * p.ldx;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int h = r.chunk * (HPW * kU) + hw + u * HPW;
      ahead[u] = make_uint4(0, 0, 0, 0);
      if (r.g < r.g1 && h < p.total_heads) ahead[u] = at.load(row + static_cast<int64_t>(h) * HD);
    }
  };
  load(run);
  Angles ang;
  int64_t slot = -1;
  int have = -1;  // the token whose angles and slot are at hand
  while (run.g < run.g1) {
    const int tok = run.tok, run_chunk = run.chunk, h0 = run_chunk * (HPW * kU) + hw;
    if (tok != have) {
      const int pos = position(p.rope, tok, p.err);
      if (at.turns) load_angles(ang, p.rope, pos, sub);
      if (DEST != kToRows) {
        slot = p.slots[tok];
        if (slot < -1 || slot >= p.n_slots) {
          set_error(p.err, kDevBadIndex);
          slot = -1;
        }
      }
      have = tok;
    }
    uint4 raw[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) raw[u] = ahead[u];
    run.next(p.chunks);
    load(run);

    const int h_first = run_chunk * (HPW * kU), h_last = h_first + HPW * kU - 1;
    const bool all_turn = h_last < p.heads + p.kv_heads;  // the group holds q and k vectors only
    uint64_t f[kU][2], s[kU][2];
    if (all_turn || DEST == kToInt8Pages || h_first < p.heads + p.kv_heads) {
#pragma unroll
      for (int u = 0; u < kU; ++u) at.unpack(raw[u], f[u], s[u]);
    }
    // Of a group of q and k vectors alone the kU chains of loads, sums and shuffles run side by
    // side; a mixed group takes them one by one.
    if (all_turn) {
      float r[kU];
      if (p.gq) {
#pragma unroll
        for (int u = 0; u < kU; ++u) r[u] = dot8(f[u], s[u], f[u], s[u]);
#pragma unroll
        for (int o = LPH / 2; o; o >>= 1)
#pragma unroll
          for (int u = 0; u < kU; ++u) r[u] += __shfl_xor_sync(0xffffffffu, r[u], o);
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          uint64_t gf[2], gs[2];
          at.gather(gam[h0 + u * HPW < p.heads ? 0 : 1], gf, gs);
          scale(f[u], s[u], rsqrtf(r[u] * (1.0f / HD) + p.eps), gf, gs);
        }
      }
      if (at.turns) {
#pragma unroll
        for (int u = 0; u < kU; ++u) rotate<false>(f[u], s[u], ang);
      }
#pragma unroll
      for (int u = 0; u < kU; ++u) raw[u] = at.pack(f[u], s[u]);
    } else if (h_first < p.heads + p.kv_heads) {
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int h = h0 + u * HPW;
        if (h >= p.heads + p.kv_heads) continue;  // a whole vector's lanes
        if (p.gq) {
          uint64_t gf[2], gs[2];
          at.gather(gam[h < p.heads ? 0 : 1], gf, gs);
          scale(f[u], s[u], rsqrtf(head_sum<LPH>(dot8(f[u], s[u], f[u], s[u]), mates) * (1.0f / HD) + p.eps), gf, gs);
        }
        if (at.turns) rotate<false>(f[u], s[u], ang);
        raw[u] = at.pack(f[u], s[u]);
      }
    }

#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int h = h0 + u * HPW;
      if (h >= p.total_heads) continue;
      const bool is_q = h < p.heads, is_v = h >= p.heads + p.kv_heads;
      if (DEST == kToRows || is_q) {
        at.store(p.out + tok * p.ldo + static_cast<int64_t>(h) * HD, raw[u]);
        continue;
      }
      const int kh = is_v ? h - p.heads - p.kv_heads : h - p.heads;
      const int64_t page = slot >> p.page_shift, off = slot & ((1 << p.page_shift) - 1);
      const int64_t row = (((page * p.kv_heads + kh) << p.page_shift) + off);
      if (DEST == kToBf16Pages) {
        if (slot >= 0) at.store(static_cast<__nv_bfloat16*>(is_v ? p.cv : p.ck) + row * HD, raw[u]);
      } else {
        float v[8], amax = 0.f;
        at.spread(f[u], s[u], v);
        bool finite = true;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          amax = fmaxf(amax, fabsf(v[i]));
          finite = finite && isfinite(v[i]);
        }
        amax = head_max<LPH>(finite ? amax : INFINITY, mates);
        const float scale = isinf(amax) ? NAN : amax / 127.0f;
        uint32_t b[2] = {0, 0};
        if (scale > 0.f) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            // |y / s| <= 127 but for the rounding of a denormal scale
            const int c = max(-127, min(127, __float2int_rn(v[i] / scale)));
            b[i >> 2] |= static_cast<uint32_t>(c & 0xff) << (8 * (i & 3));
          }
        }
        if (slot >= 0) {
          int8_t* dst = static_cast<int8_t*>(is_v ? p.cv : p.ck) + row * HD;
          if (HALF) {
            *reinterpret_cast<uint32_t*>(dst + at.a) = b[0];
            *reinterpret_cast<uint32_t*>(dst + at.b) = b[1];
          } else {
            *reinterpret_cast<uint2*>(dst + at.a) = make_uint2(b[0], b[1]);
          }
          if (sub == 0) (is_v ? p.sv : p.sk)[row] = scale;
        }
      }
    }
  }
}

// Backward.  Every warp keeps the dgamma sums of its run in registers; each CTA adds its
// warps' sums in a fixed order and writes one partial row per gamma.
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

template <int HD, bool HALF>
__global__ void __launch_bounds__(kThreads, 2) qk_rope_bwd_kernel(const BwdParams p) {
  constexpr int LPH = HD / 8, HPW = 32 / LPH;
  __shared__ float red[2][kWarps * HPW][HD];
  __shared__ __align__(16) float gam[2][HD];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % LPH, hw = lane / LPH;
  const uint32_t mates = ((1u << LPH) - 1u) << (hw * LPH);
  const Place<HALF> at(sub, p.rope.rot);
  if (p.gq) {
    for (int i = threadIdx.x; i < 2 * HD; i += kThreads) gam[i / HD][i % HD] = (i < HD ? p.gq : p.gk)[i % HD];
    __syncthreads();
  }
  uint64_t sum_f[2][2] = {}, sum_s[2][2] = {};  // dgamma of q, k
  Run run(static_cast<int64_t>(p.T) * p.chunks, p.chunks);
  uint4 ahead_d[kUb], ahead_x[kUb];
  auto load = [&](const Run& r) {
#pragma unroll
    for (int u = 0; u < kUb; ++u) {
      const int h = r.chunk * (HPW * kUb) + hw + u * HPW;
      const int64_t col = static_cast<int64_t>(h) * HD;
      ahead_d[u] = ahead_x[u] = make_uint4(0, 0, 0, 0);
      if (r.g < r.g1 && h < p.total_heads) ahead_d[u] = at.load(p.dy + r.tok * p.lddy + col);
      if (r.g < r.g1 && p.gq && h < p.heads + p.kv_heads) ahead_x[u] = at.load(p.x + r.tok * p.ldx + col);
    }
  };
  load(run);
  Angles ang;
  int have = -1;
  while (run.g < run.g1) {
    const int64_t tok = run.tok;
    const int run_chunk = run.chunk, h0 = run_chunk * (HPW * kUb) + hw;
    if (run.tok != have) {
      const int pos = position(p.rope, run.tok, p.err);
      if (at.turns) load_angles(ang, p.rope, pos, sub);
      have = run.tok;
    }
    uint4 rd[kUb], rx[kUb];
#pragma unroll
    for (int u = 0; u < kUb; ++u) {
      rd[u] = ahead_d[u];
      rx[u] = ahead_x[u];
    }
    run.next(p.chunks);
    load(run);
    // Every vector takes the same steps, so that the kUb chains run side by side; v's result
    // is its input, and vectors past the last are zeros that go nowhere.
    if (run_chunk * (HPW * kUb) < p.heads + p.kv_heads) {
      uint64_t df[kUb][2], ds[kUb][2];
#pragma unroll
      for (int u = 0; u < kUb; ++u) {
        at.unpack(rd[u], df[u], ds[u]);
        if (at.turns) rotate<true>(df[u], ds[u], ang);
      }
      if (p.gq) {
        uint64_t xf[kUb][2], xs[kUb][2];
        float r[kUb], dot[kUb];
#pragma unroll
        for (int u = 0; u < kUb; ++u) {
          at.unpack(rx[u], xf[u], xs[u]);
          r[u] = dot8(xf[u], xs[u], xf[u], xs[u]);
        }
#pragma unroll
        for (int o = LPH / 2; o; o >>= 1)
#pragma unroll
          for (int u = 0; u < kUb; ++u) r[u] += __shfl_xor_sync(0xffffffffu, r[u], o);
#pragma unroll
        for (int u = 0; u < kUb; ++u) {
          const int h = h0 + u * HPW;
          r[u] = rsqrtf(r[u] * (1.0f / HD) + p.eps);
          const uint64_t r2 = f2_pack(r[u], r[u]);
          const bool to_q = h < p.heads, to_k = !to_q && h < p.heads + p.kv_heads;
          uint64_t gf[2], gs[2];
          at.gather(gam[h < p.heads ? 0 : 1], gf, gs);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            xf[u][i] = f2_mul(xf[u][i], r2);
            xs[u][i] = f2_mul(xs[u][i], r2);
            const uint64_t tf = f2_mul(df[u][i], xf[u][i]), ts = f2_mul(ds[u][i], xs[u][i]);
            sum_f[0][i] = f2_add(sum_f[0][i], to_q ? tf : 0ull);
            sum_s[0][i] = f2_add(sum_s[0][i], to_q ? ts : 0ull);
            sum_f[1][i] = f2_add(sum_f[1][i], to_k ? tf : 0ull);
            sum_s[1][i] = f2_add(sum_s[1][i], to_k ? ts : 0ull);
            df[u][i] = f2_mul(df[u][i], gf[i]);
            ds[u][i] = f2_mul(ds[u][i], gs[i]);
          }
          dot[u] = dot8(df[u], ds[u], xf[u], xs[u]);
        }
#pragma unroll
        for (int o = LPH / 2; o; o >>= 1)
#pragma unroll
          for (int u = 0; u < kUb; ++u) dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], o);
#pragma unroll
        for (int u = 0; u < kUb; ++u) {
          const uint64_t r2 = f2_pack(r[u], r[u]), m2 = f2_pack(dot[u] * (-1.0f / HD), dot[u] * (-1.0f / HD));
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            df[u][i] = f2_mul(f2_fma(xf[u][i], m2, df[u][i]), r2);
            ds[u][i] = f2_mul(f2_fma(xs[u][i], m2, ds[u][i]), r2);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kUb; ++u)
        if (h0 + u * HPW < p.heads + p.kv_heads) rd[u] = at.pack(df[u], ds[u]);
    }
#pragma unroll
    for (int u = 0; u < kUb; ++u) {
      const int h = h0 + u * HPW;
      if (h < p.total_heads) at.store(p.dx + tok * p.lddx + static_cast<int64_t>(h) * HD, rd[u]);
    }
  }
  if (!p.gq) return;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float v[8];
    at.spread(sum_f[w], sum_s[w], v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      red[w][warp * HPW + hw][at.a + i] = v[i];
      red[w][warp * HPW + hw][at.b + i] = v[4 + i];
    }
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
        o = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                       pack_bf16x2(v[6], v[7]));
      }
      *reinterpret_cast<uint4*>((w ? p.v_out : p.k_out) + tok * p.ldo + static_cast<int64_t>(h) * HD + sub * 8) = o;
    }
  }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

inline int chunks_of(int total_heads, int hd, int u = kU) {
  const int per = (32 / (hd / 8)) * u;
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
  return {a.rope.cos, a.rope.sin, a.pos, a.rope.n_pos, a.rope.rot};
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
  const int64_t nb = (static_cast<int64_t>(a.T) * p.chunks + kWarps - 1) / kWarps;
  if (nb == 0) return 0;
  const int most = kCtasPerSm * num_sms();
  const unsigned grid = static_cast<unsigned>(nb < most ? nb : most);
#define RT_FWD(HD, DEST)                                                            \
  do {                                                                              \
    if (a.rope.half) qk_rope_fwd_kernel<HD, DEST, true><<<grid, kThreads, 0, s>>>(p); \
    else qk_rope_fwd_kernel<HD, DEST, false><<<grid, kThreads, 0, s>>>(p);          \
  } while (0)
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

// The backward's grid, a function of the sizes alone (not of the device), fixes the order of
// the dgamma sums.
int qk_rope_bwd_blocks(int T, int heads, int kv_heads) {
  if (T <= 0 || heads <= 0 || kv_heads <= 0) return 1;
  const int64_t groups = static_cast<int64_t>(T) * ((heads + 2 * static_cast<int64_t>(kv_heads) + 2 * kUb - 1) / (2 * kUb));
  const int64_t b = (groups + kWarps - 1) / kWarps;
  return static_cast<int>(b < 148 * kCtasPerSm ? b : 148 * kCtasPerSm);
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
  p.chunks = chunks_of(p.total_heads, a.hd, kUb);
  p.part = a.partials;
  p.err = a.err;
  const int blocks = qk_rope_bwd_blocks(a.T, a.heads, a.kv_heads);
  if (a.hd == 128) {
    if (a.rope.half) qk_rope_bwd_kernel<128, true><<<blocks, kThreads, 0, s>>>(p);
    else qk_rope_bwd_kernel<128, false><<<blocks, kThreads, 0, s>>>(p);
  } else {
    if (a.rope.half) qk_rope_bwd_kernel<64, true><<<blocks, kThreads, 0, s>>>(p);
    else qk_rope_bwd_kernel<64, false><<<blocks, kThreads, 0, s>>>(p);
  }
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
