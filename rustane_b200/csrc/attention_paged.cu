// Attention of each sequence's new tokens over its paged key/value cache.
//
// Sequence s has n = q_start[s+1] - q_start[s] new tokens (rows of q) and L = kv_lens[s]
// cached tokens, the new ones included: new token i sits at position L - n + i and sees
// keys (position - window, position] (window 0: all of [0, position]).
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - max);  lse2 = log2 sum exp
// A row that sees no key (L < n, or an unused batch slot) gives o = 0, lse2 = -inf.
//
// This file: up to 16 rows per key head (a decode step).  HBM-bound: K and V of every
// visible token are read once, 2 hd bytes a token and head each (int8: hd + 4).  The keys are
// the 16 rows of the m16n8k16 products (S^T = K Q^T, O^T = V^T P^T) and the query rows their 8
// columns, NT times: with the query rows as the 16, a step of 1 to 8 rows issued twice the
// products and held twice the sums.
//
// 160 threads a CTA, three CTAs an SM (NT 2: two; hd 64: one more): warp 4 streams 64-key blocks by TMA (one box
// per page and 128 bytes of head, swizzled) into a ring of 32 to 96 KB (Cfg::STAGES blocks); warps 0-3 take 16 keys
// of each block for all rows, each with its own running maximum, sum and output, which meet in
// the last block's ring slot when the item (or the CTA's part of it) ends.  A weight goes into the
// P V product as the sum of two bf16 numbers, 2^-15 of it off: its leading 8 bits, then what they leave
// (2^-7 of it).  Both are above 0 where the weight is, so that an infinite v stays infinite.
//
// Measured, of the copy rate: 8 sequences of up to 40037 tokens, 32 query and 8 key heads, 176 us
// (99%); 48 x 3000 of 16 heads 183 us (98%); 48 x up to 6011 tokens of 32 heads in int8 253 us (78%); the same
// at hd 64 191 us (100%), in int8 187 us (54%); one sequence of 512 tokens of 12 heads 9.7 us, most of
// it the launch and a chain of dependent loads (lengths, page, keys) and the join.  int8 takes two thirds
// as long at half the head: the rest is work per 16 keys (the maximum across lanes, votes, units, scales).
//
// int8: the codes become fp16, exactly (two and a half instructions a pair, one and a half of
// them on the integer pipe; bf16 takes four and three, and that pipe was the limit: 354 us
// for the int8 case above).  Each row of q is brought into fp16's range by a
// power of two, exact down to 2^-22 of its largest entry; k's scale multiplies the score in fp32.
// The weights times v's scales are rounded to fp16 (2^-11 of each) in units of 2^kv, a power of
// two of each row that moves, with the row's sums, when its largest weight leaves [2^0, 2^15)
// units.  (One power for all rows of an item lost those of much smaller q, and those before a
// token whose v is 2^26 times larger; the int8 case took 245 us.)  A step with a key whose scale lies
// far below a row's unit takes its small weights in further products of 2^-24 the unit each, so
// that columns where the large keys hold zeros keep theirs.
#include <cuda_fp16.h>

#include "attention_paged.cuh"
#include "kernels.h"

namespace rt {
namespace paged {
namespace {

constexpr int kBK = 64;   // keys per block
constexpr int kConsumers = 4;
constexpr int kThreads = (kConsumers + 1) * 32;
constexpr float kLeft = 0x1p-18f;  // of a weight, added to what its leading bits leave: never 0

template <int HD, bool I8, int NT>
struct Cfg {
  static constexpr int BM = 8 * NT;                    // rows per tile
  // As many CTAs an SM as the registers allow; they share the shared memory.  hd 64, 48 x up to 6011
  // tokens of 32 heads: four 199 us (int8 193), three 211 (227), five, with spills, 210 (225).  hd 128 in int8
  // with four: 265 against 252.
  static constexpr int CTAS = (NT == 1 ? 3 : 2) + (HD == 64 ? 1 : 0);
  static constexpr int ROW = HD * (I8 ? 1 : 2);  // bytes of a key
  static constexpr int TILE = kBK * ROW;
  static constexpr int SCALES = I8 ? kBK * 4 : 0;
  static constexpr int STAGE = 2 * TILE + 2 * SCALES;  // K, V, scales of k, of v
  static constexpr int SLOT = (STAGE + 1023) / 1024 * 1024;
  // Blocks in flight.  hd 64 in bf16 would have the shared memory for one more; 48 x 6011 tokens of 32 heads
  // take 348 us with two, 361 with three.
  static constexpr int STAGES = HD == 128 ? (NT == 1 ? (I8 ? 3 : 2) : I8 ? 5 : 3) : NT == 1 ? (I8 ? 5 : 2) : I8 ? 6 : 3;
  static constexpr int BOX = ROW < 128 ? ROW : 128;  // bytes of a row in one TMA box
  static constexpr int BOXES = ROW / BOX;
  // the four warps' outputs meet CHUNK columns at a time in the last block's slot
  static constexpr int CHUNK = 2 * TILE / (kConsumers * BM * 4) < HD ? 2 * TILE / (kConsumers * BM * 4) : HD;
  static constexpr int TPR = kConsumers * 32 / BM;  // threads per row at the end
  static constexpr int BAR = STAGES * SLOT;
  static constexpr int ML = BAR + 256;                     // float [warp][row][2]
  static constexpr int FIX = ML + kConsumers * BM * 8;    // float [row][2] of recomputed rows
  static constexpr int BYTES = FIX + BM * 8 + 64 + 1024;  // + flags, alignment slack
};

// byte offset of 16-byte chunk ch of row r in a TMA-swizzled tile of kBK rows
template <int ROW>
__device__ __forceinline__ uint32_t tile_off(int r, int ch) {
  if (ROW == 64) return r * 64 + ((ch ^ ((r >> 1) & 3)) << 4);
  return (ch >> 3) * (kBK * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816h(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Codes I and J of a word whose sign bits are flipped (codes + 128), in fp16: 1024 + (code + 128)
// is exact with the codes as the last mantissa bits, and so is the difference.
template <int I, int J>
__device__ __forceinline__ uint32_t codes_f16x2(uint32_t flipped) {
  const uint32_t x = __byte_perm(flipped, 0x64646464u, I | 0x40 | (J << 8) | 0x4000), y = 0x64806480u;  // 1152
  const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&y));
  return *reinterpret_cast<const uint32_t*>(&d);
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float power_of_2(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }
// 8 x 8 16-bit matrix, a row to 4 lanes: transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void consumer_bar() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <int HD, bool I8, int NT>
__global__ void __launch_bounds__(kThreads, Cfg<HD, I8, NT>::CTAS)
    attn_paged_few_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                          const __grid_constant__ Params p) {
  using C = Cfg<HD, I8, NT>;
  constexpr int kBM = C::BM;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BAR);
  uint64_t* empty = full + C::STAGES;
  float* ml = reinterpret_cast<float*>(smem + C::ML);
  float* fix = reinterpret_cast<float*>(smem + C::FIX);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::FIX + kBM * 8);
  volatile int* is_last = abort_flag + 1;
  volatile unsigned* nan_rows = reinterpret_cast<volatile unsigned*>(abort_flag + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PagedAttnArgs& a = p.a;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kConsumers);
    }
    *abort_flag = 0;
    *nan_rows = 0;
    fence_mbar_init();
  }
  int64_t total;
  int P;
  Walk<kBK> w = start_walk<kBK, kThreads>(p, total, P);  // its barriers cover the init above

  if (warp == kConsumers) {
    // ------------------------------------------------------------------ producer
    // lane i < boxes of a block loads `sub` keys: a page, or half of one of 128
    if (lane == 0) {
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
    const int ps = 1 << p.page_shift, sub = ps < kBK ? ps : kBK;
    int g = 0;
    bool ok = true;
    for (; ok && w.more(); w.next()) {
      if (w.empty()) continue;
      const int32_t* table = a.table + w.s * a.table_ld;
      const int cnt = w.count();
      const int key00 = (w.blk0 + w.off) * kBK;
      // this lane's page of a block (fetched one block ahead of its use), -1: no key of it is seen
      auto my_page = [&](int b) {
        const int key = key00 + b * kBK + lane * sub;
        return b < cnt && lane * sub < kBK && key < w.hi && key + sub > w.lo ? page_of(p, table, key) : -1;
      };
      int page = my_page(0);
      for (int b = 0; b < cnt; ++b, ++g) {
        const int st = g % C::STAGES;
        const int key0 = key00 + b * kBK;
        const int ahead = my_page(b + 1);
        bool go = mbar_wait(&empty[st], ((g / C::STAGES) & 1) ^ 1) && !*abort_flag;
        if (!__all_sync(0xffffffffu, go)) {
          ok = false;
          break;
        }
        const int loads = __popc(__ballot_sync(0xffffffffu, page >= 0));
        uint8_t* slot = smem + st * C::SLOT;
        if (lane == 0) mbar_arrive_expect_tx(&full[st], loads * sub * (2 * C::ROW + (I8 ? 8 : 0)));
        __syncwarp();
        if (page >= 0) {
          const int64_t row64 = ((static_cast<int64_t>(page) * a.cache.kv_heads + w.h) << p.page_shift) +
                                ((key0 + lane * sub) & (ps - 1));
          const int row = static_cast<int>(row64);
          const uint32_t at = lane * sub * C::BOX;
#pragma unroll
          for (int x = 0; x < C::BOXES; ++x) {
            tma_load_2d(slot + x * (kBK * C::BOX) + at, &tm_k, &full[st], x * C::BOX, row);
            tma_load_2d(slot + C::TILE + x * (kBK * C::BOX) + at, &tm_v, &full[st], x * C::BOX, row);
          }
          if (I8) {
            uint8_t* sc = slot + 2 * C::TILE + lane * sub * 4;
            bulk_load(sc, a.cache.k_scale + row64, sub * 4, &full[st]);
            bulk_load(sc + C::SCALES, a.cache.v_scale + row64, sub * 4, &full[st]);
          }
        }
        __syncwarp();
        page = ahead;
      }
    }
    if (!ok) {  // let copies still in flight land before the CTA exits
      if (lane == 0) set_error(a.err, kDevTimeoutProducer);
      *abort_flag = 1;
      for (int x = g > C::STAGES ? g - C::STAGES : 0; x < g; ++x)
        mbar_wait(&full[x % C::STAGES], (x / C::STAGES) & 1);
    }
    return;
  }

  // -------------------------------------------------------------------- consumers
  constexpr int KS = HD / 16;  // k-steps of K Q^T; groups of 16 output columns of V^T P^T
  const int gr = lane >> 2, c = lane & 3;
  const uint32_t ring = smem_u32(smem);
  int g = 0;
  bool ok = true;
  for (; w.more(); w.next()) {
    const int rows = w.rows(), cnt = w.count();
    const int r0 = w.t * kBM;
    auto q_ptr = [&](int r) {
      const int i = (r0 + r) / p.G, hg = w.h * p.G + (r0 + r) % p.G;
      return a.q + (w.q0 + i) * a.ldq + hg * HD;
    };
    auto write_row4 = [&](int r, int col, const float (&o)[4]) {
      const int i = (r0 + r) / p.G, hg = w.h * p.G + (r0 + r) % p.G;
      *reinterpret_cast<uint2*>(a.out + (w.q0 + i) * a.ldo + hg * HD + col) =
          make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
    };
    auto write_lse = [&](int r, float v) {
      const int i = (r0 + r) / p.G, hg = w.h * p.G + (r0 + r) % p.G;
      if (a.lse2) a.lse2[static_cast<int64_t>(w.q0 + i) * a.heads + hg] = v;
    };
    // thread's share of the rows at the end: row er, columns 4 ec + 4 TPR j
    const int er = threadIdx.x / C::TPR, ec = threadIdx.x % C::TPR;
    if (w.empty()) {
      if (er < rows) {
        const float zero[4] = {0.f, 0.f, 0.f, 0.f};
        for (int col = 4 * ec; col < HD; col += 4 * C::TPR) write_row4(er, col, zero);
        if (ec == 0) write_lse(er, -CUDART_INF_F);
      }
      continue;
    }

    // Q^T: row 8 t + gr.  An int8 key's 16 bytes of a k-step arrive 4 to a thread, so there the
    // k index 2c, 2c + 1, 2c + 8, 2c + 9 stands for entries 4c .. 4c + 3.
    uint32_t qb[KS][NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = 8 * t + gr;
      const bool in = r < rows;
      const __nv_bfloat16* q = q_ptr(in ? r : 0);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const uint32_t* x = reinterpret_cast<const uint32_t*>(q + ks * 16 + (I8 ? 4 * c : 2 * c));
        qb[ks][t][0] = in ? x[0] : 0u;
        qb[ks][t][1] = in ? x[I8 ? 1 : 4] : 0u;
      }
    }
    float s_scale[NT][2];  // of rows 8 t + 2c + x
    int kv[NT][2];         // int8: O is in units of 2^kv
    float least = 1.f;     // the smallest 2^-kv of the thread's rows
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        s_scale[t][x] = p.scale_log2;
        kv[t][x] = 0;
      }
    if (I8) {
      // each row's largest finite entry to [2^8, 2^9)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        unsigned top = 0;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const unsigned hi16 = qb[ks][t][x] >> 16 & 0x7fffu, lo16 = qb[ks][t][x] & 0x7fffu;
            top = max(top, max(hi16 < 0x7f80u ? hi16 : 0u, lo16 < 0x7f80u ? lo16 : 0u));
          }
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
        const int eq = max(-100, static_cast<int>(top >> 7) - 127 - 8);
        const float down = power_of_2(-eq);
#pragma unroll
        for (int x = 0; x < 2; ++x) s_scale[t][x] *= power_of_2(__shfl_sync(0xffffffffu, eq, (2 * c + x) * 4));
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int x = 0; x < 2; ++x) qb[ks][t][x] = pack_f16x2(bf16lo(qb[ks][t][x]) * down, bf16hi(qb[ks][t][x]) * down);
      }
    }
    // O^T of columns dg * 16 ..: entries 0, 1 (rows 8 t + 2c, + 1) of column gr (int8: 2 gr),
    // entries 2, 3 of column gr + 8 (int8: 2 gr + 1)
    float o[KS][NT][4];
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][t][e] = 0.f;
    float m[NT][2], l[NT][2];
    int hi_r[NT][2], lo_r[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = min(8 * t + 2 * c + x, rows - 1);
        m[t][x] = -CUDART_INF_F;
        l[t][x] = 0.f;
        hi_r[t][x] = w.row_hi(r);
        lo_r[t][x] = w.row_lo(r);
      }
    // keys that every row sees
    const int lo_all = w.row_lo(rows - 1), hi_all = w.row_hi(0);

    for (int b = 0; b < cnt; ++b, ++g) {
      const int st = g % C::STAGES;
      const int key0 = (w.blk0 + w.off + b) * kBK + warp * 16;  // the warp's keys
      ok = __all_sync(0xffffffffu, ok && mbar_wait(&full[st], (g / C::STAGES) & 1) && !*abort_flag);
      if (!ok) *abort_flag = 1;  // the loops run on without waiting: every warp meets the same barriers
      const uint32_t slot = ring + st * C::SLOT;
      if (ok && key0 < w.hi && key0 + 16 > w.lo) {
        float s[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[t][e] = 0.f;
        // ------------------------------------------------- S^T = K Q^T: 16 keys x 8 NT rows
        if (!I8) {
          const int key = warp * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            uint32_t ka[4];
            ldsm4(slot + tile_off<C::ROW>(key, 2 * ks + (lane >> 4)), ka);
#pragma unroll
            for (int t = 0; t < NT; ++t) mma16816(s[t], ka, qb[ks][t][0], qb[ks][t][1]);
          }
        } else {
          const int key = warp * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
#pragma unroll
          for (int ks = 0; ks < KS; ks += 2) {
            uint32_t kb[4];
            ldsm4(slot + tile_off<C::ROW>(key, ks + (lane >> 4)), kb);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const uint32_t k0 = kb[2 * x] ^ 0x80808080u, k1 = kb[2 * x + 1] ^ 0x80808080u;
              const uint32_t ka[4] = {codes_f16x2<0, 1>(k0), codes_f16x2<0, 1>(k1), codes_f16x2<2, 3>(k0),
                                      codes_f16x2<2, 3>(k1)};
#pragma unroll
              for (int t = 0; t < NT; ++t) mma16816h(s[t], ka, qb[ks + x][t][0], qb[ks + x][t][1]);
            }
          }
        }
        // ------------------------------------------------- scale, mask, running maximum
        const bool masked = key0 < lo_all || key0 + 16 > hi_all;
        float vs[2] = {1.f, 1.f}, ks2[2] = {1.f, 1.f};
        if (I8) {
          const float* sc = reinterpret_cast<const float*>(smem + st * C::SLOT + 2 * C::TILE) + warp * 16 + gr;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            ks2[x] = sc[8 * x];
            vs[x] = sc[kBK + 8 * x];
          }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[t][e] *= I8 ? s_scale[t][e & 1] * ks2[e >> 1] : p.scale_log2;
        uint32_t seen = 0xffffffffu;  // bit 4 t + e
        if (masked) {
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = key0 + gr + 8 * (e >> 1);
              if (key < lo_r[t][e & 1] || key >= hi_r[t][e & 1]) {
                s[t][e] = -CUDART_INF_F;
                seen &= ~(1u << (4 * t + e));
              }
            }
        }
        float mx[NT][2];
        bool grow = false;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            mx[t][x] = fmaxf(s[t][x], s[t][2 + x]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) mx[t][x] = fmaxf(mx[t][x], __shfl_xor_sync(0xffffffffu, mx[t][x], d));
            grow = grow || mx[t][x] > m[t][x] + kRescale;
          }
        const bool raised = __any_sync(0xffffffffu, grow);
        int fell[NT][2];  // int8: a row's O fell by 2^fell or more (255: it was 0)
#pragma unroll
        for (int t = 0; t < NT; ++t) fell[t][0] = fell[t][1] = 0;
        if (raised) {
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            float f[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const bool gx = mx[t][x] > m[t][x] + kRescale;
              f[x] = gx ? ex2_approx(m[t][x] - mx[t][x]) : 1.f;
              if (I8 && gx) fell[t][x] = m[t][x] == -CUDART_INF_F ? 255 : static_cast<int>(fminf(mx[t][x] - m[t][x], 255.f));
              if (gx) m[t][x] = mx[t][x];
              l[t][x] *= f[x];
            }
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[i][t][e] *= f[e & 1];
          }
        }
        // ------------------------------------------------------- P^T: 16 keys x 8 NT rows
        uint32_t pb[NT][2], pr[NT][2];  // pr (bf16): what pb leaves of the weight
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            // a maximum of -inf (nothing seen yet) is taken as 0: the weights come out 0
            const float mm = m[t][e & 1] == -CUDART_INF_F ? 0.f : m[t][e & 1];
            s[t][e] = ex2_approx(s[t][e] - mm);
            l[t][e & 1] += s[t][e];
            if (I8) {
              s[t][e] *= vs[e >> 1];
              if (masked && !((seen >> (4 * t + e)) & 1u)) s[t][e] = 0.f;  // whatever the scale was
            }
          }
          if (!I8) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float z0 = s[t][2 * x], z1 = s[t][2 * x + 1];
              const uint32_t lead = __byte_perm(__float_as_uint(z0), __float_as_uint(z1), 0x7632);
              pb[t][x] = transpose8(lead);
              pr[t][x] = transpose8(pack_bf16x2(fmaf(z0, kLeft, z0 - bf16lo(lead)), fmaf(z1, kLeft, z1 - bf16hi(lead))));
            }
          }
        }
        float y[NT][4];
        bool wide = false;  // int8: a key's scale lies far below a row's unit
        if (I8) {
          auto in_units = [&] {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              const float unit[2] = {power_of_2(-kv[t][0]), power_of_2(-kv[t][1])};
#pragma unroll
              for (int e = 0; e < 4; ++e) y[t][e] = s[t][e] * unit[e & 1];
            }
          };
          in_units();
          auto far_below = [&] {
            return (vs[0] != 0.f && fabsf(vs[0]) * least < 0.25f) || (vs[1] != 0.f && fabsf(vs[1]) * least < 0.25f);
          };
          bool rare = raised || far_below();
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) rare = rare || fabsf(y[t][e]) >= 32768.f;
          if (__any_sync(0xffffffffu, rare)) {
            // A row's unit follows its own largest finite weight: up where that leaves fp16, down where the
            // row's O has fallen, and no further than it fell, so that O's own numbers do not grow.
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              auto exponent = [](float w) {  // of a finite weight, else 0
                const unsigned x = __float_as_uint(w) >> 23 & 0xffu;
                return x < 255 ? x : 0u;
              };
              unsigned top = max(exponent(s[t][0]), exponent(s[t][2])) | max(exponent(s[t][1]), exponent(s[t][3])) << 16;
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, d));
              float f[2];
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const int ex = top >> 16 * x & 0xffffu, above = ex - 127 - kv[t][x];
                int to = kv[t][x];
                if (ex && above >= 15) to += above - 10;
                else if (ex && above < 0) to += max(above - 10, -fell[t][x]);
                to = max(max(-100, kv[t][x] - 120), min(120, to));
                f[x] = kv[t][x] - to < -126 ? 0.f : power_of_2(kv[t][x] - to);
                kv[t][x] = to;
              }
#pragma unroll
              for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][t][e] *= f[e & 1];
            }
            in_units();
            least = power_of_2(-kv[0][0]);
#pragma unroll
            for (int t = 0; t < NT; ++t) least = fminf(least, fminf(power_of_2(-kv[t][0]), power_of_2(-kv[t][1])));
            wide = __any_sync(0xffffffffu, far_below());
          }
        }
        // ----------------------------------------------------------------- O^T += V^T P^T
        const uint32_t vt = slot + C::TILE;
        if (!I8) {
          const int key = warp * 16 + ((lane >> 4) << 3) + (lane & 7);
          // v of keys that no row sees counts as 0, whatever is there
          uint32_t keep[2] = {~0u, ~0u};
          const bool edge = key0 < w.lo || key0 + 16 > w.hi;
          if (edge) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int k = key0 + 8 * x + 2 * c;
              keep[x] = (k >= w.lo && k < w.hi ? 0xffffu : 0u) | (k + 1 >= w.lo && k + 1 < w.hi ? 0xffff0000u : 0u);
            }
          }
#pragma unroll
          for (int dg = 0; dg < KS; ++dg) {
            uint32_t va[4];
            ldsm4t(vt + tile_off<C::ROW>(key, 2 * dg + ((lane >> 3) & 1)), va);
            if (edge) {
              va[0] &= keep[0];
              va[1] &= keep[0];
              va[2] &= keep[1];
              va[3] &= keep[1];
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              mma16816(o[dg][t], va, pb[t][0], pb[t][1]);
              mma16816(o[dg][t], va, pr[t][0], pr[t][1]);
            }
          }
        } else {
          const int key = warp * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
          auto weights = [&](const float (&z)[NT][4]) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              pb[t][0] = transpose8(pack_f16x2(z[t][0], z[t][1]));
              pb[t][1] = transpose8(pack_f16x2(z[t][2], z[t][3]));
            }
          };
          // the 16 columns are taken as their even ones, then their odd ones
          auto product = [&](auto add) {
#pragma unroll
            for (int dg = 0; dg < KS; dg += 2) {
              uint32_t vb[4];
              ldsm4t(vt + tile_off<C::ROW>(key, dg + (lane >> 4)), vb);
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const uint32_t v0 = vb[2 * x] ^ 0x80808080u, v1 = vb[2 * x + 1] ^ 0x80808080u;
                const uint32_t va[4] = {codes_f16x2<0, 2>(v0), codes_f16x2<1, 3>(v0), codes_f16x2<0, 2>(v1),
                                        codes_f16x2<1, 3>(v1)};
#pragma unroll
                for (int t = 0; t < NT; ++t) add(o[dg + x][t], va, t);
              }
            }
          };
          // Weights below 2^-10 units next to larger scales: kept back here, and taken below in units
          // of 2^-24, 2^-48, .. of the first.
          constexpr float kSmall = 0x1p-10f;
          float rest[NT][4];
          if (wide) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                rest[t][e] = fabsf(y[t][e]) < kSmall ? y[t][e] : 0.f;
                y[t][e] = rest[t][e] == 0.f ? y[t][e] : 0.f;
              }
          }
          weights(y);
          product([&](float (&d)[4], const uint32_t (&va)[4], int t) { mma16816h(d, va, pb[t][0], pb[t][1]); });
          if (wide) {
            float down = 1.f;
#pragma unroll 1
            for (int level = 1; level < 12; ++level) {
              bool left = false;
              down *= 0x1p-24f;
#pragma unroll
              for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float z = rest[t][e] * 0x1p24f;
                  left = left || z != 0.f;
                  rest[t][e] = fabsf(z) < kSmall ? z : 0.f;
                  y[t][e] = rest[t][e] == 0.f ? z : 0.f;
                }
              if (down == 0.f || !__any_sync(0xffffffffu, left)) break;
              weights(y);
              product([&](float (&d)[4], const uint32_t (&va)[4], int t) {
                float part[4] = {0.f, 0.f, 0.f, 0.f};
                mma16816h(part, va, pb[t][0], pb[t][1]);
#pragma unroll
                for (int e = 0; e < 4; ++e) d[e] = fmaf(part[e], down, d[e]);
              });
            }
          }
        }
      }
      if (b + 1 < cnt) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]);
      }
    }

    // ------------------------------------------------------------ the warps' results meet
    const int last = (g - 1) % C::STAGES;  // still held
    float* buf = reinterpret_cast<float*>(smem + last * C::SLOT);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[t][x] += __shfl_xor_sync(0xffffffffu, l[t][x], d);
        if (gr == 0) {
          ml[(warp * kBM + 8 * t + 2 * c + x) * 2] = m[t][x];
          ml[(warp * kBM + 8 * t + 2 * c + x) * 2 + 1] = l[t][x];
        }
      }
    consumer_bar();
    auto merged = [&](int r, float& mm, float& ll) {
      mm = -CUDART_INF_F;
#pragma unroll
      for (int x = 0; x < kConsumers; ++x) mm = fmaxf(mm, ml[(x * kBM + r) * 2]);
      const float base = mm == -CUDART_INF_F ? 0.f : mm;
      ll = 0.f;
#pragma unroll
      for (int x = 0; x < kConsumers; ++x) ll += ml[(x * kBM + r) * 2 + 1] * ex2_approx(ml[(x * kBM + r) * 2] - base);
    };
    float f[NT][2], dummy, em, el;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        merged(8 * t + 2 * c + x, em, dummy);
        f[t][x] = ex2_approx(m[t][x] - (em == -CUDART_INF_F ? 0.f : em));
        if (I8) f[t][x] *= power_of_2(kv[t][x]);
      }
    merged(er, em, el);
    const bool split = w.off > 0 || cnt < w.nb;
    float* part = split ? partial_slot<16, HD>(p, blockIdx.x, w.off > 0 ? 0 : 1) : nullptr;
    // columns of a row are swizzled in groups of 8 over the banks
    auto buf_at = [&](int wp, int r, int col) { return (wp * kBM + r) * C::CHUNK + (col ^ (((r >> 1) & 3) << 3)); };
    float inv = el == 0.f ? 0.f : 1.f / el;
#pragma unroll
    for (int ch = 0; ch < HD / C::CHUNK; ++ch) {
      if (ch) consumer_bar();
#pragma unroll
      for (int dg = ch * C::CHUNK / 16; dg < (ch + 1) * C::CHUNK / 16; ++dg)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 8 * t + 2 * c + (e & 1), col = dg * 16 - ch * C::CHUNK + (I8 ? 2 * gr + (e >> 1) : gr + 8 * (e >> 1));
            buf[buf_at(warp, r, col)] = o[dg][t][e] * f[t][e & 1];
          }
      consumer_bar();
      float v[C::CHUNK / (4 * C::TPR)][4];
      bool nan = false;
#pragma unroll
      for (int j = 0; j < C::CHUNK / (4 * C::TPR); ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[j][e] = 0.f;
#pragma unroll
        for (int x = 0; x < kConsumers; ++x) {
          const float4 u = *reinterpret_cast<const float4*>(buf + buf_at(x, er, 4 * (ec + C::TPR * j)));
          v[j][0] += u.x;
          v[j][1] += u.y;
          v[j][2] += u.z;
          v[j][3] += u.w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) nan = nan || isnan(v[j][e]);
      }
      if (!I8 && w.n > 1) {
        // a row may have met a NaN or an infinity of a key that only a later row sees
        if (nan && er < rows && ok) atomicOr(const_cast<unsigned*>(nan_rows), 1u << er);
        consumer_bar();
        const unsigned todo = *nan_rows;
        if (todo) {
          const int seg_lo = (w.blk0 + w.off) * kBK, seg_hi = seg_lo + cnt * kBK;
          for (int r = warp; r < kBM; r += kConsumers) {
            if (!((todo >> r) & 1u)) continue;
            float rm, rl, ro[HD / 32];
            row_attend<HD>(p, a.table + w.s * a.table_ld, w.h, q_ptr(r), max(w.row_lo(r), seg_lo),
                           min(w.row_hi(r), seg_hi), rm, rl, ro);
#pragma unroll
            for (int e = 0; e < HD / 32; ++e) buf[r * HD + lane * (HD / 32) + e] = ro[e];
            if (lane == 0) {
              fix[2 * r] = rm;
              fix[2 * r + 1] = rl;
            }
          }
          consumer_bar();
          if ((todo >> er) & 1u) {
            em = fix[2 * er];
            el = fix[2 * er + 1];
            inv = el == 0.f ? 0.f : 1.f / el;
#pragma unroll
            for (int j = 0; j < C::CHUNK / (4 * C::TPR); ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) v[j][e] = buf[er * HD + 4 * (ec + C::TPR * j) + e];
          }
          if (threadIdx.x == 0) *nan_rows = 0;
          consumer_bar();
        }
      }
#pragma unroll
      for (int j = 0; j < C::CHUNK / (4 * C::TPR); ++j) {
        const int col = ch * C::CHUNK + 4 * (ec + C::TPR * j);
        if (split) {
          if (er < rows) __stcg(reinterpret_cast<float4*>(part + er * HD + col), make_float4(v[j][0], v[j][1], v[j][2], v[j][3]));
        } else if (er < rows && ok) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[j][e] = el == 0.f ? 0.f : v[j][e] * inv;
          write_row4(er, col, v[j]);
        }
      }
    }
    fence_proxy_async_smem();  // the slot was written by threads; TMA writes it next
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[last]);
    if (ec == 0) {
      if (split) {
        __stcg(part + 16 * HD + er, em);
        __stcg(part + 16 * HD + 16 + er, el);
      } else if (er < rows && ok) {
        write_lse(er, el == 0.f ? -CUDART_INF_F : em + log2f(el));
      }
    }
    if (!split) continue;

    // -------------------------------------------- the item's CTAs: the last one joins them
    const int64_t first_block = w.g - w.off;
    const int cta0 = block_owner(first_block, total, P), cta1 = block_owner(first_block + w.nb - 1, total, P);
    int* counter = static_cast<int*>(a.workspace) + cta0;
    __threadfence();
    consumer_bar();
    if (threadIdx.x == 0) *is_last = atomicAdd(counter, 1) == cta1 - cta0;
    consumer_bar();
    if (!*is_last) continue;
    __threadfence();
    auto slot_of = [&](int cta) { return partial_slot<16, HD>(p, cta, cta == cta0 ? 1 : 0); };
    constexpr int kCols = HD / (4 * C::TPR);
    float jm = -CUDART_INF_F, jl = 0.f, v[kCols][4];
    const int parts_end = er < rows ? cta1 : cta0 - 1;
    for (int x = cta0; x <= parts_end; ++x) jm = fmaxf(jm, __ldcg(slot_of(x) + 16 * HD + er));
    const float base = jm == -CUDART_INF_F ? 0.f : jm;
#pragma unroll
    for (int j = 0; j < kCols; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j][e] = 0.f;
    for (int x = cta0; x <= parts_end; ++x) {
      const float* src = slot_of(x);
      const float wt = ex2_approx(__ldcg(src + 16 * HD + er) - base);
      jl += wt * __ldcg(src + 16 * HD + 16 + er);
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        const float4 u = __ldcg(reinterpret_cast<const float4*>(src + er * HD + 4 * (ec + C::TPR * j)));
        v[j][0] += wt * u.x;
        v[j][1] += wt * u.y;
        v[j][2] += wt * u.z;
        v[j][3] += wt * u.w;
      }
    }
    if (er < rows && ok) {
      const float jinv = jl == 0.f ? 0.f : 1.f / jl;
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[j][e] = jl == 0.f ? 0.f : v[j][e] * jinv;
        write_row4(er, 4 * (ec + C::TPR * j), v[j]);
      }
      if (ec == 0) write_lse(er, jl == 0.f ? -CUDART_INF_F : jm + log2f(jl));
    }
    if (threadIdx.x == 0) *counter = 0;
    consumer_bar();  // is_last is read before it is written again
  }
  if (!ok && threadIdx.x == 0) set_error(a.err, kDevTimeoutEpilogue);
}

int few_ctas(int per_sm) {
  const int c = per_sm * num_sms();
  return c < kMaxCtas ? c : kMaxCtas;
}

template <int HD, bool I8, int NT>
int launch(const Params& p, cudaStream_t s) {
  using C = Cfg<HD, I8, NT>;
  CUtensorMap tk, tv;
  const uint64_t rows = static_cast<uint64_t>(p.a.cache.num_pages) * p.a.cache.kv_heads * p.a.cache.page_size;
  const uint32_t box = p.a.cache.page_size < kBK ? p.a.cache.page_size : kBK;
  if (!make_tmap_rows(&tk, p.a.cache.k, C::ROW, rows, C::BOX, box) ||
      !make_tmap_rows(&tv, p.a.cache.v, C::ROW, rows, C::BOX, box))
    return -3;
  const void* fn = reinterpret_cast<const void*>(attn_paged_few_kernel<HD, I8, NT>);
  const cudaError_t attr = smem_limit_once(fn, C::BYTES);
  if (attr != cudaSuccess) return attr;
  // no more CTAs than the bounds allow blocks (a sequence without keys costs one)
  const int64_t tiles = (static_cast<int64_t>(p.a.max_q < 1 ? 1 : p.a.max_q) * p.G + C::BM - 1) / C::BM;
  const int64_t keys = p.a.max_kv < 1 ? 1 : p.a.max_kv;
  const int64_t most = p.a.nseq * static_cast<int64_t>(p.a.cache.kv_heads) * tiles * ((keys + kBK - 1) / kBK);
  const int64_t ctas = few_ctas(C::CTAS);
  attn_paged_few_kernel<HD, I8, NT><<<static_cast<unsigned>(most < ctas ? most : ctas), kThreads, C::BYTES, s>>>(tk, tv, p);
  return cudaGetLastError();
}

template <int NT>
int launch_nt(const Params& p, cudaStream_t s) {
  if (p.a.cache.hd == 128) return p.a.cache.int8 ? launch<128, true, NT>(p, s) : launch<128, false, NT>(p, s);
  return p.a.cache.int8 ? launch<64, true, NT>(p, s) : launch<64, false, NT>(p, s);
}

}  // namespace
}  // namespace paged

int attn_paged_few(const paged::Params& p, cudaStream_t s) {
  return p.bm == 8 ? paged::launch_nt<1>(p, s) : paged::launch_nt<2>(p, s);
}

int64_t attn_paged_workspace_bytes(int hd) {
  const int64_t few = int64_t(paged::kMaxCtas) * 16, many = attn_paged_many_ctas() * 256;
  return paged::kCounterBytes + (few > many ? few : many) * 2 * (hd + 2) * 4;
}

int attn_paged(const PagedAttnArgs& a, cudaStream_t s) {
  if (!kv_pages_ok(a.cache) || a.nseq < 0 || a.T < 0 || a.heads <= 0 || a.heads % a.cache.kv_heads) return -1;
  const int64_t cols = static_cast<int64_t>(a.heads) * a.cache.hd;
  if (a.ldq % 8 || a.ldo % 8 || a.ldq < cols || a.ldo < cols || a.table_ld < 0 || a.table_cols < 0 || a.window < 0) return -1;
  if (!(a.scale > 0.f)) return -1;
  if ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.workspace)) & 15)
    return -1;
  if (a.workspace_bytes < attn_paged_workspace_bytes(a.cache.hd)) return -1;
  if (static_cast<int64_t>(a.T) * a.heads >= int64_t(1) << 31) return -1;  // rows are counted in 32 bits
  if (a.T == 0 || a.nseq == 0) return 0;
  paged::Params p;
  p.a = a;
  p.G = a.heads / a.cache.kv_heads;
  p.page_shift = 31 - __builtin_clz(a.cache.page_size);
  const int64_t most_pages = (1 << 30) / a.cache.page_size;
  p.max_len = static_cast<int>((a.table_cols < most_pages ? a.table_cols : most_pages) * a.cache.page_size);
  if (a.window >= p.max_len) p.a.window = 0;  // of no length: and differences with it stay in 32 bits
  p.scale_log2 = a.scale * 1.4426950408889634f;
  // Up to 8 or 16 rows per key head and sequence fill one tile of the kernel above; more rows share
  // each block's keys in tiles of up to 2 x 128 on the tcgen05 tensor cores.  Both kernels, us (few / many), 8
  // sequences of 8 heads, hd 128 in bf16: 16 rows over 256 keys 12.5 / 15.7, over 2048 28 / 34, over 16384 96 /
  // 175; 32 rows 12.6 / 15.7, 34 / 35, 171 / 176; 64 rows 12.5 / 16.6, 49 / 36, 324 / 200.  int8: 16 rows 14 / 21,
  // 28 / 50, 86 / 223; 64 rows 15 / 23, 51 / 52, 283 / 226.  hd 64: 16 rows 11 / 15, 18 / 26, 57 / 85; 24 rows 11 / 15, 22 /
  // 27, 94 / 86.  So 16 is the last count at which the few-row kernel is ahead everywhere; up to 32 it is within
  // 10%, and ahead over int8 and short caches.
  if (static_cast<int64_t>(a.max_q) * p.G <= 16 || p.G > 128) {
    p.bm = static_cast<int64_t>(a.max_q) * p.G <= 8 ? 8 : 16;
    p.tile_tokens = p.bm % p.G ? 0 : p.bm / p.G;
    return attn_paged_few(p, s);
  }
  p.bm = 2 * (128 / p.G * p.G);  // two halves of whole tokens, so that a half of q is one TMA box
  p.tile_tokens = p.bm / p.G;
  return attn_paged_many(p, s);
}

}  // namespace rt
