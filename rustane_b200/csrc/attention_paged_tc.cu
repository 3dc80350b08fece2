// Attention over the paged cache for many rows per key head (prompts in chunks, several
// new tokens at once): tiles of up to 128 rows on tcgen05 / TMEM.  Semantics, the split of
// the work and the join as in attention_paged.cu; the products and the softmax are built
// like the training forward's (attention_tc.cu).
//
// Compute-bound on the 4 hd flop per row and visible key; in practice the softmax's issue
// slots bound it before the tensor pipe.  One persistent CTA per SM:
//   warp 0      TMA producer: Q of each item (one box: whole tokens x the G heads of the key
//               head), then the pages of 128-key blocks of K and V, two blocks deep;
//   warp 1      MMA issuer: S_j = Q K_j^T into one of two TMEM buffers, O += P_j V_j with P as
//               the TMEM operand; S_{j+1} goes before O += P_j V_j.  It also zeroes the
//               v rows of a bf16 edge block that no row of the tile sees;
//   warp 2      owns the TMEM allocation;
//   warps 4-11  softmax, two threads per row (half the keys each), P over S in TMEM, O
//               rescaled only when the running maximum grew by more than 2^8;
//   warps 12-15 (int8 cache) turn the codes into bf16 tiles, exactly, one key a thread;
//               k's scale multiplies the scores and v's the weights, in fp32.
// P is rounded to bf16 for the P V product (its sum is not).  All waits are bounded.
#include "attention_paged.cuh"
#include "kernels.h"

namespace rt {
namespace paged {
namespace {

constexpr int kBM = 128;
constexpr int kBK = 128;
constexpr int kAtomBytes = kBM * 128;  // 64 bf16 columns of 128 rows
constexpr int kStages8 = 3;            // int8 tiles (k or v) in flight
constexpr int kScaleSlots = 4;         // blocks whose scales are held

enum Bar : int {
  kQFull = 0,
  kQEmpty = 1,   // every S MMA of the item done
  kKFull = 2,    // [2]
  kKEmpty = 4,   // [2]
  kVFull = 6,    // [2]
  kVEmpty = 8,   // [2]
  kSFull = 10,   // [2]
  kSFree = 12,   // [2]
  kPFull = 14,   // [2] by S buffer: the softmax may finish block g + 1 before P of block g is waited for
  kPvDone = 16,  // [2]
  kOFree = 18,   // [2]
  kDrain = 20,
  kCodeFull = 21,                           // [kStages8]
  kCodeEmpty = kCodeFull + kStages8,        // [kStages8]
  kScaleFull = kCodeEmpty + kStages8,       // [kScaleSlots]
  kScaleEmpty = kScaleFull + kScaleSlots,   // [kScaleSlots]
  kNumBars = kScaleEmpty + kScaleSlots
};

template <int HD, bool I8>
struct Cfg {
  static constexpr int ATOMS = HD / 64;
  static constexpr int TILE = ATOMS * kAtomBytes;  // Q, K or V in bf16
  static constexpr int ROW8 = HD;                  // bytes of an int8 key
  static constexpr int CODES = kBK * ROW8;
  static constexpr int Q = 0;
  static constexpr int K = Q + TILE;      // [2]
  static constexpr int V = K + 2 * TILE;  // [2]
  static constexpr int CODE = V + 2 * TILE;
  static constexpr int SCALE = CODE + (I8 ? kStages8 * CODES : 0);              // [slot][k, v][128]
  static constexpr int RED = SCALE + (I8 ? kScaleSlots * 2 * kBK * 4 : 0);      // float [2][2 halves][128]: row max
  static constexpr int SUM = RED + 2 * 2 * kBM * 4;                             // float [2 halves][128]
  static constexpr int NANS = SUM + 2 * kBM * 4;                                // unsigned [4 quadrants][2 halves]
  static constexpr int BAR = NANS + 64;
  static constexpr int BYTES = BAR + 512 + 1024;
  static constexpr int THREADS = I8 ? 512 : 384;
};
static_assert(kNumBars * 8 + 16 <= 512, "barrier area");

__device__ __forceinline__ void softmax_bar() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ void row_pair_bar(int qw) { asm volatile("bar.sync %0, 64;" ::"r"(2 + qw) : "memory"); }

template <int HD, bool I8>
__global__ void __launch_bounds__(Cfg<HD, I8>::THREADS, 1)
    attn_paged_many_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                           const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Params p, int min_blocks) {
  using C = Cfg<HD, I8>;
  constexpr int HC = HD / 2;  // output columns per softmax thread
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + C::BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* is_last = abort_flag + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PagedAttnArgs& a = p.a;

  if (threadIdx.x == 0) {
    mbar_init(&bar[kQFull], 1);
    mbar_init(&bar[kQEmpty], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar[kKFull + i], I8 ? 4 : 1);
      mbar_init(&bar[kKEmpty + i], 1);
      mbar_init(&bar[kVFull + i], I8 ? 4 : 1);
      mbar_init(&bar[kVEmpty + i], 1);
      mbar_init(&bar[kSFull + i], 1);
      mbar_init(&bar[kSFree + i], 1);
      mbar_init(&bar[kPvDone + i], 1);
      mbar_init(&bar[kOFree + i], 8);
      mbar_init(&bar[kPFull + i], 8);
    }
    mbar_init(&bar[kDrain], 1);
    for (int i = 0; i < kStages8; ++i) {
      mbar_init(&bar[kCodeFull + i], 1);
      mbar_init(&bar[kCodeEmpty + i], 4);
    }
    for (int i = 0; i < kScaleSlots; ++i) {
      mbar_init(&bar[kScaleFull + i], 1);
      mbar_init(&bar[kScaleEmpty + i], 8);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 2) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  int64_t total;
  int P;
  Walk<kBK> w = start_walk<kBK, C::THREADS>(p, min_blocks, total, P);  // its barriers cover the set-up above
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;  // columns [0,128) S0, [128,256) S1, then O0, O1 of 128 each

  if (warp == 0) {
    // ----------------------------------------------------------------- producer
    // lane i < boxes of a block loads `ps` keys, one page
    if (lane == 0) {
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
    const int ps = 1 << p.page_shift;
    int g = 0, it = 0;
    int q_issued = 0, k_issued = 0, v_issued = 0, s_issued = 0;  // k_issued of an int8 cache: k and v tiles
    bool ok = true;
    auto wait = [&](uint64_t* b, uint32_t parity) {
      return __all_sync(0xffffffffu, mbar_wait(b, parity) && !*abort_flag);
    };
    for (; ok && w.more(); w.next()) {
      if (w.empty()) continue;
      const int32_t* table = a.table + w.s * a.table_ld;
      const int cnt = w.count();
      const int key00 = (w.blk0 + w.off) * kBK;
      auto my_page = [&](int b) {
        const int key = key00 + b * kBK + lane * ps;
        return b < cnt && lane * ps < kBK && key < w.hi && key + ps > w.lo ? page_of(p, table, key) : -1;
      };
      int page = my_page(0);
      if (it > 0 && !wait(&bar[kQEmpty], (it - 1) & 1)) {
        ok = false;
        break;
      }
      if (lane == 0) {
        mbar_arrive_expect_tx(&bar[kQFull], C::ATOMS * p.bm * 128);
#pragma unroll
        for (int x = 0; x < C::ATOMS; ++x)
          tma_load_3d(smem + C::Q + x * kAtomBytes, &tm_q, &bar[kQFull], x * 64, w.h * p.G, w.q0 + w.t * p.bm / p.G);
      }
      q_issued = ++it;
      for (int b = 0; b < cnt; ++b, ++g) {
        const int ahead = my_page(b + 1);
        const int loads = __popc(__ballot_sync(0xffffffffu, page >= 0));
        const int64_t row64 = ((static_cast<int64_t>(page < 0 ? 0 : page) * a.cache.kv_heads + w.h) << p.page_shift);
        const int row = static_cast<int>(row64);
        const int st = g & 1;
        const uint32_t ph = (g >> 1) & 1;
        if (I8) {
          const int sl = g % kScaleSlots;
          if (!wait(&bar[kScaleEmpty + sl], ((g / kScaleSlots) & 1) ^ 1)) {
            ok = false;
            break;
          }
          if (lane == 0) mbar_arrive_expect_tx(&bar[kScaleFull + sl], loads * ps * 8);
          __syncwarp();
          if (page >= 0) {
            uint8_t* sc = smem + C::SCALE + sl * (2 * kBK * 4) + lane * ps * 4;
            bulk_load(sc, a.cache.k_scale + row64, ps * 4, &bar[kScaleFull + sl]);
            bulk_load(sc + kBK * 4, a.cache.v_scale + row64, ps * 4, &bar[kScaleFull + sl]);
          }
          s_issued = g + 1;
          __syncwarp();
        }
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const CUtensorMap* tm = kv ? &tm_v : &tm_k;
          if (I8) {
            const int x = 2 * g + kv, cs = x % kStages8;
            if (!wait(&bar[kCodeEmpty + cs], ((x / kStages8) & 1) ^ 1)) {
              ok = false;
              break;
            }
            if (lane == 0) mbar_arrive_expect_tx(&bar[kCodeFull + cs], loads * ps * C::ROW8);
            __syncwarp();
            if (page >= 0)
              tma_load_2d(smem + C::CODE + cs * C::CODES + lane * ps * C::ROW8, tm, &bar[kCodeFull + cs], 0, row);
            k_issued = x + 1;
          } else {
            const int full = (kv ? kVFull : kKFull) + st, empty = (kv ? kVEmpty : kKEmpty) + st;
            if (!wait(&bar[empty], ph ^ 1)) {
              ok = false;
              break;
            }
            if (lane == 0) mbar_arrive_expect_tx(&bar[full], loads * ps * C::ATOMS * 128);
            __syncwarp();
            if (page >= 0) {
              uint8_t* dst = smem + (kv ? C::V : C::K) + st * C::TILE + lane * ps * 128;
#pragma unroll
              for (int x = 0; x < C::ATOMS; ++x) tma_load_2d(dst + x * kAtomBytes, tm, &bar[full], x * 128, row);
            }
            (kv ? v_issued : k_issued) = g + 1;
          }
          __syncwarp();
        }
        if (!ok) break;
        page = ahead;
      }
    }
    if (!ok) {  // let copies still in flight land before the CTA exits
      if (lane == 0) set_error(a.err, kDevTimeoutProducer);
      *abort_flag = 1;
      if (q_issued > 0) mbar_wait(&bar[kQFull], (q_issued - 1) & 1);
      if (I8) {
        for (int x = k_issued > kStages8 ? k_issued - kStages8 : 0; x < k_issued; ++x)
          mbar_wait(&bar[kCodeFull + x % kStages8], (x / kStages8) & 1);
        for (int x = s_issued > kScaleSlots ? s_issued - kScaleSlots : 0; x < s_issued; ++x)
          mbar_wait(&bar[kScaleFull + x % kScaleSlots], (x / kScaleSlots) & 1);
      } else {
        for (int x = k_issued > 2 ? k_issued - 2 : 0; x < k_issued; ++x) mbar_wait(&bar[kKFull + (x & 1)], (x >> 1) & 1);
        for (int x = v_issued > 2 ? v_issued - 2 : 0; x < v_issued; ++x) mbar_wait(&bar[kVFull + (x & 1)], (x >> 1) & 1);
      }
    }
  } else if (warp == 1) {
    // -------------------------------------------------------------- MMA issuer
    constexpr uint32_t idesc_s = idesc_bf16_f32(kBM, kBK, false, false);  // Q, K: both hd-contiguous
    constexpr uint32_t idesc_o = idesc_bf16_f32(kBM, HD, false, true);    // P key-contiguous, V hd-contiguous
    const uint32_t sq = smem_u32(smem + C::Q);
    auto wait = [&](uint64_t* b, uint32_t parity) {
      return __all_sync(0xffffffffu, mbar_wait(b, parity) && !*abort_flag);
    };
    auto issue_s = [&](int gg) -> bool {
      const int st = gg & 1;
      const uint32_t ph = (gg >> 1) & 1;
      if (!wait(&bar[kKFull + st], ph) || !wait(&bar[kSFree + st], ph ^ 1)) return false;
      tc_fence_after();
      if (lane == 0) {
        const uint32_t sk = smem_u32(smem + C::K + st * C::TILE);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint32_t off = (kk >> 2) * kAtomBytes + (kk & 3) * 32;
          umma_bf16(tmem + st * kBK, smem_desc_sw128(sq + off, 16, 1024), smem_desc_sw128(sk + off, 16, 1024), idesc_s,
                    kk != 0 ? 1u : 0u);
        }
        umma_commit(&bar[kKEmpty + st]);
        umma_commit(&bar[kSFull + st]);
      }
      __syncwarp();
      return true;
    };
    bool ok = true;
    int g = 0, it = 0;
    for (; ok && w.more(); w.next()) {
      if (w.empty()) continue;
      const int cnt = w.count();
      const int ob = it & 1;
      if (!wait(&bar[kQFull], it & 1) || !issue_s(g)) {
        ok = false;
        break;
      }
      for (int b = 0; b < cnt; ++b, ++g) {
        if (b + 1 < cnt) {
          if (!issue_s(g + 1)) {
            ok = false;
            break;
          }
        } else if (lane == 0) {
          umma_commit(&bar[kQEmpty]);
        }
        const int st = g & 1;
        if (!wait(&bar[kVFull + st], (g >> 1) & 1)) {
          ok = false;
          break;
        }
        uint8_t* vt = smem + C::V + st * C::TILE;
        const int key0 = (w.blk0 + w.off + b) * kBK;
        if (!I8 && (key0 < w.lo || key0 + kBK > w.hi)) {
          // keys that no row of the tile sees weigh 0, but what is there may be NaN
          const int first = max(0, w.lo - key0), last = min(kBK, w.hi - key0);
#pragma unroll
          for (int x = 0; x < C::ATOMS; ++x) {
            uint4* rows = reinterpret_cast<uint4*>(vt + x * kAtomBytes);
            for (int i = lane; i < first * 8; i += 32) rows[i] = make_uint4(0, 0, 0, 0);
            for (int i = last * 8 + lane; i < kBK * 8; i += 32) rows[i] = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (!wait(&bar[kPFull + st], (g >> 1) & 1) || (b == 0 && it >= 2 && !wait(&bar[kOFree + ob], ((it >> 1) - 1) & 1))) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (lane == 0) {
          const uint32_t sv = smem_u32(vt);
#pragma unroll
          for (int kk = 0; kk < kBK / 16; ++kk) {
            const uint32_t acol = st * kBK + (kk < 4 ? kk * 8 : 64 + (kk - 4) * 8);
            umma_bf16_ts(tmem + (2 + ob) * 128, tmem + acol, smem_desc_sw128(sv + kk * 2048, kAtomBytes, 1024), idesc_o,
                         (b | kk) != 0 ? 1u : 0u);
          }
          umma_commit(&bar[kVEmpty + st]);
          umma_commit(&bar[kPvDone + st]);
          umma_commit(&bar[kSFree + st]);
        }
        __syncwarp();
      }
      ++it;
    }
    if (!ok) {
      if (lane == 0) set_error(a.err, kDevTimeoutMma);
      *abort_flag = 1;
    }
    if (lane == 0) {
      umma_commit(&bar[kDrain]);
      mbar_wait(&bar[kDrain], 0);
    }
    __syncwarp();
  } else if (I8 && warp >= 12) {
    // ------------------------------------------------------------ int8 -> bf16
    const int r = threadIdx.x - 384;  // key of the block
    int x = 0;
    bool ok = true;
    for (; ok && w.more(); w.next()) {
      if (w.empty()) continue;
      const int cnt = w.count();
      for (int b = 0; ok && b < 2 * cnt; ++b, ++x) {
        const int g = x >> 1, st = g & 1, cs = x % kStages8;
        const bool v = x & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&bar[kCodeFull + cs], (x / kStages8) & 1) &&
                                         mbar_wait(&bar[(v ? kVEmpty : kKEmpty) + st], ((g >> 1) & 1) ^ 1) && !*abort_flag);
        if (!ok) break;
        const uint8_t* src = smem + C::CODE + cs * C::CODES + r * C::ROW8;
        uint8_t* dst = smem + (v ? C::V : C::K) + st * C::TILE + r * 128;
#pragma unroll
        for (int ch = 0; ch < HD / 16; ++ch) {
          const int sw = HD == 64 ? ch ^ ((r >> 1) & 3) : ch ^ (r & 7);
          const uint4 u = *reinterpret_cast<const uint4*>(src + sw * 16);
          uint8_t* d = dst + (ch >> 2) * kAtomBytes;
          const int c0 = (ch & 3) * 2;
          *reinterpret_cast<uint4*>(d + ((c0 ^ (r & 7)) << 4)) =
              make_uint4(i8x2_bf16x2<0, 1>(u.x), i8x2_bf16x2<2, 3>(u.x), i8x2_bf16x2<0, 1>(u.y), i8x2_bf16x2<2, 3>(u.y));
          *reinterpret_cast<uint4*>(d + (((c0 + 1) ^ (r & 7)) << 4)) =
              make_uint4(i8x2_bf16x2<0, 1>(u.z), i8x2_bf16x2<2, 3>(u.z), i8x2_bf16x2<0, 1>(u.w), i8x2_bf16x2<2, 3>(u.w));
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bar[kCodeEmpty + cs]);
          mbar_arrive(&bar[(v ? kVFull : kKFull) + st]);
        }
      }
    }
    if (!ok) {
      if (lane == 0) set_error(a.err, kDevTimeoutEpilogue);
      *abort_flag = 1;
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ softmax
    const int qw = warp & 3;               // TMEM lane quadrant
    const int hh = (warp - 4) >> 2;        // key columns [64 hh, 64 hh + 64) of the block
    const int r = qw * 32 + lane;          // row of the tile
    const uint32_t lane_off = static_cast<uint32_t>(qw * 32) << 16;
    float* red = reinterpret_cast<float*>(smem + C::RED);
    float* sum = reinterpret_cast<float*>(smem + C::SUM);
    volatile unsigned* nans = reinterpret_cast<volatile unsigned*>(smem + C::NANS);
    // A failed (timed-out) wait does not leave the loops: every softmax warp must reach the same
    // sequence of named barriers.  After the first failure every later wait returns at once.
    const float raise = kRescale / p.scale_log2;
    bool ok = true;
    auto wait = [&](uint64_t* bb, uint32_t parity) {
      bool good = !*abort_flag && mbar_wait(bb, parity);
      good = __all_sync(0xffffffffu, good);
      if (!good) {
        ok = false;
        *abort_flag = 1;
      }
    };
    int g = 0, it = 0;
    for (; w.more(); w.next()) {
      const int rows = w.rows(), cnt = w.count();
      const int rr = min(r, rows - 1);
      const int flat = w.t * p.bm + rr;
      const int64_t tok = w.q0 + flat / p.G;
      const int head = w.h * p.G + flat % p.G;
      __nv_bfloat16* orow = a.out + tok * a.ldo + head * HD + hh * HC;
      float* lse = a.lse2 ? a.lse2 + tok * a.heads + head : nullptr;
      if (w.empty()) {
        if (r < rows) {
#pragma unroll
          for (int i = 0; i < HC / 8; ++i) reinterpret_cast<uint4*>(orow)[i] = make_uint4(0, 0, 0, 0);
          if (lse && hh == 0) *lse = -CUDART_INF_F;
        }
        continue;
      }
      const int ob = it & 1;
      const uint32_t to = tmem + (2 + ob) * 128 + lane_off + hh * HC;  // this thread's O columns
      const int hi_r = w.row_hi(rr), lo_r = w.row_lo(rr);
      const int lo_all = w.row_lo(rows - 1), hi_all = w.row_hi(0);  // keys that every row sees
      float m_used = -CUDART_INF_F, l = 0.f;  // m_used: of the unscaled scores
      for (int b = 0; b < cnt; ++b, ++g) {
        const int st = g & 1;
        const int key0 = (w.blk0 + w.off + b) * kBK;
        const bool masked = key0 < lo_all || key0 + kBK > hi_all;
        wait(&bar[kSFull + st], (g >> 1) & 1);
        tc_fence_after();
        const uint32_t ts = tmem + st * kBK + lane_off + hh * 64;
        uint32_t v[64];
        tmem_ld32(ts, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
        tmem_ld32(ts + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
        const float* scales = reinterpret_cast<const float*>(smem + C::SCALE + (g % kScaleSlots) * (2 * kBK * 4)) + hh * 64;
        if (I8) wait(&bar[kScaleFull + g % kScaleSlots], (g / kScaleSlots) & 1);
        tmem_ld_wait();
        if (I8) {
#pragma unroll
          for (int e = 0; e < 64; e += 4) {
            const float4 k4 = *reinterpret_cast<const float4*>(scales + e);
            float x0, x1, x2, x3;
            f2_unpack(f2_mul(f2_pack(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), f2_pack(k4.x, k4.y)), x0, x1);
            f2_unpack(f2_mul(f2_pack(__uint_as_float(v[e + 2]), __uint_as_float(v[e + 3])), f2_pack(k4.z, k4.w)), x2, x3);
            v[e] = __float_as_uint(x0);
            v[e + 1] = __float_as_uint(x1);
            v[e + 2] = __float_as_uint(x2);
            v[e + 3] = __float_as_uint(x3);
          }
        }
        if (masked) {
          const int last = hi_r - key0 - hh * 64, first = lo_r - key0 - hh * 64;  // seen: first <= e < last
#pragma unroll
          for (int e = 0; e < 64; ++e)
            if (e >= last || e < first) v[e] = __float_as_uint(-CUDART_INF_F);
        }
        float mc[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t* u = v + 16 * q;
          mc[q] = fmax3(__uint_as_float(u[0]), __uint_as_float(u[1]), __uint_as_float(u[2]));
#pragma unroll
          for (int e = 3; e < 15; e += 2) mc[q] = fmax3(mc[q], __uint_as_float(u[e]), __uint_as_float(u[e + 1]));
          mc[q] = fmaxf(mc[q], __uint_as_float(u[15]));
        }
        float mx = fmax3(mc[0], mc[1], fmaxf(mc[2], mc[3]));
        red[(st * 2 + hh) * kBM + r] = mx;
        row_pair_bar(qw);
        mx = fmaxf(red[(st * 2) * kBM + r], red[(st * 2 + 1) * kBM + r]);
        const float m_new = fmaxf(m_used, mx);
        if (b == 0) {
          m_used = m_new;
        } else if (__any_sync(0xffffffffu, m_new > m_used + raise)) {
          wait(&bar[kPvDone + ((g - 1) & 1)], ((g - 1) >> 1) & 1);
          tc_fence_after();
          const bool grow = m_new > m_used + raise;
          const float f = grow ? exp2f((m_used - m_new) * p.scale_log2) : 1.f;
          if (grow) {
            l *= f;
            m_used = m_new;
          }
#pragma unroll 1
          for (int cc = 0; cc < HC / 32; ++cc) {
            uint32_t o[32];
            tmem_ld32(to + cc * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st32(to + cc * 32, o);
          }
          tmem_st_wait();
        }
        // a maximum of -inf (the row has seen nothing yet) is taken as 0: its weights come out 0
        const float ms = m_used == -CUDART_INF_F ? 0.f : m_used;
        // the difference first: a fused scale * s - m would leave m's rounding, which is everything
        // where scores are near the lowest value of the type
        const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2), ms2 = f2_pack(ms, ms);
        uint64_t ls2[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          uint32_t pk[16];
#pragma unroll
          for (int tt = 0; tt < 16; ++tt) {
            const int e = cc * 32 + 2 * tt;
            float x0, x1;
            f2_unpack(f2_mul(f2_sub(f2_pack(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), ms2), sc2), x0, x1);
            float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
            ls2[cc] = f2_add(ls2[cc], f2_pack(p0, p1));
            if (I8) {
              const float2 vs = *reinterpret_cast<const float2*>(scales + kBK + e);
              f2_unpack(f2_mul(f2_pack(p0, p1), f2_pack(vs.x, vs.y)), p0, p1);
              if (masked) {  // 0 whatever the scale of an unseen key is
                if (v[e] == 0xff800000u) p0 = 0.f;
                if (v[e + 1] == 0xff800000u) p1 = 0.f;
              }
            }
            pk[tt] = pack_bf16x2(p0, p1);
          }
          tmem_st16(ts + cc * 16, pk);
        }
        {
          float a0, a1, b0, b1;
          f2_unpack(ls2[0], a0, a1);
          f2_unpack(ls2[1], b0, b1);
          l += (a0 + a1) + (b0 + b1);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bar[kPFull + st]);
          if (I8) mbar_arrive(&bar[kScaleEmpty + g % kScaleSlots]);
        }
      }
      // ------------------------------------------------------------- end of the item (or part)
      wait(&bar[kPvDone + ((g - 1) & 1)], ((g - 1) >> 1) & 1);
      tc_fence_after();
      sum[hh * kBM + r] = l;
      const bool split = w.off > 0 || cnt < w.nb;
      const bool may_nan = !I8 && w.n > 1;
      if (may_nan) {
        // a row may have met a NaN or an infinity of a key that only a later row sees
        bool nan = false;
#pragma unroll 1
        for (int cc = 0; cc < HC / 32; ++cc) {
          uint32_t o[32];
          tmem_ld32(to + cc * 32, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) nan = nan || isnan(__uint_as_float(o[e]));
        }
        const unsigned word = __ballot_sync(0xffffffffu, nan && r < rows && ok);
        if (lane == 0) nans[qw * 2 + hh] = word;
      }
      row_pair_bar(qw);
      l = sum[r] + sum[kBM + r];
      const unsigned todo = may_nan ? nans[qw * 2] | nans[qw * 2 + 1] : 0u;
      float* part = split ? partial_slot<kBM, HD>(p, blockIdx.x, w.off > 0 ? 0 : 1) : nullptr;
      const float inv = l == 0.f ? 0.f : 1.f / l, m_log2 = m_used * p.scale_log2;
      const bool mine = r < rows && !((todo >> lane) & 1u);
#pragma unroll 1
      for (int cc = 0; cc < HC / 32; ++cc) {
        uint32_t o[32];
        tmem_ld32(to + cc * 32, o);
        tmem_ld_wait();
        if (mine && split) {
          float4* dst = reinterpret_cast<float4*>(part + r * HD + hh * HC + cc * 32);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            __stcg(dst + e, make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]),
                                        __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3])));
        } else if (mine && ok) {
          float f[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) f[e] = l == 0.f ? 0.f : __uint_as_float(o[e]) * inv;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            reinterpret_cast<uint4*>(orow + cc * 32)[e] =
                make_uint4(pack_bf16x2(f[8 * e], f[8 * e + 1]), pack_bf16x2(f[8 * e + 2], f[8 * e + 3]),
                           pack_bf16x2(f[8 * e + 4], f[8 * e + 5]), pack_bf16x2(f[8 * e + 6], f[8 * e + 7]));
        }
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar[kOFree + ob]);  // this O buffer can take the item after next
      if (mine && hh == 0) {
        if (split) {
          __stcg(part + kBM * HD + r, m_log2);
          __stcg(part + kBM * HD + kBM + r, l);
        } else if (lse && ok) {
          *lse = l == 0.f ? -CUDART_INF_F : m_log2 + log2f(l);
        }
      }
      if (todo) {  // the quadrant's two warps share its rows
        const int seg_lo = (w.blk0 + w.off) * kBK, seg_hi = seg_lo + cnt * kBK;
        int nth = 0;
        for (int x = 0; x < 32; ++x) {
          if (!((todo >> x) & 1u) || (nth++ & 1) != hh) continue;
          const int row = qw * 32 + x, fl = w.t * p.bm + row;
          const int64_t tk = w.q0 + fl / p.G;
          const int hd = w.h * p.G + fl % p.G;
          float rm, rl, ro[HD / 32];
          row_attend<HD>(p, a.table + w.s * a.table_ld, w.h, a.q + tk * a.ldq + hd * HD, max(w.row_lo(row), seg_lo),
                         min(w.row_hi(row), seg_hi), rm, rl, ro);
          const float rinv = rl == 0.f ? 0.f : 1.f / rl;
#pragma unroll
          for (int e = 0; e < HD / 32; ++e) {
            const int col = lane * (HD / 32) + e;
            if (split) __stcg(part + row * HD + col, ro[e]);
            else a.out[tk * a.ldo + hd * HD + col] = __float2bfloat16(rl == 0.f ? 0.f : ro[e] * rinv);
          }
          if (lane == 0) {
            if (split) {
              __stcg(part + kBM * HD + row, rm);
              __stcg(part + kBM * HD + kBM + row, rl);
            } else if (a.lse2) {
              a.lse2[tk * a.heads + hd] = rl == 0.f ? -CUDART_INF_F : rm + log2f(rl);
            }
          }
        }
      }
      ++it;
      row_pair_bar(qw);  // sum and nans are read before the next item writes them
      if (!split) continue;

      // ------------------------------------------ the item's CTAs: the last one joins them
      const int64_t first_block = w.g - w.off;
      const int cta0 = block_owner(first_block, total, P), cta1 = block_owner(first_block + w.nb - 1, total, P);
      int* counter = static_cast<int*>(a.workspace) + cta0;
      __threadfence();
      softmax_bar();
      if (threadIdx.x == 128) *is_last = atomicAdd(counter, 1) == cta1 - cta0;
      softmax_bar();
      if (*is_last) {
        __threadfence();
        if (r < rows && ok) {
          auto slot_of = [&](int cta) { return partial_slot<kBM, HD>(p, cta, cta == cta0 ? 1 : 0); };
          float jm = -CUDART_INF_F, jl = 0.f;
          for (int x = cta0; x <= cta1; ++x) jm = fmaxf(jm, __ldcg(slot_of(x) + kBM * HD + r));
          const float base = jm == -CUDART_INF_F ? 0.f : jm;
          for (int x = cta0; x <= cta1; ++x)
            jl += exp2f(__ldcg(slot_of(x) + kBM * HD + r) - base) * __ldcg(slot_of(x) + kBM * HD + kBM + r);
          const float jinv = jl == 0.f ? 0.f : 1.f / jl;
#pragma unroll 1
          for (int cc = 0; cc < HC / 32; ++cc) {
            float f[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) f[e] = 0.f;
            for (int x = cta0; x <= cta1; ++x) {
              const float* src = slot_of(x);
              const float wt = exp2f(__ldcg(src + kBM * HD + r) - base);
              const float4* s4 = reinterpret_cast<const float4*>(src + r * HD + hh * HC + cc * 32);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float4 u = __ldcg(s4 + e);
                f[4 * e] += wt * u.x;
                f[4 * e + 1] += wt * u.y;
                f[4 * e + 2] += wt * u.z;
                f[4 * e + 3] += wt * u.w;
              }
            }
#pragma unroll
            for (int e = 0; e < 32; ++e) f[e] = jl == 0.f ? 0.f : f[e] * jinv;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              reinterpret_cast<uint4*>(orow + cc * 32)[e] =
                  make_uint4(pack_bf16x2(f[8 * e], f[8 * e + 1]), pack_bf16x2(f[8 * e + 2], f[8 * e + 3]),
                             pack_bf16x2(f[8 * e + 4], f[8 * e + 5]), pack_bf16x2(f[8 * e + 6], f[8 * e + 7]));
          }
          if (lse && hh == 0) *lse = jl == 0.f ? -CUDART_INF_F : jm + log2f(jl);
        }
        if (threadIdx.x == 128) *counter = 0;
      }
      softmax_bar();  // is_last is read before it is written again
    }
    if (!ok && threadIdx.x == 128) set_error(a.err, kDevTimeoutEpilogue);
    tc_fence_before();
  }

  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int HD, bool I8>
int launch(const Params& p, cudaStream_t s) {
  using C = Cfg<HD, I8>;
  const PagedAttnArgs& a = p.a;
  CUtensorMap tq, tk, tv;
  const uint64_t rows = static_cast<uint64_t>(a.cache.num_pages) * a.cache.kv_heads * a.cache.page_size;
  const uint32_t row_bytes = I8 ? HD : 2 * HD, box = row_bytes < 128 ? row_bytes : 128;
  if (!make_tmap_heads(&tq, a.q, HD, a.heads, a.T, a.ldq, p.G, p.bm / p.G) ||
      !make_tmap_rows(&tk, a.cache.k, row_bytes, rows, box, a.cache.page_size) ||
      !make_tmap_rows(&tv, a.cache.v, row_bytes, rows, box, a.cache.page_size))
    return -3;
  const void* fn = reinterpret_cast<const void*>(attn_paged_many_kernel<HD, I8>);
  const cudaError_t attr = smem_limit_once(fn, C::BYTES);
  if (attr != cudaSuccess) return attr;
  const int64_t tiles = (static_cast<int64_t>(a.max_q < 1 ? 1 : a.max_q) * p.G + p.bm - 1) / p.bm;
  const int64_t keys = a.max_kv < 1 ? 1 : a.max_kv;
  const int64_t most = a.nseq * static_cast<int64_t>(a.cache.kv_heads) * tiles * ((keys + kBK - 1) / kBK);
  const int64_t ctas = attn_paged_many_ctas();
  attn_paged_many_kernel<HD, I8>
      <<<static_cast<unsigned>(most < ctas ? most : ctas), C::THREADS, C::BYTES, s>>>(tq, tk, tv, p, 1);
  return cudaGetLastError();
}

}  // namespace
}  // namespace paged

int64_t attn_paged_many_ctas() { return num_sms() < paged::kMaxCtas ? num_sms() : paged::kMaxCtas; }

int attn_paged_many(const paged::Params& p, cudaStream_t s) {
  if (p.a.cache.hd == 128) return p.a.cache.int8 ? paged::launch<128, true>(p, s) : paged::launch<128, false>(p, s);
  return p.a.cache.int8 ? paged::launch<64, true>(p, s) : paged::launch<64, false>(p, s);
}

}  // namespace rt
