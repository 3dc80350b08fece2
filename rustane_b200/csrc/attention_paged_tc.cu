// Attention over the paged cache for many rows per key head (prompts in chunks, several
// new tokens at once): tiles of up to 128 rows on tcgen05 / TMEM.  Semantics, the split of
// the work and the join as in attention_paged.cu; the products and the softmax are built
// like the training forward's (attention_tc.cu).
//
// Compute-bound on the 4 hd flop per row and visible key; the exponentials (one a score, 16 a
// clock and SM) take as long as the products at hd 128.  One persistent CTA per SM runs two
// streams, each with its own S and O in TMEM, its own MMA warp and its own 128 softmax
// threads, one row each.  A stream takes 64 keys at a time, into two S buffers in turn, so the
// scores of the next 64 are ready before the weights of the last are in the product.  An item is
// up to 2 x 128 rows; the streams take a half each and share every K and V tile, or, if the rows
// fit one half, take the blocks in turn and add up at the end.
//   warp 0      TMA producer: Q of each item (one box a half: whole tokens x the G heads of the
//               key head), then the pages of 128-key K and V tiles into one ring;
//   warps 1, 3  MMA issuers of the two streams: S_{n+1} = Q K^T, then O += P_n V with P (over
//               S) as the TMEM operand.  They zero the v rows of a bf16 edge tile that no row sees;
//   warp 2      owns the TMEM allocation;
//   warps 4-11  softmax, 4 warps a stream: the row's maximum, then P; O rescaled only when the
//               running maximum grew by more than 2^8;
//   warps 12-15 (int8 cache) turn the codes into bf16 tiles, exactly, one key a thread; k's scale
//               multiplies the scores and v's the weights, in fp32.
// Measured: 4 x 509 tokens over up to 4091, 20 heads, 104 us (586 TFLOP/s); 1024 over 8192, 16 heads,
// 100 us (642; int8 137 us); 1531 over 20011, 32 query and 8 key heads, int8, 809 us (597).  Per 64-key step of
// 2450 clocks the softmax waits 700 for its scores, takes 260 for the maximum and 1010 for the
// exponentials; start-up, partial results and the join of split items are a sixth of the 102 us.
// Other forms, same cases: one stream of two threads a row 115; one S buffer of 128 keys a
// stream 157; S of 128 keys into both buffers 107; P in shared memory 108; exponentials partly on the FMA
// pipe 104 and up; int8 with a branch for unseen weights inside the exponent loop +13%.
// P is rounded to bf16 for the P V product (its sum is not), 2^-8 of each weight, as in the training forward: a
// product for the remainder would add half as much again to the products of a step.  All waits are bounded.
#include <type_traits>

#include "attention_paged.cuh"
#include "kernels.h"

namespace rt {
namespace paged {
namespace {

constexpr int kBM = 128;               // rows of a half
constexpr int kBK = 128;
constexpr int kAtomBytes = kBM * 128;  // 64 bf16 columns of 128 rows
constexpr int kStages8 = 3;            // int8 tiles (k or v) in flight
constexpr int kScaleSlots = 4;         // blocks whose scales are held
constexpr int kSub = 64;               // keys that a stream takes at a time
constexpr int kMaxRing = 8;

// Every wait names a phase by its parity, so a waiter may be at most one phase behind or ahead of
// its barrier: each role waits for every phase of the barriers that it uses, in order, and both
// streams hand back every tile, taken or not.
enum Bar : int {
  kQFull = 0,
  kQEmpty = 1,                              // both streams' S MMAs of the item done
  kOFree = 2,                               // both O buffers read
  kSFull = 3,                               // [2 streams][2 buffers]
  kPFull = 7,                               // [2 streams][2 buffers]
  kPvDone = 11,                             // [2 streams][2 buffers]; the buffer is free too
  kDrain = 15,                              // [2 streams]
  kTileFull = 17,                           // [kMaxRing] K and V tiles in turn
  kTileEmpty = kTileFull + kMaxRing,        // [kMaxRing] both streams are done with it
  kCodeFull = kTileEmpty + kMaxRing,        // [kStages8]
  kCodeEmpty = kCodeFull + kStages8,        // [kStages8]
  kScaleFull = kCodeEmpty + kStages8,       // [kScaleSlots]
  kScaleEmpty = kScaleFull + kScaleSlots,   // [kScaleSlots]
  kNumBars = kScaleEmpty + kScaleSlots
};

template <int HD, bool I8>
struct Cfg {
  static constexpr int ATOMS = HD / 64;
  static constexpr int TILE = ATOMS * kAtomBytes;  // a half of Q, K or V in bf16
  static constexpr int ROW8 = HD;                  // bytes of an int8 key
  static constexpr int CODES = kBK * ROW8;
  static constexpr int RING = HD == 64 ? 8 : I8 ? 3 : 4;
  static constexpr int Q = 0;
  static constexpr int KV = Q + 2 * TILE;  // [RING]
  static constexpr int CODE = KV + RING * TILE;
  static constexpr int SCALE = CODE + (I8 ? kStages8 * CODES : 0);          // [slot][k, v][128]
  static constexpr int ML = SCALE + (I8 ? kScaleSlots * 2 * kBK * 4 : 0);   // float [2 streams][128][m, l]
  static constexpr int NANS = ML + 2 * kBM * 8;                             // unsigned [4 quadrants][2 streams]
  static constexpr int BAR = NANS + 64;
  static constexpr int BYTES = BAR + 512 + 1024;
  static constexpr int THREADS = I8 ? 512 : 384;
};
static_assert(kNumBars * 8 + 16 <= 512, "barrier area");

// tmem_ld_wait() that also orders the uses of the loaded registers after it.
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                 "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                 "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}
// One lane of a converged warp, and a value that all its lanes share, in the forms that the
// compiler keeps in uniform registers: tcgen05.mma takes its operands from there, and moving them
// over for every product took one lane 100 clocks a product.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }

__device__ __forceinline__ void softmax_bar() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
// the two softmax warps (one a stream) of TMEM lane quadrant qw
__device__ __forceinline__ void quad_bar(int qw) { asm volatile("bar.sync %0, 64;" ::"r"(2 + qw) : "memory"); }

// row_attend() 8 keys (of one page) at a time, whose loads run side by side; the lanes' sums are halved in
// number at each step, so that 4 lanes end with one key's score.  A warp does up to 32 rows over, one after
// another, while the CTA's other roles wait for it within their limit of 4 s.  4 x 509 rows over 4091 keys, 20 heads,
// one request's all done over: 14.4 ms (76 ms with row_attend(), 20 with 8 whole sums; 0.14 ms without a NaN), 0.11
// us a key and row: the limit is at 1.1M keys of one CTA's part.  (The next 8 keys' loads in flight as well: no
// faster, and its registers cost the ordinary rows 5%.)
template <int HD>
__device__ __noinline__ void redo_row(const Params& p, const int32_t* table, int h, const __nv_bfloat16* qrow, int lo,
                                      int hi, float& m_out, float& l_out, float (&o_out)[HD / 32]) {
  constexpr int E = HD / 32, KB = 8;
  const int lane = threadIdx.x & 31;
  const __nv_bfloat16 *kc = static_cast<const __nv_bfloat16*>(p.a.cache.k),
                      *vc = static_cast<const __nv_bfloat16*>(p.a.cache.v);
  float q[E], o[E], m = -CUDART_INF_F, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = __bfloat162float(qrow[lane * E + e]);
    o[e] = 0.f;
  }
  using Pair = typename std::conditional<E == 4, uint2, uint32_t>::type;
  union Row {
    Pair x;
    uint32_t w[E / 2];
  };
  auto entry = [&](int j0) { return j0 < hi ? table[j0 >> p.page_shift] : 0; };
  const int j_first = lo & ~(KB - 1);
  int page_next = entry(j_first);
  for (int j0 = j_first; j0 < hi; j0 += KB) {
    const int64_t page = checked_page(p, page_next);
    const int64_t at = ((page * p.a.cache.kv_heads + h) << p.page_shift) + (j0 & ((1 << p.page_shift) - 1));
    // all 8 keys are rows of the page, so they can be loaded whether the row sees them or not
    Row k[KB], v[KB];
#pragma unroll
    for (int i = 0; i < KB; ++i) k[i].x = *reinterpret_cast<const Pair*>(kc + (at + i) * HD + lane * E);
#pragma unroll
    for (int i = 0; i < KB; ++i) v[i].x = *reinterpret_cast<const Pair*>(vc + (at + i) * HD + lane * E);
    page_next = entry(j0 + KB);
    float s[KB];
#pragma unroll
    for (int i = 0; i < KB; ++i) {
      s[i] = 0.f;
#pragma unroll
      for (int e = 0; e < E / 2; ++e) s[i] += q[2 * e] * bf16lo(k[i].w[e]) + q[2 * e + 1] * bf16hi(k[i].w[e]);
    }
    // sums over the lanes, half as many a step: lanes 4 i .. 4 i + 3 end with key i's (bits 4, 3, 2 of the lane)
#pragma unroll
    for (int n = KB / 2, x = 16; n; n /= 2, x /= 2) {
      const bool up = lane & x;
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float keep = up ? s[i + n] : s[i], give = up ? s[i] : s[i + n];
        s[i] = keep + __shfl_xor_sync(0xffffffffu, give, x);
      }
    }
#pragma unroll
    for (int x = 2; x; x /= 2) s[0] += __shfl_xor_sync(0xffffffffu, s[0], x);
    const int mine = j0 + (lane >> 2);
    const float score = mine >= lo && mine < hi ? s[0] * p.scale_log2 : -CUDART_INF_F;
    float m2 = score;
#pragma unroll
    for (int x = 4; x < 32; x *= 2) m2 = fmaxf(m2, __shfl_xor_sync(0xffffffffu, m2, x));
    m2 = fmaxf(m, m2);
    const float f = m == m2 ? 1.f : exp2f(m - m2), weight = score == -CUDART_INF_F ? 0.f : exp2f(score - m2);
    l *= f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= f;
#pragma unroll
    for (int i = 0; i < KB; ++i) {
      const float pj = __shfl_sync(0xffffffffu, weight, 4 * i);
      const bool in = j0 + i >= lo && j0 + i < hi;  // an unseen v may be NaN
      l += pj;
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        o[2 * e] += pj * (in ? bf16lo(v[i].w[e]) : 0.f);
        o[2 * e + 1] += pj * (in ? bf16hi(v[i].w[e]) : 0.f);
      }
    }
    m = m2;
  }
  m_out = m;
  l_out = l;
#pragma unroll
  for (int e = 0; e < E; ++e) o_out[e] = o[e];
}

// Columns col .. col + 3 of row r in a partial result: rows side by side, one a thread.
__device__ __forceinline__ float4* part_at(float* part, int r, int col) {
  return reinterpret_cast<float4*>(part) + (col >> 2) * (2 * kBM) + r;
}

// How an item's part is shared by the two streams.
struct Share {
  bool pair;       // halves of the rows (else: blocks in turn)
  int rows[2];     // rows of each half
  int lo[2], hi[2];  // keys that each half sees
  int key0;        // first key of the part
  __device__ __forceinline__ Share(const Walk<kBK>& w, int half) {
    const int n = w.rows();
    pair = n > half;
    rows[0] = min(n, half);
    rows[1] = pair ? n - half : rows[0];
    key0 = (w.blk0 + w.off) * kBK;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      lo[u] = pair ? w.row_lo(u * half) : w.lo;
      hi[u] = pair ? max(0, w.row_hi(u * half + rows[u] - 1)) : w.hi;
    }
  }
  // whether any row sees the part's block b: others are not loaded (rows of a short window may
  // leave such blocks between the halves)
  __device__ __forceinline__ bool loaded(int b) const { return !pair || takes(0, b) || takes(1, b); }
  // whether stream u works on the part's block b
  __device__ __forceinline__ bool takes(int u, int b) const {
    const int k = key0 + b * kBK;
    return pair ? k < hi[u] && k + kBK > lo[u] : (b & 1) == u;
  }
  // whether block b is the last one of stream u in a part of cnt blocks
  __device__ __forceinline__ bool ends(int u, int b, int cnt) const {
    return pair ? b + 1 >= cnt || !takes(u, b + 1) : b + 2 >= cnt;
  }
  // stream u's blocks: [first, end), every one (halves) or every other one
  __device__ __forceinline__ int first(int u) const { return pair ? max(0, lo[u] - key0) / kBK : u; }
  __device__ __forceinline__ int end(int u, int cnt) const {
    return !pair ? cnt : hi[u] > lo[u] ? min(cnt, (max(0, hi[u] - key0) + kBK - 1) / kBK) : 0;
  }
  __device__ __forceinline__ int count(int u, int cnt) const {
    return pair ? max(0, end(u, cnt) - first(u)) : (cnt + 1 - u) >> 1;
  }
};

template <int HD, bool I8>
__global__ void __launch_bounds__(Cfg<HD, I8>::THREADS, 1)
    attn_paged_many_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                           const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Params p) {
  using C = Cfg<HD, I8>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + C::BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* is_last = abort_flag + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int half = p.bm / 2;
  const PagedAttnArgs& a = p.a;

  if (threadIdx.x == 0) {
    mbar_init(&bar[kQFull], 1);
    mbar_init(&bar[kQEmpty], 2);
    mbar_init(&bar[kOFree], 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar[kDrain + i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&bar[kSFull + i], 1);
      mbar_init(&bar[kPFull + i], 4);
      mbar_init(&bar[kPvDone + i], 1);
    }
    for (int i = 0; i < C::RING; ++i) {
      mbar_init(&bar[kTileFull + i], I8 ? 4 : 1);
      mbar_init(&bar[kTileEmpty + i], 2);
    }
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
  Walk<kBK> w = start_walk<kBK, C::THREADS>(p, total, P);  // its barriers cover the set-up above
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;  // columns [0,128) S0, [128,256) S1, then O0, O1 of 128 each
  auto wait_all = [&](uint64_t* b, uint32_t parity) {  // a whole warp; false: timed out or given up
    return __all_sync(0xffffffffu, mbar_wait(b, parity) && !*abort_flag);
  };

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
    int q_issued = 0, t_issued = 0, s_issued = 0;  // t_issued: tiles of the ring, or int8 tiles
    bool ok = true;
    for (; ok && w.more(); w.next()) {
      if (w.empty()) continue;
      const int32_t* table = a.table + w.s * a.table_ld;
      const int cnt = w.count();
      const int key00 = (w.blk0 + w.off) * kBK;
      const Share sh(w, half);
      auto my_page = [&](int b) {
        const int key = key00 + b * kBK + lane * ps;
        return b < cnt && lane * ps < kBK && key < w.hi && key + ps > w.lo ? page_of(p, table, key) : -1;
      };
      auto after = [&](int b) {
        do ++b;
        while (b < cnt && !sh.loaded(b));
        return b;
      };
      int page = my_page(after(-1));
      if (it > 0 && !wait_all(&bar[kQEmpty], (it - 1) & 1)) {
        ok = false;
        break;
      }
      if (lane == 0) {
        const int halves = sh.pair ? 2 : 1;
        mbar_arrive_expect_tx(&bar[kQFull], halves * C::ATOMS * half * 128);
        for (int u = 0; u < halves; ++u)
#pragma unroll
          for (int x = 0; x < C::ATOMS; ++x)
            tma_load_3d(smem + C::Q + u * C::TILE + x * kAtomBytes, &tm_q, &bar[kQFull], x * 64, w.h * p.G,
                        w.q0 + (w.t * p.bm + u * half) / p.G);
      }
      q_issued = ++it;
      for (int b = after(-1); b < cnt; b = after(b), ++g) {
        const int ahead = my_page(after(b));
        const int loads = __popc(__ballot_sync(0xffffffffu, page >= 0));
        const int64_t row64 = ((static_cast<int64_t>(page < 0 ? 0 : page) * a.cache.kv_heads + w.h) << p.page_shift);
        const int row = static_cast<int>(row64);
        if (I8) {
          const int sl = g % kScaleSlots;
          if (!wait_all(&bar[kScaleEmpty + sl], ((g / kScaleSlots) & 1) ^ 1)) {
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
          const int x = 2 * g + kv;
          const int n = I8 ? kStages8 : C::RING, st = x % n;
          uint64_t* full = &bar[(I8 ? kCodeFull : kTileFull) + st];
          if (!wait_all(&bar[(I8 ? kCodeEmpty : kTileEmpty) + st], ((x / n) & 1) ^ 1)) {
            ok = false;
            break;
          }
          if (lane == 0) mbar_arrive_expect_tx(full, loads * ps * (I8 ? C::ROW8 : C::ATOMS * 128));
          __syncwarp();
          if (page >= 0) {
            if (I8) {
              tma_load_2d(smem + C::CODE + st * C::CODES + lane * ps * C::ROW8, tm, full, 0, row);
            } else {
#pragma unroll
              for (int y = 0; y < C::ATOMS; ++y)
                tma_load_2d(smem + C::KV + st * C::TILE + y * kAtomBytes + lane * ps * 128, tm, full, y * 128, row);
            }
          }
          t_issued = x + 1;
          __syncwarp();
        }
        if (!ok) break;
        page = ahead;
      }
    }
    if (!ok) {  // let copies still in flight land before the CTA exits
      if (lane == 0) set_error(a.err, kDevTimeoutProducer);
      *abort_flag = 1;
      const int n = I8 ? kStages8 : C::RING;
      if (q_issued > 0) mbar_wait(&bar[kQFull], (q_issued - 1) & 1);
      for (int x = t_issued > n ? t_issued - n : 0; x < t_issued; ++x)
        mbar_wait(&bar[(I8 ? kCodeFull : kTileFull) + x % n], (x / n) & 1);
      for (int x = s_issued > kScaleSlots ? s_issued - kScaleSlots : 0; x < s_issued; ++x)
        mbar_wait(&bar[kScaleFull + x % kScaleSlots], (x / kScaleSlots) & 1);
    }
  } else if (warp == 1 || warp == 3) {
    // ------------------------------------------------------- MMA issuer of stream u
    constexpr uint32_t idesc_s = idesc_bf16_f32(kBM, kSub, false, false);  // Q, K: both hd-contiguous
    constexpr uint32_t idesc_o = idesc_bf16_f32(kBM, HD, false, true);    // P key-contiguous, V hd-contiguous
    const int u = uniform(warp >> 1);
    const uint32_t ts = uniform(tmem) + u * 128, to = uniform(tmem) + 256 + u * 128;
    // Descriptors of the first tile; others are a number of 16-byte units further (building one for
    // every product took one lane longer than the products themselves)
    const uint64_t q_desc = smem_desc_sw128(smem_u32(smem + C::Q), 16, 1024);
    const uint64_t kv_desc = smem_desc_sw128(smem_u32(smem + C::KV), 16, 1024);
    const uint64_t v_desc = smem_desc_sw128(smem_u32(smem + C::KV), kAtomBytes, 1024);
    bool ok = true;
    int g = 0, it = 0, n = 0;  // n: 64-key steps of this stream so far
    for (; ok && w.more(); w.next()) {
      if (w.empty()) continue;
      const int cnt = w.count();
      const Share sh(w, half);
      const uint64_t dq = q_desc + uniform(sh.pair ? u * (C::TILE >> 4) : 0);
      if (!wait_all(&bar[kQFull], it & 1)) {
        ok = false;
        break;
      }
      // block bb (the CTA's gg-th) -> the next one that the stream takes, or the end; the tiles of
      // the others are handed back
      auto forward = [&](int& bb, int& gg) {
        for (;;) {
          if (bb >= 0 && sh.loaded(bb)) ++gg;
          if (++bb >= cnt || sh.takes(u, bb)) return true;
          if (!sh.loaded(bb)) continue;
          for (int x = 2 * gg; x < 2 * gg + 2; ++x) {
            if (!wait_all(&bar[kTileFull + x % C::RING], (x / C::RING) & 1)) return false;
            if (lane == 0) mbar_arrive(&bar[kTileEmpty + x % C::RING]);
          }
          __syncwarp();
        }
      };
      // S of 64 keys into buffer nn & 1, once P V of step nn - 2 has read its weights there
      auto issue_s = [&](int bb, int gg, int h, int nn) {
        const int kx = (2 * gg) % C::RING;
        if ((h == 0 && !wait_all(&bar[kTileFull + kx], ((2 * gg) / C::RING) & 1)) ||
            (nn >= 2 && !wait_all(&bar[kPvDone + 2 * u + (nn & 1)], ((nn - 2) >> 1) & 1)))
          return false;
        tc_fence_after();
        const uint64_t dk = kv_desc + uniform(kx * (C::TILE >> 4) + h * (kSub * 128 >> 4));
        const uint32_t buf = uniform(nn & 1);
        const bool free_k = uniform(h == 1), free_q = uniform(h == 1 && sh.ends(u, bb, cnt));
        const uint32_t k_slot = uniform(kx);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint32_t off = ((kk >> 2) * kAtomBytes + (kk & 3) * 32) >> 4;
            umma_bf16(ts + buf * kSub, dq + off, dk + off, idesc_s, kk != 0 ? 1u : 0u);
          }
          umma_commit(&bar[kSFull + 2 * u + buf]);
          if (free_k) umma_commit(&bar[kTileEmpty + k_slot]);
          if (free_q) umma_commit(&bar[kQEmpty]);
        }
        __syncwarp();
        return true;
      };
      // With 3 tiles in the ring and blocks in turn, the stream's next K goes where its V is now
      const bool ahead = C::RING > 3 || sh.pair;
      int b = -1, gb = g;
      ok = forward(b, gb);
      if (ok && b < cnt) {
        ok = issue_s(b, gb, 0, n);
      } else if (lane == 0) {
        mbar_arrive(&bar[kQEmpty]);
      }
      bool first = true;
      while (ok && b < cnt) {
        int b2 = b, g2 = gb;
        const int vx = (2 * gb + 1) % C::RING;
        uint8_t* vt = smem + C::KV + vx * C::TILE;
        for (int h = 0; ok && h < 2; ++h, ++n) {
          if (h == 0) ok = issue_s(b, gb, 1, n + 1);
          else if (ahead && !sh.ends(u, b, cnt)) ok = forward(b2, g2) && issue_s(b2, g2, 0, n + 1);
          if (!ok) break;
          if (h == 0) {
            ok = wait_all(&bar[kTileFull + vx], ((2 * gb + 1) / C::RING) & 1);
            if (!ok) break;
            const int key0 = sh.key0 + b * kBK;
            if (!I8 && (key0 < w.lo || key0 + kBK > w.hi)) {
              // keys that no row of the item sees weigh 0, but what is there may be NaN (both
              // streams write the same zeros, each before its own product)
              const int from = max(0, w.lo - key0), to_row = min(kBK, w.hi - key0);
#pragma unroll
              for (int x = 0; x < C::ATOMS; ++x) {
                uint4* rows = reinterpret_cast<uint4*>(vt + x * kAtomBytes);
                for (int i = lane; i < from * 8; i += 32) rows[i] = make_uint4(0, 0, 0, 0);
                for (int i = to_row * 8 + lane; i < kBK * 8; i += 32) rows[i] = make_uint4(0, 0, 0, 0);
              }
              fence_proxy_async_smem();
              __syncwarp();
            }
          }
          ok = wait_all(&bar[kPFull + 2 * u + (n & 1)], (n >> 1) & 1) &&
               (!first || it == 0 || wait_all(&bar[kOFree], (it - 1) & 1));
          if (!ok) break;
          tc_fence_after();
          const uint64_t dv = v_desc + uniform(vx * (C::TILE >> 4) + h * (kSub * 128 >> 4));
          const uint32_t buf = uniform(n & 1), v_slot = uniform(vx);
          const bool free_v = uniform(h == 1), add0 = uniform(!first);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < kSub / 16; ++kk)
              umma_bf16_ts(to, ts + buf * kSub + kk * 8, dv + kk * (2048 >> 4), idesc_o, kk == 0 && !add0 ? 0u : 1u);
            umma_commit(&bar[kPvDone + 2 * u + buf]);
            if (free_v) umma_commit(&bar[kTileEmpty + v_slot]);
          }
          __syncwarp();
          first = false;
        }
        if (ok && b2 == b) ok = forward(b2, g2) && (b2 >= cnt || issue_s(b2, g2, 0, n));
        if (!ok) break;
        b = b2;
        gb = g2;
      }
      g = gb;  // past the part's last block: every loaded one is counted
      // a stream without a block in this item still takes part in the O hand-over
      if (ok && first && it > 0) ok = wait_all(&bar[kOFree], (it - 1) & 1);
      ++it;
    }
    if (!ok) {
      if (lane == 0) set_error(a.err, kDevTimeoutMma);
      *abort_flag = 1;
    }
    if (elect_one()) {  // the lane that issued the products
      umma_commit(&bar[kDrain + u]);
      mbar_wait(&bar[kDrain + u], 0);
    }
    __syncwarp();
  } else if (I8 && warp >= 12) {
    // ------------------------------------------------------------ int8 -> bf16
    int x = 0;
    bool ok = true;
    for (; ok && w.more(); w.next()) {
      if (w.empty()) continue;
      const int cnt = w.count();
      const Share sh(w, half);
      for (int b = 0; ok && b < 2 * cnt; ++b) {
        if (!sh.loaded(b >> 1)) continue;
        const int cs = x % kStages8, st = x % C::RING;
        ok = wait_all(&bar[kCodeFull + cs], (x / kStages8) & 1) && wait_all(&bar[kTileEmpty + st], ((x / C::RING) & 1) ^ 1);
        if (!ok) break;
        {
          const int r = threadIdx.x - 384;  // key of the block
          const uint8_t* src = smem + C::CODE + cs * C::CODES + r * C::ROW8;
          uint8_t* dst = smem + C::KV + st * C::TILE + r * 128;
          uint4 codes[HD / 16];  // all of the key's first: the compiler moves no load before a store
#pragma unroll
          for (int ch = 0; ch < HD / 16; ++ch)
            codes[ch] = *reinterpret_cast<const uint4*>(src + (HD == 64 ? ch ^ ((r >> 1) & 3) : ch ^ (r & 7)) * 16);
#pragma unroll
          for (int ch = 0; ch < HD / 16; ++ch) {
            const uint4 q = codes[ch];
            uint8_t* d = dst + (ch >> 2) * kAtomBytes;
            const int c0 = (ch & 3) * 2;
            *reinterpret_cast<uint4*>(d + ((c0 ^ (r & 7)) << 4)) =
                make_uint4(i8x2_bf16x2<0, 1>(q.x), i8x2_bf16x2<2, 3>(q.x), i8x2_bf16x2<0, 1>(q.y), i8x2_bf16x2<2, 3>(q.y));
            *reinterpret_cast<uint4*>(d + (((c0 + 1) ^ (r & 7)) << 4)) =
                make_uint4(i8x2_bf16x2<0, 1>(q.z), i8x2_bf16x2<2, 3>(q.z), i8x2_bf16x2<0, 1>(q.w), i8x2_bf16x2<2, 3>(q.w));
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bar[kCodeEmpty + cs]);
          mbar_arrive(&bar[kTileFull + st]);
        }
        ++x;
      }
    }
    if (!ok) {
      if (lane == 0) set_error(a.err, kDevTimeoutEpilogue);
      *abort_flag = 1;
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------- softmax of stream u, row r
    const int qw = warp & 3;          // TMEM lane quadrant
    const int u = (warp - 4) >> 2;
    const int r = qw * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(qw * 32) << 16;
    const uint32_t to = tmem + 256 + lane_off;
    float* ml = reinterpret_cast<float*>(smem + C::ML);
    volatile unsigned* nans = reinterpret_cast<volatile unsigned*>(smem + C::NANS);
    const float raise = kRescale / p.scale_log2;
    // A failed (timed-out) wait does not leave the loops: every softmax warp must reach the same
    // sequence of named barriers.  After the first failure every later wait returns at once.
    bool ok = true;
    auto wait = [&](uint64_t* bb, uint32_t parity) {
      bool good = !*abort_flag && mbar_wait(bb, parity);
      good = __all_sync(0xffffffffu, good);
      if (!good) {
        ok = false;
        *abort_flag = 1;
      }
    };
    int g = 0, n = 0;  // loaded blocks of the CTA, 64-key steps of the stream so far
    for (; w.more(); w.next()) {
      const int cnt = w.count();
      const Share sh(w, half);
      const int base = sh.pair ? u * half : 0;  // the stream's first row in the item
      const bool in = r < sh.rows[u];
      const int row = base + min(r, sh.rows[u] - 1);
      const int64_t tok = w.q0 + (w.t * p.bm + row) / p.G;
      const int head = w.h * p.G + (w.t * p.bm + row) % p.G;
      __nv_bfloat16* orow = a.out + tok * a.ldo + head * HD;
      float* lse = a.lse2 ? a.lse2 + tok * a.heads + head : nullptr;
      if (w.empty()) {
        if (in && (sh.pair || u == 0)) {
#pragma unroll
          for (int i = 0; i < HD / 8; ++i) reinterpret_cast<uint4*>(orow)[i] = make_uint4(0, 0, 0, 0);
          if (lse) *lse = -CUDART_INF_F;
        }
        continue;
      }
      const int hi_r = w.row_hi(row), lo_r = w.row_lo(row);
      // keys that every row of the stream sees
      const int lo_all = w.row_lo(base + sh.rows[u] - 1), hi_all = w.row_hi(base);
      float m_used = -CUDART_INF_F, l = 0.f;  // m_used: of the unscaled scores
      bool first = true;
      // a bf16 cache: the stream's own blocks; an int8 one: every loaded block's scales pass by
      const int b_step = I8 || sh.pair ? 1 : 2, b_first = I8 ? 0 : sh.first(u), b_end = I8 ? cnt : sh.end(u, cnt);
      for (int b = b_first; b < b_end; b += b_step) {
        if (I8 && !sh.loaded(b)) continue;
        if (I8) wait(&bar[kScaleFull + g % kScaleSlots], (g / kScaleSlots) & 1);
#pragma unroll 1
        for (int h = I8 && !sh.takes(u, b) ? 2 : 0; h < 2; ++h) {
          const float* scales = reinterpret_cast<const float*>(smem + C::SCALE + (g % kScaleSlots) * (2 * kBK * 4)) + h * kSub;
          const int key0 = sh.key0 + b * kBK + h * kSub;
          const bool masked = key0 < lo_all || key0 + kSub > hi_all;
          const uint32_t ts = tmem + u * 128 + (n & 1) * kSub + lane_off;
          wait(&bar[kSFull + 2 * u + (n & 1)], (n >> 1) & 1);
          tc_fence_after();
          uint32_t v[2][32];
          const int last = hi_r - key0, from = lo_r - key0;  // seen: from <= e < last
          auto scale_k = [&](uint32_t (&x)[32], int c) {
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float4 k4 = *reinterpret_cast<const float4*>(scales + c * 32 + e);
              float x0, x1, x2, x3;
              f2_unpack(f2_mul(f2_pack(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), f2_pack(k4.x, k4.y)), x0, x1);
              f2_unpack(f2_mul(f2_pack(__uint_as_float(x[e + 2]), __uint_as_float(x[e + 3])), f2_pack(k4.z, k4.w)), x2, x3);
              x[e] = __float_as_uint(x0);
              x[e + 1] = __float_as_uint(x1);
              x[e + 2] = __float_as_uint(x2);
              x[e + 3] = __float_as_uint(x3);
            }
          };
          auto top = [](const uint32_t (&x)[32]) {
            float mc[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              mc[q] = fmax3(__uint_as_float(x[16 * q]), __uint_as_float(x[16 * q + 1]), __uint_as_float(x[16 * q + 2]));
#pragma unroll
              for (int e = 3; e < 15; e += 2)
                mc[q] = fmax3(mc[q], __uint_as_float(x[16 * q + e]), __uint_as_float(x[16 * q + e + 1]));
            }
            return fmaxf(fmaxf(mc[0], __uint_as_float(x[15])), fmaxf(mc[1], __uint_as_float(x[31])));
          };
          tmem_ld32(ts, v[0]);
          tmem_ld32(ts + 32, v[1]);
          tmem_ld_wait(v[0]);
          tmem_ld_wait(v[1]);
          if (I8) {
            scale_k(v[0], 0);
            scale_k(v[1], 1);
          }
          if (masked) {
#pragma unroll
            for (int e = 0; e < 64; ++e)
              if (e >= last || e < from) v[e >> 5][e & 31] = __float_as_uint(-CUDART_INF_F);
          }
          const float m_new = fmax3(m_used, top(v[0]), top(v[1]));
          if (first) {
            m_used = m_new;
          } else if (__any_sync(0xffffffffu, m_new > m_used + raise)) {
            wait(&bar[kPvDone + 2 * u + ((n - 1) & 1)], ((n - 1) >> 1) & 1);
            tc_fence_after();
            const bool grow = m_new > m_used + raise;
            const float f = grow ? exp2f((m_used - m_new) * p.scale_log2) : 1.f;
            if (grow) {
              l *= f;
              m_used = m_new;
            }
#pragma unroll 1
            for (int cc = 0; cc < HD / 32; ++cc) {
              uint32_t o[32];
              tmem_ld32(to + u * 128 + cc * 32, o);
              tmem_ld_wait(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st32(to + u * 128 + cc * 32, o);
            }
            tmem_st_wait();
          }
          // a maximum of -inf (the row has seen nothing yet) is taken as 0: its weights come out 0.
          // The difference first: a fused scale * s - m would leave m's rounding, which is
          // everything where scores are near the lowest value of the type
          const float ms = m_used == -CUDART_INF_F ? 0.f : m_used;
          const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2), ms2 = f2_pack(ms, ms);
          uint64_t ls2[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
          // P in bf16 pairs over the row's own S columns: keys 2 i, 2 i + 1 at column i
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t(&x)[32] = v[c];
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              float pw[4];
#pragma unroll
              for (int i = 0; i < 4; i += 2) {
                float x0, x1;
                f2_unpack(f2_mul(f2_sub(f2_pack(__uint_as_float(x[e + i]), __uint_as_float(x[e + i + 1])), ms2), sc2), x0, x1);
                pw[i] = ex2_approx(x0);
                pw[i + 1] = ex2_approx(x1);
                ls2[c] = f2_add(ls2[c], f2_pack(pw[i], pw[i + 1]));
              }
              if (I8) {
                const float4 vs = *reinterpret_cast<const float4*>(scales + kBK + c * 32 + e);
                f2_unpack(f2_mul(f2_pack(pw[0], pw[1]), f2_pack(vs.x, vs.y)), pw[0], pw[1]);
                f2_unpack(f2_mul(f2_pack(pw[2], pw[3]), f2_pack(vs.z, vs.w)), pw[2], pw[3]);
              }
              pk[e / 2] = pack_bf16x2(pw[0], pw[1]);
              pk[e / 2 + 1] = pack_bf16x2(pw[2], pw[3]);
            }
            tmem_st16(ts + c * 16, pk);
          }
          {
            float a0, a1, b0, b1;
            f2_unpack(ls2[0], a0, a1);
            f2_unpack(ls2[1], b0, b1);
            l += (a0 + a1) + (b0 + b1);
          }
          tmem_st_wait();
          if (I8 && masked) {
            // 0 where unseen, whatever the scale of that key is (a branch in the loop above, which
            // keeps the compiler from mixing its two halves, cost every step 13%)
            uint32_t pw[32];
            tmem_ld32(ts, pw);
            tmem_ld_wait(pw);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              pw[i] &= (2 * i >= from && 2 * i < last ? 0xffffu : 0u) | (2 * i + 1 >= from && 2 * i + 1 < last ? 0xffff0000u : 0u);
            tmem_st32(ts, pw);
            tmem_st_wait();
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar[kPFull + 2 * u + (n & 1)]);
          ++n;
          first = false;
        }
        if (I8) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar[kScaleEmpty + g % kScaleSlots]);
        }
        ++g;
      }
      // ------------------------------------------------------------- end of the item (or part)
      // A thread has its row's HD columns (halves), or half of them from both streams' sums.
      const int c0 = sh.count(0, cnt), c1 = sh.count(1, cnt);
      if ((u ? c1 : c0) > 0) wait(&bar[kPvDone + 2 * u + ((n - 1) & 1)], ((n - 1) >> 1) & 1);
      tc_fence_after();
      float f0 = 1.f, f1 = 1.f;  // factors of O0, O1
      if (sh.pair) {
        f0 = u == 0 && c0 > 0 ? 1.f : 0.f;
        f1 = u == 1 && c1 > 0 ? 1.f : 0.f;
      } else {
        ml[(u * kBM + r) * 2] = m_used;
        ml[(u * kBM + r) * 2 + 1] = l;
        tc_fence_before();
        quad_bar(qw);  // the other stream's O is complete too
        tc_fence_after();
        const float m0 = ml[r * 2], m1 = ml[(kBM + r) * 2];
        m_used = fmaxf(m0, m1);
        const float ms = m_used == -CUDART_INF_F ? 0.f : m_used;
        f0 = exp2f((m0 - ms) * p.scale_log2);
        f1 = c1 > 0 ? exp2f((m1 - ms) * p.scale_log2) : 0.f;
        l = ml[r * 2 + 1] * f0 + ml[(kBM + r) * 2 + 1] * f1;
      }
      const int col0 = sh.pair ? 0 : u * (HD / 2), chunks = sh.pair ? HD / 32 : HD / 64;
      // 32 columns of the row's sum; O of a stream without blocks is never read
      auto column32 = [&](int cc, float (&f)[32]) {
        uint32_t o[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) f[e] = 0.f;
        if (sh.pair ? u == 0 && c0 > 0 : c0 > 0) {
          tmem_ld32(to + col0 + cc * 32, o);
          tmem_ld_wait(o);
#pragma unroll
          for (int e = 0; e < 32; ++e) f[e] = __uint_as_float(o[e]) * f0;
        }
        if (sh.pair ? u == 1 && c1 > 0 : c1 > 0) {
          tmem_ld32(to + 128 + col0 + cc * 32, o);
          tmem_ld_wait(o);
#pragma unroll
          for (int e = 0; e < 32; ++e) f[e] = fmaf(__uint_as_float(o[e]), f1, f[e]);
        }
      };
      const bool split = w.off > 0 || cnt < w.nb;
      float* part = split ? partial_slot<2 * kBM, HD>(p, blockIdx.x, w.off > 0 ? 0 : 1) : nullptr;
      const float inv = l == 0.f ? 0.f : 1.f / l, m_log2 = m_used * p.scale_log2;
      bool nan = false;
#pragma unroll 1
      for (int cc = 0; cc < chunks; ++cc) {
        float f[32];
        column32(cc, f);
        const int col = col0 + cc * 32;
#pragma unroll
        for (int e = 0; e < 32; ++e) nan = nan || isnan(f[e]);
        if (in && split) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            __stcg(part_at(part, row, col + 4 * e), make_float4(f[4 * e], f[4 * e + 1], f[4 * e + 2], f[4 * e + 3]));
        } else if (in && ok) {
#pragma unroll
          for (int e = 0; e < 32; ++e) f[e] = l == 0.f ? 0.f : f[e] * inv;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            reinterpret_cast<uint4*>(orow + col)[e] =
                make_uint4(pack_bf16x2(f[8 * e], f[8 * e + 1]), pack_bf16x2(f[8 * e + 2], f[8 * e + 3]),
                           pack_bf16x2(f[8 * e + 4], f[8 * e + 5]), pack_bf16x2(f[8 * e + 6], f[8 * e + 7]));
        }
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar[kOFree]);  // the O buffers can take the next item
      if (in && (sh.pair || u == 0)) {
        if (split) {
          __stcg(part + 2 * kBM * HD + row, m_log2);
          __stcg(part + 2 * kBM * HD + 2 * kBM + row, l);
        } else if (lse && ok) {
          *lse = l == 0.f ? -CUDART_INF_F : m_log2 + log2f(l);
        }
      }
      // a row may have met a NaN or an infinity of a key that only a later row sees: it is done
      // over, alone, and written over
      unsigned todo = 0;
      if (!I8 && w.n > 1) {
        todo = __ballot_sync(0xffffffffu, nan && in && ok);
        if (!sh.pair) {
          if (lane == 0) nans[qw * 2 + u] = todo;
          quad_bar(qw);
          todo = nans[qw * 2] | nans[qw * 2 + 1];
        }
      }
      if (todo) {
        const int seg_lo = sh.key0, seg_hi = seg_lo + cnt * kBK;
        int nth = 0;
        for (int x = 0; x < 32; ++x) {
          // of a row that both streams share, the quadrant's two warps take every other one
          if (!((todo >> x) & 1u) || (!sh.pair && (nth++ & 1) != u)) continue;
          const int rx = base + qw * 32 + x, fl = w.t * p.bm + rx;
          const int64_t tk = w.q0 + fl / p.G;
          const int hd = w.h * p.G + fl % p.G;
          float rm, rl, ro[HD / 32];
          redo_row<HD>(p, a.table + w.s * a.table_ld, w.h, a.q + tk * a.ldq + hd * HD, max(w.row_lo(rx), seg_lo),
                       min(w.row_hi(rx), seg_hi), rm, rl, ro);
          const float rinv = rl == 0.f ? 0.f : 1.f / rl;
#pragma unroll
          for (int e = 0; e < HD / 32; ++e) {
            const int col = lane * (HD / 32) + e;
            if (split) __stcg(reinterpret_cast<float*>(part_at(part, rx, col)) + (col & 3), ro[e]);
            else a.out[tk * a.ldo + hd * HD + col] = __float2bfloat16(rl == 0.f ? 0.f : ro[e] * rinv);
          }
          if (lane == 0) {
            if (split) {
              __stcg(part + 2 * kBM * HD + rx, rm);
              __stcg(part + 2 * kBM * HD + 2 * kBM + rx, rl);
            } else if (a.lse2) {
              a.lse2[tk * a.heads + hd] = rl == 0.f ? -CUDART_INF_F : rm + log2f(rl);
            }
          }
        }
      }
      if (!sh.pair) quad_bar(qw);  // ml and nans are read before the next item writes them
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
        auto slot_of = [&](int cta) { return partial_slot<2 * kBM, HD>(p, cta, cta == cta0 ? 1 : 0); };
        // a thread joins 16 or more columns of a row: rows side by side, so that loads coalesce
        const int rows = w.rows();
        int wide = 16;
        while (wide < HD && 256 / (HD / wide) < rows) wide *= 2;
        const int lanes = 256 / (HD / wide), jr = (threadIdx.x - 128) % lanes, jc = (threadIdx.x - 128) / lanes * wide;
        if (ok && jr < rows) {
          float jm = -CUDART_INF_F, jl = 0.f;
          for (int x = cta0; x <= cta1; ++x) jm = fmaxf(jm, __ldcg(slot_of(x) + 2 * kBM * HD + jr));
          const float base_m = jm == -CUDART_INF_F ? 0.f : jm;
          for (int x = cta0; x <= cta1; ++x)
            jl += exp2f(__ldcg(slot_of(x) + 2 * kBM * HD + jr) - base_m) * __ldcg(slot_of(x) + 2 * kBM * HD + 2 * kBM + jr);
          const float jinv = jl == 0.f ? 0.f : 1.f / jl;
          const int fl = w.t * p.bm + jr;
          const int64_t tk = w.q0 + fl / p.G;
          const int hd = w.h * p.G + fl % p.G;
#pragma unroll 1
          for (int col = jc; col < jc + wide; col += 16) {
            float f[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) f[e] = 0.f;
            for (int x = cta0; x <= cta1; x += 4) {  // ascending: a fixed order; 4 parts' loads together
              float wt[4];
              float4 q[4][4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                float* src = slot_of(min(x + i, cta1));
                wt[i] = x + i <= cta1 ? __ldcg(src + 2 * kBM * HD + jr) : -CUDART_INF_F;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  q[i][e] = x + i <= cta1 ? __ldcg(part_at(src, jr, col + 4 * e)) : make_float4(0.f, 0.f, 0.f, 0.f);
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                wt[i] = exp2f(wt[i] - base_m);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  f[4 * e] += wt[i] * q[i][e].x;
                  f[4 * e + 1] += wt[i] * q[i][e].y;
                  f[4 * e + 2] += wt[i] * q[i][e].z;
                  f[4 * e + 3] += wt[i] * q[i][e].w;
                }
              }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) f[e] = jl == 0.f ? 0.f : f[e] * jinv;
#pragma unroll
            for (int e = 0; e < 2; ++e)
              reinterpret_cast<uint4*>(a.out + tk * a.ldo + hd * HD + col)[e] =
                  make_uint4(pack_bf16x2(f[8 * e], f[8 * e + 1]), pack_bf16x2(f[8 * e + 2], f[8 * e + 3]),
                             pack_bf16x2(f[8 * e + 4], f[8 * e + 5]), pack_bf16x2(f[8 * e + 6], f[8 * e + 7]));
          }
          if (a.lse2 && jc == 0) a.lse2[tk * a.heads + hd] = jl == 0.f ? -CUDART_INF_F : jm + log2f(jl);
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
  if (!make_tmap_heads(&tq, a.q, HD, a.heads, a.T, a.ldq, p.G, p.bm / 2 / p.G) ||
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
      <<<static_cast<unsigned>(most < ctas ? most : ctas), C::THREADS, C::BYTES, s>>>(tq, tk, tv, p);
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
