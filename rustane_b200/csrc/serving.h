// Launch interface of the serving kernels (internal): per-head norm + rotary
// position (also used in training), the paged key/value cache, attention over
// it, and the step from logits to a token.  Every launch is asynchronous on
// `stream`; 0 = launched, -1 = a shape or alignment the kernels do not take,
// otherwise a cudaError_t.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace rt {

// Rotary tables [n_pos][rot / 2] fp32 and the layout of the rotated pairs:
// half == false: (2i, 2i + 1); half == true: (i, i + rot / 2).
struct RopeTables {
  const float* cos = nullptr;
  const float* sin = nullptr;
  int n_pos = 0, rot = 0;
  bool half = false;
};

// Paged cache, K and V each [num_pages][kv_heads][page_size][hd]: the tokens of one
// head and page are contiguous, so a page is one TMA box.  int8 caches carry one
// fp32 scale per (page, head, token).
struct KvPages {
  void* k = nullptr;
  void* v = nullptr;
  float* k_scale = nullptr;
  float* v_scale = nullptr;
  int64_t num_pages = 0;
  int page_size = 0, kv_heads = 0, hd = 0;
  bool int8 = false;
};

struct QkRopeArgs {
  const __nv_bfloat16* x = nullptr;  // [T, ldx]: heads q | kv_heads k | v_heads v, hd columns each
  int64_t ldx = 0;
  __nv_bfloat16* out = nullptr;  // forward: [T, ldo] all of it; append: q only
  int64_t ldo = 0;
  const __nv_bfloat16* dy = nullptr;  // backward: gradient of `out`
  int64_t lddy = 0;
  const int32_t* pos = nullptr;  // [T]
  RopeTables rope;
  const float* gamma_q = nullptr;  // [hd], both or neither
  const float* gamma_k = nullptr;
  float eps = 1e-5f;
  int T = 0, heads = 0, kv_heads = 0, v_heads = 0, hd = 0;
  // append
  const int32_t* slots = nullptr;  // [T], -1: not cached
  KvPages cache;
  // backward
  float* dgamma_q = nullptr;
  float* dgamma_k = nullptr;
  int accumulate = 0;
  float* partials = nullptr;  // [2][qk_rope_bwd_blocks][hd]
  int* err = nullptr;
};
int qk_rope_fwd(const QkRopeArgs& a, cudaStream_t s);
int qk_rope_bwd(const QkRopeArgs& a, cudaStream_t s);
int qk_rope_bwd_blocks(int T, int heads, int kv_heads);
int kv_append(const QkRopeArgs& a, cudaStream_t s);
// k_out, v_out [T, ldo] bf16 = the cached tokens of `slots` (-1: zeros).
int kv_gather(const KvPages& c, const int32_t* slots, __nv_bfloat16* k_out, __nv_bfloat16* v_out, int64_t ldo, int T,
              int* err, cudaStream_t s);

struct PagedAttnArgs {
  const __nv_bfloat16* q = nullptr;  // [T, ldq]
  int64_t ldq = 0;
  __nv_bfloat16* out = nullptr;  // [T, ldo]
  int64_t ldo = 0;
  float* lse2 = nullptr;  // [T, heads] or null
  KvPages cache;
  const int32_t* table = nullptr;  // [nseq, table_cols] page numbers, rows table_ld apart
  int64_t table_ld = 0;
  int64_t table_cols = 0;  // entries of a row
  const int32_t* kv_lens = nullptr;  // [nseq]
  const int32_t* q_start = nullptr;  // [nseq + 1]
  int nseq = 0, T = 0, heads = 0;
  int max_q = 0, max_kv = 0;
  int window = 0;  // 0: none
  float scale = 0.f;
  void* workspace = nullptr;
  int64_t workspace_bytes = 0;
  int* err = nullptr;
};
int attn_paged(const PagedAttnArgs& a, cudaStream_t s);
int64_t attn_paged_workspace_bytes(int hd);

struct LogitsArgs {
  const float* logits = nullptr;  // [B, ldl]
  int64_t ldl = 0;
  float* out = nullptr;  // [B, ldo], may be `logits`
  int64_t ldo = 0;
  int32_t* token = nullptr;  // [B] or null
  int B = 0, V = 0;
  const int32_t* hist = nullptr;  // [n_hist], rows by hist_start: prompt tokens, then the answer's
  int64_t n_hist = 0;
  const int32_t* hist_start = nullptr;  // [B + 1]
  const int32_t* n_prompt = nullptr;    // [B]
  const float* repetition = nullptr;    // [B]
  const float* presence = nullptr;
  const float* frequency = nullptr;
  const int32_t* bias_ids = nullptr;
  const float* bias_vals = nullptr;
  const int32_t* bias_start = nullptr;  // [B + 1]
  int64_t n_bias = 0;
  const uint32_t* mask = nullptr;       // [B, mask_ld] words
  int64_t mask_ld = 0;
  int* err = nullptr;
};
bool kv_pages_ok(const KvPages& c);
int logits_adjust(const LogitsArgs& a, cudaStream_t s);

}  // namespace rt
