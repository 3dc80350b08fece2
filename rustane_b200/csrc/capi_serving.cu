// C entry points of the serving operators: argument checks, then one launcher each.
#include <cmath>

#include "rustane_cuda.h"
#include "serving.h"

namespace {
inline int map_rc(int rc) { return rc == 0 ? RT_OK : (rc == -1 ? RT_ERR_SHAPE : RT_ERR_CUDA); }
inline cudaStream_t st(void* s) { return static_cast<cudaStream_t>(s); }
inline const __nv_bfloat16* cb(const void* p) { return static_cast<const __nv_bfloat16*>(p); }
inline __nv_bfloat16* mb(void* p) { return static_cast<__nv_bfloat16*>(p); }

rt::RopeTables tables(const rt_rope* r) { return {r->cos, r->sin, r->n_pos, r->rot, r->half != 0}; }
rt::KvPages pages(const rt_kv_pages* c) {
  return {c->k, c->v, c->k_scale, c->v_scale, c->num_pages, c->page_size, c->kv_heads, c->hd, c->int8_rows != 0};
}
bool rope_given(const rt_rope* r) { return r && r->cos && r->sin; }
bool pages_given(const rt_kv_pages* c) {
  return c && c->k && c->v && (!c->int8_rows || (c->k_scale && c->v_scale));
}
}  // namespace

extern "C" {

RT_API int rt_rope_tables(float* cos_out, float* sin_out, int n_pos, int rot, double theta, int scaling, double factor,
                          double low, double high, int trained_pos) {
  if (!cos_out || !sin_out) return RT_ERR_ARG;
  if (n_pos <= 0 || rot <= 0 || rot % 2 || !(theta > 0.0)) return RT_ERR_SHAPE;
  if (scaling != RT_ROPE_PLAIN && scaling != RT_ROPE_LINEAR && scaling != RT_ROPE_BANDS) return RT_ERR_ARG;
  if (scaling != RT_ROPE_PLAIN && !(factor > 0.0)) return RT_ERR_ARG;
  if (scaling == RT_ROPE_BANDS && (!(low > 0.0) || !(high > low) || trained_pos <= 0)) return RT_ERR_ARG;
  const double two_pi = 6.283185307179586476925286766559;
  const int pairs = rot / 2;
  for (int i = 0; i < pairs; ++i) {
    double f = std::pow(theta, -2.0 * i / rot);
    if (scaling == RT_ROPE_LINEAR) f /= factor;
    if (scaling == RT_ROPE_BANDS) {
      const double turns = trained_pos * f / two_pi;  // of this pair over the trained positions
      double keep = (turns - low) / (high - low);
      keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
      f *= keep + (1.0 - keep) / factor;
    }
    for (int p = 0; p < n_pos; ++p) {
      const double a = f * p;
      cos_out[static_cast<int64_t>(p) * pairs + i] = static_cast<float>(std::cos(a));
      sin_out[static_cast<int64_t>(p) * pairs + i] = static_cast<float>(std::sin(a));
    }
  }
  return RT_OK;
}

RT_API int rt_kernel_qk_norm_rope_fwd(const void* x, int64_t ldx, void* out, int64_t ldo, const int32_t* pos,
                                      const rt_rope* rope, const float* gamma_q, const float* gamma_k, float eps, int T,
                                      int heads, int kv_heads, int v_heads, int hd, int* dev_err, void* stream) {
  if (!rope_given(rope) || (T > 0 && (!x || !out || !pos))) return RT_ERR_ARG;
  rt::QkRopeArgs a;
  a.x = cb(x);
  a.ldx = ldx;
  a.out = mb(out);
  a.ldo = ldo;
  a.pos = pos;
  a.rope = tables(rope);
  a.gamma_q = gamma_q;
  a.gamma_k = gamma_k;
  a.eps = eps;
  a.T = T;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.v_heads = v_heads;
  a.hd = hd;
  a.err = dev_err;
  return map_rc(rt::qk_rope_fwd(a, st(stream)));
}

RT_API int rt_kernel_qk_norm_rope_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, void* dx, int64_t lddx,
                                      const int32_t* pos, const rt_rope* rope, const float* gamma_q,
                                      const float* gamma_k, float eps, float* dgamma_q, float* dgamma_k, int accumulate,
                                      float* partials, int T, int heads, int kv_heads, int v_heads, int hd, int* dev_err,
                                      void* stream) {
  if (!rope_given(rope) || (T > 0 && (!dy || !dx || !pos))) return RT_ERR_ARG;
  if (gamma_q && ((T > 0 && !x) || !dgamma_q || !dgamma_k || !partials)) return RT_ERR_ARG;
  rt::QkRopeArgs a;
  a.dy = cb(dy);
  a.lddy = lddy;
  a.x = cb(x);
  a.ldx = ldx;
  a.out = mb(dx);
  a.ldo = lddx;
  a.pos = pos;
  a.rope = tables(rope);
  a.gamma_q = gamma_q;
  a.gamma_k = gamma_k;
  a.eps = eps;
  a.dgamma_q = dgamma_q;
  a.dgamma_k = dgamma_k;
  a.accumulate = accumulate;
  a.partials = partials;
  a.T = T;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.v_heads = v_heads;
  a.hd = hd;
  a.err = dev_err;
  return map_rc(rt::qk_rope_bwd(a, st(stream)));
}

RT_API int rt_kernel_qk_norm_rope_bwd_partials(int T, int heads, int kv_heads) {
  return 2 * rt::qk_rope_bwd_blocks(T, heads, kv_heads);
}

RT_API int rt_kernel_kv_append(const void* qkv, int64_t ldqkv, void* q_out, int64_t ldq, const int32_t* pos,
                               const int32_t* slots, const rt_rope* rope, const float* gamma_q, const float* gamma_k,
                               float eps, const rt_kv_pages* cache, int T, int heads, int* dev_err, void* stream) {
  if (!rope_given(rope) || !pages_given(cache) || (T > 0 && (!qkv || !q_out || !pos || !slots))) return RT_ERR_ARG;
  rt::QkRopeArgs a;
  a.x = cb(qkv);
  a.ldx = ldqkv;
  a.out = mb(q_out);
  a.ldo = ldq;
  a.pos = pos;
  a.slots = slots;
  a.rope = tables(rope);
  a.gamma_q = gamma_q;
  a.gamma_k = gamma_k;
  a.eps = eps;
  a.cache = pages(cache);
  a.T = T;
  a.heads = heads;
  a.err = dev_err;
  return map_rc(rt::kv_append(a, st(stream)));
}

RT_API int rt_kernel_kv_gather(const rt_kv_pages* cache, const int32_t* slots, void* k_out, void* v_out, int64_t ldo,
                               int T, int* dev_err, void* stream) {
  if (!pages_given(cache) || (T > 0 && (!slots || !k_out || !v_out))) return RT_ERR_ARG;
  return map_rc(rt::kv_gather(pages(cache), slots, mb(k_out), mb(v_out), ldo, T, dev_err, st(stream)));
}

RT_API int64_t rt_kernel_attention_paged_workspace_bytes(int hd) { return rt::attn_paged_workspace_bytes(hd); }

RT_API int rt_kernel_attention_paged_cols(const void* q, int64_t ldq, void* out, int64_t ldo, float* lse2,
                                          const rt_kv_pages* cache, const int32_t* page_table, int64_t table_ld,
                                          int64_t table_cols, const int32_t* kv_lens, const int32_t* q_start, int nseq,
                                          int T, int max_q, int max_kv, int heads, int window, float scale,
                                          void* workspace, int64_t workspace_bytes, int* dev_err, void* stream) {
  if (!pages_given(cache) || !workspace) return RT_ERR_ARG;
  if (T > 0 && nseq > 0 && (!q || !out || !page_table || !kv_lens || !q_start)) return RT_ERR_ARG;
  rt::PagedAttnArgs a;
  a.q = cb(q);
  a.ldq = ldq;
  a.out = mb(out);
  a.ldo = ldo;
  a.lse2 = lse2;
  a.cache = pages(cache);
  a.table = page_table;
  a.table_ld = table_ld;
  a.table_cols = table_cols;
  a.kv_lens = kv_lens;
  a.q_start = q_start;
  a.nseq = nseq;
  a.T = T;
  a.max_q = max_q;
  a.max_kv = max_kv;
  a.heads = heads;
  a.window = window;
  a.scale = scale;
  a.workspace = workspace;
  a.workspace_bytes = workspace_bytes;
  a.err = dev_err;
  return map_rc(rt::attn_paged(a, st(stream)));
}

RT_API int rt_kernel_attention_paged(const void* q, int64_t ldq, void* out, int64_t ldo, float* lse2,
                                     const rt_kv_pages* cache, const int32_t* page_table, int64_t table_ld,
                                     const int32_t* kv_lens, const int32_t* q_start, int nseq, int T, int max_q,
                                     int max_kv, int heads, int window, float scale, void* workspace,
                                     int64_t workspace_bytes, int* dev_err, void* stream) {
  return rt_kernel_attention_paged_cols(q, ldq, out, ldo, lse2, cache, page_table, table_ld, table_ld, kv_lens, q_start,
                                        nseq, T, max_q, max_kv, heads, window, scale, workspace, workspace_bytes,
                                        dev_err, stream);
}

RT_API int rt_kernel_logits_adjust(const float* logits, int64_t ldl, float* out, int64_t ldo, int32_t* token, int B,
                                   int V, const rt_logit_rules* rules, int* dev_err, void* stream) {
  if (!rules || (B > 0 && (!logits || !out))) return RT_ERR_ARG;
  if (rules->hist && !rules->hist_start) return RT_ERR_ARG;
  if (rules->bias_ids && (!rules->bias_start || !rules->bias_vals)) return RT_ERR_ARG;
  if (rules->n_hist < 0 || rules->n_bias < 0) return RT_ERR_ARG;
  rt::LogitsArgs a;
  a.logits = logits;
  a.ldl = ldl;
  a.out = out;
  a.ldo = ldo;
  a.token = token;
  a.B = B;
  a.V = V;
  a.hist = rules->hist;
  a.n_hist = rules->n_hist;
  a.hist_start = rules->hist_start;
  a.n_prompt = rules->n_prompt;
  a.repetition = rules->repetition;
  a.presence = rules->presence;
  a.frequency = rules->frequency;
  a.bias_ids = rules->bias_ids;
  a.bias_vals = rules->bias_vals;
  a.bias_start = rules->bias_start;
  a.n_bias = rules->n_bias;
  a.mask = rules->mask;
  a.mask_ld = rules->mask_ld;
  a.err = dev_err;
  return map_rc(rt::logits_adjust(a, st(stream)));
}

}  // extern "C"
