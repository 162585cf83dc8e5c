// C-ABI of the decoder-model kernels (include/lfm_capi.h): argument checks
// and launches on the caller's stream, no host synchronisation.  Host-only
// helpers (rotary tables, synthetic tensor names) are in lfm_host.cpp; the
// model handle (lfm_model_*) wraps LFM2Model in model.cpp.
#include "lfm_capi.h"

#include <stdint.h>

#include "lfm_internal.h"

namespace {

bool al16(const void *p) { return ((uintptr_t)p & 15u) == 0; }

int launch_status(hipError_t e) {
  if (e == hipSuccess) return MOE_OK;
  (void)hipGetLastError();
  return e == hipErrorInvalidValue ? MOE_ERR_UNSUPPORTED : MOE_ERR_HIP;
}

hipStream_t S(moe_stream_t s) { return static_cast<hipStream_t>(s); }

// Checks a cache and a batch and writes them into `a`.  Tables that a call does
// not read may be NULL: new tokens with NEW false.
int kv_args(const lfm_kv_cache *c, const lfm_kv_batch *b, int *bad, lfm::KvArgs *a) {
  if (!c || !b) return MOE_ERR_INVALID_ARG;
  if (c->kv_heads <= 0 || c->num_pages <= 0 || c->page_tokens <= 0) return MOE_ERR_INVALID_ARG;
  if (c->format < LFM_KV_F32 || c->format > LFM_KV_FP8) return MOE_ERR_UNSUPPORTED;
  if (c->page_tokens < 16 || c->page_tokens > 4096 || (c->page_tokens & (c->page_tokens - 1)) != 0)
    return MOE_ERR_UNSUPPORTED;
  if (c->kv_heads > 256) return MOE_ERR_UNSUPPORTED;
  if (!c->k || !c->v || !al16(c->k) || !al16(c->v)) return MOE_ERR_INVALID_ARG;
  const bool scaled = c->format == LFM_KV_INT8 || c->format == LFM_KV_FP8;
  if (scaled != (c->k_scale != nullptr) || scaled != (c->v_scale != nullptr) || !al16(c->k_scale) ||
      !al16(c->v_scale))
    return MOE_ERR_INVALID_ARG;
  if (b->batch < 0 || b->tokens < 0 || b->max_new < 0 || b->max_len < 0 || b->max_pages < 0 ||
      b->prefix_len < 0)
    return MOE_ERR_INVALID_ARG;
  if (!b->new_start && (long long)b->batch * b->max_new != b->tokens) return MOE_ERR_INVALID_ARG;
  if (b->batch > 65535) return MOE_ERR_UNSUPPORTED;
  if (b->batch > 0 && (!b->own_len || (b->max_pages > 0 && !b->pages))) return MOE_ERR_INVALID_ARG;
  if (b->prefix_len > 0 && !b->prefix_pages) return MOE_ERR_INVALID_ARG;
  // positions, absolute ones too, are ints
  if (((long long)b->max_pages * c->page_tokens + b->prefix_len) >> 30) return MOE_ERR_UNSUPPORTED;
  int shift = 0;
  while ((1 << shift) < c->page_tokens) ++shift;
  *a = lfm::KvArgs{static_cast<char *>(c->k), static_cast<char *>(c->v), c->k_scale, c->v_scale,
                   b->new_start, b->own_len, b->pages, b->prefix_pages, bad, c->format, c->kv_heads,
                   shift, c->num_pages, b->batch, b->tokens, b->max_new, b->max_len, b->max_pages,
                   b->prefix_len};
  return MOE_OK;
}

int kv_heads_ok(const lfm::KvArgs &a, int heads) {
  if (heads <= 0 || heads % a.kv_heads != 0) return MOE_ERR_INVALID_ARG;
  if (heads / a.kv_heads > 64 || (long long)a.max_new * heads >> 24 || (long long)a.tokens * heads >> 30)
    return MOE_ERR_UNSUPPORTED;
  return MOE_OK;
}

}  // namespace

extern "C" {

int lfm_gemm_nt(const float *A, const float *B, float *C, const float *R, int M, int N, int K,
                moe_stream_t stream) {
  if (M < 0 || N <= 0 || K <= 0) return MOE_ERR_INVALID_ARG;
  if (M == 0) return MOE_OK;
  if (!A || !B || !C || !al16(A) || !al16(B) || !al16(C) || (R && !al16(R)))
    return MOE_ERR_INVALID_ARG;
  if (C == A || C == B) return MOE_ERR_INVALID_ARG;  // tiles read A/B while others write C
  if (N % 128 != 0 || K % 32 != 0) return MOE_ERR_UNSUPPORTED;
  if ((size_t)M * K >= ((size_t)1 << 30) || (size_t)M * N >= ((size_t)1 << 30))
    return MOE_ERR_UNSUPPORTED;
  return launch_status(lfm::launch_gemm_nt(A, B, C, R, M, N, K, S(stream)));
}

int lfm_embed(const int *ids, const float *table, float *h, int num_tokens, int hidden, int vocab,
              int *bad_flag, moe_stream_t stream) {
  if (num_tokens < 0 || hidden <= 0 || vocab <= 0) return MOE_ERR_INVALID_ARG;
  if (num_tokens == 0) return MOE_OK;
  if (!ids || !table || !h || !al16(table) || !al16(h)) return MOE_ERR_INVALID_ARG;
  if (hidden % 4 != 0) return MOE_ERR_UNSUPPORTED;
  return launch_status(lfm::launch_embed(ids, table, h, num_tokens, hidden, vocab, bad_flag,
                                         S(stream)));
}

int lfm_rmsnorm(const float *x, long long x_stride, const float *weight, float *y,
                long long y_stride, int rows, int dim, moe_stream_t stream) {
  if (rows < 0 || dim <= 0 || x_stride < dim || y_stride < dim) return MOE_ERR_INVALID_ARG;
  if (rows == 0) return MOE_OK;
  if (!x || !weight || !y) return MOE_ERR_INVALID_ARG;
  return launch_status(
      lfm::launch_rmsnorm_rows(x, x_stride, weight, y, y_stride, rows, dim, S(stream)));
}

int lfm_qk_norm_rope(float *qkv, int ld, const float *q_weight, const float *k_weight,
                     const float *cos_table, const float *sin_table, int batch, int seq,
                     int heads, int kv_heads, int k_col, moe_stream_t stream) {
  if (batch < 0 || seq < 0 || heads <= 0 || kv_heads <= 0) return MOE_ERR_INVALID_ARG;
  if (batch == 0 || seq == 0) return MOE_OK;
  if (!qkv || !q_weight || !k_weight || !cos_table || !sin_table) return MOE_ERR_INVALID_ARG;
  if (!al16(qkv) || !al16(q_weight) || !al16(k_weight) || !al16(cos_table) || !al16(sin_table) ||
      ld % 4 != 0 || k_col % 4 != 0)
    return MOE_ERR_INVALID_ARG;
  if (k_col < heads * 64 || ld < k_col + kv_heads * 64) return MOE_ERR_INVALID_ARG;
  if (heads + kv_heads > 64) return MOE_ERR_UNSUPPORTED;
  return launch_status(lfm::launch_qk_norm_rope(qkv, ld, q_weight, k_weight, cos_table, sin_table,
                                                batch, seq, heads, kv_heads, k_col, S(stream)));
}

int lfm_attention(const float *qkv, int ld, float *out, int batch, int seq, int heads,
                  int kv_heads, int k_col, int v_col, moe_stream_t stream) {
  if (batch < 0 || seq < 0 || heads <= 0 || kv_heads <= 0) return MOE_ERR_INVALID_ARG;
  if (batch == 0 || seq == 0) return MOE_OK;
  if (!qkv || !out || !al16(qkv) || !al16(out) || ld % 4 != 0) return MOE_ERR_INVALID_ARG;
  if (k_col < heads * 64 || v_col < k_col + kv_heads * 64 || ld < v_col + kv_heads * 64 ||
      k_col % 4 != 0 || v_col % 4 != 0)
    return MOE_ERR_INVALID_ARG;
  if (heads != 4 * kv_heads) return MOE_ERR_UNSUPPORTED;
  if ((const void *)out == (const void *)qkv) return MOE_ERR_INVALID_ARG;
  return launch_status(
      lfm::launch_attention(qkv, ld, out, batch, seq, heads, kv_heads, k_col, v_col, S(stream)));
}

int lfm_shortconv(const float *bcg, const float *conv_weight, float *y, int batch, int seq,
                  int hidden, int kernel, moe_stream_t stream) {
  if (batch < 0 || seq < 0 || hidden <= 0 || kernel <= 0) return MOE_ERR_INVALID_ARG;
  if (batch == 0 || seq == 0) return MOE_OK;
  if (!bcg || !conv_weight || !y || !al16(bcg) || !al16(y)) return MOE_ERR_INVALID_ARG;
  if ((const void *)y == (const void *)bcg) return MOE_ERR_INVALID_ARG;
  if (hidden % 4 != 0) return MOE_ERR_UNSUPPORTED;
  return launch_status(
      lfm::launch_shortconv(bcg, conv_weight, y, batch, seq, hidden, kernel, S(stream)));
}

int lfm_kv_write(const lfm_kv_cache *cache, const lfm_kv_batch *batch, float *qkv, int ld,
                 int heads, int k_col, int v_col, const float *q_weight, const float *k_weight,
                 const float *cos_table, const float *sin_table, int max_pos, int *bad_flag,
                 moe_stream_t stream) {
  lfm::KvArgs a;
  const int rc = kv_args(cache, batch, bad_flag, &a);
  if (rc != MOE_OK) return rc;
  const int given = (q_weight != nullptr) + (k_weight != nullptr) + (cos_table != nullptr) +
                    (sin_table != nullptr);
  if (given != 0 && given != 4) return MOE_ERR_INVALID_ARG;
  if (k_col < 0 || v_col < k_col || v_col - k_col < a.kv_heads * 64 || ld < v_col ||
      ld - v_col < a.kv_heads * 64 || ld % 4 != 0 || k_col % 4 != 0 || v_col % 4 != 0)
    return MOE_ERR_INVALID_ARG;
  if (given && (heads <= 0 || heads > k_col / 64 || max_pos <= 0 || !al16(q_weight) ||
                !al16(k_weight) || !al16(cos_table) || !al16(sin_table)))
    return MOE_ERR_INVALID_ARG;
  if (a.batch == 0 || a.max_new == 0 || a.tokens == 0) return MOE_OK;
  if (!qkv || !al16(qkv)) return MOE_ERR_INVALID_ARG;
  // rows of a sequence are counted in an int
  if ((long long)a.max_new * ((given ? heads : 0) + 2 * a.kv_heads) >> 30) return MOE_ERR_UNSUPPORTED;
  return launch_status(lfm::launch_kv_write(
      a, lfm::KvWriteArgs{qkv, q_weight, k_weight, cos_table, sin_table, ld, heads, k_col, v_col, max_pos},
      S(stream)));
}

int lfm_kv_read(const lfm_kv_cache *cache, const lfm_kv_batch *batch, float *k_out, float *v_out,
                int rows, int ld, int *bad_flag, moe_stream_t stream) {
  lfm::KvArgs a;
  const int rc = kv_args(cache, batch, bad_flag, &a);
  if (rc != MOE_OK) return rc;
  if (rows < 0 || ld < a.kv_heads * 64 || ld % 4 != 0) return MOE_ERR_INVALID_ARG;
  if ((k_out && !al16(k_out)) || (v_out && !al16(v_out)) || (k_out && k_out == v_out))
    return MOE_ERR_INVALID_ARG;
  if (a.batch == 0 || rows == 0 || (!k_out && !v_out)) return MOE_OK;
  if ((long long)rows * 2 * a.kv_heads >> 30) return MOE_ERR_UNSUPPORTED;
  return launch_status(lfm::launch_kv_read(a, k_out, v_out, rows, ld, S(stream)));
}

int lfm_kv_attention_workspace(const lfm_kv_cache *cache, const lfm_kv_batch *batch, int heads,
                               size_t *bytes) {
  lfm::KvArgs a;
  if (!bytes) return MOE_ERR_INVALID_ARG;
  *bytes = 0;
  int rc = kv_args(cache, batch, nullptr, &a);
  if (rc == MOE_OK) rc = kv_heads_ok(a, heads);
  if (rc == MOE_OK) *bytes = lfm::kv_attention_ws(a, heads);
  return rc;
}

int lfm_kv_attention(const lfm_kv_cache *cache, const lfm_kv_batch *batch, const float *qkv,
                     int ld, float *out, int ld_out, int heads, void *workspace,
                     size_t workspace_bytes, int *bad_flag, moe_stream_t stream) {
  lfm::KvArgs a;
  int rc = kv_args(cache, batch, bad_flag, &a);
  if (rc == MOE_OK) rc = kv_heads_ok(a, heads);
  if (rc != MOE_OK) return rc;
  if (ld < heads * 64 || ld % 4 != 0 || ld_out < heads * 64 || ld_out % 4 != 0)
    return MOE_ERR_INVALID_ARG;
  if (a.batch == 0 || a.max_new == 0 || a.tokens == 0) return MOE_OK;
  if (!qkv || !out || !al16(qkv) || !al16(out) || (const float *)out == qkv)
    return MOE_ERR_INVALID_ARG;
  const size_t need = lfm::kv_attention_ws(a, heads);
  if (need && (!workspace || !al16(workspace) || workspace_bytes < need)) return MOE_ERR_INVALID_ARG;
  return launch_status(
      lfm::launch_kv_attention(a, qkv, ld, out, ld_out, heads, workspace, S(stream)));
}

int lfm_softmax_workspace(int rows, int dim, size_t *bytes) {
  if (!bytes) return MOE_ERR_INVALID_ARG;
  *bytes = 0;
  if (rows < 0 || dim <= 0) return MOE_ERR_INVALID_ARG;
  *bytes = lfm::softmax_ws(rows, dim);
  return MOE_OK;
}

int lfm_softmax(const float *x, long long x_stride, float *y, long long y_stride, int rows, int dim,
                float temperature, void *workspace, size_t workspace_bytes, moe_stream_t stream) {
  if (rows < 0 || dim <= 0 || x_stride < dim || y_stride < dim) return MOE_ERR_INVALID_ARG;
  // 1 / temperature is finite and not 0 (this refuses NaN as well)
  if (!(temperature >= 0x1p-120f && temperature <= 0x1p120f)) return MOE_ERR_INVALID_ARG;
  if (rows == 0) return MOE_OK;
  if (!x || !y || ((uintptr_t)x & 3u) != 0 || ((uintptr_t)y & 3u) != 0) return MOE_ERR_INVALID_ARG;
  if (x == y && x_stride != y_stride) return MOE_ERR_INVALID_ARG;
  const size_t need = lfm::softmax_ws(rows, dim);
  if (need && (!workspace || !al16(workspace) || workspace_bytes < need)) return MOE_ERR_INVALID_ARG;
  return launch_status(lfm::launch_softmax(x, x_stride, y, y_stride, rows, dim, temperature,
                                           workspace, S(stream)));
}

int lfm_verify_draft_workspace(int batch, int vocab, size_t *bytes) {
  if (!bytes) return MOE_ERR_INVALID_ARG;
  *bytes = 0;
  if (batch < 0 || vocab <= 0) return MOE_ERR_INVALID_ARG;
  *bytes = lfm::verify_draft_ws(batch, vocab);
  return MOE_OK;
}

int lfm_verify_draft(const float *target, const float *draft, const int *draft_ids,
                     long long ids_stride, const float *u_accept, const float *u_sample,
                     const int *n_valid, int batch, int n_draft, int vocab, int *accepted,
                     int *tokens, void *workspace, size_t workspace_bytes, moe_stream_t stream) {
  if (batch < 0 || n_draft < 0 || vocab <= 0) return MOE_ERR_INVALID_ARG;
  if (batch == 0) return MOE_OK;
  if (batch > 65535 || n_draft > 1024) return MOE_ERR_UNSUPPORTED;
  if (!target || !u_sample || !accepted || !tokens) return MOE_ERR_INVALID_ARG;
  if (n_draft > 0 && (!draft || !draft_ids || !u_accept || ids_stride < n_draft))
    return MOE_ERR_INVALID_ARG;
  const size_t need = lfm::verify_draft_ws(batch, vocab);
  if (need && (!workspace || !al16(workspace) || workspace_bytes < need)) return MOE_ERR_INVALID_ARG;
  return launch_status(lfm::launch_verify_draft(
      lfm::VerifyArgs{target, draft, draft_ids, u_accept, u_sample, n_valid, accepted, tokens, batch,
                      n_draft, vocab, ids_stride},
      workspace, S(stream)));
}

int lfm_synth_normal(float *dst, size_t n, uint64_t seed, uint64_t stream_id, float std_dev,
                     uint64_t first, moe_stream_t stream) {
  if (n == 0) return MOE_OK;
  if (!dst) return MOE_ERR_INVALID_ARG;
  return launch_status(lfm::launch_synth_normal(dst, n, seed, stream_id, std_dev, first, S(stream)));
}

int lfm_fill(float *dst, size_t n, float value, moe_stream_t stream) {
  if (n == 0) return MOE_OK;
  if (!dst) return MOE_ERR_INVALID_ARG;
  return launch_status(lfm::launch_fill(dst, n, value, S(stream)));
}

}  // extern "C"
