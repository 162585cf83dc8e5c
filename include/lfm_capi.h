/*
 * lfm_capi.h -- C-ABI of the decoder model around the MoE block (gfx950).
 *
 * The kernels of an LFM2-8B-A1B-style decoder layer other than the MoE FFN
 * (risepower20/final src/layer.cu:144-429, 1508-1922; src/model.cu:18-116,
 * 469-559), as plain-pointer entry points the C++ layer classes
 * (include/layer.h, include/model.h) call, plus a handle on the whole
 * one-GPU model for FFI callers.  Every call returns an int status of enum
 * moe_status (include/moe_capi.h; moe_strerror names it) and never exits the
 * process.  Device pointers, fp32 row-major, 16-byte aligned; every kernel
 * call is asynchronous on `stream` with no host synchronisation.
 *
 * What is kept from the reference and what is not: the arithmetic of its
 * kernels where it is defined for the shapes (RMSNorm reduction order, rotary
 * tables and rotation, the conv's FMA chain, the gather); the projections run
 * on MFMA tiles (fp32 accumulation in another order than the reference's FMA
 * chains: results agree within fp32 rounding, not bit for bit); attention is
 * an online-softmax form of the reference's (which holds at most 16
 * positions, layer.cu:312); the 24-stage 4-GPU pipeline, P2P copies, dual
 * streams and the fp16 cuBLAS LM head are not built (one GPU, one stream).
 */
#ifndef LFM_CAPI_H
#define LFM_CAPI_H

#include <stddef.h>
#include <stdint.h>

#include "moe_capi.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- kernels ------------------------------------------------------------ */

/* C[M][N] = A[M][K] . B[N][K]^T, plus R[M][N] when R != NULL (R may alias C).
 * Replaces attn_matmul_tiled_kernel (layer.cu:9-141: the q/k/v/o, in_proj
 * and out_proj projections, "A @ B^T" with B in PyTorch Linear [out][in]
 * layout) and lm_head_gemm_kernel (model.cu:42-116); R fuses the decoder's
 * residual add_kernel (layer.cu:1860-1880 as launched at 1912-1913).
 * N % 128 == 0, K % 32 == 0, M*K and M*N below 2^30 elements. */
int lfm_gemm_nt(const float *A, const float *B, float *C, const float *R, int M, int N, int K,
                moe_stream_t stream);

/* h[t][:] = table[ids[t]][:] for t < num_tokens: embedding_lookup_kernel
 * (model.cu:18-32).  table [vocab][hidden], hidden % 4 == 0.  An id outside
 * [0, vocab) gives a zero row and sets *bad_flag (device int, may be NULL) to
 * 1; the reference reads out of bounds there. */
int lfm_embed(const int *ids, const float *table, float *h, int num_tokens, int hidden,
              int vocab, int *bad_flag, moe_stream_t stream);

/* y = RMSNorm(x) * weight for `rows` rows of `dim`: rms_norm_kernel
 * (layer.cu:144-193) as RMSNorm::forward_gpu launches it (layer.cu:1144-1148),
 * bit for bit; row r of x starts at x + r*x_stride, of y at y + r*y_stride
 * (floats; strides let the model normalise only the last token of each
 * sequence, model.cu:486-501).  y may alias x. */
int lfm_rmsnorm(const float *x, long long x_stride, const float *weight, float *y,
                long long y_stride, int rows, int dim, moe_stream_t stream);

/* In place on qkv [batch*seq][ld]: the q heads (columns [0, heads*64)) and
 * the k heads (columns [k_col, k_col + kv_heads*64)) of every token are
 * RMS-normalised over their 64 values with q_weight / k_weight [64] (the
 * q_layernorm / k_layernorm of Attention::forward_gpu, layer.cu:1638-1642)
 * and rotated for position s = t % seq with cos/sin [>= seq][64]
 * (rope_transpose_kernel, layer.cu:195-231, without its transpose).
 * head_dim 64, heads + kv_heads <= 64; qkv, the weights and tables 16-byte
 * aligned, ld and k_col multiples of 4. */
int lfm_qk_norm_rope(float *qkv, int ld, const float *q_weight, const float *k_weight,
                     const float *cos_table, const float *sin_table, int batch, int seq,
                     int heads, int kv_heads, int k_col, moe_stream_t stream);

/* out[t][h*64 + d] = sum_j softmax_j(q_h(t) . k_g(j) / 8) v_g(j)[d] over the
 * keys j <= t of t's own sequence, g = h / (heads / kv_heads): the causal GQA
 * attention of fused_attn_gqa_kernel (layer.cu:262-354), for any seq.  q, k,
 * v are read from qkv [batch*seq][ld] at columns h*64, k_col + g*64 and
 * v_col + g*64.  head_dim 64, heads == 4 * kv_heads.  out [batch*seq][heads*64]. */
int lfm_attention(const float *qkv, int ld, float *out, int batch, int seq, int heads,
                  int kv_heads, int k_col, int v_col, moe_stream_t stream);

/* ShortConv's mix (conv_transpose_split_kernel, causal_conv1d_kernel and
 * conv_gating_transpose_kernel, layer.cu:360-429, token-major, bit for bit):
 * with B, C, g the column blocks [0,H), [H,2H), [2H,3H) of bcg
 * [batch*seq][3*hidden], y[t][h] = C[t][h] * sum_{k: s-L+1+k >= 0}
 * (B*g)[t-L+1+k][h] * conv_weight[h][k], s = t % seq, L = kernel.
 * y [batch*seq][hidden], hidden % 4 == 0, kernel <= 4 (the reference's is 3,
 * config.h:29). */
int lfm_shortconv(const float *bcg, const float *conv_weight, float *y, int batch, int seq,
                  int hidden, int kernel, moe_stream_t stream);

/* ---- serving: a paged KV cache, and sampling ---------------------------- */

/* How a cache holds keys and values, in rows of 64 (one token, one kv head):
 *   F32, BF16  the values, bf16 rounded to the nearest (halves to even);
 *   INT8       s = amax / 127 in fp32, then x / s to the nearest integer
 *              (halves to even), held to [-127, 127]; a value reads as q * s;
 *   FP8        s = the least power of two, 2^-126 at least, for which amax / s
 *              <= 448, then x / s to the nearest e4m3 value; reads as q * s.
 * amax is the row's largest magnitude; a row of zeros, or so small that INT8's
 * s is 0, reads as zeros.  An INT8 or FP8 row with an infinity or a NaN reads
 * as NaN throughout (s = NaN). */
enum lfm_kv_format { LFM_KV_F32 = 0, LFM_KV_BF16 = 1, LFM_KV_INT8 = 2, LFM_KV_FP8 = 3 };

/* The caller's cache buffers: k and v [num_pages][kv_heads][page_tokens][64] of
 * the format's type; k_scale and v_scale [num_pages][kv_heads][page_tokens] fp32
 * for INT8 and FP8, NULL for the others; all 16-byte aligned.  page_tokens is a
 * power of two, 16 to 4096.  Nothing has to be initialised. */
typedef struct lfm_kv_cache {
  int format;
  int kv_heads;
  int page_tokens;
  int num_pages;
  void *k, *v;
  float *k_scale, *v_scale;
} lfm_kv_cache;

/* The sequences of a call.  Every sequence may begin with the same `prefix_len`
 * positions, held in prefix_pages [ceil(prefix_len / page_tokens)]; its own
 * positions follow, own_len[b] of them, in the pages pages[b][0 .. max_pages).
 * The last n_b own positions are this call's new tokens: rows new_start[b] ..
 * new_start[b + 1] - 1 of the call's token tensors, or, where new_start is
 * NULL, rows b * max_new .. b * max_new + max_new - 1.  Pointers are device
 * memory; own_len, new_start and the tables are read when the kernels run, so a
 * captured graph follows their contents.
 *   tokens    rows of the token tensors (new_start NULL: batch * max_new);
 *   max_new   the most new tokens a sequence has;
 *   max_len   about the most own positions a sequence has: it decides how the
 *             work is split, not what is computed.
 * A sequence whose own_len is 0 takes no part (a slot of a padded batch): its
 * rows of an output stay as they were.  So does, and sets the call's *bad_flag
 * (device int, may be NULL) to 1, one whose contents do not fit: own_len below 0
 * or beyond max_pages * page_tokens; new_start that runs backwards, past
 * `tokens` or past max_new; more new tokens than own_len.  A page outside
 * [0, num_pages) sets the flag too: its positions are not written, read as
 * zeros and take no part in attention.  Pages may be shared for reading; a
 * position that two tokens of one call are written to holds either's values or
 * a mixture. */
typedef struct lfm_kv_batch {
  int batch;
  int tokens;
  int max_new;
  int max_len;
  const int *new_start;
  const int *own_len;
  const int *pages;
  int max_pages;
  const int *prefix_pages;
  int prefix_len;
} lfm_kv_batch;

/* Stores the new tokens' keys and values: columns k_col + g*64 and v_col + g*64
 * of qkv [tokens][ld], g < kv_heads, to the tokens' own positions.  (The shared
 * prefix is written as the own positions of a batch of one.)  With q_weight,
 * k_weight, cos_table and sin_table (all or none; `heads` and max_pos are used
 * only then) q and k are first normalised and rotated as lfm_qk_norm_rope does,
 * bit for bit, for position prefix_len + own position: q in place in columns
 * [0, heads*64), k on its way to the cache (qkv keeps its own).  A position of
 * max_pos, the tables' rows, or more sets *bad_flag and leaves the token out.
 * qkv 16-byte aligned, ld, k_col and v_col multiples of 4, heads*64 <= k_col,
 * k_col + kv_heads*64 <= v_col. */
int lfm_kv_write(const lfm_kv_cache *cache, const lfm_kv_batch *batch, float *qkv, int ld,
                 int heads, int k_col, int v_col, const float *q_weight, const float *k_weight,
                 const float *cos_table, const float *sin_table, int max_pos, int *bad_flag,
                 moe_stream_t stream);

/* Reads own positions back: row b * rows + p of k_out and v_out
 * [batch * rows][ld] (columns g*64) is position p of sequence b, for p <
 * min(own_len[b], rows); the other rows stay as they were (new_start,
 * tokens and max_new play no part).  Either output may be NULL.  ld a multiple
 * of 4, at least kv_heads * 64. */
int lfm_kv_read(const lfm_kv_cache *cache, const lfm_kv_batch *batch, float *k_out, float *v_out,
                int rows, int ld, int *bad_flag, moe_stream_t stream);

/* out[t][h*64 + d] = sum_j softmax_j(q_h(t) . k_g(j) / 8) v_g(j)[d] over the
 * prefix and the own positions j up to t's own, g = h / (heads / kv_heads): the
 * attention of lfm_attention for new tokens whose keys and values, their own
 * included, are in the cache.  q is read from columns [0, heads*64) of qkv
 * [tokens][ld], out has rows of ld_out.  heads a multiple of kv_heads, at most
 * 64 of them for each.  out does not overlap the columns that q is read from.  A
 * token that sees no position (its pages are outside the cache) gets zeros.  The
 * keys and values of a prefix that is long enough are read once for all sequences.
 * Sums, maxima and weights are fp32.  A key that is not finite makes the outputs of the tokens that see
 * it, for its heads, NaN, and a value that is not finite those of its column
 * not finite; what a token does not see does not reach it.
 * workspace: lfm_kv_attention_workspace bytes, 16-byte aligned (NULL where that
 * is 0), the caller's to keep from other calls until this one has run; it needs
 * no initial contents. */
int lfm_kv_attention(const lfm_kv_cache *cache, const lfm_kv_batch *batch, const float *qkv,
                     int ld, float *out, int ld_out, int heads, void *workspace,
                     size_t workspace_bytes, int *bad_flag, moe_stream_t stream);
/* Bytes for a call with these arguments (contents of device memory play no part). */
int lfm_kv_attention_workspace(const lfm_kv_cache *cache, const lfm_kv_batch *batch, int heads,
                               size_t *bytes);

/* y[r][i] = exp((x[r][i] - max x[r]) / temperature) / sum: probabilities of the
 * logits of `rows` rows of `dim`, row r at x + r*x_stride and y + r*y_stride
 * (floats).  A logit of -infinity gives 0, a row of nothing else zeros; NaN or
 * +infinity makes its row NaN.  temperature from 2^-120 to 2^120.  y may be
 * x (with equal strides); otherwise the two do not overlap.  workspace: lfm_softmax_workspace bytes, as for
 * lfm_kv_attention. */
int lfm_softmax(const float *x, long long x_stride, float *y, long long y_stride, int rows, int dim,
                float temperature, void *workspace, size_t workspace_bytes, moe_stream_t stream);
int lfm_softmax_workspace(int rows, int dim, size_t *bytes);

/* Verification of drafted tokens.  target [batch][n_draft + 1][vocab] holds the
 * target's probabilities after each draft (row 0: before the first), draft
 * [batch][n_draft][vocab] those that draft_ids (sequence b's at draft_ids + b *
 * ids_stride, ids_stride >= n_draft) were drawn from, u_accept [batch][n_draft]
 * and u_sample [batch] random numbers of [0, 1); n_valid [batch] how many drafts
 * a sequence has (NULL: n_draft for all; held to [0, n_draft]).  Draft i is
 * accepted if all before it were and u_accept * draft[i][id] < target[i][id].
 * Then one more token is drawn: after a rejected draft i from max(target[i] -
 * draft[i], 0), or from target[i] where that has no positive sum; after n_valid
 * accepted drafts from target[n_valid].  It is the lowest id up to which the
 * weights' sum exceeds u_sample times their whole sum, in 64 bits; -1 where no
 * weight is positive.  Weights that are NaN
 * or below 0 count as 0 (an infinite one leaves -1), and an id outside [0, vocab)
 * is rejected.
 * accepted [batch] = the number of accepted drafts; tokens [batch][n_draft + 1]
 * = these, the drawn token, then -1.  n_draft = 0 draws one token from target
 * (draft, draft_ids and u_accept may then be NULL).  n_draft at most 1024.
 * workspace: lfm_verify_draft_workspace bytes, as for lfm_kv_attention. */
int lfm_verify_draft(const float *target, const float *draft, const int *draft_ids,
                     long long ids_stride, const float *u_accept, const float *u_sample,
                     const int *n_valid, int batch, int n_draft, int vocab, int *accepted,
                     int *tokens, void *workspace, size_t workspace_bytes, moe_stream_t stream);
int lfm_verify_draft_workspace(int batch, int vocab, size_t *bytes);

/* Rotary tables [max_pos][head_dim] in host memory, computed as
 * RotaryEmbedding::init_gpu does (layer.cu:1167-1178): theta_j =
 * powf(theta, -2.0f*j/head_dim), angle = (float)i * theta_j, cos/sin of the
 * float angle (cosf/sinf) in columns j and j + head_dim/2. */
int lfm_rope_tables(float *cos_out, float *sin_out, int max_pos, int head_dim, float theta);

/* ---- synthetic weights (no counterpart in the reference) --------------- */

/* dst[i] = std * N(0,1) sample (first + i) of (seed, stream): the generator
 * of include/moe_synth.h evaluated on the device (dst is device memory). */
int lfm_synth_normal(float *dst, size_t n, uint64_t seed, uint64_t stream_id, float std_dev,
                     uint64_t first, moe_stream_t stream);
/* dst[i] = value for i < n (device memory). */
int lfm_fill(float *dst, size_t n, float value, moe_stream_t stream);
/* Stream id of a tensor name: FNV-1a 64 of its bytes. */
uint64_t lfm_synth_stream_of(const char *name);
/* 1 if a synthetic model fills this tensor with ones (RMSNorm weights: names
 * ending in "norm.weight"), else 0 (N(0, std)). */
int lfm_synth_is_norm(const char *name);
/* The synthetic tensor `name` of n elements as a synthetic model holds it
 * (ones, or N(0, std) from (seed, lfm_synth_stream_of(name))), copied to host
 * memory.  Drawn on the current device; synchronous. */
int lfm_synth_tensor(uint64_t seed, const char *name, float std_dev, float *host_out, size_t n);

/* ---- the model (wraps LFM2Model, include/model.h) ---------------------- */

typedef struct lfm_model lfm_model;

/* Synthetic model: every weight drawn on the device by name (matrices and
 * expert bias N(0, weight_std), RMSNorm weights 1), embedding tied to the LM
 * head.  layer_types[i]: 0 attention, 1 short conv (NULL = the reference's
 * LAYER_TYPES, config.h:31); layers below num_dense_layers get the dense
 * SwiGLU FFN, the rest the MoE block.  Scratch for max_batch*max_seq
 * tokens, shared by all layers. */
typedef struct lfm_model_config {
  int num_layers;
  const int *layer_types;
  int num_dense_layers;
  int max_batch;
  int max_seq;
  uint64_t seed;
  float weight_std;
} lfm_model_config;

int lfm_model_create_synthetic(const lfm_model_config *cfg, lfm_model **out);
/* The reference's LFM2Model(model_file) (model.cu:124-137): tensors by name
 * from a model.bin; scratch for max_batch*max_seq tokens. */
int lfm_model_create_from_file(const char *path, int max_batch, int max_seq, lfm_model **out);
int lfm_model_destroy(lfm_model *m);

/* Last-token logits [batch][vocab] of token ids [batch][seq] (device int32):
 * embedding, every decoder layer, final RMSNorm, LM head -- the work of
 * LFM2Model::worker_stage over all stages (model.cu:403-559) on one GPU and
 * one stream. */
int lfm_model_forward(lfm_model *m, const int *ids, int batch, int seq, float *logits,
                      moe_stream_t stream);
/* The same in pieces: embedding into h [batch*seq][hidden]; decoder layer
 * `layer` in place on h (DecoderLayer::forward_gpu, layer.cu:1882-1919);
 * final norm of each sequence's last token + LM head. */
int lfm_model_embed(lfm_model *m, const int *ids, int batch, int seq, float *h,
                    moe_stream_t stream);
int lfm_model_layer_forward(lfm_model *m, int layer, float *h, int batch, int seq,
                            moe_stream_t stream);
int lfm_model_head(lfm_model *m, const float *h, int batch, int seq, float *logits,
                   moe_stream_t stream);
/* Forward of ids [batch][seq] (device int32) whose last n_draft tokens are drafts
 * (0 <= n_draft < seq, at most 1024), then verification: probs [batch][n_draft + 1][vocab] gets
 * the softmax (lfm_softmax with `temperature`) of the logits from the position
 * before the first draft on, and accepted [batch] and tokens [batch][n_draft + 1]
 * what lfm_verify_draft says of them; draft, u_accept, u_sample and n_valid are its
 * arguments.  n_draft = 0 draws each sequence's next token. */
int lfm_model_verify(lfm_model *m, const int *ids, int batch, int seq, int n_draft,
                     const float *draft, const float *u_accept, const float *u_sample,
                     const int *n_valid, float temperature, float *probs, int *accepted,
                     int *tokens, moe_stream_t stream);
/* The MoE context of a layer (NULL for a dense layer): moe_last_routing on it
 * reads that layer's routing until the next MoE layer runs (all layers share
 * one scratch). */
int lfm_model_moe(lfm_model *m, int layer, moe_ctx **out);
/* Shape queries. */
int lfm_model_info(const lfm_model *m, int *num_layers, int *hidden, int *vocab, int *max_tokens);
/* MOE_OK, MOE_ERR_INVALID_ARG if an out-of-range token id was embedded since
 * the last call, or a MoE layer's device status.  Synchronises `stream`. */
int lfm_model_status(lfm_model *m, moe_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif
