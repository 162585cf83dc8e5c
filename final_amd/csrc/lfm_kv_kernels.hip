// HIP kernels of the paged KV cache (gfx950): rows written as they are
// quantised (with the q/k norm and rotation in front where asked for), rows
// read back, and attention of new tokens over a shared prefix and their own
// pages.
#include <algorithm>

#include "lfm_kv.h"
#include "lfm_rope.h"

namespace lfm {

// ---------------------------------------------------------------------------
// Rows into the cache, and back
// ---------------------------------------------------------------------------

// 16 lanes take a row of 64 (a token's q, k or v head), four floats each, R rows
// one after the other with their loads in flight together; block (x, sequence).
template <int FMT, bool ROPE, int R>
__global__ __launch_bounds__(256) void kv_write_kernel(KvArgs a, KvWriteArgs w) {
  KvSeq s;
  if (!kv_seq<true>(a, blockIdx.y, s)) return;
  const int qrows = ROPE ? w.heads : 0, per_tok = qrows + 2 * a.kv_heads, total = s.n * per_tok;
  const int first = blockIdx.x * 16 * R;
  if (first >= total) return;
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
  f32x4 x[R];
  int tok[R], row[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int f = first + 16 * j + g;
    tok[j] = f / per_tok;
    row[j] = f - tok[j] * per_tok;
    const int col = row[j] < qrows ? row[j] * kRowDim
                    : row[j] < qrows + a.kv_heads ? w.k_col + (row[j] - qrows) * kRowDim
                                                  : w.v_col + (row[j] - qrows - a.kv_heads) * kRowDim;
    x[j] = f < total ? moe::ld4(w.qkv + (size_t)(s.row0 + tok[j]) * w.ld + col + 4 * c)
                     : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
#pragma unroll
  for (int j = 0; j < R; ++j) {
    bool ok = first + 16 * j + g < total;
    const int pos = s.len - s.n + tok[j];
    const bool is_q = row[j] < qrows, is_v = row[j] >= qrows + a.kv_heads;
    if (ROPE) {
      const int at = a.prefix_len + pos;
      if (ok && at >= w.max_pos) {
        kv_flag(a.bad);
        ok = false;
      }
      const size_t t = (size_t)(ok ? at : 0) * kRowDim + 4 * c;
      const f32x4 y = norm_rope_row(x[j], moe::ld4((is_q ? w.q_weight : w.k_weight) + 4 * c),
                                    moe::ld4(w.cos_t + t), moe::ld4(w.sin_t + t));
      if (!is_v) x[j] = y;
      if (ok && is_q) moe::st4(w.qkv + (size_t)(s.row0 + tok[j]) * w.ld + row[j] * kRowDim + 4 * c, y);
    }
    const int h = row[j] - qrows - (is_v ? a.kv_heads : 0);
    ok = ok && !is_q;
    const int page = ok ? a.pages[(size_t)blockIdx.y * a.max_pages + (pos >> a.pshift)] : 0;
    if (page < 0 || page >= a.num_pages) {
      kv_flag(a.bad);
      ok = false;
    }
    const size_t at = ok ? kv_row(a, page, h, pos & ((1 << a.pshift) - 1)) : 0;
    kv_store_row<FMT>(is_v ? a.v : a.k, is_v ? a.vs : a.ks, at, c, x[j], ok);
  }
}

template <int FMT, int R>
__global__ __launch_bounds__(256) void kv_read_kernel(KvArgs a, float *k_out, float *v_out, int rows, int ld) {
  KvSeq s;
  if (!kv_seq<false>(a, blockIdx.y, s)) return;
  const int kinds = (k_out != nullptr) + (v_out != nullptr), per_pos = kinds * a.kv_heads;
  const int total = min(s.len, rows) * per_pos, first = blockIdx.x * 16 * R;
  if (first >= total) return;
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
  f32x4 x[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int f = first + 16 * j + g, pos = f / per_pos, row = f - pos * per_pos;
    x[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (f >= total) continue;
    const bool is_v = !k_out || row >= a.kv_heads;
    const int page = a.pages[(size_t)blockIdx.y * a.max_pages + (pos >> a.pshift)];
    if (page < 0 || page >= a.num_pages) {
      kv_flag(a.bad);
      continue;
    }
    const size_t at = kv_row(a, page, row >= a.kv_heads ? row - a.kv_heads : row, pos & ((1 << a.pshift) - 1));
    x[j] = kv_load_row<FMT>(is_v ? a.v : a.k, is_v ? a.vs : a.ks, at, c);
  }
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int f = first + 16 * j + g, pos = f / per_pos, row = f - pos * per_pos;
    if (f >= total) continue;
    const bool is_v = !k_out || row >= a.kv_heads;
    float *o = is_v ? v_out : k_out;
    moe::st4(o + ((size_t)blockIdx.y * rows + pos) * ld + (row >= a.kv_heads ? row - a.kv_heads : row) * kRowDim +
                 4 * c, x[j]);
  }
}

// ---------------------------------------------------------------------------
// Attention over the cache
// ---------------------------------------------------------------------------

// One wave per (new token, query head): 64 positions at a time, a lane's
// position for the scores, a lane's column for the values.
template <int FMT>
__global__ __launch_bounds__(64) void kv_attention_kernel(KvArgs a, const float *q, int ld, float *out,
                                                          int ldo, int heads) {
  KvSeq s;
  if (!kv_seq<true>(a, blockIdx.y, s)) return;
  const int i = blockIdx.x / heads, h = blockIdx.x - i * heads;
  if (i >= s.n) return;
  const int lane = threadIdx.x, g = h / (heads / a.kv_heads);
  const int end = a.prefix_len + s.len - s.n + i + 1;
  const float *qr = q + (size_t)(s.row0 + i) * ld + h * kRowDim;
  float m = -__builtin_inff(), l = 0.0f, o = 0.0f;
  for (int j0 = 0; j0 < end; j0 += 64) {
    const int j = j0 + lane, p = j < a.prefix_len ? j : j - a.prefix_len;
    int page = -1;
    if (j < end) {
      page = j < a.prefix_len ? a.prefix_pages[p >> a.pshift]
                              : a.pages[(size_t)blockIdx.y * a.max_pages + (p >> a.pshift)];
      if (page < 0 || page >= a.num_pages) {
        kv_flag(a.bad);
        page = -1;
      }
    }
    const size_t row = page >= 0 ? kv_row(a, page, g, p & ((1 << a.pshift) - 1)) : 0;
    float sc = -__builtin_inff();
    if (page >= 0) {
      sc = 0.0f;
      for (int c = 0; c < 16; ++c) {
        const f32x4 kv = kv_load_row<FMT>(a.k, a.ks, row, c), qv = moe::ld4(qr + 4 * c);
        for (int e = 0; e < 4; ++e) sc = __builtin_fmaf(kv[e], qv[e], sc);
      }
      sc *= 0.125f;
    }
    float mt = sc;
    for (int d = 32; d > 0; d >>= 1) mt = fmaxf(mt, __shfl_xor(mt, d));
    const float mn = fmaxf(m, mt), ref = mn == -__builtin_inff() ? 0.0f : mn;
    const float al = expf(m - ref), e = page >= 0 ? expf(sc - ref) : 0.0f;
    l = l * al + e;
    o *= al;
    m = mn;
    for (int t = 0; t < 64; ++t) {
      const int pg = __shfl(page, t);
      if (pg < 0) continue;
      const int pt = __shfl(p, t);
      const float w = __shfl(e, t);
      const size_t r = kv_row(a, pg, g, pt & ((1 << a.pshift) - 1));
      o = __builtin_fmaf(w, kv_load_row<FMT>(a.v, a.vs, r, lane >> 2)[lane & 3], o);
    }
  }
  for (int d = 32; d > 0; d >>= 1) l += __shfl_xor(l, d);
  out[(size_t)(s.row0 + i) * ldo + h * kRowDim + lane] = l == 0.0f ? 0.0f : o / l;
}

// ---------------------------------------------------------------------------
// Launchers
// ---------------------------------------------------------------------------

template <int FMT, bool ROPE>
static hipError_t kv_write_launch(const KvArgs &a, const KvWriteArgs &w, hipStream_t st) {
  const int rows = a.max_new * ((ROPE ? w.heads : 0) + 2 * a.kv_heads);
  hipLaunchKernelGGL((kv_write_kernel<FMT, ROPE, 4>), dim3((rows + 63) / 64, a.batch), dim3(256), 0, st, a, w);
  return hipGetLastError();
}

template <int FMT>
static hipError_t kv_read_launch(const KvArgs &a, float *k_out, float *v_out, int rows, int ld, hipStream_t st) {
  const int n = std::min<long long>(rows, (long long)a.max_pages << a.pshift) *
                ((k_out != nullptr) + (v_out != nullptr)) * a.kv_heads;
  if (n == 0) return hipSuccess;
  hipLaunchKernelGGL((kv_read_kernel<FMT, 4>), dim3((n + 63) / 64, a.batch), dim3(256), 0, st, a, k_out, v_out, rows,
                     ld);
  return hipGetLastError();
}

// f with the cache's format as a compile-time constant.
template <typename F>
static hipError_t by_format(int format, F &&f) {
  switch (format) {
    case LFM_KV_F32: return f(std::integral_constant<int, LFM_KV_F32>{});
    case LFM_KV_BF16: return f(std::integral_constant<int, LFM_KV_BF16>{});
    case LFM_KV_INT8: return f(std::integral_constant<int, LFM_KV_INT8>{});
    default: return f(std::integral_constant<int, LFM_KV_FP8>{});
  }
}

hipError_t launch_kv_write(const KvArgs &a, const KvWriteArgs &w, hipStream_t st) {
  return by_format(a.format, [&](auto f) {
    return w.q_weight ? kv_write_launch<f(), true>(a, w, st) : kv_write_launch<f(), false>(a, w, st);
  });
}

hipError_t launch_kv_read(const KvArgs &a, float *k_out, float *v_out, int rows, int ld, hipStream_t st) {
  return by_format(a.format, [&](auto f) { return kv_read_launch<f()>(a, k_out, v_out, rows, ld, st); });
}

size_t kv_attention_ws(const KvArgs &, int) { return 0; }

hipError_t launch_kv_attention(const KvArgs &a, const float *q, int ld, float *out, int ldo, int heads, void *,
                               hipStream_t st) {
  return by_format(a.format, [&](auto f) {
    hipLaunchKernelGGL((kv_attention_kernel<f()>), dim3(a.max_new * heads, a.batch), dim3(64), 0, st, a, q, ld, out,
                       ldo, heads);
    return hipGetLastError();
  });
}

}  // namespace lfm
