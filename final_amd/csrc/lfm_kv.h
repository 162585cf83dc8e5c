// The paged KV cache on the device: a call's arguments, the sequences' checks,
// and rows of 64 in and out of the cache's formats (include/lfm_capi.h).
#pragma once

#include "gpu_common.h"
#include "lfm_capi.h"
#include "lfm_internal.h"

namespace lfm {

using moe::f32x4;
typedef __bf16 kv_bf16x2 __attribute__((ext_vector_type(2)));
typedef float kv_f32x2 __attribute__((ext_vector_type(2)));

constexpr int kRowDim = 64;  // head_dim

__device__ __forceinline__ void kv_flag(int *bad) {
  if (bad) __hip_atomic_store(bad, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Sequence b's new tokens (rows row0 .. row0 + n) and own length; false where
// it takes no part in the call.  With NEW false the new tokens are not looked at.
struct KvSeq {
  int row0, n, len;
};

template <bool NEW>
__device__ __forceinline__ bool kv_seq(const KvArgs &a, int b, KvSeq &s) {
  s.len = a.own_len[b];
  s.row0 = b * a.max_new;
  s.n = a.max_new;
  if (NEW && a.new_start) {
    s.row0 = a.new_start[b];
    const long long n = (long long)a.new_start[b + 1] - s.row0;
    s.n = n < 0 || n > a.max_new ? -1 : (int)n;
  }
  if (s.len == 0) return false;
  bool ok = s.len > 0 && s.len <= (long long)a.max_pages << a.pshift;
  if (NEW) ok = ok && s.row0 >= 0 && s.n >= 0 && s.n <= s.len && s.row0 <= a.tokens - s.n;
  if (!ok) kv_flag(a.bad);
  return ok;
}

// Row index of (page, kv head, offset) in the pools; the page is inside them.
__device__ __forceinline__ size_t kv_row(const KvArgs &a, int page, int h, int off) {
  return (((size_t)page * a.kv_heads + h) << a.pshift) + off;
}

template <int FMT>
constexpr int kv_size() {
  return FMT == LFM_KV_F32 ? 4 : FMT == LFM_KV_BF16 ? 2 : 1;
}

// Largest of the 16 lanes of a row (DPP row rotations), on the bits of
// magnitudes: NaN orders above infinity, infinity above every number.
__device__ __forceinline__ uint32_t row_max_bits(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xf, 0xf, true));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x124, 0xf, 0xf, true));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x122, 0xf, 0xf, true));
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x121, 0xf, 0xf, true));
}

// x / s to the nearest integer, halves to even, of the real quotient: the
// rounded product with 1 / s is that integer or, next to a half, one beside it;
// the remainder x - q s is exact in fp32 (|q| <= 127) and says which.
__device__ __forceinline__ float nearest_quotient(float x, float s, float inv) {
  float q = rintf(x * inv);
  const float e = __builtin_fmaf(-q, s, x), half = 0.5f * s;
  const bool odd = ((int)q & 1) != 0;
  if (e > half || (e == half && odd)) q += 1.0f;
  if (e < -half || (e == -half && odd)) q -= 1.0f;
  return q;
}

// Lane c of a row's 16 stores elements 4c .. 4c+3 (x) of pool row `row`; all 16
// take part, `ok` or not.
template <int FMT>
__device__ __forceinline__ void kv_store_row(char *pool, float *scale, size_t row, int c, f32x4 x,
                                             bool ok) {
  char *p = pool + (row * kRowDim + 4 * c) * kv_size<FMT>();
  if constexpr (FMT == LFM_KV_F32) {
    if (ok) *reinterpret_cast<f32x4 *>(p) = x;
  } else if constexpr (FMT == LFM_KV_BF16) {
    uint2 w;
    w.x = __builtin_bit_cast(uint32_t, __builtin_convertvector(kv_f32x2{x[0], x[1]}, kv_bf16x2));
    w.y = __builtin_bit_cast(uint32_t, __builtin_convertvector(kv_f32x2{x[2], x[3]}, kv_bf16x2));
    if (ok) *reinterpret_cast<uint2 *>(p) = w;
  } else {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float e = x[i];  // not x[i] itself: a bit cast of a vector's element takes the first
      m = max(m, __builtin_bit_cast(uint32_t, e) & 0x7FFFFFFFu);
    }
    m = row_max_bits(m);
    const float amax = __builtin_bit_cast(float, m);
    const bool fin = m < 0x7F800000u;
    float s;
    uint32_t w = 0;
    if constexpr (FMT == LFM_KV_INT8) {
      s = amax / 127.0f;
      // away from the subnormals the remainder's products would round in
      const float up = s < 0x1p-60f ? 0x1p80f : 1.0f, ss = s * up, inv = 1.0f / ss;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float q = __builtin_fminf(__builtin_fmaxf(nearest_quotient(x[i] * up, ss, inv), -127.0f), 127.0f);
        w |= ((uint32_t)(int)q & 0xFFu) << (8 * i);
      }
      if (s == 0.0f) w = 0;
    } else {
      // 448 = 1.75 * 2^8: amax = f 2^E needs 2^(E - 8), or one more for f > 1.75
      const int e = max((int)(m >> 23) - 127 - 8 + ((m & 0x7FFFFFu) > 0x600000u ? 1 : 0), -126);
      s = __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
      const float inv = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);  // 2^-e, exact
      w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false);
      w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, (int)w, true);
    }
    if (!fin) {
      s = __builtin_nanf("");
      w = 0;
    }
    if (ok) {
      *reinterpret_cast<uint32_t *>(p) = w;
      if (c == 0) scale[row] = s;
    }
  }
}

// The values of elements 4c .. 4c+3 of pool row `row`.
template <int FMT>
__device__ __forceinline__ f32x4 kv_load_row(const char *pool, const float *scale, size_t row, int c) {
  const char *p = pool + (row * kRowDim + 4 * c) * kv_size<FMT>();
  if constexpr (FMT == LFM_KV_F32) {
    return *reinterpret_cast<const f32x4 *>(p);
  } else if constexpr (FMT == LFM_KV_BF16) {
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    return f32x4{__builtin_bit_cast(float, w.x << 16), __builtin_bit_cast(float, w.x & 0xFFFF0000u),
                 __builtin_bit_cast(float, w.y << 16), __builtin_bit_cast(float, w.y & 0xFFFF0000u)};
  } else {
    const uint32_t w = *reinterpret_cast<const uint32_t *>(p);
    const float s = scale[row];
    f32x4 v;
    if constexpr (FMT == LFM_KV_INT8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = (float)(signed char)(w >> (8 * i));
    } else {
      const kv_f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
      const kv_f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
      v = f32x4{lo[0], lo[1], hi[0], hi[1]};
    }
    return v * s;
  }
}

}  // namespace lfm
