// HIP kernels of the paged KV cache (gfx950): rows written as they are
// quantised (with the q/k norm and rotation in front where asked for), rows
// read back, and attention of new tokens over a shared prefix and their own
// pages.
#include <algorithm>
#include <type_traits>

#include "lfm_kv.h"
#include "lfm_rope.h"
#include "split_tile.h"

namespace lfm {

// ---------------------------------------------------------------------------
// Rows into the cache, and back
// ---------------------------------------------------------------------------

// 16 lanes take a row of 64 (a token's q, k or v head), four floats each, R rows
// one after the other; block (x, sequence).  A row's largest magnitude is found
// over its 16 lanes by DPP moves, so nothing goes through LDS and no block waits.
// What bounds them is memory: every load that hangs on nothing but the sequence
// stands in front, without a branch, pages and then R rows, so that four rows a
// lane are in flight.  64 ragged sequences of up to 512 tokens and 8 heads in fp8 (117
// MB): written in 32 us (3.7 TB/s, three quarters of it reads), read back in 21 us
// (5.6 TB/s); 20011 bf16 tokens (123 MB) are read in 26 us.  A single token takes 2.4
// and 37 take 3.1 us: a launch, and the table, page and row one after the other.

// The page, or -1 (and the flag) where it is outside the cache.
__device__ __forceinline__ int kv_page(const KvArgs &a, int page) {
  if (page >= 0 && page < a.num_pages) return page;
  kv_flag(a.bad);
  return -1;
}

// Which of a sequence's `blocks` this one is, or `blocks` and more: block x is on XCD x % 8
// (gridDim.x is a multiple of 8), and an XCD takes neighbouring rows, whose scales share
// lines of 32 tokens (64 ragged fp8 prompts in and out: 34.0 + 22.7 us in block order).
__device__ __forceinline__ int neighbours(int blocks) {
  const int per = (blocks + 7) / 8, at = blockIdx.x >> 3;
  return at < per ? (blockIdx.x & 7) * per + at : blocks;
}

template <int FMT, bool ROPE, int R>
__global__ __launch_bounds__(256) void kv_write_kernel(KvArgs a, KvWriteArgs w) {
  KvSeq s;
  if (!kv_seq<true>(a, blockIdx.y, s)) return;
  const int qrows = ROPE ? w.heads : 0, per_tok = qrows + 2 * a.kv_heads, total = s.n * per_tok;
  const int first = neighbours((total + 16 * R - 1) / (16 * R)) * 16 * R;
  if (first >= total) return;
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
  f32x4 x[R], cs[R], sn[R];
  int tok[R], row[R], page[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int f = min(first + 16 * j + g, total - 1);  // a surplus row repeats the last, and is not stored
    tok[j] = f / per_tok;
    row[j] = f - tok[j] * per_tok;
    const int pos = s.len - s.n + tok[j];
    page[j] = a.pages[(size_t)blockIdx.y * a.max_pages + (pos >> a.pshift)];
    const int col = row[j] < qrows ? row[j] * kRowDim
                    : row[j] < qrows + a.kv_heads ? w.k_col + (row[j] - qrows) * kRowDim
                                                  : w.v_col + (row[j] - qrows - a.kv_heads) * kRowDim;
    x[j] = moe::ld4(w.qkv + (size_t)(s.row0 + tok[j]) * w.ld + col + 4 * c);
    if (ROPE) {
      const size_t t = (size_t)min(a.prefix_len + pos, w.max_pos - 1) * kRowDim + 4 * c;
      cs[j] = moe::ld4(w.cos_t + t);
      sn[j] = moe::ld4(w.sin_t + t);
    }
  }
  f32x4 wq, wk;
  if (ROPE) {
    wq = moe::ld4(w.q_weight + 4 * c);
    wk = moe::ld4(w.k_weight + 4 * c);
  }
#pragma unroll
  for (int j = 0; j < R; ++j) {
    bool ok = first + 16 * j + g < total;
    const int pos = s.len - s.n + tok[j];
    const bool is_q = row[j] < qrows, is_v = row[j] >= qrows + a.kv_heads;
    if (ROPE) {
      if (ok && a.prefix_len + pos >= w.max_pos) {
        kv_flag(a.bad);
        ok = false;
      }
      const f32x4 y = norm_rope_row(x[j], is_q ? wq : wk, cs[j], sn[j]);
      if (!is_v) x[j] = y;
      if (ok && is_q) moe::st4(w.qkv + (size_t)(s.row0 + tok[j]) * w.ld + row[j] * kRowDim + 4 * c, y);
    }
    const int h = row[j] - qrows - (is_v ? a.kv_heads : 0);
    ok = ok && !is_q;
    if (ok) ok = kv_page(a, page[j]) >= 0;
    const size_t at = ok ? kv_row(a, page[j], h, pos & ((1 << a.pshift) - 1)) : 0;
    kv_store_row<FMT>(is_v ? a.v : a.k, is_v ? a.vs : a.ks, at, c, x[j], ok);
  }
}

template <int FMT, int R>
__global__ __launch_bounds__(256) void kv_read_kernel(KvArgs a, float *k_out, float *v_out, int rows, int ld) {
  KvSeq s;
  if (!kv_seq<false>(a, blockIdx.y, s)) return;
  const int kinds = (k_out != nullptr) + (v_out != nullptr), per_pos = kinds * a.kv_heads;
  const int total = min(s.len, rows) * per_pos, first = neighbours((total + 16 * R - 1) / (16 * R)) * 16 * R;
  if (first >= total) return;
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
  int pos[R], row[R], page[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int f = min(first + 16 * j + g, total - 1);  // a surplus row repeats the last
    pos[j] = f / per_pos;
    row[j] = f - pos[j] * per_pos;
    page[j] = a.pages[(size_t)blockIdx.y * a.max_pages + (pos[j] >> a.pshift)];
  }
  f32x4 x[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    page[j] = kv_page(a, page[j]);
    const bool is_v = !k_out || row[j] >= a.kv_heads;
    const size_t at = kv_row(a, max(page[j], 0), row[j] >= a.kv_heads ? row[j] - a.kv_heads : row[j],
                             pos[j] & ((1 << a.pshift) - 1));
    x[j] = kv_load_row<FMT>(is_v ? a.v : a.k, is_v ? a.vs : a.ks, at, c);
  }
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const bool is_v = !k_out || row[j] >= a.kv_heads;
    float *o = (is_v ? v_out : k_out) + ((size_t)blockIdx.y * rows + pos[j]) * ld +
               (row[j] >= a.kv_heads ? row[j] - a.kv_heads : row[j]) * kRowDim + 4 * c;
    if (first + 16 * j + g < total) moe::st4(o, page[j] >= 0 ? x[j] : f32x4{0.0f, 0.0f, 0.0f, 0.0f});
  }
}

// ---------------------------------------------------------------------------
// Attention over the cache
// ---------------------------------------------------------------------------
//
// A wave computes S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_bf16 for
// tiles of 32 keys and CT tiles of 16 columns, a column being one query head of
// one token that attends the kv head's keys: the heads of a group and the new
// tokens of a sequence (or, for the prefix, of all sequences) stand next to each
// other.  q is the exact sum of three bf16 parts, as is a weight p, and int8,
// e4m3 and bf16 keys and values are bf16 values as they are (an fp32 cache's are
// split too, six of the nine products taken), so the products are exact, their
// sums fp32, and the rows' scales are applied to scores and weights in fp32.
//
// Nothing is staged in LDS and nothing transposed: a lane (c = l % 16, g = l / 16)
// loads 16 bytes of key c of each half tile, which is its operand of S^T up to a
// permutation of the dimensions (the same in q's), and four values, dimensions 4c
// .. 4c+3, of the keys 4g + i, whose weights S^T leaves in this lane: block db of
// O^T takes dimension 4c + db from each.  The tiles are dealt to the waves of a
// part's blocks in turn, which join their sums through LDS at the end; a part that
// is not the only one leaves them in the workspace to kv_join_kernel.
//
// The running maximum is only raised when a score passes it by kRaise: weights
// then reach 2^kRaise, and most tiles need no exchange between lanes and no
// scaling of O.  A weight is 2 to the power of one FMA, score * scale - maximum.

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kKeys = 32;           // keys per tile
constexpr int kMinTiles = 8;        // tiles of a split, at least
constexpr float kRaise = 8.0f;      // log2
constexpr int kFewCols = 4;         // columns of a kernel whose 16 hold four columns' three parts
constexpr int kJoinPitch = 68;      // floats per column of the joined O
constexpr float kNoScore = -__builtin_inff();

struct FlashArgs {
  const float *q;
  float *out;
  float *po;   // [parts][rows][64]: sums of p v of a part
  float2 *pm;  // [parts][rows]: its maximum (log2) and sum of p
  int ld, ldo, heads, group;
  int own_parts, prefix_parts;  // parts 0 .. own_parts are the own positions'
  size_t rows;                  // tokens * heads
};

// Parts that `keys` keys are split into, of at most `parts`.
__host__ __device__ inline int active_parts(int keys, int parts) {
  const int most = (keys + kKeys - 1) / kKeys / kMinTiles;
  return most < 1 ? 1 : most < parts ? most : parts;
}

// Waves of a block without a prefix beside it: few columns leave room for eight.
__host__ __device__ constexpr int own_waves(int ct) { return ct == 0 ? 8 : 4; }

// A block of W waves with CT tiles of 16 columns; CT = 0: kFewCols columns, whose
// three parts fill a tile.
template <int CT, int W>
struct FlashShape {
  static constexpr bool FEW = CT == 0;
  static constexpr int NT = FEW ? 1 : CT, COLS = FEW ? kFewCols : 16 * CT, QP = FEW ? 1 : 3;
  static constexpr int kSumFloats = W * COLS * kJoinPitch, kPartFloats = NT * 2 * QP * 64 * 4;
  static constexpr int kFloats = kSumFloats > kPartFloats ? kSumFloats : kPartFloats;
  static constexpr int kBytes = kFloats * 4 + W * COLS * 8;
};

// What a part's sums (maximum, sum of weights) count under the maximum of all:
// without a score as they are, 0 or NaN.
__device__ __forceinline__ float part_scale(float2 part, float mx) {
  if (part.x == kNoScore) return part.y == 0.0f ? 0.0f : 1.0f;
  return __builtin_amdgcn_exp2f(part.x - mx);
}

// Keys and values of a tile as they were loaded.
template <int FMT>
struct RawTile {
  static constexpr int KW = FMT == LFM_KV_F32 ? 4 : FMT == LFM_KV_BF16 ? 2 : 1;  // 16-byte loads of a key's quarter
  static constexpr bool SCALED = FMT == LFM_KV_INT8 || FMT == LFM_KV_FP8;
  u32x4 k[2][KW];
  uint32_t v[2][4][KW];  // [half][key 4g + i][dwords]
  f32x4 ks[2], vs[2];    // scales of keys 4g .. 4g+3
  bool ok[2];            // the half's page is inside the cache
};

// Dimension of element j of k-step s in a lane of group g (K's loads decide it).
template <int FMT>
__device__ __forceinline__ constexpr int key_dim(int s, int g, int j) {
  return FMT == LFM_KV_F32    ? 32 * s + 16 * (j >> 2) + 4 * g + (j & 3)
         : FMT == LFM_KV_BF16 ? 32 * s + 8 * g + j
                              : 16 * g + 8 * s + j;
}

__device__ __forceinline__ uint32_t pack_hi(uint32_t lo, uint32_t hi) {  // upper halves of two floats
  return __builtin_amdgcn_perm(hi, lo, 0x07060302u);
}

__device__ __forceinline__ uint32_t byte_pair(float lo, float hi) {  // two small integers as bf16, exactly
  return pack_hi(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
}

// Bits 0 and 1 as masks of a dword's halves.
__device__ __forceinline__ uint32_t half_mask(uint32_t bits) {
  return (bits & 1u ? 0xFFFFu : 0u) | (bits & 2u ? 0xFFFF0000u : 0u);
}

// Four bytes of an 8-bit format -> two dwords of bf16.
template <int FMT>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t &lo, uint32_t &hi) {
  if constexpr (FMT == LFM_KV_FP8) {
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true));
  } else {
    lo = byte_pair((float)(signed char)w, (float)(signed char)(w >> 8));
    hi = byte_pair((float)(signed char)(w >> 16), (float)(signed char)(w >> 24));
  }
}

// x - the low (high) bf16 of a pair: exact where that is x rounded.  The factor
// stands in a register: as an inline constant -1.0 the instruction takes it for
// the upper half.
__device__ __forceinline__ float less(float x, uint32_t pair, uint32_t minus_one) {
  asm("" : "+s"(minus_one));
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(kv_bf16x2, pair),
                                         __builtin_bit_cast(kv_bf16x2, minus_one), x, false);
}
__device__ __forceinline__ float less_lo(float x, uint32_t pair) { return less(x, pair, 0xBF80u); }
__device__ __forceinline__ float less_hi(float x, uint32_t pair) { return less(x, pair, 0xBF800000u); }
__device__ __forceinline__ uint32_t round_pair(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(kv_f32x2{lo, hi}, kv_bf16x2));
}

// Three parts of eight floats, exact together: 8 bits each, rounded to nearest.
// 28 instructions (the remainders by the bf16 dot product) where masks, subtractions
// and byte permutes take 44.
__device__ __forceinline__ void split8_exact(const float (&x)[8], bf16x8 (&part)[3]) {
  u32x4 p[3];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float a = x[2 * j], b = x[2 * j + 1];
    p[0][j] = round_pair(a, b);
    a = less_lo(a, p[0][j]);
    b = less_hi(b, p[0][j]);
    p[1][j] = round_pair(a, b);
    p[2][j] = round_pair(less_lo(a, p[1][j]), less_hi(b, p[1][j]));
  }
#pragma unroll
  for (int q = 0; q < 3; ++q) part[q] = __builtin_bit_cast(bf16x8, p[q]);
}

// One of three parts of eight floats (0, 1, 2; zeros for 3), 8 bits each, truncated.
__device__ __forceinline__ bf16x8 part8(const float (&x)[8], int which) {
  const uint32_t m1 = which == 0 ? 0u : which == 3 ? 0xFFFFFFFFu : 0xFFFF0000u, m2 = which == 2 ? 0xFFFF0000u : 0u;
  u32x4 p;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t w[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float v = x[2 * j + e], a = v - __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & m1);
      const float b = a - __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, a) & m2);
      w[e] = __builtin_bit_cast(uint32_t, b);
    }
    p[j] = pack_hi(w[0], w[1]);
  }
  return __builtin_bit_cast(bf16x8, p);
}

// Sum over the four columns c, c ^ 4, ... of a row of 16 lanes.
__device__ __forceinline__ float sum_parts(float v) {
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x128, 0xf, 0xf, true));
  return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x124, 0xf, 0xf, true));
}

// acc += the product of an operand of NP parts with one of QP: the six largest
// products of three parts by three; where one side has one part, all.
template <size_t NP, size_t QP>
__device__ __forceinline__ f32x4 mfma_parts(const bf16x8 (&x)[NP], const bf16x8 (&y)[QP], f32x4 acc) {
  if constexpr (NP == 3 && QP == 3) {
#pragma unroll
    for (int m = 0; m < moe::kSplitProducts; ++m)
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[moe::kSplitA[m]], y[moe::kSplitB[m]], acc, 0, 0, 0);
  } else {
#pragma unroll
    for (int n = (int)(NP * QP) - 1; n >= 0; --n)
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[NP == 1 ? 0 : n], y[QP == 1 ? 0 : n], acc, 0, 0, 0);
  }
  return acc;
}

// The operand of K for half tile hb and k-step st.
template <int FMT, int NP>
__device__ __forceinline__ void key_operand(const RawTile<FMT> &r, int hb, int st, bf16x8 (&op)[NP]) {
  if constexpr (FMT == LFM_KV_F32) {
    const f32x4 x[2] = {__builtin_bit_cast(f32x4, r.k[hb][2 * st]), __builtin_bit_cast(f32x4, r.k[hb][2 * st + 1])};
    moe::split8(x, op);
  } else if constexpr (FMT == LFM_KV_BF16) {
    op[0] = __builtin_bit_cast(bf16x8, r.k[hb][st]);
  } else {
    uint32_t w[4];
    widen4<FMT>(r.k[hb][0][2 * st], w[0], w[1]);
    widen4<FMT>(r.k[hb][0][2 * st + 1], w[2], w[3]);
    op[0] = __builtin_bit_cast(bf16x8, u32x4{w[0], w[1], w[2], w[3]});
  }
}

// The operands of V: block db takes dimension 4c + db of the lane's eight keys.
template <int FMT, int NP>
__device__ __forceinline__ void value_operands(const RawTile<FMT> &r, bf16x8 (&op)[4][NP]) {
  if constexpr (FMT == LFM_KV_F32) {
#pragma unroll
    for (int db = 0; db < 4; ++db) {
      f32x4 x[2];
#pragma unroll
      for (int hb = 0; hb < 2; ++hb)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[hb][i] = __builtin_bit_cast(float, r.v[hb][i][db]);
      moe::split8(x, op[db]);
    }
  } else {
    u32x4 w[4];
#pragma unroll
    for (int hb = 0; hb < 2; ++hb) {
      const uint32_t(&v)[4][RawTile<FMT>::KW] = r.v[hb];
#pragma unroll
      for (int p = 0; p < 2; ++p) {  // keys 4g + 2p and 4g + 2p + 1
        if constexpr (FMT == LFM_KV_BF16) {
#pragma unroll
          for (int db = 0; db < 4; ++db)
            w[db][2 * hb + p] = __builtin_amdgcn_perm(v[2 * p + 1][db >> 1], v[2 * p][db >> 1],
                                                      db & 1 ? 0x07060302u : 0x05040100u);
        } else if constexpr (FMT == LFM_KV_FP8) {
          // dimensions (0, 1) and (2, 3), the two keys byte by byte
          const uint32_t q[2] = {__builtin_amdgcn_perm(v[2 * p + 1][0], v[2 * p][0], 0x05010400u),
                                 __builtin_amdgcn_perm(v[2 * p + 1][0], v[2 * p][0], 0x07030602u)};
#pragma unroll
          for (int db = 0; db < 4; ++db)
            w[db][2 * hb + p] = __builtin_bit_cast(
                uint32_t, db & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[db >> 1], 1.0f, true)
                                 : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[db >> 1], 1.0f, false));
        } else {
#pragma unroll
          for (int db = 0; db < 4; ++db)
            w[db][2 * hb + p] = byte_pair((float)(signed char)(v[2 * p][0] >> (8 * db)),
                                          (float)(signed char)(v[2 * p + 1][0] >> (8 * db)));
        }
      }
    }
#pragma unroll
    for (int db = 0; db < 4; ++db) op[db][0] = __builtin_bit_cast(bf16x8, w[db]);
  }
}

// Which positions a block takes: a sequence's own, the shared prefix's for all
// sequences, or a sequence's own with the prefix's tiles in front of them.
enum FlashKeys { kOwnKeys, kPrefixKeys, kBothKeys };

// One block's part of a product: columns col0 .. of kv head h, every `stride`-th
// tile of KEYS (of sequence b).  Tiles are dealt to the parts' waves in turn, so that
// a wave knows its first tile, and looks up its page, before it knows how long the
// sequence is.
template <int FMT, int CT, FlashKeys KEYS, int W>
__device__ __forceinline__ void flash_part(const KvArgs &a, const FlashArgs &f, int h, int part, int group, int b,
                                           float *s_lds) {
  using Raw = RawTile<FMT>;
  using SH = FlashShape<CT, W>;
  constexpr int NP = FMT == LFM_KV_F32 ? 3 : 1, NT = SH::NT, COLS = SH::COLS, QP = SH::QP;
  constexpr bool FEW = SH::FEW, PREFIX = KEYS == kPrefixKeys, BOTH = KEYS == kBothKeys;
  // q's parts as operands [column tile][k-step][part][lane], then the waves' sums
  bf16x8 *const s_q = reinterpret_cast<bf16x8 *>(s_lds);
  float2 *const s_m = reinterpret_cast<float2 *>(s_lds + SH::kFloats);  // [W][COLS]
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lc = FEW ? c & 3 : c;  // the lane's column in its tile
  const int col0 = group * COLS;
  const int t0 = part * W + wave;

  // tiles of the prefix in front of the own ones; a tile's number among its own kind
  const int front = BOTH ? (a.prefix_len + kKeys - 1) / kKeys : 0;
  auto in_front = [&](int t) { return BOTH && t < front; };
  auto number = [&](int t) { return in_front(t) ? t : t - front; };
  const int *own_table = a.pages + (size_t)b * a.max_pages;
  auto table_of = [&](int t) { return PREFIX || in_front(t) ? a.prefix_pages : own_table; };
  const int most_pages = PREFIX || in_front(t0) ? (a.prefix_len - 1) >> a.pshift : a.max_pages - 1;
  int first_pages = 0;  // of the first tile's halves, in lanes 0 and 1
  if (most_pages >= 0)
    first_pages = table_of(t0)[min((number(t0) * kKeys + 16 * (lane & 1)) >> a.pshift, most_pages)];
  KvSeq s;
  int len, first_seen;  // keys; those below first_seen are seen by every column of the block
  if (PREFIX) {
    s.row0 = 0;
    s.n = a.tokens;
    len = first_seen = a.prefix_len;
  } else {
    if (!kv_seq<true>(a, b, s)) return;
    len = s.len;
    first_seen = len - s.n + col0 / f.group + 1;
  }
  const int parts = active_parts(len, PREFIX ? f.prefix_parts : f.own_parts), stride = parts * W;
  if (part >= parts || col0 >= s.n * f.group) return;
  const bool direct = !PREFIX && f.prefix_parts == 0 && parts == 1;
  // the last position a column of the block sees
  const int seen = PREFIX ? len : min(len, len - s.n + (col0 + COLS - 1) / f.group + 1);
  const int t_end = front + (seen + kKeys - 1) / kKeys;
  auto keys_of = [&](int t) { return in_front(t) ? a.prefix_len : len; };

  // q, for the column tiles' k-steps w, w + W, ... in wave w
  constexpr int QE = (2 * NT + W - 1) / W;
  f32x4 qv[QE][2];
  int last[NT];  // last position the lane's columns see
#pragma unroll
  for (int ct = 0; ct < NT; ++ct) last[ct] = PREFIX ? len - 1 : len - s.n + (col0 + ct * 16 + lc) / f.group;
#pragma unroll
  for (int n = 0; n < QE; ++n) {
    const int e = min(wave + n * W, 2 * NT - 1), col = col0 + (e >> 1) * 16 + lc, tok = col / f.group;
    const bool valid = tok < s.n;
    const float *qr = f.q + (size_t)(s.row0 + (valid ? tok : 0)) * f.ld + (h * f.group + col - tok * f.group) * kRowDim;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      qv[n][j] = moe::ld4(qr + key_dim<FMT>(e & 1, g, 4 * j));
      if (!valid) qv[n][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }

  auto load = [&](int t, int page0, int page1, Raw &r) {
#pragma unroll
    for (int hb = 0; hb < 2; ++hb) {
      // a half tile behind the last key repeats the one with that key
      const int k0 = min(number(t) * kKeys + 16 * hb, (keys_of(t) - 1) & ~15), page = hb ? page1 : page0;
      r.ok[hb] = page >= 0;
      const size_t row = kv_row(a, max(page, 0), h, k0 & ((1 << a.pshift) - 1));
      // the half tile's 16 rows as buffers: a scalar base, and offsets of the lane alone
      constexpr int kRowBytes = kRowDim * kv_size<FMT>(), kBytes = 16 * kRowBytes;
      const auto kr = __builtin_amdgcn_make_buffer_rsrc(a.k + row * kRowBytes, 0, kBytes, moe::kBufferRsrcWord3);
      const auto vr = __builtin_amdgcn_make_buffer_rsrc(a.v + row * kRowBytes, 0, kBytes, moe::kBufferRsrcWord3);
#pragma unroll
      for (int w = 0; w < Raw::KW; ++w)
        r.k[hb][w] = __builtin_amdgcn_raw_buffer_load_b128(kr, c * kRowBytes + 16 * g + 64 * w, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = (4 * g + i) * kRowBytes + 4 * c * kv_size<FMT>();
        if constexpr (Raw::KW == 1) {
          r.v[hb][i][0] = __builtin_amdgcn_raw_buffer_load_b32(vr, at, 0, 0);
        } else if constexpr (Raw::KW == 2) {
          const auto x = __builtin_amdgcn_raw_buffer_load_b64(vr, at, 0, 0);
          r.v[hb][i][0] = x[0];
          r.v[hb][i][1] = x[1];
        } else {
          const auto x = __builtin_amdgcn_raw_buffer_load_b128(vr, at, 0, 0);
#pragma unroll
          for (int w = 0; w < 4; ++w) r.v[hb][i][w] = x[w];
        }
      }
      if constexpr (Raw::SCALED) {
        const auto ksr = __builtin_amdgcn_make_buffer_rsrc(a.ks + row, 0, 64, moe::kBufferRsrcWord3);
        const auto vsr = __builtin_amdgcn_make_buffer_rsrc(a.vs + row, 0, 64, moe::kBufferRsrcWord3);
        r.ks[hb] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(ksr, 16 * g, 0, 0));
        r.vs[hb] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(vsr, 16 * g, 0, 0));
      }
    }
  };
  // Pages of 32 of the wave's tiles, a half tile's in each lane (-1 outside the cache).
  auto page_of = [&](int t) {
    t += stride * (lane >> 1);
    return table_of(t)[min(number(t) * kKeys + 16 * (lane & 1), (keys_of(t) - 1) & ~15) >> a.pshift];
  };

  f32x4 o[NT][4];
  // ref: the running maximum, 0 before there is one; limit: what a score may pass it by
  float ref[NT], limit[NT], l[NT];
#pragma unroll
  for (int ct = 0; ct < NT; ++ct) {
    ref[ct] = l[ct] = 0.0f;
    limit[ct] = kNoScore;
#pragma unroll
    for (int d = 0; d < 4; ++d) o[ct][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // Tile t from r, while `next` (on pages next0 and next1) is loaded to rn.  The
  // values become operands after the scores, for the registers.
  auto tile = [&](int t, Raw &r, Raw &rn, int next, int next0, int next1) {
    const int k0 = number(t) * kKeys;
    auto last_of = [&](int ct) { return in_front(t) ? a.prefix_len - 1 : last[ct]; };
    const bool ok[2] = {r.ok[0], r.ok[1]};
    // some keys are behind the end, behind a column's own position or on no page (wave-uniform)
    const bool cut = k0 + kKeys > (in_front(t) ? a.prefix_len : first_seen) || !ok[0] || !ok[1];
    if constexpr (Raw::SCALED) {
      // or the compiler takes the bytes apart as they arrive, in three steps each
#pragma unroll
      for (int hb = 0; hb < 2; ++hb) asm("" : "+v"(r.k[hb][0]));
    }
    load(next, next0, next1, rn);
    bf16x8 kop[2][2][NP];
#pragma unroll
    for (int hb = 0; hb < 2; ++hb)
#pragma unroll
      for (int st = 0; st < 2; ++st) key_operand<FMT>(r, hb, st, kop[hb][st]);

    // scores of keys 16 hb + 4g + i against the running maximum
    float p[NT][8];
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      bf16x8 qp[2][QP];
#pragma unroll
      for (int e = 0; e < 2 * QP; ++e) qp[e / QP][e % QP] = s_q[(ct * 2 * QP + e) * 64 + lane];
#pragma unroll
      for (int hb = 0; hb < 2; ++hb) {
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int st = 0; st < 2; ++st) acc = mfma_parts(kop[hb][st], qp[st], acc);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float sc = FEW ? sum_parts(acc[i]) : (float)acc[i];
          p[ct][4 * hb + i] = Raw::SCALED ? __builtin_fmaf(sc, r.ks[hb][i], -ref[ct]) : sc - ref[ct];
        }
      }
    }
    if (cut) {
#pragma unroll
      for (int ct = 0; ct < NT; ++ct)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          p[ct][e] = !ok[e >> 2] || k0 + 16 * (e >> 2) + 4 * g + (e & 3) > last_of(ct) ? kNoScore : p[ct][e];
    }
    bool raise = false;
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      float top = __builtin_elementwise_maximum(p[ct][0], p[ct][1]);
#pragma unroll
      for (int e = 2; e < 8; e += 2)
        top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(p[ct][e], p[ct][e + 1]), top);
      raise = raise || top > limit[ct];
    }
    if (__any(raise)) {
#pragma unroll
      for (int ct = 0; ct < NT; ++ct) {
        float mt = kNoScore;
#pragma unroll
        for (int e = 0; e < 8; ++e) mt = fmaxf(mt, p[ct][e]);
        mt = fmaxf(mt, __shfl_xor(mt, 16));
        mt = fmaxf(mt, __shfl_xor(mt, 32));
        const bool had = limit[ct] != kNoScore;
        if (had) mt = fmaxf(mt, 0.0f);
        if (mt != kNoScore) {
          const float to = ref[ct] + mt, by = to - ref[ct];  // what the rounded maximum is above the old one
          const float scale = had ? __builtin_amdgcn_exp2f(-by) : 0.0f;
          ref[ct] = to;
          limit[ct] = kRaise;
          l[ct] *= scale;
#pragma unroll
          for (int d = 0; d < 4; ++d) o[ct][d] *= scale;
          // of scores beyond 2^27 the FMA keeps more than their maximum's rounding left
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            p[ct][e] -= by;
            p[ct][e] = p[ct][e] > kRaise ? kRaise : p[ct][e];
          }
        }
      }
    }
    bf16x8 vop[4][NP];
    value_operands<FMT>(r, vop);
    // A value (or its row's scale) that is not finite must not meet the zero
    // weight of a column that does not see it, nor what stands behind the end or
    // on no page: such values (a bit each in nf) leave the product and make the
    // outputs of the columns that do see them NaN.
    uint32_t nf = 0;
    bool apart = false;
    if (cut) {
      if constexpr (FMT != LFM_KV_INT8) {
#pragma unroll
        for (int db = 0; db < 4; ++db) {
          const u32x4 w = __builtin_bit_cast(u32x4, vop[db][0]);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            nf |= ((w[j] & 0x7F80u) == 0x7F80u ? 1u : 0u) << (8 * db + 2 * j) |
                  ((w[j] & 0x7F800000u) == 0x7F800000u ? 2u : 0u) << (8 * db + 2 * j);
        }
      }
      if constexpr (Raw::SCALED) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (!(__builtin_fabsf(r.vs[e >> 2][e & 3]) <= __FLT_MAX__)) nf |= 0x01010101u << e;
      }
      apart = __any(nf != 0);
      if (apart) {
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
          for (int q = 0; q < NP; ++q) {
            u32x4 w = __builtin_bit_cast(u32x4, vop[db][q]);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] &= ~half_mask(nf >> (8 * db + 2 * j));
            vop[db][q] = __builtin_bit_cast(bf16x8, w);
          }
        if constexpr (Raw::SCALED) {
#pragma unroll
          for (int e = 0; e < 8; ++e) r.vs[e >> 2][e & 3] = nf >> e & 1u ? 0.0f : r.vs[e >> 2][e & 3];
        }
      }
    }

#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[ct][e] = __builtin_amdgcn_exp2f(p[ct][e]);
        l[ct] += p[ct][e];
        if constexpr (Raw::SCALED) p[ct][e] *= r.vs[e >> 2][e & 3];
      }
      bf16x8 pp[QP];
      if constexpr (FEW)
        pp[0] = part8(p[ct], c >> 2);
      else
        split8_exact(p[ct], pp);
#pragma unroll
      for (int d = 0; d < 4; ++d) o[ct][d] = mfma_parts(vop[d], pp, o[ct][d]);
    }
    if (apart) {
#pragma unroll
      for (int ct = 0; ct < NT; ++ct) {
        // how many of them a column sees: a product of ones
        u32x4 see;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int k = k0 + 16 * (j >> 1) + 4 * g + 2 * (j & 1);
          see[j] = (k <= last_of(ct) ? 0x3F80u : 0u) | (k + 1 <= last_of(ct) ? 0x3F800000u : 0u);
          see[j] = ok[j >> 1] ? see[j] : 0u;
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          u32x4 w;
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = half_mask(nf >> (8 * d + 2 * j)) & 0x3F803F80u;
          const f32x4 n = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w),
                                                                  __builtin_bit_cast(bf16x8, see),
                                                                  f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[ct][d][i] = n[i] > 0.0f ? __builtin_nanf("") : o[ct][d][i];
        }
      }
    }
  };

  Raw ra, rb;  // two tiles: one computed, one on its way
  int pages = 0;
  if (t0 < t_end) {
    pages = kv_page(a, page_of(t0));
    const int half0 = __builtin_amdgcn_readlane(first_pages, 0);
    const int half1 = number(t0) * kKeys + 16 < keys_of(t0) ? __builtin_amdgcn_readlane(first_pages, 1) : half0;
    load(t0, kv_page(a, half0), kv_page(a, half1), ra);
  }
  // q's parts, scaled so that a score is the log2 of its weight
#pragma unroll
  for (int n = 0; n < QE; ++n) {
    const int e = min(wave + n * W, 2 * NT - 1);  // a surplus wave repeats the last
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = qv[n][j >> 2][j & 3] * (0.125f * 1.44269504088896340736f);
    if constexpr (FEW) {
      s_q[e * 64 + lane] = part8(x, c >> 2);
    } else {
      bf16x8 part3[3];
      split8_exact(x, part3);
#pragma unroll
      for (int q = 0; q < 3; ++q) s_q[(e * 3 + q) * 64 + lane] = part3[q];
    }
  }
  __syncthreads();  // q's parts are there
  int t = t0, n = 0;
  // behind the wave's last tile that one is loaded again (its lines are in L2)
  auto step = [&](Raw &r, Raw &rn) {
    const bool more = t + stride < t_end;
    const int next = more ? t + stride : t, i = (n + (more ? 1 : 0)) & 31;
    if (more && i == 0) pages = kv_page(a, page_of(next));
    tile(t, r, rn, next, __builtin_amdgcn_readlane(pages, 2 * i), __builtin_amdgcn_readlane(pages, 2 * i + 1));
    t += stride;
    ++n;
  };
  while (t < t_end) {
    step(ra, rb);
    if (t >= t_end) break;
    step(rb, ra);
  }
  __syncthreads();  // and read for the last time

  // Join the waves: a common maximum, then sums.  O^T row 4g + i of block db is
  // dimension 16g + 4i + db.
#pragma unroll
  for (int ct = 0; ct < NT; ++ct) {
    l[ct] += __shfl_xor(l[ct], 16);
    l[ct] += __shfl_xor(l[ct], 32);
    if (FEW) {
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[ct][d][i] = sum_parts(o[ct][d][i]);
    }
    if (c < COLS) {
      if (g == 0) s_m[wave * COLS + ct * 16 + c] = float2{limit[ct] == kNoScore ? kNoScore : ref[ct], l[ct]};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        moe::st4(&s_lds[(wave * COLS + ct * 16 + c) * kJoinPitch + 16 * g + 4 * i],
                 f32x4{o[ct][0][i], o[ct][1][i], o[ct][2][i], o[ct][3][i]});
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < (COLS * 16 + 64 * W - 1) / (64 * W); ++n) {
    const int e = n * 64 * W + threadIdx.x, cc = e >> 4, d = (e & 15) * 4;
    const int col = col0 + cc, tok = col / f.group, qh = h * f.group + col - tok * f.group;
    if (cc >= COLS || tok >= s.n) continue;
    float mx = kNoScore, lt = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) mx = fmaxf(mx, s_m[w * COLS + cc].x);
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float2 ml = s_m[w * COLS + cc];
      const float sc = part_scale(ml, mx);
      lt += ml.y * sc;
      v += moe::ld4(&s_lds[(w * COLS + cc) * kJoinPitch + d]) * sc;
    }
    const size_t row = (size_t)(s.row0 + tok) * f.heads + qh;
    if (direct) {
      moe::st4(f.out + (size_t)(s.row0 + tok) * f.ldo + qh * kRowDim + d,
               lt == 0.0f ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : v * (1.0f / lt));
    } else {
      const size_t at = (size_t)(PREFIX ? f.own_parts + part : part) * f.rows + row;
      moe::st4(f.po + at * kRowDim + d, v);
      if (d == 0) f.pm[at] = float2{mx, lt};
    }
  }
}

// What bounds it, by the columns (8 kv heads, 4 heads each):
// - one token a sequence: the cache's bytes.  64 ragged sequences of up to 2048 int8
//   positions (88 MB) take 22 us, 4.0 TB/s with the start of the launch and of the
//   loads, 4 of 65536 bf16 positions (537 MB) 93 us, 5.8 TB/s: two tiles a wave are
//   on their way with no branch between their loads.
// - 4 column tiles (a prefix of 64 sequences, or a prompt): the exponentials, the
//   splits of weights and the matrix instructions, which keep a SIMD's vector unit
//   from issuing for half of their 16 cycles.  8192 fp8 positions for 64 x 1 token:
//   11.5 us of 22; the rest is the launch, the first loads, the join of the waves and
//   the own positions beside.
// - short caches: a chain of loads (length, page, rows), 10 us for 300 positions.

// Waves a SIMD holds, by the registers a tile's columns take.
constexpr int flash_waves(int fmt, int ct) { return fmt == LFM_KV_F32 ? 2 : ct == 0 ? 4 : ct == 1 ? 3 : 2; }

// A sequence's positions alone.  kv head fastest: with 8 of them a head's keys stay in
// one XCD's L2.
template <int FMT, int CT, FlashKeys KEYS, int W>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(flash_waves(FMT, CT))))
void kv_flash_kernel(KvArgs a, FlashArgs f) {
  __shared__ float s_lds[FlashShape<CT, W>::kBytes / 4];
  flash_part<FMT, CT, KEYS, W>(a, f, blockIdx.x % a.kv_heads, blockIdx.x / a.kv_heads, blockIdx.y,
                                            blockIdx.z, s_lds);
}

// The prefix, whose blocks are the grid's first, and the own positions beside it.
template <int FMT, int PCT, int CT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(flash_waves(FMT, PCT))))
void kv_prefix_flash_kernel(KvArgs a, FlashArgs f, int prefix_blocks, int own_groups) {
  constexpr int W = 4;
  using P = FlashShape<PCT, W>;
  using O = FlashShape<CT, W>;
  __shared__ float s_lds[(P::kBytes > O::kBytes ? P::kBytes : O::kBytes) / 4];
  int at = blockIdx.x;
  if (at < prefix_blocks) {
    const int h = at % a.kv_heads;
    at /= a.kv_heads;
    flash_part<FMT, PCT, kPrefixKeys, W>(a, f, h, at % f.prefix_parts, at / f.prefix_parts, 0, s_lds);
  } else {
    at -= prefix_blocks;
    const int h = at % a.kv_heads;
    at /= a.kv_heads;
    const int part = at % f.own_parts;
    at /= f.own_parts;
    flash_part<FMT, CT, kOwnKeys, W>(a, f, h, part, at % own_groups, at / own_groups, s_lds);
  }
}

// Joins the parts of a token's head, a wave per row: 16 lanes take a part's 64
// sums, so 16 parts are on their way at a time, and a lane a part's maximum.  Latency
// bounds it: 64 x 32 rows of 9 parts 4.1 us, 4 x 32 rows of 16 parts 4.8 us, half of
// it the launch.
__global__ __launch_bounds__(256) void kv_join_kernel(KvArgs a, FlashArgs f) {
  KvSeq s;
  if (!kv_seq<true>(a, blockIdx.y, s)) return;
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (r >= s.n * f.heads) return;
  const int own = active_parts(s.len, f.own_parts);
  int parts = own;
  if (f.prefix_parts > 0)
    parts += active_parts(a.prefix_len, f.prefix_parts);
  else if (own == 1)
    return;  // written by its one block
  const size_t row = (size_t)s.row0 * f.heads + r;
  const int tok = r / f.heads, qh = r - tok * f.heads;
  auto at = [&](int p) { return (size_t)(p < own ? p : f.own_parts + p - own) * f.rows + row; };
  float mx = kNoScore, lt = 0.0f;
  f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  const int mine = lane >> 4;
  // sums of parts p, p + 4, p + 8, p + 12 of the lane's group, the last where there are none
  auto load = [&](int p, f32x4 (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = moe::ld4(f.po + at(min(p + 4 * i + mine, parts - 1)) * kRowDim + (lane & 15) * 4);
  };
  f32x4 x[4];
  load(0, x);
  for (int p0 = 0; p0 < parts; p0 += 64) {
    float2 ml = f.pm[at(min(p0 + lane, parts - 1))];
    if (p0 + lane >= parts) ml = float2{kNoScore, 0.0f};
    float mn = ml.x;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) mn = fmaxf(mn, __shfl_xor(mn, d));
    mn = fmaxf(mn, mx);
    const float old = part_scale(float2{mx, lt}, mn), sc = part_scale(ml, mn);
    mx = mn;
    float sum = ml.y * sc;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    lt = lt * old + sum;
    v *= old;
    const int n = min(parts - p0, 64);
    for (int p = 0; p < n; p += 16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float w = __shfl(sc, p + 4 * i + mine);
        const f32x4 sum = v + x[i] * w;
        if (p + 4 * i + mine < n) v = sum;
      }
      if (p0 + p + 16 < parts) load(p0 + p + 16, x);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] += __shfl_xor(v[i], 16);
    v[i] += __shfl_xor(v[i], 32);
  }
  if (lane < 16)
    moe::st4(f.out + (size_t)(s.row0 + tok) * f.ldo + qh * kRowDim + lane * 4,
             lt == 0.0f ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : v * (1.0f / lt));
}

// ---------------------------------------------------------------------------
// Launchers
// ---------------------------------------------------------------------------

// Rows a group of 16 lanes takes: four where they fill the CUs, else one.
constexpr long long kSplitRows = 32768;

static unsigned blocks_of(int rows, int each) { return ((unsigned)(rows + each - 1) / each + 7) / 8 * 8; }

template <int FMT, bool ROPE>
static hipError_t kv_write_launch(const KvArgs &a, const KvWriteArgs &w, hipStream_t st) {
  const int rows = a.max_new * ((ROPE ? w.heads : 0) + 2 * a.kv_heads);
  if ((long long)rows * a.batch <= kSplitRows)
    hipLaunchKernelGGL((kv_write_kernel<FMT, ROPE, 1>), dim3(blocks_of(rows, 16), a.batch), dim3(256), 0, st, a, w);
  else
    hipLaunchKernelGGL((kv_write_kernel<FMT, ROPE, 4>), dim3(blocks_of(rows, 64), a.batch), dim3(256), 0, st, a, w);
  return hipGetLastError();
}

template <int FMT>
static hipError_t kv_read_launch(const KvArgs &a, float *k_out, float *v_out, int rows, int ld, hipStream_t st) {
  const int n = (int)std::min<long long>(rows, (long long)a.max_pages << a.pshift) *
                ((k_out != nullptr) + (v_out != nullptr)) * a.kv_heads;
  if (n == 0) return hipSuccess;
  if ((long long)n * a.batch <= kSplitRows)
    hipLaunchKernelGGL((kv_read_kernel<FMT, 1>), dim3(blocks_of(n, 16), a.batch), dim3(256), 0, st, a, k_out, v_out, rows, ld);
  else
    hipLaunchKernelGGL((kv_read_kernel<FMT, 4>), dim3(blocks_of(n, 64), a.batch), dim3(256), 0, st, a, k_out, v_out, rows, ld);
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

// How a call is split: column tiles a wave holds, and parts of the own positions
// and of the prefix.  Parts are added where a wave has most to do, as long as the
// blocks fit the CUs at once, since a second round of blocks begins with the same
// chain of loads (6-8 us) as the first: 16 x 5 tokens of 1000 int8 positions behind
// 2000 shared ones take 18.8 us in 416 blocks, 22.1 in 536, 24.5 in 792.  Where the
// sequences alone fill the CUs the prefix gets half as many blocks beside them, or
// as many where it is longer than kLongPrefix (64 x 1 token behind fp8 positions, us
// in 256 / 512 blocks: 8192 23.9 / 27.8, 16384 37.0 / 39.4, 32768 63.6 / 58.0; 8192
// in 128: 34.9).
struct FlashPlan {
  int own_ct, prefix_ct, own_groups, prefix_groups, own_parts, prefix_parts;
  bool wide;  // own positions by blocks of kWideWaves
};

constexpr int kFlashCUs = 256, kMostParts = 256, kLongPrefix = 20480;

static int columns_of(int ct) { return ct == 0 ? kFewCols : 16 * ct; }

static int widest(int format) { return format == LFM_KV_F32 ? 2 : 4; }

// A tile's time, to that of one column tile.
static float tile_cost(int ct) { return ct <= 1 ? 1.0f : ct == 2 ? 1.6f : 2.8f; }

// Waves of a block of column tiles that has a CU to itself: 5 tokens over 1000 int8
// positions 12.6 us, 4 waves in two launches 16.2 (twice the 8 of a single token's blocks
// wait for the CU's loads: 900 positions 10.7 us, 9.7 with 8).
constexpr int kWideWaves = 8;

// Tiles of a block below which a sequence's positions are not split, nor the prefix
// shared (each sequence then reads it for itself): the parts' join is a second launch, 4
// to 5 us and what the host takes.  By the call's longest sequence, since it waits for the
// slowest; for blocks that have a CU to themselves, half of it where two share one.  8
// sequences, us in one launch / two: 1 token over int8 900 positions 9.8 / 14.0, 2000 14.0
// / 14.4, 3000 17.9 / 15; bf16 900 10.9 / 13.8, 2000 16.4 / 16.8; fp32 700 14.4 / 16.4,
// 1500 21 / 17; 3 tokens over int8 1000 9.9 / 15.3, 1800 13.6 / 15.6, 5 tokens 1000 12.6 /
// 16.2, 1800 17.5 / 16.3, 20 tokens 500 13.1 / 17, 1000 18.9 / 17.8; 5 tokens over fp32
// 500 14.1 / 18.7, 900 20.1 / 17.4.  1 token over 300 int8 positions behind 700 shared
// 10.4 / 16.8, 700 behind 1700 15.6 / 16.3, 100 behind 3000 18.5 / 16.6; 64 sequences of
// 300 bf16 behind 1200 23.1 / 18.7, 100 behind 300 12.7 / 17.2.
static int whole_tiles(int format, int ct, int waves) {
  return waves * (format == LFM_KV_F32 ? (ct <= 1 ? 4 : 3) : ct <= 1 ? 8 : ct == 2 ? 6 : 3);
}

static FlashPlan flash_plan(const KvArgs &a, int heads) {
  FlashPlan p{};
  const long long group = heads / a.kv_heads, cap = (long long)a.max_pages << a.pshift;
  const long long own = a.max_new * group, all = a.tokens * group;
  p.own_ct = own <= kFewCols ? 0 : own <= 16 ? 1 : std::min(widest(a.format), own <= 32 ? 2 : 4);
  p.own_groups = (int)((own + columns_of(p.own_ct) - 1) / columns_of(p.own_ct));
  p.own_parts = 1;
  const int keys = (int)std::min<long long>(a.max_len ? a.max_len : cap, cap);
  const long long own_base = (long long)p.own_groups * a.kv_heads * std::max(a.batch, 1);
  const int most = active_parts(keys, kMostParts);
  const float own_time = (float)keys * tile_cost(p.own_ct);  // of a wave
  const long long own_slots = kFlashCUs * flash_waves(a.format, p.own_ct) * 4 / own_waves(p.own_ct);
  const int tiles = (keys + kKeys - 1) / kKeys + (a.prefix_len + kKeys - 1) / kKeys;
  p.wide = p.own_ct > 0 && own_base <= kFlashCUs;
  if (own_base <= own_slots && tiles * ((own_base + kFlashCUs - 1) / kFlashCUs) <
                                   whole_tiles(a.format, p.own_ct, p.wide ? kWideWaves : own_waves(p.own_ct)))
    return p;
  p.wide = false;
  if (a.prefix_len == 0) {
    p.own_parts = (int)std::min<long long>(most, std::max<long long>(1, own_slots / own_base));
    return p;
  }
  p.prefix_ct = all <= 16 && p.own_ct <= 1 ? 1 : widest(a.format);
  p.prefix_groups = (int)((all + columns_of(p.prefix_ct) - 1) / columns_of(p.prefix_ct));
  p.prefix_parts = 1;
  const long long prefix_base = (long long)p.prefix_groups * a.kv_heads;
  const int prefix_most = active_parts(a.prefix_len, kMostParts);
  const float prefix_time = (float)a.prefix_len * tile_cost(p.prefix_ct);
  const long long slots = kFlashCUs * flash_waves(a.format, p.prefix_ct);
  const long long budget = std::max(slots, own_base + (a.prefix_len > kLongPrefix ? slots : slots / 2));
  for (;;) {
    const bool prefix = prefix_time * p.own_parts >= own_time * p.prefix_parts;
    int &parts = prefix ? p.prefix_parts : p.own_parts;
    if (parts >= (prefix ? prefix_most : most)) break;
    if (own_base * p.own_parts + prefix_base * p.prefix_parts + (prefix ? prefix_base : own_base) > budget) break;
    ++parts;
  }
  return p;
}

static size_t flash_rows(const KvArgs &a, int heads) { return (size_t)a.tokens * heads; }

size_t kv_attention_ws(const KvArgs &a, int heads) {
  const FlashPlan p = flash_plan(a, heads);
  const int parts = p.own_parts + p.prefix_parts;
  return parts == 1 ? 0 : flash_rows(a, heads) * parts * (kRowDim + 2) * sizeof(float);
}

// f with `ct` as a compile-time constant.
template <int MOST, typename F>
static hipError_t by_columns(int ct, F &&f) {
  switch (ct) {
    case 0: return f(std::integral_constant<int, 0>{});
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    default: return f(std::integral_constant<int, MOST>{});
  }
}

hipError_t launch_kv_attention(const KvArgs &a, const float *q, int ld, float *out, int ldo, int heads, void *ws,
                               hipStream_t st) {
  const FlashPlan p = flash_plan(a, heads);
  const size_t rows = flash_rows(a, heads);
  float *po = static_cast<float *>(ws);
  const FlashArgs f{q, out, po, reinterpret_cast<float2 *>(po + rows * (p.own_parts + p.prefix_parts) * kRowDim),
                    ld, ldo, heads, heads / a.kv_heads, p.own_parts, p.prefix_parts, rows};
  const long long own_blocks = (long long)a.kv_heads * p.own_parts * p.own_groups * a.batch;
  const long long prefix_blocks = (long long)a.kv_heads * p.prefix_parts * p.prefix_groups;
  // beside a prefix all blocks are in x, whose threads are counted in 32 bits
  if (p.own_groups > 65535 || own_blocks + prefix_blocks > (p.prefix_parts ? 0xFFFFFF : 0x7FFFFFFF))
    return hipErrorInvalidValue;
  return by_format(a.format, [&](auto fmt) -> hipError_t {
    constexpr int FMT = fmt(), MOST = FMT == LFM_KV_F32 ? 2 : 4;
    hipError_t e = by_columns<MOST>(p.own_ct, [&](auto own) -> hipError_t {
      constexpr int CT = own();
      constexpr int W = own_waves(CT), WIDE = CT == 0 ? W : kWideWaves;
      const dim3 grid(a.kv_heads * p.own_parts, p.own_groups, a.batch), block(64 * (p.wide ? WIDE : W));
      if (a.prefix_len == 0 && p.wide)
        hipLaunchKernelGGL((kv_flash_kernel<FMT, CT, kOwnKeys, WIDE>), grid, block, 0, st, a, f);
      else if (a.prefix_len == 0)
        hipLaunchKernelGGL((kv_flash_kernel<FMT, CT, kOwnKeys, W>), grid, block, 0, st, a, f);
      else if (p.wide)
        hipLaunchKernelGGL((kv_flash_kernel<FMT, CT, kBothKeys, WIDE>), grid, block, 0, st, a, f);
      else if (p.prefix_parts == 0)
        hipLaunchKernelGGL((kv_flash_kernel<FMT, CT, kBothKeys, W>), grid, block, 0, st, a, f);
      else if (p.prefix_ct == 1)
        hipLaunchKernelGGL((kv_prefix_flash_kernel<FMT, 1, CT < 1 ? CT : 1>), dim3((unsigned)(prefix_blocks + own_blocks)),
                           dim3(256), 0, st, a, f, (int)prefix_blocks, p.own_groups);
      else
        hipLaunchKernelGGL((kv_prefix_flash_kernel<FMT, MOST, CT>), dim3((unsigned)(prefix_blocks + own_blocks)),
                           dim3(256), 0, st, a, f, (int)prefix_blocks, p.own_groups);
      return hipGetLastError();
    });
    if (e == hipSuccess && p.own_parts + p.prefix_parts > 1) {
      hipLaunchKernelGGL(kv_join_kernel, dim3((unsigned)((a.max_new * (long long)heads + 3) / 4), a.batch), dim3(256), 0,
                         st, a, f);
      e = hipGetLastError();
    }
    return e;
  });
}

}  // namespace lfm
