// HIP kernels from logits to tokens (gfx950): softmax with a temperature, and
// verification of drafted tokens against the target's probabilities.
#include <algorithm>

#include "gpu_common.h"
#include "lfm_internal.h"

namespace lfm {

using moe::f32x4;

// ---------------------------------------------------------------------------
// Softmax
// ---------------------------------------------------------------------------
//
// A row's maximum and its sum of exponentials under that maximum, in fp32, then
// the quotients.  A block's threads keep the values they loaded, so a row of up to
// 65536 is read once; longer rows are split over blocks that leave their maximum and
// sum in the workspace to a second kernel, which reads the row again (from L2).  An
// exponential is 2 to the power of the rounded difference times c = log2(e) /
// temperature: v_exp_f32 does it in one instruction, where expf's 15 made a row's
// 65536 values 9 us of arithmetic.  Memory bounds many rows (320 of 65536, 168 MB: 33
// us, 5.1 TB/s; a CU holds one row, so the first 256 all read and then all write), and
// the chain load, maximum, sum, store few (1 row: 6.9 us).

constexpr int kSoftThreads = 1024;
constexpr int kSoftRegs = 64;        // values a thread keeps
constexpr int kSoftRow = kSoftThreads * kSoftRegs;
constexpr int kSliceThreads = 256;   // a slice of a split row
constexpr int kSliceRegs = 16;
constexpr int kSlice = kSliceThreads * kSliceRegs;

struct MaxSum {
  float m, l;
};

// What a sum under maximum `m` counts under `mx` (a part with nothing but
// -infinity has sum 0, or NaN with a NaN in it).
__device__ __forceinline__ float rescale(float m, float mx, float c) {
  return m == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f((m - mx) * c);
}

// Over groups of N lanes.
template <int N = 64>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int d = N / 2; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}

template <int N = 64>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int d = N / 2; d > 0; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// A thread's values of a row: groups of four, the j-th at 4 (j * threads + t), and one
// of the last n % 4.  Groups are loaded and stored as they lie: a row of odd length
// puts the next one's at any multiple of 4 bytes, and a wave's 1 KiB then touches one
// cache line more (320 rows of 31999: 14.9 us, as of 32000; value by value 45).
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

template <int NR>
struct RowValues {
  f32x4 v[NR / 4];
  float tail;
};

// Values [0, n) of x; -infinity where there are none.
template <int NW, int NR>
__device__ __forceinline__ void load_values(const float *x, int n, RowValues<NR> &r) {
  const int groups = n >> 2, tid = threadIdx.x;
#pragma unroll
  for (int j = 0; j < NR / 4; ++j) {
    const int i = j * NW * 64 + tid;
    r.v[j] = i < groups ? f32x4(*reinterpret_cast<const f32x4_any *>(x + 4 * i)) : f32x4(-__builtin_inff());
  }
  r.tail = tid < (n & 3) ? x[4 * groups + tid] : -__builtin_inff();
}

// Stores past the caches, so that the logits, which the head has just written, are not
// driven out of the last one (256 MB) while they are read: 320 rows of 65536 take 33
// us instead of 41 where they are there, 39 either way where they come from HBM.  A copy
// of the logits, this and verification of 64 x 5 rows together 77 us instead of 84
// (in place 76 either way).
template <int NW, int NR>
__device__ __forceinline__ void store_values(float *y, int n, const RowValues<NR> &r, float scale) {
  const int groups = n >> 2, tid = threadIdx.x;
#pragma unroll
  for (int j = 0; j < NR / 4; ++j) {
    const int i = j * NW * 64 + tid;
    if (i < groups) __builtin_nontemporal_store(f32x4_any(r.v[j] * scale), reinterpret_cast<f32x4_any *>(y + 4 * i));
  }
  if (tid < (n & 3)) y[4 * groups + tid] = r.tail * scale;
}

// The values become exp((v - ref) / t); their sum.  -infinity gives 0 whatever ref is.
template <int NR>
__device__ __forceinline__ float exp_values(RowValues<NR> &r, float ref, float c) {
  r.tail = __builtin_amdgcn_exp2f((r.tail - ref) * c);
  float l = r.tail;
#pragma unroll
  for (int j = 0; j < NR / 4; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      r.v[j][e] = __builtin_amdgcn_exp2f((r.v[j][e] - ref) * c);
      l += r.v[j][e];
    }
  return l;
}

// A block's maximum and its sum of exponentials under it.  The values become
// exponentials under their thread's own maximum, with no barrier between loads and
// exponentials, so that a wave's run while others still load; `mine` is what they
// count under the block's.
template <int NW, int NR>
__device__ __forceinline__ MaxSum block_exp(RowValues<NR> &r, float c, float2 *s_part, float &mine) {
  float m = r.tail;
#pragma unroll
  for (int j = 0; j < NR / 4; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) m = fmaxf(m, r.v[j][e]);
  float l = exp_values(r, m == -__builtin_inff() ? 0.0f : m, c);
  float mx = lanes_max(m);
  l = lanes_sum(l * rescale(m, mx, c));
  if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = float2{mx, l};
  __syncthreads();
  const float2 p = s_part[threadIdx.x & (NW - 1)];  // a wave's in each of NW lanes
  mx = lanes_max<NW>(p.x);
  l = lanes_sum<NW>(p.y * rescale(p.x, mx, c));
  mine = rescale(m, mx, c);
  return {mx, l};
}

__device__ __forceinline__ float inverse_sum(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }

// A row a block, NR values a thread.
template <int NR>
__global__ __launch_bounds__(kSoftThreads) __attribute__((amdgpu_waves_per_eu(NR <= 32 ? 8 : 4)))
void softmax_row_kernel(const float *x, long long xs, float *y, long long ys, int dim, float c) {
  constexpr int NW = kSoftThreads / 64;
  __shared__ float2 s_part[NW];
  x += blockIdx.x * xs;
  y += blockIdx.x * ys;
  RowValues<NR> v;
  load_values<NW, NR>(x, dim, v);
  float mine;
  const MaxSum r = block_exp<NW, NR>(v, c, s_part, mine);
  store_values<NW, NR>(y, dim, v, mine * inverse_sum(r.l));
}

// A slice of a row a block: its maximum and sum.
__global__ __launch_bounds__(kSliceThreads) void softmax_part_kernel(const float *x, long long xs, float2 *part, int dim,
                                                                     float c) {
  constexpr int NW = kSliceThreads / 64;
  __shared__ float2 s_part[NW];
  const int first = blockIdx.x * kSlice, n = min(dim - first, kSlice);
  RowValues<kSliceRegs> v;
  load_values<NW, kSliceRegs>(x + blockIdx.y * xs + first, n, v);
  float mine;
  const MaxSum r = block_exp<NW, kSliceRegs>(v, c, s_part, mine);
  if (threadIdx.x == 0) part[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = float2{r.m, r.l};
}

__global__ __launch_bounds__(kSliceThreads) void softmax_finish_kernel(const float *x, long long xs, float *y,
                                                                       long long ys, const float2 *part, int dim,
                                                                       float c) {
  constexpr int NW = kSliceThreads / 64;
  const int first = blockIdx.x * kSlice, n = min(dim - first, kSlice), lane = threadIdx.x & 63;
  RowValues<kSliceRegs> v;
  load_values<NW, kSliceRegs>(x + blockIdx.y * xs + first, n, v);
  // every wave joins the row's parts by itself
  const float2 *p = part + (size_t)blockIdx.y * gridDim.x;
  float m = -__builtin_inff();
  for (int i = lane; i < (int)gridDim.x; i += 64) m = fmaxf(m, p[i].x);
  m = lanes_max(m);
  const float ref = m == -__builtin_inff() ? 0.0f : m;
  float l = 0.0f;
  for (int i = lane; i < (int)gridDim.x; i += 64) l += p[i].y * rescale(p[i].x, ref, c);
  const float inv = inverse_sum(lanes_sum(l));
  exp_values(v, ref, c);
  store_values<NW, kSliceRegs>(y + blockIdx.y * ys + first, n, v, inv);
}

// A row of up to kSoftRow values is one block's, however few the rows: split over
// blocks that leave their sums to a second launch, 1 row of 65536 takes 6.5 us and 8
// blocks that read it all and write an eighth each 7.1, one block 6.9; 64 rows 12.0 /
// 12.1 / 11.3, 320 rows 46 split, 42 in blocks, 43 with the last 64 split (all with
// stores through the caches).
constexpr int kShortRow = 8 * kSoftThreads, kMidRow = 32 * kSoftThreads;

size_t softmax_ws(int rows, int dim) {
  return dim <= kSoftRow ? 0 : (size_t)rows * ((dim + kSlice - 1) / kSlice) * sizeof(float2);
}

static void softmax_rows_launch(const float *x, long long xs, float *y, long long ys, int rows, int dim, float c,
                                hipStream_t st) {
  const dim3 grid(rows), block(kSoftThreads);
  if (dim <= kShortRow)
    hipLaunchKernelGGL(softmax_row_kernel<8>, grid, block, 0, st, x, xs, y, ys, dim, c);
  else if (dim <= kMidRow)
    hipLaunchKernelGGL(softmax_row_kernel<32>, grid, block, 0, st, x, xs, y, ys, dim, c);
  else
    hipLaunchKernelGGL(softmax_row_kernel<64>, grid, block, 0, st, x, xs, y, ys, dim, c);
}

hipError_t launch_softmax(const float *x, long long xs, float *y, long long ys, int rows, int dim,
                          float temperature, void *ws, hipStream_t st) {
  const float c = (float)(1.4426950408889634 / (double)temperature);
  if (dim <= kSoftRow) {
    constexpr int kMostRows = 1 << 21;  // of a launch: its threads are counted in 32 bits
    for (long long r0 = 0; r0 < rows; r0 += kMostRows)
      softmax_rows_launch(x + r0 * xs, xs, y + r0 * ys, ys, (int)std::min<long long>(rows - r0, kMostRows), dim, c, st);
    return hipGetLastError();
  }
  const int slices = (dim + kSlice - 1) / kSlice;
  float2 *part = static_cast<float2 *>(ws);
  for (long long r0 = 0; r0 < rows; r0 += 65535) {  // rows a launch may have
    const dim3 grid(slices, (unsigned)std::min<long long>(rows - r0, 65535));
    float2 *p = part + (size_t)r0 * slices;
    hipLaunchKernelGGL(softmax_part_kernel, grid, dim3(kSliceThreads), 0, st, x + r0 * xs, xs, p, dim, c);
    hipLaunchKernelGGL(softmax_finish_kernel, grid, dim3(kSliceThreads), 0, st, x + r0 * xs, xs, y + r0 * ys, ys, p, dim,
                       c);
  }
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Verification of drafted tokens
// ---------------------------------------------------------------------------
//
// Only the row that a token is drawn from is read, and the draft's at a
// rejection.  Sums are 64-bit, so that which id a random number falls on does
// not hang on their order: a slice of kDrawSlice weights a block leaves two
// sums (of the weights after a rejection, and of the target alone, for where
// those have no positive sum), and a second kernel finds the slice, then the id
// in it.  Every block of the first decides by itself which row that is.  64
// sequences' rows of 65536 (up to 34 MB) take 8.0 + 4.5 us, near memory's rate in the
// first; one sequence's 3.6 + 3.3, two launches and their chains of loads.

constexpr int kDrawThreads = 256;
constexpr int kDrawRegs = 8;
constexpr int kDrawSlice = kDrawThreads * kDrawRegs;

// Accepted drafts of sequence b, found by one wave, 64 drafts at a time (exact:
// a product of two fp32 values is exact in 64 bits).
__device__ __forceinline__ int accepted_drafts(const VerifyArgs &a, int b, int n) {
  const int lane = threadIdx.x & 63;
  for (int i0 = 0; i0 < a.n_draft; i0 += 64) {
    const int i = i0 + lane;
    bool ok = i < a.n_draft;
    if (ok) {
      const size_t at = (size_t)b * a.n_draft + i;
      const int id = a.ids[b * a.ids_stride + i];
      const float u = a.u_accept[at];
      ok = id >= 0 && id < a.vocab;
      if (ok) {
        const float q = a.draft[at * a.vocab + id];
        const float p = a.target[(at + b) * a.vocab + id];  // [b][n_draft + 1]
        ok = (double)u * (double)q < (double)p;
      }
    }
    const unsigned long long no = __ballot(!ok);
    if (no) return min(i0 + __builtin_ctzll(no), n);
  }
  return n;
}

// max(p - q, 0); NaN counts as 0.
__device__ __forceinline__ double weight(float p, float q) {
  const double d = (double)p - (double)q;
  return d > 0.0 ? d : 0.0;
}

// Four of a row's neighbouring values a thread and step; 0 behind the row.
template <int NW, int NR>
__device__ __forceinline__ void load_weights(const float *x, int n, RowValues<NR> &r) {
#pragma unroll
  for (int j = 0; j < NR / 4; ++j) {
    const int i = 4 * (j * NW * 64 + (int)threadIdx.x);
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (i + 4 <= n) {
      v = *reinterpret_cast<const f32x4_any *>(x + i);
    } else {
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (i + e < n) v[e] = x[i + e];
    }
    r.v[j] = v;
  }
}

struct DrawRow {
  const float *p, *q;  // q null: the target alone
};

__device__ __forceinline__ int drafts_of(const VerifyArgs &a, int b) {
  return a.n_valid ? min(max(a.n_valid[b], 0), a.n_draft) : a.n_draft;
}

// The row that the token after `acc` accepted drafts is drawn from.
__device__ __forceinline__ DrawRow row_after(const VerifyArgs &a, int b, int acc, int n) {
  return {a.target + ((size_t)b * (a.n_draft + 1) + acc) * a.vocab,
          acc < n ? a.draft + ((size_t)b * a.n_draft + acc) * a.vocab : nullptr};
}

// Inclusive running sum over a wave, and its total: row shifts by 1, 2, 4, 8,
// then the sums of a row of 16 and of the lower half broadcast upwards.  (DPP
// moves of the two halves; shuffles through LDS took twice the kernel's time.)
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_up(double v) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}

__device__ __forceinline__ double scan(double v) {
  v += dpp_up<0x111, 0xf>(v);
  v += dpp_up<0x112, 0xf>(v);
  v += dpp_up<0x114, 0xf>(v);
  v += dpp_up<0x118, 0xf>(v);
  v += dpp_up<0x142, 0xa>(v);
  return v + dpp_up<0x143, 0xc>(v);
}

__device__ __forceinline__ double lane_value(double v, int lane) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}

// Sum of one value of each thread, the same order in every thread.
__device__ __forceinline__ double block_sum(double v, double *s_part) {
  v = lane_value(scan(v), 63);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = s_part[0];
#pragma unroll
  for (int w = 1; w < kDrawThreads / 64; ++w) v += s_part[w];
  return v;
}

__global__ __launch_bounds__(kDrawThreads) void draw_sums_kernel(VerifyArgs a, double2 *sums) {
  __shared__ double s_part[kDrawThreads / 64];
  const int b = blockIdx.y, first = blockIdx.x * kDrawSlice;
  const int n = drafts_of(a, b);
  const int acc = accepted_drafts(a, b, n);
  const DrawRow r = row_after(a, b, acc, n);
  if (blockIdx.x == 0 && threadIdx.x == 0) a.accepted[b] = acc;
  double rest = 0.0, whole = 0.0;
  const float *q = r.q ? r.q : r.p;
  float pv[kDrawRegs], qv[kDrawRegs];  // every load without a branch: they are in flight together
#pragma unroll
  for (int j = 0; j < kDrawRegs; ++j) {
    const int v = min(first + j * kDrawThreads + (int)threadIdx.x, a.vocab - 1);
    pv[j] = r.p[v];
    qv[j] = q[v];
  }
#pragma unroll
  for (int j = 0; j < kDrawRegs; ++j) {
    const bool there = first + j * kDrawThreads + (int)threadIdx.x < a.vocab;
    whole += there ? weight(pv[j], 0.0f) : 0.0;
    rest += there ? weight(pv[j], qv[j]) : 0.0;
  }
  whole = block_sum(whole, s_part);
  if (r.q) rest = block_sum(rest, s_part);
  if (threadIdx.x == 0) sums[(size_t)b * gridDim.x + blockIdx.x] = double2{rest, whole};
}

// The lowest id up to which the weights sum to more than u times their whole
// sum; one block per sequence.  Every wave finds the slice, then each of the
// 1024 threads takes two of its weights.  (With LDS atomics for the lowest id,
// which the compiler turns into a loop over a wave's lanes, it took 8.5 us.)
constexpr int kTokenThreads = 1024, kTokenRegs = kDrawSlice / kTokenThreads;

__global__ __launch_bounds__(kTokenThreads) void draw_token_kernel(VerifyArgs a, const double2 *sums, int slices) {
  __shared__ double s_part[kTokenThreads / 64];
  __shared__ int s_token[kTokenThreads / 64], s_last[kTokenThreads / 64];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int acc = a.accepted[b];
  const float u = a.u_sample[b];
  const int n = drafts_of(a, b);  // every load that hangs on nothing stands in front
  const int id = tid < a.n_draft ? a.ids[b * a.ids_stride + tid] : -1;
  sums += (size_t)b * slices;
  // lane l holds the sums of `each` neighbouring slices
  const int each = (slices + 63) / 64, i0 = lane * each, i1 = min(i0 + each, slices);
  double rest = 0.0, whole = 0.0;
  for (int i = i0; i < i1; ++i) {
    rest += sums[i].x;
    whole += sums[i].y;
  }
  const DrawRow r = row_after(a, b, acc, n);
  bool use_rest = r.q != nullptr;
  double mine = use_rest ? rest : whole, incl, total;
  for (;;) {
    incl = scan(mine);
    total = lane_value(incl, 63);
    if (!use_rest || total > 0.0) break;
    use_rest = false;
    mine = whole;
  }
  const double bar = (double)u * total;
  const unsigned long long hit = __ballot(incl > bar && mine > 0.0);
  int token = -1;
  if (hit) {
    const int at = __builtin_ctzll(hit);
    double run = lane_value(incl - mine, at);
    int slice = at * each;
    for (int i = slice; i < min(slice + each, slices) - 1; ++i) {  // uniform
      const double next = run + (use_rest ? sums[i].x : sums[i].y);
      if (next > bar) break;
      run = next;
      ++slice;
    }
    const int v0 = slice * kDrawSlice + tid * kTokenRegs;
    const float *q = r.q ? r.q : r.p;
    float pv[kTokenRegs], qv[kTokenRegs];
#pragma unroll
    for (int j = 0; j < kTokenRegs; ++j) {
      pv[j] = r.p[min(v0 + j, a.vocab - 1)];
      qv[j] = q[min(v0 + j, a.vocab - 1)];
    }
    double w[kTokenRegs], sum = 0.0;
#pragma unroll
    for (int j = 0; j < kTokenRegs; ++j) {
      w[j] = v0 + j < a.vocab ? weight(pv[j], use_rest ? qv[j] : 0.0f) : 0.0;
      sum += w[j];
    }
    const double upto = scan(sum);
    if (lane == 63) s_part[tid >> 6] = upto;
    __syncthreads();
    // a wave's first id past the bar and its last id of any weight, by lane order
    const int wave = tid >> 6;
    sum = run + (upto - sum);
    for (int i = 0; i < wave; ++i) sum += s_part[i];
    int past = -1, last = -1;
#pragma unroll
    for (int j = 0; j < kTokenRegs; ++j) {
      sum += w[j];
      if (w[j] > 0.0) {
        last = v0 + j;
        if (past < 0 && sum > bar) past = v0 + j;
      }
    }
    const unsigned long long is_past = __ballot(past >= 0), is_last = __ballot(last >= 0);
    const int first_past = is_past ? __builtin_amdgcn_readlane(past, __builtin_ctzll(is_past)) : -1;
    const int at_last = is_last ? __builtin_amdgcn_readlane(last, 63 - __builtin_clzll(is_last)) : -1;
    if (lane == 0) {
      s_token[wave] = first_past;
      s_last[wave] = at_last;
    }
    __syncthreads();
    // the slice's sum was taken in another order: where only that passes the
    // bar, the slice's last id it is
    for (int i = kTokenThreads / 64 - 1; i >= 0; --i) token = max(token, s_last[i]);
    for (int i = kTokenThreads / 64 - 1; i >= 0; --i)
      if (s_token[i] >= 0) token = s_token[i];
  }
  int *out = a.tokens + (size_t)b * (a.n_draft + 1);
  if (tid <= a.n_draft) out[tid] = tid < acc ? id : tid == acc ? token : -1;
  if (tid == 0 && a.n_draft == kTokenThreads) out[a.n_draft] = acc == a.n_draft ? token : -1;
}

// The same in one launch where a block's threads hold the row (and the draft's): four
// ids a thread, 4096 a step of the block, so that a wave's four of a step are a segment
// of 256 neighbouring ids.  Every wave finds the segment from the segments' sums, and
// the one that holds it the id.  Calls one after the other, 64 sequences of 16384 ids: 5.0
// us, of which the launch on the host is most, two launches 7.8.  With 32 ids a thread
// (24000 to 32768) the registers do not hold the 64-bit sums as well: 10.3 us, two
// launches 8.6.
template <int NR>
__global__ __launch_bounds__(kTokenThreads) void draw_whole_kernel(VerifyArgs a) {
  constexpr int NW = kTokenThreads / 64, G = NR / 4, SEGS = G * NW, EACH = (SEGS + 63) / 64;
  __shared__ double s_seg[SEGS];
  __shared__ int s_token;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float u = a.u_sample[b];
  const int n = drafts_of(a, b);
  const int id = tid < a.n_draft ? a.ids[b * a.ids_stride + tid] : -1;
  const int acc = accepted_drafts(a, b, n);
  const DrawRow r = row_after(a, b, acc, n);
  RowValues<NR> p, q;
  load_weights<NW, NR>(r.p, a.vocab, p);
  load_weights<NW, NR>(r.q ? r.q : r.p, r.q ? a.vocab : 0, q);  // zeros without one
  bool use_rest = r.q != nullptr;
  auto four = [&](int j, double (&w)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = weight(p.v[j][e], q.v[j][e]);
  };
  double mine[EACH], sum, incl, total;
  for (;;) {
#pragma unroll
    for (int j = 0; j < G; ++j) {
      double w[4];
      four(j, w);
      const double seg = scan((w[0] + w[1]) + (w[2] + w[3]));
      if (lane == 63) s_seg[j * NW + wave] = seg;
      __builtin_amdgcn_sched_barrier(0);  // or every step's 64-bit sums are held at once, and spill
    }
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int at = lane * EACH + i;
      mine[i] = at < SEGS ? s_seg[at] : 0.0;
      sum += mine[i];
    }
    incl = scan(sum);
    total = lane_value(incl, 63);
    if (!use_rest || total > 0.0) break;
    use_rest = false;
#pragma unroll
    for (int j = 0; j < G; ++j) q.v[j] = f32x4(0.0f);
    __syncthreads();
  }
  const double bar = (double)u * total;
  const unsigned long long hit = __ballot(incl > bar && sum > 0.0);
  int token = -1;
  if (hit) {  // the same in every wave
    const int at = __builtin_ctzll(hit);
    double run = lane_value(incl - sum, at);
    int seg = at * EACH;
#pragma unroll
    for (int i = 0; i < EACH - 1; ++i) {
      const double next = run + lane_value(mine[i], at);
      if (seg == at * EACH + i && !(next > bar)) {
        run = next;
        ++seg;
      }
    }
    if (seg % NW == wave) {
      double w[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
      for (int j = 0; j < G; ++j) {
        asm("" : "+v"(p.v[j]));  // or the weights, of 64 bits each, are kept from above
        if (j == seg / NW) four(j, w);
      }
      const double own = (w[0] + w[1]) + (w[2] + w[3]);
      double upto = run + (scan(own) - own);
      const int first = seg / NW * (4 * kTokenThreads) + 4 * tid;
      int past = -1, last = -1;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        upto += w[e];
        if (w[e] > 0.0) {
          last = first + e;
          if (past < 0 && upto > bar) past = first + e;
        }
      }
      // the segment's sum was taken in another order: where only that passes the
      // bar, the segment's last id it is
      const unsigned long long is_past = __ballot(past >= 0), is_last = __ballot(last >= 0);
      if (is_past)
        token = __builtin_amdgcn_readlane(past, __builtin_ctzll(is_past));
      else if (is_last)
        token = __builtin_amdgcn_readlane(last, 63 - __builtin_clzll(is_last));
      if (lane == 0) s_token = token;
    }
    __syncthreads();
    token = s_token;
  }
  if (tid == 0) a.accepted[b] = acc;
  int *out = a.tokens + (size_t)b * (a.n_draft + 1);
  if (tid <= a.n_draft) out[tid] = tid < acc ? id : tid == acc ? token : -1;
  if (tid == 0 && a.n_draft == kTokenThreads) out[a.n_draft] = acc == a.n_draft ? token : -1;
}

constexpr int kWholeVocab = 16 * kTokenThreads;  // ids of a row that a block holds

size_t verify_draft_ws(int batch, int vocab) {
  if (vocab <= kWholeVocab) return 0;
  return (size_t)batch * (((size_t)vocab + kDrawSlice - 1) / kDrawSlice) * sizeof(double2);
}

hipError_t launch_verify_draft(const VerifyArgs &a, void *ws, hipStream_t st) {
  if (a.vocab <= kWholeVocab) {
    const dim3 grid(a.batch), block(kTokenThreads);
    if (a.vocab <= 8 * kTokenThreads)
      hipLaunchKernelGGL(draw_whole_kernel<8>, grid, block, 0, st, a);
    else
      hipLaunchKernelGGL(draw_whole_kernel<16>, grid, block, 0, st, a);
    return hipGetLastError();
  }
  const int slices = (int)(((size_t)a.vocab + kDrawSlice - 1) / kDrawSlice);
  double2 *sums = static_cast<double2 *>(ws);
  hipLaunchKernelGGL(draw_sums_kernel, dim3(slices, a.batch), dim3(kDrawThreads), 0, st, a, sums);
  hipLaunchKernelGGL(draw_token_kernel, dim3(a.batch), dim3(kTokenThreads), 0, st, a, sums, slices);
  return hipGetLastError();
}

}  // namespace lfm
