// HIP kernels from logits to tokens (gfx950): softmax with a temperature, and
// verification of drafted tokens against the target's probabilities.
#include "gpu_common.h"
#include "lfm_internal.h"

namespace lfm {

// ---------------------------------------------------------------------------
// Softmax
// ---------------------------------------------------------------------------

constexpr int kSoftThreads = 1024;

template <typename F>
__device__ __forceinline__ float block_fold(float v, float *s_part, F f) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = f(v, __shfl_xor(v, d));
  __syncthreads();  // readers of the fold before this one are done
  if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = s_part[0];
  for (int i = 1; i < kSoftThreads / 64; ++i) v = f(v, s_part[i]);
  return v;
}

__global__ __launch_bounds__(kSoftThreads) void softmax_kernel(const float *x, long long xs, float *y, long long ys,
                                                               int dim, float inv_t) {
  __shared__ float s_part[kSoftThreads / 64];
  x += blockIdx.x * xs;
  y += blockIdx.x * ys;
  float m = -__builtin_inff();
  for (int i = threadIdx.x; i < dim; i += kSoftThreads) m = fmaxf(m, x[i]);
  m = block_fold(m, s_part, [](float p, float q) { return fmaxf(p, q); });
  if (m == -__builtin_inff()) m = 0.0f;
  float l = 0.0f;
  for (int i = threadIdx.x; i < dim; i += kSoftThreads) l += expf((x[i] - m) * inv_t);
  l = block_fold(l, s_part, [](float p, float q) { return p + q; });
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  for (int i = threadIdx.x; i < dim; i += kSoftThreads) y[i] = expf((x[i] - m) * inv_t) * inv;
}

size_t softmax_ws(int, int) { return 0; }

hipError_t launch_softmax(const float *x, long long xs, float *y, long long ys, int rows, int dim,
                          float temperature, void *, hipStream_t st) {
  hipLaunchKernelGGL(softmax_kernel, dim3(rows), dim3(kSoftThreads), 0, st, x, xs, y, ys, dim, 1.0f / temperature);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Verification of drafted tokens
// ---------------------------------------------------------------------------

// Accepted drafts of sequence b (one thread's work; exact: a product of two
// fp32 values is exact in 64 bits).
__device__ inline int accepted_drafts(const VerifyArgs &a, int b, int n) {
  for (int i = 0; i < n; ++i) {
    const int id = a.ids[(size_t)b * a.n_draft + i];
    if (id < 0 || id >= a.vocab) return i;
    const float q = a.draft[((size_t)b * a.n_draft + i) * a.vocab + id];
    const float p = a.target[((size_t)b * (a.n_draft + 1) + i) * a.vocab + id];
    if (!((double)a.u_accept[(size_t)b * a.n_draft + i] * (double)q < (double)p)) return i;
  }
  return n;
}

// max(p - q, 0) in 64 bits, where the difference of two fp32 values of like
// size is exact; NaN counts as 0.
__device__ __forceinline__ double weight(float p, float q) {
  const double d = (double)p - (double)q;
  return d > 0.0 ? d : 0.0;
}

// One thread per sequence.
__global__ __launch_bounds__(64) void verify_kernel(VerifyArgs a) {
  const int b = blockIdx.x * 64 + threadIdx.x;
  if (b >= a.batch) return;
  const int n = a.n_valid ? min(max(a.n_valid[b], 0), a.n_draft) : a.n_draft;
  const int acc = accepted_drafts(a, b, n);
  const float *p = a.target + ((size_t)b * (a.n_draft + 1) + acc) * a.vocab;
  const float *q = acc < n ? a.draft + ((size_t)b * a.n_draft + acc) * a.vocab : nullptr;
  double total = 0.0;
  for (int v = 0; v < a.vocab; ++v) total += weight(p[v], q ? q[v] : 0.0f);
  if (q && !(total > 0.0)) {
    q = nullptr;
    total = 0.0;
    for (int v = 0; v < a.vocab; ++v) total += weight(p[v], 0.0f);
  }
  const double bar = (double)a.u_sample[b] * total;
  int token = -1;
  double sum = 0.0;
  for (int v = 0; v < a.vocab && token < 0; ++v) {
    sum += weight(p[v], q ? q[v] : 0.0f);
    if (sum > bar) token = v;
  }
  a.accepted[b] = acc;
  for (int i = 0; i <= a.n_draft; ++i)
    a.tokens[(size_t)b * (a.n_draft + 1) + i] = i < acc ? a.ids[(size_t)b * a.n_draft + i] : i == acc ? token : -1;
}

size_t verify_draft_ws(int, int) { return 0; }

hipError_t launch_verify_draft(const VerifyArgs &a, void *, hipStream_t st) {
  hipLaunchKernelGGL(verify_kernel, dim3((a.batch + 63) / 64), dim3(64), 0, st, a);
  return hipGetLastError();
}

}  // namespace lfm
