// RMSNorm and rotation of a head's row of 64 held by 16 lanes, bit for bit the
// reference's (rms_norm_kernel, layer.cu:144-193, on a 64-wide row;
// rope_transpose_kernel, layer.cu:217-228).
#pragma once

#include "gpu_common.h"

namespace lfm {

// Lane l of 16 holds elements 4l .. 4l+3 of x, the norm weight w and the
// position's cos and sin rows; every lane of the wave takes part.  The norm
// is launched with 256 threads there (layer.cu:1146): threads 0..63 hold one
// square each (fmaf(x, x, 0) = x*x), warps 0 and 1 fold elements 0..31 and
// 32..63 with shuffle-down at 16..1, and the 8-warp fold adds warps 2..7's
// zeros, which leaves warp0 + warp1.  The same binary tree runs here over the
// float4 layout (16 -> 4 lanes down, 8 -> 2 lanes, 4 -> 1 lane, then 2 and 1
// across a lane's components), so every addition is the reference's.  Then
// out[d] = q1*c1 - q2*s1, out[d+32] = q2*c2 + q1*s2 with q1 = x[d], q2 =
// x[d+32] (element d + 32 is 8 lanes up); nvcc's contraction of each line is
// restated as fmaf(first product, -/+ second product).
__device__ __forceinline__ moe::f32x4 norm_rope_row(moe::f32x4 x, moe::f32x4 w, moe::f32x4 cs,
                                                    moe::f32x4 sn) {
#pragma clang fp contract(off)
  using moe::f32x4;
  const int lane = threadIdx.x & 63, r = lane >> 4;
  f32x4 sq, a, b, cc, y, other, o;
#pragma unroll
  for (int i = 0; i < 4; ++i) sq[i] = x[i] * x[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = sq[i] + __shfl_down(sq[i], 4, 16);
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = a[i] + __shfl_down(a[i], 2, 16);
#pragma unroll
  for (int i = 0; i < 4; ++i) cc[i] = b[i] + __shfl_down(b[i], 1, 16);
  const float f = (cc[0] + cc[2]) + (cc[1] + cc[3]);
  const float total = __shfl(f, 16 * r) + __shfl(f, 16 * r + 8);
  const float rms = 1.0f / sqrtf(total / 64.0f + moe::kNormEps);
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = (x[i] * rms) * w[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) other[i] = __shfl_xor(y[i], 8);
  const bool lo = (lane & 15) < 8;  // elements d < 32
#pragma unroll
  for (int i = 0; i < 4; ++i)
    o[i] = lo ? __builtin_fmaf(y[i], cs[i], -(other[i] * sn[i])) : __builtin_fmaf(y[i], cs[i], other[i] * sn[i]);
  return o;
}

}  // namespace lfm
