// 4-bit projections of a few rows (bg_linear.h states the weight's format). f32 throughout: a wave owns an
// output row and its lanes the row's words, eight weights each.
#include <hip/hip_fp16.h>

#include "bg_common.h"
#include "bg_linear.h"

namespace bg {

namespace {

template <int M, bool F16>
__global__ __launch_bounds__(256) void gemv4_kernel(Gemv4Args a, int m0) {
  const int N = a.N0 + a.N1 + a.N2;
  const int n = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (n >= N) return;
  const int words = a.K / 8, groups = a.K / a.group;
  float acc[M];
#pragma unroll
  for (int m = 0; m < M; m++) acc[m] = 0.0f;
  for (int w = lane; w < words; w += 64) {
    const uint32_t c = a.codes[(size_t)n * words + w];
    const size_t at = (size_t)n * groups + 8 * w / a.group;
    const float s = F16 ? __half2float(((const __half*)a.scales)[at]) : ((const float*)a.scales)[at];
    float lo = -8.0f * s;
    if (a.mins) lo = F16 ? __half2float(((const __half*)a.mins)[at]) : ((const float*)a.mins)[at];
    float wt[8];
#pragma unroll
    for (int i = 0; i < 8; i++) wt[i] = fmaf((float)((c >> (4 * i)) & 15), s, lo);
#pragma unroll
    for (int m = 0; m < M; m++) {
      const int row = min(m0 + m, a.M - 1);
      const float4* x = (const float4*)(a.x + (size_t)row * a.K + 8 * w);
      const float4 p = x[0], q = x[1];
      acc[m] = fmaf(wt[0], p.x, fmaf(wt[1], p.y, fmaf(wt[2], p.z, fmaf(wt[3], p.w, acc[m]))));
      acc[m] = fmaf(wt[4], q.x, fmaf(wt[5], q.y, fmaf(wt[6], q.z, fmaf(wt[7], q.w, acc[m]))));
    }
  }
#pragma unroll
  for (int m = 0; m < M; m++) {
    const float t = wave_sum(acc[m]);
    const int row = m0 + m;
    if (lane || row >= a.M) continue;
    const float y = a.resid ? t + a.resid[(size_t)row * N + n] : t;
    if (n < a.N0) a.out0[(size_t)row * a.N0 + n] = y;
    else if (n < a.N0 + a.N1) a.out1[(size_t)row * a.N1 + n - a.N0] = y;
    else a.out2[(size_t)row * a.N2 + n - a.N0 - a.N1] = y;
  }
}

}  // namespace

hipError_t launch_gemv4(const Gemv4Args& a, hipStream_t st) {
  const int N = a.N0 + a.N1 + a.N2;
  if (N <= 0 || a.M <= 0) return hipSuccess;
  const dim3 g((N + 3) / 4);
  for (int m0 = 0; m0 < a.M; m0 += 4) {
    if (a.M == 1) {
      if (a.scale_f16) hipLaunchKernelGGL((gemv4_kernel<1, true>), g, dim3(256), 0, st, a, m0);
      else hipLaunchKernelGGL((gemv4_kernel<1, false>), g, dim3(256), 0, st, a, m0);
    } else {
      if (a.scale_f16) hipLaunchKernelGGL((gemv4_kernel<4, true>), g, dim3(256), 0, st, a, m0);
      else hipLaunchKernelGGL((gemv4_kernel<4, false>), g, dim3(256), 0, st, a, m0);
    }
  }
  return hipGetLastError();
}

}  // namespace bg
