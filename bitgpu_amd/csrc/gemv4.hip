// 4-bit projections of up to 16 rows (bg_linear.h states the weight's format).
//
//   contraction  on the int8 matrix cores (v_mfma_i32_16x16x32_i8), exactly: a row of x becomes, 128 weights at a time,
//           a 31-bit fixed-point number over the block's largest power of two in four signed int8 digits; a
//           weight's code, its top bit turned, is 16 (c - 8) as the high half of a signed byte (two bit operations
//           a word give its odd codes and, shifted, its even ones). The operand of x has four rows a token, one a
//           digit, so a product takes four tokens; its result leaves lane 16 g + n with the four digit sums of
//           weight row n and token g, exact integers that are joined in f32 once a scale group, scaled back and
//           multiplied by the group's scale. With minima, a weight is (c - 8) s + (8 s + m): the groups' sums of
//           x come from the same products over all-ones weights. What a row of x gives does not depend on the
//           rows beside it: how K is split depends on K alone, and the rest is exact.
//   lanes   16 weight rows x 128 weights: lane 16 g + n holds words 4 g .. 4 g + 3 of row n (one 16-byte load). A
//           product contracts one word of each of the four lane groups: of the same scale group with groups of 128;
//           for 64 and 32 the words change lane groups (v_permlane32_swap, v_permlane16_swap) until that holds. The
//           digits of x are read in the order that this gives.
//   split   the waves of a workgroup split K, each taking 512 weights at a time and preparing x for those alone, in
//           LDS; every wave runs the workgroup's tiles over its part, and the parts meet in LDS. A wave's loads of
//           weights and scales are in flight before x is prepared.
//   values  a block of x with an infinity or a NaN is summed directly in f32.
#include <hip/hip_fp16.h>

#include <algorithm>
#include <type_traits>

#include "bg_common.h"
#include "bg_linear.h"

namespace bg {

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kStep = 512;            // weights of a wave's step: four blocks of 128
constexpr int kWaves = 8;
constexpr int kDigit = 528;           // bytes of a digit's row: 64 words of 8, and a pad that spreads 16 rows over the banks
constexpr int kToken = 4 * kDigit;

// The word of a 128-weight block (0 to 15) that lane group g holds as its j-th after the exchange.
template <int G>
__device__ inline int word_of(int j, int g) {
  if constexpr (G == 128) return 4 * g + j;
  if constexpr (G == 64) return 8 * (j >> 1) + (j & 1) + 4 * (g & 1) + 2 * (g >> 1);
  return 4 * j + g;
}
template <int G>
__device__ inline void exchange(u32x4_t& w) {
  if constexpr (G <= 64) {
    auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
    auto b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    if constexpr (G == 64) {
      w = u32x4_t{a[0], b[0], a[1], b[1]};
    } else {
      auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
      auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
      w = u32x4_t{c[0], c[1], d[0], d[1]};
    }
  }
}

// a word's eight codes as signed bytes 16 (c - 8): its even ones, then its odd ones
__device__ inline long weight_operand(uint32_t w) {
  const uint32_t even = (w << 4 ^ 0x80808080u) & 0xf0f0f0f0u, odd = (w ^ 0x80808080u) & 0xf0f0f0f0u;
  return (long)((uint64_t)odd << 32 | even);
}

// floor(v + 0.5) in one instruction
__device__ inline int round_i32(float v) {
  int r;
  asm("v_cvt_rpi_i32_f32 %0, %1" : "=v"(r) : "v"(v));
  return r;
}

// One group's scale of a row (or its minimum)
__device__ inline float scale_at(const void* p, size_t at, int f16) {
  return f16 ? __half2float(((const __half*)p)[at]) : ((const float*)p)[at];
}
// The 128 / G scales of a block, as loaded: 2 to 16 bytes
template <int G>
struct Scales {
  uint32_t raw[128 / G];
};
template <int G>
__device__ inline void load_scales(Scales<G>& s, const void* p, size_t at, int f16) {
  constexpr int N = 128 / G;
  if (f16) {  // (rows hold a multiple of 128 / G groups: aligned)
    if constexpr (N == 1) s.raw[0] = ((const uint16_t*)p)[at];
    if constexpr (N == 2) s.raw[0] = *(const uint32_t*)((const uint16_t*)p + at);
    if constexpr (N == 4) {
      const uint2 v = *(const uint2*)((const uint16_t*)p + at);
      s.raw[0] = v.x;
      s.raw[1] = v.y;
    }
  } else {
    if constexpr (N == 1) s.raw[0] = ((const uint32_t*)p)[at];
    if constexpr (N == 2) {
      const uint2 v = *(const uint2*)((const uint32_t*)p + at);
      s.raw[0] = v.x;
      s.raw[1] = v.y;
    }
    if constexpr (N == 4) {
      const uint4 v = *(const uint4*)((const uint32_t*)p + at);
      s.raw[0] = v.x;
      s.raw[1] = v.y;
      s.raw[2] = v.z;
      s.raw[3] = v.w;
    }
  }
}
template <int G>
__device__ inline float scale_of(const Scales<G>& s, int i, int f16) {
  if (!f16) return __uint_as_float(s.raw[i]);
  return __half2float(__ushort_as_half((unsigned short)(s.raw[i >> 1] >> (16 * (i & 1)))));
}

// A block of 128 weights in f32, for a row of x that holds an infinity or a NaN there
__device__ __noinline__ float block_f32(const float* x, const uint32_t* words, const void* scales, const void* mins, size_t at, int group,
                                        int f16) {
  float sum = 0.0f;
#pragma unroll 1
  for (int k = 0; k < 128; k++) {
    const float s = scale_at(scales, at + k / group, f16);
    const float lo = mins ? scale_at(mins, at + k / group, f16) : -8.0f * s;
    sum = fmaf(fmaf((float)(words[k >> 3] >> (4 * (k & 7)) & 15), s, lo), x[k], sum);
  }
  return sum;
}

constexpr int kOdd = 1 << 20;  // in the place of a block's exponent: it is not finite

// Rows of x as loaded: lane 16 b + l has weights 8 l .. + 7 of the step's block b.
template <int MT>
struct XLoad {
  f32x4_t v[MT][2];
};

// T tiles of 16 weight rows a workgroup, P passes of MT tokens over a step's weights (MT 1: one token).
template <int T, int MT, int P, int G>
__global__ __launch_bounds__(64 * kWaves) void gemv4_kernel(Gemv4Args a) {
  constexpr int NG = 128 / G;
  constexpr int kBytes = MT * kToken + kDigit;  // a wave's digits, then zeros for the tokens that are not there
  constexpr int kRed = T * 16 * MT * P * 4;     // a wave's sums
  __shared__ __align__(16) char lds[kWaves * (kBytes > kRed ? kBytes : kRed)];
  __shared__ int exps[kWaves][MT][4];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n = lane & 15, g = lane >> 4;
  const int N = a.N0 + a.N1 + a.N2, n0 = blockIdx.x * 16 * T;
  const int steps = (a.K + kStep - 1) / kStep, waves = blockDim.x >> 6;
  const int blocks = a.K >> 7, words = a.K >> 3, groups = a.K / G;
  char* dig = lds + wave * kBytes;
  float* red = (float*)lds;

  size_t row[T];
#pragma unroll
  for (int t = 0; t < T; t++) row[t] = min(n0 + 16 * t + n, N - 1);
  auto load_x = [&](XLoad<MT>& x, int step, int m0) {
    const int blk = min(4 * step + g, blocks - 1);
#pragma unroll
    for (int m = 0; m < MT; m++) {
      const float* p = a.x + (size_t)min(m0 + m, a.M - 1) * a.K + 128 * blk + 8 * n;
      x.v[m][0] = *(const f32x4_t*)p;
      x.v[m][1] = *(const f32x4_t*)(p + 4);
    }
  };
  float acc[P][T];
#pragma unroll
  for (int p = 0; p < P; p++)
#pragma unroll
    for (int t = 0; t < T; t++) acc[p][t] = 0.0f;
  for (int i = lane; i < kDigit / 4; i += 64) ((int*)(dig + MT * kToken))[i] = 0;

  for (int step = wave; step < steps; step += waves) {
    // x first: it is needed first, and loads arrive in order
    XLoad<MT> x;
    load_x(x, step, 0);
    __builtin_amdgcn_sched_barrier(0);
    u32x4_t w[T][4];
    Scales<G> sc[T][4], mn[T][4];
#pragma unroll
    for (int b = 0; b < 4; b++) {
      const int blk = min(4 * step + b, blocks - 1);  // past the end: x counts as zero there
#pragma unroll
      for (int t = 0; t < T; t++) {
        w[t][b] = *(const u32x4_t*)(a.codes + row[t] * words + 16 * blk + 4 * g);
        load_scales<G>(sc[t][b], a.scales, row[t] * groups + NG * blk, a.scale_f16);
        if (a.mins) load_scales<G>(mn[t][b], a.mins, row[t] * groups + NG * blk, a.scale_f16);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int p = 0; p < P; p++) {
      const int m0 = p * MT;
      if (p && m0 >= a.M) break;
      bool bad = false;
      // the reads of the pass before are done; a wave's LDS accesses complete in order
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int m = 0; m < MT; m++) {
        const bool on = 4 * step + g < blocks && m0 + m < a.M;
        const f32x4_t x0 = x.v[m][0], x1 = x.v[m][1];
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) top = max(top, max(__float_as_uint(x0[e]) & 0x7fffffffu, __float_as_uint(x1[e]) & 0x7fffffffu));
        auto dppmax = [&](auto ctrl) { top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, decltype(ctrl)::value, 0xf, 0xf, false)); };
        dppmax(std::integral_constant<int, kDppXor1>{});
        dppmax(std::integral_constant<int, kDppXor2>{});
        dppmax(std::integral_constant<int, kDppHalfMirror>{});
        dppmax(std::integral_constant<int, kDppMirror>{});
        const bool odd = top >= 0x7f800000u;
        bad = bad || (on && odd);
        const int e = (int)(top >> 23) - 126;  // |x| < 2^e
        const int shift = on && !odd ? 30 - e : -1024;  // (an infinity or NaN leaves some integer, cleared below)
        uint32_t y[2][4];  // even weights, odd weights
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float u = i < 2 ? x0[2 * i] : x1[2 * i - 4], v = i < 2 ? x0[2 * i + 1] : x1[2 * i - 3];
          y[0][i] = ((uint32_t)(odd ? 0 : round_i32(ldexpf(u, shift))) + 0x80808080u) ^ 0x80808080u;  // signed base-256 digits
          y[1][i] = ((uint32_t)(odd ? 0 : round_i32(ldexpf(v, shift))) + 0x80808080u) ^ 0x80808080u;
        }
        uint32_t d[2][4];
#pragma unroll
        for (int u = 0; u < 2; u++) {  // dword of digit q = byte q of the four
          const uint32_t p01 = __builtin_amdgcn_perm(y[u][1], y[u][0], 0x05010400u);
          const uint32_t p23 = __builtin_amdgcn_perm(y[u][3], y[u][2], 0x05010400u);
          const uint32_t q01 = __builtin_amdgcn_perm(y[u][1], y[u][0], 0x07030602u);
          const uint32_t q23 = __builtin_amdgcn_perm(y[u][3], y[u][2], 0x07030602u);
          d[u][0] = __builtin_amdgcn_perm(p23, p01, 0x05040100u);
          d[u][1] = __builtin_amdgcn_perm(p23, p01, 0x07060302u);
          d[u][2] = __builtin_amdgcn_perm(q23, q01, 0x05040100u);
          d[u][3] = __builtin_amdgcn_perm(q23, q01, 0x07060302u);
        }
#pragma unroll
        for (int q = 0; q < 4; q++) *(uint2*)(dig + m * kToken + q * kDigit + 128 * g + 8 * n) = make_uint2(d[0][q], d[1][q]);
        if (n == 0) exps[wave][m][g] = odd ? kOdd : e - 34;
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      if (p + 1 < P) load_x(x, step, m0 + MT);
      const int token = n >> 2;  // of the operand's row n; its digit is n & 3
      const char* src = dig + (token < MT ? token * kToken + (n & 3) * kDigit : MT * kToken);
      const int mine = g < MT ? g : 0;  // the token of this lane's results
#pragma unroll
      for (int b = 0; b < 4; b++) {
        long xd[4];
#pragma unroll
        for (int j = 0; j < 4; j++) xd[j] = *(const long*)(src + 128 * b + 8 * word_of<G>(j, g));
        const int e = exps[wave][mine][b];
        auto joined = [&](const i32x4_t& d) {  // digits 0, 1 and 2, 3 as integers (|d| <= 2^21), then in f32
          return ldexpf(fmaf((float)(d[2] + (d[3] << 8)), 65536.0f, (float)(d[0] + (d[1] << 8))), e);
        };
        float sums[NG];  // of x, by group
        if (a.mins) {
#pragma unroll
          for (int i = 0; i < NG; i++) {
            i32x4_t d = {0, 0, 0, 0};
#pragma unroll
            for (int j = i * G / 32; j < (i + 1) * G / 32; j++)
              d = __builtin_amdgcn_mfma_i32_16x16x32_i8(xd[j], 0x1010101010101010l, d, 0, 0, 0);
            sums[i] = joined(d);
          }
        }
#pragma unroll
        for (int t = 0; t < T; t++) {
          u32x4_t v = w[t][b];
          exchange<G>(v);
#pragma unroll
          for (int i = 0; i < NG; i++) {
            i32x4_t d = {0, 0, 0, 0};
#pragma unroll
            for (int j = i * G / 32; j < (i + 1) * G / 32; j++)
              d = __builtin_amdgcn_mfma_i32_16x16x32_i8(xd[j], weight_operand(v[j]), d, 0, 0, 0);
            const float s = scale_of<G>(sc[t][b], i, a.scale_f16);
            acc[p][t] = fmaf(joined(d), s, acc[p][t]);
            if (a.mins) acc[p][t] = fmaf(sums[i], fmaf(8.0f, s, scale_of<G>(mn[t][b], i, a.scale_f16)), acc[p][t]);
          }
        }
      }
      if (__any(bad)) {
#pragma unroll 1
        for (int b = 0; b < 4; b++) {
          const int k = 4 * step + b;
          if (k >= blocks || g >= MT || m0 + g >= a.M || exps[wave][mine][b] != kOdd) continue;
#pragma unroll
          for (int t = 0; t < T; t++)
            acc[p][t] += block_f32(a.x + (size_t)(m0 + g) * a.K + 128 * k, a.codes + row[t] * words + 16 * k, a.scales, a.mins,
                                   row[t] * groups + NG * k, G, a.scale_f16);
        }
      }
    }
  }
  __syncthreads();  // every wave is done with its digits
  if (g < MT)
#pragma unroll
    for (int p = 0; p < P; p++)
#pragma unroll
      for (int t = 0; t < T; t++) red[(wave * T * 16 + 16 * t + n) * (MT * P) + p * MT + g] = acc[p][t];
  __syncthreads();
  for (int i = threadIdx.x; i < T * 16 * MT * P; i += blockDim.x) {
    const int m = i / (T * 16), r = i % (T * 16), at = n0 + r;
    if (at >= N || m >= a.M) continue;
    float y = 0.0f;
    for (int k = 0; k < waves; k++) y += red[(k * T * 16 + r) * (MT * P) + m];
    if (a.resid) y += a.resid[(size_t)m * N + at];
    if (at < a.N0) a.out0[(size_t)m * a.N0 + at] = y;
    else if (at < a.N0 + a.N1) a.out1[(size_t)m * a.N1 + at - a.N0] = y;
    else a.out2[(size_t)m * a.N2 + at - a.N0 - a.N1] = y;
  }
}

template <int T, int MT, int P, int G>
hipError_t launch_t(const Gemv4Args& a, hipStream_t st) {
  const int N = a.N0 + a.N1 + a.N2, steps = (a.K + kStep - 1) / kStep;
  hipLaunchKernelGGL((gemv4_kernel<T, MT, P, G>), dim3((N + 16 * T - 1) / (16 * T)), dim3(64 * std::min(steps, kWaves)), 0, st, a);
  return hipGetLastError();
}

template <int G>
hipError_t launch_g(const Gemv4Args& a, hipStream_t st) {
  const bool few = (a.N0 + a.N1 + a.N2 + 15) / 16 <= 512;
  if (a.M == 1) return few ? launch_t<1, 1, 1, G>(a, st) : launch_t<2, 1, 1, G>(a, st);
  if (a.M <= 4) return few ? launch_t<1, 4, 1, G>(a, st) : launch_t<2, 4, 1, G>(a, st);
  if (a.M <= 8) return few ? launch_t<1, 4, 2, G>(a, st) : launch_t<2, 4, 2, G>(a, st);
  return few ? launch_t<1, 4, 4, G>(a, st) : launch_t<2, 4, 4, G>(a, st);
}

}  // namespace

hipError_t launch_gemv4(const Gemv4Args& a, hipStream_t st) {
  if (a.N0 + a.N1 + a.N2 <= 0 || a.M <= 0) return hipSuccess;
  return a.group == 32 ? launch_g<32>(a, st) : a.group == 64 ? launch_g<64>(a, st) : launch_g<128>(a, st);
}

}  // namespace bg
