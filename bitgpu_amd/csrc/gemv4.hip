// 4-bit projections of up to 16 rows (bg_linear.h states the weight's format).
//
//   contraction  on the int8 matrix cores, exactly: a row of x becomes, 128 weights at a time, a 31-bit fixed-point
//           number over the block's largest power of two in four signed int8 digits; a weight's code, its top bit turned, is
//           16 (c - 8) as the high half of a signed byte (two bit operations a word give its odd codes and, shifted,
//           its even ones). The operand of x has four rows a token, one a digit, so a product takes four tokens; its
//           result leaves lane 16 g + n with the four digit sums of weight row n and token g, exact integers that are
//           joined in f32 once a scale group, multiplied by the group's scale and scaled back once a block. With
//           minima, codes enter as they are (c), and the minima times the groups' sums of x, 16 tokens at once, are a
//           product on the f32 matrix cores.
//   order   what a row of x gives does not depend on the rows beside it: how K is split depends on K alone, the integers
//           are exact, and the f32 sums are taken in one order, groups, blocks (0 + 1) + (2 + 3), steps, waves.
//   lanes   16 weight rows x 128 weights: lane 16 g + n holds words 4 g .. 4 g + 3 of row n (one 16-byte load). A
//           product contracts words of the four lane groups: of the same scale group with groups of 128; for 64 and 32
//           the words change lane groups (v_permlane32_swap, v_permlane16_swap) until that holds. The digits of x are
//           read in the order that this gives.
//   split   the waves of a workgroup split K, 512 weights at a time. A wave has x for its 512 in registers (or LDS) and
//           runs the workgroup's tiles of 16 rows over it, the next tile's weights and scales in flight while one is
//           multiplied; the parts meet in LDS at the end.
//   x       up to four tokens: every wave prepares x for its 512, through LDS. More: a kernel of its own does, once for
//           all workgroups, in the order in which they read it. That launch takes 2.5 us (five rows of 4096 x 4096 8.4
//           us, four 6.5), but 16 rows prepared in every workgroup took longer than all products: 15 rows of K = 6144,
//           N = 4096 22 us, so 11 + 4.7.
//   bounds  one token: 24576 rows of K = 4096 in groups of 32 with minima (63 MB) 13.4 us, 4.7 TB/s, what a large copy
//           reaches; 4096 x 4096 in groups of 128 (8.7 MB) 5.1 us, the latency of a launch and one pass over K. More tokens:
//           the joining of the integers: ten rows of K = 4096, N = 16480 16.6 + 2.6 us.
//           (Of two to four tokens 24576 rows of K = 4096 take 19 to 20 us, of 16 30.)
//   values  x is rounded to 2^-31 of its block's largest value: below the rounding of an f32 sum that this value takes part
//           in. Where its weight is exactly zero (code 8, no minima) the others keep only that: values 2^-7 of the largest
//           have an f32's 24 bits, smaller ones fewer. A block with an infinity or a NaN is summed directly in f32.
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
// Workgroups that a launch aims at, with up to kMaxTiles tiles of 16 rows each. One token, two a CU: 4096 x 4096 takes
// 5.1 us and 6176 x 2048 6.5 us, with half as many 5.1 and 7.0, with twice as many 5.1 and 6.3 (but 24576 rows of 4096
// 13.9 against 13.4). More tokens prepare x longer, so one a CU: 16 rows of 16480 x 4096 21 us, with twice as many 28;
// waves of half as many: 25.
constexpr int kTargetOne = 512, kTarget = 256, kMaxTiles = 8;
constexpr int kDigit = 528;           // bytes of a digit's row: 64 words of 8, and a pad that spreads 16 rows over the banks
constexpr int kToken = 4 * kDigit;
// x prepared for more than four tokens: of a step of 512 weights, kPassBytes for every four tokens (operands
// [block][word pair][lane], 16 bytes each, then powers of two [token][block]), behind all of them kSumBytes a step (the
// groups' sums [16 rows][block][group])
constexpr int kOperand = 8192, kPassBytes = kOperand + 64, kSumBytes = 1024;
// A block's joined digits count 2^(e - kUnit) (codes without minima 16 times as much), |x| < 2^e there: a digit of weight
// 2^0 counts 2^(e - 30), and digits 2 and 3 are the whole part. A group's sum is at most about 2^28 so, and may be multiplied by
// a scale of 2^90.
constexpr int kUnit = 14;
constexpr int kOdd = 0x7fffffff;      // the power of two of a block with an infinity or a NaN (its digits are zero)

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

// a word's eight codes as signed bytes, its even ones, then its odd ones: 16 (c - 8), or c where there are minima
template <bool MINS>
__device__ inline long weight_operand(uint32_t w) {
  const uint32_t even = MINS ? w & 0x0f0f0f0fu : (w << 4 ^ 0x80808080u) & 0xf0f0f0f0u;
  const uint32_t odd = MINS ? w >> 4 & 0x0f0f0f0fu : (w ^ 0x80808080u) & 0xf0f0f0f0u;
  return (long)((uint64_t)odd << 32 | even);
}

__device__ inline i32x4_t pair(long a, long b) {
  return i32x4_t{(int)(uint32_t)(uint64_t)a, (int)(uint32_t)((uint64_t)a >> 32), (int)(uint32_t)(uint64_t)b, (int)(uint32_t)((uint64_t)b >> 32)};
}

// floor(v + 0.5) in one instruction
__device__ inline int round_i32(float v) {
  int r;
  asm("v_cvt_rpi_i32_f32 %0, %1" : "=v"(r) : "v"(v));
  return r;
}

// One group's scale of a row (or its minimum)
template <bool F16>
__device__ inline float scale_at(const void* p, size_t at) {
  return F16 ? __half2float(((const __half*)p)[at]) : ((const float*)p)[at];
}
// The 128 / G scales of a block, as loaded: 2 to 16 bytes (rows hold a multiple of 128 / G groups: aligned)
template <int G, bool F16>
struct Scales {
  static constexpr int N = 128 / G, W = F16 ? (N + 1) / 2 : N;
  uint32_t raw[W];
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, int at, int more) {  // bytes
    if constexpr (F16 && N == 1) {
      raw[0] = __builtin_amdgcn_raw_buffer_load_b16(r, at, more, 0);
    } else if constexpr (W == 1) {
      raw[0] = __builtin_amdgcn_raw_buffer_load_b32(r, at, more, 0);
    } else if constexpr (W == 2) {
      const auto v = __builtin_amdgcn_raw_buffer_load_b64(r, at, more, 0);
      raw[0] = v[0];
      raw[1] = v[1];
    } else {
      const auto v = __builtin_amdgcn_raw_buffer_load_b128(r, at, more, 0);
      raw[0] = v[0];
      raw[1] = v[1];
      raw[2] = v[2];
      raw[3] = v[3];
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (!F16) return __uint_as_float(raw[i]);
    else return __half2float(__ushort_as_half((unsigned short)(raw[i >> 1] >> (16 * (i & 1)))));
  }
};

// A block of 128 weights in f32, for a row of x that holds an infinity or a NaN there
template <int G, bool F16>
__device__ __forceinline__ float block_f32(const float* x, const uint32_t* words, const void* scales, const void* mins, size_t at) {
  float sum = 0.0f;
#pragma unroll 1
  for (int k = 0; k < 128; k++) {
    const float s = scale_at<F16>(scales, at + k / G);
    const float lo = mins ? scale_at<F16>(mins, at + k / G) : -8.0f * s;
    sum = fmaf(fmaf((float)(words[k >> 3] >> (4 * (k & 7)) & 15), s, lo), x[k], sum);
  }
  return sum;
}

// A lane's eight values of x (its block's other 15 lanes hold the rest) as digits: d[0] of its even ones, d[1] of its
// odd ones, digit q in d[.][q]; |x| < 2^e in the block, and a digit of weight 2^0 counts 2^(e - 30). Where not `on`, or
// the block is not finite (returned), all are zero.
__device__ inline bool digits(f32x4_t x0, f32x4_t x1, bool on, uint32_t (&d)[2][4], int& e) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) top = max(top, max(__float_as_uint(x0[i]) & 0x7fffffffu, __float_as_uint(x1[i]) & 0x7fffffffu));
  auto dppmax = [&](auto ctrl) { top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, decltype(ctrl)::value, 0xf, 0xf, false)); };
  dppmax(std::integral_constant<int, kDppXor1>{});
  dppmax(std::integral_constant<int, kDppXor2>{});
  dppmax(std::integral_constant<int, kDppHalfMirror>{});
  dppmax(std::integral_constant<int, kDppMirror>{});
  const bool odd = top >= 0x7f800000u;
  e = (int)(top >> 23) - 126;
  const uint32_t use = on && !odd ? ~0u : 0u;  // (an infinity or NaN leaves some integer)
  uint32_t y[2][4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float u = i < 2 ? x0[2 * i] : x1[2 * i - 4], v = i < 2 ? x0[2 * i + 1] : x1[2 * i - 3];
    y[0][i] = (((uint32_t)round_i32(ldexpf(u, 30 - e)) & use) + 0x80808080u) ^ 0x80808080u;  // signed base-256 digits
    y[1][i] = (((uint32_t)round_i32(ldexpf(v, 30 - e)) & use) + 0x80808080u) ^ 0x80808080u;
  }
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
  return odd;
}

// the sum over a lane's scale group, in all of the group's lanes
template <int G>
__device__ inline float block_sums(f32x4_t x0, f32x4_t x1) {
  return group_sum<G / 8>(((x0[0] + x0[1]) + (x0[2] + x0[3])) + ((x1[0] + x1[1]) + (x1[2] + x1[3])));
}

// four registers of the four lane groups transposed: afterwards w[i] of group g is what w[g] of group i was
__device__ inline void transpose(uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  auto ac = __builtin_amdgcn_permlane32_swap(a, c, false, false);
  auto bd = __builtin_amdgcn_permlane32_swap(b, d, false, false);
  auto lo = __builtin_amdgcn_permlane16_swap(ac[0], bd[0], false, false);
  auto hi = __builtin_amdgcn_permlane16_swap(ac[1], bd[1], false, false);
  a = lo[0];
  b = lo[1];
  c = hi[0];
  d = hi[1];
}

__device__ inline __amdgpu_buffer_rsrc_t buffer(const void* p, size_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, (short)0, (int)(uint32_t)(bytes < 0xffffffffu ? bytes : 0xffffffffu), 0x00020000);
}

// The blocks of x that hold an infinity or a NaN, left out of a wave's sums red[wave][tile][16 rows][M] so far
template <int G, bool MINS, bool F16>
__device__ __forceinline__ void odd_blocks(const Gemv4Args& a, float* red, int T, int n0, int wave, int waves, int lane) {
  const int n = lane & 15, g = lane >> 4, N = a.N0 + a.N1 + a.N2;
  const int blocks = a.K >> 7, words = a.K >> 3, groups = a.K / G;
#pragma unroll 1
  for (int blk = 0; blk < blocks; blk++) {
    if ((blk >> 2) % waves != wave) continue;
#pragma unroll 1
    for (int m = g; m < a.M; m += 4) {
      const float* xp = a.x + (size_t)m * a.K + 128 * blk;
      uint32_t top = 0;
#pragma unroll 1
      for (int k = 0; k < 128; k++) top = max(top, __float_as_uint(xp[k]) & 0x7fffffffu);
      if (top < 0x7f800000u) continue;
#pragma unroll 1
      for (int u = 0; u < T; u++) {
        const size_t r = min(n0 + 16 * u + n, N - 1);
        red[(size_t)((wave * T + u) * 16 + n) * a.M + m] +=
            block_f32<G, F16>(xp, a.codes + r * words + 16 * blk, a.scales, MINS ? a.mins : nullptr, r * groups + 128 / G * blk);
      }
    }
  }
}

// The workgroup's rows: the waves' sums in their order
__device__ __forceinline__ void store(const Gemv4Args& a, const float* red, int T, int n0, int waves) {
  const int N = a.N0 + a.N1 + a.N2;
  for (int i = threadIdx.x; i < T * 16 * a.M; i += blockDim.x) {
    const int m = i / (T * 16), r = i % (T * 16), at = n0 + r;
    if (at >= N) continue;
    float y = 0.0f;
    for (int k = 0; k < waves; k++) y += red[(size_t)(k * T * 16 + r) * a.M + m];
    if (a.resid) y += a.resid[(size_t)m * N + at];
    if (at < a.N0) a.out0[(size_t)m * a.N0 + at] = y;
    else if (at < a.N0 + a.N1) a.out1[(size_t)m * a.N1 + at - a.N0] = y;
    else a.out2[(size_t)m * a.N2 + at - a.N0 - a.N1] = y;
  }
}

// x of more than four tokens, prepared once for all workgroups in the order in which they read it: a wave takes 512
// weights of a token (of 4 P, those behind the last are zero).
template <int G, bool MINS>
__global__ __launch_bounds__(64) void gemv4_digits_kernel(Gemv4Args a, int P) {
  constexpr int NG = 128 / G;
  const int lane = threadIdx.x, n = lane & 15, g = lane >> 4, step = blockIdx.x, token = blockIdx.y;
  const int steps = (a.K + kStep - 1) / kStep, blocks = a.K >> 7;
  const bool on = token < a.M && 4 * step + g < blocks;
  const float* xp = a.x + (size_t)min(token, a.M - 1) * a.K + 128 * min(4 * step + g, blocks - 1) + 8 * n;
  const f32x4_t x0 = *(const f32x4_t*)xp, x1 = *(const f32x4_t*)(xp + 4);
  uint32_t d[2][4];
  int e;
  const bool odd = digits(x0, x1, on, d, e);
  char* to = a.room + ((size_t)step * P + (token >> 2)) * kPassBytes;
  // word n of block g: the j-th that lane group `at` holds (word_of)
  const int j = G == 128 ? n & 3 : G == 64 ? 2 * (n >> 3) + (n & 1) : n >> 2;
  const int at = G == 128 ? n >> 2 : G == 64 ? ((n >> 2) & 1) + 2 * ((n >> 1) & 1) : n & 3;
  if (token < 4 * P) {
#pragma unroll
    for (int q = 0; q < 4; q++)
      *(uint2*)(to + (2 * g + (j >> 1)) * 1024 + (16 * at + 4 * (token & 3) + q) * 16 + 8 * (j & 1)) = make_uint2(d[0][q], d[1][q]);
    if (n == 0) ((int*)(to + kOperand))[4 * (token & 3) + g] = on && odd ? kOdd : odd ? 0 : e - (MINS ? kUnit : kUnit + 4);
  }
  if constexpr (MINS) {
    const float t = block_sums<G>(x0, x1);
    float* sums = (float*)(a.room + (size_t)steps * P * kPassBytes + (size_t)step * kSumBytes);
    if (n % (G / 8) == 0) sums[((4 * (token & 3) + (token >> 2)) * 4 + g) * NG + n / (G / 8)] = on && !odd ? t : 0.0f;
  }
}

// P: groups of four tokens.
template <int P, int G, bool MINS, bool F16>
__global__ __launch_bounds__(64 * kWaves, P == 1 ? 4 : 2) void gemv4_kernel(Gemv4Args a, int T) {
  constexpr int NG = 128 / G;
  extern __shared__ __align__(16) char lds[];
  __shared__ int exps[kWaves][4][4];
  __shared__ float xsum[MINS && P == 1 ? kWaves : 1][4][4 * NG];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n = lane & 15, g = lane >> 4;
  const int N = a.N0 + a.N1 + a.N2, n0 = blockIdx.x * 16 * T;
  const int steps = (a.K + kStep - 1) / kStep, waves = blockDim.x >> 6;
  const int blocks = a.K >> 7, words = a.K >> 3, groups = a.K / G;
  const int held = min(a.M, 4);                         // tokens of the digits in LDS, then zeros for the others
  char* dig = lds + wave * (held * kToken + kDigit);
  float* red = (float*)(lds + (P == 1 ? waves * (held * kToken + kDigit) : 0));  // [wave][tile][16 rows][M]

  long xd[P][4][4];    // the operand of x: four words of each of the step's blocks (of one pass: read where used)
  int ex[P][4];        // the blocks' powers of two, of this lane's token 4 p + g
  float xs[NG];        // the groups' sums of x: token 4 (n % 4) + n / 4, group i of the step's block g
  bool odd_any = false;
  f32x4_t x0[4], x1[4];  // the rows of x as loaded: lane 16 b + l has weights 8 l .. + 7 of block b
  auto load_x = [&](int step) {
#pragma unroll
    for (int m = 0; m < 4; m++) {
      if (m >= a.M) break;
      const float* xp = a.x + (size_t)m * a.K + 128 * min(4 * step + g, blocks - 1) + 8 * n;
      x0[m] = *(const f32x4_t*)xp;
      x1[m] = *(const f32x4_t*)(xp + 4);
    }
  };
  auto prepare = [&](int step) {  // four tokens: x is loaded
    for (int i = lane; i < kDigit / 4; i += 64) ((int*)(dig + held * kToken))[i] = 0;
#pragma unroll
    for (int m = 0; m < 4; m++) {
      if (m >= a.M) {
        if constexpr (MINS)
          if (lane < 4 * NG) xsum[wave][m][lane] = 0.0f;
        continue;
      }
      const bool on = 4 * step + g < blocks;
      uint32_t d[2][4];
      int e;
      const bool odd = digits(x0[m], x1[m], on, d, e);
      odd_any = odd_any || (on && odd);
      if constexpr (MINS) {
        const float t = block_sums<G>(x0[m], x1[m]);
        if (n % (G / 8) == 0) xsum[wave][m][NG * g + n / (G / 8)] = on && !odd ? t : 0.0f;
      }
#pragma unroll
      for (int q = 0; q < 4; q++) *(uint2*)(dig + m * kToken + q * kDigit + 128 * g + 8 * n) = make_uint2(d[0][q], d[1][q]);
      if (n == 0) exps[wave][m][g] = odd ? 0 : e - (MINS ? kUnit : kUnit + 4);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int b = 0; b < 4; b++) ex[0][b] = g < a.M ? exps[wave][g][b] : 0;
    if constexpr (MINS)
#pragma unroll
      for (int i = 0; i < NG; i++) xs[i] = (n & 3) == 0 ? xsum[wave][n >> 2][NG * g + i] : 0.0f;
  };
  auto take = [&](int step) {  // more tokens: as gemv4_digits_kernel left it
    const char* at = a.room + (size_t)step * P * kPassBytes;
#pragma unroll
    for (int p = 0; p < P; p++) {
#pragma unroll
      for (int b = 0; b < 4; b++)
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          const i32x4_t v = *(const i32x4_t*)(at + p * kPassBytes + (2 * b + j / 2) * 1024 + lane * 16);
          xd[p][b][j] = (long)((uint64_t)(uint32_t)v[1] << 32 | (uint32_t)v[0]);
          xd[p][b][j + 1] = (long)((uint64_t)(uint32_t)v[3] << 32 | (uint32_t)v[2]);
        }
      const i32x4_t e = *(const i32x4_t*)(at + p * kPassBytes + kOperand + g * 16);
#pragma unroll
      for (int b = 0; b < 4; b++) {
        ex[p][b] = e[b];
        odd_any = odd_any || e[b] == kOdd;
      }
    }
    if constexpr (MINS) {
      const float* sums = (const float*)(a.room + (size_t)steps * P * kPassBytes + (size_t)step * kSumBytes) + (n * 4 + g) * NG;
#pragma unroll
      for (int i = 0; i < NG; i++) xs[i] = sums[i];
    }
  };

  struct Tile {
    u32x4_t w[4];
    Scales<G, F16> s[4];
    Scales<G, F16> lo;  // of block g
  };
  // The workgroup's rows as buffers: 32-bit offsets from its first (rows behind the last are the last again)
  const int rows = min(16 * T, N - n0);
  constexpr int kScale = F16 ? 2 : 4;
  const auto rw = buffer(a.codes + (size_t)n0 * words, (size_t)rows * words * 4);
  const auto rs = buffer((const char*)a.scales + (size_t)n0 * groups * kScale, (size_t)rows * groups * kScale);
  const auto rm = buffer((const char*)(MINS ? a.mins : a.scales) + (size_t)n0 * groups * kScale, (size_t)rows * groups * kScale);
  auto load = [&](Tile& x, int step, int t, int b) {
    const int r = min(16 * t + n, rows - 1), blk = min(4 * step + b, blocks - 1);  // past the end: x counts as zero there
    x.w[b] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rw, r * words * 4 + 16 * g, 64 * blk, 0));
    x.s[b].load(rs, r * groups * kScale, NG * kScale * blk);
  };
  auto load_lo = [&](Tile& x, int step, int t) {
    const int r = min(16 * t + n, rows - 1);
    if constexpr (MINS) x.lo.load(rm, kScale * (r * groups + NG * min(4 * step + g, blocks - 1)), 0);
  };
  // A tile's products; the next one's (step1, t1) loads go into the registers of each block as it is done
  auto multiply = [&](Tile& x, int step, int t, int step1, int t1) {
    float acc[P], two[P];  // of the blocks so far; of the pair of blocks under way
    f32x4_t lo = {0, 0, 0, 0};
    if constexpr (MINS) {
#pragma unroll
      for (int i = 0; i < NG; i++) lo = __builtin_amdgcn_mfma_f32_16x16x4f32(xs[i], x.lo.get(i), lo, 0, 0, 0);
      if (step1 < steps) load_lo(x, step1, t1);
    }
#pragma unroll
    for (int b = 0; b < 4; b++) {
      u32x4_t v = x.w[b];
      exchange<G>(v);
      long w[4];
#pragma unroll
      for (int j = 0; j < 4; j++) w[j] = weight_operand<MINS>(v[j]);
      if constexpr (P == 1) {
        const char* src = dig + ((n >> 2) < held ? (n >> 2) * kToken + (n & 3) * kDigit : held * kToken);
#pragma unroll
        for (int j = 0; j < 4; j++) xd[0][b][j] = *(const long*)(src + 128 * b + 8 * word_of<G>(j, g));
      }
      float sum[P];
#pragma unroll
      for (int i = 0; i < NG; i++) {
        const float s = x.s[b].get(i);
        i32x4_t d[P];
#pragma unroll
        for (int p = 0; p < P; p++) d[p] = i32x4_t{0, 0, 0, 0};
        if constexpr (G == 32) {
#pragma unroll
          for (int p = 0; p < P; p++) d[p] = __builtin_amdgcn_mfma_i32_16x16x32_i8(xd[p][b][i], w[i], d[p], 0, 0, 0);
        } else {  // two words a lane at once
#pragma unroll
          for (int j = i * G / 32; j < (i + 1) * G / 32; j += 2)
#pragma unroll
            for (int p = 0; p < P; p++)
              d[p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(pair(xd[p][b][j], xd[p][b][j + 1]), pair(w[j], w[j + 1]), d[p], 0, 0, 0);
        }
#pragma unroll
        for (int p = 0; p < P; p++) {  // digits 0, 1 and 2, 3 as integers (|d| <= 2^21), then in f32
          const float low = (float)(d[p][0] + (d[p][1] << 8)), hi = (float)(d[p][2] + (d[p][3] << 8));
          const float all = fmaf(low, 0x1p-16f, hi);
          sum[p] = i ? fmaf(all, s, sum[p]) : all * s;
        }
      }
#pragma unroll
      for (int p = 0; p < P; p++) {  // (blocks 0 + 1) + (2 + 3)
        const float v = ldexpf(sum[p], ex[p][b]);
        two[p] = b & 1 ? two[p] + v : v;
        if (b == 1) acc[p] = two[p];
        if (b == 3) acc[p] += two[p];
      }
      // the sums of a block here, and not where a lane stores its part: all blocks' digits at once do not fit
#pragma unroll
      for (int p = 0; p < P; p++) asm volatile("" : "+v"(two[p]));
      if (step1 < steps) load(x, step1, t1, b);
    }
    if constexpr (MINS)
#pragma unroll
      for (int p = 0; p < P; p++) acc[p] += lo[p];
    float* to = red + (size_t)((wave * T + t) * 16 + n) * a.M + g;
#pragma unroll
    for (int p = 0; p < P; p++)
      if (4 * p + g < a.M) to[4 * p] = step == wave ? acc[p] : to[4 * p] + acc[p];
  };

  if (wave < steps) {
    // x first: it is needed first, and loads arrive in order
    Tile x;
    if constexpr (P == 1) load_x(wave);
    else take(wave);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int b = 0; b < 4; b++) load(x, wave, 0, b);
    load_lo(x, wave, 0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll 1
    for (int step = wave, t = 0; step < steps;) {
      if (t == 0) {
        if constexpr (P == 1) {
          if (step != wave) load_x(step);
          prepare(step);
        } else if (step != wave) {
          take(step);
        }
      }
      const bool end = t + 1 == T;
      const int step1 = end ? step + waves : step, t1 = end ? 0 : t + 1;
      multiply(x, step, t, step1, t1);
      step = step1;
      t = t1;
    }
    if (__any(odd_any)) odd_blocks<G, MINS, F16>(a, red, T, n0, wave, waves, lane);
  }
  __syncthreads();
  store(a, red, T, n0, waves);
}

// One token: the operand of x is block diagonal. Its row 4 b + q holds digit q of the step's block b, in the k of lane
// group b and zeros elsewhere, so lane 16 g + n gets its row's sums over block g, and the joining, scaling and adding
// of sums (half of the instructions with four tokens, of which three would be missing) is a quarter. A lane needs the
// words of its own block: what 16-byte loads of 64 contiguous bytes a row bring is transposed between lane groups.
template <int G, bool MINS, bool F16>
__global__ __launch_bounds__(64 * kWaves, 4) void gemv4_one_kernel(Gemv4Args a, int T) {
  constexpr int NG = 128 / G;
  constexpr int kRow = 144;                             // bytes of a (block, digit) row: 16 words of 8, and a pad
  constexpr int kBytes = 16 * kRow + 128;               // then zeros
  __shared__ __align__(16) char lds[kWaves * kBytes];
  __shared__ float red[kWaves * kMaxTiles * 16];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n = lane & 15, g = lane >> 4;
  const int N = a.N0 + a.N1 + a.N2, n0 = blockIdx.x * 16 * T;
  const int steps = (a.K + kStep - 1) / kStep, waves = blockDim.x >> 6;
  const int blocks = a.K >> 7, words = a.K >> 3, groups = a.K / G;
  char* dig = lds + wave * kBytes;
  const int rows = min(16 * T, N - n0);
  constexpr int kScale = F16 ? 2 : 4;
  const auto rw = buffer(a.codes + (size_t)n0 * words, (size_t)rows * words * 4);
  const auto rs = buffer((const char*)a.scales + (size_t)n0 * groups * kScale, (size_t)rows * groups * kScale);
  const auto rm = buffer((const char*)(MINS ? a.mins : a.scales) + (size_t)n0 * groups * kScale, (size_t)rows * groups * kScale);

  i32x4_t xd[8];       // the operand of x: words 2 i, 2 i + 1 of the lane's block
  int ex = 0;          // the block's power of two
  float xs[NG];        // the sums of x over the block's groups, as row 0 of an operand
  bool odd_any = false;
  f32x4_t x0, x1;
  u32x4_t w[4];
  Scales<G, F16> sc, lo;
  auto load_x = [&](int step) {
    const float* xp = a.x + 128 * min(4 * step + g, blocks - 1) + 8 * n;
    x0 = *(const f32x4_t*)xp;
    x1 = *(const f32x4_t*)(xp + 4);
  };
  auto load = [&](int step, int t) {
    const int r = min(16 * t + n, rows - 1);
#pragma unroll
    for (int b = 0; b < 4; b++)  // past the end: x counts as zero there
      w[b] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rw, r * words * 4 + 16 * g, 64 * min(4 * step + b, blocks - 1), 0));
    const int at = kScale * (r * groups + NG * min(4 * step + g, blocks - 1));
    sc.load(rs, at, 0);
    if constexpr (MINS) lo.load(rm, at, 0);
  };
  if (wave < steps) {
    load_x(wave);
    __builtin_amdgcn_sched_barrier(0);
    load(wave, 0);
    __builtin_amdgcn_sched_barrier(0);
    if (lane < 8) *(uint4*)(dig + 16 * kRow + 16 * lane) = make_uint4(0, 0, 0, 0);
#pragma unroll 1
    for (int step = wave, t = 0; step < steps;) {
      if (t == 0) {
        if (step != wave) load_x(step);
        const bool on = 4 * step + g < blocks;
        uint32_t d[2][4];
        int e;
        const bool odd = digits(x0, x1, on, d, e);
        odd_any = odd_any || (on && odd);
        ex = odd ? 0 : e - (MINS ? kUnit : kUnit + 4);
        if constexpr (MINS) {
          float v = block_sums<G>(x0, x1);
          v = on && !odd ? v : 0.0f;
#pragma unroll
          for (int i = 0; i < NG; i++) {
            const float all = __shfl(v, 16 * g + (G / 8) * i);
            xs[i] = n == 0 ? all : 0.0f;
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int q = 0; q < 4; q++) *(uint2*)(dig + (4 * g + q) * kRow + 8 * n) = make_uint2(d[0][q], d[1][q]);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        const char* src = dig + ((n >> 2) == g ? n * kRow : 16 * kRow);
#pragma unroll
        for (int i = 0; i < 8; i++) xd[i] = *(const i32x4_t*)(src + 16 * i);
      }
      const bool end = t + 1 == T;
      const int step1 = end ? step + waves : step, t1 = end ? 0 : t + 1;
      u32x4_t v[4];
      float s[NG], m[NG];
#pragma unroll
      for (int b = 0; b < 4; b++) v[b] = w[b];
#pragma unroll
      for (int i = 0; i < NG; i++) {
        s[i] = sc.get(i);
        m[i] = MINS ? lo.get(i) : 0.0f;
      }
#pragma unroll
      for (int j = 0; j < 4; j++) {
        uint32_t p0 = v[0][j], p1 = v[1][j], p2 = v[2][j], p3 = v[3][j];
        transpose(p0, p1, p2, p3);
        v[0][j] = p0;
        v[1][j] = p1;
        v[2][j] = p2;
        v[3][j] = p3;
      }
      if (step1 < steps) load(step1, t1);
      float acc = 0.0f;
#pragma unroll
      for (int i = 0; i < NG; i++) {
        i32x4_t d = {0, 0, 0, 0};
#pragma unroll
        for (int j = i * G / 16; j < (i + 1) * G / 16; j++)
          d = __builtin_amdgcn_mfma_i32_16x16x64_i8(xd[j], pair(weight_operand<MINS>(v[j >> 1][2 * (j & 1)]), weight_operand<MINS>(v[j >> 1][2 * (j & 1) + 1])), d, 0, 0, 0);
        const float all = fmaf((float)(d[0] + (d[1] << 8)), 0x1p-16f, (float)(d[2] + (d[3] << 8)));
        acc = i ? fmaf(all, s[i], acc) : all * s[i];
      }
      acc = ldexpf(acc, ex);
      float2 r = pair16(acc);
      r = pair32(r.x + r.y);
      acc = r.x + r.y;  // the step's four blocks
      if constexpr (MINS) {
        f32x4_t d = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < NG; i++) d = __builtin_amdgcn_mfma_f32_16x16x4f32(xs[i], m[i], d, 0, 0, 0);
        acc += d[0];  // (of lanes 0 to 15)
      }
      float* to = red + (wave * T + t) * 16 + n;
      if (g == 0) *to = step == wave ? acc : *to + acc;
      step = step1;
      t = t1;
    }
    if (__any(odd_any)) odd_blocks<G, MINS, F16>(a, red, T, n0, wave, waves, lane);
  }
  __syncthreads();
  store(a, red, T, n0, waves);
}

template <int P, int G, bool MINS, bool F16>
hipError_t launch_t(const Gemv4Args& a, hipStream_t st) {
  const int tiles = (a.N0 + a.N1 + a.N2 + 15) / 16, waves = std::min((a.K + kStep - 1) / kStep, kWaves);
  const int T = std::min(kMaxTiles, (tiles + kTarget - 1) / kTarget);
  const size_t lds = waves * ((P == 1 ? (size_t)(a.M * kToken + kDigit) : 0) + (size_t)T * 16 * a.M * sizeof(float));
  if constexpr (P > 1) {
    // (the sums are an operand of 16 rows)
    hipLaunchKernelGGL((gemv4_digits_kernel<G, MINS>), dim3((a.K + kStep - 1) / kStep, MINS ? 16 : 4 * P), dim3(64), 0, st, a, P);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((gemv4_kernel<P, G, MINS, F16>), dim3((tiles + T - 1) / T), dim3(64 * waves), lds, st, a, T);
  return hipGetLastError();
}

template <int G, bool MINS, bool F16>
hipError_t launch_one_t(const Gemv4Args& a, hipStream_t st) {
  const int tiles = (a.N0 + a.N1 + a.N2 + 15) / 16, waves = std::min((a.K + kStep - 1) / kStep, kWaves);
  const int T = std::min(kMaxTiles, (tiles + kTargetOne - 1) / kTargetOne);
  hipLaunchKernelGGL((gemv4_one_kernel<G, MINS, F16>), dim3((tiles + T - 1) / T), dim3(64 * waves), 0, st, a, T);
  return hipGetLastError();
}

template <int G>
hipError_t launch_one(const Gemv4Args& a, hipStream_t st) {
  if (a.mins) return a.scale_f16 ? launch_one_t<G, true, true>(a, st) : launch_one_t<G, true, false>(a, st);
  return a.scale_f16 ? launch_one_t<G, false, true>(a, st) : launch_one_t<G, false, false>(a, st);
}

template <int P, int G>
hipError_t launch_p(const Gemv4Args& a, hipStream_t st) {
  if (a.mins) return a.scale_f16 ? launch_t<P, G, true, true>(a, st) : launch_t<P, G, true, false>(a, st);
  return a.scale_f16 ? launch_t<P, G, false, true>(a, st) : launch_t<P, G, false, false>(a, st);
}

template <int G>
hipError_t launch_g(const Gemv4Args& a, hipStream_t st) {
  if (a.M == 1) return launch_one<G>(a, st);
  switch ((a.M + 3) / 4) {
    case 1: return launch_p<1, G>(a, st);
    case 2: return launch_p<2, G>(a, st);
    case 3: return launch_p<3, G>(a, st);
    default: return launch_p<4, G>(a, st);
  }
}

}  // namespace

size_t gemv4_room(int M, int K) {
  return M <= 4 ? 0 : (size_t)((K + kStep - 1) / kStep) * ((size_t)(M + 3) / 4 * kPassBytes + kSumBytes);
}

hipError_t launch_gemv4(const Gemv4Args& a, hipStream_t st) {
  if (a.N0 + a.N1 + a.N2 <= 0 || a.M <= 0) return hipSuccess;
  return a.group == 32 ? launch_g<32>(a, st) : a.group == 64 ? launch_g<64>(a, st) : launch_g<128>(a, st);
}

}  // namespace bg
