// Linear attention with a decay for each head, 64 rows at a time (prompts).
//
// Within a chunk, with G_i the sum of its log decays up to row i and S the state before it:
//   A_ij = beta_i e^(G_i - G_j) k_i . k_j  (i > j)       T = (I + A)^-1 diag(beta)
//   V'   = T (V - e^G K S)                               P_ij = e^(G_i - G_j) q_i . k_j  (i >= j)
//   O    = scale (e^G Q S + P V')                        S  <- e^(G_n) S + K^T (e^(G_n - G) V')
// ("sum": V' = V). Everything that does not need S is one launch over all chunks (linear_chunk_prepare); the
// scan (linear_chunk_scan) then walks a sequence's chunks with 32 value dims of a head a workgroup.
//
// Precision: products run on the bf16 matrix cores with each f32 operand as three bf16 parts, which hold all of its 24
// bits and, down to 2^-109, its exponents: six products of nine, the others being below 2^-23 of a product, summed
// in f32. Every row and value dim is as good as an f32 sum makes it, whatever its neighbours' sizes. (Two f16 parts
// and three products are faster, prompt of 8192 rows 490 us instead of 617, but want one power of two for all rows of
// a value dim: a large state or value that the rows behind it have forgotten leaves those with as many bits fewer.) The
// decays' sums are taken in f64: their differences over a chunk would lose 2^-24 of the sums. T is found in f32: its
// diagonal blocks of 16 rows by substitution, the others from them with f32 matrix products. Values below 2^-109 count in
// steps of 2^-133, the smallest bf16.
//
// A column whose V or S is not finite, or so large that a sum on the way could overflow, and every column of a chunk
// whose K, Q, decays or strengths are not finite, is done again row by row: zero times infinity would reach
// rows before it. Its other columns keep their results (a matrix product's columns do not mix).
#include <algorithm>
#include <cstddef>

#include "bg_common.h"
#include "bg_linear.h"

namespace bg {

namespace {

typedef __bf16 part8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int kParts = 3;     // of an operand: largest first
constexpr int kFewScans = 128;  // workgroups of 32 value dims
constexpr int kPrepared = 768;   // workgroups that the preparation is split into, at most
constexpr int kPad = 68;      // row stride of 64 x 64 matrices in LDS
constexpr double kLowest = -1e4;  // of a log decay: e^g is 0 in f32 from -104 on

// What the scan needs of a chunk and head beside its operands: e^G_n, and the size (as bits) from which on a value of S
// or V could overflow a sum on its way; 0 where something is not finite.
struct ChunkMeta {
  float whole;
  uint32_t limit;
  int pad[30];
};
static_assert(sizeof(ChunkMeta) == 128, "meta");

// Operands of a chunk in the order the matrix instructions take them: [tile of 16 rows][32 of k][part][lane], a
// lane's k values being 16 (j / 4) + 4 g + j % 4 of the 32 for j = 0..7 (g = lane / 16), so that a product's
// result (rows 4 g + r of a tile) is the next one's operand without leaving its lane.
template <int DK>
struct ChunkSpace {
  static constexpr int NKB = DK / 32;
  static constexpr int K = 0, Q = K + 4 * NKB * kParts * 64, KT = Q + 4 * NKB * kParts * 64, PER_K = KT + (DK / 16) * 2 * kParts * 64;  // in part8
  static constexpr int T = 0, P = T + 4 * 2 * kParts * 64, G = P + 4 * 2 * kParts * 64, META = G + 128 / 4, PER_H = META + 8;          // in 16 bytes
};

// The workspace, as memory that is known to be the device's: through a pointer of no known kind its loads would
// count as LDS accesses too, and every barrier wait for them.
#define BG_GLOBAL __attribute__((address_space(1)))
typedef BG_GLOBAL part8 gpart8;
__device__ inline gpart8* workspace(const LinBatchView& b) { return (gpart8*)(b.ws ? b.ws : b.hdr->ws); }

__device__ inline int top_exponent(float x) { return __builtin_amdgcn_frexp_expf(x); }  // x < 2^e; 0 for 0
__device__ inline uint32_t mag(float x) { return __float_as_uint(x) & 0x7fffffffu; }
constexpr uint32_t kInf = 0x7f800000u;

// two values as bf16, rounded to nearest: the first in the low half
__device__ inline uint32_t round2(float a, float b) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), b2));
}
__device__ inline void split2(float a, float b, uint32_t (&to)[kParts]) {
#pragma unroll
  for (int p = 0; p < kParts; p++) {
    to[p] = round2(a, b);
    a -= __uint_as_float(to[p] << 16);
    b -= __uint_as_float(to[p] & 0xffff0000u);
  }
}
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
__device__ inline void split4(float a, float b, float c, float d, u2 (&to)[kParts]) {
  uint32_t x[kParts], y[kParts];
  split2(a, b, x);
  split2(c, d, y);
#pragma unroll
  for (int p = 0; p < kParts; p++) to[p] = u2{x[p], y[p]};
}
__device__ inline void split8(const float (&x)[8], part8 (&to)[kParts]) {
  uint32_t h[4][kParts];
#pragma unroll
  for (int i = 0; i < 4; i++) split2(x[2 * i], x[2 * i + 1], h[i]);
#pragma unroll
  for (int p = 0; p < kParts; p++) to[p] = __builtin_bit_cast(part8, u4{h[0][p], h[1][p], h[2][p], h[3][p]});
}
// c += a b for N tiles of columns, their chains side by side, the smallest products first
template <int N>
__device__ inline void products(const part8 (&a)[kParts], const part8 (&b)[N][kParts], f4 (&c)[N]) {
#pragma unroll
  for (int both = 2; both >= 0; both--)
#pragma unroll
    for (int p = both; p >= 0; p--)
#pragma unroll
      for (int i = 0; i < N; i++) c[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[p], b[i][both - p], c[i], 0, 0, 0);
}
__device__ inline f4 product(const part8 (&a)[kParts], const part8 (&b)[kParts], f4 c) {
#pragma unroll
  for (int both = 2; both >= 0; both--)
#pragma unroll
    for (int p = both; p >= 0; p--) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[p], b[both - p], c, 0, 0, 0);
  return c;
}
// e^x, x in 64 bits: the float next to x alone would leave 2^-25 of x
__device__ inline float exp_of(double x) {
  const float h = (float)x, e = expf(h);
  return fmaf(e, (float)(x - (double)h), e);
}
// over the four lane groups that hold a column's rows (or a row's k values)
__device__ inline uint32_t groups_max(uint32_t v) {
  auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(r[0], r[1]);
  r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(r[0], r[1]);
}
__device__ inline float groups_sum(float v) {
  float2 r = pair16(v);
  r = pair32(r.x + r.y);
  return r.x + r.y;
}
__device__ inline uint32_t wave_umax(uint32_t v) {
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, m));
  return groups_max(v);
}

__device__ inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ inline __amdgpu_buffer_rsrc_t buffer(const void* p, uint32_t bytes) {
  const uint64_t a = (uint64_t)p;
  const uint64_t u = (uint64_t)(uint32_t)uniform((int)(uint32_t)a) | (uint64_t)(uint32_t)uniform((int)(uint32_t)(a >> 32)) << 32;
  return __builtin_amdgcn_make_buffer_rsrc((void*)u, (short)0, (int)bytes, 0x00020000);
}
__device__ inline part8 load8(__amdgpu_buffer_rsrc_t r, int offset, int at) {  // `at` part8s behind byte `offset`
  return __builtin_bit_cast(part8, __builtin_amdgcn_raw_buffer_load_b128(r, offset, 16 * at, 0));
}
// x, copied here: a copy that the compiler puts at its next use would wait there for what x is loaded with anew
__device__ inline float moved(float x) {
  float y;
  asm volatile("v_mov_b32 %0, %1" : "=v"(y) : "v"(x));
  return y;
}
// x, which the compiler may not keep ready beside its multiples for the whole loop (those spilled)
__device__ inline int afresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// One chunk and key head, and `each` of its value heads: blockIdx.x a unit from u0 on, blockIdx.y the key head and which of
// its value heads.
template <int DK, bool DELTA>
__global__ __launch_bounds__(256, 3) void linear_chunk_prepare(LinLayer L, LinBatchView b, LinAttnArgs a, int u0, int each) {
  using W = ChunkSpace<DK>;
  constexpr int NKB = W::NKB;
  constexpr int kMat = 64 * kPad * 4, kFrag = 4 * NKB * kParts * 64 * 16;
  __shared__ __align__(16) char mem[2 * kMat > kFrag ? 2 * kMat : kFrag];
  __shared__ double gsums[4][64];            // of four value heads at a time, a wave each
  __shared__ float strengths[4][64], gtop[4][3];
  __shared__ int gbad[4];
  __shared__ uint32_t most[4], bits[4];
  __shared__ float sums[4];
  part8* frag = (part8*)mem;                 // K, while products with it run
  float* Am = (float*)mem;                   // then A
  float* Tm = (float*)(mem + kMat);          // P, then T
  const LinUnit u = b.units[u0 + blockIdx.x];
  if (u0 + (int)blockIdx.x >= b.hdr->n_chunk_units) return;
  const int rep = L.v_heads / L.k_heads, parts = (rep + each - 1) / each, kh = blockIdx.y / parts;
  const int i0 = blockIdx.y % parts * each, i1 = min(i0 + each, rep);
  const int wave = uniform(threadIdx.x >> 6), lane_ = threadIdx.x & 63;
  gpart8* wk = workspace(b) + (size_t)blockIdx.x * (L.k_heads * W::PER_K + L.v_heads * W::PER_H);
  gpart8* wh0 = wk + (size_t)L.k_heads * W::PER_K;
  wk += (size_t)kh * W::PER_K;

  f4 kk[4], qk[4];
  float kmax, qmax;
  bool bad_k;
  {
  const int lane = lane_, m = lane & 15, g = lane >> 4;
  // this wave's 16 rows of K and Q as operands
  const int row = 16 * wave + m;
  const bool live = row < u.n;
  const size_t at = ((size_t)(u.row0 + (live ? row : 0)) * L.k_heads + kh) * DK + 4 * g;
  float kx[NKB][8], qx[NKB][8];
  uint32_t km = 0, qm = 0;
#pragma unroll
  for (int kb = 0; kb < NKB; kb++)
#pragma unroll
    for (int half = 0; half < 2; half++) {
      const f4 k = *(const f4*)(a.k + at + 32 * kb + 16 * half), q = *(const f4*)(a.q + at + 32 * kb + 16 * half);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        kx[kb][4 * half + e] = live ? k[e] : 0.0f;
        qx[kb][4 * half + e] = live ? q[e] : 0.0f;
        km = max(km, mag(kx[kb][4 * half + e]));
        qm = max(qm, mag(qx[kb][4 * half + e]));
      }
    }
  km = wave_umax(km);
  qm = wave_umax(qm);
  if (lane == 0) {
    most[wave] = km;
    bits[wave] = qm;
  }
  const int mine = wave * NKB * kParts * 64 + lane;  // this wave's operands
#pragma unroll
  for (int kb = 0; kb < NKB; kb++) {
    part8 x[kParts];
    split8(kx[kb], x);
#pragma unroll
    for (int p = 0; p < kParts; p++) {
      frag[mine + (kb * kParts + p) * 64] = x[p];
      if constexpr (DELTA)
        if (i0 == 0) wk[W::K + mine + (kb * kParts + p) * 64] = x[p];
    }
  }
  __syncthreads();
  const uint32_t kall = max(max(most[0], most[1]), max(most[2], most[3]));
  const uint32_t qall = max(max(bits[0], bits[1]), max(bits[2], bits[3]));
  bad_k = kall >= kInf || qall >= kInf;
  kmax = __uint_as_float(kall);
  qmax = __uint_as_float(qall);
  // K^T: this wave's tiles of 16 key dims
  if (i0 == 0) {
    const __bf16* e = (const __bf16*)frag;
#pragma unroll
    for (int i = 0; i < DK / 64; i++) {
      const int td = wave * (DK / 64) + i;
#pragma unroll
      for (int kb2 = 0; kb2 < 2; kb2++)
#pragma unroll
        for (int p = 0; p < kParts; p++) {
          asm volatile("" ::: "memory");
          part8 x;
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const int tile = 2 * kb2 + (j >> 2), from = 4 * g + (j & 3) + 16 * (m >> 2);
            x[j] = e[(((tile * NKB + (td >> 1)) * kParts + p) * 64 + from) * 8 + 4 * (td & 1) + (m & 3)];
          }
          wk[W::KT + ((td * 2 + kb2) * kParts + p) * 64 + lane] = x;
        }
    }
  }
  // row tile `wave` of K K^T and Q K^T (its operands made or read where they are used: kept through the loop they spilled)
#pragma unroll
  for (int ct = 0; ct < 4; ct++) kk[ct] = qk[ct] = f4{0, 0, 0, 0};
#pragma unroll
  for (int kb = 0; kb < NKB; kb++) {
    asm volatile("" ::: "memory");
    part8 kp[kParts], qp[kParts];
    split8(qx[kb], qp);
#pragma unroll
    for (int p = 0; p < kParts; p++) {
      kp[p] = frag[mine + (kb * kParts + p) * 64];
      if (i0 == 0) wk[W::Q + mine + (kb * kParts + p) * 64] = qp[p];
    }
#pragma unroll
    for (int ct = 0; ct < 4; ct++) {
      if (ct > wave) continue;
      part8 x[kParts];
#pragma unroll
      for (int p = 0; p < kParts; p++) x[p] = frag[((ct * NKB + kb) * kParts + p) * 64 + lane];
      if constexpr (DELTA) kk[ct] = product(kp, x, kk[ct]);
      qk[ct] = product(qp, x, qk[ct]);
    }
  }
  }

#pragma unroll 1
  for (int i = i0; i < i1; i++) {
    const int h = kh * rep + i;
    gpart8* wh = wh0 + (size_t)h * W::PER_H;
    const auto rh = buffer((const void*)wh, 16 * W::PER_H);
    const int lane = afresh(lane_), m = lane & 15, g = lane >> 4, row = 16 * wave + m;
    __syncthreads();  // the frag reads, or the head before
    if ((i - i0 & 3) == 0) {
      if (i + wave < i1) {  // the decays' sums: lane = row
        const bool on = lane < u.n;
        const size_t rr = u.row0 + (on ? lane : 0);
        const int hh = h + wave;
        const float gv = on ? a.g[(a.g_stride ? rr * a.g_stride : 0) + hh] : 0.0f;
        double s = gv < (float)kLowest ? kLowest : (double)gv;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const double o = __shfl_up(s, d);
          if (lane >= d) s += o;
        }
        const double end = __shfl(s, 63);
        const float be = DELTA ? (on ? a.beta[rr * L.v_heads + hh] : 0.0f) : 1.0f;
        gsums[wave][lane] = s;
        strengths[wave][lane] = be;
        const float eg = exp_of(s), fg = exp_of(end - s);
        BG_GLOBAL float* gg = (BG_GLOBAL float*)(wh + (size_t)wave * W::PER_H + W::G);
        gg[lane] = eg;
        gg[64 + lane] = on ? fg : 0.0f;
        const float gm = __uint_as_float(wave_umax(mag(eg))), fm = __uint_as_float(wave_umax(mag(fg)));
        const bool odd = __any(mag(eg) >= kInf || mag(fg) >= kInf || mag(be) >= kInf);
        if (lane == 0) {
          gtop[wave][0] = gm;
          gtop[wave][1] = fm;
          gtop[wave][2] = exp_of(end);
          gbad[wave] = odd;
        }
      }
      __syncthreads();
    }
    const double* gsum = gsums[i - i0 & 3];
    const float* strength = strengths[i - i0 & 3];
    const float gmax = gtop[i - i0 & 3][0], fmax_ = gtop[i - i0 & 3][1], whole = gtop[i - i0 & 3][2];
    bool bad = bad_k || gbad[i - i0 & 3];
    // A and P of this wave's rows
    uint32_t pm = 0;
#pragma unroll
    for (int ct = 0; ct < 4; ct++) {
      if (ct > wave) continue;
      const int c = 16 * ct + m;
      const double gc = gsum[c];
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int w = 16 * wave + 4 * g + r;
        const float fade = expf(c <= w ? (float)(gsum[w] - gc) : -__builtin_inff());  // 0 above the diagonal
        const float p = c <= w ? fade * qk[ct][r] : 0.0f;
        Tm[w * kPad + c] = p;
        pm = max(pm, mag(p));
        if constexpr (DELTA) Am[w * kPad + c] = c < w ? strength[w] * (fade * kk[ct][r]) : 0.0f;
      }
    }
    pm = wave_umax(pm);
    if (lane == 0) bits[wave] = pm;
    // P's operands: rows written by this wave itself
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    auto operand = [&](const float* M, int kb, bool strong, float& sum, float (&x)[8]) {
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const int ct = 2 * kb + half;
        f4 v = f4{0, 0, 0, 0};
        if (ct <= wave) v = *(const f4*)(M + row * kPad + 16 * ct + 4 * g);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float y = ct <= wave && strong ? v[e] * strength[16 * ct + 4 * g + e] : v[e];
          x[4 * half + e] = y;
          sum += fabsf(y);
        }
      }
    };
    auto put = [&](int base, int kb, const float (&x)[8]) {
      part8 parts[kParts];
      split8(x, parts);
      const int at = 16 * lane + 2 * kParts * 1024 * wave;
#pragma unroll
      for (int p = 0; p < kParts; p++)
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, parts[p]), rh, at, 16 * (base + (kb * kParts + p) * 64), 0);
    };
#pragma unroll
    for (int kb = 0; kb < 2; kb++) {
      float x[8], none = 0;
      if (2 * kb > wave) continue;
      operand(Tm, kb, false, none, x);
      put(W::P, kb, x);
    }
    float tsum = 1.0f;
    if constexpr (DELTA) {
      __syncthreads();  // P is read; A is there
      {  // the diagonal block of this wave, a column a lane (four lanes alike)
        float x[16];
#pragma unroll
        for (int q = 0; q < 8; q++) {
          // two rows' values at a time: all sixteen rows' at once do not fit
          asm volatile("" ::: "memory");
          f4 w[2][4];
#pragma unroll
          for (int r = 0; r < 2; r++)
#pragma unroll
            for (int c = 0; c <= q / 2; c++) w[r][c] = *(const f4*)(Am + (16 * wave + 2 * q + r) * kPad + 16 * wave + 4 * c);
#pragma unroll
          for (int r = 0; r < 2; r++) {
            float y = 2 * q + r == m ? 1.0f : 0.0f;
#pragma unroll
            for (int c = 0; c < 2 * q + r; c++) y = fmaf(-w[r][c >> 2][c & 3], x[c], y);
            asm volatile("" : "+v"(y));  // here, and not where a lane stores it: the values it is made of go
            x[2 * q + r] = y;
          }
        }
#pragma unroll
        for (int r = 0; r < 16; r++)
          if ((r >> 2) == g) Tm[(16 * wave + r) * kPad + 16 * wave + m] = x[r];
      }
      __syncthreads();
      {  // the blocks below it: column block `wave`
        f4 t[4];
#pragma unroll
        for (int r = 0; r < 4; r++) t[0][r] = Tm[(16 * wave + 4 * g + r) * kPad + 16 * wave + m];
#pragma unroll
        for (int d = 1; d < 4; d++) {
          const int I = wave + d;
          if (I > 3) break;
          f4 acc = f4{0, 0, 0, 0};
#pragma unroll
          for (int k = 0; k < d; k++) {
            const f4 x = *(const f4*)(Am + (16 * I + m) * kPad + 16 * (wave + k) + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; r++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[r], t[k][r], acc, 0, 0, 0);
          }
          const f4 x = *(const f4*)(Tm + (16 * I + m) * kPad + 16 * I + 4 * g);
          t[d] = f4{0, 0, 0, 0};
#pragma unroll
          for (int r = 0; r < 4; r++) t[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[r], -acc[r], t[d], 0, 0, 0);
#pragma unroll
          for (int r = 0; r < 4; r++) Tm[(16 * I + 4 * g + r) * kPad + 16 * wave + m] = t[d][r];
        }
      }
      __syncthreads();
      float sum = 0.0f;
#pragma unroll
      for (int kb = 0; kb < 2; kb++) {
        float x[8];
        if (2 * kb > wave) continue;
        operand(Tm, kb, true, sum, x);
        put(W::T, kb, x);
      }
      sum = __uint_as_float(wave_umax(mag(groups_sum(sum))));  // (a NaN counts as the largest)
      if (lane == 0) sums[wave] = sum;
      __syncthreads();
      tsum = fmaxf(fmaxf(sums[0], sums[1]), fmaxf(sums[2], sums[3]));
      for (int w = 0; w < 4; w++) bad = bad || !(sums[w] < 0x1p60f);
    } else {
      __syncthreads();
    }
    for (int w = 0; w < 4; w++) bad = bad || !(__uint_as_float(bits[w]) < 0x1p60f);
    if (threadIdx.x == 0) {
      // what a value of S or V may grow by: through e^G Q S; through Y, T and e^(G_n - G) to K^T V' or P V'
      const float pmax = __uint_as_float(max(max(bits[0], bits[1]), max(bits[2], bits[3])));
      constexpr int kSum = DK == 64 ? 6 : 7;
      const int eg = max(0, top_exponent(gmax)), ek = top_exponent(kmax), y = DELTA ? max(0, kSum + ek + eg) + 1 : 0;
      const int v = y + max(0, top_exponent(tsum)) + max(0, top_exponent(fmax_));
      const int grow = max(max(eg, kSum + top_exponent(qmax) + eg), v + max(0, 6 + max(ek, top_exponent(pmax)))) + 1;
      BG_GLOBAL ChunkMeta* meta = (BG_GLOBAL ChunkMeta*)(wh + W::META);
      meta->whole = whole;
      meta->limit = bad || grow > 220 ? 0 : __float_as_uint(ldexpf(1.0f, 126 - grow));
    }
  }
}

// A sequence's chunks from u0 up to u1 (its window of the workspace) for 16 NT value dims of a head. Four waves carry
// the state: wave w has rows 16 w .. of K S, Y and V' and a quarter of the key dims of S, all in registers; what
// the next product needs of the others goes through LDS, three barriers a chunk. Four more waves, a SIMD's second,
// make the output from what lies in LDS between those barriers. The next chunk's operands are loaded into the
// registers of this one's as soon as their last product has been issued: by buffer loads, whose one lane
// offset and scalar rest leave the registers to the operands. (A register too many costs a wait for everything
// in flight when it is read back; with two f16 parts an operand: 64-bit addresses in vector registers 14 us a chunk, the
// row offsets of V and the output kept through the loop 6.8, without 4.0, two sets of waves 2.9.) 4.1 us a chunk: the
// chain of three products of six matrix instructions a tile and step, each with its operand's way through LDS. By
// count the matrix cores and LDS are a third busy.
template <int DK, int DV, bool DELTA, int NT>
__global__ __launch_bounds__(512, 2) void linear_chunk_scan(LinLayer L, LinBatchView b, LinAttnArgs a, int u0, int u1) {
  using W = ChunkSpace<DK>;
  constexpr int NKB = W::NKB, MT = DK / 64, kCols = 16 * NT, SLICES = DV / kCols;
  constexpr int kRows = 2 * NT * kParts * 64;    // of an operand whose k are the chunk's rows
  __shared__ part8 Sb[NKB * NT * kParts * 64];   // the state as an operand
  __shared__ part8 Yb[kRows], Vb[2][kRows], Fb[kRows];  // Y, V' (of this chunk and the one before), e^(G_n - G) V'
  __shared__ uint32_t sout[4], vout[4];          // the waves' columns with a value of S, of V past the chunk's limit
  __shared__ float plain[kCols][DK + 4];        // columns that are done row by row: the state before
  __shared__ int slow_from[kCols];              // this chunk of the sequence
  // a key head's value heads and slices, which read the same operands, run on one XCD
  const int rep = L.v_heads / L.k_heads, members = rep * SLICES;
  const int x = blockIdx.x & 7, j = blockIdx.x >> 3;
  const int group = x + 8 * (j / members), member = j % members;
  const int seq = group / L.k_heads, kh = group % L.k_heads;
  if (seq >= b.hdr->n_chunked) return;
  const LinSeq* sp = b.seqs + seq;
  const int row0 = uniform(sp->row0), rows = uniform(sp->rows), unit0 = uniform(sp->unit0);
  const int first = max(unit0, u0), last = min(unit0 + uniform(sp->n_units), u1);
  if (first >= last) return;
  const int h = kh * rep + member / SLICES, col0 = (member % SLICES) * kCols;
  const int role = uniform(threadIdx.x >> 8), wave = uniform((threadIdx.x >> 6) & 3);
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const size_t per_unit = (size_t)L.k_heads * W::PER_K + (size_t)L.v_heads * W::PER_H;
  const part8* ws = (const part8*)(b.ws ? b.ws : b.hdr->ws);

  const int at_k = 16 * lane + wave * (NKB * kParts * 64 * 16), at_t = 16 * lane + wave * (2 * kParts * 64 * 16);
  static_assert(NKB == 2 * MT, "the operands of a wave's rows and of its key dims lie alike");
  auto keys = [&](int u) { return buffer(ws + (size_t)(u - u0) * per_unit + (size_t)kh * W::PER_K, 16 * W::PER_K); };
  auto head = [&](int u) {
    return buffer(ws + (size_t)(u - u0) * per_unit + (size_t)L.k_heads * W::PER_K + (size_t)h * W::PER_H, 16 * W::PER_H);
  };
  const int vrow = L.v_heads * DV * 4;  // bytes of a row of V and of the output
  const int vlane = (16 * wave + 4 * g) * vrow + 4 * n;
  auto values = [&](const float* p, int u) {  // the chunk's rows: those behind them read as zero and are not stored
    const int r = kLinChunk * (u - unit0);
    return buffer(p + ((size_t)(row0 + r) * L.v_heads + h) * DV + col0, (min(kLinChunk, rows - r) - 1) * vrow + 4 * kCols);
  };
  u2 meta;  // the chunk's ChunkMeta, in every lane
  auto load_meta = [&](int u) { meta = __builtin_bit_cast(u2, __builtin_amdgcn_raw_buffer_load_b64(head(u), 0, 16 * W::META, 0)); };
  auto load_fade = [&](int u, int at) {  // this wave's rows' e^G (at 0) or e^(G_n - G) (256)
    return __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(head(u), 64 * wave + 16 * (afresh(lane) >> 4), 16 * W::G + at, 0));
  };
  // bit c: column c, of which a lane's largest value (as bits) is in top[c / 16], is not for the chunk's products
  auto marked = [&](const uint32_t (&top)[NT]) {
    const uint32_t limit = uniform((int)meta[1]);
    uint32_t m = 0;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const uint64_t b = __ballot(top[nt] >= limit);
      const uint32_t w = (uint32_t)b | (uint32_t)(b >> 32);
      m |= ((w | w >> 16) & 0xffffu) << (16 * nt);
    }
    return m;
  };
  auto marks = [&]() { return (uint32_t)uniform((int)(sout[0] | sout[1] | sout[2] | sout[3] | vout[0] | vout[1] | vout[2] | vout[3])); };
  auto load_v = [&](int u, float (&to)[NT][4]) {
    const auto r = values(a.v, u);
    int at = afresh(vlane);
#pragma unroll
    for (int e = 0; e < 4; e++, at += vrow)
#pragma unroll
      for (int nt = 0; nt < NT; nt++) to[nt][e] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, at + 64 * nt, 0, 0));
  };
  auto operands = [&](const part8* from, int kb, part8 (&x)[NT][kParts]) {  // all column tiles
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int p = 0; p < kParts; p++) x[nt][p] = from[((kb * NT + nt) * kParts + p) * 64 + lane];
  };
  uint32_t slow = 0;  // the columns that are done row by row
  f4 S[MT][NT];

  if (role == 0) {
    __builtin_amdgcn_s_setprio(2);  // the state is what everything waits for
    part8 fk[NKB][kParts], ft[2][kParts], fkt[MT][2][kParts];
    float v[2][NT][4];  // this chunk's and the next one's
    f4 eg, fg;
    auto load_k = [&](int u) {
      const auto r = keys(u);
      if constexpr (DELTA)
#pragma unroll
        for (int kb = 0; kb < NKB; kb++)
#pragma unroll
          for (int p = 0; p < kParts; p++) fk[kb][p] = load8(r, at_k, W::K + (kb * kParts + p) * 64);
    };
    auto load_t = [&](int u) {
      const auto r = head(u);
      if constexpr (DELTA)
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
          for (int p = 0; p < kParts; p++) ft[kb][p] = load8(r, at_t, W::T + (kb * kParts + p) * 64);  // (also what no product takes)
    };
    auto load_kt = [&](int u) {
      const auto r = keys(u);
#pragma unroll
      for (int i = 0; i < MT; i++)
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
          for (int p = 0; p < kParts; p++) fkt[i][kb][p] = load8(r, at_k, W::KT + ((i * 2 + kb) * kParts + p) * 64);
    };
    auto note = [&]() {  // this wave's key dims
      uint32_t top[NT] = {};
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
          for (int r = 0; r < 4; r++) top[nt] = max(top[nt], mag(S[i][nt][r]));
      sout[wave] = marked(top);
    };
    auto put4 = [&](part8* to, int tile, int nt, float a, float b, float c, float d) {
      u2 x[kParts];
      split4(a, b, c, d, x);
      char* at = (char*)(to + (((tile >> 1) * NT + nt) * kParts) * 64 + lane) + 8 * (tile & 1);
#pragma unroll
      for (int p = 0; p < kParts; p++) *(u2*)(at + p * 64 * 16) = x[p];
    };
    auto put_state = [&]() {
#pragma unroll
      for (int i = 0; i < MT; i++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++) put4(Sb, wave * MT + i, nt, S[i][nt][0], S[i][nt][1], S[i][nt][2], S[i][nt][3]);
    };
    const int from = uniform(first == unit0 ? sp->src : sp->dst);
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
        S[i][nt] = from >= 0 ? *(const f4*)(L.state + (((size_t)from * L.v_heads + h) * DV + col0 + 16 * nt + n) * DK + 16 * (wave * MT + i) + 4 * g)
                             : f4{0, 0, 0, 0};
    load_v(first, v[0]);
    load_meta(first);
    load_k(first);
    eg = load_fade(first, 0);
    fg = load_fade(first, 256);
    load_t(first);
    load_kt(first);
    load_v(min(first + 1, last - 1), v[1]);
    note();
    put_state();
#pragma unroll 1
    for (int u = first; u < last; u++) {
      const int next = min(u + 1, last - 1);
      const float whole = __uint_as_float(uniform((int)meta[0]));
      __syncthreads();  // the state, and what is noted of it and of V
      const uint32_t out = marks();
      load_meta(next);
      f4 vp[NT];
      if constexpr (DELTA) {
        f4 ks[NT] = {};
#pragma unroll
        for (int kb = 0; kb < NKB; kb++) {
          part8 x[NT][kParts];
          operands(Sb, kb, x);
          products(fk[kb], x, ks);
        }
        __builtin_amdgcn_sched_barrier(0);
        load_k(next);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          float y[4];
#pragma unroll
          for (int r = 0; r < 4; r++) y[r] = fmaf(-eg[r], ks[nt][r], v[0][nt][r]);
          put4(Yb, wave, nt, y[0], y[1], y[2], y[3]);
        }
        eg = load_fade(next, 0);
        __syncthreads();
        for (int nt = 0; nt < NT; nt++) vp[nt] = f4{0, 0, 0, 0};
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
          if (2 * kb <= wave) {
            part8 x[NT][kParts];
            operands(Yb, kb, x);
            products(ft[kb], x, vp);
          }
        __builtin_amdgcn_sched_barrier(0);
        load_t(next);
        __builtin_amdgcn_sched_barrier(0);
      } else {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int r = 0; r < 4; r++) vp[nt][r] = v[0][nt][r];
      }
#pragma unroll
      for (int nt = 0; nt < NT; nt++) put4(Fb, wave, nt, fg[0] * vp[nt][0], fg[1] * vp[nt][1], fg[2] * vp[nt][2], fg[3] * vp[nt][3]);
      fg = load_fade(next, 256);
      __syncthreads();
      f4 acc[MT][NT] = {};
#pragma unroll
      for (int kb = 0; kb < 2; kb++) {
        part8 x[NT][kParts];
        operands(Fb, kb, x);
#pragma unroll
        for (int i = 0; i < MT; i++) products(fkt[i][kb], x, acc[i]);
      }
      __builtin_amdgcn_sched_barrier(0);
      load_kt(next);
      __builtin_amdgcn_sched_barrier(0);
      if (const uint32_t todo = out & ~slow) {  // columns that leave the chunks here
        const int l = afresh(lane);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          const int c = 16 * nt + (l & 15);
          if (!(todo >> c & 1)) continue;
#pragma unroll
          for (int i = 0; i < MT; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) plain[c][16 * (wave * MT + i) + 4 * (l >> 4) + r] = S[i][nt][r];
          if (wave == 0) slow_from[c] = u - unit0;
        }
        slow |= todo;
      }
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
          for (int r = 0; r < 4; r++) S[i][nt][r] = fmaf(whole, S[i][nt][r], acc[i][nt][r]);
#pragma unroll
        for (int r = 0; r < 4; r++) v[0][nt][r] = moved(v[1][nt][r]);
      }
      note();
      put_state();
      // V' for the output waves, which take it behind the next barrier
#pragma unroll
      for (int nt = 0; nt < NT; nt++) put4(Vb[u & 1], wave, nt, vp[nt][0], vp[nt][1], vp[nt][2], vp[nt][3]);
      __builtin_amdgcn_sched_barrier(0);
      load_v(min(u + 2, last - 1), v[1]);
      __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
  } else {
    part8 fq[NKB][kParts], fp[2][kParts];
    f4 eg;
    auto load_q = [&](int u) {
      const auto r = keys(u);
#pragma unroll
      for (int kb = 0; kb < NKB; kb++)
#pragma unroll
        for (int p = 0; p < kParts; p++) fq[kb][p] = load8(r, at_k, W::Q + (kb * kParts + p) * 64);
    };
    auto load_p = [&](int u) {
      const auto r = head(u);
#pragma unroll
      for (int kb = 0; kb < 2; kb++)
#pragma unroll
        for (int p = 0; p < kParts; p++) fp[kb][p] = load8(r, at_t, W::P + (kb * kParts + p) * 64);
    };
    auto note_v = [&](const float (&of)[NT][4]) {
      uint32_t top[NT] = {};
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int r = 0; r < 4; r++) top[nt] = max(top[nt], mag(of[nt][r]));
      vout[wave] = marked(top);
    };
    float v[NT][4];
    f4 o[NT] = {};
    // what V' (in Vb[half]) adds to the rows of chunk u, and their store, but for the columns `left_out`
    auto finish = [&](int u, int half, uint32_t left_out) {
      const auto ro = values(a.out, u);
      f4 acc[NT] = {};
#pragma unroll
      for (int kb = 0; kb < 2; kb++)
        if (2 * kb <= wave) {
          part8 x[NT][kParts];
          operands(Vb[half], kb, x);
          products(fp[kb], x, acc);
        }
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int r = 0; r < 4; r++) acc[nt][r] = fmaf(a.scale, acc[nt][r], o[nt][r]);
      }
      // (A column that is left out, and with the first chunk every one, is stored past the buffer's end, which drops it:
      // with a branch there a wait for what was loaded before would not know how many stores came after, and wait for them.)
      int at[NT];
#pragma unroll
      for (int nt = 0; nt < NT; nt++) at[nt] = left_out >> (16 * nt + n) & 1 ? 0x40000000 : afresh(vlane) + 64 * nt;
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++, at[nt - 1] += vrow)
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(acc[nt][r]), ro, at[nt], 0, 0);
    };
    load_v(first, v);
    load_meta(first);
    load_q(first);
    eg = load_fade(first, 0);
    load_p(first);
    note_v(v);
    load_v(min(first + 1, last - 1), v);
#pragma unroll 1
    for (int u = first; u < last; u++) {
      const int next = min(u + 1, last - 1);
      __syncthreads();
      const uint32_t out = marks();
      load_meta(next);
      f4 now[NT] = {};
#pragma unroll
      for (int kb = 0; kb < NKB; kb++) {
        part8 x[NT][kParts];
        operands(Sb, kb, x);
        products(fq[kb], x, now);
      }
      __builtin_amdgcn_sched_barrier(0);
      load_q(next);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (DELTA) __syncthreads();
      // the state waves hurry from here to the third barrier: the chunk before is finished behind it
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
          now[nt][r] = a.scale * (eg[r] * now[nt][r]);
          asm volatile("" : "+v"(now[nt][r]));  // here: moved to where it is read next, it would keep eg from its next load
        }
      }
      eg = load_fade(next, 0);
      __syncthreads();
      note_v(v);
      finish(max(u - 1, first), u & 1 ^ 1, u > first ? slow : ~0u);
      __builtin_amdgcn_sched_barrier(0);
      load_p(u);
      __builtin_amdgcn_sched_barrier(0);
      load_v(min(u + 2, last - 1), v);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int nt = 0; nt < NT; nt++) o[nt] = now[nt];
      slow |= out;
    }
    __syncthreads();
    finish(last - 1, (last - 1) & 1, slow);
  }
  float* left = L.state + (((size_t)uniform(sp->dst) * L.v_heads + h) * DV + col0) * DK;
  if (role == 0)
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
        if (!(slow >> (16 * nt + n) & 1)) *(f4*)(left + (16 * nt + n) * DK + 16 * (wave * MT + i) + 4 * g) = S[i][nt];
  if (!slow) return;
  // the other columns, eight lanes each, as linear_attn.hip does them
  __syncthreads();
  const int c = threadIdx.x >> 3, l = threadIdx.x & 7;
  if (c >= kCols || !(slow >> c & 1)) return;
  f4 st[DK / 32];
#pragma unroll
  for (int i = 0; i < DK / 32; i++) st[i] = *(const f4*)&plain[c][32 * i + 4 * l];
  const int end = min(rows, kLinChunk * (last - unit0));
#pragma unroll 1
  for (int t = kLinChunk * slow_from[c]; t < end; t++) {
    const size_t r = row0 + t;
    const float* kp = a.k + (r * L.k_heads + kh) * DK + 4 * l;
    const float* qp = a.q + (r * L.k_heads + kh) * DK + 4 * l;
    float hi, lo;
    fade_of(a.g[(a.g_stride ? r * a.g_stride : 0) + h], hi, lo);
    float sum = 0.0f;
    f4 kx[DK / 32];
#pragma unroll
    for (int i = 0; i < DK / 32; i++) {
      kx[i] = *(const f4*)(kp + 32 * i);
#pragma unroll
      for (int e = 0; e < 4; e++) sum = fmaf(st[i][e], kx[i][e], sum);
    }
    float d = a.v[(r * L.v_heads + h) * DV + col0 + c];
    if constexpr (DELTA) d = a.beta[r * L.v_heads + h] * (d - hi * group_sum<8>(sum));
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < DK / 32; i++) {
      const f4 q = *(const f4*)(qp + 32 * i);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        st[i][e] = fmaf(hi, st[i][e], fmaf(lo, st[i][e], kx[i][e] * d));
        sum = fmaf(st[i][e], q[e], sum);
      }
    }
    sum = group_sum<8>(sum);
    if (l == 0) a.out[(r * L.v_heads + h) * DV + col0 + c] = a.scale * sum;
  }
#pragma unroll
  for (int i = 0; i < DK / 32; i++) *(f4*)(left + c * DK + 32 * i + 4 * l) = st[i];
}

// The output norm of the chunks' rows, in place: DV / 4 lanes a row and head.
template <int DV>
__global__ __launch_bounds__(256) void linear_norm_kernel(LinLayer L, LinBatchView b, LinAttnArgs a) {
  constexpr int LG = DV / 4;
  const LinUnit u = b.units[blockIdx.x];
  if ((int)blockIdx.x >= b.hdr->n_chunk_units) return;
  const int grp = threadIdx.x / LG, c = 4 * (threadIdx.x % LG);
  const f4 w = *(const f4*)(a.norm + c);
  for (int i = blockIdx.y * (256 / LG) + grp; i < u.n * L.v_heads; i += gridDim.y * (256 / LG)) {
    const size_t at = ((size_t)u.row0 * L.v_heads + i) * DV + c;
    f4 o = *(const f4*)(a.out + at);
    const float inv = 1.0f / sqrtf(group_sum<LG>(fmaf(o[0], o[0], fmaf(o[1], o[1], fmaf(o[2], o[2], o[3] * o[3])))) / DV + a.eps);
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = o[e] * inv * w[e];
    if (a.gate) {
      const f4 z = *(const f4*)(a.gate + at);
#pragma unroll
      for (int e = 0; e < 4; e++) o[e] *= z[e] / (1.0f + expf(-z[e]));
    }
    *(f4*)(a.out + at) = o;
  }
}

template <int DK, int DV, bool DELTA, int NT>
void launch_scan(const LinLayer& L, const LinBatchView& b, const LinAttnArgs& a, int u0, int u1, hipStream_t st) {
  const int groups = b.n_chunked * L.k_heads, members = L.v_heads / L.k_heads * (DV / (16 * NT));
  hipLaunchKernelGGL((linear_chunk_scan<DK, DV, DELTA, NT>), dim3(8 * ((groups + 7) / 8) * members), dim3(512), 0, st, L, b, a, u0, u1);
}

template <int DK, int DV, bool DELTA>
hipError_t launch_t(const LinLayer& L, const LinBatchView& b, const LinAttnArgs& a, hipStream_t st) {
  // as few passes as the workspace allows, of one size
  const int most = b.n_chunked > 1 ? b.window : std::min<int>(b.window, std::max<size_t>(1, kLinCached / linear_unit_bytes(DK, L.k_heads, L.v_heads)));
  const int passes = (b.n_chunk_units + most - 1) / most, step = (b.n_chunk_units + passes - 1) / passes;
  for (int u0 = 0; u0 < b.n_chunk_units; u0 += step) {
    const int u1 = std::min(u0 + step, b.n_chunk_units);
    // A workgroup's value heads one after the other, or, where that leaves most of the GPU idle, workgroups of their own
    // that share a key head's products (16 key and 48 value heads, one chunk: prompt of 64 rows 36 us, so 27; four
    // prompts of 256, 16 chunks, 91 and 88; 32 chunks 160 and 169, 8192 rows 604 and 637).
    const int rep = L.v_heads / L.k_heads, parts = std::max(1, std::min(rep, kPrepared / ((u1 - u0) * L.k_heads)));
    const int each = (rep + parts - 1) / parts;
    hipLaunchKernelGGL((linear_chunk_prepare<DK, DELTA>), dim3(u1 - u0, L.k_heads * ((rep + each - 1) / each)), dim3(256), 0, st, L, b, a, u0, each);
    // 32 value dims a workgroup, or 16 where that still leaves one workgroup a CU (delta rule, 2048 rows of 16 heads, 64
    // workgroups of 32: 130 us, 128 of 16: 104; of two such prompts 176 and 163; three of 1024 rows 95 and 120. Sum, two of
    // 2048, k_dim 64: 78 and 59; three 103 and 116). More workgroups, each reading the same operands, take longer.
    if (b.n_chunked * L.v_heads * (DV / 32) <= kFewScans) launch_scan<DK, DV, DELTA, 1>(L, b, a, u0, u1, st);
    else launch_scan<DK, DV, DELTA, 2>(L, b, a, u0, u1, st);
  }
  if (a.norm)
    hipLaunchKernelGGL((linear_norm_kernel<DV>), dim3(b.n_chunk_units, (kLinChunk * L.v_heads * DV / 4 + 1023) / 1024), dim3(256), 0, st, L, b, a);
  return hipGetLastError();
}

template <int DK>
size_t unit_bytes(int k_heads, int v_heads) {
  return 16 * ((size_t)k_heads * ChunkSpace<DK>::PER_K + (size_t)v_heads * ChunkSpace<DK>::PER_H);
}

}  // namespace

size_t linear_unit_bytes(int DK, int k_heads, int v_heads) {
  return DK == 64 ? unit_bytes<64>(k_heads, v_heads) : unit_bytes<128>(k_heads, v_heads);
}

hipError_t launch_linear_chunks(const LinLayer& L, const LinBatchView& b, const LinAttnArgs& a, hipStream_t st) {
  if (a.beta) {
    if (L.DK == 64) return L.DV == 64 ? launch_t<64, 64, true>(L, b, a, st) : launch_t<64, 128, true>(L, b, a, st);
    return L.DV == 64 ? launch_t<128, 64, true>(L, b, a, st) : launch_t<128, 128, true>(L, b, a, st);
  }
  if (L.DK == 64) return L.DV == 64 ? launch_t<64, 64, false>(L, b, a, st) : launch_t<64, 128, false>(L, b, a, st);
  return L.DV == 64 ? launch_t<128, 64, false>(L, b, a, st) : launch_t<128, 128, false>(L, b, a, st);
}

}  // namespace bg
