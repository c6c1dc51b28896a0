// Attention of a batch over a paged KV cache on gfx950: any mix of single tokens, verifies and prompts,
// pages that sequences share scanned once for the rows of all of them.
//
// The plan (bg_paged_plan.h) hands every workgroup a unit: a tile of rows (row = (token, head of one kv
// head's group), so a loaded key serves G heads of every member token) times a chunk of positions. Two
// bodies, chosen by the unit's segment:
//   few     <= 32 rows (a token, a verify): bound by the cache's bytes. Each of the four waves takes
//           every fourth 32-position tile straight from the pages into matrix-core operand registers (no
//           LDS, no barrier), the next tile's K in flight under the softmax and its V under the next
//           scores; the waves' (o, m, l) meet in LDS at the end.
//   many    more rows (a shared prefix, a prompt): bound by the matrix cores. 128 rows, 32 a wave; the
//           positions staged through LDS once for all four waves, double-buffered.
//
// Results are f32-accurate, as the f32 activations and outputs are: an f16 operand holds 11 bits, so the
// query and the probabilities enter the f16 matrix cores as two parts each (hi = f16(x), lo = f16(x -
// hi): 22 bits), while what the pages hold is exact in one part (f16 values as they are, q8 codes as
// integers, their scales applied in f32). f32 pages run on the f32 matrix cores.
//   query   a row is scaled by a power of two that brings its largest value into [2^10, 2^11) (any
//           magnitude keeps its 22 bits; undone in the score's f32 factor);
//   p       2^(s - m + 8), m raised only when a tile's maximum passes it by 6 (most tiles skip the
//           rescale): p <= 2^14 stays below f16's 65504, and the smallest f16 step is 2^-32 of the
//           largest p;
//   q8 V    p is multiplied by the block scale of its position, over a power of two 2^ev that is at least
//           every scale so far (raised like m).
// S^T = K Q^T and O^T += V^T P^T: the score registers of a lane hold positions of one row, in exactly the
// order in which the V tile stores them (bg_common.h), so P enters the second product as it lies.
// Masked positions: scores are replaced, not added to; V beyond the positions written so far (a page's
// stale or never written slots, possibly NaN) is replaced by zero, its q8 scales too.
#include <algorithm>

#include "bg_paged.h"

namespace bg {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef __fp16 fp16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void* lds_ptr;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPShift = 8.0f;   // p = 2^(s - m + 8)
constexpr float kLazy = 6.0f;     // m is raised when a score passes it by this

union H8 {
  half8 h;
  u32x4 u;
  _Float16 e[8];
  fp16x2 p[4];
};

struct PagedKernelArgs {
  const char* k; const char* v;
  const float* ks; const float* vs;
  int kv_heads;
  PagedBatchView b;
  const float* q;
  float qscale;      // scale * log2(e)
  const float* gate; int gate_stride;
  float* out;
  int first, n_blocks;  // a launch's first unit and its units * kv heads; n_blocks 0: read the header
};

__device__ inline float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// x[0..7] as hi and lo f16 parts (each conversion truncates; lo holds what hi lost)
__device__ inline void split8(const float (&x)[8], H8& hi, H8& lo) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    hi.p[i] = __builtin_amdgcn_cvt_pkrtz(x[2 * i], x[2 * i + 1]);
    lo.p[i] = __builtin_amdgcn_cvt_pkrtz(x[2 * i] - (float)hi.e[2 * i], x[2 * i + 1] - (float)hi.e[2 * i + 1]);
  }
}

// 2^e with 2^e * top in [2^10, 2^11) for a row's largest |value|; 1 for zero, infinite and NaN rows
__device__ inline float row_factor(float top, float* undo) {
  const int e = (int)((__float_as_uint(top) >> 23) & 0xff);
  if (e == 0xff || top == 0.0f) {
    *undo = 1.0f;
    return 1.0f;
  }
  const int s = min(max(137 - e, -100), 100);  // both powers normal
  *undo = __uint_as_float((uint32_t)(127 - s) << 23);
  return __uint_as_float((uint32_t)(127 + s) << 23);
}

// 8 int8 codes as exact f16 values: byte + 128 placed under the exponent of 1024, less 1152
__device__ inline half8 codes8(u32x2 w) {
  H8 o;
  const half8 bias = {-1152, -1152, -1152, -1152, -1152, -1152, -1152, -1152};
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const uint32_t u = w[i] ^ 0x80808080u;
    o.u[2 * i] = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u);
    o.u[2 * i + 1] = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
  }
  return o.h + bias;
}

// what a unit's body needs to know of one of its rows
struct RowAt {
  int t, head, part;
  bool on;
};
__device__ inline RowAt row_at(const PagedKernelArgs& p, const PagedUnit& u, int kvh, int i) {
  RowAt r;
  r.on = i < u.n_rho;
  const int rho = u.rho0 + (r.on ? i : 0);
  const int j = rho / p.b.G;
  const PagedTok tok = p.b.toks[u.tok + j];
  r.t = tok.t;
  r.part = tok.part < 0 ? -1 : tok.part + u.chunk;
  r.head = kvh * p.b.G + rho - j * p.b.G;
  return r;
}

// a row's o at dims d .. d+3: the output (normalized, gated) or the unit's partial
template <int D>
__device__ inline void store_o(const PagedKernelArgs& p, float* ws_o, const RowAt& r, int d, f32x4 o, float l) {
  if (r.part >= 0) {
    *(f32x4*)(ws_o + ((size_t)r.part * p.b.H + r.head) * D + d) = o;
    return;
  }
  const size_t row = (size_t)r.t * p.b.H + r.head;
  const float inv = 1.0f / l;
  o *= inv;
  if (p.gate) {
    const float* g = p.gate + row * p.gate_stride + d;
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = o[e] / (1.0f + __expf(-g[e]));
  }
  *(f32x4*)(p.out + row * D + d) = o;
}

// slot of register i (0..7) of lane group g in a 32-slot tile, 16-row matrix products: the V tile's own
// order (tile_slot)
__device__ inline int slot16(int g, int i) { return 16 * (g >> 1) + 8 * (i >> 2) + 4 * (g & 1) + (i & 3); }

// ------------------------------------------------------------------------------------------ few
template <int D, int DT>
struct FewK {  // a lane's K operand of a 32-slot tile
  static constexpr int N = DT == KV_F32 ? 2 * (D / 16) : 2 * (D / 32);
  f32x4 f[DT == KV_F32 ? N : 1];
  u32x4 h[DT == KV_F16 ? N : 1];
  u32x2 c[DT == KV_Q8 ? N : 1];
  f32x4 s[DT == KV_Q8 ? 8 * (D / 128) : 1];
};
template <int D, int DT>
struct FewV {
  static constexpr int N = D / 16;
  f32x4 f[DT == KV_F32 ? 2 * N : 1];
  u32x4 h[DT == KV_F16 ? N : 1];
  u32x2 c[DT == KV_Q8 ? N : 1];
  f32x4 s[DT == KV_Q8 ? 8 * (D / 128) : 1];
};

template <int D, int DT>
__device__ __forceinline__ void few_load_k(const PagedKernelArgs& p, size_t row, int c, int g, FewK<D, DT>& k) {
  // operand row c of product i is slot slot16(c / 4, 4 i + c % 4); the k dimension of a lane group is
  // 8 g + e of every 32 dims (f32: 4 g + e of every 16)
  const int s0 = 16 * (c >> 3) + 4 * ((c >> 2) & 1) + (c & 3);
  if constexpr (DT == KV_F32) {
    const float* b = (const float*)p.k + row * D + (size_t)s0 * D + 4 * g;
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int j = 0; j < D / 16; j++) k.f[i * (D / 16) + j] = *(const f32x4*)(b + 8 * i * D + 16 * j);
  } else if constexpr (DT == KV_F16) {
    const _Float16* b = (const _Float16*)p.k + row * D + (size_t)s0 * D + 8 * g;
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int j = 0; j < D / 32; j++) k.h[i * (D / 32) + j] = *(const u32x4*)(b + 8 * i * D + 32 * j);
  } else {
    const int8_t* b = (const int8_t*)p.k + row * D + (size_t)s0 * D + 8 * g;
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int j = 0; j < D / 32; j++) k.c[i * (D / 32) + j] = *(const u32x2*)(b + 8 * i * D + 32 * j);
    // the scales of the 8 slots this lane's scores are of
    const float* sc = p.ks + (row + slot16(g, 0)) * (D / 32);
#pragma unroll
    for (int e = 0; e < 8; e++)
#pragma unroll
      for (int j = 0; j < D / 128; j++)
        k.s[e * (D / 128) + j] = *(const f32x4*)(sc + (size_t)(8 * (e >> 2) + (e & 3)) * (D / 32) + 4 * j);
  }
}

template <int D, int DT>
__device__ __forceinline__ void few_load_v(const PagedKernelArgs& p, size_t row, int c, int g, FewV<D, DT>& v) {
  if constexpr (DT == KV_F32) {
    const float* b = (const float*)p.v + row * D + (size_t)(g * D + c) * 8;
#pragma unroll
    for (int j = 0; j < D / 16; j++) {
      v.f[2 * j] = *(const f32x4*)(b + 128 * j);
      v.f[2 * j + 1] = *(const f32x4*)(b + 128 * j + 4);
    }
  } else if constexpr (DT == KV_F16) {
    const _Float16* b = (const _Float16*)p.v + row * D + (size_t)(g * D + c) * 8;
#pragma unroll
    for (int j = 0; j < D / 16; j++) v.h[j] = *(const u32x4*)(b + 128 * j);
  } else {
    const int8_t* b = (const int8_t*)p.v + row * D + (size_t)(g * D + c) * 8;
#pragma unroll
    for (int j = 0; j < D / 16; j++) v.c[j] = *(const u32x2*)(b + 128 * j);
    const float* sc = p.vs + (row + slot16(g, 0)) * (D / 32);
#pragma unroll
    for (int e = 0; e < 8; e++)
#pragma unroll
      for (int j = 0; j < D / 128; j++)
        v.s[e * (D / 128) + j] = *(const f32x4*)(sc + (size_t)(8 * (e >> 2) + (e & 3)) * (D / 32) + 4 * j);
  }
}

constexpr int kFewPad = 4;  // floats between the LDS rows of the waves' o

template <int D, int DT, int NSET>
__device__ __forceinline__ void few_unit(const PagedKernelArgs& p, const PagedUnit& u, int kvh, float* ws_o, float2* ws_ml,
                                         float (*lo)[16 * NSET][D + kFewPad], float2 (*lml)[16 * NSET]) {
  constexpr int NK = DT == KV_F32 ? D / 16 : D / 32;
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int shift = p.b.page_shift, P = 1 << shift;
  const int n_tiles = (u.key1 - u.key0 + 31) >> 5;
  const int* pages = p.b.pages + u.table;

  // ---- the queries
  int pos[NSET];
  float qs[NSET];
  H8 qh[NSET][DT == KV_F32 ? 1 : NK], ql[NSET][DT == KV_F32 ? 1 : NK];
  f32x4 qf[NSET][DT == KV_F32 ? NK : 1];
#pragma unroll
  for (int s = 0; s < NSET; s++) {
    const int i = 16 * s + c;
    const bool on = i < u.n_rho;
    const int rho = u.rho0 + (on ? i : 0);
    const int j = rho / p.b.G;
    const PagedTok tok = p.b.toks[u.tok + j];
    pos[s] = tok.pos;
    const float* q = p.q + ((size_t)tok.t * p.b.H + kvh * p.b.G + rho - j * p.b.G) * D;
    if constexpr (DT == KV_F32) {
#pragma unroll
      for (int n = 0; n < NK; n++) qf[s][n] = *(const f32x4*)(q + 16 * n + 4 * g);
      qs[s] = p.qscale;
    } else {
      float x[NK][8];
      float top = 0.0f;
#pragma unroll
      for (int n = 0; n < NK; n++) {
        const f32x4 a = *(const f32x4*)(q + 32 * n + 8 * g), b = *(const f32x4*)(q + 32 * n + 8 * g + 4);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          x[n][e] = a[e];
          x[n][4 + e] = b[e];
          top = fmaxf(top, fmaxf(fabsf(a[e]), fabsf(b[e])));
        }
      }
      float2 r = pair16(top);
      top = fmaxf(r.x, r.y);
      r = pair32(top);
      top = fmaxf(r.x, r.y);
      float undo;
      const float f = row_factor(top, &undo);
      qs[s] = p.qscale * undo;
#pragma unroll
      for (int n = 0; n < NK; n++) {
#pragma unroll
        for (int e = 0; e < 8; e++) x[n][e] *= f;
        split8(x[n], qh[s][n], ql[s][n]);
      }
    }
    if constexpr (DT == KV_Q8) qs[s] *= 1.0f / 127.0f;
  }

  f32x4 o[NSET][D / 16];
  float m[NSET], l[NSET];
#pragma unroll
  for (int s = 0; s < NSET; s++) {
    m[s] = -INFINITY;
    l[s] = 0.0f;
#pragma unroll
    for (int j = 0; j < D / 16; j++) o[s][j] = f32x4{0, 0, 0, 0};
  }
  float vscale = 0.0f;   // q8: 2^-ev, 0 before the first tile

  auto row_of = [&](int t) -> size_t {
    const int key = u.key0 + 32 * t;
    const int id = uniform(pages[key >> shift]);
    return ((size_t)id * p.kv_heads + kvh) * P + (key & (P - 1));
  };
  FewK<D, DT> k;
  FewV<D, DT> v;
  if (wave < n_tiles) {
    const size_t row = row_of(wave);
    few_load_k<D, DT>(p, row, c, g, k);
    few_load_v<D, DT>(p, row, c, g, v);
  }
  for (int t = wave; t < n_tiles; t += 4) {
    const int key = u.key0 + 32 * t;
    const int tn = min(t + 4, n_tiles - 1);   // past the end: a tile of the unit, unused
    const size_t next = row_of(tn);
    // ---- scores: s[set][e] of slot slot16(g, e), row c
    float sc[NSET][8];
    if constexpr (DT == KV_F32) {
#pragma unroll
      for (int s = 0; s < NSET; s++) {
        f32x4 a[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int n = 0; n < NK; n++)
#pragma unroll
          for (int e = 0; e < 4; e++)
#pragma unroll
            for (int i = 0; i < 2; i++)
              a[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(k.f[i * NK + n][e], qf[s][n][e], a[i], 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 8; e++) sc[s][e] = a[e >> 2][e & 3];
      }
    } else if constexpr (DT == KV_F16) {
      f32x4 a[NSET][2];
#pragma unroll
      for (int s = 0; s < NSET; s++) a[s][0] = a[s][1] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int n = 0; n < NK; n++) {
        H8 k0, k1;
        k0.u = k.h[n];
        k1.u = k.h[NK + n];
#pragma unroll
        for (int s = 0; s < NSET; s++) {
          a[s][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0.h, qh[s][n].h, a[s][0], 0, 0, 0);
          a[s][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1.h, qh[s][n].h, a[s][1], 0, 0, 0);
          a[s][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0.h, ql[s][n].h, a[s][0], 0, 0, 0);
          a[s][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1.h, ql[s][n].h, a[s][1], 0, 0, 0);
        }
      }
#pragma unroll
      for (int s = 0; s < NSET; s++)
#pragma unroll
        for (int e = 0; e < 8; e++) sc[s][e] = a[s][e >> 2][e & 3];
    } else {
      // a product's 32 dims are one scale block: its exact code sums, then the block scale in f32
#pragma unroll
      for (int s = 0; s < NSET; s++)
#pragma unroll
        for (int e = 0; e < 8; e++) sc[s][e] = 0.0f;
#pragma unroll
      for (int n = 0; n < NK; n++) {
        const half8 k0 = codes8(k.c[n]), k1 = codes8(k.c[NK + n]);
#pragma unroll
        for (int s = 0; s < NSET; s++) {
          f32x4 a0 = {0, 0, 0, 0}, a1 = {0, 0, 0, 0};
          a0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qh[s][n].h, a0, 0, 0, 0);
          a1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qh[s][n].h, a1, 0, 0, 0);
          a0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, ql[s][n].h, a0, 0, 0, 0);
          a1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, ql[s][n].h, a1, 0, 0, 0);
#pragma unroll
          for (int e = 0; e < 8; e++)
            sc[s][e] = fmaf(e < 4 ? a0[e & 3] : a1[e & 3], k.s[e * (D / 128) + n / 4][n & 3], sc[s][e]);
        }
      }
    }
    few_load_k<D, DT>(p, next, c, g, k);
    const bool masked = key + 32 > u.mask0;
    if (masked) {
#pragma unroll
      for (int s = 0; s < NSET; s++)
#pragma unroll
        for (int e = 0; e < 8; e++) sc[s][e] = key + slot16(g, e) <= pos[s] ? sc[s][e] : -INFINITY;
    }
    const bool stale = key + 32 > u.key1;  // slots past the written positions
    if (stale) {
      if constexpr (DT == KV_F32) {
#pragma unroll
        for (int j = 0; j < D / 16; j++)
#pragma unroll
          for (int e = 0; e < 8; e++)
            v.f[2 * j + (e >> 2)][e & 3] = key + slot16(g, e) < u.key1 ? v.f[2 * j + (e >> 2)][e & 3] : 0.0f;
      } else if constexpr (DT == KV_F16) {
        u32x4 keep;
#pragma unroll
        for (int w = 0; w < 4; w++)
          keep[w] = (key + slot16(g, 2 * w) < u.key1 ? 0xffffu : 0u) | (key + slot16(g, 2 * w + 1) < u.key1 ? 0xffff0000u : 0u);
#pragma unroll
        for (int j = 0; j < D / 16; j++) v.h[j] &= keep;
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
#pragma unroll
          for (int j = 0; j < D / 128; j++)
            if (key + slot16(g, e) >= u.key1) v.s[e * (D / 128) + j] = f32x4{0, 0, 0, 0};
      }
    }
    // ---- running maximum and sum
    float pr[NSET][8];
#pragma unroll
    for (int s = 0; s < NSET; s++) {
      float top = sc[s][0];
#pragma unroll
      for (int e = 1; e < 8; e++) top = fmaxf(top, sc[s][e]);
      float2 r = pair16(top);
      top = fmaxf(r.x, r.y);
      r = pair32(top);
      top = fmaxf(r.x, r.y) * qs[s];
      if (__any(top > m[s] + kLazy)) {
        const float mn = fmaxf(m[s], top);
        const float f = mn == -INFINITY ? 1.0f : exp2_hw(m[s] - mn);
        m[s] = mn;
        l[s] *= f;
#pragma unroll
        for (int j = 0; j < D / 16; j++) o[s][j] *= f;
      }
      const float base = m[s] == -INFINITY ? 0.0f : kPShift - m[s];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        pr[s][e] = exp2_hw(fmaf(sc[s][e], qs[s], base));
        l[s] += pr[s][e];
      }
    }
    // ---- o
    if constexpr (DT == KV_F32) {
#pragma unroll
      for (int s = 0; s < NSET; s++)
#pragma unroll
        for (int e = 0; e < 8; e++)
#pragma unroll
          for (int j = 0; j < D / 16; j++)
            o[s][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v.f[2 * j + (e >> 2)][e & 3], pr[s][e], o[s][j], 0, 0, 0);
    } else if constexpr (DT == KV_F16) {
      H8 ph[NSET], pl[NSET];
#pragma unroll
      for (int s = 0; s < NSET; s++) split8(pr[s], ph[s], pl[s]);
#pragma unroll
      for (int s = 0; s < NSET; s++) {
#pragma unroll
        for (int j = 0; j < D / 16; j++) {
          H8 a;
          a.u = v.h[j];
          o[s][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h, ph[s].h, o[s][j], 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < D / 16; j++) {
          H8 a;
          a.u = v.h[j];
          o[s][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h, pl[s].h, o[s][j], 0, 0, 0);
        }
      }
    } else {
      // 2^ev at least every scale of the tile (and of those before): p * scale / 2^ev <= p
      float top = 0.0f;
#pragma unroll
      for (int e = 0; e < 8 * (D / 128); e++)
#pragma unroll
        for (int w = 0; w < 4; w++) top = fmaxf(top, v.s[e][w]);
      float2 r = pair16(top);
      top = fmaxf(r.x, r.y);
      r = pair32(top);
      top = fmaxf(r.x, r.y);
      if (vscale == 0.0f || top * vscale > 1.0f) {  // the same in every lane
        const int ex = min(max((int)((__float_as_uint(top) >> 23) & 0xff) + 1, 28), 226);
        const float vn = __uint_as_float((uint32_t)(254 - ex) << 23);
        const float f = vscale == 0.0f ? 1.0f : vn / vscale;
        vscale = vn;
#pragma unroll
        for (int s = 0; s < NSET; s++)
#pragma unroll
          for (int j = 0; j < D / 16; j++) o[s][j] *= f;
      }
#pragma unroll
      for (int n = 0; n < D / 32; n++) {
        const half8 a0 = codes8(v.c[2 * n]), a1 = codes8(v.c[2 * n + 1]);
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; e++) w[e] = v.s[e * (D / 128) + n / 4][n & 3] * vscale;
#pragma unroll
        for (int s = 0; s < NSET; s++) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; e++) x[e] = pr[s][e] * w[e];
          H8 ph, pl;
          split8(x, ph, pl);
          o[s][2 * n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, ph.h, o[s][2 * n], 0, 0, 0);
          o[s][2 * n + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, ph.h, o[s][2 * n + 1], 0, 0, 0);
          o[s][2 * n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, pl.h, o[s][2 * n], 0, 0, 0);
          o[s][2 * n + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, pl.h, o[s][2 * n + 1], 0, 0, 0);
        }
      }
    }
    few_load_v<D, DT>(p, next, c, g, v);
  }

  // ---- the four waves' results meet in LDS
  const float oscale = DT == KV_Q8 ? (vscale == 0.0f ? 0.0f : 1.0f / (127.0f * vscale)) : 1.0f;
#pragma unroll
  for (int s = 0; s < NSET; s++) {
    float2 r = pair16(l[s]);
    l[s] = r.x + r.y;
    r = pair32(l[s]);
    l[s] = r.x + r.y;
    if (g == 0) lml[wave][16 * s + c] = make_float2(m[s], l[s]);
#pragma unroll
    for (int j = 0; j < D / 16; j++) *(f32x4*)(&lo[wave][16 * s + c][16 * j + 4 * g]) = o[s][j] * oscale;
  }
  __syncthreads();
  for (int x = threadIdx.x; x < u.n_rho * (D / 4); x += 256) {
    const int i = x / (D / 4), d = 4 * (x % (D / 4));
    float mw[4], lw[4], top = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const float2 ml = lml[w][i];
      mw[w] = ml.x;
      lw[w] = ml.y;
      top = fmaxf(top, ml.x);
    }
    f32x4 sum = {0, 0, 0, 0};
    float lsum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const float f = mw[w] == -INFINITY ? 0.0f : exp2_hw(mw[w] - top);
      lsum += lw[w] * f;
      sum += *(const f32x4*)(&lo[w][i][d]) * f;
    }
    const RowAt r = row_at(p, u, kvh, i);
    store_o<D>(p, ws_o, r, d, sum, lsum);
    if (d == 0 && r.part >= 0) ws_ml[(size_t)r.part * p.b.H + r.head] = make_float2(top, lsum);
  }
}

// ------------------------------------------------------------------------------------------ many
template <int D, int DT>
struct Many {
  static constexpr int EB = DT == KV_F32 ? 4 : 2;               // bytes of a staged value (q8 codes as f16)
  static constexpr int KT = DT == KV_F32 || D == 256 ? 32 : 64; // positions a step
  static constexpr int NSUB = KT / 32;
  static constexpr int SUB = 32 * D * EB;                       // bytes of a staged 32-position tile of K (or V)
  static constexpr int CPR = D * EB / 16;                       // 16-byte chunks of a K row
  static constexpr int SCALES = DT == KV_Q8 ? KT * (D / 32) * 4 : 0;  // bytes of a step's K (or V) scales
};

// where a staged K row keeps its chunk x: rows of one bank phase spread over all banks
__device__ inline int swz(int r, int x) { return x ^ (r & 15); }

template <int D, int DT>
__device__ __forceinline__ void many_stage(const PagedKernelArgs& p, size_t row, char* kd, char* vd) {
  // f16 / f32: 16-byte chunks copied straight into LDS, no registers. A wave instruction fills 64
  // consecutive chunks; the lane reads the chunk that belongs there.
  using M = Many<D, DT>;
  constexpr int CH = M::SUB / 16;
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void*)(p.k + row * D * M::EB), (short)0, M::SUB, 0x00020000);
  const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void*)(p.v + row * D * M::EB), (short)0, M::SUB, 0x00020000);
#pragma unroll
  for (int i = 0; i < CH / 256; i++) {
    const int at = (4 * i + wave) * 64;
    const int x = at + lane, r = x / M::CPR, cc = swz(r, x % M::CPR);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_ptr)(kd + at * 16), 16, (r * M::CPR + cc) * 16, 0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_ptr)(vd + at * 16), 16, x * 16, 0, 0, 0);
  }
}

// q8: a thread's share of a staged 32-position tile, through registers
template <int D>
struct ManyQ8 {
  static constexpr int N = 32 * D / 16 / 256 > 0 ? 32 * D / 16 / 256 : 1;
  u32x4 k[N], v[N];
  float ks, vs;
};
template <int D>
__device__ __forceinline__ void many_load_q8(const PagedKernelArgs& p, size_t row, ManyQ8<D>& r) {
  const int t = threadIdx.x;
#pragma unroll
  for (int i = 0; i < ManyQ8<D>::N; i++) {
    r.k[i] = *(const u32x4*)(p.k + row * D + (size_t)(t + 256 * i) * 16);
    r.v[i] = *(const u32x4*)(p.v + row * D + (size_t)(t + 256 * i) * 16);
  }
  const int n = t & (D - 1);  // 32 positions x D / 32 scales
  r.ks = p.ks[row * (D / 32) + n];
  r.vs = p.vs[row * (D / 32) + n];
}
// scales are staged [block][position], so that a lane reads the four positions of a register group at once
template <int D>
__device__ __forceinline__ void many_store_q8(const ManyQ8<D>& r, char* kd, char* vd, float* ksd, float* vsd, int KT) {
  const int t = threadIdx.x;
#pragma unroll
  for (int i = 0; i < ManyQ8<D>::N; i++) {
    const int x = t + 256 * i;              // 16 codes: half a K row's 32 ..., two dims' 8 slots of V
    const int row = x / (D / 16), c0 = 2 * (x % (D / 16));
    H8 a, b;
    a.h = codes8(u32x2{r.k[i][0], r.k[i][1]});
    b.h = codes8(u32x2{r.k[i][2], r.k[i][3]});
    *(u32x4*)(kd + (row * (D / 8) + swz(row, c0)) * 16) = a.u;
    *(u32x4*)(kd + (row * (D / 8) + swz(row, c0 + 1)) * 16) = b.u;
    a.h = codes8(u32x2{r.v[i][0], r.v[i][1]});
    b.h = codes8(u32x2{r.v[i][2], r.v[i][3]});
    *(u32x4*)(vd + (size_t)x * 32) = a.u;
    *(u32x4*)(vd + (size_t)x * 32 + 16) = b.u;
  }
  if (t < D) {
    const int s = t / (D / 32), blk = t % (D / 32);
    ksd[blk * KT + s] = r.ks;
    vsd[blk * KT + s] = r.vs;
  }
}

template <int D, int DT>
__device__ __forceinline__ void many_unit(const PagedKernelArgs& p, const PagedUnit& u, int kvh, float* ws_o, float2* ws_ml,
                                          char* k0, char* k1, char* v0, char* v1, float* scales) {
  using M = Many<D, DT>;
  constexpr int KT = M::KT, NSUB = M::NSUB;
  constexpr int NK = DT == KV_F32 ? D / 8 : D / 16;   // f32: 16-byte chunks a lane; else 16-dim products
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int shift = p.b.page_shift, P = 1 << shift;
  const int n_tiles = (u.key1 - u.key0 + 31) >> 5, n_steps = (n_tiles + NSUB - 1) / NSUB;
  const int* pages = p.b.pages + u.table;
  const bool active = 32 * wave < u.n_rho;

  const RowAt ra = row_at(p, u, kvh, 32 * wave + c);
  int pos;
  float qs;
  H8 qh[DT == KV_F32 ? 1 : NK], ql[DT == KV_F32 ? 1 : NK];
  f32x4 qf[DT == KV_F32 ? NK : 1];
  {
    const int rho = u.rho0 + (ra.on ? 32 * wave + c : 0);
    pos = p.b.toks[u.tok + rho / p.b.G].pos;
    const float* q = p.q + ((size_t)ra.t * p.b.H + ra.head) * D;
    if constexpr (DT == KV_F32) {
#pragma unroll
      for (int n = 0; n < NK; n++) qf[n] = *(const f32x4*)(q + 8 * n + 4 * h);
      qs = p.qscale;
    } else {
      float top = 0.0f;
#pragma unroll
      for (int n = 0; n < NK; n++) {
        const f32x4 a = *(const f32x4*)(q + 16 * n + 8 * h), b = *(const f32x4*)(q + 16 * n + 8 * h + 4);
#pragma unroll
        for (int e = 0; e < 4; e++) top = fmaxf(top, fmaxf(fabsf(a[e]), fabsf(b[e])));
      }
      const float2 r = pair32(top);
      top = fmaxf(r.x, r.y);
      float undo;
      const float f = row_factor(top, &undo);
      qs = p.qscale * undo * (DT == KV_Q8 ? 1.0f / 127.0f : 1.0f);
#pragma unroll
      for (int n = 0; n < NK; n++) {  // read again: half the registers of holding the row in f32
        const f32x4 a = *(const f32x4*)(q + 16 * n + 8 * h), b = *(const f32x4*)(q + 16 * n + 8 * h + 4);
        float x[8];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          x[e] = a[e] * f;
          x[4 + e] = b[e] * f;
        }
        split8(x, qh[n], ql[n]);
      }
    }
  }
  f32x16 o[D / 32];
#pragma unroll
  for (int j = 0; j < D / 32; j++)
#pragma unroll
    for (int e = 0; e < 16; e++) o[j][e] = 0.0f;
  float m = -INFINITY, l = 0.0f, vscale = 0.0f;

  auto row_of = [&](int t) -> size_t {
    const int key = u.key0 + 32 * min(t, n_tiles - 1);  // past the end: staged again, masked
    const int id = uniform(pages[key >> shift]);
    return ((size_t)id * p.kv_heads + kvh) * P + (key & (P - 1));
  };

  // one step over staged tiles; key: its first position
  auto step = [&](const char* kb, const char* vb, const float* ksb, const float* vsb, int key) __attribute__((always_inline)) {
    float s[NSUB][16];
#pragma unroll
    for (int sub = 0; sub < NSUB; sub++) {
      const char* kt = kb + sub * M::SUB + c * M::CPR * 16;
      if constexpr (DT == KV_F32) {
        f32x16 a;
#pragma unroll
        for (int e = 0; e < 16; e++) a[e] = 0.0f;
#pragma unroll
        for (int n = 0; n < NK; n++) {
          const f32x4 x = *(const f32x4*)(kt + swz(c, 2 * n + h) * 16);
#pragma unroll
          for (int e = 0; e < 4; e++) a = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], qf[n][e], a, 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 16; e++) s[sub][e] = a[e];
      } else if constexpr (DT == KV_F16) {
        f32x16 a, b;
#pragma unroll
        for (int e = 0; e < 16; e++) a[e] = b[e] = 0.0f;
#pragma unroll
        for (int n = 0; n < NK; n++) {
          H8 x;
          x.u = *(const u32x4*)(kt + swz(c, 2 * n + h) * 16);
          a = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.h, qh[n].h, a, 0, 0, 0);
          b = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.h, ql[n].h, b, 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 16; e++) s[sub][e] = a[e] + b[e];
      } else {
#pragma unroll
        for (int e = 0; e < 16; e++) s[sub][e] = 0.0f;
#pragma unroll
        for (int blk = 0; blk < D / 32; blk++) {
          f32x16 a;
#pragma unroll
          for (int e = 0; e < 16; e++) a[e] = 0.0f;
#pragma unroll
          for (int n = 2 * blk; n < 2 * blk + 2; n++) {
            H8 x;
            x.u = *(const u32x4*)(kt + swz(c, 2 * n + h) * 16);
            a = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.h, qh[n].h, a, 0, 0, 0);
            a = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.h, ql[n].h, a, 0, 0, 0);
          }
#pragma unroll
          for (int w = 0; w < 4; w++) {
            const f32x4 z = *(const f32x4*)(ksb + blk * KT + 32 * sub + 8 * w + 4 * h);
#pragma unroll
            for (int e = 0; e < 4; e++) s[sub][4 * w + e] = fmaf(a[4 * w + e], z[e], s[sub][4 * w + e]);
          }
        }
      }
    }
    if (key + KT > u.mask0) {
#pragma unroll
      for (int sub = 0; sub < NSUB; sub++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const int at = key + 32 * sub + 8 * (e >> 2) + 4 * h + (e & 3);
          s[sub][e] = at <= pos && at < u.key1 ? s[sub][e] : -INFINITY;
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int sub = 0; sub < NSUB; sub++)
#pragma unroll
      for (int e = 0; e < 16; e++) top = fmaxf(top, s[sub][e]);
    const float2 r = pair32(top);
    top = fmaxf(r.x, r.y) * qs;
    if (__any(top > m + kLazy)) {
      const float mn = fmaxf(m, top);
      const float f = mn == -INFINITY ? 1.0f : exp2_hw(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int j = 0; j < D / 32; j++) o[j] *= f;
    }
    const float base = m == -INFINITY ? 0.0f : kPShift - m;
#pragma unroll
    for (int sub = 0; sub < NSUB; sub++)
#pragma unroll
      for (int e = 0; e < 16; e++) {
        s[sub][e] = exp2_hw(fmaf(s[sub][e], qs, base));
        l += s[sub][e];
      }
    if constexpr (DT == KV_Q8) {
      // 2^ev at least every scale of the step
      float big = 0.0f;
#pragma unroll
      for (int i = 0; i < KT * (D / 32) / 64; i++) big = fmaxf(big, vsb[lane + 64 * i]);
      big = wave_max(big);
      if (vscale == 0.0f || big * vscale > 1.0f) {
        const int ex = min(max((int)((__float_as_uint(big) >> 23) & 0xff) + 1, 28), 226);
        const float vn = __uint_as_float((uint32_t)(254 - ex) << 23);
        const float f = vscale == 0.0f ? 1.0f : vn / vscale;
        vscale = vn;
#pragma unroll
        for (int j = 0; j < D / 32; j++) o[j] *= f;
      }
    }
#pragma unroll
    for (int sub = 0; sub < NSUB; sub++) {
      const char* vt = vb + sub * M::SUB;
      if constexpr (DT == KV_F32) {
#pragma unroll
        for (int x = 0; x < 4; x++) {  // half a panel pair: registers 4 x .. 4 x + 3
#pragma unroll
          for (int j = 0; j < D / 32; j++) {
            const f32x4 a = *(const f32x4*)(vt + (((2 * (x >> 1) + h) * D + 32 * j + c) * 8 + 4 * (x & 1)) * 4);
#pragma unroll
            for (int e = 0; e < 4; e++) o[j] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], s[sub][4 * x + e], o[j], 0, 0, 0);
          }
        }
      } else if constexpr (DT == KV_F16) {
#pragma unroll
        for (int x = 0; x < 2; x++) {
          float w[8];
#pragma unroll
          for (int e = 0; e < 8; e++) w[e] = s[sub][8 * x + e];
          H8 ph, pl;
          split8(w, ph, pl);
#pragma unroll
          for (int j = 0; j < D / 32; j++) {
            H8 a;
            a.u = *(const u32x4*)(vt + ((2 * x + h) * D + 32 * j + c) * 16);
            o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, ph.h, o[j], 0, 0, 0);
            o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, pl.h, o[j], 0, 0, 0);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < D / 32; j++) {
#pragma unroll
          for (int x = 0; x < 2; x++) {
            float w[8];
#pragma unroll
            for (int y = 0; y < 2; y++) {
              const f32x4 z = *(const f32x4*)(vsb + j * KT + 32 * sub + 16 * x + 8 * y + 4 * h);
#pragma unroll
              for (int e = 0; e < 4; e++) w[4 * y + e] = s[sub][8 * x + 4 * y + e] * (z[e] * vscale);
            }
            H8 ph, pl, a;
            split8(w, ph, pl);
            a.u = *(const u32x4*)(vt + ((2 * x + h) * D + 32 * j + c) * 16);
            o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, ph.h, o[j], 0, 0, 0);
            o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, pl.h, o[j], 0, 0, 0);
          }
        }
      }
    }
  };
  // V (or its q8 scales) past the written positions becomes zero
  auto clear_stale = [&](char* vb, float* vsb, int key) __attribute__((always_inline)) {
    for (int x = threadIdx.x; x < KT * (DT == KV_Q8 ? D / 32 : D); x += 256) {
      if constexpr (DT == KV_Q8) {
        if (key + x % KT >= u.key1) vsb[x] = 0.0f;
      } else {
        const int sub = x / (32 * D), y = x % (32 * D), panel = y / (8 * D), e = y % 8;
        if (key + 32 * sub + tile_slot(panel, e) >= u.key1) {
          if constexpr (DT == KV_F32) ((float*)vb)[x] = 0.0f;
          else ((uint16_t*)vb)[x] = 0;
        }
      }
    }
    __syncthreads();
  };

  // k0, k1: K of even and odd steps; v0, v1: V. scales: [step parity][K, V][block][KT]
  ManyQ8<D> r8[DT == KV_Q8 ? NSUB : 1];
  auto begin = [&](int st, char* kd, char* vd) __attribute__((always_inline)) {
#pragma unroll
    for (int sub = 0; sub < NSUB; sub++) {
      const size_t row = row_of(NSUB * st + sub);
      if constexpr (DT == KV_Q8) many_load_q8<D>(p, row, r8[sub]);
      else many_stage<D, DT>(p, row, kd + sub * M::SUB, vd + sub * M::SUB);
    }
  };
  auto finish = [&](char* kd, char* vd, float* sc) __attribute__((always_inline)) {
    if constexpr (DT == KV_Q8) {
#pragma unroll
      for (int sub = 0; sub < NSUB; sub++)
        many_store_q8<D>(r8[sub], kd + sub * M::SUB, vd + sub * M::SUB, sc + 32 * sub, sc + KT * (D / 32) + 32 * sub, KT);
    }
  };
  constexpr int SC = DT == KV_Q8 ? 2 * KT * (D / 32) : 0;
  auto one = [&](int st, char* kb, char* vb, float* sb, char* kn, char* vn, float* sn) __attribute__((always_inline)) {
    // the step's tiles have landed; the other buffers' readers are done
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const bool more = st + 1 < n_steps;
    if (more) begin(st + 1, kn, vn);
    const int key = u.key0 + KT * st;
    if (key + KT > u.key1) clear_stale(vb, sb + SC / 2, key);
    if (active) step(kb, vb, sb, sb + SC / 2, key);
    if (more) finish(kn, vn, sn);
  };
  if (n_steps > 0) {
    begin(0, k0, v0);
    finish(k0, v0, scales);
  }
  for (int st = 0; st < n_steps; st += 2) {
    one(st, k0, v0, scales, k1, v1, scales + SC);
    if (st + 1 < n_steps) one(st + 1, k1, v1, scales + SC, k0, v0, scales);
  }
  const float2 r = pair32(l);
  l = r.x + r.y;
  const float oscale = DT == KV_Q8 ? (vscale == 0.0f ? 0.0f : 1.0f / (127.0f * vscale)) : 1.0f;
  if (ra.on) {
#pragma unroll
    for (int j = 0; j < D / 32; j++)
#pragma unroll
      for (int w = 0; w < 4; w++)
        store_o<D>(p, ws_o, ra, 32 * j + 8 * w + 4 * h,
                   f32x4{o[j][4 * w], o[j][4 * w + 1], o[j][4 * w + 2], o[j][4 * w + 3]} * oscale, l);
    if (h == 0 && ra.part >= 0) ws_ml[(size_t)ra.part * p.b.H + ra.head] = make_float2(m, l);
  }
}

// Kernels: the 128-row units and the few-row units are launches of their own, each with its own registers.
template <int D, int DT>
__global__ __launch_bounds__(256, D == 128 ? 2 : 1) void paged_many_kernel(PagedKernelArgs p) {
  using M = Many<D, DT>;
  // four distinct arrays: a copy into one buffer then cannot alias the reads of another, and the
  // compiler adds no waits between them
  __shared__ __align__(16) char k0[M::SUB * M::NSUB];
  __shared__ __align__(16) char k1[M::SUB * M::NSUB];
  __shared__ __align__(16) char v0[M::SUB * M::NSUB];
  __shared__ __align__(16) char v1[M::SUB * M::NSUB];
  __shared__ __align__(16) float scales[DT == KV_Q8 ? 4 * M::KT * (D / 32) : 4];
  const int total = p.n_blocks ? p.n_blocks : p.b.hdr->n_many * p.kv_heads;
  float* ws_o = p.b.hdr->ws_o;
  float2* ws_ml = p.b.hdr->ws_ml;
  for (int b = blockIdx.x; b < total; b += gridDim.x) {
    const PagedUnit u = p.b.units[b / p.kv_heads];
    many_unit<D, DT>(p, u, b % p.kv_heads, ws_o, ws_ml, k0, k1, v0, v1, scales);
    __syncthreads();  // the unit's LDS is read before the next one's is written
  }
}

template <int D, int DT, int NSET>
__global__ __launch_bounds__(256, D == 128 ? 2 : 1) void paged_few_kernel(PagedKernelArgs p) {
  __shared__ __align__(16) float lo[4][16 * NSET][D + kFewPad];
  __shared__ float2 lml[4][16 * NSET];
  const PagedHeader* h = p.b.hdr;
  const int first = p.n_blocks ? p.first : NSET == 1 ? h->n_units - h->n_few1 : h->n_many;
  const int total = p.n_blocks ? p.n_blocks : (NSET == 1 ? h->n_few1 : h->n_units - h->n_few1 - h->n_many) * p.kv_heads;
  float* ws_o = h->ws_o;
  float2* ws_ml = h->ws_ml;
  for (int b = blockIdx.x; b < total; b += gridDim.x) {
    const PagedUnit u = p.b.units[first + b / p.kv_heads];
    few_unit<D, DT, NSET>(p, u, b % p.kv_heads, ws_o, ws_ml, lo, lml);
    __syncthreads();  // the unit's LDS is read before the next one's is written
  }
}

// lane groups that share a row's partials
__host__ __device__ inline int merge_groups(int most_parts) { return most_parts <= 8 ? 1 : 4; }

// A row's partials joined. D / 4 lanes hold a partial's row (16 bytes a lane); PP lane groups a row take
// every PP-th partial, eight at a time, all loaded before any is used (a row of 55 partials: two rounds of
// memory latency instead of 55), and meet in LDS. PP is 1 where no row has more than eight, else 4: the
// same for a replay as for a call, so both give the same bits.
template <int D>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedKernelArgs p, int n_merges, int most_parts) {
  constexpr int LPR = D / 4, N = 8, MAXP = 4;
  __shared__ f32x4 lo[256 / (LPR * MAXP)][MAXP][LPR];
  __shared__ float2 lml[256 / (LPR * MAXP)][MAXP];
  const int PP = merge_groups(n_merges ? most_parts : p.b.hdr->most_parts), RPW = 256 / (LPR * PP);
  const int c = threadIdx.x % LPR, g = threadIdx.x / LPR % PP, rw = threadIdx.x / (LPR * PP);
  const int H = p.b.H;
  const long total = (long)(n_merges ? n_merges : p.b.hdr->n_merges) * H;
  const float* ws_o = p.b.hdr->ws_o;
  const float2* ws_ml = p.b.hdr->ws_ml;
  for (long first = (long)blockIdx.x * RPW; first < total; first += (long)gridDim.x * RPW) {
    const long x = min(first + rw, total - 1);  // past the end: the last row again, not stored
    const PagedMerge mg = p.b.merges[x / H];
    const int head = (int)(x % H);
    float m = -INFINITY, l = 0.0f;
    f32x4 acc = {0, 0, 0, 0};
    for (int i0 = g; i0 < mg.n; i0 += N * PP) {
      f32x4 o[N];
      float2 ml[N];
      float top = m;
#pragma unroll
      for (int u = 0; u < N; u++) {
        const size_t row = (size_t)(mg.part + min(i0 + u * PP, mg.n - 1)) * H + head;
        ml[u] = ws_ml[row];
        o[u] = *(const f32x4*)(ws_o + row * D + 4 * c);
      }
#pragma unroll
      for (int u = 0; u < N; u++) {
        if (i0 + u * PP >= mg.n) ml[u] = make_float2(-INFINITY, 0.0f);
        top = fmaxf(top, ml[u].x);
      }
      const float f0 = m == -INFINITY ? 0.0f : exp2_hw(m - top);
      l *= f0;
      acc *= f0;
#pragma unroll
      for (int u = 0; u < N; u++) {
        const float f = ml[u].x == -INFINITY ? 0.0f : exp2_hw(ml[u].x - top);
        l += ml[u].y * f;
        if (ml[u].x != -INFINITY) acc += o[u] * f;  // an empty part's o is zero, a padding one's any row's
      }
      m = top;
    }
    if (PP > 1) {
      lo[rw][g][c] = acc;
      if (c == 0) lml[rw][g] = make_float2(m, l);
      __syncthreads();
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < MAXP; i++) top = fmaxf(top, lml[rw][i].x);
      l = 0.0f;
      acc = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < MAXP; i++) {
        const float2 ml = lml[rw][i];
        const float f = ml.x == -INFINITY ? 0.0f : exp2_hw(ml.x - top);
        l += ml.y * f;
        acc += lo[rw][i][c] * f;
      }
      __syncthreads();
    }
    if (g == 0 && first + rw < total) {
      RowAt r;
      r.t = mg.t;
      r.head = head;
      r.part = -1;
      store_o<D>(p, nullptr, r, 4 * c, acc, l);
    }
  }
}

template <int D, int DT>
static hipError_t launch_attn(const PagedKernelArgs& k, const PagedAttnArgs& a, hipStream_t st) {
  const PagedBatchView& b = k.b;
  if (!b.captured && b.n_units == 0) return hipSuccess;
  // Under capture a grid that fills the GPU walks the units of whatever batch is set at replay, of every
  // kind. Units lie by kind: 128 rows, two sets, one set.
  PagedKernelArgs x = k;
  const unsigned full = (unsigned)(a.num_cus * (D == 128 ? 2 : 1));
  if (b.captured || b.n_many) {
    x.n_blocks = b.n_many * k.kv_heads;
    hipLaunchKernelGGL((paged_many_kernel<D, DT>), dim3(b.captured ? full : (unsigned)x.n_blocks), dim3(256), 0, st, x);
  }
  if constexpr (DT != KV_F32) {
    const int n2 = b.n_units - b.n_many - b.n_few1;
    if (b.captured || n2) {
      x.first = b.n_many;
      x.n_blocks = n2 * k.kv_heads;
      hipLaunchKernelGGL((paged_few_kernel<D, DT, 2>), dim3(b.captured ? full : (unsigned)x.n_blocks), dim3(256), 0, st, x);
    }
  }
  if (b.captured || b.n_few1) {
    x.first = b.n_units - b.n_few1;
    x.n_blocks = b.n_few1 * k.kv_heads;
    hipLaunchKernelGGL((paged_few_kernel<D, DT, 1>), dim3(b.captured ? full : (unsigned)x.n_blocks), dim3(256), 0, st, x);
  }
  if (b.captured || b.n_merges) {
    const int rpw = 256 / (D / 4 * merge_groups(b.most_parts));
    const unsigned grid = b.captured ? (unsigned)(a.num_cus * 4) : (unsigned)(((long)b.n_merges * b.H + rpw - 1) / rpw);
    hipLaunchKernelGGL((paged_merge_kernel<D>), dim3(grid), dim3(256), 0, st, k, b.captured ? 0 : b.n_merges, b.most_parts);
  }
  return hipGetLastError();
}

template <int D>
static hipError_t launch_attn_d(const LayerView& pool, const PagedKernelArgs& k, const PagedAttnArgs& a, hipStream_t st) {
  switch (pool.dtype) {
    case KV_F32: return launch_attn<D, KV_F32>(k, a, st);
    case KV_F16: return launch_attn<D, KV_F16>(k, a, st);
    default: return launch_attn<D, KV_Q8>(k, a, st);
  }
}

hipError_t launch_paged_attention(const LayerView& pool, const PagedBatchView& b, const PagedAttnArgs& a, hipStream_t st) {
  PagedKernelArgs k;
  k.k = (const char*)pool.k;
  k.v = (const char*)pool.v;
  k.ks = pool.ks;
  k.vs = pool.vs;
  k.kv_heads = pool.kv_heads;
  k.b = b;
  k.q = a.q;
  k.qscale = a.scale * kLog2e;
  k.gate = a.gate;
  k.gate_stride = a.gate_stride;
  k.out = a.out;
  k.first = k.n_blocks = 0;
  return pool.D == 128 ? launch_attn_d<128>(pool, k, a, st) : launch_attn_d<256>(pool, k, a, st);
}

}  // namespace bg
