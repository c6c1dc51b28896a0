// Attention of a batch over a paged KV cache on gfx950: any mix of single tokens, verifies and prompts,
// pages that sequences share scanned once for the rows of all of them.
//
// The plan (bg_paged_plan.h) hands every workgroup a unit: a tile of rows (row = (token, head of one kv
// head's group), so a loaded key serves G heads of every member token) times a chunk of positions, for one
// kv head. Kv heads are the fastest index of the grid: with eight of them each XCD's L2 sees one head's
// pages. Three kinds of units, each a kernel with its own registers and LDS (one kernel of all bodies
// spilled: 64 ragged q8 sequences 278 us against 191):
//   few     16 rows, a token's or two's. Bound by the pages' bytes: four waves take every fourth 32-position
//           tile straight from the pages into matrix operand registers, the next tile's K in flight under
//           the softmax and its V under the next scores. Three workgroups a CU (queries and q8 scales in
//           LDS) keep enough of them in flight: 64 sequences of up to 8,192 q8 positions, 712 MB in
//           136-142 us, 5.0-5.2 TB/s (two a CU 180 us; a device copy 5.1).
//   mid     32 rows: verifies, short prompts, a prefix that a batch shares. As few, on the 32-row matrix
//           products; one unit's four waves split the positions, so a chunk of them costs a quarter of the
//           partials that four waves of different rows would need for the same parallelism. 128 rows behind
//           16,384 shared f16 positions and their own tails, 144 MB: 48 us; bound by its waves' chains
//           (two a SIMD; matrix cores a quarter, loads alone 31 us, products alone 27) and a start and an
//           end of 9 us (descriptor, queries, first tile, exchange). Tried and slower: double-buffered K,
//           64 rows over the same registers (50 us), three workgroups a CU for f16 (spills, 67).
//   many    128 rows, 32 a wave: prompts, and prefixes with enough work for them. Positions staged through
//           LDS once for all four waves, double-buffered by asynchronous copies. Bound by the matrix
//           cores: two prompts of 777 and their 2,048 shared positions, 113 GFLOP in two parts a product,
//           120 us, 0.94 PFLOP/s (a plain f16 product of 8,192 cubed: 1.1).
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
//   q8 V    p is multiplied by the block scale of its position in units of 2^e, e the block's own, 2^e above
//           every scale of that block so far (o counts in the same units, rescaled when e is raised): the
//           products stay as small, and a block keeps its bits whatever the other blocks hold.
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

// x less the low (high) half of h: one mixed-precision fma, exact
__device__ inline float less_lo(float x, uint32_t h) {
  float r;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
  return r;
}
__device__ inline float less_hi(float x, uint32_t h) {
  float r;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
  return r;
}

// x[0..7] as hi and lo f16 parts (each conversion truncates; lo holds what hi lost)
__device__ inline void split8(const float (&x)[8], H8& hi, H8& lo) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    hi.p[i] = __builtin_amdgcn_cvt_pkrtz(x[2 * i], x[2 * i + 1]);
    lo.p[i] = __builtin_amdgcn_cvt_pkrtz(less_lo(x[2 * i], hi.u[i]), less_hi(x[2 * i + 1], hi.u[i]));
  }
}

// ---- q8 value scales. A lane loads D / 64 of a tile's, of blocks (lane * D / 64 + i) % (D / 32): the same
// ones for every second lane. unit[i] holds 2^-e of its block, 2^e above every scale of the block so far. e
// from -120 (zeros) to 126 (a scale of up to 2^128 is then below 4, its products below 2^16: two f16 parts
// still hold them).
constexpr float kUnit0 = 0x1p120f;
constexpr int kDppRor4 = 0x124, kDppRor8 = 0x128;  // row_ror, within 16 lanes
// o's blocks to the units that this tile's scales need: a power of two each, seldom anything
template <int D, class V>
__device__ __forceinline__ void raise_units(const float (&vs)[D / 64], float (&unit)[D / 64], V* o) {
  constexpr int N = D / 64, PER = sizeof(V) == 16 ? 2 : 1;  // vectors of o a block
  bool over = false;
#pragma unroll
  for (int i = 0; i < N; i++) over |= fabsf(vs[i] * unit[i]) > 1.0f;
  if (!__any(over)) return;
  float f[N];
#pragma unroll
  for (int i = 0; i < N; i++) {
    float big = fabsf(vs[i]);
    big = fmaxf(big, dpp_mov<kDppXor2>(big));  // over the lanes of this one's parity
    big = fmaxf(big, dpp_mov<kDppRor4>(big));
    big = fmaxf(big, dpp_mov<kDppRor8>(big));
    float2 r = pair16(big);
    r = pair32(fmaxf(r.x, r.y));
    const int e = min(max((int)((__float_as_uint(fmaxf(r.x, r.y)) >> 23) & 0xff) - 126, -120), 126);
    const float up = fminf(unit[i], __uint_as_float((uint32_t)(127 - e) << 23));
    f[i] = __int_as_float(max((127 << 23) + __float_as_int(up) - __float_as_int(unit[i]), 0));  // up / unit
    unit[i] = up;
  }
#pragma unroll
  for (int b = 0; b < D / 32; b++) {
    const float fb = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f[b % N]), b / N));
#pragma unroll
    for (int j = 0; j < PER; j++) o[PER * b + j] *= fb;
  }
}
// what block b of o is to be multiplied by in the end (a value is code * scale / 127)
template <int D>
__device__ __forceinline__ float unit_of(const float (&unit)[D / 64], int b) {
  const int u = __builtin_amdgcn_readlane(__float_as_int(unit[b % (D / 64)]), b / (D / 64));
  return __int_as_float((254 << 23) - u) * (1.0f / 127.0f);
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

// A score's factor from the products' one. Never zero, which a masked score (-inf) would turn into NaN.
__device__ inline float score_factor(float qs, float undo) { return fmaxf(qs * undo, 0x1p-149f); }

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

// A value the compiler takes as new here: what is computed from it for a unit's end is not computed before
// the walk over units and held (or spilled) through all of it.
__device__ __forceinline__ int afresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// what a unit's body needs to know of one of its rows
struct RowAt {
  int t, head, part, pos;
};
// (rows past the unit's: its first one)
__device__ inline RowAt row_at(const PagedKernelArgs& p, const PagedUnit& u, int kvh, int i) {
  RowAt r;
  const int rho = u.rho0 + (i < u.n_rho ? i : 0);
  const int j = rho / p.b.G;
  const PagedTok tok = p.b.toks[u.tok + j];
  r.t = tok.t;
  r.pos = tok.pos;
  r.part = tok.part < 0 ? -1 : tok.part + u.chunk;
  r.head = kvh * p.b.G + rho - j * p.b.G;
  return r;
}

// row (of D values) at which tile t of a unit begins, t one of the first four
__device__ inline size_t first_row(const PagedKernelArgs& p, const PagedUnit& u, int kvh, int t) {
  const int key = u.key0 + 32 * t, P = 1 << p.b.page_shift;
  const int id = t == 0 ? u.page[0] : t == 1 ? u.page[1] : t == 2 ? u.page[2] : u.page[3];
  return ((size_t)id * p.kv_heads + kvh) * P + (key & (P - 1));
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

// 32 rows of o between waves and threads, in LDS: 16-byte chunk ch of row c lies in line ch / 2, where the
// lanes of a matrix result (row c, dims 8 w + 4 h + e of every 32) write it without bank conflicts, and 16
// chunks of one row are read without.
__device__ inline int chunk_at(int c, int line, int h) { return line * 64 + ((c + 2 * (line & 7) + h) & 31) + 32 * h; }
template <int J>
__device__ __forceinline__ void put_o(f32x4* x, const f32x16* o, int c, int h) {
#pragma unroll
  for (int j = 0; j < J; j++)
#pragma unroll
    for (int w = 0; w < 4; w++)
      x[chunk_at(c, 4 * j + w, h)] = f32x4{o[j][4 * w], o[j][4 * w + 1], o[j][4 * w + 2], o[j][4 * w + 3]};
}
template <int J>
__device__ __forceinline__ void add_o(const f32x4* x, f32x16* o, int c, int h) {
#pragma unroll
  for (int j = 0; j < J; j++)
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const f32x4 y = x[chunk_at(c, 4 * j + w, h)];
#pragma unroll
      for (int e = 0; e < 4; e++) o[j][4 * w + e] += y[e];
    }
}
__device__ inline f32x4 get_o(const f32x4* x, int c, int ch) { return x[chunk_at(c, ch >> 1, ch & 1)]; }

// slot of register i (0..7) of lane group g in a 32-slot tile, 16-row matrix products: the V tile's own
// order (tile_slot)
__device__ inline int slot16(int g, int i) { return 16 * (g >> 1) + 8 * (i >> 2) + 4 * (g & 1) + (i & 3); }

// a 128-row unit's staging
template <int D, int DT>
struct Many {
  static constexpr int EB = DT == KV_F32 ? 4 : 2;               // bytes of a staged value
  static constexpr int KT = DT == KV_F32 || D == 256 ? 32 : 64; // positions a step
  static constexpr int NSUB = KT / 32;
  static constexpr int SUB = 32 * D * EB;                       // bytes of a staged 32-position tile of K (or V)
  static constexpr int CPR = D * EB / 16;                       // 16-byte chunks of a K row
};

// ------------------------------------------------------------------------------------------ few
// A wave's 32-position tile in matrix operand registers. All loads are buffer loads over the tile's 32
// rows: one descriptor a tile (scalars), constant lane offsets, and a tile past the wave's last one has a
// descriptor of no bytes, so that the loop needs no branch around its loads and moves nothing for them.
template <int D, int DT>
struct FewTile {
  static constexpr int NK = DT == KV_F32 ? 2 * (D / 16) : 2 * (D / 32), NV = D / 16;
  u32x4 k[DT == KV_Q8 ? 1 : NK], v[DT == KV_F32 ? 2 * NV : DT == KV_F16 ? NV : 1];
  u32x2 kc[DT == KV_Q8 ? NK : 1], vc[DT == KV_Q8 ? NV : 1];
  float ks[DT == KV_Q8 ? D / 64 : 1], vs[DT == KV_Q8 ? D / 64 : 1];  // the lane's share of the tile's scales
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const void* base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, bytes, 0x00020000);
}
template <int AUX = 0>
__device__ __forceinline__ u32x4 ld16(__amdgpu_buffer_rsrc_t r, int off, int more) {
  return __builtin_amdgcn_raw_buffer_load_b128(r, off, more, AUX);
}
__device__ __forceinline__ u32x2 ld8(__amdgpu_buffer_rsrc_t r, int off, int more) {
  return __builtin_amdgcn_raw_buffer_load_b64(r, off, more, 0);
}

template <int D, int DT>
__device__ __forceinline__ void few_load_scales(const float* base, size_t row, bool on, int lane, float (&s)[D / 64]) {
  const __amdgpu_buffer_rsrc_t r = tile_rsrc(base + row * (D / 32), on ? D * 4 : 0);
  if constexpr (D == 128) {
    const u32x2 w = ld8(r, lane * 8, 0);
    s[0] = __uint_as_float(w[0]);
    s[1] = __uint_as_float(w[1]);
  } else {
    const u32x4 w = ld16(r, lane * 16, 0);
#pragma unroll
    for (int i = 0; i < 4; i++) s[i] = __uint_as_float(w[i]);
  }
}

template <int D, int DT, int AUX>
__device__ __forceinline__ void few_load_k(const PagedKernelArgs& p, size_t row, bool on, int c, int g, FewTile<D, DT>& t) {
  // operand row c of product i is slot slot16(c / 4, 4 i + c % 4); the k dimension of a lane group is
  // 8 g + e of every 32 dims (f32: 4 g + e of every 16)
  constexpr int EB = DT == KV_F32 ? 4 : DT == KV_F16 ? 2 : 1;
  const int s0 = 16 * (c >> 3) + 4 * ((c >> 2) & 1) + (c & 3);
  const __amdgpu_buffer_rsrc_t r = tile_rsrc(p.k + row * D * EB, on ? 32 * D * EB : 0);
  if constexpr (DT == KV_F32) {
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int j = 0; j < D / 16; j++) t.k[i * (D / 16) + j] = ld16<AUX>(r, (s0 * D + 4 * g) * 4, (8 * i * D + 16 * j) * 4);
  } else if constexpr (DT == KV_F16) {
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int j = 0; j < D / 32; j++) t.k[i * (D / 32) + j] = ld16<AUX>(r, (s0 * D + 8 * g) * 2, (8 * i * D + 32 * j) * 2);
  } else {
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int j = 0; j < D / 32; j++) t.kc[i * (D / 32) + j] = ld8(r, s0 * D + 8 * g, 8 * i * D + 32 * j);
    few_load_scales<D, DT>(p.ks, row, on, c + 16 * g, t.ks);
  }
}

template <int D, int DT, int AUX>
__device__ __forceinline__ void few_load_v(const PagedKernelArgs& p, size_t row, bool on, int c, int g, FewTile<D, DT>& t) {
  constexpr int EB = DT == KV_F32 ? 4 : DT == KV_F16 ? 2 : 1;
  const __amdgpu_buffer_rsrc_t r = tile_rsrc(p.v + row * D * EB, on ? 32 * D * EB : 0);
  const int off = (g * D + c) * 8 * EB;
  if constexpr (DT == KV_F32) {
#pragma unroll
    for (int j = 0; j < D / 16; j++) {
      t.v[2 * j] = ld16<AUX>(r, off, 128 * 4 * j);
      t.v[2 * j + 1] = ld16<AUX>(r, off, 128 * 4 * j + 16);
    }
  } else if constexpr (DT == KV_F16) {
#pragma unroll
    for (int j = 0; j < D / 16; j++) t.v[j] = ld16<AUX>(r, off, 128 * 2 * j);
  } else {
#pragma unroll
    for (int j = 0; j < D / 16; j++) t.vc[j] = ld8(r, off, 128 * j);
    few_load_scales<D, DT>(p.vs, row, on, c + 16 * g, t.vs);
  }
}

// where an LDS row keeps its 16-byte chunk x: 16 rows of one chunk spread over all banks
__device__ inline int swz(int r, int x) { return x ^ (r & 15); }

// LDS of a few-row unit
template <int D, int DT>
struct FewLds {
  static constexpr int NQ = DT == KV_F32 ? D / 16 : 2 * (D / 32);
  union {
    struct {
      u32x4 q[NQ][64];                         // the queries as matrix operands, the same for every wave
      float s[DT == KV_Q8 ? 4 : 1][2][DT == KV_Q8 ? D : 1];  // q8: K and V scales of the tile a wave is at
    } in;
    struct {
      float o[4][16 * D];                      // the waves' results
      float2 ml[4][16];
    } out;
  };
  float top[4][16];                            // largest |q| of a wave's dims
  RowAt row[16];
};

// workgroups of few-row units a CU holds (waves a SIMD)
template <int D, int DT>
constexpr int few_waves() { return D == 256 ? (DT == KV_F32 ? 1 : 2) : DT == KV_F32 ? 2 : 3; }

template <int D, int DT, int AUX>
__device__ __forceinline__ void few_unit(const PagedKernelArgs& p, const PagedUnit& u, int kvh, float* ws_o, float2* ws_ml,
                                         FewLds<D, DT>& lds) {
  constexpr int NK = DT == KV_F32 ? D / 16 : D / 32;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int shift = p.b.page_shift, P = 1 << shift;
  const int n_tiles = (u.key1 - u.key0 + 31) >> 5;
  const int* pages = p.b.pages + u.table;

  auto row_of = [&](int t) -> size_t {
    const int key = u.key0 + 32 * min(t, n_tiles - 1);
    const int id = uniform(pages[key >> shift]);
    return ((size_t)id * p.kv_heads + kvh) * P + (key & (P - 1));
  };
  // the first tiles are on their way before the queries are looked at
  FewTile<D, DT> tl;
  if (n_tiles > 0) {
    const size_t row = first_row(p, u, kvh, wave);
    few_load_k<D, DT, AUX>(p, row, wave < n_tiles, c, g, tl);
    few_load_v<D, DT, AUX>(p, row, wave < n_tiles, c, g, tl);
  }

  // ---- the queries: a wave prepares every fourth operand; a row's factor needs all of them
  int pos;
  float qs = p.qscale;
  {
    const int tid = afresh(threadIdx.x), c = tid & 15, g = (tid >> 4) & 3, lane = tid & 63;
    const RowAt ra = row_at(p, u, kvh, c);
    pos = ra.pos;
    if (wave == 0 && g == 0) lds.row[c] = ra;
    const float* q = p.q + ((size_t)ra.t * p.b.H + ra.head) * D;
    if constexpr (DT == KV_F32) {
#pragma unroll
      for (int i = 0; i < NK / 4; i++) lds.in.q[4 * i + wave][lane] = *(const u32x4*)(q + 16 * (4 * i + wave) + 4 * g);
    } else {
      f32x4 x[NK / 4][2];
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < NK / 4; i++) {
        const float* at = q + 32 * (4 * i + wave) + 8 * g;
        x[i][0] = *(const f32x4*)at;
        x[i][1] = *(const f32x4*)(at + 4);
#pragma unroll
        for (int e = 0; e < 4; e++) top = fmaxf(top, fmaxf(fabsf(x[i][0][e]), fabsf(x[i][1][e])));
      }
      float2 r = pair16(top);
      top = fmaxf(r.x, r.y);
      r = pair32(top);
      lds.top[wave][c] = fmaxf(r.x, r.y);
      __syncthreads();
      float undo;
      const float f = row_factor(fmaxf(fmaxf(lds.top[0][c], lds.top[1][c]), fmaxf(lds.top[2][c], lds.top[3][c])), &undo);
      qs = score_factor(qs, undo * (DT == KV_Q8 ? 1.0f / 127.0f : 1.0f));
#pragma unroll
      for (int i = 0; i < NK / 4; i++) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = x[i][e >> 2][e & 3] * f;
        H8 hi, lo;
        split8(y, hi, lo);
        lds.in.q[2 * (4 * i + wave)][lane] = hi.u;
        lds.in.q[2 * (4 * i + wave) + 1][lane] = lo.u;
      }
    }
  }
  __syncthreads();
  // part 0: hi (f32: the values), 1: lo
  auto q_at = [&](int n, int part) __attribute__((always_inline)) {
    H8 h;
    h.u = lds.in.q[2 * n + part][lane];
    return h.h;
  };

  f32x4 o[D / 16];
  float m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int j = 0; j < D / 16; j++) o[j] = f32x4{0, 0, 0, 0};
  float unit[DT == KV_Q8 ? D / 64 : 1];  // q8: of the value scales
  if constexpr (DT == KV_Q8) {
#pragma unroll
    for (int i = 0; i < D / 64; i++) unit[i] = kUnit0;
  }

  for (int t = wave; t < n_tiles; t += 4) {
    const int key = u.key0 + 32 * t;
    const bool more = t + 4 < n_tiles;
    const size_t next = row_of(t + 4);
    float* lk = lds.in.s[DT == KV_Q8 ? wave : 0][0];
    float* lv = lds.in.s[DT == KV_Q8 ? wave : 0][1];
    if constexpr (DT == KV_Q8) {
      if (key + 32 > u.key1) {  // slots past the written positions; this lane's scales are of slot x / (D / 32)
#pragma unroll
        for (int i = 0; i < D / 64; i++)
          if (key + (lane * (D / 64) + i) / (D / 32) >= u.key1) tl.vs[i] = 0.0f;
      }
      raise_units<D>(tl.vs, unit, o);
      // a wave's LDS accesses complete in order: the tile before is done with them
#pragma unroll
      for (int i = 0; i < D / 64; i++) {
        lk[lane * (D / 64) + i] = tl.ks[i];
        lv[lane * (D / 64) + i] = tl.vs[i] * unit[i];
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    // ---- scores: sc[e] of slot slot16(g, e), row c
    float sc[8];
    if constexpr (DT == KV_F32) {
      f32x4 a[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
      for (int n = 0; n < NK; n++) {
        const f32x4 qn = *(const f32x4*)&lds.in.q[n][lane];
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
          for (int i = 0; i < 2; i++)
            a[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(tl.k[i * NK + n][e]), qn[e], a[i], 0, 0, 0);
      }
#pragma unroll
      for (int e = 0; e < 8; e++) sc[e] = a[e >> 2][e & 3];
    } else if constexpr (DT == KV_F16) {
      f32x4 a[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}}, b[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
      for (int n = 0; n < NK; n++) {
        H8 k0, k1;
        k0.u = tl.k[n];
        k1.u = tl.k[NK + n];
        const half8 qh = q_at(n, 0), ql = q_at(n, 1);
        a[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0.h, qh, a[0], 0, 0, 0);
        a[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1.h, qh, a[1], 0, 0, 0);
        b[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0.h, ql, b[0], 0, 0, 0);
        b[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1.h, ql, b[1], 0, 0, 0);
      }
#pragma unroll
      for (int e = 0; e < 8; e++) sc[e] = a[e >> 2][e & 3] + b[e >> 2][e & 3];
    } else {
      // a product's 32 dims are one scale block: its exact code sums, then the block scale in f32
#pragma unroll
      for (int e = 0; e < 8; e++) sc[e] = 0.0f;
#pragma unroll
      for (int n4 = 0; n4 < NK; n4 += 4) {
        f32x4 a[4][2];
#pragma unroll
        for (int n = 0; n < 4; n++) {
          const half8 k0 = codes8(tl.kc[n4 + n]), k1 = codes8(tl.kc[NK + n4 + n]);
          const half8 qh = q_at(n4 + n, 0), ql = q_at(n4 + n, 1);
          a[n][0] = a[n][1] = f32x4{0, 0, 0, 0};
          a[n][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qh, a[n][0], 0, 0, 0);
          a[n][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qh, a[n][1], 0, 0, 0);
          a[n][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, ql, a[n][0], 0, 0, 0);
          a[n][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, ql, a[n][1], 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const f32x4 z = *(const f32x4*)(lk + slot16(g, e) * (D / 32) + n4);
#pragma unroll
          for (int n = 0; n < 4; n++) sc[e] = fmaf(a[n][e >> 2][e & 3], z[n], sc[e]);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // into the registers just used: not before, which would take a second set
    few_load_k<D, DT, AUX>(p, next, more, c, g, tl);
    __builtin_amdgcn_sched_barrier(0);
    if (key + 32 > u.mask0) {
#pragma unroll
      for (int e = 0; e < 8; e++) sc[e] = key + slot16(g, e) <= pos ? sc[e] : -INFINITY;
    }
    if (DT != KV_Q8 && key + 32 > u.key1) {  // slots past the written positions
      if constexpr (DT == KV_F32) {
#pragma unroll
        for (int j = 0; j < D / 16; j++)
#pragma unroll
          for (int e = 0; e < 8; e++)
            tl.v[2 * j + (e >> 2)][e & 3] = key + slot16(g, e) < u.key1 ? tl.v[2 * j + (e >> 2)][e & 3] : 0u;
      } else if constexpr (DT == KV_F16) {
        u32x4 keep;
#pragma unroll
        for (int w = 0; w < 4; w++)
          keep[w] = (key + slot16(g, 2 * w) < u.key1 ? 0xffffu : 0u) | (key + slot16(g, 2 * w + 1) < u.key1 ? 0xffff0000u : 0u);
#pragma unroll
        for (int j = 0; j < D / 16; j++) tl.v[j] &= keep;
      }
    }
    // ---- running maximum and sum
    float top = sc[0];
#pragma unroll
    for (int e = 1; e < 8; e++) top = fmaxf(top, sc[e]);
    float2 r = pair16(top);
    top = fmaxf(r.x, r.y);
    r = pair32(top);
    top = fmaxf(r.x, r.y) * qs;
    if (__any(top > m + kLazy)) {
      const float mn = top > m + kLazy ? top : m;
      const float f = m == -INFINITY ? 1.0f : exp2_hw(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int j = 0; j < D / 16; j++) o[j] *= f;
    }
    const float base = m == -INFINITY ? 0.0f : kPShift - m;
    float pr[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      pr[e] = exp2_hw(fmaf(sc[e], qs, base));
      l += pr[e];
    }
    // ---- o
    if constexpr (DT == KV_F32) {
#pragma unroll
      for (int e = 0; e < 8; e++)
#pragma unroll
        for (int j = 0; j < D / 16; j++)
          o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(tl.v[2 * j + (e >> 2)][e & 3]), pr[e], o[j], 0, 0, 0);
    } else if constexpr (DT == KV_F16) {
      H8 ph, pl;
      split8(pr, ph, pl);
#pragma unroll
      for (int j = 0; j < D / 16; j++) {
        H8 a;
        a.u = tl.v[j];
        o[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h, ph.h, o[j], 0, 0, 0);
      }
#pragma unroll
      for (int j = 0; j < D / 16; j++) {
        H8 a;
        a.u = tl.v[j];
        o[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h, pl.h, o[j], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int n4 = 0; n4 < D / 32; n4 += 4) {
        f32x4 z[8];
#pragma unroll
        for (int e = 0; e < 8; e++) z[e] = *(const f32x4*)(lv + slot16(g, e) * (D / 32) + n4);
#pragma unroll
        for (int n = 0; n < 4; n++) {
          const half8 a0 = codes8(tl.vc[2 * (n4 + n)]), a1 = codes8(tl.vc[2 * (n4 + n) + 1]);
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; e++) x[e] = pr[e] * z[e][n];
          H8 ph, pl;
          split8(x, ph, pl);
          f32x4 &o0 = o[2 * (n4 + n)], &o1 = o[2 * (n4 + n) + 1];
          o0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, ph.h, o0, 0, 0, 0);
          o1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, ph.h, o1, 0, 0, 0);
          o0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, pl.h, o0, 0, 0, 0);
          o1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, pl.h, o1, 0, 0, 0);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    few_load_v<D, DT, AUX>(p, next, more, c, g, tl);
    __builtin_amdgcn_sched_barrier(0);
  }

  // ---- the four waves' results meet in LDS
  const int tid = afresh(threadIdx.x), ec = tid & 15, eg = (tid >> 4) & 3;
  if constexpr (DT == KV_Q8) {
#pragma unroll
    for (int j = 0; j < D / 16; j++) o[j] *= unit_of<D>(unit, j / 2);
  }
  __syncthreads();  // every wave is done with the queries and its scales
  {
    float2 r = pair16(l);
    l = r.x + r.y;
    r = pair32(l);
    l = r.x + r.y;
    if (eg == 0) lds.out.ml[wave][ec] = make_float2(m, l);
#pragma unroll
    for (int j = 0; j < D / 16; j++) *(f32x4*)&lds.out.o[wave][ec * D + swz(ec, 4 * j + eg) * 4] = o[j];
  }
  __syncthreads();
  for (int x = tid; x < u.n_rho * (D / 4); x += 256) {
    const int i = x / (D / 4), ch = x % (D / 4);
    float mw[4], lw[4], top = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const float2 z = lds.out.ml[w][i];
      mw[w] = z.x;
      lw[w] = z.y;
      top = fmaxf(top, z.x);
    }
    f32x4 sum = {0, 0, 0, 0};
    float lsum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const float f = mw[w] == -INFINITY ? 0.0f : exp2_hw(mw[w] - top);
      lsum += lw[w] * f;
      sum += *(const f32x4*)&lds.out.o[w][i * D + swz(i, ch) * 4] * f;
    }
    const RowAt r = lds.row[i];
    store_o<D>(p, ws_o, r, 4 * ch, sum, lsum);
    if (ch == 0 && r.part >= 0) ws_ml[(size_t)r.part * p.b.H + r.head] = make_float2(top, lsum);
  }
}

// ------------------------------------------------------------------------------------------ mid
// A wave's 32-position tile as operands of the 32-row products (descriptors as for the few-row units): K
// row c, dims 16 n + 8 h + e (f32 8 n + 4 h + e, q8 32 n + 16 h + e); V dim 32 j + c, panel 2 x + h.
template <int D, int DT>
struct MidK {
  static constexpr int N = DT == KV_F32 ? D / 8 : DT == KV_F16 ? D / 16 : D / 32;
  u32x4 k[N];
  float ks[DT == KV_Q8 ? D / 64 : 1];
};
template <int D, int DT>
struct MidV {
  static constexpr int N = 2 * (D / 32);
  u32x4 v[DT == KV_F32 ? 2 * N : DT == KV_F16 ? N : 1];
  u32x2 vc[DT == KV_Q8 ? N : 1];
  float vs[DT == KV_Q8 ? D / 64 : 1];
};

template <int D, int DT>
__device__ __forceinline__ void mid_load_k(const PagedKernelArgs& p, size_t row, bool on, int c, int h, MidK<D, DT>& t) {
  constexpr int EB = DT == KV_F32 ? 4 : DT == KV_F16 ? 2 : 1;
  const __amdgpu_buffer_rsrc_t r = tile_rsrc(p.k + row * D * EB, on ? 32 * D * EB : 0);
#pragma unroll
  for (int n = 0; n < MidK<D, DT>::N; n++) t.k[n] = ld16(r, c * D * EB + 16 * h, 32 * n);
  if constexpr (DT == KV_Q8) few_load_scales<D, DT>(p.ks, row, on, c + 32 * h, t.ks);
}
template <int D, int DT>
__device__ __forceinline__ void mid_load_v(const PagedKernelArgs& p, size_t row, bool on, int c, int h, MidV<D, DT>& t) {
  constexpr int EB = DT == KV_F32 ? 4 : DT == KV_F16 ? 2 : 1;
  const __amdgpu_buffer_rsrc_t r = tile_rsrc(p.v + row * D * EB, on ? 32 * D * EB : 0);
  const int off = (h * D + c) * 8 * EB;
#pragma unroll
  for (int x = 0; x < 2; x++)
#pragma unroll
    for (int j = 0; j < D / 32; j++) {
      const int at = (2 * x * D + 32 * j) * 8 * EB;
      if constexpr (DT == KV_F32) {
        t.v[2 * (x * (D / 32) + j)] = ld16(r, off, at);
        t.v[2 * (x * (D / 32) + j) + 1] = ld16(r, off, at + 16);
      } else if constexpr (DT == KV_F16) {
        t.v[x * (D / 32) + j] = ld16(r, off, at);
      } else {
        t.vc[x * (D / 32) + j] = ld8(r, off, at);
      }
    }
  if constexpr (DT == KV_Q8) few_load_scales<D, DT>(p.vs, row, on, c + 32 * h, t.vs);
}

template <int D, int DT>
struct MidLds {
  static constexpr int NQ = DT == KV_F32 ? D / 8 : 2 * (D / 16);
  union {
    struct {
      u32x4 q[NQ][64];                         // the queries as matrix operands, the same for every wave
      float s[DT == KV_Q8 ? 4 : 1][2][DT == KV_Q8 ? D : 1];  // q8: K and V scales of the tile a wave is at
    } in;
    f32x4 x[2][D / 8 * 64];                    // two waves' o
  };
  float2 ml[4][32];                            // the waves' (m, l)
  float2 all[32];                              // the rows' (m, l)
  RowAt row[32];
  float top[4][32];                            // largest |q| of a wave's dims
};

template <int D, int DT>
__device__ __forceinline__ void mid_unit(const PagedKernelArgs& p, const PagedUnit& u, int kvh, float* ws_o, float2* ws_ml,
                                         MidLds<D, DT>& lds) {
  constexpr int ND = D / 32;
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int shift = p.b.page_shift, P = 1 << shift;
  const int n_tiles = (u.key1 - u.key0 + 31) >> 5;
  const int* pages = p.b.pages + u.table;
  auto row_of = [&](int t) -> size_t {
    const int key = u.key0 + 32 * min(t, n_tiles - 1);
    const int id = uniform(pages[key >> shift]);
    return ((size_t)id * p.kv_heads + kvh) * P + (key & (P - 1));
  };
  MidK<D, DT> tk;
  MidV<D, DT> tv;
  if (n_tiles > 0) {
    const size_t row = first_row(p, u, kvh, wave);
    mid_load_k<D, DT>(p, row, wave < n_tiles, c, h, tk);
    mid_load_v<D, DT>(p, row, wave < n_tiles, c, h, tv);
  }
  // ---- the queries: a wave prepares every fourth operand; a row's factor needs all of them
  int pos;
  float qs = p.qscale;
  {
    const int tid = afresh(threadIdx.x), c = tid & 31, h = (tid >> 5) & 1, lane = tid & 63;
    const RowAt ra = row_at(p, u, kvh, c);
    pos = ra.pos;
    if (wave == 0 && h == 0) lds.row[c] = ra;
    const float* q = p.q + ((size_t)ra.t * p.b.H + ra.head) * D;
    if constexpr (DT == KV_F32) {
#pragma unroll
      for (int i = 0; i < D / 32; i++) lds.in.q[4 * i + wave][lane] = *(const u32x4*)(q + 8 * (4 * i + wave) + 4 * h);
    } else {
      // product n: f16 dims 16 n + 8 h + e; q8 block n / 2, dims 16 h + 8 (n & 1) + e
      f32x4 x[D / 64][2];
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 64; i++) {
        const int n = 4 * i + wave;
        const float* at = q + (DT == KV_F16 ? 16 * n + 8 * h : 32 * (n >> 1) + 16 * h + 8 * (n & 1));
        x[i][0] = *(const f32x4*)at;
        x[i][1] = *(const f32x4*)(at + 4);
#pragma unroll
        for (int e = 0; e < 4; e++) top = fmaxf(top, fmaxf(fabsf(x[i][0][e]), fabsf(x[i][1][e])));
      }
      const float2 r = pair32(top);
      lds.top[wave][c] = fmaxf(r.x, r.y);
      __syncthreads();
      float undo;
      const float f = row_factor(fmaxf(fmaxf(lds.top[0][c], lds.top[1][c]), fmaxf(lds.top[2][c], lds.top[3][c])), &undo);
      qs = score_factor(qs, undo * (DT == KV_Q8 ? 1.0f / 127.0f : 1.0f));
#pragma unroll
      for (int i = 0; i < D / 64; i++) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = x[i][e >> 2][e & 3] * f;
        H8 hi, lo;
        split8(y, hi, lo);
        lds.in.q[2 * (4 * i + wave)][lane] = hi.u;
        lds.in.q[2 * (4 * i + wave) + 1][lane] = lo.u;
      }
    }
  }
  __syncthreads();
  auto q_at = [&](int n, int part) __attribute__((always_inline)) {
    H8 x;
    x.u = lds.in.q[2 * n + part][lane];
    return x.h;
  };

  f32x16 o[ND];
#pragma unroll
  for (int j = 0; j < ND; j++)
#pragma unroll
    for (int e = 0; e < 16; e++) o[j][e] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  float unit[DT == KV_Q8 ? D / 64 : 1];  // q8: of the value scales
  if constexpr (DT == KV_Q8) {
#pragma unroll
    for (int i = 0; i < D / 64; i++) unit[i] = kUnit0;
  }

  for (int t = wave; t < n_tiles; t += 4) {
    const int key = u.key0 + 32 * t;
    const bool more = t + 4 < n_tiles;
    const size_t next = row_of(t + 4);
    float* lk = lds.in.s[DT == KV_Q8 ? wave : 0][0];
    float* lv = lds.in.s[DT == KV_Q8 ? wave : 0][1];
    if constexpr (DT == KV_Q8) {
      if (key + 32 > u.key1) {  // slots past the written positions
#pragma unroll
        for (int i = 0; i < D / 64; i++)
          if (key + (lane * (D / 64) + i) / (D / 32) >= u.key1) tv.vs[i] = 0.0f;
      }
      raise_units<D>(tv.vs, unit, o);
      // [block][position], so that a lane reads the four positions of a register group at once; a wave's
      // LDS accesses complete in order: the tile before is done with them
#pragma unroll
      for (int i = 0; i < D / 64; i++) {
        const int x = lane * (D / 64) + i, at = x % (D / 32) * 32 + x / (D / 32);
        lk[at] = tk.ks[i];
        lv[at] = tv.vs[i] * unit[i];
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    // ---- scores: s[e] of slot 8 (e / 4) + 4 h + e % 4, row c
    float s[16];
    if constexpr (DT == KV_F32) {
      f32x16 a;
#pragma unroll
      for (int e = 0; e < 16; e++) a[e] = 0.0f;
#pragma unroll
      for (int n = 0; n < D / 8; n++) {
        const f32x4 qn = *(const f32x4*)&lds.in.q[n][lane];
#pragma unroll
        for (int e = 0; e < 4; e++) a = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(tk.k[n][e]), qn[e], a, 0, 0, 0);
      }
#pragma unroll
      for (int e = 0; e < 16; e++) s[e] = a[e];
    } else if constexpr (DT == KV_F16) {
      f32x16 a;
#pragma unroll
      for (int e = 0; e < 16; e++) a[e] = 0.0f;
#pragma unroll
      for (int n = 0; n < D / 16; n++) {
        H8 x;
        x.u = tk.k[n];
        a = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.h, q_at(n, 0), a, 0, 0, 0);
        a = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.h, q_at(n, 1), a, 0, 0, 0);
      }
#pragma unroll
      for (int e = 0; e < 16; e++) s[e] = a[e];
    } else {
#pragma unroll
      for (int e = 0; e < 16; e++) s[e] = 0.0f;
#pragma unroll
      for (int b = 0; b < ND; b++) {
        const half8 x0 = codes8(u32x2{tk.k[b][0], tk.k[b][1]}), x1 = codes8(u32x2{tk.k[b][2], tk.k[b][3]});
        f32x16 a;
#pragma unroll
        for (int e = 0; e < 16; e++) a[e] = 0.0f;
        a = __builtin_amdgcn_mfma_f32_32x32x16_f16(x0, q_at(2 * b, 0), a, 0, 0, 0);
        a = __builtin_amdgcn_mfma_f32_32x32x16_f16(x0, q_at(2 * b, 1), a, 0, 0, 0);
        a = __builtin_amdgcn_mfma_f32_32x32x16_f16(x1, q_at(2 * b + 1, 0), a, 0, 0, 0);
        a = __builtin_amdgcn_mfma_f32_32x32x16_f16(x1, q_at(2 * b + 1, 1), a, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < 4; w++) {
          const f32x4 z = *(const f32x4*)(lk + 32 * b + 8 * w + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; e++) s[4 * w + e] = fmaf(a[4 * w + e], z[e], s[4 * w + e]);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // into the registers just used: not before, which would take a second set
    mid_load_k<D, DT>(p, next, more, c, h, tk);
    __builtin_amdgcn_sched_barrier(0);
    if (key + 32 > u.mask0) {
#pragma unroll
      for (int e = 0; e < 16; e++) s[e] = key + 8 * (e >> 2) + 4 * h + (e & 3) <= pos ? s[e] : -INFINITY;
    }
    if (DT != KV_Q8 && key + 32 > u.key1) {  // slots past the written positions
      if constexpr (DT == KV_F32) {
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
          for (int j = 0; j < ND; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
              const int i = 2 * (x * ND + j) + (e >> 2);
              tv.v[i][e & 3] = key + 16 * x + 8 * (e >> 2) + 4 * h + (e & 3) < u.key1 ? tv.v[i][e & 3] : 0u;
            }
      } else if constexpr (DT == KV_F16) {
#pragma unroll
        for (int x = 0; x < 2; x++) {
          u32x4 keep;
#pragma unroll
          for (int w = 0; w < 4; w++) {
            const int at = key + 16 * x + 8 * (w >> 1) + 4 * h + 2 * (w & 1);
            keep[w] = (at < u.key1 ? 0xffffu : 0u) | (at + 1 < u.key1 ? 0xffff0000u : 0u);
          }
#pragma unroll
          for (int j = 0; j < ND; j++) tv.v[x * ND + j] &= keep;
        }
      }
    }
    // ---- running maximum and sum
    float top = s[0];
#pragma unroll
    for (int e = 1; e < 16; e++) top = fmaxf(top, s[e]);
    const float2 r = pair32(top);
    top = fmaxf(r.x, r.y) * qs;
    if (__any(top > m + kLazy)) {
      const float mn = top > m + kLazy ? top : m;
      const float f = m == -INFINITY ? 1.0f : exp2_hw(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int j = 0; j < ND; j++) o[j] *= f;
    }
    const float base = m == -INFINITY ? 0.0f : kPShift - m;
#pragma unroll
    for (int e = 0; e < 16; e++) {
      s[e] = exp2_hw(fmaf(s[e], qs, base));
      l += s[e];
    }
    // ---- o
#pragma unroll
    for (int x = 0; x < 2; x++) {
      if constexpr (DT == KV_F32) {
#pragma unroll
        for (int e = 0; e < 8; e++)
#pragma unroll
          for (int j = 0; j < ND; j++)
            o[j] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(tv.v[2 * (x * ND + j) + (e >> 2)][e & 3]), s[8 * x + e],
                                                        o[j], 0, 0, 0);
      } else if constexpr (DT == KV_F16) {
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; e++) w[e] = s[8 * x + e];
        H8 ph, pl;
        split8(w, ph, pl);
#pragma unroll
        for (int j = 0; j < ND; j++) {
          H8 a;
          a.u = tv.v[x * ND + j];
          o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, ph.h, o[j], 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < ND; j++) {
          H8 a;
          a.u = tv.v[x * ND + j];
          o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, pl.h, o[j], 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int j = 0; j < ND; j++) {
          float w[8];
#pragma unroll
          for (int y = 0; y < 2; y++) {
            const f32x4 z = *(const f32x4*)(lv + 32 * j + 16 * x + 8 * y + 4 * h);
#pragma unroll
            for (int e = 0; e < 4; e++) w[4 * y + e] = s[8 * x + 4 * y + e] * z[e];
          }
          H8 ph, pl;
          split8(w, ph, pl);
          const half8 a = codes8(tv.vc[x * ND + j]);
          o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph.h, o[j], 0, 0, 0);
          o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl.h, o[j], 0, 0, 0);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    mid_load_v<D, DT>(p, next, more, c, h, tv);
    __builtin_amdgcn_sched_barrier(0);
  }

  // ---- the four waves' results, weighted by one maximum: two waves' o through LDS to the other two, their
  // sums through LDS to all threads, which store whole rows
  const int tid = afresh(threadIdx.x), ec = tid & 31, eh = (tid >> 5) & 1;
  {
    const float2 r = pair32(l);
    l = r.x + r.y;
  }
  if (eh == 0) lds.ml[wave][ec] = make_float2(m, l);
  __syncthreads();  // and every wave is done with the queries and its scales
  float top = -INFINITY, lsum = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; w++) top = fmaxf(top, lds.ml[w][ec].x);
#pragma unroll
  for (int w = 0; w < 4; w++) {
    const float2 z = lds.ml[w][ec];
    lsum += z.y * (z.x == -INFINITY ? 0.0f : exp2_hw(z.x - top));  // a sum that is NaN stays one
  }
  const float mine = m == -INFINITY ? 0.0f : exp2_hw(m - top);
#pragma unroll
  for (int j = 0; j < ND; j++) {
    if constexpr (DT == KV_Q8) o[j] *= mine * unit_of<D>(unit, j);
    else o[j] *= mine;
  }
  if (wave == 0 && eh == 0) lds.all[ec] = make_float2(top, lsum);
  if (wave >= 2) put_o<ND>(lds.x[wave - 2], o, ec, eh);
  __syncthreads();
  if (wave < 2) {
    add_o<ND>(lds.x[wave], o, ec, eh);
    put_o<ND>(lds.x[wave], o, ec, eh);  // a lane's own places
  }
  __syncthreads();
#pragma unroll 1
  for (int x = tid; x < u.n_rho * (D / 4); x += 256) {
    const int i = x / (D / 4), ch = x % (D / 4);
    const RowAt r = lds.row[i];
    const float2 z = lds.all[i];
    store_o<D>(p, ws_o, r, 4 * ch, get_o(lds.x[0], i, ch) + get_o(lds.x[1], i, ch), z.y);
    if (ch == 0 && r.part >= 0) ws_ml[(size_t)r.part * p.b.H + r.head] = z;
  }
}

// ------------------------------------------------------------------------------------------ many
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

template <int D, int DT>
__device__ __forceinline__ void many_unit(const PagedKernelArgs& p, const PagedUnit& u, int kvh, float* ws_o, float2* ws_ml,
                                          char* k0, char* k1, char* v0, char* v1) {
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
    pos = ra.pos;
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
      qs = score_factor(p.qscale, undo);
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
  float m = -INFINITY, l = 0.0f;

  auto row_of = [&](int t) -> size_t {
    const int key = u.key0 + 32 * min(t, n_tiles - 1);  // past the end: staged again, masked
    const int id = uniform(pages[key >> shift]);
    return ((size_t)id * p.kv_heads + kvh) * P + (key & (P - 1));
  };

  // one step over staged tiles; key: its first position
  auto step = [&](const char* kb, const char* vb, int key) __attribute__((always_inline)) {
    float s[NSUB][16];
    if constexpr (DT == KV_F16) {
      // both sub-tiles' chains side by side, their operands read two chunks ahead
      f32x16 a[NSUB];
#pragma unroll
      for (int sub = 0; sub < NSUB; sub++)
#pragma unroll
        for (int e = 0; e < 16; e++) a[sub][e] = 0.0f;
      int at = c * M::CPR * 16 + swz(c, h) * 16;  // chunk 2 n + h lies at at ^ 32 n
      asm volatile("" : "+v"(at));                // made here, not kept in a register a chunk
#pragma unroll
      for (int n = 0; n < NK; n++) {
        H8 x[NSUB];
#pragma unroll
        for (int sub = 0; sub < NSUB; sub++) x[sub].u = *(const u32x4*)(kb + sub * M::SUB + (at ^ (32 * n)));
#pragma unroll
        for (int sub = 0; sub < NSUB; sub++) a[sub] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[sub].h, qh[n].h, a[sub], 0, 0, 0);
#pragma unroll
        for (int sub = 0; sub < NSUB; sub++) a[sub] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[sub].h, ql[n].h, a[sub], 0, 0, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, 2 * NSUB, 0);
#pragma unroll
      for (int n = 0; n < NK; n++) {
        __builtin_amdgcn_sched_group_barrier(0x008, 2 * NSUB, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, NSUB, 0);
      }
#pragma unroll
      for (int sub = 0; sub < NSUB; sub++)
#pragma unroll
        for (int e = 0; e < 16; e++) s[sub][e] = a[sub][e];
    }
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
      const float mn = top > m + kLazy ? top : m;
      const float f = m == -INFINITY ? 1.0f : exp2_hw(m - mn);
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
          for (int j = 0; j < D / 32; j += 2) {
            H8 a, b;
            a.u = *(const u32x4*)(vt + ((2 * x + h) * D + 32 * j + c) * 16);
            b.u = *(const u32x4*)(vt + ((2 * x + h) * D + 32 * j + 32 + c) * 16);
            o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, ph.h, o[j], 0, 0, 0);
            o[j + 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b.h, ph.h, o[j + 1], 0, 0, 0);
            o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, pl.h, o[j], 0, 0, 0);
            o[j + 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b.h, pl.h, o[j + 1], 0, 0, 0);
          }
        }
      }
    }
  };
  // V past the written positions becomes zero
  auto clear_stale = [&](char* vb, int key) __attribute__((always_inline)) {
    for (int x = threadIdx.x; x < KT * D; x += 256) {
      const int sub = x / (32 * D), y = x % (32 * D), panel = y / (8 * D), e = y % 8;
      if (key + 32 * sub + tile_slot(panel, e) >= u.key1) {
        if constexpr (DT == KV_F32) ((float*)vb)[x] = 0.0f;
        else ((uint16_t*)vb)[x] = 0;
      }
    }
    __syncthreads();
  };
  auto begin = [&](int st, char* kd, char* vd) __attribute__((always_inline)) {
#pragma unroll
    for (int sub = 0; sub < NSUB; sub++) many_stage<D, DT>(p, row_of(NSUB * st + sub), kd + sub * M::SUB, vd + sub * M::SUB);
  };
  auto one = [&](int st, char* kb, char* vb, char* kn, char* vn) __attribute__((always_inline)) {
    // the step's tiles have landed; the other buffers' readers are done
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (st + 1 < n_steps) begin(st + 1, kn, vn);
    const int key = u.key0 + KT * st;
    if (key + KT > u.key1) clear_stale(vb, key);
    if (active) step(kb, vb, key);
  };
  if (n_steps > 0) begin(0, k0, v0);
  for (int st = 0; st < n_steps; st += 2) {
    one(st, k0, v0, k1, v1);
    if (st + 1 < n_steps) one(st + 1, k1, v1, k0, v0);
  }
  const float2 r = pair32(l);
  l = r.x + r.y;
  if (32 * wave + c < u.n_rho) {
#pragma unroll
    for (int j = 0; j < D / 32; j++)
#pragma unroll
      for (int w = 0; w < 4; w++)
        store_o<D>(p, ws_o, ra, 32 * j + 8 * w + 4 * h,
                   f32x4{o[j][4 * w], o[j][4 * w + 1], o[j][4 * w + 2], o[j][4 * w + 3]}, l);
    if (h == 0 && ra.part >= 0) ws_ml[(size_t)ra.part * p.b.H + ra.head] = make_float2(m, l);
  }
}

// A workgroup a unit and kv head; a launch under capture walks the units of whatever batch is set.
template <int D, int DT>
__global__ __launch_bounds__(256, D == 128 ? 2 : 1) void paged_many_kernel(PagedKernelArgs p) {
  using M = Many<D, DT>;
  // K and V tiles of even and odd steps. Distinct arrays: a copy into one buffer then cannot alias the
  // reads of another, and the compiler adds no waits between them.
  __shared__ __align__(16) char k0[M::SUB * M::NSUB];
  __shared__ __align__(16) char k1[M::SUB * M::NSUB];
  __shared__ __align__(16) char v0[M::SUB * M::NSUB];
  __shared__ __align__(16) char v1[M::SUB * M::NSUB];
  const int total = p.n_blocks ? p.n_blocks : p.b.hdr->n_many * p.kv_heads;
  float* ws_o = p.b.hdr->ws_o;
  float2* ws_ml = p.b.hdr->ws_ml;
  for (int b = blockIdx.x; b < total; b += gridDim.x) {
    const PagedUnit u = p.b.units[b / p.kv_heads];
    many_unit<D, DT>(p, u, b % p.kv_heads, ws_o, ws_ml, k0, k1, v0, v1);
    __syncthreads();  // the unit's LDS is read before the next one's is written
  }
}

// workgroups of 32-row units a CU holds
template <int D, int DT>
constexpr int mid_waves() { return D == 256 && DT != KV_Q8 ? 1 : D == 128 && DT == KV_Q8 ? 3 : 2; }

template <int D, int DT>
__global__ __launch_bounds__(256, (mid_waves<D, DT>())) void paged_mid_kernel(PagedKernelArgs p) {
  __shared__ MidLds<D, DT> lds;
  const PagedHeader* h = p.b.hdr;
  const int first = p.n_blocks ? p.first : h->n_many;
  const int total = p.n_blocks ? p.n_blocks : h->n_mid * p.kv_heads;
  float* ws_o = h->ws_o;
  float2* ws_ml = h->ws_ml;
  for (int b = blockIdx.x; b < total; b += gridDim.x) {
    const PagedUnit u = p.b.units[first + b / p.kv_heads];
    mid_unit<D, DT>(p, u, b % p.kv_heads, ws_o, ws_ml, lds);
    __syncthreads();  // the unit's LDS is read before the next one's is written
  }
}

// AUX: cache policy of the page loads (2: nontemporal)
template <int D, int DT, int AUX>
__global__ __launch_bounds__(256, (few_waves<D, DT>())) void paged_few_kernel(PagedKernelArgs p) {
  __shared__ FewLds<D, DT> lds;
  const PagedHeader* h = p.b.hdr;
  const int first = p.n_blocks ? p.first : h->n_many + h->n_mid;
  const int total = p.n_blocks ? p.n_blocks : (h->n_units - first) * p.kv_heads;
  float* ws_o = h->ws_o;
  float2* ws_ml = h->ws_ml;
  for (int b = blockIdx.x; b < total; b += gridDim.x) {
    const PagedUnit u = p.b.units[first + b / p.kv_heads];
    few_unit<D, DT, AUX>(p, u, b % p.kv_heads, ws_o, ws_ml, lds);
    __syncthreads();  // the unit's LDS is read before the next one's is written
  }
}

template <int D>
__host__ __device__ inline long merge_blocks(long rows, int groups) {
  const int rpw = 256 / (D / 4 * groups);
  return (rows + rpw - 1) / rpw;
}

// A row's partials joined. D / 4 lanes hold a partial's row (16 bytes a lane); PP lane groups a row take
// every PP-th partial, eight at a time, all loaded before any is used (a row of 55 partials: two rounds of
// memory latency instead of 55), and meet in LDS. The merges of at most kMergeFew partials come first and
// take one group a row (a row of two would leave three of four groups idle), the others four; a workgroup
// has rows of one kind.
template <int D>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedKernelArgs p) {
  constexpr int LPR = D / 4, N = 8, MAXP = 4;
  static_assert(N >= kMergeFew, "one round takes a row of few partials");
  __shared__ f32x4 lo[256 / (LPR * MAXP)][MAXP][LPR];
  __shared__ float2 lml[256 / (LPR * MAXP)][MAXP];
  const int H = p.b.H;
  const PagedHeader* hdr = p.b.hdr;
  const long n_few = (long)(p.b.captured ? hdr->n_merge_few : p.b.n_merge_few) * H;
  const long n_all = (long)(p.b.captured ? hdr->n_merges : p.b.n_merges) * H;
  const long few_blocks = merge_blocks<D>(n_few, 1), blocks = few_blocks + merge_blocks<D>(n_all - n_few, MAXP);
  const float* ws_o = p.b.hdr->ws_o;
  const float2* ws_ml = p.b.hdr->ws_ml;
  for (long blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const bool few = blk < few_blocks;
    const int PP = few ? 1 : MAXP, RPW = 256 / (LPR * PP);
    const int c = threadIdx.x % LPR, g = few ? 0 : threadIdx.x / LPR % MAXP, rw = threadIdx.x / (LPR * PP);
    const long first = few ? blk * RPW : n_few + (blk - few_blocks) * RPW, total = few ? n_few : n_all;
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
  // Under capture grids that fill the GPU walk the units of whatever batch is set at replay, of every kind (a
  // kind without units takes 0.7-1.6 us, q8's few rows 4.5).
  PagedKernelArgs x = k;
  if constexpr (paged_has_many(D, DT)) {
    if (b.captured || b.n_many) {
      x.n_blocks = b.n_many * k.kv_heads;
      const unsigned grid = (unsigned)(b.captured ? a.num_cus * (D == 128 ? 2 : 1) : x.n_blocks);
      hipLaunchKernelGGL((paged_many_kernel<D, DT>), dim3(grid), dim3(256), 0, st, x);
    }
  }
  if (b.captured || b.n_mid) {
    x.first = b.n_many;
    x.n_blocks = b.n_mid * k.kv_heads;
    const unsigned grid = (unsigned)(b.captured ? a.num_cus * mid_waves<D, DT>() : x.n_blocks);
    hipLaunchKernelGGL((paged_mid_kernel<D, DT>), dim3(grid), dim3(256), 0, st, x);
  }
  if (b.captured || b.n_units > b.n_many + b.n_mid) {
    x.first = b.n_many + b.n_mid;
    x.n_blocks = (b.n_units - x.first) * k.kv_heads;
    const unsigned grid = (unsigned)(b.captured ? a.num_cus * few_waves<D, DT>() : x.n_blocks);
    // Pages that one unit reads once, more of them than caches keep from call to call: nontemporal, which
    // leaves the shared pages there (64 sequences of 2,000, 524 MB: 94 -> 83 us; a shared 16k document
    // beside tails of 71 MB 61 -> 57). Two row tiles that share a page want it kept (115 -> 149), and q8's
    // 8-byte and head_dim 256's strided pieces of a line come one after the other (138 -> 157, 137 -> 151).
    bool stream = false;
    if constexpr (paged_has_stream(D, DT)) {
      stream = b.stream_few;
      if (stream) hipLaunchKernelGGL((paged_few_kernel<D, DT, 2>), dim3(grid), dim3(256), 0, st, x);
    }
    if (!stream) hipLaunchKernelGGL((paged_few_kernel<D, DT, 0>), dim3(grid), dim3(256), 0, st, x);
  }
  if (b.captured || b.n_merges) {
    const long few = (long)b.n_merge_few * b.H, all = (long)b.n_merges * b.H;
    const long grid = b.captured ? a.num_cus * 4L : merge_blocks<D>(few, 1) + merge_blocks<D>(all - few, 4);
    hipLaunchKernelGGL((paged_merge_kernel<D>), dim3((unsigned)grid), dim3(256), 0, st, k);
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
