// Storing one cache row (D values spread D/64 per lane over a wave) in the storage mode's
// format: f32 copy (shaders/copy.wgsl), f16 RNE (shaders/copy_kv16.wgsl:13) or q8 codes with
// one f32 scale per 32 values (shaders/copy_kv8.wgsl:24-40).
#pragma once

#include "bg_kernels.h"

namespace bg {

template <int D, int DT>
__device__ inline void store_row(const LayerView& L, int which, int slot, int kvh, const float (&v)[D / 64], int lane) {
  constexpr int EPL = D / 64;
  const int d0 = lane * EPL;
  if constexpr (DT == KV_Q8) {
    constexpr int LPB = kBlock / EPL;  // lanes per q8 block
    float m = 0.0f;
#pragma unroll
    for (int e = 0; e < EPL; e++) m = fmaxf(m, fabsf(v[e]));
    m = group_max<LPB>(m);
    if (L.q8_row) m = wave_max(m);  // per-row scale: the row's 64 lanes
    const float s = q8_scale_of(m);
    float* sc = which == 0 ? L.ks : L.vs;
    if ((lane % LPB) == 0) sc[scale_offset(kvh, slot, d0 / kBlock, L.cap, D)] = s;
    int8_t* base = (int8_t*)(which == 0 ? L.k : L.v);
#pragma unroll
    for (int e = 0; e < EPL; e++) {
      const int8_t c = (int8_t)q8_code(v[e], s);
      const size_t off = which == 0 ? k_offset(kvh, slot, d0 + e, L.cap, D) : v_offset(kvh, slot, d0 + e, L.cap, D);
      base[off] = c;
    }
  } else if constexpr (DT == KV_F16) {
    __half* base = (__half*)(which == 0 ? L.k : L.v);
#pragma unroll
    for (int e = 0; e < EPL; e++) {
      const size_t off = which == 0 ? k_offset(kvh, slot, d0 + e, L.cap, D) : v_offset(kvh, slot, d0 + e, L.cap, D);
      base[off] = __float2half_rn(v[e]);
    }
  } else {
    float* base = (float*)(which == 0 ? L.k : L.v);
#pragma unroll
    for (int e = 0; e < EPL; e++) {
      const size_t off = which == 0 ? k_offset(kvh, slot, d0 + e, L.cap, D) : v_offset(kvh, slot, d0 + e, L.cap, D);
      base[off] = v[e];
    }
  }
}

// Slot (within a 16-slot group) of entry i of the group's panel b: tile_slot(2a + b, i) - 16a,
// which does not depend on the half a of the tile. A compile-time index keeps the group's values
// in fixed registers (an index through a, known only at run time, makes the compiler select
// among all 16 rows for every entry).
__host__ __device__ constexpr int vgroup_slot(int b, int i) { return 8 * (i >> 2) + 4 * b + (i & 3); }

// Store panel b of a 16-slot group (its 8 slots, v[i] = slot vgroup_slot(b, i) of the group, D/64
// consecutive dims a lane) into the transposed V tile: every (dim, panel) is one contiguous
// 16-byte (f16) / 8-byte (q8) / 32-byte (f32) store; q8 scales are per (slot, 32 dims).
template <int D, int DT, int B>
__device__ inline void store_vpanel(const LayerView& L, int kvh, int slot_base, const float (&v)[8][D / 64], int lane) {
  constexpr int EPL = D / 64;
  const int d0 = lane * EPL;
  const int t_base = slot_base & ~31;   // first slot of the 32-slot tile
  const int a = (slot_base >> 4) & 1;   // which half of the tile: panels 2a, 2a+1
  const size_t off0 = v_offset(kvh, t_base + tile_slot(2 * a + B, 0), d0, L.cap, D);  // entry 0 of dim d0
  if constexpr (DT == KV_Q8) {
    constexpr int LPB = kBlock / EPL;   // lanes per q8 block
    float sc[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      float m = 0.0f;
#pragma unroll
      for (int e = 0; e < EPL; e++) m = fmaxf(m, fabsf(v[i][e]));
      m = group_max<LPB>(m);
      if (L.q8_row) m = wave_max(m);  // per-row scale: the row's 64 lanes
      sc[i] = q8_scale_of(m);
      if ((lane % LPB) == 0) L.vs[scale_offset(kvh, slot_base + vgroup_slot(B, i), d0 / kBlock, L.cap, D)] = sc[i];
    }
    int8_t* base = (int8_t*)L.v + off0;
#pragma unroll
    for (int e = 0; e < EPL; e++) {
      uint32_t w[2] = {0u, 0u};
#pragma unroll
      for (int i = 0; i < 8; i++) w[i >> 2] |= (uint32_t)(uint8_t)(int8_t)q8_code(v[i][e], sc[i]) << (8 * (i & 3));
      st_stream8(base + 8 * e, w[0], w[1]);
    }
  } else if constexpr (DT == KV_F16) {
    __half* base = (__half*)L.v + off0;
#pragma unroll
    for (int e = 0; e < EPL; e++) {
      union { __half h[8]; uint4 u; } o;
#pragma unroll
      for (int i = 0; i < 8; i++) o.h[i] = __float2half_rn(v[i][e]);
      st_stream16(base + 8 * e, o.u.x, o.u.y, o.u.z, o.u.w);
    }
  } else {
    float* base = (float*)L.v + off0;
#pragma unroll
    for (int e = 0; e < EPL; e++) {
      st_stream16f(base + 8 * e, v[0][e], v[1][e], v[2][e], v[3][e]);
      st_stream16f(base + 8 * e + 4, v[4][e], v[5][e], v[6][e], v[7][e]);
    }
  }
}

// Nontemporal loads of f32 rows that are read once
typedef float floatx4_t __attribute__((ext_vector_type(4)));
__device__ inline float4 ld_stream4(const float* p) {
  const floatx4_t v = __builtin_nontemporal_load((const floatx4_t*)p);
  return make_float4(v[0], v[1], v[2], v[3]);
}

// EPL consecutive floats (EPL = 2 or 4), nontemporal
template <int EPL>
__device__ inline void ld_stream(const float* p, float (&v)[EPL]) {
  if constexpr (EPL == 4) {
    const float4 f = ld_stream4(p);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  } else {
    typedef float floatx2_t __attribute__((ext_vector_type(2)));
    const floatx2_t f = __builtin_nontemporal_load((const floatx2_t*)p);
    v[0] = f[0]; v[1] = f[1];
  }
}

}  // namespace bg
