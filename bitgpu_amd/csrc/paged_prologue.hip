// The attention prologue of a batch on a paged cache: per-head RMSNorm + rotary position for the new
// tokens' Q (to an f32 buffer) and K (to its page, in the storage format), and the V append, one launch
// for any mix of sequences.
//
// Rows, norms, rotation and stores are bg_qkrow.h's and bg_store.h's, so a row's bits equal those the
// one-sequence prologue (norm_rope.hip) gives it. What is the batch's own:
//   * a token's slot and its rotary positions come from arrays (dst, pos), read before the row's data so
//     that the table entries follow one load behind;
//   * with several axes each rotary pair j takes its angle from the table row of axis pair_axis[j]
//     (2 bits a pair, in the kernel's arguments): sections and interleaved forms are one map. One axis
//     reads its table entries 16 bytes a lane; several read them one by one (a lane's four pairs may
//     have three axes), from table rows that the L2 holds: an image's tokens share most of them.
// A wave an item, 64 threads a workgroup: NI loads of Q / K rows (few rows are bound by latency and
// spread over the most waves), one V row, or 16 tokens' V rows that fill 16 aligned slots.
#include <algorithm>

#include "bg_paged.h"
#include "bg_qkrow.h"
#include "bg_store.h"

namespace bg {

// the page holding flat slot `at` as a layer view of `page` slots, and the slot within it
__device__ inline LayerView page_view(const LayerView& pool, int at, int shift, int D, int eb, int* slot) {
  LayerView L = pool;
  const size_t page = (size_t)(at >> shift);
  const size_t rows = page * (size_t)pool.kv_heads * pool.cap;
  L.k = (char*)pool.k + rows * D * eb;
  L.v = (char*)pool.v + rows * D * eb;
  if (pool.ks) {
    L.ks = pool.ks + rows * (D / kBlock);
    L.vs = pool.vs + rows * (D / kBlock);
  }
  *slot = at & ((1 << shift) - 1);
  return L;
}

template <int D, int DT, int NI>
__global__ __launch_bounds__(64) void paged_prologue_kernel(LayerView pool, PagedBatchView b, PagedAppendArgs a) {
  constexpr int EPL = D / 64;
  constexpr int LPR = D / 4, RPI = 64 / LPR, RB = RPI * NI;
  constexpr int EB = DT == KV_F32 ? 4 : DT == KV_F16 ? 2 : 1;
  __shared__ __align__(16) float rowbuf[RB][D];
  const int lane = threadIdx.x;
  const int KV = pool.kv_heads, H = b.H;
  const int T = b.captured ? b.hdr->n_tokens : b.n_tokens;
  const int nvs = a.v ? (b.captured ? b.hdr->n_v_single : b.n_v_single) : 0;
  const int ng = a.v ? (b.captured ? b.hdr->n_v_group : b.n_v_group) : 0;
  const int nq = a.q ? T * H : 0, nk = a.k ? T * KV : 0, nqk = nq + nk;
  const int nqk_items = (nqk + RB - 1) / RB;
  const int n_items = nqk_items + (nvs + ng) * KV;
  for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
    if (item < nqk_items) {
      const int h = lane / LPR, c = lane % LPR;
      const int rot = a.rot_dim, half = rot >> 1;
      float x[NI][4], cs[NI][4], sn[NI][4];
      int tok[NI];
#pragma unroll
      for (int i = 0; i < NI; i++) {
        const int r = min(item * RB + RPI * i + h, nqk - 1);  // past the end: the last row again, not stored
        const float* src;
        if (r < nq) {
          tok[i] = r / H;
          src = a.q + ((size_t)tok[i] * H + r % H) * a.q_stride;
        } else {
          tok[i] = (r - nq) / KV;
          src = a.k + (size_t)(r - nq) * D;
        }
        const float4 v4 = ld_stream4(src + 4 * c);
        x[i][0] = v4.x; x[i][1] = v4.y; x[i][2] = v4.z; x[i][3] = v4.w;
      }
#pragma unroll
      for (int i = 0; i < NI; i++) {
        if (a.axes == 1) {
          row_tables(a.cos_tab, a.sin_tab, b.pos[tok[i]], rot, c, cs[i], sn[i]);
        } else {
          int at[4];
#pragma unroll
          for (int x4 = 0; x4 < 4; x4++) at[x4] = x4 < a.axes ? b.pos[(size_t)x4 * b.pos_stride + tok[i]] : 0;
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int d = 4 * c + e;
            const bool on = d < rot;
            const int j = on ? (d < half ? d : d - half) : 0;
            const int ax = (a.pair_axis[j >> 4] >> (2 * (j & 15))) & 3;
            const int p = ax == 0 ? at[0] : ax == 1 ? at[1] : ax == 2 ? at[2] : at[3];
            cs[i][e] = on ? a.cos_tab[(size_t)p * half + j] : 0.0f;
            sn[i][e] = on ? a.sin_tab[(size_t)p * half + j] : 0.0f;
          }
        }
      }
      float gq[4] = {0, 0, 0, 0}, gk[4] = {0, 0, 0, 0};
      if (a.q_gamma) load4(a.q_gamma + 4 * c, gq);
      if (a.k_gamma) load4(a.k_gamma + 4 * c, gk);
#pragma unroll
      for (int i = 0; i < NI; i++) {
        const bool isq = item * RB + RPI * i + h < nq;
        float g4[4];
#pragma unroll
        for (int e = 0; e < 4; e++) g4[e] = isq ? gq[e] : gk[e];
        row_scale(x[i], row_inv_rms<D, LPR>(x[i], a.eps), g4);
      }
      float pr[NI][4];
      bool lanes = true;
#pragma unroll
      for (int i = 0; i < NI; i++) lanes = rope_partner_lanes(x[i], rot, pr[i]);
      if (!lanes) {
#pragma unroll
        for (int i = 0; i < NI; i++)
          *(float4*)(&rowbuf[RPI * i + h][4 * c]) = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < NI; i++) {
        const int r = item * RB + RPI * i + h;
        if (lanes) row_rope_lanes(x[i], pr[i], c, rot, cs[i], sn[i]);
        else row_rope(x[i], &rowbuf[RPI * i + h][0], c, rot, cs[i], sn[i]);
        if (r < nq) {
          st_stream16f(a.q_out + (size_t)r * D + 4 * c, x[i][0], x[i][1], x[i][2], x[i][3]);
        } else if (r < nqk) {
          int slot;
          const LayerView L = page_view(pool, b.dst[tok[i]], b.page_shift, D, EB, &slot);
          store_k4<D, DT>(L, slot, (r - nq) % KV, x[i], c);
        }
      }
      if (!lanes) __syncthreads();  // the rows are read before the next item writes its own
      continue;
    }
    const int vi = item - nqk_items;
    if (vi < nvs * KV) {
      const int head = vi % KV, t = b.v_single[vi / KV];
      float v[EPL];
      ld_stream<EPL>(a.v + ((size_t)t * KV + head) * D + lane * EPL, v);
      int slot;
      const LayerView L = page_view(pool, b.dst[t], b.page_shift, D, EB, &slot);
      store_row<D, DT>(L, 1, slot, head, v, lane);
      continue;
    }
    const int gi = vi - nvs * KV;
    const int head = gi % KV, t = b.v_group[gi / KV];
    int slot;
    const LayerView L = page_view(pool, b.dst[t], b.page_shift, D, EB, &slot);
    float v[8][EPL];
#pragma unroll
    for (int i = 0; i < 8; i++) ld_stream<EPL>(a.v + ((size_t)(t + vgroup_slot(0, i)) * KV + head) * D + lane * EPL, v[i]);
    store_vpanel<D, DT, 0>(L, head, slot, v, lane);
#pragma unroll
    for (int i = 0; i < 8; i++) ld_stream<EPL>(a.v + ((size_t)(t + vgroup_slot(1, i)) * KV + head) * D + lane * EPL, v[i]);
    store_vpanel<D, DT, 1>(L, head, slot, v, lane);
  }
}

template <int D, int DT, int NI>
static void launch_rows(const LayerView& pool, const PagedBatchView& b, const PagedAppendArgs& a, hipStream_t st) {
  constexpr int RB = 64 / (D / 4) * NI;
  const long rows = (long)b.n_tokens * ((a.q ? b.H : 0) + (a.k ? pool.kv_heads : 0));
  long items = (rows + RB - 1) / RB + (a.v ? (long)(b.n_v_single + b.n_v_group) * pool.kv_heads : 0);
  // under capture the items are counted on the device: a grid that fills the GPU walks them
  if (b.captured) items = (long)a.num_cus * 16;
  if (items == 0) return;
  hipLaunchKernelGGL((paged_prologue_kernel<D, DT, NI>), dim3((unsigned)std::min(items, 0x7fffffffL)), dim3(64), 0, st, pool, b, a);
}

template <int D, int DT>
static void launch_dt(const LayerView& pool, const PagedBatchView& b, const PagedAppendArgs& a, hipStream_t st) {
  const long rows = (long)b.n_tokens * ((a.q ? b.H : 0) + (a.k ? pool.kv_heads : 0));
  if (b.captured || rows <= 8192) launch_rows<D, DT, 1>(pool, b, a, st);
  else launch_rows<D, DT, 2>(pool, b, a, st);
}

template <int D>
static hipError_t launch_d(const LayerView& pool, const PagedBatchView& b, const PagedAppendArgs& a, hipStream_t st) {
  switch (pool.dtype) {
    case KV_F32: launch_dt<D, KV_F32>(pool, b, a, st); break;
    case KV_F16: launch_dt<D, KV_F16>(pool, b, a, st); break;
    default: launch_dt<D, KV_Q8>(pool, b, a, st);
  }
  return hipGetLastError();
}

hipError_t launch_paged_prologue(const LayerView& pool, const PagedBatchView& b, const PagedAppendArgs& a, hipStream_t st) {
  return pool.D == 128 ? launch_d<128>(pool, b, a, st) : launch_d<256>(pool, b, a, st);
}

// One launch brings a set's arrays to the device: workgroups read the pinned staging memory over the bus
// 16 bytes a lane. A handful of copies of some KB each would cost as many launches.
__global__ __launch_bounds__(256) void paged_upload_kernel(PagedUpload u) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const u32x4* src = (const u32x4*)u.src[blockIdx.y];
  u32x4* dst = (u32x4*)u.dst[blockIdx.y];
  const unsigned n = u.n16[blockIdx.y];
  for (unsigned i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) dst[i] = src[i];
}

hipError_t launch_paged_upload(const PagedUpload& u, hipStream_t st) {
  unsigned most = 1;
  for (unsigned n : u.n16) most = std::max(most, n);
  hipLaunchKernelGGL(paged_upload_kernel, dim3(std::min((most + 255) / 256, 64u), 9), dim3(256), 0, st, u);
  return hipGetLastError();
}

}  // namespace bg
