// The attention prologue of a batch on a paged cache: per-head RMSNorm + rotary position for the new
// tokens' Q (to an f32 buffer) and K (to its page, in the storage format), and the V append, one launch
// for any mix of sequences. Bound by memory: every row is read once and written once (5,905 tokens of 24 +
// 4 heads of 256 into q8 pages, three axes: 354 MB in 65 us, 5.5 TB/s; 3,241 of 16 + 8 heads of 128 into
// f32 ones 108 MB in 21.6 us, 5.0 TB/s; a device copy reaches 5.1), a decode step by its chain of loads
// (one token 3.0 us, 64 tokens 3.4, with three axes 4.4).
//
// Norms, rotation and stores are bg_qkrow.h's and bg_store.h's, so a row's bits equal those the
// one-sequence prologue (norm_rope.hip) gives it. What is the batch's own:
//   * items are rows of one token, so its position, page and table entries are loaded once for all;
//   * a token's slot and rotary positions come from arrays (dst, pos) that the batch uploads;
//   * with several axes each rotary pair j takes its angle from the table row of axis pair_axis[j]
//     (2 bits a pair, in the kernel's arguments): sections and interleaved forms are one map. One axis
//     reads its table entries 16 bytes a lane; several read them one by one (a lane's four pairs may
//     have three axes), from table rows that the L2 holds: an image's tokens share most of them.
// A wave an item, 64 threads a workgroup: RB rows of a token (NI loads), one V row, or 16 tokens' V rows
// that fill 16 aligned slots.
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

// 16 tokens' V rows of one head (src: the first one's, `step` values from token to token) into the 16
// aligned slots from `slot`: every store instruction writes one contiguous run of its panel. f16: a lane a
// dim, its 8 slots 16 bytes; f32: two lanes a dim, 4 slots each. (Two neighbouring dims a lane, as a q8
// row's scale wants them, leave every second 16 bytes to the next instruction: f32 11.8 us for 26 MB.)
template <int D, int DT>
__device__ __forceinline__ void store_v16(const LayerView& L, int head, int slot, const float* src, size_t step, int lane) {
  const int tile = slot & ~31, a = (slot >> 4) & 1;
  constexpr int PL = DT == KV_F32 ? 2 : 1, N = D * PL / 64, S = 8 / PL;  // lanes a dim, dims a lane, slots a lane
  const int c = lane / PL, hf = lane % PL;
  float v[2][N][S];
#pragma unroll
  for (int p = 0; p < 2; p++)
#pragma unroll
    for (int i = 0; i < S; i++)
#pragma unroll
      for (int n = 0; n < N; n++)
        v[p][n][i] = __builtin_nontemporal_load(src + (size_t)(vgroup_slot(p, i) + 8 * hf) * step + c + 64 / PL * n);
#pragma unroll
  for (int p = 0; p < 2; p++) {
    const size_t off = v_offset(head, tile + tile_slot(2 * a + p, 0), c, L.cap, D) + S * hf;
#pragma unroll
    for (int n = 0; n < N; n++) {
      if constexpr (DT == KV_F32) {
        st_stream16f((float*)L.v + off + (size_t)8 * 32 * n, v[p][n][0], v[p][n][1], v[p][n][2], v[p][n][3]);
      } else {
        union { __half h[8]; uint4 u; } o;
#pragma unroll
        for (int i = 0; i < 8; i++) o.h[i] = __float2half_rn(v[p][n][i % S]);
        st_stream16((__half*)L.v + off + (size_t)8 * 64 * n, o.u.x, o.u.y, o.u.z, o.u.w);
      }
    }
  }
}

// What a launch works through: a token's rows (its Q heads, then its K heads) in items of RB, then V.
struct PrologueItems {
  int hq, hqk, per_tok, nqk, nvs, n;
};
template <int RB>
__device__ inline PrologueItems count_items(const PagedAppendArgs& a, int H, int KV, int T, int nvs, int ng) {
  PrologueItems it;
  it.hq = a.q ? H : 0;
  it.hqk = it.hq + (a.k ? KV : 0);
  it.per_tok = (it.hqk + RB - 1) / RB;
  it.nqk = T * it.per_tok;
  it.nvs = a.v ? nvs : 0;
  it.n = it.nqk + (it.nvs + (a.v ? ng : 0)) * KV;
  return it;
}

template <int D, int DT, int NI, bool AXES>
__device__ __forceinline__ void prologue_item(const LayerView& pool, const PagedBatchView& b, const PagedAppendArgs& a,
                                              const PrologueItems& it, int item, float (*rowbuf)[D]) {
  constexpr int EPL = D / 64;
  constexpr int LPR = D / 4, RPI = 64 / LPR, RB = RPI * NI;
  constexpr int EB = DT == KV_F32 ? 4 : DT == KV_F16 ? 2 : 1;
  const int lane = threadIdx.x;
  const int KV = pool.kv_heads, H = b.H;
  // q8: the V items first, which divide and reduce the most (images' 5,905 rows 69.2 -> 64.7 us; f32 and
  // f16 the rows first, 21.6 against 22.1)
  if constexpr (DT == KV_Q8) item = item < it.n - it.nqk ? item + it.nqk : item - (it.n - it.nqk);
  if (item < it.nqk) {
    // ---------------- RB rows of one token: its position's table entries serve them all
    const int t = item / it.per_tok, h0 = (item - t * it.per_tok) * RB;
    const int h = lane / LPR, c = lane % LPR;
    const int rot = a.rot_dim, half = rot >> 1;
    float x[NI][4], cs[4], sn[4];
#pragma unroll
    for (int i = 0; i < NI; i++) {
      const int r = min(h0 + RPI * i + h, it.hqk - 1);  // past the last head: that one again, not stored
      const float* src = r < it.hq ? a.q + ((size_t)t * H + r) * a.q_stride : a.k + ((size_t)t * KV + r - it.hq) * D;
      const float4 v4 = ld_stream4(src + 4 * c);
      x[i][0] = v4.x; x[i][1] = v4.y; x[i][2] = v4.z; x[i][3] = v4.w;
    }
    if constexpr (!AXES) {
      row_tables(a.cos_tab, a.sin_tab, b.pos[t], rot, c, cs, sn);
    } else {
      int at[4];
#pragma unroll
      for (int x4 = 0; x4 < 4; x4++) at[x4] = x4 < a.axes ? b.pos[(size_t)x4 * b.pos_stride + t] : 0;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int d = 4 * c + e;
        const bool on = d < rot;
        const int j = on ? (d < half ? d : d - half) : 0;
        const int ax = (a.pair_axis[j >> 4] >> (2 * (j & 15))) & 3;
        const int p = ax == 0 ? at[0] : ax == 1 ? at[1] : ax == 2 ? at[2] : at[3];
        cs[e] = on ? a.cos_tab[(size_t)p * half + j] : 0.0f;
        sn[e] = on ? a.sin_tab[(size_t)p * half + j] : 0.0f;
      }
    }
    float gq[4] = {0, 0, 0, 0}, gk[4] = {0, 0, 0, 0};
    if (a.q_gamma) load4(a.q_gamma + 4 * c, gq);
    if (a.k_gamma) load4(a.k_gamma + 4 * c, gk);
#pragma unroll
    for (int i = 0; i < NI; i++) {
      const bool isq = h0 + RPI * i + h < it.hq;
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
      const int r = h0 + RPI * i + h;
      if (lanes) row_rope_lanes(x[i], pr[i], c, rot, cs, sn);
      else row_rope(x[i], &rowbuf[RPI * i + h][0], c, rot, cs, sn);
      if (r < it.hq) {
        st_stream16f(a.q_out + ((size_t)t * H + r) * D + 4 * c, x[i][0], x[i][1], x[i][2], x[i][3]);
      } else if (r < it.hqk) {
        int slot;
        const LayerView L = page_view(pool, b.dst[t], b.page_shift, D, EB, &slot);
        store_k4<D, DT>(L, slot, r - it.hq, x[i], c);
      }
    }
    return;
  }
  const int vi = item - it.nqk;
  int slot;
  if (vi < it.nvs * KV) {
    // ---------------- a single V row
    const int head = vi % KV, t = b.v_single[vi / KV];
    float v[EPL];
    ld_stream<EPL>(a.v + ((size_t)t * KV + head) * D + lane * EPL, v);
    const LayerView L = page_view(pool, b.dst[t], b.page_shift, D, EB, &slot);
    store_row<D, DT>(L, 1, slot, head, v, lane);
    return;
  }
  // ---------------- 16 tokens' V rows of one head, 16 aligned slots, one panel at a time
  const int gi = vi - it.nvs * KV;
  const int head = gi % KV, t = b.v_group[gi / KV];
  const LayerView L = page_view(pool, b.dst[t], b.page_shift, D, EB, &slot);
  const float* src = a.v + ((size_t)t * KV + head) * D;
  if constexpr (DT != KV_Q8) {
    store_v16<D, DT>(L, head, slot, src, (size_t)KV * D, lane);
  } else {
    float v[8][EPL];
#pragma unroll
    for (int i = 0; i < 8; i++) ld_stream<EPL>(src + (size_t)vgroup_slot(0, i) * KV * D + lane * EPL, v[i]);
    store_vpanel<D, DT, 0>(L, head, slot, v, lane);
#pragma unroll
    for (int i = 0; i < 8; i++) ld_stream<EPL>(src + (size_t)vgroup_slot(1, i) * KV * D + lane * EPL, v[i]);
    store_vpanel<D, DT, 1>(L, head, slot, v, lane);
  }
}

// An item a workgroup.
template <int D, int DT, int NI, bool AXES>
__global__ __launch_bounds__(64) void paged_prologue_kernel(LayerView pool, PagedBatchView b, PagedAppendArgs a) {
  constexpr int RB = 64 / (D / 4) * NI;
  __shared__ __align__(16) float rowbuf[RB][D];
  const PrologueItems it = count_items<RB>(a, b.H, pool.kv_heads, b.n_tokens, b.n_v_single, b.n_v_group);
  if ((int)blockIdx.x < it.n) prologue_item<D, DT, NI, AXES>(pool, b, a, it, blockIdx.x, rowbuf);
}

// Under capture: the items of whatever batch is set at replay, counted on the device, walked by a grid
// that fills the GPU (the walk holds about 100 registers where one item holds 30 to 60: one token and 64 take as
// long as outside a capture, 3,241 f32 rows 27-28 us instead of 21.6).
template <int D, int DT, bool AXES>
__global__ __launch_bounds__(64) void paged_prologue_walk_kernel(LayerView pool, PagedBatchView b, PagedAppendArgs a) {
  constexpr int RB = 64 / (D / 4);
  __shared__ __align__(16) float rowbuf[RB][D];
  const PrologueItems it = count_items<RB>(a, b.H, pool.kv_heads, b.hdr->n_tokens, b.hdr->n_v_single, b.hdr->n_v_group);
  for (int item = blockIdx.x; item < it.n; item += gridDim.x) {
    prologue_item<D, DT, 1, AXES>(pool, b, a, it, item, rowbuf);
    __syncthreads();  // the rows in LDS are read before the next item writes its own
  }
}

template <int D, int DT, int NI, bool AXES>
static void launch_rows(const LayerView& pool, const PagedBatchView& b, const PagedAppendArgs& a, hipStream_t st) {
  constexpr int RB = 64 / (D / 4) * NI;
  const long heads = (a.q ? b.H : 0) + (a.k ? pool.kv_heads : 0);
  const long items = b.n_tokens * ((heads + RB - 1) / RB) + (a.v ? (long)(b.n_v_single + b.n_v_group) * pool.kv_heads : 0);
  if (items) hipLaunchKernelGGL((paged_prologue_kernel<D, DT, NI, AXES>), dim3((unsigned)items), dim3(64), 0, st, pool, b, a);
}

template <int D, int DT, bool AXES>
static void launch_axes(const LayerView& pool, const PagedBatchView& b, const PagedAppendArgs& a, hipStream_t st) {
  const long rows = (long)b.n_tokens * ((a.q ? b.H : 0) + (a.k ? pool.kv_heads : 0));
  if (b.captured) hipLaunchKernelGGL((paged_prologue_walk_kernel<D, DT, AXES>), dim3(a.num_cus * 16), dim3(64), 0, st, pool, b, a);
  // Few rows are bound by latency and spread over the most waves; many share a position's table entries
  // and keep four loads in flight a wave (us, one / two / four loads: 5,905 tokens q8 at head_dim 256 109 /
  // 79 / 70, 3,241 f16 23.5 / 19.5 / 18.5, one and 64 tokens equal).
  else if (rows <= 8192) launch_rows<D, DT, 1, AXES>(pool, b, a, st);
  else launch_rows<D, DT, 4, AXES>(pool, b, a, st);
}

template <int D, int DT>
static void launch_dt(const LayerView& pool, const PagedBatchView& b, const PagedAppendArgs& a, hipStream_t st) {
  if (a.axes > 1) launch_axes<D, DT, true>(pool, b, a, st);
  else launch_axes<D, DT, false>(pool, b, a, st);
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
