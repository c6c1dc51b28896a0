// Linear attention with a decay for each head, one row after the other (sequences of few new rows).
//
//   S <- e^g S + k (beta (v - e^g S^T k))^T   ("sum": S <- e^g S + k v^T),   o = scale S^T q
// and behind it, where asked for, the layer's output norm o / rms(o) * weight * silu(gate).
//
// One workgroup holds a head's whole state in registers while it walks the sequence's rows. Eight lanes share
// a column (a value dim): lane l has key dims 32 i + 4 l .. + 3, so a load of the state covers whole 128-byte
// lines, and both dot products of a row (with k and with q, against the state before the row's own write) are
// one pass over the registers and three exchanges inside eight lanes: o = scale (e^g S^T q + (q . k) delta).
#include "bg_common.h"
#include "bg_linear.h"

namespace bg {

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
constexpr int kThreads = 512;

template <int DK>
struct RowIn {
  f4 k[DK / 32], q[DK / 32];
};

template <int DK, int DV, bool DELTA>
__global__ __launch_bounds__(kThreads) void linear_recurrent_kernel(LinLayer L, LinBatchView b, LinAttnArgs a, int first) {
  constexpr int CPL = DV * 8 / kThreads;  // columns of a lane group
  constexpr int NI = DK / 32;
  constexpr int WAVES = kThreads / 64;
  static_assert(CPL >= 1 && NI >= 1, "state split");
  __shared__ float part[2][WAVES];
  const int s_at = first + blockIdx.y;
  const LinSeq s = b.seqs[s_at];
  if (s_at >= b.hdr->n_seqs || s.rows >= kLinChunkFrom) return;
  const int h = blockIdx.x, kh = h / (L.v_heads / L.k_heads);
  const int l = threadIdx.x & 7, col = (threadIdx.x >> 3) * CPL, wave = threadIdx.x >> 6;

  f4 S[CPL][NI];
#pragma unroll
  for (int c = 0; c < CPL; c++)
#pragma unroll
    for (int i = 0; i < NI; i++) S[c][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  if (s.src >= 0) {
    const float* p = L.state + (((size_t)s.src * L.v_heads + h) * DV + col) * DK + 4 * l;
#pragma unroll
    for (int c = 0; c < CPL; c++)
#pragma unroll
      for (int i = 0; i < NI; i++) S[c][i] = *(const f4*)(p + c * DK + 32 * i);
  }
  float weight[CPL];
#pragma unroll
  for (int c = 0; c < CPL; c++) weight[c] = a.norm ? a.norm[col + c] : 1.0f;

  const size_t kstride = (size_t)L.k_heads * DK, vstride = (size_t)L.v_heads * DV;
  const float* kp = a.k + (size_t)s.row0 * kstride + kh * DK + 4 * l;
  const float* qp = a.q + (size_t)s.row0 * kstride + kh * DK + 4 * l;
  const float* vp = a.v + (size_t)s.row0 * vstride + h * DV + col;
  RowIn<DK> in;
  float v[CPL], z[CPL], g, beta;
  auto load = [&](int t) {
#pragma unroll
    for (int i = 0; i < NI; i++) {
      in.k[i] = *(const f4*)(kp + t * kstride + 32 * i);
      in.q[i] = *(const f4*)(qp + t * kstride + 32 * i);
    }
#pragma unroll
    for (int c = 0; c < CPL; c++) v[c] = vp[t * vstride + c];
#pragma unroll
    for (int c = 0; c < CPL; c++) z[c] = a.gate ? a.gate[((size_t)(s.row0 + t) * L.v_heads + h) * DV + col + c] : 0.0f;
    g = a.g[(a.g_stride ? (size_t)(s.row0 + t) * a.g_stride : 0) + h];
    beta = DELTA ? a.beta[(size_t)(s.row0 + t) * L.v_heads + h] : 1.0f;
  };
  load(0);
  for (int t = 0; t < s.rows; t++) {
    const RowIn<DK> x = in;
    float vv[CPL], zz[CPL];
#pragma unroll
    for (int c = 0; c < CPL; c++) {
      vv[c] = v[c];
      zz[c] = z[c];
    }
    float fade, rest;
    fade_of(g, fade, rest);
    const float strength = beta;
    if (t + 1 < s.rows) load(t + 1);
    float ks[CPL], qs[CPL], qk = 0.0f;
#pragma unroll
    for (int c = 0; c < CPL; c++) ks[c] = qs[c] = 0.0f;
#pragma unroll
    for (int i = 0; i < NI; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        qk = fmaf(x.q[i][e], x.k[i][e], qk);
#pragma unroll
        for (int c = 0; c < CPL; c++) {
          if constexpr (DELTA) ks[c] = fmaf(S[c][i][e], x.k[i][e], ks[c]);
          qs[c] = fmaf(S[c][i][e], x.q[i][e], qs[c]);
        }
      }
    qk = group_sum<8>(qk);
    float o[CPL], ss = 0.0f;
#pragma unroll
    for (int c = 0; c < CPL; c++) {
      qs[c] = group_sum<8>(qs[c]);
      float delta = vv[c];
      if constexpr (DELTA) delta = strength * (vv[c] - fade * group_sum<8>(ks[c]));
      o[c] = a.scale * fmaf(qk, delta, fade * qs[c]);
      ss = fmaf(o[c], o[c], ss);
#pragma unroll
      for (int i = 0; i < NI; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) S[c][i][e] = fmaf(fade, S[c][i][e], fmaf(rest, S[c][i][e], x.k[i][e] * delta));
    }
    if (a.norm) {
      // the eight lanes of a column hold the same value: sum over the wave's eight groups, then its waves
      ss += dpp_mov<0x128>(ss);  // row_ror:8: the row's other group
      float2 r = pair16(ss);
      r = pair32(r.x + r.y);
      ss = r.x + r.y;
      if ((threadIdx.x & 63) == 0) part[t & 1][wave] = ss;
      __syncthreads();
      ss = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; w++) ss += part[t & 1][w];
      const float inv = 1.0f / sqrtf(ss / DV + a.eps);
#pragma unroll
      for (int c = 0; c < CPL; c++) {
        o[c] = o[c] * inv * weight[c];
        if (a.gate) o[c] *= zz[c] / (1.0f + expf(-zz[c]));
      }
    }
    if (l == 0) {
      float* op = a.out + ((size_t)(s.row0 + t) * L.v_heads + h) * DV + col;
#pragma unroll
      for (int c = 0; c < CPL; c++) op[c] = o[c];
    }
  }
  float* p = L.state + (((size_t)s.dst * L.v_heads + h) * DV + col) * DK + 4 * l;
#pragma unroll
  for (int c = 0; c < CPL; c++)
#pragma unroll
    for (int i = 0; i < NI; i++) *(f4*)(p + c * DK + 32 * i) = S[c][i];
}

template <int DK, int DV>
hipError_t launch_t(const LinLayer& L, const LinBatchView& b, const LinAttnArgs& a, hipStream_t st) {
  const int first = b.ws || !b.n_chunked ? b.n_chunked : 0;  // (under capture the counts are of the replay)
  const dim3 g(L.v_heads, b.n_seqs - first);
  if (a.beta) hipLaunchKernelGGL((linear_recurrent_kernel<DK, DV, true>), g, dim3(kThreads), 0, st, L, b, a, first);
  else hipLaunchKernelGGL((linear_recurrent_kernel<DK, DV, false>), g, dim3(kThreads), 0, st, L, b, a, first);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_linear_rows(const LinLayer& L, const LinBatchView& b, const LinAttnArgs& a, hipStream_t st) {
  if (L.DK == 64) return L.DV == 64 ? launch_t<64, 64>(L, b, a, st) : launch_t<64, 128>(L, b, a, st);
  return L.DV == 64 ? launch_t<128, 64>(L, b, a, st) : launch_t<128, 128>(L, b, a, st);
}

}  // namespace bg
