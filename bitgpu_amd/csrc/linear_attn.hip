// Linear attention with a decay for each head, one row after the other (sequences of few new rows).
//
//   S <- e^g S + k (beta (v - e^g S^T k))^T   ("sum": S <- e^g S + k v^T),   o = scale S^T q
// and behind it, where asked for, the layer's output norm o / rms(o) * weight * silu(gate).
//
// One workgroup holds a head's whole state in registers while it walks the sequence's rows. Eight lanes share
// a column (a value dim): lane l has key dims 32 i + 4 l .. + 3, so a load of the state covers whole 128-byte
// lines, and both dot products of a row (with k and with q, against the state before the row's own write) are
// one pass over the registers and three exchanges inside eight lanes: o = scale (e^g S^T q + (q . k) delta).
//
// Few sequences are bound by latency (one row, 48 heads 5.5 us), then by instructions: 0.87 us a row and CU, where a row
// that waits for the one before costs no memory, its decay's exponential in 64 bits is taken once for all rows and the
// output norm runs behind the last row, all rows at once (five rows of three sequences 11.9 us, with both in the rows'
// order 14.1). Many are bound by the states' bytes: 64 x 48 heads of 128 x 128 read and written, 403 MB, 83 us, 4.9 TB/s.
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
  constexpr int ROW = 2 * DK + DV, PIECES = ROW / 4;      // of a row in LDS: k | q | v
  constexpr int EACH = DV / 64;                           // values of a lane that normalizes a row
  constexpr int HELD = (kLinChunkFrom - 2) * PIECES / kThreads + 1;
  const int s_at = first + blockIdx.y;
  const LinSeq s = b.seqs[s_at];
  if (s_at >= b.hdr->n_seqs || s.rows >= kLinChunkFrom) return;
  extern __shared__ __align__(16) float lds[];
  float* made = lds;                                      // the rows' outputs, where they are to be normalized
  float* rows = lds + (a.norm ? s.rows * DV : 0);   // the rows behind the first
  const int h = blockIdx.x, kh = h / (L.v_heads / L.k_heads);
  const int l = threadIdx.x & 7, col = (threadIdx.x >> 3) * CPL, wave = threadIdx.x >> 6;

  // All rows but the first go through LDS, requested together ahead of the state.
  f4 held[HELD];
  const int pieces = (s.rows - 1) * PIECES;
#pragma unroll
  for (int i = 0; i < HELD; i++) {
    const int at = i * kThreads + threadIdx.x, t = at / PIECES, e = at % PIECES * 4;
    if (at >= pieces) continue;
    const size_t row = s.row0 + 1 + t;
    held[i] = e < 2 * DK ? *(const f4*)((e < DK ? a.k : a.q) + (row * L.k_heads + kh) * DK + (e & (DK - 1)))
                         : *(const f4*)(a.v + (row * L.v_heads + h) * DV + e - 2 * DK);
  }
  __builtin_amdgcn_sched_barrier(0);
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
  RowIn<DK> in;
  float v[CPL];
  {
    const float* kp = a.k + ((size_t)s.row0 * L.k_heads + kh) * DK + 4 * l;
    const float* qp = a.q + ((size_t)s.row0 * L.k_heads + kh) * DK + 4 * l;
    const size_t vat = ((size_t)s.row0 * L.v_heads + h) * DV + col;
#pragma unroll
    for (int i = 0; i < NI; i++) {
      in.k[i] = *(const f4*)(kp + 32 * i);
      in.q[i] = *(const f4*)(qp + 32 * i);
    }
#pragma unroll
    for (int c = 0; c < CPL; c++) v[c] = a.v[vat + c];
  }
  // a wave normalizes rows wave, wave + 8 ..: the first one's gate, and the weight
  const int mine = EACH * (threadIdx.x & 63);
  float weight[EACH], z[EACH];
  auto load_gate = [&](int t) {
#pragma unroll
    for (int c = 0; c < EACH; c++) z[c] = a.gate[((size_t)(s.row0 + t) * L.v_heads + h) * DV + mine + c];
  };
  if (a.norm && wave < s.rows) {
#pragma unroll
    for (int c = 0; c < EACH; c++) weight[c] = a.norm[mine + c];
    if (a.gate) load_gate(wave);
  }
  // the rows' decays and write strengths: lane t has row t's (an exponential in 64 bits a wave, not one a row)
  static_assert(kLinChunkFrom <= 64, "a lane a row");
  float fades, rests, betas = 1.0f;
  {
    const size_t t = s.row0 + min((int)(threadIdx.x & 63), s.rows - 1);
    if constexpr (DELTA) betas = a.beta[t * L.v_heads + h];
    fade_of(a.g[(a.g_stride ? t * a.g_stride : 0) + h], fades, rests);
  }
  auto of_row = [&](float x, int t) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), t)); };
  __builtin_amdgcn_sched_barrier(0);
  if (pieces) {
#pragma unroll
    for (int i = 0; i < HELD; i++)
      if (i * kThreads + (int)threadIdx.x < pieces) *(f4*)(rows + 4 * (i * kThreads + threadIdx.x)) = held[i];
    __syncthreads();
  }
  auto load = [&](int t) {
    const float* r = rows + (t - 1) * ROW;
#pragma unroll
    for (int i = 0; i < NI; i++) {
      in.k[i] = *(const f4*)(r + 4 * l + 32 * i);
      in.q[i] = *(const f4*)(r + DK + 4 * l + 32 * i);
    }
#pragma unroll
    for (int c = 0; c < CPL; c++) v[c] = r[2 * DK + col + c];
  };
  for (int t = 0; t < s.rows; t++) {
    const RowIn<DK> x = in;
    float vv[CPL];
#pragma unroll
    for (int c = 0; c < CPL; c++) vv[c] = v[c];
    const float fade = of_row(fades, t), rest = of_row(rests, t), strength = of_row(betas, t);
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
    float o[CPL];
#pragma unroll
    for (int c = 0; c < CPL; c++) {
      qs[c] = group_sum<8>(qs[c]);
      float delta = vv[c];
      if constexpr (DELTA) delta = strength * (vv[c] - fade * group_sum<8>(ks[c]));
      o[c] = a.scale * fmaf(qk, delta, fade * qs[c]);
#pragma unroll
      for (int i = 0; i < NI; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) S[c][i][e] = fmaf(fade, S[c][i][e], fmaf(rest, S[c][i][e], x.k[i][e] * delta));
    }
    if (l == 0) {
      float* op = a.norm ? made + t * DV + col : a.out + ((size_t)(s.row0 + t) * L.v_heads + h) * DV + col;
#pragma unroll
      for (int c = 0; c < CPL; c++) op[c] = o[c];
    }
  }
  float* p = L.state + (((size_t)s.dst * L.v_heads + h) * DV + col) * DK + 4 * l;
#pragma unroll
  for (int c = 0; c < CPL; c++)
#pragma unroll
    for (int i = 0; i < NI; i++) *(f4*)(p + c * DK + 32 * i) = S[c][i];
  if (!a.norm) return;
  __syncthreads();
  for (int t = wave; t < s.rows; t += WAVES) {
    if (t != wave && a.gate) load_gate(t);
    float o[EACH], ss = 0.0f;
#pragma unroll
    for (int c = 0; c < EACH; c++) {
      o[c] = made[t * DV + mine + c];
      ss = fmaf(o[c], o[c], ss);
    }
    const float inv = 1.0f / sqrtf(wave_sum(ss) / DV + a.eps);
    float* op = a.out + ((size_t)(s.row0 + t) * L.v_heads + h) * DV + mine;
#pragma unroll
    for (int c = 0; c < EACH; c++) {
      const float y = o[c] * inv * weight[c];
      op[c] = a.gate ? y * (z[c] / (1.0f + expf(-z[c]))) : y;
    }
  }
}

template <int DK, int DV>
hipError_t launch_t(const LinLayer& L, const LinBatchView& b, const LinAttnArgs& a, hipStream_t st) {
  const int first = b.ws || !b.n_chunked ? b.n_chunked : 0;  // (under capture the counts are of the replay)
  const dim3 g(L.v_heads, b.n_seqs - first);
  const size_t lds = ((size_t)(b.most - 1) * (2 * DK + DV) + (a.norm ? b.most * DV : 0)) * sizeof(float);
  if (a.beta) hipLaunchKernelGGL((linear_recurrent_kernel<DK, DV, true>), g, dim3(kThreads), lds, st, L, b, a, first);
  else hipLaunchKernelGGL((linear_recurrent_kernel<DK, DV, false>), g, dim3(kThreads), lds, st, L, b, a, first);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_linear_rows(const LinLayer& L, const LinBatchView& b, const LinAttnArgs& a, hipStream_t st) {
  if (L.DK == 64) return L.DV == 64 ? launch_t<64, 64>(L, b, a, st) : launch_t<64, 128>(L, b, a, st);
  return L.DV == 64 ? launch_t<128, 64>(L, b, a, st) : launch_t<128, 128>(L, b, a, st);
}

}  // namespace bg
